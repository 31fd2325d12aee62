// int8 KV caches: rows are quantised as they are written and read back into
// f16 or f32 caches.
//
// Layout of one I8 cache of K (or V): cap * kv_heads * 128 bytes c + 128,
// [cap][kv_heads][128], then f32 scales [kv_heads][cap]; position p lives in
// slot p % cap as in the other caches.  One scale serves one head of one row:
//   s = max|x| / 127 rounded to f32 (0 when below 2^-126, NaN when an element
//   is not finite), c = the integer nearest to x / s (ties to even), value c*s.
// A head is the unit that attention multiplies, so a key's scale is one factor
// of its score and a value's scale one factor of its weight.  The scales of
// a head lie side by side over the rows: a decode warp reads 16 of them as
// 64 contiguous bytes (row-major scales would cost it a 32-byte sector each).
//
// Both kernels move bytes and compute a few operations for each; HBM bounds
// them, at (2 or 4) + 1.03 bytes for each element in either direction.
#include "batch_internal.cuh"

namespace sf37kv {

extern unsigned long long g_launches;

// ------------------------------------------------------------ append
struct AppendI8Job {
    uint8_t *k_cache, *v_cache;
    const void *k, *v;   // [n_tok][heads][128], f32 or bf16
    uint32_t pos0, cap;  // the rows that stay: at most cap
};
struct AppendI8Params {
    AppendI8Job job[kMaxJobs];
    uint32_t row_begin[kMaxJobs + 1];
    uint32_t n_jobs, heads, rows_each;  // rows_each: of every job, or 0 where they differ
};

// Job of row `row` (or block, by its begin array).
template <typename Begin>
__device__ __forceinline__ uint32_t job_of(const Begin &begin, uint32_t n, uint32_t each, uint32_t row) {
    if (each) return row / each;
    uint32_t lo = 0;
    for (uint32_t hi = n; hi - lo > 1;) {
        const uint32_t mid = (lo + hi) >> 1;
        if (begin[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Eight lanes per head of one row, K and V together: 16 elements a lane in
// 128-byte runs, all loads first; a head's maximum is three shuffles, and a code
// four instructions, with one test of a lane's 16 remainders for a tie.  8192 rows of
// 8 heads, bf16: 14 us, 3.6 TB/s (a warp a head with integer conversions took 30,
// a test for each element 16; K and V in blocks of their own 17).  Latency and
// instructions bound it: 50 MB are 8 us of HBM.
constexpr uint32_t kAppendThreads = 128;
template <bool BF16>
__global__ void __launch_bounds__(kAppendThreads) append_i8_kernel(const __grid_constant__ AppendI8Params P) {
    after_previous();
    const uint32_t lane8 = threadIdx.x & 7u, unit = blockIdx.x * (kAppendThreads / 8u) + (threadIdx.x >> 3);
    const uint32_t row = unit / P.heads, head = unit - row * P.heads;
    const bool live = row < P.row_begin[P.n_jobs];
    const uint32_t j = live ? job_of(P.row_begin, P.n_jobs, P.rows_each, row) : 0u;
    const AppendI8Job &J = P.job[j];
    const uint32_t t = live ? row - P.row_begin[j] : 0u;
    const uint64_t src = ((uint64_t)t * P.heads + head) * 128u;
    const uint64_t kv_dim = (uint64_t)P.heads * 128u;
    constexpr uint32_t kRun = BF16 ? 8 : 4, kRuns = 16 / kRun;  // elements of a load, loads
    uint4 raw[2][kRuns];
    if (live) {
#pragma unroll
        for (uint32_t i = 0; i < kRuns; i++) {
            const uint64_t at = src + (i * 8u + lane8) * kRun;
            const uint32_t size = BF16 ? 2u : 4u;
            raw[0][i] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(J.k) + at * size);
            raw[1][i] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(J.v) + at * size);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kRuns; i++) raw[0][i] = raw[1][i] = make_uint4(0u, 0u, 0u, 0u);
    }
    const uint32_t slot = (J.pos0 + t) % J.cap;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        float x[16];
#pragma unroll
        for (uint32_t i = 0; i < kRuns; i++) {
            const uint32_t w[4] = {raw[which][i].x, raw[which][i].y, raw[which][i].z, raw[which][i].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (BF16) {
                    x[(8 * i + 2 * e) & 15] = __uint_as_float(w[e] << 16);
                    x[(8 * i + 2 * e + 1) & 15] = __uint_as_float(w[e] & 0xffff0000u);
                } else {
                    x[(4 * i + e) & 15] = __uint_as_float(w[e]);
                }
            }
        }
        float a = fabsf(x[0]);
#pragma unroll
        for (int e = 1; e < 16; e++) a = max_abs_nan(a, x[e]);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) a = max_abs_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        const float s = i8_scale(a), inv = s > 0.f ? __frcp_rn(s) : 0.f;
        uint32_t codes[4];
        float worst = 0.f;
#pragma unroll
        for (int q = 0; q < 4; q++) codes[q] = i8_pack_near(x + 4 * q, s, inv, worst);
        if (!(worst + worst < s)) {  // a tie or one off, or a scale of 0 or NaN
#pragma unroll
            for (int q = 0; q < 4; q++)
                codes[q] = s > 0.f ? i8_pack(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3], s, inv) : kI8Zero;
        }
        if (!live) continue;
        uint8_t *cache = which ? J.v_cache : J.k_cache, *dst = cache + slot * kv_dim + head * 128u;
#pragma unroll
        for (uint32_t i = 0; i < kRuns; i++) {
            if (BF16) *reinterpret_cast<uint2 *>(dst + (i * 8u + lane8) * 8u) = make_uint2(codes[(2 * i) & 3], codes[(2 * i + 1) & 3]);
            else *reinterpret_cast<uint32_t *>(dst + (i * 8u + lane8) * 4u) = codes[i & 3];
        }
        if (lane8 == 0) reinterpret_cast<float *>(cache + J.cap * kv_dim)[(uint64_t)head * J.cap + slot] = s;
    }
}

// ------------------------------------------------------------ read back
struct ReadI8Job {
    const uint8_t *k_src, *v_src;
    void *k_dst, *v_dst;
    uint32_t first, rows, src_cap, dst_cap;
};
struct ReadI8Params {
    ReadI8Job job[kMaxJobs];
    uint32_t blk_begin[kMaxJobs + 1];
    uint32_t n_jobs, heads, blks_each;
};

// One CTA per kReadRows rows of one job's K (blockIdx.y 0) or V (1).  A thread
// writes 16 bytes at a time, so stores are coalesced and loads are 4 (f32) or
// 8 (f16) contiguous codes; 32 or 16 neighbouring threads share a scale.  A
// code becomes f32 as the low bits of 2^23 + c + 128, less 2^23 + 128.  32768 rows of 8
// heads to f16: 36 us, 5.6 TB/s (0.86 of the measured copy rate).
constexpr uint32_t kReadRows = 16;

template <bool F16>
__global__ void __launch_bounds__(256) read_i8_kernel(const __grid_constant__ ReadI8Params P) {
    constexpr uint32_t E = F16 ? 8u : 4u, kAtOnce = 4;  // elements a thread and step, steps at once
    after_previous();
    const uint32_t j = job_of(P.blk_begin, P.n_jobs, P.blks_each, blockIdx.x);
    const ReadI8Job &J = P.job[j];
    const uint32_t r0 = (blockIdx.x - P.blk_begin[j]) * kReadRows;
    const uint32_t nr = min(kReadRows, J.rows - r0);
    const uint8_t *src = blockIdx.y ? J.v_src : J.k_src;
    void *dst = blockIdx.y ? J.v_dst : J.k_dst;
    const uint64_t kv_dim = (uint64_t)P.heads * 128u;
    const float *scales = reinterpret_cast<const float *>(src + kv_dim * J.src_cap);
    const uint32_t per_row = P.heads * (128u / E), n = nr * per_row;
    const uint32_t s_src = (J.first + r0) % J.src_cap, s_dst = (J.first + r0) % J.dst_cap;
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += 256u * kAtOnce) {
        uint2 w[kAtOnce];
        float s[kAtOnce];
        uint64_t to[kAtOnce];
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; k++) {
            const uint32_t i = i0 + k * 256u;
            if (i < n) {
                const uint32_t r = i / per_row, c = i - r * per_row;
                uint32_t a = s_src + r, b = s_dst + r;
                if (a >= J.src_cap) a = a - J.src_cap < J.src_cap ? a - J.src_cap : a % J.src_cap;
                if (b >= J.dst_cap) b = b - J.dst_cap < J.dst_cap ? b - J.dst_cap : b % J.dst_cap;
                s[k] = scales[(uint64_t)(c / (128u / E)) * J.src_cap + a];
                const uint8_t *p = src + a * kv_dim + c * E;
                if (F16) w[k] = *reinterpret_cast<const uint2 *>(p);
                else w[k].x = *reinterpret_cast<const uint32_t *>(p);
                to[k] = b * kv_dim + c * E;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; k++) {
            if (i0 + k * 256u >= n) continue;
            float x[8];
#pragma unroll
            for (uint32_t e = 0; e < E; e++)
                x[e] = (__uint_as_float(__byte_perm(e < 4 ? w[k].x : w[k].y, 0x4B000000u, 0x7650u | (e & 3u))) - 8388736.0f) * s[k];
            if (F16) {
                *reinterpret_cast<uint4 *>(reinterpret_cast<__half *>(dst) + to[k]) =
                    make_uint4(h2_bits(x[0], x[1]), h2_bits(x[2], x[3]), h2_bits(x[4 % E], x[5 % E]), h2_bits(x[6 % E], x[7 % E]));
            } else {
                *reinterpret_cast<float4 *>(reinterpret_cast<float *>(dst) + to[k]) = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
    }
}

}  // namespace sf37kv

using namespace sf37kv;

extern "C" uint64_t sf37kv_i8_cache_bytes(uint32_t cap, uint32_t kv_heads, uint32_t head_dim) {
    if (head_dim != 128) return 0;
    return ((uint64_t)cap * kv_heads * 132u + 255u) / 256u * 256u;
}

extern "C" int sf37kv_append_i8(const sf37kv_append_i8_layer *layers, uint32_t n_layers, uint32_t kv_heads,
                                uint32_t head_dim, int row_type, void *stream) {
    if (!layers && n_layers) return set_error(SF37KV_EINVAL, "append_i8: layers is NULL");
    if (int rc = check_heads("append_i8", kv_heads, kv_heads, head_dim)) return rc;
    if (row_type != SF37KV_Q_F32 && row_type != SF37KV_Q_BF16)
        return set_error(SF37KV_EINVAL, "append_i8: unknown row type %d", row_type);
    cudaStream_t s = stream ? (cudaStream_t)stream : current_stream();
    // All checks run before the first launch, so a refused call changes nothing.
    for (uint32_t i = 0; i < n_layers; i++) {
        const sf37kv_append_i8_layer &L = layers[i];
        if (int rc = check_cache("append_i8", i, L.cache)) return rc;
        if (L.n_tok == 0) continue;
        if (!L.k || !L.v || !aligned16(L.k) || !aligned16(L.v))
            return set_error(SF37KV_EINVAL, "append_i8: layer %u rows must be non-NULL and 16-byte aligned", i);
        if ((uint64_t)L.pos0 + L.n_tok > kMaxPos)
            return set_error(SF37KV_EINVAL, "append_i8: layer %u positions exceed %u", i, kMaxPos);
        if ((uint64_t)(L.n_tok < L.cache.cap ? L.n_tok : L.cache.cap) * kv_heads > kMaxUnits)
            return set_error(SF37KV_EINVAL, "append_i8: layer %u has too many rows for one call", i);
    }
    try {
        if (parts_conflict((size_t)n_layers * 2, [&](const auto &add) {
                for (uint32_t i = 0; i < n_layers; i++) {
                    const sf37kv_cache &c = layers[i].cache;
                    const uint64_t bytes = layers[i].n_tok ? (uint64_t)c.cap * kv_heads * 132u : 0u;
                    add(0, c.k_cache, bytes, true);
                    add(1, c.v_cache, bytes, true);
                }
            }))
            return set_error(SF37KV_EINVAL, "append_i8: one cache is written twice in one call, or overlaps another");
    } catch (const std::bad_alloc &) {
        return set_error(SF37KV_ENOMEM, "append_i8: no memory to compare %u layers", n_layers);
    }
    for (uint32_t base = 0; base < n_layers;) {
        AppendI8Params P;
        P.n_jobs = 0;
        P.heads = kv_heads;
        const bool bf16 = row_type == SF37KV_Q_BF16;
        P.rows_each = 0;
        uint64_t rows = 0;
        uint32_t i = base;
        for (; i < n_layers && P.n_jobs < (uint32_t)kMaxJobs; i++) {
            const sf37kv_append_i8_layer &L = layers[i];
            if (L.n_tok == 0) continue;
            // With n_tok > cap only the last cap rows stay, as in a sequential append.
            const uint32_t keep = L.n_tok < L.cache.cap ? L.n_tok : L.cache.cap, skip = L.n_tok - keep;
            if ((rows + keep) * kv_heads > kMaxUnits) break;
            const uint64_t off = (uint64_t)skip * kv_heads * 128u * (bf16 ? 2u : 4u);
            P.job[P.n_jobs] = AppendI8Job{(uint8_t *)L.cache.k_cache, (uint8_t *)L.cache.v_cache,
                                          (const char *)L.k + off, (const char *)L.v + off, L.pos0 + skip,
                                          L.cache.cap};
            P.rows_each = P.n_jobs == 0 || P.rows_each == keep ? keep : 0u;
            P.row_begin[P.n_jobs++] = (uint32_t)rows;
            rows += keep;
        }
        base = i;
        if (P.n_jobs == 0) continue;
        P.row_begin[P.n_jobs] = (uint32_t)rows;
        const unsigned grid = (unsigned)((rows * kv_heads + kAppendThreads / 8u - 1u) / (kAppendThreads / 8u));
        g_launches++;
        if (int rc = launch_early("append_i8 launch", bf16 ? append_i8_kernel<true> : append_i8_kernel<false>, grid,
                                  kAppendThreads, 0,
                                  s, P))
            return rc;
    }
    return SF37KV_OK;
}

extern "C" int sf37kv_read_i8(const sf37kv_read_i8_layer *layers, uint32_t n_layers, uint32_t kv_heads,
                              uint32_t head_dim, int dst_dtype, void *stream) {
    if (!layers && n_layers) return set_error(SF37KV_EINVAL, "read_i8: layers is NULL");
    if (int rc = check_heads("read_i8", kv_heads, kv_heads, head_dim)) return rc;
    if (dst_dtype != SF37KV_F16 && dst_dtype != SF37KV_F32)
        return set_error(SF37KV_EINVAL, "read_i8: destination dtype %d is neither f16 nor f32", dst_dtype);
    cudaStream_t s = stream ? (cudaStream_t)stream : current_stream();
    for (uint32_t i = 0; i < n_layers; i++) {
        const sf37kv_read_i8_layer &L = layers[i];
        if (int rc = check_cache("read_i8", i, L.src)) return rc;
        if (int rc = check_cache("read_i8", i, L.dst)) return rc;
        if (L.rows > L.src.cap || L.rows > L.dst.cap)
            return set_error(SF37KV_EINVAL, "read_i8: layer %u has %u rows for caches of %u and %u", i, L.rows,
                             L.src.cap, L.dst.cap);
        if ((uint64_t)L.first_pos + L.rows > kMaxPos)
            return set_error(SF37KV_EINVAL, "read_i8: layer %u positions exceed %u", i, kMaxPos);
        if (L.src.k_cache == L.dst.k_cache || L.src.v_cache == L.dst.v_cache || L.src.k_cache == L.dst.v_cache ||
            L.src.v_cache == L.dst.k_cache)
            return set_error(SF37KV_EINVAL, "read_i8: layer %u reads and writes the same cache", i);
    }
    try {
        // Destinations by the rows that are written: layers may fill parts of one cache.
        const uint64_t row = (uint64_t)kv_heads * 128u * (uint64_t)dst_dtype;
        if (parts_conflict((size_t)n_layers * 6, [&](const auto &add) {
                for (uint32_t i = 0; i < n_layers; i++) {
                    const sf37kv_read_i8_layer &L = layers[i];
                    if (L.rows == 0) continue;
                    const uint64_t slot = L.first_pos % L.dst.cap, head = std::min<uint64_t>(L.rows, L.dst.cap - slot),
                                   bytes = (uint64_t)L.src.cap * kv_heads * 132u;
                    add(0, L.dst.k_cache, (L.rows - head) * row, true);
                    add(0, (const char *)L.dst.k_cache + slot * row, head * row, true);
                    add(1, L.dst.v_cache, (L.rows - head) * row, true);
                    add(1, (const char *)L.dst.v_cache + slot * row, head * row, true);
                    add(2, L.src.k_cache, bytes, false);
                    add(3, L.src.v_cache, bytes, false);
                }
            }))
            return set_error(SF37KV_EINVAL, "read_i8: rows that one layer writes are another's, read or written");
    } catch (const std::bad_alloc &) {
        return set_error(SF37KV_ENOMEM, "read_i8: no memory to compare %u layers", n_layers);
    }
    for (uint32_t base = 0; base < n_layers;) {
        ReadI8Params P;
        P.n_jobs = 0;
        P.heads = kv_heads;
        P.blks_each = 0;
        uint64_t blks = 0;
        uint32_t i = base;
        for (; i < n_layers && P.n_jobs < (uint32_t)kMaxJobs; i++) {
            const sf37kv_read_i8_layer &L = layers[i];
            if (L.rows == 0) continue;
            const uint32_t nb = (L.rows + kReadRows - 1u) / kReadRows;
            if (blks + nb > kMaxUnits) break;
            P.job[P.n_jobs] = ReadI8Job{(const uint8_t *)L.src.k_cache, (const uint8_t *)L.src.v_cache, L.dst.k_cache,
                                        L.dst.v_cache, L.first_pos, L.rows, L.src.cap, L.dst.cap};
            P.blks_each = P.n_jobs == 0 || P.blks_each == nb ? nb : 0u;
            P.blk_begin[P.n_jobs++] = (uint32_t)blks;
            blks += nb;
        }
        base = i;
        if (P.n_jobs == 0) continue;
        P.blk_begin[P.n_jobs] = (uint32_t)blks;
        g_launches++;
        if (int rc = launch_early("read_i8 launch", dst_dtype == SF37KV_F16 ? read_i8_kernel<true> : read_i8_kernel<false>,
                                  dim3((unsigned)blks, 2), 256, 0, s, P))
            return rc;
    }
    return SF37KV_OK;
}
