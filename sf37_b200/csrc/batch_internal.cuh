// Declarations shared by the int8 cache and the batched decode kernels
// (cache_i8.cu, batch_decode.cu, prefix_tc05.cu).
#pragma once

#include <algorithm>
#include <new>
#include <vector>

#include <cuda_bf16.h>

#include "kv_internal.cuh"

namespace sf37kv {

// Positions stay below 2^31 so that pos + 1 and slot sums fit 32 bits.
constexpr uint32_t kMaxPos = 0x7fffffffu;
constexpr uint64_t kMaxUnits = 0x7fffff00ull;  // grid size bound

static inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

// Head counts and head_dim that the kernels of this file family take.
static inline int check_heads(const char *what, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim) {
    if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads)
        return set_error(SF37KV_EINVAL, "%s: %u query heads do not divide over %u KV heads", what, q_heads, kv_heads);
    if (head_dim != 128) return set_error(SF37KV_EUNSUPPORTED, "%s: head_dim must be 128", what);
    if (kv_heads > 4096) return set_error(SF37KV_EUNSUPPORTED, "%s: more than 4096 KV heads", what);
    if (q_heads / kv_heads > 16)
        return set_error(SF37KV_EUNSUPPORTED, "%s: more than 16 query heads for each KV head", what);
    return SF37KV_OK;
}

static inline int check_cache(const char *what, uint32_t i, const sf37kv_cache &c) {
    if (!c.k_cache || !c.v_cache || !aligned16(c.k_cache) || !aligned16(c.v_cache))
        return set_error(SF37KV_EINVAL, "%s: cache %u must be non-NULL and 16-byte aligned", what, i);
    if (c.cap == 0 || c.cap > kMaxPos) return set_error(SF37KV_EINVAL, "%s: cache %u has cap %u", what, i, c.cap);
    if (c.k_cache == c.v_cache) return set_error(SF37KV_EINVAL, "%s: cache %u has one buffer for K and V", what, i);
    return SF37KV_OK;
}

// Whether memory that one part of a call writes overlaps what another part reads or
// writes.  each(add) calls add(list, address, bytes, writes) for every part, at most n
// of them; `list` (below kLists) tells parts apart that lie in order, each list in a
// range of its own, as a rule: K and V caches in one allocation each.  Then two
// comparisons a part settle it; otherwise the parts are sorted (std::bad_alloc).
constexpr uint32_t kLists = 4;
template <typename Each>
static bool parts_conflict(size_t n, const Each &each) {
    struct Span {
        uintptr_t lo, hi;
        bool writes;
    };
    Span list[kLists] = {};  // from the lowest byte to the highest
    bool in_order[kLists] = {true, true, true, true};
    each([&](uint32_t i, const void *p, uint64_t bytes, bool writes) {
        if (!bytes) return;
        Span &x = list[i];
        const uintptr_t lo = (uintptr_t)p, hi = lo + (uintptr_t)bytes;
        x.writes |= writes;
        in_order[i] &= lo >= x.hi;
        x.lo = x.hi ? std::min(x.lo, lo) : lo;
        x.hi = std::max(x.hi, hi);
    });
    bool apart = true;
    for (uint32_t i = 0; i < kLists; i++) {
        apart &= in_order[i] || !list[i].writes;
        for (uint32_t k = 0; k < i; k++)
            apart &= !(list[i].writes || list[k].writes) || list[i].hi <= list[k].lo || list[k].hi <= list[i].lo;
    }
    if (apart) return false;
    std::vector<Span> s;
    s.reserve(n);
    each([&](uint32_t, const void *p, uint64_t bytes, bool writes) {
        if (bytes) s.push_back(Span{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, writes});
    });
    std::sort(s.begin(), s.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
    uintptr_t any = 0, written = 0;  // ends of the spans so far
    for (const Span &x : s) {
        if (x.lo < written || (x.writes && x.lo < any)) return true;
        any = std::max(any, x.hi);
        if (x.writes) written = std::max(written, x.hi);
    }
    return false;
}

// Launches a kernel that starts while the one before it on the stream drains
// (programmatic dependent launch) and so calls after_previous() before it touches
// memory.  sf37kv_decode, whose kernels read some caches before they wait, is
// told that its successor's start is no longer ordered behind this one's end.
template <typename Kernel, typename Params>
static int launch_early(const char *what, Kernel kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t stream,
                        const Params &params) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    stream_record_drop(stream);
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params);
    if (e == cudaSuccess) e = cudaGetLastError();
    return check_cuda(e, what);
}
// Waits for the kernel before, then lets the next one start.  What the kernel before
// wrote is read by plain loads from here on: a kernel that starts early may not
// read it as data that is constant for its whole run (ld.global.nc).
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
}

// Two words of a workspace, zero between calls: `ready` is set by the prefix launch once
// all work before it is complete and visible to it, and read by the decode launch that
// runs beside it; `done` counts that launch's CTAs, the last of which clears both.
struct PrefixSync {
    uint32_t ready, done;
};
// Of one thread, after griddepcontrol.wait.
__device__ __forceinline__ void publish_previous(PrefixSync *sync) {
    asm volatile("st.release.gpu.global.u32 [%0], 1;" ::"l"(&sync->ready) : "memory");
}
// Of a warp of the launch that starts while the prefix launch runs: orders what follows
// after all work that the prefix launch waited for.  The release above and this
// acquire do so, and as a rule the flag is there at the first look, since the launch
// starts after it; where it is not, the warp waits for the prefix launch itself.
__device__ __forceinline__ void after_published(const PrefixSync *sync) {
    uint32_t seen = 0;
    if ((threadIdx.x & 31u) == 0)
        for (int i = 0; i < 16 && !seen; i++)
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(&sync->ready) : "memory");
    if (!__shfl_sync(0xffffffffu, seen, 0)) asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncwarp();
}
// Of one thread of each CTA of that launch, when its warps are past after_published().
__device__ __forceinline__ void leave_published(PrefixSync *sync) {
    uint32_t prev;
    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;"
                 : "=r"(prev) : "l"(&sync->done), "r"(gridDim.x - 1u) : "memory");
    if (prev == gridDim.x - 1u) sync->ready = 0u;
}

__device__ __forceinline__ uint32_t h2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Four consecutive elements of an f32 or bf16 array (16- or 8-byte aligned).
__device__ __forceinline__ float4 load_row4(const void *p, uint64_t i, bool bf16) {
    if (!bf16) return *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + i);
    const uint2 w = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(p) + i);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}

// max(a, |x|), NaN where either is.
__device__ __forceinline__ float max_abs_nan(float a, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(x)));
    return r;
}
// The scale of a head whose largest |element| (NaN if one is) is a.
__device__ __forceinline__ float i8_scale(float a) {
    if (!(a <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    const float s = __fdiv_rn(a, 127.0f);
    return s < 1.17549435e-38f ? 0.f : s;
}
// Byte c + 128 in the low bits: c the integer nearest to x / s, ties to even,
// decided exactly.  inv = 1 / s.  x * inv + 1.5 * 2^23 rounds to an integer that
// is at most one off; the remainder x - c*s is an exact f32 (a multiple of the
// smaller of ulp(x), ulp(s) and at most 1.5 s), so comparing 2r with s is exact too.
__device__ __forceinline__ uint32_t i8_byte(float x, float s, float inv) {
    constexpr float kMagic = 12582912.0f + 128.0f;  // the integer's low byte is c + 128
    const float t = fmaf(x, inv, kMagic), c = t - kMagic;
    const float r = fmaf(-c, s, x), r2 = r + r;
    uint32_t b = __float_as_uint(t);
    if (fabsf(r2) >= s) {  // a tie, or one off (rare)
        const bool odd = (b & 1u) != 0;
        if (r2 > s || (r2 == s && odd)) b++;
        else if (-r2 > s || (-r2 == s && odd)) b--;
    }
    return b;
}
// Four codes to a word.
__device__ __forceinline__ uint32_t i8_pack(float x, float y, float z, float w, float s, float inv) {
    const uint32_t a = __byte_perm(i8_byte(x, s, inv), i8_byte(y, s, inv), 0x0040);
    const uint32_t b = __byte_perm(i8_byte(z, s, inv), i8_byte(w, s, inv), 0x0040);
    return __byte_perm(a, b, 0x5410);
}
// The same without the decision; `worst` becomes the largest |remainder|.  The
// codes are right if that is below s / 2 (all but those within 2^-16 of a tie).
__device__ __forceinline__ uint32_t i8_pack_near(const float *x, float s, float inv, float &worst) {
    constexpr float kMagic = 12582912.0f + 128.0f;
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float t = fmaf(x[i], inv, kMagic);
        b[i] = __float_as_uint(t);
        worst = fmaxf(worst, fabsf(fmaf(kMagic - t, s, x[i])));
    }
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
constexpr uint32_t kI8Zero = 0x80808080u;  // four zeros: also the codes of a NaN scale

// Quantises one head (four elements a lane, all 32 lanes) and stores its codes
// and scale in slot `slot` of an I8 cache.
__device__ __forceinline__ void store_i8_head(uint8_t *cache, uint32_t cap, uint32_t heads, uint32_t head, uint32_t slot,
                                              uint32_t lane, float4 x) {
    float a = max_abs_nan(max_abs_nan(max_abs_nan(fabsf(x.x), x.y), x.z), x.w);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = max_abs_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
    const float s = i8_scale(a);
    const uint64_t kv_dim = (uint64_t)heads * 128u;
    *reinterpret_cast<uint32_t *>(cache + slot * kv_dim + head * 128u + lane * 4u) =
        s > 0.f ? i8_pack(x.x, x.y, x.z, x.w, s, __frcp_rn(s)) : kI8Zero;
    if (lane == 0) reinterpret_cast<float *>(cache + cap * kv_dim)[(uint64_t)head * cap + slot] = s;
}

// ------------------------------------------------------------ shared prefix
constexpr int kPrefixGroups = 8;    // groups per prefix launch
constexpr int kPrefixSeqs = 256;    // sequences per prefix launch
constexpr uint32_t kPlanSms = 148;  // B200

struct PrefixSeq {
    const void *q;     // [q_heads][128]
    uint32_t start;    // first prefix row that the sequence attends to
    uint32_t pad;
};
// One group: all sequences over the rows [lo, len) of one f16 prefix cache.
struct PrefixGroup {
    const void *k, *v;
    uint32_t lo, len;
    uint32_t seq0, n_seqs;      // its sequences in the launch's list
    // filled by prefix_plan()
    uint32_t m_tiles, splits, tiles_per_split;
    uint32_t part0;             // first partial tile of the group
};

// Sequences of one 128-row tile: row sl * G + hl holds head hl of sequence sl.
static inline uint32_t prefix_seqs_per_tile(uint32_t group) { return 128u / group; }

// Splits each group's rows over CTAs, considering that the launch that follows
// reads own_rows own rows (f16 or I8) on the SMs left; returns the number of CTAs.  A partial tile is
// 128 x 128 f32 (unnormalised outputs) and 128 (reference, sum) pairs; that of
// (kv head h, m tile t, split s) is part0 + (h * m_tiles + t) * splits + s.
uint32_t prefix_plan(PrefixGroup *groups, uint32_t n, uint32_t q_heads, uint32_t kv_heads, bool f32, uint64_t own_rows,
                     bool own_i8);
// Partial tiles that prefix_plan() stays within.
uint64_t prefix_tiles_bound(uint64_t n_groups, uint64_t n_seqs, uint32_t q_heads, uint32_t kv_heads);
int prefix_attention(const PrefixGroup *groups, uint32_t n, const PrefixSeq *seqs, uint32_t n_seqs, uint32_t q_heads,
                     uint32_t kv_heads, bool f32, float *part, float *ml, PrefixSync *sync, cudaStream_t stream);

}  // namespace sf37kv
