// Attention of a batch of decode queries over one shared f16 prefix, on the
// tcgen05 tensor cores: each K/V tile is read once for up to 32 sequences.
//
// M folds the batch and the GQA group: row sl * G + hl of a 128-row Q tile is
// query head hl of sequence sl (128 / G sequences a tile), so one UMMA serves
// all of a KV head's queries.  A CTA takes one KV head, a run of 128-key tiles
// (a split) and one or two Q tiles, and leaves its unnormalised O with a
// (reference, sum) pair for each row; batch_decode.cu joins the splits with each
// sequence's own rows.
//
// Two streams of a CTA ping-pong, so that one's softmax overlaps the other's
// MMAs.  With two Q tiles (pair) each stream is a Q tile and both use every
// K/V tile; with one (solo) the streams take alternate K/V tiles of the same
// Q tile and are joined through shared memory at the end.
//
// The first 16 warps are the softmax, eight for each stream and two threads for
// each row; they weigh a tile in one pass, with the reference of the tiles
// before it (one thread a row and two passes over S took 108 us where this took
// 101, 64 sequences over 32768 rows).  F32 has 8 and one thread a row: two leave it no registers.  Then
// one warp issues the MMAs and one the TMA loads.  TMEM: S_0, S_1, O_0, O_1 (128
// columns each); P (f16) overwrites its S.  F32 (f32 queries and outputs): q and P
// are two f16 parts each, q_hi + q_lo and P_hi + P_lo, 22 bits: twice the MMAs;
// P_lo takes the second half of S's columns.
//
// Weights are 2^(x - m) with the reference m 7 below a running row maximum,
// raised when x - m passes 15: f16 holds them up to 2^15, and down to 2^-32 of
// the largest.  S and O accumulate in f32 (TMEM), m and l in f32 registers.
//
// Bound by the MMA thread and the tensor pipe: a step (S and PV of one stream and
// key tile) is 1024 cycles of MMA, issues in 1300-1500 (8 MMAs and their commits
// take 600 on an idle SM, more beside the softmax) and takes 1850; its softmax takes
// 1700 and is hidden by the other stream's.  64 sequences x 64 heads, bf16: this
// launch takes 292 us over 131072 rows, 0.94 PFLOP/s (0.56 of the measured burst
// bf16 rate); 86 us over 32768, of which 15 are a CTA's start and end (64 KB of q and
// the first tiles, a 128 KB partial out).
#include <algorithm>
#include <type_traits>

#include "batch_internal.cuh"
#include "tc05.cuh"

namespace sf37kv {

extern unsigned long long g_launches;

static __device__ int g_prefix_error;  // 1: a bounded wait gave up

struct PrefixDev {
    CUtensorMap kmap, vmap;  // rows [0, len): later rows read as zeros
    const __half *k, *v;
    uint32_t lo, len, seq0, n_seqs, m_tiles, splits, tps, part0, cta0, pairs;
};
template <int NS>
struct PrefixParams {
    PrefixDev group[kPrefixGroups];
    PrefixSeq seq[NS];
    float *part, *ml;
    PrefixSync *sync;
    uint32_t take0;  // first of one partial tile for each CTA, for stream 1's sums (F32)
    uint32_t n_groups, heads_per_kv, kv_heads, tpt;
};

constexpr float kHead = 7.0f, kRaise = 15.0f;
// x * qs - m as one fma keeps the product's last bits, which m's rounding lacks: 0.125 at
// references up to this, beyond which product and difference are rounded one by one.
constexpr float kFused = 2097152.0f;
constexpr float kNone = -3.402823466e38f;  // reference of a row without keys: no finite score is below it
// The tensor core truncates its f32 sums: O loses 1.7e-8 of itself with each MMA (measured).
// F32 takes O into sums in memory after this many key tiles of a stream (256 MMAs,
// 4e-6; 16000 keys, 40 sequences: 99 us with half as many, 85 with none).
constexpr uint32_t kTake = 16;

// Threads of a row in the softmax, and its warps.
__host__ __device__ constexpr uint32_t row_threads(bool f32) { return f32 ? 1 : 2; }
__host__ __device__ constexpr uint32_t soft_warps(bool f32) { return 8 * row_threads(f32); }

// Q tiles: scaled by a power of two for each row so that its largest element is
// in [1, 2): f16 then holds a bf16 row exactly and hi + lo 22 bits.  Of the
// 8 warps each reads whole rows, 16 lanes (bf16) or 32 (f32) each: with a row a
// thread, 32 lines a load, this took 8 us.  `rows` is 128 or 256 (two tiles).
template <bool F32>
__device__ __forceinline__ void load_q(const PrefixSeq *tab, uint32_t n_seqs, uint32_t mt0, uint32_t rows, uint32_t kvh,
                                       uint32_t G, uint32_t T, uint8_t *tiles, float *qscale) {
    using namespace tc05;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    constexpr uint32_t kLanes = F32 ? 32 : 16, kAtOnce = 32 / kLanes;
    constexpr uint32_t kWarps = soft_warps(F32);
    const uint32_t c = lane % kLanes, n = rows / (kWarps * kAtOnce);  // trips of a warp
    for (uint32_t i0 = 0; i0 < n; i0 += 8u) {
        const uint32_t x0 = (warp * n + i0) * kAtOnce;
        uint4 raw[8];
        float scale[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i0 + i >= n) break;
            const uint32_t x = x0 + i * kAtOnce + lane / kLanes;  // row of both tiles
            const uint32_t sl = (x & 127u) / G, hl = (x & 127u) - sl * G;
            const PrefixSeq q = tab[min((mt0 + (x >> 7)) * T + sl, n_seqs - 1u)];
            raw[i] = reinterpret_cast<const uint4 *>(q.q)[(uint64_t)(kvh * G + hl) * kLanes + c];
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i0 + i >= n) break;
            const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++)
                top = F32 ? fmaxf(top, fabsf(__uint_as_float(u[k])))
                          : fmaxf(top, fmaxf(fabsf(__uint_as_float(u[k] << 16)), fabsf(__uint_as_float(u[k] & 0xffff0000u))));
#pragma unroll
            for (uint32_t k = kLanes / 2; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
            scale[i] = top;
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i0 + i >= n) break;
            const uint32_t x = x0 + i * kAtOnce + lane / kLanes, r = x & 127u;
            const int e = max(-126, min(126, (int)((__float_as_uint(scale[i]) >> 23) & 255u) - 127));
            const float f = __int_as_float((127 - e) << 23);
            if (c == 0) qscale[x] = __int_as_float((127 + e) << 23) * (1.4426950408889634f * 0.08838834764831845f);
            const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            uint8_t *qt = tiles + (x >> 7) * kTile;
            if (F32) {
                uint32_t hv[2], lv[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float a = __uint_as_float(u[2 * k]) * f, b = __uint_as_float(u[2 * k + 1]) * f;
                    hv[k] = pack_h2(a, b);
                    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hv[k]));
                    lv[k] = pack_h2(a - h.x, b - h.y);
                }
                *reinterpret_cast<uint2 *>(qt + tile_off(r, c >> 1) + 8u * (c & 1u)) = make_uint2(hv[0], hv[1]);
                *reinterpret_cast<uint2 *>(qt + kTile + tile_off(r, c >> 1) + 8u * (c & 1u)) = make_uint2(lv[0], lv[1]);
            } else {
                uint4 hv;
                uint32_t *ho = &hv.x;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    ho[k] = pack_h2(__uint_as_float(u[k] << 16) * f, __uint_as_float(u[k] & 0xffff0000u) * f);
                *reinterpret_cast<uint4 *>(qt + tile_off(r, c)) = hv;
            }
        }
    }
    fence_async_smem();
}

// The weight of a raw score x under the reference m.
template <bool FUSED>
__device__ __forceinline__ float weight(float x, float qs, float m) {
    return fast_exp2(FUSED ? fmaf(x, qs, -m) : __fsub_rn(__fmul_rn(x, qs), m));
}

// Whether any thread of two warps (named barrier `id`), or of all softmax warps, says so.
__device__ __forceinline__ bool bar_any(uint32_t id, uint32_t threads, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((uint32_t)x), "r"(id), "r"(threads) : "memory");
    return r != 0;
}
__device__ __forceinline__ bool pair_any(uint32_t id, bool x) { return bar_any(id, 64, x); }
__device__ __forceinline__ bool soft_any(uint32_t threads, bool x) { return bar_any(9, threads, x); }

__device__ __forceinline__ bool all_finite(const float4 &x) {
    return fmaf(x.x, 0.f, x.y * 0.f) + fmaf(x.z, 0.f, x.w * 0.f) == 0.f;
}

// One row of a partial tile again, by a warp: query head q [128] over the keys
// [first, end) of K and V (`stride` elements a row).  PV multiplies every V row of a
// tile by every weight, and 0 times a V that is not finite is NaN for sequences that do
// not attend to it; so is q_hi K + q_lo K where K is infinite.  A row of O that is not
// finite is therefore taken again by the formula, unless its query is the reason.
__device__ __noinline__ void redo_row(const void *q, bool bf16, const __half *k, const __half *v, uint64_t stride,
                                      uint32_t first, uint32_t end, float *o, float *ml) {
    const uint32_t lane = threadIdx.x & 31u;
    const float4 x = load_row4(q, lane * 4u, bf16);
    if (__any_sync(0xffffffffu, !all_finite(x))) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = kNone, l = 0.f;
    auto row4 = [&](const __half *base, uint32_t r) {
        const uint2 w = *reinterpret_cast<const uint2 *>(base + r * stride + lane * 4u);
        const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)),
                     hi = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        return make_float4(lo.x, lo.y, hi.x, hi.y);
    };
    for (uint32_t r = first; r < end; r += 4u) {
        float s[4];
        float4 y[4];
        float mn = m;
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t at = min(r + i, end - 1u);
            const float4 z = row4(k, at);
            y[i] = row4(v, at);
            s[i] = fmaf(x.x, z.x, fmaf(x.y, z.y, fmaf(x.z, z.z, x.w * z.w)));
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
            s[i] *= 1.4426950408889634f * 0.08838834764831845f;
            mn = fmaxf(mn, s[i]);
        }
        const float f = fast_exp2(m - mn);
        m = mn;
        l *= f;
        a = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            if (r + i >= end) break;
            const float p = fast_exp2(s[i] - m);
            l += p;
            a = make_float4(fmaf(p, y[i].x, a.x), fmaf(p, y[i].y, a.y), fmaf(p, y[i].z, a.z), fmaf(p, y[i].w, a.w));
        }
    }
    *reinterpret_cast<float4 *>(o + lane * 4u) = a;
    if (lane == 0) *reinterpret_cast<float2 *>(ml) = make_float2(m, l);
}

template <bool F32, int NS>
__global__ void __launch_bounds__(soft_warps(F32) * 32 + 64, 1) prefix_tc05_kernel(const __grid_constant__ PrefixParams<NS> P) {
    using namespace tc05;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    enum { B_KFULL = 0, B_KEMPTY = 3, B_VFULL = 6, B_VEMPTY = 8, B_SFULL = 10, B_PFULL = 12, B_ODONE = 14, B_DRAIN = 16, N_BARS = 17 };
    enum { T_Q = 0, T_K = 2, T_V = 4 };  // 32 KB tiles; Q: two tiles (pair) or hi and lo (F32), else a third K tile
    __shared__ __align__(8) uint64_t bars[N_BARS];
    __shared__ uint32_t tmem_base_sh;
    __shared__ volatile int abort_sh;
    constexpr uint32_t H = row_threads(F32), kSoft = soft_warps(F32);
    __shared__ float2 ml_sh[2][H][128];  // [stream][half][row] (m, l)
    __shared__ float top_sh[2][H][128];
    __shared__ float qscale_sh[2][128];

    const uint32_t sraw = (uint32_t)__cvta_generic_to_shared(smem_raw);
    const uint32_t s0 = (sraw + 1023u) & ~1023u;
    uint8_t *gsm = smem_raw + (s0 - sraw);
    auto tile = [&](uint32_t i) { return s0 + i * kTile; };
    auto bar = [&](uint32_t i) { return (uint32_t)__cvta_generic_to_shared(&bars[i]); };
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;

    uint32_t gi = 0;
    while (gi + 1 < P.n_groups && P.group[gi + 1].cta0 <= blockIdx.x) gi++;
    const PrefixDev &Gr = P.group[gi];
    const uint32_t local = blockIdx.x - Gr.cta0;
    const uint32_t pr = local % Gr.pairs, kvh = (local / Gr.pairs) % P.kv_heads, split = local / (Gr.pairs * P.kv_heads);
    const uint32_t mt0 = F32 ? pr : 2u * pr;
    const bool solo = F32 || mt0 + 1u >= Gr.m_tiles;
    const uint32_t G = P.heads_per_kv, T = P.tpt;
    const uint32_t kbeg = Gr.lo + split * Gr.tps * 128u;
    const uint32_t kend = min(kbeg + Gr.tps * 128u, Gr.len);
    const uint32_t nt = (kend - kbeg + 127u) / 128u;
    const uint32_t steps = solo ? nt : 2u * nt;

    const bool loads = tid == (kSoft + 1u) * 32u;  // the thread that issues the TMA loads
    if (loads) {
        for (uint32_t t = 0; t < 3; t++) {
            bar_init(bar(B_KFULL + t), 1);
            bar_init(bar(B_KEMPTY + t), 1);
        }
        for (uint32_t t = 0; t < 2; t++) {
            bar_init(bar(B_VFULL + t), 1);
            bar_init(bar(B_VEMPTY + t), 1);
            bar_init(bar(B_SFULL + t), 1);
            bar_init(bar(B_PFULL + t), 128 * H);
            bar_init(bar(B_ODONE + t), 1);
        }
        bar_init(bar(B_DRAIN), 1);
        asm volatile("fence.mbarrier_init.release.cluster;");
        abort_sh = 0;
    }
    if (warp == 0) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(&tmem_base_sh);
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // The next kernel reads this one's partials after a wait of its own, and what was written
    // before this one after the flag.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x == 0 && tid == 0) publish_previous(P.sync);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto load = [&](uint32_t full, uint32_t dst, const CUtensorMap *map, uint32_t j) {
        const int32_t x = (int32_t)(kvh * 128u), y = (int32_t)(kbeg + j * 128u);
        bar_expect_tx(full, kTile);
        tma_load_2d(dst, map, x, y, full);
        tma_load_2d(dst + kHalf, map, x + 64, y, full);
    };
    // The first K tile is asked for beside q (4 sequences over 512 rows: 10.2 -> 9.9 us); more
    // would queue ahead of q.
    if (loads) load(bar(B_KFULL), tile(solo && !F32 ? 1u : T_K), &Gr.kmap, 0);

    // The sequences' table is read by generic loads: lane-divergent constant loads replay.
    const PrefixSeq *tab = P.seq;
    asm volatile("" : "+l"(tab));
    if (warp < kSoft)
        load_q<F32>(tab + Gr.seq0, Gr.n_seqs, mt0, solo ? 128u : 256u, kvh, G, T, gsm + T_Q * kTile, &qscale_sh[0][0]);
    const uint32_t st = warp / (4u * H), half = (warp >> 2) % H;  // of a softmax warp
    const uint32_t r = ((warp & 3u) << 5) | lane;
    const uint32_t sl = r / G;
    const uint32_t mt = solo ? mt0 : mt0 + (st & 1u);
    const uint32_t si = mt * T + sl;  // sequence within the group
    const bool valid = sl < T && si < Gr.n_seqs;
    const uint32_t first = tab[Gr.seq0 + min(si, Gr.n_seqs - 1u)].start;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base_sh;

    uint32_t k_loads = 0, v_loads = 0;  // issued, of the thread that does

    if (warp == kSoft + 1) {
        // ---------------- TMA loader: a ring of K tiles and one of V tiles ----------------
        auto loader = [&](auto kind) {
            constexpr uint32_t kRing = decltype(kind)::value && !F32 ? 3 : 2, kTile0 = kRing == 3 ? 1 : T_K;
            auto load_k = [&](uint32_t j) {
                load(bar(B_KFULL + j % kRing), tile(kTile0 + j % kRing), &Gr.kmap, j);
                k_loads = j + 1u;
            };
            auto load_v = [&](uint32_t j) {
                load(bar(B_VFULL + (j & 1u)), tile(T_V + (j & 1u)), &Gr.vmap, j);
                v_loads = j + 1u;
            };
            k_loads = 1u;
            for (uint32_t j = 0; j < kRing && j < nt; j++) {
                if (j > 0) load_k(j);
                if (j < 2) load_v(j);
            }
            for (uint32_t j = 0; j + 2 < nt && !abort_sh; j++) {
                if (j + kRing < nt) {
                    if (!wait_bar(bar(B_KEMPTY + j % kRing), (j / kRing) & 1u)) { abort_sh = 1; break; }
                    load_k(j + kRing);
                }
                if (!wait_bar(bar(B_VEMPTY + (j & 1u)), (j >> 1) & 1u)) { abort_sh = 1; break; }
                load_v(j + 2);
            }
        };
        if (loads) {
            if (solo) loader(std::true_type());
            else loader(std::false_type());
        }
    } else if (warp == kSoft) {
        // ---------------- MMA issuer ----------------
        // Step i belongs to stream i & 1 and takes key tile i (solo) or i / 2 (pair).  S
        // of step i + 2 overwrites the columns from which PV of step i reads P: MMAs
        // issued by one thread execute in order.  The streams wait for this thread,
        // so it computes little: each kind has its own loop, descriptors are a base
        // and an offset, and tiles are waited for before P (100 cycles more a step took
        // 64 x 32768 from 123 to 129 us).
        auto issuer = [&](auto kind) -> bool {
            constexpr bool kSolo = decltype(kind)::value;
            constexpr uint32_t kRing = kSolo && !F32 ? 3 : 2, kTile0 = kRing == 3 ? 1 : T_K, kSteps = F32 ? 16 : 8;
            const uint64_t qd = sdesc(tile(T_Q), 16, 1024), kd = sdesc(tile(kTile0), 16, 1024),
                           vd = sdesc(tile(T_V), kHalf, 1024);
            uint32_t ks = 0, kp = 0, vs = 0, vp = 0;  // next K tile's and V tile's slot and phase
            auto issue_s = [&](uint32_t t) {
                const uint64_t a = qd + (kSolo ? 0u : t * (kTile >> 4)), b = kd + ks * (kTile >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < kSteps; kk++) {
                    // F32: the remainders' products first, so that they are not cut off a large sum
                    const uint32_t off = (((kk >> 2) & 1u) * kHalf + (kk & 3u) * 32u) >> 4, lo = F32 ? 1u - (kk >> 3) : 0u;
                    mma(tmem + t * 128u, a + lo * (kTile >> 4) + off, b + off, idesc(0), kk > 0);
                }
                commit(bar(B_SFULL + t));
                if (kSolo || t == 1) {
                    commit(bar(B_KEMPTY + ks));
                    if (++ks == kRing) {
                        ks = 0;
                        kp ^= 1u;
                    }
                }
            };
            auto issue_pv = [&](uint32_t t, uint32_t acc, bool last) {
                const uint64_t b = vd + vs * (kTile >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < kSteps; kk++)
                    mma_ts(tmem + 256u + t * 128u, tmem + t * 128u + kk * 8u, b + (kk & 7u) * 128u, idesc(1), kk > 0 ? 1u : acc);
                if (last) commit(bar(B_ODONE + t));
                if (kSolo || t == 1) {
                    commit(bar(B_VEMPTY + vs));
                    vs ^= 1u;
                    vp ^= vs == 0;
                }
            };
            for (uint32_t i = 0; i < 2 && i < steps; i++) {
                if ((kSolo || i == 0) && !wait_bar(bar(B_KFULL + ks), kp)) return false;
                fence_after();
                issue_s(i);
            }
            for (uint32_t i = 0; i < steps && !abort_sh; i++) {
                const uint32_t t = i & 1u;
                const bool more = i + 2 < steps;
                if (kSolo || t == 0) {
                    if (!wait_bar(bar(B_VFULL + vs), vp)) return false;
                    if (more && !wait_bar(bar(B_KFULL + ks), kp)) return false;
                }
                if (!wait_bar(bar(B_PFULL + t), (i >> 1) & 1u)) return false;
                fence_after();
                issue_pv(t, F32 ? (i >> 1) % kTake != 0 : i > 1, !more);
                if (more) issue_s(t);
            }
            return true;
        };
        if (lane == 0 && !(solo ? issuer(std::true_type()) : issuer(std::false_type()))) abort_sh = 1;
    } else {
        // ---------------- softmax of stream st, H threads a row ----------------
        const uint32_t lane_off = ((warp & 3u) * 32u) << 16;
        const uint32_t t_s = tmem + st * 128u + lane_off, t_o = tmem + 256u + st * 128u + lane_off;
        const uint32_t s_row = max(first, kbeg);
        const float qs = qscale_sh[solo ? 0 : st][r];
        const uint32_t n_steps = solo ? (nt + 1u - st) >> 1 : nt;
        float m = kNone, l = 0.f;
        bool ok = true;
        // Partial tile of (kv head, m tile, split); F32: this thread's sums of O, relative to
        // 2^m_taken (stream 0's in the partial tile that it writes at the end).
        const uint64_t row = ((uint64_t)Gr.part0 + ((uint64_t)kvh * Gr.m_tiles + mt) * Gr.splits + split) * 128u + r;
        float *sums = P.part + (st == 0 ? row - r : ((uint64_t)P.take0 + blockIdx.x) * 128u) * 128u + r;  // [column][row]
        float m_taken = kNone;
        // 32 columns of O and of the sums
        auto read_o = [&](uint32_t c, bool add, float scale, float (&v)[32]) {
            tmem_ld32(t_o + c * 32u, v);
            tmem_wait_ld();
            if (add) {
#pragma unroll
                for (int i = 0; i < 32; i++) v[i] = fmaf(sums[(c * 32 + i) * 128], scale, v[i]);
            }
        };
        for (uint32_t s = 0; s < n_steps; s++) {
            const uint32_t k0 = kbeg + (solo ? 2u * s + st : s) * 128u;
            __syncwarp();
            ok = !abort_sh && wait_bar_warp(bar(B_SFULL + st), s & 1u);
            if (H == 1 && !ok) break;
            fence_after();
            if (F32 && s > 0 && s % kTake == 0) {  // PV of this step starts O anew
                const float scale = fast_exp2(m_taken - m);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float v[32];
                    read_o(c, s > kTake, scale, v);
#pragma unroll
                    for (int i = 0; i < 32; i++) sums[(c * 32 + i) * 128] = v[i];
                }
                m_taken = m;
            }
            const bool edge = __any_sync(0xffffffffu, k0 < s_row || k0 + 128u > kend);
            // scores 32c .. 32c+31, -inf outside the row's keys
            auto mask = [&](uint32_t c, float (&x)[32]) {
                if (edge)
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (k0 + 32u * c + (uint32_t)i < s_row || k0 + 32u * c + (uint32_t)i >= kend) x[i] = -INFINITY;
            };
            auto top_of = [&](const float (&x)[32]) {
                float a = x[0], b = x[1];
#pragma unroll
                for (int i = 2; i < 32; i += 2) {
                    a = fmaxf(a, x[i]);
                    b = fmaxf(b, x[i + 1]);
                }
                return fmaxf(a, b);
            };
            float la = 0.f, lb = 0.f;
            if constexpr (H == 1) {
                // The first half is read twice, the second half stays in registers.
                float v[2][32], u[2][32];
                tmem_ld32(t_s, u[0]);
                tmem_ld32(t_s + 32u, u[1]);
                tmem_wait_ld();
                tmem_ld32(t_s + 64u, v[0]);
                tmem_ld32(t_s + 96u, v[1]);
                mask(0, u[0]);
                mask(1, u[1]);
                float mx = fmaxf(top_of(u[0]), top_of(u[1]));
                tmem_wait_ld();
                tmem_ld32(t_s, u[0]);
                mask(2, v[0]);
                mask(3, v[1]);
                const float top = fmaxf(mx, fmaxf(top_of(v[0]), top_of(v[1]))) * qs;
                const bool raise = top - m > kRaise;
                if (__any_sync(0xffffffffu, raise)) {
                    const float mn = raise ? top - kHead : m, alpha = fast_exp2(m - mn);
                    if (s > 0) {
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            float o[32];
                            tmem_ld32(t_o + c * 32u, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] *= alpha;
                            tmem_st32(t_o + c * 32u, o);
                        }
                    }
                    l *= alpha;
                    m = mn;
                }
                // P over S: keys 32c .. 32c+31 in columns 16c .. 16c+15 (remainders 64 columns on)
                auto weigh = [&](int c, const float (&x)[32]) {
                    uint32_t w[16], wl[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p0 = weight<false>(x[2 * i], qs, m), p1 = weight<false>(x[2 * i + 1], qs, m);
                        la += p0;
                        lb += p1;
                        w[i] = pack_h2(p0, p1);
                        if (F32) {
                            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                            wl[i] = pack_h2(p0 - h.x, p1 - h.y);
                        }
                    }
                    tmem_st16u(t_s + c * 16u, w);
                    if (F32) tmem_st16u(t_s + 64u + c * 16u, wl);
                };
                tmem_wait_ld();
                mask(0, u[0]);
                weigh(0, u[0]);
                tmem_ld32(t_s + 32u, u[1]);
                tmem_wait_ld();
                mask(1, u[1]);
                weigh(1, u[1]);
                weigh(2, v[0]);
                weigh(3, v[1]);
            } else {
                // Columns 64 * half on.  The weights are taken with the reference of the tiles
                // before, which holds as a rule; where a row's does not, or is beyond kFused, both
                // threads of every row of the warp pair begin again (P is not written yet).
                uint32_t w[32];
                auto weigh = [&](auto fused, int c, const float (&x)[32]) {
                    constexpr bool kF = decltype(fused)::value;
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p0 = weight<kF>(x[2 * i], qs, m), p1 = weight<kF>(x[2 * i + 1], qs, m);
                        la += p0;
                        lb += p1;
                        w[16 * c + i] = pack_h2(p0, p1);
                    }
                };
                const uint32_t t_h = t_s + 64u * half;
                bool raise = false;
                float top = 0.f;
                if (ok) {
                    float v[32], u[32];
                    tmem_ld32(t_h, v);
                    tmem_wait_ld();
                    tmem_ld32(t_h + 32u, u);
                    mask(2 * half, v);
                    top = top_of(v);
                    weigh(std::true_type(), 0, v);
                    tmem_wait_ld();
                    mask(2 * half + 1, u);
                    top = fmaxf(top, top_of(u)) * qs;
                    weigh(std::true_type(), 1, u);
                    raise = top - m > kRaise || (fabsf(m) > kFused && m != kNone);
                }
                const uint32_t pair = 1u + st * 4u + (warp & 3u);
                fence_before();
                if (pair_any(pair, raise || !ok)) {
                    fence_after();
                    top_sh[st][half][r] = top;
                    if (pair_any(pair, !ok)) {
                        ok = false;
                        break;
                    }
                    top = fmaxf(top, top_sh[st][half ^ 1u][r]);
                    raise = top - m > kRaise;
                    const float mn = raise ? top - kHead : m, alpha = fast_exp2(m - mn);
                    if (s > 0) {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            float o[32];
                            tmem_ld32(t_o + 64u * half + c * 32u, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] *= alpha;
                            tmem_st32(t_o + 64u * half + c * 32u, o);
                        }
                    }
                    l *= alpha;
                    m = mn;
                    la = lb = 0.f;
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float v[32];
                        tmem_ld32(t_h + c * 32u, v);
                        tmem_wait_ld();
                        mask(2 * half + c, v);
                        weigh(std::false_type(), c, v);
                    }
                    fence_before();
                    pair_any(pair, false);
                }
                fence_after();
#pragma unroll
                for (int c = 0; c < 2; c++) tmem_st16u(t_s + 32u * half + c * 16u, *reinterpret_cast<uint32_t(*)[16]>(&w[16 * c]));
            }
            l += la + lb;
            tmem_wait_st();
            fence_before();
            bar_arrive(bar(B_PFULL + st));
        }
        if (ok && n_steps > 0) ok = !abort_sh && wait_bar_warp(bar(B_ODONE + st), 0);
        if (!ok) abort_sh = 1;
        const bool took = F32 && n_steps > kTake;
        const float w_taken = fast_exp2(m_taken - m);
        const float *ob = reinterpret_cast<const float *>(gsm + T_K * kTile);  // stream 1's O, [128 columns][128 rows]
        float wA = 1.f;
        ml_sh[st][half][r] = make_float2(m, l);
        // Both streams' MMAs are done: the K and V tiles are free.  All go on, or none.
        ok = !soft_any(kSoft * 32u, abort_sh);
        fence_after();
        if (H == 2) l = ml_sh[st][0][r].y + ml_sh[st][H - 1][r].y;
        if (solo) {
            // Join the streams: stream 1 leaves its O, scaled, in the K tiles.
            float2 a = ml_sh[0][0][r], b = ml_sh[1][0][r];
            if (H == 2) {
                a.y += ml_sh[0][H - 1][r].y;
                b.y += ml_sh[1][H - 1][r].y;
            }
            m = fmaxf(a.x, b.x);
            wA = fast_exp2(a.x - m);
            const float wB = fast_exp2(b.x - m);
            l = a.y * wA + b.y * wB;
            if (st == 1 && nt > 1 && ok) {
#pragma unroll
                for (uint32_t k = 0; k < 4 / H; k++) {
                    const uint32_t c = half * (4 / H) + k;
                    float v[32];
                    read_o(c, took, w_taken, v);
#pragma unroll
                    for (int i = 0; i < 32; i++) const_cast<float *>(ob)[(c * 32u + i) * 128u + r] = v[i] * wB;
                }
            }
            soft_any(kSoft * 32u, false);
        }
        if (ok && (!solo || st == 0)) {
            // O goes through shared memory (16-byte chunk c of row r at c ^ (r & 31)), so that
            // the global stores are whole rows: stream 0 by the V tiles, stream 1 by the K tiles
            // (solo: stream 1's O is there until it is added).
            uint8_t *tile_sm = gsm + (st == 0 ? T_V : T_K) * kTile;
#pragma unroll
            for (uint32_t k = 0; k < 4 / H; k++) {
                const uint32_t c = half * (4 / H) + k;
                float v[32];
                read_o(c, took, w_taken, v);
                if (solo) {
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        v[i] *= wA;
                        if (nt > 1) v[i] += ob[(c * 32u + i) * 128u + r];
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < 8; i++)
                    *reinterpret_cast<float4 *>(tile_sm + r * 512u + (((c * 8u + i) ^ lane) << 4)) =
                        make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
            if (valid && half == 0) *reinterpret_cast<float2 *>(P.ml + row * 2u) = make_float2(m, l);
            if (took) asm volatile("bar.sync 10, 128;" ::: "memory");  // (the sums of all columns are read)
            // a warp stores its own 32 rows, two that share them half of them each
            if (H == 1) __syncwarp();
            else pair_any(1u + st * 4u + (warp & 3u), false);
            const uint32_t rows = min(T, Gr.n_seqs - mt * T) * G;  // of the tile's, those that hold a head
            const uint32_t r0 = (warp & 3u) * 32u + half * (32u / H);
            float *tile_out = P.part + (row - r) * 128u;
            uint32_t bad = 0;  // rows with an element that is not finite
#pragma unroll 8
            for (uint32_t x = r0; x < min(r0 + 32u / H, rows); x++) {
                const float4 y = *reinterpret_cast<const float4 *>(tile_sm + x * 512u + ((lane ^ (x & 31u)) << 4));
                *reinterpret_cast<float4 *>(tile_out + x * 128u + lane * 4u) = y;
                if (!all_finite(y)) bad |= 1u << (x - r0);
            }
            bad = __reduce_or_sync(0xffffffffu, bad);
            for (; bad; bad &= bad - 1u) {
                const uint32_t x = r0 + (uint32_t)__ffs((int)bad) - 1u, hl = x % G;
                const PrefixSeq sq = tab[Gr.seq0 + mt * T + x / G];
                const uint64_t at = (uint64_t)kvh * 128u;
                redo_row(reinterpret_cast<const char *>(sq.q) + (uint64_t)(kvh * G + hl) * (F32 ? 512u : 256u), !F32, Gr.k + at,
                         Gr.v + at, (uint64_t)P.kv_heads * 128u, max(sq.start, kbeg), kend, tile_out + x * 128u, P.ml + (row - r + x) * 2u);
            }
        }
    }
    fence_before();
    __syncthreads();
    if (abort_sh) {
        // The loads and MMAs in flight end before the shared memory and TMEM go, as far as
        // another bounded wait for each tells.
        if (loads) {
            const uint32_t ring = solo && !F32 ? 3u : 2u;
#pragma unroll 1
            for (uint32_t t = 0; t < ring && t < k_loads; t++) (void)wait_bar(bar(B_KFULL + t), ((k_loads - 1u - t) / ring) & 1u);
#pragma unroll 1
            for (uint32_t t = 0; t < 2u && t < v_loads; t++) (void)wait_bar(bar(B_VFULL + t), ((v_loads - 1u - t) / 2u) & 1u);
        }
        if (warp == kSoft && lane == 0) {
            commit(bar(B_DRAIN));
            (void)wait_bar(bar(B_DRAIN), 0);
        }
        __syncthreads();
        if (tid == 0) atomicExch(&g_prefix_error, 1);
    }
    fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ------------------------------------------------------------ planning
// Every CTA takes the same number of key tiles (splits of a group differ by
// its last).  More CTAs shorten this launch; fewer leave SMs to the launch that
// reads the sequences' own rows, which runs beside it.  The plan minimises the
// time of both by measured rates (us): a CTA's start and end, a key tile of two
// Q tiles or of one (bf16, f32), and the own rows at the rate of HBM or of the SMs left.
constexpr double kCtaUs = 15.0, kPairUs = 2.35, kSoloUs = 1.5, kSoloF32Us = 2.5;
constexpr double kHbmBytesUs = 5.8e6, kSmI8BytesUs = 4.6e4, kSmF16BytesUs = 7e4, kOwnUs = 12.0;

uint32_t prefix_plan(PrefixGroup *groups, uint32_t n, uint32_t q_heads, uint32_t kv_heads, bool f32, uint64_t own_rows,
                     bool own_i8) {
    const uint32_t T = prefix_seqs_per_tile(q_heads / kv_heads);
    const double own_bytes = (double)own_rows * kv_heads * (own_i8 ? 264.0 : 512.0);
    const double sm_bytes_us = own_i8 ? kSmI8BytesUs : kSmF16BytesUs;
    uint64_t units = 0, work = 0, most = 1, pairs = 0;
    bool pair = false;
    for (uint32_t i = 0; i < n; i++) {
        PrefixGroup &X = groups[i];
        X.m_tiles = (X.n_seqs + T - 1) / T;
        pair = pair || (!f32 && X.m_tiles > 1);
        const uint64_t ctas = (uint64_t)kv_heads * (f32 ? X.m_tiles : (X.m_tiles + 1) / 2);
        const uint64_t nt = (X.len - X.lo + 127) / 128;
        pairs += (uint64_t)X.n_seqs * kv_heads;
        units += ctas;
        work += ctas * nt;
        most = std::max(most, nt);
    }
    auto ctas_at = [&](uint64_t tps) {
        uint64_t c = 0;
        for (uint32_t i = 0; i < n; i++) {
            const PrefixGroup &X = groups[i];
            c += (uint64_t)kv_heads * (f32 ? X.m_tiles : (X.m_tiles + 1) / 2) * (((X.len - X.lo + 127) / 128 + tps - 1) / tps);
        }
        return c;
    };
    const double tile_us = f32 ? kSoloF32Us : pair ? kPairUs : kSoloUs;
    uint64_t best_tps = most;
    double best = 1e300;
    const uint64_t w0 = (units + kPlanSms - 1) / kPlanSms;
    for (uint64_t room = (w0 + 1) * kPlanSms; room >= units && room > 0;) {
        uint64_t tps = std::max<uint64_t>(1, (work + room - 1) / room);
        while (tps < most && ctas_at(tps) > room) tps += std::max<uint64_t>(1, tps / 32);
        tps = std::min(tps, most);
        const uint64_t c = ctas_at(tps), waves = (c + kPlanSms - 1) / kPlanSms;
        const double prefix_us = (double)waves * (kCtaUs + (double)tps * tile_us);
        // few pairs: wide CTAs, one an SM, which wait for this launch themselves
        const bool wide = pairs <= kPlanSms / 4;
        const uint64_t free_sms = waves == 1 ? kPlanSms - c : 0, slots = wide ? free_sms : 3 * free_sms;
        const double alone = kOwnUs + own_bytes / kHbmBytesUs;
        double beside = 1e300;
        if (free_sms && !(wide && pairs > slots)) {
            // more (sequence, KV head) pairs than CTAs run in whole waves of them
            const double uneven = pairs > slots ? (double)((pairs + slots - 1) / slots * slots) / (double)pairs : 1.0;
            beside = kOwnUs + std::max(own_bytes / kHbmBytesUs, uneven * own_bytes / ((double)free_sms * sm_bytes_us));
        }
        const double cost = std::min(prefix_us + alone, std::max(prefix_us, beside));
        if (cost < best) {
            best = cost;
            best_tps = tps;
        }
        // Next: a second wave's room, a full one, then eight SMs less each time.
        const uint64_t next = room > w0 * kPlanSms ? w0 * kPlanSms : room - 8;
        if (room <= 8 || c < room - 8) room = std::min(next, std::max<uint64_t>(c, 1) - 1);
        else room = next;
        if (w0 > 1 && room < w0 * kPlanSms) break;
    }
    uint64_t tiles = 0, ctas = 0;
    for (uint32_t i = 0; i < n; i++) {
        PrefixGroup &X = groups[i];
        X.tiles_per_split = (uint32_t)best_tps;
        X.splits = (uint32_t)(((X.len - X.lo + 127) / 128 + best_tps - 1) / best_tps);
        X.part0 = (uint32_t)tiles;
        tiles += (uint64_t)kv_heads * X.m_tiles * X.splits;
        ctas += (uint64_t)kv_heads * (f32 ? X.m_tiles : (X.m_tiles + 1) / 2) * X.splits;
    }
    return (uint32_t)ctas;
}

// CTAs stay within units + 2 * kPlanSms, and a CTA has at most two tiles: two Q
// tiles (units are KV heads x pairs of m tiles), or, in F32, one and its stream 1's sums.
uint64_t prefix_tiles_bound(uint64_t n_groups, uint64_t n_seqs, uint32_t q_heads, uint32_t kv_heads) {
    const uint64_t m_tiles = n_seqs / prefix_seqs_per_tile(q_heads / kv_heads) + n_groups;
    return (uint64_t)kv_heads * 2u * m_tiles + 4u * kPlanSms;
}

template <bool F32, int NS>
static int launch(const PrefixGroup *groups, uint32_t n, const PrefixSeq *seqs, uint32_t n_seqs, uint32_t q_heads,
                  uint32_t kv_heads, float *part, float *ml, PrefixSync *sync, cudaStream_t stream) {
    constexpr size_t smem = 6 * tc05::kTile + 1024;
    static bool ready[64];
    int dev = 0;
    if (int rc = check_cuda(cudaGetDevice(&dev), "prefix get device")) return rc;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (int rc = check_cuda(cudaFuncSetAttribute(prefix_tc05_kernel<F32, NS>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                "prefix shared memory"))
            return rc;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    PrefixParams<NS> P;
    uint32_t ctas = 0;
    for (uint32_t i = 0; i < n; i++) {
        const PrefixGroup &X = groups[i];
        PrefixDev &D = P.group[i];
        if (!tc05::make_map(&D.kmap, X.k, kv_heads * 128u, X.len) || !tc05::make_map(&D.vmap, X.v, kv_heads * 128u, X.len))
            return set_error(SF37KV_ECUDA, "prefix: tensor map encoding failed");
        D.k = (const __half *)X.k;
        D.v = (const __half *)X.v;
        D.lo = X.lo;
        D.len = X.len;
        D.seq0 = X.seq0;
        D.n_seqs = X.n_seqs;
        D.m_tiles = X.m_tiles;
        D.splits = X.splits;
        D.tps = X.tiles_per_split;
        D.part0 = X.part0;
        D.pairs = F32 ? X.m_tiles : (X.m_tiles + 1) / 2;
        D.cta0 = ctas;
        ctas += D.pairs * kv_heads * X.splits;
    }
    std::copy(seqs, seqs + n_seqs, P.seq);
    P.part = part;
    P.ml = ml;
    P.sync = sync;
    const PrefixGroup &last = groups[n - 1];
    P.take0 = last.part0 + kv_heads * last.m_tiles * last.splits;
    P.n_groups = n;
    P.heads_per_kv = q_heads / kv_heads;
    P.kv_heads = kv_heads;
    P.tpt = prefix_seqs_per_tile(P.heads_per_kv);
    g_launches++;
    return launch_early("prefix launch", prefix_tc05_kernel<F32, NS>, dim3(ctas), soft_warps(F32) * 32 + 64, smem, stream, P);
}

int prefix_attention(const PrefixGroup *groups, uint32_t n, const PrefixSeq *seqs, uint32_t n_seqs, uint32_t q_heads,
                     uint32_t kv_heads, bool f32, float *part, float *ml, PrefixSync *sync, cudaStream_t stream) {
    if (n_seqs <= 32)
        return f32 ? launch<true, 32>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, sync, stream)
                   : launch<false, 32>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, sync, stream);
    return f32 ? launch<true, kPrefixSeqs>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, sync, stream)
               : launch<false, kPrefixSeqs>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, sync, stream);
}

int prefix_device_error(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_prefix_error, sizeof(int)) != cudaSuccess) {
        (void)cudaGetLastError();
        return -1;
    }
    const int zero = 0;
    if (clear && v) (void)cudaMemcpyToSymbol(g_prefix_error, &zero, sizeof(int));
    return v;
}

}  // namespace sf37kv
