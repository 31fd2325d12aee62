// Batched decode over int8 caches and over shared prefixes: the kernel for a
// sequence's own rows, the merge, the split planning and the entry points.
// The attention over a shared prefix itself is in prefix_tc05.cu.
//
// For query head h of KV head h / G over rows r (log2 domain, base-2 exps):
//   s_r = (q[h] . K[r]) log2(e) / sqrt(128),  out = sum_r 2^(s_r - m) V[r] / l,
// one pass with a running reference m that is raised only when a score exceeds
// it by more than 8.  I8 rows enter as their integer codes: a key's scale
// multiplies its score, a value's scale its weight.  q . codes is a product of
// integers (q as three 8-bit digits, s8 x u8 tiles, exact in s32), so
// keys need no conversion; value codes become f16, exactly.
//
// One CTA serves one KV head of one sequence over a run of rows (a split), so
// each K/V byte is read once for all G query heads.  Its warps stream
// interleaved 16-row blocks through private rings of cp.async stages; S = qK^T
// and O += PV are mma.sync tiles on fragments that the lanes load straight from
// the stage.  The bytes bound it, not the products (tcgen05 would need 64 rows of
// queries or more): 16 rows of I8 are 4224 bytes and about 330 warp instructions,
// and an SM receives those bytes in 180 cycles, in which it can issue 720.  The
// CTAs of a (sequence, KV head) leave unnormalised partials; the last one to
// finish (an atomic counter) or join_kernel joins them, and the shared prefix's,
// in a fixed order, so results do not depend on which CTA is last.
//
// Measured (one B200, graph replay; of the measured copy rate): 48 layers x 32769
// rows of I8, 8 KV heads, f32: 520-560 us (0.91-0.98); 64 sequences of 1 to 8192
// rows, bf16: 96 us (0.89); one of 131072: 47 us (0.90); 128 windows of 512 rows,
// 96 query heads: 42 us (0.50: a CTA's start and end are as long as its 512
// rows); one of 2049: 9.2 us.  Under seconds of load the card's power cap lowers the
// SMs to 1.55 GHz, and the 48 layers take 660 us (bf16 queries: 648), 64 sequences
// 112: the integer and f16 tiles then bound it.
//
// Sixteen M rows of a tile hold, by MODE:
//   kPair  G <= 8, f32: eight heads twice, f16 "hi" and remainder "lo" of the weights
//          (and of an f16 path's q), 22 bits at no extra cost;
//   kHalf  G <= 8, bf16: the same without sums of their own (kTake);
//   kWide  G <= 16 and bf16: sixteen heads, weights rounded to f16 (half a step is
//          2^-11 of a weight; the output's own rounding has 2^-8);
//   kTwo   G <= 16 and f32: two kPair tiles on the same K/V fragments.
// I8 takes q in three 8-bit digits throughout, off by at most 2^-22 of the head's
// largest power of two.  Two digits (2^-14 of it) would be 7% faster with bf16 (64
// sequences of 1 to 8192 rows 98.5 us against 105.8, one of 131072 48.0 against 52.7),
// but a channel of 100 times the rest then puts the output off by more than its rounding.
#include <algorithm>
#include <climits>
#include <cstring>

#include "batch_internal.cuh"

namespace sf37kv {

extern unsigned long long g_launches;

enum { kPair = 0, kHalf = 1, kWide = 2, kTwo = 3 };

constexpr float kSlack = 8.0f;
constexpr float kNone = -3.402823466e38f;  // reference of a state without rows: no finite score is below it
// The tensor core truncates its f32 sums: O loses 1.7e-8 of itself with each block
// (measured), 9e-6 over 512 of them.  f32 outputs take O into sums of their own
// after this many.
constexpr uint32_t kTake = 32;
constexpr uint64_t kCounters = 16384;  // u32 counters at the start of a workspace
constexpr uint32_t kSmallSeqs = 16, kSomeSeqs = 64, kMaxSeqs = 256;  // sequences per launch
constexpr uint32_t kMapped = 1024;     // slots with a direct map to their sequence
// Range of the weights' power of two (kernel below): value scales from 2^-113 to 2^121, the largest.
constexpr int kFMin = -114, kFMax = 120;

struct SeqDev {
    const void *k, *v, *q;
    const float *gate;
    void *out;
    const void *k_new, *v_new;
    uint32_t start, end, cap;            // own rows [start, end)
    uint32_t split_rows, n_splits, slot;  // its splits are slots slot, slot + 1, ...
    // partials of the shared prefix: tile pre_tile + kvh * pre_kvh + split, row pre_row on
    uint32_t pre_tile, pre_kvh, pre_splits, pre_row;
};
__host__ __device__ constexpr uint32_t part_stride(uint32_t g) { return g * 128u + ((2u * g + 3u) & ~3u); }

template <int NJ>
struct BatchParams {
    uint8_t seq_of[kMapped];  // sequence of a slot; CTA = slot * kv_heads + KV head
    SeqDev seq[NJ];
    uint32_t n, slots, group, kv_heads, bf16;
    uint32_t after_prefix, join;  // sequences with a prefix are joined by join_kernel
    float *part;          // [cta][part_stride(G)]: O [G][128], then (m, l) [G]
    uint32_t *counters;   // [sequence][kv head]
    PrefixSync *sync;
    const float *pre_part, *pre_ml;
};

// ------------------------------------------------------------ device helpers
namespace bd {

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(int (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {  // s8 x u8
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
    return r;
}
__device__ __forceinline__ float2 lds64f(uint32_t addr) {
    float2 r;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(addr));
    return r;
}
__device__ __forceinline__ uint32_t word(const uint4 &u, int w) {
    return w == 0 ? u.x : w == 1 ? u.y : w == 2 ? u.z : u.w;
}
// Two bytes u (in the low and high half's low byte of an 0x64uu pair) to f16
// u - 128: 0x6400 + u is the f16 1024 + u, and 1152 is subtracted exactly.
__device__ __forceinline__ uint32_t unbias(uint32_t h) {
    const uint32_t bias = 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), *reinterpret_cast<const __half2 *>(&bias));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return unbias(prmt(w, 0x64646464u, 0x4140u)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return unbias(prmt(w, 0x64646464u, 0x4342u)); }

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint64_t pol) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(pol) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 2^-e for a positive f32 x in [2^e, 2^(e+1)), e clamped to [-126, 126].
__device__ __forceinline__ float pow2_below(float x, int &e) {
    e = (int)((__float_as_uint(x) >> 23) & 255u) - 127;
    e = max(-126, min(126, e));
    return __int_as_float((127 - e) << 23);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }

// Float index of dimension d of row `row` in the merge buffer: 16-byte chunks
// permuted so that the fragment stores spread over the banks and float4 reads
// stay whole.
__device__ __forceinline__ uint32_t os_at(uint32_t row, uint32_t d) {
    const uint32_t c = d >> 2;
    return row * 128u + ((c ^ (row & 7u) ^ ((c >> 3) & 3u)) << 2) + (d & 3u);
}
__device__ __forceinline__ void store_out4(void *out, uint64_t i, float4 x, bool bf16) {
    if (!bf16) {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(out) + i) = x;
        return;
    }
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    uint2 w;
    w.x = *reinterpret_cast<const uint32_t *>(&a);
    w.y = *reinterpret_cast<const uint32_t *>(&b);
    *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(out) + i) = w;
}
// (a, l) += (x, lx) * w
__device__ __forceinline__ void fold(float4 &a, float &l, const float4 &x, float lx, float w) {
    a.x = fmaf(x.x, w, a.x);
    a.y = fmaf(x.y, w, a.y);
    a.z = fmaf(x.z, w, a.z);
    a.w = fmaf(x.w, w, a.w);
    l = fmaf(lx, w, l);
}
// Of a head with the sum l of its weights; a sequence without rows gets zeros, one
// whose scores are all -inf NaN (0 / 0).
__device__ __forceinline__ float4 normalise(float4 a, float l, float g, bool no_rows) {
    if (no_rows) return make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(a.x / l * g, a.y / l * g, a.z / l * g, a.w / l * g);
}

// One float4 (index idx of [G][128], head h) of the partials of a (sequence, KV
// head): n_own of its own, `step` floats apart, then n_pre of the prefix's, a 128-row tile
// apart, always in this order.  Eight partials' values and (m, l) pairs are loaded at once:
// a trip to L2 for each eight, and no barrier.
struct Joined {
    float4 o;
    float l;
};
__device__ __forceinline__ Joined join_one(const float *own, uint64_t step, uint32_t n_own, const float *pre,
                                           const float *pre_ml, uint64_t row, uint32_t n_pre, uint32_t G, uint32_t h,
                                           uint32_t idx) {
    Joined r;
    r.o = make_float4(0.f, 0.f, 0.f, 0.f);
    r.l = 0.f;
    float M = kNone;
    const uint32_t n = n_own + n_pre;
    for (uint32_t s = 0; s < n; s += 8u) {
        float4 x[8];
        float2 ml[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t k = s + i;
            ml[i] = make_float2(-INFINITY, 0.f);
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < n) {
                const bool mine = k < n_own;
                const float *po = mine ? own + k * step : pre + (row + (uint64_t)(k - n_own) * 128u) * 128u;
                const float *pm = mine ? po + G * 128u : pre_ml + (row + (uint64_t)(k - n_own) * 128u) * 2u;
                x[i] = __ldcg(reinterpret_cast<const float4 *>(po) + idx);
                ml[i] = __ldcg(reinterpret_cast<const float2 *>(pm) + h);
            }
        }
        float mn = M;
#pragma unroll
        for (int i = 0; i < 8; i++) mn = fmaxf(mn, ml[i].x);
        const float sc = fast_exp2(M - mn);
        M = mn;
        r.l *= sc;
        r.o = make_float4(r.o.x * sc, r.o.y * sc, r.o.z * sc, r.o.w * sc);
#pragma unroll
        for (int i = 0; i < 8; i++) fold(r.o, r.l, x[i], ml[i].y, fast_exp2(ml[i].x - mn));
    }
    return r;
}

}  // namespace bd

// ------------------------------------------------------------ the stage
// One stage: 16 rows of K, 16 of V (I8: then 16 + 16 scales).  16-byte chunk ch
// of row r sits at ch ^ k_swz(r) (K) or ch ^ v_swz(r) (V), which keeps the
// eight lanes of a load phase on distinct banks:
//   K: lane (g, t) reads row g (+8), chunk t + 4c; V: rows 2t + {0,1,8,9}, chunk g (+8).
template <bool I8>
struct Stage {
    static constexpr uint32_t kRow = I8 ? 128 : 256;
    static constexpr uint32_t kV = 16 * kRow;
    static constexpr uint32_t kScales = 32 * kRow;
    static constexpr uint32_t kBytes = 32 * kRow + (I8 ? 128 : 0);
    static __device__ __forceinline__ uint32_t k_swz(uint32_t r) {
        return I8 ? (r & 1u) << 2 : ((r & 1u) << 2) ^ (((r >> 1) & 3u) << 1);
    }
    static __device__ __forceinline__ uint32_t v_swz(uint32_t r) {
        return I8 ? ((r >> 1) & 3u) << 1 : ((r & 1u) << 2) ^ (((r >> 1) & 3u) << 1);
    }
    // Dimension of element e (0..3) that lane t holds in k-step kk: the order
    // inside a head is permuted so that the loaded words are the fragments.
    static __device__ __forceinline__ uint32_t k_dim(uint32_t kk, uint32_t t, uint32_t e) {
        if (I8) return 64u * (kk >> 2) + 16u * t + 4u * (kk & 3u) + e;
        const uint32_t w = 2u * kk + (e >> 1);
        return (4u * (w >> 2) + t) * 8u + 2u * (w & 3u) + (e & 1u);
    }
    // Dimension of column c (0..7) of output tile jt.
    static __device__ __forceinline__ uint32_t v_dim(uint32_t jt, uint32_t c) {
        return I8 ? 16u * c + jt : jt < 8 ? 8u * c + jt : 64u + 8u * c + jt - 8u;
    }
};

// Warps of a CTA, CTAs of an SM and stages of a warp.  An SM runs 12 warps (8 in
// kTwo, for their registers, and with f32 outputs over f16 caches, for the sums'
// memory), either as CTAs of four, which hide each other's starts and ends, or
// as one wide CTA, which leaves fewer partials to join.
// More stages only lengthen the queue to HBM, and with it every other access:
// 8 layers x 32769 rows of I8 took 95 us with three stages, 100 with four, 102
// with two; f16 rows 76 us with two stages of 12 warps, 80 with three of 8.
template <int MODE, bool I8, bool WIDE>
struct Shape {
    static constexpr int kSmWarps = MODE == kTwo || (MODE == kPair && !I8) ? 8 : 12;
    static constexpr int kWarps = WIDE ? kSmWarps : 4;
    static constexpr int kThreads = kWarps * 32;
    static constexpr int kCtas = kSmWarps / kWarps;
    static constexpr int kStages = !I8 ? 2 : MODE == kTwo ? 4 : 3;
    static constexpr uint32_t kUnit = kWarps * 16;  // rows that the warps take at once
    static constexpr uint32_t kArea = kWarps * kStages * Stage<I8>::kBytes;
    // q: an I8 q in kDigits digits of 8 bits, eight rows (a group) each, two groups a
    // tile of 16 rows; an f16 q in tiles of the weights' layout
    static constexpr int kDigits = 3;
    static constexpr int kGroups = kDigits * (MODE == kWide || MODE == kTwo ? 2 : 1);
    static constexpr int kQTiles = I8 ? (kGroups + 1) / 2 : MODE == kTwo ? 2 : 1;
    static constexpr uint32_t kQArea = (8 * 32 * 16) * (!I8 && MODE == kTwo ? 2 : I8 && kQTiles > 2 ? 2 : 1);
    // f32 outputs: sums of O out of the tensor core's accumulators, one float a lane each
    static constexpr int kSums = MODE == kPair ? 32 : MODE == kTwo ? 64 : 0;
    static constexpr uint32_t kSmem = kArea + kQArea + kWarps * kSums * 32 * 4;
    static_assert(kCtas * (kSmem + 2048) <= 228 * 1024, "CTAs of an SM");
};

template <int MODE, bool I8, bool WIDE, int NJ>
__global__ void __launch_bounds__(Shape<MODE, I8, WIDE>::kThreads, Shape<MODE, I8, WIDE>::kCtas)
    batch_decode_kernel(const __grid_constant__ BatchParams<NJ> P) {
    using namespace bd;
    using St = Stage<I8>;
    using Sh = Shape<MODE, I8, WIDE>;
    constexpr int NT = MODE == kTwo ? 2 : 1;   // M tiles
    constexpr int NH = MODE == kWide || MODE == kTwo ? 2 : 1;  // heads of a lane
    constexpr int ND = Sh::kDigits, NQ = Sh::kQTiles;
    constexpr int S = Sh::kStages, kWarps = Sh::kWarps, kThreads = Sh::kThreads;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float qfac[16], gate_s[16];
    __shared__ int qoff[2 * NQ][8];  // I8: -128 times the sum of a group's row
    __shared__ uint32_t s_last;

    // Launched early (programmatic dependent launch), the CTAs wait here for the
    // kernel before, whatever it was; after a prefix launch, which has itself waited
    // and writes partials only, they may read caches and q once its flag tells that.
    if (P.after_prefix) after_published(P.sync);
    else asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t slot_id = blockIdx.x / P.kv_heads, kvh = blockIdx.x - slot_id * P.kv_heads;
    uint32_t lo = 0;
    if (P.slots <= kMapped) {
        lo = P.seq_of[slot_id];
    } else {
        for (uint32_t hi = P.n; hi - lo > 1;) {
            const uint32_t mid = (lo + hi) >> 1;
            if (P.seq[mid].slot <= slot_id) lo = mid;
            else hi = mid;
        }
    }
    const SeqDev &J = P.seq[lo];
    const uint32_t G = P.group, split = slot_id - J.slot;
    const uint32_t row0 = J.start + split * J.split_rows;
    const uint32_t row1 = min(row0 + J.split_rows, J.end);
    const uint64_t row_bytes = (uint64_t)P.kv_heads * St::kRow;
    const uint8_t *kbase = reinterpret_cast<const uint8_t *>(J.k), *vbase = reinterpret_cast<const uint8_t *>(J.v);
    const float *sbase = reinterpret_cast<const float *>((lane < 16 ? kbase : vbase) + row_bytes * J.cap) +
                         (uint64_t)kvh * J.cap;
    const uint32_t wbuf = (uint32_t)__cvta_generic_to_shared(smem) + warp * S * St::kBytes;
    uint4 *Qs = reinterpret_cast<uint4 *>(smem + Sh::kArea);  // [tile][kk][lane]

    const uint32_t b_first = row0 + warp * 16u;
    constexpr uint32_t kStep = Sh::kUnit;
    const uint32_t nblk = b_first < row1 ? (row1 - b_first + kStep - 1) / kStep : 0u;
    uint64_t pol;  // a step reads more than L2 holds: the stream is marked to leave first
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    // Lane's part of a block: 16-byte chunk c_ch of rows c_row + kRows * i.
    constexpr uint32_t kCh = St::kRow / 16, kRows = 32 / kCh;
    const uint32_t c_ch = lane % kCh, c_row = lane / kCh;
    const uint64_t lane_off = c_row * row_bytes + kvh * St::kRow + c_ch * 16u;
    uint32_t slot_next = b_first % J.cap;  // slot of the next block to issue
    auto issue = [&](uint32_t it) {
        if (it < nblk) {
            const uint32_t bb = b_first + it * kStep, sb = slot_next, st = wbuf + (it % S) * St::kBytes;
            slot_next += kStep;
            if (slot_next >= J.cap) slot_next = slot_next - J.cap < J.cap ? slot_next - J.cap : slot_next % J.cap;
            if (sb + 16u <= J.cap && bb + 16u <= row1) {  // 16 rows side by side
                const uint8_t *kp = kbase + sb * row_bytes + lane_off, *vp = vbase + sb * row_bytes + lane_off;
#pragma unroll
                for (uint32_t i = 0; i < kCh / 2; i++) {
                    const uint32_t r = c_row + kRows * i;
                    cp16(st + r * St::kRow + ((c_ch ^ St::k_swz(r)) << 4), kp, pol);
                    cp16(st + St::kV + r * St::kRow + ((c_ch ^ St::v_swz(r)) << 4), vp, pol);
                    kp += kRows * row_bytes;
                    vp += kRows * row_bytes;
                }
                if (I8) cp4(st + St::kScales + lane * 4u, sbase + sb + (lane & 15u));
            } else {
                // the ring's end or the last rows: past row1 a row that is read anyway, masked below
                auto slot_of = [&](uint32_t r) {
                    uint32_t slot = sb + r;
                    if (slot >= J.cap) slot %= J.cap;
                    return bb + r < row1 ? slot : sb;
                };
#pragma unroll
                for (uint32_t i = 0; i < kCh / 2; i++) {
                    const uint32_t r = c_row + kRows * i;
                    const uint64_t go = slot_of(r) * row_bytes + kvh * St::kRow + c_ch * 16u;
                    cp16(st + r * St::kRow + ((c_ch ^ St::k_swz(r)) << 4), kbase + go, pol);
                    cp16(st + St::kV + r * St::kRow + ((c_ch ^ St::v_swz(r)) << 4), vbase + go, pol);
                }
                if (I8) cp4(st + St::kScales + lane * 4u, sbase + slot_of(lane & 15u));
            }
        }
        cp_commit();
    };
    // q is asked for before the stream, so that it does not queue behind it.
    float4 qx[8];
    if (warp < NH) {
        const uint64_t at = (uint64_t)(kvh * G + min(warp * 8u + g, G - 1u)) * 128u;
#pragma unroll
        for (uint32_t kk = 0; kk < 8; kk++) qx[kk] = load_row4(J.q, at + St::k_dim(kk, t, 0), P.bf16);
    }
    const float gate = tid < G && J.gate ? J.gate[kvh * G + tid] : 0.f;
    // The CTA that covers the last row stores the appended one first, K and V by its
    // last two warps.  A warp whose first stages hold that row starts to load after it.
    const bool appends = J.k_new && row0 < row1 && row1 == J.end;
    const bool late = appends && b_first < row1 && (J.end - 1u - b_first) % kStep < 16u &&
                      (J.end - 1u - b_first) / kStep < S - 1;
    if (!late) {
#pragma unroll
        for (int s = 0; s < S - 1; s++) issue(s);
    }
    if (appends && warp >= kWarps - 2) {
        const bool value = warp == kWarps - 1;
        uint8_t *cache = const_cast<uint8_t *>(value ? vbase : kbase);
        const float4 x = load_row4(value ? J.v_new : J.k_new, kvh * 128u + lane * 4u, P.bf16);
        const uint32_t slot = (J.end - 1u) % J.cap;
        if (I8) {
            store_i8_head(cache, J.cap, P.kv_heads, kvh, slot, lane, x);
        } else {
            uint2 w;
            w.x = h2_bits(x.x, x.y);
            w.y = h2_bits(x.z, x.w);
            *reinterpret_cast<uint2 *>(cache + slot * row_bytes + kvh * 256u + lane * 8u) = w;
        }
    }

    // q, scaled by a power of two for each head so that its largest element is in
    // [1, 2): as f16 (a bf16 q exactly, an f32 one in two parts), or, for I8, as
    // integers q * 2^21 in signed digits of 8 bits.
    if (warp < NH) {
        const uint32_t h = warp * 8u + g;
        float top = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; kk++) {
            const float x[4] = {qx[kk].x, qx[kk].y, qx[kk].z, qx[kk].w};
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(x[e]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e2;
        const float f = pow2_below(top, e2);
        constexpr int kBits = 21;
        if (t == 0) qfac[h] = pow2(e2) * (1.4426950408889634f * 0.08838834764831845f) * (I8 ? 1.f / (1 << kBits) : 1.f);
        uint32_t *Q32 = reinterpret_cast<uint32_t *>(Qs);
        if (I8) {
            bool finite = true;
            int sum[ND];
#pragma unroll
            for (int d = 0; d < ND; d++) sum[d] = 0;
#pragma unroll
            for (int kk = 0; kk < 8; kk++) {  // four dimensions: register kk & 1 of half a of step kk / 2
                uint32_t w[ND];
#pragma unroll
                for (int d = 0; d < ND; d++) w[d] = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = (e == 0 ? qx[kk].x : e == 1 ? qx[kk].y : e == 2 ? qx[kk].z : qx[kk].w) * f;
                    finite = finite && fabsf(x) < 2.f;
                    // bytes of v + 0x80..80 are the digits of v plus 128
                    const uint32_t v = (uint32_t)(__float2int_rn(x * (float)(1 << kBits)) + 0x808080);
#pragma unroll
                    for (int d = 0; d < ND; d++) {  // digit 0 is the highest
                        const uint32_t byte = (v >> (8 * (ND - 1 - d))) & 255u;
                        sum[d] += (int)byte - 128;
                        w[d] |= (byte ^ 128u) << (8 * e);
                    }
                }
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const int grp = (int)warp * ND + d;
                    Q32[(((grp >> 1) * 4 + (kk >> 1)) * 32 + lane) * 4 + (grp & 1) + 2 * (kk & 1)] = w[d];
                }
                if (Sh::kGroups & 1) Q32[(((Sh::kGroups >> 1) * 4 + (kk >> 1)) * 32 + lane) * 4 + 1 + 2 * (kk & 1)] = 0;
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                sum[d] += __shfl_xor_sync(0xffffffffu, sum[d], 1);
                sum[d] += __shfl_xor_sync(0xffffffffu, sum[d], 2);
                if (t == 0) qoff[warp * ND + d][g] = -128 * sum[d];
            }
            if ((Sh::kGroups & 1) && t == 0) qoff[Sh::kGroups][g] = 0;
            __syncwarp();
            // a q that is not finite has no digits: its scores are NaN
            if (!finite) qfac[h] = __int_as_float(0x7fc00000);
        } else {
#pragma unroll
            for (int kk = 0; kk < 8; kk++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const float x0 = (half ? qx[kk].z : qx[kk].x) * f, x1 = (half ? qx[kk].w : qx[kk].y) * f;
                    const __half2 hv = __floats2half2_rn(x0, x1);
                    const float2 hf = __half22float2(hv);
                    const uint32_t hi = *reinterpret_cast<const uint32_t *>(&hv), lo = h2_bits(x0 - hf.x, x1 - hf.y);
                    if (MODE == kWide) {
                        Q32[(kk * 32 + lane) * 4 + 2 * half + warp] = hi;
                    } else {
                        Q32[((warp * 8 + kk) * 32 + lane) * 4 + 2 * half] = hi;
                        Q32[((warp * 8 + kk) * 32 + lane) * 4 + 2 * half + 1] = lo;
                    }
                }
        }
    }
    if (tid < 16) gate_s[tid] = J.gate ? sigmoid_dev(gate) : 1.f;
    __syncthreads();
    if (late) {
#pragma unroll
        for (int s = 0; s < S - 1; s++) issue(s);
    }
    float qf[NH];
#pragma unroll
    for (int h = 0; h < NH; h++) qf[h] = qfac[g + 8u * h];
    const uint32_t qaddr = (uint32_t)__cvta_generic_to_shared(Qs + lane);
    int q0[2 * NQ];
#pragma unroll
    for (int x = 0; x < 2 * NQ; x++) q0[x] = I8 ? qoff[x][g] : 0;

    float o[NT][16][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    // Per head: reference m, sum l, and f, a power of two that brings the
    // weights p * (value scale) into f16's range: the largest is kept in
    // [2^7, 2^15], so weights down to 2^-32 of it are held.  When m rises, f does at most
    // by what the weights so far lose (8 bits or more, rounded up to a whole one), so O
    // gains less than a bit for each 8 of f's 234, and its largest weights stay in range.
    float m[NH], l[NH], f[NH];
#pragma unroll
    for (int h = 0; h < NH; h++) {
        m[h] = kNone;
        l[h] = 0.f;
        f[h] = I8 ? pow2(kFMax) : 128.f;
    }

    // f32 outputs: this lane's sums of O (the two parts of a weight joined)
    float *sums = reinterpret_cast<float *>(smem + Sh::kArea + Sh::kQArea) + warp * (Sh::kSums * 32) + lane;
    bool taken = false;
    auto take = [&]() {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 16; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float *x = sums + ((n * 16 + i) * 2 + e) * 32;
                    *x = (taken ? *x : 0.f) + (o[n][i][e] + o[n][i][e + 2]);
                    o[n][i][e] = o[n][i][e + 2] = 0.f;
                }
        taken = true;
    };

    for (uint32_t it = 0; it < nblk; it++) {
        if (Sh::kSums && it > 0 && it % kTake == 0) take();
        cp_wait<S - 2>();
        __syncwarp();
        issue(it + S - 1);
        const uint32_t b = b_first + it * kStep, st = wbuf + (it % S) * St::kBytes;

        // scores of the lane's keys 8i + 2t + e, and the scales of the same values
        float sc[NH][2][2], vs[2][2], ks[2][2];
        if (I8) {
            int s[NQ][2][4];
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[n][i][e] = q0[2 * n + (e >> 1)];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint4 u[2];
#pragma unroll
                for (uint32_t i = 0; i < 2; i++) {
                    const uint32_t r = 8u * i + g;
                    u[i] = lds128(st + r * St::kRow + (((4u * c + t) ^ St::k_swz(r)) << 4));
                }
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    const uint4 a0 = lds128(qaddr + (n * 4 + 2 * c) * 512), a1 = lds128(qaddr + (n * 4 + 2 * c + 1) * 512);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        mma(s[n][i], a0, u[i].x, u[i].y);
                        mma(s[n][i], a1, u[i].z, u[i].w);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float2 k2 = lds64f(st + St::kScales + (8u * i + 2u * t) * 4u);
                const float2 v2 = lds64f(st + St::kScales + 64u + (8u * i + 2u * t) * 4u);
                ks[i][0] = k2.x;
                ks[i][1] = k2.y;
                vs[i][0] = v2.x;
                vs[i][1] = v2.y;
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int h = 0; h < NH; h++) {
                        auto digit = [&](int d) { return s[(h * ND + d) >> 1][i][e + 2 * ((h * ND + d) & 1)]; };
                        // two digits: below 2^31; the third: two f32 roundings of the sum
                        sc[h][i][e] = fmaf((float)(digit(0) * 256 + digit(1)), 256.f, (float)digit(2));
                    }
            }
        } else {
            float s[NT][2][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) s[n][i][0] = s[n][i][1] = s[n][i][2] = s[n][i][3] = 0.f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint4 u[2];
#pragma unroll
                for (uint32_t i = 0; i < 2; i++) {
                    const uint32_t r = 8u * i + g;
                    u[i] = lds128(st + r * St::kRow + (((4u * c + t) ^ St::k_swz(r)) << 4));
                }
#pragma unroll
                for (int w = 0; w < 2; w++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint4 q4 = lds128(qaddr + (n * 8 + 2 * c + w) * 512);
                        const uint32_t a[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
                        for (int i = 0; i < 2; i++) mma(s[n][i], a, word(u[i], 2 * w), word(u[i], 2 * w + 1));
                    }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    ks[i][e] = vs[i][e] = 1.f;
#pragma unroll
                    for (int h = 0; h < NH; h++)
                        sc[h][i][e] = MODE == kWide ? s[0][i][e + 2 * h] : s[h % NT][i][e] + s[h % NT][i][e + 2];
                }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int h = 0; h < NH; h++) sc[h][i][e] *= I8 ? qf[h] * ks[i][e] : qf[h];
        if (b + 16u > row1) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (b + 8u * i + 2u * t + e >= row1) {
                        vs[i][e] = 0.f;
#pragma unroll
                        for (int h = 0; h < NH; h++) sc[h][i][e] = -INFINITY;
                    }
        }
        float p[NH][2][2], w[NH][2][2];
        bool need[NH];
        auto weigh = [&](int h) {
            float xm = -INFINITY, wm = 0.f;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float x = sc[h][i][e] - m[h];
                    xm = fmaxf(xm, x);
                    p[h][i][e] = fast_exp2(x);
                    w[h][i][e] = I8 ? p[h][i][e] * vs[i][e] * f[h] : p[h][i][e] * f[h];  // (vs * f may overflow where p is 0)
                    wm = fmaxf(wm, w[h][i][e]);
                }
            need[h] = xm > kSlack || (I8 && wm > 32768.f);
        };
        bool any = false;
#pragma unroll
        for (int h = 0; h < NH; h++) {
            weigh(h);
            any |= need[h];
        }
        if (__any_sync(0xffffffffu, any)) {
            float fac[NH];
#pragma unroll
            for (int h = 0; h < NH; h++) {
                uint32_t nd = need[h];
                nd |= __shfl_xor_sync(0xffffffffu, nd, 1);
                nd |= __shfl_xor_sync(0xffffffffu, nd, 2);
                float mx = fmaxf(fmaxf(sc[h][0][0], sc[h][0][1]), fmaxf(sc[h][1][0], sc[h][1][1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = nd ? fmaxf(m[h], mx) : m[h];
                const float m_old = m[h];
                fac[h] = fast_exp2(m_old - mn);
                l[h] *= fac[h];
                m[h] = mn;
                if (I8) {
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int e = 0; e < 2; e++) top = fmaxf(top, fast_exp2(sc[h][i][e] - mn) * vs[i][e]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    int top_e, f_e;
                    pow2_below(top, top_e);
                    pow2_below(f[h], f_e);
                    const int grow = (int)ceilf(fminf(mn - m_old, 256.f));  // powers of two that the weights so far lose
                    const int fe = nd ? max(kFMin, min(min(kFMax, 7 - top_e), f_e + grow)) : f_e;
                    fac[h] *= pow2(max(-126, min(126, fe - f_e)));
                    f[h] = pow2(fe);
                }
                weigh(h);
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 16; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][i][e] *= MODE == kWide ? fac[(e >> 1) % NH] : fac[n % NH];
            if (Sh::kSums && taken)
#pragma unroll 4
                for (int x = 0; x < Sh::kSums; x++) sums[x * 32] *= fac[(x >> 5) % NH];
        }
        uint32_t pa[NT][4];
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                l[h] += p[h][i][0] + p[h][i][1];
                const __half2 hv = __floats2half2_rn(w[h][i][0], w[h][i][1]);
                const uint32_t hb = *reinterpret_cast<const uint32_t *>(&hv);
                if (MODE == kWide) {
                    pa[0][2 * i + h] = hb;
                } else {
                    const float2 b2 = __half22float2(hv);
                    pa[h % NT][2 * i] = hb;
                    pa[h % NT][2 * i + 1] = h2_bits(w[h][i][0] - b2.x, w[h][i][1] - b2.y);
                }
            }

        // O += P V: rows 2t, 2t+1 (B register 0) and 2t+8, 2t+9 (B register 1)
        const uint32_t vt = st + St::kV;
        if (I8) {
            uint4 v[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const uint32_t r = 2u * t + (x & 1) + (x >> 1) * 8u;
                v[x] = lds128(vt + r * St::kRow + ((g ^ St::v_swz(r)) << 4));
            }
#pragma unroll
            for (int wd = 0; wd < 4; wd++) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const uint32_t sel = hf ? 0x7362u : 0x5140u;  // {a2,b2,a3,b3} or {a0,b0,a1,b1}
                    const uint32_t x = prmt(word(v[0], wd), word(v[1], wd), sel);
                    const uint32_t y = prmt(word(v[2], wd), word(v[3], wd), sel);
                    const uint32_t x0 = codes_lo(x), x1 = codes_hi(x), y0 = codes_lo(y), y1 = codes_hi(y);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        mma(o[n][4 * wd + 2 * hf], pa[n], x0, y0);
                        mma(o[n][4 * wd + 2 * hf + 1], pa[n], x1, y1);
                    }
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint4 v[4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const uint32_t r = 2u * t + (x & 1) + (x >> 1) * 8u;
                    v[x] = lds128(vt + r * St::kRow + (((g + 8u * u) ^ St::v_swz(r)) << 4));
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
                    const uint32_t b0 = prmt(word(v[0], e >> 1), word(v[1], e >> 1), sel);
                    const uint32_t b1 = prmt(word(v[2], e >> 1), word(v[3], e >> 1), sel);
#pragma unroll
                    for (int n = 0; n < NT; n++) mma(o[n][8 * u + e], pa[n], b0, b1);
                }
            }
        }
        __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();  // the stages become the merge buffer
    if (P.after_prefix && tid == 0) leave_published(P.sync);

    // ---- the warps' states to one ----
    float *Os = reinterpret_cast<float *>(smem);  // [warp*16 + head][128]
    float2 *MLs = reinterpret_cast<float2 *>(Os + kWarps * 16 * 128);  // [warp*16 + head] (m, l)
#pragma unroll
    for (int h = 0; h < NH; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const uint32_t row = warp * 16u + g + 8u * h;
        const float inv = 1.f / f[h];
#pragma unroll
        for (uint32_t jt = 0; jt < 16; jt++)
#pragma unroll
            for (uint32_t e = 0; e < 2; e++) {
                float x = MODE == kWide ? o[0][jt][e + 2 * h] : o[h % NT][jt][e] + o[h % NT][jt][e + 2];
                if (Sh::kSums && taken) x += sums[((h % NT) * 32 + jt * 2 + e) * 32];
                Os[os_at(row, St::v_dim(jt, 2u * t + e))] = x * inv;
            }
        if (t == 0) MLs[row] = make_float2(m[h], l[h]);
    }
    __syncthreads();
    const bool single = J.n_splits == 1 && J.pre_splits == 0;
    const uint32_t stride = part_stride(G);
    float *part = P.part + (uint64_t)blockIdx.x * stride;
    const uint64_t out0 = (uint64_t)kvh * G * 128u;
    for (uint32_t idx = tid; idx < G * 32u; idx += kThreads) {
        const uint32_t h = idx >> 5, d4 = (idx & 31u) * 4u;
        float M = kNone, L = 0.f;
#pragma unroll
        for (int s = 0; s < kWarps; s++) M = fmaxf(M, MLs[s * 16 + h].x);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < kWarps; s++) {
            const float2 ml = MLs[s * 16 + h];
            fold(a, L, *reinterpret_cast<const float4 *>(Os + os_at(s * 16u + h, d4)), ml.y, fast_exp2(ml.x - M));
        }
        if (single) store_out4(J.out, out0 + idx * 4u, normalise(a, L, gate_s[h], J.start == J.end), P.bf16);
        else __stcg(reinterpret_cast<float4 *>(part + idx * 4u), a);
        if (!single && (idx & 31u) == 0) __stcg(reinterpret_cast<float2 *>(part + G * 128u + 2u * h), make_float2(M, L));
    }
    // A shared prefix's partials come from the launch before this one, which
    // this kernel may overlap until here (programmatic dependent launch).  With
    // join_kernel to follow, CTAs do not wait for it but make room for others; the last one
    // waits, so that this launch does not end before that one.
    if (!P.join || blockIdx.x + 1u == gridDim.x) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (single || (P.join && J.pre_splits)) return;
    __syncthreads();
    uint32_t *ctr = P.counters + (uint64_t)lo * P.kv_heads + kvh;
    if (tid == 0) {
        uint32_t prev;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(prev) : "l"(ctr) : "memory");
        s_last = prev == J.n_splits - 1u;
    }
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) *ctr = 0u;  // ready for the next call

    // ---- the last CTA joins all partials of (sequence, KV head) ----
    const uint64_t row_pre = ((uint64_t)J.pre_tile + (uint64_t)kvh * J.pre_kvh) * 128u + J.pre_row;
    const float *own = P.part + ((uint64_t)J.slot * P.kv_heads + kvh) * stride;
    for (uint32_t idx = tid; idx < G * 32u; idx += kThreads) {
        const uint32_t h = idx >> 5;
        const Joined x = join_one(own, (uint64_t)P.kv_heads * stride, J.n_splits, P.pre_part, P.pre_ml, row_pre, J.pre_splits, G,
                                  h, idx);
        store_out4(J.out, out0 + idx * 4u, normalise(x.o, x.l, gate_s[h], false), P.bf16);
    }
}

// ------------------------------------------------------------ join
// One CTA per (sequence, KV head) with a shared prefix: its own partials and the
// prefix's, in that order.  Bound by trips to L2: one for every eight partials.
template <int NJ>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ BatchParams<NJ> P) {
    using namespace bd;
    const uint32_t tid = threadIdx.x, G = P.group;
    const uint32_t lo = blockIdx.x / P.kv_heads, kvh = blockIdx.x - lo * P.kv_heads;
    const SeqDev &J = P.seq[lo];
    after_previous();
    if (J.pre_splits == 0) return;
    const uint32_t stride = part_stride(G);
    const float *own = P.part + ((uint64_t)J.slot * P.kv_heads + kvh) * stride;
    const uint64_t row_pre = ((uint64_t)J.pre_tile + (uint64_t)kvh * J.pre_kvh) * 128u + J.pre_row;
    for (uint32_t idx = tid; idx < G * 32u; idx += 256u) {
        const uint32_t h = idx >> 5;
        const float gate = J.gate ? J.gate[kvh * G + h] : 0.f;
        const Joined x = join_one(own, (uint64_t)P.kv_heads * stride, J.n_splits, P.pre_part, P.pre_ml, row_pre, J.pre_splits, G,
                                  h, idx);
        store_out4(J.out, (uint64_t)kvh * G * 128u + idx * 4u, normalise(x.o, x.l, J.gate ? sigmoid_dev(gate) : 1.f, false),
                   P.bf16);
    }
}

// ------------------------------------------------------------ planning
// Rows of a split.  Few pairs (sequence, KV head): one wave of wide CTAs, with
// as many splits as fill it (131072 rows, 8 KV heads: 56 us when this was chosen,
// 119 in CTAs of four warps).  More pairs: the split whose CTAs, in whole waves of
// `resident`, cost least, a CTA's start and end counting as kFixedRows rows; a
// pair's splits are even, and a short pair is one (8 layers x 32769 rows: 101 us
// with 13 splits, 1.9 waves, 113 with 17, 2.5 waves, 123 with 7, 1.01).
constexpr uint32_t kMaxCtas = 4096, kFixedRows = 256, kWaves = 4;

struct Plan {
    bool wide;
    uint32_t slots;
    uint8_t order[kMaxSeqs];  // of the sequences' slots
};
static uint64_t plan_ctas(const SeqDev *seqs, uint32_t n, uint64_t rows) {
    const uint32_t r = (uint32_t)std::min<uint64_t>(rows, kMaxPos);
    uint64_t c = 0;
    for (uint32_t i = 0; i < n; i++) {
        const uint32_t len = seqs[i].end - seqs[i].start;
        c += len <= r ? 1u : (len - 1u) / r + 1u;
    }
    return c;
}
static Plan plan_splits(SeqDev *seqs, uint32_t n, uint32_t kv_heads, uint32_t wide_unit, uint32_t unit,
                        uint32_t ctas_per_sm, uint32_t sms) {
    Plan plan;
    const uint32_t resident = ctas_per_sm * sms;
    uint64_t total = 0, longest = 1;
    for (uint32_t i = 0; i < n; i++) {
        total += seqs[i].end - seqs[i].start;
        longest = std::max<uint64_t>(longest, seqs[i].end - seqs[i].start);
    }
    total *= kv_heads;
    plan.wide = (uint64_t)n * kv_heads <= kPlanSms / 4;
    const uint64_t u = plan.wide ? wide_unit : unit;
    uint64_t rows;
    if (plan.wide) {
        const uint64_t room = std::max<uint64_t>(sms, (uint64_t)n * kv_heads);
        rows = std::max<uint64_t>(1, (total / room + u - 1) / u) * u;
        while (plan_ctas(seqs, n, rows) * kv_heads > room) rows += std::max<uint64_t>(1, rows / (32 * u)) * u;
    } else {
        // The smallest split whose CTAs fit w waves, for the w that costs least.  A
        // guess of half a split lost for each pair keeps the search short.
        const uint64_t half = (uint64_t)n * kv_heads / 2, least = (total + kMaxCtas - 1) / kMaxCtas;
        uint64_t best = UINT64_MAX;
        rows = longest;
        const uint64_t w0 = std::max<uint64_t>(1, ((uint64_t)n * kv_heads + resident - 1) / resident);
        for (uint64_t w = w0; w < w0 + kWaves; w++) {
            const uint64_t room = w * resident;
            uint64_t r = std::max<uint64_t>(least, total / (room - half));
            r = std::max<uint64_t>(1, (r + u - 1) / u) * u;
            uint64_t c = plan_ctas(seqs, n, r) * kv_heads;
            for (int k = 0; c > room && r < longest; k++, c = plan_ctas(seqs, n, r) * kv_heads)
                r += std::max<uint64_t>(1, r / ((k < 8 ? 16 : 2) * u)) * u;
            const uint64_t cost = (c + resident - 1) / resident * (total / c + kFixedRows);
            if (cost < best) {
                best = cost;
                rows = r;
            }
        }
        rows = std::max(rows, least);
        rows = std::max<uint64_t>(1, (rows + u - 1) / u) * u;
    }
    for (uint32_t i = 0; i < n; i++) {
        SeqDev &J = seqs[i];
        const uint64_t len = J.end - J.start;
        J.n_splits = (uint32_t)std::max<uint64_t>(1, (len + rows - 1) / rows);
        J.split_rows = (uint32_t)std::max<uint64_t>(u, ((len + J.n_splits - 1) / J.n_splits + u - 1) / u * u);
    }
    // The longest first: the short ones even out the end.
    uint64_t key[kMaxSeqs];
    for (uint32_t i = 0; i < n; i++) key[i] = (uint64_t)(plan.wide ? 0u : ~seqs[i].split_rows) << 32 | i;
    if (!std::is_sorted(key, key + n)) std::sort(key, key + n);
    plan.slots = 0;
    for (uint32_t i = 0; i < n; i++) {
        plan.order[i] = (uint8_t)key[i];
        SeqDev &J = seqs[plan.order[i]];
        J.slot = plan.slots;
        plan.slots += J.n_splits;
    }
    return plan;
}

// Sequences of a launch: the counters bound them with many KV heads.
static uint32_t seqs_per_launch(uint32_t kv_heads) {
    return (uint32_t)std::min<uint64_t>(kMaxSeqs, kCounters / kv_heads);
}

// Workspace: counters, a PrefixSync, own partials, prefix partial tiles, their (max, sum) pairs.
struct Layout {
    uint64_t sync, part, pre, ml, bytes;
};
static Layout layout(uint64_t n_groups, uint64_t n_seqs, uint32_t q_heads, uint32_t kv_heads, bool shared) {
    const uint64_t n = std::min<uint64_t>(n_seqs, seqs_per_launch(kv_heads)), g = std::min<uint64_t>(n_groups, kPrefixGroups);
    const uint64_t ctas = n * kv_heads + kMaxCtas;
    const uint64_t tiles = shared ? prefix_tiles_bound(g, n, q_heads, kv_heads) : 0;
    Layout w;
    w.sync = kCounters * 4u;
    w.part = w.sync + 256u;
    w.pre = (w.part + ctas * part_stride(q_heads / kv_heads) * 4u + 255u) / 256u * 256u;
    w.ml = w.pre + tiles * 128u * 128u * 4u;
    w.bytes = w.ml + tiles * 128u * 2u * 4u;
    return w;
}

// ------------------------------------------------------------ launches
template <int MODE, bool I8, bool WIDE, int NJ>
static int launch(const SeqDev *seqs, uint32_t n, const Plan &plan, const BatchParams<1> &head, bool after_prefix,
                  cudaStream_t stream) {
    using Sh = Shape<MODE, I8, WIDE>;
    static bool ready[64];
    int dev = 0;
    if (int rc = check_cuda(cudaGetDevice(&dev), "decode get device")) return rc;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (int rc = check_cuda(cudaFuncSetAttribute(batch_decode_kernel<MODE, I8, WIDE, NJ>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Sh::kSmem),
                                "decode shared memory"))
            return rc;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    BatchParams<NJ> P;
    for (uint32_t i = 0; i < n; i++) {
        const SeqDev &J = P.seq[i] = seqs[plan.order[i]];
        if (plan.slots <= kMapped) std::memset(P.seq_of + J.slot, (int)i, J.n_splits);
    }
    P.slots = plan.slots;
    P.n = n;
    P.group = head.group;
    P.kv_heads = head.kv_heads;
    P.bf16 = head.bf16;
    P.part = head.part;
    P.counters = head.counters;
    P.sync = head.sync;
    P.pre_part = head.pre_part;
    P.pre_ml = head.pre_ml;
    // After a prefix launch the CTAs start on the SMs that it leaves, and stream their own
    // rows meanwhile; every CTA waits for that launch before it reads its
    // partials.  Otherwise they start as the kernel before drains, and wait for it.
    P.after_prefix = after_prefix;
    P.join = after_prefix && !WIDE;
    g_launches++;
    if (int rc = launch_early("decode launch", batch_decode_kernel<MODE, I8, WIDE, NJ>, dim3(plan.slots * head.kv_heads),
                              Sh::kThreads, Sh::kSmem, stream, P))
        return rc;
    if (!P.join) return SF37KV_OK;
    g_launches++;
    return launch_early("join launch", join_kernel<NJ>, dim3(n * head.kv_heads), 256, 0, stream, P);
}

template <int MODE, bool I8>
static int launch_n(SeqDev *seqs, uint32_t n, const BatchParams<1> &head, uint32_t prefix_ctas,
                    cudaStream_t stream) {
    const Plan plan = plan_splits(seqs, n, head.kv_heads, Shape<MODE, I8, true>::kUnit, Shape<MODE, I8, false>::kUnit,
                                  Shape<MODE, I8, false>::kCtas,
                                  prefix_ctas < kPlanSms ? kPlanSms - prefix_ctas : kPlanSms);
    const bool after_prefix = prefix_ctas > 0;
    // The descriptors travel as kernel parameters (30 KB for kMaxSeqs, whose copies take
    // the host some us); a small launch carries few, and a wide plan has few.
    static_assert(kPlanSms / 4 <= kSomeSeqs, "sequences of a wide plan");
    if (plan.wide) {
        if (n <= kSmallSeqs) return launch<MODE, I8, true, kSmallSeqs>(seqs, n, plan, head, after_prefix, stream);
        return launch<MODE, I8, true, kSomeSeqs>(seqs, n, plan, head, after_prefix, stream);
    }
    if (n <= kSmallSeqs) return launch<MODE, I8, false, kSmallSeqs>(seqs, n, plan, head, after_prefix, stream);
    if (n <= kSomeSeqs) return launch<MODE, I8, false, kSomeSeqs>(seqs, n, plan, head, after_prefix, stream);
    return launch<MODE, I8, false, kMaxSeqs>(seqs, n, plan, head, after_prefix, stream);
}

template <bool I8>
static int launch_mode(SeqDev *seqs, uint32_t n, const BatchParams<1> &head, uint32_t prefix_ctas,
                    cudaStream_t stream) {
    if (head.group <= 8 && head.bf16) return launch_n<kHalf, I8>(seqs, n, head, prefix_ctas, stream);
    if (head.group <= 8) return launch_n<kPair, I8>(seqs, n, head, prefix_ctas, stream);
    if (head.bf16) return launch_n<kWide, I8>(seqs, n, head, prefix_ctas, stream);
    return launch_n<kTwo, I8>(seqs, n, head, prefix_ctas, stream);
}

static int check_seq(const char *what, uint32_t i, const sf37kv_decode_seq &L, uint32_t prefix_len, bool ring_clamp) {
    if (int rc = check_cache(what, i, L.cache)) return rc;
    if (!L.q || !L.out || !aligned16(L.q) || !aligned16(L.out))
        return set_error(SF37KV_EINVAL, "%s: sequence %u q and out must be non-NULL and 16-byte aligned", what, i);
    if ((L.k_new != nullptr) != (L.v_new != nullptr))
        return set_error(SF37KV_EINVAL, "%s: sequence %u has only one of k_new/v_new", what, i);
    if (!aligned16(L.k_new) || !aligned16(L.v_new) || ((uintptr_t)L.gate & 3u))
        return set_error(SF37KV_EINVAL, "%s: sequence %u k_new/v_new must be 16-byte and gate 4-byte aligned", what, i);
    if (L.pos >= kMaxPos) return set_error(SF37KV_EINVAL, "%s: sequence %u position %u exceeds %u", what, i, L.pos, kMaxPos);
    if (L.k_new && L.cache.sliding && L.cache.window == 0)
        return set_error(SF37KV_EINVAL, "%s: sequence %u appends to a window of no rows", what, i);
    if (ring_clamp) return SF37KV_OK;
    const uint32_t have = L.pos + 1u;
    if (have < prefix_len)
        return set_error(SF37KV_EINVAL, "%s: sequence %u position %u is inside the prefix of %u", what, i, L.pos, prefix_len);
    if (L.k_new && have == prefix_len)
        return set_error(SF37KV_EINVAL, "%s: sequence %u appends at position %u, which is the prefix's", what, i, L.pos);
    uint32_t first = L.cache.sliding && have > L.cache.window ? have - L.cache.window : 0u;
    if (first < prefix_len) first = prefix_len;
    if (have > first && have - first > L.cache.cap)
        return set_error(SF37KV_EINVAL, "%s: sequence %u attends to %u own rows, its cache holds %u", what, i, have - first,
                         L.cache.cap);
    return SF37KV_OK;
}

// Whether a cache that one sequence of a call appends to overlaps another one's (rows of
// `row` bytes), or any group's prefix, which is read beside the appends.
static bool append_conflict(const sf37kv_shared_group *groups, uint32_t n_groups, uint64_t total, uint64_t row,
                            uint64_t prefix_row) {
    bool any = false;
    for (uint32_t i = 0; i < n_groups; i++)
        for (uint32_t k = 0; k < groups[i].n_seqs; k++) any |= groups[i].seqs[k].k_new != nullptr;
    if (!any) return false;
    return parts_conflict((size_t)(total + n_groups) * 2u, [&](const auto &add) {
        for (uint32_t i = 0; i < n_groups; i++) {
            const sf37kv_shared_group &Gr = groups[i];
            const uint64_t bytes = Gr.n_seqs ? Gr.prefix_len * prefix_row : 0u;
            add(2, Gr.prefix.k_cache, bytes, false);
            add(3, Gr.prefix.v_cache, bytes, false);
            for (uint32_t k = 0; k < Gr.n_seqs; k++) {
                const sf37kv_decode_seq &L = Gr.seqs[k];
                add(0, L.cache.k_cache, L.cache.cap * row, L.k_new != nullptr);
                add(1, L.cache.v_cache, L.cache.cap * row, L.k_new != nullptr);
            }
        }
    });
}

// Decode of all groups; ring_clamp (sf37kv_decode_i8): no prefixes, and a full cache's
// oldest rows drop out as in sf37kv_decode.
static int decode_groups(const char *what, const sf37kv_shared_group *groups, uint32_t n_groups, uint32_t q_heads,
                         uint32_t kv_heads, uint32_t head_dim, int dtype, int io_type, void *workspace,
                         uint64_t workspace_bytes, bool ring_clamp, cudaStream_t stream) {
    if (int rc = check_heads(what, q_heads, kv_heads, head_dim)) return rc;
    if (dtype != SF37KV_F16 && dtype != SF37KV_I8)
        return set_error(SF37KV_EUNSUPPORTED, "%s: cache dtype %d is neither f16 nor i8", what, dtype);
    if (io_type != SF37KV_Q_F32 && io_type != SF37KV_Q_BF16)
        return set_error(SF37KV_EINVAL, "%s: unknown io type %d", what, io_type);
    uint64_t total = 0;
    for (uint32_t i = 0; i < n_groups; i++) {
        const sf37kv_shared_group &Gr = groups[i];
        if (Gr.n_seqs == 0) continue;
        if (!Gr.seqs) return set_error(SF37KV_EINVAL, "%s: group %u has no sequences array", what, i);
        if (Gr.prefix_len) {
            if (int rc = check_cache(what, i, Gr.prefix)) return rc;
            if (Gr.prefix_len > Gr.prefix.cap)
                return set_error(SF37KV_EINVAL, "%s: group %u prefix of %u rows exceeds its cache of %u", what, i,
                                 Gr.prefix_len, Gr.prefix.cap);
        }
        for (uint32_t k = 0; k < Gr.n_seqs; k++) {
            const sf37kv_decode_seq &L = Gr.seqs[k];
            if (int rc = check_seq(what, k, L, Gr.prefix_len, ring_clamp)) return rc;
            if (Gr.prefix_len && L.k_new &&
                (L.cache.k_cache == Gr.prefix.k_cache || L.cache.v_cache == Gr.prefix.v_cache))
                return set_error(SF37KV_EINVAL, "%s: sequence %u appends to its prefix's cache", what, k);
        }
        total += Gr.n_seqs;
    }
    if (total == 0) return SF37KV_OK;
    try {
        if (append_conflict(groups, n_groups, total, (uint64_t)kv_heads * (dtype == SF37KV_I8 ? 132u : 256u), kv_heads * 256ull))
            return set_error(SF37KV_EINVAL,
                             "%s: a cache that one sequence appends to is given twice, or overlaps another or a group's prefix",
                             what);
    } catch (const std::bad_alloc &) {
        return set_error(SF37KV_ENOMEM, "%s: no memory to compare %llu sequences", what, (unsigned long long)total);
    }
    const Layout W = layout(n_groups, total, q_heads, kv_heads, !ring_clamp);
    if (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < W.bytes)
        return set_error(SF37KV_EINVAL, "%s: the workspace must be 256-byte aligned and hold %llu bytes", what,
                         (unsigned long long)W.bytes);
    char *ws = (char *)workspace;
    BatchParams<1> head;
    head.group = q_heads / kv_heads;
    head.kv_heads = kv_heads;
    head.bf16 = io_type == SF37KV_Q_BF16;
    head.counters = (uint32_t *)ws;
    head.sync = (PrefixSync *)(ws + W.sync);
    head.part = (float *)(ws + W.part);
    head.pre_part = (const float *)(ws + W.pre);
    head.pre_ml = (const float *)(ws + W.ml);
    const uint32_t most = seqs_per_launch(kv_heads), T = prefix_seqs_per_tile(head.group);
    uint32_t gi = 0, k0 = 0;  // next group, and its next sequence
    while (gi < n_groups) {
        PrefixGroup pg[kPrefixGroups];
        PrefixSeq ps[kMaxSeqs];
        SeqDev sd[kMaxSeqs];
        uint32_t owner[kMaxSeqs];  // the sequence's prefix group, or n_pg
        uint32_t n = 0, n_pg = 0;
        while (gi < n_groups && n < most && n_pg < (uint32_t)kPrefixGroups) {
            const sf37kv_shared_group &Gr = groups[gi];
            const uint32_t take = std::min(Gr.n_seqs - k0, most - n);
            PrefixGroup &X = pg[n_pg];
            X = PrefixGroup{Gr.prefix.k_cache, Gr.prefix.v_cache, Gr.prefix_len, Gr.prefix_len, n, take};
            for (uint32_t k = 0; k < take; k++, n++) {
                const sf37kv_decode_seq &L = Gr.seqs[k0 + k];
                const uint32_t have = L.pos + 1u;
                uint32_t first = L.cache.sliding && have > L.cache.window ? have - L.cache.window : 0u;
                if (ring_clamp) first = start_at(L.pos, L.cache.cap, (int)L.cache.sliding, L.cache.window);
                ps[n] = PrefixSeq{L.q, std::min(first, Gr.prefix_len), 0};
                X.lo = std::min(X.lo, ps[n].start);
                SeqDev &J = sd[n];
                J = SeqDev{L.cache.k_cache, L.cache.v_cache, L.q, L.gate, L.out, L.k_new, L.v_new};
                J.start = std::min(std::max(first, Gr.prefix_len), have);
                J.end = have;
                J.cap = L.cache.cap;
                owner[n] = n_pg;
            }
            if (X.lo < X.len) n_pg++;
            else for (uint32_t k = n - take; k < n; k++) owner[k] = UINT32_MAX;
            k0 += take;
            if (k0 == Gr.n_seqs) {
                gi++;
                k0 = 0;
            }
        }
        if (n == 0) continue;
        uint64_t own = 0;  // rows
        for (uint32_t k = 0; k < n; k++) own += sd[k].end - sd[k].start;
        const uint32_t prefix_ctas =
            n_pg ? prefix_plan(pg, n_pg, q_heads, kv_heads, !head.bf16, own, dtype == SF37KV_I8) : 0;
        for (uint32_t k = 0; k < n; k++) {
            SeqDev &J = sd[k];
            J.pre_tile = J.pre_kvh = J.pre_splits = J.pre_row = 0;
            if (owner[k] == UINT32_MAX || ps[k].start >= pg[owner[k]].len) continue;
            const PrefixGroup &X = pg[owner[k]];
            const uint32_t i = k - X.seq0;
            J.pre_tile = X.part0 + i / T * X.splits;
            J.pre_kvh = X.m_tiles * X.splits;
            J.pre_splits = X.splits;
            J.pre_row = i % T * head.group;
        }
        if (n_pg)
            if (int rc = prefix_attention(pg, n_pg, ps, n, q_heads, kv_heads, !head.bf16, (float *)(ws + W.pre),
                                          (float *)(ws + W.ml), head.sync, stream))
                return rc;
        const int rc = dtype == SF37KV_I8 ? launch_mode<true>(sd, n, head, prefix_ctas, stream)
                                          : launch_mode<false>(sd, n, head, prefix_ctas, stream);
        if (rc) return rc;
    }
    return SF37KV_OK;
}

}  // namespace sf37kv

using namespace sf37kv;

extern "C" uint64_t sf37kv_decode_i8_workspace(uint32_t n_seqs, uint32_t q_heads, uint32_t kv_heads) {
    if (check_heads("decode_i8_workspace", q_heads, kv_heads, 128)) return 0;
    return layout(1, n_seqs, q_heads, kv_heads, false).bytes;
}

extern "C" int sf37kv_decode_i8(const sf37kv_decode_seq *seqs, uint32_t n_seqs, uint32_t q_heads, uint32_t kv_heads,
                                uint32_t head_dim, int io_type, void *workspace, uint64_t workspace_bytes,
                                void *stream) {
    if (!seqs && n_seqs) return set_error(SF37KV_EINVAL, "decode_i8: seqs is NULL");
    sf37kv_shared_group one = {};
    one.n_seqs = n_seqs;
    one.seqs = seqs;
    return decode_groups("decode_i8", &one, 1, q_heads, kv_heads, head_dim, SF37KV_I8, io_type, workspace,
                         workspace_bytes, true, stream ? (cudaStream_t)stream : current_stream());
}

extern "C" uint64_t sf37kv_decode_shared_workspace(uint32_t n_groups, uint32_t n_seqs, uint32_t q_heads,
                                                   uint32_t kv_heads) {
    if (check_heads("decode_shared_workspace", q_heads, kv_heads, 128)) return 0;
    return layout(n_groups, n_seqs, q_heads, kv_heads, true).bytes;
}

extern "C" int sf37kv_decode_shared(const sf37kv_shared_group *groups, uint32_t n_groups, uint32_t q_heads,
                                    uint32_t kv_heads, uint32_t head_dim, int dtype, int io_type, void *workspace,
                                    uint64_t workspace_bytes, void *stream) {
    if (!groups && n_groups) return set_error(SF37KV_EINVAL, "decode_shared: groups is NULL");
    return decode_groups("decode_shared", groups, n_groups, q_heads, kv_heads, head_dim, dtype, io_type, workspace,
                         workspace_bytes, false, stream ? (cudaStream_t)stream : current_stream());
}
