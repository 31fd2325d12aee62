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
// Warps 0-7 and 8-15 are the softmax of stream 0 and 1, two threads for each
// row (64 score columns each); warp 16 issues the MMAs, warp 17 the TMA loads,
// as in prefill_tc05.cu.  TMEM: S_0, S_1, O_0, O_1 (128 columns each); P
// (f16) overwrites its S.  F32 (f32 queries and outputs): q and P are two
// f16 parts each, q_hi + q_lo and P_hi + P_lo, 22 bits: twice the MMAs; P_lo
// takes the second half of S's columns.
//
// Weights are 2^(x - m) with the reference m 7 below a running row maximum,
// raised when x - m passes 15: f16 holds them up to 2^15, and down to 2^-32 of
// the largest.  S and O accumulate in f32 (TMEM), m and l in f32 registers.
#include <algorithm>
#include <type_traits>

#include "batch_internal.cuh"
#include "tc05.cuh"

namespace sf37kv {

extern unsigned long long g_launches;

static __device__ int g_prefix_error;  // 1: a bounded wait gave up

struct PrefixDev {
    CUtensorMap kmap, vmap;  // rows [0, len): later rows read as zeros
    uint32_t lo, len, seq0, n_seqs, m_tiles, splits, tps, part0, cta0, pairs;
};
template <int NS>
struct PrefixParams {
    PrefixDev group[kPrefixGroups];
    PrefixSeq seq[NS];
    float *part, *ml;
    uint32_t n_groups, heads_per_kv, kv_heads, tpt;
};

constexpr float kHead = 7.0f, kRaise = 15.0f;

template <bool F32, int NS>
__global__ void __launch_bounds__(576, 1) prefix_tc05_kernel(const __grid_constant__ PrefixParams<NS> P) {
    using namespace tc05;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    enum { B_KFULL = 0, B_KEMPTY = 3, B_VFULL = 6, B_VEMPTY = 8, B_SFULL = 10, B_PFULL = 12, B_ODONE = 14, N_BARS = 16 };
    enum { T_Q = 0, T_K = 2, T_V = 4 };  // 32 KB tiles; Q: two tiles (pair) or hi and lo (F32), else a third K tile
    __shared__ __align__(8) uint64_t bars[N_BARS];
    __shared__ uint32_t tmem_base_sh;
    __shared__ volatile int abort_sh;
    __shared__ float xch[2][2][2][128];  // [parity][stream][half][row]
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

    if (tid == 0) {
        for (uint32_t t = 0; t < 3; t++) {
            bar_init(bar(B_KFULL + t), 1);
            bar_init(bar(B_KEMPTY + t), 1);
        }
        for (uint32_t t = 0; t < 2; t++) {
            bar_init(bar(B_VFULL + t), 1);
            bar_init(bar(B_VEMPTY + t), 1);
            bar_init(bar(B_SFULL + t), 1);
            bar_init(bar(B_PFULL + t), 256);
            bar_init(bar(B_ODONE + t), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;");
        abort_sh = 0;
    }
    if (warp == 0) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(&tmem_base_sh);
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // The kernel before (which may still drain: programmatic dependent launch) is
    // waited for; then the next one, which reads this kernel's partials after a
    // wait of its own, may start as SMs become free.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    // Q tiles: scaled by a power of two for each row so that its largest element
    // is in [1, 2): f16 then holds a bf16 row exactly and hi + lo 22 bits.  A warp
    // reads whole rows, 16 lanes (bf16) or 32 (f32) each: with a row a thread,
    // 32 lines a load, this start took 8 us.  Rows belong to several sequences;
    // their table is read by generic loads (lane-divergent constant loads replay).
    const PrefixSeq *tab = P.seq;
    asm volatile("" : "+l"(tab));
    if (warp < 16) {
        constexpr uint32_t kLanes = F32 ? 32 : 16, kAtOnce = 32 / kLanes;
        const uint32_t per_warp = (solo ? 128u : 256u) / 16u, c = lane % kLanes;
        uint4 raw[8];
        float scale[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            const uint32_t x = warp * per_warp + i * kAtOnce + lane / kLanes;  // row of both tiles
            if (i * kAtOnce < per_warp) {
                const uint32_t sl = (x & 127u) / G, hl = (x & 127u) - sl * G;
                const PrefixSeq q = tab[Gr.seq0 + min((mt0 + (x >> 7)) * T + sl, Gr.n_seqs - 1u)];
                raw[i] = __ldg(reinterpret_cast<const uint4 *>(q.q) + (uint64_t)(kvh * G + hl) * kLanes + c);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i * kAtOnce < per_warp) {
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
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i * kAtOnce < per_warp) {
                const uint32_t x = warp * per_warp + i * kAtOnce + lane / kLanes, r = x & 127u;
                const int e = max(-126, min(126, (int)((__float_as_uint(scale[i]) >> 23) & 255u) - 127));
                const float f = __int_as_float((127 - e) << 23);
                if (c == 0)
                    qscale_sh[x >> 7][r] = __int_as_float((127 + e) << 23) * (1.4426950408889634f * 0.08838834764831845f);
                const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                uint8_t *qt = gsm + (T_Q + (x >> 7)) * kTile;
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
    const uint32_t st = warp >> 3;               // stream of a softmax warp
    const uint32_t hh = (warp >> 2) & 1u;        // column half
    const uint32_t r = ((warp & 3u) << 5) | lane;
    const uint32_t sl = r / G;
    const uint32_t mt = solo ? mt0 : mt0 + (st & 1u);
    const uint32_t si = mt * T + sl;             // sequence within the group
    const bool valid = sl < T && si < Gr.n_seqs;
    const uint32_t first = tab[Gr.seq0 + min(si, Gr.n_seqs - 1u)].start;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base_sh;

    if (warp == 17) {
        // ---------------- TMA loader: a ring of K tiles and one of V tiles ----------------
        auto loader = [&](auto kind) {
            constexpr uint32_t kRing = decltype(kind)::value && !F32 ? 3 : 2, kTile0 = kRing == 3 ? 1 : T_K;
            const int32_t x0 = (int32_t)(kvh * 128u);
            auto load = [&](uint32_t full, uint32_t dst, const CUtensorMap *map, uint32_t j) {
                const int32_t y = (int32_t)(kbeg + j * 128u);
                bar_expect_tx(full, kTile);
                tma_load_2d(dst, map, x0, y, full);
                tma_load_2d(dst + kHalf, map, x0 + 64, y, full);
            };
            auto load_k = [&](uint32_t j) { load(bar(B_KFULL + j % kRing), tile(kTile0 + j % kRing), &Gr.kmap, j); };
            auto load_v = [&](uint32_t j) { load(bar(B_VFULL + (j & 1u)), tile(T_V + (j & 1u)), &Gr.vmap, j); };
            for (uint32_t j = 0; j < kRing && j < nt; j++) {
                load_k(j);
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
        if (lane == 0) {
            if (solo) loader(std::true_type());
            else loader(std::false_type());
        }
    } else if (warp == 16) {
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
                    const uint32_t off = (((kk >> 2) & 1u) * kHalf + (kk & 3u) * 32u) >> 4;
                    mma(tmem + t * 128u, a + (kk >> 3) * (kTile >> 4) + off, b + off, idesc(0), kk > 0);
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
                issue_pv(t, i > 1, !more);
                if (more) issue_s(t);
            }
            return true;
        };
        if (lane == 0 && !(solo ? issuer(std::true_type()) : issuer(std::false_type()))) abort_sh = 1;
    } else {
        // ---------------- softmax of stream st, column half hh ----------------
        const uint32_t lane_off = ((warp & 3u) * 32u) << 16;
        const uint32_t cb = 64u * hh;
        const uint32_t t_s = tmem + st * 128u + lane_off, t_o = tmem + 256u + st * 128u + lane_off;
        const uint32_t pair_bar = 1u + st * 4u + (warp & 3u);  // the two warps that share these rows
        // Pair barrier that also ORs a flag, so both warps take the same exit.
        auto pair_any = [&](bool v) -> bool {
            uint32_t rr;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                "bar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
                : "=r"(rr)
                : "r"((uint32_t)v), "r"(pair_bar)
                : "memory");
            return rr != 0;
        };
        const uint32_t s_row = max(first, kbeg);
        const float qs = qscale_sh[solo ? 0 : st][r];
        const uint32_t n_steps = solo ? (nt + 1u - st) >> 1 : nt;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        // One pass over this thread's 64 scores with reference mu: weights (f16 pairs,
        // and their remainders) into w and wl, their sum, the largest x - mu.
        auto pass_of = [&](auto masked, uint32_t k0, float mu, uint32_t (&w)[2][16], uint32_t (&wl)[2][16], float &la,
                           float &xm) {
            float lb = 0.f, xa = -INFINITY, xb = -INFINITY;
            la = 0.f;
#pragma unroll
            for (int q2 = 0; q2 < 2; q2++) {
                float v[32];
                tmem_ld32(t_s + cb + q2 * 32u, v);
                tmem_wait_ld();
                const uint32_t kb = k0 + cb + (uint32_t)(q2 * 32);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float x0 = fmaf(v[2 * i], qs, -mu), x1 = fmaf(v[2 * i + 1], qs, -mu);
                    if (decltype(masked)::value) {
                        const uint32_t kp = kb + 2u * i;
                        if (kp < s_row || kp >= kend) x0 = -INFINITY;
                        if (kp + 1u < s_row || kp + 1u >= kend) x1 = -INFINITY;
                    }
                    xa = fmaxf(xa, x0);
                    xb = fmaxf(xb, x1);
                    const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                    la += p0;
                    lb += p1;
                    w[q2][i] = pack_h2(p0, p1);
                    if (F32) {
                        const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[q2][i]));
                        wl[q2][i] = pack_h2(p0 - h.x, p1 - h.y);
                    }
                }
            }
            la += lb;
            xm = fmaxf(xa, xb);
        };
        auto pass = [&](uint32_t k0, bool full, float mu, uint32_t (&w)[2][16], uint32_t (&wl)[2][16], float &la, float &xm) {
            if (full) pass_of(std::false_type(), k0, mu, w, wl, la, xm);
            else pass_of(std::true_type(), k0, mu, w, wl, la, xm);
        };
        for (uint32_t s = 0; s < n_steps; s++) {
            const uint32_t k0 = kbeg + (solo ? 2u * s + st : s) * 128u;
            __syncwarp();
            const bool got = !abort_sh && wait_bar_warp(bar(B_SFULL + st), s & 1u);
            fence_after();
            const bool full = __all_sync(0xffffffffu, k0 >= s_row && k0 + 128u <= kend);
            uint32_t w[2][16], wl[2][16];
            float la = 0.f, xm = -INFINITY;
            const float mu0 = m == -INFINITY ? 0.f : m;
            if (got && (F32 || s > 0)) pass(k0, full, mu0, w, wl, la, xm);
            if (!F32 && got && s == 0) {  // no reference yet: the largest score alone (F32: no registers for it)
#pragma unroll
                for (int q2 = 0; q2 < 2; q2++) {
                    float v[32];
                    tmem_ld32(t_s + cb + q2 * 32u, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const uint32_t kp = k0 + cb + (uint32_t)(q2 * 32 + i);
                        if (full || (kp >= s_row && kp < kend)) xm = fmaxf(xm, v[i]);
                    }
                }
                xm *= qs;
            }
            if (pair_any(!got)) { abort_sh = 1; ok = false; break; }
            const bool need = (m == -INFINITY && xm > -INFINITY) || xm > kRaise;
            if (pair_any(need || (!F32 && s == 0))) {
                // raise the rows' references: exchange the maximum with the other half, rescale O, redo P
                xch[s & 1u][st][hh][r] = xm + mu0;
                pair_any(false);
                const float mx = fmaxf(xch[s & 1u][st][0][r], xch[s & 1u][st][1][r]) - kHead;
                const bool raise = mx > -INFINITY && (m == -INFINITY || mx > m + (kRaise - kHead));
                if (__any_sync(0xffffffffu, raise || (!F32 && s == 0))) {
                    const float alpha = !raise ? 1.f : m == -INFINITY ? 0.f : fast_exp2(m - mx);
                    if (s > 0) {
#pragma unroll
                        for (int q2 = 0; q2 < 2; q2++) {
                            float v[32];
                            tmem_ld32(t_o + cb + q2 * 32u, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] *= alpha;
                            tmem_st32(t_o + cb + q2 * 32u, v);
                        }
                        tmem_wait_st();
                    }
                    if (raise) {
                        l *= alpha;
                        m = mx;
                    }
                    pass(k0, full, m == -INFINITY ? 0.f : m, w, wl, la, xm);
                }
                pair_any(false);  // both halves have re-read S
            }
            // (both halves have read S: P overwrites columns of either)
            l += la;
            tmem_st16u(t_s + cb / 2u, w[0]);
            tmem_st16u(t_s + cb / 2u + 16u, w[1]);
            if (F32) {
                tmem_st16u(t_s + 64u + cb / 2u, wl[0]);
                tmem_st16u(t_s + 64u + cb / 2u + 16u, wl[1]);
            }
            tmem_wait_st();
            fence_before();
            bar_arrive(bar(B_PFULL + st));
        }
        const bool got_e = n_steps == 0 || (ok && !abort_sh && wait_bar_warp(bar(B_ODONE + st), 0));
        if (ok) {
            xch[0][st][hh][r] = l;
            if (pair_any(!got_e)) ok = false;
        }
        if (!ok) abort_sh = 1;
        if (ok) l = xch[0][st][0][r] + xch[0][st][1][r];
        // Partial tile of (kv head, m tile, split).
        const uint64_t row = ((uint64_t)Gr.part0 + ((uint64_t)kvh * Gr.m_tiles + mt) * Gr.splits + split) * 128u + r;
        float wA = 1.f;
        const float *ob = reinterpret_cast<const float *>(gsm + T_K * kTile);  // stream 1's O, [128 columns][128 rows]
        if (hh == 0) {
            xch[1][st][0][r] = m;
            xch[1][st][1][r] = l;
        }
        asm volatile("bar.sync 9, 512;" ::: "memory");  // both streams' MMAs are done: the K and V tiles are free
        if (solo) {
            // Join the streams: stream 1 leaves (m, l) and its O, scaled, in the K tiles.
            const float m0 = xch[1][0][0][r], m1 = xch[1][1][0][r], l0 = xch[1][0][1][r], l1 = xch[1][1][1][r];
            const float mj = fmaxf(m0, m1);
            wA = m0 == -INFINITY ? (l0 == 0.f ? 0.f : 1.f) : fast_exp2(m0 - mj);
            const float wB = m1 == -INFINITY ? (l1 == 0.f ? 0.f : 1.f) : fast_exp2(m1 - mj);
            if (st == 1 && n_steps > 0 && !abort_sh) {
                fence_after();
#pragma unroll
                for (int q2 = 0; q2 < 2; q2++) {
                    float v[32];
                    tmem_ld32(t_o + cb + q2 * 32u, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i++) const_cast<float *>(ob)[(cb + q2 * 32u + i) * 128u + r] = v[i] * wB;
                }
            }
            asm volatile("bar.sync 9, 512;" ::: "memory");
            m = mj;
            l = l0 * wA + l1 * wB;
        }
        if (!abort_sh && (!solo || st == 0)) {
            // O goes through shared memory (16-byte chunk c of row r at c ^ (r & 31)), so that
            // the global stores are whole rows: stream 0 by the V tiles, stream 1 by the K tiles
            // (solo: stream 1's O is there until it is added).
            fence_after();
            uint8_t *stage = gsm + (st == 0 ? T_V : T_K) * kTile + r * 512u;
#pragma unroll
            for (int q2 = 0; q2 < 2; q2++) {
                float v[32];
                tmem_ld32(t_o + cb + q2 * 32u, v);
                tmem_wait_ld();
                if (solo) {
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        v[i] *= wA;
                        if (nt > 1) v[i] += ob[(cb + q2 * 32u + i) * 128u + r];
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < 8; i++)
                    *reinterpret_cast<float4 *>(stage + (((cb / 4u + q2 * 8u + i) ^ (r & 31u)) << 4)) =
                        make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
            pair_any(false);  // the two warps' halves of 32 rows are in place; each stores 16 of them
            const uint32_t rows = min(T, Gr.n_seqs - mt * T) * G;  // of the tile's, those that hold a head
            const uint32_t r0 = (warp & 3u) * 32u + hh * 16u;
            const uint8_t *tile_sm = gsm + (st == 0 ? T_V : T_K) * kTile;
            float *tile_out = P.part + (row - r) * 128u;
#pragma unroll 4
            for (uint32_t x = r0; x < min(r0 + 16u, rows); x++)
                *reinterpret_cast<float4 *>(tile_out + x * 128u + lane * 4u) =
                    *reinterpret_cast<const float4 *>(tile_sm + x * 512u + ((lane ^ (x & 31u)) << 4));
            if (valid && hh == 0) *reinterpret_cast<float2 *>(P.ml + row * 2u) = make_float2(m, l);
        }
    }
    fence_before();
    __syncthreads();
    if (abort_sh && tid == 0) atomicExch(&g_prefix_error, 1);
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

// CTAs stay within units + 2 * kPlanSms, a CTA has at most two tiles, and
// 2 * (KV heads x tile pairs) within KV heads x (m tiles + groups).
uint64_t prefix_tiles_bound(uint64_t n_groups, uint64_t n_seqs, uint32_t q_heads, uint32_t kv_heads) {
    const uint64_t m_tiles = n_seqs / prefix_seqs_per_tile(q_heads / kv_heads) + n_groups;
    return (uint64_t)kv_heads * (m_tiles + n_groups) + 4u * kPlanSms;
}

template <bool F32, int NS>
static int launch(const PrefixGroup *groups, uint32_t n, const PrefixSeq *seqs, uint32_t n_seqs, uint32_t q_heads,
                  uint32_t kv_heads, float *part, float *ml, cudaStream_t stream) {
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
    P.n_groups = n;
    P.heads_per_kv = q_heads / kv_heads;
    P.kv_heads = kv_heads;
    P.tpt = prefix_seqs_per_tile(P.heads_per_kv);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(576);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, prefix_tc05_kernel<F32, NS>, P);
    if (e == cudaSuccess) e = cudaGetLastError();
    g_launches++;
    return check_cuda(e, "prefix launch");
}

int prefix_attention(const PrefixGroup *groups, uint32_t n, const PrefixSeq *seqs, uint32_t n_seqs, uint32_t q_heads,
                     uint32_t kv_heads, bool f32, float *part, float *ml, cudaStream_t stream) {
    if (n_seqs <= 32)
        return f32 ? launch<true, 32>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, stream)
                   : launch<false, 32>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, stream);
    return f32 ? launch<true, kPrefixSeqs>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, stream)
               : launch<false, kPrefixSeqs>(groups, n, seqs, n_seqs, q_heads, kv_heads, part, ml, stream);
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
