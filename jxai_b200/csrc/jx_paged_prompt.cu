// jx_paged_prompt.cu -- causal prompt attention on the tensor cores (tcgen05) for
// the paged 8-bit cache, whose rows were brought to fp16 (widen_kernel).
//
//  * Work item: 2 * 128/G consecutive tokens of a sequence, one layer, one kv
//    head: two tiles X = 0, 1 of 128 query rows (row r = token r/G, head r%G)
//    that read the same K and V tiles.
//  * What bounds it: per 128 x 128 scores, 2 * 128*128*HD multiply-adds for each of S
//    and P.V (q and p in two fp16 parts; 1024 cycles each at head_dim 128, at 4096
//    per cycle) against 16384 exponentials at 16 per cycle (1024 cycles) and about 6
//    instructions per score on four schedulers.  Measured: 8192 tokens of two
//    Mistral-7B-shaped layers 2.33 ms with append and widening (472 TFLOP/s by the
//    attention's formula, twice that in products; tensor pipe 47 % active), 2048
//    tokens of the Llama-3.2-1B shape 1.13 ms (tensor pipe 25 %).  The three overlap
//    only if there is always a tile for each, so two tiles take turns: while one's
//    softmax runs, the tensor cores work on the other.
//  * Warp 0 streams K and V tiles (128 rows, TMA, 128-byte swizzle) through a
//    ring.  Warp 1 issues the MMAs of both tiles from one thread.  Warps 2-9 and
//    10-17 are the softmax of tile 0 and 1: two threads per row, each with half of
//    its scores, weights and dims; they exchange the row's maximum per tile.
//  * TMEM (512 columns): S of both tiles, 128 each, and O of both.  The weights
//    replace the scores they came from -- as fp16, both parts take exactly S's
//    columns -- and are the A operand of P.V from there; no weight passes through
//    shared memory, which Q (two parts, both tiles) and the ring fill.
//  * A tile's next S overwrites its P: it is issued once that P.V has completed,
//    while the other tile's work is in the queue.
//  * Weights are taken against a reference 2^7 below the largest score when it is
//    set, and it moves only when a weight would exceed 2^15 (fp16 ends at 2^16; its
//    floor then lies 2^-32 below the largest weight).  O is then rescaled in TMEM,
//    its P.V known complete from the S that follows it.
//  * The tensor cores cut the sum they add to towards zero (about 1e-8 of it per
//    MMA of 16 rows), which over thousands of rows adds up to 1e-5.  So O sums
//    a few tiles, then the softmax threads add it to an fp32 total of their own
//    in global memory (L2; [dim][row], so that a warp's accesses are whole lines),
//    while the next S is being computed, and P.V begins anew.
//  * Every mbarrier wait is bounded; one that runs out raises the abort flag and
//    the device error word, and every role finishes its control flow.
#include "jx_internal.h"
#include "jx_paged.h"
#include "jx_tcgen05.cuh"

namespace jx {
namespace {

constexpr int kThreads = 32 * 18;
constexpr float kLog2 = 1.4426950408889634f;
constexpr float kFar = 1048576.0f;  // scores beyond: a difference of a few is no longer exact


template <int HD>
struct PromptCfg {
    static constexpr int BN = 128;
    static constexpr int NSLAB = HD / 64;        // 128-byte slabs of a head row
    static constexpr int SLAB = 128 * 128;       // 128 rows of one slab
    static constexpr int TILE = SLAB * NSLAB;    // a K or V tile, or one part of a Q tile
    static constexpr int NS = HD == 64 ? 8 : 3;  // ring stages (K0, V0, K1, ...)
    static constexpr int OFF_Q = 0;              // [tile][part]
    static constexpr int OFF_KV = 4 * TILE;
    static constexpr int OFF_BAR = OFF_KV + NS * TILE;
    static constexpr int B_KVF = 0, B_KVE = NS, B_QF = 2 * NS, B_SF = B_QF + 2, B_PF = B_SF + 2, B_PV = B_PF + 2,
                         B_OE = B_PV + 2, B_DONE = B_OE + 2, NBARS = B_DONE + 1;
    static constexpr int OFF_MISC = OFF_BAR + NBARS * 8;
    static constexpr int OFF_XCH = OFF_MISC + 16;      // [tile][half][128] floats: row exchanges
    static constexpr int SMEM = OFF_XCH + 2 * 2 * 128 * 4;
    static constexpr int COL_S = 0, COL_O = 256;       // tile X: + 128 X
    static constexpr int DRAIN = HD == 64 ? 4 : 6;     // K/V tiles that O sums before it is added to the total
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

template <int HD, int G>
__global__ void __launch_bounds__(kThreads, 1)
    paged_prompt_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const PromptArgs a) {
    using C = PromptCfg<HD>;
    constexpr int BN = C::BN, TQ = 128 / G;
    // 128-byte-swizzled tiles: 1024-byte aligned (nothing else is in shared memory)
    extern __shared__ __align__(1024) unsigned char base[];
    const uint32_t sbase = smem_u32(base);
    if (sbase & 1023u) {  // every thread takes this branch together
        if (threadIdx.x == 0) atomicExch(a.err, kDevErrCheck);
        return;
    }
    const uint32_t bars = sbase + C::OFF_BAR;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + C::OFF_MISC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(base + C::OFF_MISC + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int it_begin = a.cta_first[blockIdx.x], it_end = a.cta_first[blockIdx.x + 1];
#define BAR(i) (bars + 8u * static_cast<uint32_t>(i))
#define WAIT(i, par, site, idx) \
    mbar_wait_bounded(BAR(i), (par), abort_flag, a.err, a.dbg, (site), (idx), true, a.wait_limit)

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::NS; ++s) {
            mbar_init(BAR(C::B_KVF + s), 1);
            mbar_init(BAR(C::B_KVE + s), 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(BAR(C::B_QF + x), 8);
            mbar_init(BAR(C::B_SF + x), 1);
            mbar_init(BAR(C::B_PF + x), 8);
            mbar_init(BAR(C::B_PV + x), 1);
            mbar_init(BAR(C::B_OE + x), 8);
        }
        mbar_init(BAR(C::B_DONE), 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // K/V tiles that tile x of an item reads (it has no later rows to attend)
    auto tiles_of = [](const PrefillTile& t, int x) {
        const int tok = x == 0 ? min(t.ntok, TQ) : t.ntok - TQ;
        return tok <= 0 ? 0 : (t.tok_row0 + x * TQ + tok - t.kv_lo + BN - 1) / BN;
    };

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            prefetch_tensormap(&tmK);
            prefetch_tensormap(&tmV);
        }
        int n = 0, issued = 0;  // tiles of the ring so far
        for (int it = it_begin; it < it_end; ++it) {
            const PrefillTile tl = a.tiles[it];
            const int nt = max(tiles_of(tl, 0), tiles_of(tl, 1));
            for (int t = 0; t < 2 * nt; ++t, ++n) {
                const int st = n % C::NS;
                if (n >= C::NS) WAIT(C::B_KVE + st, ((n / C::NS) & 1) ^ 1u, 50, n);
                if (__shfl_sync(0xffffffffu, *abort_flag, 0)) continue;
                issued = n + 1;
                if (lane == 0) {
                    mbar_arrive_expect_tx(BAR(C::B_KVF + st), C::TILE);
#pragma unroll
                    for (int b = 0; b < C::NSLAB; ++b)
                        tma_load_4d(sbase + C::OFF_KV + st * C::TILE + b * C::SLAB, (t & 1) ? &tmV : &tmK,
                                    BAR(C::B_KVF + st), tl.kvh * HD + b * 64, tl.kv_lo + t / 2 * BN, tl.cache_layer, tl.seq);
                }
                __syncwarp();
            }
        }
        // every issued tile lands before the CTA exits
        for (int k = max(0, issued - C::NS); k < issued; ++k)
            mbar_wait_bounded(BAR(C::B_KVF + k % C::NS), (k / C::NS) & 1, abort_flag, a.err, a.dbg, 51, k, false,
                              kDrainLimitCycles);
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t ID_S = idesc_f16(DT_F16T, 128, BN, false);
        constexpr uint32_t ID_PV = idesc_f16(DT_F16T, 128, HD, true);
        int n0 = 0, itc = 0;          // first ring tile of the item, items so far
        int pf[2] = {0, 0};           // weights taken, and P.V issued, of each tile
        for (int it = it_begin; it < it_end; ++it, ++itc) {
            const PrefillTile tl = a.tiles[it];
            const int cnt[2] = {tiles_of(tl, 0), tiles_of(tl, 1)};
            const int nt = max(cnt[0], cnt[1]);
            auto kv_at = [&](int n) { return sbase + C::OFF_KV + (n % C::NS) * C::TILE; };
            auto issue_s = [&](int x, int t) {  // S = Q_lo.K^T + Q_hi.K^T
                const int n = n0 + 2 * t;
                WAIT(C::B_KVF + n % C::NS, (n / C::NS) & 1, 52, n);
                tc_fence_after();
                if (lane == 0) {
                    // the small parts first: what the sum loses is in proportion to its size
#pragma unroll
                    for (int part = 1; part >= 0; --part)
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ++ks) {
                            const uint32_t off = (ks / 4) * C::SLAB + (ks % 4) * 32;
                            tc_mma(tmem + C::COL_S + x * 128,
                                   sw128_desc(sbase + C::OFF_Q + (2 * x + part) * C::TILE + off, 16, 1024),
                                   sw128_desc(kv_at(n) + off, 16, 1024), ID_S, part == 0 || ks != 0 ? 1u : 0u);
                        }
                    tc_commit(BAR(C::B_SF + x));
                }
                __syncwarp();
            };
            auto release = [&](int n) {  // a ring tile, once all MMAs issued so far are done
                if (lane == 0) tc_commit(BAR(C::B_KVE + n % C::NS));
                __syncwarp();
            };
            for (int x = 0; x < 2; ++x) {
                WAIT(C::B_QF + x, itc & 1, 53, itc);
                if (cnt[x] == 0) {
                    // no rows in this tile: its softmax is let on to the next item (it
                    // would otherwise run ahead of the barriers' phases)
                    if (lane == 0) tc_commit(BAR(C::B_SF + x));
                    __syncwarp();
                    continue;
                }
                // S takes the place of the item before's last P
                if (pf[x] > 0) WAIT(C::B_PV + x, (pf[x] - 1) & 1, 61, itc);
                issue_s(x, 0);
            }
            if (nt > 0) release(n0);
            for (int t = 0; t < nt; ++t) {
                for (int x = 0; x < 2; ++x) {
                    if (t < cnt[x]) {
                        WAIT(C::B_PF + x, pf[x] & 1, 54, t);
                        // the first P.V overwrites O: the item before has read it
                        if (t == 0 && itc > 0) WAIT(C::B_OE + x, (itc - 1) & 1, 55, itc);
                        const int n = n0 + 2 * t + 1;
                        WAIT(C::B_KVF + n % C::NS, (n / C::NS) & 1, 56, n);
                        tc_fence_after();
                        if (lane == 0) {
#pragma unroll
                            for (int part = 1; part >= 0; --part)
#pragma unroll
                                for (int kb = 0; kb < BN / 16; ++kb)
                                    tc_mma_ts(tmem + C::COL_O + x * 128, tmem + C::COL_S + x * 128 + part * 64 + kb * 8,
                                              sw128_desc(kv_at(n) + kb * 16 * 128, C::SLAB, 1024), ID_PV,
                                              t % C::DRAIN != 0 || part == 0 || kb != 0 ? 1u : 0u);
                            tc_commit(BAR(C::B_PV + x));
                        }
                        __syncwarp();
                        if (t + 1 < cnt[x]) {
                            WAIT(C::B_PV + x, pf[x] & 1, 57, t);  // S takes the place of P
                            issue_s(x, t + 1);
                        }
                        ++pf[x];
                    }
                }
                release(n0 + 2 * t + 1);
                if (t + 1 < nt) release(n0 + 2 * t + 2);
            }
            n0 += 2 * nt;
        }
        // every MMA completes before TMEM is freed
        if (lane == 0) tc_commit(BAR(C::B_DONE));
        __syncwarp();
        mbar_wait_bounded(BAR(C::B_DONE), 0u, abort_flag, a.err, a.dbg, 58, 0, false, kDrainLimitCycles);
    } else {
        // ------------------------------------------------------------ softmax, two threads per row
        constexpr int SW = BN / 2, HW = HD / 2;  // scores and dims of a thread
        const int x = (warp - 2) >> 3, hf = ((warp - 2) >> 2) & 1;
        const int q4 = warp & 3;
        float* mine = reinterpret_cast<float*>(base + C::OFF_XCH) + (x * 2 + hf) * 128 + q4 * 32 + lane;
        const float* other = reinterpret_cast<const float*>(base + C::OFF_XCH) + (x * 2 + (hf ^ 1)) * 128 + q4 * 32 + lane;
        auto meet = [&]() { named_bar_sync(1 + x * 4 + q4, 64); };
        // The other thread's value for this row.  A write must not meet the partner's
        // read of the value before it: per tile the S in between sees to that, else
        // the barriers do.
        auto swap = [&](float v, bool before, bool after) {
            if (before) meet();
            *mine = v;
            meet();
            const float o = *other;
            if (after) meet();
            return o;
        };
        const int r = q4 * 32 + lane;  // row of the tile = TMEM lane
        // this thread's running totals, dim c of its half at total[c * 128]
        float* total = a.totals + ((static_cast<long long>(blockIdx.x) * 2 + x) * HD + hf * HW) * 128 + r;
        const int j = r / G, h = r % G;
        const uint32_t lane_addr = static_cast<uint32_t>(q4 * 32) << 16;
        const uint32_t ts = tmem + lane_addr + C::COL_S + x * 128;
        const uint32_t to = tmem + lane_addr + C::COL_O + x * 128;
        const bool capped = a.softcap > 0.0f;
        // This row of item tl's Q tile: rotated, brought into [2^14, 2^15), split into
        // two fp16 parts.  Returns what undoes it, times the scale of scores.
        auto stage_q = [&](const PrefillTile& tl) -> float {
            const int tok = x * TQ + j;
            float qr[HW];
            if (tok < tl.ntok) {
                const long long io = static_cast<long long>(tl.io0) + static_cast<long long>(tok) * tl.io_step;
                const float* src = a.q + io * a.q_stride + static_cast<long long>(tl.kvh * G + h) * HD;
                const float2* cs = a.rope + static_cast<long long>(tl.rope_row0 + tok) * (HD / 2);
                const bool vec = a.q_vec && tl.rope_half % 4 == 0;
#pragma unroll
                for (int d = 0; d < HW; d += 4) {
                    const float4 v = rope4(src, hf * HW + d, tl.rope_half, cs, a.neox != 0, vec);
                    qr[d] = v.x;
                    qr[d + 1] = v.y;
                    qr[d + 2] = v.z;
                    qr[d + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int d = 0; d < HW; ++d) qr[d] = 0.0f;
            }
            float mx = 0.0f;
#pragma unroll
            for (int d = 0; d < HW; ++d) mx = fmaxf(mx, fabsf(qr[d]));
            mx = fmaxf(mx, swap(mx, true, false));
            const int sh = query_exp(mx);
            const float up = exp2_int(sh);
            unsigned char* q = base + C::OFF_Q + 2 * x * C::TILE;
#pragma unroll
            for (int cc = 0; cc < HW / 8; ++cc) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    split_pair<DT_F16T>(qr[8 * cc + 2 * i] * up, qr[8 * cc + 2 * i + 1] * up, hi[i], lo[i]);
                const int c = hf * (HW / 8) + cc;
                const int off = (c / 8) * C::SLAB + r * 128 + (((c % 8) ^ (r & 7)) * 16);
                *reinterpret_cast<uint4*>(q + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(q + C::TILE + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(C::B_QF + x));
            return query_unit(sh, a.scale * kLog2);
        };
        int g = 0, pv = 0;  // phases of S, and of P.V, so far
        float unscale = it_begin < it_end ? stage_q(a.tiles[it_begin]) : 1.0f;
        for (int it = it_begin; it < it_end; ++it) {
            const PrefillTile tl = a.tiles[it];
            const int nt = tiles_of(tl, x);
            const int tok = x * TQ + j;
            const bool live = tok < tl.ntok;
            const int row0 = tl.tok_row0 + x * TQ, row_n = row0 + min(TQ, tl.ntok - x * TQ) - 1;  // of the tile's tokens
            const int hi_r = live ? row0 + j : -1;
            const int lo_r = live && tl.window > 0 ? max(0, hi_r - tl.window + 1) : 0;
            const int lo_all = tl.window > 0 ? max(0, row_n - tl.window + 1) : 0;
            const float2 hs = __ldg(a.head_scale + (static_cast<long long>(tl.seq) * a.scale_layers + tl.cache_layer) *
                                                       a.scale_heads + tl.kvh);
            // raw S -> score, in units of log2; not 0, which times a masked -inf is NaN
            const float mul2 = fmaxf(unscale * hs.x, 1.17549435e-38f);
            float m = -INFINITY, l = 0.0f;  // what weights are taken against (in units of log2)
            float behind = 1.0f;            // what the total is to be multiplied by since it was written
            for (int t = 0; t < nt; ++t, ++g, ++pv) {
                if (t > 0 && t % C::DRAIN == 0) {
                    // O of the tiles so far to the total, while S is being computed; 32
                    // dims at a time, the first ones' totals fetched during the wait
                    float sum[32];
#pragma unroll
                    for (int c = 0; c < HW; ++c) {
                        if (c % 32 == 0) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum[i] = t > C::DRAIN ? __ldcg(total + (c + i) * 128) : 0.0f;
                            if (c == 0) {
                                WAIT(C::B_PV + x, (pv - 1) & 1, 62, g);
                                __syncwarp();
                                tc_fence_after();
                            }
                        }
                        if (c % 16 == 0) {
                            uint32_t o[16];
                            tmem_ld16(to + hf * HW + c, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                __stcg(total + (c + i) * 128, fmaf(sum[c % 32 + i], behind, __uint_as_float(o[i])));
                        }
                    }
                    behind = 1.0f;
                    tc_fence_before();
                }
                WAIT(C::B_SF + x, g & 1, 59, g);
                __syncwarp();
                tc_fence_after();
                const int c0 = tl.kv_lo + t * BN + hf * SW;
                const bool masked = c0 + SW - 1 > row0 || c0 < lo_all;
                uint32_t s[SW];
                tmem_ld64(ts + hf * SW, s);
                tc_fence_before();
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (masked) {
#pragma unroll
                    for (int i = 0; i < SW; ++i) {
                        if (c0 + i < lo_r || c0 + i > hi_r) s[i] = 0xFF800000u;  // -inf
                        mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i]));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < SW; i += 2)
                        mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                }
                float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                mt = fmaxf(mt, swap(mt, false, false));  // both have read their scores, too
                // the score's soft cap is monotone: the capped maximum is the maximum's cap
                mt = capped ? (mt == -INFINITY ? mt : a.cap_out * tanhf(mt * mul2 * a.cap_in)) : mt * mul2;
                const bool move = mt - m > 15.0f;  // (an empty m is -inf, an empty tile's maximum, too)
                if (__any_sync(0xffffffffu, move)) {
                    const float ref = mt - (fabsf(mt) > kFar ? 0.0f : 7.0f);
                    const float f = !move ? 1.0f : (m == -INFINITY ? 0.0f : ex2_approx(m - ref));
                    if (move) {
                        l *= f;
                        behind *= f;
                        m = ref;
                    }
                    // this S was issued after the P.V before it had completed
                    if (t % C::DRAIN != 0) {
#pragma unroll
                        for (int c = 0; c < HW; c += 16) {
                            uint32_t o[16];  // (few: the scores are live)
                            tmem_ld16(to + hf * HW + c, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st16(to + hf * HW + c, o);
                        }
                    }
                }
                const float add = m == -INFINITY ? 0.0f : -m;
                float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                // The fused product below is exact where m is a rounded number: far from
                // zero the difference could leave fp16's range, so such scores are
                // rounded first, as m was.
                const bool far = __any_sync(0xffffffffu, fabsf(m) > kFar && m > -INFINITY);
                if (capped || far) {
#pragma unroll
                    for (int i = 0; i < SW; ++i) {
                        float v = __fmul_rn(__uint_as_float(s[i]), mul2);
                        if (capped) v = v == -INFINITY ? v : a.cap_out * tanhf(v * a.cap_in);
                        s[i] = __float_as_uint(v);
                    }
                }
                const float k = capped || far ? 1.0f : mul2;
#pragma unroll
                for (int c = 0; c < SW; c += 32) {
                    uint32_t hw[16], lw[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float x0 = add, x1 = add;
                        fma_x2(x0, x1, __uint_as_float(s[c + i]), __uint_as_float(s[c + i + 1]), k, k);
                        const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                        add_x2(ls[i & 2], ls[(i & 2) + 1], p0, p1);
                        split_pair<DT_F16T>(p0, p1, hw[i / 2], lw[i / 2]);
                    }
                    // over the scores, which are all in registers
                    tmem_st16(ts + (hf * SW + c) / 2, hw);
                    tmem_st16(ts + 64 + (hf * SW + c) / 2, lw);
                }
                l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(BAR(C::B_PF + x));
            }
            if (nt == 0) {
                WAIT(C::B_SF + x, g & 1, 63, g);
                ++g;
            }
            // the next item's Q while the last P.V runs: every S of this one is done
            const float next = it + 1 < it_end ? stage_q(a.tiles[it + 1]) : 1.0f;
            if (nt > 0) {
                WAIT(C::B_PV + x, (pv - 1) & 1, 60, g);
                __syncwarp();
                tc_fence_after();
                const long long io = static_cast<long long>(tl.io0) + static_cast<long long>(tok) * tl.io_step;
                float* dst = a.out + io * a.q_stride + static_cast<long long>(tl.kvh * G + h) * HD;
                const float lt = l + swap(l, true, true);
                const float inv = lt > 0.0f ? hs.y / lt : 0.0f;
#pragma unroll
                for (int c = 0; c < HW; c += 16) {
                    float sum[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[i] = nt > C::DRAIN ? __ldcg(total + (c + i) * 128) : 0.0f;
                    uint32_t o[16];
                    tmem_ld16(to + hf * HW + c, o);
                    if (live) {
#pragma unroll
                        for (int d = 0; d < 16; d += 4)
                            *reinterpret_cast<float4*>(dst + hf * HW + c + d) = make_float4(
                                fmaf(sum[d], behind, __uint_as_float(o[d])) * inv,
                                fmaf(sum[d + 1], behind, __uint_as_float(o[d + 1])) * inv,
                                fmaf(sum[d + 2], behind, __uint_as_float(o[d + 2])) * inv,
                                fmaf(sum[d + 3], behind, __uint_as_float(o[d + 3])) * inv);
                    }
                    __syncwarp();  // converged for the next .sync.aligned load
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(BAR(C::B_OE + x));  // O may be overwritten
            unscale = next;
        }
    }
#undef WAIT
#undef BAR
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int HD, int G>
cudaError_t launch_one(const PromptArgs& a, const CUtensorMap* tk, const CUtensorMap* tv, int grid, cudaStream_t st) {
    constexpr int smem = PromptCfg<HD>::SMEM;
    static bool set[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !set[dev]) {
        e = cudaFuncSetAttribute(paged_prompt_kernel<HD, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) set[dev] = true;
    }
    paged_prompt_kernel<HD, G><<<grid, kThreads, smem, st>>>(*tk, *tv, a);
    return cudaGetLastError();
}

template <int HD>
cudaError_t launch_g(const PromptArgs& a, const CUtensorMap* tk, const CUtensorMap* tv, int G, int grid, cudaStream_t st) {
    switch (G) {
        case 1: return launch_one<HD, 1>(a, tk, tv, grid, st);
        case 2: return launch_one<HD, 2>(a, tk, tv, grid, st);
        case 4: return launch_one<HD, 4>(a, tk, tv, grid, st);
        case 8: return launch_one<HD, 8>(a, tk, tv, grid, st);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

bool paged_prompt_supported(int hd, int G) {
    return (hd == 64 || hd == 128) && (G == 1 || G == 2 || G == 4 || G == 8);
}

cudaError_t paged_prompt_launch(const PromptArgs& a, const CUtensorMap* tmK, const CUtensorMap* tmV, int hd, int G,
                                int grid, cudaStream_t st) {
    if (!paged_prompt_supported(hd, G)) return cudaErrorInvalidValue;
    return hd == 64 ? launch_g<64>(a, tmK, tmV, G, grid, st) : launch_g<128>(a, tmK, tmV, G, grid, st);
}

}  // namespace jx
