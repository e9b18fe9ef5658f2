// jx_paged_step.cuh -- attention over the paged 8-bit cache for few query rows:
// a decode step (one token per sequence, its k and v appended in the same
// launch), and prompts whose shape the prompt kernel does not take (blocks of
// up to 8 / G tokens of a sequence, rows appended before).
//
//  * Bound by the codes it reads: one byte per element, 2 G multiply-adds each.
//    So every record (32 rows of one kv head: K, V and scales, one contiguous
//    run) goes to shared memory in one bulk copy (head_dim 128 and 256: two, scales
//    and K, then V, so that 8 or 12 warps per SM have three or four in flight) and is
//    read once.  Measured (one B200, kernel alone, int8 or e4m3): 131072 rows of the
//    Mistral-7B shape (8.6 GB) 1.32-1.35 ms = 6.4-6.5 TB/s; 64 ragged sequences of
//    the Llama-3.2-1B shape (4.4 GB) 0.73 ms = 5.95 TB/s (head_dim 64: 420 instructions
//    per 4 KB record, 2.35 per cycle; 128: 770 per 8 KB record, 2.15); one such
//    sequence of 4096 rows (68 MB) 23 us; 100 rows of one layer 8.4 to 11 us.
//  * Work.  Units are (kv head, page) pairs, flattened over sequences, layers
//    and heads; each CTA takes an equal run of them, cut into pieces at segment
//    boundaries (a segment: one kv head of one layer and sequence).  Unit x of
//    a piece goes to warp x % W.  A warp keeps its own ring of records: it waits
//    only for its own copies and refills a stage as soon as it has read it, so
//    no barrier stands between memory and arithmetic within a piece.
//  * Arithmetic: warp-level m16n8k16 products in fp16 with fp32 sums.
//      S^T[row][col] = K[row][:] . q[col][:]    O^T[d][col] += V^T[d][row] P[row][col]
//    A code is exact in fp16: int8 u = code + 128 becomes 1024 + u by one byte
//    permute and code by one subtraction, e4m3 by the conversion instruction.
//    q and the weights are fp32, split into two fp16 parts each (2^-22): the 8
//    columns are (part, head), so a group of 4 heads costs no extra product.
//    The dims of a 16-byte chunk feed four k-steps as they lie in memory (q is
//    laid out to match); V comes through transposed 8x8 loads whose 16-bit
//    elements are pairs of codes, and the permute that builds fp16 numbers also
//    separates the pair: no transposition is paid for.
//  * Scales.  s = q.k 2^kK enters as a factor of the exponent; the weight of a
//    row is taken as 2^(s log2e + kV - m) with kV the exponent of its V block and m
//    a whole number, so that kV - m is exact and one fused multiply-add gives the
//    exponent.  Where scores are beyond 2^22 the reference is a pair, a score m and
//    an exponent c, and the weight 2^((s log2e - m) + (kV - c)): kV would be rounded
//    away in a sum with such a score.  P stays at most 2^15 in fp16 whatever the
//    scales are, O needs no factor per row, and the softmax sum takes back 2^-kV in
//    fp32, once per block.
//  * Split segments: a CTA has at most two pieces that are not whole segments
//    (its first and its last), so two slots of scratch per CTA hold their
//    (o, m, l, c); the CTA that counts in last joins them.
#pragma once

#include <algorithm>
#include <type_traits>

#include "jx_device.cuh"
#include "jx_paged.h"

namespace jx {

template <int HD, int GP>
struct StepCfg {
    static constexpr int W = 4;  // warps per CTA
    // Resident CTAs per SM, as many as the accumulators' registers allow.  (Groups of
    // 5 to 8 heads, 131072 rows: head_dim 128 three CTAs with spills 159 us, two
    // without 131; head_dim 64 four 80, three 73.  Eight columns of head_dim 256 spill
    // 470 bytes all the same.)
    static constexpr int CTAS = HD == 256 ? 2 : HD == 128 ? (GP == 8 ? 2 : 3) : HD == 64 && GP == 8 ? 3 : 4;
    // A stage holds a record, or (wide heads) half of one: scales and K, or V.
    static constexpr bool SPLIT = HD >= 128;
    static constexpr int STAGE = SPLIT ? tile_at(HD, 1) : record_bytes(HD);
    static constexpr int MISC = W * GP * 4 * 4 + 64;  // (m, l, c) of each warp and column; flags
    static constexpr int budget = (227 * 1024) / CTAS - 1024 - MISC - 8;
    static constexpr int fit = budget / (W * (STAGE + 8));
    static constexpr int NS = fit > 8 ? 8 : fit;  // stages per warp
    // floats of a partial result: o [GP][HD], then (m, l, c, -) [GP]; 16-byte aligned
    static constexpr int PART = GP * (HD + 4);
    static_assert(PART <= kStepCols * (HD + 4), "scratch");
    static constexpr int OFF_MISC = W * NS * STAGE;
    static constexpr int OFF_BAR = OFF_MISC + MISC;
    static constexpr int SMEM = OFF_BAR + W * NS * 8 + 8;  // (+ the barrier of test_wait_cta)
    static_assert(NS >= (SPLIT ? 3 : 2), "ring");
    static_assert(OFF_BAR % 8 == 0 && OFF_MISC % 16 == 0, "alignment");
    // a warp's part of a finished piece lies in the stage it read last
    static_assert(GP * HD * 4 <= kPageRows * HD, "result in a V tile");
};

// Rows of an 8-row matrix in the order the lanes take them: two rows read by
// one phase of a 16-byte load then lie in different halves of the banks.
template <int HD>
__device__ __forceinline__ int row_perm(int g) {
    return HD >= 128 ? (g & 1) * 4 + (g >> 1) : g;
}

// One piece: pages page0 .. page0+n-1 of a sequence for one layer and kv head.
struct Piece {
    int run, layer, h;
    int page0, n;
    int in_seg;         // pages of the segment before it
    int seg_x0, seg_n;  // the segment's first unit, and its pages
    int rot;            // its first page goes to warp rot
    bool coop;          // read by all warps of the CTA, page by page in turn; else by warp rot alone
};

// Walks the pieces of units [x, end).  A segment takes kPieceCost units before
// its pages' own: what it costs to start and finish one is counted into a CTA's
// share, which matters where sequences are short.
// A piece that is a whole segment of at most 1/16 of the share is one warp's
// (the next in turn): it starts and ends without a barrier, and without all
// four warps preparing the same q.  The others are read by all warps together.
struct PieceWalk {
    int x, end, r, cls, small, owned;

    __device__ __forceinline__ void init(int x_, int end_) {
        x = x_;
        end = end_;
        r = 0;
        cls = 0;
        small = (end_ - x_) / 16;
        owned = 0;
    }
    // Layers [0, n_full) attend everything, [n_full, n_layers) a window; the
    // windowed ones' units stand behind the others'.
    __device__ __forceinline__ bool next(const PagedArgs& a, Piece& p) {
        while (x < end) {
            if (cls == 0 && x >= a.total0) {
                cls = 1;
                r = 0;
            }
            const int per = (cls ? a.n_layers - a.n_full : a.n_full) * a.n_kv;  // segments of a run
            const int y = x - (cls ? a.total0 : 0);
            auto off = [&](int i) {
                return i < a.n_runs ? (cls ? a.runs[i].off1 : a.runs[i].off) : (cls ? a.units1 : a.units0);
            };
            if (y >= off(r + 1) * per) {  // the run that holds y
                int lo = r + 1, hi = a.n_runs - 1;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (y >= off(mid + 1) * per) lo = mid + 1;
                    else hi = mid;
                }
                r = lo;
            }
            const int first = off(r), len = off(r + 1) - first;
            const int rem = y - first * per;
            const int seg = rem / len, u = rem - seg * len;
            const int n = min(len - u, end - x);
            const int pg = max(0, u - kPieceCost);
            p.n = u + n - kPieceCost - pg;
            p.seg_x0 = x - u;
            x += n;
            if (p.n <= 0) continue;
            p.run = r;
            p.layer = (cls ? a.n_full : 0) + seg / a.n_kv;
            p.h = seg % a.n_kv;
            p.in_seg = pg;
            p.seg_n = len - kPieceCost;
            p.page0 = (cls ? max(0, a.runs[r].pos0 - a.window + 1) / kPageRows : 0) + pg;
            p.coop = p.n < p.seg_n || p.n > small;
            p.rot = (p.coop ? x : owned++) & 3;
            return true;
        }
        return false;
    }
};

// 16-bit pairs from a 32-bit word of codes.
template <int DT>
__device__ __forceinline__ void codes_in_order(uint32_t w, uint32_t& lo, uint32_t& hi) {  // (b0,b1), (b2,b3)
    if constexpr (DT == DT_I8) {
        lo = __byte_perm(w, 0x64646464u, 0x4140);
        hi = __byte_perm(w, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(0x64806480u));
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    }
}
template <int DT>
__device__ __forceinline__ void codes_split(uint32_t w, uint32_t& ev, uint32_t& od) {  // (b0,b2), (b1,b3)
    if constexpr (DT == DT_I8) {
        ev = __byte_perm(w, 0x64646464u, 0x4240);
        od = __byte_perm(w, 0x64646464u, 0x4341);
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(ev) : "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(od) : "r"(0x64806480u));
    } else {
        codes_in_order<DT>(__byte_perm(w, 0u, 0x3120), ev, od);
    }
}

template <int HD, int GP, int DT>
struct StepWarp {
    static constexpr int NBC = (2 * GP + 7) / 8;  // column blocks: (part, head) pairs
    static constexpr int KS = HD / 16;
    // Weights are taken against a reference m + c, about 2^10 below the largest when it
    // is set and moved when a weight would exceed 2^15 (fp16 ends at 2^16).  m is a whole
    // number and c 0, or, scores beyond kFar, m the largest of them.
    static constexpr float kBase = 10.0f, kTop = 15.0f, kFar = 4194304.0f;
    // Parts are joined with their c where the largest m is beyond this: a part whose m
    // is beyond kFar has no weight otherwise.
    static constexpr float kFarJoin = kFar / 2;

    uint32_t qf[KS][NBC][2];
    float o[KS][NBC][4];
    float m[2], l[2];  // m is 0 before the column's first row
    float top[2];      // what a weight's exponent may be: kTop, or -inf before the first row
    float unscale[2];  // of this lane's two columns: a.scale log2(e), and what q was scaled by taken back
    int lo[2], hi[2];  // attended rows of this lane's two columns
    bool far;          // a column of the warp has scores beyond kFar; then each has a c, in shared memory

    __device__ __forceinline__ static float col_sum(const float (&x)[NBC][4], int r) {
        float v = x[0][r];
        if constexpr (NBC == 2) v += x[1][r];
        if constexpr (GP == 1) v += x[0][r ^ 1];
        if constexpr (GP <= 2) v += __shfl_xor_sync(0xffffffffu, v, 1);
        if constexpr (GP <= 4) v += __shfl_xor_sync(0xffffffffu, v, 2);
        return v;
    }
    __device__ __forceinline__ static uint32_t pick(uint32_t h, uint32_t w, int nb, int t) {
        if constexpr (GP == 8) return nb == 0 ? h : w;
        else if constexpr (GP == 4) return t < 2 ? h : w;
        else if constexpr (GP == 2) return t == 0 ? h : (t == 1 ? w : 0u);
        else return t == 0 ? ((h & 0xFFFFu) | (w << 16)) : 0u;
    }

    // Prepares q of a piece: rotated into `tmp` (GP * HD floats of shared memory,
    // this warp's own) by a compact loop, then read back as operands.
    __device__ __forceinline__ void begin(const PagedArgs& a, const Piece& p, float* tmp, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const PagedRun& run = a.runs[p.run];
        const PagedLayer L = a.layers[p.layer];
        const int ncol = run.n * a.G;
        const bool vec = a.q_vec && L.half % 4 == 0;
#pragma unroll 2
        for (int i = lane; i < GP * HD / 4; i += 32) {
            const int col = i / (HD / 4), d = i % (HD / 4) * 4;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (col < ncol) {
                const int tok = run.n > 1 ? col / a.G : 0;
                const long long io = static_cast<long long>(run.io0 + tok) * a.n_io_layers + L.io;
                x = rope4(a.q + io * a.q_stride + (p.h * a.G + col - tok * a.G) * HD, d, L.half,
                          a.rope[L.cfg] + static_cast<long long>(run.pos0 + tok) * (HD / 2), a.neox != 0, vec);
            }
            *reinterpret_cast<float4*>(tmp + 4 * i) = x;
        }
        __syncwarp();
        auto mine = [&](int ks) {  // what this lane takes of column g % GP; its four lanes have all dims
            const int d = HD >= 64 ? (t + 4 * (ks / 4)) * 16 + (ks % 4) * 4 : t * 8 + ks * 4;
            return *reinterpret_cast<const float4*>(tmp + (g % GP) * HD + d);
        };
        // A column's largest |q| is brought into [2^14, 2^15): no bits of the second part
        // are lost to fp16's range.  Each column by itself: a query that is infinite,
        // or far larger than those of the other heads and tokens, is no matter of theirs.
        float mx = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const float4 x = mine(ks);
            mx = fmaxf(fmaxf(mx, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int sh = query_exp(mx);
        const float up = exp2_int(sh);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            unscale[j] = query_unit(__shfl_sync(0xffffffffu, sh, (2 * t + j) % GP * 4), a.scale * 1.4426950408889634f);
        const int part = g / GP;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const float4 x = mine(ks);
            uint32_t h01, l01, h23, l23;
            split_pair<DT_F16T>(x.x * up, x.y * up, h01, l01);
            split_pair<DT_F16T>(x.z * up, x.w * up, h23, l23);
            if constexpr (NBC == 2) {
                qf[ks][0][0] = h01;
                qf[ks][0][1] = h23;
                qf[ks][1][0] = l01;
                qf[ks][1][1] = l23;
            } else {
                qf[ks][0][0] = part == 0 ? h01 : (part == 1 ? l01 : 0u);
                qf[ks][0][1] = part == 0 ? h23 : (part == 1 ? l23 : 0u);
            }
        }
        __syncwarp();  // tmp is read before it is used for something else
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = (2 * t + j) % GP;
            const int pos = run.pos0 + min(col, ncol - 1) / a.G;
            hi[j] = pos;
            lo[j] = (L.flags & kLayerWindow) ? max(0, pos - a.window + 1) : 0;
            m[j] = 0.0f;
            top[j] = -INFINITY;
            l[j] = 0.0f;
        }
        far = false;
#pragma unroll
        for (int mh = 0; mh < KS; ++mh)
#pragma unroll
            for (int nb = 0; nb < NBC; ++nb)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[mh][nb][r] = 0.0f;
    }

    uint32_t bp[2][NBC][2];  // weights of a page as operands

    // l and O by a factor of each column.
    __device__ __forceinline__ void rescale(const float (&w)[2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            l[j] *= w[j];
#pragma unroll
            for (int mh = 0; mh < KS; ++mh)
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb) {
                    o[mh][nb][j] *= w[j];
                    o[mh][nb][j + 2] *= w[j];
                }
        }
    }

    // The largest of a column's rows of a page.
    __device__ __forceinline__ static float largest(const float (&v)[2][4], int j) {
        float t = fmaxf(fmaxf(v[0][j], v[0][j + 2]), fmaxf(v[1][j], v[1][j + 2]));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        return fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
    }

    // What a page does to the references where scores are beyond kFar: x [block][row]
    // (scores) becomes the weights' exponents, w what l and O are to be multiplied by.  A
    // call of its own: inline it would cost the ordinary page registers.
    struct FarPage {
        float x[2][4], kv[2], m[2], c[2], top[2], w[2];
    };
    __device__ __noinline__ static void far_page(FarPage& p) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float z[2][4];
            auto against = [&](float mj, float cj) {
                for (int b = 0; b < 2; ++b)
                    for (int r = j; r < 4; r += 2) z[b][r] = (p.x[b][r] - mj) + (p.kv[b] - cj);
                return largest(z, j);
            };
            const float mx = largest(p.x, j);
            const bool move = against(p.m[j], p.c[j]) > p.top[j], beyond = fabsf(mx) > kFar;
            p.w[j] = 1.0f;
            const float e = against(beyond ? mx : 0.0f, 0.0f);
            if (move) {
                const float m1 = beyond ? mx : rintf(e) - kBase, c1 = beyond ? e - kBase : 0.0f;
                p.w[j] = p.top[j] == -INFINITY ? 0.0f : ex2_approx((p.m[j] - m1) + (p.c[j] - c1));
                p.m[j] = m1;
                p.c[j] = c1;
                p.top[j] = kTop;
            }
            against(p.m[j], p.c[j]);
            for (int b = 0; b < 2; ++b)
                for (int r = j; r < 4; r += 2) p.x[b][r] = z[b][r];
        }
    }

    // Weights of rows row0 .. row0+31 from their K tile and scales.  mlc: where the
    // warp's columns keep their c while `far`.
    __device__ __forceinline__ void scores(const PagedArgs& a, const unsigned char* rec, const float4 sc, int row0,
                                           bool edge, float4* mlc, int lane) {
        const int g = lane >> 2, t = lane & 3;
        float acc[2][NBC][4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int nb = 0; nb < NBC; ++nb)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[b][nb][r] = 0.0f;
        const int rp = row_perm<HD>(g);
        if constexpr (HD >= 64) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int cc = 0; cc < HD / 64; ++cc) {
                    const uint4 k0 = *reinterpret_cast<const uint4*>(rec + tile_byte(HD, b * 16 + rp, (t + 4 * cc) * 16));
                    const uint4 k1 = *reinterpret_cast<const uint4*>(rec + tile_byte(HD, b * 16 + 8 + rp, (t + 4 * cc) * 16));
                    const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        codes_in_order<DT>(w0[i], a0, a2);
                        codes_in_order<DT>(w1[i], a1, a3);
#pragma unroll
                        for (int nb = 0; nb < NBC; ++nb)
                            mma_16816<DT_F16T>(acc[b][nb], a0, a1, a2, a3, qf[cc * 4 + i][nb][0], qf[cc * 4 + i][nb][1]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint2 k0 = *reinterpret_cast<const uint2*>(rec + tile_byte(HD, b * 16 + rp, t * 8));
                const uint2 k1 = *reinterpret_cast<const uint2*>(rec + tile_byte(HD, b * 16 + 8 + rp, t * 8));
                const uint32_t w0[2] = {k0.x, k0.y}, w1[2] = {k1.x, k1.y};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t a0, a1, a2, a3;
                    codes_in_order<DT>(w0[i], a0, a2);
                    codes_in_order<DT>(w1[i], a1, a3);
#pragma unroll
                    for (int nb = 0; nb < NBC; ++nb)
                        mma_16816<DT_F16T>(acc[b][nb], a0, a1, a2, a3, qf[i][nb][0], qf[i][nb][1]);
                }
            }
        }
        // s log2e = d * f; rows b*16 + (r>>1)*8 + perm(g), column slot r&1
        float d[2][4], f[2][2], kv[2], vinv[2], y[2][4];
        const bool capped = a.softcap > 0.0f;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t ve = __float_as_uint(b ? sc.w : sc.z) >> 23;
            kv[b] = static_cast<float>(static_cast<int>(ve) - 127);
            vinv[b] = __uint_as_float((254u - ve) << 23);
            f[b][0] = unscale[0] * (b ? sc.y : sc.x);
            f[b][1] = unscale[1] * (b ? sc.y : sc.x);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                d[b][r] = col_sum(acc[b], r);
            }
        }
        if (capped) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int r = 0; r < 4; ++r) d[b][r] = a.cap_out * tanhf(d[b][r] * f[b][r & 1] * a.cap_in);
                f[b][0] = f[b][1] = 1.0f;
            }
        }
        auto exponents = [&]() {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) y[b][r] = fmaf(d[b][r], f[b][r & 1], kv[b] - m[r & 1]);
            if (edge) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = row0 + b * 16 + (r >> 1) * 8 + rp;
                        if (row < lo[r & 1] || row > hi[r & 1]) y[b][r] = -INFINITY;
                    }
            }
        };
        exponents();
        const float big[2] = {largest(y, 0), largest(y, 1)};
        if (__any_sync(0xffffffffu, far || big[0] > top[0] || big[1] > top[1])) {
            float w[2], mn[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                mn[j] = big[j] > top[j] ? rintf(m[j] + big[j]) - kBase : m[j];
                w[j] = top[j] == -INFINITY ? 0.0f : ex2_approx(m[j] - mn[j]);
            }
            if (__any_sync(0xffffffffu, far || fabsf(mn[0]) > kFar || fabsf(mn[1]) > kFar)) {
                FarPage p;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    p.m[j] = m[j];
                    p.c[j] = far ? mlc[(2 * t + j) % GP].z : 0.0f;
                    p.top[j] = top[j];
                    p.kv[j] = kv[j];
#pragma unroll
                    for (int r = 0; r < 4; ++r)  // scores as rounded numbers (a fused product would
                        // tell equal ones apart from their rounded maximum)
                        p.x[j][r] = y[j][r] == -INFINITY ? -INFINITY : __fmul_rn(d[j][r], f[j][r & 1]);
                }
                far_page(p);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    m[j] = p.m[j];
                    top[j] = p.top[j];
                    w[j] = p.w[j];
                    mlc[(2 * t + j) % GP].z = p.c[j];  // (the lanes of a column write the same)
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[j][r] = p.x[j][r];
                }
                __syncwarp();
                far = __any_sync(0xffffffffu, fabsf(m[0]) > kFar || fabsf(m[1]) > kFar);
                rescale(w);
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    m[j] = mn[j];
                    if (big[j] > top[j]) top[j] = kTop;
                }
                rescale(w);
                exponents();
            }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float pr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) pr[r] = ex2_approx(y[b][r]);
            l[0] = fmaf(pr[0] + pr[2], vinv[b], l[0]);
            l[1] = fmaf(pr[1] + pr[3], vinv[b], l[1]);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                uint32_t h, w;
                split_pair<DT_F16T>(pr[2 * hf], pr[2 * hf + 1], h, w);
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb) bp[b][nb][hf] = movmatrix_trans(pick(h, w, nb, t));
            }
        }
    }

    // O += P V for the page whose weights `scores` left.
    __device__ __forceinline__ void values(uint32_t vbase, int lane) {
        const int i8 = lane >> 3, vr = (i8 & 1) * 8 + row_perm<HD>(lane & 7);
        // A page's 32 rows are summed from zero and then added: the tensor cores cut
        // the sum they add to towards zero (about 1e-8 of it each time), which over
        // the rows of a long cache would add up; an fp32 addition rounds.
#pragma unroll
        for (int c = 0; c < KS; c += 2) {  // chunks of 16 dims, two per load
            float acc[2][NBC][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][nb][r] = 0.0f;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t r0, r1, r2, r3;
                ldsm_x4<true>(vbase + tile_byte(HD, b * 16 + vr, (c + (i8 >> 1)) * 16), r0, r1, r2, r3);
                uint32_t e0, d0, e1, d1;
                codes_split<DT>(r0, e0, d0);
                codes_split<DT>(r1, e1, d1);
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb) mma_16816<DT_F16T>(acc[0][nb], e0, d0, e1, d1, bp[b][nb][0], bp[b][nb][1]);
                codes_split<DT>(r2, e0, d0);
                codes_split<DT>(r3, e1, d1);
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb) mma_16816<DT_F16T>(acc[1][nb], e0, d0, e1, d1, bp[b][nb][0], bp[b][nb][1]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb) {
                    add_x2(o[c + i][nb][0], o[c + i][nb][1], acc[i][nb][0], acc[i][nb][1]);
                    add_x2(o[c + i][nb][2], o[c + i][nb][3], acc[i][nb][2], acc[i][nb][3]);
                }
        }
    }

    // This warp's part of a piece to shared memory: o_s [col][HD], mlc [col](m, l, c), m
    // -inf of a column without rows.
    __device__ __forceinline__ void finish(float* o_s, float4* mlc, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const bool w0 = GP == 8 || (GP == 4 && t < 2) || (GP <= 2 && t == 0);
        const bool w1 = w0 && GP != 1;
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = col_sum(o[c], r);
                if ((r & 1) == 0 ? w0 : w1) o_s[((2 * t + (r & 1)) % GP) * HD + c * 16 + 2 * g + (r >> 1)] = v;
            }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float v = l[j];
            v += __shfl_xor_sync(0xffffffffu, v, 4);
            v += __shfl_xor_sync(0xffffffffu, v, 8);
            v += __shfl_xor_sync(0xffffffffu, v, 16);
            if (g == 0 && (j == 0 ? w0 : w1)) {
                float4& at = mlc[(2 * t + j) % GP];
                at = make_float4(top[j] == -INFINITY ? -INFINITY : m[j], v, far ? at.z : 0.0f, 0.0f);
            }
        }
    }
};

// The step's new row, by the warp whose record (in shared memory: scales, K and
// V tile; in the pool at `home`) receives it: append_kernel's arithmetic, four
// values per lane and turn.  At head_dim up to 64 the warp's halves take K and V
// at once, else one after the other.
template <int HD, int DT>
__device__ __forceinline__ void step_append(const PagedArgs& a, const Piece& p, unsigned char* scales,
                                            unsigned char* kt, unsigned char* vt, unsigned char* home, int lane) {
    constexpr int TURNS = HD <= 64 ? 1 : 2;              // tensors one after the other
    constexpr int SPAN = HD / 4 < 32 ? HD / 4 : 32;      // lanes of a tensor
    constexpr int NG = HD / 4 / SPAN;                    // groups of four per lane
    const PagedRun& run = a.runs[p.run];
    const PagedLayer L = a.layers[p.layer];
    const int row = run.pos0 % kPageRows, blk = row / kBlockRows;
    const bool joins = row % kBlockRows != 0;
    const long long io = static_cast<long long>(run.io0) * a.n_io_layers + L.io;
    const float2* cs = a.rope[L.cfg] + static_cast<long long>(run.pos0) * (HD / 2);
    const bool vec = a.kv_vec && L.half % 4 == 0;
#pragma unroll 1
    for (int turn = 0; turn < TURNS; ++turn) {
        const int which = TURNS == 2 ? turn : lane / SPAN;
        const bool on = which < 2;
        const float* src = (which == 0 ? a.k_in : a.v_in) + io * a.kv_stride + p.h * HD;
        unsigned char* rec = which == 0 ? kt : vt;
        unsigned char* tile = home + tile_at(HD, which & 1);
        float* scale = reinterpret_cast<float*>(scales) + (which & 1) * 2 + blk;
        float4 x[NG];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int d = (lane % SPAN + i * SPAN) * 4;
            x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (on) x[i] = rope4(src, d, which == 0 ? L.half : 0, cs, a.neox != 0, vec);
            x[i] = make_float4(cache_value(x[i].x), cache_value(x[i].y), cache_value(x[i].z), cache_value(x[i].w));
            m = fmaxf(fmaxf(m, fmaxf(fabsf(x[i].x), fabsf(x[i].y))), fmaxf(fabsf(x[i].z), fabsf(x[i].w)));
        }
#pragma unroll
        for (int s = 1; s < SPAN; s <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        const int k_old = joins ? max(kMinExp, scale_exp(*scale)) : kMinExp;
        const int k = max(k_old, block_exp<DT>(m));
        __syncwarp();  // the old scale is read by all before one lane replaces it
        if (on) {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const int d = (lane % SPAN + i * SPAN) * 4;
                const uint32_t c = pack4<DT>(x[i].x, x[i].y, x[i].z, x[i].w, exp2_int(-k));
                *reinterpret_cast<uint32_t*>(rec + tile_byte(HD, row, d)) = c;
                *reinterpret_cast<uint32_t*>(tile + tile_byte(HD, row, d)) = c;
                if (joins && k > k_old) {
                    const float f = exp2_int(k_old - k);
#pragma unroll 1
                    for (int r = blk * kBlockRows; r < row; ++r) {
                        const uint32_t at = tile_byte(HD, r, d);
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + at);
                        const float4 v = unpack4<DT>(w);
                        const uint32_t n = pack4<DT>(v.x, v.y, v.z, v.w, f);
                        *reinterpret_cast<uint32_t*>(rec + at) = n;
                        *reinterpret_cast<uint32_t*>(tile + at) = n;
                    }
                }
            }
            if (lane % SPAN == 0) {
                *scale = exp2_int(k);
                reinterpret_cast<float*>(home)[which * 2 + blk] = exp2_int(k);
            }
        }
    }
    __syncwarp();
    fence_proxy_async_shared();  // these writes before the stages' next bulk copies
    __syncwarp();
}

// The inputs a piece begins with (q, the position's cosines and sines, the new
// k and v) into L2 while the pieces before it are still being read.
template <int HD>
__device__ __forceinline__ void warm_inputs(const PagedArgs& a, const Piece& p, int lane) {
    const PagedRun& run = a.runs[p.run];
    const PagedLayer L = a.layers[p.layer];
    auto warm = [&](const void* at, int bytes) {
        for (int b = lane * 128; b < bytes; b += 32 * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const char*>(at) + b));
    };
    for (int j = 0; j < run.n; ++j) {
        const long long io = static_cast<long long>(run.io0 + j) * a.n_io_layers + L.io;
        warm(a.q + io * a.q_stride + p.h * a.G * HD, a.G * HD * 4);
        warm(a.rope[L.cfg] + static_cast<long long>(run.pos0 + j) * (HD / 2), HD * 4);
        if (a.append && (L.flags & kLayerAppend)) {
            warm(a.k_in + io * a.kv_stride + p.h * HD, HD * 4);
            warm(a.v_in + io * a.kv_stride + p.h * HD, HD * 4);
        }
    }
}

// Elements e .. e+3 of a split segment's sum where m is beyond kFarJoin: each
// part's c counts, too.  Rare, so one part after the other, in a call of its own.
template <int HD, int GP>
__device__ __noinline__ float4 join_far(const float* scratch, int c0, int c1, int e, float* sum) {
    float M = -INFINITY, Cm = 0.0f, Ls = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int c = c0; c <= c1; ++c) {
        const float* src = scratch + static_cast<long long>(c == c0 ? 2 * c0 + 1 : 2 * c) * StepCfg<HD, GP>::PART;
        const float4 mlc = __ldcg(reinterpret_cast<const float4*>(src + GP * HD + 4 * (e / HD)));
        const float4 o = __ldcg(reinterpret_cast<const float4*>(src + e));
        if (mlc.x == -INFINITY) continue;
        const float Mn = fmaxf(M, mlc.x);
        const float x = (M - Mn) + Cm, y = (mlc.x - Mn) + mlc.z, Cn = fmaxf(x, y);
        const float f0 = ex2_approx(x - Cn), f = ex2_approx(y - Cn);
        Ls = fmaf(mlc.y, f, Ls * f0);
        O = make_float4(fmaf(o.x, f, O.x * f0), fmaf(o.y, f, O.y * f0), fmaf(o.z, f, O.z * f0), fmaf(o.w, f, O.w * f0));
        M = Mn;
        Cm = Cn;
    }
    *sum = Ls;
    return O;
}

template <int HD, int GP, int DT>
__global__ void __launch_bounds__(StepCfg<HD, GP>::W * 32, StepCfg<HD, GP>::CTAS)
    paged_step_kernel(const __grid_constant__ PagedArgs a) {
    using C = StepCfg<HD, GP>;
    using SW = StepWarp<HD, GP, DT>;
    constexpr int W = C::W, NS = C::NS;
    static_assert(W == 4, "PieceWalk's rotation");
    extern __shared__ __align__(16) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float4* mlc_s = reinterpret_cast<float4*>(smem + C::OFF_MISC);              // [warp][col](m, l, c)
    int* o_at = reinterpret_cast<int*>(smem + C::OFF_MISC + W * GP * 4 * 4);    // [warp]: its o in smem
    volatile int* abort_flag = o_at + W;
    int* flag = o_at + W + 1;
    unsigned char* ring = smem + warp * NS * C::STAGE;
    const uint32_t ring_u32 = smem_u32(ring);
    const uint32_t bars = smem_u32(smem + C::OFF_BAR) + warp * NS * 8;
    const uint32_t test_bar = smem_u32(smem + C::OFF_BAR) + W * NS * 8;  // nothing ever arrives here
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        mbar_init(test_bar, 1);
    }
    if (lane == 0) {
        for (int s = 0; s < NS; ++s) mbar_init(bars + 8 * s, 1);
        fence_barrier_init();
    }
    __syncthreads();

    const int P = gridDim.x, c = blockIdx.x;
    const int b0 = static_cast<int>(static_cast<long long>(a.total) * c / P);
    const int b1 = static_cast<int>(static_cast<long long>(a.total) * (c + 1) / P);

    // ---- the prefetch cursor: this warp's records (halves), in the order it reads them
    PieceWalk cw;
    cw.init(b0, b1);
    Piece p;
    bool more = cw.next(a, p);
    PieceWalk pw = cw;
    Piece pp = p;
    bool p_more = more;
    int p_i = 0, p_cnt = 0, p_first = 0, p_step = 1, ids = 0;
    const unsigned char* p_base = nullptr;
    const unsigned char* p_src = nullptr;
    bool p_half = false;  // V of the record at p_src is next
    int issued = 0, p_st = 0;
    bool dead = false;    // a wait ran out: nothing more is issued
    auto enter = [&]() {  // the cursor takes up piece pp
        p_i = 0;
        p_step = pp.coop ? W : 1;
        p_first = pp.coop ? (warp - pp.rot) & (W - 1) : 0;  // first own page of the piece
        p_cnt = pp.coop ? (pp.n - p_first + W - 1) / W : (warp == pp.rot ? pp.n : 0);
        p_base = a.pool + a.layers[pp.layer].cache_layer * a.layer_bytes +
                 static_cast<long long>(pp.h) * record_bytes(HD);
    };
    if (more) enter();
    auto prefetch = [&]() {
        if (dead || !p_more) return;
        if (!p_half) {
            while (p_i >= p_cnt) {
                p_more = pw.next(a, pp);
                if (!p_more) return;
                enter();
                if (warp == pp.rot) warm_inputs<HD>(a, pp, lane);
            }
            if (p_i % 32 == 0) {
                const int own = p_i + lane;
                ids = own < p_cnt
                          ? a.table[static_cast<long long>(a.runs[pp.run].seq) * a.max_pages + pp.page0 + p_first + own * p_step]
                          : 0;
            }
            p_src = p_base + __shfl_sync(0xffffffffu, ids, p_i % 32) * a.page_bytes;
            ++p_i;
        }
        if (lane == 0) {
            const uint32_t bytes = C::SPLIT && p_half ? kPageRows * HD : C::STAGE;
            mbar_arrive_expect_tx(bars + 8 * p_st, bytes);
            bulk_load(ring_u32 + p_st * C::STAGE, p_half ? p_src + tile_at(HD, 1) : p_src, bytes, bars + 8 * p_st);
        }
        if constexpr (C::SPLIT) p_half = !p_half;
        ++issued;
        p_st = p_st + 1 == NS ? 0 : p_st + 1;
    };
    // Stages that may be refilled; one of them is kept back at the start and end of
    // a piece, for its q and its result.
    int free_stages = NS;
    auto refill = [&](int keep) {
#pragma unroll 1
        for (; free_stages > keep; --free_stages) prefetch();
    };
    refill(1);

    int c_st = 0;
    uint32_t c_par = 0;  // the stage read next, and its phase
    auto wait = [&](int at, uint32_t par) {
        const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(bars + 8 * at, par, abort_flag, a.err, a.dbg, 40,
                                                                  issued, true, a.wait_limit));
        dead = dead || !ok;
    };
    auto advance = [&]() {
        ++free_stages;
        if (++c_st == NS) {
            c_st = 0;
            c_par ^= 1u;
        }
    };
    if (a.test_wait_cta == c + 1 && warp == 0)
        dead = !__all_sync(0xffffffffu, mbar_wait_bounded(test_bar, 0u, abort_flag, a.err, a.dbg, 42, 0, true, a.wait_limit));
    SW sw;
    for (; more; more = cw.next(a, p)) {
        if (!p.coop && warp != p.rot) continue;
        // the stage kept back: the one read last (at the start, the last one)
        const int l_st = c_st == 0 ? NS - 1 : c_st - 1;
        unsigned char* o_mine = ring + l_st * C::STAGE + (C::SPLIT ? 0 : tile_at(HD, 1));
        const int step = p.coop ? W : 1;
        const int first = p.coop ? (warp - p.rot) & (W - 1) : 0;
        const bool any = first < p.n;
        if (any) {
            sw.begin(a, p, reinterpret_cast<float*>(o_mine), lane);
            fence_proxy_async_shared();  // what the stage held, before its next bulk copy
            __syncwarp();
        }
        const PagedRun& run = a.runs[p.run];
        const PagedLayer L = a.layers[p.layer];
        const int last_row = run.pos0 + run.n - 1;
        // pages every column attends in full need no test of their rows
        const int lo_all = (L.flags & kLayerWindow) ? max(0, last_row - a.window + 1) : 0;
        const int append_page = a.append && (L.flags & kLayerAppend) ? run.pos0 / kPageRows - p.page0 : -1;
        for (int i = first; i < p.n; i += step) {
            refill(0);
            wait(c_st, c_par);
            unsigned char* rec = ring + c_st * C::STAGE;
            unsigned char* vt = rec + tile_at(HD, 1);
            if constexpr (C::SPLIT) {
                const int v_st = c_st + 1 == NS ? 0 : c_st + 1;
                vt = ring + v_st * C::STAGE;
                if (i == append_page) wait(v_st, v_st == 0 ? c_par ^ 1u : c_par);
            }
            const int row0 = (p.page0 + i) * kPageRows;
            if (!dead) {
                if (i == append_page) {
                    const int id = a.table[static_cast<long long>(run.seq) * a.max_pages + p.page0 + i];
                    step_append<HD, DT>(a, p, rec, rec + tile_at(HD, 0), vt,
                                        a.pool + id * a.page_bytes + L.cache_layer * a.layer_bytes +
                                            static_cast<long long>(p.h) * record_bytes(HD), lane);
                }
                sw.scores(a, rec + tile_at(HD, 0), *reinterpret_cast<const float4*>(rec), row0,
                          row0 < lo_all || row0 + kPageRows - 1 > run.pos0, mlc_s + warp * GP, lane);
            }
            if constexpr (C::SPLIT) {
                advance();
                __syncwarp();
                refill(0);  // the K half at once: 131072 rows of the Mistral-7B shape 1.40 -> 1.33 ms
                wait(c_st, c_par);
            }
            if (!dead) sw.values(smem_u32(vt), lane);
            advance();
            __syncwarp();  // every lane has read the stages before they are refilled
        }
        // the last stage read carries the result; the others are refilled meanwhile
        const int r_st = c_st == 0 ? NS - 1 : c_st - 1;
        o_mine = ring + r_st * C::STAGE + (C::SPLIT ? 0 : tile_at(HD, 1));
        refill(1);
        const int ncol = run.n * a.G;
        auto out_at = [&](int col, int d) {  // of a column: a head, or a token's head
            const int tok = run.n > 1 ? col / a.G : 0;
            const long long io = static_cast<long long>(run.io0 + tok) * a.n_io_layers + L.io;
            return a.out + io * a.q_stride + (p.h * a.G + col - tok * a.G) * HD + d;
        };
        if (!p.coop) {
            // a whole segment, read by this warp alone
            float4* mlc = mlc_s + warp * GP;
            sw.finish(reinterpret_cast<float*>(o_mine), mlc, lane);
            __syncwarp();
            for (int e = lane; e < ncol * HD; e += 32) {
                *out_at(e / HD, e % HD) = __fdividef(reinterpret_cast<const float*>(o_mine)[e], mlc[e / HD].y);
            }
            __syncwarp();
            continue;
        }
        if (any) {
            sw.finish(reinterpret_cast<float*>(o_mine), mlc_s + warp * GP, lane);
        } else if (lane < GP) {
            mlc_s[warp * GP + lane] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        }
        if (lane == 0) o_at[warp] = any ? static_cast<int>(o_mine - smem) : -1;
        __syncthreads();
        // ---- the warps' parts joined: the segment's output, or a partial of it
        const bool whole = p.n == p.seg_n;
        float* part = a.scratch + static_cast<long long>(p.in_seg == 0 ? 2 * c + 1 : 2 * c) * C::PART;
#pragma unroll 1
        for (int e = threadIdx.x * 2; e < ncol * HD; e += W * 32 * 2) {
            const int col = e / HD, d = e % HD;
            float2 ml[W];
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                ml[w] = *reinterpret_cast<const float2*>(mlc_s + w * GP + col);
                M = fmaxf(M, ml[w].x);
            }
#pragma unroll
            for (int w = 0; w < W; ++w) ml[w].x = ml[w].x == -INFINITY ? -INFINITY : ml[w].x - M;
            float Cm = 0.0f;  // of the sum, as M
            if (fabsf(M) > SW::kFarJoin && M > -INFINITY) {
                Cm = -INFINITY;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    ml[w].x += mlc_s[w * GP + col].z;
                    Cm = fmaxf(Cm, ml[w].x);
                }
#pragma unroll
                for (int w = 0; w < W; ++w) ml[w].x -= Cm;
            }
            float Ls = 0.0f;
            float2 O = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (o_at[w] < 0 || ml[w].x == -INFINITY) continue;  // no pages, or no rows of them
                const float f = ex2_approx(ml[w].x);
                const float2 o = *reinterpret_cast<const float2*>(smem + o_at[w] + e * 4);
                Ls = fmaf(ml[w].y, f, Ls);
                O = make_float2(fmaf(o.x, f, O.x), fmaf(o.y, f, O.y));
            }
            if (whole) {
                float* dst = out_at(col, d);
                const float inv = __fdividef(1.0f, Ls);
                dst[0] = O.x * inv;
                dst[1] = O.y * inv;
            } else {
                *reinterpret_cast<float2*>(part + e) = O;
                if (d == 0) *reinterpret_cast<float4*>(part + GP * HD + 4 * col) = make_float4(M, Ls, Cm, 0.0f);
            }
        }
        if (!whole) {
            const int c0 = static_cast<int>(owner_of(p.seg_x0 + kPieceCost, a.total, P));
            const int c1 = static_cast<int>(owner_of(p.seg_x0 + kPieceCost + p.seg_n - 1, a.total, P));
            __syncthreads();
            if (threadIdx.x == 0) *flag = atomic_add_acq_rel_gpu(a.counters + c0, 1) == c1 - c0;
            __syncthreads();
            if (*flag) {
                // the last of the segment's CTAs
                if (threadIdx.x == 0) a.counters[c0] = 0;
                fence_acq_rel_gpu();
                constexpr int Q = 8;  // parts whose loads are in flight together
                for (int e = threadIdx.x * 4; e < ncol * HD; e += W * 32 * 4) {
                    const int col = e / HD, d = e % HD;
                    float M = -INFINITY, Ls = 0.0f;
                    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int q0 = c0; q0 <= c1; q0 += Q) {
                        float2 ml[Q];
                        float4 ov[Q];
#pragma unroll
                        for (int q = 0; q < Q; ++q) {
                            // beyond the last part: the last one again, with no weight
                            const int cq = min(q0 + q, c1);
                            const float* src = a.scratch + static_cast<long long>(cq == c0 ? 2 * c0 + 1 : 2 * cq) * C::PART;
                            ml[q] = __ldcg(reinterpret_cast<const float2*>(src + GP * HD + 4 * col));
                            ov[q] = __ldcg(reinterpret_cast<const float4*>(src + e));
                            if (q0 + q > c1) ml[q].x = -INFINITY;
                        }
                        float Mn = M;
#pragma unroll
                        for (int q = 0; q < Q; ++q) Mn = fmaxf(Mn, ml[q].x);
                        if (Mn == -INFINITY) continue;
                        const float f0 = M == -INFINITY ? 0.0f : ex2_approx(M - Mn);
                        Ls *= f0;
                        O = make_float4(O.x * f0, O.y * f0, O.z * f0, O.w * f0);
#pragma unroll
                        for (int q = 0; q < Q; ++q) {
                            const float f = ml[q].x == -INFINITY ? 0.0f : ex2_approx(ml[q].x - Mn);
                            Ls = fmaf(ml[q].y, f, Ls);
                            O = make_float4(fmaf(ov[q].x, f, O.x), fmaf(ov[q].y, f, O.y), fmaf(ov[q].z, f, O.z),
                                            fmaf(ov[q].w, f, O.w));
                        }
                        M = Mn;
                    }
                    if (fabsf(M) > SW::kFarJoin && M > -INFINITY) O = join_far<HD, GP>(a.scratch, c0, c1, e, &Ls);
                    float* dst = out_at(col, d);
                    const float inv = __fdividef(1.0f, Ls);
                    dst[0] = O.x * inv;
                    dst[1] = O.y * inv;
                    dst[2] = O.z * inv;
                    dst[3] = O.w * inv;
                }
            }
        }
        __syncthreads();  // o, mlc_s and flag are read before they are written again
    }
    // every copy has landed before the CTA exits, after a wait that ran out too
    for (int k = max(0, issued - NS); k < issued; ++k)
        mbar_wait_bounded(bars + 8 * (k % NS), (k / NS) & 1, abort_flag, a.err, a.dbg, 41, k, false, kDrainLimitCycles);
}

template <int HD, int DT, int GP>
cudaError_t step_launch_one(const PagedArgs& a, int num_sms, cudaStream_t st) {
    using C = StepCfg<HD, GP>;
    static_assert(C::CTAS <= kStepCtasPerSm, "scratch holds two slots for each CTA");
    static bool set[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !set[dev]) {
        e = cudaFuncSetAttribute(paged_step_kernel<HD, GP, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) set[dev] = true;
    }
    // no more CTAs than give each warp a page
    const int per = C::W + kPieceCost;
    const int grid = std::max(1, std::min(num_sms * C::CTAS, (a.total + per - 1) / per));
    paged_step_kernel<HD, GP, DT><<<grid, C::W * 32, C::SMEM, st>>>(a);
    return cudaGetLastError();
}

// Launches the kernel for head_dim and columns (heads, times a block's tokens).
template <int DT>
cudaError_t step_launch_dt(const PagedArgs& a, int hd, int cols, int num_sms, cudaStream_t st) {
    auto with_gp = [&](auto hdv) {
        constexpr int HD = decltype(hdv)::value;
        if (cols <= 1) return step_launch_one<HD, DT, 1>(a, num_sms, st);
        if (cols <= 2) return step_launch_one<HD, DT, 2>(a, num_sms, st);
        if (cols <= 4) return step_launch_one<HD, DT, 4>(a, num_sms, st);
        return step_launch_one<HD, DT, 8>(a, num_sms, st);
    };
    switch (hd) {
        case 32: return with_gp(std::integral_constant<int, 32>{});
        case 64: return with_gp(std::integral_constant<int, 64>{});
        case 128: return with_gp(std::integral_constant<int, 128>{});
        default: return with_gp(std::integral_constant<int, 256>{});
    }
}

}  // namespace jx
