// jx_paged_step.cuh -- attention over the paged 8-bit cache for few query rows:
// a decode step (one token per sequence, its k and v appended in the same
// launch), and prompts whose shape the prompt kernel does not take (blocks of
// up to 8 / G tokens of a sequence, rows appended before).
//
//  * Bound by the codes it reads: one byte per element, 2 G multiply-adds each.
//    So every record (32 rows of one kv head: K, V and scales, one contiguous
//    run) goes to shared memory in ONE bulk copy and is read once.
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
//    row is taken as 2^(s log2e + kV - m) with kV the exponent of its V block,
//    and the running maximum m is over that sum.  P stays at most 2^15 in
//    fp16 whatever the scales are, O needs no factor per row, and the softmax
//    sum takes back 2^-kV in fp32, once per block.
//  * Split segments: a CTA has at most two pieces that are not whole segments
//    (its first and its last), so two slots of scratch per CTA hold their
//    (o, m, l); the CTA that counts in last joins them.
#pragma once

#include <algorithm>
#include <type_traits>

#include "jx_device.cuh"
#include "jx_paged.h"

namespace jx {

template <int HD, int GP>
struct StepCfg {
    static constexpr int R = record_bytes(HD);
    static constexpr int W = 4;                        // warps
    static constexpr int CTAS = HD == 256 ? 1 : 2;  // resident per SM
    // ring stages per warp: as many records as the SM's shared memory holds
    static constexpr int O_BYTES = W * GP * HD * 4;
    static constexpr int ML_BYTES = W * GP * 2 * 4;
    static constexpr int MISC = 64;
    static constexpr int budget = (227 * 1024) / CTAS - 1024 - O_BYTES - ML_BYTES - MISC;
    static constexpr int fit = budget / (W * (R + 8));
    static constexpr int NS = fit > 8 ? 8 : fit;
    static constexpr int OFF_O = W * NS * R;
    static constexpr int OFF_ML = OFF_O + O_BYTES;
    static constexpr int OFF_BAR = OFF_ML + ML_BYTES;
    static constexpr int OFF_MISC = OFF_BAR + W * NS * 8;
    static constexpr int SMEM = OFF_MISC + MISC;
    static_assert(NS >= 2, "ring");
    static_assert(OFF_BAR % 8 == 0 && OFF_O % 16 == 0, "alignment");
};

// Rows of an 8-row matrix in the order the lanes take them: two rows read by
// one phase of a 16-byte load then lie in different halves of the banks.
template <int HD>
__device__ __forceinline__ int row_perm(int g) {
    return HD >= 128 ? (g & 1) * 4 + (g >> 1) : g;
}

// One piece: units [x0, x0 + n) of the flattened space, pages page0 .. of a segment.
struct Piece {
    int run, layer, h;
    int page0, n;
    int x0;
    int seg_x0, seg_n;  // the whole segment
};

// Walks the pieces of units [x, end).
struct PieceWalk {
    int x, end, r, cls;

    __device__ __forceinline__ void init(int x_, int end_) {
        x = x_;
        end = end_;
        r = 0;
        cls = 0;
    }
    // Layers [0, n_full) attend everything, [n_full, n_layers) a window; the
    // windowed ones' units stand behind the others'.
    __device__ __forceinline__ bool next(const PagedArgs& a, Piece& p) {
        if (x >= end) return false;
        if (cls == 0 && x >= a.total0) {
            cls = 1;
            r = 0;
        }
        const int base = cls ? a.total0 : 0;
        const int per = (cls ? a.n_layers - a.n_full : a.n_full) * a.n_kv;  // segments of a run
        const int y = x - base;
        int first = cls ? a.runs[r].off1 : a.runs[r].off;
        int next_off = r + 1 < a.n_runs ? (cls ? a.runs[r + 1].off1 : a.runs[r + 1].off) : (cls ? a.pages1 : a.pages0);
        while (y >= next_off * per) {
            ++r;
            first = next_off;
            next_off = r + 1 < a.n_runs ? (cls ? a.runs[r + 1].off1 : a.runs[r + 1].off) : (cls ? a.pages1 : a.pages0);
        }
        const int np = next_off - first;
        const int rem = y - first * per;
        const int seg = rem / np, pg = rem - seg * np;
        p.run = r;
        p.layer = (cls ? a.n_full : 0) + seg / a.n_kv;
        p.h = seg % a.n_kv;
        const int pos0 = a.runs[r].pos0;
        p.page0 = (cls ? max(0, pos0 - a.window + 1) / kPageRows : 0) + pg;
        p.x0 = x;
        p.seg_x0 = x - pg;
        p.seg_n = np;
        p.n = min(np - pg, end - x);
        x += p.n;
        return true;
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

// Four consecutive dims of a rotated head.  vec: 16-byte loads are possible and
// a group of four does not cross the end of the rotated part.
__device__ __forceinline__ float4 rope4(const float* x, int d, int half, const float2* cs, bool neox, bool vec) {
    if (!vec)
        return make_float4(rope_plain(x, d, half, cs, neox), rope_plain(x, d + 1, half, cs, neox),
                           rope_plain(x, d + 2, half, cs, neox), rope_plain(x, d + 3, half, cs, neox));
    const float4 v = *reinterpret_cast<const float4*>(x + d);
    if (d >= 2 * half) return v;
    if (neox) {
        const bool first = d < half;
        const int j = first ? d : d - half;
        const float4 w = *reinterpret_cast<const float4*>(x + (first ? d + half : d - half));
        const float4 c0 = *reinterpret_cast<const float4*>(cs + j);
        const float4 c1 = *reinterpret_cast<const float4*>(cs + j + 2);
        auto rot = [&](float mine, float other, float c, float s) {
            return first ? __fsub_rn(__fmul_rn(mine, c), __fmul_rn(other, s))
                         : __fadd_rn(__fmul_rn(other, s), __fmul_rn(mine, c));
        };
        return make_float4(rot(v.x, w.x, c0.x, c0.y), rot(v.y, w.y, c0.z, c0.w), rot(v.z, w.z, c1.x, c1.y),
                           rot(v.w, w.w, c1.z, c1.w));
    }
    const float4 c = *reinterpret_cast<const float4*>(cs + d / 2);
    return make_float4(__fsub_rn(__fmul_rn(v.x, c.x), __fmul_rn(v.y, c.y)),
                       __fadd_rn(__fmul_rn(v.x, c.y), __fmul_rn(v.y, c.x)),
                       __fsub_rn(__fmul_rn(v.z, c.z), __fmul_rn(v.w, c.w)),
                       __fadd_rn(__fmul_rn(v.z, c.w), __fmul_rn(v.w, c.z)));
}

template <int HD, int GP, int DT>
struct StepWarp {
    static constexpr int NBC = (2 * GP + 7) / 8;  // column blocks: (part, head) pairs
    static constexpr int KS = HD / 16;
    static constexpr int kBase = 10;              // a weight of 1 is 2^10 in fp16 (at most 2^15)
    static constexpr float kLazy = 5.0f;          // the maximum moves when exceeded by 2^5

    uint32_t qf[KS][NBC][2];
    float o[KS][NBC][4];
    float m[2], l[2];
    float unscale[2];
    int lo[2], hi[2];  // attended rows of this lane's two columns

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

    __device__ __forceinline__ void begin(const PagedArgs& a, const Piece& p, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const PagedRun& run = a.runs[p.run];
        const PagedLayer L = a.layers[p.layer];
        const int ncol = run.n * a.G;
        float mx = 0.0f;
        float4 x[KS];
        {
            const int col = g % GP, part = g / GP;
            const int tok = col / a.G;
            const bool use = col < ncol && (NBC == 2 || part < 2);
            const long long io = static_cast<long long>(run.io0 + tok) * a.n_io_layers + L.io;
            const float* src = a.q + io * a.q_stride + (p.h * a.G + col % a.G) * HD;
            const float2* cs = a.rope[L.cfg] + static_cast<long long>(run.pos0 + tok) * (HD / 2);
            const bool vec = a.q_vec && L.half % 4 == 0;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = HD >= 64 ? (t + 4 * (ks / 4)) * 16 + (ks % 4) * 4 : t * 8 + ks * 4;
                x[ks] = use ? rope4(src, d, L.half, cs, a.neox != 0, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
                mx = fmaxf(fmaxf(mx, fmaxf(fabsf(x[ks].x), fabsf(x[ks].y))), fmaxf(fabsf(x[ks].z), fabsf(x[ks].w)));
            }
            // each head's largest |q| is brought into [2^14, 2^15): no bits of the
            // second part are lost to fp16's range
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const int e = static_cast<int>((__float_as_uint(mx) >> 23) & 0xFFu) - 127;
            const int sh = min(60, max(-60, 14 - e));
            const float up = exp2_int(sh), down = exp2_int(-sh);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t h01, l01, h23, l23;
                split_pair<DT_F16T>(x[ks].x * up, x[ks].y * up, h01, l01);
                split_pair<DT_F16T>(x[ks].z * up, x[ks].w * up, h23, l23);
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
#pragma unroll
            for (int j = 0; j < 2; ++j) unscale[j] = __shfl_sync(0xffffffffu, down, ((2 * t + j) % GP) * 4);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int col = (2 * t + j) % GP;
            const int pos = run.pos0 + min(col, ncol - 1) / a.G;
            hi[j] = pos;
            lo[j] = (L.flags & kLayerWindow) ? max(0, pos - a.window + 1) : 0;
            m[j] = -INFINITY;
            l[j] = 0.0f;
        }
#pragma unroll
        for (int mh = 0; mh < KS; ++mh)
#pragma unroll
            for (int nb = 0; nb < NBC; ++nb)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[mh][nb][r] = 0.0f;
    }

    // One record in shared memory at `rec`, rows row0 .. row0+31.
    __device__ __forceinline__ void page(const PagedArgs& a, const unsigned char* rec, int row0, bool edge, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const float4 sc = *reinterpret_cast<const float4*>(rec + 2 * kPageRows * HD);
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
        // exponents: x = s log2e + kV; rows b*16 + (r>>1)*8 + perm(g), column slot r&1
        float x[2][4];
        float vinv[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const float ks = b ? sc.y : sc.x;
            const uint32_t ve = __float_as_uint(b ? sc.w : sc.z) >> 23;
            const float kv = static_cast<float>(static_cast<int>(ve) - 127);
            vinv[b] = __uint_as_float((254u - ve) << 23);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float s = col_sum(acc[b], r) * (unscale[r & 1] * ks);
                s *= a.scale;
                if (a.softcap > 0.0f) s = a.softcap * tanhf(s * a.inv_softcap);
                s = fmaf(s, 1.4426950408889634f, kv);
                if (edge) {
                    const int row = row0 + b * 16 + (r >> 1) * 8 + rp;
                    if (row < lo[r & 1] || row > hi[r & 1]) s = -INFINITY;
                }
                x[b][r] = s;
            }
        }
        float mt[2];
        bool move = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            mt[j] = fmaxf(fmaxf(x[0][j], x[0][j + 2]), fmaxf(x[1][j], x[1][j + 2]));
            mt[j] = fmaxf(mt[j], __shfl_xor_sync(0xffffffffu, mt[j], 4));
            mt[j] = fmaxf(mt[j], __shfl_xor_sync(0xffffffffu, mt[j], 8));
            mt[j] = fmaxf(mt[j], __shfl_xor_sync(0xffffffffu, mt[j], 16));
            move = move || mt[j] > m[j] + kLazy || (m[j] == -INFINITY && mt[j] > -INFINITY);
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float mn = fmaxf(m[j], mt[j]);
                const float f = m[j] == -INFINITY ? 0.0f : ex2_approx(m[j] - mn);
                m[j] = mn;
                l[j] *= f;
#pragma unroll
                for (int mh = 0; mh < KS; ++mh)
#pragma unroll
                    for (int nb = 0; nb < NBC; ++nb) {
                        o[mh][nb][j] *= f;
                        o[mh][nb][j + 2] *= f;
                    }
            }
        }
        uint32_t bp[2][NBC][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float pr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float mr = m[r & 1] == -INFINITY ? 0.0f : m[r & 1];
                pr[r] = ex2_approx(x[b][r] - mr + static_cast<float>(kBase));
            }
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
        const int i8 = lane >> 3, vr = (i8 & 1) * 8 + row_perm<HD>(lane & 7);
        const uint32_t vbase = smem_u32(rec) + kPageRows * HD;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int c = 0; c < KS; c += 2) {  // chunks of 16 dims, two per load
                uint32_t r0, r1, r2, r3;
                ldsm_x4<true>(vbase + tile_byte(HD, b * 16 + vr, (c + (i8 >> 1)) * 16), r0, r1, r2, r3);
                uint32_t e0, d0, e1, d1;
                codes_split<DT>(r0, e0, d0);
                codes_split<DT>(r1, e1, d1);
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb) mma_16816<DT_F16T>(o[c][nb], e0, d0, e1, d1, bp[b][nb][0], bp[b][nb][1]);
                codes_split<DT>(r2, e0, d0);
                codes_split<DT>(r3, e1, d1);
#pragma unroll
                for (int nb = 0; nb < NBC; ++nb)
                    mma_16816<DT_F16T>(o[c + 1][nb], e0, d0, e1, d1, bp[b][nb][0], bp[b][nb][1]);
            }
        }
    }

    // This warp's (o, m, l) of the piece to shared memory: o_s [warp][col][HD],
    // ml_s [warp][col][2].
    __device__ __forceinline__ void finish(float* o_s, float* ml_s, int lane) {
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
                ml_s[((2 * t + j) % GP) * 2] = m[j];
                ml_s[((2 * t + j) % GP) * 2 + 1] = v;
            }
        }
    }
};

// The step's new row, by the warp whose record (in shared memory at `rec`, in
// the pool at `home`) receives it: the same arithmetic and thread layout as
// append_kernel, one lane per 16 values.
template <int HD, int DT>
__device__ __forceinline__ void step_append(const PagedArgs& a, const Piece& p, unsigned char* rec,
                                            unsigned char* home, int lane) {
    constexpr int CPR = HD / 16;
    const PagedRun& run = a.runs[p.run];
    const PagedLayer L = a.layers[p.layer];
    const int which = lane / CPR, d0 = lane % CPR * 16;
    const int row = run.pos0 % kPageRows, blk = row / kBlockRows;
    const uint32_t tile = static_cast<uint32_t>(which * kPageRows * HD);
    const uint32_t at_scale = 2 * kPageRows * HD + (which * 2 + blk) * 4;
    const bool on = which < 2;
    float x[16];
    float m = 0.0f;
    if (on) {
        const long long io = static_cast<long long>(run.io0) * a.n_io_layers + L.io;
        const float* src = (which ? a.v_in : a.k_in) + io * a.kv_stride + p.h * HD;
        const float2* cs = a.rope[L.cfg] + static_cast<long long>(run.pos0) * (HD / 2);
        const bool vec = a.kv_vec && L.half % 4 == 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = rope4(src, d0 + 4 * i, which ? 0 : L.half, cs, a.neox != 0, vec);
            x[4 * i] = cache_value(v.x);
            x[4 * i + 1] = cache_value(v.y);
            x[4 * i + 2] = cache_value(v.z);
            x[4 * i + 3] = cache_value(v.w);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(x[i]));
    }
#pragma unroll
    for (int s = 1; s < CPR; s <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    const bool joins = row % kBlockRows != 0;
    const int k_old = on && joins ? max(kMinExp, scale_exp(*reinterpret_cast<float*>(rec + at_scale))) : kMinExp;
    __syncwarp();  // the old scale is read by all before one lane replaces it
    if (on) {
        const int k = max(k_old, block_exp<DT>(m));
        const uint4 c = pack_codes<DT>(x, exp2_int(-k));
        *reinterpret_cast<uint4*>(rec + tile + tile_byte(HD, row, d0)) = c;
        *reinterpret_cast<uint4*>(home + tile + tile_byte(HD, row, d0)) = c;
        if (joins && k > k_old)
            for (int r = blk * kBlockRows; r < row; ++r) {
                const uint32_t at = tile + tile_byte(HD, r, d0);
                unpack_codes<DT>(*reinterpret_cast<const uint4*>(rec + at), x);
                const uint4 cr = pack_codes<DT>(x, exp2_int(k_old - k));
                *reinterpret_cast<uint4*>(rec + at) = cr;
                *reinterpret_cast<uint4*>(home + at) = cr;
            }
        if (d0 == 0) {
            *reinterpret_cast<float*>(rec + at_scale) = exp2_int(k);
            *reinterpret_cast<float*>(home + at_scale) = exp2_int(k);
        }
    }
    __syncwarp();
    fence_proxy_async_shared();  // these writes before the stage's next bulk copy
    __syncwarp();
}

template <int HD, int GP, int DT>
__global__ void __launch_bounds__(StepCfg<HD, GP>::W * 32, StepCfg<HD, GP>::CTAS)
    paged_step_kernel(const __grid_constant__ PagedArgs a) {
    using C = StepCfg<HD, GP>;
    constexpr int W = C::W, NS = C::NS;
    extern __shared__ __align__(16) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* o_s = reinterpret_cast<float*>(smem + C::OFF_O);
    float* ml_s = reinterpret_cast<float*>(smem + C::OFF_ML);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
    int* flag = reinterpret_cast<int*>(smem + C::OFF_MISC) + 1;
    unsigned char* ring = smem + warp * NS * C::R;
    const uint32_t ring_u32 = smem_u32(ring);
    const uint32_t bars = smem_u32(smem + C::OFF_BAR) + warp * NS * 8;
    if (threadIdx.x == 0) *abort_flag = 0;
    if (lane == 0) {
        for (int s = 0; s < NS; ++s) mbar_init(bars + 8 * s, 1);
        fence_barrier_init();
    }
    __syncthreads();

    const int P = gridDim.x, c = blockIdx.x;
    const int b0 = static_cast<int>(static_cast<long long>(a.total) * c / P);
    const int b1 = static_cast<int>(static_cast<long long>(a.total) * (c + 1) / P);

    // ---- the prefetch cursor: this warp's records, in the order it reads them
    PieceWalk pw;
    pw.init(b0, b1);
    Piece pp;
    pp.n = 0;
    int p_i = 0, p_cnt = 0, p_first = 0, ids = 0;
    const unsigned char* p_base = nullptr;
    int issued = 0, used = 0;
    auto prefetch = [&]() {
        while (p_i >= p_cnt) {
            if (!pw.next(a, pp)) return;
            p_first = (warp - pp.x0 % W + W) % W;  // first own page of the piece
            p_cnt = (pp.n - p_first + W - 1) / W;
            p_i = 0;
            p_base = a.pool + a.layers[pp.layer].cache_layer * a.layer_bytes + static_cast<long long>(pp.h) * C::R;
        }
        if (p_i % 32 == 0) {
            const int own = p_i + lane;
            ids = own < p_cnt ? a.table[static_cast<long long>(a.runs[pp.run].seq) * a.max_pages + pp.page0 + p_first + own * W] : 0;
        }
        const int id = __shfl_sync(0xffffffffu, ids, p_i % 32);
        ++p_i;
        if (__shfl_sync(0xffffffffu, *abort_flag, 0)) return;
        const int st = issued % NS;
        ++issued;
        if (lane == 0) {
            mbar_arrive_expect_tx(bars + 8 * st, C::R);
            bulk_load(ring_u32 + st * C::R, p_base + id * a.page_bytes, C::R, bars + 8 * st);
        }
    };
#pragma unroll 1
    for (int s = 0; s < NS; ++s) prefetch();

    PieceWalk cw;
    cw.init(b0, b1);
    Piece p;
    StepWarp<HD, GP, DT> sw;
    while (cw.next(a, p)) {
        sw.begin(a, p, lane);
        const PagedRun& run = a.runs[p.run];
        const PagedLayer L = a.layers[p.layer];
        const int last_row = run.pos0 + run.n - 1;
        // pages every column attends in full need no test of their rows
        const int lo_all = (L.flags & kLayerWindow) ? max(0, last_row - a.window + 1) : 0;
        for (int i = (warp - p.x0 % W + W) % W; i < p.n; i += W) {
            const int st = used % NS;
            const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(bars + 8 * st, (used / NS) & 1, abort_flag, a.err,
                                                                      a.dbg, 40, used, true, a.wait_limit));
            ++used;
            unsigned char* rec = ring + st * C::R;
            const int row0 = (p.page0 + i) * kPageRows;
            if (ok) {
                if (a.append && (L.flags & kLayerAppend) && run.pos0 / kPageRows == p.page0 + i) {
                    const int id = a.table[static_cast<long long>(run.seq) * a.max_pages + p.page0 + i];
                    step_append<HD, DT>(a, p, rec, a.pool + id * a.page_bytes + L.cache_layer * a.layer_bytes +
                                                       static_cast<long long>(p.h) * C::R, lane);
                }
                sw.page(a, rec, row0, row0 < lo_all || row0 + kPageRows - 1 > run.pos0, lane);
            }
            __syncwarp();  // every lane has read the record before it is overwritten
            prefetch();
        }
        sw.finish(o_s + warp * GP * HD, ml_s + warp * GP * 2, lane);
        __syncthreads();
        // ---- the warps' parts joined: the segment's output, or a partial of it
        const bool whole = p.n == p.seg_n;
        const int ncol = run.n * a.G;
        float* part = a.scratch + static_cast<long long>(p.x0 == b0 ? 2 * c : 2 * c + 1) * (GP * (HD + 2));
        for (int e = threadIdx.x; e < ncol * HD; e += W * 32) {
            const int col = e / HD, d = e % HD;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; ++w) M = fmaxf(M, ml_s[(w * GP + col) * 2]);
            float Ls = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float mw = ml_s[(w * GP + col) * 2];
                const float f = mw == -INFINITY ? 0.0f : ex2_approx(mw - M);
                Ls = fmaf(ml_s[(w * GP + col) * 2 + 1], f, Ls);
                O = fmaf(o_s[(w * GP + col) * HD + d], f, O);
            }
            if (whole) {
                const long long io = static_cast<long long>(run.io0 + col / a.G) * a.n_io_layers + L.io;
                a.out[io * a.q_stride + (p.h * a.G + col % a.G) * HD + d] = O / Ls;
            } else {
                part[col * (HD + 2) + d] = O;
                if (d == 0) {
                    part[col * (HD + 2) + HD] = M;
                    part[col * (HD + 2) + HD + 1] = Ls;
                }
            }
        }
        if (!whole) {
            const int c0 = static_cast<int>(owner_of(p.seg_x0, a.total, P));
            const int c1 = static_cast<int>(owner_of(p.seg_x0 + p.seg_n - 1, a.total, P));
            __syncthreads();
            if (threadIdx.x == 0) *flag = atomic_add_acq_rel_gpu(a.counters + c0, 1) == c1 - c0;
            __syncthreads();
            if (*flag) {
                // the last of the segment's CTAs
                if (threadIdx.x == 0) a.counters[c0] = 0;
                fence_acq_rel_gpu();
                const int s0 = p.seg_x0 == static_cast<int>(static_cast<long long>(a.total) * c0 / P) ? 2 * c0 : 2 * c0 + 1;
                constexpr int Q = 8;
                for (int e = threadIdx.x; e < ncol * HD; e += W * 32) {
                    const int col = e / HD, d = e % HD;
                    float M = -INFINITY, Ls = 0.0f, O = 0.0f;
                    for (int q0 = c0; q0 <= c1; q0 += Q) {
                        float mv[Q], lv[Q], ov[Q];
#pragma unroll
                        for (int q = 0; q < Q; ++q) {
                            const bool on = q0 + q <= c1;
                            const float* src = a.scratch + static_cast<long long>(q0 + q == c0 ? s0 : 2 * (q0 + q)) * (GP * (HD + 2)) + col * (HD + 2);
                            mv[q] = on ? __ldcg(src + HD) : -INFINITY;
                            lv[q] = on ? __ldcg(src + HD + 1) : 0.0f;
                            ov[q] = on ? __ldcg(src + d) : 0.0f;
                        }
                        float Mn = M;
#pragma unroll
                        for (int q = 0; q < Q; ++q) Mn = fmaxf(Mn, mv[q]);
                        if (Mn == -INFINITY) continue;
                        const float f0 = M == -INFINITY ? 0.0f : ex2_approx(M - Mn);
                        Ls *= f0;
                        O *= f0;
#pragma unroll
                        for (int q = 0; q < Q; ++q) {
                            const float f = mv[q] == -INFINITY ? 0.0f : ex2_approx(mv[q] - Mn);
                            Ls = fmaf(lv[q], f, Ls);
                            O = fmaf(ov[q], f, O);
                        }
                        M = Mn;
                    }
                    const long long io = static_cast<long long>(run.io0 + col / a.G) * a.n_io_layers + L.io;
                    a.out[io * a.q_stride + (p.h * a.G + col % a.G) * HD + d] = O / Ls;
                }
            }
        }
        __syncthreads();  // o_s, ml_s and flag before the next piece writes them
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
    const int grid = std::max(1, std::min(num_sms * C::CTAS, (a.total + C::W - 1) / C::W));
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
