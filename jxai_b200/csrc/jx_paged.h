// jx_paged.h -- types and device helpers of the paged 8-bit KV cache, shared by
// its host side and its kernels.
//
// A page holds kPageRows consecutive rows of one sequence for every layer.  It
// is a run of records, one per (layer, kv head):
//   scales {K0, K1, V0, V1}, K codes [32][HD] bytes, V codes [32][HD] bytes
// where K0 / V0 scale rows 0-15 and K1 / V1 rows 16-31 (fp32 powers of two).
// Inside a 32-row tile the 16-byte chunks of each 128-byte line are permuted
// (chunk ^= line & 7; by row at head_dim 256), so that both the row-wise reads
// of K and the 8x8 matrix loads of V are free of bank conflicts once a record
// lies in shared memory.
// A record is one contiguous, 16-byte aligned run (HD*64 + 16 bytes): one bulk
// copy, or two (scales and K, then V), bring all that attention needs of 32 rows.
// int8 codes are stored offset by 128 (one byte permute then builds the fp16
// number 1024 + u); e4m3 codes as they are.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace jx {

enum { DT_I8 = 3, DT_E4M3 = 4 };  // = jx_dtype JX_I8, JX_E4M3

constexpr int kPageRows = 32;
constexpr int kBlockRows = 16;     // rows that share a scale
constexpr int kMinExp = -40;       // scale exponents: a block of zeros has the smallest
constexpr int kMaxExp = 56;
constexpr float kClip = 4.611686018427387904e18f;  // 2^62: larger magnitudes are held as this one

constexpr int kMaxRuns = 128;      // runs and layers of one launch: its plan travels in the
constexpr int kMaxCallLayers = 64; // kernel's parameters (no upload, nothing to outlive the call)
constexpr int kMaxRopeCfgs = 8;
constexpr int kStepCtasPerSm = 4;  // at most
// What a segment costs a CTA beside its pages, in pages.  (3 / 8 / 16: ragged batch 239 / 220 / 216 us,
// Gemma-3-1B shape 63 / 59 / 49 us, 131072-row Mistral-7B shape 110 / 108 / 105 us; 24: as 16.)
constexpr int kPieceCost = 16;
constexpr int kStepCols = 8;       // columns of the step kernel

// Consecutive tokens of one sequence: rows io0 .. io0+n-1 of the call, at
// positions pos0 .. pos0+n-1.
struct PagedRun {
    int seq;
    int pos0;
    int n;
    int io0;
    int off;  // first work unit of the run (meaning: the kernel's)
    int off1;
};

struct PagedLayer {
    uint16_t cache_layer;
    uint16_t io;    // layer index within the call's rows
    uint16_t half;  // rotated pairs per head
    uint8_t cfg;    // rope table
    uint8_t flags;  // kLayerWindow | kLayerAppend
};
constexpr int kLayerWindow = 1, kLayerAppend = 2;

struct PagedArgs {
    unsigned char* pool;
    const int* table;       // [n_seqs][max_pages] page of every 32 rows
    long long page_bytes;
    long long layer_bytes;  // n_kv * record
    int max_pages;
    int n_kv;
    int G;
    int n_io_layers;        // layers of the call: row r, layer l is io row r*n_io_layers + l
    const float* q;
    const float* k_in;
    const float* v_in;
    float* out;
    long long q_stride;
    long long kv_stride;
    float scale;
    float softcap;
    float cap_in, cap_out;  // softcap on x = s log2(e): cap_out tanh(x cap_in)
    int window;
    int neox;
    int n_runs;
    int n_layers;
    int n_full;             // step: layers without a window stand first
    int total;              // work units
    int total0;             // step: units of those layers
    int units0, units1;     // step: units of a segment, over all runs, without and with the window
    int append;             // step: write the run's row, too
    int q_vec, kv_vec;      // 16-byte loads of q / of k and v are possible
    int test_wait_cta;      // step: CTA + 1 that waits on a barrier nothing arrives at (test hook)
    const float2* rope[kMaxRopeCfgs];  // [capacity][HD/2] (cos, sin)
    float* scratch;
    int* counters;
    int* err;
    int* dbg;
    long long wait_limit;
    PagedLayer layers[kMaxCallLayers];
    PagedRun runs[kMaxRuns];
};
static_assert(sizeof(PagedArgs) <= 4096, "kernel parameters");

constexpr int kScaleBytes = 16;
__host__ __device__ constexpr int record_bytes(int hd) { return kScaleBytes + 2 * kPageRows * hd; }
// The K (0) or V (1) tile of a record.
__host__ __device__ constexpr int tile_at(int hd, int which) { return kScaleBytes + which * kPageRows * hd; }

// Byte of (row, dim) inside a K or V tile of a record.
__host__ __device__ __forceinline__ uint32_t tile_byte(int hd, int row, int d) {
    const uint32_t off = static_cast<uint32_t>(row * hd + d);
    return off ^ (((off >> (hd == 256 ? 8 : 7)) & 7u) << 4);
}

#ifdef __CUDACC__

// ---------------------------------------------------------------- the format
// A value as the cache takes it: NaN is 0, magnitudes are cut at 2^62.
__device__ __forceinline__ float cache_value(float x) {
    return x != x ? 0.0f : fminf(fmaxf(x, -kClip), kClip);
}

// Exponent k of a block whose largest magnitude is `amax`: the smallest with
// amax <= M * 2^k (M = 127: 1.984375 * 2^6; 448: 1.75 * 2^8), cut to the range.
template <int DT>
__device__ __forceinline__ int block_exp(float amax) {
    if (!(amax > 0.0f)) return kMinExp;
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 127;  // subnormals end up below kMinExp all the same
    const uint32_t man = u & 0x7FFFFFu;
    const int k = DT == DT_I8 ? e - 6 + (man > 0x7E0000u ? 1 : 0) : e - 8 + (man > 0x600000u ? 1 : 0);
    return min(kMaxExp, max(kMinExp, k));
}

__device__ __forceinline__ float exp2_int(int k) {  // 2^k, k in the normal range
    return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}
__device__ __forceinline__ int scale_exp(float s) {  // k of a stored scale 2^k
    return static_cast<int>(__float_as_uint(s) >> 23) - 127;
}

// Exponent of the power of two that brings a query whose largest magnitude is `amax`
// into [2^14, 2^15), to the end of fp32's range; at most 2^60 for small ones, of which
// what lies below 2^-84 is lost.
__device__ __forceinline__ int query_exp(float amax) {
    return min(60, 14 - (static_cast<int>((__float_as_uint(amax) >> 23) & 0xFFu) - 127));
}
// What takes that (and the scale of scores) back, no larger than 2^70: times a block's
// scale it then stays in range.  (That cuts scores of queries beyond 2^84, by a common
// factor: they stay far apart.)
__device__ __forceinline__ float query_unit(int sh, float scale) {
    constexpr float kMost = 1.180591620717411303424e21f;
    const float u = exp2_int(-sh) * scale;
    return u > kMost ? kMost : u < -kMost ? -kMost : u;
}

// One element of a rotated head; each operation's result is an fp32 number
// (no fused multiply-add), so that what the cache holds does not depend on
// how the compiler contracts.  cs[j] = (cos, sin).
__device__ __forceinline__ float rope_plain(const float* x, int d, int half, const float2* cs,
                                            bool neox) {
    if (d >= 2 * half) return x[d];
    const int j = neox ? (d < half ? d : d - half) : d >> 1;
    const bool first = neox ? d < half : (d & 1) == 0;
    const float a = x[neox ? j : 2 * j], b = x[neox ? j + half : 2 * j + 1];
    const float2 t = cs[j];
    return first ? __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y))
                 : __fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
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

// Four values to codes (nearest to x * inv, ties to even; inv a power of two and
// |x * inv| within the codes' range) and back; 16 likewise.  int8: adding
// 1.5 * 2^23 + 128 leaves the rounded code plus 128 in the sum's low byte, and a
// byte under the exponent of 2^23 is that number plus its value: no conversion
// instruction, of which an SM does 16 a cycle.
template <int DT>
__device__ __forceinline__ uint32_t pack4(float x, float y, float z, float w, float inv) {
    if constexpr (DT == DT_I8) {
        constexpr float kMagic = 12582912.0f + 128.0f;
        const uint32_t a = __float_as_uint(__fmaf_rn(x, inv, kMagic)), b = __float_as_uint(__fmaf_rn(y, inv, kMagic));
        const uint32_t c = __float_as_uint(__fmaf_rn(z, inv, kMagic)), d = __float_as_uint(__fmaf_rn(w, inv, kMagic));
        return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x * inv, y * inv), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(z * inv, w * inv), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}
template <int DT>
__device__ __forceinline__ float4 unpack4(uint32_t w) {
    if constexpr (DT == DT_I8) {
        auto at = [&](uint32_t sel) { return __uint_as_float(__byte_perm(w, 0x4B000000u, sel)) - (8388608.0f + 128.0f); };
        return make_float4(at(0x7540), at(0x7541), at(0x7542), at(0x7543));
    } else {
        const __half2_raw l = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFFu), __NV_E4M3);
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
        const float2 a = __half22float2(__half2(l)), b = __half22float2(__half2(h));
        return make_float4(a.x, a.y, b.x, b.y);
    }
}
template <int DT>
__device__ __forceinline__ uint4 pack_codes(const float (&x)[16], float inv) {
    return make_uint4(pack4<DT>(x[0], x[1], x[2], x[3], inv), pack4<DT>(x[4], x[5], x[6], x[7], inv),
                      pack4<DT>(x[8], x[9], x[10], x[11], inv), pack4<DT>(x[12], x[13], x[14], x[15], inv));
}
template <int DT>
__device__ __forceinline__ void unpack_codes(const uint4& c, float (&x)[16]) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 v = unpack4<DT>(w[i]);
        x[4 * i] = v.x;
        x[4 * i + 1] = v.y;
        x[4 * i + 2] = v.z;
        x[4 * i + 3] = v.w;
    }
}

// CTA that owns unit x when CTA c of P takes units [c*total/P, (c+1)*total/P).
__device__ __forceinline__ long long owner_of(long long x, long long total, long long P) {
    return ((x + 1) * P - 1) / total;
}

#endif  // __CUDACC__

// The prompt kernel (jx_paged_prompt.cu): items of up to 2 * 128/G tokens over
// fp16 rows (tensor maps of 128-row boxes), whose K and V of a head are to be
// multiplied by head_scale [seq][layer][kv head] (K, V).
struct PrefillTile;
struct PromptArgs {
    const PrefillTile* tiles;
    const int* cta_first;   // CTA b runs tiles [cta_first[b], cta_first[b + 1])
    const float* q;
    float* out;
    long long q_stride;
    const float2* rope;     // rows of HD/2 (cos, sin) pairs, by position
    const float2* head_scale;
    float* totals;          // [grid][2][HD][128]
    int scale_layers, scale_heads;
    int neox, q_vec;
    float scale, softcap, cap_in, cap_out;
    int* err;
    int* dbg;
    long long wait_limit;
};
constexpr int kPromptRows = 128;  // rows of a K or V tile, and of a query tile
bool paged_prompt_supported(int hd, int G);
cudaError_t paged_prompt_launch(const PromptArgs& a, const CUtensorMap* tmK, const CUtensorMap* tmV, int hd, int G,
                                int grid, cudaStream_t st);

// The step kernel (jx_paged_step.cuh) for `cols` columns: query heads of a kv
// head, times the tokens of a block.
cudaError_t paged_step_i8(const PagedArgs& a, int hd, int cols, int num_sms, cudaStream_t st);
cudaError_t paged_step_e4m3(const PagedArgs& a, int hd, int cols, int num_sms, cudaStream_t st);

}  // namespace jx
