// jx_paged.cu -- the paged 8-bit KV cache: its host side (pages, page tables,
// argument checks, launch plans) and the kernels that write, move and read rows.
//
// Pages, their reference counts and the page table live on the host; a device
// copy of the table ([n_seqs][max_pages]) is brought up to date by small kernels
// on the caller's stream.  A launch's plan (which sequences, positions and
// layers) travels in the kernel's parameters; only the work items of a
// tensor-core prompt and the row list of a keep are uploaded, from two buffers
// that are used in turn.
#include "jx_paged.h"

#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <map>
#include <memory>
#include <mutex>
#include <new>
#include <string>
#include <vector>

#include "jx_attn.h"
#include "jx_device.cuh"
#include "jx_internal.h"

using namespace jx;

namespace {

int pfail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int pfail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_last_error(buf);
    return code;
}

#define PKV_CUDA(call)                                                                    \
    do {                                                                                  \
        cudaError_t e_ = (call);                                                          \
        if (e_ != cudaSuccess)                                                            \
            return pfail(JX_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));    \
    } while (0)

using TensorMapEncode = PFN_cuTensorMapEncodeTiled_v12000;
TensorMapEncode tensor_map_encode() {
    static TensorMapEncode fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<TensorMapEncode>(p);
    });
    return fn;
}

struct OnDevice {  // the handle's device for the duration of a call
    int prev = -1;
    bool ok = false;
    explicit OnDevice(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) return;
        ok = prev == dev || cudaSetDevice(dev) == cudaSuccess;
    }
    ~OnDevice() {
        if (ok && prev >= 0) cudaSetDevice(prev);
    }
};

// ------------------------------------------------------------------ kernels

constexpr int kTableBatch = 480;
struct TableSet {
    int* table;
    int n;
    int at[kTableBatch];
    int page[kTableBatch];
};
static_assert(sizeof(TableSet) <= 4096, "kernel parameters");

__global__ void table_set_kernel(const __grid_constant__ TableSet t) {
    for (int i = threadIdx.x; i < t.n; i += blockDim.x) t.table[t.at[i]] = t.page[i];
}

__global__ void table_copy_kernel(int* dst, const int* src, int n) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x)
        dst[i] = src[i];
}

constexpr int kCopyBatch = 480;
struct PageCopies {
    unsigned char* pool;
    long long page_bytes;
    int n;
    int src[kCopyBatch];
    int dst[kCopyBatch];
};
static_assert(sizeof(PageCopies) <= 4096, "kernel parameters");

// Whole pages, 16 bytes per thread and turn: a page is one contiguous run, so
// this is a plain copy whatever the layers and heads are (67 MB and back: 24 us =
// 5.6 TB/s; the call with its table entries 38 us).
__global__ void page_copy_kernel(const __grid_constant__ PageCopies c) {
    const long long n16 = c.page_bytes / 16;
    for (int p = blockIdx.y; p < c.n; p += gridDim.y) {
        const uint4* s = reinterpret_cast<const uint4*>(c.pool + c.src[p] * c.page_bytes);
        uint4* d = reinterpret_cast<uint4*>(c.pool + c.dst[p] * c.page_bytes);
        for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < n16;
             i += static_cast<long long>(gridDim.x) * blockDim.x)
            d[i] = s[i];
    }
}

// (cos, sin) of every rotated pair at every position of the cache, from angles
// in 64 bits: at position 100000 an fp32 angle is off by up to 4e-3.
struct RopeTable {
    float2* out;
    int rows, width, half;
    double freq[128];
};
__global__ void rope_table_kernel(const __grid_constant__ RopeTable t) {
    const long long n = static_cast<long long>(t.rows) * t.width;
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < n;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int j = static_cast<int>(i % t.width);
        float2 r = make_float2(1.0f, 0.0f);
        if (j < t.half) {
            const double a = static_cast<double>(i / t.width) * t.freq[j];
            r = make_float2(static_cast<float>(cos(a)), static_cast<float>(sin(a)));
        }
        t.out[i] = r;
    }
}

// Largest value over the `n` threads (a multiple of 32, starting at a warp) of
// one half of the CTA: `red` has one slot per warp.
__device__ __forceinline__ float half_max(float v, float* red, int n) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int w0 = threadIdx.x / n * (n / 32);
    float m = 0.0f;
    for (int w = 0; w < n / 32; ++w) m = fmaxf(m, red[w0 + w]);
    return m;
}

// Rows of a call written to the cache.  One CTA per (block of 16 rows, layer,
// kv head): its first half takes K, its second V, one thread per 16 values of
// a row.  The block's largest magnitude gives the scale; rows that were in the
// block before the call are re-rounded where the scale grows.  Reads 4 bytes and
// writes 1 per element: 2048 tokens of four Llama-3.2-1B-shaped layers (42 MB) in
// 15 us (16-byte loads; with scalar ones 41).
template <int HD, int DT>
__global__ void __launch_bounds__(2 * HD) append_kernel(const __grid_constant__ PagedArgs a) {
    constexpr int CPR = HD / 16;  // threads per row
    __shared__ float red[2 * HD / 32];
    const int which = threadIdx.x / HD, tid = threadIdx.x % HD;
    const int row = tid / CPR, d0 = tid % CPR * 16;
    int r = 0;
    while (r + 1 < a.n_runs && a.runs[r + 1].off <= static_cast<int>(blockIdx.x)) ++r;
    const PagedRun run = a.runs[r];
    const int h = blockIdx.y % a.n_kv;
    const PagedLayer L = a.layers[blockIdx.y / a.n_kv];
    const int blk = run.pos0 / kBlockRows + (static_cast<int>(blockIdx.x) - run.off);
    const int t = blk * kBlockRows + row;
    const bool is_new = t >= run.pos0 && t < run.pos0 + run.n;
    const bool kept = t < run.pos0;
    const int page = a.table[static_cast<long long>(run.seq) * a.max_pages + blk / 2];
    unsigned char* rec = a.pool + page * a.page_bytes + L.cache_layer * a.layer_bytes +
                         static_cast<long long>(h) * record_bytes(HD);
    unsigned char* dst = rec + tile_at(HD, which) + tile_byte(HD, (blk & 1) * kBlockRows + row, d0);
    float* scale = reinterpret_cast<float*>(rec) + which * 2 + (blk & 1);
    float x[16];
    float m = 0.0f;
    if (is_new) {
        const long long io = static_cast<long long>(run.io0 + t - run.pos0) * a.n_io_layers + L.io;
        const float* src = (which == 0 ? a.k_in : a.v_in) + io * a.kv_stride + h * HD;
        const float2* cs = a.rope[L.cfg] + static_cast<long long>(t) * (HD / 2);
        const int half = which == 0 ? L.half : 0;
        const bool vec = a.kv_vec && half % 4 == 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = rope4(src, d0 + 4 * i, half, cs, a.neox != 0, vec);
            x[4 * i] = cache_value(v.x);
            x[4 * i + 1] = cache_value(v.y);
            x[4 * i + 2] = cache_value(v.z);
            x[4 * i + 3] = cache_value(v.w);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(x[i]));
    }
    m = half_max(m, red, HD);
    int k = block_exp<DT>(m);
    const bool joins = blk * kBlockRows < run.pos0;  // earlier rows stay in the block
    const int k_old = joins ? max(kMinExp, scale_exp(*scale)) : kMinExp;
    k = max(k, k_old);
    __syncthreads();  // the old scale is read by all before one thread replaces it
    if (is_new) *reinterpret_cast<uint4*>(dst) = pack_codes<DT>(x, exp2_int(-k));
    if (kept && k > k_old) {
        unpack_codes<DT>(*reinterpret_cast<const uint4*>(dst), x);
        *reinterpret_cast<uint4*>(dst) = pack_codes<DT>(x, exp2_int(k_old - k));
    }
    if (tid == 0) *scale = exp2_int(k);
}

struct KeepArgs {
    unsigned char* pool;
    const int* src_table;  // [pages] of the sequence as it is
    const int* dst_table;  // [pages] of the result
    const int* rows;       // [n_rows] kept rows, ascending
    long long page_bytes;
    int n_rec;             // records of a page
    int n_rows;
    int blk0;              // first block to write
    int n_blk;             // blocks to write
    int serial;            // one CTA per record, block after block (in place)
};

constexpr int kKeepRecords = 4;  // records of a block that a CTA moves together

// Kept rows gathered into dense blocks: each is scaled and rounded anew from
// the values held.  One CTA per (block of 16 rows, kKeepRecords records); its
// first half takes K, its second V, one thread per 16 values of a row.  Where a
// row lies is looked up once for all records, and their loads are in flight
// together: a block alone is 8 KB behind three dependent loads.  Row i of the
// result comes from a row >= i, and a CTA reads all of a block before it writes
// it: in place (serial) no row is overwritten before it has been read.  5000 of
// 16384 rows, 16 Mistral-7B-shaped layers (328 MB both ways): 77 us = 4.3 TB/s (one
// record at a time and conversion instructions: 126); the call 102 us, of 32 layers
// 176.
template <int HD, int DT>
__global__ void __launch_bounds__(2 * HD) keep_kernel(const KeepArgs a) {
    constexpr int CPR = HD / 16, R = kKeepRecords, WARPS = 2 * HD / 32;
    __shared__ float red[R][WARPS];
    const int which = threadIdx.x / HD, tid = threadIdx.x % HD;
    const int row = tid / CPR, d0 = tid % CPR * 16;
    const int rec0 = blockIdx.y * R, n_rec = min(R, a.n_rec - rec0);
    const int last = a.serial ? a.n_blk : static_cast<int>(blockIdx.x) + 1;
    for (int b = a.serial ? 0 : static_cast<int>(blockIdx.x); b < last; ++b) {
        const int blk = a.blk0 + b;
        const int i = blk * kBlockRows + row;
        const bool on = i < a.n_rows;
        uint4 c[R];
        float s[R];
        if (on) {
            const int t = a.rows[i];
            const unsigned char* rec = a.pool + a.src_table[t / kPageRows] * a.page_bytes +
                                       static_cast<long long>(rec0) * record_bytes(HD);
            const uint32_t at = tile_at(HD, which) + tile_byte(HD, t % kPageRows, d0);
            const int k = which * 2 + (t / kBlockRows & 1);
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (j < n_rec) {
                    c[j] = *reinterpret_cast<const uint4*>(rec + j * record_bytes(HD) + at);
                    s[j] = reinterpret_cast<const float*>(rec + j * record_bytes(HD))[k];
                }
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float m = 0.0f;
            if (on && j < n_rec) {
                float x[16];
                unpack_codes<DT>(c[j], x);
#pragma unroll
                for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(x[e]));
                m *= s[j];
            }
            m = warp_max(m);
            if (threadIdx.x % 32 == 0) red[j][threadIdx.x / 32] = m;
        }
        __syncthreads();  // this block's reads are done before its writes begin, too
        unsigned char* rec = a.pool + a.dst_table[blk / 2] * a.page_bytes + static_cast<long long>(rec0) * record_bytes(HD);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (j >= n_rec) break;
            float m = 0.0f;
            for (int w = 0; w < WARPS / 2; ++w) m = fmaxf(m, red[j][which * (WARPS / 2) + w]);
            const int k = block_exp<DT>(m);
            if (on) {
                float x[16];
                unpack_codes<DT>(c[j], x);
                // the scale's change alone: code 2^ks to code 2^k
                *reinterpret_cast<uint4*>(rec + j * record_bytes(HD) + tile_at(HD, which) +
                                          tile_byte(HD, (blk & 1) * kBlockRows + row, d0)) =
                    pack_codes<DT>(x, s[j] * exp2_int(-k));
            }
            if (tid == 0)
                reinterpret_cast<float*>(rec + j * record_bytes(HD))[which * 2 + (blk & 1)] = exp2_int(k);
        }
        __syncthreads();  // this block's writes before the next one's reads; red is free
    }
}

struct LoadArgs {
    unsigned char* pool;
    const int* table;  // of the sequence
    const unsigned char* codes[2];
    const float* scales[2];
    long long page_bytes;
    int row0, n_rows, n_kv, n_layers;
};

template <int HD, int DT>
__global__ void load_kernel(const LoadArgs a) {
    constexpr int CPR = HD / 16;
    const int n_blk = (a.n_rows + kBlockRows - 1) / kBlockRows;
    const long long n = static_cast<long long>(a.n_layers) * a.n_rows * a.n_kv * CPR;
    const int which = blockIdx.y;
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < n;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int c = static_cast<int>(i % CPR);
        const int h = static_cast<int>(i / CPR % a.n_kv);
        const long long lr = i / CPR / a.n_kv;
        const int r = static_cast<int>(lr % a.n_rows), l = static_cast<int>(lr / a.n_rows);
        const int t = a.row0 + r;
        unsigned char* rec = a.pool + a.table[t / kPageRows] * a.page_bytes +
                             (static_cast<long long>(l) * a.n_kv + h) * record_bytes(HD);
        const uint4 v = *reinterpret_cast<const uint4*>(a.codes[which] + i * 16);
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t o = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                uint32_t u = (w[j] >> (8 * b)) & 0xFFu;
                if constexpr (DT == DT_I8) u = max(u ^ 0x80u, 1u);  // offset by 128; -128 -> -127
                else u = (u & 0x7Fu) == 0x7Fu ? 0u : u;             // NaN -> 0
                o |= u << (8 * b);
            }
            w[j] = o;
        }
        *reinterpret_cast<uint4*>(rec + tile_at(HD, which) + tile_byte(HD, t % kPageRows, c * 16)) =
            make_uint4(w[0], w[1], w[2], w[3]);
        if (c == 0 && r % kBlockRows == 0) {
            const float s = a.scales[which][(static_cast<long long>(l) * n_blk + r / kBlockRows) * a.n_kv + h];
            reinterpret_cast<float*>(rec)[which * 2 + (t / kBlockRows & 1)] =
                exp2_int(min(kMaxExp, max(kMinExp, scale_exp(fabsf(s)))));
        }
    }
}

struct ReadArgs {
    const unsigned char* pool;
    const int* table;
    void* out;
    long long page_bytes;
    int max_pages, n_kv, n_layers, n_rows, n;
    int r0, rows;  // the rows of this launch, of n_rows
    int seq[kMaxRuns];
    int row0[kMaxRuns];
};
static_assert(sizeof(ReadArgs) <= 4096, "kernel parameters");

// Values of rows; one (sequence, layer, K or V) per (z, y) of the grid, a thread
// per 16 codes of a row, in the order of the output: 5000 rows of 16 layers (492 MB
// both ways) in 87 us = 5.7 TB/s.
template <int HD, int DT, bool F32>
__global__ void read_kernel(const __grid_constant__ ReadArgs a) {
    constexpr uint32_t CPR = HD / 16;
    const int s = blockIdx.z, which = blockIdx.y & 1, l = blockIdx.y >> 1;
    const int* table = a.table + static_cast<long long>(a.seq[s]) * a.max_pages;
    const uint32_t per_row = a.n_kv * CPR, n = a.rows * per_row;
    const long long out0 = (((static_cast<long long>(s) * a.n_layers + l) * 2 + which) * a.n_rows + a.r0) * per_row;
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
        const uint32_t r = i / per_row, c = i % CPR, h = (i - r * per_row) / CPR;
        const int t = a.row0[s] + a.r0 + static_cast<int>(r);
        const unsigned char* rec = a.pool + table[t / kPageRows] * a.page_bytes +
                                   (static_cast<long long>(l) * a.n_kv + h) * record_bytes(HD);
        const float sc = reinterpret_cast<const float*>(rec)[which * 2 + (t / kBlockRows & 1)];
        float x[16];
        unpack_codes<DT>(*reinterpret_cast<const uint4*>(rec + tile_at(HD, which) + tile_byte(HD, t % kPageRows, c * 16)), x);
        const long long o = (out0 + i) * 16;
        if constexpr (F32) {
            float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + o);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                dst[j] = make_float4(x[4 * j] * sc, x[4 * j + 1] * sc, x[4 * j + 2] * sc, x[4 * j + 3] * sc);
        } else {
            // a code has at most 7 significant bits: its value is a bf16 number,
            // the upper half of the fp32 one
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                w[j] = __byte_perm(__float_as_uint(x[2 * j] * sc), __float_as_uint(x[2 * j + 1] * sc), 0x7632);
            uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + o);
            dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
            dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
}

// Rows of a prompt's sequences from codes to fp16, for the tensor-core prompt
// kernel: out [slot][layer][rows][n_kv * HD], K and V.
struct WidenArgs {
    const unsigned char* pool;
    const int* table;
    uint16_t* out[2];
    float2* head_scale;   // [slot][layer][kv head]
    long long page_bytes;
    long long layer_bytes;
    long long slot_elems; // elements of a slot (all layers) and of a layer in `out`
    long long layer_elems;
    int max_pages, n_kv, n_layers, n_runs, window, rows;
    PagedLayer layers[kMaxCallLayers];
    PagedRun runs[kMaxRuns];  // off: first row chunk
};
static_assert(sizeof(WidenArgs) <= 4096, "kernel parameters");

constexpr int kWidenRows = 64;
constexpr int kMaxWideExp = 16;

// A code times 2^(k - K), K so that the head's largest block exponent becomes 8
// (int8; e4m3: 7) and no value exceeds 448 * 2^7.  fp16 has bits down to 2^-24, an
// e4m3 code down to 2^-9: exact for blocks down to 2^-32 (e4m3: 2^-22) of the largest
// scale, below that off by at most 2^-33 (2^-32) of it.  K is at most 8 (9): a row
// that holds infinities (2^62 in the cache) is taken as 65504 * 2^8 = 1.7e7 (3.4e7),
// so that it cannot wipe out the rows of tokens that do not attend it; beside it a
// value is off by at most 2^-17 (2^-16).  The factor 2^K of each head goes to the
// prompt kernel, which multiplies scores and outputs by it.  One CTA per (64 rows,
// layer, kv head); the exponents of the sequence's blocks (16 bytes per page) are
// read by every one of them.
template <int HD, int DT>
__global__ void __launch_bounds__(256) widen_kernel(const __grid_constant__ WidenArgs a) {
    constexpr int kTop = DT == DT_I8 ? 8 : 7;
    __shared__ int red[2][8];
    int s = 0;
    while (s + 1 < a.n_runs && a.runs[s + 1].off <= static_cast<int>(blockIdx.x)) ++s;
    const PagedRun run = a.runs[s];
    const int l = blockIdx.y / a.n_kv, h = blockIdx.y % a.n_kv;
    const PagedLayer L = a.layers[l];
    const int end = run.pos0 + run.n;
    const int lo = (L.flags & kLayerWindow) ? max(0, run.pos0 - a.window + 1) : 0;
    const int first = lo / kPageRows, last = (end - 1) / kPageRows;
    const int row0 = lo / kWidenRows * kWidenRows + (static_cast<int>(blockIdx.x) - run.off) * kWidenRows;
    // rows behind the last one that share its tile are zeros: their weights are 0,
    // but 0 times what the buffer held before might not be
    const int zeros = min(a.rows, end + kPromptRows);
    if (row0 >= zeros) return;
    const int* table = a.table + static_cast<long long>(run.seq) * a.max_pages;
    const unsigned char* base = a.pool + L.cache_layer * a.layer_bytes + static_cast<long long>(h) * record_bytes(HD);
    int ek = kMinExp, ev = kMinExp;
    for (int p = first + threadIdx.x; p <= last; p += 256) {
        const float4 sc = *reinterpret_cast<const float4*>(base + table[p] * a.page_bytes);
        // a page's first block may lie before the rows, its second behind them
        const bool one = p * kPageRows + kBlockRows > lo, two = p * kPageRows + kBlockRows < end;
        ek = max(ek, max(one ? scale_exp(sc.x) : kMinExp, two ? scale_exp(sc.y) : kMinExp));
        ev = max(ev, max(one ? scale_exp(sc.z) : kMinExp, two ? scale_exp(sc.w) : kMinExp));
    }
    ek = __reduce_max_sync(0xffffffffu, ek);
    ev = __reduce_max_sync(0xffffffffu, ev);
    if (threadIdx.x % 32 == 0) {
        red[0][threadIdx.x / 32] = ek;
        red[1][threadIdx.x / 32] = ev;
    }
    __syncthreads();
    for (int w = 0; w < 8; ++w) {
        ek = max(ek, red[0][w]);
        ev = max(ev, red[1][w]);
    }
    ek = min(ek, kMaxWideExp) - kTop;
    ev = min(ev, kMaxWideExp) - kTop;
    if (blockIdx.x == static_cast<unsigned>(run.off) && threadIdx.x == 0)
        a.head_scale[(static_cast<long long>(s) * a.n_layers + l) * a.n_kv + h] = make_float2(exp2_int(ek), exp2_int(ev));
    constexpr int CPR = HD / 16;
    for (int i = threadIdx.x; i < kWidenRows * CPR * 2; i += 256) {
        const int which = i / (kWidenRows * CPR), c = i % CPR, t = row0 + i / CPR % kWidenRows;
        if (t < lo || t >= zeros) continue;
        uint4* dst = reinterpret_cast<uint4*>(a.out[which] + s * a.slot_elems + l * a.layer_elems +
                                              (static_cast<long long>(t) * a.n_kv + h) * HD + c * 16);
        if (t >= end) {
            dst[0] = dst[1] = make_uint4(0u, 0u, 0u, 0u);
            continue;
        }
        const unsigned char* rec = base + table[t / kPageRows] * a.page_bytes;
        const int k = scale_exp(reinterpret_cast<const float*>(rec)[which * 2 + (t / kBlockRows & 1)]) - (which ? ev : ek);
        const float f = exp2_int(max(k, -60));
        float x[16];
        unpack_codes<DT>(*reinterpret_cast<const uint4*>(rec + tile_at(HD, which) + tile_byte(HD, t % kPageRows, c * 16)), x);
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __half2 v = __floats2half2_rn(fminf(fmaxf(x[2 * j] * f, -65504.0f), 65504.0f),
                                                fminf(fmaxf(x[2 * j + 1] * f, -65504.0f), 65504.0f));
            w[j] = *reinterpret_cast<const uint32_t*>(&v);
        }
        dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
        dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// Calls f(integral_constant<HD>, integral_constant<DT>) for a cache's format.
template <int V>
using Int = std::integral_constant<int, V>;
template <typename F>
void dispatch(const jx_pkv_desc& d, F&& f) {
    auto with_hd = [&](auto dt) {
        switch (d.head_dim) {
            case 32: f(Int<32>{}, dt); break;
            case 64: f(Int<64>{}, dt); break;
            case 128: f(Int<128>{}, dt); break;
            default: f(Int<256>{}, dt); break;
        }
    };
    if (d.dtype == JX_I8) with_hd(Int<DT_I8>{});
    else with_hd(Int<DT_E4M3>{});
}

struct RopeCfg {
    uint32_t rdim, base_bits, yarn_bits;
    std::vector<float> factors;
    float2* d_tab;
};

}  // namespace

struct jx_pkv {
    jx_pkv_desc d{};
    long long page_bytes = 0, layer_bytes = 0;
    uint32_t max_pages = 0;
    unsigned char* pool = nullptr;
    int* d_table = nullptr;
    std::vector<int> free_pages;          // a stack
    std::vector<int> refs;                // sequences that hold the page
    std::vector<std::vector<int>> pages;  // of each sequence
    std::vector<uint32_t> rows;           // rows held by each sequence
    std::vector<RopeCfg> ropes;
    float* d_scratch = nullptr;           // two partial results per CTA of the step kernel
    int* d_counters = nullptr;
    int* d_err = nullptr;
    int* d_dbg = nullptr;
    struct Upload {                       // a list for a kernel: pinned, and its device copy
        void* h = nullptr;
        void* d = nullptr;
        size_t bytes = 0;
        cudaEvent_t done = nullptr;       // the kernels that read the device copy
        bool pending = false;
    } up[2];
    int up_next = 0;
    uint16_t* d_wide = nullptr;           // prompts: fp16 rows of a group of layers
    size_t wide_bytes = 0;
    float2* d_head_scale = nullptr;
    size_t head_scales = 0;
    float* d_totals = nullptr;            // prompts: the CTAs' running sums
    size_t totals_bytes = 0;
    int num_sms = 0;
    int opt_wait_limit_ms = 0;
    int opt_test_wait_cta = 0;
    int opt_test_fail = 0;                // test hook: workspaces (1), a keep's launch (2) fail
    int opt_prefill_tc = -1;              // prompts on the tensor cores: 1 / 0, -1: by estimate
    int last_launches = 0;
};

namespace {

int launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? JX_OK : pfail(JX_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}

int refuse_capture(cudaStream_t st) {
    cudaStreamCaptureStatus c = cudaStreamCaptureStatusNone;
    PKV_CUDA(cudaStreamIsCapturing(st, &c));
    return c == cudaStreamCaptureStatusNone
               ? JX_OK
               : pfail(JX_ERR_UNSUPPORTED,
                       "calls on a paged cache cannot be captured into a graph (pages are "
                       "assigned on the host, call by call)");
}

uint32_t pages_for(uint32_t rows) { return (rows + kPageRows - 1) / kPageRows; }

void give_back(jx_pkv* kv, int page) {
    if (--kv->refs[page] == 0) kv->free_pages.push_back(page);
}

int take_page(jx_pkv* kv) {  // the caller has checked that one is free
    const int p = kv->free_pages.back();
    kv->free_pages.pop_back();
    kv->refs[p] = 1;
    return p;
}

void drop_rows(jx_pkv* kv, uint32_t seq, uint32_t rows) {
    auto& pg = kv->pages[seq];
    while (pg.size() > pages_for(rows)) {
        give_back(kv, pg.back());
        pg.pop_back();
    }
    kv->rows[seq] = std::min(kv->rows[seq], rows);
}

struct TableEntry {
    uint32_t seq, idx;
    int page;
};

int set_table(jx_pkv* kv, const std::vector<TableEntry>& e, cudaStream_t st) {
    for (size_t i = 0; i < e.size();) {
        TableSet t;
        t.table = kv->d_table;
        t.n = 0;
        for (; i < e.size() && t.n < kTableBatch; ++i, ++t.n) {
            t.at[t.n] = static_cast<int>(e[i].seq * kv->max_pages + e[i].idx);
            t.page[t.n] = e[i].page;
        }
        table_set_kernel<<<1, 128, 0, st>>>(t);
        if (int rc = launched("page table")) return rc;
    }
    return JX_OK;
}

int copy_pages(jx_pkv* kv, const std::vector<std::pair<int, int>>& c, cudaStream_t st) {
    for (size_t i = 0; i < c.size();) {
        PageCopies p;
        p.pool = kv->pool;
        p.page_bytes = kv->page_bytes;
        p.n = 0;
        for (; i < c.size() && p.n < kCopyBatch; ++i, ++p.n) {
            p.src[p.n] = c[i].first;
            p.dst[p.n] = c[i].second;
        }
        const long long per = std::max<long long>(1, (kv->page_bytes / 16 + 255) / 256);
        const dim3 grid(static_cast<unsigned>(std::min<long long>(per, 64)), p.n);
        page_copy_kernel<<<grid, 256, 0, st>>>(p);
        if (int rc = launched("page copy")) return rc;
    }
    return JX_OK;
}

struct Span {  // rows [begin, end) of a sequence that a call writes
    uint32_t seq, begin, end;
};

// Pages for the rows that a call writes: new ones, and copies of shared ones
// (the page is shared by a fork: the writer gets its own).  All or nothing: what can
// fail for lack of memory comes before the first page moves.
int make_room(jx_pkv* kv, const std::vector<Span>& spans, cudaStream_t st) {
    size_t need = 0;
    std::map<int, int> left;  // holders of a shared page after those before have their own
    for (const Span& s : spans) {
        auto& pg = kv->pages[s.seq];
        pg.reserve(pages_for(s.end));
        for (uint32_t i = s.begin / kPageRows; i < pages_for(s.end); ++i) {
            if (i >= pg.size()) {
                ++need;
            } else if (kv->refs[pg[i]] > 1) {
                int& holders = left.emplace(pg[i], kv->refs[pg[i]]).first->second;
                if (holders > 1) {
                    ++need;
                    --holders;
                }
            }
        }
    }
    if (need > kv->free_pages.size())
        return pfail(JX_ERR_NOMEM, "%zu pages are needed, %zu of %u are free", need,
                     kv->free_pages.size(), kv->d.n_pages);
    std::vector<TableEntry> table;
    std::vector<std::pair<int, int>> copies;
    table.reserve(need);
    copies.reserve(need);
    for (const Span& s : spans) {
        auto& pg = kv->pages[s.seq];
        for (uint32_t i = s.begin / kPageRows; i < pages_for(s.end); ++i) {
            if (i < pg.size() && kv->refs[pg[i]] == 1) continue;
            const int p = take_page(kv);
            if (i < pg.size()) {
                copies.emplace_back(pg[i], p);
                give_back(kv, pg[i]);
                pg[i] = p;
            } else {
                pg.push_back(p);
            }
            table.push_back({s.seq, i, p});
        }
    }
    if (int rc = copy_pages(kv, copies, st)) return rc;
    return set_table(kv, table, st);
}

// The table of (cos, sin) rows for a layer's RoPE setting, built on first use.
int rope_table(jx_pkv* kv, const jx_layer_desc& L, float yarn, bool neox, cudaStream_t st, int* cfg) {
    const uint32_t rdim = std::min(L.head_dim, L.rope_dim);  // (odd: its frequencies, one pair fewer)
    const float* rf = neox && !L.is_swa ? L.rope_freqs : nullptr;
    uint32_t bb, yb;
    std::memcpy(&bb, &L.rope_freq_base, 4);
    std::memcpy(&yb, &yarn, 4);
    for (size_t i = 0; i < kv->ropes.size(); ++i) {
        const RopeCfg& r = kv->ropes[i];
        if (r.rdim == rdim && r.base_bits == bb && r.yarn_bits == yb &&
            r.factors.size() == (rf ? rdim / 2 : 0) &&
            (!rf || std::memcmp(r.factors.data(), rf, rdim / 2 * sizeof(float)) == 0)) {
            *cfg = static_cast<int>(i);
            return JX_OK;
        }
    }
    if (kv->ropes.size() == kMaxRopeCfgs)
        return pfail(JX_ERR_UNSUPPORTED, "more than %d RoPE settings on one paged cache", kMaxRopeCfgs);
    RopeCfg r{rdim, bb, yb, {}, nullptr};
    if (rf) r.factors.assign(rf, rf + rdim / 2);
    RopeTable t;
    t.rows = static_cast<int>(kv->d.capacity);
    t.width = static_cast<int>(kv->d.head_dim / 2);
    t.half = static_cast<int>(rdim / 2);
    for (int j = 0; j < t.half; ++j) {
        t.freq[j] = std::pow(static_cast<double>(L.rope_freq_base), -2.0 * j / rdim) /
                    static_cast<double>(std::max(1e-4f, yarn));
        if (rf) t.freq[j] /= static_cast<double>(rf[j]);
    }
    const size_t n = static_cast<size_t>(t.rows) * t.width;
    if (cudaMalloc(&r.d_tab, n * sizeof(float2)) != cudaSuccess) {
        cudaGetLastError();
        return pfail(JX_ERR_NOMEM, "RoPE table of %zu bytes failed", n * sizeof(float2));
    }
    t.out = r.d_tab;
    rope_table_kernel<<<static_cast<unsigned>(std::min<size_t>((n + 255) / 256, 4096)), 256, 0, st>>>(t);
    if (int rc = launched("RoPE table")) {
        cudaFree(r.d_tab);
        return rc;
    }
    kv->ropes.push_back(std::move(r));
    *cfg = static_cast<int>(kv->ropes.size()) - 1;
    return JX_OK;
}

int check_device_ptr(const void* p, const char* name, int device, int align) {
    if (reinterpret_cast<uintptr_t>(p) % align != 0) return pfail(JX_ERR_INVALID, "%s must be aligned to %d bytes", name, align);
    cudaPointerAttributes at{};
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return pfail(JX_ERR_INVALID, "%s: not a CUDA-visible pointer (%s)", name, cudaGetErrorString(e));
    }
    if ((at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged) && at.device == device)
        return JX_OK;
    return pfail(JX_ERR_INVALID, "%s must be memory of device %d", name, device);
}

// A pinned buffer of `bytes` and its device copy, free to be written: used in
// turn, so that a call prepares its list while the previous one's is in use.
int take_upload(jx_pkv* kv, size_t bytes, jx_pkv::Upload** out) {
    jx_pkv::Upload& u = kv->up[kv->up_next];
    kv->up_next ^= 1;
    if (!u.done) PKV_CUDA(cudaEventCreateWithFlags(&u.done, cudaEventDisableTiming));
    if (u.pending) PKV_CUDA(cudaEventSynchronize(u.done));
    u.pending = false;
    if (u.bytes < bytes) {
        if (kv->opt_test_fail == 1) return pfail(JX_ERR_NOMEM, "list of %zu bytes failed (test_fail)", bytes);
        if (u.h) PKV_CUDA(cudaFreeHost(u.h));
        u.h = nullptr;
        if (u.d) PKV_CUDA(cudaFree(u.d));
        u.d = nullptr;
        u.bytes = 0;
        if (cudaHostAlloc(&u.h, 2 * bytes, cudaHostAllocDefault) != cudaSuccess ||
            cudaMalloc(&u.d, 2 * bytes) != cudaSuccess) {
            cudaGetLastError();
            return pfail(JX_ERR_NOMEM, "list of %zu bytes failed", 2 * bytes);
        }
        u.bytes = 2 * bytes;
    }
    *out = &u;
    return JX_OK;
}

// A list on its way: copied to the device, and the buffer's release queued behind the
// kernels that read it, whichever way the call ends.
struct SentUpload {
    jx_pkv::Upload* u;
    cudaStream_t st;
    SentUpload(jx_pkv::Upload* u_, cudaStream_t st_) : u(u_), st(st_) {}
    SentUpload(const SentUpload&) = delete;
    ~SentUpload() { u->pending = cudaEventRecord(u->done, st) == cudaSuccess; }
    int copy(size_t bytes) const {
        PKV_CUDA(cudaMemcpyAsync(u->d, u->h, bytes, cudaMemcpyHostToDevice, st));
        return JX_OK;
    }
};

int grow_device(jx_pkv* kv, void** p, size_t* have, size_t need, const char* what) {
    if (*have >= need) return JX_OK;
    if (kv->opt_test_fail == 1) return pfail(JX_ERR_NOMEM, "%s of %zu bytes failed (test_fail)", what, need);
    if (*p) {
        PKV_CUDA(cudaDeviceSynchronize());  // earlier calls may still be reading it
        PKV_CUDA(cudaFree(*p));
    }
    *p = nullptr;
    *have = 0;
    need = (need + (size_t{1} << 20) - 1) >> 20 << 20;
    if (cudaMalloc(p, need) != cudaSuccess) {
        cudaGetLastError();
        return pfail(JX_ERR_NOMEM, "%s of %zu bytes failed", what, need);
    }
    *have = need;
    return JX_OK;
}

// The rows of a call written to the given layers.
int append_rows(jx_pkv* kv, PagedArgs& A, const std::vector<PagedLayer>& part, const std::vector<PagedRun>& runs,
                cudaStream_t st, int* launches) {
    for (size_t l0 = 0; l0 < part.size(); l0 += kMaxCallLayers) {
        A.n_layers = static_cast<int>(std::min<size_t>(kMaxCallLayers, part.size() - l0));
        std::copy_n(part.begin() + l0, A.n_layers, A.layers);
        for (size_t r0 = 0; r0 < runs.size(); r0 += kMaxRuns) {
            A.n_runs = static_cast<int>(std::min<size_t>(kMaxRuns, runs.size() - r0));
            A.total = 0;
            for (int i = 0; i < A.n_runs; ++i) {
                PagedRun r = runs[r0 + i];
                r.off = A.total;
                A.total += (r.pos0 + r.n - 1) / kBlockRows - r.pos0 / kBlockRows + 1;
                A.runs[i] = r;
            }
            const dim3 grid(A.total, static_cast<unsigned>(A.n_layers * A.n_kv));
            dispatch(kv->d, [&](auto hd, auto dt) {
                append_kernel<hd.value, dt.value><<<grid, 2 * hd.value, 0, st>>>(A);
            });
            ++*launches;
            if (int rc = launched("append")) return rc;
        }
    }
    return JX_OK;
}

// The step kernel over the given layers and runs (of at most 8 / G tokens),
// in as many launches as their plan takes: at most 64 layers, 128 runs and 2^30
// units (of one layer a sequence cannot have more: 2^30 records are 2 TB).
int step_rows(jx_pkv* kv, PagedArgs& A, const std::vector<PagedLayer>& part, const std::vector<PagedRun>& runs,
              cudaStream_t st, int* launches) {
    constexpr long long kMaxUnits = 1ll << 30;
    long long longest = 1;
    for (const PagedRun& r : runs) longest = std::max<long long>(longest, (r.pos0 + r.n - 1) / kPageRows + 1 + kPieceCost);
    const size_t most = static_cast<size_t>(
        std::min<long long>(kMaxCallLayers, std::max<long long>(1, kMaxUnits / (longest * A.n_kv))));
    for (size_t l0 = 0; l0 < part.size(); l0 += most) {
        A.n_layers = static_cast<int>(std::min(most, part.size() - l0));
        std::copy_n(part.begin() + l0, A.n_layers, A.layers);
        std::stable_partition(A.layers, A.layers + A.n_layers,
                              [](const PagedLayer& L) { return !(L.flags & kLayerWindow); });
        A.n_full = static_cast<int>(std::count_if(A.layers, A.layers + A.n_layers, [](const PagedLayer& L) {
            return !(L.flags & kLayerWindow);
        }));
        const long long seg0 = static_cast<long long>(A.n_full) * A.n_kv;
        const long long seg1 = static_cast<long long>(A.n_layers - A.n_full) * A.n_kv;
        for (size_t r0 = 0; r0 < runs.size();) {
            long long p0 = 0, p1 = 0;
            int cols = 1;
            A.n_runs = 0;
            for (; A.n_runs < kMaxRuns && r0 < runs.size(); ++r0) {
                PagedRun r = runs[r0];
                const int last = r.pos0 + r.n - 1;
                const int n0 = last / kPageRows + 1 + kPieceCost;
                const int n1 = last / kPageRows - std::max(0, r.pos0 - A.window + 1) / kPageRows + 1 + kPieceCost;
                if (A.n_runs > 0 && (p0 + n0) * seg0 + (p1 + n1) * seg1 > kMaxUnits) break;
                r.off = static_cast<int>(p0);
                r.off1 = static_cast<int>(p1);
                p0 += n0;
                p1 += n1;
                cols = std::max(cols, r.n * A.G);
                A.runs[A.n_runs++] = r;
            }
            A.units0 = static_cast<int>(p0);
            A.units1 = static_cast<int>(p1);
            A.total0 = static_cast<int>(p0 * seg0);
            A.total = static_cast<int>(p0 * seg0 + p1 * seg1);
            const auto launch = kv->d.dtype == JX_I8 ? paged_step_i8 : paged_step_e4m3;
            const cudaError_t e = launch(A, static_cast<int>(kv->d.head_dim), cols, kv->num_sms, st);
            if (e != cudaSuccess) return pfail(JX_ERR_CUDA, "step launch failed: %s", cudaGetErrorString(e));
            ++*launches;
        }
    }
    return JX_OK;
}

// fp16 rows held at one time.  A group of layers grows until its rows would
// leave L2 (126 MB) before they are read, but not before its work items give
// every CTA several; never beyond the second figure.
constexpr size_t kWideL2 = size_t{64} << 20, kWideMost = size_t{1} << 30;
constexpr size_t kItemsPerCta = 8;
// K/V streams (one kv head of a layer and sequence) that CTAs read at one time
// where a group's rows exceed L2: as many as fit this.
constexpr size_t kStreamL2 = size_t{32} << 20;

// Whether a prompt goes to the tensor-core kernel or, in blocks of tokens, to the
// step kernel: by what each takes, in microseconds.  The step kernel reads a
// sequence's pages once per block, spread over all SMs (0.0135 ns per head_dim
// element and unit); the prompt kernel walks the tiles of an item one by one on
// one SM (3.4 us per 128 rows at head_dim 64, 4.6 at 128), after bringing the rows
// to fp16.  Measured, one layer of 8 kv heads and 4 heads each, blocks / tensor
// cores: head_dim 64, 256 tokens 35 / 32 us, behind 8192 rows 242 / 240 us, 64
// tokens behind them 74 / 235 us; head_dim 128, 96 tokens behind 8192 rows 193 /
// 310 us, 256 tokens 480 / 316 us.
bool prompt_on_tensor_cores(const jx_pkv* kv, const PagedArgs& A, const std::vector<PagedLayer>& all,
                            const std::vector<PagedRun>& runs) {
    const int hd = static_cast<int>(kv->d.head_dim), nq = kStepCols / A.G, TQ = 2 * kPromptRows / A.G;
    double windowed = 0.0;
    for (const PagedLayer& L : all) windowed += (L.flags & kLayerWindow) ? 1.0 : 0.0;
    const double full = static_cast<double>(all.size()) - windowed;
    double units = 0.0, tiles = 0.0, longest = 0.0, rows = 0.0;
    for (const PagedRun& r : runs) {
        const double end = r.pos0 + r.n, mid = r.pos0 + 0.5 * r.n, win = A.window;
        const double blocks = (r.n + nq - 1) / nq, items = (r.n + TQ - 1) / TQ;
        units += blocks * (full * (mid / kPageRows + 1 + kPieceCost) +
                           windowed * (std::min(mid, win) / kPageRows + 2 + kPieceCost));
        tiles += items * (full * (mid / kPromptRows + 1) + windowed * ((std::min(mid, win) + TQ) / kPromptRows + 1));
        longest = std::max(longest, (full > 0 ? end : std::min(end, win + TQ)) / kPromptRows + 1);
        rows += full * end + windowed * std::min(end, win + r.n);
    }
    units *= A.n_kv;
    tiles *= A.n_kv;
    const double by_blocks = 12.0 + units * hd * 1.35e-5;
    const double by_tiles = 18.0 + rows * A.n_kv * hd * 6 / 5e6 +
                            std::max(longest, tiles / std::max(kv->num_sms, 1)) * (hd == 64 ? 3.4 : 4.6);
    return by_tiles < by_blocks;
}

// Prompt attention on the tensor cores: the rows of a group of layers are
// brought to fp16 (see widen_kernel), then paged_prompt_kernel runs over them.
struct PromptPlan {
    struct Group {
        size_t r0, nr;
        std::vector<PagedLayer> layers;
        long long rows;          // per slot
        size_t items, at_items, at_first;
        int grid;
    };
    std::vector<Group> groups;
    jx_pkv::Upload* list = nullptr;  // items, then each CTA's first, of all groups
    size_t bytes = 0, first_at = 0;
};

// Groups, work items (laid out for the persistent CTAs: longest first, dealt in
// turn and back) and workspaces: all that can fail for lack of memory.  Changes
// nothing of the cache.
int plan_prompt(jx_pkv* kv, const PagedArgs& A, const std::vector<PagedLayer>& all, const std::vector<PagedRun>& runs,
                PromptPlan* plan) {
    const jx_pkv_desc& D = kv->d;
    const int hd = static_cast<int>(D.head_dim), G = A.G, TQ = 2 * kPromptRows / G, BN = kPromptRows;
    if (!tensor_map_encode()) return pfail(JX_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    using Group = PromptPlan::Group;
    std::vector<Group>& groups = plan->groups;
    const size_t row_bytes = static_cast<size_t>(D.n_kv_heads) * hd * 2;
    for (size_t r0 = 0; r0 < runs.size();) {
        // sequences whose rows of one layer fit the budget go together (one at least)
        long long rows = 0;
        size_t nr = 0;
        while (r0 + nr < runs.size() && nr < kMaxRuns) {
            const long long t = (static_cast<long long>(runs[r0 + nr].pos0) + runs[r0 + nr].n + 127) / 128 * 128;
            const long long m = std::max<long long>(rows, t);
            if (nr > 0 && 2 * row_bytes * m * (nr + 1) > kWideMost) break;
            rows = m;
            ++nr;
        }
        const size_t layer_bytes = 2 * row_bytes * rows * nr;
        size_t layer_items = 0;
        for (size_t i = 0; i < nr; ++i) layer_items += (runs[r0 + i].n + TQ - 1) / TQ * D.n_kv_heads;
        const size_t enough = kItemsPerCta * std::max(kv->num_sms, 1);
        const size_t per = std::min<size_t>(
            std::min<size_t>(kMaxCallLayers, std::max<size_t>(1, kWideMost / layer_bytes)),
            std::max<size_t>(std::max<size_t>(1, kWideL2 / layer_bytes), (enough + layer_items - 1) / layer_items));
        // layers of one RoPE setting share a launch
        std::vector<PagedLayer> order = all;
        std::stable_sort(order.begin(), order.end(), [](const PagedLayer& x, const PagedLayer& y) { return x.cfg < y.cfg; });
        for (size_t l0 = 0; l0 < order.size();) {
            Group g{r0, nr, {}, rows, 0, 0, 0, 0};
            while (l0 < order.size() && g.layers.size() < per && (g.layers.empty() || order[l0].cfg == g.layers[0].cfg))
                g.layers.push_back(order[l0++]);
            groups.push_back(std::move(g));
        }
        r0 += nr;
    }
    // the work items of every group, in one list
    std::vector<PrefillTile> items;
    std::vector<int> firsts;
    std::vector<PrefillTile> tiles;
    std::vector<std::pair<uint32_t, uint32_t>> order;  // (tile, kv head) of each item
    for (Group& g : groups) {
        tiles.clear();
        order.clear();
        for (size_t i = 0; i < g.nr; ++i) {
            const PagedRun& r = runs[g.r0 + i];
            for (int j = 0; j < r.n; j += TQ)
                for (size_t l = 0; l < g.layers.size(); ++l) {
                    const PagedLayer& L = g.layers[l];
                    PrefillTile t{};
                    t.seq = static_cast<int>(i);
                    t.cache_layer = static_cast<int>(l);
                    t.io0 = (r.io0 + j) * A.n_io_layers + L.io;
                    t.io_step = A.n_io_layers;
                    t.tok_row0 = r.pos0 + j;
                    t.ntok = std::min(TQ, r.n - j);
                    t.window = (L.flags & kLayerWindow) ? A.window : 0;
                    t.rope_row0 = t.tok_row0;
                    t.rope_half = L.half;
                    t.kv_lo = t.window > 0 ? std::max(0, t.tok_row0 - t.window + 1) : 0;
                    t.n_tiles = (t.tok_row0 + t.ntok - t.kv_lo + BN - 1) / BN;
                    tiles.push_back(t);
                }
        }
        std::stable_sort(tiles.begin(), tiles.end(), [](const PrefillTile& x, const PrefillTile& y) { return x.n_tiles > y.n_tiles; });
        const size_t n = tiles.size() * D.n_kv_heads;
        g.items = n;
        g.grid = static_cast<int>(std::min<size_t>(std::max(kv->num_sms, 1), n));
        g.at_items = items.size();
        g.at_first = firsts.size();
        for (uint32_t i = 0; i < tiles.size(); ++i)
            for (uint32_t h = 0; h < D.n_kv_heads; ++h) order.emplace_back(i, h);
        if (2 * row_bytes * g.rows * g.nr * g.layers.size() > 2 * kWideL2) {
            // more than L2 holds: stream by stream, a batch of streams at a time; the
            // last rounds longest first again, so that the CTAs end together
            const size_t batch = std::max<size_t>(1, kStreamL2 / (4 * static_cast<size_t>(g.rows) * hd));
            auto of = [&](const std::pair<uint32_t, uint32_t>& x) {
                const PrefillTile& t = tiles[x.first];
                return ((static_cast<size_t>(t.seq) * g.layers.size() + t.cache_layer) * D.n_kv_heads + x.second) / batch;
            };
            std::stable_sort(order.begin(), order.end(), [&](const auto& x, const auto& y) { return of(x) < of(y); });
            std::stable_sort(order.end() - static_cast<std::ptrdiff_t>(std::min<size_t>(n, 3 * g.grid)), order.end(),
                             [](const auto& x, const auto& y) { return x.first < y.first; });
        }
        const size_t P = static_cast<size_t>(g.grid);
        items.resize(items.size() + n);
        // CTA c runs the items at its place in each round of P, every other round reversed
        size_t at = g.at_items;
        for (size_t c = 0; c < P; ++c) {
            firsts.push_back(static_cast<int>(at - g.at_items));
            for (size_t round = 0;; ++round) {
                const size_t i = round * P + (round % 2 ? P - 1 - c : c);
                if (round * P >= n) break;
                if (i >= n) continue;
                items[at] = tiles[order[i].first];
                items[at++].kvh = static_cast<int>(order[i].second);
            }
        }
        firsts.push_back(static_cast<int>(at - g.at_items));
    }
    const size_t first_at = plan->first_at = items.size() * sizeof(PrefillTile);
    const size_t bytes = plan->bytes = first_at + firsts.size() * sizeof(int);
    size_t wide = 0, heads = 0;
    for (const Group& g : groups) {
        wide = std::max<size_t>(wide, 2 * row_bytes * g.rows * g.nr * g.layers.size());
        heads = std::max<size_t>(heads, g.nr * g.layers.size() * D.n_kv_heads);
    }
    if (int rc = grow_device(kv, reinterpret_cast<void**>(&kv->d_wide), &kv->wide_bytes, wide, "fp16 rows")) return rc;
    if (int rc = grow_device(kv, reinterpret_cast<void**>(&kv->d_head_scale), &kv->head_scales, heads * sizeof(float2), "head scales")) return rc;
    if (int rc = grow_device(kv, reinterpret_cast<void**>(&kv->d_totals), &kv->totals_bytes,
                             static_cast<size_t>(std::max(kv->num_sms, 1)) * 2 * hd * kPromptRows * sizeof(float), "totals"))
        return rc;
    if (int rc = take_upload(kv, bytes, &plan->list)) return rc;
    std::memcpy(plan->list->h, items.data(), first_at);
    std::memcpy(static_cast<char*>(plan->list->h) + first_at, firsts.data(), firsts.size() * sizeof(int));
    return JX_OK;
}

int run_prompt(jx_pkv* kv, const PagedArgs& A, const std::vector<PagedRun>& runs, const PromptPlan& plan,
               cudaStream_t st, int* launches) {
    const jx_pkv_desc& D = kv->d;
    const int hd = static_cast<int>(D.head_dim), G = A.G, BN = kPromptRows;
    const size_t row_bytes = static_cast<size_t>(D.n_kv_heads) * hd * 2;
    const TensorMapEncode enc = tensor_map_encode();
    jx_pkv::Upload* u = plan.list;
    const SentUpload sent(u, st);
    if (int rc = sent.copy(plan.bytes)) return rc;
    for (const PromptPlan::Group& g : plan.groups) {
        const size_t nl = g.layers.size();
        WidenArgs w{};
        w.pool = kv->pool;
        w.table = kv->d_table;
        w.page_bytes = kv->page_bytes;
        w.layer_bytes = kv->layer_bytes;
        w.layer_elems = static_cast<long long>(g.rows) * D.n_kv_heads * hd;
        w.slot_elems = w.layer_elems * static_cast<long long>(nl);
        w.out[0] = kv->d_wide;
        w.out[1] = kv->d_wide + w.slot_elems * static_cast<long long>(g.nr);
        w.head_scale = kv->d_head_scale;
        w.max_pages = A.max_pages;
        w.n_kv = A.n_kv;
        w.n_layers = static_cast<int>(nl);
        w.n_runs = static_cast<int>(g.nr);
        w.window = A.window;
        w.rows = static_cast<int>(g.rows);
        std::copy(g.layers.begin(), g.layers.end(), w.layers);
        int chunks = 0;
        for (size_t i = 0; i < g.nr; ++i) {
            w.runs[i] = runs[g.r0 + i];
            w.runs[i].off = chunks;
            chunks += (w.runs[i].pos0 + w.runs[i].n + kPromptRows + kWidenRows - 1) / kWidenRows;
        }
        const dim3 grid(chunks, static_cast<unsigned>(nl * A.n_kv));
        dispatch(D, [&](auto h, auto dt) { widen_kernel<h.value, dt.value><<<grid, 256, 0, st>>>(w); });
        if (int rc = launched("widen")) return rc;
        CUtensorMap maps[2];
        const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D.n_kv_heads) * hd, static_cast<cuuint64_t>(g.rows), nl, g.nr};
        const cuuint64_t strides[3] = {row_bytes, row_bytes * g.rows, row_bytes * g.rows * nl};
        const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(BN), 1, 1};
        const cuuint32_t one[4] = {1, 1, 1, 1};
        for (int k = 0; k < 2; ++k)
            if (enc(&maps[k], CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, w.out[k], dims, strides, box, one,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
                return pfail(JX_ERR_CUDA, "cuTensorMapEncodeTiled failed");
        PromptArgs p{};
        p.tiles = reinterpret_cast<const PrefillTile*>(u->d) + g.at_items;
        p.cta_first = reinterpret_cast<const int*>(static_cast<const char*>(u->d) + plan.first_at) + g.at_first;
        p.q = A.q;
        p.out = A.out;
        p.q_stride = A.q_stride;
        p.rope = A.rope[g.layers[0].cfg];
        p.head_scale = kv->d_head_scale;
        p.totals = kv->d_totals;
        p.scale_layers = static_cast<int>(nl);
        p.scale_heads = A.n_kv;
        p.neox = A.neox;
        p.q_vec = A.q_vec;
        p.scale = A.scale;
        p.softcap = A.softcap;
        p.cap_in = A.cap_in;
        p.cap_out = A.cap_out;
        p.err = A.err;
        p.dbg = A.dbg;
        p.wait_limit = A.wait_limit;
        const cudaError_t e = paged_prompt_launch(p, &maps[0], &maps[1], hd, G, g.grid, st);
        if (e != cudaSuccess) return pfail(JX_ERR_CUDA, "prompt launch failed: %s", cudaGetErrorString(e));
        *launches += 2;
    }
    return JX_OK;
}

int attn_call(jx_pkv* kv, const jx_layer_desc* layers, uint32_t n_layers, const jx_step_args* a,
              cudaStream_t st, bool prompt) {
    if (!kv || !layers || !a) return pfail(JX_ERR_INVALID, "null handle, layers or args");
    if (n_layers == 0 || a->n_seqs == 0) return pfail(JX_ERR_INVALID, "empty step");
    if (n_layers > 65535) return pfail(JX_ERR_INVALID, "more than 65535 layers");
    if (!a->pos || !a->q || !a->k || !a->v || !a->out)
        return pfail(JX_ERR_INVALID, "null pos/q/k/v/out");
    const jx_pkv_desc& D = kv->d;
    if (a->n_kv_heads != D.n_kv_heads || a->n_heads == 0 || a->n_heads % a->n_kv_heads != 0)
        return pfail(JX_ERR_INVALID, "n_kv_heads %u (the cache has %u) must match and divide n_heads %u",
                     a->n_kv_heads, D.n_kv_heads, a->n_heads);
    const uint32_t G = a->n_heads / a->n_kv_heads;
    if (G > 8) return pfail(JX_ERR_UNSUPPORTED, "query group of %u heads exceeds 8", G);
    if (!(a->yarn_scale >= 0.0f)) return pfail(JX_ERR_INVALID, "yarn_scale must not be negative or NaN");
    const uint64_t q_row = static_cast<uint64_t>(a->n_heads) * D.head_dim;
    const uint64_t kv_row = static_cast<uint64_t>(a->n_kv_heads) * D.head_dim;
    if (a->q_stride < q_row || a->kv_stride < kv_row)
        return pfail(JX_ERR_INVALID, "q_stride/kv_stride smaller than the layer's rows");
    if (static_cast<uint64_t>(a->n_seqs) * n_layers > 0x7FFFFFFFull)
        return pfail(JX_ERR_INVALID, "too many rows");
    std::vector<int> writer(D.n_layers, -1);
    for (uint32_t l = 0; l < n_layers; ++l) {
        const jx_layer_desc& L = layers[l];
        if (L.head_dim != D.head_dim)
            return pfail(JX_ERR_UNSUPPORTED, "layer %u: head_dim %u, the cache has %u", l, L.head_dim, D.head_dim);
        if (L.kv_source_layer >= D.n_layers)
            return pfail(JX_ERR_INVALID, "layer %u: kv_source_layer %u >= %u", l, L.kv_source_layer, D.n_layers);
        if (std::min(L.head_dim, L.rope_dim) >= 2 && (!(L.rope_freq_base > 0.0f) || !std::isfinite(L.rope_freq_base)))
            return pfail(JX_ERR_INVALID, "layer %u: rope_freq_base must be positive", l);
        if (!L.shares_kv) {
            if (writer[L.kv_source_layer] >= 0)
                return pfail(JX_ERR_INVALID, "layers %d and %u both write cache layer %u",
                             writer[L.kv_source_layer], l, L.kv_source_layer);
            writer[L.kv_source_layer] = static_cast<int>(l);
        }
    }
    // runs: rows of one sequence at consecutive positions
    std::vector<PagedRun> runs;
    std::vector<char> seen(D.n_seqs, 0);
    bool any_write = false;
    for (uint32_t l = 0; l < n_layers; ++l) any_write = any_write || !layers[l].shares_kv;
    for (uint32_t i = 0; i < a->n_seqs; ++i) {
        const int sid = a->seq_ids ? a->seq_ids[i] : (prompt ? 0 : static_cast<int>(i));
        if (sid < 0 || static_cast<uint32_t>(sid) >= D.n_seqs)
            return pfail(JX_ERR_INVALID, "sequence id %d outside [0, %u)", sid, D.n_seqs);
        const int p = a->pos[i];
        if (p < 0) return pfail(JX_ERR_INVALID, "negative position");
        if (static_cast<uint32_t>(p) >= D.capacity)
            return pfail(JX_ERR_RANGE, "position %d is beyond the capacity of %u rows", p, D.capacity);
        if (!runs.empty() && runs.back().seq == sid) {
            if (!prompt) return pfail(JX_ERR_INVALID, "sequence id %d listed twice", sid);
            PagedRun& r = runs.back();
            if (p != r.pos0 + r.n)
                return pfail(JX_ERR_INVALID, "a prompt's rows of one sequence must ascend by one "
                             "(sequence %d: position %d after %d)", sid, p, r.pos0 + r.n - 1);
            ++r.n;
            continue;
        }
        if (seen[sid]) return pfail(JX_ERR_INVALID, prompt ? "the rows of sequence %d must stand together"
                                                           : "sequence id %d listed twice", sid);
        seen[sid] = 1;
        runs.push_back(PagedRun{sid, p, 1, static_cast<int>(i), 0, 0});
    }
    std::vector<Span> spans;
    for (const PagedRun& r : runs) {
        const uint32_t held = kv->rows[r.seq], end = static_cast<uint32_t>(r.pos0 + r.n);
        if (any_write ? static_cast<uint32_t>(r.pos0) > held : end > held)
            return pfail(JX_ERR_RANGE, "sequence %d holds %u rows: position %d leaves a gap", r.seq, held, r.pos0);
        spans.push_back(Span{static_cast<uint32_t>(r.seq), static_cast<uint32_t>(r.pos0), end});
    }
    const void* ptrs[4] = {a->q, a->k, a->v, a->out};
    const char* names[4] = {"q", "k", "v", "out"};
    OnDevice on(D.device);
    if (!on.ok) return pfail(JX_ERR_CUDA, "cannot select device %d", D.device);
    for (int i = 0; i < 4; ++i)
        if (int rc = check_device_ptr(ptrs[i], names[i], D.device, 4)) return rc;
    if (int rc = refuse_capture(st)) return rc;
    std::vector<PagedLayer> all(n_layers);
    PagedArgs A{};
    for (uint32_t l = 0; l < n_layers; ++l) {
        const jx_layer_desc& L = layers[l];
        int cfg = 0;
        if (int rc = rope_table(kv, L, a->yarn_scale, a->rope_neox != 0, st, &cfg)) return rc;
        all[l].cache_layer = static_cast<uint16_t>(L.kv_source_layer);
        all[l].io = static_cast<uint16_t>(l);
        all[l].half = static_cast<uint16_t>(std::min(L.head_dim, L.rope_dim) / 2);
        all[l].cfg = static_cast<uint8_t>(cfg);
        all[l].flags = static_cast<uint8_t>((L.is_swa && a->sliding_window > 0 ? kLayerWindow : 0) |
                                            (L.shares_kv ? 0 : kLayerAppend));
    }
    for (size_t i = 0; i < kv->ropes.size(); ++i) A.rope[i] = kv->ropes[i].d_tab;
    A.pool = kv->pool;
    A.table = kv->d_table;
    A.page_bytes = kv->page_bytes;
    A.layer_bytes = kv->layer_bytes;
    A.max_pages = static_cast<int>(kv->max_pages);
    A.n_kv = static_cast<int>(D.n_kv_heads);
    A.G = static_cast<int>(G);
    A.n_io_layers = static_cast<int>(n_layers);
    A.q = a->q;
    A.k_in = a->k;
    A.v_in = a->v;
    A.out = a->out;
    A.q_stride = a->q_stride;
    A.kv_stride = a->kv_stride;
    A.scale = a->scale;
    A.softcap = a->softcap;
    A.cap_out = a->softcap * 1.4426950408889634f;
    A.cap_in = a->softcap > 0.0f ? 1.0f / A.cap_out : 0.0f;
    A.window = static_cast<int>(std::min<uint32_t>(a->sliding_window, 0x7FFFFFFFu));
    A.neox = a->rope_neox != 0 ? 1 : 0;
    A.err = kv->d_err;
    A.dbg = kv->d_dbg;
    A.wait_limit = wait_limit_cycles(kv->opt_wait_limit_ms);
    A.test_wait_cta = kv->opt_test_wait_cta;
    A.q_vec = reinterpret_cast<uintptr_t>(a->q) % 16 == 0 && a->q_stride % 4 == 0;
    A.kv_vec = reinterpret_cast<uintptr_t>(a->k) % 16 == 0 && reinterpret_cast<uintptr_t>(a->v) % 16 == 0 &&
               a->kv_stride % 4 == 0;
    // the prompt kernel writes its rows 16 bytes at a time
    const bool out_vec = reinterpret_cast<uintptr_t>(a->out) % 16 == 0 && a->q_stride % 4 == 0;
    A.scratch = kv->d_scratch;
    A.counters = kv->d_counters;
    // Attention of a prompt: on the tensor cores, or (few tokens, or a shape that kernel
    // does not take) for blocks of as many tokens as fill the step kernel's columns.
    const bool tc = prompt && paged_prompt_supported(static_cast<int>(D.head_dim), static_cast<int>(G)) && out_vec &&
                    a->scale > 0.0f &&
                    (kv->opt_prefill_tc < 0 ? prompt_on_tensor_cores(kv, A, all, runs) : kv->opt_prefill_tc > 0);
    // What can fail for lack of memory comes before the rows of the call are claimed.
    PromptPlan plan;
    std::vector<PagedLayer> first, second;
    std::vector<PagedRun> blocks;
    if (tc)
        if (int rc = plan_prompt(kv, A, all, runs, &plan)) return rc;
    for (const PagedLayer& L : all) {
        if (prompt) {
            if (L.flags & kLayerAppend) first.push_back(L);  // written before any attention
        } else {
            // a layer that reads rows another layer of the call writes goes second
            const bool later = !(L.flags & kLayerAppend) && writer[L.cache_layer] >= 0;
            (later ? second : first).push_back(L);
        }
    }
    if (prompt && !tc) {
        const int nq = std::max(1, kStepCols / static_cast<int>(G));
        for (const PagedRun& r : runs)
            for (int j = 0; j < r.n; j += nq)
                blocks.push_back(PagedRun{r.seq, r.pos0 + j, std::min(nq, r.n - j), r.io0 + j, 0, 0});
    }
    if (any_write) {
        if (int rc = make_room(kv, spans, st)) return rc;
        for (const Span& s : spans) {
            drop_rows(kv, s.seq, s.end);
            kv->rows[s.seq] = s.end;
        }
    }
    int launches = 0;
    if (prompt) {
        if (int rc = append_rows(kv, A, first, runs, st, &launches)) return rc;
        if (int rc = tc ? run_prompt(kv, A, runs, plan, st, &launches) : step_rows(kv, A, all, blocks, st, &launches))
            return rc;
    } else {
        A.append = 1;
        if (int rc = step_rows(kv, A, first, runs, st, &launches)) return rc;
        if (int rc = step_rows(kv, A, second, runs, st, &launches)) return rc;
    }
    kv->last_launches = launches;
    return JX_OK;
}

int keep_impl(jx_pkv* kv, uint32_t seq, const int32_t* rows, uint32_t n_rows, cudaStream_t st) {
    const jx_pkv_desc& D = kv->d;
    OnDevice on(D.device);
    if (!on.ok) return pfail(JX_ERR_CUDA, "cannot select device %d", D.device);
    if (int rc = refuse_capture(st)) return rc;
    uint32_t same = 0;  // leading rows that stay in place
    while (same < n_rows && rows[same] == static_cast<int32_t>(same)) ++same;
    if (same == n_rows) {  // nothing moves
        drop_rows(kv, seq, n_rows);
        return JX_OK;
    }
    auto& pg = kv->pages[seq];
    const uint32_t keep_pages = same / kPageRows, n_pages = pages_for(n_rows);
    const uint32_t fresh = n_pages - keep_pages;
    bool shared = false;
    for (uint32_t i = keep_pages; i < n_pages; ++i) shared = shared || kv->refs[pg[i]] > 1;
    const bool in_place = fresh > kv->free_pages.size();
    if (in_place && shared)
        return pfail(JX_ERR_NOMEM, "%u pages are needed (the sequence shares its own), %zu of %u are free",
                     fresh, kv->free_pages.size(), D.n_pages);
    // [rows][source pages][result pages]
    const size_t n_src = pg.size(), n_list = n_rows + n_src + n_pages;
    jx_pkv::Upload* u = nullptr;
    if (int rc = take_upload(kv, n_list * sizeof(int), &u)) return rc;
    int* list = static_cast<int*>(u->h);
    std::memcpy(list, rows, n_rows * sizeof(int));
    std::memcpy(list + n_rows, pg.data(), n_src * sizeof(int));
    std::vector<int> result(pg.begin(), pg.begin() + n_pages);
    std::vector<TableEntry> table;
    table.reserve(fresh);
    struct Fresh {  // pages taken for the result, given back unless the call succeeds
        jx_pkv* kv;
        std::vector<int>& result;
        uint32_t first;
        bool taken;
        ~Fresh() {
            if (taken)
                for (size_t i = result.size(); i > first; --i) give_back(kv, result[i - 1]);
        }
    } hold{kv, result, keep_pages, false};
    if (!in_place) {
        for (uint32_t i = keep_pages; i < n_pages; ++i) result[i] = take_page(kv);
        hold.taken = true;
    }
    std::memcpy(list + n_rows + n_src, result.data(), n_pages * sizeof(int));
    const SentUpload sent(u, st);
    if (int rc = sent.copy(n_list * sizeof(int))) return rc;
    const int* d_list = static_cast<const int*>(u->d);
    KeepArgs k{};
    k.pool = kv->pool;
    k.rows = d_list;
    k.src_table = d_list + n_rows;
    k.dst_table = d_list + n_rows + n_src;
    k.page_bytes = kv->page_bytes;
    k.n_rec = static_cast<int>(D.n_layers * D.n_kv_heads);
    k.n_rows = static_cast<int>(n_rows);
    k.blk0 = static_cast<int>(keep_pages * (kPageRows / kBlockRows));
    k.n_blk = static_cast<int>((n_rows + kBlockRows - 1) / kBlockRows) - k.blk0;
    k.serial = in_place ? 1 : 0;
    if (kv->opt_test_fail == 2) return pfail(JX_ERR_CUDA, "keep launch failed (test_fail)");
    const dim3 grid(in_place ? 1 : k.n_blk, (k.n_rec + kKeepRecords - 1) / kKeepRecords);
    dispatch(D, [&](auto hd, auto dt) {
        keep_kernel<hd.value, dt.value><<<grid, 2 * hd.value, 0, st>>>(k);
    });
    if (int rc = launched("keep")) return rc;
    if (in_place) {
        drop_rows(kv, seq, n_rows);
        return JX_OK;
    }
    hold.taken = false;
    for (uint32_t i = keep_pages; i < n_pages; ++i) table.push_back({seq, i, result[i]});
    for (size_t i = keep_pages; i < pg.size(); ++i) give_back(kv, pg[i]);
    pg = std::move(result);
    kv->rows[seq] = n_rows;
    return set_table(kv, table, st);
}

bool bad_seq(const jx_pkv* kv, uint32_t seq) { return !kv || seq >= kv->d.n_seqs; }

// No C++ exception crosses the C boundary.
template <typename F>
int guarded(F&& f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return pfail(JX_ERR_NOMEM, "out of host memory");
    } catch (...) {
        return pfail(JX_ERR_INVALID, "unexpected exception");
    }
}

}  // namespace

// ================================================================== C ABI

extern "C" {

int jx_pkv_create(const jx_pkv_desc* desc, jx_pkv** out) {
    return guarded([&]() -> int {
        if (!desc || !out) return pfail(JX_ERR_INVALID, "null desc/out");
        *out = nullptr;
        const jx_pkv_desc& d = *desc;
        if (d.n_seqs == 0 || d.n_layers == 0 || d.capacity == 0 || d.n_kv_heads == 0 || d.n_pages == 0)
            return pfail(JX_ERR_INVALID, "n_seqs, n_layers, capacity, n_kv_heads and n_pages must be positive");
        if (d.dtype != JX_I8 && d.dtype != JX_E4M3)
            return pfail(JX_ERR_INVALID, "dtype %d: a paged cache holds JX_I8 or JX_E4M3", d.dtype);
        if (d.head_dim != 32 && d.head_dim != 64 && d.head_dim != 128 && d.head_dim != 256)
            return pfail(JX_ERR_UNSUPPORTED, "head_dim %u (compiled: 32, 64, 128, 256)", d.head_dim);
        if (d.n_layers > 32767 || d.n_kv_heads > 512 ||
            static_cast<uint64_t>(d.n_layers) * d.n_kv_heads > 65535)
            return pfail(JX_ERR_UNSUPPORTED, "n_layers must be at most 32767, n_kv_heads 512, their product 65535");
        if (d.capacity > (1u << 30) || d.n_pages > (1u << 30) ||
            static_cast<uint64_t>(d.n_seqs) * ((d.capacity + kPageRows - 1) / kPageRows) > (1ull << 30))
            return pfail(JX_ERR_INVALID, "capacity, n_pages and the page table must stay below 2^30 entries");
        int ndev = 0;
        if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) {
            cudaGetLastError();
            return pfail(JX_ERR_CUDA, "no CUDA device (this library has no CPU path)");
        }
        if (d.device < 0 || d.device >= ndev) return pfail(JX_ERR_INVALID, "device %d absent", d.device);
        OnDevice on(d.device);
        if (!on.ok) return pfail(JX_ERR_CUDA, "cannot select device %d", d.device);
        int major = 0, sms = 0;
        PKV_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, d.device));
        PKV_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, d.device));
        if (major < 10) return pfail(JX_ERR_UNSUPPORTED, "device %d is older than this build's target, sm_100a", d.device);
        struct Destroy {
            void operator()(jx_pkv* k) const { jx_pkv_destroy(k); }
        };
        std::unique_ptr<jx_pkv, Destroy> owner(new jx_pkv());
        jx_pkv* kv = owner.get();
        kv->d = d;
        kv->num_sms = sms;
        kv->layer_bytes = static_cast<long long>(d.n_kv_heads) * record_bytes(static_cast<int>(d.head_dim));
        kv->page_bytes = kv->layer_bytes * d.n_layers;
        kv->max_pages = pages_for(d.capacity);
        kv->refs.assign(d.n_pages, 0);
        kv->pages.resize(d.n_seqs);
        kv->rows.assign(d.n_seqs, 0);
        kv->free_pages.resize(d.n_pages);
        for (uint32_t i = 0; i < d.n_pages; ++i) kv->free_pages[i] = static_cast<int>(d.n_pages - 1 - i);
        const size_t bytes = static_cast<size_t>(kv->page_bytes) * d.n_pages;
        const size_t tb = static_cast<size_t>(d.n_seqs) * kv->max_pages * sizeof(int);
        if (cudaMalloc(&kv->pool, bytes) != cudaSuccess || cudaMalloc(&kv->d_table, tb) != cudaSuccess) {
            cudaGetLastError();
            return pfail(JX_ERR_NOMEM, "page pool of %zu bytes failed", bytes);
        }
        const size_t ctas = static_cast<size_t>(sms) * kStepCtasPerSm;
        const size_t part = 2 * ctas * kStepCols * (d.head_dim + 4) * sizeof(float);
        if (cudaMalloc(&kv->d_scratch, part) != cudaSuccess || cudaMalloc(&kv->d_counters, ctas * sizeof(int)) != cudaSuccess ||
            cudaMemset(kv->d_counters, 0, ctas * sizeof(int)) != cudaSuccess) {
            cudaGetLastError();
            return pfail(JX_ERR_NOMEM, "scratch of %zu bytes failed", part);
        }
        if (cudaMemset(kv->pool, 0, bytes) != cudaSuccess || cudaMemset(kv->d_table, 0, tb) != cudaSuccess ||
            cudaMalloc(&kv->d_err, sizeof(int)) != cudaSuccess || cudaMemset(kv->d_err, 0, sizeof(int)) != cudaSuccess ||
            cudaMalloc(&kv->d_dbg, 8 * sizeof(int)) != cudaSuccess ||
            cudaMemset(kv->d_dbg, 0, 8 * sizeof(int)) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) {
            cudaGetLastError();
            return pfail(JX_ERR_CUDA, "cache initialisation failed");
        }
        *out = owner.release();
        return JX_OK;
    });
}

int jx_pkv_destroy(jx_pkv* kv) {
    if (!kv) return JX_OK;
    OnDevice on(kv->d.device);
    cudaDeviceSynchronize();
    cudaFree(kv->pool);
    cudaFree(kv->d_table);
    cudaFree(kv->d_scratch);
    cudaFree(kv->d_counters);
    cudaFree(kv->d_err);
    cudaFree(kv->d_dbg);
    cudaFree(kv->d_wide);
    cudaFree(kv->d_head_scale);
    cudaFree(kv->d_totals);
    for (auto& u : kv->up) {
        cudaFree(u.d);
        if (u.h) cudaFreeHost(u.h);
        if (u.done) cudaEventDestroy(u.done);
    }
    for (RopeCfg& r : kv->ropes) cudaFree(r.d_tab);
    delete kv;
    return JX_OK;
}

int jx_pkv_get_desc(const jx_pkv* kv, jx_pkv_desc* desc) {
    if (!kv || !desc) return pfail(JX_ERR_INVALID, "null argument");
    *desc = kv->d;
    return JX_OK;
}

int jx_pkv_get_seq_pos(const jx_pkv* kv, uint32_t seq, uint32_t* seq_pos) {
    if (bad_seq(kv, seq) || !seq_pos) return pfail(JX_ERR_INVALID, "bad handle/sequence");
    *seq_pos = kv->rows[seq];
    return JX_OK;
}

int jx_pkv_set_seq_pos(jx_pkv* kv, uint32_t seq, uint32_t seq_pos) {
    if (bad_seq(kv, seq)) return pfail(JX_ERR_INVALID, "bad handle/sequence");
    if (seq_pos > kv->rows[seq])
        return pfail(JX_ERR_RANGE, "sequence %u holds %u rows, not %u", seq, kv->rows[seq], seq_pos);
    return jx_pkv_rollback(kv, seq, seq_pos);
}

int jx_pkv_free_pages(const jx_pkv* kv, uint32_t* n) {
    if (!kv || !n) return pfail(JX_ERR_INVALID, "null argument");
    *n = static_cast<uint32_t>(kv->free_pages.size());
    return JX_OK;
}

int jx_pkv_held_pages(const jx_pkv* kv, uint32_t seq, uint32_t* n) {
    if (bad_seq(kv, seq) || !n) return pfail(JX_ERR_INVALID, "bad handle/sequence");
    *n = static_cast<uint32_t>(kv->pages[seq].size());
    return JX_OK;
}

int jx_pkv_clear(jx_pkv* kv, uint32_t seq) { return jx_pkv_rollback(kv, seq, 0); }

int jx_pkv_rollback(jx_pkv* kv, uint32_t seq, uint32_t new_seq_pos) {
    return guarded([&]() -> int {
        if (bad_seq(kv, seq)) return pfail(JX_ERR_INVALID, "bad handle/sequence");
        if (new_seq_pos < kv->rows[seq]) drop_rows(kv, seq, new_seq_pos);
        return JX_OK;
    });
}

int jx_pkv_fork(jx_pkv* kv, uint32_t src, uint32_t dst, uint32_t n_rows, void* stream) {
    return guarded([&]() -> int {
        if (bad_seq(kv, src) || bad_seq(kv, dst) || src == dst)
            return pfail(JX_ERR_INVALID, "bad handle/sequence, or a sequence forked into itself");
        if (n_rows > kv->rows[src])
            return pfail(JX_ERR_RANGE, "sequence %u holds %u rows, not %u", src, kv->rows[src], n_rows);
        OnDevice on(kv->d.device);
        if (!on.ok) return pfail(JX_ERR_CUDA, "cannot select device %d", kv->d.device);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (int rc = refuse_capture(st)) return rc;
        const uint32_t n = pages_for(n_rows);
        std::vector<int> pg(kv->pages[src].begin(), kv->pages[src].begin() + n);
        for (int p : pg) ++kv->refs[p];  // before dst's are given back: it may hold the same pages
        drop_rows(kv, dst, 0);
        kv->pages[dst] = std::move(pg);
        kv->rows[dst] = n_rows;
        if (n == 0) return JX_OK;
        table_copy_kernel<<<std::min<uint32_t>((n + 255) / 256, 148), 256, 0, st>>>(
            kv->d_table + static_cast<size_t>(dst) * kv->max_pages,
            kv->d_table + static_cast<size_t>(src) * kv->max_pages, static_cast<int>(n));
        return launched("page table copy");
    });
}

int jx_pkv_copy(jx_pkv* kv, uint32_t src, uint32_t dst, void* stream) {
    return guarded([&]() -> int {
        if (bad_seq(kv, src) || bad_seq(kv, dst) || src == dst)
            return pfail(JX_ERR_INVALID, "bad handle/sequence, or a sequence copied into itself");
        OnDevice on(kv->d.device);
        if (!on.ok) return pfail(JX_ERR_CUDA, "cannot select device %d", kv->d.device);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (int rc = refuse_capture(st)) return rc;
        const auto& from = kv->pages[src];
        size_t freed = 0;  // pages that only dst holds come free first
        for (int p : kv->pages[dst]) freed += kv->refs[p] == 1;
        if (from.size() > kv->free_pages.size() + freed)
            return pfail(JX_ERR_NOMEM, "%zu pages are needed, %zu of %u are free", from.size(),
                         kv->free_pages.size() + freed, kv->d.n_pages);
        std::vector<TableEntry> table;
        std::vector<std::pair<int, int>> copies;
        table.reserve(from.size());
        copies.reserve(from.size());
        kv->pages[dst].reserve(from.size());
        drop_rows(kv, dst, 0);
        for (size_t i = 0; i < from.size(); ++i) {
            const int p = take_page(kv);
            kv->pages[dst].push_back(p);
            copies.emplace_back(from[i], p);
            table.push_back({dst, static_cast<uint32_t>(i), p});
        }
        kv->rows[dst] = kv->rows[src];
        if (int rc = copy_pages(kv, copies, st)) return rc;
        return set_table(kv, table, st);
    });
}

int jx_pkv_keep(jx_pkv* kv, uint32_t seq, const int32_t* rows, uint32_t n_rows, void* stream) {
    return guarded([&]() -> int {
        if (bad_seq(kv, seq) || (!rows && n_rows > 0)) return pfail(JX_ERR_INVALID, "bad handle/sequence/rows");
        for (uint32_t i = 0; i < n_rows; ++i)
            if (rows[i] < 0 || static_cast<uint32_t>(rows[i]) >= kv->rows[seq] || (i > 0 && rows[i] <= rows[i - 1]))
                return pfail(JX_ERR_INVALID, "rows must ascend and stay below %u (entry %u is %d)", kv->rows[seq], i, rows[i]);
        return keep_impl(kv, seq, rows, n_rows, static_cast<cudaStream_t>(stream));
    });
}

int jx_pkv_compact(jx_pkv* kv, uint32_t seq, uint32_t keep_recent, void* stream) {
    return guarded([&]() -> int {
        if (bad_seq(kv, seq)) return pfail(JX_ERR_INVALID, "bad handle/sequence");
        const uint32_t sink = 4, sp = kv->rows[seq];
        if (static_cast<uint64_t>(sp) <= static_cast<uint64_t>(sink) + keep_recent) return JX_OK;
        std::vector<int32_t> rows;
        rows.reserve(sink + keep_recent);
        for (uint32_t i = 0; i < sink; ++i) rows.push_back(static_cast<int32_t>(i));
        for (uint32_t i = sp - keep_recent; i < sp; ++i) rows.push_back(static_cast<int32_t>(i));
        return keep_impl(kv, seq, rows.data(), static_cast<uint32_t>(rows.size()), static_cast<cudaStream_t>(stream));
    });
}

int jx_pkv_load_rows(jx_pkv* kv, uint32_t seq, uint32_t row0, uint32_t n_rows, const void* k_codes,
                     const float* k_scales, const void* v_codes, const float* v_scales, void* stream) {
    return guarded([&]() -> int {
        if (bad_seq(kv, seq)) return pfail(JX_ERR_INVALID, "bad handle/sequence");
        const jx_pkv_desc& D = kv->d;
        if (n_rows == 0) return JX_OK;
        if (row0 % kBlockRows != 0) return pfail(JX_ERR_INVALID, "row0 must be a multiple of %d", kBlockRows);
        if (static_cast<uint64_t>(row0) + n_rows > D.capacity || row0 > kv->rows[seq])
            return pfail(JX_ERR_RANGE, "rows [%u, %llu): the sequence holds %u, its capacity is %u", row0,
                         static_cast<unsigned long long>(row0) + n_rows, kv->rows[seq], D.capacity);
        OnDevice on(D.device);
        if (!on.ok) return pfail(JX_ERR_CUDA, "cannot select device %d", D.device);
        const void* ptrs[4] = {k_codes, k_scales, v_codes, v_scales};
        const char* names[4] = {"k_codes", "k_scales", "v_codes", "v_scales"};
        for (int i = 0; i < 4; ++i)
            if (int rc = check_device_ptr(ptrs[i], names[i], D.device, i % 2 ? 4 : 16)) return rc;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (int rc = refuse_capture(st)) return rc;
        if (int rc = make_room(kv, {Span{seq, row0, row0 + n_rows}}, st)) return rc;
        drop_rows(kv, seq, row0 + n_rows);
        kv->rows[seq] = row0 + n_rows;
        LoadArgs a{};
        a.pool = kv->pool;
        a.table = kv->d_table + static_cast<size_t>(seq) * kv->max_pages;
        a.codes[0] = static_cast<const unsigned char*>(k_codes);
        a.codes[1] = static_cast<const unsigned char*>(v_codes);
        a.scales[0] = k_scales;
        a.scales[1] = v_scales;
        a.page_bytes = kv->page_bytes;
        a.row0 = static_cast<int>(row0);
        a.n_rows = static_cast<int>(n_rows);
        a.n_kv = static_cast<int>(D.n_kv_heads);
        a.n_layers = static_cast<int>(D.n_layers);
        const long long n = static_cast<long long>(D.n_layers) * n_rows * D.n_kv_heads * (D.head_dim / 16);
        const dim3 grid(static_cast<unsigned>(std::min<long long>((n + 255) / 256, 8ll * kv->num_sms)), 2);
        dispatch(D, [&](auto hd, auto dt) { load_kernel<hd.value, dt.value><<<grid, 256, 0, st>>>(a); });
        return launched("load");
    });
}

int jx_pkv_read_rows(jx_pkv* kv, const int32_t* seq_ids, const int32_t* row0, uint32_t n, uint32_t n_rows,
                     int32_t dtype, void* out, void* stream) {
    return guarded([&]() -> int {
        if (!kv || !seq_ids || !row0) return pfail(JX_ERR_INVALID, "null argument");
        const jx_pkv_desc& D = kv->d;
        if (dtype != JX_F32 && dtype != JX_BF16) return pfail(JX_ERR_INVALID, "rows are read as JX_F32 or JX_BF16");
        for (uint32_t i = 0; i < n; ++i) {
            if (seq_ids[i] < 0 || bad_seq(kv, static_cast<uint32_t>(seq_ids[i])))
                return pfail(JX_ERR_INVALID, "sequence id %d outside [0, %u)", seq_ids[i], D.n_seqs);
            if (row0[i] < 0 || static_cast<uint64_t>(row0[i]) + n_rows > kv->rows[seq_ids[i]])
                return pfail(JX_ERR_RANGE, "sequence %d holds %u rows, not [%d, %lld)", seq_ids[i],
                             kv->rows[seq_ids[i]], row0[i], static_cast<long long>(row0[i]) + n_rows);
        }
        if (n == 0 || n_rows == 0) return JX_OK;
        OnDevice on(D.device);
        if (!on.ok) return pfail(JX_ERR_CUDA, "cannot select device %d", D.device);
        if (int rc = check_device_ptr(out, "out", D.device, 16)) return rc;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (int rc = refuse_capture(st)) return rc;
        ReadArgs a{};
        a.pool = kv->pool;
        a.table = kv->d_table;
        a.page_bytes = kv->page_bytes;
        a.max_pages = static_cast<int>(kv->max_pages);
        a.n_kv = static_cast<int>(D.n_kv_heads);
        a.n_layers = static_cast<int>(D.n_layers);
        a.n_rows = static_cast<int>(n_rows);
        const long long per = static_cast<long long>(D.n_layers) * 2 * n_rows * D.n_kv_heads * (D.head_dim / 16);
        const uint32_t per_row = D.n_kv_heads * (D.head_dim / 16);
        const uint32_t most = (1u << 30) / per_row;  // rows of a launch: 32-bit indices
        for (uint32_t s0 = 0; s0 < n; s0 += kMaxRuns) {
            a.n = static_cast<int>(std::min<uint32_t>(kMaxRuns, n - s0));
            std::copy_n(seq_ids + s0, a.n, a.seq);
            std::copy_n(row0 + s0, a.n, a.row0);
            a.out = static_cast<char*>(out) + static_cast<size_t>(s0) * per * 16 * (dtype == JX_F32 ? 4 : 2);
            for (uint32_t r0 = 0; r0 < n_rows; r0 += most) {
                a.r0 = static_cast<int>(r0);
                a.rows = static_cast<int>(std::min(most, n_rows - r0));
                const uint32_t work = static_cast<uint32_t>(a.rows) * per_row;
                const dim3 grid(std::min<uint32_t>((work + 255) / 256, 4096), D.n_layers * 2, a.n);
                dispatch(D, [&](auto hd, auto dt) {
                    if (dtype == JX_F32) read_kernel<hd.value, dt.value, true><<<grid, 256, 0, st>>>(a);
                    else read_kernel<hd.value, dt.value, false><<<grid, 256, 0, st>>>(a);
                });
                if (int rc = launched("read")) return rc;
            }
        }
        return JX_OK;
    });
}

int jx_pkv_attn_step(jx_pkv* kv, const jx_layer_desc* layers, uint32_t n_layers, const jx_step_args* args,
                     void* stream) {
    return guarded([&]() -> int {
        return attn_call(kv, layers, n_layers, args, static_cast<cudaStream_t>(stream), false);
    });
}

int jx_pkv_attn_prefill(jx_pkv* kv, const jx_layer_desc* layers, uint32_t n_layers, const jx_step_args* args,
                        void* stream) {
    return guarded([&]() -> int {
        return attn_call(kv, layers, n_layers, args, static_cast<cudaStream_t>(stream), true);
    });
}

int jx_pkv_check_device_error(jx_pkv* kv, int* code, void* stream) {
    if (!kv || !code) return pfail(JX_ERR_INVALID, "null argument");
    OnDevice on(kv->d.device);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int h = 0, dbg[8] = {0};
    PKV_CUDA(cudaMemcpyAsync(&h, kv->d_err, sizeof(int), cudaMemcpyDeviceToHost, st));
    PKV_CUDA(cudaMemcpyAsync(dbg, kv->d_dbg, sizeof dbg, cudaMemcpyDeviceToHost, st));
    PKV_CUDA(cudaStreamSynchronize(st));
    PKV_CUDA(cudaMemsetAsync(kv->d_err, 0, sizeof(int), st));
    PKV_CUDA(cudaMemsetAsync(kv->d_dbg, 0, sizeof dbg, st));
    PKV_CUDA(cudaStreamSynchronize(st));
    *code = h;
    if (h)
        return pfail(JX_ERR_DEVICE, "a kernel's bounded wait ran out: site %d block %d thread %d index %d (error %d)",
                     dbg[0] - 100, dbg[1], dbg[2], dbg[5], h);
    return JX_OK;
}

int jx_pkv_set_option(jx_pkv* kv, const char* key, int value) {
    if (!kv || !key) return pfail(JX_ERR_INVALID, "null argument");
    if (std::strcmp(key, "prefill_tc") == 0) {
        if (value < -1 || value > 1) return pfail(JX_ERR_INVALID, "prefill_tc must be 1, 0 or -1");
        kv->opt_prefill_tc = value;
        return JX_OK;
    }
    if (value < 0) return pfail(JX_ERR_INVALID, "%s must not be negative", key);
    if (std::strcmp(key, "wait_limit_ms") == 0) {
        kv->opt_wait_limit_ms = value;
        return JX_OK;
    }
    if (std::strcmp(key, "test_fail") == 0) {
        kv->opt_test_fail = value;
        return JX_OK;
    }
    if (std::strcmp(key, "test_wait_cta") == 0) {
        kv->opt_test_wait_cta = value;
        return JX_OK;
    }
    return pfail(JX_ERR_INVALID, "unknown option '%s'", key);
}

int jx_pkv_last_launch_count(const jx_pkv* kv, int* count) {
    if (!kv || !count) return pfail(JX_ERR_INVALID, "null argument");
    *count = kv->last_launches;
    return JX_OK;
}

}  // extern "C"
