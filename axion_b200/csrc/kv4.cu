// The paged KV cache in 4 bits (include/axkv.h): append, read, and attention
// over its pages.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "axkv.h"
#include "common.cuh"
#include "kv4.cuh"
#include "kv4_narrow.cuh"
#include "kv4_wide.cuh"
#include "runtime.h"

using namespace axq8;

namespace {

// The page of position p of sequence s, or null outside the table or the pool.
template <int HD>
__device__ __forceinline__ uint8_t* kv4_at(const Kv4Pages& c, int s, int p, int h) {
    if (s < 0 || s >= c.n_seqs || p < 0 || p >= c.max_blocks * kKv4Tokens) return nullptr;
    const int page = __ldcg(c.table + (int64_t)s * c.max_blocks + p / kKv4Tokens);
    if (page < 0 || page >= c.n_pages) return nullptr;
    return c.pages + ((int64_t)page * c.n_kv + h) * Kv4<HD>::BYTES;
}

// Append and read move 4 dims per lane: HD / 4 lanes to a (row, KV head), 8 lanes
// to a block.  Lane i of a head (dims 4 i ..) has half a K word, and one nibble of
// 4 bytes of V, whose other nibble is lane i ^ 2's.
template <int HD>
struct Kv4Lane {
    using F = Kv4<HD>;
    int b, k_at, v_at;   // block, byte offsets of the 4 K codes and of the first V byte in slot 0
    bool high;           // V codes are the high nibbles
    __device__ __forceinline__ explicit Kv4Lane(int i) {
        b = i / 8;
        k_at = F::k_byte(0, b, 2 * (i % 8));
        v_at = F::v_byte(0, i / 4, 4 * (i & 1));
        high = i & 2;
    }
    static constexpr int V_STEP = 16 * F::TPG;   // bytes from dim g to g + 1
    __device__ __forceinline__ int k(int slot) const { return k_at + slot * (HD / 2); }
    __device__ __forceinline__ int v(int slot) const { return v_at + F::v_byte(slot, 0, 0) - F::V; }
};

// Bound: HBM (4 + 0.5625 bytes a value); one read of the rows, all in registers.
// 4095 rows of 8 x 128: 20.7 us for 38 MB, 0.28 of the copy bandwidth, at 0.75 of
// the issue slots (rounding and packing); a warp per row and 32 dims took 38 us.
template <int HD>
__global__ void __launch_bounds__(256)
    kv4_append_kernel(Kv4Pages c, const float* __restrict__ k_rows, const float* __restrict__ v_rows,
                      int64_t ld, int n_rows, const int* __restrict__ row_seq,
                      const int* __restrict__ row_pos, int* __restrict__ status) {
    using F = Kv4<HD>;
    constexpr int LPR = HD / 4;
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LPR;
    const int i = threadIdx.x % LPR;
    const bool in = unit < (int64_t)n_rows * c.n_kv;
    const int r = in ? (int)(unit / c.n_kv) : 0, h = in ? (int)(unit % c.n_kv) : 0;
    const int64_t src = (int64_t)r * ld + (int64_t)h * HD + 4 * i;
    const float4 kx = __ldg(reinterpret_cast<const float4*>(k_rows + src));
    const float4 vx = __ldg(reinterpret_cast<const float4*>(v_rows + src));
    const int p = row_pos[r], slot = p & (kKv4Tokens - 1);
    uint8_t* base = in ? kv4_at<HD>(c, row_seq[r], p, h) : nullptr;
    if (in && !base && i == 0) record_status(status, AXQ8_ERR_INVALID);
    const Kv4Lane<HD> at(i);
    bool bad = false;
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        float x[4] = {kv ? vx.x : kx.x, kv ? vx.y : kx.y, kv ? vx.z : kx.z, kv ? vx.w : kx.w};
        float lo = 0.0f, hi = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] = kv4_clean(x[e], bad);
            lo = fminf(lo, x[e]);
            hi = fmaxf(hi, x[e]);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const int code = kv4_step_code(hi - lo);
        const float d = code ? kv4_step(code) : 1.0f;   // all zero: any step does
        const float inv = kv4_inverse(d);
        const float z = -kv4_round(lo, d, inv);
        uint32_t q = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) q |= kv4_whole(fminf(kv4_round(x[e], d, inv) + z, 15.0f)) << (4 * e);
        const uint32_t other = __shfl_xor_sync(0xffffffffu, q, 2);
        if (!base) continue;
        if (i % 8 == 0)
            *reinterpret_cast<uint16_t*>(base + (kv ? F::VS : F::KS) + F::scale(slot, at.b)) =
                (uint16_t)((code << 4) | kv4_whole(z));
        if (kv == 0) {
            *reinterpret_cast<uint16_t*>(base + at.k(slot)) = (uint16_t)q;
        } else {
            // the pair of lanes writes two of the four bytes each
            const uint32_t l = at.high ? other : q, u = at.high ? q : other;
            uint8_t* to = base + at.v(slot);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int g = e + (at.high ? 2 : 0);
                to[g * at.V_STEP] = (uint8_t)(((l >> (4 * g)) & 15) | ((u >> (4 * g)) & 15) << 4);
            }
        }
    }
    if (in && base && bad) record_status(status, AXQ8_ERR_INVALID);
}

// The same lanes the other way; 4095 rows: 13.4 us, waits on the page's loads.
template <int HD>
__global__ void __launch_bounds__(256)
    kv4_read_kernel(Kv4Pages c, float* __restrict__ k_rows, float* __restrict__ v_rows, int64_t ld,
                    int n_rows, const int* __restrict__ row_seq, const int* __restrict__ row_pos,
                    int* __restrict__ status) {
    using F = Kv4<HD>;
    constexpr int LPR = HD / 4;
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LPR;
    const int i = threadIdx.x % LPR;
    if (unit >= (int64_t)n_rows * c.n_kv) return;
    const int r = (int)(unit / c.n_kv), h = (int)(unit % c.n_kv);
    const int p = row_pos[r], slot = p & (kKv4Tokens - 1);
    const uint8_t* base = kv4_at<HD>(c, row_seq[r], p, h);
    float k[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (base) {
        const Kv4Lane<HD> at(i);
        const int ks = *reinterpret_cast<const uint16_t*>(base + F::KS + F::scale(slot, at.b));
        const int vs = *reinterpret_cast<const uint16_t*>(base + F::VS + F::scale(slot, at.b));
        const int kq = *reinterpret_cast<const uint16_t*>(base + at.k(slot));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int vq = base[at.v(slot) + e * at.V_STEP] >> (at.high ? 4 : 0);
            k[e] = kv4_step(ks >> 4) * (float)(((kq >> (4 * e)) & 15) - (ks & 15));
            v[e] = kv4_step(vs >> 4) * (float)((vq & 15) - (vs & 15));
        }
    } else if (i == 0) {
        record_status(status, AXQ8_ERR_INVALID);
    }
    const int64_t to = (int64_t)r * ld + (int64_t)h * HD + 4 * i;
    *reinterpret_cast<float4*>(k_rows + to) = make_float4(k[0], k[1], k[2], k[3]);
    *reinterpret_cast<float4*>(v_rows + to) = make_float4(v[0], v[1], v[2], v[3]);
}

int check_cache4(const axkv4_cache_t* c, const char* what) {
    if (!c || !c->pages || !c->block_table) return fail(AXQ8_ERR_INVALID, "%s: null cache pointer", what);
    if (c->page_tokens != kKv4Tokens)
        return fail(AXQ8_ERR_UNSUPPORTED, "%s: page_tokens must be 16", what);
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128)
        return fail(AXQ8_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64, 128)", what, c->head_dim);
    if (c->n_seqs <= 0 || c->n_pages <= 0 || c->max_blocks <= 0 || c->n_kv_heads <= 0)
        return fail(AXQ8_ERR_INVALID, "%s: non-positive cache dimension", what);
    if (c->n_kv_heads > 65535) return fail(AXQ8_ERR_UNSUPPORTED, "%s: %d KV heads", what, c->n_kv_heads);
    if (c->max_blocks > (1 << 26)) return fail(AXQ8_ERR_UNSUPPORTED, "%s: max_blocks %d", what, c->max_blocks);
    if (reinterpret_cast<uintptr_t>(c->pages) & 15)
        return fail(AXQ8_ERR_INVALID, "%s: pages not 16-byte aligned", what);
    return AXQ8_OK;
}

Kv4Pages pages_of(const axkv4_cache_t* c) {
    return {static_cast<uint8_t*>(c->pages), c->block_table, c->n_seqs, c->max_blocks, c->n_pages,
            c->n_kv_heads};
}

int check_rows(const axkv4_cache_t* c, const char* what, const void* k, const void* v, int64_t ld,
               int32_t n_rows, const void* seq, const void* pos) {
    int rc = check_cache4(c, what);
    if (rc) return rc;
    if (n_rows < 0) return fail(AXQ8_ERR_INVALID, "%s: n_rows < 0", what);
    if (n_rows == 0) return AXQ8_OK;
    if (!k || !v || !seq || !pos) return fail(AXQ8_ERR_INVALID, "%s: null pointer", what);
    if (ld < (int64_t)c->n_kv_heads * c->head_dim || ld % 4 ||
        ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15))
        return fail(AXQ8_ERR_INVALID, "%s: rows must be 16-byte aligned and %d floats or more apart", what,
                    c->n_kv_heads * c->head_dim);
    if (((int64_t)n_rows * c->n_kv_heads + 7) / 8 > 0x7fffffff)
        return fail(AXQ8_ERR_UNSUPPORTED, "%s: too many rows", what);
    return AXQ8_OK;
}

int check_attn(const axkv4_cache_t* c, const char* what, int32_t n_heads) {
    int rc = check_cache4(c, what);
    if (rc) return rc;
    if (n_heads <= 0 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 16)
        return fail(AXQ8_ERR_INVALID, "%s: n_heads must be a multiple of n_kv_heads (<= 16x)", what);
    return AXQ8_OK;
}

// fn<HD>(...) for the cache's head dim.
#define KV4_BY_HEAD_DIM(hd, fn, ...)               \
    ((hd) == 32   ? fn<32>(__VA_ARGS__)            \
     : (hd) == 64 ? fn<64>(__VA_ARGS__)            \
                  : fn<128>(__VA_ARGS__))

template <int HD>
cudaError_t launch_append(const axkv4_cache_t* c, const float* k, const float* v, int64_t ld, int n_rows,
                          const int* seq, const int* pos, int* status, cudaStream_t s) {
    const int64_t threads = (int64_t)n_rows * c->n_kv_heads * (HD / 4);
    return launch_k(kv4_append_kernel<HD>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, false,
                    pages_of(c), k, v, ld, n_rows, seq, pos, status);
}

template <int HD>
cudaError_t launch_read(const axkv4_cache_t* c, float* k, float* v, int64_t ld, int n_rows,
                        const int* seq, const int* pos, int* status, cudaStream_t s) {
    const int64_t threads = (int64_t)n_rows * c->n_kv_heads * (HD / 4);
    return launch_k(kv4_read_kernel<HD>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, false,
                    pages_of(c), k, v, ld, n_rows, seq, pos, status);
}

int narrow_cols(int64_t cols) { return cols <= 4 ? 4 : cols <= 8 ? 8 : 16; }

// Whether the column tiles' units of work (runs of them rounded up: at most twice as
// many) count in 32 bits.
int check_narrow(const axkv4_cache_t* c, const char* what, int entries, int rows, int G) {
    const int64_t cols = (int64_t)rows * G, per = narrow_cols(cols);
    const double tiles = (double)((cols + per - 1) / per) * c->n_kv_heads * entries;
    if (tiles * (c->max_blocks + kNarrowTileCost) * 2 > 2147483647.0)
        return fail(AXQ8_ERR_UNSUPPORTED, "%s: %d chunks of at most %d rows over %d pages", what, entries, rows,
                    c->max_blocks);
    return AXQ8_OK;
}

int check_decode(const axkv4_cache_t* c, const char* what, int32_t n_rows, int32_t n_heads) {
    const int rc = check_attn(c, what, n_heads);
    if (rc) return rc;
    if (n_rows < 0 || n_rows > (1 << 20)) return fail(AXQ8_ERR_INVALID, "%s: n_rows %d", what, n_rows);
    return check_narrow(c, what, n_rows, 1, n_heads / c->n_kv_heads);
}

int check_chunks(const axkv4_cache_t* c, const char* what, int32_t n_chunks, int32_t max_rows, int32_t n_heads) {
    const int rc = check_attn(c, what, n_heads);
    if (rc) return rc;
    if (n_chunks < 0 || max_rows < 0 || n_chunks > 65535 || max_rows > (1 << 24))
        return fail(AXQ8_ERR_INVALID, "%s: %d chunks of at most %d rows", what, n_chunks, max_rows);
    return AXQ8_OK;
}

// Columns of a tile, CTAs, and workspace bytes: a record per CTA, then two
// partial states per CTA.
struct NarrowPlan {
    int cols, ctas, aligned;
    int64_t records, workspace;
};

NarrowPlan narrow_plan(DeviceState* ds, const axkv4_cache_t* c, int entries, int rows, int G) {
    NarrowPlan p;
    const int64_t cols = (int64_t)rows * G;
    p.cols = narrow_cols(cols);
    const int slots = ds->sm_count * (p.cols <= 8 ? 3 : 2);
    const int64_t tiles = (cols + p.cols - 1) / p.cols * c->n_kv_heads * entries;
    // every tile starts a run where that leaves half of the runs; with the most
    // tiles a call can have (it may have fewer), this many runs are never exceeded
    p.aligned = 2 * tiles <= slots ? (int)tiles : 0;
    const int64_t runs = p.aligned ? (tiles * c->max_blocks + kNarrowMinPages - 1) / kNarrowMinPages + p.aligned
                                   : (tiles * (c->max_blocks + kNarrowTileCost) + kNarrowMinUnits - 1) / kNarrowMinUnits;
    p.ctas = (int)std::min<int64_t>(slots, runs);
    p.records = ((int64_t)p.ctas * sizeof(NarrowPart) + 15) / 16 * 16;
    p.workspace = p.records + (int64_t)p.ctas * 2 * p.cols * (c->head_dim + 2) * 4;
    return p;
}

template <int HD, int COLS>
cudaError_t launch_narrow_cols(DeviceState* ds, const NarrowArgs& a, int ctas, cudaStream_t s) {
    static_assert(NarrowCfg<HD, COLS>::CTAS == (COLS <= 8 ? 3 : 2), "narrow_plan");
    constexpr size_t smem = NarrowCfg<HD, COLS>::SMEM;
    auto kern = kv4_attn_narrow_kernel<HD, COLS>;
    static std::atomic<int> configured[64] = {};   // by device
    const int dev = ds->device < 64 ? ds->device : 63;
    if (dev == 63 || !configured[dev]) {   // with the kernel's static part, from less than 48 KB
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        configured[dev] = 1;
    }
    const cudaError_t e = launch_k(kern, dim3(ctas), dim3(kNarrowWarps * 32), smem, s, false, a);
    if (e != cudaSuccess) return e;
    constexpr int blocks = COLS * HD / 4 / NarrowCfg<HD, COLS>::JOIN_ITEMS;
    return launch_k(kv4_attn_join_kernel<HD, COLS>, dim3(ctas, blocks), dim3(kJoinThreads), 0, s, true, a);
}

template <int HD>
cudaError_t launch_narrow(DeviceState* ds, const NarrowPlan& p, const axkv4_cache_t* c, const float* q, int64_t ldq,
                          int n_rows, int chunks, int max_rows, int n_heads, const int* q_seq,
                          const int* q_start, const int* q_pos, float* out, void* ws, cudaStream_t s) {
    NarrowArgs a = {};
    a.c = pages_of(c);
    a.q = q;
    a.ldq = ldq;
    a.n_rows = n_rows;
    a.max_rows = max_rows;
    a.n_heads = n_heads;
    a.G = n_heads / c->n_kv_heads;
    a.n_entries = chunks;
    a.aligned = p.aligned;
    a.q_seq = q_seq;
    a.q_start = q_start;
    a.q_pos = q_pos;
    a.scale = 1.4426950408889634f / std::sqrt((float)HD);
    a.out = out;
    a.split = static_cast<NarrowPart*>(ws);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + p.records);
    a.status = ds->status;
    return p.cols == 4   ? launch_narrow_cols<HD, 4>(ds, a, p.ctas, s)
           : p.cols == 8 ? launch_narrow_cols<HD, 8>(ds, a, p.ctas, s)
                         : launch_narrow_cols<HD, 16>(ds, a, p.ctas, s);
}

template <int HD>
cudaError_t launch_wide(DeviceState* ds, const axkv4_cache_t* c, const float* q, int64_t ldq, int n_rows, int chunks,
                        int max_rows, int n_heads, const int* q_seq, const int* q_start,
                        const int* q_pos, float* out, cudaStream_t s) {
    WideArgs a = {};
    a.c = pages_of(c);
    a.q = q;
    a.ldq = ldq;
    a.n_rows = n_rows;
    a.max_rows = max_rows;
    a.n_heads = n_heads;
    a.G = n_heads / c->n_kv_heads;
    a.q_seq = q_seq;
    a.q_start = q_start;
    a.q_pos = q_pos;
    a.scale = 1.4426950408889634f / std::sqrt((float)HD);
    a.out = out;
    a.status = ds->status;
    constexpr size_t smem = WideCfg<HD>::SMEM;
    static std::atomic<int> configured[64] = {};   // by device
    const int dev = ds->device < 64 ? ds->device : 63;
    if (dev == 63 || !configured[dev]) {
        // the roles' register split draws on what the launch has
        cudaFuncAttributes fa;
        cudaError_t e = cudaFuncGetAttributes(&fa, kv4_attn_wide_kernel<HD>);
        if (e == cudaSuccess && fa.numRegs < kWideRegs) e = cudaErrorInvalidConfiguration;
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kv4_attn_wide_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)smem);
        if (e != cudaSuccess) return e;
        configured[dev] = 1;
    }
    const int64_t rows = (int64_t)std::min(max_rows, n_rows) * a.G;
    return launch_k(kv4_attn_wide_kernel<HD>, dim3((unsigned)((rows + 255) / 256), c->n_kv_heads, chunks),
                    dim3(kWideThreads), smem, s, false, a);
}

// Whether the tensor-core tiles of 256 rows (kv4_wide.cuh) take a chunk call, or the
// column tiles of 16 (kv4_narrow.cuh), which share a long context among all SMs.
// Measured per page of context at head dim 128 (64 and 32): a CTA of the first takes
// 0.67 us (0.48, 0.44), whatever its rows, one to an SM, and no other SM helps it; a tile
// of the second 0.18 us of an SM (0.12, 0.10), so the head dim hardly matters.  From a
// prompt's start a tile of the second walks twice the pages it needs, and short contexts
// cost it more beside the pages: 61 to 27 lies between the two.  18 chunks of 12 rows of
// 32/8 heads: 349 us (the second 276) over 8192 tokens, 61 (62) over 1024, 14.5 (20.8)
// from the start; 2 chunks of 64 rows over 8192 tokens 324 (171, taken), of 100 rows from
// the start 16.5 (26.7).  Furthest off: 4 prompts of 40 rows take 22.6, 15.6 by the first.
bool wide_takes(DeviceState* ds, const axkv4_cache_t* c, int chunks, int rows, int G) {
    const int64_t cols = (int64_t)rows * G, lists = (int64_t)chunks * c->n_kv_heads;
    const int64_t waves = (lists * ((cols + 255) / 256) + ds->sm_count - 1) / ds->sm_count;
    return 61 * waves * ds->sm_count < 27 * lists * ((cols + 15) / 16);
}

}  // namespace

extern "C" {

int64_t axkv4_pages_bytes(const axkv4_cache_t* c) {
    if (!c) return 0;
    return (int64_t)c->n_pages * c->n_kv_heads * 18 * c->head_dim;
}

int axkv4_append(const axkv4_cache_t* c, const float* k_rows, const float* v_rows, int64_t ld,
                 int32_t n_rows, const int32_t* row_seq, const int32_t* row_pos, void* stream) {
    int rc = check_rows(c, "axkv4_append", k_rows, v_rows, ld, n_rows, row_seq, row_pos);
    if (rc || n_rows == 0) return rc;
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    AXQ8_CUDA_TRY(KV4_BY_HEAD_DIM(c->head_dim, launch_append, c, k_rows, v_rows, ld, n_rows, row_seq,
                                  row_pos, ds->status, static_cast<cudaStream_t>(stream)),
                  "axkv4_append launch");
    return AXQ8_OK;
}

int axkv4_read(const axkv4_cache_t* c, float* k_rows, float* v_rows, int64_t ld, int32_t n_rows,
               const int32_t* row_seq, const int32_t* row_pos, void* stream) {
    int rc = check_rows(c, "axkv4_read", k_rows, v_rows, ld, n_rows, row_seq, row_pos);
    if (rc || n_rows == 0) return rc;
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    AXQ8_CUDA_TRY(KV4_BY_HEAD_DIM(c->head_dim, launch_read, c, k_rows, v_rows, ld, n_rows, row_seq,
                                  row_pos, ds->status, static_cast<cudaStream_t>(stream)),
                  "axkv4_read launch");
    return AXQ8_OK;
}

int64_t axkv4_decode_attn_workspace(const axkv4_cache_t* c, int32_t n_rows, int32_t n_heads) {
    if (check_decode(c, "axkv4_decode_attn_workspace", n_rows, n_heads) || n_rows == 0) return -1;
    DeviceState* ds = device_state();
    if (!ds) return -1;
    return narrow_plan(ds, c, n_rows, 1, n_heads / c->n_kv_heads).workspace;
}

int axkv4_decode_attn(const axkv4_cache_t* c, const float* q, int64_t ldq, int32_t n_rows,
                      int32_t n_heads, const int32_t* q_seq, const int32_t* q_pos, float* out,
                      void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_decode(c, "axkv4_decode_attn", n_rows, n_heads);
    if (rc) return rc;
    if (n_rows == 0) return AXQ8_OK;
    if (!q || !q_pos || !out || !workspace) return fail(AXQ8_ERR_INVALID, "axkv4_decode_attn: null pointer");
    if (ldq < (int64_t)n_heads * c->head_dim || ldq % 4 ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
          reinterpret_cast<uintptr_t>(workspace)) & 15))
        return fail(AXQ8_ERR_INVALID, "axkv4_decode_attn: q, out and workspace must be 16-byte aligned");
    if (!q_seq && n_rows > c->n_seqs)
        return fail(AXQ8_ERR_INVALID, "axkv4_decode_attn: %d rows of %d sequences", n_rows, c->n_seqs);
    if (workspace_bytes <= 0) return fail(AXQ8_ERR_INVALID, "axkv4_decode_attn: no workspace");
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    const NarrowPlan p = narrow_plan(ds, c, n_rows, 1, n_heads / c->n_kv_heads);
    if (workspace_bytes < p.workspace)
        return fail(AXQ8_ERR_INVALID, "axkv4_decode_attn: workspace %lld B < %lld B",
                    (long long)workspace_bytes, (long long)p.workspace);
    AXQ8_CUDA_TRY(KV4_BY_HEAD_DIM(c->head_dim, launch_narrow, ds, p, c, q, ldq, n_rows, n_rows, 1, n_heads,
                                  q_seq, nullptr, q_pos, out, workspace, static_cast<cudaStream_t>(stream)),
                  "axkv4_decode_attn launch");
    return AXQ8_OK;
}

int64_t axkv4_chunk_attn_workspace(const axkv4_cache_t* c, int32_t n_chunks, int32_t max_rows,
                                   int32_t n_heads) {
    if (check_chunks(c, "axkv4_chunk_attn_workspace", n_chunks, max_rows, n_heads) || n_chunks == 0 || max_rows == 0)
        return -1;
    DeviceState* ds = device_state();
    if (!ds) return -1;
    if (wide_takes(ds, c, n_chunks, max_rows, n_heads / c->n_kv_heads)) return 16;
    if (check_narrow(c, "axkv4_chunk_attn_workspace", n_chunks, max_rows, n_heads / c->n_kv_heads)) return -1;
    return narrow_plan(ds, c, n_chunks, max_rows, n_heads / c->n_kv_heads).workspace;
}

int axkv4_chunk_attn(const axkv4_cache_t* c, const float* q, int64_t ldq, int32_t n_rows,
                     int32_t n_chunks, int32_t max_rows, int32_t n_heads, const int32_t* q_seq,
                     const int32_t* q_start, const int32_t* q_pos, float* out, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    int rc = check_chunks(c, "axkv4_chunk_attn", n_chunks, max_rows, n_heads);
    if (rc) return rc;
    if (n_rows < 0) return fail(AXQ8_ERR_INVALID, "axkv4_chunk_attn: %d rows", n_rows);
    if (n_rows == 0 || n_chunks == 0 || max_rows == 0) return AXQ8_OK;
    if (!q || !q_start || !q_pos || !out || !workspace)
        return fail(AXQ8_ERR_INVALID, "axkv4_chunk_attn: null pointer");
    if (ldq < (int64_t)n_heads * c->head_dim || ldq % 4 ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
          reinterpret_cast<uintptr_t>(workspace)) & 15))
        return fail(AXQ8_ERR_INVALID, "axkv4_chunk_attn: q, out and workspace must be 16-byte aligned");
    if (!q_seq && n_chunks > c->n_seqs)
        return fail(AXQ8_ERR_INVALID, "axkv4_chunk_attn: %d chunks of %d sequences", n_chunks, c->n_seqs);
    if (workspace_bytes <= 0) return fail(AXQ8_ERR_INVALID, "axkv4_chunk_attn: no workspace");
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    if (wide_takes(ds, c, n_chunks, max_rows, n_heads / c->n_kv_heads)) {
        AXQ8_CUDA_TRY(KV4_BY_HEAD_DIM(c->head_dim, launch_wide, ds, c, q, ldq, n_rows, n_chunks, max_rows, n_heads,
                                      q_seq, q_start, q_pos, out,
                                      static_cast<cudaStream_t>(stream)),
                      "axkv4_chunk_attn launch");
        return AXQ8_OK;
    }
    if ((rc = check_narrow(c, "axkv4_chunk_attn", n_chunks, max_rows, n_heads / c->n_kv_heads))) return rc;
    const NarrowPlan p = narrow_plan(ds, c, n_chunks, max_rows, n_heads / c->n_kv_heads);
    if (workspace_bytes < p.workspace)
        return fail(AXQ8_ERR_INVALID, "axkv4_chunk_attn: workspace %lld B < %lld B",
                    (long long)workspace_bytes, (long long)p.workspace);
    AXQ8_CUDA_TRY(KV4_BY_HEAD_DIM(c->head_dim, launch_narrow, ds, p, c, q, ldq, n_rows, n_chunks, max_rows,
                                  n_heads, q_seq, q_start, q_pos, out, workspace,
                                  static_cast<cudaStream_t>(stream)),
                  "axkv4_chunk_attn launch");
    return AXQ8_OK;
}

}  // extern "C"
