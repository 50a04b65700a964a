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

// One warp per (row, KV head); lane l holds dim 32 b + l of every block b.
template <int HD>
__global__ void __launch_bounds__(256)
    kv4_append_kernel(Kv4Pages c, const float* __restrict__ k_rows, const float* __restrict__ v_rows,
                      int64_t ld, int n_rows, const int* __restrict__ row_seq,
                      const int* __restrict__ row_pos, int* __restrict__ status) {
    using F = Kv4<HD>;
    const int64_t gw = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (gw >= (int64_t)n_rows * c.n_kv) return;
    const int r = (int)(gw / c.n_kv), h = (int)(gw % c.n_kv);
    const int p = row_pos[r];
    uint8_t* base = kv4_at<HD>(c, row_seq[r], p, h);
    if (!base) {
        if (lane == 0) record_status(status, AXQ8_ERR_INVALID);
        return;
    }
    const int slot = p % kKv4Tokens;
    bool bad = false;
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        const float* src = (kv ? v_rows : k_rows) + (int64_t)r * ld + (int64_t)h * HD;
#pragma unroll
        for (int b = 0; b < F::NB; b++) {
            const float x = kv4_clean(src[32 * b + lane], bad);
            float lo = fminf(x, 0.0f), hi = fmaxf(x, 0.0f);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            const int code = kv4_step_code(hi - lo);
            const float d = code ? kv4_step(code) : 1.0f;   // all zero: any step does
            const float inv = 1.0f / d;
            const float z = -kv4_round(lo, d, inv);
            const uint32_t q = (uint32_t)fminf(kv4_round(x, d, inv) + z, 15.0f);
            if (lane == 0)
                *reinterpret_cast<uint16_t*>(base + (kv ? F::VS : F::KS) + F::scale(slot, b)) =
                    (uint16_t)((code << 4) | (int)z);
            if (kv == 0) {
                const uint32_t pair = q | (__shfl_down_sync(0xffffffffu, q, 1) << 4);
                if ((lane & 1) == 0) base[F::k_byte(slot, b, lane >> 1)] = (uint8_t)pair;
            } else {
                const uint32_t pair = q | (__shfl_down_sync(0xffffffffu, q, 8) << 4);
                if ((lane & 8) == 0) base[F::v_byte(slot, 2 * b + (lane >> 4), lane & 7)] = (uint8_t)pair;
            }
        }
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0) record_status(status, AXQ8_ERR_INVALID);
}

// Dim 32 b + lane of token r of a (page, KV head).
template <int HD>
__device__ __forceinline__ float kv4_value(const uint8_t* base, bool v, int r, int b, int lane) {
    using F = Kv4<HD>;
    const uint32_t w = *reinterpret_cast<const uint16_t*>(base + (v ? F::VS : F::KS) + F::scale(r, b));
    const int q = v ? (base[F::v_byte(r, 2 * b + (lane >> 4), lane & 7)] >> ((lane & 8) >> 1)) & 15
                    : (base[F::k_byte(r, b, lane >> 1)] >> (4 * (lane & 1))) & 15;
    return kv4_step(w >> 4) * (float)(q - (int)(w & 15));
}

template <int HD>
__global__ void __launch_bounds__(256)
    kv4_read_kernel(Kv4Pages c, float* __restrict__ k_rows, float* __restrict__ v_rows, int64_t ld,
                    int n_rows, const int* __restrict__ row_seq, const int* __restrict__ row_pos,
                    int* __restrict__ status) {
    const int64_t gw = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (gw >= (int64_t)n_rows * c.n_kv) return;
    const int r = (int)(gw / c.n_kv), h = (int)(gw % c.n_kv);
    const int p = row_pos[r];
    const uint8_t* base = kv4_at<HD>(c, row_seq[r], p, h);
    if (!base && lane == 0) record_status(status, AXQ8_ERR_INVALID);
#pragma unroll
    for (int b = 0; b < Kv4<HD>::NB; b++) {
        const int64_t at = (int64_t)r * ld + (int64_t)h * HD + 32 * b + lane;
        k_rows[at] = base ? kv4_value<HD>(base, false, p % kKv4Tokens, b, lane) : 0.0f;
        v_rows[at] = base ? kv4_value<HD>(base, true, p % kKv4Tokens, b, lane) : 0.0f;
    }
}

int check_cache4(const axkv4_cache_t* c, const char* what) {
    if (!c || !c->pages || !c->block_table) return fail(AXQ8_ERR_INVALID, "%s: null cache pointer", what);
    if (c->page_tokens != kKv4Tokens)
        return fail(AXQ8_ERR_UNSUPPORTED, "%s: page_tokens must be 16", what);
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128)
        return fail(AXQ8_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64, 128)", what, c->head_dim);
    if (c->n_seqs <= 0 || c->n_pages <= 0 || c->max_blocks <= 0 || c->n_kv_heads <= 0)
        return fail(AXQ8_ERR_INVALID, "%s: non-positive cache dimension", what);
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
    const int64_t warps = (int64_t)n_rows * c->n_kv_heads;
    return launch_k(kv4_append_kernel<HD>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, s, false,
                    pages_of(c), k, v, ld, n_rows, seq, pos, status);
}

template <int HD>
cudaError_t launch_read(const axkv4_cache_t* c, float* k, float* v, int64_t ld, int n_rows,
                        const int* seq, const int* pos, int* status, cudaStream_t s) {
    const int64_t warps = (int64_t)n_rows * c->n_kv_heads;
    return launch_k(kv4_read_kernel<HD>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, s, false,
                    pages_of(c), k, v, ld, n_rows, seq, pos, status);
}

// Columns of a tile, CTAs, and workspace bytes: a record per CTA, then two
// partial states per CTA.
struct NarrowPlan {
    int cols, ctas, aligned;
    int64_t records, workspace;
    int64_t units;   // of work, at most
};

NarrowPlan narrow_plan(DeviceState* ds, const axkv4_cache_t* c, int entries, int rows, int G) {
    NarrowPlan p;
    const int64_t cols = (int64_t)rows * G;
    p.cols = cols <= 4 ? 4 : cols <= 8 ? 8 : 16;
    const int slots = ds->sm_count * (p.cols == 4 ? 4 : p.cols == 8 ? 3 : 2);
    const int64_t tiles = (cols + p.cols - 1) / p.cols * c->n_kv_heads * entries;
    // every tile starts a run where that leaves half of the runs; with the most
    // tiles a call can have (it may have fewer), this many runs are never exceeded
    p.aligned = 2 * tiles <= slots ? (int)tiles : 0;
    const int64_t runs = (tiles * c->max_blocks + kNarrowMinPages - 1) / kNarrowMinPages + p.aligned;
    p.ctas = (int)std::min<int64_t>(slots, runs);
    p.units = tiles * (c->max_blocks + kNarrowTileCost) * 2;
    p.records = ((int64_t)p.ctas * sizeof(NarrowPart) + 15) / 16 * 16;
    p.workspace = p.records + (int64_t)p.ctas * 2 * p.cols * (c->head_dim + 2) * 4;
    return p;
}

template <int HD, int COLS>
cudaError_t launch_narrow_cols(DeviceState* ds, const NarrowArgs& a, int ctas, cudaStream_t s) {
    static_assert(NarrowCfg<HD, COLS>::CTAS == (COLS == 4 ? 4 : COLS == 8 ? 3 : 2), "narrow_plan");
    constexpr size_t smem = NarrowCfg<HD, COLS>::SMEM;
    auto kern = kv4_attn_narrow_kernel<HD, COLS>;
    static std::atomic<int> configured[64] = {};   // by device
    const int dev = ds->device < 64 ? ds->device : 63;
    if (smem > 48 * 1024 && (dev == 63 || !configured[dev])) {
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

// Columns (rows x heads of a KV head) of a chunk from which the tensor-core
// tiles of 128 rows take it.
constexpr int kWideCols = 33;

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
    if (check_attn(c, "axkv4_decode_attn_workspace", n_heads) || n_rows <= 0) return -1;
    DeviceState* ds = device_state();
    if (!ds) return -1;
    return narrow_plan(ds, c, n_rows, 1, n_heads / c->n_kv_heads).workspace;
}

int axkv4_decode_attn(const axkv4_cache_t* c, const float* q, int64_t ldq, int32_t n_rows,
                      int32_t n_heads, const int32_t* q_seq, const int32_t* q_pos, float* out,
                      void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_attn(c, "axkv4_decode_attn", n_heads);
    if (rc) return rc;
    if (n_rows < 0 || n_rows > 65535) return fail(AXQ8_ERR_INVALID, "axkv4_decode_attn: n_rows %d", n_rows);
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
    if (p.units > 0x7fffffff)
        return fail(AXQ8_ERR_UNSUPPORTED, "axkv4_decode_attn: %d rows of %d pages", n_rows, c->max_blocks);
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
    if (check_attn(c, "axkv4_chunk_attn_workspace", n_heads) || n_chunks <= 0 || max_rows <= 0) return -1;
    if ((int64_t)max_rows * (n_heads / c->n_kv_heads) >= kWideCols) return 16;
    DeviceState* ds = device_state();
    if (!ds) return -1;
    return narrow_plan(ds, c, n_chunks, max_rows, n_heads / c->n_kv_heads).workspace;
}

int axkv4_chunk_attn(const axkv4_cache_t* c, const float* q, int64_t ldq, int32_t n_rows,
                     int32_t n_chunks, int32_t max_rows, int32_t n_heads, const int32_t* q_seq,
                     const int32_t* q_start, const int32_t* q_pos, float* out, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    int rc = check_attn(c, "axkv4_chunk_attn", n_heads);
    if (rc) return rc;
    if (n_rows < 0 || n_chunks < 0 || max_rows < 0 || n_chunks > 65535 || max_rows > 65535)
        return fail(AXQ8_ERR_INVALID, "axkv4_chunk_attn: %d rows, %d chunks of at most %d", n_rows, n_chunks,
                    max_rows);
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
    if ((int64_t)max_rows * (n_heads / c->n_kv_heads) >= kWideCols) {
        if (c->n_kv_heads > 65535) return fail(AXQ8_ERR_UNSUPPORTED, "axkv4_chunk_attn: %d KV heads", c->n_kv_heads);
        AXQ8_CUDA_TRY(KV4_BY_HEAD_DIM(c->head_dim, launch_wide, ds, c, q, ldq, n_rows, n_chunks, max_rows, n_heads,
                                      q_seq, q_start, q_pos, out,
                                      static_cast<cudaStream_t>(stream)),
                      "axkv4_chunk_attn launch");
        return AXQ8_OK;
    }
    const NarrowPlan p = narrow_plan(ds, c, n_chunks, max_rows, n_heads / c->n_kv_heads);
    if (p.units > 0x7fffffff)
        return fail(AXQ8_ERR_UNSUPPORTED, "axkv4_chunk_attn: %d chunks of %d rows, %d pages", n_chunks,
                    max_rows, c->max_blocks);
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
