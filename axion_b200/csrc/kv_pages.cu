// Pages of a cache (include/axkv.h, axkv_pages): reserve, fork, free, compact
// and copy over the block table, the reference counts and every layer's pools.
//
// A call that allocates or compacts is two kernels.  The first, one CTA, reads
// the counts and the request and writes what is to be done (a plan) to the
// workspace; the second carries it out over the whole GPU: table rows, counts
// and the page copies.  Nothing is decided by the order of atomics.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "axkv.h"
#include "common.cuh"
#include "runtime.h"

using namespace axq8;

namespace {

constexpr int kPageTokens = 16;
constexpr int kPlanThreads = 1024;
constexpr int kScanPages = 8;     // consecutive pages of a thread in a scan over the counts
constexpr int kCopyThreads = 256;
constexpr int kCopyAhead = 4;    // 16-byte loads of a thread on their way
constexpr int kPiece = kCopyThreads * kCopyAhead * 16;   // bytes of a page that one CTA copies at a time

// Workspace: header, then claim [n_seqs], first [n + 1], src and dst [n_pages]
// each (compact: + to [n_pages]).
struct Plan {
    int* header;   // [0] page copies, [1] call is valid, [2] live pages
    int* claim;    // entry that names the sequence as its child (reserve: at all)
    int* first;    // entry i's new pages are dst[first[i]] .. dst[first[i + 1] - 1]
    int* src;
    int* dst;
    int* to;
};

__host__ __device__ inline int64_t plan_ints(int n_seqs, int n, int n_pages) {
    return 16 + (int64_t)n_seqs + (n + 1) + 3 * (int64_t)n_pages;
}

__device__ __host__ inline Plan plan_of(void* ws, int n_seqs, int n, int n_pages) {
    int* p = static_cast<int*>(ws);
    Plan a;
    a.header = p;
    a.claim = p + 16;
    a.first = a.claim + n_seqs;
    a.src = a.first + n + 1;
    a.dst = a.src + n_pages;
    a.to = a.dst + n_pages;
    return a;
}

// Exclusive prefix sum of v over the CTA, and the total.
__device__ __forceinline__ int cta_scan(int v, int* sm, int* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    __syncthreads();   // sm is free
    if (lane == 31) sm[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int w = lane < nw ? sm[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += t;
        }
        if (lane < nw) sm[lane] = w;
    }
    __syncthreads();
    *total = sm[nw - 1];
    return inc - v + (warp ? sm[warp - 1] : 0);
}

// Pages that row `row` of the table holds (its pages come first): the first
// negative entry, by bisection.
__device__ __forceinline__ int held_pages(const int* row, int max_blocks) {
    int lo = 0, hi = max_blocks;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (__ldcg(row + mid) >= 0) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// The plan of a reserve (FORK false) or a fork: the request is checked, new
// pages are counted, and the lowest free pages are dealt out in its order.
template <bool FORK>
__global__ void __launch_bounds__(kPlanThreads)
    pages_plan_kernel(axkv_pages_t p, const int* __restrict__ parents, const int* __restrict__ seqs,
                      const int* __restrict__ tokens, int n, void* ws, int* __restrict__ status) {
    __shared__ int sm[32];
    __shared__ int bad;
    const Plan a = plan_of(ws, p.n_seqs, n, p.n_pages);
    const int tid = threadIdx.x;
    pdl_launch_dependents();
    for (int i = tid; i < p.n_seqs; i += kPlanThreads) a.claim[i] = 0x7fffffff;
    if (tid == 0) bad = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPlanThreads) {
        const int s = seqs[i];
        if (s < 0 || s >= p.n_seqs) bad = 1;
        else atomicMin(a.claim + s, i);
    }
    __syncthreads();
    int total = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int need = 0;
        if (i < n) {
            const int s = seqs[i], t = tokens[i];
            bool ok = s >= 0 && s < p.n_seqs && t >= 0 && t <= p.max_blocks * kPageTokens &&
                      __ldcg(a.claim + s) == i;
            if (ok) {
                const int* row = p.block_table + (int64_t)s * p.max_blocks;
                const int blocks = (t + kPageTokens - 1) / kPageTokens;
                if (FORK) {
                    const int par = parents[i];
                    ok = __ldcg(row) < 0 && par >= 0 && par < p.n_seqs &&
                         __ldcg(a.claim + par) == 0x7fffffff &&
                         (blocks == 0 ||
                          __ldcg(p.block_table + (int64_t)par * p.max_blocks + blocks - 1) >= 0);
                    need = t % kPageTokens ? 1 : 0;
                } else {
                    need = min(max(0, blocks - held_pages(row, p.max_blocks)), p.n_pages + 1);
                }
            }
            if (!ok) {
                bad = 1;
                need = 0;
            }
        }
        int sum;
        const int at = cta_scan(need, sm, &sum);
        // the page that a fork copies in part; none for a child without one
        if (FORK && i < n && need && total + at < p.n_pages)
            a.src[total + at] = __ldcg(p.block_table + (int64_t)parents[i] * p.max_blocks + tokens[i] / kPageTokens);
        if (i < n) a.first[i] = (int)min((int64_t)total + at, (int64_t)p.n_pages + 1);
        total = (int)min((int64_t)total + sum, (int64_t)p.n_pages + 1);
    }
    if (tid == 0) a.first[n] = total;
    // the lowest `total` free pages
    int found = 0;
    for (int g0 = 0; g0 < p.n_pages && found < total; g0 += kPlanThreads * kScanPages) {
        const int g = g0 + tid * kScanPages;
        unsigned free = 0;
#pragma unroll
        for (int k = 0; k < kScanPages; k++)
            if (g + k < p.n_pages && __ldcg(p.ref_count + g + k) == 0) free |= 1u << k;
        int sum;
        int at = found + cta_scan(__popc(free), sm, &sum);
        for (; free && at < total; free &= free - 1) a.dst[at++] = g + __ffs(free) - 1;
        found += sum;
    }
    __syncthreads();
    if (tid == 0) {
        const int code = bad ? AXQ8_ERR_INVALID : found < total ? AXQ8_ERR_ALLOC : AXQ8_OK;
        if (code) record_status(status, code);
        a.header[0] = code ? 0 : total;
        a.header[1] = code == AXQ8_OK;
    }
}

// Pages src[i] to dst[i] in every pool, i < n, over the whole grid in pieces.  Bound:
// HBM, twice the pages' bytes; the next piece's page numbers are read while a
// piece is copied.  984 MB in 153 us of a compaction's 174 (0.98 of the copy
// bandwidth).  Pairs outside the pool are left out; reported, if status is.
__device__ __forceinline__ void copy_pages(const axkv_pages_t& p, const int* src, const int* dst, int n,
                                           int* status) {
    if (p.n_pools == 0) return;
    const int pieces = (int)((p.page_bytes + kPiece - 1) / kPiece);
    const int64_t items = (int64_t)n * p.n_pools * pieces;
    int64_t it = blockIdx.x;
    if (it >= items) return;
    int i = (int)(it / pieces / p.n_pools), s = __ldcg(src + i), d = __ldcg(dst + i);
    for (;;) {
        const int piece = (int)(it % pieces), pool = (int)(it / pieces % p.n_pools);
        const int64_t next = it + gridDim.x;
        const int i2 = next < items ? (int)(next / pieces / p.n_pools) : i;
        const int s2 = __ldcg(src + i2), d2 = __ldcg(dst + i2);
        if ((unsigned)s < (unsigned)p.n_pages && (unsigned)d < (unsigned)p.n_pages) {
            const int64_t at = (int64_t)piece * kPiece;
            uint8_t* base = static_cast<uint8_t*>(p.pools[pool]);
            const uint4* from = reinterpret_cast<const uint4*>(base + (int64_t)s * p.page_bytes + at);
            uint4* to = reinterpret_cast<uint4*>(base + (int64_t)d * p.page_bytes + at);
            const int words = (int)min((int64_t)kPiece, p.page_bytes - at) / 16;
            uint4 v[kCopyAhead];
#pragma unroll
            for (int k = 0; k < kCopyAhead; k++)
                if (threadIdx.x + k * kCopyThreads < words) v[k] = __ldcg(from + threadIdx.x + k * kCopyThreads);
#pragma unroll
            for (int k = 0; k < kCopyAhead; k++)
                if (threadIdx.x + k * kCopyThreads < words) to[threadIdx.x + k * kCopyThreads] = v[k];
        } else if (status && threadIdx.x == 0) {
            record_status(status, AXQ8_ERR_INVALID);
        }
        if (next >= items) return;
        it = next;
        s = s2;
        d = d2;
    }
}

// Reserve: the new pages into the rows.  Fork: the children's rows, the counts
// of the shared pages, and the copies of the partly filled ones.
template <bool FORK>
__global__ void __launch_bounds__(kCopyThreads)
    pages_apply_kernel(axkv_pages_t p, const int* __restrict__ parents, const int* __restrict__ seqs,
                       const int* __restrict__ tokens, int n, void* ws) {
    const Plan a = plan_of(ws, p.n_seqs, n, p.n_pages);
    pdl_wait();
    if (!__ldcg(a.header + 1)) return;
    const int step = gridDim.x * (blockDim.x >> 5);
    const int lane = threadIdx.x & 31;
    for (int i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < n; i += step) {
        int* row = p.block_table + (int64_t)seqs[i] * p.max_blocks;
        const int f0 = __ldcg(a.first + i), f1 = __ldcg(a.first + i + 1);
        if (FORK) {
            const int* par = p.block_table + (int64_t)parents[i] * p.max_blocks;
            const int full = tokens[i] / kPageTokens;
            for (int j = lane; j < full; j += 32) {
                const int page = __ldcg(par + j);
                row[j] = page;
                if (page >= 0 && page < p.n_pages) atomicAdd(p.ref_count + page, 1);
            }
            if (lane == 0 && f1 > f0) {
                const int page = __ldcg(a.dst + f0);
                row[full] = page;
                p.ref_count[page] = 1;
            }
        } else {
            const int held = (tokens[i] + kPageTokens - 1) / kPageTokens - (f1 - f0);
            for (int j = lane; j < f1 - f0; j += 32) {
                const int page = __ldcg(a.dst + f0 + j);
                row[held + j] = page;
                p.ref_count[page] = 1;
            }
        }
    }
    if (FORK) copy_pages(p, a.src, a.dst, __ldcg(a.header), nullptr);
}

__global__ void __launch_bounds__(kCopyThreads)
    pages_free_kernel(axkv_pages_t p, const int* __restrict__ seqs, int n, int* __restrict__ status) {
    const int lane = threadIdx.x & 31;
    const int step = gridDim.x * (blockDim.x >> 5);
    for (int i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < n; i += step) {
        const int s = seqs[i];
        if (s < 0 || s >= p.n_seqs) {
            if (lane == 0) record_status(status, AXQ8_ERR_INVALID);
            continue;
        }
        int* row = p.block_table + (int64_t)s * p.max_blocks;
        for (int j0 = lane; j0 < p.max_blocks; j0 += 128) {   // four entries on their way
            int page[4];
#pragma unroll
            for (int k = 0; k < 4; k++) page[k] = j0 + 32 * k < p.max_blocks ? atomicExch(row + j0 + 32 * k, -1) : -1;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (page[k] >= 0 && page[k] < p.n_pages) atomicSub(p.ref_count + page[k], 1);
        }
    }
}

// The moves of a compaction: live pages from n_live on, free ones below it,
// each in ascending order, paired.
__global__ void __launch_bounds__(kPlanThreads)
    pages_moves_kernel(axkv_pages_t p, int* __restrict__ n_live, void* ws) {
    __shared__ int sm[32];
    const Plan a = plan_of(ws, p.n_seqs, 0, p.n_pages);
    const int tid = threadIdx.x;
    pdl_launch_dependents();
    int mine = 0, live;
#pragma unroll 8
    for (int g = tid; g < p.n_pages; g += kPlanThreads) {
        mine += __ldcg(p.ref_count + g) > 0;
        a.to[g] = g;
    }
    cta_scan(mine, sm, &live);
    int ns = 0, nd = 0;
    for (int g0 = 0; g0 < p.n_pages; g0 += kPlanThreads * kScanPages) {
        const int g = g0 + tid * kScanPages;
        unsigned src = 0, dst = 0;
#pragma unroll
        for (int k = 0; k < kScanPages; k++) {
            if (g + k >= p.n_pages) continue;
            const bool used = __ldcg(p.ref_count + g + k) > 0;
            if (used && g + k >= live) src |= 1u << k;
            if (!used && g + k < live) dst |= 1u << k;
        }
        int sum;
        const int at = cta_scan(__popc(src) | (__popc(dst) << 16), sm, &sum);   // at most 8192 of each
        int i = ns + (at & 0xffff), j = nd + (at >> 16);
        for (; src; src &= src - 1) a.src[i++] = g + __ffs(src) - 1;
        for (; dst; dst &= dst - 1) a.dst[j++] = g + __ffs(dst) - 1;
        ns += sum & 0xffff;
        nd += sum >> 16;
    }
    __syncthreads();
    for (int k = tid; k < ns; k += kPlanThreads) {
        const int s = __ldcg(a.src + k), d = __ldcg(a.dst + k);
        a.to[s] = d;
        p.ref_count[d] = __ldcg(p.ref_count + s);
        p.ref_count[s] = 0;
    }
    if (tid == 0) {
        a.header[0] = ns;
        a.header[2] = live;
        *n_live = live;
    }
}

__global__ void __launch_bounds__(kCopyThreads) pages_move_kernel(axkv_pages_t p, void* ws) {
    const Plan a = plan_of(ws, p.n_seqs, 0, p.n_pages);
    pdl_wait();
    const int ns = __ldcg(a.header), live = __ldcg(a.header + 2);
    const int64_t entries = (int64_t)p.n_seqs * p.max_blocks;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < entries;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int page = p.block_table[i];
        if (page >= live && page < p.n_pages) p.block_table[i] = __ldcg(a.to + page);
    }
    copy_pages(p, a.src, a.dst, ns, nullptr);
}

__global__ void __launch_bounds__(kCopyThreads)
    pages_copy_kernel(axkv_pages_t p, const int* __restrict__ src, const int* __restrict__ dst, int n,
                      int* __restrict__ status) {
    copy_pages(p, src, dst, n, status);
}

int check_pages(const axkv_pages_t* p, const char* what) {
    if (!p || !p->block_table || !p->ref_count || (p->n_pools > 0 && !p->pools))
        return fail(AXQ8_ERR_INVALID, "%s: null pointer", what);
    if (p->n_pools < 0 || p->n_seqs <= 0 || p->max_blocks <= 0 || p->n_pages <= 0)
        return fail(AXQ8_ERR_INVALID, "%s: non-positive dimension", what);
    // 1024 requests of n_pages + 1 pages still sum in 32 bits
    if (p->max_blocks > (1 << 26) || p->n_pages > 2000000)
        return fail(AXQ8_ERR_UNSUPPORTED, "%s: %d blocks, %d pages", what, p->max_blocks, p->n_pages);
    if (p->n_pools > 0 && (p->page_bytes <= 0 || p->page_bytes % 16))
        return fail(AXQ8_ERR_INVALID, "%s: page_bytes %lld is not a multiple of 16", what,
                    (long long)p->page_bytes);
    return AXQ8_OK;
}

int check_workspace(const axkv_pages_t* p, int32_t n, const void* ws, int64_t bytes, const char* what) {
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15))
        return fail(AXQ8_ERR_INVALID, "%s: workspace null or not 16-byte aligned", what);
    const int64_t need = axkv_pages_workspace(p, n);
    if (bytes < need)
        return fail(AXQ8_ERR_INVALID, "%s: workspace %lld B < %lld B", what, (long long)bytes,
                    (long long)need);
    return AXQ8_OK;
}

// CTAs of a kernel that walks `items` copy pieces (or as many as the GPU holds).
unsigned copy_ctas(DeviceState* ds, int64_t items) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(items, 8ll * ds->sm_count));
}
int64_t pieces_of(const axkv_pages_t* p) { return p->n_pools ? (p->page_bytes + kPiece - 1) / kPiece : 0; }

template <bool FORK>
int allocate(const axkv_pages_t* p, const char* what, const int32_t* parents, const int32_t* seqs,
             const int32_t* tokens, int32_t n, void* ws, int64_t ws_bytes, void* stream) {
    int rc = check_pages(p, what);
    if (rc) return rc;
    if (n < 0) return fail(AXQ8_ERR_INVALID, "%s: n < 0", what);
    if (n == 0) return AXQ8_OK;
    if (!seqs || !tokens || (FORK && !parents)) return fail(AXQ8_ERR_INVALID, "%s: null pointer", what);
    if ((rc = check_workspace(p, n, ws, ws_bytes, what))) return rc;
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    AXQ8_CUDA_TRY(launch_k(pages_plan_kernel<FORK>, dim3(1), dim3(kPlanThreads), 0, s, false, *p, parents,
                           seqs, tokens, (int)n, ws, ds->status),
                  "axkv_pages plan launch");
    const int64_t items = FORK ? (int64_t)n * p->n_pools * pieces_of(p) : 0;
    AXQ8_CUDA_TRY(launch_k(pages_apply_kernel<FORK>, dim3(copy_ctas(ds, std::max<int64_t>(items, (n + 7) / 8))),
                           dim3(kCopyThreads), 0, s, true, *p, parents, seqs, tokens, (int)n, ws),
                  "axkv_pages apply launch");
    return AXQ8_OK;
}

}  // namespace

extern "C" {

int64_t axkv_pages_workspace(const axkv_pages_t* p, int32_t n) {
    if (check_pages(p, "axkv_pages_workspace") || n < 0) return -1;
    return plan_ints(p->n_seqs, n, p->n_pages) * 4;
}

int axkv_pages_reserve(const axkv_pages_t* p, const int32_t* seqs, const int32_t* tokens, int32_t n,
                       void* workspace, int64_t workspace_bytes, void* stream) {
    return allocate<false>(p, "axkv_pages_reserve", nullptr, seqs, tokens, n, workspace, workspace_bytes,
                           stream);
}

int axkv_pages_fork(const axkv_pages_t* p, const int32_t* parents, const int32_t* children,
                    const int32_t* tokens, int32_t n, void* workspace, int64_t workspace_bytes,
                    void* stream) {
    return allocate<true>(p, "axkv_pages_fork", parents, children, tokens, n, workspace, workspace_bytes,
                          stream);
}

int axkv_pages_free(const axkv_pages_t* p, const int32_t* seqs, int32_t n, void* stream) {
    int rc = check_pages(p, "axkv_pages_free");
    if (rc) return rc;
    if (n < 0) return fail(AXQ8_ERR_INVALID, "axkv_pages_free: n < 0");
    if (n == 0) return AXQ8_OK;
    if (!seqs) return fail(AXQ8_ERR_INVALID, "axkv_pages_free: null pointer");
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    AXQ8_CUDA_TRY(launch_k(pages_free_kernel, dim3(copy_ctas(ds, (n + 7) / 8)), dim3(kCopyThreads), 0,
                           static_cast<cudaStream_t>(stream), false, *p, seqs, (int)n, ds->status),
                  "axkv_pages_free launch");
    return AXQ8_OK;
}

int axkv_pages_compact(const axkv_pages_t* p, int32_t* n_live, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    int rc = check_pages(p, "axkv_pages_compact");
    if (rc) return rc;
    if (!n_live) return fail(AXQ8_ERR_INVALID, "axkv_pages_compact: null pointer");
    if ((rc = check_workspace(p, 0, workspace, workspace_bytes, "axkv_pages_compact"))) return rc;
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    AXQ8_CUDA_TRY(launch_k(pages_moves_kernel, dim3(1), dim3(kPlanThreads), 0, s, false, *p, n_live, workspace),
                  "axkv_pages_compact plan launch");
    const int64_t items = std::max<int64_t>((int64_t)p->n_pages * p->n_pools * pieces_of(p) / 2,
                                            ((int64_t)p->n_seqs * p->max_blocks + 255) / 256);
    AXQ8_CUDA_TRY(launch_k(pages_move_kernel, dim3(copy_ctas(ds, items)), dim3(kCopyThreads), 0, s, true, *p,
                           workspace),
                  "axkv_pages_compact launch");
    return AXQ8_OK;
}

int axkv_pages_copy(const axkv_pages_t* p, const int32_t* src, const int32_t* dst, int32_t n,
                    void* stream) {
    int rc = check_pages(p, "axkv_pages_copy");
    if (rc) return rc;
    if (n < 0) return fail(AXQ8_ERR_INVALID, "axkv_pages_copy: n < 0");
    if (n == 0 || p->n_pools == 0) return AXQ8_OK;
    if (!src || !dst) return fail(AXQ8_ERR_INVALID, "axkv_pages_copy: null pointer");
    DeviceState* ds = device_state();
    if (!ds) return AXQ8_ERR_CUDA;
    AXQ8_CUDA_TRY(launch_k(pages_copy_kernel, dim3(copy_ctas(ds, (int64_t)n * p->n_pools * pieces_of(p))),
                           dim3(kCopyThreads), 0, static_cast<cudaStream_t>(stream), false, *p, src, dst, (int)n,
                           ds->status),
                  "axkv_pages_copy launch");
    return AXQ8_OK;
}

}  // extern "C"
