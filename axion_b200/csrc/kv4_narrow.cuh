// Attention of few columns over the 4-bit cache: decode steps and short chunks.
//
// The (row, head) pairs that read one KV head of one sequence are columns; a
// page's 16 tokens are the rows of m16n8k16 products:
//   S^T [16 tokens x 8] = K Q^T,  O^T [HD x 8] += V^T P^T.
// The cache words are laid out as the products' A operands, so a code goes
// from shared memory to the tensor core through registers only:
//   K: a nibble in place is the fp16 subnormal q 2^-24 (low nibbles) or q 2^-20
//      (high ones), which the product takes as it is; Q is divided by 16 in the
//      high nibbles' k-steps.  A block's 32 dims are two k-steps, and
//      s = sum_b d_b (acc_b - z_b sum_b(q)) puts step and zero point in after
//      the integer product, in fp32.
//   V: a nibble in place times D plus Z is (q - z) d 2^(e - 24) in one fused
//      multiply-add, with D = d 2^e (high nibbles: d 2^(e - 4)) and Z = -z d
//      2^(e - 24): exact while D is 2^6 to 2^16.  e is kept from step to step and
//      moves when a step's d leave that window.  Where they are too far apart for one
//      (a factor of 2^9: tokens or blocks of dims of very different size, or a draft
//      row's token that the others do not see), the smaller ones' (q - z) d are formed by
//      a subtraction and a product, exact for every d, in a pass of their own.  O is the
//      plain sum.  (With one e for all tokens so far, small d lost bits.)
// Q (scaled by a power of two to below 2^11) is a whole number plus an fp16 residual:
// whole numbers times codes sum without loss, so only the residual's products are cut
// (with an fp16 high part instead, 257 tokens were 1.8e-6 off and 64 x 2176 9e-7; now
// 5.5e-7 and 2.7e-7, and sums in fp32 5.8e-7 and 1.0e-6).  P (2^7 times the softmax
// weight) is an fp16 high part plus an fp16 residual.  Up to four columns, the two parts
// are two columns of one product (no padding, half the products); beyond, two products
// into one accumulator.  Softmax in base 2 with a running reference; it moves (and O is
// rescaled) only when a score exceeds it by more than 8, so that weights stay within fp16.
//
// The pages of all tiles (entry, column tile, KV head) in a row are dealt out in
// equal runs to as many CTAs as the GPU holds at once, whatever the sequences'
// lengths; a CTA walks the parts of tiles that its run covers.  Where there are at
// least twice as many CTAs as tiles, a tile's length is rounded up to whole runs, so
// that every tile starts one and a CTA has one part.  Its
// kNarrowWarps warps take a part's pages in turn, two at a time where registers
// allow (one softmax step and twice the independent products).  Each has its
// own ring of page buffers, filled by bulk copies (a page's 18 HD bytes of one
// KV head are contiguous); the next part's first copies are under way while a
// part is written.  The warps' states merge in shared memory, the parts of a
// tile through the workspace in a second kernel, in page order.
//
// Bound: issue slots.  64 sequences of 2176 tokens (32 query, 8 KV heads of 128):
// 55 us, 162 MB, 0.46 of the measured copy bandwidth, about 414 instructions a
// page at 0.59 of the slots; one sequence of 131072 tokens: 50 us.  Three CTAs an
// SM measured 51 us there, four (fewer registers) 54; one page a step 56 against
// 55 us at batch 64.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"
#include "decode_ops.cuh"
#include "kv4.cuh"

namespace axq8 {

constexpr int kNarrowWarps = 4;
constexpr int kNarrowPages = 4;       // page buffers of a warp
constexpr int kNarrowMinPages = 24;   // pages of a run at least, where every tile starts one
constexpr int kNarrowMinUnits = 14;   // units of a run at least elsewhere
constexpr int kNarrowMaxParts = 96;   // a run is at least that share of the longest tile: 97 parts at most
constexpr int kJoinThreads = 256;
constexpr int kNarrowTileCost = 16;   // what a tile costs beside its pages, in pages
// Pages of a part at most.  Weights and values that are alike round the same way at every
// addition, so a CTA takes longer stretches of a tile in pieces and joins their states:
// 64 sequences of 131072 equal tokens were 3.9e-5 off in one piece, 7.4e-6 now.  (Pieces
// within a part, kept in shared memory by a rare branch of the loop, cost 3 % at any length.)
constexpr int kNarrowPiece = 1024;
constexpr int kNarrowKept = 128;      // entries kept in shared memory (else read again)

struct Kv4Pages {
    uint8_t* pages;
    const int* table;
    int n_seqs, max_blocks, n_pages, n_kv;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// fp16 pair of (x, y) and of what it leaves.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = pack_f16(x, y);
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = pack_f16(x - h.x, y - h.y);
}
__device__ __forceinline__ float2 f16_pair(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t hsub2u(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2u(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfma2u(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Bounded wait for a copy: the hardware suspends the warp for up to 20 us at a
// time, a second in all.
__device__ __forceinline__ bool copy_wait(uint64_t* bar, uint32_t parity) {
    for (int i = 0; i < 50000; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(20000)
            : "memory");
        if (ok) return true;
    }
    return false;
}

// c = a b, the first product of a sum.
__device__ __forceinline__ void mma_f16_16816_first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// 2^k as fp16 in both halves, -14 <= k <= 15.
__device__ __forceinline__ uint32_t f16_pow2(int k) { return (uint32_t)(k + 15) * 0x04000400u; }

// N 32-bit words from shared memory, as wide as N allows (aligned to 4 N bytes, 16 at most).
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], const uint8_t* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(p + 4 * i);
    } else if constexpr (N == 2) {
        *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// The NB scales of token r: 16-bit words, in pairs.
template <int NB>
struct Scales {
    static constexpr int W = NB > 1 ? NB / 2 : 1;
    uint32_t w[W];
    __device__ __forceinline__ void load(const uint8_t* p, int r) {
        if constexpr (NB == 1) w[0] = *reinterpret_cast<const uint16_t*>(p + 2 * r);
        else lds_words<W>(w, p + 2 * NB * r);
    }
    __device__ __forceinline__ uint32_t word(int b) const {   // scale b in the low half (NB 1, even b)
        return w[b / 2];
    }
};

struct NarrowArgs {
    Kv4Pages c;
    const float* q;
    int64_t ldq;
    int n_rows, n_entries, max_rows, n_heads, G;
    int aligned;          // every tile starts a run
    const int* q_seq;
    const int* q_start;   // null: one row per entry
    const int* q_pos;
    float scale;          // softmax scale times log2(e)
    float* out;
    struct NarrowPart* split;   // [CTA]: the tile whose first part is this CTA's, if it has more
    float* part;          // [CTA][2][COLS][HD], then [CTA][2][COLS][2]
    int* status;
};

// Entry i of the request: its rows, sequence, and the pages of its tiles.
struct NarrowEntry {
    int r0, T, seq, pos0, ctx, nblk, segs;   // segs: tiles of nblk pages each
};
__device__ __forceinline__ NarrowEntry narrow_entry(const NarrowArgs& a, int i, int cols, bool report) {
    NarrowEntry e;
    const int room = a.c.max_blocks * kKv4Tokens;
    e.r0 = i;
    e.T = 1;
    bool ok = true;
    if (a.q_start) {
        e.r0 = a.q_start[i];
        e.T = a.q_start[i + 1] - e.r0;
        ok = e.T <= 0 || (e.r0 >= 0 && e.r0 <= a.n_rows - e.T && e.T <= a.max_rows);
        if (!ok) e.T = 0;
    }
    e.seq = a.q_seq ? a.q_seq[i] : i;
    e.pos0 = min(a.q_pos[i], room);
    const bool seq_ok = e.seq >= 0 && e.seq < a.c.n_seqs;
    if (report && (!ok || (e.T > 0 && (!seq_ok || e.pos0 + e.T > room))))
        record_status(a.status, AXQ8_ERR_INVALID);
    e.ctx = seq_ok ? max(0, min(e.pos0 + e.T, room)) : 0;
    if (!seq_ok) e.seq = 0;
    // no token at all: one page that nothing sees, so that the zeros are written
    e.nblk = max(1, (e.ctx + kKv4Tokens - 1) / kKv4Tokens);
    e.segs = e.T > 0 ? (e.T * a.G + cols - 1) / cols * a.c.n_kv : 0;
    return e;
}

// A part of a tile: what a CTA works on at a time.
struct NarrowPart {
    int r0, cols, seq, pos0, ctx;   // the entry's first row, columns, sequence, first position, tokens
    int kvh, col0;                  // the tile
    int b0, b1;                     // pages of the part
    int follows, ends;              // the CTA had the pages before in a part of its own; has none behind
    int c0, c1;                     // CTAs with parts of the tile; b0 == b1: no part
};

// A CTA's run: units [p, end) of all tiles' units in a row.  A tile's units are
// `before` of no page (what a tile costs beside its pages), its pages, and in
// the aligned case more of no page up to a multiple of the run.
struct NarrowRun {
    int p, end, run, before;
    int entry, first;   // the entry at p, and its first unit
    __device__ __forceinline__ int units(const NarrowArgs& a, int nblk) const {
        return a.aligned ? (nblk + run - 1) / run * run : nblk + before;
    }
};

// The part at r.p, and r.p past it (one thread); d.b0 == d.b1: none is left.
template <int COLS>
__device__ __noinline__ void narrow_next_part(const NarrowArgs& a, const NarrowEntry* kept, NarrowRun& r,
                                              NarrowPart& d) {
    int p = r.p, first = r.first, i = r.entry;
    d.b0 = d.b1 = 0;
    while (p < r.end) {
        const NarrowEntry e = kept ? kept[i] : narrow_entry(a, i, COLS, false);
        const int units = r.units(a, e.nblk);
        if (p >= first + units * e.segs) {
            first += units * e.segs;
            i++;
            continue;
        }
        const int seg = (p - first) / units;
        const int tile = first + seg * units + r.before;   // its first page
        const int stop = min(r.end, first + (seg + 1) * units), last = min(stop, tile + e.nblk);
        if (last > max(tile, p)) {
            d.r0 = e.r0;
            d.cols = e.T * a.G;
            d.seq = e.seq;
            d.pos0 = e.pos0;
            d.ctx = e.ctx;
            d.kvh = seg % a.c.n_kv;
            d.col0 = seg / a.c.n_kv * COLS;
            d.b0 = max(0, p - tile);
            d.b1 = min(last - tile, d.b0 + kNarrowPiece);
            d.follows = d.b0 > 0 && p > (int)blockIdx.x * r.run;
            d.ends = d.b1 == last - tile;
            d.c0 = tile / r.run;
            d.c1 = (tile + e.nblk - 1) / r.run;
            p = d.ends ? stop : tile + d.b1;
            break;
        }
        p = stop;
    }
    r.p = p;
    r.first = first;
    r.entry = i;
}

__device__ __forceinline__ void narrow_write(const NarrowArgs& a, const NarrowPart& d, int HD, int col, int dim,
                                             float4 v, float sum) {
    const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;   // nothing seen: zeros
    const int c = d.col0 + col, j = c / a.G;
    *reinterpret_cast<float4*>(a.out + (int64_t)(d.r0 + j) * a.n_heads * HD +
                               (int64_t)(d.kvh * a.G + c - j * a.G) * HD + dim) =
        make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
}

// COLS columns of a tile: 4 (both parts of Q and P in one n-tile), 8 or 16.
template <int HD, int COLS_>
struct NarrowCfg {
    static constexpr int COLS = COLS_;
    static constexpr bool PACK = COLS == 4;
    static constexpr int NT = COLS <= 8 ? 1 : 2;        // n-tiles of 8
    static constexpr int PP = COLS <= 8 ? 2 : 1;        // pages of a step
    static constexpr int NBUF = kNarrowPages / PP;      // steps in flight
    static constexpr int PITCH = HD + 4;                // merge rows, conflict-free
    static constexpr size_t RING = (size_t)kNarrowWarps * kNarrowPages * Kv4<HD>::BYTES;
    static constexpr size_t MERGE = RING;               // the warps' states
    static constexpr size_t VSC = MERGE + (size_t)kNarrowWarps * COLS * (PITCH + 2) * 4;   // V factors
    static constexpr size_t VSC_PAGE = 4 * 2 * Kv4<HD>::NB * 8;  // [t][block][u] {D, Z}
    static constexpr size_t QBUF = VSC + kNarrowWarps * PP * VSC_PAGE;   // Q of this and the next part
    static constexpr size_t KEPT = QBUF + 2 * COLS * HD * 4;
    static constexpr size_t BAR = KEPT + kNarrowKept * sizeof(NarrowEntry);
    static constexpr size_t PIECE = BAR + kNarrowWarps * NBUF * 8;   // of the pieces so far, in turn
    static constexpr size_t PARTS = PIECE + 2 * COLS * 8;
    static constexpr size_t SMEM = PARTS + 3 * sizeof(NarrowPart);
    static constexpr int JOIN_ITEMS = COLS * HD / 4 < 64 ? COLS * HD / 4 : 64;   // 4 dims of a column each
    static constexpr int CTAS = COLS <= 8 ? 3 : 2;   // resident per SM
    // d below a step's window in a pass after the others', so that no branch stands before
    // the products (64 x 2176 tokens of 32/4 heads of 64: 27.2 us, else 28.7); where 168
    // registers do not hold that, all of the step's d instead (64/8 heads of 128: 39.3, else 40.7)
    static constexpr bool AFTER = !(HD == 128 && COLS == 8);
};

// The parts of the tile that begins in run blockIdx.x, joined in page order by one CTA
// for every JOIN_ITEMS groups of 4 dims: the
// second slot of CTA c0, then the first slots of c0 + 1 .. c1.  Groups of threads
// take every S-th part of a column's 4 dims each; group states join the same way.
template <int HD, int COLS>
__global__ void __launch_bounds__(kJoinThreads) kv4_attn_join_kernel(const __grid_constant__ NarrowArgs a) {
    constexpr int PER = NarrowCfg<HD, COLS>::JOIN_ITEMS, S = kJoinThreads / PER;
    __shared__ float4 acc_s[S][PER];
    __shared__ float2 ml_s[S][PER];
    pdl_wait();
    const NarrowPart& d = a.split[blockIdx.x];
    const int c0 = d.c0, c1 = d.c1;
    if (c1 <= c0) return;
    const float* pml = a.part + (int64_t)gridDim.x * 2 * COLS * HD;
    const int live = min(COLS, d.cols - d.col0), group = threadIdx.x / PER, item = threadIdx.x % PER;
    const int idx = blockIdx.y * PER + item, col = idx / (HD / 4), dim = idx % (HD / 4) * 4;
    if (blockIdx.y * PER >= live * (HD / 4)) return;
    float mx = -CUDART_INF_F, sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float2 ml, float4 x) {
        if (ml.x == -CUDART_INF_F && ml.y == 0.0f) return;   // saw nothing (a NaN query: sum NaN, which stays)
        const float m = fmaxf(mx, ml.x), f = ex2(mx - m), h = ex2(ml.x - m);
        mx = m;
        v.x = fmaf(v.x, f, x.x * h);
        v.y = fmaf(v.y, f, x.y * h);
        v.z = fmaf(v.z, f, x.z * h);
        v.w = fmaf(v.w, f, x.w * h);
        sum = fmaf(sum, f, ml.y * h);
    };
    for (int k0 = c0 + group; k0 <= c1; k0 += 8 * S) {
        float2 ml[8];
        float4 x[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int k = k0 + u * S;
            ml[u] = make_float2(-CUDART_INF_F, 0.0f);
            if (k <= c1) {
                const int64_t at = ((int64_t)k * 2 + (k == c0)) * COLS + col;
                ml[u] = ld_cg2(pml + at * 2);
                x[u] = ld_cg4(a.part + at * HD + dim);
            }
        }
#pragma unroll
        for (int u = 0; u < 8; u++) add(ml[u], x[u]);
    }
    acc_s[group][item] = v;
    ml_s[group][item] = make_float2(mx, sum);
    __syncthreads();
    if (group == 0 && idx < live * (HD / 4)) {
#pragma unroll
        for (int k = 1; k < S; k++) add(ml_s[k][item], acc_s[k][item]);
        narrow_write(a, d, HD, col, dim, v, sum);
    }
}

// The warps' states of a part, joined: out, or to the workspace where the tile has more.
// A piece of a longer stretch joins those before it, whose sum rests in the same place (a
// thread reads what itself wrote) and whose references and sums take turns in shared
// memory.
template <int HD, int COLS>
__device__ __forceinline__ void narrow_merge(const NarrowArgs& a, int which, int turn) {
    using C = NarrowCfg<HD, COLS>;
    constexpr int W = kNarrowWarps;
    extern __shared__ __align__(16) uint8_t nar_sm[];
    const NarrowPart part = reinterpret_cast<const NarrowPart*>(nar_sm + C::PARTS)[which];
    const float* acc_s = reinterpret_cast<const float*>(nar_sm + C::MERGE);
    const float* ml_s = acc_s + (size_t)W * COLS * C::PITCH;
    const float2* had = reinterpret_cast<const float2*>(nar_sm + C::PIECE) + turn * COLS;
    float2* has = reinterpret_cast<float2*>(nar_sm + C::PIECE) + (turn ^ 1) * COLS;
    const int c0 = part.c0, c1 = part.c1, live = min(COLS, part.cols - part.col0);
    const int64_t slot = (int64_t)blockIdx.x * 2 + (c0 == (int)blockIdx.x);
    const bool out = c1 == c0 && part.ends;
    for (int idx = threadIdx.x; idx < live * (HD / 4); idx += W * 32) {
        const int col = idx / (HD / 4), d = idx % (HD / 4) * 4;
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < W; w++) mx = fmaxf(mx, ml_s[(w * COLS + col) * 2]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float mw = ml_s[(w * COLS + col) * 2];
            const float f = mw == -CUDART_INF_F ? 0.0f : ex2(mw - mx);
            const float4 x = *reinterpret_cast<const float4*>(acc_s + ((size_t)w * COLS + col) * C::PITCH + d);
            v.x = fmaf(x.x, f, v.x);
            v.y = fmaf(x.y, f, v.y);
            v.z = fmaf(x.z, f, v.z);
            v.w = fmaf(x.w, f, v.w);
            sum = fmaf(ml_s[(w * COLS + col) * 2 + 1], f, sum);
        }
        float* at = a.part + (slot * COLS + col) * HD + d;
        if (part.follows) {
            const float2 ml = had[col];
            if (ml.x != -CUDART_INF_F || ml.y != 0.0f) {   // else they saw nothing
                const float4 was = *reinterpret_cast<const float4*>(at);
                const float m = fmaxf(mx, ml.x), f = ex2(mx - m), h = ex2(ml.x - m);
                v = make_float4(fmaf(v.x, f, was.x * h), fmaf(v.y, f, was.y * h), fmaf(v.z, f, was.z * h),
                                fmaf(v.w, f, was.w * h));
                sum = fmaf(sum, f, ml.y * h);
                mx = m;
            }
        }
        if (!out) {
            *reinterpret_cast<float4*>(at) = v;
            if (d == 0) {
                has[col] = make_float2(mx, sum);
                *reinterpret_cast<float2*>(a.part + (int64_t)gridDim.x * 2 * COLS * HD + (slot * COLS + col) * 2) =
                    make_float2(mx, sum);
            }
        } else {
            narrow_write(a, part, HD, col, d, v, sum);
        }
    }
    if (c1 > c0 && c0 == (int)blockIdx.x && threadIdx.x == 0) a.split[blockIdx.x] = part;
}

// A function of its own leaves the page loop of 4 columns its registers: 131072 tokens
// 51.0 us inlined, 50.5 called.  With 8 and 16 columns it is the other way: 32 x 2176 tokens
// of 64/8 heads 39.2 and 39.8 us, 24 x 5 draft rows 35.9 and 36.9.
template <int HD, int COLS>
__device__ __noinline__ void narrow_merge_call(const NarrowArgs& a, int which, int turn) {
    narrow_merge<HD, COLS>(a, which, turn);
}

template <int HD, int COLS>
__global__ void __launch_bounds__(kNarrowWarps * 32, NarrowCfg<HD, COLS>::CTAS)
    kv4_attn_narrow_kernel(const __grid_constant__ NarrowArgs a) {
    using F = Kv4<HD>;
    using C = NarrowCfg<HD, COLS>;
    constexpr int NB = F::NB, MT = F::TILES, W = kNarrowWarps, NBUF = C::NBUF, NT = C::NT, PP = C::PP;
    constexpr bool PACK = C::PACK;
    constexpr int STEP = PP * F::BYTES;
    extern __shared__ __align__(16) uint8_t nar_sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // this lane's column of Q^T operands, and the first of its two in the accumulators
    const int gq = PACK ? g & 3 : g, tq = PACK ? 2 * (t & 1) : 2 * t;
    const int room = a.c.max_blocks * kKv4Tokens;
    if (threadIdx.x == 0) {   // no tile of several parts begins here, as yet
        a.split[blockIdx.x].c0 = a.split[blockIdx.x].c1 = 0;
        pdl_launch_dependents();
    }
    uint8_t* ring = nar_sm + (size_t)warp * NBUF * STEP;
    uint64_t* full = reinterpret_cast<uint64_t*>(nar_sm + C::BAR) + warp * NBUF;
    uint8_t* vsc = nar_sm + C::VSC + warp * (PP * C::VSC_PAGE);
    float* acc_s = reinterpret_cast<float*>(nar_sm + C::MERGE);         // [W][COLS][PITCH]
    float* ml_s = acc_s + (size_t)W * COLS * C::PITCH;                  // [W][COLS][2]
    if (lane == 0) {
        for (int s = 0; s < NBUF; s++) mbar_init(full + s, 1);
        fence_mbar_init();
    }

    float* qbuf = reinterpret_cast<float*>(nar_sm + C::QBUF);          // [2][COLS][HD]
    NarrowEntry* kept = a.n_entries <= kNarrowKept ? reinterpret_cast<NarrowEntry*>(nar_sm + C::KEPT) : nullptr;
    __shared__ int scan_sm[2][2][W];
    __shared__ NarrowRun run_s;
    NarrowPart* parts = reinterpret_cast<NarrowPart*>(nar_sm + C::PARTS);   // the last, this and the next one
    {
        const int per = (a.n_entries + W * 32 - 1) / (W * 32), i0 = threadIdx.x * per;
        const int before = a.aligned ? 0 : kNarrowTileCost;
        // pass 0: all units without alignment give the run; pass 1: the units of
        // the threads up to this one
        int run = 1, total = 0, longest = 1, mine = 0, upto = 0;
#pragma unroll 1
        for (int pass = 0; pass < 2; pass++) {
            mine = 0;
            for (int i = i0; i < min(i0 + per, a.n_entries); i++) {
                const NarrowEntry e = kept && pass ? kept[i] : narrow_entry(a, i, COLS, blockIdx.x == 0 && !pass);
                if (kept && !pass) kept[i] = e;
                const int n = e.nblk + before;
                mine += (a.aligned ? (n + run - 1) / run * run : n) * e.segs;
                longest = max(longest, n);
            }
            upto = mine;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, s);
                if (lane >= s) upto += v;
            }
            longest = __reduce_max_sync(0xffffffffu, longest);
            if (lane == 31) {
                scan_sm[pass][0][warp] = upto;
                scan_sm[pass][1][warp] = longest;
            }
            __syncthreads();
            upto -= mine;
            total = 0;
#pragma unroll
            for (int w = 0; w < W; w++) {
                if (w < warp) upto += scan_sm[pass][0][w];
                total += scan_sm[pass][0][w];
                longest = max(longest, scan_sm[pass][1][w]);
            }
            if (pass) break;
            // aligned: at most `tiles` more runs than the units fill
            const int ctas = gridDim.x - a.aligned;
            run = max(max(a.aligned ? kNarrowMinPages : kNarrowMinUnits, (total + ctas - 1) / ctas), (longest + kNarrowMaxParts - 1) / kNarrowMaxParts);
            if (!a.aligned) break;
        }
        const int p = blockIdx.x * run;
        if (p >= total) return;
        if (p >= upto && p < upto + mine) {   // one thread: the entry that holds unit p
            NarrowRun r;
            r.p = p;
            r.end = min(total, p + run);
            r.run = run;
            r.before = before;
            r.first = upto;
            r.entry = i0;
            run_s = r;
            narrow_next_part<COLS>(a, kept, run_s, parts[0]);
        }
        __syncthreads();
    }
    if (parts[0].b1 <= parts[0].b0) return;   // no page of a tile in the run
    // the part's Q rows to buffer `to`, zeros behind its columns
    auto fetch_q = [&](const NarrowPart& d, int to) {
        for (int idx = threadIdx.x; idx < COLS * (HD / 4); idx += W * 32) {
            const int col = idx / (HD / 4), c = d.col0 + col, j = c / a.G;
            const bool ok = c < d.cols;
            const float* src = a.q + (ok ? (int64_t)(d.r0 + j) * a.ldq + (int64_t)(d.kvh * a.G + c - j * a.G) * HD +
                                               idx % (HD / 4) * 4 : 0);
            cp_async16_zfill(qbuf + to * COLS * HD + idx * 4, src, ok);
        }
        cp_async_commit();
    };
    fetch_q(parts[0], 0);

    int ids = -1;            // lane l: the id of the l-th page from step n / (32 / PP) * (32 / PP) on
    uint32_t bad = 0;        // bit PP s + k: page k of buffer s is none
    unsigned used = 0;       // steps of this warp so far, over all parts
    bool lost = false;       // a copy never came: compute nothing more
    auto steps_of = [&](const NarrowPart& d) {
        const int steps = (d.b1 - d.b0 + PP - 1) / PP;
        return steps > warp && !lost ? (steps - warp + W - 1) / W : 0;
    };
    // step n of this warp in part d: pages b0 + (n W + warp) PP + 0 .. PP - 1
    auto issue = [&](const NarrowPart& d, int n) {
        if (n % (32 / PP) == 0) {
            const int blk = d.b0 + ((n + lane / PP) * W + warp) * PP + lane % PP;
            const bool live = blk < d.b1 && blk * kKv4Tokens < d.ctx;
            ids = live ? __ldg(a.c.table + (int64_t)d.seq * a.c.max_blocks + blk) : -1;
            if (live && (unsigned)ids >= (unsigned)a.c.n_pages) record_status(a.status, AXQ8_ERR_INVALID);
        }
        const int s = (used + n) % NBUF;
        int page[PP], bytes = 0;
#pragma unroll
        for (int k = 0; k < PP; k++) {
            page[k] = __shfl_sync(0xffffffffu, ids, (n * PP + k) & 31);
            const bool ok = (unsigned)page[k] < (unsigned)a.c.n_pages;
            bad = (bad & ~(1u << (PP * s + k))) | ((ok ? 0u : 1u) << (PP * s + k));
            if (!ok) page[k] = -1;
            else bytes += F::BYTES;
        }
        if (lane == 0) {
            const uint8_t* src = a.c.pages + d.kvh * F::BYTES;
            const int pitch = a.c.n_kv * F::BYTES;
            mbar_arrive_expect_tx(full + s, bytes);
#pragma unroll
            for (int k = 0; k < PP; k++)
                if (page[k] >= 0)
                    bulk_g2s(ring + s * STEP + k * F::BYTES, src + (int64_t)page[k] * pitch, F::BYTES, full + s);
        }
    };
    for (int n = 0; n < min(steps_of(parts[0]), NBUF); n++) issue(parts[0], n);
    if (threadIdx.x == 0) narrow_next_part<COLS>(a, kept, run_s, parts[1]);
    cp_async_wait_all();
    __syncthreads();   // Q is there, and the second part

  int turn = 0;
  for (int which = 0, qb = 0;; which = which == 2 ? 0 : which + 1, qb ^= 1) {
    const NarrowPart& part = parts[which];
    const NarrowPart& next = parts[which == 2 ? 0 : which + 1];
    const int part_steps = steps_of(part), part_b0 = part.b0, ctx = part.ctx;

    // Q^T operands (column gq), their block sums and scales (columns tq, tq + 1)
    uint32_t qh[NT][NB][4], ql[PACK ? 1 : NT][PACK ? 1 : NB][4];
    float qs[NT][2][NB], mul[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        float x[NB][8], mx = 0.0f;
        const float* qp = qbuf + (qb * COLS + 8 * n + gq) * HD;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 v = *reinterpret_cast<const float4*>(qp + 32 * b + 8 * t + e);
                x[b][e] = v.x;
                x[b][e + 1] = v.y;
                x[b][e + 2] = v.z;
                x[b][e + 3] = v.w;
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^k with max |q| 2^k in [2^10, 2^11)
        const int ex = max((int)(__float_as_uint(mx) >> 23), 40) - 127;
        const float up = __uint_as_float((uint32_t)(127 + 10 - ex) << 23);
        const float down = __uint_as_float((uint32_t)(127 - 10 + ex) << 23) * 16777216.0f * a.scale;
        float sum[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            constexpr int first[4] = {0, 2, 1, 3};   // elements of operand register k: (first, first + 4)
            sum[b] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float f = k < 2 ? 1.0f : 0.0625f;
                const float x0 = x[b][first[k]] * up, x1 = x[b][first[k] + 4] * up;
                // rounded to whole numbers by the addition
                const float r0 = (x0 + 12582912.0f) - 12582912.0f, r1 = (x1 + 12582912.0f) - 12582912.0f;
                const uint32_t hi = pack_f16(r0 * f, r1 * f), lo = pack_f16((x0 - r0) * f, (x1 - r1) * f);
                if (PACK) {   // columns 4 .. 7 are the residuals of columns 0 .. 3
                    qh[n][b][k] = g < 4 ? hi : lo;
                    const float2 v = f16_pair(qh[n][b][k]);
                    sum[b] += (v.x + v.y) * (k < 2 ? 1.0f : 16.0f);
                } else {
                    qh[n][b][k] = hi;
                    ql[n][b][k] = lo;
                    sum[b] += x0 + x1;
                }
            }
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 1);
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 2);
        }
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {
            const int src = (2 * t + hh) * 4;
#pragma unroll
            for (int b = 0; b < NB; b++) qs[n][hh][b] = __shfl_sync(0xffffffffu, sum[b], src);
            mul[n][hh] = __shfl_sync(0xffffffffu, down, src);
            const int cc = part.col0 + 8 * n + tq + hh;
            lim[n][hh] = cc < part.cols ? min(part.pos0 + cc / a.G + 1, room) : 0;
        }
    }
    int low = ctx;   // tokens that every live column sees
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int hh = 0; hh < 2; hh++)
            if (part.col0 + 8 * n + tq + hh < part.cols) low = min(low, lim[n][hh]);
    low = __reduce_min_sync(0xffffffffu, low);

    const float rest = t < 2 ? 0.0f : -1.0f;
    // e, and the scale words that it takes: dlow .. dlow + dspan - 1.  At first d of 2^-8 to
    // 2^2, where the steps of values around 1 lie.
    int dexp = 14;
    uint32_t dlow = 7u << 10, dspan = 10u << 10;
    float o[NT][MT][4], base[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        base[n][0] = base[n][1] = -CUDART_INF_F;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int m = 0; m < MT; m++) o[n][m][0] = o[n][m][1] = o[n][m][2] = o[n][m][3] = 0.0f;
    }

    for (int it = 0; it < part_steps; it++) {
        const int s = (used + it) % NBUF;
        if (!__all_sync(0xffffffffu, copy_wait(full + s, ((used + it) / NBUF) & 1))) {
            // a copy was lost: no other may still be landing when the CTA ends
            if (lane == 0) record_status(a.status, AXQ8_ERR_WAIT_TIMEOUT);
            for (unsigned n = used + it + 1; n < used + min(part_steps, it + NBUF); n++)
                copy_wait(full + n % NBUF, (n / NBUF) & 1);
            lost = true;   // and none is started
            break;
        }
        const uint8_t* buf = ring + s * STEP;
        int tok0[PP];   // first token of a page; no page: one that nothing sees
#pragma unroll
        for (int p = 0; p < PP; p++)
            tok0[p] = (bad >> (PP * s + p)) & 1 ? 0x40000000
                                                : (part_b0 + (it * W + warp) * PP + p) * kKv4Tokens;
        // V factors: lane (g, t) makes those of block b = g % NB, tokens 2t + 8u, 2t + 1 + 8u
        uint32_t wa[PP], wb[PP];
        auto scale_words = [&](uint32_t hidden) {
#pragma unroll
            for (int p = 0; p < PP; p++) {
                const uint8_t* vs = buf + p * F::BYTES + F::VS;
                const int u = g / NB, r = 2 * t + 8 * (u & 1), b = g % NB;
                wa[p] = *reinterpret_cast<const uint16_t*>(vs + F::scale(r, b));
                wb[p] = *reinterpret_cast<const uint16_t*>(vs + F::scale(r + 1, b));
                if (tok0[p] + kKv4Tokens > ctx) {   // slots behind the last token, any bits: their weights are 0
                    if (tok0[p] + r >= ctx) wa[p] = hidden;
                    if (tok0[p] + r + 1 >= ctx) wb[p] = hidden;
                }
            }
        };
        auto put_factors = [&] {
            const uint32_t up1 = f16_pow2(dexp / 2), up2 = f16_pow2(dexp - dexp / 2);
#pragma unroll
            for (int p = 0; p < PP; p++) {
                const uint32_t w = __byte_perm(wa[p], wb[p], 0x5410);
                const uint32_t D = hmul2u(hmul2u(w & 0x7ff07ff0u, up1), up2);
                if (g < 2 * NB)
                    *reinterpret_cast<uint2*>(vsc + p * C::VSC_PAGE + ((t * NB + g % NB) * 2 + g / NB) * 8) =
                        make_uint2(D, hmul2u(w & 0x000f000fu, D) ^ 0x80008000u);
            }
        };
        auto put_far_factors = [&](uint32_t limit) {   // d below it
#pragma unroll
            for (int p = 0; p < PP; p++) {
                const uint32_t w = __byte_perm(wa[p] < limit ? wa[p] : 0, wb[p] < limit ? wb[p] : 0, 0x5410);
                if (g < 2 * NB)
                    *reinterpret_cast<uint2*>(vsc + p * C::VSC_PAGE + ((t * NB + g % NB) * 2 + g / NB) * 8) =
                        make_uint2(w & 0x7ff07ff0u, (w & 0x000f000fu) | 0x64006400u);
            }
        };
        scale_words(dlow);
        bool out = false, left = false;
#pragma unroll
        for (int p = 0; p < PP; p++) out |= wa[p] - dlow >= dspan || wb[p] - dlow >= dspan;
        if (__builtin_expect(__any_sync(0xffffffffu, out), 0)) {
            // a window for the largest d, and for all the smaller ones if there is one
            uint32_t top = 0, low = 0xffffffffu;
#pragma unroll
            for (int p = 0; p < PP; p++) {
                top = max(top, max(wa[p], wb[p]));
                low = min(low, min(wa[p] - 16u, wb[p] - 16u));   // zeros aside
            }
            top = __reduce_max_sync(0xffffffffu, top) >> 10;
            low = __reduce_min_sync(0xffffffffu, low) + 16u;
            low = low < 16 ? top : low >> 10;   // binades, 0 below 2^-14
            const uint32_t spare = low == 0 || top > low + 9 ? 0 : (9 - (top - low)) / 2;
            dexp = 30 - (int)(top + spare);
            dlow = dexp >= 26 ? 16 : (uint32_t)max(1, 21 - dexp) << 10;
            dspan = ((uint32_t)(31 - dexp) << 10) - dlow;
#pragma unroll
            for (int p = 0; p < PP; p++) {
                left |= (wa[p] < dlow && wa[p] >= 16) || (wb[p] < dlow && wb[p] >= 16);
                if (C::AFTER && wa[p] < dlow) wa[p] = 0;
                if (C::AFTER && wb[p] < dlow) wb[p] = 0;
            }
            left = __any_sync(0xffffffffu, left);
        }
        if (C::AFTER || !left) put_factors();
        else put_far_factors(0x10000u);
        // scores: tokens g (sc[..][0], [1]) and g + 8 ([2], [3]), columns tq, tq + 1
        float sc[PP][NT][4];
#pragma unroll
        for (int p = 0; p < PP; p++) {
            const uint8_t* pg = buf + p * F::BYTES;
#pragma unroll
            for (int n = 0; n < NT; n++) sc[p][n][0] = sc[p][n][1] = sc[p][n][2] = sc[p][n][3] = 0.0f;
            uint32_t w0[NB], w1[NB];
            lds_words<NB>(w0, pg + g * (HD / 2) + t * (HD / 8));
            lds_words<NB>(w1, pg + (g + 8) * (HD / 2) + t * (HD / 8));
            Scales<NB> s0, s1;
            s0.load(pg + F::KS, g);
            s1.load(pg + F::KS, g + 8);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t u0 = w0[b] >> 8, u1 = w1[b] >> 8;
                const uint32_t lowa[4] = {w0[b] & 0x000f000fu, w1[b] & 0x000f000fu,
                                          u0 & 0x000f000fu, u1 & 0x000f000fu};
                const uint32_t higha[4] = {w0[b] & 0x00f000f0u, w1[b] & 0x00f000f0u,
                                           u0 & 0x00f000f0u, u1 & 0x00f000f0u};
                const float2 d0p = f16_pair(s0.word(b) & 0x7ff07ff0u), z0p = f16_pair(s0.word(b) & 0x000f000fu);
                const float2 d1p = f16_pair(s1.word(b) & 0x7ff07ff0u), z1p = f16_pair(s1.word(b) & 0x000f000fu);
                const float d0 = b & 1 ? d0p.y : d0p.x, z0 = b & 1 ? z0p.y : z0p.x;
                const float d1 = b & 1 ? d1p.y : d1p.x, z1 = b & 1 ? z1p.y : z1p.x;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float c[4];
                    if constexpr (PACK) {
                        mma_f16_16816_first(c, lowa, qh[n][b][0], qh[n][b][1]);
                    } else {
                        // residuals last: the sum before them is exact
                        mma_f16_16816_first(c, lowa, qh[n][b][0], qh[n][b][1]);
                        mma_f16_16816(c, higha, qh[n][b][2], qh[n][b][3]);
                        mma_f16_16816(c, lowa, ql[n][b][0], ql[n][b][1]);
                        mma_f16_16816(c, higha, ql[n][b][2], ql[n][b][3]);
                    }
                    if constexpr (PACK) mma_f16_16816(c, higha, qh[n][b][2], qh[n][b][3]);
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
                        sc[p][n][hh] = fmaf(d0, fmaf(-z0, qs[n][hh][b], c[hh]), sc[p][n][hh]);
                        sc[p][n][2 + hh] = fmaf(d1, fmaf(-z1, qs[n][hh][b], c[2 + hh]), sc[p][n][2 + hh]);
                    }
                }
            }
            if (PACK)
#pragma unroll
                for (int k = 0; k < 4; k++) sc[p][0][k] += __shfl_xor_sync(0xffffffffu, sc[p][0][k], 2);
            if (tok0[p] + kKv4Tokens > low) {   // some column does not see all of the page
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (tok0[p] + g + 4 * (k & 2) >= lim[n][k & 1]) sc[p][n][k] = -CUDART_INF_F;
            }
        }
        float mx[NT][2];
        bool over = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
                mx[n][hh] = fmaxf(sc[0][n][hh], sc[0][n][2 + hh]);
#pragma unroll
                for (int p = 1; p < PP; p++)
                    mx[n][hh] = fmaxf(mx[n][hh], fmaxf(sc[p][n][hh], sc[p][n][2 + hh]));
                mx[n][hh] *= mul[n][hh];
                over |= mx[n][hh] > base[n][hh] + 8.0f;
            }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    float m = mx[n][hh];
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(m, base[n][hh]);
                    const float f = m == -CUDART_INF_F ? 1.0f : ex2(base[n][hh] - m);   // 0 from -inf
                    base[n][hh] = m;
                    l[n][hh] *= f;
#pragma unroll
                    for (int k = 0; k < MT; k++) {
                        o[n][k][hh] *= f;
                        o[n][k][2 + hh] *= f;
                    }
                }
        }
        __syncwarp();   // V factors are written
        // weights, as P^T operands: tokens 2t, 2t + 1 and + 8, column g
        uint32_t ph[PP][NT][2], pl[PP][PACK ? 1 : NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float b7[2];
#pragma unroll
            for (int hh = 0; hh < 2; hh++) b7[hh] = base[n][hh] == -CUDART_INF_F ? 0.0f : base[n][hh] - 7.0f;
#pragma unroll
            for (int p = 0; p < PP; p++) {
                float w[4];
#pragma unroll
                for (int k = 0; k < 4; k++) w[k] = ex2(fmaf(sc[p][n][k], mul[n][k & 1], -b7[k & 1]));
                l[n][0] += w[0] + w[2];
                l[n][1] += w[1] + w[3];
                if constexpr (PACK) {   // the high parts (t < 2), or what they leave
                    const float2 a0 = f16_pair(pack_f16(w[0], w[1])), a1 = f16_pair(pack_f16(w[2], w[3]));
                    ph[p][n][0] = movmatrix_t(pack_f16(fmaf(rest, a0.x, w[0]), fmaf(rest, a0.y, w[1])));
                    ph[p][n][1] = movmatrix_t(pack_f16(fmaf(rest, a1.x, w[2]), fmaf(rest, a1.y, w[3])));
                } else {
                    uint32_t h0, l0, h1, l1;
                    split2(w[0], w[1], h0, l0);
                    split2(w[2], w[3], h1, l1);
                    ph[p][n][0] = movmatrix_t(h0);
                    ph[p][n][1] = movmatrix_t(h1);
                    pl[p][n][0] = movmatrix_t(l0);
                    pl[p][n][1] = movmatrix_t(l1);
                }
            }
        }
        // O^T += V^T P^T.  A product truncates what it adds to about 24 bits of the
        // largest term, so a step's products are summed from zero and added in fp32.
        constexpr int TPG = F::TPG;
        auto add_values = [&](auto by_window) {
            constexpr bool WINDOW = decltype(by_window)::value;
            const float back = __uint_as_float((uint32_t)(127 + 24 - dexp) << 23);
            // factors of tokens (2t, 2t + 1), (2t + 8, 2t + 9), and what high nibbles take instead
            uint32_t f2[PP][4], fh[PP][2];
#pragma unroll
            for (int m0 = 0; m0 < MT; m0 += TPG) {
                uint32_t x[PP][TPG];
#pragma unroll
                for (int p = 0; p < PP; p++)
                    lds_words<TPG>(x[p], buf + p * F::BYTES + F::V + (m0 / TPG) * (128 * TPG) + lane * (4 * TPG));
#pragma unroll
                for (int k = 0; k < TPG; k++) {
                    const int m = m0 + k, b = m / 2;
                    float c[NT][4];
#pragma unroll
                    for (int p = 0; p < PP; p++) {
                        if (m % 2 == 0) {
                            lds_words<4>(f2[p], vsc + p * C::VSC_PAGE + (t * NB + b) * 16);
#pragma unroll
                            for (int u = 0; u < 2; u++)   // D / 16, or 64 + z
                                fh[p][u] = WINDOW ? hmul2u(f2[p][2 * u], 0x2c002c00u)
                                                  : (f2[p][2 * u + 1] & 0x000f000fu) * 16 + 0x54005400u;
                        }
                        uint32_t v[4];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const uint32_t y = u ? x[p][k] >> 8 : x[p][k], d = f2[p][2 * u], z = f2[p][2 * u + 1];
                            if constexpr (WINDOW) {
                                v[2 * u] = hfma2u(y & 0x000f000fu, d, z);
                                v[2 * u + 1] = hfma2u(y & 0x00f000f0u, fh[p][u], z);
                            } else {
                                v[2 * u] = hmul2u(hsub2u((y & 0x000f000fu) | 0x64006400u, z), d);
                                v[2 * u + 1] = hmul2u(hsub2u((y & 0x00f000f0u) | 0x54005400u, fh[p][u]), d);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            if (p == 0) mma_f16_16816_first(c[n], v, ph[p][n][0], ph[p][n][1]);
                            else mma_f16_16816(c[n], v, ph[p][n][0], ph[p][n][1]);
                            if constexpr (!PACK) mma_f16_16816(c[n], v, pl[p][n][0], pl[p][n][1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) o[n][m][j] = fmaf(c[n][j], WINDOW ? back : 1.0f, o[n][m][j]);
                }
            }
        };
        if (C::AFTER || !left) add_values(std::true_type{});
        if (__builtin_expect(left, 0)) {
            if (C::AFTER) {
                scale_words(0);
                __syncwarp();   // the factors are read
                put_far_factors(dlow);
                __syncwarp();
            }
            add_values(std::false_type{});
        }
        __syncwarp();   // buffer s is read
        if (it + NBUF < part_steps) issue(part, it + NBUF);
    }

    // the warp's state to shared memory
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {
            l[n][hh] += __shfl_xor_sync(0xffffffffu, l[n][hh], 4);
            l[n][hh] += __shfl_xor_sync(0xffffffffu, l[n][hh], 8);
            l[n][hh] += __shfl_xor_sync(0xffffffffu, l[n][hh], 16);
        }
    if (PACK)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int k = 0; k < 4; k++) o[0][m][k] += __shfl_xor_sync(0xffffffffu, o[0][m][k], 2);
    // the next part's first copies land while this one is written
    used += part_steps;
    const bool more = next.b1 > next.b0;
    if (more) {
        for (int n = 0; n < min(steps_of(next), NBUF); n++) issue(next, n);
        fetch_q(next, qb ^ 1);
    }
    __syncthreads();   // the states of the last part are read
    if (threadIdx.x == 0 && more)
        narrow_next_part<COLS>(a, kept, run_s, parts[which == 0 ? 2 : which - 1]);
    if (!PACK || t < 2) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int hh = 0; hh < 2; hh++) {
                const int col = 8 * n + tq + hh;
                float* row = acc_s + ((size_t)warp * COLS + col) * C::PITCH;
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    row[16 * m + g] = o[n][m][hh];
                    row[16 * m + g + 8] = o[n][m][2 + hh];
                }
                if (g == 0) {
                    ml_s[(warp * COLS + col) * 2] = base[n][hh];
                    ml_s[(warp * COLS + col) * 2 + 1] = l[n][hh];
                }
            }
    }
    cp_async_wait_all();
    __syncthreads();   // states, and the next part's Q
    if constexpr (COLS <= 4) narrow_merge_call<HD, COLS>(a, which, turn);
    else narrow_merge<HD, COLS>(a, which, turn);
    turn ^= 1;
    if (!more) break;
  }
}

}  // namespace axq8
