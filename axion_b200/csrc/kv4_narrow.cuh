// Attention of few columns over the 4-bit cache: decode steps and short chunks.
//
// The (row, head) pairs that read one KV head of one sequence are columns of a
// tile of 8 NT; a page's 16 tokens are the rows of m16n8k16 products:
//   S^T [16 tokens x 8] = K Q^T,  O^T [HD x 8] += V^T P^T.
// The cache words are laid out as the products' A operands, so a code goes
// from shared memory to the tensor core through registers only:
//   K: a nibble in place is the fp16 subnormal q 2^-24 (low nibbles) or q 2^-20
//      (high ones), which the product takes as it is; Q is divided by 16 in the
//      high nibbles' k-steps.  A block's 32 dims are two k-steps, and
//      s = sum_b d_b (acc_b - z_b sum_b(q)) puts step and zero point in after
//      the integer product, in fp32.
//   V: (q - z) d is formed in registers, exact in fp16 (the format's steps have
//      7 significant bits).
// Q (scaled by a power of two to below 2^14) and P (2^7 times the softmax
// weight) are split into an fp16 high part and an fp16 residual, multiplied
// one after the other: results keep fp32 accuracy.  Softmax in base 2 with a
// running reference; it moves (and O is rescaled) only when a score exceeds it
// by more than 8, so that weights stay within fp16.
//
// kNarrowWarps warps take the split's pages in turn.  Each has its own ring of
// page buffers, filled by one bulk copy per page (a page's 18 HD bytes of one
// KV head are contiguous).  The warps' states merge in shared memory, splits of
// the context through the workspace in the last CTA of a tile, in split order.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"
#include "decode_ops.cuh"
#include "kv4.cuh"

namespace axq8 {

constexpr int kNarrowWarps = 4;
constexpr int kNarrowBufs = 4;        // pages in flight per warp
constexpr int kNarrowMinPages = 8;    // pages of a split at least
constexpr int kNarrowMaxSplits = 128;

struct Kv4Pages {
    uint8_t* pages;
    const int* table;
    int n_seqs, max_blocks, n_pages, n_kv;
};

struct NarrowArgs {
    Kv4Pages c;
    const float* q;
    int64_t ldq;
    int n_rows, max_rows, n_heads, G, nsplit;
    const int* q_seq;
    const int* q_start;   // null: one row per entry
    const int* q_pos;
    float scale;          // softmax scale times log2(e)
    float* out;
    float* part;          // [tile][split][8 NT][HD], then [tile][split][8 NT][2]
    int* counters;        // one per tile
    int* status;
};

template <int HD, int NT>
struct NarrowCfg {
    static constexpr int COLS = 8 * NT;
    static constexpr int PITCH = HD + 4;   // merge rows, conflict-free
    static constexpr size_t RING = (size_t)kNarrowWarps * kNarrowBufs * Kv4<HD>::BYTES;
    static constexpr size_t MERGE = (size_t)kNarrowWarps * COLS * (PITCH + 2) * 4;
    static constexpr size_t BAR = RING > MERGE ? RING : MERGE;
    static constexpr size_t SMEM = BAR + kNarrowWarps * kNarrowBufs * 8;
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

template <int HD, int NT>
__global__ void __launch_bounds__(kNarrowWarps * 32) kv4_attn_narrow_kernel(const NarrowArgs a) {
    using F = Kv4<HD>;
    using C = NarrowCfg<HD, NT>;
    constexpr int NB = F::NB, MT = F::TILES, W = kNarrowWarps, NBUF = kNarrowBufs;
    extern __shared__ __align__(16) uint8_t nar_sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.x % a.c.n_kv, ct = blockIdx.x / a.c.n_kv;
    const int i = blockIdx.y, sp = blockIdx.z;
    const int tile = (i * (gridDim.x / a.c.n_kv) + ct) * a.c.n_kv + kvh;

    // the entry's rows, sequence and positions
    int r0 = i, T = 1;
    if (a.q_start) {
        r0 = __ldg(a.q_start + i);
        T = __ldg(a.q_start + i + 1) - r0;
        if (T <= 0) return;
        if (r0 < 0 || r0 > a.n_rows - T || T > a.max_rows) {
            if (threadIdx.x == 0) record_status(a.status, AXQ8_ERR_INVALID);
            return;
        }
    }
    const int cols = T * a.G, col0 = ct * C::COLS;
    if (col0 >= cols) return;
    const int seq = a.q_seq ? __ldg(a.q_seq + i) : i;
    const int room = a.c.max_blocks * kKv4Tokens;
    const bool seq_ok = seq >= 0 && seq < a.c.n_seqs;
    const int pos0 = min(__ldg(a.q_pos + i), room);
    if ((!seq_ok || pos0 + T > room) && threadIdx.x == 0) record_status(a.status, AXQ8_ERR_INVALID);
    const int jmax = min(T - 1, (col0 + C::COLS - 1) / a.G);
    const int ctx = seq_ok ? max(0, min(pos0 + jmax + 1, room)) : 0;
    const int nblk = (ctx + kKv4Tokens - 1) / kKv4Tokens;
    const int pps = max(kNarrowMinPages, (nblk + a.nsplit - 1) / a.nsplit);
    const int ns = max(1, (nblk + pps - 1) / pps);
    if (sp >= ns) return;
    const int b0 = sp * pps, b1 = min(nblk, b0 + pps);

    // page ring of this warp
    uint8_t* ring = nar_sm + (size_t)warp * NBUF * F::BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(nar_sm + C::BAR) + warp * NBUF;
    if (lane == 0) {
        for (int s = 0; s < NBUF; s++) mbar_init(full + s, 1);
        fence_mbar_init();
    }
    __syncwarp();
    const int npw = b1 > b0 + warp ? (b1 - b0 - warp + W - 1) / W : 0;
    const int* row_table = a.c.table + (int64_t)(seq_ok ? seq : 0) * a.c.max_blocks;
    int ids = -1;            // lane l: the id of this warp's page 32 (n / 32) + l
    uint32_t bad = 0;        // bit s: the page of buffer s is outside the pool
    auto issue = [&](int n) {
        if ((n & 31) == 0) {
            const int blk = b0 + warp + (n + lane) * W;
            ids = blk < b1 ? __ldg(row_table + blk) : 0;
        }
        const int page = __shfl_sync(0xffffffffu, ids, n & 31), s = n % NBUF;
        const bool ok = page >= 0 && page < a.c.n_pages;
        bad = (bad & ~(1u << s)) | ((ok ? 0u : 1u) << s);
        if (lane == 0) {
            if (ok) {
                mbar_arrive_expect_tx(full + s, F::BYTES);
                bulk_g2s(ring + s * F::BYTES, a.c.pages + ((int64_t)page * a.c.n_kv + kvh) * F::BYTES,
                         F::BYTES, full + s);
            } else {
                record_status(a.status, AXQ8_ERR_INVALID);
                mbar_arrive(full + s);
            }
        }
    };
    for (int n = 0; n < min(npw, NBUF); n++) issue(n);

    // Q^T operands (column g), their block sums and scales (columns 2t, 2t + 1)
    uint32_t qh[NT][NB][4], ql[NT][NB][4];
    float qs[NT][2][NB], mul[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int col = col0 + 8 * n + g, j = col / a.G;
        float x[NB][8], mx = 0.0f;
        const float* qp = a.q + (int64_t)(r0 + j) * a.ldq + (int64_t)(kvh * a.G + col - j * a.G) * HD;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (col < cols) v = __ldg(reinterpret_cast<const float4*>(qp + 32 * b + 8 * t + e));
                x[b][e] = v.x;
                x[b][e + 1] = v.y;
                x[b][e + 2] = v.z;
                x[b][e + 3] = v.w;
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^k with max |q| 2^k in [2^13, 2^14)
        const int ex = max((int)(__float_as_uint(mx) >> 23), 40) - 127;
        const float up = __uint_as_float((uint32_t)(127 + 13 - ex) << 23);
        const float down = __uint_as_float((uint32_t)(127 - 13 + ex) << 23) * 16777216.0f * a.scale;
        float sum[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            sum[b] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[b][e] *= up;
                sum[b] += x[b][e];
            }
            split2(x[b][0], x[b][4], qh[n][b][0], ql[n][b][0]);
            split2(x[b][2], x[b][6], qh[n][b][1], ql[n][b][1]);
            split2(x[b][1] * 0.0625f, x[b][5] * 0.0625f, qh[n][b][2], ql[n][b][2]);
            split2(x[b][3] * 0.0625f, x[b][7] * 0.0625f, qh[n][b][3], ql[n][b][3]);
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 1);
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 2);
        }
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {
            const int src = (2 * t + hh) * 4;
#pragma unroll
            for (int b = 0; b < NB; b++) qs[n][hh][b] = __shfl_sync(0xffffffffu, sum[b], src);
            mul[n][hh] = __shfl_sync(0xffffffffu, down, src);
            const int cc = col0 + 8 * n + 2 * t + hh;
            lim[n][hh] = cc < cols ? min(pos0 + cc / a.G + 1, room) : 0;
        }
    }
    int low = ctx;   // tokens that every live column sees
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int hh = 0; hh < 2; hh++)
            if (col0 + 8 * n + 2 * t + hh < cols) low = min(low, lim[n][hh]);
    low = __reduce_min_sync(0xffffffffu, low);

    float o[NT][MT][4], base[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        base[n][0] = base[n][1] = -CUDART_INF_F;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int m = 0; m < MT; m++) o[n][m][0] = o[n][m][1] = o[n][m][2] = o[n][m][3] = 0.0f;
    }

    for (int it = 0; it < npw; it++) {
        const int s = it % NBUF;
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(full + s, (it / NBUF) & 1, a.status,
                                                       AXQ8_ERR_WAIT_TIMEOUT))) {
            // no copy may still be landing when the CTA reuses its shared memory
            for (int n = it + 1; n < min(npw, it + NBUF); n++)
                mbar_wait_bounded(full + n % NBUF, (n / NBUF) & 1, a.status, AXQ8_ERR_WAIT_TIMEOUT);
            break;
        }
        const uint8_t* pg = ring + s * F::BYTES;
        const int tok0 = (b0 + warp + it * W) * kKv4Tokens;
        if (!((bad >> s) & 1)) {
            // scores: tokens g (sc[..][0], [1]) and g + 8 ([2], [3]), columns 2t, 2t + 1
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
            {
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
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        // residuals first: the product truncates each sum to the
                        // accumulator's 24 bits, which costs less while it is small
                        mma_f16_16816(c, lowa, ql[n][b][0], ql[n][b][1]);
                        mma_f16_16816(c, higha, ql[n][b][2], ql[n][b][3]);
                        mma_f16_16816(c, lowa, qh[n][b][0], qh[n][b][1]);
                        mma_f16_16816(c, higha, qh[n][b][2], qh[n][b][3]);
#pragma unroll
                        for (int hh = 0; hh < 2; hh++) {
                            sc[n][hh] = fmaf(d0, fmaf(-z0, qs[n][hh][b], c[hh]), sc[n][hh]);
                            sc[n][2 + hh] = fmaf(d1, fmaf(-z1, qs[n][hh][b], c[2 + hh]), sc[n][2 + hh]);
                        }
                    }
                }
            }
            bool over = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    sc[n][hh] *= mul[n][hh];
                    sc[n][2 + hh] *= mul[n][hh];
                }
            if (tok0 + kKv4Tokens > low) {   // some column does not see all of the page
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
                        if (tok0 + g >= lim[n][hh]) sc[n][hh] = -CUDART_INF_F;
                        if (tok0 + g + 8 >= lim[n][hh]) sc[n][2 + hh] = -CUDART_INF_F;
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int hh = 0; hh < 2; hh++)
                    over |= fmaxf(sc[n][hh], sc[n][2 + hh]) > base[n][hh] + 8.0f;
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
                        float mx = fmaxf(sc[n][hh], sc[n][2 + hh]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        if (mx > base[n][hh]) {
                            const float f = ex2(base[n][hh] - mx);   // 0 from -inf
                            base[n][hh] = mx;
                            l[n][hh] *= f;
#pragma unroll
                            for (int m = 0; m < MT; m++) {
                                o[n][m][hh] *= f;
                                o[n][m][2 + hh] *= f;
                            }
                        }
                    }
            }
            // weights, as P^T operands: tokens 2t, 2t + 1 and + 8, column g
            uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float p[4];
#pragma unroll
                for (int hh = 0; hh < 2; hh++) {
                    const float b7 = base[n][hh] == -CUDART_INF_F ? 0.0f : base[n][hh] - 7.0f;
                    p[hh] = ex2(sc[n][hh] - b7);
                    p[2 + hh] = ex2(sc[n][2 + hh] - b7);
                    l[n][hh] += p[hh] + p[2 + hh];
                }
                uint32_t h0, l0, h1, l1;
                split2(p[0], p[1], h0, l0);
                split2(p[2], p[3], h1, l1);
                ph[n][0] = movmatrix_t(h0);
                ph[n][1] = movmatrix_t(h1);
                pl[n][0] = movmatrix_t(l0);
                pl[n][1] = movmatrix_t(l1);
            }
            // steps and zero points of tokens (2t, 2t + 1) and (2t + 8, 2t + 9)
            uint32_t d2[2][NB], z2[2][NB], z2h[2][NB];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                Scales<NB> sa, sb;
                sa.load(pg + F::VS, 2 * t + 8 * u);
                sb.load(pg + F::VS, 2 * t + 1 + 8 * u);
                if (tok0 + kKv4Tokens > ctx) {   // slots behind the last token: any bits
#pragma unroll
                    for (int w = 0; w < Scales<NB>::W; w++) {
                        if (tok0 + 2 * t + 8 * u >= ctx) sa.w[w] = 0;
                        if (tok0 + 2 * t + 1 + 8 * u >= ctx) sb.w[w] = 0;
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const uint32_t w = __byte_perm(sa.word(b), sb.word(b), b & 1 ? 0x7632 : 0x5410);
                    d2[u][b] = w & 0x7ff07ff0u;
                    z2[u][b] = (w & 0x000f000fu) | 0x64006400u;           // 1024 + z
                    z2h[u][b] = ((w << 4) & 0x00f000f0u) | 0xd400d400u;   // -(64 + z)
                }
            }
            // O^T += V^T P^T
            constexpr int TPG = F::TPG;
#pragma unroll
            for (int m0 = 0; m0 < MT; m0 += TPG) {
                uint32_t w[TPG];
                lds_words<TPG>(w, pg + F::V + (m0 / TPG) * (128 * TPG) + lane * (4 * TPG));
#pragma unroll
                for (int k = 0; k < TPG; k++) {
                    const int m = m0 + k, b = m / 2;
                    const uint32_t x = w[k], y = w[k] >> 8;
                    uint32_t v[4];
                    v[0] = hmul2u(hsub2u((x & 0x000f000fu) | 0x64006400u, z2[0][b]), d2[0][b]);
                    v[1] = hmul2u(hfma2u((x & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, z2h[0][b]), d2[0][b]);
                    v[2] = hmul2u(hsub2u((y & 0x000f000fu) | 0x64006400u, z2[1][b]), d2[1][b]);
                    v[3] = hmul2u(hfma2u((y & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, z2h[1][b]), d2[1][b]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        mma_f16_16816(o[n][m], v, ph[n][0], ph[n][1]);
                        mma_f16_16816(o[n][m], v, pl[n][0], pl[n][1]);
                    }
                }
            }
        }
        __syncwarp();   // buffer s is read
        if (it + NBUF < npw) issue(it + NBUF);
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
    __syncthreads();   // every ring is read
    float* acc_s = reinterpret_cast<float*>(nar_sm);                       // [W][COLS][PITCH]
    float* ml_s = acc_s + (size_t)W * C::COLS * C::PITCH;                  // [W][COLS][2]
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int hh = 0; hh < 2; hh++) {
            const int col = 8 * n + 2 * t + hh;
            float* row = acc_s + ((size_t)warp * C::COLS + col) * C::PITCH;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                row[16 * m + g] = o[n][m][hh];
                row[16 * m + g + 8] = o[n][m][2 + hh];
            }
            if (g == 0) {
                ml_s[(warp * C::COLS + col) * 2] = base[n][hh];
                ml_s[(warp * C::COLS + col) * 2 + 1] = l[n][hh];
            }
        }
    __syncthreads();
    const int live = min(C::COLS, cols - col0);
    float* pacc = a.part + ((int64_t)tile * a.nsplit + sp) * C::COLS * HD;
    float* pml = a.part + (int64_t)gridDim.x * gridDim.y * a.nsplit * C::COLS * HD +
                 ((int64_t)tile * a.nsplit + sp) * C::COLS * 2;
    for (int idx = threadIdx.x; idx < live * (HD / 4); idx += W * 32) {
        const int col = idx / (HD / 4), d = idx % (HD / 4) * 4;
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < W; w++) mx = fmaxf(mx, ml_s[(w * C::COLS + col) * 2]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float mw = ml_s[(w * C::COLS + col) * 2];
            const float f = mw == -CUDART_INF_F ? 0.0f : ex2(mw - mx);
            const float4 x = *reinterpret_cast<const float4*>(acc_s + ((size_t)w * C::COLS + col) * C::PITCH + d);
            v.x = fmaf(x.x, f, v.x);
            v.y = fmaf(x.y, f, v.y);
            v.z = fmaf(x.z, f, v.z);
            v.w = fmaf(x.w, f, v.w);
            sum = fmaf(ml_s[(w * C::COLS + col) * 2 + 1], f, sum);
        }
        if (ns > 1) {
            *reinterpret_cast<float4*>(pacc + col * HD + d) = v;
            if (d == 0) {
                pml[col * 2] = mx;
                pml[col * 2 + 1] = sum;
            }
            continue;
        }
        const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;   // nothing seen: zeros
        const int c = col0 + col, j = c / a.G;
        *reinterpret_cast<float4*>(a.out + (int64_t)(r0 + j) * a.n_heads * HD +
                                   (int64_t)(kvh * a.G + c - j * a.G) * HD + d) =
            make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
    if (ns == 1) return;

    // the last split's CTA joins them, in split order
    __threadfence();
    __syncthreads();
    __shared__ int last;
    if (threadIdx.x == 0) {
        last = atomicAdd(a.counters + tile, 1) == ns - 1;
        if (last) a.counters[tile] = 0;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    pacc = a.part + (int64_t)tile * a.nsplit * C::COLS * HD;
    pml = a.part + (int64_t)gridDim.x * gridDim.y * a.nsplit * C::COLS * HD + (int64_t)tile * a.nsplit * C::COLS * 2;
    float* fac = acc_s;                      // [ns][COLS] factors, then [COLS] 1 / sum
    for (int col = warp; col < live; col += W) {
        float mx = -CUDART_INF_F, sum = 0.0f;
        for (int k = lane; k < ns; k += 32) mx = fmaxf(mx, __ldcg(pml + ((int64_t)k * C::COLS + col) * 2));
        mx = warp_max(mx);
        for (int k = lane; k < ns; k += 32) {
            const float mk = __ldcg(pml + ((int64_t)k * C::COLS + col) * 2);
            const float f = mk == -CUDART_INF_F ? 0.0f : ex2(mk - mx);
            fac[k * C::COLS + col] = f;
            sum = fmaf(__ldcg(pml + ((int64_t)k * C::COLS + col) * 2 + 1), f, sum);
        }
        sum = warp_sum(sum);
        if (lane == 0) fac[ns * C::COLS + col] = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < live * (HD / 4); idx += W * 32) {
        const int col = idx / (HD / 4), d = idx % (HD / 4) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int k = 0; k < ns; k++) {
            const float f = fac[k * C::COLS + col];
            const float4 x = ld_cg4(pacc + ((int64_t)k * C::COLS + col) * HD + d);
            v.x = fmaf(x.x, f, v.x);
            v.y = fmaf(x.y, f, v.y);
            v.z = fmaf(x.z, f, v.z);
            v.w = fmaf(x.w, f, v.w);
        }
        const float inv = fac[ns * C::COLS + col];
        const int c = col0 + col, j = c / a.G;
        *reinterpret_cast<float4*>(a.out + (int64_t)(r0 + j) * a.n_heads * HD +
                                   (int64_t)(kvh * a.G + c - j * a.G) * HD + d) =
            make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
}

}  // namespace axq8
