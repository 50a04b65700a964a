// Causal attention of long chunks over the 4-bit cache on the 5th-generation
// tensor cores (tcgen05.mma kind::f16, accumulators in TMEM).
//
// The (row, head) pairs that read one KV head of one chunk are the rows of
// 128-row tiles; a CTA takes two tiles (256 rows: 64 positions of 4 heads) and
// walks the tokens 0 .. its last position in steps of 128 (8 pages):
//   S [128 x 128] = Q K^T     A = Q from shared memory, B = K
//   O [128 x HD] += P V       A = P from TMEM, B = V^T
// A cache value d (q - z) is an fp16 number, so K and V^T tiles are formed in
// shared memory without rounding (128-byte-swizzled K-major rows), once for
// both tiles.  Q (scaled per row by a power of two to below 2^14) and P (2^7
// times the softmax weight) are an fp16 high part plus an fp16 residual,
// multiplied one after the other, at twice the products: 4 x 2048 prompt rows are
// 1.2e-6 off (fp32 sums 5.5e-7), most of it the sums of O.  Dims within 8 stand in the order 0 4 1 5 2 6 3 7 in both Q and K:
// the order in which a code word's nibbles come out in pairs.
//
// Roles: warps 0-3 and 4-7 the softmax of tile 0 and 1 (a thread is a row),
// warps 8-11 form the K tiles and 12-15 the V^T tiles from page words that they
// read a step ahead, warp 16 issues the products in the order
//   PV(tile 0, step j)  QK(tile 0, j + 1)  PV(tile 1, j)  QK(tile 1, j + 1)
// so that each tile's softmax runs under the other tile's products.  P takes
// the place of S in TMEM, 32 tokens at a time, in one pass: the softmax
// reference (base 2, a whole number) moves only when a score exceeds it by more
// than 8, and then O and the step's earlier P are multiplied by a power of two.
// O rows go out through shared memory.  Every kWideKeep steps O is added to an fp32 sum
// (kept where the rows of the output will stand) and starts anew.
//
// Bound: 4 x 128 x 128 x HD multiply-adds a step and tile, 5.2k cycles a step at
// HD 128; a step takes 8.5k to 9.1k (a tile's softmax and products follow one
// another), 9.3k with the fp32 sums of O among 16, and a CTA 29k beside its steps.
// Four prompts of 2048 tokens (32 query, 8 KV heads of 128): 478 us, 287 TFLOP/s of
// the algorithm's operations, tensor pipe active 0.31 of the time.  Every wait is
// bounded; a role that gives up raises a flag, and all stop.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"
#include "kv4.cuh"
#include "kv4_narrow.cuh"
#include "tcgen05.cuh"

namespace axq8 {

constexpr int kWideTok = 128;                      // tokens of a step
constexpr int kWidePages = kWideTok / kKv4Tokens;
// Steps summed in TMEM at a time.  The tensor cores' sums drop what lies below their
// last place, always the same way: over 16,000 tokens of values of one sign an O summed
// throughout was 1.2e-4 off, 16 steps at a time 1.3e-5, 8 below 1e-5 (values of both
// signs: 3.8e-5, 4.9e-6, 2.7e-6; all tokens alike: 8 at most 2.1e-5).  The fp32 sums of these pieces cost 4 us each.
constexpr int kWideKeep = 8;
constexpr int kWideThreads = 20 * 32;              // five warpgroups, the last one for the products
// Registers of a thread by role (setmaxnreg); at launch each has 96.
constexpr int kWideRegs = 96, kWideRegsSoft = 128, kWideRegsTiles = 80, kWideRegsMma = 64;
static_assert(2 * kWideRegsSoft + 2 * kWideRegsTiles + kWideRegsMma <= 5 * kWideRegs, "registers of the launch");

struct WideArgs {
    Kv4Pages c;
    const float* q;
    int64_t ldq;
    int n_rows, max_rows, n_heads, G;
    const int* q_seq;
    const int* q_start;
    const int* q_pos;
    float scale;          // softmax scale times log2(e)
    float* out;
    int* status;
};

template <int HD>
struct WideCfg {
    static constexpr int ATOMS = HD > 64 ? 2 : 1;           // 64 dims of a Q or K row
    static constexpr int ATOM = kWideTok * 128;             // bytes: 128 rows of 128
    static constexpr int Q = 2 * 2 * ATOMS * ATOM;          // [tile][high, residual][atom]
    static constexpr int K = ATOMS * ATOM;
    static constexpr int VATOM = HD * 128;                  // 64 tokens of a V^T row
    static constexpr int V = 2 * VATOM;
    static constexpr int OFF_K = Q, OFF_V = Q + K;
    static constexpr int OFF_VS = OFF_V + V;                // V scales [2][page][block][16]
    static constexpr int VS = kWidePages * (HD / 32) * 32;
    static constexpr int OFF_MUL = OFF_VS + 2 * VS;         // score factors of the rows [2][128]
    static constexpr int OFF_BAR = OFF_MUL + 2 * 128 * 4;
    static constexpr int SMEM = 1024 + OFF_BAR + 256;
    static constexpr int OROW = HD * 4 + 16;                // bytes of an output row on its way out
    static_assert(256 * OROW <= OFF_VS, "output rows");
    static constexpr int TILE_COLS = 128 + (HD < 32 ? 32 : HD);   // S (P), then O
    static constexpr int TMEM_COLS = 512;
};

template <int N>
__device__ __forceinline__ void wide_regs_dec() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void wide_regs_inc() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Instruction descriptor, kind::f16: D fp32 (bits 4-5 = 1), A and B fp16, both
// K-major, N >> 3 at bit 17, M >> 4 at bit 24.
__host__ __device__ constexpr uint32_t wide_idesc(int M, int N) {
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// 8 codes of a word as 4 fp16 pairs (q0 q4) (q1 q5) (q2 q6) (q3 q7), minus the
// zero points z (1024 + z pair), zh (-(64 + z) pair), times the steps d.
__device__ __forceinline__ void kv4_word(uint32_t w, uint32_t d, uint32_t z, uint32_t zh, uint32_t* v) {
    const uint32_t y = w >> 8;
    v[0] = hmul2u(hsub2u((w & 0x000f000fu) | 0x64006400u, z), d);
    v[1] = hmul2u(hfma2u((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, zh), d);
    v[2] = hmul2u(hsub2u((y & 0x000f000fu) | 0x64006400u, z), d);
    v[3] = hmul2u(hfma2u((y & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, zh), d);
}

// Wait for a phase; false (and all roles stop) when it does not come, or when
// another role has given up.
__device__ __forceinline__ bool wide_wait(uint64_t* bar, uint32_t parity, volatile int* stop, int* status) {
    for (int i = 0; i < 200000; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(10000)
            : "memory");
        if (ok) return true;
        if (*stop) return false;
    }
    *stop = 1;
    record_status(status, AXQ8_ERR_WAIT_TIMEOUT);
    return false;
}

// The softmax reference has moved: n16 times 16 columns of O (fp32) times f, and
// `pages` 16-token pieces of P (fp16 pairs) times 2^down.
__device__ __noinline__ void wide_rescale(int n16, uint32_t o, int pages, uint32_t ts, int down, float f) {
    uint32_t v[16];
    tmem_wait_st();   // P as written so far
#pragma unroll 1
    for (int c = 0; c < n16; c++) {
        tmem_ld16(o + 16 * c, v);
        tmem_wait_ld16(v);
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
        tmem_st16(o + 16 * c, v);
    }
#pragma unroll 1
    for (int p = 0; p < pages; p++) {
        tmem_ld16(ts + 16 * p, v);
        tmem_wait_ld16(v);
        for (int k = down; k < 0; k += 14) {   // fp16 factors go down to 2^-14
            const uint32_t h = f16_pow2(max(k, -14));
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = hmul2u(v[e], h);
        }
        tmem_st16(ts + 16 * p, v);
    }
    tmem_wait_st();
}

// O of the last steps plus f times the row's sum so far (`kept`: there is one) goes to
// memory, or (`back`) to O for the end.  A sum rests where the warp's rows of the output
// come to stand; with 32 rows, chunk c of every lane's row side by side in row c, so
// that a warp's access is 512 bytes in one piece.  A lane reads what itself wrote.
template <int HD>
__device__ __noinline__ void wide_keep(uint32_t o, float* out, int64_t row, bool live, bool kept, bool back, float f) {
    constexpr int OL = HD / 4;
    const int lane = threadIdx.x & 31;
    const bool full = __all_sync(0xffffffffu, live);
    uint32_t v[16];
#pragma unroll 1
    for (int c = 0; c < HD / 16; c++) {
        float4* at[4];
        float4 was[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int ch = 4 * c + e;
            const int64_t r = __shfl_sync(0xffffffffu, row, full ? ch * (32 / OL) + lane / OL : lane);
            at[e] = reinterpret_cast<float4*>(out + r) + (full ? lane % OL : ch);
            was[e] = live && kept ? *at[e] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        tmem_ld16(o + 16 * c, v);
        tmem_wait_ld16(v);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            was[e].x = fmaf(was[e].x, f, __uint_as_float(v[4 * e]));
            was[e].y = fmaf(was[e].y, f, __uint_as_float(v[4 * e + 1]));
            was[e].z = fmaf(was[e].z, f, __uint_as_float(v[4 * e + 2]));
            was[e].w = fmaf(was[e].w, f, __uint_as_float(v[4 * e + 3]));
        }
        if (back) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[4 * e] = __float_as_uint(was[e].x);
                v[4 * e + 1] = __float_as_uint(was[e].y);
                v[4 * e + 2] = __float_as_uint(was[e].z);
                v[4 * e + 3] = __float_as_uint(was[e].w);
            }
            tmem_st16(o + 16 * c, v);
        } else if (live) {
#pragma unroll
            for (int e = 0; e < 4; e++) *at[e] = was[e];
        }
    }
    if (back) tmem_wait_st();
}

// 2^(from - to) for two references, at least 2^-120; 2^-120 too where one is infinite.
__device__ __forceinline__ float wide_down(float from, float to) {
    return __uint_as_float((uint32_t)(127 + (int)fmaxf(from - to, -120.0f)) << 23);
}

template <int HD>
__global__ void __launch_bounds__(kWideThreads, 1) kv4_attn_wide_kernel(const __grid_constant__ WideArgs a) {
    using F = Kv4<HD>;
    using C = WideCfg<HD>;
    constexpr int NB = F::NB;
    extern __shared__ uint8_t wide_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wide_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t *kfull = bars, *vfull = bars + 1, *kfree = bars + 2, *vfree = bars + 3, *qfull = bars + 4,
             *sfull = bars + 5, *pfull = bars + 7, *odone = bars + 9;   // sfull, pfull, odone: [tile]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12);
    volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile uint32_t* present = reinterpret_cast<volatile uint32_t*>(tmem_slot + 2);   // [2] pages of a step
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // the chunk's rows and positions; the last tiles, with the most tokens, first
    const int i = blockIdx.z, kvh = blockIdx.y;
    const int r0 = a.q_start[i], T = a.q_start[i + 1] - r0;
    if (T <= 0) return;
    if (r0 < 0 || r0 > a.n_rows - T || T > a.max_rows) {
        if (threadIdx.x == 0) record_status(a.status, AXQ8_ERR_INVALID);
        return;
    }
    const int rows = T * a.G, m0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * 256;
    if (m0 >= rows) return;
    const int room = a.c.max_blocks * kKv4Tokens;
    const int seq_in = a.q_seq ? a.q_seq[i] : i;
    const bool seq_ok = seq_in >= 0 && seq_in < a.c.n_seqs;
    const int seq = seq_ok ? seq_in : 0, pos0 = min(a.q_pos[i], room);
    if ((!seq_ok || pos0 + T > room) && threadIdx.x == 0 && m0 == 0) record_status(a.status, AXQ8_ERR_INVALID);
    const int tiles = rows - m0 > 128 ? 2 : 1;
    const int jlast = min(rows - 1, m0 + 255) / a.G;
    const int ctx = seq_ok ? max(0, min(pos0 + jlast + 1, room)) : 0;
    const int steps = max(1, (ctx + kWideTok - 1) / kWideTok);

    if (threadIdx.x == 0) {
        mbar_init(kfull, 128);
        mbar_init(vfull, 128);
        mbar_init(kfree, 1);
        mbar_init(vfree, 1);
        mbar_init(qfull, 128 * tiles);
        for (int x = 0; x < 2; x++) {
            mbar_init(sfull + x, 1);
            mbar_init(pfull + x, 128);
            mbar_init(odone + x, 1);
        }
        *stop = 0;
        fence_mbar_init();
    }
    if (warp == 16) tmem_alloc(tmem_slot, C::TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp < 8) {
        // ---- softmax: thread = row of tile x --------------------------------------
        wide_regs_inc<kWideRegsSoft>();
        const int x = warp >> 2;
        if (x < tiles) {
            // Q rows of this warp, LPR lanes (8 dims each) to a row, as many rows on their
            // way as registers hold
            constexpr int LPR = HD / 8, RPI = 32 / LPR, ITS = 32 / RPI, AHEAD = ITS < 8 ? ITS : 8;
            float* mul_s = reinterpret_cast<float*>(sm + C::OFF_MUL) + x * 128;
            const int r = (warp & 3) * 32 + lane, m = m0 + 128 * x + r;   // this thread's row
            const bool live = m < rows;
            const int j = min(m, rows - 1) / a.G;
            const int64_t mine = (int64_t)(r0 + j) * a.ldq + (int64_t)(kvh * a.G + min(m, rows - 1) - j * a.G) * HD;
            const int ch = lane % LPR;
#pragma unroll 1
            for (int i0 = 0; i0 < ITS; i0 += AHEAD) {
                float4 u[AHEAD], v[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {
                    const float* qp = a.q + __shfl_sync(0xffffffffu, mine, (i0 + k) * RPI + lane / LPR) + 8 * ch;
                    u[k] = __ldg(reinterpret_cast<const float4*>(qp));
                    v[k] = __ldg(reinterpret_cast<const float4*>(qp + 4));
                }
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {
                    const int rr = (warp & 3) * 32 + (i0 + k) * RPI + lane / LPR;
                    float mx = fmaxf(fmaxf(fmaxf(fabsf(u[k].x), fabsf(u[k].y)), fmaxf(fabsf(u[k].z), fabsf(u[k].w))),
                                     fmaxf(fmaxf(fabsf(v[k].x), fabsf(v[k].y)), fmaxf(fabsf(v[k].z), fabsf(v[k].w))));
#pragma unroll
                    for (int o = 1; o < LPR; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    // 2^k with max |q| 2^k in [2^13, 2^14); rows behind the last are zero
                    const int ex = max((int)(__float_as_uint(mx) >> 23), 40) - 127;
                    const float up = m0 + 128 * x + rr < rows ? __uint_as_float((uint32_t)(127 + 13 - ex) << 23) : 0.0f;
                    if (ch == 0) mul_s[rr] = __uint_as_float((uint32_t)(127 - 13 + ex) << 23) * a.scale;
                    uint4 hi, lo;
                    split2(u[k].x * up, v[k].x * up, hi.x, lo.x);
                    split2(u[k].y * up, v[k].y * up, hi.y, lo.y);
                    split2(u[k].z * up, v[k].z * up, hi.z, lo.z);
                    split2(u[k].w * up, v[k].w * up, hi.w, lo.w);
                    uint8_t* at = sm + (x * 2 * C::ATOMS + (ch >> 3)) * C::ATOM + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4);
                    *reinterpret_cast<uint4*>(at) = hi;
                    *reinterpret_cast<uint4*>(at + C::ATOMS * C::ATOM) = lo;
                }
            }
            bool lost = false;   // a wait gave up: go on without waiting
            fence_async_smem();
            __syncwarp();
            mbar_arrive(qfull);

            const float mul = mul_s[r];
            const int pos = live && seq_ok ? min(pos0 + j, room - 1) : -1;   // the last token seen
            const int sees = __reduce_min_sync(0xffffffffu, live ? pos : 0x7fffffff);
            const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + x * C::TILE_COLS, to = ts + 128;
            const int64_t oat = (int64_t)(r0 + j) * a.n_heads * HD + (int64_t)(kvh * a.G + min(m, rows - 1) - j * a.G) * HD;
            // the weights' sum and what its additions put over (equal weights round the same way at
            // each: a plain sum was 1.3e-4 off at 16,000 tokens), and the sum of a step
            float base = -CUDART_INF_F, l = 0.0f, l_over = 0.0f, l_step[2] = {0.0f, 0.0f};
            float kept = -CUDART_INF_F;   // the reference of the sum in `out`
            uint32_t s[2][32];   // 32 tokens each, the next ones on their way
            for (int st = 0; st < steps; st++) {
                if (!lost) lost = !wide_wait(sfull + x, st & 1, stop, a.status);
                __syncwarp();
                tc_fence_after();
                const bool fresh = st % kWideKeep == 0;   // O starts from zero in this step
                if (fresh && st) {
                    wide_keep<HD>(to, a.out, oat, live, st > kWideKeep, false, wide_down(kept, base));
                    kept = base;
                }
                tmem_ld32(ts, s[0]);
                const int tok0 = st * kWideTok;
                const uint32_t pages = present[st & 1];
                const bool whole = tok0 + kWideTok - 1 <= sees && pages == (1u << kWidePages) - 1;
#pragma unroll
                for (int c = 0; c < kWideTok / 32; c++) {
                    uint32_t* v = s[c & 1];
                    tmem_wait_ld32(v);
                    if (c + 1 < kWideTok / 32) tmem_ld32(ts + 32 * (c + 1), s[(c + 1) & 1]);
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            const int tok = 32 * c + e;
                            if (tok0 + tok > pos || !((pages >> (tok / kKv4Tokens)) & 1)) v[e] = 0xff800000u;
                        }
                    }
                    float t4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                    for (int e = 0; e < 32; e++) t4[e & 3] = fmaxf(t4[e & 3], __uint_as_float(v[e]));
                    const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * mul;
                    const bool over = top > base + 8.0f;
                    if (__any_sync(0xffffffffu, over)) {
                        const float to_base = over ? ceilf(top) : base;
                        // the factor 2^down; nothing so far: any
                        const int down = over && base != -CUDART_INF_F ? (int)fmaxf(base - to_base, -120.0f) : 0;
                        base = to_base;
                        const float f = __uint_as_float((uint32_t)(127 + down) << 23);
                        l *= f;
                        l_over *= f;
                        l_step[0] *= f;
                        l_step[1] *= f;
                        // what is on its way has to arrive before its registers can be moved
                        if (c + 1 < kWideTok / 32) tmem_wait_ld32(s[(c + 1) & 1]);
                        if (!fresh || c) wide_rescale(fresh ? 0 : HD / 16, to, 2 * c, ts, down, f);
                    }
                    const float b7 = base == -CUDART_INF_F ? 0.0f : base - 7.0f;
#pragma unroll
                    for (int p = 0; p < 2; p++) {   // 16 tokens: 8 columns of high pairs, 8 of residuals
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float w0 = ex2(fmaf(__uint_as_float(v[16 * p + 2 * e]), mul, -b7));
                            const float w1 = ex2(fmaf(__uint_as_float(v[16 * p + 2 * e + 1]), mul, -b7));
                            l_step[0] = c || p || e ? l_step[0] + w0 : w0;
                            l_step[1] = c || p || e ? l_step[1] + w1 : w1;
                            split2(w0, w1, hi[e], lo[e]);
                        }
                        tmem_st8(ts + 32 * c + 8 * p, hi);
                        tmem_st8(ts + 32 * c + 16 + 8 * p, lo);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(pfull + x);
                const float add = l_step[0] + l_step[1] - l_over, sum = l + add;
                l_over = (sum - l) - add;
                l = sum;
            }
            // O / l: the tile's rows to shared memory (Q and K are read), from there to `out`
            if (!lost) lost = !wide_wait(odone + x, 0, stop, a.status);
            __syncwarp();
            tc_fence_after();
            if (steps > kWideKeep) wide_keep<HD>(to, a.out, oat, live, true, true, wide_down(kept, base));
            const float sum = l - l_over;
            const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;   // nothing seen: zeros
            uint8_t* orow = sm + (128 * x + r) * C::OROW;
#pragma unroll
            for (int c = 0; c < HD / 32; c++) {
                tmem_ld32(to + 32 * c, s[0]);
                tmem_wait_ld32(s[0]);
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<float4*>(orow + (32 * c + e) * 4) =
                        make_float4(__uint_as_float(s[0][e]) * inv, __uint_as_float(s[0][e + 1]) * inv,
                                    __uint_as_float(s[0][e + 2]) * inv, __uint_as_float(s[0][e + 3]) * inv);
            }
            __syncwarp();
            // this warp's rows, HD / 4 lanes to a row
            constexpr int OL = HD / 4;
#pragma unroll 4
            for (int k = 0; k < OL; k++) {
                const int rr = k * (32 / OL) + lane / OL;
                const int64_t at = __shfl_sync(0xffffffffu, oat, rr);
                if (m0 + 128 * x + (warp & 3) * 32 + rr < rows)
                    *reinterpret_cast<float4*>(a.out + at + 4 * (lane % OL)) = *reinterpret_cast<const float4*>(
                        sm + (128 * x + (warp & 3) * 32 + rr) * C::OROW + 16 * (lane % OL));
            }
        }
    } else if (warp < 16) {
        // ---- K tiles (warps 8-11) and V^T tiles (12-15) --------------------------------
        wide_regs_dec<kWideRegsTiles>();
        const int w = warp & 3, th = threadIdx.x & 127;
        const int* row = a.c.table + (int64_t)seq * a.c.max_blocks;
        bool lost = false;   // a wait gave up: go on without waiting, to the same barriers
        int ids = -1;
        auto page_ids = [&](int st) {      // lane p: page p of step st; a bit for each that is there
            const int blk = st * kWidePages + (lane & 7);
            const bool in = blk * kKv4Tokens < ctx;
            ids = in ? __ldg(row + blk) : -1;
            if ((unsigned)ids >= (unsigned)a.c.n_pages) {
                if (in && th < 8) record_status(a.status, AXQ8_ERR_INVALID);
                ids = -1;
            }
            return __ballot_sync(0xffffffffu, lane < 8 && ids >= 0);
        };
        auto page_at = [&](int p) {
            const int id = __shfl_sync(0xffffffffu, ids, p);
            return id < 0 ? nullptr : a.c.pages + ((int64_t)id * a.c.n_kv + kvh) * F::BYTES;
        };
        if (warp < 12) {
            uint32_t kw[4][NB], there = 0;
            Scales<NB> ksc[4];
            auto read_k = [&](int st) {        // tokens 32 w + 8 k + lane / 4, chunk lane % 4
                there = page_ids(st);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int tok = 32 * w + 8 * k + (lane >> 2), slot = tok % kKv4Tokens;
                    const uint8_t* pg = page_at(tok / kKv4Tokens);
                    const bool in = pg && st * kWideTok + tok < ctx;
#pragma unroll
                    for (int b = 0; b < NB; b++) kw[k][b] = 0;
#pragma unroll
                    for (int b = 0; b < Scales<NB>::W; b++) ksc[k].w[b] = 0;
                    if (in) {
                        lds_words<NB>(kw[k], pg + slot * (HD / 2) + (lane & 3) * (HD / 8));
                        ksc[k].load(pg + F::KS, slot);
                    }
                }
            };
            read_k(0);
            for (int st = 0; st < steps; st++) {
                // half of the values first, so that little stands between the old tile's last
                // product and the new tile's first
                uint4 kv[2][NB];
                auto form = [&](int k) {
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint32_t sc = b & 1 ? ksc[k].word(b) >> 16 : ksc[k].word(b) & 0xffffu;
                        const uint32_t two = sc | (sc << 16);
                        kv4_word(kw[k][b], two & 0x7ff07ff0u, (two & 0x000f000fu) | 0x64006400u,
                                 ((two << 4) & 0x00f000f0u) | 0xd400d400u, reinterpret_cast<uint32_t*>(&kv[k & 1][b]));
                    }
                };
                auto store = [&](int k) {
                    const int tok = 32 * w + 8 * k + (lane >> 2);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const int ch = 4 * b + (lane & 3);
                        *reinterpret_cast<uint4*>(sm + C::OFF_K + (ch >> 3) * C::ATOM + tok * 128 +
                                                  (((ch & 7) ^ (tok & 7)) << 4)) = kv[k & 1][b];
                    }
                };
                form(0);
                form(1);
                if (st && !lost) lost = !wide_wait(kfree, (st - 1) & 1, stop, a.status);
                if (th == 0) present[st & 1] = there;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    store(k);
                    if (k < 2) form(k + 2);
                }
                fence_async_smem();
                mbar_arrive(kfull);
                __syncwarp();
                if (st + 1 < steps) read_k(st + 1);
            }
        } else {
            constexpr int VT = HD / 2, VI = HD / 32;           // threads of a page, pages of a thread
            const int vp = th / VT, vm = (th % VT) / 8, vg = th % 8;
            uint32_t vw[VI][4];
            Scales<NB> vsc;
            auto read_v = [&](int st) {
                page_ids(st);
#pragma unroll
                for (int k = 0; k < VI; k++) {
                    const uint8_t* pg = page_at(vp + k * (kWidePages / VI));
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        vw[k][t] = pg ? __ldg(reinterpret_cast<const uint32_t*>(
                                            pg + F::V + (vm / F::TPG) * (128 * F::TPG) + (vg * 4 + t) * (4 * F::TPG) +
                                            (vm % F::TPG) * 4))
                                      : 0u;
                }
                // the scales of token th; slots behind the last token hold any bits
                const uint8_t* pg = page_at(th / kKv4Tokens);
#pragma unroll
                for (int b = 0; b < Scales<NB>::W; b++) vsc.w[b] = 0;
                if (pg && st * kWideTok + th < ctx) vsc.load(pg + F::VS, th % kKv4Tokens);
            };
            read_v(0);
            for (int st = 0; st < steps; st++) {
                // scales to [page][block][token]
                uint16_t* vs = reinterpret_cast<uint16_t*>(sm + C::OFF_VS + (st & 1) * C::VS);
#pragma unroll
                for (int b = 0; b < NB; b++)
                    vs[(th / kKv4Tokens * NB + b) * 16 + th % kKv4Tokens] =
                        (uint16_t)(b & 1 ? vsc.word(b) >> 16 : vsc.word(b));
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (st && !lost) lost = !wide_wait(vfree, (st - 1) & 1, stop, a.status);
#pragma unroll
                for (int k = 0; k < VI; k++) {
                    const int p = vp + k * (kWidePages / VI), b = vm / 2;
                    uint32_t sc[8];   // tokens 2t, 2t + 1
                    lds_words<8>(sc, reinterpret_cast<const uint8_t*>(vs + (p * NB + b) * 16));
                    uint32_t lo[8], hi[8];   // dims 16 vm + vg and + 8, token pairs
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const uint32_t x = vw[k][t], y = x >> 8;
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const uint32_t q = u ? y : x, s2 = sc[t + 4 * u];
                            const uint32_t d = s2 & 0x7ff07ff0u;
                            lo[t + 4 * u] = hmul2u(hsub2u((q & 0x000f000fu) | 0x64006400u,
                                                          (s2 & 0x000f000fu) | 0x64006400u), d);
                            hi[t + 4 * u] = hmul2u(hfma2u((q & 0x00f000f0u) | 0x64006400u, 0x2c002c00u,
                                                          ((s2 << 4) & 0x00f000f0u) | 0xd400d400u), d);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const int ch = (p & 3) * 2 + u;
                        uint8_t* at = sm + C::OFF_V + (p >> 2) * C::VATOM + (16 * vm + vg) * 128 + ((ch ^ vg) << 4);
                        *reinterpret_cast<uint4*>(at) = make_uint4(lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]);
                        *reinterpret_cast<uint4*>(at + 8 * 128) =
                            make_uint4(hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]);
                    }
                }
                fence_async_smem();
                mbar_arrive(vfull);
                __syncwarp();
                if (st + 1 < steps) read_v(st + 1);
            }
        }
    } else {
      wide_regs_dec<kWideRegsMma>();
      if (warp == 16 && lane == 0) {
        // ---- products -------------------------------------------------------------
        constexpr uint32_t iqk = wide_idesc(128, kWideTok), ipv = wide_idesc(128, HD);
        const uint32_t qa = smem_u32(sm), ka = smem_u32(sm + C::OFF_K), va = smem_u32(sm + C::OFF_V);
        auto qk = [&](int x) {
            const uint32_t d = tmem + x * C::TILE_COLS;
            // residuals first: what a product drops below its largest term is smaller
            // then (with P's the same way: 1.6e-6 of the result, 2.0e-6 the other way)
#pragma unroll 1
            for (int part = 0; part < 2; part++)
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint64_t qd = sw128_kmajor_desc(qa + ((x * 2 + 1 - part) * C::ATOMS + k / 4) * C::ATOM) + 2 * (k & 3);
                    const uint64_t kd = sw128_kmajor_desc(ka + (k / 4) * C::ATOM) + 2 * (k & 3);
                    mma_f16_ss(d, qd, kd, iqk, part | k);
                }
            tc_commit(sfull + x);
        };
        auto pv = [&](int x, int st) {
            const uint32_t d = tmem + x * C::TILE_COLS + 128;
#pragma unroll 1
            for (int part = 0; part < 2; part++)
#pragma unroll
                for (int p = 0; p < kWidePages; p++) {
                    const uint64_t vd = sw128_kmajor_desc(va + (p / 4) * C::VATOM) + 2 * (p & 3);
                    mma_f16_ts(d, tmem + x * C::TILE_COLS + (p / 2) * 32 + (1 - part) * 16 + (p & 1) * 8, vd, ipv,
                               st % kWideKeep | part | p);
                }
        };
        bool ok = wide_wait(qfull, 0, stop, a.status) && wide_wait(kfull, 0, stop, a.status);
        tc_fence_after();
        if (ok) {
            for (int x = 0; x < tiles; x++) qk(x);
            tc_commit(kfree);
        }
        for (int st = 0; ok && st < steps; st++) {
            for (int x = 0; x < tiles; x++) {   // tile 1's last product ends last
                ok = wide_wait(pfull + x, st & 1, stop, a.status) &&
                     (x || wide_wait(vfull, st & 1, stop, a.status));
                if (!ok) break;
                tc_fence_after();
                pv(x, st);
                if (x == tiles - 1) tc_commit(vfree);
                else if (st + 1 == steps) tc_commit(odone);
                if (st + 1 < steps) {
                    if (x == 0 && !(ok = wide_wait(kfull, (st + 1) & 1, stop, a.status))) break;
                    tc_fence_after();
                    qk(x);
                    if (x == tiles - 1) tc_commit(kfree);
                }
            }
        }
        tc_commit(odone + tiles - 1);
      }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        // every product has retired before TMEM is released
        mbar_wait_bounded(odone + tiles - 1, 0, a.status, AXQ8_ERR_WAIT_TIMEOUT);
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

}  // namespace axq8
