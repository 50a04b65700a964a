// The 4-bit KV page format (include/axkv.h, axkv4_cache): offsets of a page's
// parts, the block quantizer, and the word layouts of the K and V codes.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace axq8 {

constexpr int kKv4Tokens = 16;          // tokens of a page
constexpr float kKv4Limit = 32768.0f;   // values are clamped to it

// Byte offsets inside one (page, KV head): K codes, V codes, K scales, V scales.
template <int HD>
struct Kv4 {
    static_assert(HD == 32 || HD == 64 || HD == 128, "head dim");
    static constexpr int NB = HD / 32;                 // blocks of a token
    static constexpr int TILES = HD / 16;              // 16-dim tiles of V
    static constexpr int TPG = TILES < 4 ? TILES : 4;  // tiles of a V group
    static constexpr int V = 8 * HD;
    static constexpr int KS = 16 * HD;
    static constexpr int VS = 17 * HD;
    static constexpr int BYTES = 18 * HD;
    // The byte of token r that holds K dim 32 b + 2 i (low nibble) and + 1.
    __host__ __device__ static constexpr int k_byte(int r, int b, int i) {
        return r * (HD / 2) + (i >> 2) * (HD / 8) + 4 * b + (i & 3);
    }
    // The byte of token r that holds V dim 16 tile + g (low nibble) and + 8.
    __host__ __device__ static constexpr int v_byte(int r, int tile, int g) {
        return V + (tile / TPG) * (128 * TPG) + (g * 4 + ((r & 7) >> 1)) * (4 * TPG) +
               (tile % TPG) * 4 + 2 * (r & 1) + (r >> 3);
    }
    __host__ __device__ static constexpr int scale(int r, int b) { return (r * NB + b) * 2; }
};

__device__ __forceinline__ float kv4_step(int code) {   // fp16 with the low 4 bits clear
    return __half2float(__ushort_as_half((unsigned short)(code << 4)));
}

// The code of the smallest step d with 15 d >= R.  15 d has 11 significant
// bits, so the comparisons are exact; the guess is at most two codes low (the
// quotient's rounding and the truncation) and never too high.
__device__ __forceinline__ int kv4_step_code(float R) {
    int c = __half_as_ushort(__float2half_rz(R * (1.0f / 15.0f))) >> 4;
    if (15.0f * kv4_step(c) < R) c++;
    if (15.0f * kv4_step(c) < R) c++;
    return c;
}

// 1/d to a unit or so in the last place: kv4_round needs no more.
__device__ __forceinline__ float kv4_inverse(float d) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return r;
}

// floor(x / d + 1/2), exactly: the product with 1/d, rounded to a whole number by
// the addition of 1.5 * 2^23, is at most one off, and the remainder x - n d of a
// value near a border is an fp32 number.
__device__ __forceinline__ float kv4_round(float x, float d, float inv) {
    float n = fmaf(x, inv, 12582912.0f) - 12582912.0f;
    const float r = fmaf(-n, d, x);
    if (r >= 0.5f * d) n += 1.0f;
    if (r < -0.5f * d) n -= 1.0f;
    return n;
}

// A whole number of 0 .. 15 as an integer.
__device__ __forceinline__ uint32_t kv4_whole(float n) { return __float_as_uint(n + 8388608.0f) & 15u; }

__device__ __forceinline__ float kv4_clean(float x, bool& bad) {
    if (!(fabsf(x) <= kKv4Limit)) {
        bad = true;
        return isnan(x) ? 0.0f : copysignf(kKv4Limit, x);
    }
    return x;
}

}  // namespace axq8
