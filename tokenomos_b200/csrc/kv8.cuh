// The 8-bit cache of keys and values: pages [pages, 2 (K|V), Hkv, P, D] of e4m3 bytes and one scale per (page, K|V, head),
// [pages, 2, Hkv] float32, always a power of two between 2^-40 and 2^40. A byte b of such a block stands for s * e4m3(b).
//
// Why powers of two: e4m3 keeps its relative precision over 2^-6 .. 448, so a finer scale buys nothing but the last bit of that
// range, while with a power of two (1) a block whose scale has to grow as tokens join it is rescaled without a second
// rounding (but for bytes at or below 2^-6, e4m3's smallest normal number, under the new scale), and (2) the scale joins the attention's exponents as an addend.
// Why bounded: the attention folds a value block's scale into its softmax weights in base-2 logarithms, and 2^+-40 leaves
// a weight 46 bits before the 32-bit exponent runs out. 448 * 2^40 = 4.9e14 is the largest magnitude the cache takes.
//
// A token one of whose keys or values (of one head) is not finite, or beyond that magnitude, is marked: its key is stored as
// NaN and its value as 0. Queries that see it get NaN from its score; queries that do not see it never multiply a NaN.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int KV8_EXP_MIN = -40, KV8_EXP_MAX = 40;
constexpr float KV8_MOST = 448.0f * 1099511627776.0f;       // 448 * 2^40

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }       // -126 <= e <= 127

// two e4m3 bytes (the low one first) as half2, exactly
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}

// two values as e4m3 bytes, `lo` in the low one, to the nearest (ties to even)
__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// The exponent of the smallest power of two s with most / s <= 448 = 1.75 * 2^8.
__device__ __forceinline__ int kv8_exponent(float most) {
    const int bits = __float_as_int(most);
    const int e = (bits >> 23) - 127 - ((bits & 0x7fffff) <= 0x600000 ? 8 : 7);
    return min(max(e, KV8_EXP_MIN), KV8_EXP_MAX);
}

}  // namespace
