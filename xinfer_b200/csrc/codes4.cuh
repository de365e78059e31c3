// Numbers held in 4 bits: groups of consecutive numbers x with a scale s and a least value m in bfloat16; a number is m + s * code.
//   lo, hi = the group's least and largest number,  s = bf16((hi - lo) / 15),  m = bf16(lo),  code = round((x - m) / s) within 0..15 (s = 0: 0)
// s and m are bfloat16 because they have float32's range (float16 would turn large keys into infinities): m's rounding moves the whole group by
// at most 2^-9 |lo| and s's the upper codes by at most 15 * 2^-9 s, both below the half step that the codes themselves are off.
// A group that holds an infinity, no number, or numbers whose spread float32 does not hold has s = m = NaN: all of it reads as NaN.
//
// A page of the cache holds `ps` tokens of one key/value head: for every group of 32 channels the codes of its slots, 16 bytes each (channel 2 i of
// the group in the low half of byte i, 2 i + 1 in the high half), then for every slot the words of its groups (s in the low 16 bits, m in the
// high ones).  Heads are padded to a whole group: 20 bytes for 32 channels.  Groups apart, so that eight slots' codes of a group are 128 bytes
// that ldmatrix takes without bank conflicts.
#pragma once
#include "common.cuh"

namespace xb4 {

constexpr int GROUP = 32;                 // channels of a group in the cache
constexpr int GROUP_BYTES = GROUP / 2;
constexpr int TILE_ROWS = 16, TILE_COLS = 128, TILE_CODES = TILE_ROWS * TILE_COLS / 2;      // a tile of a weight (linear4.cu)

__host__ __device__ constexpr int groups_of(int d) { return (d + GROUP - 1) / GROUP; }
__host__ __device__ constexpr int row_bytes(int d) { return groups_of(d) * (GROUP_BYTES + 4); }

__device__ __forceinline__ float scale_of(uint32_t word) { return __uint_as_float(word << 16); }
__device__ __forceinline__ float least_of(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }

// The larger and the smaller of two numbers; one that is no number wins.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// a / b by a reciprocal of b and one step of correction (Markstein: the remainder a - q b is exact, so what it adds rounds the quotient
// correctly): halves of whole numbers come out exactly.  `inv` may be off by a unit of its last place.
__device__ __forceinline__ float corrected(float a, float b, float inv) {
    const float q = a * inv;
    return fmaf(fmaf(-q, b, a), inv, q);
}
__device__ __forceinline__ float reciprocal(float s) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(s));
    return r;
}

// The group's word from its least and largest number.
__device__ __forceinline__ uint32_t word_of(float lo, float hi) {
    const __nv_bfloat16 s = __float2bfloat16_rn(corrected(hi - lo, 15.f, 1.f / 15.f)), m = __float2bfloat16_rn(lo);
    const uint32_t su = __bfloat16_as_ushort(s), mu = __bfloat16_as_ushort(m);
    return (su & 0x7f80u) == 0x7f80u || (mu & 0x7f80u) == 0x7f80u ? 0x7fff7fffu : su | (mu << 16);
}
// A number's code in a group of that scale and least value, plus 1.5 * 2^23, which rounds it to a whole number (halves to even) and leaves it in the
// lowest bits; `inv` is the scale's reciprocal.  Where the scale is zero or no number the quotient is no number, or none that counts, and the code is zero.
// Below TINY a scale's reciprocal, or a remainder, is no ordinary number: scale, least value and numbers are taken LIFT times their size then, which is exact.
constexpr float CODE_UP = 12582912.f, TINY = 0x1p-100f, LIFT = 0x1p100f;
__device__ __forceinline__ float raised_code(float x, float s, float m, float inv) { return fminf(fmaxf(corrected(x - m, s, inv), 0.f), 15.f) + CODE_UP; }
__device__ __forceinline__ float value_of(uint32_t code, uint32_t word) { return fmaf(scale_of(word), (float)code, least_of(word)); }

}  // namespace xb4
