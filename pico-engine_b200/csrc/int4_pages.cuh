// How keys and values lie in a page of 4-bit codes, and the arithmetic of the codes.
//
// A head's row of D channels (64 or 128) is cut into groups of 32 channels.  Of a group with largest and smallest number max and min (bfloat16)
//   mid = (max + min) / 2, step = (max - min) / 15, both rounded to bfloat16;  level L = floor((x - mid) / step), between -8 and 7 (0 where step is 0)
// and x is held as the 4 bits of L: it stands for mid + step * (L + 1/2).  5 bits a channel with step and mid.  A group with a number that is none
// (an infinity, NaN, or a sum or spread that float32 or bfloat16 does not hold) has step = mid = NaN.
//
// A block holds the 64 positions of one page and one head, 80 D bytes:
//   [0, 32 D)     codes of the keys: position p, part t (4), group b: one word of the channels 32 b + 8 t + 2 i + e (i of 4, e of 2)
//   [32 D, 64 D)  codes of the values: tile of 16 positions, half h of the groups (D / 64), g (8), t (4), w (4): with m = 4 h + w one word of the
//                 positions 16 tile + 8 f + 2 t + e and the channels 32 (m / 2) + 4 g + 2 (m % 2) + n, i = 2 f + n
//   [64 D, 72 D)  of the keys' groups: position p: step of every group, then mid of every group
//   [72 D, 80 D)  of the values' groups: tile, then step and mid, group b, and the 16 positions as t, f, e
// In a word the element (i, e) has its sign in bit 15 + 16 e and a magnitude of three bits k in bits 4..6 + 16 e, all turned left by 4 i: k = L for L >= 0,
// k = -1 - L below.  Turned back, masked and with bits 3 and 19 set, a word is a pair of bfloat16 numbers +-(k + 1/2) 2^-129: operands of a product on the
// tensor cores as they stand (which keep subnormal operands), two instructions a pair, with no conversion and no offset to take off afterwards.
// The words are in the order of the fragments of mma.sync m16n8k16, keys as rows and channels as rows, so that a warp reads them 16 or 8 bytes a thread.
#pragma once
#include "common.cuh"

template <int D>
struct Int4Block {
    static constexpr int groups = D / 32, halves = D / 64, key_words = D / 8;
    static constexpr int values = 32 * D, key_meta = 64 * D, value_meta = 72 * D, bytes = 80 * D;
    static constexpr int tile_bytes = 8 * D;                   // the values' codes of 16 positions
};

#define Q4_MASK 0x80708070u
#define Q4_HALF 0x00080008u

// elements (i, 0) and (i, 1) of a word as two bfloat16 numbers, in units of 2^-129
__device__ __forceinline__ unsigned q4_pair(unsigned word, int i) {
    unsigned r;                                                // (one instruction; written as operators it becomes two)
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(__funnelshift_r(word, word, 4 * i)), "r"(Q4_MASK), "r"(Q4_HALF));
    return r;
}
// the level + 1/2 of element (i, e)
__device__ __forceinline__ float q4_level(unsigned word, int i, int e) {
    const unsigned r = __funnelshift_r(word, word, 4 * i) >> (16 * e);
    const float k = (float)((r >> 4) & 7u) + 0.5f;
    return (r & 0x8000u) ? -k : k;
}
// the 16 bits of a level, for element (i, e): field << 16 e, turned left by 4 i
__device__ __forceinline__ unsigned q4_field(int level) { return ((unsigned)level & 0x8000u) | (unsigned)((level ^ (level >> 31)) << 4); }
__device__ __forceinline__ unsigned q4_turn(unsigned pair, int i) { return __funnelshift_l(pair, pair, 4 * i); }
// the bits of a values' word that belong to its position (f, e): elements i = 2 f and 2 f + 1
__device__ __forceinline__ unsigned q4_position_bits(int f, int e) {
    const unsigned own = 0x8070u << (16 * e);
    return q4_turn(own, 2 * f) | q4_turn(own, 2 * f + 1);
}

__device__ __forceinline__ float q4_min(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float q4_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// step and mid of a group from its largest and smallest number
__device__ __forceinline__ void q4_scale(float lo, float hi, bf16& step, bf16& mid) {
    const float m = __bfloat162float(__float2bfloat16_rn((hi + lo) * 0.5f)), s = __bfloat162float(__float2bfloat16_rn((hi - lo) / 15.f));
    const bool none = !(fabsf(m) < INFINITY) || !(s < INFINITY);
    mid = none ? __ushort_as_bfloat16(0x7fffu) : __float2bfloat16_rn(m);
    step = none ? __ushort_as_bfloat16(0x7fffu) : __float2bfloat16_rn(s);
}
// What numbers, middle and step of a group are multiplied by before they meet: a power of two with which the step has a reciprocal in float32 (subnormal ones do not), or 0 for a step of 0,
// whose levels are 0 then.  (A number is less than 2^12 steps in size, where the step is none of the smallest of all: numbers have 8 bits.)
__device__ __forceinline__ float q4_up(float step) { return step == 0.f ? 0.f : step < 5.421010862427522e-20f ? 18446744073709551616.f : 1.f; }
// floor((x - mid) / step) within the levels; `by`: 1 / step (0 for a step of 0).  The quotient is rounded to the nearest integer n through its last bits, and is one less where x lies below
// mid + n step.  That is a float32 without rounding: where they are not 0, 2^-12 < step / mid < 2^7, since numbers have 8 bits, and n has 4.  (x - mid, which float32 rounds where x is far
// smaller than mid, would not tell the side.)
__device__ __forceinline__ int q4_quantise(float x, float step, float mid, float by) {
    const float r = __fmaf_rn(x - mid, by, 12582912.f), n = r - 12582912.f;
    const int l = __float_as_int(r) - 0x4b400000 - (x < __fmaf_rn(n, step, mid) ? 1 : 0);
    return min(max(l, -8), 7);
}

// byte offsets within a block
template <int D> __device__ __forceinline__ int q4_key_word(int p, int b, int t) { return (p * Int4Block<D>::key_words + t * Int4Block<D>::groups + b) * 4; }
template <int D> __device__ __forceinline__ int q4_value_words(int tile, int h, int g, int t) { return Int4Block<D>::values + ((tile * Int4Block<D>::halves + h) * 32 + g * 4 + t) * 16; }
template <int D> __device__ __forceinline__ int q4_key_step(int p, int b) { return Int4Block<D>::key_meta + (p * 2 * Int4Block<D>::groups + b) * 2; }
template <int D> __device__ __forceinline__ int q4_value_step(int p, int b) {
    const int tile = p >> 4, r = p & 15;
    return Int4Block<D>::value_meta + ((tile * 2 * Int4Block<D>::groups + b) * 16 + ((r & 7) >> 1) * 4 + (r >> 3) * 2 + (r & 1)) * 2;
}
