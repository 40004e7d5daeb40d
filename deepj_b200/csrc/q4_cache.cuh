// The 4-bit K/V cache: its layout in memory and the quantization of a row, shared by the kernels that fill it, read it and move its rows.
//
// A row (the key or the value of one position and key/value head) of hd = 32·NB values is NB blocks of 32: a bf16 scale
//     s = bf16(max|w| · fp32(1/7)), at least 2^-17 and at most 2^13; 0 where the block is all zeros
// and 32 codes clamp(round_half_even(w / s), -7, 7), NaN → 0.  A code has 3 bits and a sign, s has 8 bits: code · s is exact in fp16 over the whole
// range of s, which is what lets the tensor cores multiply stored values without a correction term.
// Rows lie in pages of 32 consecutive positions, 1152·NB contiguous bytes that one bulk copy brings:
//     K codes [32][16·NB] | K scales [32][NB] bf16 | V codes [32][16·NB] | V scales [32][NB] bf16
// Word (t, j) of a row, t < 4, j < NB, holds the codes as two's complement nibbles: byte i the dims 32j + 4t + i (low) and 32j + 16 + 4t + i (high).
// Masked, a word gives two int8 operand registers of m16n8k32 whose bytes are 16 times the codes.  The words of one t are a piece of 4·NB bytes; piece t of row r sits in slot t ^ (r/2 % 4): with
// rows of 64 bytes the warp that reads one piece of four consecutive rows finds them in different banks.
#pragma once
#include <cuda_bf16.h>

#include "q8_common.cuh"

namespace dj {

constexpr int kQ4Page = 32;
constexpr int kQ4PageBytes = 1152;               // … times NB
constexpr float kQ4ScaleMin = 1.0f / 131072.0f, kQ4ScaleMax = 8192.0f;

template <int NB> struct Q4Page {
    static constexpr int kBytes = kQ4PageBytes * NB, kHalf = kBytes / 2, kRow = 16 * NB;
    static constexpr int kKs = kQ4Page * kRow, kV = kHalf, kVs = kV + kKs;                     // offsets of the scales and of the V half
    static __device__ __forceinline__ int word(int row, int t, int j) { return row * kRow + (t ^ ((row >> 1) & 3)) * (4 * NB) + 4 * j; }
};

// A length, position or place, which travel as floats: -1 for what is below 0 or no number, so that differences of two never leave 32 bits.
__device__ __forceinline__ int q4_int(float x) { return x >= 0.0f ? (int)x : -1; }
// Rows starts[b] … starts[b + 1] - 1 of the M packed rows: the first one, and how many.
__device__ __forceinline__ int q4_rows(float start, float next, int M, int& first) {
    first = min(max(q4_int(start), 0), M);
    return max(0, min(q4_int(next), M) - first);
}
// Rows that a sequence has room for and positions that its tables have, of `tokens` new ones: 0 for a length or position outside its range.
__device__ __forceinline__ int q4_room(int tokens, int len, int maxSeq, int pos, int maxPos) {
    if (len < 0 || len >= maxSeq || pos < 0 || pos >= maxPos) return 0;
    return max(0, min(tokens, min(maxSeq - len, maxPos - pos)));
}

// The scale of a block whose largest magnitude is `most` (of the values that are no NaN).
__device__ __forceinline__ float q4_scale(float most) { return fminf(fmaxf(__bfloat162float(__float2bfloat16_rn(most * (1.0f / 7.0f))), kQ4ScaleMin), kQ4ScaleMax); }
__device__ __forceinline__ float q4_most(const float4& x) { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))); }
// Four values' codes in the low nibbles of a word's bytes.  The code is the rounded quotient; a product with the reciprocal is within 2e-6 of it, so only
// values that close to the middle of two codes need the division (2048 rows of 64 × 128, with the rotation: 33 µs dividing all).  The sum with 1.5 · 2^23
// ends in the rounded quotient, in two's complement.  off: raised to the largest distance from a whole number.
__device__ __forceinline__ uint32_t q4_near(const float4& x, float inverse, float& off) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float q = v[i] * inverse, sum = q + 12582912.0f;
        off = fmaxf(off, fabsf(q - (sum - 12582912.0f)));
        codes |= ((uint32_t)__float_as_int(sum) & 15u) << (8 * i);
    }
    return codes;
}
__device__ __forceinline__ uint32_t q4_divided(const float4& x, float s) {
    auto code = [](float v) { return (uint32_t)min(max(__float2int_rn(v), -7), 7) & 15u; };     // NaN → 0
    return code(x.x / s) | code(x.y / s) << 8 | code(x.z / s) << 16 | code(x.w / s) << 24;
}

// 8·NB consecutive lanes (all lanes of the warp are here) put one row into its page: lane e of them holds the values 4e … 4e + 3.
template <int NB>
__device__ __forceinline__ void q4_put_row(unsigned char* page, int row, bool value, int e, const float4& x, bool on) {
    float most = q4_most(x);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    most = most == most ? most : 0.0f;
    const float s = q4_scale(most);
    float off = 0.0f;
    uint32_t mine = q4_near(x, __frcp_rn(s), off);
    const float all = (x.x + x.y) + (x.z + x.w);  // blocks that saturate, NaN and infinities are divided too
    if (__any_sync(0xffffffffu, off > 0.4999f || most > 7.0f * kQ4ScaleMax || all != all)) mine = q4_divided(x, s);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 4);
    if (!on) return;
    const int j = e >> 3, t = e & 3;
    if ((e & 4) == 0) *reinterpret_cast<uint32_t*>(page + (value ? Q4Page<NB>::kV : 0) + Q4Page<NB>::word(row, t, j)) = mine | other << 4;
    if ((e & 7) == 0) *reinterpret_cast<__nv_bfloat16*>(page + (value ? Q4Page<NB>::kVs : Q4Page<NB>::kKs) + (row * NB + j) * 2) = __float2bfloat16_rn(most > 0.0f ? s : 0.0f);
}
// 4·NB lanes: lane f holds the values 32j + 4t … + 3 (x) and 16 values on (y), j = f / 4, t = f % 4: a word of the page.
template <int NB>
__device__ __forceinline__ void q4_put_words(unsigned char* page, int row, bool value, int f, const float4& x, const float4& y, bool on) {
    float most = fmaxf(q4_most(x), q4_most(y));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    most = most == most ? most : 0.0f;
    const float s = q4_scale(most), inverse = __frcp_rn(s);
    float off = 0.0f;
    uint32_t word = q4_near(x, inverse, off);
    word |= q4_near(y, inverse, off) << 4;
    const float all = ((x.x + x.y) + (x.z + x.w)) + ((y.x + y.y) + (y.z + y.w));
    if (__any_sync(0xffffffffu, off > 0.4999f || most > 7.0f * kQ4ScaleMax || all != all)) word = q4_divided(x, s) | q4_divided(y, s) << 4;
    if (!on) return;
    const int j = f >> 2, t = f & 3;
    unsigned char* const half = page + (value ? Q4Page<NB>::kV : 0);
    *reinterpret_cast<uint32_t*>(half + Q4Page<NB>::word(row, t, j)) = word;
    if (t == 0) *reinterpret_cast<__nv_bfloat16*>(half + Q4Page<NB>::kKs + (row * NB + j) * 2) = __float2bfloat16_rn(most > 0.0f ? s : 0.0f);
}

// interleaved pairs (x0, x1) → (x0·c − x1·s, x0·s + x1·c), every product and sum rounded (RotaryEmbedding.java:81-122)
__device__ __forceinline__ float4 q4_rotate(const float4& x, const float2& c, const float2& s) {
    return make_float4(x.x * c.x - x.y * s.x, x.x * s.x + x.y * c.x, x.z * c.y - x.w * s.y, x.z * s.y + x.w * c.y);
}

// A word's codes in the high (low: shifted there) nibbles of its bytes: int8 values of 16 times the code.
__device__ __forceinline__ uint32_t q4_high(uint32_t w) { return w & 0xf0f0f0f0u; }
__device__ __forceinline__ uint32_t q4_low(uint32_t w) { return (w << 4) & 0xf0f0f0f0u; }
// one code of a word: bit 0 of its nibble is at `shift`
__device__ __forceinline__ int q4_code(uint32_t w, int shift) { return (int)(w << (28 - shift)) >> 28; }

}  // namespace dj
