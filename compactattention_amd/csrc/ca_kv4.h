// A KV cache held in 4 bits: the layout of a page and the conversions.
//
// Format.  The 128 dims of a token of one KV head are four groups of 32.  An element is an E2M1 code
// (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit), a group has a scale 2^(byte - 127): the operands of
// CDNA4's v_cvt_scalef32_pk_bf16_fp4, which turns a byte of codes and a scale into two bf16 values in
// one instruction at full rate.  Every value is exact in bf16.
//  - Scale: the power of two that brings the group's largest magnitude into (3.5, 7].  Up to 7 a value
//    rounds to 6 with an error of at most 1, as between 4 and 6.  With a the bits of that magnitude in
//    bf16, byte = ((a + 0x1f) >> 7) - 2: a mantissa above 1.75 carries into the exponent.  Bytes are
//    kept in [2, 252]: below, codes would stand for subnormal bf16 values, above for values beyond bf16
//    (what is larger saturates).
//  - Code: round to nearest, ties to the even code (v_cvt_scalef32_pk_fp4_bf16 rounds so).
//  - A group with an infinity or a NaN gets the byte 255 and is read as NaN.
//
// Page (64 tokens of one KV head, K or V): 4096 bytes of codes, then 256 scale bytes.
//  - K codes: token t at 64 t, dims in order, the lower dim in the low nibble.  16 bytes are a group, and
//    one lane's share of the A operand of S^T = K Q^T.
//  - V codes: dims 8 m .. 8 m + 7 of token t at 256 (t / 4) + 16 m + 4 (t % 4): 16 bytes hold 8 dims of
//    four tokens, one lane's share of the A operand of O^T = V^T P^T.
//  - Scale of group g of token t, from byte 4096 on: K at 64 g + 4 (t % 16) + t / 16, so that the four
//    tokens that a lane meets in a page are one word; V at 64 g + 16 (t % 16 / 4) + 4 (t / 16) + t % 4, so
//    that a lane's sixteen are 16 bytes.
#pragma once

#include "ca_common.h"

namespace ca {

constexpr int kPage4 = CA_PAGE4_BYTES;
constexpr int kPage4Scales = 4096;
constexpr uint32_t kScaleNan = 255;

typedef __bf16 bf16x2v_t __attribute__((ext_vector_type(2)));

struct Kv4Addr {
    uint8_t* data;
    int64_t stride;  // bytes from page to page
    const int32_t* page_table;
    int64_t pts;
    int32_t max_page;
};

__device__ __forceinline__ int k4_code(int t, int d) { return 64 * t + (d >> 1); }
__device__ __forceinline__ int v4_code(int t, int d) {
    return 256 * (t >> 2) + 16 * (d >> 3) + 4 * (t & 3) + ((d & 7) >> 1);
}
__device__ __forceinline__ int k4_scale(int t, int g) { return kPage4Scales + 64 * g + 4 * (t & 15) + (t >> 4); }
__device__ __forceinline__ int v4_scale(int t, int g) {
    return kPage4Scales + 64 * g + 16 * ((t & 15) >> 2) + 4 * (t >> 4) + (t & 3);
}

// The scale operand of the conversions from byte I of a word: they read the operand's exponent bits alone
// (all 256 exponents with 64 patterns in the other bits give the same values), so one shift will do.
template <int I>
__device__ __forceinline__ float scale_of(uint32_t word) {
    return __uint_as_float(I == 3 ? word >> 1 : word << (23 - 8 * I));
}
__device__ __forceinline__ float scale_of(uint32_t word, int i) {  // i a constant after unrolling
    return __uint_as_float(i == 3 ? word >> 1 : word << (23 - 8 * i));
}
// Two values of byte I of a word of codes, bf16 (the lower dim in the low half).
template <int I>
__device__ __forceinline__ uint32_t decode2(uint32_t word, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, I));
}

// The scale byte of a group whose largest bf16 magnitude has the bits a.
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
    if (a >= 0x7f80u) return kScaleNan;
    const int e = static_cast<int>((a + 0x1fu) >> 7) - 2;
    return static_cast<uint32_t>(min(max(e, 2), 252));
}

}  // namespace ca
