// Codes of a quantized cache as operands of the bfloat16 matrix instructions, and float32 values as sums of bfloat16 terms.
#pragma once

#include "nvq_device.h"
#include "qmf_kernel.h"

namespace nvq {
namespace {

typedef float floatx4_t __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ floatx4_t mfma16(uint4 a, uint4 b, floatx4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qmf::bf16x8_t, a), __builtin_bit_cast(qmf::bf16x8_t, b), c, 0, 0, 0);
}

// A value from any address, in as few loads as it has dwords.
template <typename V>
__device__ __forceinline__ V load_any(const void *p) {
    struct __attribute__((packed)) Raw { uint8_t b[sizeof(V)]; };
    return __builtin_bit_cast(V, *reinterpret_cast<const Raw *>(p));
}

// An operand is kOffset + code.  WIDE: float32.
template <int BITS, bool WIDE> constexpr float kOffset = WIDE ? -(float)(1 << (BITS - 1)) : BITS == 8 ? 0.0f : (float)(1 << BITS);
template <int BITS> constexpr uint32_t kMagic = BITS == 4 ? 0x41804180u : 0x41004100u;  // two of 2^BITS, BITS < 8
// Codes at bit `at` of both halves of a word as 2^BITS + code.  The constants come in registers, a scalar one and a vector one: then the
// mask and the exponent are one instruction (v_and_or_b32, which takes no literal; from constants they were two).
template <int BITS>
struct CodeConstants {
    uint32_t mask = ((1u << BITS) - 1u) * 0x00010001u << (BITS < 7 ? 7 - BITS : 0), magic = kMagic<BITS>;
    __device__ __forceinline__ CodeConstants() {
        asm("" : "+s"(mask));
        asm("" : "+v"(magic));
    }
};
template <int BITS>
__device__ __forceinline__ uint32_t two_codes(const CodeConstants<BITS> &c, uint32_t z, int at) {
    constexpr int to = 7 - BITS;  // the code's place in the mantissa
    return ((at >= to ? z >> (at - to) : z << (to - at)) & c.mask) | c.magic;
}

// Two exact bfloat16 values from two floats that bfloat16 holds.
__device__ __forceinline__ uint32_t pack_exact(float lo, float hi) { return __builtin_amdgcn_perm(f2u(hi), f2u(lo), 0x07060302u); }

// Which of eight consecutive codes element j of an operand is.
template <int BITS> constexpr int code_at(int j) { return BITS == 8 ? j : (j >> 1) + 4 * (j & 1); }

// Eight consecutive codes of a row (BITS bytes in the low bits of w0, w1) as an operand, in the order of code_at.
template <int BITS, bool WIDE>
__device__ __forceinline__ uint4 eight_codes(const CodeConstants<BITS> &c, uint32_t w0, uint32_t w1) {
    if constexpr (WIDE) {
        auto at = [&](int j) {
            const int i = code_at<BITS>(j);
            const uint32_t code = BITS == 8 ? (i < 4 ? w0 >> (8 * i) : w1 >> (8 * (i - 4))) & 0xFFu : (w0 >> (BITS * i)) & ((1u << BITS) - 1u);
            return (float)code + kOffset<BITS, true>;
        };
        return make_uint4(pack_exact(at(0), at(1)), pack_exact(at(2), at(3)), pack_exact(at(4), at(5)), pack_exact(at(6), at(7)));
    } else if constexpr (BITS == 8) {
        return make_uint4(pack_exact(qmf::ubyte_to_float<0>(w0), qmf::ubyte_to_float<1>(w0)), pack_exact(qmf::ubyte_to_float<2>(w0), qmf::ubyte_to_float<3>(w0)),
                          pack_exact(qmf::ubyte_to_float<0>(w1), qmf::ubyte_to_float<1>(w1)), pack_exact(qmf::ubyte_to_float<2>(w1), qmf::ubyte_to_float<3>(w1)));
    } else {
        const uint32_t z = BITS == 4 ? w0 : (w0 & 0xFFFu) | ((w0 & 0xFFF000u) << 4);  // code i at bit BITS i, code i + 4 sixteen above
        return make_uint4(two_codes(c, z, 0), two_codes(c, z, BITS), two_codes(c, z, 2 * BITS), two_codes(c, z, 3 * BITS));
    }
}

// A float as a sum of N bfloat16 terms (8 bits each), two floats at a time: term i of both in t[i].
template <int N>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&t)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        t[i] = f32_to_bf16_pair(a, b);
        a -= u2f(t[i] << 16), b -= u2f(t[i] & 0xFFFF0000u);
    }
}

}  // namespace
}  // namespace nvq
