// Matrix instructions over fragments of rows as they lie in memory.
//
// A Frag is a lane's share of an operand of 16 lines (rows of one operand, columns of the other): line lane % 16, of a step's values the
// run quarter lane / 16.  Both operands hold the contraction in one order, which is all that a product needs; what it leaves is the usual
// accumulator: column lane % 16, rows 4 (lane / 16) + i.
#pragma once

#include "nvq_device.h"

namespace nvq {
namespace {

typedef float acc4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

// Values of a line that a lane holds, and those of a whole step.
template <typename T> constexpr int kFragRun = 16 / (int)sizeof(T);
template <typename T> constexpr int kFragStep = 4 * kFragRun<T>;

template <typename T>
__device__ __forceinline__ acc4_t product16(uint4 a, uint4 b, acc4_t c) {
    if constexpr (Elem<T>::code == NVQ_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else if constexpr (Elem<T>::code == NVQ_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(a.x), u2f(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(a.y), u2f(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(a.z), u2f(b.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(a.w), u2f(b.w), c, 0, 0, 0);
    }
}

// The run of values at p, at any address, of which `left` lie in the line; zeros behind them.
template <typename T>
__device__ __forceinline__ uint4 load_run(const T *p) {
    struct __attribute__((packed)) Run { uint32_t w[4]; };
    const Run r = *reinterpret_cast<const Run *>(p);
    return make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
}
template <typename T>
__device__ __forceinline__ uint4 load_run(const T *p, int64_t left) {
    if (left >= kFragRun<T>) return load_run(p);
    T t[kFragRun<T>];
#pragma unroll
    for (int i = 0; i < kFragRun<T>; i++) {
        Elem<T>::store(t, i, 0.0f);
        if (i < left) t[i] = p[i];
    }
    uint4 w;
    __builtin_memcpy(&w, t, 16);
    return w;
}

}  // namespace
}  // namespace nvq
