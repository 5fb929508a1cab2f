// Eight consecutive values of a head a lane: loads and stores, the norm over a head, the rotation of its positions, the affine
// codes of its groups.  P lanes (a power of two, 8 .. 64) hold a head of at most 8 P values.
#pragma once

#include "nvq_device.h"

namespace nvq {
namespace {

constexpr int kHeadBlock = 256;

template <typename T>
__device__ __forceinline__ void store_run(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 w;
        if constexpr (Elem<T>::code == NVQ_BF16) {
            w = make_uint4(f32_to_bf16_pair(v[0], v[1]), f32_to_bf16_pair(v[2], v[3]), f32_to_bf16_pair(v[4], v[5]), f32_to_bf16_pair(v[6], v[7]));
        } else {
            T t[8];
#pragma unroll
            for (int i = 0; i < 8; i++) Elem<T>::store(t, i, v[i]);
            __builtin_memcpy(&w, t, 16);
        }
        *reinterpret_cast<uint4 *>(p) = w;
    }
}

// Values across the lanes of a head.  Within 16 lanes by data-parallel moves: pairs, quads, then mirrors, which meet another quad or
// half each time, so that after a step all lanes that have met hold the same bits (addition and the extremes commute).
template <int CTRL> __device__ __forceinline__ float moved(float v) {
    return u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL> __device__ __forceinline__ double moved(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}
constexpr int kPairs = 0xB1, kQuads = 0x4E, kHalfRow = 0x141, kRow = 0x140;
template <int LANES, typename V, typename F>
__device__ __forceinline__ V across(V v, F f) {
    v = f(v, moved<kPairs>(v));
    v = f(v, moved<kQuads>(v));
    if constexpr (LANES >= 8) v = f(v, moved<kHalfRow>(v));
    if constexpr (LANES >= 16) v = f(v, moved<kRow>(v));
    if constexpr (LANES >= 32) v = f(v, __shfl_xor(v, 16));
    if constexpr (LANES >= 64) v = f(v, __shfl_xor(v, 32));
    return v;
}

// 1 / sqrt(mean of squares + eps) of the head whose values lie in P lanes, 0 where a lane has none.  The sum is 64 bits wide and so
// the factor is the correctly rounded one for any order of the sum: a cache's codes turn over on its last bit.
template <int P>
__device__ __forceinline__ float norm_factor(const float (&v)[8], int dim, double eps) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) sum = __builtin_fma((double)v[i], (double)v[i], sum);
    sum = across<P>(sum, [](double a, double b) { return a + b; });
    const double x = sum / (double)dim + eps;
    double y = __builtin_amdgcn_rsq(x);  // (half its digits; each step doubles them)
#pragma unroll
    for (int i = 0; i < 2; i++) y = y * __builtin_fma(-0.5 * x * y, y, 1.5);
    return x == (double)INFINITY ? 0.0f : (float)y;  // (the steps make infinity x 0 of it)
}

// Which values of a head the rotation turns and with which others, for the lane's run of eight.
struct Turn {
    float c[8], n[8];  // cosine, and sine with the sign of the partner's share; 1 and 0 where nothing turns
};
// How a lane's run of eight is read.  kWhole: whole runs turn or stay, and their partners are one run (half layout) or in the same run
// (interleaved).  kRuns: runs as such, their partners, which lie across two runs, through LDS.  kSingle: value by value.  (4096 positions of 32 heads of
// 128, bfloat16, 64 values rotated as kWhole 13.0 us; 50 rotated as kRuns 15.0, value by value 41.8.)
enum { kSingle, kRuns, kWhole };

template <int READ>
__device__ __forceinline__ Turn read_turn(const float2 *__restrict__ angles, int j0, int half, bool interleaved) {
    Turn t;
    if (READ == kWhole) {
        const bool turns = j0 < 2 * half, second = !interleaved && j0 >= half;
        if (turns) {
            if (interleaved) {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float4 a = *reinterpret_cast<const float4 *>(angles + (j0 >> 1) + i);
                    t.c[2 * i] = t.c[2 * i + 1] = a.x, t.n[2 * i] = -a.y, t.n[2 * i + 1] = a.y;
                    t.c[2 * i + 2] = t.c[2 * i + 3] = a.z, t.n[2 * i + 2] = -a.w, t.n[2 * i + 3] = a.w;
                }
            } else {
                const float2 *from = angles + (second ? j0 - half : j0);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float4 a = *reinterpret_cast<const float4 *>(from + i);
                    t.c[i] = a.x, t.n[i] = second ? a.y : -a.y;
                    t.c[i + 1] = a.z, t.n[i + 1] = second ? a.w : -a.w;
                }
            }
            return t;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) t.c[i] = 1.0f, t.n[i] = 0.0f;
        return t;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int j = j0 + i;
        t.c[i] = 1.0f, t.n[i] = 0.0f;
        if (j < 2 * half) {
            const float2 a = angles[interleaved ? j >> 1 : j < half ? j : j - half];
            const bool second = interleaved ? (j & 1) != 0 : j >= half;
            t.c[i] = a.x, t.n[i] = second ? a.y : -a.y;
        }
    }
    return t;
}

// The lane's values of a head and those that the rotation mixes into them, as they lie in memory: a head's are requested before the one in front of it is
// worked on.
template <typename T, int READ>
struct HeadRaw {
    T v[8], p[8];
    __device__ __forceinline__ void load(const T *row, int j0, int dim, int half, bool interleaved) {
        if (READ != kSingle) {
            struct alignas(16) Run { T t[8]; };
            if (j0 < dim) {
                __builtin_memcpy(v, reinterpret_cast<const Run *>(row + j0), sizeof(Run));
                if (READ == kWhole && !interleaved && j0 < 2 * half) __builtin_memcpy(p, reinterpret_cast<const Run *>(row + (j0 < half ? j0 + half : j0 - half)), sizeof(Run));
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = j0 + i;
            if (j < dim) v[i] = row[j];
            if (j < 2 * half) p[i] = row[interleaved ? j ^ 1 : j < half ? j + half : j - half];
        }
    }
};
// kRuns: the heads that a block's lanes hold, eight values' room around each; a head's lanes are of one wavefront, whose LDS operations are in order.
template <typename T, int P, int READ> constexpr int kHeldHeads = READ == kRuns ? kHeadBlock / P : 1;
template <typename T, int P, int READ>
struct HeldHeads {
    struct alignas(16) Run { T t[8]; };
    Run runs[kHeldHeads<T, P, READ>][P + 2];
};
template <typename T, int READ>
struct HeadRun {
    float v[8], p[8];
    template <int FROM>
    __device__ __forceinline__ explicit HeadRun(const HeadRaw<T, FROM> &raw) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = Elem<T>::load(raw.v, i), p[i] = Elem<T>::load(raw.p, i);
    }
    // kRuns, half layout: the partners, `half` values further or before, from the other lanes of the head.
    template <int P>
    __device__ __forceinline__ void meet(const HeadRaw<T, READ> &raw, HeldHeads<T, P, READ> &held, int half) {
        struct __attribute__((packed)) Any { T t[8]; };
        auto &head = held.runs[threadIdx.x / P];
        const int lane = threadIdx.x % P, j0 = 8 * lane;
        __builtin_memcpy(&head[1 + lane], raw.v, sizeof(head[0]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const T *at = head[1].t;
        const int further = j0 + half < 8 * P ? j0 + half : 8 * P, before = j0 - half > -8 ? j0 - half : -8;  // (in the room around: of no use)
        const Any a = *reinterpret_cast<const Any *>(at + further), b = *reinterpret_cast<const Any *>(at + before);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = j0 + i < half ? Elem<T>::load(a.t, i) : Elem<T>::load(b.t, i);
    }
    // times the factor and the weight: two roundings in float32, those of the partners likewise
    __device__ __forceinline__ void scale(float r, const HeadRun &w) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = v[i] * r * w.v[i], p[i] = p[i] * r * w.p[i];
    }
    __device__ __forceinline__ void turn(const Turn &t, int j0, int half, bool interleaved) {
        if (j0 >= 2 * half) return;  // (nothing of this run; not times 1 plus times 0, which an infinite partner would spoil)
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float other = READ != kSingle && interleaved ? v[i ^ 1] : p[i];
            const float turned = v[i] * t.c[i] + other * t.n[i];
            y[i] = READ == kWhole || j0 + i < 2 * half ? turned : v[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = y[i];
    }
};

// How heads are read whose rows are 16-byte aligned where `aligned`, and their weights and the table of angles where `all_aligned`.
inline int read_of(int dim, int half, bool interleaved, bool aligned, bool all_aligned) {
    if (dim % 8 != 0 || !aligned) return kSingle;
    return all_aligned && (interleaved ? half % 4 == 0 : half % 8 == 0) ? kWhole : kRuns;
}

}  // namespace
}  // namespace nvq
