// The choice of experts from a router's logits: of a row l of them
//     p = softmax(l) or sigmoid(l),  c = p + bias,
// a group's score is the sum of its one or two largest c, the best groups stay, the k largest c of their experts are chosen, and their
// weights are p, divided by (their sum + 1e-20) where asked, times a scale.
//
// What is chosen is decided on 64 bits: two values of c that float32 makes one, or turns round, are an expert of difference.  Without a bias
// (and groups by their best alone) c's order is the logits', and nothing is computed to find it.  Values are compared as whole numbers of the
// same order, 0 for what is not to be chosen, 1 for a NaN.
//
// One wavefront a row, a lane holding V consecutive experts; the maximum over the lanes by data-parallel moves, its place by a ballot.
#include "heads.h"
#include "nvq_internal.h"
#include "wave_reduce.h"

namespace nvq {
namespace {

constexpr int kSelectWaves = 4;

struct SelectArgs {
    const void *logits;
    const float *bias;
    int32_t *indices;
    void *weights;
    int64_t rows;
    int32_t experts, k, groups, top_groups, group_best, normalize, sigmoid;
    double scale;
};

// The larger of own and moved whole numbers; 0 from lanes that feed nothing.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t larger(uint32_t v) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
    return v > other ? v : other;
}
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
    v = larger<0x111, 0xF>(v);
    v = larger<0x112, 0xF>(v);
    v = larger<0x114, 0xF>(v);
    v = larger<0x118, 0xF>(v);
    v = larger<0x142, 0xA>(v);
    v = larger<0x143, 0xC>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Whole numbers in the values' order, above 1; a NaN is 1.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = f2u(v + 0.0f);  // (-0 is 0)
    return v != v ? 1u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return v != v ? 1u : b >> 63 ? ~b : b | 1ull << 63;
}

__device__ __forceinline__ double from_lane(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}

// WIDE: c is computed, and compared in 64 bits; else the logits are compared.
template <typename T, int V, bool WIDE>
__global__ void __launch_bounds__(64 * kSelectWaves) moe_select_kernel(const SelectArgs a) {
    __shared__ double held[WIDE ? kSelectWaves : 1][WIDE ? 64 * V : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * kSelectWaves + wave;
    if (row >= a.rows) return;
    const int n = a.experts, first = lane * V;
    const T *logits = (const T *)a.logits + row * n;
    float l[V];
    if (n % V == 0 && first < n) {
        struct __attribute__((packed)) Run { T t[V]; };
        const Run run = *reinterpret_cast<const Run *>(logits + first);
#pragma unroll
        for (int j = 0; j < V; j++) l[j] = Elem<T>::load(run.t, j);
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) l[j] = first + j < n ? Elem<T>::load(logits, first + j) : 0.0f;
    }
    // p = e / total
    double e[V], total = 1.0;
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < V; j++) e[j] = 1.0 / (1.0 + exp(-(double)l[j]));
    } else {
        float top = -INFINITY;
        bool wild = false;
#pragma unroll
        for (int j = 0; j < V; j++)
            if (first + j < n) top = fmaxf(top, l[j]), wild |= l[j] != l[j];
        top = across<64>(top, [](float x, float y) { return fmaxf(x, y); });
        const bool none = top == -INFINITY && !__any(wild);  // (a row of -inf alone: zeros)
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; j++) {
            e[j] = none ? 0.0 : exp((double)l[j] - (double)top);
            if (first + j < n) sum += e[j];
        }
        sum = across<64>(sum, [](double x, double y) { return x + y; });
        total = none ? 1.0 : sum;
#pragma unroll
        for (int j = 0; j < V; j++) e[j] = e[j] / total;
    }
    uint32_t hi[V], lo[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const bool real = first + j < n;
        if (WIDE) {
            const double c = a.bias != nullptr && real ? e[j] + (double)a.bias[first + j] : e[j];
            const uint64_t b = real ? ordered(c) : 0;
            hi[j] = (uint32_t)(b >> 32), lo[j] = (uint32_t)b;
            held[wave][first + j] = c != c ? -INFINITY : c;
        } else {
            hi[j] = real ? ordered(l[j]) : 0, lo[j] = 0;
        }
    }
    if (a.groups > 1) {
        const int each = n / a.groups;
        uint32_t group_hi = 0, group_lo = 0;
        if constexpr (WIDE) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (lane < a.groups) {
                double best = -INFINITY, second = -INFINITY;
                for (int i = 0; i < each; i++) {
                    const double c = held[wave][lane * each + i];
                    second = c > best ? best : c > second ? c : second, best = c > best ? c : best;
                }
                const uint64_t b = ordered(a.group_best == 2 && each > 1 ? best + second : best);
                group_hi = (uint32_t)(b >> 32), group_lo = (uint32_t)b;
            }
        } else {
            for (int g = 0; g < a.groups; g++) {
                uint32_t best = 0;
#pragma unroll
                for (int j = 0; j < V; j++) best = (first + j) / each == g && hi[j] > best ? hi[j] : best;
                best = wave_largest(best);
                if (lane == g) group_hi = best;
            }
        }
        uint64_t kept = 0;
        for (int i = 0; i < a.top_groups; i++) {
            const uint32_t h = wave_largest(group_hi), w = WIDE ? wave_largest(group_hi == h ? group_lo : 0) : 0;
            const int at = __builtin_ctzll(__ballot(group_hi == h && group_lo == w));
            kept |= 1ull << at;
            if (lane == at) group_hi = 0, group_lo = 0;
        }
#pragma unroll
        for (int j = 0; j < V; j++)
            if (first + j < n && (kept >> ((first + j) / each) & 1) == 0) hi[j] = 0, lo[j] = 0;
    }
    // round r's choice and its weight: lane r's
    int chosen = 0;
    double weight = 0.0, sum = 0.0;
    for (int r = 0; r < a.k; r++) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < V; j++) best = hi[j] > best ? hi[j] : best;
        const uint32_t h = wave_largest(best);
        uint32_t w = 0;
        if (WIDE) {
#pragma unroll
            for (int j = 0; j < V; j++) w = hi[j] == h && lo[j] > w ? lo[j] : w;
            w = wave_largest(w);
        }
        int mine = V;
        double p = 0.0;
#pragma unroll
        for (int j = V - 1; j >= 0; j--)
            if (hi[j] == h && lo[j] == w) mine = j, p = e[j];
        const int at = __builtin_ctzll(__ballot(mine < V));
#pragma unroll
        for (int j = 0; j < V; j++)
            if (lane == at && j == mine) hi[j] = 0, lo[j] = 0;
        const int index = __builtin_amdgcn_readlane(first + mine, at);
        p = from_lane(p, at);
        sum += p;
        if (lane == r) chosen = index, weight = p;
    }
    if (lane < a.k) {
        a.indices[row * a.k + lane] = chosen;
        if (a.normalize) weight /= sum + 1e-20;
        Elem<T>::store((T *)a.weights, row * a.k + lane, (float)(weight * a.scale));
    }
}

template <typename T, int V>
void run_select(const SelectArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)((a.rows + kSelectWaves - 1) / kSelectWaves)), block(64 * kSelectWaves);
    if (a.bias != nullptr || (a.groups > 1 && a.group_best == 2)) hipLaunchKernelGGL((moe_select_kernel<T, V, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((moe_select_kernel<T, V, false>), grid, block, 0, s, a);
}

template <typename T>
void run_select_type(const SelectArgs &a, hipStream_t s) {
    if (a.experts <= 64) run_select<T, 1>(a, s);
    else if (a.experts <= 128) run_select<T, 2>(a, s);
    else if (a.experts <= 256) run_select<T, 4>(a, s);
    else if (a.experts <= 512) run_select<T, 8>(a, s);
    else run_select<T, 16>(a, s);
}

}  // namespace

int32_t launch_moe_select(const nvq_moe_select_desc &d, const void *logits, const float *bias, int32_t *indices, void *weights, hipStream_t s) {
    const SelectArgs a{logits, bias, indices, weights, d.rows, d.experts, d.k, d.groups, d.top_groups, d.group_best, d.normalize, d.scores == NVQ_SCORES_SIGMOID, d.scale};
    if (d.dtype == NVQ_F32) run_select_type<float>(a, s);
    else if (d.dtype == NVQ_BF16) run_select_type<bf16_t>(a, s);
    else run_select_type<f16_t>(a, s);
    NVQ_LAUNCH_CHECK("moe_select");
    return NVQ_OK;
}

}  // namespace nvq
