// The choice of experts from a router's logits: of a row l of them
//     p = softmax(l) or sigmoid(l),  c = p + bias,
// a group's score is the sum of its one or two largest c, the best groups stay, the k largest c of their experts are chosen, and their
// weights are p, divided by (their sum + 1e-20) where asked, times a scale.
//
// What is chosen is decided as by real numbers.  Without a bias (and groups by their best alone) c's order is the logits', and nothing is computed to find it.
// Otherwise c is computed in float32, off by less than kNear: where two values that follow one another among the chosen, or at the border of what is chosen,
// are further apart than that their order is certain, and where they are not (or a value is not finite) the row is decided again in 64 bits.  The
// weights are computed for the chosen alone, for float32 results in 64 bits, as a softmax's sum is.
//
// One wavefront a row.  A group has a power of two of the lanes, a lane V consecutive experts, so that (lane, place) is the experts' order and a group's
// score a few exchanges among its lanes.  Values are compared as whole numbers of the same order, 0 for what is not to be chosen, whose low bits are their
// places: a round is one maximum over the wavefront, by data-parallel moves, and knows whose it is.
//
// Bound by the vector unit's instructions, 427 a row of 256 experts; memory would allow 1.9 us for the first of these.  Measured (us): 16384 rows of
// 256 in eight groups, bfloat16, sigmoid, a bias 16.5 (all of it in 64 bits 35; ballots for a maximum's place, and weights of 64 bits 19.6; every lane's
// values sorted beforehand 21.5); 1333 rows of 60 in float16 5.0 and eight rows of 256 4.6 to 5.4, a launch.
#include <type_traits>

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
    int32_t experts, k, groups, top_groups, group_best, normalize, sigmoid, lanes_shift;  // lanes of a group: a power of two
    double scale;
};

// Whole numbers in the values' order, above 1; a NaN is 1.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = f2u(v + 0.0f);  // (-0 is 0)
    return v != v ? 1u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return v != v ? 1u : b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint32_t ordered_number(float v) {  // (of what is a number)
    const uint32_t b = f2u(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return u2f(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

// exp(x) with the product's rounding put back: off by a step of float32.
__device__ __forceinline__ float exponential(float x) {
    constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
    const float y = x * kLog2e, e = __builtin_amdgcn_exp2f(y);
    return fabsf(y) < 200.0f ? __builtin_fmaf(e, __builtin_fmaf(x, kLog2e, -y) * kLn2, e) : e;  // (0, infinite or not a number as it is)
}

// The lane's place: of the group `group` of `each` experts the expert `first` and those behind it, `count` of the V.
struct Place {
    int group, first, count;
};

// The row decided in 64 bits: lane r's round r, its expert.
template <int V>
__device__ __forceinline__ int select_wide(const SelectArgs &a, const float (&l)[V], const Place &at_place, double *held) {
    const int lane = threadIdx.x & 63, each = a.experts / a.groups;
    double c[V];
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < V; j++) c[j] = 1.0 / (1.0 + exp(-(double)l[j]));
    } else {
        float top = -INFINITY;
        bool wild = false;
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j < at_place.count) top = fmaxf(top, l[j]), wild |= l[j] != l[j];
        top = across<64>(top, [](float x, float y) { return fmaxf(x, y); });
        const bool none = top == -INFINITY && !__any(wild);  // (a row of -inf alone: zeros)
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; j++) {
            c[j] = none ? 0.0 : exp((double)l[j] - (double)top);
            if (j < at_place.count) sum += c[j];
        }
        sum = across<64>(sum, [](double x, double y) { return x + y; });
#pragma unroll
        for (int j = 0; j < V; j++) c[j] = none ? 0.0 : c[j] / sum;
    }
    const bool by_logits = a.bias == nullptr && (a.groups == 1 || a.group_best == 1);
    uint32_t hi[V], lo[V];
#pragma unroll
    for (int j = 0; j < V; j++) {
        const bool real = j < at_place.count;
        if (a.bias != nullptr && real) c[j] += (double)a.bias[at_place.first + j];
        if (by_logits) c[j] = (double)l[j];
        const uint64_t b = real ? ordered(c[j]) : 0;
        hi[j] = (uint32_t)(b >> 32), lo[j] = (uint32_t)b;
        if (real) held[at_place.first + j] = c[j] != c[j] ? -INFINITY : c[j];
    }
    if (a.groups > 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint32_t group_hi = 0, group_lo = 0;
        if (lane < a.groups) {
            double best = -INFINITY, second = -INFINITY;
            for (int i = 0; i < each; i++) {
                const double v = held[lane * each + i];
                second = v > best ? best : v > second ? v : second, best = v > best ? v : best;
            }
            const uint64_t b = ordered(a.group_best == 2 && each > 1 ? best + second : best);
            group_hi = (uint32_t)(b >> 32), group_lo = (uint32_t)b;
        }
        uint64_t kept = 0;
        for (int i = 0; i < a.top_groups; i++) {
            const uint32_t h = wave_largest(group_hi), w = wave_largest(group_hi == h ? group_lo : 0);
            const int at = __builtin_ctzll(__ballot(group_hi == h && group_lo == w));
            kept |= 1ull << at;
            if (lane == at) group_hi = 0, group_lo = 0;
        }
        if ((kept >> at_place.group & 1) == 0)
#pragma unroll
            for (int j = 0; j < V; j++) hi[j] = 0, lo[j] = 0;
    }
    if (a.bias == nullptr && !by_logits)  // (groups by c, but their experts by the logits, whose order c's is as far as 64 bits hold it)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const uint64_t b = (hi[j] | lo[j]) != 0 ? ordered((double)l[j]) : 0;
            hi[j] = (uint32_t)(b >> 32), lo[j] = (uint32_t)b;
        }
    int chosen = 0;
    for (int r = 0; r < a.k; r++) {
        uint32_t best = 0, w = 0;
#pragma unroll
        for (int j = 0; j < V; j++) best = hi[j] > best ? hi[j] : best;
        const uint32_t h = wave_largest(best);
#pragma unroll
        for (int j = 0; j < V; j++) w = hi[j] == h && lo[j] > w ? lo[j] : w;
        w = wave_largest(w);
        int mine = V;
#pragma unroll
        for (int j = V - 1; j >= 0; j--)
            if (hi[j] == h && lo[j] == w) mine = j;
        const int at = __builtin_ctzll(__ballot(mine < V));
#pragma unroll
        for (int j = 0; j < V; j++)
            if (lane == at && j == mine) hi[j] = 0, lo[j] = 0;
        const int expert = __builtin_amdgcn_readlane(at_place.first + mine, at);
        if (lane == r) chosen = expert;
    }
    return chosen;
}

// Float32's error of c, relative to 1 and to c: sigmoids and softmaxes (at most 1) are off by 2^-21 at most, products with 64 lanes' sums among it, and the sum
// with the bias by half a step; a group's score by that of its two and another half step of their sum.  What is as near as this is decided again.
constexpr float kNear = 1.0f / (1 << 19);

// The weight of the expert that lane r of k has, from its logit.
template <typename Real>
__device__ __forceinline__ float weight_of(const SelectArgs &a, float x, float top, bool none, double total) {
    constexpr bool kWide = sizeof(Real) == 8;
    Real p = 0;
    if ((int)(threadIdx.x & 63) < a.k) {
        if constexpr (kWide) p = a.sigmoid ? 1.0 / (1.0 + exp(-(double)x)) : none ? 0.0 : exp((double)x - (double)top) / total;
        else p = a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + exponential(-x)) : none ? 0.0f : exponential(x - top) * __builtin_amdgcn_rcpf((float)total);
    }
    if (a.normalize) {
        auto add = [](Real x, Real y) { return x + y; };
        const Real sum = (a.k <= 16 ? across<16>(p, add) : across<64>(p, add)) + (Real)1e-20;
        if constexpr (kWide) p /= sum;
        else p *= __builtin_amdgcn_rcpf(sum);
    }
    return (float)(p * (Real)a.scale);
}

// BIASED: c is computed; else the logits are compared, and nothing is in doubt but what is not a number.
template <typename T, int V, bool BIASED>
__global__ void __launch_bounds__(64 * kSelectWaves) moe_select_kernel(const SelectArgs a) {
    __shared__ double held[kSelectWaves][64 * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * kSelectWaves + wave;
    if (row >= a.rows) return;
    const int each = a.experts / a.groups, per = 1 << a.lanes_shift;  // lanes of a group
    Place place;
    place.group = lane >> a.lanes_shift;
    const int within = (lane & (per - 1)) * V;
    place.first = place.group * each + within;
    place.count = place.group < a.groups ? each - within : 0;
    place.count = place.count < 0 ? 0 : place.count < V ? place.count : V;
    const T *logits = (const T *)a.logits + row * a.experts;
    const bool biased = BIASED && a.bias != nullptr;
    float l[V], bias[V];
    if (each % V == 0) {  // a lane's are all there or none
        struct __attribute__((packed)) Run { T t[V]; };
        struct __attribute__((packed)) Biases { float t[V]; };
        const int from = place.count > 0 ? place.first : 0;
        const Run run = *reinterpret_cast<const Run *>(logits + from);
        Biases b{};
        if (biased) b = *reinterpret_cast<const Biases *>(a.bias + from);
#pragma unroll
        for (int j = 0; j < V; j++) l[j] = Elem<T>::load(run.t, j), bias[j] = b.t[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int from = j < place.count ? place.first + j : 0;
            l[j] = Elem<T>::load(logits, from), bias[j] = biased ? a.bias[from] : 0.0f;
        }
    }
    constexpr float kLog2e = 1.44269504088896340736f;
    double total = 1.0;  // softmax: of exp(l - top)
    bool none = false;   // a row of -inf alone: zeros
    float top = 0.0f;
    float c[V];
    if (!a.sigmoid) {
        top = -INFINITY;
#pragma unroll
        for (int j = 0; j < V; j++) top = j < place.count ? fmaxf(top, l[j]) : top;
        top = across<64>(top, [](float x, float y) { return fmaxf(x, y); });
        if (top == -INFINITY) {
            asm volatile("");  // (a branch, the same for all lanes)
            bool wild = false;
#pragma unroll
            for (int j = 0; j < V; j++) wild |= j < place.count && l[j] != l[j];
            none = !__any(wild);
        }
        if (BIASED || !a.normalize) {  // (normalized weights do without the sum, but for what keeps them from 0 / 0)
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < V; j++) {
                c[j] = exponential(l[j] - top);
                sum += j >= place.count ? 0.0 : sizeof(T) == 4 ? exp((double)l[j] - (double)top) : (double)c[j];
            }
            total = across<64>(sum, [](double x, double y) { return x + y; });
        }
    }
    uint32_t key[V];
    float wild = 0.0f;  // NaN where a value is not finite (not a number)
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (BIASED) c[j] = (a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[j] * -kLog2e)) : c[j] * __builtin_amdgcn_rcpf((float)total)) + bias[j];
        else c[j] = l[j];
        const float v = j < place.count ? c[j] : 0.0f;
        wild = BIASED ? __builtin_fmaf(v, 0.0f, wild) : v != v ? v : wild;
        key[j] = j < place.count ? ordered_number(c[j]) : 0u;
    }
    bool doubt = wild != wild;
    if (a.groups > 1) {
        // a group's two best, among its lanes
        float best = -INFINITY, second = -INFINITY;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float v = j < place.count ? c[j] : -INFINITY;
            second = fmaxf(second, fminf(best, v)), best = fmaxf(best, v);
        }
        auto meet = [&](float b, float s) __attribute__((always_inline)) { second = fmaxf(fminf(best, b), fmaxf(second, s)), best = fmaxf(best, b); };
        if (a.lanes_shift > 0) meet(moved<kPairs>(best), moved<kPairs>(second));
        if (a.lanes_shift > 1) meet(moved<kQuads>(best), moved<kQuads>(second));
        if (a.lanes_shift > 2) meet(moved<kHalfRow>(best), moved<kHalfRow>(second));
        if (a.lanes_shift > 3) meet(moved<kRow>(best), moved<kRow>(second));
        if (a.lanes_shift > 4) meet(__shfl_xor(best, 16), __shfl_xor(second, 16));
        const bool two = a.group_best == 2 && each > 1;
        const float score = two ? best + second : best;
        const float off = kNear * (1.0f + fabsf(best) + (two ? fabsf(second) : 0.0f));  // (of what is added up: the sum may be far smaller)
        const bool real = place.group < a.groups;
        const uint32_t mine = real ? ordered_number(score) : 0u;
        int before = 0;  // groups that come first
        for (int g0 = 0; g0 < a.groups; g0 += 4)
#pragma unroll
            for (int g = g0; g < g0 + 4; g++) {  // (of two groups those behind the last would be lanes 64 and 96)
                const uint32_t other = g < a.groups ? (uint32_t)__builtin_amdgcn_readlane((int)mine, g << a.lanes_shift) : 0u;
                before += other + (g < place.group ? 1u : 0u) > mine ? 1 : 0;  // (no key is the largest number)
            }
        const bool kept = before < a.top_groups;
        if (BIASED && a.top_groups < a.groups) {
            const int last = __builtin_ctzll(__ballot(before == a.top_groups - 1) | 1ull << 63);
            const float least = value_of((uint32_t)__builtin_amdgcn_readlane((int)mine, last)), least_off = from_lane(off, last);
            doubt |= !kept && real && !(score < least - (off + least_off));
        }
#pragma unroll
        for (int j = 0; j < V; j++) key[j] = kept ? key[j] : 0u;
    }
    // A value's place among the wavefront's (V a lane, in the experts' order) replaces its key's low bits, the first the largest: a round is the largest key
    // below the last one's, and holds its place.  Keys that have come wrap round to less than all others when the last is taken off.
    constexpr uint32_t kPlaces = 64 * V - 1;
    constexpr bool kWhole = !BIASED && sizeof(T) == 2;  // no key has lost a bit that it had (the 13 lowest are alike in all of float16's, 16 in bfloat16's)
    static_assert(kPlaces < 1u << 13);
#pragma unroll
    for (int j = 0; j < V; j++) key[j] = key[j] == 0u ? 0u : (key[j] & ~kPlaces) | (kPlaces - (uint32_t)(lane * V + j));
    int slot = 0;  // lane r's of round r
    uint32_t h = 0;
    auto round = [&]() __attribute__((always_inline)) {
        uint32_t best = key[0] - h;
#pragma unroll
        for (int j = 1; j < V; j++) best = key[j] - h > best ? key[j] - h : best;
        h += wave_largest(best);
    };
    for (int r = 0; r < a.k; r++) {
        round();
        slot = lane == r ? (int)(kPlaces - (h & kPlaces)) : slot;
    }
    float2 *both = reinterpret_cast<float2 *>(held[wave]);  // logits, and what decided
#pragma unroll
    for (int j = 0; j < V; j++) both[lane * V + j] = make_float2(l[j], c[j]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const float2 mine_of = both[slot];
    int chosen = __shfl(place.first, slot / V) + slot % V;
    if (!kWhole) {
        // What the keys have lost: those chosen have to be in order by themselves, and the last of them in front of all that the key behind it can stand for.
        round();
        const float v = mine_of.y, next = __shfl_down(v, 1), w = lane == a.k - 1 ? value_of(h | kPlaces) : next;
        const bool last = lane == a.k - 1, sure = BIASED ? w < v - kNear * (1.0f + fabsf(v)) : last ? w < v : w <= v;
        doubt |= lane < a.k && !sure && !(last && (h & ~kPlaces) == 0u);
    }
    float x = mine_of.x;
    if (__any(doubt)) {
        asm volatile("");  // (a branch, the same for all lanes)
        if (!BIASED && __any(wild != wild)) total = NAN;  // (the sum that was not needed: a softmax with a NaN is NaN)
        chosen = select_wide<V>(a, l, place, held[wave]);
        x = lane < a.k ? Elem<T>::load(logits, chosen) : 0.0f;
    }
    // Results of 16 bits from float32, off by less than 2^-20, but where an exponential would leave its normal range; of 32 from 64 bits.
    const bool far = lane < a.k && (a.sigmoid ? -x : top - x) > 80.0f;
    const float weight = sizeof(T) == 4 || __builtin_expect(__any(far), 0) ? weight_of<double>(a, x, top, none, total) : weight_of<float>(a, x, top, none, total);
    if (lane < a.k) {
        a.indices[row * a.k + lane] = chosen;
        Elem<T>::store((T *)a.weights, row * a.k + lane, weight);
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
    const int each = a.experts / a.groups, of_lane = (each + (1 << a.lanes_shift) - 1) >> a.lanes_shift;
    if (of_lane <= 1) run_select<T, 1>(a, s);
    else if (of_lane <= 2) run_select<T, 2>(a, s);
    else if (of_lane <= 4) run_select<T, 4>(a, s);
    else if (of_lane <= 8) run_select<T, 8>(a, s);
    else if (of_lane <= 16) run_select<T, 16>(a, s);
    else run_select<T, 32>(a, s);  // (31 at most: 1024 experts over the more than 32 lanes that the groups have together)
}

}  // namespace

int32_t launch_moe_select(const nvq_moe_select_desc &d, const void *logits, const float *bias, int32_t *indices, void *weights, hipStream_t s) {
    SelectArgs a{logits, bias, indices, weights, d.rows, d.experts, d.k, d.groups, d.top_groups, d.group_best, d.normalize, d.scores == NVQ_SCORES_SIGMOID, 0, d.scale};
    while (a.groups << (a.lanes_shift + 1) <= 64) a.lanes_shift++;
    if (d.dtype == NVQ_F32) run_select_type<float>(a, s);
    else if (d.dtype == NVQ_BF16) run_select_type<bf16_t>(a, s);
    else run_select_type<f16_t>(a, s);
    NVQ_LAUNCH_CHECK("moe_select");
    return NVQ_OK;
}

}  // namespace nvq
