// Attention of whole prompts over keys and values as the projections leave them:
//     out[row, h, :] = softmax(scale * q[row, h, :] . K^T [masked] [, sink[h]]) . V
// over the keys and values of the row's sequence.
//
// A block has 128 lines (line r of a sequence: row r / rep, query head r % rep of the key head, so that the heads that share keys share their tile), a
// wavefront 32 of them, and walks the keys it sees in tiles in LDS: S^T = K . Q^T on v_mfma_f32_32x32x16 leaves a lane with half of a tile's scores of
// ONE line, its maximum and sum are in-lane but for an exchange of two lanes, and the weights of 16 keys are already the operand of
// O^T = V^T . P^T, whose V is read from LDS through the transposing read in the order in which the lanes hold the keys.  float32 runs the same way on
// v_mfma_f32_32x32x2_f32.
//
// Terms.  Queries, keys and values are exact operands in their own type.  The weights are two terms of it, 16 bits in bfloat16 and 22 in float16 (one term
// leaves an error beside the result's own rounding; float16's are relative to a reference that follows the tiles' maxima up and down, so that small ones have
// them too: a weight is off by 2^-22 of itself or 2^-21 of its tile's largest), in float32 themselves.  Scores, maxima, sums and accumulators are float32.  bfloat16 values as float16
// operands would take one term, but a power of two that brings a tile's values into float16's range is one for lines that see the largest of them and for
// lines that do not, whose own would be lost.
//
// Masked keys (behind the sequence's end, in front of a row or outside its window) have no weight whatever their keys hold.  A block whose sums are not finite
// walks its keys again: values that are not finite are zeros in the tile then, so that lines that do not see them stay clean, and the lines that do are given them
// afterwards; and the weights are 2^-32 at most, so that sums of the largest finite values stay finite.
//
// The bound of long prompts of 128 values is the matrix cores at the clock that the chip's power leaves them: busy for 60 % of the cycles that a compute unit is,
// vector instructions for as many, at 1.70 GHz (GRBM_GUI_ACTIVE over the time; launches that are short or wait more run at 2.05 and more).  That of small heads
// is the instructions beside the products: 32 fused multiply-adds, exponentials (eight cycles each, others five, and eight beside the other wavefront's
// products), additions, 16 maxima and conversions a lane for 64 keys of a line, and 48 more for the weights' second terms (80 in bfloat16, which has no
// instruction that takes a pair's half off).  Two wavefronts a SIMD take turns on the matrix cores (three of heads of 64 values); what is
// written between the products runs beside them: the next tile's way into LDS in those of the scores, the next keys' weights in those of the values.
//
// Measured (us; a large product of the types runs at 1235 and 1183 TFLOP/s; boxes differ by 3 to 5 %): 8192 rows of 32 heads of 128 over 8 key heads in bfloat16
// 701 to 737, 746 to 784 TFLOP/s; nine ragged prompts of up to 1500 rows in float16, 20 heads of 64, sinks and a window 69 to 70, 370 TFLOP/s: vector
// instructions for 61 % of a busy compute unit's cycles, and a fifth of the launch in which it is not busy (920 blocks on 768 places); seven prompts of up to 61
// rows 9.5, a chain of first loads.  4096 rows of 16 heads over 4 (512 blocks, all on the chip at once): bfloat16 heads of 64 423 TFLOP/s, 128 557 to 585, 256 561;
// float16 426, 560, 539; float32 110, 123, 67 (of 154).  One row over 32768 keys 39 to 41 us, 3.3 to 3.5 TB/s.
//
// Weights of one float16 term over values taken as float16 were 576 to 605 us in the first of these, and wrong where a row does not see the largest values
// (paragraph on terms).  Timed without its parts in that form: the tile's way into LDS 23 % (half of it the loads), the products of the values 15 %.  Tried with it
// and not kept: 64 lines a wavefront at one a SIMD (690 us: one wavefront issues no more than an instruction in five cycles), blocks of eight wavefronts (3 %
// faster, half of the blocks empty in short prompts), tiles of 32 keys (652, at three wavefronts a SIMD 700 with spills), the branches of the rare cases in
// the loop (714: their loads made every tile wait for its successor's).
#pragma once

#include <type_traits>

#include "matrix.h"
#include "nvq_device.h"
#include "nvq_internal.h"
#include "prompt_attention.h"

namespace nvq {
namespace prompt {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.4e38f;  // where maxima start (paged_rows_kernel.h says why it is finite)

template <typename T>
struct PromptArgs {
    PromptBatch batch;
    const T *q, *k, *v, *sinks;
    T *out;
    int32_t *length;  // of the plan, for the merge; NULL: no merge
    float *states;    // [slots][kLines][D + 4]: maximum of the base-2 scores, denominator, two unused, D weighted means
    int64_t q_strides[2], k_strides[2], v_strides[2], out_strides[2];
    int32_t dim, turn, back, slots;  // (starts that are not ascending may ask for more states than there are: those are left out)
    float scale;
};

namespace {

typedef float acc16_t __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));

template <int D> constexpr int kState = D + 4;

// K's rows have a 16-byte run more than their values, an odd number of them: the 16 lanes that read one run of 16 rows meet different banks.  V's
// rows are an odd number of 64 bytes apart: the 32 lanes that read 64 bytes of four rows.
template <typename T, int D>
struct Tile {
    static constexpr int kKeys = sizeof(T) == 4 || D > 128 ? 32 : 64;  // (of a lane 32 at most: the bits of a word)
    static constexpr int kRuns = D * (int)sizeof(T) / 16;  // of a row
    static constexpr int kKeyRow = 16 * (kRuns + 1), kValueRow = 64 * (kRuns / 4 + (kRuns / 4 % 2 == 0 ? 1 : 0));
    static constexpr int kShare = kKeys * kRuns / (64 * kWaves);  // runs of a thread
    static_assert(kKeys * kRuns % (64 * kWaves) == 0);
    struct Stage {
        uint8_t keys[kKeys * kKeyRow], values[kKeys * kValueRow];
    };
};

template <typename T>
__device__ __forceinline__ acc16_t product32(uint4 k, uint4 q, acc16_t c) {
    if constexpr (Elem<T>::code == NVQ_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q), c, 0, 0, 0);
    } else if constexpr (Elem<T>::code == NVQ_F16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, k), __builtin_bit_cast(half8_t, q), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(k.x), u2f(q.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(k.y), u2f(q.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(k.z), u2f(q.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(k.w), u2f(q.w), c, 0, 0, 0);
    }
}

// Two values as a pair of the (16-bit) element type.
template <typename T>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t v = {a, b};
    if constexpr (Elem<T>::code == NVQ_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
}
// v less half I of the pair w.
template <typename T, int I>
__device__ __forceinline__ float behind(float v, uint32_t w) {
    if constexpr (Elem<T>::code == NVQ_BF16) return v - u2f(I == 0 ? w << 16 : w & 0xFFFF0000u);
    float d;
    if constexpr (I == 0) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(w), "v"(v));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(w), "v"(v));
    return d;
}

// The keys that a block's lines see, from `begin` to `end`, and how its items share them: evenly, `keys` each.  An item that has them all writes the result.
struct Span {
    int32_t begin, end, keys, items;
};
__device__ __forceinline__ Span span_of(const PromptBatch &a, const PagedItem &item, int part) {
    const int32_t from = part * kLines, lines = item.s.rows * a.rep, to = lines - from < kLines ? lines : from + kLines;
    int32_t begin = 0, end = item.s.length;
    if (a.causal) {
        const int32_t before = item.s.length - item.s.rows, seen = before + (to - 1) / a.rep + 1;
        const int64_t first = a.window > 0 ? before + from / a.rep + 1 - a.window : 0;
        end = seen < end ? seen : end, begin = first > 0 ? (int32_t)first / kScheduleKeys * kScheduleKeys : 0;
    }
    Span s{uniform(begin), uniform(end), 0, 1};
    const int32_t tiles = end > begin ? (end - begin + kScheduleKeys - 1) / kScheduleKeys : 0;
    int32_t per = (tiles + item.splits - 1) / item.splits;
    per = ((per > a.least ? per : a.least) + 1) & ~1;
    s.keys = uniform(item.splits == 1 ? tiles * kScheduleKeys : per * kScheduleKeys);
    s.items = uniform(item.splits == 1 || tiles <= per ? 1 : (tiles + per - 1) / per);
    return s;
}

// The item of a block.  Items come with the longest of a sequence first, a block on each compute unit in turn, and where they are all on the chip at once the unit
// that has the longest would have the longest of the second turn too: the second turn goes back, eight at a time, so that a key head stays with its XCD.
// (4096 rows of 16 heads over 4: float32, 128 values 754 -> 556 us, bfloat16 130 -> 123, float16, 64 values 87.0 -> 80.5; where more blocks follow, which
// go where one has ended, it is of no use: 3000 rows of 32 heads over 8 114.4 and 114.5.)
__device__ __forceinline__ int32_t turned(uint32_t block, int32_t turn, int32_t back) {
    const int32_t r = (int32_t)block - turn;
    return r >= 0 && r < back ? turn + back - 8 - (r & ~7) + (r & 7) : (int32_t)block;
}

template <typename T, int D>
__global__ void __launch_bounds__(64 * kWaves, blocks_of((int)sizeof(T), D)) prompt_kernel(const PromptArgs<T> a) {
    using Of = Tile<T, D>;
    using Stage = typename Of::Stage;
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int KT = Of::kKeys, TB = KT / 32, RUN = kFragRun<T>;      // keys of a tile, blocks of 32; values of a run
    constexpr int KS = D / (2 * RUN), ND = D / 32;                     // steps of a score (a run of both halves of the wavefront), blocks of D
    constexpr int SHARE = Of::kShare;
    // With care maxima stand 2^kLift above the scores' own (not float16's, whose sums stay in float32's range anyway).
    constexpr float kLift = Elem<T>::code == NVQ_F16 ? 0.0f : 40.0f;
    __shared__ alignas(16) Stage stages[2];
    __shared__ uint32_t flags[2];             // of a stage: a value that is not finite
    __shared__ uint32_t again;                // sums that are not finite
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
    PagedItem item;
    const int32_t at_item = turned(blockIdx.x, a.turn, a.back);
    if (a.length != nullptr) {
        if (!paged_item<kLines, 1, false>(a.batch, lane, at_item, a.length, item)) return;
    } else if (!paged_item_of<kLines, 1, false>(a.batch, PagedPlan{1 << 26, INT32_MAX}, lane, paged_sequence<kLines, 1>(a.batch, lane), at_item, item)) {
        return;  // (nothing is split: no plan to work out)
    }
    const int rep = a.batch.rep, hk = item.head, S = item.s.length, n = item.s.rows;
    const int part = item.s.parts - 1 - item.part;  // (the lines that see most first)
    const int lines = n * rep;
    const int window = (int)(a.batch.window < S + 1 ? a.batch.window : S + 1);
    auto last_of = [&](int i) { return a.batch.causal ? S - n + i : S - 1; };
    auto first_of = [&](int i) { return window > 0 && a.batch.causal ? last_of(i) - window + 1 : 0; };
    const Span span = span_of(a.batch, item, part);
    if (item.split >= span.items || (span.items > 1 && item.slot >= a.slots)) return;
    const int s_begin = uniform(span.begin + item.split * span.keys), s_end = uniform(span.end < s_begin + span.keys ? span.end : s_begin + span.keys);
    // the wavefront's lines
    const int r0 = part * kLines + wave * 32, r = r0 + col;
    const bool live = r < lines;
    const int my_row = (live ? r : lines - 1) / rep, my_head = hk * rep + (live ? r % rep : 0);
    const int my_last = last_of(my_row), my_first = first_of(my_row);
    const int w_first = (r0 < lines ? r0 : lines - 1) / rep, w_last = (r0 + 31 < lines ? r0 + 31 : lines - 1) / rep;
    const int all_last = uniform(last_of(w_first)), all_first = uniform(first_of(w_last));                    // keys up to / from which all of them see
    const int any_last = uniform(r0 < lines ? last_of(w_last) : -1), any_first = uniform(first_of(w_first));  // and any does

    // ── staging: run i of a thread is run tid + 256 i of the tile ──
    const int64_t first_key = a.batch.first_key(item.b);
    const T *keys = a.k + first_key * a.k_strides[0] + (int64_t)hk * a.k_strides[1], *values = a.v + first_key * a.v_strides[0] + (int64_t)hk * a.v_strides[1];
    uint4 kr[SHARE], vr[SHARE];
    auto place = [&](int i, int &row, int &run) __attribute__((always_inline)) {
        const int at = tid + 64 * kWaves * i;
        row = at / Of::kRuns, run = at % Of::kRuns;
    };
    // A run's offset from its tile's first row is below 2^32 (the entry refuses strides beyond that), so that a load adds it to a scalar address.  It is
    // worked out from the first run's where the runs of a thread lie whole rows apart.
    constexpr bool kEven = 64 * kWaves % Of::kRuns == 0;
    constexpr int kApart = 64 * kWaves / Of::kRuns;  // rows
    auto offset = [&](int64_t stride, int row, int run) __attribute__((always_inline)) {
        return ((uint32_t)row * (uint32_t)stride + (uint32_t)(run * RUN < a.dim ? run * RUN : 0)) * (uint32_t)sizeof(T);
    };
    uint32_t k_offset[kEven ? 1 : SHARE], v_offset[kEven ? 1 : SHARE];
#pragma unroll
    for (int i = 0; i < (kEven ? 1 : SHARE); i++) {
        int row, run;
        place(i, row, run);
        k_offset[i] = offset(a.k_strides[0], row, run), v_offset[i] = offset(a.v_strides[0], row, run);
    }
    const bool whole_rows = a.dim == D;
    // (keys behind the sequence's last are read as the last; loads under a condition would be waited for at its end)
    auto load_tile = [&](uint4 (&to)[SHARE], const T *from, int64_t stride, uint32_t (&of)[kEven ? 1 : SHARE], int s0) __attribute__((always_inline)) {
        const uint8_t *first = reinterpret_cast<const uint8_t *>(from + (int64_t)s0 * stride);
        const uint32_t step = (uint32_t)stride * (uint32_t)sizeof(T), last = (uint32_t)(S - 1 - s0 < KT - 1 ? S - 1 - s0 : KT - 1) * step;
        asm volatile("" : "+v"(of[0]));  // (what follows from it is not worth a register each)
#pragma unroll
        for (int i = 0; i < SHARE; i++) {
            int row, run;
            place(kEven ? 0 : i, row, run);
            const uint32_t at = kEven ? of[0] + (uint32_t)(i * kApart) * step : of[kEven ? 0 : i], end = last + (uint32_t)(run * RUN < a.dim ? run * RUN : 0) * (uint32_t)sizeof(T);
            to[i] = load_run(reinterpret_cast<const T *>(first + (at < end ? at : end)));
        }
    };
    auto request_values = [&](int s0) __attribute__((always_inline)) { load_tile(vr, values, a.v_strides[0], v_offset, s0); };
    auto request = [&](int s0) __attribute__((always_inline)) {
        load_tile(kr, keys, a.k_strides[0], k_offset, s0);
        request_values(s0);
    };
    if (s_begin < s_end) request(s_begin);  // (the queries come behind it)
    // Scores are kept positive multiples of the product: a negative scale's sign goes to the queries, and of a scale of 0 they are zeros.
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    uint4 qf[KS];
    {
        const T *query = a.q + (int64_t)(item.s.start + my_row) * a.q_strides[0] + (int64_t)my_head * a.q_strides[1];
        const uint32_t sign = a.scale < 0.0f ? (kWide ? 0x80000000u : 0x80008000u) : 0u, keep = a.scale == 0.0f ? 0u : ~0u;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const int d = (2 * s + half) * RUN;
            const uint4 w = load_run(query + (d < a.dim ? d : 0));
            const uint32_t k = d < a.dim ? keep : 0u;
            qf[s] = make_uint4((w.x ^ sign) & k, (w.y ^ sign) & k, (w.z ^ sign) & k, (w.w ^ sign) & k);
        }
    }
    // What lies behind the head's values and behind the sequence's end: zeros.
    auto real = [&](int s0, int i) __attribute__((always_inline)) {
        int row, run;
        place(i, row, run);
        return s0 + row < S && run * RUN < a.dim;
    };
    auto value_place = [&](Stage &to, int i) __attribute__((always_inline)) {
        int row, run;
        place(i, row, run);
        return reinterpret_cast<uint4 *>(to.values + row * Of::kValueRow + 16 * run);
    };
    // The tile's rows into a stage, in pieces: run i of the values and of the keys by turns.  First what takes a branch; last (CAREFUL) the stage's flag where a
    // value is not finite there.
    float wild;
    auto lay_first = [&](int s0) __attribute__((always_inline)) {
        wild = 0.0f;
        if (__builtin_expect(!whole_rows || s0 + KT > S, 0)) {
            asm volatile("");  // (a branch, the same for all)
#pragma unroll
            for (int i = 0; i < SHARE; i++) {
                int row, run;
                place(i, row, run);
                // (keys behind the head's values meet zeros of the queries, which an infinite value would spoil)
                const uint32_t k = run * RUN < a.dim ? ~0u : 0u, v = real(s0, i) ? ~0u : 0u;
                kr[i] = make_uint4(kr[i].x & k, kr[i].y & k, kr[i].z & k, kr[i].w & k), vr[i] = make_uint4(vr[i].x & v, vr[i].y & v, vr[i].z & v, vr[i].w & v);
            }
        }
    };
    auto lay_piece = [&](auto careful, Stage &to, int piece) __attribute__((always_inline)) {
        const int i = piece >> 1;
        int row, run;
        place(i, row, run);
        if (piece & 1) {
            *reinterpret_cast<uint4 *>(to.keys + row * Of::kKeyRow + 16 * run) = kr[i];
            return;
        }
        *value_place(to, i) = vr[i];
        if constexpr (!decltype(careful)::value) return;
        T t[RUN];
        __builtin_memcpy(t, &vr[i], 16);
#pragma unroll
        for (int j = 0; j < RUN; j++) wild = __builtin_fmaf(Elem<T>::load(t, j), 0.0f, wild);  // (x 0 is NaN of what is not finite)
    };
    auto lay_last = [&](auto careful, uint32_t &flag) __attribute__((always_inline)) {
        if constexpr (!decltype(careful)::value) return;
        if (wild != wild) flag = 1u;
    };

    acc16_t o[ND];
    float m, l;
    auto clear = [&]() __attribute__((always_inline)) {
        m = kLowest, l = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    };

    // V^T . P^T of 16 keys (float32: of two), their weights in `p` as the scores' accumulators hold them.
    auto value_run = [&](const Stage &from, int c, int d) __attribute__((always_inline)) {
        const uint8_t *at = from.values + (16 * c + 4 * half + ((lane & 15) >> 2)) * Of::kValueRow + 2 * (32 * d + 16 * (lane >> 4 & 1) + 4 * (lane & 3));
        typedef __attribute__((address_space(3))) short4_t *Lds;
        const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(uintptr_t)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(uintptr_t)(at + 8 * Of::kValueRow));
        struct { short4_t v[2]; } both = {{lo, hi}};
        return __builtin_bit_cast(uint4, both);
    };
    auto value_at = [&](const Stage &from, int i, int d) __attribute__((always_inline)) {
        return reinterpret_cast<const float *>(from.values + (8 * (i >> 2) + 4 * half + (i & 3)) * Of::kValueRow)[32 * d + col];
    };
    // Exponentials, sums and products.  16-bit types: the weights of 16 keys are worked out, and the values of the next 16 read, between the products of the
    // 16 before them (in the order written: products wait for neither, and the vector unit works beside them).
    auto weigh = [&](const Stage &from, float (&x)[TB][16], auto careful, uint32_t &seen) __attribute__((always_inline)) {
        float sum = 0.0f;  // (a tile's by itself: beside a large sum many small weights would be lost one by one)
        auto weight = [&](int i) __attribute__((always_inline)) {
            const float e = __builtin_amdgcn_exp2f(x[i >> 4][i & 15]);
            sum += e;
            if constexpr (decltype(careful)::value) seen |= (x[i >> 4][i & 15] < -126.0f - kLift ? 0u : 1u) << i;  // (as without the lift)
            return e;
        };
        if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[0][i] = weight(i);
#pragma unroll
            for (int i = 0; i < 16; i++)
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(value_at(from, i, d), x[0][i], o[d], 0, 0, 0);
        } else {
            constexpr int NC = KT / 16;
            uint32_t high[2][4], low[2][4];
            uint4 v[2][ND];
            auto prepare = [&](int c, int j) __attribute__((always_inline)) {
                const float e0 = weight(8 * c + 2 * j), e1 = weight(8 * c + 2 * j + 1);
                uint32_t &h = high[c & 1][j];
                h = pair_of<T>(e0, e1);
                low[c & 1][j] = pair_of<T>(behind<T, 0>(e0, h), behind<T, 1>(e1, h));
            };
            auto operand_of = [&](const uint32_t (&w)[4]) __attribute__((always_inline)) { return make_uint4(w[0], w[1], w[2], w[3]); };
#pragma unroll
            for (int d = 0; d < ND; d++) v[0][d] = value_run(from, 0, d);
#pragma unroll
            for (int j = 0; j < 4; j++) prepare(0, j);
            __builtin_amdgcn_s_setprio(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    o[d] = product32<T>(v[c & 1][d], operand_of(high[c & 1]), o[d]);
                    if (c + 1 < NC) v[(c + 1) & 1][d] = value_run(from, c + 1, d);
                    o[d] = product32<T>(v[c & 1][d], operand_of(low[c & 1]), o[d]);
                    if (c + 1 < NC)
#pragma unroll
                        for (int j = 4 * d / ND; j < 4 * (d + 1) / ND; j++) prepare(c + 1, j);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
        l += sum;
    };
    // One tile: the scores, one look at their maximum, the weights and their products.  x[t][i]: key 32 t + 8 (i / 4) + 4 half + i % 4 of the lane's line.
    // The next tile is laid between the scores' products, whose keys are read kAhead products before them.  `seen` (CAREFUL): a bit for each of these
    // keys that has a weight.
    auto tile = [&](const Stage &from, Stage &next, int s0, auto careful, uint32_t &seen) __attribute__((always_inline)) {
        constexpr int STEPS = TB * KS, PIECES = 2 * SHARE, kAhead = 8;
        float x[TB][16];
        {
            acc16_t s[TB];
#pragma unroll
            for (int t = 0; t < TB; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[t][i] = 0.0f;
            uint4 k[STEPS];
            auto read = [&](int step) __attribute__((always_inline)) {
                k[step] = *reinterpret_cast<const uint4 *>(from.keys + (32 * (step / KS) + col) * Of::kKeyRow + 16 * half + 32 * (step % KS));
            };
#pragma unroll
            for (int step = 0; step < kAhead && step < STEPS; step++) read(step);
            __builtin_amdgcn_s_setprio(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int step = 0; step < STEPS; step++) {
                s[step / KS] = product32<T>(k[step], qf[step % KS], s[step / KS]);
                if (step + kAhead < STEPS) read(step + kAhead);
#pragma unroll
                for (int piece = (PIECES * step + STEPS - 1) / STEPS; piece < (PIECES * (step + 1) + STEPS - 1) / STEPS; piece++) lay_piece(careful, next, piece);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int t = 0; t < TB; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[t][i] = s[t][i];
        }
        __builtin_amdgcn_s_setprio(0);
        if (__builtin_expect(s0 + KT - 1 > all_last || s0 < all_first || s0 + KT > s_end, 0)) {
            asm volatile("");  // (a branch: as selects it would cost every tile)
#pragma unroll
            for (int t = 0; t < TB; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int key = s0 + 32 * t + 8 * (i >> 2) + 4 * half + (i & 3);
                    if (key > my_last || key < my_first || key >= s_end) x[t][i] = -INFINITY;
                }
        }
        float top = x[0][0];
#pragma unroll
        for (int i = 1; i < 16 * TB; i++) top = fmaxf(top, x[i >> 4][i & 15]);
        top *= scale;
        // Rescaled only when a maximum has grown by more than 2^8: until then the weights are at most 2^8 (with care 2^8 less the lift).
        // float16: weights of a tile have to lie high in its range, 2^-24 to 2^16, to keep their bits however many small ones there are.  `m` is 7 below the tile's
        // maximum then, rises where a weight would leave 2^15, and falls where the tile's largest would be below 2^-4 (not for a score that is masked, and only as
        // far as the sums, which grow by that much, stay below 2^60).  Scores that are multiples of 16 and more have weights of at most 1 so: 7 is rounded to 0, and
        // differences are exact where sums are not.
        constexpr bool kFalls = Elem<T>::code == NVQ_F16;
        constexpr float kBelow = kFalls ? 7.0f : decltype(careful)::value ? -kLift : 0.0f, kMost = kFalls ? 15.0f : 8.0f + kBelow;
        auto leaves = [&]() __attribute__((always_inline)) {
            const float above = top - m;
            return above > kMost || (kFalls && above < -4.0f && top > kLowest);
        };
        const bool moves = leaves();
        if (__builtin_expect(__any(moves), 0)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            float m_new = fmaxf(m, top - kBelow);
            if constexpr (kFalls) {
                const float sum = l + __shfl_xor(l, 32), least = sum > 0.0f ? m + __builtin_amdgcn_logf(sum) - 60.0f : kLowest;  // (the same in both halves)
                m_new = leaves() ? fmaxf(top - kBelow, least) : m;
            }
            const float f = exp2f(m - m_new);
            m = m_new, l *= f;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= f;
        }
        // The maximum is a rounded product, which the fused one is not: the difference is a factor that all weights of a line share, but one that grows
        // with the scores' size.  From 2^20 on both are rounded.
        if (__builtin_expect(__any(fabsf(m) > 1048576.0f), 0)) {
            asm volatile("");
#pragma unroll
            for (int i = 0; i < 16 * TB; i++) x[i >> 4][i & 15] = x[i >> 4][i & 15] * scale - m;
        } else {
#pragma unroll
            for (int i = 0; i < 16 * TB; i++) x[i >> 4][i & 15] = __builtin_fmaf(x[i >> 4][i & 15], scale, -m);
        }
        weigh(from, x, careful, seen);
        __builtin_amdgcn_s_setprio(0);
    };

    // A flagged tile laid out again: the values that are not finite as zeros.
    auto lay_again = [&](Stage &to, int s0) __attribute__((always_inline)) {
        request_values(s0);
#pragma unroll
        for (int i = 0; i < SHARE; i++) {
            T t[RUN];
            __builtin_memcpy(t, &vr[i], 16);
            const bool used = real(s0, i);
#pragma unroll
            for (int j = 0; j < RUN; j++)
                if (!used || !(fabsf(Elem<T>::load(t, j)) < INFINITY)) Elem<T>::store(t, j, 0.0f);
            uint4 w;
            __builtin_memcpy(&w, t, 16);
            *value_place(to, i) = w;
        }
        __syncthreads();
    };
    // What is not finite, to the lines that see it: by a product of ones at the places of one kind with ones at the keys that are seen.
    auto add_wild = [&](Stage &to, int s0, const uint32_t &seen) __attribute__((always_inline)) {
        constexpr uint32_t kOne = Elem<T>::code == NVQ_BF16 ? 0x3F80u : 0x3C00u;
        request_values(s0);
        for (int kind = 0; kind < 3; kind++) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < SHARE; i++) {
                T t[RUN];
                __builtin_memcpy(t, &vr[i], 16);
                const bool used = real(s0, i);
                uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < RUN; j++) {
                    const float v = Elem<T>::load(t, j);
                    const bool is = used && (kind == 0 ? v == INFINITY : kind == 1 ? v == -INFINITY : v != v);
                    if constexpr (kWide) w[j] = is ? f2u(1.0f) : 0u;
                    else w[j >> 1] |= (is ? kOne : 0u) << (16 * (j & 1));
                }
                *value_place(to, i) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncthreads();
            const float special = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
#pragma unroll
            for (int d = 0; d < ND; d++) {
                acc16_t count;
#pragma unroll
                for (int i = 0; i < 16; i++) count[i] = 0.0f;
                if constexpr (kWide) {
#pragma unroll
                    for (int i = 0; i < 16; i++) count = __builtin_amdgcn_mfma_f32_32x32x2f32(value_at(to, i, d), (float)(seen >> i & 1u), count, 0, 0, 0);
                } else {
#pragma unroll
                    for (int c = 0; c < KT / 16; c++) {
                        uint32_t p[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) p[j] = (seen >> (8 * c + 2 * j) & 1u) * kOne | (seen >> (8 * c + 2 * j + 1) & 1u) * (kOne << 16);
                        count = product32<T>(value_run(to, c, d), make_uint4(p[0], p[1], p[2], p[3]), count);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (count[i] > 0.0f) o[d][i] += special;
            }
        }
    };

    // The keys of the item.  First without a look at what the values hold: where one is not finite, or sums leave float32's range, those of some line are
    // not finite, and the block walks its keys again with care.  (In one loop the rare paths' loads would be waited for in every tile.)
    // Tile s lies in a stage while tile s + 1 is on its way through registers and tile s + 2 is requested; behind the item's last tile
    // that one again (loads under a condition cost registers that spilled: 5% of the time).
    auto walk = [&](auto careful) __attribute__((always_inline)) {
        constexpr bool kCareful = decltype(careful)::value;
        auto behind_of = [&](int s0) { return s0 + KT < s_end ? s0 + KT : s0; };
        lay_first(s_begin);
#pragma unroll
        for (int piece = 0; piece < 2 * SHARE; piece++) lay_piece(careful, stages[0], piece);
        lay_last(careful, flags[0]);
        request(behind_of(s_begin));
        __syncthreads();
        int at = 0;
        for (int s0 = s_begin; s0 < s_end; s0 += KT) {
            const int next = behind_of(s0);
            bool wild_tile = false;
            if constexpr (kCareful) {
                if (uniform((int32_t)flags[at]) != 0) {
                    asm volatile("");
                    __syncthreads();
                    if (tid == 0) flags[at] = 0u;
                    wild_tile = true;
                    lay_again(stages[at], s0);
                    request_values(next);
                }
            }
            uint32_t seen = 0;
            lay_first(next);
            if (__builtin_expect(s0 <= any_last && s0 + KT > any_first, 1)) {  // (uniform in the wavefront)
                tile(stages[at], stages[at ^ 1], s0, careful, seen);
            } else {
#pragma unroll
                for (int piece = 0; piece < 2 * SHARE; piece++) lay_piece(careful, stages[at ^ 1], piece);
            }
            lay_last(careful, flags[at ^ 1]);
            if constexpr (kCareful) {
                if (wild_tile) add_wild(stages[at], s0, seen);
            }
            request(behind_of(next));
            __syncthreads();
            at ^= 1;
        }
    };
    clear();
    if (tid < 3) (tid < 2 ? flags[tid] : again) = 0u;
    if (s_begin < s_end) {
        walk(std::false_type{});
        float odd = 0.0f;
        odd = __builtin_fmaf(l, 0.0f, odd);
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) odd = __builtin_fmaf(o[d][i], 0.0f, odd);
        if (__any(odd != odd) && lane == 0) again = 1u;
        __syncthreads();
        if (__builtin_expect(uniform((int32_t)again) != 0, 0)) {
            clear();
            request(s_begin);
            walk(std::true_type{});
        }
    }
    l += __shfl_xor(l, 32);
    if (!live) return;
    const bool whole = span.items == 1;
    float factor = 1.0f;
    float *state = nullptr;  // of this line and split: maximum, denominator, weighted means
    if (whole) {
        float denom = l, f = 1.0f;
        if (a.sinks != nullptr) {
            const float sink = Elem<T>::load(a.sinks, my_head) * kLog2e, top = fmaxf(m, sink);
            f = exp2f(m - top), denom = denom * f + exp2f(sink - top);
        }
        factor = denom == 0.0f ? 0.0f : f / denom;  // (a row that sees nothing: zeros)
    } else {
        factor = l == 0.0f ? 0.0f : 1.0f / l;  // (divided here, so that sums of the largest values do not leave float32)
        state = a.states + ((int64_t)item.slot * kLines + wave * 32 + col) * kState<D>;
        if (half == 0) *reinterpret_cast<float2 *>(state) = make_float2(m, l);
    }
    T *out = a.out + (int64_t)(item.s.start + my_row) * a.out_strides[0] + (int64_t)my_head * a.out_strides[1];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int c = 32 * d + 8 * g + 4 * half;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = o[d][4 * g + i] * factor;
            if (!whole) {
                *reinterpret_cast<float4 *>(state + 4 + c) = make_float4(v[0], v[1], v[2], v[3]);
            } else if (c < a.dim) {
                struct __attribute__((packed)) Four { T t[4]; };
                Four four;
#pragma unroll
                for (int i = 0; i < 4; i++) Elem<T>::store(four.t, i, v[i]);
                *reinterpret_cast<Four *>(out + c) = four;
            }
        }
}

// The splits' states merged: D / 4 threads a line, four splits' loads under way at a time.
template <int D> constexpr int kMergeLines = 256 / (D / 4);  // of a block
constexpr uint32_t kMergeBlocks = 2048;
template <typename T, int D>
__device__ __forceinline__ void merge_line(const PromptArgs<T> &a, const PagedItem &item, const Span &span, int part, int ln, int at) {
    const int rep = a.batch.rep, line = part * kLines + ln;
    if (ln >= kLines || line >= item.s.rows * rep) return;
    const int64_t stride = (int64_t)a.batch.key_heads * kLines * kState<D>;  // of a split's states
    const float *src = a.states + ((int64_t)item.slot * kLines + ln) * kState<D>;
    float top = kLowest, total = 0.0f, sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int z0 = 0; z0 < span.items; z0 += 4) {
        float2 m[4];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float *state = src + (z0 + i < span.items ? z0 + i : z0) * stride;
            m[i] = *reinterpret_cast<const float2 *>(state), v[i] = *reinterpret_cast<const float4 *>(state + 4 + at);
        }
        float most = top;
#pragma unroll
        for (int i = 0; i < 4; i++) most = fmaxf(most, m[i].x);
        // (the means' weights add up to 1 as they come, for the same reason)
        float w[4], all = total * exp2f(top - most);
        const float before = all;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = z0 + i < span.items ? m[i].y * exp2f(m[i].x - most) : 0.0f, all += w[i];
        top = most, total = all;
        const float share = all == 0.0f ? 0.0f : 1.0f / all, kept = before * share;
#pragma unroll
        for (int i = 0; i < 4; i++) sum[i] = kept == 0.0f ? 0.0f : sum[i] * kept;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float part = w[i] * share;
            if (part == 0.0f) continue;  // (a split that sees nothing, or nothing beside the others)
            sum[0] = __builtin_fmaf(v[i].x, part, sum[0]), sum[1] = __builtin_fmaf(v[i].y, part, sum[1]);
            sum[2] = __builtin_fmaf(v[i].z, part, sum[2]), sum[3] = __builtin_fmaf(v[i].w, part, sum[3]);
        }
    }
    const int head = item.head * rep + line % rep;
    float inv = 1.0f;
    if (a.sinks != nullptr) {
        const float sink = Elem<T>::load(a.sinks, head) * kLog2e, most = fmaxf(top, sink);
        total *= exp2f(top - most);
        inv = total == 0.0f ? 0.0f : total / (total + exp2f(sink - most));
    }
    struct __attribute__((packed)) Four { T t[4]; };
    Four four;
#pragma unroll
    for (int i = 0; i < 4; i++) Elem<T>::store(four.t, i, sum[i] * inv);
    *reinterpret_cast<Four *>(a.out + (int64_t)(item.s.start + line / rep) * a.out_strides[0] + (int64_t)head * a.out_strides[1] + at) = four;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const PromptArgs<T> a, uint32_t units) {
    constexpr int kThreads = D / 4;
    PagedItem item;
    if (!paged_item<kLines, 1, true>(a.batch, threadIdx.x & 63, blockIdx.x % units, a.length, item)) return;
    const int at = (int)threadIdx.x % kThreads * 4;
    const int part = item.s.parts - 1 - item.part;  // (items count the parts from the last)
    const Span span = span_of(a.batch, item, part);
    if ((int)threadIdx.x >= kMergeLines<D> * kThreads || span.items == 1 || at >= a.dim ||
        item.slot + (span.items - 1) * a.batch.key_heads >= a.slots)
        return;
    for (int first = (int)(blockIdx.x / units) * kMergeLines<D>; first < kLines; first += (int)(gridDim.x / units) * kMergeLines<D>)
        merge_line<T, D>(a, item, span, part, first + (int)threadIdx.x / kThreads, at);
}

template <typename T, int D>
int32_t launch_sized(const PromptArgs<T> &a, const PromptLaunch &r, hipStream_t s) {
    hipLaunchKernelGGL((prompt_kernel<T, D>), dim3(r.grid), dim3(64 * kWaves), 0, s, a);
    NVQ_LAUNCH_CHECK("prompt_attention");
    if (r.merge_units == 0) return NVQ_OK;
    // (blocks of several passes over a unit's lines from where they would be more than the chip holds: often nothing is split)
    const uint32_t all = (kLines + kMergeLines<D> - 1) / kMergeLines<D>, some = kMergeBlocks / r.merge_units, blocks = some < 1 ? 1 : some < all ? some : all;
    hipLaunchKernelGGL((prompt_merge_kernel<T, D>), dim3(r.merge_units * blocks), dim3(256), 0, s, a, r.merge_units);
    NVQ_LAUNCH_CHECK("prompt_attention merge");
    return NVQ_OK;
}

template <typename T>
int32_t launch_type(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, const PromptLaunch &r, hipStream_t s) {
    PromptArgs<T> a{};
    a.batch = r.batch;
    a.q = (const T *)o.q, a.k = (const T *)o.k, a.v = (const T *)o.v, a.sinks = (const T *)o.sinks, a.out = (T *)o.out;
    a.length = r.merge_units > 0 ? (int32_t *)o.workspace : nullptr;
    a.states = o.workspace == nullptr ? nullptr : (float *)((uint8_t *)o.workspace + kPlanBytes);
    for (int i = 0; i < 2; i++)
        a.q_strides[i] = d.q_strides[i], a.k_strides[i] = d.k_strides[i], a.v_strides[i] = d.v_strides[i], a.out_strides[i] = d.out_strides[i];
    a.dim = d.head_dim, a.turn = r.turn, a.back = r.back, a.slots = r.slots, a.scale = d.scale;
    switch (padded_dim(d.head_dim)) {
    case 64: return launch_sized<T, 64>(a, r, s);
    case 96: return launch_sized<T, 96>(a, r, s);
    case 128: return launch_sized<T, 128>(a, r, s);
    default: return launch_sized<T, 256>(a, r, s);
    }
}

}  // namespace
}  // namespace prompt
}  // namespace nvq
