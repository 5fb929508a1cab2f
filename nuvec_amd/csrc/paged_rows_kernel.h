// Attention of few lines (query rows x query heads of a key head) over a paged, affine-quantized key / value cache:
//     out[row, h, :] = softmax(scale * q[row, h, :] . K^T [masked] [, sink[h]]) . V
// K and V of the row's sequence, read through its page table, lengths and all from device memory.
//
// The bound is the stream of the cache.  Both products run on the matrix cores over the codes, which bfloat16 holds exactly, as in
// qattn.hip (its weights are three terms in every type, though): the 16 columns of v_mfma_f32_16x16x32 are (group of D, line), S^T = K . Q^T
// with zeros of Q outside a column's group, scale and bias of the group applied to the partial score, O^T = V^T . P^T with the weights times the
// column's group's scale.  A lane holds in S^T the keys 4 quarter .. + 3 of two halves of 16 keys, which are the eight keys of its operand P^T.
// Half a tile lies within one page (pages have 16 positions at least), so a tile's addresses are two scalars, looked up a tile ahead.
//
// Terms.  Queries are exact: one bfloat16 term, two in float16, three in float32.  The weights p x scale are two terms in bfloat16 and float16
// (16 bits: the result's own rounding is all that is left of the error; one term in bfloat16 was 1 to 3% faster and a result's error 1.4 times
// its rounding's), three in float32.  The codes of V count from the middle of their range: the operands themselves in float32, else by an
// operand of ones whose products with the same, rounded weights are taken off.  Scores, maxima, sums and accumulators are float32.
//
// Masked keys (behind the sequence's end, in front of a row or outside its window) are given no weight whatever their pages hold: their
// scores are replaced and their values' scales and biases too, which may be infinite or NaN.
#pragma once

#include "attention_codes.h"
#include "nvq_device.h"
#include "nvq_internal.h"
#include "paged_attention.h"
#include "paged_schedule.h"

namespace nvq {
namespace paged {

constexpr int kWaves = 4;
constexpr int kTile = kScheduleKeys;
// Where maxima start: under every score but the last thousandth of float32's range, and finite, so that a masked score's weight is
// exp2(-inf - m) = 0 from the first tile on.
constexpr float kLowest = -3.4e38f;

template <typename T>
struct RowsArgs {
    PagedBatch batch;
    const T *q, *ks, *kb, *vs, *vb, *sinks;
    const uint32_t *kw, *vw;
    T *out;
    int32_t *length;  // of the plan, for the merge; NULL: no merge
    float *states;    // [slots][LINES][kState<D>]: maximum of the base-2 scores, denominator, two unused, D weighted sums
    int64_t q_strides[2], out_strides[2];
    float scale;
};

namespace {

template <int D> constexpr int kState = D + 4;  // (rows of 16 bytes)

// Blocks on a compute unit.  Three need 168 registers at most: heads of 128 read their queries from LDS in every tile there.
template <typename T, int G> constexpr int rows_blocks() { return sizeof(T) == 4 || G == 4 ? 2 : 3; }
template <typename T, int D, int G> constexpr bool rows_queries_in_lds() { return rows_blocks<T, G>() == 3 && D == 128; }
template <typename T> constexpr int weight_terms() { return sizeof(T) == 4 ? 3 : 2; }

template <typename T, int BITS, int D, int G>
__global__ void __launch_bounds__(64 * kWaves, (rows_blocks<T, G>())) paged_rows_kernel(const RowsArgs<T> a, const int32_t *__restrict__ table) {
    constexpr int TQ = sizeof(T) == 4 ? 3 : Elem<T>::code == NVQ_BF16 ? 1 : 2, TP = weight_terms<T>();
    constexpr int R = 16 / G, KS = D / 32, ND = D / 16;  // lines; instructions of K per 16 keys; values of D per lane
    constexpr int kRowBytes = D * BITS / 8, kChunk = kRowBytes / 4, kSlot = BITS * ND;  // bytes of a quarter's codes; bits of a lane's slot
    constexpr bool kWide = sizeof(T) == 4, kOnes = !kWide;
    constexpr float kOff = kOffset<BITS, kWide>, kMiddle = 1 << (BITS - 1);
    constexpr uint32_t kOne = BITS == 8 ? 0x43004300u : 0x41C041C0u;  // two of kOff + kMiddle: 128, 24 (at 8 and 4 bits)
    __shared__ float part[kWaves][R][D + 1];
    __shared__ float wave_m[kWaves][R], wave_l[kWaves][R];
    constexpr bool kLdsQueries = rows_queries_in_lds<T, D, G>();
    __shared__ uint4 queries[kLdsQueries ? KS * TQ : 1][64];  // (the same in all wavefronts)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l = lane & 15, quarter = lane >> 4, g = l / R, line = l % R;
    const float scale = a.scale * kLog2e;
    const CodeConstants<BITS> constants;
    PagedItem item;
    if (!paged_item<R, 0, false>(a.batch, lane, blockIdx.x, a.length, item)) return;
    const int rep = a.batch.rep, hk = item.head, S = item.s.length, n = item.s.rows;
    const int lines = n * rep - item.part * R < R ? n * rep - item.part * R : R;  // of this unit
    // the keys that row i of n sees
    const int window = (int)(a.batch.window < S + 1 ? a.batch.window : S + 1);
    auto last_of = [&](int i) { return a.batch.causal ? S - n + i : S - 1; };
    auto first_of = [&](int i) { return window > 0 && a.batch.causal ? last_of(i) - window + 1 : 0; };
    const int i_first = item.part * R / rep, i_last = (item.part * R + lines - 1) / rep;
    const bool real = line < lines;
    const int r = item.part * R + (real ? line : 0), my_row = r / rep, my_head = hk * rep + r % rep;
    const int my_last = real ? last_of(my_row) : -1, my_first = first_of(my_row);
    const int all_last = uniform(last_of(i_first)), all_first = uniform(first_of(i_last));  // keys up to / from which all lines see
    const int split_begin = item.s.base + item.split * item.per * kTile;
    int s_begin = split_begin, s_end = item.splits == 1 ? S : split_begin + item.per * kTile < S ? split_begin + item.per * kTile : S;
    if (last_of(i_last) + 1 < s_end) s_end = last_of(i_last) + 1;
    if (first_of(i_first) / kTile * kTile > s_begin) s_begin = first_of(i_first) / kTile * kTile;
    s_begin = uniform(s_begin), s_end = uniform(s_end);

    // What a tile of 32 keys reads; the next tile's keys are requested when this one's have become operands, its values likewise.  Behind
    // the last tile an earlier one is requested again: under a condition the wait for this tile's values would be one for all requests.
    constexpr int kRun = G * (int)sizeof(T);  // bytes of a key's scales
    constexpr bool kOwn = kRun == 16;         // float32, four groups: the lane's own group alone
    struct Quad { uint32_t w[kOwn ? 4 : kRun]; };  // of four consecutive keys
    struct KeyTile {
        uint32_t c[2][kChunk / 4];
        Quad s[2], b[2];
    } kt;
    struct ValueTile {
        uint32_t c[8][(kSlot + 31) / 32];
        Quad s[2], b[2];
    } vt;
    // The rows (of all pages and heads) at which the halves of the tile at s0 lie, and the pages' ids before that, which are requested an
    // iteration ahead.  A half behind the end reads the last page.
    struct Halves { int64_t row[2]; };
    struct Ids { int32_t id[2], s0; };
    const int shift = a.batch.place.page_shift, last_column = S > 0 ? (S - 1) >> shift : 0, pages = (int)a.batch.place.pages;
    // (constant memory: the page table's entries are scalar loads, and the addresses that follow from them scalar)
    typedef const int32_t __attribute__((address_space(4))) *Columns;
    const Columns columns = (Columns)(uintptr_t)table + item.b * a.batch.place.stride;
    auto look_up = [&](int s0) __attribute__((always_inline)) {
        Ids o;
#pragma unroll
        for (int h = 0; h < 2; h++) o.id[h] = columns[uniform((s0 + 16 * h) >> shift < last_column ? (s0 + 16 * h) >> shift : last_column)];
        o.s0 = s0;
        return o;
    };
    auto place = [&](const Ids &of) __attribute__((always_inline)) {
        Halves o;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int32_t id = of.id[h], page = id < 0 ? 0 : id < pages ? id : pages - 1;
            o.row[h] = (((int64_t)page * a.batch.key_heads + hk) << shift) + ((of.s0 + 16 * h) & ((1 << shift) - 1));
        }
        return o;
    };
    auto four = [&](const T *p, const Halves &of, int h) __attribute__((always_inline)) {
        const uint8_t *at = reinterpret_cast<const uint8_t *>(p) + of.row[h] * kRun;
        Quad o;
        if constexpr (kOwn) {
#pragma unroll
            for (int i = 0; i < 4; i++) o.w[i] = load_any<uint32_t>(at + (uint32_t)(4 * quarter * kRun + 4 * g) + i * kRun);
        } else {
            o = load_any<Quad>(at + (uint32_t)(4 * quarter * kRun));
        }
        return o;
    };
    auto fetch_keys = [&](const Halves &of) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            struct Words { uint32_t w[kChunk / 4]; };
            const uint8_t *half = reinterpret_cast<const uint8_t *>(a.kw) + of.row[h] * kRowBytes;
            const Words w = *reinterpret_cast<const Words *>(half + (uint32_t)(l * kRowBytes + quarter * kChunk));
#pragma unroll
            for (int i = 0; i < kChunk / 4; i++) kt.c[h][i] = w.w[i];
            kt.s[h] = four(a.ks, of, h), kt.b[h] = four(a.kb, of, h);
        }
    };
    auto fetch_values = [&](const Halves &of) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint8_t *row = reinterpret_cast<const uint8_t *>(a.vw) + (of.row[j >> 2] + (j & 3)) * kRowBytes + (uint32_t)(4 * quarter * kRowBytes);
            if constexpr (kSlot == 64) {
                const uint2 w = *reinterpret_cast<const uint2 *>(row + 8 * l);
                vt.c[j][0] = w.x, vt.c[j][1] = w.y;
            } else if constexpr (kSlot == 32) {
                vt.c[j][0] = *reinterpret_cast<const uint32_t *>(row + 4 * l);
            } else {
                vt.c[j][0] = *reinterpret_cast<const uint16_t *>(row + 2 * l);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) vt.s[h] = four(a.vs, of, h), vt.b[h] = four(a.vb, of, h);
    };
    // Zeros for key i.
    auto clear = [](Quad &o, int i) {
        if constexpr (kRun == 2) o.w[i >> 1] &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
        for (int w = 0; w < (kOwn ? 1 : kRun / 4); w++) o.w[(kOwn ? 1 : kRun / 4) * i + w] = 0;
    };
    // The lane's own group of key i.
    const int down = 16 * (g & 1);
    const uint32_t half_of = g & 1 ? 0x03020C0Cu : 0x01000C0Cu;  // (its 16 bits above zeros: one byte permutation)
    auto pick = [&](const Quad &o, int i) {
        if constexpr (kOwn) {
            return u2f(o.w[i]);
        } else if constexpr (sizeof(T) == 4) {
            uint32_t w = o.w[G * i];
#pragma unroll
            for (int e = 1; e < G; e++) w = g == e ? o.w[G * i + e] : w;
            return u2f(w);
        } else {
            uint32_t w = o.w[G * i / 2];
            if constexpr (G == 4) w = g >= 2 ? o.w[2 * i + 1] : w;
            if constexpr (Elem<T>::code == NVQ_BF16) {
                if constexpr (G == 1) return u2f(i & 1 ? w & 0xFFFF0000u : w << 16);
                return u2f(__builtin_amdgcn_perm(0u, w, half_of));
            } else {
                return (float)__builtin_bit_cast(f16_t, (uint16_t)(w >> (G == 1 ? 16 * (i & 1) : down)));
            }
        }
    };

    floatx4_t acc[ND], ones = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = kLowest, denom = 0.0f, accb = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; i++) acc[i] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int step = kWaves * kTile;
    const int s_wave = s_begin + wave * kTile;
    Halves next{};
    if (s_wave < s_end) {
        const Ids first = look_up(s_wave), second = look_up(s_wave + step < s_end ? s_wave + step : s_wave);
        const Halves here = place(first);
        fetch_keys(here);
        fetch_values(here);
        next = place(second);
    }
    // The queries' operands: column (g, line), zeros outside the group; their sums per column.
    uint4 qf[KS][TQ];
    float qsum = 0.0f;
    const T *query = a.q + (int64_t)(item.s.start + my_row) * a.q_strides[0] + (int64_t)my_head * a.q_strides[1];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int at = quarter * (D / 4) + 8 * s;  // (eight values of one group)
        struct __attribute__((packed)) Eight { T v[8]; };
        const Eight eight = *reinterpret_cast<const Eight *>(query + at);
        const bool mine = real && at / (D / G) == g;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = mine ? Elem<T>::load(eight.v, code_at<BITS>(j)) : 0.0f, qsum += v[j];
        uint32_t t[4][TQ];
#pragma unroll
        for (int j = 0; j < 4; j++) split_pair<TQ>(v[2 * j], v[2 * j + 1], t[j]);
#pragma unroll
        for (int i = 0; i < TQ; i++) {
            qf[s][i] = make_uint4(t[0][i], t[1][i], t[2][i], t[3][i]);
            if (kLdsQueries && wave == 0) queries[s * TQ + i][lane] = qf[s][i];
        }
    }
    if (kLdsQueries) __syncthreads();
    qsum += __shfl_xor(qsum, 16);
    qsum += __shfl_xor(qsum, 32);

    for (int s0 = s_wave; s0 < s_end; s0 += step) {
        const Ids behind = look_up(s0 + 2 * step < s_end ? s0 + 2 * step : s0);
        float score[8];
        if constexpr (kLdsQueries) {
            asm volatile("" ::: "memory");  // (not kept from the tile before)
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < TQ; i++) qf[s][i] = queries[s * TQ + i][lane];
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            floatx4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const uint4 kf = BITS == 8 ? eight_codes<BITS, kWide>(constants, kt.c[h][2 * s], kt.c[h][2 * s + 1]) : eight_codes<BITS, kWide>(constants, kt.c[h][s], 0);
#pragma unroll
                for (int i = 0; i < TQ; i++) sum = mfma16(kf, qf[s][i], sum);
            }
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++) {
                const float sk = pick(kt.s[h], r4), bk = pick(kt.b[h], r4);
                float v = __builtin_fmaf(sk, sum[r4], __builtin_fmaf(-kOff, sk, bk) * qsum);
                // the groups of a row: columns R apart
                if constexpr (G == 4) v += u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), 0x124, 0xF, 0xF, true));
                if constexpr (G >= 2) v += u2f((uint32_t)__builtin_amdgcn_mov_dpp((int)f2u(v), 0x128, 0xF, 0xF, true));
                score[4 * h + r4] = v * scale;
            }
        }
        if (s0 + kTile - 1 > all_last || s0 < all_first || s0 + kTile > S) {
            asm volatile("");  // (a branch: as selects it would cost every tile)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = s0 + 16 * (j >> 2) + 4 * quarter + (j & 3);
                if (key > my_last || key < my_first || key >= S) {
                    score[j] = -INFINITY;
                    clear(vt.s[j >> 2], j & 3), clear(vt.b[j >> 2], j & 3);
                }
            }
        }
        fetch_keys(next);
        float top = score[0];
#pragma unroll
        for (int j = 1; j < 8; j++) top = fmaxf(top, score[j]);
        // The sums are rescaled only when a maximum has grown by more than 2^8; until then weights are at most 2^8.
        if (__any(top > m + 8.0f)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float m_new = fmaxf(m, top), f = exp2f(m - m_new);
            m = m_new, denom *= f, accb *= f;
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++) {
                ones[r4] *= f;
#pragma unroll
                for (int i = 0; i < ND; i++) acc[i][r4] *= f;
            }
        }
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float p = __builtin_amdgcn_exp2f(score[j] - m);
            denom += p;
            const float sv = pick(vt.s[j >> 2], j & 3), bv = pick(vt.b[j >> 2], j & 3);
            accb = __builtin_fmaf(p, __builtin_fmaf(kMiddle, sv, bv), accb);
            w[j] = p * sv;
        }
        uint32_t t[4][TP];
        uint4 pf[TP];
#pragma unroll
        for (int j = 0; j < 4; j++) split_pair<TP>(w[2 * j], w[2 * j + 1], t[j]);
#pragma unroll
        for (int e = 0; e < TP; e++) {
            pf[e] = make_uint4(t[0][e], t[1][e], t[2][e], t[3][e]);
            if constexpr (kOnes) ones = mfma16(make_uint4(kOne, kOne, kOne, kOne), pf[e], ones);
        }
        // value i of the lane's slot, two keys a word
#pragma unroll
        for (int i = 0; i < ND; i++) {
            uint32_t p[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (kWide) {
                    const int at = BITS * i / 32, sh = BITS * i % 32;
                    constexpr uint32_t mask = (1u << BITS) - 1u;
                    p[j] = pack_exact((float)((vt.c[2 * j][at] >> sh) & mask) + kOff, (float)((vt.c[2 * j + 1][at] >> sh) & mask) + kOff);
                } else if constexpr (BITS == 8) {
                    const uint32_t x = vt.c[2 * j][i / 4] >> (8 * (i % 4)), y = vt.c[2 * j + 1][i / 4] >> (8 * (i % 4));
                    p[j] = pack_exact((float)(x & 0xFFu), (float)(y & 0xFFu));
                } else {
                    // sixteen bits of each key that hold the code, side by side
                    const bool high = BITS * i + BITS > 16;
                    const uint32_t both = __builtin_amdgcn_perm(vt.c[2 * j + 1][0], vt.c[2 * j][0], high ? 0x07060302u : 0x05040100u);
                    p[j] = two_codes(constants, both, BITS * i - (high ? 16 : 0));
                }
            }
            const uint4 vf = make_uint4(p[0], p[1], p[2], p[3]);
#pragma unroll
            for (int e = 0; e < TP; e++) acc[i] = mfma16(vf, pf[e], acc[i]);
        }
        fetch_values(next);
        next = place(behind);
    }

    // merge: the block's maximum, every wavefront scaled to it, the wavefronts added up
    denom += __shfl_xor(denom, 16), accb += __shfl_xor(accb, 16);
    denom += __shfl_xor(denom, 32), accb += __shfl_xor(accb, 32);
    if (lane < R) wave_m[wave][line] = m, wave_l[wave][line] = denom;
#pragma unroll
    for (int i = 0; i < ND; i++)
#pragma unroll
        for (int r4 = 0; r4 < 4; r4++) {
            const int at = ND * (4 * quarter + r4) + i;  // of D: this column's group has it or another column's
            if (at / (D / G) == g) part[wave][line][at] = acc[i][r4] - (kOnes ? ones[r4] : 0.0f) + accb;
        }
    __syncthreads();
    for (int e = tid; e < lines * D; e += 64 * kWaves) {
        const int ln = e / D, at = e % D;
        float top = kLowest;
#pragma unroll
        for (int w = 0; w < kWaves; w++) top = fmaxf(top, wave_m[w][ln]);
        float sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float f = exp2f(wave_m[w][ln] - top);
            total = __builtin_fmaf(wave_l[w][ln], f, total);
            sum = __builtin_fmaf(part[w][ln][at], f, sum);
        }
        if (item.splits == 1) {
            const int rr = item.part * R + ln, head = hk * rep + rr % rep;
            if (a.sinks != nullptr) {
                const float sink = Elem<T>::load(a.sinks, head) * kLog2e, t2 = fmaxf(top, sink), f = exp2f(top - t2);
                sum *= f, total = total * f + exp2f(sink - t2);
            }
            // (a row that sees nothing: zeros)
            Elem<T>::store(a.out + (int64_t)(item.s.start + rr / rep) * a.out_strides[0] + (int64_t)head * a.out_strides[1], at, total == 0.0f ? 0.0f : sum / total);
        } else {
            float *dst = a.states + ((int64_t)item.slot * R + ln) * kState<D>;
            if (at == 0) dst[0] = top, dst[1] = total;
            dst[4 + at] = sum;
        }
    }
}

// The splits of a line merged, one block a line: its wavefronts take them in turn, eight loads under way at a time, and add up through LDS.
template <typename T, int D, int LINES>
__device__ __forceinline__ void merge_few(const RowsArgs<T> &a, int32_t unit, int ln) {
    constexpr int V = D / 64;
    __shared__ float sums[kWaves][D], tops[kWaves], totals[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PagedItem item;
    if (!paged_item<LINES, 0, true>(a.batch, lane, unit, a.length, item)) return;
    const int rep = a.batch.rep, line = item.part * LINES + ln;
    if (line >= item.s.rows * rep) return;
    const int64_t stride = (int64_t)a.batch.key_heads * LINES * kState<D>;  // of a split's states
    const float *src = a.states + ((int64_t)item.slot * LINES + ln) * kState<D>;
    float top = kLowest, total = 0.0f, sum[V] = {};
    for (int z0 = wave; z0 < item.splits; z0 += 8 * kWaves) {
        float m[8], d[8], v[8][V];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int z = z0 + kWaves * i < item.splits ? z0 + kWaves * i : z0;
            const float *state = src + z * stride;
            m[i] = state[0], d[i] = state[1];
#pragma unroll
            for (int e = 0; e < V; e++) v[i][e] = state[4 + V * lane + e];
        }
        float most = top;
#pragma unroll
        for (int i = 0; i < 8; i++) most = fmaxf(most, m[i]);
        const float f = exp2f(top - most);
        top = most, total *= f;
#pragma unroll
        for (int e = 0; e < V; e++) sum[e] *= f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float w = z0 + kWaves * i < item.splits ? exp2f(m[i] - top) : 0.0f;
            total = __builtin_fmaf(d[i], w, total);
#pragma unroll
            for (int e = 0; e < V; e++) sum[e] = __builtin_fmaf(v[i][e], w, sum[e]);
        }
    }
    tops[wave] = top, totals[wave] = total;
#pragma unroll
    for (int e = 0; e < V; e++) sums[wave][V * lane + e] = sum[e];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; w++) top = fmaxf(top, tops[w]);
    total = 0.0f;
#pragma unroll
    for (int e = 0; e < V; e++) sum[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        const float f = exp2f(tops[w] - top);
        total = __builtin_fmaf(totals[w], f, total);
#pragma unroll
        for (int e = 0; e < V; e++) sum[e] = __builtin_fmaf(sums[w][V * lane + e], f, sum[e]);
    }
    const int head = item.head * rep + line % rep;
    if (a.sinks != nullptr) {
        const float sink = Elem<T>::load(a.sinks, head) * kLog2e, most = fmaxf(top, sink), f = exp2f(top - most);
        total = __builtin_fmaf(total, f, exp2f(sink - most));
#pragma unroll
        for (int e = 0; e < V; e++) sum[e] *= f;
    }
    T *out = a.out + (int64_t)(item.s.start + line / rep) * a.out_strides[0] + (int64_t)head * a.out_strides[1];
#pragma unroll
    for (int e = 0; e < V; e++) Elem<T>::store(out, V * lane + e, total == 0.0f ? 0.0f : sum[e] / total);
}

template <typename T, int D, int LINES>
__global__ void __launch_bounds__(64 * kWaves) paged_merge_kernel(const RowsArgs<T> a) { merge_few<T, D, LINES>(a, blockIdx.x, blockIdx.y); }

template <typename T, int BITS, int D, int G>
int32_t launch_rows_sized(const RowsArgs<T> &a, const PagedLaunch &r, hipStream_t s) {
    hipLaunchKernelGGL((paged_rows_kernel<T, BITS, D, G>), dim3(r.grid), dim3(64 * kWaves), 0, s, a, a.batch.place.table);
    NVQ_LAUNCH_CHECK("paged_attention");
    if (r.merge_units > 0 && !r.merged_later) {
        hipLaunchKernelGGL((paged_merge_kernel<T, D, 16 / G>), dim3(r.merge_units, r.merge_lines), dim3(64 * kWaves), 0, s, a);
        NVQ_LAUNCH_CHECK("paged_attention merge");
    }
    return NVQ_OK;
}

template <typename T, int BITS>
int32_t launch_rows_bits(const RowsArgs<T> &a, const nvq_paged_desc &c, const PagedLaunch &r, hipStream_t s) {
    if (c.head_dim == 64) return c.group_size == 32 ? launch_rows_sized<T, BITS, 64, 2>(a, r, s) : launch_rows_sized<T, BITS, 64, 1>(a, r, s);
    if (c.group_size == 32) return launch_rows_sized<T, BITS, 128, 4>(a, r, s);
    return c.group_size == 64 ? launch_rows_sized<T, BITS, 128, 2>(a, r, s) : launch_rows_sized<T, BITS, 128, 1>(a, r, s);
}

template <typename T>
RowsArgs<T> rows_args(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &r) {
    RowsArgs<T> a{};
    a.batch = r.batch;
    a.q = (const T *)o.q, a.ks = (const T *)o.ks, a.kb = (const T *)o.kb, a.vs = (const T *)o.vs, a.vb = (const T *)o.vb, a.sinks = (const T *)o.sinks;
    a.kw = (const uint32_t *)o.kw, a.vw = (const uint32_t *)o.vw, a.out = (T *)o.out, a.states = (float *)((char *)o.workspace + r.states + kPlanBytes);
    a.length = r.merge_units > 0 ? (int32_t *)((char *)o.workspace + r.states) : nullptr;
    for (int i = 0; i < 2; i++) a.q_strides[i] = d.q_strides[i], a.out_strides[i] = d.out_strides[i];
    a.scale = d.scale;
    return a;
}

template <typename T>
int32_t launch_rows(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &r, hipStream_t s) {
    const RowsArgs<T> a = rows_args<T>(d, o, r);
    return d.cache.bits == 4 ? launch_rows_bits<T, 4>(a, d.cache, r, s) : launch_rows_bits<T, 8>(a, d.cache, r, s);
}

}  // namespace
}  // namespace paged
}  // namespace nvq
