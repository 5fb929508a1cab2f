// Attention of many lines (query rows x query heads of a key head) over a paged, affine-quantized key / value cache, float16 and bfloat16.
//
// The products run on the matrix cores over the codes, as for few lines (paged_rows_kernel.h): scale and bias of a key's groups
// are applied to the float32 scores, those of a value's to the softmax's weights, so that no key or value is rounded.
// A block has 128 lines, a wavefront 16 of them: S^T = K . Q^T with v_mfma_f32_16x16x32, a group of the head at a time, leaves a lane
// with 4 of 16 keys of ONE line; its maximum and sum are in-lane but for two exchanges, and the weights of 32 keys are already the operand of
// O^T = V^T . P^T, whose keys are stored in the order in which the lanes hold them.
//
// 64 keys at a time become operands in LDS, once for the block: expanded by each wavefront for itself they would cost it six times
// the instructions.  The next 64 keys' codes are requested before, and expanded after, this tile's products; two buffers, one barrier a tile.  A
// code becomes an element in two instructions for two of them (16 + code in the mantissa; 8 bits through float32); the 16 is taken off the sums
// again, by the biases (in float16 the outputs', and the middle of V's codes with it, by the sum of the rounded weights).  The keys'
// biases are one more product (qb below).
//
// Terms: queries are exact in their own type.  Weights x scale are two terms of bfloat16, 16 bits (one where the element type is bfloat16: 123 us
// instead of 140 below, and the results' error 1.4 times that of their rounding; with two it is that of the rounding).
//
// Measured: 1024 rows of 32 heads of 128 over 4096 positions, 8 key heads, 4 bits in groups of 64, bfloat16: 140 us, 430 TFLOP/s (groups of 128:
// 121, of 32: 180: each group of a head has its own scaling of scores and weights); 2048 rows over as many positions 114 us, 1024 47 us, 512
// 28 us.  While a compute unit is busy its vector units are at 61%, LDS at 50%, the matrix cores at 34%.  With one term a block alone took nearly
// as long for a tile as two that share a compute unit, and the same with 32 lines a wavefront (v_mfma_f32_32x32x16, four wavefronts of 256
// registers) is as fast over a long prefix and 2 to 15% slower on the diagonal; eight of those wavefronts with 256 lines to a block 5% faster at
// 1024 rows over 4096 and 15% slower at 2048 over 2048; sixteen wavefronts of 16 lines and tiles of 128 keys 15 to 30% slower; scales laid out
// by products instead of read from LDS: no faster.
#pragma once

#include "paged_rows_kernel.h"

namespace nvq {
namespace paged {
namespace {

constexpr int kPromptWaves = 8, kPromptLines = 16 * kPromptWaves, kStageKeys = 64;

// Eight codes of a row as an operand of the element type, value code_at<BITS>(j) of them in place j, each plus key_offset.
template <typename T, int BITS> constexpr float key_offset = BITS == 4 ? 16.0f : Elem<T>::code == NVQ_BF16 ? 0.0f : 1024.0f;
template <typename T, int BITS>
__device__ __forceinline__ uint4 key_codes(const CodeConstants<BITS == 8 ? 4 : BITS> &c, uint32_t w0, uint32_t w1) {
    if constexpr (BITS == 8 && Elem<T>::code == NVQ_BF16) {
        return make_uint4(pack_exact(qmf::ubyte_to_float<0>(w0), qmf::ubyte_to_float<1>(w0)), pack_exact(qmf::ubyte_to_float<2>(w0), qmf::ubyte_to_float<3>(w0)),
                          pack_exact(qmf::ubyte_to_float<0>(w1), qmf::ubyte_to_float<1>(w1)), pack_exact(qmf::ubyte_to_float<2>(w1), qmf::ubyte_to_float<3>(w1)));
    } else if constexpr (BITS == 8) {  // 1024 + code: the low bits of the mantissa
        auto two = [](uint32_t w, bool high) { return __builtin_amdgcn_perm(0u, w, high ? 0x0C030C02u : 0x0C010C00u) | 0x64006400u; };
        return make_uint4(two(w0, false), two(w0, true), two(w1, false), two(w1, true));
    } else if constexpr (Elem<T>::code == NVQ_BF16) {
        return make_uint4(two_codes(c, w0, 0), two_codes(c, w0, 4), two_codes(c, w0, 8), two_codes(c, w0, 12));
    } else {  // 16 + code, in float16 at bit 6
        auto two = [](uint32_t z, int at) { return ((at >= 6 ? z >> (at - 6) : z << (6 - at)) & 0x03C003C0u) | 0x4C004C00u; };
        return make_uint4(two(w0, 0), two(w0, 4), two(w0, 8), two(w0, 12));
    }
}

// What a unit's lines see, keys from `begin` (rounded down to a tile) to `end`, and how its items share them: evenly, `keys` each, so that the first lines of
// a prompt, which see less than the last, are shorter items rather than some whole and some empty ones (the 1024 rows above 137 us so).  An item
// that has them all writes the result.
struct PromptSpan {
    int32_t begin, end, keys, items;
};
__device__ __forceinline__ PromptSpan prompt_span(const PagedBatch &a, const PagedItem &item, int part) {
    const int32_t from = part * kPromptLines, lines = item.s.rows * a.rep, to = lines - from < kPromptLines ? lines : from + kPromptLines;
    int32_t begin = 0, end = item.s.length;
    if (a.causal) {
        const int32_t before = item.s.length - item.s.rows, seen = before + (to - 1) / a.rep + 1;
        const int64_t first = a.window > 0 ? before + from / a.rep + 1 - a.window : 0;
        end = seen < end ? seen : end, begin = first > 0 ? (int32_t)first / kTile * kTile : 0;
    }
    PromptSpan s{uniform(begin), uniform(end), 0, 1};
    const int32_t tiles = end > begin ? (end - begin + kTile - 1) / kTile : 0;
    int32_t per = (tiles + item.splits - 1) / item.splits;
    per = per > a.least ? per : a.least;
    s.keys = uniform(item.splits == 1 ? tiles * kTile : per * kTile), s.items = uniform(item.splits == 1 || tiles <= per ? 1 : (tiles + per - 1) / per);
    return s;
}

// Keys x queries, in the element type.
template <typename T>
__device__ __forceinline__ floatx4_t key_product(uint4 k, uint4 q, floatx4_t c) {
    if constexpr (Elem<T>::code == NVQ_BF16) {
        return mfma16(k, q, c);
    } else {
        typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, k), __builtin_bit_cast(f16x8_t, q), c, 0, 0, 0);
    }
}

template <typename T, int BITS, int D, int G>
__global__ void __launch_bounds__(64 * kPromptWaves, 4) paged_prompt_kernel(const RowsArgs<T> a, const int32_t *__restrict__ table) {
    constexpr int TP = weight_terms<T>();
    constexpr int KS = D / 32, ND = D / 16, GS = KS / G, GB = ND / G;                  // steps of K, blocks of D; of a group
    constexpr int kRowBytes = D * BITS / 8, kQuarter = kRowBytes / 4, kShare = kQuarter / 2;  // a row; a quarter; a thread's share of the keys' codes
    constexpr int kChunks = D / 64, kVals = D / 32, kSlot = BITS * kVals;              // of a thread: eight-code chunks; values of a row and their bits
    // Where the values' codes count from: float16, the middle of their range, taken off by the sum of the same, rounded weights; bfloat16, whose two terms
    // hold 16 bits where the result has 8, the operands' own zero, taken off the bias.
    constexpr bool kOnes = Elem<T>::code != NVQ_BF16;
    constexpr float kOff = key_offset<T, BITS>, kValueOff = BITS == 4 ? 16.0f : 0.0f, kMiddle = kOnes ? 1 << (BITS - 1) : -kValueOff;
    // Operands, 16 bytes a lane, with gaps, so that what 16 lanes write at once falls on different banks.
    struct Stage {
        uint4 keys[4][KS][64 + 2];         // [16 keys][step][quarter of the step x key]
        uint4 values[2][ND][64 + 1];       // [32 keys][block][run of four keys of each half x value]
        uint4 key_bias[4][64];             // [16 keys][group x key]: terms of their products with the queries' sums
        float scale[3][G][kStageKeys];     // of keys, of values, the values' biases
        uint16_t wild[2][G][2];            // a bit for every key whose value's scale or bias is not finite
    };
    static_assert(4 * sizeof(Stage) <= 160 * 1024);
    __shared__ Stage stages[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quarter = lane >> 4;
    PagedItem item;
    if (!paged_item<kPromptLines, 1, false>(a.batch, lane, blockIdx.x, a.length, item)) return;
    const int rep = a.batch.rep, hk = item.head, S = item.s.length, n = item.s.rows;
    const int part = item.s.parts - 1 - item.part;  // (the lines that see most first)
    const int lines = n * rep;
    const int window = (int)(a.batch.window < S + 1 ? a.batch.window : S + 1);
    auto last_of = [&](int i) { return a.batch.causal ? S - n + i : S - 1; };
    auto first_of = [&](int i) { return window > 0 && a.batch.causal ? last_of(i) - window + 1 : 0; };
    // the block's keys
    const PromptSpan span = prompt_span(a.batch, item, part);
    if (item.split >= span.items) return;
    const int s_begin = uniform(span.begin + item.split * span.keys), s_end = uniform(span.end < s_begin + span.keys ? span.end : s_begin + span.keys);
    // the wavefront's lines
    const int r0 = part * kPromptLines + wave * 16, r = r0 + col;
    const bool live = r < lines;
    const int my_row = (live ? r : lines - 1) / rep, my_head = hk * rep + (live ? r % rep : 0);
    const int my_last = last_of(my_row), my_first = first_of(my_row);
    const int w_first = (r0 < lines ? r0 : lines - 1) / rep, w_last = (r0 + 15 < lines ? r0 + 15 : lines - 1) / rep;
    const int all_last = uniform(last_of(w_first)), all_first = uniform(first_of(w_last));                       // keys up to / from which all of them see
    const int any_last = uniform(r0 < lines ? last_of(w_last) : -1), any_first = uniform(first_of(w_first));  // and any does

    uint4 qf[KS];
    float qsum[G];
#pragma unroll
    for (int g = 0; g < G; g++) qsum[g] = 0.0f;
    const T *query = a.q + (int64_t)(item.s.start + my_row) * a.q_strides[0] + (int64_t)my_head * a.q_strides[1];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const uint4 w = load_any<uint4>(query + 32 * s + 8 * quarter);
        T t[8], to[8];
        __builtin_memcpy(t, &w, 16);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) to[j] = t[code_at<BITS>(j)], sum += Elem<T>::load(t, j);
        __builtin_memcpy(&qf[s], to, 16);
        qsum[s / GS] += sum;
    }
    // The biases' share of a score, sum over the groups of bias x (sum of the group's queries), is one more product: both as three bfloat16 terms
    // h, m, l, whose six largest products are the contraction (h h, h m, m h, h l, l h, m m), a group in each quarter of it.
    uint4 qb = make_uint4(0u, 0u, 0u, 0u);
    {
        float sum = 0.0f;
#pragma unroll
        for (int g = 0; g < G; g++) {
            float all = qsum[g] + __shfl_xor(qsum[g], 16);
            all += __shfl_xor(all, 32);
            if (quarter == g) sum = all;
        }
        uint32_t t[3];
        split_pair<3>(sum, sum, t);
        const uint32_t hm = (t[0] & 0xFFFFu) | (t[1] & 0xFFFF0000u), hl = (t[0] & 0xFFFFu) | (t[2] & 0xFFFF0000u);
        qb = make_uint4(hm, hl, hm, 0u);
    }

    // ── staging ──
    const CodeConstants<4> constants;
    const float scale = a.scale * kLog2e;
    // The 16 keys that two wavefronts expand lie in one page: their place is a scalar, whose page is looked up a tile ahead.
    const int my_keys = wave >> 1, share = wave & 1;
    const int shift = a.batch.place.page_shift, last_column = S > 0 ? (S - 1) >> shift : 0, pages = (int)a.batch.place.pages;
    typedef const int32_t __attribute__((address_space(4))) *Columns;  // (constant memory: scalar loads)
    const Columns columns = (Columns)(uintptr_t)table + item.b * a.batch.place.stride;
    auto look_up = [&](int s0) __attribute__((always_inline)) {
        const int column = (s0 + 16 * my_keys) >> shift;
        return columns[uniform(column < last_column ? column : last_column)];  // (a tile behind the end reads the last page)
    };
    // This lane's: a share of a quarter of a key's codes; of four values (keys 4 v_run .. + 3 of the sixteen) a share of a sixteenth of the
    // codes; a scale and a bias of one group, of a key in the one wavefront and of a value in the other.
    const int k_key = lane >> 2, k_quarter = lane & 3;
    const int v_slot = lane & 15, v_run = lane >> 4;
    const int s_key = lane & 15, s_group = lane >> 4 < G ? lane >> 4 : 0;
    uint32_t kc[(kShare + 3) / 4], vc[4][(kSlot + 31) / 32];
    T sc, bc;
    bool s_real;
    auto request = [&](int32_t id, int s0) __attribute__((always_inline)) {
        const int32_t page = id < 0 ? 0 : id < pages ? id : pages - 1;
        const int64_t row = (((int64_t)page * a.batch.key_heads + hk) << shift) + ((s0 + 16 * my_keys) & ((1 << shift) - 1));
        struct Words { uint32_t w[kShare / 4]; };
        const Words w = *reinterpret_cast<const Words *>(reinterpret_cast<const uint8_t *>(a.kw) + row * kRowBytes + (uint32_t)(lane * kQuarter + share * kShare));
#pragma unroll
        for (int i = 0; i < kShare / 4; i++) kc[i] = w.w[i];
        const uint8_t *rows = reinterpret_cast<const uint8_t *>(a.vw) + row * kRowBytes;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint8_t *at = rows + (uint32_t)(4 * v_run * kRowBytes + (kRowBytes / 16) * v_slot + share * (kSlot / 8)) + j * kRowBytes;
            if constexpr (kSlot == 64) {
                const uint2 v = *reinterpret_cast<const uint2 *>(at);
                vc[j][0] = v.x, vc[j][1] = v.y;
            } else if constexpr (kSlot == 32) {
                vc[j][0] = *reinterpret_cast<const uint32_t *>(at);
            } else if constexpr (kSlot == 16) {
                vc[j][0] = *reinterpret_cast<const uint16_t *>(at);
            } else {
                vc[j][0] = *at;
            }
        }
        const int64_t from = (row + s_key) * G + s_group;
        sc = (share != 0 ? a.vs : a.ks)[from], bc = (share != 0 ? a.vb : a.kb)[from];
        s_real = s0 + 16 * my_keys + s_key < S;
    };
    auto expand = [&](Stage &to) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kChunks; j++) {
            const int c = (D / 32) * k_quarter + kChunks * share + j;  // (step c / 4, quarter c % 4)
            to.keys[my_keys][c >> 2][16 * (c & 3) + k_key] = key_codes<T, BITS>(constants, kc[BITS == 8 ? 2 * j : j], BITS == 8 ? kc[2 * j + 1] : 0u);
        }
#pragma unroll
        for (int i = 0; i < kVals; i++) {
            const int d = (D / 16) * v_slot + kVals * share + i;
            uint32_t p[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if constexpr (BITS == 8) {
                    const uint32_t x = vc[2 * j][i / 4] >> (8 * (i % 4)), y = vc[2 * j + 1][i / 4] >> (8 * (i % 4));
                    p[j] = pack_exact((float)(x & 0xFFu), (float)(y & 0xFFu));
                } else {
                    const uint32_t both = __builtin_amdgcn_perm(vc[2 * j + 1][0], vc[2 * j][0], i >= 4 ? 0x07060302u : 0x05040100u);
                    p[j] = two_codes(constants, both, 4 * (i & 3));
                }
            }
            reinterpret_cast<uint2 *>(&to.values[my_keys >> 1][d >> 4][16 * v_run + (d & 15)])[my_keys & 1] = make_uint2(p[0], p[1]);
        }
        // Keys: both with the softmax's scale, the bias without the codes' offset; values: the bias from the middle of the codes' range.  What lies
        // behind the sequence's end may hold anything: zeros.
        const float v = Elem<T>::load(&sc, 0), b = Elem<T>::load(&bc, 0);
        float own = share != 0 ? v : v * scale, with = share != 0 ? __builtin_fmaf(kMiddle, v, b) : __builtin_fmaf(-kOff, v, b) * scale;
        const bool wild = share != 0 && !(fabsf(with) < INFINITY && fabsf(own) < INFINITY), used = s_real && !wild;
        own = used ? own : 0.0f, with = used ? with : 0.0f;
        const uint64_t all = __ballot(wild && s_real);
        if (lane >> 4 < G) {
            to.scale[share][s_group][16 * my_keys + s_key] = own;
            if (share != 0) {
                to.scale[2][s_group][16 * my_keys + s_key] = with;
                if (s_key == 0) to.wild[my_keys >> 1][s_group][my_keys & 1] = (uint16_t)(all >> (lane & 48));
            }
        }
        if (share == 0) {
            with = lane >> 4 < G ? with : 0.0f;  // (no more groups: zeros)
            uint32_t t[3];
            split_pair<3>(with, with, t);
            to.key_bias[my_keys][lane] = make_uint4(t[0], (t[1] & 0xFFFFu) | (t[0] & 0xFFFF0000u), (t[2] & 0xFFFFu) | (t[1] & 0xFFFF0000u), 0u);
        }
    };

    const floatx4_t zeros = {0.0f, 0.0f, 0.0f, 0.0f};
    floatx4_t o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = zeros;
    float m = kLowest, l = 0.0f, ones[G], accb[G];
#pragma unroll
    for (int g = 0; g < G; g++) ones[g] = accb[g] = 0.0f;

    // The weights of 32 keys, half `sub` of the stage, times their values.
    auto values = [&](const Stage &from, int sub, const float (&x)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            uint32_t p[TP][4];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int at = 32 * sub + 16 * t + 4 * quarter;
                const float4 sv = *reinterpret_cast<const float4 *>(&from.scale[1][g][at]), bv = *reinterpret_cast<const float4 *>(&from.scale[2][g][at]);
                const float *e = x + 4 * t;
                accb[g] = __builtin_fmaf(e[0], bv.x, accb[g]), accb[g] = __builtin_fmaf(e[1], bv.y, accb[g]);
                accb[g] = __builtin_fmaf(e[2], bv.z, accb[g]), accb[g] = __builtin_fmaf(e[3], bv.w, accb[g]);
                uint32_t w[TP];
                split_pair<TP>(sv.x * e[0], sv.y * e[1], w);
#pragma unroll
                for (int i = 0; i < TP; i++) p[i][2 * t] = w[i];
                split_pair<TP>(sv.z * e[2], sv.w * e[3], w);
#pragma unroll
                for (int i = 0; i < TP; i++) p[i][2 * t + 1] = w[i];
            }
            if constexpr (kOnes) {
                typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
                const pair_t one2 = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
                for (int i = 0; i < TP; i++)
#pragma unroll
                    for (int w = 0; w < 4; w++) ones[g] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair_t, p[i][w]), one2, ones[g], false);
            }
#pragma unroll
            for (int d = g * GB; d < (g + 1) * GB; d += 2) {  // (two at a time: no product waits for the one in front of it; 142 -> 140 us)
                const uint4 v0 = from.values[sub][d][lane], v1 = from.values[sub][d + 1][lane];
#pragma unroll
                for (int i = 0; i < TP; i++) {
                    const uint4 w = make_uint4(p[i][0], p[i][1], p[i][2], p[i][3]);
                    o[d] = mfma16(v0, w, o[d]), o[d + 1] = mfma16(v1, w, o[d + 1]);
                }
            }
        }
    };
    // A tile of 64 keys from s0 on: the scores, one look at their maximum, the weights and their products.  x[u][4 t + e]: key 32 u + 16 t + 4 quarter + e.
    auto tile = [&](const Stage &from, int s0) __attribute__((always_inline)) {
        float x[2][8];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            floatx4_t sum = mfma16(from.key_bias[t][lane], qb, zeros);
#pragma unroll
            for (int g = 0; g < G; g++) {
                floatx4_t s = zeros;
#pragma unroll
                for (int k = g * GS; k < (g + 1) * GS; k++) s = key_product<T>(from.keys[t][k][lane], qf[k], s);
                const float4 sk = *reinterpret_cast<const float4 *>(&from.scale[0][g][16 * t + 4 * quarter]);
                sum[0] = __builtin_fmaf(sk.x, s[0], sum[0]), sum[1] = __builtin_fmaf(sk.y, s[1], sum[1]);
                sum[2] = __builtin_fmaf(sk.z, s[2], sum[2]), sum[3] = __builtin_fmaf(sk.w, s[3], sum[3]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) x[t >> 1][4 * (t & 1) + e] = sum[e];
        }
        if (s0 + kStageKeys - 1 > all_last || s0 < all_first || s0 + kStageKeys > s_end) {
            asm volatile("");  // (a branch: as selects it would cost every tile)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = s0 + 32 * u + 16 * (e >> 2) + 4 * quarter + (e & 3);
                    if (key > my_last || key < my_first || key >= s_end) x[u][e] = -INFINITY;
                }
        }
        float top = x[0][0];
#pragma unroll
        for (int e = 1; e < 16; e++) top = fmaxf(top, x[e >> 3][e & 7]);
        // Rescaled only when a maximum has grown by more than 2^8: until then the weights are at most 2^8.
        if (__any(top > m + 8.0f)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float m_new = fmaxf(m, top), f = exp2f(m - m_new);
            m = m_new, l *= f;
#pragma unroll
            for (int g = 0; g < G; g++) ones[g] *= f, accb[g] *= f;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[d][e] *= f;
        }
        // Values whose scales are not finite were made zeros, so that lines that do not see them stay clean: those that do get a NaN.
        uint32_t any = 0;
#pragma unroll
        for (int g = 0; g < G; g++) any |= *reinterpret_cast<const uint32_t *>(from.wild[0][g]) | *reinterpret_cast<const uint32_t *>(from.wild[1][g]);
        if (uniform((int32_t)any) != 0) {
            asm volatile("");
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int bit = 16 * (e >> 2 & 1) + 4 * quarter + (e & 3);
                    if (x[e >> 3][e & 7] > -INFINITY && (*reinterpret_cast<const uint32_t *>(from.wild[e >> 3][g]) >> bit & 1) != 0) accb[g] = NAN;
                }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[u][e] = __builtin_amdgcn_exp2f(x[u][e] - m), l += x[u][e];
            values(from, u, x[u]);
        }
    };

    int32_t next = 0;
    if (s_begin < s_end) {
        const int32_t first = look_up(s_begin);
        next = look_up(s_begin + kStageKeys);
        request(first, s_begin);
        expand(stages[0]);
    }
    __syncthreads();
    int at = 0;
    for (int s0 = s_begin; s0 < s_end; s0 += kStageKeys) {
        const bool more = s0 + kStageKeys < s_end;
        if (more) request(next, s0 + kStageKeys);
        next = look_up(s0 + 2 * kStageKeys);
        if (s0 <= any_last && s0 + kStageKeys > any_first) tile(stages[at], s0);  // (uniform in the wavefront)
        if (more) expand(stages[at ^ 1]);
        __syncthreads();
        at ^= 1;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
#pragma unroll
    for (int g = 0; g < G; g++) {
        ones[g] += __shfl_xor(ones[g], 16), accb[g] += __shfl_xor(accb[g], 16);
        ones[g] += __shfl_xor(ones[g], 32), accb[g] += __shfl_xor(accb[g], 32);
        if constexpr (kOnes) accb[g] = __builtin_fmaf(-(kValueOff + kMiddle), ones[g], accb[g]);  // (the operands and kValueOff + kMiddle went through the same weights)
    }
    if (!live) return;
    const bool whole = span.items == 1;
    float inv = 1.0f;
    float *state = nullptr;  // of this line and split: maximum, denominator, weighted sums
    if (whole) {
        float denom = l, f = 1.0f;
        if (a.sinks != nullptr) {
            const float sink = Elem<T>::load(a.sinks, my_head) * kLog2e, top = fmaxf(m, sink);
            f = exp2f(m - top), denom = denom * f + exp2f(sink - top);
        }
        inv = denom == 0.0f ? 0.0f : f / denom;  // (a row that sees nothing: zeros)
    } else {
        state = a.states + ((int64_t)item.slot * kPromptLines + wave * 16 + col) * kState<D>;
        if (quarter == 0) *reinterpret_cast<float2 *>(state) = make_float2(m, l);
    }
    T *out = a.out + (int64_t)(item.s.start + my_row) * a.out_strides[0] + (int64_t)my_head * a.out_strides[1];
#pragma unroll
    for (int d = 0; d < ND; d++) {
        const int c = 16 * d + 4 * quarter;
        const float b = accb[d / GB];
        const float v0 = o[d][0] + b, v1 = o[d][1] + b, v2 = o[d][2] + b, v3 = o[d][3] + b;
        if (whole) {
            struct __attribute__((packed)) Four { uint32_t w[2]; };
            *reinterpret_cast<Four *>(out + c) = Four{{qmf::Ops<T>::pack(v0 * inv, v1 * inv), qmf::Ops<T>::pack(v2 * inv, v3 * inv)}};
        } else {
            *reinterpret_cast<float4 *>(state + 4 + c) = make_float4(v0, v1, v2, v3);
        }
    }
}

// The splits of many lines merged: D / 4 threads a line, four splits' loads under way at a time.
template <int D> constexpr int kMergeLines = 64 * kWaves / (D / 4);  // of a block
template <typename T, int D>
__device__ __forceinline__ void merge_many(const RowsArgs<T> &a, int32_t unit, int block) {
    constexpr int kThreads = D / 4;
    PagedItem item;
    if (!paged_item<kPromptLines, 1, true>(a.batch, threadIdx.x & 63, unit, a.length, item)) return;
    const int rep = a.batch.rep, ln = block * kMergeLines<D> + (int)threadIdx.x / kThreads, at = (int)threadIdx.x % kThreads * 4;
    const int part = item.s.parts - 1 - item.part, line = part * kPromptLines + ln;  // (items count the parts from the last)
    const PromptSpan span = prompt_span(a.batch, item, part);
    if (line >= item.s.rows * rep || span.items == 1) return;
    const int64_t stride = (int64_t)a.batch.key_heads * kPromptLines * kState<D>;  // of a split's states
    const float *src = a.states + ((int64_t)item.slot * kPromptLines + ln) * kState<D>;
    float top = kLowest, total = 0.0f;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
        const float f = exp2f(top - most);
        top = most, total *= f, sum.x *= f, sum.y *= f, sum.z *= f, sum.w *= f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float w = z0 + i < span.items ? exp2f(m[i].x - top) : 0.0f;
            total = __builtin_fmaf(m[i].y, w, total);
            sum.x = __builtin_fmaf(v[i].x, w, sum.x), sum.y = __builtin_fmaf(v[i].y, w, sum.y);
            sum.z = __builtin_fmaf(v[i].z, w, sum.z), sum.w = __builtin_fmaf(v[i].w, w, sum.w);
        }
    }
    const int head = item.head * rep + line % rep;
    float inv = 1.0f;
    if (a.sinks != nullptr) {
        const float sink = Elem<T>::load(a.sinks, head) * kLog2e, most = fmaxf(top, sink);
        inv = exp2f(top - most), total = __builtin_fmaf(total, inv, exp2f(sink - most));
    }
    inv = total == 0.0f ? 0.0f : inv / total;
    struct __attribute__((packed)) Four { uint32_t w[2]; };
    *reinterpret_cast<Four *>(a.out + (int64_t)(item.s.start + line / rep) * a.out_strides[0] + (int64_t)head * a.out_strides[1] + at) =
        Four{{qmf::Ops<T>::pack(sum.x * inv, sum.y * inv), qmf::Ops<T>::pack(sum.z * inv, sum.w * inv)}};
}

// Both kernels' splits in one launch (nine sequences of one to 200 rows 49 -> 46 us): the blocks of few lines, a line each, behind those of many.
template <typename T, int D, int LINES>
__global__ void __launch_bounds__(64 * kWaves) paged_merge_both_kernel(const RowsArgs<T> few, const RowsArgs<T> many, uint32_t many_units, uint32_t few_units) {
    const uint32_t many_blocks = many_units * (kPromptLines / kMergeLines<D>), at = blockIdx.x - many_blocks;
    if (blockIdx.x < many_blocks) merge_many<T, D>(many, blockIdx.x % many_units, blockIdx.x / many_units);
    else merge_few<T, D, LINES>(few, at % few_units, at / few_units);
}

template <typename T, int BITS, int D, int G>
int32_t launch_prompt_sized(const RowsArgs<T> &few, const RowsArgs<T> &a, const PagedLaunch &f, const PagedLaunch &r, hipStream_t s) {
    hipLaunchKernelGGL((paged_prompt_kernel<T, BITS, D, G>), dim3(r.grid), dim3(64 * kPromptWaves), 0, s, a, a.batch.place.table);
    NVQ_LAUNCH_CHECK("paged_attention");
    if (r.merge_units == 0) return NVQ_OK;
    const uint32_t blocks = r.merge_units * (kPromptLines / kMergeLines<D>) + f.merge_units * f.merge_lines;
    hipLaunchKernelGGL((paged_merge_both_kernel<T, D, 16 / G>), dim3(blocks), dim3(64 * kWaves), 0, s, few, a, r.merge_units, f.merge_units);
    NVQ_LAUNCH_CHECK("paged_attention merge");
    return NVQ_OK;
}

template <typename T, int BITS>
int32_t launch_prompt_bits(const nvq_paged_desc &c, const RowsArgs<T> &few, const RowsArgs<T> &a, const PagedLaunch &f, const PagedLaunch &r, hipStream_t s) {
    if (c.head_dim == 64) return c.group_size == 32 ? launch_prompt_sized<T, BITS, 64, 2>(few, a, f, r, s) : launch_prompt_sized<T, BITS, 64, 1>(few, a, f, r, s);
    if (c.group_size == 32) return launch_prompt_sized<T, BITS, 128, 4>(few, a, f, r, s);
    return c.group_size == 64 ? launch_prompt_sized<T, BITS, 128, 2>(few, a, f, r, s) : launch_prompt_sized<T, BITS, 128, 1>(few, a, f, r, s);
}

template <typename T>
int32_t launch_prompt(const nvq_paged_attention_desc &d, const PagedAttentionOperands &o, const PagedLaunch &f, const PagedLaunch &r, hipStream_t s) {
    const RowsArgs<T> few = rows_args<T>(d, o, f), a = rows_args<T>(d, o, r);
    return d.cache.bits == 4 ? launch_prompt_bits<T, 4>(d.cache, few, a, f, r, s) : launch_prompt_bits<T, 8>(d.cache, few, a, f, r, s);
}

}  // namespace
}  // namespace paged
}  // namespace nvq
