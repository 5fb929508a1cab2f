// New keys and values into a paged, affine-quantized cache, and rows of it back as values.
//
// Append.  A token's queries are normed and rotated (heads.h), its keys normed, rotated and quantized, its values quantized, in one
// launch: what a decode step has between its projections and its attention.  The codes are made from the float32 results, which are
// never rounded to the element type on the way.  Of a group of a head's values with extremes lo, hi:
//     edge = lo where |lo| > |hi|, else hi;  steps = rint(|edge| (2^bits - 1) / (hi - lo));  scale = edge / steps (negative from hi), bias = edge
// (no steps: scale (hi - lo) / (2^bits - 1), bias 0; a range under 1e-7 (2^bits - 1) counts as that), both rounded to the element type, and
//     code = clamp(rint((x - bias) / scale))
// to the scale and bias as they are stored, so that each code is the nearest of those that the attention will read.  (`quantize` takes
// the unrounded ones, as the reference does.)  Quotients are correctly rounded: 16-bit inputs meet the middle between two codes
// exactly, and float32 then decides as real numbers would.
//
// Bound by memory when there are many tokens, by one round trip for the table, one for the inputs and one for the page's id when there
// are few.  A block takes 256 / P tokens of a head at a time (P lanes a head), so that the codes, scales and biases of consecutive
// positions, which lie together, are written by one block; a head is requested before the one in front of it is quantized.  Measured,
// bfloat16 to 4 bits in groups of 64: 6000 tokens of 32 query heads and 8 key heads of 128 in 32 us, 4.1 TB/s; 64 tokens with norms in 5 us, a
// launch; the 6000 tokens read back in 11 us, 2.9 TB/s.
#include "heads.h"
#include "nvq_internal.h"
#include "paged.h"

namespace nvq {
namespace {

template <typename T>
struct AppendArgs {
    PagedPlace place;
    const int32_t *sequences, *positions;
    const float2 *table;
    int64_t table_rows, tokens;
    const T *q, *k, *v, *q_weight, *k_weight;
    T *q_out;
    uint32_t *kw, *vw;
    T *ks, *kb, *vs, *vb;
    int64_t qs[2], kst[2], vst[2];  // strides of tokens and heads
    int32_t query_heads, key_heads, per_block, dim, half, interleaved, group;
    double eps;
};

// Codes, scale and bias of the lane's eight values, of a group in LANES adjacent lanes.
template <typename T, int BITS, int LANES>
__device__ __forceinline__ void quantize_run(const float (&x)[8], uint32_t (&words)[BITS / 4], float &scale, float &bias) {
    constexpr float bins = (float)((1u << BITS) - 1u);
    float lo = INFINITY, hi = -INFINITY;  // (NaN is skipped and gets code 0)
#pragma unroll
    for (int i = 0; i < 8; i++) lo = __builtin_fminf(lo, x[i]), hi = __builtin_fmaxf(hi, x[i]);
    lo = across<LANES>(lo, [](float a, float b) { return __builtin_fminf(a, b); });
    hi = across<LANES>(hi, [](float a, float b) { return __builtin_fmaxf(a, b); });
    const bool wide = fabsf(lo) > fabsf(hi);
    const float span = hi - lo, edge = wide ? lo : hi, size = fabsf(edge);
    const float steps = rintf(span > 1e-7f * bins ? size * bins / span : size / 1e-7f);
    const float step = steps == 0.0f ? __builtin_fmaxf(span / bins, 1e-7f) : size / steps;
    scale = rounded<T>(wide ? step : -step), bias = steps == 0.0f ? 0.0f : rounded<T>(edge);
    // t = (x - bias) / scale, correctly rounded: with y the correctly rounded reciprocal the second step t <- fma(fma(-scale, t, d), y, t)
    // gives the quotient itself (Markstein) wherever nothing leaves the normal range; elsewhere the division.  1.5 x 2^23 added rounds to
    // the nearest integer, ties to even, in the low mantissa bits.
    constexpr float kMagic = 12582912.0f;
    const float y = 1.0f / scale, mag = fabsf(scale);
    const bool plain = mag > 1e-20f && mag < 1e20f && span * fabsf(y) < 1024.0f;
    uint32_t raw[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float d = x[i] - bias;
        float t = d * y;
        if (plain) {
            t = __builtin_fmaf(__builtin_fmaf(-scale, t, d), y, t);
            t = __builtin_fmaf(__builtin_fmaf(-scale, t, d), y, t);
        } else {
            t = d / scale;
        }
        raw[i] = f2u(__builtin_amdgcn_fmed3f(t + kMagic, kMagic, kMagic + bins)) - 0x4B400000u;
    }
#pragma unroll
    for (int w = 0; w < BITS / 4; w++) {
        constexpr int kPer = 32 / BITS;
        uint32_t word = 0;
#pragma unroll
        for (int i = kPer - 1; i >= 0; i--) word = word << BITS | raw[w * kPer + i];
        words[w] = word;
    }
}

// The row of a head's first position and the place in the page; -1 where the token is not written: padding, or outside the cache.
template <typename T>
__device__ __forceinline__ int64_t row_of(const PagedPlace &p, const int32_t *sequences, const int32_t *positions, int64_t token, int64_t key_heads, int64_t most) {
    const int64_t position = positions[token], sequence = sequences == nullptr ? token : (int64_t)sequences[token];
    if (position < 0 || position >= p.capacity() || position >= most || sequence < 0 || sequence >= p.sequences) return -1;
    const int64_t id = p.table[sequence * p.stride + (position >> p.page_shift)];
    if (id < 0 || id >= p.pages) return -1;
    return (id * key_heads << p.page_shift) + (position & ((1 << p.page_shift) - 1));
}

template <typename T, int P, int BITS, int READ>
__global__ void __launch_bounds__(kHeadBlock) append_paged_kernel(const AppendArgs<T> a) {
    constexpr int kSlots = kHeadBlock / P, kWords = BITS / 4;
    __shared__ HeldHeads<T, P, READ> held;
    const int lane = threadIdx.x % P, j0 = 8 * lane;
    const int64_t token = (int64_t)blockIdx.x * kSlots + threadIdx.x / P;
    if (token >= a.tokens) return;
    const bool interleaved = a.interleaved != 0;
    const int64_t row = row_of<T>(a.place, a.sequences, a.positions, token, a.key_heads, a.half > 0 ? a.table_rows : INT64_MAX);
    Turn turn{};
    if (a.half > 0) {
        int64_t position = a.positions[token];
        position = position < 0 ? 0 : position < a.table_rows ? position : a.table_rows - 1;
        turn = read_turn<READ>(a.table + position * a.half, j0, a.half, interleaved);
    }
    const int h0 = blockIdx.y * a.per_block, h1 = min(h0 + a.per_block, a.query_heads + 2 * a.key_heads);
    auto normed = [&](HeadRun<T, READ> &run, const T *w, const HeadRun<T, READ> &weight) __attribute__((always_inline)) {
        if (w != nullptr) run.scale(norm_factor<P>(run.v, a.dim, a.eps), weight);
        run.turn(turn, j0, a.half, interleaved);
    };
    auto weight_of = [&](const T *w) __attribute__((always_inline)) {
        HeadRaw<T, READ == kWhole ? kWhole : kSingle> raw{};
        if (w != nullptr) raw.load(w, j0, a.dim, a.half, interleaved);
        return HeadRun<T, READ>(raw);
    };
    HeadRaw<T, READ> raw{};
    if (h0 < a.query_heads) {
        const HeadRun<T, READ> weight = weight_of(a.q_weight);
        const T *x = a.q + token * a.qs[0];
        T *y = a.q_out + token * a.query_heads * a.dim + j0;
        const int to = min(h1, a.query_heads);
        raw.load(x + h0 * a.qs[1], j0, a.dim, a.half, interleaved);
        for (int64_t head = h0; head < to; head++) {
            HeadRun<T, READ> run(raw);
            if (READ == kRuns && !interleaved) run.template meet<P>(raw, held, a.half);
            raw.load(x + (head + 1 < to ? head + 1 : head) * a.qs[1], j0, a.dim, a.half, interleaved);
            normed(run, a.q_weight, weight);
            store_run(y + head * a.dim, run.v);
        }
    }
    const int from = max(h0 - a.query_heads, 0), to = h1 - a.query_heads;
    if (row < 0 || from >= to) return;
    const HeadRun<T, READ> weight = weight_of(a.k_weight);
    auto row_at = [&](int h) { return h < a.key_heads ? a.k + token * a.kst[0] + h * a.kst[1] : a.v + token * a.vst[0] + (h - a.key_heads) * a.vst[1]; };
    raw.load(row_at(from), j0, a.dim, a.half, interleaved);
    for (int h = from; h < to; h++) {
        const bool is_v = h >= a.key_heads;
        const int64_t head = is_v ? h - a.key_heads : h;
        HeadRun<T, READ> run(raw);
        if (READ == kRuns && !interleaved && !is_v) run.template meet<P>(raw, held, a.half);
        raw.load(row_at(h + 1 < to ? h + 1 : h), j0, a.dim, a.half, interleaved);
        if (!is_v) normed(run, a.k_weight, weight);
        uint32_t words[kWords];
        float scale, bias;
        if (a.group == 32) quantize_run<T, BITS, 4>(run.v, words, scale, bias);
        else if (a.group == 64) quantize_run<T, BITS, 8>(run.v, words, scale, bias);
        else quantize_run<T, BITS, P < 16 ? 8 : 16>(run.v, words, scale, bias);
        const int64_t r = row + (head << a.place.page_shift);
        uint32_t *code = (is_v ? a.vw : a.kw) + r * (P * kWords) + lane * kWords;
        if constexpr (kWords == 1) *code = words[0];
        else *reinterpret_cast<uint2 *>(code) = make_uint2(words[0], words[1]);
        if (j0 % a.group == 0) {
            const int64_t g = r * (a.dim / a.group) + j0 / a.group;
            Elem<T>::store(is_v ? a.vs : a.ks, g, scale);
            Elem<T>::store(is_v ? a.vb : a.kb, g, bias);
        }
    }
}

template <typename T>
struct ReadArgs {
    PagedPlace place;
    const int32_t *sequences, *positions;
    int64_t tokens;
    const uint32_t *kw, *vw;
    const T *ks, *kb, *vs, *vb;
    T *keys, *values;
    int32_t key_heads, per_block, group;
};

// code x scale + bias, rounded once; zeros for a token that is not in the cache.
template <typename T, int P, int BITS>
__global__ void __launch_bounds__(kHeadBlock) read_paged_kernel(const ReadArgs<T> a) {
    constexpr int kSlots = kHeadBlock / P, kWords = BITS / 4, D = 8 * P;
    const int lane = threadIdx.x % P, j0 = 8 * lane;
    const int64_t token = (int64_t)blockIdx.x * kSlots + threadIdx.x / P;
    if (token >= a.tokens) return;
    const int64_t row = row_of<T>(a.place, a.sequences, a.positions, token, a.key_heads, INT64_MAX);
    const int h1 = min((int)(blockIdx.y + 1) * a.per_block, 2 * a.key_heads);
    for (int h = blockIdx.y * a.per_block; h < h1; h++) {
        const bool is_v = h >= a.key_heads;
        const int64_t head = is_v ? h - a.key_heads : h;
        float y[8] = {};
        if (row >= 0) {
            const int64_t r = row + (head << a.place.page_shift), g = r * (D / a.group) + j0 / a.group;
            const uint32_t *code = (is_v ? a.vw : a.kw) + r * (P * kWords) + lane * kWords;
            uint32_t words[kWords];
            if constexpr (kWords == 1) words[0] = *code;
            else words[0] = reinterpret_cast<const uint2 *>(code)->x, words[1] = reinterpret_cast<const uint2 *>(code)->y;
            const float scale = Elem<T>::load(is_v ? a.vs : a.ks, g), bias = Elem<T>::load(is_v ? a.vb : a.kb, g);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t c = words[i * BITS / 32] >> (i * BITS % 32) & ((1u << BITS) - 1u);
                y[i] = __builtin_fmaf((float)c, scale, bias);
            }
        }
        store_run((is_v ? a.values : a.keys) + (token * a.key_heads + head) * D + j0, y);
    }
}

PagedPlace place_of(const nvq_paged_desc &d, const int32_t *page_table) {
    PagedPlace p{};
    p.table = page_table, p.stride = d.table_stride, p.pages = d.pages;
    p.sequences = (int32_t)d.sequences, p.columns = (int32_t)d.columns;
    while ((1LL << p.page_shift) < d.page_size) p.page_shift++;
    return p;
}

// Heads of a block: all that leave four blocks a compute unit, one where even that does not fill them.  (The 6000 tokens, two blocks a
// compute unit 58 us appended and read back, four 43, eight 48.)
int32_t heads_of_block(int64_t blocks, int64_t heads) {
    const int64_t per = blocks * heads / (4 * (int64_t)compute_units());
    return (int32_t)(per < 1 ? 1 : per < heads ? per : heads);
}

template <typename T, int P, int BITS>
int32_t run_append(AppendArgs<T> &a, int read, hipStream_t s) {
    const int64_t blocks = (a.tokens + kHeadBlock / P - 1) / (kHeadBlock / P);
    const int32_t all = a.query_heads + 2 * a.key_heads;
    a.per_block = heads_of_block(blocks, all);
    const dim3 grid((unsigned)blocks, (unsigned)((all + a.per_block - 1) / a.per_block));
    if (read == kWhole) hipLaunchKernelGGL((append_paged_kernel<T, P, BITS, kWhole>), grid, dim3(kHeadBlock), 0, s, a);
    else if (read == kRuns) hipLaunchKernelGGL((append_paged_kernel<T, P, BITS, kRuns>), grid, dim3(kHeadBlock), 0, s, a);
    else hipLaunchKernelGGL((append_paged_kernel<T, P, BITS, kSingle>), grid, dim3(kHeadBlock), 0, s, a);
    NVQ_LAUNCH_CHECK("append_paged");
    return NVQ_OK;
}

template <typename T>
int32_t run_append_type(const nvq_paged_append_desc &d, const PagedAppendOperands &o, hipStream_t s) {
    AppendArgs<T> a{};
    const nvq_paged_desc &c = d.cache;
    a.place = place_of(c, o.page_table);
    a.sequences = o.sequences, a.positions = o.positions, a.table = (const float2 *)o.table, a.table_rows = d.table_rows, a.tokens = d.tokens;
    a.q = (const T *)o.q, a.k = (const T *)o.k, a.v = (const T *)o.v, a.q_weight = (const T *)o.q_weight, a.k_weight = (const T *)o.k_weight;
    a.q_out = (T *)o.q_out;
    a.kw = (uint32_t *)o.kw, a.ks = (T *)o.ks, a.kb = (T *)o.kb, a.vw = (uint32_t *)o.vw, a.vs = (T *)o.vs, a.vb = (T *)o.vb;
    a.query_heads = o.q == nullptr ? 0 : (int32_t)d.query_heads, a.key_heads = (int32_t)c.key_heads;
    a.dim = c.head_dim, a.half = d.rotary_dims / 2, a.interleaved = d.interleaved, a.group = c.group_size, a.eps = d.eps;
    uintptr_t rows = (uintptr_t)o.q | (uintptr_t)o.k | (uintptr_t)o.v;  // addresses and strides in bytes: their lowest bits
    for (int i = 0; i < 2; i++) {
        a.qs[i] = d.q_strides[i], a.kst[i] = d.k_strides[i], a.vst[i] = d.v_strides[i];
        rows |= (uintptr_t)a.kst[i] * sizeof(T) | (uintptr_t)a.vst[i] * sizeof(T);
        if (a.query_heads > 0) rows |= (uintptr_t)a.qs[i] * sizeof(T);
    }
    const uintptr_t others = (uintptr_t)o.q_weight | (uintptr_t)o.k_weight | (uintptr_t)o.table;
    const int read = read_of(a.dim, a.half, a.interleaved != 0, rows % 16 == 0, others % 16 == 0);
    if (c.head_dim == 64) return c.bits == 4 ? run_append<T, 8, 4>(a, read, s) : run_append<T, 8, 8>(a, read, s);
    return c.bits == 4 ? run_append<T, 16, 4>(a, read, s) : run_append<T, 16, 8>(a, read, s);
}

template <typename T, int P, int BITS>
int32_t run_read(const nvq_paged_desc &c, int64_t tokens, const PagedAppendOperands &o, void *keys, void *values, hipStream_t s) {
    ReadArgs<T> a{};
    a.place = place_of(c, o.page_table);
    a.sequences = o.sequences, a.positions = o.positions, a.tokens = tokens;
    a.kw = (const uint32_t *)o.kw, a.ks = (const T *)o.ks, a.kb = (const T *)o.kb, a.vw = (const uint32_t *)o.vw, a.vs = (const T *)o.vs, a.vb = (const T *)o.vb;
    a.keys = (T *)keys, a.values = (T *)values, a.key_heads = (int32_t)c.key_heads, a.group = c.group_size;
    const int64_t blocks = (tokens + kHeadBlock / P - 1) / (kHeadBlock / P);
    a.per_block = heads_of_block(blocks, 2 * c.key_heads);
    hipLaunchKernelGGL((read_paged_kernel<T, P, BITS>), dim3((unsigned)blocks, (unsigned)((2 * a.key_heads + a.per_block - 1) / a.per_block)),
                       dim3(kHeadBlock), 0, s, a);
    NVQ_LAUNCH_CHECK("read_paged");
    return NVQ_OK;
}

template <typename T, typename... A>
int32_t run_read_type(const nvq_paged_desc &c, A... args) {
    if (c.head_dim == 64) return c.bits == 4 ? run_read<T, 8, 4>(c, args...) : run_read<T, 8, 8>(c, args...);
    return c.bits == 4 ? run_read<T, 16, 4>(c, args...) : run_read<T, 16, 8>(c, args...);
}

}  // namespace

int32_t launch_append_paged(const nvq_paged_append_desc &d, const PagedAppendOperands &o, hipStream_t s) {
    switch (d.cache.dtype) {
    case NVQ_F32: return run_append_type<float>(d, o, s);
    case NVQ_BF16: return run_append_type<bf16_t>(d, o, s);
    default: return run_append_type<f16_t>(d, o, s);
    }
}

int32_t launch_read_paged(const nvq_paged_desc &c, int64_t tokens, const PagedAppendOperands &o, void *keys, void *values, hipStream_t s) {
    switch (c.dtype) {
    case NVQ_F32: return run_read_type<float>(c, tokens, o, keys, values, s);
    case NVQ_BF16: return run_read_type<bf16_t>(c, tokens, o, keys, values, s);
    default: return run_read_type<f16_t>(c, tokens, o, keys, values, s);
    }
}

}  // namespace nvq
