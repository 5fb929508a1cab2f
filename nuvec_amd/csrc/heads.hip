// Rotary positions of heads, with or without the norm over each head: what a model does to its queries and keys between the
// projections and the attention.  With c, n the cosine and sine of position x frequency i from a table,
//     half layout:  y[i] = x[i] c - x[i + pairs] n,  y[i + pairs] = x[i + pairs] c + x[i] n;  interleaved: the pairs are (2 i, 2 i + 1)
// over the first 2 x pairs values of a head, the others as they are; the norm before it is x / sqrt(mean(x^2) + eps) * weight over the
// whole head.  float32 throughout, rounded once.  (The reference's model code composes them of its array operations.)
//
// Bound by memory: each value is read and written once, but for the partner's run of eight, which the lane that turns it reads
// too, from lines that are in the L1 by then.  A block takes 256 / P tokens and walks heads of them, so that a token's angles (eight bytes a
// pair, more than a 16-bit head itself) are read once for all of a block's heads, and the norm's weight too; a head is requested before the one
// in front of it is worked on.  Measured, bfloat16, 2 x 2049 tokens, 40 heads of 128 with norms: 20.2 us, 4.3 TB/s (a large copy: 4.9; the weight
// read for each head: 23.5 us); a call of few tokens is one launch, 4.6 to 5 us.
#include "heads.h"
#include "nvq_internal.h"

namespace nvq {
namespace {

template <typename T>
struct Operand {
    const T *x, *weight;
    T *y;
    int64_t xs[3], ys[3];  // strides of batches, heads, positions
};

template <typename T>
struct HeadArgs {
    Operand<T> of[2];
    int32_t first_heads, all_heads, per_block;
    const float2 *table;
    const int32_t *offsets;
    int64_t offset, table_rows, tokens, length;
    int32_t per_position, dim, half, interleaved;
    double eps;
};

template <typename T, int P, int READ>
__global__ void __launch_bounds__(kHeadBlock) head_norm_rope_kernel(const HeadArgs<T> a) {
    constexpr int kSlots = kHeadBlock / P;
    __shared__ HeldHeads<T, P, READ> held;
    const int j0 = 8 * (threadIdx.x % P);
    const int64_t token = (int64_t)blockIdx.x * kSlots + threadIdx.x / P;
    if (token >= a.tokens) return;  // (whole heads: the lanes that are left meet all of theirs)
    const int64_t b = token / a.length, l = token - b * a.length;
    const bool interleaved = a.interleaved != 0;
    Turn turn{};
    if (a.half > 0) {
        int64_t position = a.offsets == nullptr ? a.offset + l : a.per_position ? (int64_t)a.offsets[token] : (int64_t)a.offsets[b] + l;
        position = position < 0 ? 0 : position < a.table_rows ? position : a.table_rows - 1;  // (outside the table is the caller's error: clamped)
        turn = read_turn<READ>(a.table + position * a.half, j0, a.half, interleaved);
    }
    const int h0 = blockIdx.y * a.per_block, h1 = min(h0 + a.per_block, a.all_heads);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const Operand<T> &o = a.of[i];
        const int from = i == 0 ? h0 : max(h0 - a.first_heads, 0), to = i == 0 ? min(h1, a.first_heads) : h1 - a.first_heads;
        if (from >= to) continue;
        HeadRaw<T, READ == kWhole ? kWhole : kSingle> weights{};
        if (o.weight != nullptr) weights.load(o.weight, j0, a.dim, a.half, interleaved);
        const HeadRun<T, READ> weight(weights);
        HeadRaw<T, READ> raw{};
        const T *x = o.x + b * o.xs[0] + l * o.xs[2];
        T *y = o.y + b * o.ys[0] + l * o.ys[2];
        raw.load(x + from * o.xs[1], j0, a.dim, a.half, interleaved);
        for (int64_t head = from; head < to; head++) {
            HeadRun<T, READ> run(raw);
            if (READ == kRuns && !interleaved) run.template meet<P>(raw, held, a.half);
            raw.load(x + (head + 1 < to ? head + 1 : head) * o.xs[1], j0, a.dim, a.half, interleaved);
            if (o.weight != nullptr) run.scale(norm_factor<P>(run.v, a.dim, a.eps), weight);
            run.turn(turn, j0, a.half, interleaved);
            T *to_y = y + head * o.ys[1];
            if (READ != kSingle) {
                if (j0 < a.dim) store_run(to_y + j0, run.v);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (j0 + k < a.dim) Elem<T>::store(to_y, j0 + k, run.v[k]);
            }
        }
    }
}

template <typename T, int P>
int32_t run_heads(const HeadArgs<T> &a, int read, hipStream_t s) {
    const dim3 grid((unsigned)((a.tokens + kHeadBlock / P - 1) / (kHeadBlock / P)), (unsigned)((a.all_heads + a.per_block - 1) / a.per_block));
    if (read == kWhole) hipLaunchKernelGGL((head_norm_rope_kernel<T, P, kWhole>), grid, dim3(kHeadBlock), 0, s, a);
    else if (read == kRuns) hipLaunchKernelGGL((head_norm_rope_kernel<T, P, kRuns>), grid, dim3(kHeadBlock), 0, s, a);
    else hipLaunchKernelGGL((head_norm_rope_kernel<T, P, kSingle>), grid, dim3(kHeadBlock), 0, s, a);
    NVQ_LAUNCH_CHECK("head_norm_rope");
    return NVQ_OK;
}

template <typename T>
int32_t run_type(const nvq_head_rope_desc &d, const float *table, const int32_t *offsets, const void *const (&x)[2], const void *const (&w)[2],
                 void *const (&y)[2], hipStream_t s) {
    HeadArgs<T> a{};
    uintptr_t rows = 0, others = (uintptr_t)table;  // addresses and strides in bytes: their lowest bits
    for (int i = 0; i < 2; i++) {
        if (d.heads[i] == 0) continue;
        Operand<T> &o = a.of[i];
        o.x = (const T *)x[i], o.weight = (const T *)w[i], o.y = (T *)y[i];
        rows |= (uintptr_t)x[i] | (uintptr_t)y[i], others |= (uintptr_t)w[i];
        for (int k = 0; k < 3; k++) {
            o.xs[k] = d.x_strides[i][k], o.ys[k] = d.y_strides[i][k];
            rows |= (uintptr_t)o.xs[k] * sizeof(T) | (uintptr_t)o.ys[k] * sizeof(T);
        }
    }
    a.first_heads = (int32_t)d.heads[0], a.all_heads = (int32_t)(d.heads[0] + d.heads[1]);
    a.table = (const float2 *)table, a.offsets = offsets, a.offset = d.offset, a.table_rows = d.table_rows;
    a.tokens = d.batch * d.length, a.length = d.length, a.per_position = d.per_position;
    a.dim = d.head_dim, a.half = d.rotary_dims / 2, a.interleaved = d.interleaved, a.eps = d.eps;
    const int read = read_of(a.dim, a.half, a.interleaved != 0, rows % 16 == 0, others % 16 == 0);
    const int p = head_lanes(d.head_dim);
    // Heads of a block: all that leave four blocks a compute unit, one where even that does not fill them.  (The 2 x 2049 tokens above: two blocks
    // a compute unit 23.5 us, four 20.2, eight 21.6.)
    const int64_t blocks = (a.tokens + kHeadBlock / p - 1) / (kHeadBlock / p), want = 4 * (int64_t)compute_units();
    const int64_t per = blocks * a.all_heads / want;
    a.per_block = (int32_t)(per < 1 ? 1 : per < a.all_heads ? per : a.all_heads);
    switch (p) {
    case 8: return run_heads<T, 8>(a, read, s);
    case 16: return run_heads<T, 16>(a, read, s);
    case 32: return run_heads<T, 32>(a, read, s);
    default: return run_heads<T, 64>(a, read, s);
    }
}

// angle = scale x position / wavelength's base i, in 64 bits: at position 100000 a float32 angle is off by 0.004, and one of frequencies that were
// rounded to float32 by 0.0016.
template <typename F>
__global__ void __launch_bounds__(256) rotation_table_kernel(const F *__restrict__ freqs, int half, int64_t rows, double base, double scale,
                                                             double magnitude, float2 *__restrict__ table) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= rows * half) return;
    const int64_t position = at / half;
    const int i = (int)(at - position * half);
    const double f = freqs != nullptr ? (double)freqs[i] : pow(base, (double)i / (double)half);
    double n, c;
    sincos((double)position * scale / f, &n, &c);
    table[at] = make_float2((float)(c * magnitude), (float)(n * magnitude));
}

}  // namespace

int32_t launch_head_rope(const nvq_head_rope_desc &d, const float *table, const int32_t *offsets, const void *const (&x)[2],
                         const void *const (&w)[2], void *const (&y)[2], hipStream_t s) {
    switch (d.dtype) {
    case NVQ_F32: return run_type<float>(d, table, offsets, x, w, y, s);
    case NVQ_BF16: return run_type<bf16_t>(d, table, offsets, x, w, y, s);
    default: return run_type<f16_t>(d, table, offsets, x, w, y, s);
    }
}

template <typename F>
int32_t launch_rotation_table(const F *freqs, int half, int64_t rows, double base, double scale, double magnitude, float *table, hipStream_t s) {
    hipLaunchKernelGGL((rotation_table_kernel<F>), dim3((unsigned)((rows * half + 255) / 256)), dim3(256), 0, s, freqs, half, rows, base, scale, magnitude,
                       (float2 *)table);
    NVQ_LAUNCH_CHECK("rotation_table");
    return NVQ_OK;
}
template int32_t launch_rotation_table<float>(const float *, int, int64_t, double, double, double, float *, hipStream_t);
template int32_t launch_rotation_table<double>(const double *, int, int64_t, double, double, double, float *, hipStream_t);

}  // namespace nvq
