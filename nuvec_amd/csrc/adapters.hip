// Low-rank adapters of many requests beside a shared projection:
//     out[r] = y[r] + scale[a] (x[r] . down[a]^T) . up[a]^T,  a the adapter of row r.
//
// Two kernels, both on the matrix cores.  The first leaves t = x . down^T (float32, the contraction split over wavefronts and over the grid,
// whose shares the second adds up), the second takes t . up^T, adds it to y and rounds once.  A block has 16 rows of x and takes the adapters that
// occur among them one after the other, each for all of its rows at once, so that no order or plan of the rows is needed beforehand: requests' rows lie
// together, and an adapter that occurs in one tile of rows is read there once.  A product's columns are rows of x, which do not meet: what a row's
// x holds, or another adapter's weights, reaches no other row.
//
// Terms: x, down and up are exact operands.  t is two terms of the element type, high and low (16 bits in bfloat16, 22 in float16, there scaled by
// a power of two into its range), side by side in one contraction of 32 beside 16 values of up twice; float32 runs on the float32 instruction.
//
// Both are bound by memory: the adapters' weights where there are few rows, x and y where there are many.
#include "matrix.h"
#include "nvq_internal.h"

namespace nvq {
namespace {

constexpr int kTileRows = 16, kAdapterWaves = 4, kWaveColumns = 64;

template <typename T>
struct AdapterArgs {
    const T *x, *down, *up, *y;
    const float *scales;
    const int32_t *ids;
    T *out;
    float *low;  // [splits][rows][padded]: shares of x . down^T
    int64_t rows, inputs, outputs, x_stride, y_stride, out_stride;
    int32_t adapters, rank, padded, splits, slots;  // slots: of a block, of a tile's 16 rows
};

// The adapter of the lane's row (lane % 16) of the tile; -1: none, or no row.
template <typename T>
__device__ __forceinline__ int32_t adapter_of(const AdapterArgs<T> &a, int64_t row) {
    const int32_t id = row < a.rows ? a.ids[row] : -1;
    return id >= 0 && id < a.adapters ? id : -1;
}
// Whether slot `s` of the tile is the first row of its adapter; the adapter.
__device__ __forceinline__ bool leads(int32_t id, int s, int32_t &adapter) {
    adapter = __builtin_amdgcn_readlane(id, s);
    return adapter >= 0 && __builtin_ctzll(__ballot(id == adapter)) == s;
}

// RT tiles of 16 ranks at a time.
template <typename T, int RT>
__global__ void __launch_bounds__(64 * kAdapterWaves) adapters_down_kernel(const AdapterArgs<T> a) {
    __shared__ acc4_t shares[kAdapterWaves][RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quarter = lane >> 4;
    const int64_t row = (int64_t)blockIdx.x * kTileRows + col;
    const int32_t id = adapter_of(a, row);
    const int64_t steps = (a.inputs + kFragStep<T> - 1) / kFragStep<T>, whole = a.inputs / kFragStep<T>;
    const int64_t per = (steps + a.splits * kAdapterWaves - 1) / (a.splits * kAdapterWaves);
    const int64_t from = ((int64_t)blockIdx.y * kAdapterWaves + wave) * per, to = from + per < steps ? from + per : steps, to_whole = to < whole ? to : whole;
    const T *x = a.x + (row < a.rows ? row : a.rows - 1) * a.x_stride + quarter * kFragRun<T>;
    for (int s = blockIdx.z * a.slots; s < (int)(blockIdx.z + 1) * a.slots; s++) {
        int32_t adapter;
        if (!leads(id, s, adapter)) continue;
        for (int t0 = 0; t0 < a.padded; t0 += 16 * RT) {
            const T *down[RT];
            acc4_t acc[RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int r = t0 + 16 * t + col;
                down[t] = a.down + ((int64_t)adapter * a.rank + (r < a.rank ? r : a.rank - 1)) * a.inputs + quarter * kFragRun<T>;
                acc[t] = acc4_t{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll 4
            for (int64_t k = from; k < to_whole; k++) {
                const uint4 xf = load_run(x + k * kFragStep<T>);
#pragma unroll
                for (int t = 0; t < RT; t++) acc[t] = product16<T>(load_run(down[t] + k * kFragStep<T>), xf, acc[t]);
            }
            if (from < to && to > whole) {  // the last, ragged step
                const int64_t at = whole * kFragStep<T>, left = a.inputs - at - quarter * kFragRun<T>;
                const uint4 xf = load_run(x + at, left);
#pragma unroll
                for (int t = 0; t < RT; t++) acc[t] = product16<T>(load_run(down[t] + at, left), xf, acc[t]);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) shares[wave][t][lane] = acc[t];
            __syncthreads();
            for (int t = wave; t < RT; t += kAdapterWaves) {
                const int r = t0 + 16 * t + 4 * quarter;
                acc4_t sum = shares[0][t][lane];
#pragma unroll
                for (int w = 1; w < kAdapterWaves; w++) sum += shares[w][t][lane];
#pragma unroll
                for (int i = 0; i < 4; i++) sum[i] = r + i < a.rank ? sum[i] : 0.0f;
                if (id == adapter && r < a.padded) *reinterpret_cast<acc4_t *>(a.low + (blockIdx.y * a.rows + row) * a.padded + r) = sum;
            }
            __syncthreads();
        }
    }
}

// 16 consecutive values of a row, of which `left` lie in it.
template <typename T>
__device__ __forceinline__ void load_sixteen(const T *p, int64_t left, float (&v)[16]) {
    if (left >= 16) {
        struct __attribute__((packed)) Run { T t[16]; };
        const Run run = *reinterpret_cast<const Run *>(p);
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = Elem<T>::load(run.t, i);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = i < left ? Elem<T>::load(p, i) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store_sixteen(T *p, int64_t left, const float (&v)[16]) {
    if (left >= 16) {
        struct __attribute__((packed)) Run { T t[16]; };
        Run run;
#pragma unroll
        for (int i = 0; i < 16; i++) Elem<T>::store(run.t, i, v[i]);
        *reinterpret_cast<Run *>(p) = run;
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i < left) Elem<T>::store(p, i, v[i]);
    }
}

// A lane's share of 16 ranks of t as an operand: float32, ranks 4 quarter .. + 3; else the terms of ranks 8 (quarter % 2) .. + 7, the high ones in
// the first two quarters and the low ones in the others.
template <typename T> constexpr int kLowRun = sizeof(T) == 4 ? 4 : 8;
template <typename T>
__device__ __forceinline__ uint4 low_terms(const float (&t)[kLowRun<T>], bool low) {
    if constexpr (sizeof(T) == 4) {
        return make_uint4(f2u(t[0]), f2u(t[1]), f2u(t[2]), f2u(t[3]));
    } else {
        T terms[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float high = rounded<T>(t[j]), rest = fabsf(high) < INFINITY ? t[j] - high : 0.0f;  // (what has no finite high term has no low one)
            Elem<T>::store(terms, j, low ? rest : high);
        }
        uint4 w;
        __builtin_memcpy(&w, terms, 16);
        return w;
    }
}

template <typename T>
__global__ void __launch_bounds__(64 * kAdapterWaves) adapters_up_kernel(const AdapterArgs<T> a) {
    constexpr int R = kLowRun<T>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quarter = lane >> 4;
    const int64_t row = (int64_t)blockIdx.x * kTileRows + col;
    const int64_t n0 = ((int64_t)blockIdx.y * kAdapterWaves + wave) * kWaveColumns;
    if (n0 >= a.outputs) return;
    const int32_t id = adapter_of(a, row);
    const int rank0 = sizeof(T) == 4 ? 4 * quarter : 8 * (quarter & 1);
    // Tile c of the columns: line m of the operand is column 16 (m / 4) + 4 c + m % 4, so that a lane's four accumulators are 16 consecutive ones.
    int64_t column[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int64_t n = n0 + 16 * (col >> 2) + 4 * c + (col & 3);
        column[c] = n < a.outputs ? n : a.outputs - 1;
    }
    bool mine = id < 0 && blockIdx.z == 0;  // (a row without an adapter: y as it is)
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; i++) sum[i] = 0.0f;
    for (int s = blockIdx.z * a.slots; s < (int)(blockIdx.z + 1) * a.slots; s++) {
        int32_t adapter;
        if (!leads(id, s, adapter)) continue;
        const bool match = id == adapter;
        const float scale = a.scales == nullptr ? 1.0f : a.scales[adapter];
        const float *low = a.low + (match ? row : (int64_t)blockIdx.x * kTileRows + s) * a.padded + rank0;  // (a row that has been written)
        auto low_at = [&](int b, float (&t)[R]) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < R; j++) t[j] = 0.0f;
            for (int z = 0; z < a.splits; z++) {
                const float *p = low + z * a.rows * a.padded + 16 * b;
#pragma unroll
                for (int j = 0; j < R; j += 4) {
                    const acc4_t v = *reinterpret_cast<const acc4_t *>(p + j);
#pragma unroll
                    for (int i = 0; i < 4; i++) t[j + i] += v[i];
                }
            }
#pragma unroll
            for (int j = 0; j < R; j++) t[j] *= scale;
        };
        int exponent = 0;  // of the row's largest t, taken out of float16's terms
        if constexpr (Elem<T>::code == NVQ_F16) {
            float top = 0.0f;
            for (int b = 0; b < a.padded / 16; b++) {
                float t[R];
                low_at(b, t);
#pragma unroll
                for (int j = 0; j < R; j++) top = fabsf(t[j]) < INFINITY ? fmaxf(top, fabsf(t[j])) : top;
            }
            top = fmaxf(top, __shfl_xor(top, 16));
            exponent = top > 0.0f ? ilogbf(top) : 0;
        }
        acc4_t acc[4];
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] = acc4_t{0.0f, 0.0f, 0.0f, 0.0f};
        const T *up = a.up + (int64_t)adapter * a.outputs * a.rank + rank0;
        for (int b = 0; b < a.padded / 16; b++) {
            float t[R];
            low_at(b, t);
            if constexpr (Elem<T>::code == NVQ_F16)
#pragma unroll
                for (int j = 0; j < R; j++) t[j] = ldexpf(t[j], -exponent);
            const uint4 tf = low_terms<T>(t, quarter >= 2);
#pragma unroll
            for (int c = 0; c < 4; c++) acc[c] = product16<T>(load_run(up + column[c] * a.rank + 16 * b, (int64_t)a.rank - 16 * b - rank0), tf, acc[c]);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float v = acc[i >> 2][i & 3];
            if constexpr (Elem<T>::code == NVQ_F16) v = ldexpf(v, exponent);
            sum[i] = match ? v : sum[i];
        }
        mine |= match;
    }
    const int64_t n = n0 + 16 * quarter, left = a.outputs - n;
    if (!mine || row >= a.rows || left <= 0) return;
    float v[16];
    load_sixteen(a.y + row * a.y_stride + n, left, v);
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] += sum[i];
    store_sixteen(a.out + row * a.out_stride + n, left, v);
}

int32_t padded_rank(const nvq_adapters_desc &d) { return (d.rank + 15) / 16 * 16; }

// A tile's adapters go to blocks of their own where the tiles alone leave compute units without work.
int32_t slots_of_block(const nvq_adapters_desc &d) {
    const int64_t tiles = (d.rows + kTileRows - 1) / kTileRows;
    return tiles * kTileRows <= 4 * (int64_t)compute_units() ? 1 : kTileRows;
}
int32_t splits_of(const nvq_adapters_desc &d) {
    const int64_t tiles = (d.rows + kTileRows - 1) / kTileRows, step = d.dtype == NVQ_F32 ? 16 : 32;
    const int64_t steps = (d.inputs + step - 1) / step, most = steps / (4 * kAdapterWaves);  // (four steps a wavefront at least)
    const int64_t blocks = slots_of_block(d) == 1 ? (d.rows < kTileRows ? d.rows : d.rows) : tiles;
    const int64_t want = (4 * (int64_t)compute_units() + blocks - 1) / blocks;
    const int64_t splits = want < most ? want : most;
    return (int32_t)(splits < 1 ? 1 : splits < 16 ? splits : 16);
}

template <typename T>
int32_t run_adapters(const nvq_adapters_desc &d, const void *x, const void *down, const void *up, const float *scales, const int32_t *ids, const void *y,
                     void *out, void *workspace, hipStream_t s) {
    AdapterArgs<T> a{};
    a.x = (const T *)x, a.down = (const T *)down, a.up = (const T *)up, a.y = (const T *)y, a.scales = scales, a.ids = ids, a.out = (T *)out;
    a.low = (float *)workspace, a.rows = d.rows, a.inputs = d.inputs, a.outputs = d.outputs;
    a.x_stride = d.x_stride, a.y_stride = d.y_stride, a.out_stride = d.out_stride;
    a.adapters = (int32_t)d.adapters, a.rank = d.rank, a.padded = padded_rank(d), a.splits = splits_of(d), a.slots = slots_of_block(d);
    const unsigned tiles = (unsigned)((d.rows + kTileRows - 1) / kTileRows);
    const unsigned slots = a.slots == 1 ? (unsigned)(d.rows < kTileRows ? d.rows : kTileRows) : 1;
    const dim3 block(64 * kAdapterWaves), grid(tiles, (unsigned)a.splits, slots);
    if (a.padded <= 16) hipLaunchKernelGGL((adapters_down_kernel<T, 1>), grid, block, 0, s, a);
    else if (a.padded <= 32) hipLaunchKernelGGL((adapters_down_kernel<T, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((adapters_down_kernel<T, 4>), grid, block, 0, s, a);
    NVQ_LAUNCH_CHECK("apply_adapters");
    const dim3 wide(tiles, (unsigned)((d.outputs + kAdapterWaves * kWaveColumns - 1) / (kAdapterWaves * kWaveColumns)), slots);
    hipLaunchKernelGGL((adapters_up_kernel<T>), wide, block, 0, s, a);
    NVQ_LAUNCH_CHECK("apply_adapters");
    return NVQ_OK;
}

}  // namespace

size_t adapters_workspace_bytes(const nvq_adapters_desc &d) { return (size_t)splits_of(d) * (size_t)d.rows * (size_t)padded_rank(d) * sizeof(float); }

int32_t launch_adapters(const nvq_adapters_desc &d, const void *x, const void *down, const void *up, const float *scales, const int32_t *ids, const void *y,
                        void *out, void *workspace, hipStream_t s) {
    if (d.dtype == NVQ_F32) return run_adapters<float>(d, x, down, up, scales, ids, y, out, workspace, s);
    if (d.dtype == NVQ_BF16) return run_adapters<bf16_t>(d, x, down, up, scales, ids, y, out, workspace, s);
    return run_adapters<f16_t>(d, x, down, up, scales, ids, y, out, workspace, s);
}

}  // namespace nvq
