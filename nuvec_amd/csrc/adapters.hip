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
// Both are bound by memory: the adapters' weights where there are few rows, x and y where there are many; a call of one row is two launches, 7.4 us.
// Measured (bfloat16, us): 64 rows of 64 adapters of rank 16 beside [4096, 4096] 12.4 (kernels 5.6 and 7.8; the weights alone, 17 MB, at the rate of a large copy
// 3.4); 4096 rows of four of rank 32 beside [14336, 4096] 87 to 94 (19 and 70; x, y and out, 268 MB, 55); float16, 517 rows of nine of rank 12 beside [2880, 2880] 14.7.
// A product's tile goes through LDS so that y and out are moved in runs of 512 bytes a row: 64 bytes a row and wavefront took 140 us in the second of these.
#include "matrix.h"
#include "nvq_internal.h"

namespace nvq {
namespace {

constexpr int kDownWaves = 8, kUpWaves = 4, kBlockColumns = 256;  // (64 a wavefront)

template <typename T>
struct AdapterArgs {
    const T *x, *down, *up, *y;
    const float *scales;
    const int32_t *ids;
    T *out;
    float *low;  // [splits][rows][padded]: shares of x . down^T
    int64_t rows, inputs, outputs, x_stride, y_stride, out_stride;
    int32_t adapters, rank, padded, splits, chunks;  // chunks: of 256 columns of a block
};

// The adapters that occur in a tile of up to 64 rows, one after the other in the order of their first rows: every `step`th from number `first` on.
struct Occurring {
    int32_t id;     // of row `lane` of the tile; -1: none, or no row
    uint64_t left;  // rows whose adapters are still to come
    int step;
    template <typename T>
    __device__ __forceinline__ Occurring(const AdapterArgs<T> &a, int64_t row0, int rows, int first, int every) {
        const int lane = threadIdx.x & 63;
        id = lane < rows && row0 + lane < a.rows ? a.ids[row0 + lane] : -1;
        id = id >= 0 && id < a.adapters ? id : -1;
        left = __ballot(id >= 0), step = every;
        for (int i = 0; i < first && left != 0; i++) skip();
    }
    __device__ __forceinline__ void skip() { left &= ~__ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(left))); }
    __device__ __forceinline__ bool any() const { return left != 0; }
    __device__ __forceinline__ int32_t now() const { return __builtin_amdgcn_readlane(id, __builtin_ctzll(left)); }
    __device__ __forceinline__ void next() {
        for (int i = 0; i < step && left != 0; i++) skip();
    }
    // The adapter of row `row` of the tile.
    __device__ __forceinline__ int32_t of(int row) const { return __shfl(id, row); }
};

template <int N>
struct Count {
    static constexpr int value = N;
};

// RW tiles of 16 rows, RT tiles of 16 ranks at a time.
template <typename T, int RW, int RT>
__global__ void __launch_bounds__(64 * kDownWaves) adapters_down_kernel(const AdapterArgs<T> a) {
    __shared__ acc4_t shares[kDownWaves][RW * RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quarter = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * RW);
    const int32_t steps = (int32_t)((a.inputs + kFragStep<T> - 1) / kFragStep<T>), whole = (int32_t)(a.inputs / kFragStep<T>);
    const int32_t per = (steps + a.splits * kDownWaves - 1) / (a.splits * kDownWaves);
    const int32_t from = ((int32_t)blockIdx.y * kDownWaves + wave) * per, to = from + per < steps ? from + per : steps, to_whole = to < whole ? to : whole;
    const T *x[RW];
#pragma unroll
    for (int i = 0; i < RW; i++) {
        const int64_t row = row0 + 16 * i + col;
        x[i] = a.x + (row < a.rows ? row : a.rows - 1) * a.x_stride + quarter * kFragRun<T>;
    }
    uint4 ahead[4][RW];  // of x, the first four steps, requested before the rows' adapters are known
    const bool four = from + 4 <= to_whole;
    if (four)
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int i = 0; i < RW; i++) ahead[u][i] = load_run(x[i] + (int64_t)(from + u) * kFragStep<T>);
    for (Occurring at(a, row0, 16 * RW, blockIdx.z, gridDim.z); at.any(); at.next()) {
        const int32_t adapter = at.now();
        for (int t0 = 0; t0 < a.padded; t0 += 16 * RT) {
            const T *down[RT];
            acc4_t acc[RW][RT];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int r = t0 + 16 * t + col;
                down[t] = a.down + ((int64_t)adapter * a.rank + (r < a.rank ? r : a.rank - 1)) * a.inputs + quarter * kFragRun<T>;
#pragma unroll
                for (int i = 0; i < RW; i++) acc[i][t] = acc4_t{0.0f, 0.0f, 0.0f, 0.0f};
            }
            auto some = [&](int32_t k, auto count, bool first) __attribute__((always_inline)) {  // that many steps' loads under way at a time
                constexpr int U = decltype(count)::value;
                uint4 xf[U][RW], df[U][RT];
#pragma unroll
                for (int u = 0; u < U; u++) {
#pragma unroll
                    for (int i = 0; i < RW; i++) xf[u][i] = first ? ahead[u][i] : load_run(x[i] + (int64_t)(k + u) * kFragStep<T>);
#pragma unroll
                    for (int t = 0; t < RT; t++) df[u][t] = load_run(down[t] + (int64_t)(k + u) * kFragStep<T>);
                }
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int t = 0; t < RT; t++)
#pragma unroll
                        for (int i = 0; i < RW; i++) acc[i][t] = product16<T>(df[u][t], xf[u][i], acc[i][t]);
            };
            int32_t k = from;
            if (four) some(k, Count<4>{}, true), k += 4;
            for (; k + 4 <= to_whole; k += 4) some(k, Count<4>{}, false);
            for (; k < to_whole; k++) some(k, Count<1>{}, false);
            if (from < to && to > whole) {  // the last, ragged step
                const int64_t k = (int64_t)whole * kFragStep<T>, left = a.inputs - k - quarter * kFragRun<T>;
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const uint4 xf = load_run(x[i] + k, left);
#pragma unroll
                    for (int t = 0; t < RT; t++) acc[i][t] = product16<T>(load_run(down[t] + k, left), xf, acc[i][t]);
                }
            }
#pragma unroll
            for (int i = 0; i < RW; i++)
#pragma unroll
                for (int t = 0; t < RT; t++) shares[wave][i * RT + t][lane] = acc[i][t];
            __syncthreads();
            for (int s = wave; s < RW * RT; s += kDownWaves) {
                const int tile = s / RT, r = t0 + 16 * (s % RT) + 4 * quarter;
                acc4_t sum = shares[0][s][lane];
#pragma unroll
                for (int w = 1; w < kDownWaves; w++) sum += shares[w][s][lane];
#pragma unroll
                for (int i = 0; i < 4; i++) sum[i] = r + i < a.rank ? sum[i] : 0.0f;
                const int64_t row = row0 + 16 * tile + col;
                if (at.of(16 * tile + col) == adapter && r < a.padded) *reinterpret_cast<acc4_t *>(a.low + (blockIdx.y * a.rows + row) * a.padded + r) = sum;
            }
            __syncthreads();
        }
    }
}

// Eight consecutive values of a row, of which `left` lie in it.
template <typename T>
struct __attribute__((packed)) Eight {
    T t[8];
};
template <typename T>
__device__ __forceinline__ void load_eight(const T *p, int64_t left, float *v) {
    if (left >= 8) {
        const Eight<T> e = *reinterpret_cast<const Eight<T> *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = Elem<T>::load(e.t, i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < left ? Elem<T>::load(p, i) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store_eight(T *p, int64_t left, const float *v) {
    if (left >= 8) {
        Eight<T> e;
#pragma unroll
        for (int i = 0; i < 8; i++) Elem<T>::store(e.t, i, v[i]);
        *reinterpret_cast<Eight<T> *>(p) = e;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) Elem<T>::store(p, i, v[i]);
    }
}

// Runs of ranks, as long as a lane's 16 bytes of up.  The last one of a rank that is no whole number of them begins as much earlier, so that it is read as the
// others are; what it has in common with the one in front of it is taken for zeros, of t and of up.  (Ranks shorter than a run are read value by value.)
struct RankRun {
    int from, skip;  // the first rank; how many of the run are not its own
    bool any;
};
template <typename T>
__device__ __forceinline__ RankRun rank_run(int rank, int run) {
    constexpr int L = kFragRun<T>;
    const int first = L * run, last = rank > L ? rank - L : 0;
    return RankRun{first < last ? first : last, first < last ? 0 : first - last, first < rank};
}

// The rows' own t as operands of 16 ranks, a kilobyte a tile of rows and block of ranks.  float32: lane (row, quarter) holds the block's run `quarter`; else
// the terms of its run quarter % 2, the high ones in the first two quarters and the low ones in the others.  (Of a row without an adapter they are whatever
// the workspace holds, and are not used.)
template <typename T>
__device__ __forceinline__ void put_terms(uint4 *block, int row, int run, const float (&t)[kFragRun<T>]) {
    if constexpr (sizeof(T) == 4) {
        block[row + 16 * run] = make_uint4(f2u(t[0]), f2u(t[1]), f2u(t[2]), f2u(t[3]));
    } else {
        T high[8], low[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float h = rounded<T>(t[j]);
            Elem<T>::store(high, j, h);
            Elem<T>::store(low, j, fabsf(h) < INFINITY ? t[j] - h : 0.0f);  // (what has no finite high term has no low one)
        }
        __builtin_memcpy(&block[row + 16 * run], high, 16);
        __builtin_memcpy(&block[row + 16 * (run + 2)], low, 16);
    }
}

// RW tiles of 16 rows.  The products' tile goes through LDS, so that y and out are read and written in runs of 512 bytes a row.
template <typename T, int RW>
__global__ void __launch_bounds__(64 * kUpWaves, RW == 2 ? 3 : 4) adapters_up_kernel(const AdapterArgs<T> a) {
    constexpr bool kScaled = Elem<T>::code == NVQ_F16;
    extern __shared__ uint4 terms[];  // [RW][padded / 16][64]
    __shared__ float sums[16 * RW][kBlockColumns + 4];
    __shared__ uint32_t largest[16 * RW];  // float16: of a row's t, its bits
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quarter = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * RW);
    const int blocks = a.padded / 16;
    constexpr int L = kFragRun<T>, kRuns = 16 / L;  // runs of a block of ranks
    const Occurring occurring(a, row0, 16 * RW, blockIdx.z, gridDim.z);
    // The rows that this block writes, a bit each: those of its adapters, and the first block's without one.
    const uint64_t bare = blockIdx.z == 0 ? __ballot(occurring.id < 0 && lane < 16 * RW && row0 + lane < a.rows) : 0;
    uint64_t mine = bare;
    for (Occurring at = occurring; at.any(); at.next()) mine |= __ballot(occurring.id == at.now());
    if (mine == 0) return;
    // y of 256 columns: eight rows at a time, eight values a thread, requested before the columns in front of them are worked on.
    const int y_row = tid >> 5, y_col = 8 * (tid & 31);
    Eight<T> ahead[2 * RW];
    auto request = [&](int64_t n0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2 * RW; i++) {
            const int64_t r = row0 + 8 * i + y_row;
            ahead[i] = *reinterpret_cast<const Eight<T> *>(a.y + (r < a.rows ? r : a.rows - 1) * a.y_stride + n0 + y_col);
        }
    };
    const int64_t n_first = (int64_t)blockIdx.y * a.chunks * kBlockColumns, n_most = n_first + a.chunks * kBlockColumns, n_end = n_most < a.outputs ? n_most : a.outputs;
    const int64_t n_whole = n_first + (n_end - n_first) / kBlockColumns * kBlockColumns;
    if (n_first < n_whole) request(n_first);

    // ── the weights ──
    // Tile c of a wavefront's 64 columns: line m of the operand is column 32 (c / 2) + 8 (m / 4) + 4 (c % 2) + m % 4.
    const int line = 8 * (col >> 2) + (col & 3), run0 = sizeof(T) == 4 ? quarter : quarter & 1;
    const RankRun last_run = rank_run<T>(a.rank, kRuns * (blocks - 1) + run0);
    uint32_t last_kept[4];  // what is its own of the last block's run
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t low = last_run.any && (sizeof(T) == 4 ? j : 2 * j) >= last_run.skip ? (sizeof(T) == 4 ? ~0u : 0xFFFFu) : 0u;
        last_kept[j] = sizeof(T) == 4 ? low : low | (last_run.any && 2 * j + 1 >= last_run.skip ? 0xFFFF0000u : 0u);
    }
    // Of an adapter, `U` blocks of ranks from b0 on, 64 columns from n0 on.  KIND 0: value by value; 1: they are whole and so are the runs, so that no load stands
    // under a condition; 2: and so are the blocks of ranks.
    auto weights = [&](int32_t adapter, int64_t n0, int b0, auto &w, auto kind) __attribute__((always_inline)) {
        constexpr int KIND = decltype(kind)::value;
        constexpr int U = sizeof(w) / sizeof(w[0]);
        const T *up = a.up + ((int64_t)adapter * a.outputs + n0) * a.rank;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool last = KIND < 2 && b0 + u == blocks - 1;
            const int r = last ? last_run.from : 16 * (b0 + u) + L * run0;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int shift = 32 * (c >> 1) + 4 * (c & 1);
                if constexpr (KIND > 0) {
                    const uint4 v = load_run(reinterpret_cast<const T *>(reinterpret_cast<const uint8_t *>(up + shift * a.rank) + (uint32_t)(line * a.rank + r) * (uint32_t)sizeof(T)));
                    w[u][c] = last ? make_uint4(v.x & last_kept[0], v.y & last_kept[1], v.z & last_kept[2], v.w & last_kept[3]) : v;
                } else {
                    const int64_t n = n0 + shift + line;
                    const uint4 v = load_run(a.up + ((int64_t)adapter * a.outputs + (n < a.outputs ? n : a.outputs - 1)) * a.rank + r, (int64_t)a.rank - r);
                    w[u][c] = last ? make_uint4(v.x & last_kept[0], v.y & last_kept[1], v.z & last_kept[2], v.w & last_kept[3]) : v;
                }
            }
        }
    };
    // ── the terms: a thread's runs are all of one row ──
    static_assert(64 * kUpWaves % (16 * RW) == 0);
    const int runs = kRuns * blocks, my_row = tid % (16 * RW);
    const int32_t my_id = occurring.of(my_row);
    const float my_scale = a.scales != nullptr && my_id >= 0 ? a.scales[my_id] : 1.0f;
    auto each = [&](auto f) __attribute__((always_inline)) {
        const int64_t row = row0 + my_row < a.rows ? row0 + my_row : a.rows - 1, split = a.rows * a.padded;
        for (int run = tid / (16 * RW); run < runs; run += 64 * kUpWaves / (16 * RW)) {
            const RankRun of = rank_run<T>(a.rank, run);
            const float *p = a.low + row * a.padded + of.from;
            float t[L];
#pragma unroll
            for (int j = 0; j < L; j++) t[j] = 0.0f;
            for (int z = 0; z < a.splits; z += 4) {  // (four splits' loads under way at a time)
                uint4 v[4][L / 4];
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int j = 0; j < L / 4; j++) v[s][j] = load_run(p + (z + s < a.splits ? z + s : z) * split + 4 * j);
#pragma unroll
                for (int s = 0; s < 4; s++)
#pragma unroll
                    for (int j = 0; j < L / 4; j++) {
                        const float w[4] = {u2f(v[s][j].x), u2f(v[s][j].y), u2f(v[s][j].z), u2f(v[s][j].w)};
#pragma unroll
                        for (int e = 0; e < 4; e++) t[4 * j + e] += z + s < a.splits ? w[e] : 0.0f;
                    }
            }
#pragma unroll
            for (int j = 0; j < L; j++) t[j] = of.any && j >= of.skip ? t[j] * my_scale : 0.0f;
            f(run, t);
        }
    };
    if constexpr (kScaled) {  // a row's t is scaled by a power of two, so that its largest is between 1 and 2
        if (tid < 16 * RW) largest[tid] = 0u;
        __syncthreads();
        each([&](int, const float (&t)[L]) __attribute__((always_inline)) {
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < L; j++) top = fabsf(t[j]) < INFINITY ? fmaxf(top, fabsf(t[j])) : top;
            atomicMax(&largest[my_row], f2u(top));
        });
        __syncthreads();
    }
    auto exponent_of = [&](int r) __attribute__((always_inline)) { return largest[r] != 0u ? ilogbf(u2f(largest[r])) : 0; };
    each([&](int run, float (&t)[L]) __attribute__((always_inline)) {
        if constexpr (kScaled) {
            const int e = exponent_of(my_row);
#pragma unroll
            for (int j = 0; j < L; j++) t[j] = ldexpf(t[j], -e);
        }
        put_terms<T>(terms + ((my_row >> 4) * blocks + run / kRuns) * 64, my_row & 15, run % kRuns, t);
    });
    int32_t id[RW];
    int exponent[RW] = {};
#pragma unroll
    for (int i = 0; i < RW; i++) id[i] = occurring.of(16 * i + col);
    __syncthreads();
    if constexpr (kScaled)
#pragma unroll
        for (int i = 0; i < RW; i++) exponent[i] = exponent_of(16 * i + col);

    // ── the products ──
    auto products = [&](int64_t n0, auto kind) __attribute__((always_inline)) {
        for (Occurring at = occurring; at.any(); at.next()) {
            const int32_t adapter = at.now();
            acc4_t acc[RW][4];
#pragma unroll
            for (int i = 0; i < RW; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[i][c] = acc4_t{0.0f, 0.0f, 0.0f, 0.0f};
            auto add = [&](int b, const uint4 (&w)[4]) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const uint4 t = terms[(i * blocks + b) * 64 + lane];
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[i][c] = product16<T>(w[c], t, acc[i][c]);
                }
            };
            int b = 0;
            for (; b + 2 <= blocks; b += 2) {
                uint4 w[2][4];
                weights(adapter, n0, b, w, kind);
                add(b, w[0]), add(b + 1, w[1]);
            }
            if (b < blocks) {
                uint4 w[1][4];
                weights(adapter, n0, b, w, kind);
                add(b, w[0]);
            }
#pragma unroll
            for (int i = 0; i < RW; i++) {
                if constexpr (kScaled)
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[i][c][e] = ldexpf(acc[i][c][e], exponent[i]);
                if (id[i] == adapter)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        *reinterpret_cast<acc4_t *>(&sums[16 * i + col][64 * wave + 32 * (c >> 1) + 8 * quarter + 4 * (c & 1)]) = acc[i][c];
            }
        }
    };
    for (int64_t n0 = n_first; n0 < n_end; n0 += kBlockColumns) {
        const int64_t from = n0 + 64 * wave;
        if (a.rank % 16 == 0 && from + 64 <= a.outputs) products(from, Count<2>{});
        else if (a.rank >= L && from + 64 <= a.outputs) products(from, Count<1>{});
        else if (from < a.outputs) products(from, Count<0>{});
        __syncthreads();
        const bool whole = n0 < n_whole;
#pragma unroll
        for (int i = 0; i < 2 * RW; i++) {
            const int r = 8 * i + y_row;
            const int64_t n = n0 + y_col, left = a.outputs - n;
            float v[8];
            if (whole) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = Elem<T>::load(ahead[i].t, e);
            }
            if ((mine >> r & 1) == 0) continue;
            if (!whole) load_eight(a.y + (row0 + r) * a.y_stride + (left > 0 ? n : 0), left, v);
            if ((bare >> r & 1) == 0) {
                const acc4_t s0 = *reinterpret_cast<const acc4_t *>(&sums[r][y_col]), s1 = *reinterpret_cast<const acc4_t *>(&sums[r][y_col + 4]);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += s0[e], v[4 + e] += s1[e];
            }
            store_eight(a.out + (row0 + r) * a.out_stride + n, whole ? 8 : left, v);
        }
        if (whole) request(n0 + kBlockColumns < n_whole ? n0 + kBlockColumns : n0);
        __syncthreads();
    }
}

// How the rows, columns and the contraction are dealt to blocks.
struct Shape {
    // Tiles of 16 rows of a block: 2 where there are many rows, so that the adapters' weights are read half as often.  (4096 rows beside [14336, 4096] 90 us,
    // with 1 113; 2048 beside [4096, 4096] 21.7 and 23.6, where the rule changes; 1024 23.4 with 2, 18.8 with 1; 64 rows 63 with 2, 12.4 with 1.)
    int32_t wide;
    int32_t splits, down_slots, up_slots, chunks;
    int64_t tiles;
};
int64_t at_most(int64_t v, int64_t most) { return v < 1 ? 1 : v < most ? v : most; }
Shape shape_of(const nvq_adapters_desc &d) {
    Shape s{};
    const int64_t cus = compute_units();
    s.wide = d.rows >= 32 * cus / 4 ? 2 : 1;
    s.tiles = (d.rows + 16 * s.wide - 1) / (16 * s.wide);
    const int64_t most = d.adapters < 16 * s.wide ? d.adapters : 16 * s.wide, occurring = at_most(most < d.rows ? most : d.rows, 32);
    const int64_t step = d.dtype == NVQ_F32 ? 16 : 32, steps = (d.inputs + step - 1) / step;
    // A tile's adapters go to blocks of their own where the tiles alone leave compute units without work, and the contraction is split, four steps a
    // wavefront at least.  (The 64 rows: one block for all adapters 34 us, four 17, sixteen 12.6; one split 17.9, two 14.4, four 12.7, eight 12.7.  4096 rows:
    // slots of 1, 4 and 8 89, 96 and 110, splits of 1, 2, 4 and 8 110, 92, 89 and 98.)
    s.down_slots = s.wide == 2 ? 1 : (int32_t)at_most(cus / s.tiles, occurring);
    s.splits = (int32_t)at_most(2 * cus / (s.tiles * s.down_slots), at_most(steps / (4 * kDownWaves), 16));
    const int64_t columns = (d.outputs + kBlockColumns - 1) / kBlockColumns;
    // The second kernel: slots in the same way (the 64 rows: 1, 4, 8 and 16 21, 13.8, 12.5 and 12.7), and two or three times 256 columns a block, whose terms are
    // then worked out once, where blocks are several times what the chip holds (4096 rows beside [14336, 4096]: 1, 2, 3, 4 and 6 times 103, 90.8, 87.5, 89.4 and
    // 92.5; 2048 beside [4096, 4096] 24.6, 21.6, 24.8 and 26.4; 1024, in blocks of 16 rows, 18.9, 20.2 and 23; the 64 rows 12.5, 13.3 and 15.5).
    s.up_slots = (int32_t)at_most(4 * cus / (s.tiles * columns), occurring);
    s.chunks = (int32_t)at_most(s.tiles * columns * s.up_slots / ((s.wide == 2 ? 2 : 4) * cus), 3);
    return s;
}
int32_t padded_rank(const nvq_adapters_desc &d) { return d.adapters == 0 ? 0 : (d.rank + 15) / 16 * 16; }

template <typename T, int RW>
int32_t run_sized(const AdapterArgs<T> &a, const Shape &shape, hipStream_t s) {
    const dim3 grid((unsigned)shape.tiles, (unsigned)shape.splits, (unsigned)shape.down_slots), block(64 * kDownWaves);
    if (a.padded > 0) {  // (without adapters there are no shares, nor need there be an x)
        if (a.padded <= 16) hipLaunchKernelGGL((adapters_down_kernel<T, RW, 1>), grid, block, 0, s, a);
        else if (a.padded <= 32) hipLaunchKernelGGL((adapters_down_kernel<T, RW, 2>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((adapters_down_kernel<T, RW, 4>), grid, block, 0, s, a);
        NVQ_LAUNCH_CHECK("apply_adapters");
    }
    const int64_t columns = kBlockColumns * (int64_t)shape.chunks;
    const dim3 wide((unsigned)shape.tiles, (unsigned)((a.outputs + columns - 1) / columns), (unsigned)shape.up_slots);
    const size_t terms = (size_t)RW * (a.padded / 16) * 64 * sizeof(uint4), sums = 16 * RW * (kBlockColumns + 5) * sizeof(float);
    static std::atomic<bool> configured = false;
    if (terms + sums > 64 * 1024 && !configured) {  // (32 rows and ranks from 241 on)
        NVQ_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(adapters_up_kernel<T, RW>), hipFuncAttributeMaxDynamicSharedMemorySize, RW * 16 * 1024));
        configured = true;
    }
    hipLaunchKernelGGL((adapters_up_kernel<T, RW>), wide, dim3(64 * kUpWaves), terms, s, a);
    NVQ_LAUNCH_CHECK("apply_adapters");
    return NVQ_OK;
}

template <typename T>
int32_t run_adapters(const nvq_adapters_desc &d, const void *x, const void *down, const void *up, const float *scales, const int32_t *ids, const void *y,
                     void *out, void *workspace, hipStream_t s) {
    const Shape shape = shape_of(d);
    AdapterArgs<T> a{};
    a.x = (const T *)x, a.down = (const T *)down, a.up = (const T *)up, a.y = (const T *)y, a.scales = scales, a.ids = ids, a.out = (T *)out;
    a.low = (float *)workspace, a.rows = d.rows, a.inputs = d.inputs, a.outputs = d.outputs;
    a.x_stride = d.x_stride, a.y_stride = d.y_stride, a.out_stride = d.out_stride;
    a.adapters = (int32_t)d.adapters, a.rank = d.adapters == 0 ? 0 : d.rank, a.padded = padded_rank(d), a.splits = shape.splits, a.chunks = shape.chunks;
    return shape.wide == 2 ? run_sized<T, 2>(a, shape, s) : run_sized<T, 1>(a, shape, s);
}

}  // namespace

size_t adapters_workspace_bytes(const nvq_adapters_desc &d) { return (size_t)shape_of(d).splits * (size_t)d.rows * (size_t)padded_rank(d) * sizeof(float); }

int32_t launch_adapters(const nvq_adapters_desc &d, const void *x, const void *down, const void *up, const float *scales, const int32_t *ids, const void *y,
                        void *out, void *workspace, hipStream_t s) {
    if (d.dtype == NVQ_F32) return run_adapters<float>(d, x, down, up, scales, ids, y, out, workspace, s);
    if (d.dtype == NVQ_BF16) return run_adapters<bf16_t>(d, x, down, up, scales, ids, y, out, workspace, s);
    return run_adapters<f16_t>(d, x, down, up, scales, ids, y, out, workspace, s);
}

}  // namespace nvq
