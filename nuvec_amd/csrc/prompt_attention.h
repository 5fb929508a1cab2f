// The launches of attention over keys and values as the projections leave them, one translation unit per element type.
#pragma once

#include "nvq_internal.h"
#include "paged_schedule.h"

namespace nvq {
namespace prompt {

constexpr int kWaves = 4;               // of a block
constexpr int kLines = 32 * kWaves;     // (rows x query heads of a key head) of a block
constexpr size_t kPlanBytes = 64;       // in front of the states

// Sequences behind one another (paged_schedule.h deals their lines to blocks).
struct PromptBatch {
    const int32_t *starts, *key_starts;  // NULL: one sequence of all rows; of all keys
    int64_t rows, keys, window;
    int32_t sequences, key_heads, rep, causal, few, target, least;

    __device__ __forceinline__ int64_t first_row(int b) const { return starts == nullptr ? 0 : starts[b]; }
    __device__ __forceinline__ int64_t end_row(int b) const { return starts == nullptr ? rows : starts[b + 1]; }
    __device__ __forceinline__ int64_t within(int64_t key) const { return key < 0 ? 0 : key < keys ? key : keys; }
    __device__ __forceinline__ int64_t first_key(int b) const { return key_starts == nullptr ? 0 : within(key_starts[b]); }
    __device__ __forceinline__ int64_t length(int b) const { return (key_starts == nullptr ? keys : within(key_starts[b + 1])) - first_key(b); }
    __device__ __forceinline__ int64_t most() const { return keys; }
};

struct PromptLaunch {
    PromptBatch batch;
    uint32_t grid, merge_units;  // merge_units 0: nothing can be split
    int32_t slots;               // states that the workspace holds
    int32_t turn, back;          // where the order of blocks turns back (turned), and for how many: eights
};

int32_t launch_bf16(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, const PromptLaunch &r, hipStream_t s);
int32_t launch_f16(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, const PromptLaunch &r, hipStream_t s);
int32_t launch_f32(const nvq_prompt_attention_desc &d, const PromptAttentionOperands &o, const PromptLaunch &r, hipStream_t s);

// The head sizes that kernels are made for: a head lies in the next of them, with zeros behind it.
constexpr int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256; }

// Blocks of a compute unit: three where the accumulators of 64 values leave room for them (8192 rows of 32 heads of 64 over 8: bfloat16 441 us
// with two, 433 with three, float16 457 and 448), two of heads up to 128, one behind that.
constexpr int blocks_of(int bytes, int padded) { return bytes == 2 && padded == 64 ? 3 : padded <= 128 ? 2 : 1; }

}  // namespace prompt
}  // namespace nvq
