// How the rows of a batch of sequences, whose lengths the device alone knows, are dealt to blocks.
//
// A unit is one key head of one sequence and up to LINES of its lines (a line: one query row of one query head, line r of a sequence
// being row r / rep, head r % rep of the key head); its keys are walked in tiles of 32, in one item or, where the call has few units
// for the chip, in several items of `per` tiles each, whose states are merged.  Every wavefront works the same plan out for itself from
// the lengths (one round trip and two scans over them), so that nothing is laid out beforehand, a captured launch follows its
// lengths, and the items are equally long however the lengths differ.
#pragma once

#include "nvq_device.h"
#include "paged.h"

namespace nvq {

struct PagedBatch {
    PagedPlace place;
    const int32_t *lengths, *starts;  // starts NULL: sequence b has row b alone
    int64_t rows, window;
    int32_t sequences, key_heads, rep, causal;
    int32_t few;     // lines of a sequence that the kernel of few rows takes; more are the other kernel's
    int32_t target;  // items that fill the chip
};

namespace {

constexpr int kScheduleKeys = 32;   // keys of a tile
constexpr int kScheduleTiles = 8;   // of an item at least, where a unit is more than one item

struct PagedSequence {
    int32_t start, rows, length, base, tiles, parts;  // base: the first key that a row sees, rounded down to a tile
};

// KIND 0: the sequences of few lines, 1: the others (parts 0: not this kernel's).
template <int LINES, int KIND>
__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch &a, int b) {
    PagedSequence s{};
    if (b >= a.sequences) return s;
    const int64_t first = a.starts == nullptr ? b : a.starts[b], end = a.starts == nullptr ? b + 1 : a.starts[b + 1];
    const int64_t from = first < 0 ? 0 : first < a.rows ? first : a.rows, to = end < from ? from : end < a.rows ? end : a.rows;
    const int64_t length = a.lengths[b], most = a.place.capacity();
    s.start = (int32_t)from, s.rows = (int32_t)(to - from);
    s.length = (int32_t)(length < 0 ? 0 : length < most ? length : most);
    const int64_t seen = (int64_t)s.length - s.rows - a.window + 1;
    s.base = a.causal && a.window > 0 && seen > 0 ? (int32_t)(seen / kScheduleKeys * kScheduleKeys) : 0;
    s.tiles = (s.length - s.base + kScheduleKeys - 1) / kScheduleKeys;
    const int64_t lines = (int64_t)s.rows * a.rep;
    s.parts = (lines <= a.few) == (KIND == 0) ? (int32_t)((lines + LINES - 1) / LINES) : 0;
    return s;
}

template <typename V> __device__ __forceinline__ V wave_total(V v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ int32_t wave_prefix(int32_t v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int32_t u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

struct PagedPlan {
    int32_t per, items;  // tiles of an item; items of all sequences
    __device__ __forceinline__ int32_t splits(const PagedSequence &s) const { return s.tiles <= per ? 1 : (s.tiles + per - 1) / per; }
};

template <int LINES, int KIND>
__device__ __forceinline__ PagedPlan paged_plan(const PagedBatch &a, int lane, const PagedSequence &first) {
    int64_t total = 0, units = 0;
    for (int b0 = 0; b0 < a.sequences; b0 += 64) {
        const PagedSequence s = b0 == 0 ? first : paged_sequence<LINES, KIND>(a, b0 + lane);
        const int64_t u = (int64_t)s.parts * a.key_heads;
        units += u, total += u * s.tiles;
    }
    units = wave_total(units), total = wave_total(total);
    // Every unit's last item may be short.  The shortest items of three whose number is within the target: none, half an item, or one of
    // every unit left for that, half of the target at most.
    PagedPlan p[3];
#pragma unroll
    for (int i = 0; i < 3; i++) {
        const int64_t left = a.target - units * i / 2 > a.target / 2 ? a.target - units * i / 2 : a.target / 2, per = (total + left - 1) / left;
        p[i].per = (int32_t)(per < kScheduleTiles ? kScheduleTiles : per < (1 << 26) ? per : 1 << 26), p[i].items = 0;
    }
    for (int b0 = 0; b0 < a.sequences; b0 += 64) {
        const PagedSequence s = b0 == 0 ? first : paged_sequence<LINES, KIND>(a, b0 + lane);
#pragma unroll
        for (int i = 0; i < 3; i++) p[i].items += s.parts * p[i].splits(s) * a.key_heads;
    }
#pragma unroll
    for (int i = 0; i < 3; i++) p[i].items = wave_total(p[i].items);
    return p[0].items <= a.target ? p[0] : p[1].items <= a.target ? p[1] : p[2];
}

struct PagedItem {
    PagedSequence s;      // uniform in the wavefront
    int32_t b, splits, per, part, split, head;
    int32_t slot;         // of the item's state among the items of sequences with several splits
};

// Item `at`, or (UNITS) unit `at` of the sequences with several splits, its `slot` that of its first split.
template <int LINES, int KIND, bool UNITS>
__device__ __forceinline__ bool paged_find(const PagedBatch &a, const PagedPlan &p, int lane, const PagedSequence &first, int32_t at, PagedItem &item) {
    int32_t slots = 0;
    for (int b0 = 0; b0 < a.sequences; b0 += 64) {
        const PagedSequence s = b0 == 0 ? first : paged_sequence<LINES, KIND>(a, b0 + lane);
        const int32_t splits = p.splits(s), own = s.parts * a.key_heads, count = UNITS ? (splits > 1 ? own : 0) : own * splits;
        const int32_t state = splits > 1 ? own * splits : 0;
        const int32_t end = wave_prefix(count, lane), state_end = wave_prefix(state, lane);
        const uint64_t behind = __ballot(end > at);
        if (behind != 0) {
            const int l = __builtin_ctzll(behind);
            auto of = [&](int32_t v) { return __builtin_amdgcn_readlane(v, l); };
            item.s = PagedSequence{of(s.start), of(s.rows), of(s.length), of(s.base), of(s.tiles), of(s.parts)};
            item.b = b0 + l, item.splits = of(splits), item.per = p.per;
            const int32_t within = at - of(end - count), first_slot = slots + of(state_end - state);
            // (part, split, head), heads fastest: a key head's parts lie key_heads x splits apart, on one XCD where that is a multiple of 8
            item.head = within % a.key_heads;
            const int32_t rest = within / a.key_heads;
            if (UNITS) item.part = rest, item.split = 0;
            else item.split = rest % item.splits, item.part = rest / item.splits;
            item.slot = first_slot + (item.part * item.splits + item.split) * a.key_heads + item.head;
            return true;
        }
        at -= __builtin_amdgcn_readlane(end, 63), slots += __builtin_amdgcn_readlane(state_end, 63);
    }
    return false;
}

// Item (or unit) `at` of the whole plan; false behind the last.
template <int LINES, int KIND, bool UNITS>
__device__ __forceinline__ bool paged_item(const PagedBatch &a, int lane, int32_t at, PagedItem &item) {
    const PagedSequence first = paged_sequence<LINES, KIND>(a, lane);
    const PagedPlan plan = paged_plan<LINES, KIND>(a, lane, first);
    return at < plan.items && paged_find<LINES, KIND, UNITS>(a, plan, lane, first, at, item);
}

}  // namespace
}  // namespace nvq
