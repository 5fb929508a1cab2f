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
    int32_t least;   // tiles of an item, where a unit is more than one
};

namespace {

constexpr int kScheduleKeys = 32;   // keys of a tile

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

// Scans on the vector unit alone (data-parallel moves; the same through LDS took 1 us of a call): shifts by 1, 2, 4, 8 in each row of 16
// lanes, then the rows' totals carried into the next rows.
template <int CTRL, int ROWS> __device__ __forceinline__ int32_t scan_step(int32_t v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true); }
__device__ __forceinline__ int32_t wave_prefix(int32_t v) {  // inclusive
    v = scan_step<0x111, 0xF>(v);
    v = scan_step<0x112, 0xF>(v);
    v = scan_step<0x114, 0xF>(v);
    v = scan_step<0x118, 0xF>(v);
    v = scan_step<0x142, 0xA>(v);
    return scan_step<0x143, 0xC>(v);
}
__device__ __forceinline__ int32_t wave_total(int32_t v) { return __builtin_amdgcn_readlane(wave_prefix(v), 63); }
// Of whole numbers below 2^53.
template <int CTRL, int ROWS> __device__ __forceinline__ double scan_step(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xF, true);
    return v + __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}
__device__ __forceinline__ double wave_total(double v) {
    v = scan_step<0x111, 0xF>(v);
    v = scan_step<0x112, 0xF>(v);
    v = scan_step<0x114, 0xF>(v);
    v = scan_step<0x118, 0xF>(v);
    v = scan_step<0x142, 0xA>(v);
    v = scan_step<0x143, 0xC>(v);
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}

// What all lanes hold, as the compiler can see: in a scalar register, and branches on it without masks of lanes.  (Of a value that has come
// through the search for an item the move alone is folded away, and the value taken for one that differs by lane.)
__device__ __forceinline__ int32_t uniform(int32_t v) {
    v = __builtin_amdgcn_readfirstlane(v);
    asm("" : "+s"(v));
    return v;
}

struct PagedPlan {
    int32_t per, items;  // tiles of an item; items of all sequences
    __device__ __forceinline__ int32_t splits(const PagedSequence &s) const { return s.tiles <= per ? 1 : (s.tiles + per - 1) / per; }
};

template <int LINES, int KIND>
__device__ __forceinline__ PagedPlan paged_plan(const PagedBatch &a, int lane, const PagedSequence &first) {
    double total = 0.0;
    int32_t units = 0;
    for (int b0 = 0; b0 < a.sequences; b0 += 64) {
        const PagedSequence s = b0 == 0 ? first : paged_sequence<LINES, KIND>(a, b0 + lane);
        const int32_t u = s.parts * a.key_heads;
        units += u, total += (double)u * (double)s.tiles;
    }
    units = wave_total(units), total = wave_total(total);
    // Every unit's last item may be short.  The shortest items of three whose number is within the target: none, half an item, or one of
    // every unit left for that, half of the target at most.
    PagedPlan p[3];
#pragma unroll
    for (int i = 0; i < 3; i++) {
        const int32_t spare = units > a.target ? a.target : units, left = a.target - spare * i / 2 > a.target / 2 ? a.target - spare * i / 2 : a.target / 2;
        const double per = ceil(total / (double)left);
        p[i].per = per < a.least ? a.least : per < (double)(1 << 26) ? (int32_t)per : 1 << 26, p[i].items = 0;
    }
    for (int b0 = 0; b0 < a.sequences; b0 += 64) {
        const PagedSequence s = b0 == 0 ? first : paged_sequence<LINES, KIND>(a, b0 + lane);
#pragma unroll
        for (int i = 0; i < 3; i++) p[i].items += s.parts * p[i].splits(s) * a.key_heads;
    }
#pragma unroll
    for (int i = 0; i < 3; i++) p[i].items = wave_total(p[i].items), p[i].per = __builtin_amdgcn_readfirstlane(p[i].per);
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
        const int32_t end = wave_prefix(count), state_end = wave_prefix(state);
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

// Item (or unit, which comes after the items) `at` of the whole plan; false behind the last.  `length`: where the first block of the items leaves the
// plan's length for the units'; NULL: nothing is split.
template <int LINES, int KIND, bool UNITS>
__device__ __forceinline__ bool paged_item(const PagedBatch &a, int lane, int32_t at, int32_t *length, PagedItem &item) {
    const PagedSequence first = paged_sequence<LINES, KIND>(a, lane);
    PagedPlan plan;
    if constexpr (UNITS) {
        plan.per = *length, plan.items = INT32_MAX;
    } else {
        plan = paged_plan<LINES, KIND>(a, lane, first);
        if (at == 0 && threadIdx.x == 0 && length != nullptr) *length = plan.per;
    }
    const bool found = at < plan.items && paged_find<LINES, KIND, UNITS>(a, plan, lane, first, at, item);
    if (uniform(found) == 0) return false;
    const PagedSequence &s = item.s;
    item = PagedItem{{uniform(s.start), uniform(s.rows), uniform(s.length), uniform(s.base), uniform(s.tiles), uniform(s.parts)},
                     uniform(item.b), uniform(item.splits), uniform(item.per), uniform(item.part), uniform(item.split), uniform(item.head), uniform(item.slot)};
    return true;
}

}  // namespace
}  // namespace nvq
