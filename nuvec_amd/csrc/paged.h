// Where a sequence's positions lie in a pool of pages: page table[sequence][position / page], and in it the position's place.
// Keys and values are [pages, key heads, page, ...]: a head's rows of a page are consecutive.
#pragma once

#include "nvq_device.h"

namespace nvq {

struct PagedPlace {
    const int32_t *table;   // [sequences, columns], rows `stride` apart
    int64_t stride, pages;
    int32_t sequences, columns, page_shift;

    __host__ __device__ __forceinline__ int64_t capacity() const { return (int64_t)columns << page_shift; }
    // Row of a head's first position of the page, of [pages x heads x page] rows; an id outside the pool is the caller's error: clamped.
    __device__ __forceinline__ int64_t page_of(int64_t sequence, int64_t column) const {
        const int64_t id = table[sequence * stride + column];
        return id < 0 ? 0 : id < pages ? id : pages - 1;
    }
};

}  // namespace nvq
