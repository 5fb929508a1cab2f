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
};

}  // namespace nvq
