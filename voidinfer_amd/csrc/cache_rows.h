// cache_rows.h — device-side view of a paged cache and of the rows that a call
// brings to it, shared by the append and the attention kernels.
#pragma once

#include "vi_device.h"
#include "vi_internal.h"

namespace vi {

// The lane whose rows hold row r: the last with row_offsets[lane] <= r.
__device__ __forceinline__ int lane_of_row(const int32_t* offsets, int lanes, int r) {
    int lo = 0, hi = lanes - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offsets[mid] <= r) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Page of a lane's cache index, or -1 where the table or the page is out of range.
__device__ __forceinline__ int page_of(const vi_lane_rows& l, int pages, int page_size, int lane, int64_t index) {
    const int64_t e = index / page_size;
    if (index < 0 || e >= l.table_width) return -1;
    const int p = l.tables[int64_t(lane) * l.table_stride + e];
    return uint32_t(p) < uint32_t(pages) ? p : -1;
}

}  // namespace vi
