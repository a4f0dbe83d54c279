// Where the packed tokens of a call over a paged KV cache lie.
#pragma once

#include "paged_internal.h"

namespace nmi {
namespace {

// Where packed token n lies: page -1 where its row has none; seq -1 where no sequence has the token.
struct Place {
    int32_t seq;
    int32_t page;
    int32_t row;
};

__device__ __forceinline__ Place place_of(int64_t n, const int32_t* starts, const int32_t* history, const PagedRef& c) {
    int lo = 0, hi = c.B; // the last sequence that starts at or before n
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= n) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    Place p{-1, -1, 0};
    if (starts[lo] < 0 || n < starts[lo] || n >= starts[lo + 1]) { return p; }
    p.seq = lo;
    const int64_t pos = static_cast<int64_t>(history[lo]) + (n - starts[lo]);
    if (history[lo] < 0 || (pos >> c.page_shift) >= c.max_pages) { return p; }
    const int32_t page = c.table[lo * c.table_row + (pos >> c.page_shift)];
    p.page = page >= 0 && page < c.pages ? page : -1;
    p.row = static_cast<int32_t>(pos & ((int64_t{1} << c.page_shift) - 1));
    return p;
}

} // namespace
} // namespace nmi
