// Where the packed tokens of a call over a paged KV cache lie.
#pragma once

#include "device_utils.h"
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

// Lanes of a wave exchange data through LDS: everything written before is there for the others.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Sequence b's tokens [start, start + tokens), the first at position history; no tokens where the scalars are out of range.
struct Span {
    int32_t start;
    int32_t tokens;
    int32_t history;
};

__device__ __forceinline__ Span span_of(const int32_t* starts, const int32_t* history, int b, int64_t total) {
    Span s{starts[b], 0, history[b]};
    const int32_t end = starts[b + 1];
    if (s.start >= 0 && end >= s.start && end <= total && s.history >= 0) { s.tokens = end - s.start; }
    return s;
}

// Units of work dealt out by sequence, `units(span(b))` for each: the sequence that holds unit u and u's place in it (b -1: past the
// last). For the whole wave, 64 sequences at a time.
struct Found {
    int b;
    int at;
    Span s;
};

template <typename S, typename F>
__device__ __forceinline__ Found find_unit(int B, int u, int lane, S span, F units) {
    int sum = 0;
    for (int base = 0; base < B; base += 64) {
        Span s{0, 0, 0};
        int n = 0;
        if (base + lane < B) {
            s = span(base + lane);
            n = units(s);
        }
        const int end = sum + wave_inclusive_scan(n);
        const uint64_t past = __ballot(end > u);
        if (past != 0u) {
            const int l = __ffsll(static_cast<long long>(past)) - 1;
            const int count = __builtin_amdgcn_readlane(n, l), at = u - (__builtin_amdgcn_readlane(end, l) - count);
            if (at < 0 || at >= count) { break; } // (starts that descend may promise more units than whole numbers count)
            return Found{base + l, at,
                         Span{__builtin_amdgcn_readlane(s.start, l), __builtin_amdgcn_readlane(s.tokens, l), __builtin_amdgcn_readlane(s.history, l)}};
        }
        sum = __builtin_amdgcn_readlane(end, 63);
    }
    return Found{-1, 0, Span{0, 0, 0}};
}

} // namespace
} // namespace nmi
