// The pages of a paged KV cache on gfx950: copied, handed out, given back, shared and moved together.
//
// `refs` counts the table entries of every page; a page without any is free. Who gets which page is defined: the lowest free
// pages in the order of the sequences and their entries. Counts change by atomic adds of whole numbers, whose order
// does not matter.
// What bounds it: copies by HBM; the rest by latency: one workgroup (its own barriers order its steps, and a second launch would cost
// more than its waves) reads the counts once, 64 pages to a word of bits in LDS, and finds the k-th free page there by
// a search over the words' sums. Handing out pages to 64 sequences takes 7.9 us, a compaction of a pool of 6,144 pages 6.7 and 5.3 for
// its table, a fork of 48 sequences 6.3 in a table 12 pages wide. A fork writes every entry of the children's rows, so it grows with the
// table's width, whatever the sequences hold: with the call 8.1 us at 12 pages, 17.6 at 512, 87.5 at 4,096.
#include "common.h"
#include "device_utils.h"
#include "paged_internal.h"

#include <algorithm>

namespace nmi {
namespace {

// ---- copies --------------------------------------------------------------------------------------

constexpr int kMostPlanes = 6; // K, V, their scales, the block means' codes and scales
constexpr int kPiece = 16384;  // bytes of a workgroup's piece

struct CopyArgs {
    PagePlane plane[kMostPlanes];
    int32_t first[kMostPlanes + 1]; // pieces of a page: plane i has first[i] .. first[i + 1] - 1
    int32_t planes;
    int32_t pages;
    const int32_t* src;
    const int32_t* dst;
};

// A workgroup copies 16 KiB, four loads a thread ahead of the stores: 300 MB read and written in 49 us (6.1 TB/s).
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyArgs a) {
    const int pieces = a.first[a.planes];
    const int pair = blockIdx.x / pieces;
    const int piece = blockIdx.x - pair * pieces;
    const int32_t from = a.src[pair], to = a.dst[pair];
    if (from < 0 || from >= a.pages || to < 0 || to >= a.pages || from == to) { return; }
    int p = 0;
    while (piece >= a.first[p + 1]) { ++p; }
    const int64_t at = static_cast<int64_t>(piece - a.first[p]) * kPiece;
    const int64_t left = a.plane[p].bytes - at;
    const char* s = a.plane[p].data + from * a.plane[p].stride + at;
    char* d = a.plane[p].data + to * a.plane[p].stride + at;
    if (left >= kPiece && a.plane[p].wide) {
        i4 v[kPiece / 4096];
#pragma unroll
        for (int i = 0; i < kPiece / 4096; ++i) { v[i] = *reinterpret_cast<const i4*>(s + 4096 * i + 16 * threadIdx.x); }
#pragma unroll
        for (int i = 0; i < kPiece / 4096; ++i) { *reinterpret_cast<i4*>(d + 4096 * i + 16 * threadIdx.x) = v[i]; }
        return;
    }
    if (a.plane[p].wide) {
        for (int64_t i = 16 * threadIdx.x; i < left; i += 4096) { *reinterpret_cast<i4*>(d + i) = *reinterpret_cast<const i4*>(s + i); }
    } else {
        for (int64_t i = 4 * threadIdx.x; i < min(left, static_cast<int64_t>(kPiece)); i += 1024) {
            *reinterpret_cast<int32_t*>(d + i) = *reinterpret_cast<const int32_t*>(s + i);
        }
    }
}

// ---- free pages ----------------------------------------------------------------------------------

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

// A bit per page in dynamic LDS, set for the free ones, 64 pages a word, and the words' running sums.
struct Bits {
    uint64_t* word;
    int32_t* sum; // free pages before the word
    int words;
    int pages;
    int total; // free pages
};

// For the whole workgroup. `part` is scratch.
__device__ Bits free_pages(const int32_t* refs, int pages, uint64_t* lds, int32_t* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Bits b{lds, nullptr, (pages + 63) / 64, pages, 0};
    b.sum = reinterpret_cast<int32_t*>(lds + b.words);
    constexpr int kAhead = 16; // words of a wave on their way
    for (int w0 = wave; w0 < b.words; w0 += kAhead * kWaves) {
        int32_t n[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) { n[i] = refs[min(64 * (w0 + i * kWaves) + lane, pages - 1)]; }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int w = w0 + i * kWaves;
            const uint64_t m = __ballot(64 * w + lane < pages && n[i] == 0);
            if (lane == 0 && w < b.words) { b.word[w] = m; }
        }
    }
    __syncthreads();
    // running sums: a run of words for each thread
    const int each = (b.words + kThreads - 1) / kThreads;
    const int w0 = min(static_cast<int>(threadIdx.x) * each, b.words), w1 = min(w0 + each, b.words);
    int n = 0;
    for (int w = w0; w < w1; ++w) { n += __popcll(b.word[w]); }
    const int end = wave_inclusive_scan(n);
    if (lane == 63) { part[wave] = end; }
    __syncthreads();
    int before = end - n;
    for (int i = 0; i < kWaves; ++i) {
        before += i < wave ? part[i] : 0;
        b.total += part[i];
    }
    for (int w = w0; w < w1; ++w) {
        b.sum[w] = before;
        before += __popcll(b.word[w]);
    }
    __syncthreads();
    return b;
}

// The k-th free page (USED: page in use) from 0, the lowest first; -1 where there is none.
template <bool USED>
__device__ int nth_page(const Bits& b, int k) {
    if (k < 0 || k >= (USED ? b.pages - b.total : b.total)) { return -1; }
    const auto before = [&](int w) { return USED ? 64 * w - b.sum[w] : b.sum[w]; };
    int lo = 0, hi = b.words; // the last word with at most k of them before it
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before(mid) <= k) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    uint64_t m = USED ? ~b.word[lo] : b.word[lo]; // (pages past the last one stand behind all others)
    int left = k - before(lo);
    int at = 0;
#pragma unroll
    for (int half = 32; half > 0; half /= 2) {
        const int n = __popcll(m & ((uint64_t{1} << half) - 1));
        if (left >= n) {
            left -= n;
            m >>= half;
            at += half;
        }
    }
    return 64 * lo + at;
}

// Exclusive sum of v over the workgroup's threads, and the total.
struct Sum {
    int before;
    int total;
};

__device__ Sum block_sum(int v, int32_t* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int end = wave_inclusive_scan(v);
    __syncthreads();
    if (lane == 63) { part[wave] = end; }
    __syncthreads();
    Sum s{end - v, 0};
    for (int i = 0; i < kWaves; ++i) {
        s.before += i < wave ? part[i] : 0;
        s.total += part[i];
    }
    return s;
}

size_t bits_bytes(int32_t pages) { return static_cast<size_t>((pages + 63) / 64) * 12; }

// ---- handing out ---------------------------------------------------------------------------------

// The entries of a sequence's new rows: first .. first + count - 1.
struct Entries {
    int32_t first;
    int32_t count;
    int32_t tokens;
    int32_t history;
};

__device__ Entries entries_of(const PageTable& t, const int32_t* starts, const int32_t* history, int b) {
    const int32_t s = starts[b], e = starts[b + 1], h = history[b];
    if (s < 0 || e <= s || h < 0) { return Entries{0, 0, 0, 0}; }
    const int64_t last = (static_cast<int64_t>(h) + (e - s) - 1) >> t.shift;
    const int32_t first = h >> t.shift;
    return Entries{first, static_cast<int32_t>(max(int64_t{0}, min(last, static_cast<int64_t>(t.max_pages) - 1) - first + 1)), e - s, h};
}

__global__ __launch_bounds__(kThreads) void pages_reserve_kernel(PageTable t, const int32_t* starts, const int32_t* history, int32_t* granted) {
    extern __shared__ uint64_t lds[];
    __shared__ int32_t part[kWaves];
    __shared__ int32_t begin[kPagedMaxBatch + 1]; // of a sequence's entries among all
    __shared__ int32_t first[kPagedMaxBatch];     // entry of its new rows
    __shared__ int32_t lacking[kPagedMaxBatch];   // the first entry that got no page
    const int b0 = threadIdx.x;
    const Entries mine = b0 < t.B ? entries_of(t, starts, history, b0) : Entries{0, 0, 0, 0};
    const Bits free = free_pages(t.refs, t.pages, lds, part);
    const Sum s = block_sum(mine.count, part);
    if (b0 < t.B) {
        begin[b0] = s.before;
        first[b0] = mine.first;
        lacking[b0] = 0x7fffffff;
    }
    if (b0 == 0) { begin[t.B] = s.total; }
    __syncthreads();
    int handed = 0; // pages so far
    for (int i0 = 0; i0 < s.total; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        int b = 0, entry = 0, need = 0;
        if (i < s.total) {
            int lo = 0, hi = t.B; // the last sequence whose entries begin at or before i
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (begin[mid] <= i) {
                    lo = mid;
                } else {
                    hi = mid;
                }
            }
            b = lo;
            entry = first[b] + i - begin[b];
            // (starts that descend may promise more entries than whole numbers count)
            if (i >= begin[b] && i < begin[b + 1] && entry >= 0 && entry < t.max_pages) {
                const int32_t page = t.table[b * t.row + entry];
                need = page < 0 || page >= t.pages ? 1 : 0;
            }
        }
        const Sum n = block_sum(need, part);
        if (need) {
            const int page = nth_page<false>(free, handed + n.before);
            if (page >= 0) {
                t.table[b * t.row + entry] = page;
                t.refs[page] = 1;
            } else {
                atomicMin(&lacking[b], entry);
            }
        }
        handed += n.total;
    }
    __syncthreads();
    if (b0 < t.B) {
        // the tokens whose rows lie before the first page that is missing, or before the table's end
        const int64_t rows = static_cast<int64_t>(min(lacking[b0], t.max_pages)) << t.shift;
        granted[b0] = static_cast<int32_t>(max(int64_t{0}, min(static_cast<int64_t>(mine.tokens), rows - mine.history)));
    }
}

// ---- giving back ---------------------------------------------------------------------------------

__global__ __launch_bounds__(256) void pages_release_kernel(PageTable t, const int32_t* sequences, const int32_t* keep) {
    const int i = blockIdx.x;
    const int32_t b = sequences[i], rows = keep[i];
    if (b < 0 || b >= t.B || rows < 0) { return; }
    const int64_t from = (static_cast<int64_t>(rows) + (int64_t{1} << t.shift) - 1) >> t.shift;
    for (int64_t e = from + threadIdx.x; e < t.max_pages; e += 256) {
        // taken out by whoever comes first, where a sequence stands twice
        const int32_t page = atomicExch(&t.table[b * t.row + e], -1);
        if (page >= 0 && page < t.pages) { atomicSub(&t.refs[page], 1); }
    }
}

// ---- sharing -------------------------------------------------------------------------------------

__global__ __launch_bounds__(kThreads) void pages_fork_kernel(PageTable t, const int32_t* parents, const int32_t* children, int n, int32_t* history,
                                                              int32_t* src, int32_t* dst) {
    extern __shared__ uint64_t lds[];
    __shared__ int32_t part[kWaves];
    __shared__ int32_t of[kPagedMaxBatch], to[kPagedMaxBatch], rows[kPagedMaxBatch], fresh[kPagedMaxBatch];
    __shared__ int32_t claim[kPagedMaxBatch]; // of a sequence: the first pair whose child it is, -1 for a parent
    const int i = threadIdx.x;
    int32_t parent = -1, child = -1, length = 0;
    if (i < n) {
        parent = parents[i];
        child = children[i];
        if (parent >= 0 && parent < t.B) { length = max(0, history[parent]); }
        of[i] = parent;
        to[i] = child;
    }
    claim[i] = 0x7fffffff;
    __syncthreads();
    // (a pair that names no sequence as its parent claims its child all the same: it is left out for an earlier pair's sake)
    if (i < n && child >= 0 && child < t.B) { atomicMin(&claim[child], i); }
    if (i < n && parent >= 0 && parent < t.B) { atomicMin(&claim[parent], -1); }
    const Bits free = free_pages(t.refs, t.pages, lds, part); // before anything is given back
    const bool ok = i < n && parent >= 0 && parent < t.B && child >= 0 && child < t.B && claim[child] == i;
    const int whole = min(length >> t.shift, t.max_pages);
    // the last page's rows, where a page holds them
    int32_t last = -1;
    if (ok && whole < t.max_pages && (length & ((1 << t.shift) - 1)) != 0) {
        last = t.table[parent * t.row + whole];
        last = last >= 0 && last < t.pages ? last : -1;
    }
    const Sum s = block_sum(last >= 0 ? 1 : 0, part);
    const int page = last >= 0 ? nth_page<false>(free, s.before) : -1;
    if (i < n) {
        rows[i] = ok ? (page >= 0 ? length : whole << t.shift) : -1;
        fresh[i] = page;
        src[i] = page >= 0 ? last : -1;
        dst[i] = page;
    }
    __syncthreads();
    for (int64_t k = threadIdx.x; k < static_cast<int64_t>(n) * t.max_pages; k += kThreads) {
        const int j = static_cast<int>(k / t.max_pages), e = static_cast<int>(k - static_cast<int64_t>(j) * t.max_pages);
        if (rows[j] < 0) { continue; }
        const int full = rows[j] >> t.shift;
        int32_t* at = t.table + to[j] * t.row + e;
        const int32_t old = *at;
        int32_t now = -1;
        if (e < full) {
            now = t.table[of[j] * t.row + e];
        } else if (e == full) {
            now = fresh[j];
        }
        if (old >= 0 && old < t.pages) { atomicSub(&t.refs[old], 1); }
        if (now >= 0 && now < t.pages) { atomicAdd(&t.refs[now], 1); }
        *at = now;
    }
    if (ok) { history[child] = rows[i]; }
}

// ---- moving together -----------------------------------------------------------------------------

// The k-th highest page in use goes to the k-th lowest free one while that lies below it.
__global__ __launch_bounds__(kThreads) void pages_compact_kernel(PageTable t, int32_t* src, int32_t* dst, int n, int32_t* moved) {
    extern __shared__ uint64_t lds[];
    __shared__ int32_t part[kWaves];
    const Bits free = free_pages(t.refs, t.pages, lds, part);
    // as many moves as free pages lie below the number of those in use
    const int used = t.pages - free.total;
    int holes = 0;
    if (used < t.pages) { holes = free.sum[used / 64] + __popcll(free.word[used / 64] & ((uint64_t{1} << (used & 63)) - 1)); }
    const int count = min(holes, n);
    for (int k = threadIdx.x; k < n; k += kThreads) {
        int32_t from = -1, to = -1;
        if (k < count) {
            to = nth_page<false>(free, k);
            from = nth_page<true>(free, used - 1 - k);
            t.refs[to] = t.refs[from];
            t.refs[from] = 0;
        }
        src[k] = from;
        dst[k] = to;
    }
    if (threadIdx.x == 0) { *moved = count; }
}

// Entries of pages that moved; `src` descends.
__global__ __launch_bounds__(256) void pages_follow_kernel(PageTable t, const int32_t* src, const int32_t* dst, const int32_t* moved) {
    const int count = *moved;
    if (count == 0) { return; }
    const int32_t lowest = src[count - 1];
    const int64_t total = static_cast<int64_t>(t.B) * t.max_pages;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t b = i / t.max_pages;
        int32_t* at = t.table + b * t.row + (i - b * t.max_pages);
        const int32_t page = *at;
        if (page < lowest) { continue; }
        int lo = 0, hi = count; // the last source at or above the page
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (src[mid] >= page) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        if (src[lo] == page) { *at = dst[lo]; }
    }
}

} // namespace

void launch_copy_pages(const PagePlane* planes, int32_t count, const int32_t* src, const int32_t* dst, int32_t n, int32_t pages, hipStream_t stream) {
    CopyArgs a{};
    a.planes = count;
    a.pages = pages;
    a.src = src;
    a.dst = dst;
    int64_t pieces = 0;
    for (int32_t i = 0; i < count; ++i) {
        a.plane[i] = planes[i];
        a.first[i] = static_cast<int32_t>(pieces);
        pieces += (planes[i].bytes + kPiece - 1) / kPiece;
    }
    a.first[count] = static_cast<int32_t>(pieces);
    if (pieces * n > 0xFFFFFF) { throw Unsupported("paged page copies: more than 2^24 pieces of 16 KiB in one call are not built"); }
    hipLaunchKernelGGL(copy_pages_kernel, dim3(static_cast<uint32_t>(pieces * n)), dim3(256), 0, stream, a);
    check_launch("copy_pages_kernel");
}

void launch_pages_reserve(const PageTable& t, const int32_t* starts, const int32_t* history, int32_t* granted, hipStream_t stream) {
    hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(kThreads), bits_bytes(t.pages), stream, t, starts, history, granted);
    check_launch("pages_reserve_kernel");
}

void launch_pages_release(const PageTable& t, const int32_t* sequences, const int32_t* keep, int32_t n, hipStream_t stream) {
    hipLaunchKernelGGL(pages_release_kernel, dim3(n), dim3(256), 0, stream, t, sequences, keep);
    check_launch("pages_release_kernel");
}

void launch_pages_fork(const PageTable& t, const int32_t* parents, const int32_t* children, int32_t n, int32_t* history, int32_t* src, int32_t* dst,
                       hipStream_t stream) {
    hipLaunchKernelGGL(pages_fork_kernel, dim3(1), dim3(kThreads), bits_bytes(t.pages), stream, t, parents, children, n, history, src, dst);
    check_launch("pages_fork_kernel");
}

void launch_pages_compact(const PageTable& t, int32_t* src, int32_t* dst, int32_t n, int32_t* moved, hipStream_t stream) {
    hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(kThreads), bits_bytes(t.pages), stream, t, src, dst, n, moved);
    check_launch("pages_compact_kernel");
    const int64_t entries = static_cast<int64_t>(t.B) * t.max_pages;
    const uint32_t grid = static_cast<uint32_t>(std::min<int64_t>(1024, (entries + 255) / 256));
    hipLaunchKernelGGL(pages_follow_kernel, dim3(grid), dim3(256), 0, stream, t, src, dst, moved);
    check_launch("pages_follow_kernel");
}

} // namespace nmi
