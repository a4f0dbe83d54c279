// Attention of packed new tokens over selected blocks of a paged KV cache on gfx950.
//
// Mathematics: token n at position p has for every KV head a list of blocks; it sees the rows j <= p of those blocks whose page
// exists (one that stands twice counts once), out = sum_j softmax_j(scale * q . K_j) V_j in one pass with a running
// maximum and sum, zero where no row is seen. Numbers as in paged_attention.hip, whose walk over 32 keys at a time this
// is: the query heads of the token's KV head are the rows of a 16-row tile, K and V go straight from the cache to the matrix
// cores' operands.
//
// Few tokens: a token and KV head for a wave, or four, or several workgroups' waves, where the tokens alone do not fill the
// chip (sparse_attn_kernel). Prompts: tokens next to each other mostly select the same blocks, so a workgroup of eight waves
// merges the lists of up to 64 of them and walks the blocks that any of them takes, decoded once (sparse_many_kernel).
#include "common.h"
#include "paged_internal.h"
#include "paged_place.h"
#include "paged_tile.h"
#include "paged_walk.h"

#include <algorithm>
#include <cmath>

namespace nmi {
namespace {

struct SparseArgs {
    PagedAttnArgs x;
    const int32_t* selected; // [token][KV head][count]
    int32_t count;
    int32_t block_shift;
    int32_t row_tiles; // of 16 NT query heads
    int32_t parts;     // workgroups of an item
    int64_t items;     // tokens (or groups of tokens) x KV heads x row tiles, at most
    int32_t tokens;    // of a group
    int32_t per_tile;  // of a 16-row tile of a group
};

// A token, KV head and row tile.
struct Item {
    int32_t token;
    int32_t h;
    int32_t row0;
    int32_t b; // its sequence, -1: none
    int32_t pos;
};

// KV heads next to each other: workgroups go round the XCDs in turn, so with eight heads each L2 serves one.
__device__ __forceinline__ Item item_of(const SparseArgs& y, int64_t id, int rows) {
    Item it{0, static_cast<int32_t>(id % y.x.c.Hkv), 0, -1, 0};
    const int64_t rest = id / y.x.c.Hkv;
    it.row0 = static_cast<int32_t>(rest % y.row_tiles) * rows;
    it.token = static_cast<int32_t>(rest / y.row_tiles);
    return it;
}

// Lane l: sequence base + l, loaded and not looked at yet.
struct Loaded {
    int32_t start;
    int32_t end;
    int32_t history;
};

__device__ __forceinline__ Loaded load_sequences(const PagedAttnArgs& x, int base, int lane) {
    Loaded l{0x7fffffff, 0, 0};
    if (base + lane < x.c.B) { l = Loaded{x.a.starts[base + lane], x.a.starts[base + lane + 1], x.a.history[base + lane]}; }
    return l;
}

// The item's sequence, the last that starts at or before its token, and position; `l` holds the first 64 sequences. Every lane of
// the wave is there.
__device__ __forceinline__ void place(const PagedAttnArgs& x, Loaded l, Item& it, int lane) {
    for (int base = 0; base < x.c.B; base += 64) {
        if (base > 0) { l = load_sequences(x, base, lane); }
        const int before = __popcll(__ballot(base + lane < x.c.B && l.start <= it.token));
        if (before == 0) { continue; }
        const Seq s = lane_seq(checked(x, l.start, l.end, l.history), before - 1);
        const bool has = s.start <= it.token && it.token - s.start < s.tokens;
        it.b = has ? base + before - 1 : -1;
        it.pos = has ? s.history + it.token - s.start : 0;
    }
}

// An item's list: lane l of the wave that walks it holds entry l, and in bit i whether entry 64 i + l repeats an earlier one.
struct Listed {
    const int32_t* at;
    int32_t entry;
    uint32_t again;
};

__device__ __forceinline__ Listed list_of(const SparseArgs& y, const Item& it, int lane) {
    Listed l{y.selected + (static_cast<int64_t>(it.token) * y.x.c.Hkv + it.h) * y.count, -1, 0u};
    if (lane < y.count) { l.entry = l.at[lane]; }
    return l;
}

// Which entries repeat an earlier one. An ascending list has none; in any other every entry is compared with those before it, by every
// wave that walks the list: one token at 40/8/128 INT8 over 64, 256 and 1,024 blocks of 64 rows 15.5, 25.2 and 44.9 us with ascending
// lists, 19.4, 63.6 and 585 with shuffled ones.
static_assert(kPagedMaxSelected <= 64 * 32);
__device__ __forceinline__ void find_repeats(Listed& l, int count, int lane) {
    const int first = __shfl_up(l.entry, 1);
    bool ascends = lane == 0 || l.entry < 0 || (first >= 0 && first < l.entry); // no entry in the lane: -1
    for (int i = 64 + lane; i < count; i += 64) {
        const int e = l.at[i], before = l.at[i - 1];
        ascends &= e < 0 || (before >= 0 && before < e);
    }
    if (__builtin_expect(!__all(ascends), 0)) {
        for (int i = lane; i < count; i += 64) {
            const int e = l.at[i];
            bool again = false;
            for (int j = 0; j < i && !again; ++j) { again = l.at[j] == e; }
            l.again |= again ? 1u << (i >> 6) : 0u;
        }
    }
}

// A half tile of the walk: its first key's tile of 32, and its page.
struct Half {
    int32_t tile;
    int32_t page;
};

// Tiles [j0, j1) of the item's list, 32 keys each.
template <int D, bool BF, int NT, bool CARE>
__device__ __forceinline__ void sparse_walk(const SparseArgs& y, const Item& it, const Listed& l, int j0, int j1, int c, int g, Rows<D, BF, NT>& r, float down) {
    const PagedAttnArgs& x = y.x;
    const int lane = threadIdx.x & 63;
    const int lt = y.block_shift - 5; // log2(tiles of a block)
    const int32_t* table = x.c.table + it.b * x.c.table_row;
    // 64 halves (32 tiles) at a time, one per lane, the next 64 fetched ahead
    const auto fetch = [&](int j) {
        const int v = j + (lane >> 1);
        const int entry = v >> lt;
        const uint32_t twice = static_cast<uint32_t>(__shfl(static_cast<int>(l.again), entry & 63)) >> ((entry >> 6) & 31);
        const int early = __shfl(l.entry, entry & 63);
        Half f{0, -1};
        if (v < j1) {
            const int blk = entry < 64 ? early : l.at[entry];
            if (blk >= 0 && blk <= (it.pos >> y.block_shift) && (twice & 1u) == 0u) {
                f.tile = (blk << lt) + (v & ((1 << lt) - 1));
                const int key = 32 * f.tile + 16 * (lane & 1);
                if (key <= it.pos && (key >> x.c.page_shift) < x.c.max_pages) {
                    const int page = table[key >> x.c.page_shift];
                    f.page = page >= 0 && page < x.c.pages ? page : -1;
                }
            }
        }
        return f;
    };
    Half ids = fetch(j0), next_ids = fetch(j0 + 32);
    const auto refill = [&](int j) {
        if (((j - j0) & 63) == 30) { ids = fetch(j + 34); }
        if (((j - j0) & 63) == 62) { next_ids = fetch(j + 34); }
    };
    struct Tile {
        int tile;
        Halves hv;
    };
    const auto tile_at = [&](int j) { // past the end no page
        const int i = 2 * (j - j0);
        const Half& f = (i & 127) < 64 ? ids : next_ids;
        Tile t;
        t.tile = __builtin_amdgcn_readlane(f.tile, i & 63);
        t.hv.page[0] = __builtin_amdgcn_readlane(f.page, i & 63);
        t.hv.page[1] = __builtin_amdgcn_readlane(f.page, (i & 63) + 1);
        return t;
    };
    Probs<NT> pr;
    uint32_t large = 0u; // known already
    ChunkK<D, BF> ka;
    ChunkV<D, BF> va;
    Tile ta = tile_at(j0);
    load_keys<D, BF>(x, it.h, ta.tile, ta.hv, c, g, ka);
    load_values<D, BF>(x, it.h, ta.tile, ta.hv, c, g, va);
    init_rows<D, BF, NT>(x, Seq{it.token, 1, it.pos}, it.h, it.row0, c, g, r);
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
        const bool some = (ta.hv.page[0] & ta.hv.page[1]) >= 0; // a tile without a page adds nothing
        if (some) { chunk_probs<D, BF, NT>(x, ta.tile, ta.hv, g, ka, r, pr); }
        const Tile tb = tile_at(j + 1); // before the refill: tile 31 of a fetch is still in it
        if (((j - j0) & 1) == 0) { refill(j); }
        __builtin_amdgcn_sched_barrier(0);
        load_keys<D, BF>(x, it.h, tb.tile, tb.hv, c, g, ka);
        __builtin_amdgcn_sched_barrier(0);
        if (some) { chunk_values<D, BF, NT, CARE>(ta.tile, ta.hv, g, pr, va, r, down, large); }
        __builtin_amdgcn_sched_barrier(0);
        load_values<D, BF>(x, it.h, tb.tile, tb.hv, c, g, va);
        ta = tb;
    }
}

// The walk, and for BF16 caches the careful one after it where a sum passed 2^100 or is not finite. M, L: the rows' log2-domain
// maxima and sums.
template <int D, bool BF, int NT>
__device__ __forceinline__ void walk_rows(const SparseArgs& y, const Item& it, const Listed& l, int j0, int j1, int c, int g, Rows<D, BF, NT>& r, float (&M)[NT],
                                          float (&L)[NT]) {
    const PagedAttnArgs& x = y.x;
    sparse_walk<D, BF, NT, false>(y, it, l, j0, j1, c, g, r, 1.0f);
    bool lower = false;
    if constexpr (BF) {
        uint32_t top = 0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) { top = max(top, __float_as_uint(r.O[nt][t][e]) << 1); }
            }
        }
        if (__builtin_expect(__any(top >= static_cast<uint32_t>(127 + 100) << 24), 0)) {
            uint32_t large = 0u;
            const int lt = y.block_shift - 5;
            const int32_t* table = x.c.table + it.b * x.c.table_row;
#pragma unroll 1
            for (int j = j0; j < j1; ++j) {
                const int blk = __builtin_amdgcn_readfirstlane(l.at[j >> lt]);
                if (blk < 0 || blk > (it.pos >> y.block_shift)) { continue; }
                const int tile = (blk << lt) + (j & ((1 << lt) - 1));
                ChunkV<D, BF> cv;
                load_values<D, BF>(x, it.h, tile, halves_of(x, table, tile, it.pos), c, g, cv);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
#pragma unroll
                    for (int i = 0; i < Chunk<D, BF>::VP; ++i) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) { large = max(large, larger_bits(finite_word(cv.v[k][i][e]))); }
                    }
                }
            }
            lower = __any(large >= kCareTop);
            sparse_walk<D, BF, NT, true>(y, it, l, j0, j1, c, g, r, lower ? kCareDown : 1.0f);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        M[nt] = r.m[nt] == -INFINITY ? -INFINITY : r.m[nt] * r.rowmul[nt];
        L[nt] = group4_sum(r.l[nt]);
        if (lower) { care_units(M[nt], L[nt]); }
    }
}

// WAVES: four waves, a token and KV head each; otherwise four waves share one, and `parts` workgroups may.
// What bounds it: HBM for many rows (32 tokens over 64 blocks of 64 rows at 40/8/128 INT8, 277 MB, 59 us with the merge, 4.7 TB/s);
// for one token the chain list -> page -> rows, a tile's products in one wave (1.1 us, at head_dim 256 up to 3) and the merge's launch: over
// 32 blocks 13.1 us, with two tiles a wave 13.4, with four 15.5; at 24/4/256 17.0, 18.4 and 24.6. Tiles two ahead instead of one: 1 to 8%
// more.
template <int D, bool BF, int NT, bool WAVES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 128 ? 2 : 1, D == 128 ? 2 : 1))) void sparse_attn_kernel(SparseArgs y) {
    const PagedAttnArgs& x = y.x;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int tiles = y.count << (y.block_shift - 5);
    Rows<D, BF, NT> r;
    float M[NT], L[NT];
    if constexpr (WAVES) {
        // neighbouring waves: neighbouring tokens of one head, whose lists are much alike
        const int64_t group = blockIdx.x / x.c.Hkv, per = x.c.Hkv;
        const int64_t id = (group * 4 + wave) * per + blockIdx.x % x.c.Hkv;
        if (id >= y.items) { return; }
        Item it = item_of(y, id, 16 * NT);
        const Loaded first = load_sequences(x, 0, lane);
        Listed l = list_of(y, it, lane);
        place(x, first, it, lane);
        if (it.b < 0) { return; }
        find_repeats(l, y.count, lane);
        walk_rows<D, BF, NT>(y, it, l, 0, tiles, c, g, r, M, L);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = it.row0 + 16 * nt + c;
            if (row < x.G) { store_out<D, BF, NT>(x, it.token, it.h, row, r, nt, L[nt], g); }
        }
    } else {
        __shared__ f4 xo[2][NT * (D / 16) * 64];
        __shared__ float2 xm[2][NT * 64];
        const int64_t id = blockIdx.x % y.items;
        const int part = static_cast<int>(blockIdx.x / y.items);
        Item it = item_of(y, id, 16 * NT);
        const Loaded first = load_sequences(x, 0, lane);
        Listed l = list_of(y, it, lane);
        place(x, first, it, lane);
        if (it.b < 0) { return; }
        find_repeats(l, y.count, lane);
        const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * part / y.parts), t1 = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / y.parts);
        const int j0 = t0 + (t1 - t0) * wave / 4, j1 = t0 + (t1 - t0) * (wave + 1) / 4;
        walk_rows<D, BF, NT>(y, it, l, j0, j1, c, g, r, M, L);
        join_waves<D, BF, NT, 4>(r, M, L, wave, lane, xo, xm);
        if (wave != 0) { return; }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = it.row0 + 16 * nt + c;
            if (row >= x.G) { continue; }
            if (y.parts > 1) {
                store_part<D, BF, NT>(x, r, nt, M[nt], L[nt], (id * (16 * NT) + 16 * nt + c) * y.parts + part, g);
            } else {
                store_out<D, BF, NT>(x, it.token, it.h, row, r, nt, L[nt], g);
            }
        }
    }
}

// The parts of an item's rows, one after another: D / 4 threads a row, `rows` rows an item.
template <int D>
__global__ __launch_bounds__(256) void sparse_merge_kernel(SparseArgs y, int rows) {
    const PagedAttnArgs& x = y.x;
    constexpr int TPR = D / 4, RPB = 256 / TPR;
    const int64_t id = blockIdx.x / (rows / RPB);
    const int row = static_cast<int>(blockIdx.x % (rows / RPB)) * RPB + threadIdx.x / TPR;
    Item it = item_of(y, id, rows);
    const Loaded first = load_sequences(x, 0, threadIdx.x & 63); // looked at behind the parts' loads
    const bool there = it.row0 + row < x.G;
    const int d = 4 * (threadIdx.x % TPR);
    Merge m;
#pragma unroll 4
    for (int k = 0; k < (there ? y.parts : 0); ++k) {
        const int64_t at = (id * rows + row) * y.parts + k;
        const float2 ml = *reinterpret_cast<const float2*>(x.part_ml + 2 * at);
        m.add(ml.x, ml.y, *reinterpret_cast<const f4*>(x.part_o + at * D + d));
    }
    place(x, first, it, threadIdx.x & 63);
    if (it.b < 0 || !there) { return; }
    uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + it.token * x.a.out.token_stride) + (it.h * x.G + it.row0 + row) * D + d;
    *reinterpret_cast<u2*>(out) = out_pair(m.O, m.L);
}

// ---- prompts: groups of tokens over blocks that a workgroup decodes once ----------------------------
//
// A workgroup of eight waves: 8 / WK of them have NT row tiles of per_tile whole tokens each, times WK waves that take
// different chunks of 32 keys. The lists of its tokens become one, ascending, of (block, tokens that take it) in LDS, through a bit
// field per block; its chunks are walked in tiles as the many-row kernel of paged_attention.hip does it (decoding, ranges of the
// FP16 operands and the apart walk of tiles beyond them stand there). A wave skips the chunks that none of its tokens takes,
// and a row whose token does not take a chunk sees none of it.
// What bounds it: the waves of a workgroup wait for each other at every tile, whichever of them have work there (the matrix cores are
// busy 14% of the time, the VALU 36%, LDS 23%). 2,048 tokens over 16 blocks of 64 rows each at 24/4/256 BF16: 310 to 334 us; every token by
// itself 816.

constexpr int kListMost = 2048;               // blocks of a workgroup's list
constexpr int kGroupMost = 64;                // tokens of a workgroup: bits
constexpr int kManyBlock = 256;               // rows of a block, at most: bounds the tiles of a list
constexpr int kManyTiles = kListMost * (kManyBlock / 32) / 2;
constexpr int kTableBlocks = 16384;           // blocks of a pass over the lists

// Tokens token .. token + count - 1 of sequence b, the first at position pos, and a KV head.
struct Group {
    int32_t token;
    int32_t count;
    int32_t h;
    int32_t b; // -1: none
    int32_t pos;
};

__device__ __forceinline__ Group group_of(const SparseArgs& y, int64_t id, int lane) {
    const PagedAttnArgs& x = y.x;
    Group q{0, 0, static_cast<int32_t>(id % x.c.Hkv), -1, 0};
    const Found f = find_unit(
        x.c.B, static_cast<int>(id / x.c.Hkv), lane,
        [&](int b) {
            const Seq s = sequence(x, b);
            return Span{s.start, s.tokens, s.history};
        },
        [&](const Span& s) { return (s.tokens + y.tokens - 1) / y.tokens; });
    if (f.b < 0) { return q; }
    const int t0 = f.at * y.tokens;
    q.token = f.s.start + t0;
    q.count = min(y.tokens, f.s.tokens - t0);
    q.b = f.b;
    q.pos = f.s.history + t0;
    return q;
}

// The merged list in LDS.
struct List {
    uint64_t tokens[kListMost];
    int32_t block[kListMost];
    int count;
};

// For the whole workgroup; `table`: scratch of kTableBlocks words.
__device__ __forceinline__ void merge_lists(const SparseArgs& y, const Group& q, List& list, uint64_t* table) {
    const int32_t* from = y.selected + (static_cast<int64_t>(q.token) * y.x.c.Hkv + q.h) * y.count;
    const int64_t next = static_cast<int64_t>(y.x.c.Hkv) * y.count;
    const int entries = q.count * y.count;
    const int blocks = ((q.pos + q.count - 1) >> y.block_shift) + 1;
    const int lane = threadIdx.x & 63;
    int n = 0; // of the first wave
    for (int b0 = 0; b0 < blocks; b0 += kTableBlocks) {
        const int some = min(kTableBlocks, blocks - b0);
        for (int i = threadIdx.x; i < some; i += kManyThreads) { table[i] = 0u; }
        __syncthreads();
        for (int e = threadIdx.x; e < entries; e += kManyThreads) {
            const int t = e / y.count;
            const int blk = from[t * next + (e - t * y.count)];
            if (blk >= b0 && blk < b0 + some && blk <= ((q.pos + t) >> y.block_shift)) {
                atomicOr(reinterpret_cast<unsigned long long*>(&table[blk - b0]), 1ull << t);
            }
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            for (int i0 = 0; i0 < some; i0 += 64) {
                const uint64_t m = i0 + lane < some ? table[i0 + lane] : 0u;
                const uint64_t all = __ballot(m != 0u);
                const int at = n + __popcll(all & ((uint64_t{1} << lane) - 1));
                if (m != 0u && at < kListMost) { // (as many blocks or entries as the host allows fit)
                    list.block[at] = b0 + i0 + lane;
                    list.tokens[at] = m;
                }
                n += __popcll(all);
            }
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) { list.count = min(n, kListMost); }
    __syncthreads();
}

template <int D, bool BF, int WK>
__global__ __launch_bounds__(kManyThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void sparse_many_kernel(SparseArgs y) {
    using MG = ManyGeo<D, WK>;
    constexpr int NT = MG::NT, NCH = MG::NCH;
    constexpr int WPC = 32 / MG::RW; // waves that stage a chunk's rows
    __shared__ __attribute__((aligned(256))) char smem[2 * MG::kBuf];
    __shared__ List list;
    __shared__ uint32_t marks[kManyTiles / 32]; // tiles that need care
    __shared__ uint32_t state[2][8];            // per buffer and wave: bit 0 its page exists, bit 1 care
    __shared__ float tops[2][8];
    static_assert(kTableBlocks * 8 <= 2 * MG::kBuf);
    const PagedAttnArgs& x = y.x;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int wr = wave / WK, wk = wave % WK;
    const Group q = group_of(y, blockIdx.x, lane);
    if (q.b < 0) { return; }
    merge_lists(y, q, list, reinterpret_cast<uint64_t*>(smem));
    const int lt = y.block_shift - 5; // log2(chunks of a block)
    const int chunks = list.count << lt;
    const int tiles = (chunks + NCH - 1) / NCH;
    const int p1 = q.pos + q.count - 1;

    // the first key and the page of the wave's rows, 64 tiles at a time
    const int32_t* table = x.c.table + q.b * x.c.table_row;
    struct Place {
        int key, page;
    };
    const auto chunk_key = [&](int v) { return ((list.block[v >> lt] << lt) + (v & ((1 << lt) - 1))) * 32; };
    const auto places_from = [&](int j) {
        const int v = (j + lane) * NCH + wave / WPC;
        Place p{0, -1};
        if (v < chunks) {
            p.key = chunk_key(v) + wave % WPC * MG::RW;
            if (p.key <= p1 && (p.key >> x.c.page_shift) < x.c.max_pages) {
                const int page = table[p.key >> x.c.page_shift];
                p.page = page >= 0 && page < x.c.pages ? page : -1;
            }
        }
        return p;
    };
    Place ids = places_from(0), next_ids = places_from(64);
    StageRegs<D, BF> sr;
    int key = 0, page = -1; // of the rows in `sr`
    const auto fetch = [&](int j) {
        if ((j & 63) == 0 && j > 0) { // a new 64: they were fetched 64 tiles ago
            ids = next_ids;
            next_ids = places_from(j + 64);
        }
        key = __builtin_amdgcn_readlane(ids.key, j & 63);
        page = __builtin_amdgcn_readlane(ids.page, j & 63);
        stage_load<D, BF>(x, q.h, key, page, lane, sr);
    };
    ManyScale sc{1.0f, 1.0f, INFINITY, INFINITY, 0u};
    const auto trim = [&] {
        const int live = p1 + 1 - key;
        if (live < MG::RW) { stage_trim<D, BF>(sr, live, lane); }
    };
    const auto put = [&](int j) {
        trim();
        const bool care = stage_store<D, BF>(sr, sc, smem + (j & 1) * MG::kBuf, wave * MG::RW, lane);
        const uint32_t st = (page >= 0 ? 1u : 0u) | (__any(care) ? 2u : 0u);
        if (lane == 0) { state[j & 1][wave] = st; }
    };

    if (tiles > 0) { fetch(0); }
    Rows<D, BF, NT> r;
    int pos[NT];       // the row's position, -1: no row
    uint32_t bit[NT];  // its token's bit among the wave's
    const int first = wr * NT * y.per_tile; // the wave's first token
    const int mine = max(0, min(NT * y.per_tile, q.count - first));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int in = c / x.G, t = nt * y.per_tile + in;
        const bool valid = in < y.per_tile && t < mine;
        pos[nt] = valid ? q.pos + first + t : -1;
        bit[nt] = valid ? 1u << t : 0u;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(x.a.q.data + static_cast<int64_t>(q.token + (valid ? first + t : 0)) * x.a.q.token_stride) +
                              (q.h * x.G + (valid ? c - in * x.G : 0)) * D;
        init_row<D, BF, NT>(x, src, valid, nt, g, r);
    }
    const uint32_t every = (1u << mine) - 1u;
    r.hi = q.pos + first + mine - 1;
    // the wave's tokens that take chunk v; sets what its rows see of it
    const auto takes = [&](int v) {
        const uint64_t all = list.tokens[v >> lt];
        const uint32_t m = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(all >> first)) & every;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) { r.pos[nt] = (m & bit[nt]) != 0u ? pos[nt] : -1; }
        r.lo = m == every ? q.pos + first : -1;
        return m != 0u;
    };
    bool cared = false;
    if (tiles > 0) {
        for (int i = threadIdx.x; 32 * i < tiles; i += kManyThreads) { marks[i] = 0u; }
        // the first tile that holds a value tells how large they are: absent pages and zero rows say nothing
        float kt = 0.0f, vt = 0.0f;
        int js = 0;
        for (;; ++js) {
            if (js > 0) {
                const Place p = places_from(js);
                key = __builtin_amdgcn_readfirstlane(p.key);
                stage_load<D, BF>(x, q.h, key, __builtin_amdgcn_readfirstlane(p.page), lane, sr);
            }
            trim();
            const StageSize z = stage_size<D, BF>(sr);
            const float kw = wave_max(z.k < INFINITY ? z.k : 0.0f), vw = wave_max(z.v < INFINITY ? z.v : 0.0f);
            if (lane == 0) {
                tops[0][wave] = kw;
                tops[1][wave] = vw;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                kt = fmaxf(kt, tops[0][i]);
                vt = fmaxf(vt, tops[1][i]);
            }
            if (__any(vt > 0.0f) || js + 1 == tiles) { break; }
            __syncthreads(); // the tops are read
        }
        if (js > 0) { fetch(0); }
        pick(kt, 8, sc.k, sc.klim);
        pick(vt, BF ? 15 : 8, sc.v, sc.vlim);
        sc.vleast = __float_as_uint(0x1p-6f / sc.v) - 1u;
        put(0);
        if (tiles > 1) { fetch(1); }
        __syncthreads();
    }
    ManyState<D, BF, NT> ms;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        ms.mul[nt] = BF ? r.rowmul[nt] : fminf(r.rowmul[nt] / sc.k, kLargest);
        ms.ref[nt] = {};
        ms.lim[nt] = -INFINITY;
        ms.l[nt] = f4{0.f, 0.f, 0.f, 0.f};
    }
    // the wave's V^T reads: lane (c, g) addresses key 4 g + (c >> 2), dims 4 (c & 3) .. of a 16-dim segment
    const int vkey = 4 * g + (c >> 2);
    const int voff = vkey * 2 * D + 32 * (vkey & 7) + 8 * (c & 3);
    // waves w and w + 4 share a SIMD: one decodes the next tile before its products, one after them
    const bool early = wave < 4;
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
        const char* buf = smem + (j & 1) * MG::kBuf;
        const uint32_t st = lane < 8 ? state[j & 1][lane] : 0u;
        const uint32_t here = static_cast<uint32_t>(__ballot((st & 1u) != 0u));
        const bool care = __any((st & 2u) != 0u);
        const auto stage = [&] {
            if (j + 1 < tiles) {
                put(j + 1);
                if (j + 2 < tiles) { fetch(j + 2); }
            }
        };
        if (early) { stage(); }
        if (care) {
            cared = true;
            if (threadIdx.x == 0) { marks[j >> 5] |= 1u << (j & 31); }
        } else {
#pragma unroll 1
            for (int cw = 0; cw < NCH / WK; ++cw) {
                const int ci = cw * WK + wk;
                const int v = j * NCH + ci;
                // the halves' pages: two waves' rows each at head_dim 256
                const uint32_t bits = D == 128 ? here >> (2 * ci) : (here >> (4 * ci) & 1u) | (here >> (4 * ci + 1) & 2u);
                // by arithmetic: hipcc 7.2 inverted a select on a bit of a scalar here (s_bitcmp0 for s_bitcmp1)
                const Halves hv{{static_cast<int>(bits & 1u) - 1, static_cast<int>((bits >> 1) & 1u) - 1}};
                if (v >= chunks || (hv.page[0] & hv.page[1]) < 0 || !takes(v)) { continue; }
                const int c0 = __builtin_amdgcn_readfirstlane(chunk_key(v));
                if (c0 > r.hi) { continue; }
                many_chunk<D, BF, NT>(x, buf, ci, c0, hv, c, g, voff, r, ms);
            }
        }
        if (!early) { stage(); }
        __syncthreads(); // this buffer is free, the next tile is in place
    }
    const float unit_v = 1.0f / sc.v; // an exact power of two
    float M[NT], L[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float neg;
        if constexpr (kFromRef<D, BF>) { neg = ms.ref[nt][0]; } else { neg = ms.ref[nt]; }
        M[nt] = ms.lim[nt] == -INFINITY ? -INFINITY : -neg * ms.mul[nt];
        L[nt] = ms.l[nt][0];
#pragma unroll
        for (int t = 0; t < D / 16; ++t) { r.O[nt][t] *= unit_v; }
    }
    if (__builtin_expect(cared, 0)) {
        // the state so far to LDS (each wave its own part), then the marked tiles with a new one
        float* keep = reinterpret_cast<float*>(smem) + wave * (16 * NT * D);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) { *reinterpret_cast<f4*>(keep + (16 * nt + c) * D + 16 * t + 4 * g) = r.O[nt][t]; }
        }
        __syncthreads();
        uint32_t large = 0u;
        bool lower = false;
#pragma unroll 1
        for (;;) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) { r.O[nt][t] = f4{0.f, 0.f, 0.f, 0.f}; }
                r.m[nt] = -INFINITY;
                r.l[nt] = 0.0f;
            }
#pragma unroll 1
            for (int base = 0; base < tiles; base += 32) {
                uint32_t bits = __builtin_amdgcn_readfirstlane(marks[base >> 5]);
#pragma unroll 1
                for (; bits != 0u; bits &= bits - 1u) {
                    const int v0 = (base + __builtin_ctz(bits)) * NCH;
#pragma unroll 1
                    for (int cw = 0; cw < NCH / WK; ++cw) {
                        const int v = v0 + cw * WK + wk;
                        if (v >= chunks || !takes(v)) { continue; }
                        const int tile = __builtin_amdgcn_readfirstlane(chunk_key(v)) >> 5;
                        if (32 * tile > r.hi) { continue; }
                        const Halves hv = halves_of(x, table, tile, p1);
                        Probs<NT> pr;
                        {
                            ChunkK<D, BF> ck;
                            load_keys<D, BF>(x, q.h, tile, hv, c, g, ck);
                            chunk_probs<D, BF, NT>(x, tile, hv, g, ck, r, pr);
                        }
                        __builtin_amdgcn_sched_barrier(0); // the registers hold one plane's rows at a time
                        ChunkV<D, BF> cv;
                        load_values<D, BF>(x, q.h, tile, hv, c, g, cv);
                        chunk_values<D, BF, NT, BF>(tile, hv, g, pr, cv, r, lower ? kCareDown : 1.0f, large);
                    }
                }
            }
            if (!BF || lower || !__any(large >= kCareTop)) { break; }
            lower = true; // again, by the lower weights
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float m2 = r.m[nt] == -INFINITY ? -INFINITY : r.m[nt] * r.rowmul[nt], l2 = group4_sum(r.l[nt]);
            if (lower) { care_units(m2, l2); }
            const Weights w = weights(M[nt], L[nt], m2, l2);
            L[nt] = L[nt] * w.a + l2 * w.b;
            M[nt] = w.M;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) { // back in the first walk's order of dims, so that what follows is the same
                    float* o = keep + (16 * nt + c) * D + out_dim<BF>(t, 4 * g + e);
                    *o = (w.a == 0.0f ? 0.0f : *o * w.a) + (w.b == 0.0f ? 0.0f : r.O[nt][t][e] * w.b);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) { r.O[nt][t] = *reinterpret_cast<const f4*>(keep + (16 * nt + c) * D + 16 * t + 4 * g); }
        }
        __syncthreads();
    }
    // ---- the WK key waves of a row tile through LDS
    if constexpr (WK > 1) {
        f4* xo = reinterpret_cast<f4*>(smem);
        constexpr int kPer = NT * (D / 16) * 64;
        static_assert((WK - 1) * MG::WR * kPer * 16 + (WK - 1) * MG::WR * NT * 64 * 8 <= 2 * MG::kBuf, "merge exceeds the buffers");
        float2* xm = reinterpret_cast<float2*>(smem + (WK - 1) * MG::WR * kPer * 16);
        if (wk > 0) {
            const int at = (wk - 1) * MG::WR + wr;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) { xo[at * kPer + (nt * (D / 16) + t) * 64 + lane] = r.O[nt][t]; }
                xm[(at * NT + nt) * 64 + lane] = float2{M[nt], L[nt]};
            }
        }
        __syncthreads();
        if (wk > 0) { return; }
#pragma unroll
        for (int i = 0; i < WK - 1; ++i) {
            const int at = i * MG::WR + wr;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float2 o = xm[(at * NT + nt) * 64 + lane];
                const Weights w = weights(M[nt], L[nt], o.x, o.y);
                L[nt] = L[nt] * w.a + o.y * w.b;
                M[nt] = w.M;
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    const f4 z = xo[at * kPer + (nt * (D / 16) + t) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) { r.O[nt][t][e] = (w.a == 0.0f ? 0.0f : r.O[nt][t][e] * w.a) + (w.b == 0.0f ? 0.0f : z[e] * w.b); }
                }
            }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (pos[nt] < 0) { continue; }
        uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + static_cast<int64_t>(q.token + pos[nt] - q.pos) * x.a.out.token_stride) +
                        (q.h * x.G + c % x.G) * D + 4 * g;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) { *reinterpret_cast<u2*>(out + 16 * t) = out_pair(r.O[nt][t], L[nt]); }
    }
}

// How a call is cut.
struct SparsePlan {
    int32_t nt = 1;
    int32_t row_tiles = 1;
    int64_t items = 0;
    bool waves = false; // a wave per item
    int32_t parts = 1;  // workgroups per item
    int32_t wk = 0;     // groups of tokens, waves of a row tile over the keys (0: none are formed)
    int32_t tokens = 1; // of a group
    int32_t per_tile = 1;
    size_t ml_offset = 0;
    size_t bytes = 0;
};

constexpr int kCus = 256;

SparsePlan plan_sparse(int32_t Hq, int32_t Hkv, int32_t D, bool bf16, int64_t tokens, int32_t B, int32_t max_new, int32_t max_keys, int32_t selected,
                       int32_t block_shift) {
    SparsePlan p;
    const int32_t G = Hq / Hkv;
    // More than 16 query heads: two row tiles at once. One after the other reads a list's rows twice (from L2 the second time) and takes,
    // for 32 tokens over 64 blocks, INT8 and BF16, 25.1 and 31.8 us instead of 28.4 and 34.0 at 32/1/128, 39.1 and 53.4 instead of 39.9
    // and 76.5 at 32/1/256, 59.4 and 81.9 instead of 53.9 and 116.3 at 40/1/256: the registers of two tiles do not hold at head_dim 256.
    p.nt = G <= 16 ? 1 : 2;
    p.row_tiles = (G + 16 * p.nt - 1) / (16 * p.nt);
    p.items = tokens * Hkv * p.row_tiles;
    const int64_t tiles = static_cast<int64_t>(selected) << (block_shift - 5);
    const int64_t slots = kCus * (D == 128 ? 2 : 1); // workgroups of four waves at a time
    p.waves = p.items >= 4 * slots || tiles < 4;
    if (!p.waves) {
        // a tile for a wave, if that takes no more workgroups than run at a time
        p.parts = static_cast<int32_t>(std::max<int64_t>(1, std::min(slots / p.items, tiles / 4)));
    }
    if (p.parts > 1) {
        const size_t rows = static_cast<size_t>(p.items) * 16 * p.nt * p.parts;
        p.ml_offset = (rows * D * sizeof(float) + 255) & ~size_t{255};
        p.bytes = p.ml_offset + rows * 2 * sizeof(float);
    }
    // Groups, where they are estimated to be faster.
    const int64_t blocks = ((static_cast<int64_t>(max_keys) - 1) >> block_shift) + 1;
    if (G > 16 || max_new < 2 || (1 << block_shift) > kManyBlock) { return p; }
    const int32_t nt = D == 128 ? 2 : 1;
    const int32_t per_tile = std::min(16 / G, 8 / nt);
    // In us on MI355X. A chunk of 32 keys for one token and KV head (2,048 tokens over 16 blocks of 64), a third more where the tokens
    // do not fill the chip: 100 and 300 tokens at 40/8/128 INT8 reckoned 48 and 120, took 51 and 114; at 24/4/256 BF16 66 and 172, 65 and
    // 176; 24 verify rounds of 4 tokens over 43 blocks 105, 101.
    const double chunk_us = (D == 128 ? (bf16 ? 1.4e-3 : 1.04e-3) : (bf16 ? 3.1e-3 : 2.55e-3)) * (p.waves ? 1.0 : 1.35);
    double best = 12.0 + static_cast<double>(p.items * tiles) * chunk_us;
    for (int32_t wk = 1; wk <= (D == 128 ? 4 : 2); wk *= 2) {
        const int32_t most = std::min(8 / wk * nt * per_tile, kGroupMost);
        const int32_t t = std::min(most, max_new);
        if (std::min<int64_t>(blocks, static_cast<int64_t>(t) * selected) > kListMost) { continue; }
        const int64_t groups = (tokens + static_cast<int64_t>(B) * (most - 1)) / most * Hkv;
        // Tokens next to each other mostly take the same blocks: reckoned as if 2 of them took 1.34 times as many as one, 16 3.2 times (where
        // they agree less the tiles are more, up to as many as there are blocks). The host does not see the lists: 1,024 tokens at 40/8/128
        // INT8 over 60,000 rows with lists that agree, agree in part (16 tokens 60 blocks) and do not (190) take 58, 271 and 899 us so,
        // every token by itself 292, 302 and 396. A round of workgroups with WK = 1, 2, 4 at 40/8/128 INT8 over 16 blocks each: 190, 111
        // and 76 us; at 24/4/256 BF16 165 and 98.
        const double merged = std::min<double>(static_cast<double>(blocks), selected * std::pow(static_cast<double>(t), 0.42));
        const double us_tile = D == 128 ? (wk == 1 ? 4.4 : wk == 2 ? 3.35 : 2.95) : (wk == 1 ? 3.05 : 2.35);
        const double us = static_cast<double>((groups + kCus - 1) / kCus) * (10.0 + merged * (1 << block_shift) / (16384 / D) * us_tile);
        if (us < best) {
            best = us;
            p.wk = wk;
            p.tokens = most;
            p.per_tile = per_tile;
        }
    }
    if (p.wk > 0) {
        p.items = (tokens + static_cast<int64_t>(B) * (p.tokens - 1)) / p.tokens * Hkv;
        p.parts = 1;
    }
    return p;
}

template <int D, bool BF, int NT>
void launch(const SparseArgs& y, const SparsePlan& p, hipStream_t stream) {
    const int64_t per = y.x.c.Hkv;
    const int64_t grid = p.waves ? (p.items / per + 3) / 4 * per : p.items * p.parts;
    if (grid > 0x7FFFFF) { throw Unsupported("paged sparse attention: more than 2^23 workgroups are not built"); }
    const dim3 blocks(static_cast<uint32_t>(grid));
    if (p.waves) {
        hipLaunchKernelGGL((sparse_attn_kernel<D, BF, NT, true>), blocks, dim3(256), 0, stream, y);
    } else {
        hipLaunchKernelGGL((sparse_attn_kernel<D, BF, NT, false>), blocks, dim3(256), 0, stream, y);
    }
    check_launch("sparse_attn_kernel");
    if (p.parts > 1) {
        const uint32_t groups = static_cast<uint32_t>(p.items * (16 * NT / (1024 / D)));
        hipLaunchKernelGGL((sparse_merge_kernel<D>), dim3(groups), dim3(256), 0, stream, y, 16 * NT);
        check_launch("sparse_merge_kernel");
    }
}

template <int D, bool BF>
void launch_groups(const SparseArgs& y, const SparsePlan& p, hipStream_t stream) {
    if (p.items > 0x3FFFFF) { throw Unsupported("paged sparse attention: more than 2^22 workgroups are not built"); }
    const dim3 blocks(static_cast<uint32_t>(p.items));
    if (p.wk == 1) {
        hipLaunchKernelGGL((sparse_many_kernel<D, BF, 1>), blocks, dim3(kManyThreads), 0, stream, y);
    } else if (p.wk == 2) {
        hipLaunchKernelGGL((sparse_many_kernel<D, BF, 2>), blocks, dim3(kManyThreads), 0, stream, y);
    } else if constexpr (D == 128) {
        hipLaunchKernelGGL((sparse_many_kernel<D, BF, 4>), blocks, dim3(kManyThreads), 0, stream, y);
    }
    check_launch("sparse_many_kernel");
}

} // namespace

size_t sparse_attention_bytes(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t selected, int32_t block_shift) {
    return plan_sparse(Hq, Hkv, D, false, tokens, B, 1, 1, selected, block_shift).bytes; // groups take none
}

void launch_sparse_attention(const PagedAttention& a, const int32_t* selected, int32_t count, int32_t block_shift, const PagedRef& c,
                             void* workspace, hipStream_t stream) {
    const SparsePlan p = plan_sparse(a.Hq, c.Hkv, c.D, c.bf16, a.tokens, c.B, a.max_new, a.max_keys, count, block_shift);
    SparseArgs y{};
    y.x.a = a;
    y.x.a.window = 0x7FFFFFFF; // every row of a listed block up to the token's own
    y.x.c = c;
    y.x.G = a.Hq / c.Hkv;
    y.x.scale_log2 = a.scale * 1.4426950408889634f;
    y.x.part_o = static_cast<float*>(workspace);
    y.x.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.ml_offset);
    y.selected = selected;
    y.count = count;
    y.block_shift = block_shift;
    y.row_tiles = p.row_tiles;
    y.parts = p.parts;
    y.items = p.items;
    y.tokens = p.tokens;
    y.per_tile = p.per_tile;
    const auto pick = [&](auto d, auto bf) {
        constexpr int D = decltype(d)::value;
        constexpr bool BF = decltype(bf)::value;
        if (p.wk > 0) {
            launch_groups<D, BF>(y, p, stream);
        } else {
            p.nt == 1 ? launch<D, BF, 1>(y, p, stream) : launch<D, BF, 2>(y, p, stream);
        }
    };
    const auto cache = [&](auto d) { c.bf16 ? pick(d, std::true_type{}) : pick(d, std::false_type{}); };
    c.D == 128 ? cache(std::integral_constant<int, 128>{}) : cache(std::integral_constant<int, 256>{});
}

} // namespace nmi
