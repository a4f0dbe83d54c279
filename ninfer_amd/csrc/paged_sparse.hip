// Attention of packed new tokens over selected blocks of a paged KV cache on gfx950.
//
// Mathematics: token n at position p has for every KV head a list of blocks; it sees the rows j <= p of those blocks whose page
// exists (an entry that stands twice counts twice), out = sum_j softmax_j(scale * q . K_j) V_j in one pass with a running
// maximum and sum, zero where no row is seen. Numbers as in paged_attention.hip, whose walk over 32 keys at a time this
// is: the query heads of the token's KV head are the rows of a 16-row tile, K and V go straight from the cache to the matrix
// cores' operands.
//
// Single tokens: a token and KV head for a wave, or four, or several workgroups' waves, where the tokens alone do not fill the
// chip. Tokens of one sequence next to each other, up to eight: their lists are merged, since neighbours mostly select the same
// blocks, and a tile of 32 keys is fetched once for all the tokens that take it.
#include "common.h"
#include "paged_internal.h"
#include "paged_place.h"
#include "paged_walk.h"

#include <algorithm>

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
    int32_t tokens;    // of a group (1: none are formed)
    int32_t per_tile;  // tokens of a 16-row tile of a group
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
__device__ __forceinline__ Item item_of(const SparseArgs& y, int64_t id, int rows, int lane) {
    const PagedAttnArgs& x = y.x;
    Item it{0, static_cast<int32_t>(id % x.c.Hkv), 0, -1, 0};
    const int64_t rest = id / x.c.Hkv;
    it.row0 = static_cast<int32_t>(rest % y.row_tiles) * rows;
    it.token = static_cast<int32_t>(rest / y.row_tiles);
    int before = 0; // sequences that start at or before the token
    for (int base = 0; base < x.c.B; base += 64) {
        const bool in = base + lane < x.c.B && x.a.starts[base + lane] <= it.token;
        before += __popcll(__ballot(in));
    }
    if (before == 0) { return it; }
    const Seq s = sequence(x, before - 1);
    if (it.token - s.start < s.tokens) {
        it.b = before - 1;
        it.pos = s.history + it.token - s.start;
    }
    return it;
}

// A half tile of the walk: its first key's tile of 32, and its page.
struct Half {
    int32_t tile;
    int32_t page;
};

// Tiles [j0, j1) of the item's list, 32 keys each.
template <int D, bool BF, int NT, bool CARE>
__device__ __forceinline__ void sparse_walk(const SparseArgs& y, const Item& it, int j0, int j1, int c, int g, Rows<D, BF, NT>& r, float down) {
    const PagedAttnArgs& x = y.x;
    const int lane = threadIdx.x & 63;
    const int lt = y.block_shift - 5; // log2(tiles of a block)
    const int32_t* list = y.selected + (static_cast<int64_t>(it.token) * x.c.Hkv + it.h) * y.count;
    const int32_t* table = x.c.table + it.b * x.c.table_row;
    // 64 halves (32 tiles) at a time, one per lane, the next 64 fetched ahead
    const auto fetch = [&](int j) {
        const int v = j + (lane >> 1);
        Half f{0, -1};
        if (v < j1) {
            const int blk = list[v >> lt];
            if (blk >= 0 && blk <= (it.pos >> y.block_shift)) {
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
__device__ __forceinline__ void walk_rows(const SparseArgs& y, const Item& it, int j0, int j1, int c, int g, Rows<D, BF, NT>& r, float (&M)[NT],
                                          float (&L)[NT]) {
    const PagedAttnArgs& x = y.x;
    sparse_walk<D, BF, NT, false>(y, it, j0, j1, c, g, r, 1.0f);
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
            const int32_t* list = y.selected + (static_cast<int64_t>(it.token) * x.c.Hkv + it.h) * y.count;
            const int32_t* table = x.c.table + it.b * x.c.table_row;
#pragma unroll 1
            for (int j = j0; j < j1; ++j) {
                const int blk = __builtin_amdgcn_readfirstlane(list[j >> lt]);
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
            sparse_walk<D, BF, NT, true>(y, it, j0, j1, c, g, r, lower ? kCareDown : 1.0f);
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
        const Item it = item_of(y, id, 16 * NT, lane);
        if (it.b < 0) { return; }
        walk_rows<D, BF, NT>(y, it, 0, tiles, c, g, r, M, L);
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
        const Item it = item_of(y, id, 16 * NT, lane);
        if (it.b < 0) { return; }
        const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * part / y.parts), t1 = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / y.parts);
        const int j0 = t0 + (t1 - t0) * wave / 4, j1 = t0 + (t1 - t0) * (wave + 1) / 4;
        walk_rows<D, BF, NT>(y, it, j0, j1, c, g, r, M, L);
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

// ---- groups of tokens ------------------------------------------------------------------------------
//
// The rows of a wave: per_tile tokens' heads in each of NT 16-row tiles (token t of the group: tile t / per_tile, its head q row
// (t % per_tile) G + q). The group's lists become one list of (block, tokens that take it) in LDS, through a bit field
// of the blocks; a tile of keys is multiplied for the row tiles that take it, and a row whose token does not sees none of it.
// Lists with an entry twice are not merged: their entries stand one after another, for one token each.
// A wave stages 32 keys in LDS, whole rows by DMA: straight from the cache, as single tokens do it, every 16-byte piece of K
// is a cache access of its own, and those bounded it (2,048 tokens over 16 blocks of 64 at 24/4/256 BF16 807 us, the
// caches busy 70% of that). K makes room for the next tile's as soon as it is in registers, then V; DMAs land in order.

constexpr int kListMost = 512;  // entries of a group's lists
constexpr int kGroupMost = 8;   // tokens of a group: bits above a block's number
constexpr int kBlockBits = 24;
static_assert(kPagedMaxKeys / 32 <= (1 << kBlockBits));

template <int D, bool BF>
struct Stage {
    static constexpr int kRow = BF ? 2 * D : D;
    static constexpr int kPlane = 32 * kRow;
    static constexpr int kBytes = 2 * kPlane;
    static constexpr int kHalfDma = 16 * kRow / 1024; // 1 KiB DMAs of a plane's half tile
    static constexpr int kOps = 2 * kHalfDma + (BF ? 0 : 2 * (D / 128)); // loads of a plane's tile, its scales included
    static constexpr int kRowsPerDma = 1024 / kRow;
    static constexpr int kVariants = 8 / kRowsPerDma;
    static constexpr int kTable = kBytes / 4 < 2048 ? kBytes / 4 : 2048; // blocks of a pass over the lists
};

// s_waitcnt with at most n vector loads outstanding, and with no LDS operation.
constexpr int waitcnt_vm(int n) { return (n & 0xf) | ((n >> 4) << 14) | (0x7 << 4) | (0xf << 8); }
constexpr int kWaitLgkm0 = 0xc07f;

// The 16-byte piece p of LDS row r holds piece p ^ (r & 7) of the cache's row: eight rows' same pieces lie in different banks.
template <int D, bool BF>
__device__ __forceinline__ void dma_plane(const PagedAttnArgs& x, const char* plane, int64_t page_stride, int h, int tile, Halves hv, NMI_AS3 char* to, int lane) {
    using ST = Stage<D, BF>;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        const __amdgpu_buffer_rsrc_t rows = half_rows(x, plane, page_stride, ST::kRow, h, tile, kt, hv);
#pragma unroll
        for (int q = 0; q < ST::kHalfDma; ++q) {
            const int in_row = 16 * lane % ST::kRow, row = ST::kRowsPerDma * (q % ST::kVariants) + 16 * lane / ST::kRow;
            dma16(rows, to + (kt * ST::kHalfDma + q) * 1024, (16 * lane - in_row) + (in_row ^ ((row & 7) * 16)), q * 1024);
        }
    }
}

template <int D, bool BF>
__device__ __forceinline__ void stage_keys(const PagedAttnArgs& x, int h, int tile, Halves hv, NMI_AS3 char* st, int lane, int g, ChunkK<D, BF>& r) {
    if constexpr (!BF) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const __amdgpu_buffer_rsrc_t ksb = half_rows(x, x.c.ks, x.c.ks_page, D / 32, h, tile, kt, hv);
#pragma unroll
            for (int w = 0; w < D / 128; ++w) {
                r.ks[kt][w] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(ksb, 4 * g * (D / 32) + 16 * w, 0, 0));
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    dma_plane<D, BF>(x, x.c.k, x.c.k_page, h, tile, hv, st, lane);
    __builtin_amdgcn_sched_barrier(0);
}

template <int D, bool BF>
__device__ __forceinline__ void stage_values(const PagedAttnArgs& x, int h, int tile, Halves hv, NMI_AS3 char* st, int lane, int g, ChunkV<D, BF>& r) {
    if constexpr (!BF) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const __amdgpu_buffer_rsrc_t vsb = half_rows(x, x.c.vs, x.c.vs_page, D / 32, h, tile, kt, hv);
#pragma unroll
            for (int w = 0; w < D / 128; ++w) {
                r.vs[kt][w] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vsb, 4 * g * (D / 32) + 16 * w, 0, 0));
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    dma_plane<D, BF>(x, x.c.v, x.c.v_page, h, tile, hv, st + Stage<D, BF>::kPlane, lane);
    __builtin_amdgcn_sched_barrier(0);
}

template <int D, bool BF>
__device__ __forceinline__ void read_keys(const NMI_AS3 char* st, int c, int g, ChunkK<D, BF>& r) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int i = 0; i < Chunk<D, BF>::KP; ++i) {
            r.k[kt][i] = *reinterpret_cast<const NMI_AS3 u4*>(st + (16 * kt + c) * Stage<D, BF>::kRow + (((4 * i + g) ^ (c & 7)) * 16));
        }
    }
}

template <int D, bool BF>
__device__ __forceinline__ void read_values(const NMI_AS3 char* st, int c, int g, ChunkV<D, BF>& r) {
    st += Stage<D, BF>::kPlane;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = 4 * g + j;
#pragma unroll
            for (int i = 0; i < Chunk<D, BF>::VP; ++i) {
                const NMI_AS3 char* at = st + (16 * kt + row) * Stage<D, BF>::kRow;
                if constexpr (BF) {
                    const u4 w = *reinterpret_cast<const NMI_AS3 u4*>(at + (((16 * i + c) ^ (row & 7)) * 16));
#pragma unroll
                    for (int e = 0; e < 4; ++e) { r.v[4 * kt + j][i][e] = w[e]; }
                } else {
                    r.v[4 * kt + j][i][0] = *reinterpret_cast<const NMI_AS3 uint32_t*>(at + (((4 * i + (c >> 2)) ^ (row & 7)) * 16) + 4 * (c & 3));
                }
            }
        }
    }
}

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

// The group's blocks, each with the tokens that take it, in `list`; how many. `table`: scratch of `most` words.
__device__ __forceinline__ int merge_lists(const SparseArgs& y, const Group& q, uint32_t* list, uint32_t* table, int most, int lane) {
    const int32_t* from = y.selected + (static_cast<int64_t>(q.token) * y.x.c.Hkv + q.h) * y.count;
    const int64_t next = static_cast<int64_t>(y.x.c.Hkv) * y.count;
    const int entries = q.count * y.count;
    const int blocks = ((q.pos + q.count - 1) >> y.block_shift) + 1;
    bool twice = false;
    int n = 0;
    for (int b0 = 0; b0 < blocks; b0 += most) {
        const int some = min(most, blocks - b0);
        for (int i = lane; i < some; i += 64) { table[i] = 0u; }
        wave_sync();
        for (int e = lane; e < entries; e += 64) {
            const int t = e / y.count;
            const int blk = from[t * next + (e - t * y.count)];
            if (blk >= b0 && blk < b0 + some && blk <= ((q.pos + t) >> y.block_shift)) { twice |= ((atomicOr(&table[blk - b0], 1u << t) >> t) & 1u) != 0u; }
        }
        wave_sync();
        for (int i0 = 0; i0 < some; i0 += 64) {
            const uint32_t m = i0 + lane < some ? table[i0 + lane] : 0u;
            const uint64_t all = __ballot(m != 0u);
            if (m != 0u) { list[n + __popcll(all & ((uint64_t{1} << lane) - 1))] = static_cast<uint32_t>(b0 + i0 + lane) | (m << kBlockBits); }
            n += __popcll(all);
        }
        wave_sync();
    }
    if (__any(twice)) {
        n = entries;
        for (int e = lane; e < entries; e += 64) {
            const int t = e / y.count;
            const int blk = from[t * next + (e - t * y.count)];
            list[e] = blk >= 0 && blk <= ((q.pos + t) >> y.block_shift) ? static_cast<uint32_t>(blk) | (1u << (kBlockBits + t)) : 0u;
        }
        wave_sync();
    }
    return n;
}

// The lane's rows of the group.
template <int D, bool BF, int NT>
struct GroupRows {
    Rows<D, BF, NT> r;
    int pos[NT];       // the row's position, -1: no row
    uint32_t bit[NT];  // its token's bit
    int head[NT];
    uint32_t tokens;   // all rows' bits
};

// Row tiles nt0 .. of the group.
template <int D, bool BF, int NT>
__device__ __forceinline__ void init_group(const SparseArgs& y, const Group& q, int nt0, int c, int g, GroupRows<D, BF, NT>& z) {
    const PagedAttnArgs& x = y.x;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int in = c / x.G, before = (nt0 + nt) * y.per_tile, t = before + in;
        const bool valid = in < y.per_tile && t < q.count;
        z.head[nt] = c - in * x.G;
        z.pos[nt] = valid ? q.pos + t : -1;
        z.bit[nt] = valid ? 1u << t : 0u;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(x.a.q.data + static_cast<int64_t>(q.token + (valid ? t : 0)) * x.a.q.token_stride) +
                              (q.h * x.G + (valid ? z.head[nt] : 0)) * D;
        init_row<D, BF, NT>(x, src, valid, nt, g, z.r);
    }
    z.tokens = ((1u << min(q.count, (nt0 + NT) * y.per_tile)) - 1u) & ~((1u << min(q.count, nt0 * y.per_tile)) - 1u);
    z.r.hi = q.pos + q.count - 1;
}

// Tiles [j0, j1) of the merged list, for the row tiles nt0 ..
template <int D, bool BF, int NT, bool CARE>
__device__ __forceinline__ void group_walk(const SparseArgs& y, const Group& q, const uint32_t* list, int j0, int j1, NMI_AS3 char* st, int nt0, int lane,
                                           int c, int g, GroupRows<D, BF, NT>& z, float down) {
    using ST = Stage<D, BF>;
    const PagedAttnArgs& x = y.x;
    const int lt = y.block_shift - 5;
    const int32_t* table = x.c.table + q.b * x.c.table_row;
    const int last = q.pos + q.count - 1;
    struct Half {
        int tile, page;
        uint32_t mask;
    };
    const auto fetch = [&](int j) {
        const int v = j + (lane >> 1);
        Half f{0, -1, 0u};
        if (v < j1) {
            const uint32_t e = list[v >> lt];
            f.mask = e >> kBlockBits;
            f.tile = static_cast<int>((e & ((1u << kBlockBits) - 1u)) << lt) + (v & ((1 << lt) - 1));
            const int key = 32 * f.tile + 16 * (lane & 1);
            if (f.mask != 0u && key <= last && (key >> x.c.page_shift) < x.c.max_pages) {
                const int page = table[key >> x.c.page_shift];
                f.page = page >= 0 && page < x.c.pages ? page : -1;
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
        uint32_t mask;
    };
    const auto tile_at = [&](int j) { // past the end no page
        const int i = 2 * (j - j0);
        const bool now = (i & 127) < 64;
        Tile t;
        t.tile = __builtin_amdgcn_readlane(now ? ids.tile : next_ids.tile, i & 63);
        t.mask = __builtin_amdgcn_readlane(now ? ids.mask : next_ids.mask, i & 63);
        t.hv.page[0] = __builtin_amdgcn_readlane(now ? ids.page : next_ids.page, i & 63);
        t.hv.page[1] = __builtin_amdgcn_readlane(now ? ids.page : next_ids.page, (i & 63) + 1);
        return t;
    };
    Probs<NT> pr;
    uint32_t large = 0u; // known already
    ChunkK<D, BF> ka;
    ChunkV<D, BF> va;
    init_group<D, BF, NT>(y, q, nt0, c, g, z);
    Tile ta = tile_at(j0);
    stage_keys<D, BF>(x, q.h, ta.tile, ta.hv, st, lane, g, ka);
    stage_values<D, BF>(x, q.h, ta.tile, ta.hv, st, lane, g, va);
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
        const bool some = (ta.hv.page[0] & ta.hv.page[1]) >= 0 && (ta.mask & z.tokens) != 0u; // otherwise the tile adds nothing
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) { z.r.pos[nt] = (ta.mask & z.bit[nt]) != 0u ? z.pos[nt] : -1; }
        z.r.lo = (ta.mask & z.tokens) == z.tokens ? q.pos : -1;
        const Tile tb = tile_at(j + 1); // before the refill: tile 31 of a fetch is still in it
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(ST::kOps)); // the keys have landed
        read_keys<D, BF>(st, c, g, ka);
        __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
        ChunkK<D, BF> kb;
        stage_keys<D, BF>(x, q.h, tb.tile, tb.hv, st, lane, g, kb);
        if (some) { chunk_probs<D, BF, NT>(x, ta.tile, ta.hv, g, ka, z.r, pr); }
        if constexpr (!BF) { __builtin_memcpy(ka.ks, kb.ks, sizeof(ka.ks)); }
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(ST::kOps)); // the values have landed
        read_values<D, BF>(st, c, g, va);
        __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
        ChunkV<D, BF> vb;
        stage_values<D, BF>(x, q.h, tb.tile, tb.hv, st, lane, g, vb);
        if (some) { chunk_values<D, BF, NT, CARE>(ta.tile, ta.hv, g, pr, va, z.r, down, large); }
        if constexpr (!BF) { __builtin_memcpy(va.vs, vb.vs, sizeof(va.vs)); }
        if (((j - j0) & 1) == 0) { refill(j); }
        ta = tb;
    }
    __builtin_amdgcn_s_waitcnt(0); // no DMA may land after this point
}

// WAVES: a wave per group; otherwise four waves share one, and `parts` workgroups may.
template <int D, bool BF, int NT, bool WAVES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 128 ? 2 : 1, D == 128 ? 2 : 1))) void sparse_group_kernel(SparseArgs y) {
    using ST = Stage<D, BF>;
    static_assert(2 * NT * (D / 16) * 64 * 16 <= 4 * ST::kBytes, "the join exceeds the stages");
    __shared__ __attribute__((aligned(1024))) char smem[4 * ST::kBytes];
    __shared__ uint32_t lists[4][kListMost];
    __shared__ float2 xm[2][NT * 64];
    const PagedAttnArgs& x = y.x;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    int64_t id;
    int part = 0;
    if constexpr (WAVES) {
        // neighbouring waves: neighbouring groups of one head, whose lists are much alike
        id = (static_cast<int64_t>(blockIdx.x / x.c.Hkv) * 4 + wave) * x.c.Hkv + blockIdx.x % x.c.Hkv;
        if (id >= y.items) { return; }
    } else {
        id = blockIdx.x % y.items;
        part = static_cast<int>(blockIdx.x / y.items);
    }
    const Group q = group_of(y, id, lane);
    if (q.b < 0) { return; }
    char* own = smem + wave * ST::kBytes;
    const int entries = merge_lists(y, q, lists[wave], reinterpret_cast<uint32_t*>(own), ST::kTable, lane);
    const int tiles = entries << (y.block_shift - 5);
    int j0 = 0, j1 = tiles;
    if constexpr (!WAVES) {
        const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * part / y.parts), t1 = static_cast<int>(static_cast<int64_t>(tiles) * (part + 1) / y.parts);
        j0 = t0 + (t1 - t0) * wave / 4;
        j1 = t0 + (t1 - t0) * (wave + 1) / 4;
    }
    NMI_AS3 char* st = (NMI_AS3 char*)own;
    GroupRows<D, BF, NT> z;
    group_walk<D, BF, NT, false>(y, q, lists[wave], j0, j1, st, 0, lane, c, g, z, 1.0f);
    bool lower = false;
    if constexpr (BF) {
        uint32_t top = 0u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) { top = max(top, __float_as_uint(z.r.O[nt][t][e]) << 1); }
            }
        }
        // sums from 2^100 up, infinite ones or NaN: the careful walk
        if (__builtin_expect(__any(top >= static_cast<uint32_t>(127 + 100) << 24), 0)) {
            uint32_t large = 0u;
            const int lt = y.block_shift - 5;
            const int32_t* table = x.c.table + q.b * x.c.table_row;
#pragma unroll 1
            for (int j = j0; j < j1; ++j) {
                const uint32_t e = __builtin_amdgcn_readfirstlane(lists[wave][j >> lt]);
                if ((e >> kBlockBits) == 0u) { continue; }
                const int tile = static_cast<int>((e & ((1u << kBlockBits) - 1u)) << lt) + (j & ((1 << lt) - 1));
                ChunkV<D, BF> cv;
                load_values<D, BF>(x, q.h, tile, halves_of(x, table, tile, q.pos + q.count - 1), c, g, cv);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
#pragma unroll
                    for (int i = 0; i < Chunk<D, BF>::VP; ++i) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) { large = max(large, larger_bits(finite_word(cv.v[k][i][w]))); }
                    }
                }
            }
            lower = __any(large >= kCareTop);
            // a row tile at a time: two and the care do not fit the registers
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                GroupRows<D, BF, 1> one;
                group_walk<D, BF, 1, true>(y, q, lists[wave], j0, j1, st, nt, lane, c, g, one, lower ? kCareDown : 1.0f);
                z.r.m[nt] = one.r.m[0];
                z.r.l[nt] = one.r.l[0];
#pragma unroll
                for (int t = 0; t < D / 16; ++t) { z.r.O[nt][t] = one.r.O[0][t]; }
            }
        }
    }
    float M[NT], L[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        M[nt] = z.r.m[nt] == -INFINITY ? -INFINITY : z.r.m[nt] * z.r.rowmul[nt];
        L[nt] = group4_sum(z.r.l[nt]);
        if (lower) { care_units(M[nt], L[nt]); }
    }
    if constexpr (!WAVES) {
        __syncthreads(); // every wave's stage is done with
        join_waves<D, BF, NT, 4>(z.r, M, L, wave, lane, *reinterpret_cast<f4(*)[2][NT * (D / 16) * 64]>(smem), xm);
        if (wave != 0) { return; }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        if (z.pos[nt] < 0) { continue; }
        if (!WAVES && y.parts > 1) {
            store_part<D, BF, NT>(x, z.r, nt, M[nt], L[nt], (id * (16 * NT) + 16 * nt + c) * y.parts + part, g);
        } else {
            store_out<D, BF, NT>(x, q.token + z.pos[nt] - q.pos, q.h, z.head[nt], z.r, nt, L[nt], g);
        }
    }
}

// The parts of an item's rows, one after another: D / 4 threads a row, 16 nt rows an item.
template <int D>
__global__ __launch_bounds__(256) void sparse_merge_kernel(SparseArgs y, int rows) {
    const PagedAttnArgs& x = y.x;
    constexpr int TPR = D / 4, RPB = 256 / TPR;
    const int lane = threadIdx.x & 63;
    const int64_t id = blockIdx.x / (rows / RPB);
    const int row = static_cast<int>(blockIdx.x % (rows / RPB)) * RPB + threadIdx.x / TPR;
    int64_t token;
    int head;
    if (y.tokens > 1) {
        const Group q = group_of(y, id, lane);
        const int in = (row & 15) / x.G, t = (row >> 4) * y.per_tile + in;
        if (q.b < 0 || in >= y.per_tile || t >= q.count) { return; }
        token = q.token + t;
        head = q.h * x.G + (row & 15) - in * x.G;
    } else {
        const Item it = item_of(y, id, rows, lane);
        if (it.b < 0 || it.row0 + row >= x.G) { return; }
        token = it.token;
        head = it.h * x.G + it.row0 + row;
    }
    const int d = 4 * (threadIdx.x % TPR);
    Merge m;
#pragma unroll 4
    for (int k = 0; k < y.parts; ++k) {
        const int64_t at = (id * rows + row) * y.parts + k;
        const float2 ml = *reinterpret_cast<const float2*>(x.part_ml + 2 * at);
        m.add(ml.x, ml.y, *reinterpret_cast<const f4*>(x.part_o + at * D + d));
    }
    uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + token * x.a.out.token_stride) + head * D + d;
    *reinterpret_cast<u2*>(out) = out_pair(m.O, m.L);
}

// How a call is cut.
struct SparsePlan {
    int32_t nt = 1;
    int32_t row_tiles = 1;
    int32_t tokens = 1;   // of a group
    int32_t per_tile = 1;
    int64_t items = 0;
    bool waves = false; // a wave per item
    int32_t parts = 1;  // workgroups per item
    size_t ml_offset = 0;
    size_t bytes = 0;
};

constexpr int kCus = 256;

SparsePlan plan_sparse(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t max_new, int32_t selected, int32_t block_shift) {
    SparsePlan p;
    const int32_t G = Hq / Hkv;
    const int64_t tiles = static_cast<int64_t>(selected) << (block_shift - 5);
    if (G <= 16) {
        // one or two row tiles of whole tokens, as many as the lists leave room for
        p.per_tile = std::min(16 / G, G <= 2 ? 8 : 4);
        p.tokens = std::min({p.per_tile * (G <= 2 ? 1 : 2), max_new, kListMost / selected});
    }
    if (p.tokens > 1) {
        p.nt = p.tokens > p.per_tile ? 2 : 1;
        p.items = (tokens + static_cast<int64_t>(B) * (p.tokens - 1)) / p.tokens * Hkv;
    } else {
        p.tokens = 1;
        p.nt = G <= 16 ? 1 : 2;
        p.row_tiles = (G + 16 * p.nt - 1) / (16 * p.nt);
        p.items = tokens * Hkv * p.row_tiles;
    }
    const int64_t slots = kCus * (D == 128 ? 2 : 1); // workgroups of four waves at a time
    p.waves = p.items >= 4 * slots || tiles < 4;
    if (!p.waves) {
        // at least two tiles for a wave
        p.parts = static_cast<int32_t>(std::max<int64_t>(1, std::min(slots / p.items, tiles / 8)));
    }
    if (p.parts > 1) {
        const size_t rows = static_cast<size_t>(p.items) * 16 * p.nt * p.parts;
        p.ml_offset = (rows * D * sizeof(float) + 255) & ~size_t{255};
        p.bytes = p.ml_offset + rows * 2 * sizeof(float);
    }
    return p;
}

template <int D, bool BF, int NT>
void launch(const SparseArgs& y, const SparsePlan& p, hipStream_t stream) {
    const int64_t per = y.x.c.Hkv;
    const int64_t grid = p.waves ? (p.items / per + 3) / 4 * per : p.items * p.parts;
    if (grid > 0x7FFFFF) { throw Unsupported("paged sparse attention: more than 2^23 workgroups are not built"); }
    const dim3 blocks(static_cast<uint32_t>(grid));
    if (p.tokens > 1) {
        if (p.waves) {
            hipLaunchKernelGGL((sparse_group_kernel<D, BF, NT, true>), blocks, dim3(256), 0, stream, y);
        } else {
            hipLaunchKernelGGL((sparse_group_kernel<D, BF, NT, false>), blocks, dim3(256), 0, stream, y);
        }
        check_launch("sparse_group_kernel");
    } else {
        if (p.waves) {
            hipLaunchKernelGGL((sparse_attn_kernel<D, BF, NT, true>), blocks, dim3(256), 0, stream, y);
        } else {
            hipLaunchKernelGGL((sparse_attn_kernel<D, BF, NT, false>), blocks, dim3(256), 0, stream, y);
        }
        check_launch("sparse_attn_kernel");
    }
    if (p.parts > 1) {
        const uint32_t groups = static_cast<uint32_t>(p.items * (16 * NT / (1024 / D)));
        hipLaunchKernelGGL((sparse_merge_kernel<D>), dim3(groups), dim3(256), 0, stream, y, 16 * NT);
        check_launch("sparse_merge_kernel");
    }
}

} // namespace

size_t sparse_attention_bytes(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t selected, int32_t block_shift) {
    size_t most = 0; // over every envelope
    for (int32_t max_new = 1; max_new <= kGroupMost; ++max_new) {
        most = std::max(most, plan_sparse(Hq, Hkv, D, tokens, B, max_new, selected, block_shift).bytes);
    }
    return most;
}

void launch_sparse_attention(const PagedAttention& a, const int32_t* selected, int32_t count, int32_t block_shift, const PagedRef& c,
                             void* workspace, hipStream_t stream) {
    const SparsePlan p = plan_sparse(a.Hq, c.Hkv, c.D, a.tokens, c.B, a.max_new, count, block_shift);
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
        p.nt == 1 ? launch<D, BF, 1>(y, p, stream) : launch<D, BF, 2>(y, p, stream);
    };
    const auto cache = [&](auto d) { c.bf16 ? pick(d, std::true_type{}) : pick(d, std::false_type{}); };
    c.D == 128 ? cache(std::integral_constant<int, 128>{}) : cache(std::integral_constant<int, 256>{});
}

} // namespace nmi
