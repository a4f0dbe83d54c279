// Attention of packed new tokens over selected blocks of a paged KV cache on gfx950.
//
// Mathematics: token n at position p has for every KV head a list of blocks; it sees the rows j <= p of those blocks whose page
// exists (an entry that stands twice counts twice), out = sum_j softmax_j(scale * q . K_j) V_j in one pass with a running
// maximum and sum, zero where no row is seen. Numbers as in paged_attention.hip, whose walk over 32 keys at a time this
// is: the query heads of the token's KV head are the rows of a 16-row tile, K and V go straight from the cache to the matrix
// cores' operands.
//
// A token has a list of its own, so nothing of K and V is shared between tokens but through the caches: a wave (or four, or
// several workgroups' waves, where the tokens alone do not fill the chip) takes a token and KV head.
// What bounds it: HBM for decode steps; for prompts the VALU, which decodes every row for one token's heads.
#include "common.h"
#include "paged_internal.h"
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
    int32_t parts;     // workgroups of a token, KV head and row tile
    int64_t items;     // tokens x KV heads x row tiles
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
            if (row < x.G) { store_out<D, BF, NT>(x, Seq{it.token, 1, it.pos}, it.h, row, r, nt, L[nt], g); }
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
                const int64_t out_row = static_cast<int64_t>(it.token) * x.a.Hq + it.h * x.G + row;
                store_part<D, BF, NT>(x, r, nt, M[nt], L[nt], out_row * y.parts + part, g);
            } else {
                store_out<D, BF, NT>(x, Seq{it.token, 1, it.pos}, it.h, row, r, nt, L[nt], g);
            }
        }
    }
}

// The parts of a row, one after another: D / 4 threads a row.
template <int D>
__global__ __launch_bounds__(256) void sparse_merge_kernel(SparseArgs y) {
    const PagedAttnArgs& x = y.x;
    constexpr int TPR = D / 4;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR; // token * Hq + head
    const int64_t token = row / x.a.Hq;
    const int head = static_cast<int>(row - token * x.a.Hq);
    // the sequence that holds the token; the rows of a wave may be of several tokens
    int lo = 0, hi = x.c.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (x.a.starts[mid] <= token) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    if (token >= x.a.tokens) { return; }
    const Seq s = sequence(x, lo);
    if (token < s.start || token - s.start >= s.tokens) { return; }
    const int d = 4 * (threadIdx.x % TPR);
    Merge m;
#pragma unroll 4
    for (int k = 0; k < y.parts; ++k) {
        const int64_t at = row * y.parts + k;
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
    int64_t items = 0;
    bool waves = false; // a wave per item
    int32_t parts = 1;  // workgroups per item
    size_t ml_offset = 0;
    size_t bytes = 0;
};

constexpr int kCus = 256;

SparsePlan plan_sparse(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t selected, int32_t block_shift) {
    SparsePlan p;
    const int32_t G = Hq / Hkv;
    p.nt = G <= 16 ? 1 : 2;
    p.row_tiles = (G + 16 * p.nt - 1) / (16 * p.nt);
    p.items = tokens * Hkv * p.row_tiles;
    const int64_t tiles = static_cast<int64_t>(selected) << (block_shift - 5);
    const int64_t slots = kCus * (D == 128 ? 2 : 1); // workgroups of four waves at a time
    p.waves = p.items >= 4 * slots || tiles < 4;
    if (!p.waves) {
        // at least two tiles for a wave
        p.parts = static_cast<int32_t>(std::max<int64_t>(1, std::min(slots / p.items, tiles / 8)));
    }
    if (p.parts > 1) {
        const size_t rows = static_cast<size_t>(tokens) * Hq * p.parts;
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
    if (p.waves) {
        hipLaunchKernelGGL((sparse_attn_kernel<D, BF, NT, true>), dim3(static_cast<uint32_t>(grid)), dim3(256), 0, stream, y);
    } else {
        hipLaunchKernelGGL((sparse_attn_kernel<D, BF, NT, false>), dim3(static_cast<uint32_t>(grid)), dim3(256), 0, stream, y);
    }
    check_launch("sparse_attn_kernel");
    if (p.parts > 1) {
        const int64_t rows = y.x.a.tokens * y.x.a.Hq;
        hipLaunchKernelGGL((sparse_merge_kernel<D>), dim3(static_cast<uint32_t>((rows * (D / 4) + 255) / 256)), dim3(256), 0, stream, y);
        check_launch("sparse_merge_kernel");
    }
}

} // namespace

size_t sparse_attention_bytes(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t selected, int32_t block_shift) {
    return plan_sparse(Hq, Hkv, D, tokens, selected, block_shift).bytes;
}

void launch_sparse_attention(const PagedAttention& a, const int32_t* selected, int32_t count, int32_t block_shift, const PagedRef& c,
                             void* workspace, hipStream_t stream) {
    const SparsePlan p = plan_sparse(a.Hq, c.Hkv, c.D, a.tokens, count, block_shift);
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
    const auto pick = [&](auto d, auto bf) {
        constexpr int D = decltype(d)::value;
        constexpr bool BF = decltype(bf)::value;
        p.nt == 1 ? launch<D, BF, 1>(y, p, stream) : launch<D, BF, 2>(y, p, stream);
    };
    const auto cache = [&](auto d) { c.bf16 ? pick(d, std::true_type{}) : pick(d, std::false_type{}); };
    c.D == 128 ? cache(std::integral_constant<int, 128>{}) : cache(std::integral_constant<int, 256>{});
}

} // namespace nmi
