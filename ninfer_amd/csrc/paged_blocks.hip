// Blocks of keys of a paged KV cache on gfx950: a mean for each, and the blocks that a token's queries score highest.
//
// Mathematics: a block's rows are summed in 64 bits (sums of stored values, exact while INT8 scales lie within 2^29 / rows of each other:
// a lane adds at most rows / 2 products, each below 2^12.1 times the largest scale and a multiple of 2^-11 of the smallest; BF16 values
// within 2^45 / rows), step = max |sum| * FP64(1 / 127), code = rne(sum * (1 / step)), scale = FP32(step / rows): code *
// scale is the mean with 8 bits. A token's query for a KV head is the sum of its group's heads, made codes the same way; a block's score is scale * <codes, codes>, the product of
// whole numbers exact on the matrix cores (up to 2^22), so it does not depend on any order, and which blocks are
// selected is defined to the bit. A token always takes the first blocks and the last ones up to its own; of those
// between it takes the `top` highest scores, the lower index of equals. A block with an infinite or NaN key has an infinite scale
// and scores +infinity.
#include "common.h"
#include "device_utils.h"
#include "paged_internal.h"
#include "paged_place.h"

#include <algorithm>

namespace nmi {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr double kStep = 1.0 / 127.0; // a product, not a quotient: part of the definition, since it decides ties of codes

// max |x| over the D / 8 lanes of a head in every one of them, infinite where a value is infinite or NaN.
template <int D>
__device__ __forceinline__ double head_amax(const double (&x)[8]) {
    double m = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) { m = fabs(x[e]) < INFINITY ? fmax(m, fabs(x[e])) : static_cast<double>(INFINITY); }
#pragma unroll
    for (int d = 1; d < D / 8; d *= 2) { m = fmax(m, __shfl_xor(m, d)); }
    return m;
}

// Eight codes of x at 1 / step, none where there is nothing to tell (amax zero or infinite).
__device__ __forceinline__ i2 codes_of(const double (&x)[8], double amax, double step) {
    uint32_t code[2] = {0u, 0u};
    if (amax > 0.0 && amax < INFINITY) {
        const double inv = 1.0 / step;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double r = fmin(127.0, fmax(-127.0, rint(x[e] * inv)));
            code[e >> 2] |= (static_cast<uint32_t>(static_cast<int32_t>(r)) & 0xffu) << (8 * (e & 3));
        }
    }
    return i2{static_cast<int>(code[0]), static_cast<int>(code[1])};
}

// ---- means ---------------------------------------------------------------------------------------
//
// A wave per touched block and head: D / 8 lanes a row, eight values a lane, so 512 values (four or two rows) at a time.
// What bounds it: latency and launch. 27,090 rows of 8 x 128 INT8 in blocks of 64 (30.9 MB) take 14.9 us (with
// codes made FP32, times the scale, made FP64 and added 15.8); with 4 or 16 rows' loads on their way instead of 8, one wave a
// workgroup, or two waves a block the same, with four waves a block 18.2.

struct UpdateArgs {
    int64_t tokens;
    const int32_t* starts;
    const int32_t* history;
    PagedRef c;
    BlocksRef b;
    int64_t units; // waves
};

template <int D, bool BF>
__global__ __launch_bounds__(256) void block_update_kernel(UpdateArgs x) {
    constexpr int L = D / 8;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (unit >= x.units) { return; }
    const int h = static_cast<int>(unit % x.c.Hkv);
    const int bs = x.b.shift;
    // the blocks that hold new rows
    const Found f = find_unit(x.c.B, static_cast<int>(unit / x.c.Hkv), lane, [&](int b) { return span_of(x.starts, x.history, b, x.tokens); }, [&](const Span& s) {
        return s.tokens > 0 ? static_cast<int>(((static_cast<int64_t>(s.history) + s.tokens - 1) >> bs) - (s.history >> bs)) + 1 : 0;
    });
    if (f.b < 0) { return; }
    const int64_t row0 = static_cast<int64_t>((f.s.history >> bs) + f.at) << bs;
    const int rows = static_cast<int>(min(static_cast<int64_t>(1) << bs, f.s.history + static_cast<int64_t>(f.s.tokens) - row0));
    if ((row0 >> x.c.page_shift) >= x.c.max_pages) { return; }
    const int32_t page = x.c.table[f.b * x.c.table_row + (row0 >> x.c.page_shift)];
    if (page < 0 || page >= x.c.pages) { return; }
    const int in_page = static_cast<int>(row0 & ((int64_t{1} << x.c.page_shift) - 1));
    const int64_t first = (static_cast<int64_t>(h) << x.c.page_shift) + in_page;
    const int li = lane & (L - 1), group = lane / L;
    constexpr int GROUPS = 64 / L;
    const char* k = x.c.k + page * x.c.k_page + first * (BF ? 2 * D : D) + li * (BF ? 16 : 8);
    const char* ks = x.c.ks + page * x.c.ks_page + first * (D / 32) + (li >> 3) * 2;
    double sum[8] = {}, scales = 0.0;
#pragma unroll 8
    for (int r = group; r < rows; r += GROUPS) {
        if constexpr (BF) {
            const i4 raw = *reinterpret_cast<const i4*>(k + r * (2 * D));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t w = static_cast<uint32_t>(raw[e >> 1]);
                sum[e] += __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
            }
        } else {
            const i2 raw = *reinterpret_cast<const i2*>(k + r * D);
            const double s = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(ks + r * (D / 32)));
            scales += s;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // the byte code + 128 in the high word of 4096: 4224 + code without a conversion
                const uint32_t high = __builtin_amdgcn_perm(0x40b00000u, static_cast<uint32_t>(raw[e >> 2]) ^ 0x80808080u,
                                                            0x0706000cu | static_cast<uint32_t>(e & 3) << 8);
                sum[e] = fma(__hiloint2double(static_cast<int>(high), 0), s, sum[e]);
            }
        }
    }
    if constexpr (!BF) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { sum[e] = fma(-4224.0, scales, sum[e]); }
    }
#pragma unroll
    for (int d = L; d < 64; d *= 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { sum[e] += __shfl_xor(sum[e], d); }
    }
    const double amax = head_amax<D>(sum);
    const double step = amax * kStep;
    const i2 code = codes_of(sum, amax, step);
    const int64_t slot = (static_cast<int64_t>(h) << (x.c.page_shift - bs)) + (in_page >> bs);
    if (group == 0) { *reinterpret_cast<i2*>(x.b.codes + page * x.b.code_page + slot * D + 8 * li) = code; }
    if (lane == 0) { *reinterpret_cast<float*>(x.b.scales + page * x.b.scale_page + slot * 4) = static_cast<float>(step / rows); }
}

// ---- selection -----------------------------------------------------------------------------------
//
// A workgroup per (tile of up to 16 tokens of a sequence, KV head): the tile's query codes, then 16 blocks at a time as
// 16x16x64 products of whole numbers (rows: tokens, columns: blocks), the scores to LDS as ordered keys; then the keys of a
// token, in registers, are counted against a middle that closes in on the `top`-th largest, and the list is written in order.
// What bounds it: for single tokens the means' reads (9 of 23 us at 4.6 TB/s for 32 tokens over up to 2,001 blocks), the choice (6 us
// of reductions and barriers) and launch; for prompts the choice's VALU (14 of 37 us for 4,096 tokens over 320 blocks, the VALU busy 89%).
// A sequence's blocks are not split over workgroups, so few tokens over many blocks leave CUs idle: one token at 40/8/128 over 2,049, 4,065
// and 15,626 blocks 20.5, 31.3 and 93.3 us (eight workgroups); and past 2,032 blocks a tile has fewer tokens and reads the means again
// for each: 4,096 tokens over 60,000, 131,072 and 260,096 rows in blocks of 64 121, 965 and 1,705 us. The forms of the choice share one
// kernel, whose scalars do not fit: 380 of them spilled to lanes of vector registers with four waves, 696 with eight.

struct SelectArgs {
    BlockSelect a;
    PagedRef c;
    BlocksRef b;
    int32_t G;
    int32_t tile_shift; // log2(tokens of a tile)
    int32_t cap;        // keys of a token in LDS
};

// FP32 as an unsigned number of the same order; zero is left for blocks that are not to choose.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f); // -0 as +0
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

// Which of a token's keys are chosen: those above `than`, and the first `equal` of those that equal it.
struct Threshold {
    uint32_t than;
    int equal;
};

__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ ((key & 0x80000000u) != 0u ? 0x80000000u : 0xffffffffu));
}

// Where the `under` largest of over + under values end if they are spread as normal ones with this sum and these squares'. (log2(x) 0.407
// is close to the normal quantile of 1 / (1 + x).)
__device__ __forceinline__ float normal_end(float sum, float squares, float over, float under) {
    const float inv = __builtin_amdgcn_rcpf(over + under), mean = sum * inv;
    const float deviation = __builtin_amdgcn_sqrtf(fmaxf(0.0f, fmaf(squares, inv, -mean * mean)));
    return fmaf(__builtin_amdgcn_logf(over * __builtin_amdgcn_rcpf(under)) * 0.407f, deviation, mean);
}

// The `want` largest of `there` keys from lo to hi (zeros are none); `count_from` says how many there are from a key on. The interval of the
// smallest chosen key closes in from both sides until as many keys as are wanted lie at its middle or above, or one value is
// left: at `guess`, then where the counts at its ends put the middle among the scores' values (four to five steps for scores spread
// as sums are, without a guess six to nine; halving takes 14), then, for scores that are not, at the keys' own middle.
template <typename F>
__device__ __forceinline__ Threshold top_keys(F count_from, int there, int want, uint32_t lo, uint32_t hi, float guess) {
    float over = static_cast<float>(there - want), under = static_cast<float>(want); // keys from lo on that are too many, above hi too few
    int side = 0;
#pragma unroll 1
    for (int step = 0; lo < hi; ++step) {
        uint32_t mid = lo + (hi - lo) / 2 + 1;
        if (step < 12) {
            const float a = value_of(lo), b = value_of(hi);
            const float share = fminf(0.984375f, fmaxf(0.015625f, over * __builtin_amdgcn_rcpf(over + under)));
            const float v = step == 0 && guess > a && guess < b ? guess : a + (b - a) * share;
            if (v > a && v < b) { mid = __builtin_amdgcn_readfirstlane(max(lo + 1u, min(hi, ordered(v)))); } // (not for infinite ends)
        }
        const int n = count_from(mid);
        if (n == want) { return Threshold{mid - 1u, 0}; } // (a key of mid - 1 is not chosen: none is counted)
        // an end that stays twice counts half: the middle moves towards it
        if (n > want) {
            lo = mid;
            over = static_cast<float>(n - want);
            under *= side > 0 ? 0.5f : 1.0f;
            side = 1;
        } else {
            hi = mid - 1u;
            under = static_cast<float>(want - n);
            over *= side < 0 ? 0.5f : 1.0f;
            side = -1;
        }
    }
    return Threshold{lo, want - (lo == 0xffffffffu ? 0 : count_from(lo + 1u))};
}

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t max_step(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROW_MASK, 0xf, true)));
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max_step<0x111, 0xf>(v);
    v = max_step<0x112, 0xf>(v);
    v = max_step<0x114, 0xf>(v);
    v = max_step<0x118, 0xf>(v);
    v = max_step<0x142, 0xa>(v);
    v = max_step<0x143, 0xc>(v);
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

// What the waves that choose for one token share.
struct Shared {
    int count[2][8]; // by turns: a wave may be a step ahead
    uint32_t least[8], most[8];
    float sum[8], squares[8];
    int taken[8], equal[8];
};

// The list of one token from its keys of = [0, count) by WAVES waves, R keys a lane; block `first` + i has key i. Returns how many.
template <int R, int WAVES>
__device__ __forceinline__ int choose(const uint32_t* of, int count, int want, int first, int32_t* out, int lane, int wave, Shared& sh) {
    uint32_t k[R];
    uint32_t most = 0u, least = 0u; // least as its complement
    float sum = 0.0f, squares = 0.0f;
    int there = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int at = (wave * R + i) * 64 + lane; // a wave's keys stand together, so lists come out in order
        k[i] = at < count ? of[at] : 0u;
        there += static_cast<int>(__popcll(__ballot(k[i] != 0u)));
        most = max(most, k[i]);
        least = max(least, k[i] != 0u ? ~k[i] : 0u);
        const float v = k[i] != 0u ? value_of(k[i]) : 0.0f;
        sum += v;
        squares = fmaf(v, v, squares);
    }
    int turn = 0;
    const auto total = [&](int n) {
        if constexpr (WAVES == 1) {
            return n;
        } else {
            if (lane == 0) { sh.count[turn][wave] = n; }
            __syncthreads();
            int s = 0;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) { s += sh.count[turn][i]; }
            turn ^= 1;
            return __builtin_amdgcn_readfirstlane(s);
        }
    };
    most = wave_max_u32(most);
    least = wave_max_u32(least);
    sum = wave_sum(sum);
    squares = wave_sum(squares);
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            sh.most[wave] = most;
            sh.least[wave] = least;
            sh.sum[wave] = sum;
            sh.squares[wave] = squares;
        }
    }
    there = total(there);
    if constexpr (WAVES > 1) { // every wave the same sums in the same order: they have to go the same ways
        sum = squares = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            most = max(most, sh.most[i]);
            least = max(least, sh.least[i]);
            sum += sh.sum[i];
            squares += sh.squares[i];
        }
    }
    Threshold y{0u, 0};
    if (there > want) {
        y = top_keys(
            [&](uint32_t from) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < R; ++i) { n += static_cast<int>(__popcll(__ballot(k[i] >= from))); }
                return total(n);
            },
            there, want, __builtin_amdgcn_readfirstlane(~least), __builtin_amdgcn_readfirstlane(most),
            normal_end(sum, squares, static_cast<float>(there - want), static_cast<float>(want)));
    }
    // what the waves before take, of both kinds
    int taken = 0, equal = 0;
    if constexpr (WAVES > 1) {
        int above = 0, same = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            above += static_cast<int>(__popcll(__ballot(k[i] > y.than)));
            same += static_cast<int>(__popcll(__ballot(k[i] == y.than && k[i] != 0u)));
        }
        if (lane == 0) {
            sh.taken[wave] = above;
            sh.equal[wave] = same;
        }
        __syncthreads();
        for (int i = 0; i < wave; ++i) {
            const int e = min(sh.equal[i], y.equal - equal);
            taken += sh.taken[i] + e;
            equal += e;
        }
    }
    int left = y.equal - equal;
    const uint64_t below = (uint64_t{1} << lane) - 1;
    if (left == 0) { // no choice among equals
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool take = k[i] > y.than;
            const uint64_t all = __ballot(take);
            if (take) { out[taken + __popcll(all & below)] = first + (wave * R + i) * 64 + lane; }
            taken += static_cast<int>(__popcll(all));
        }
        return min(there, want);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const uint64_t same = __ballot(k[i] == y.than && k[i] != 0u);
        const bool take = k[i] > y.than || (((same >> lane) & 1u) != 0u && static_cast<int>(__popcll(same & below)) < left);
        const uint64_t all = __ballot(take);
        if (take) { out[taken + __popcll(all & below)] = first + (wave * R + i) * 64 + lane; }
        taken += static_cast<int>(__popcll(all));
        left = max(0, left - static_cast<int>(__popcll(same)));
    }
    return min(there, want);
}

template <int WAVES>
__device__ __forceinline__ int choose(const uint32_t* of, int count, int want, int first, int32_t* out, int lane, int wave, Shared& sh) {
    const int r = (count + 64 * WAVES - 1) / (64 * WAVES);
    if constexpr (WAVES > 1) { // (a wave alone has more keys)
        if (r <= 1) { return choose<1, WAVES>(of, count, want, first, out, lane, wave, sh); }
        if (r <= 2) { return choose<2, WAVES>(of, count, want, first, out, lane, wave, sh); }
        if (r <= 4) { return choose<4, WAVES>(of, count, want, first, out, lane, wave, sh); }
        if (r <= 8) { return choose<8, WAVES>(of, count, want, first, out, lane, wave, sh); }
    }
    if (r <= 16) { return choose<16, WAVES>(of, count, want, first, out, lane, wave, sh); }
    if (WAVES == 1 || r <= 32) { return choose<32, WAVES>(of, count, want, first, out, lane, wave, sh); }
    return choose<64, WAVES>(of, count, want, first, out, lane, wave, sh);
}

// ---- four tokens of a wave, one a row of 16 lanes

template <typename F>
__device__ __forceinline__ uint32_t row_all(uint32_t v, F op) {
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xf, 0xf, true)));  // lane ^ 1
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xf, 0xf, true)));  // lane ^ 2
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xf, 0xf, true))); // the other four of eight
    return op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x140, 0xf, 0xf, true)));
}

__device__ __forceinline__ int row_sum(int v) {
    return static_cast<int>(row_all(static_cast<uint32_t>(v), [](uint32_t a, uint32_t b) { return a + b; }));
}

__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    return row_all(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// As `choose`, for the token of the lane's row of 16, with R keys a lane: every row has its own interval, and the wave goes on until
// the last one's is closed.
template <int R>
__device__ __forceinline__ int choose_rows(const uint32_t* of, int count, int want, int first, int32_t* out, int lane) {
    const int li = lane & 15;
    asm("" : "+v"(want)); // in a vector register: as a scalar it is spilled and read back at every use
    uint32_t k[R];
    uint32_t most = 0u, least = 0u; // least as its complement
    int there = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        k[i] = 16 * i + li < count ? of[16 * i + li] : 0u;
        there += k[i] != 0u ? 1 : 0;
        most = max(most, k[i]);
        least = max(least, k[i] != 0u ? ~k[i] : 0u);
    }
    there = row_sum(there);
    uint32_t lo = ~row_max(least), hi = row_max(most), than = 0u;
    bool open = there > want;
    float over = static_cast<float>(there - want), under = static_cast<float>(want);
    int side = 0;
#pragma unroll 1
    for (int step = 0; __any(open); ++step) {
        uint32_t mid = lo + (hi - lo) / 2 + 1;
        if (step < 12) {
            const float a = value_of(lo), b = value_of(hi);
            const float share = fminf(0.984375f, fmaxf(0.015625f, over * __builtin_amdgcn_rcpf(over + under)));
            const float v = a + (b - a) * share;
            const uint32_t between = ordered(v); // lo < between < hi where a < v < b (not so for infinite ends)
            mid = ((v > a) & (v < b)) ? between : mid;
        }
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) { n += k[i] >= mid ? 1 : 0; }
        n = row_sum(n);
        // as in top_keys, without branches; a row whose interval has closed stays as it is
        const int d = n - want;
        const float f = static_cast<float>(d);
        const float fewer_under = under * (side > 0 ? 0.5f : 1.0f), fewer_over = over * (side < 0 ? 0.5f : 1.0f);
        const uint32_t low = mid - 1u, closed = lo >= hi ? lo : low;
        const bool met = (d == 0) | (lo >= hi);
        than = (open & met) ? closed : than;
        open = open & !met;
        lo = (open & (d > 0)) ? mid : lo;
        hi = (open & (d < 0)) ? low : hi;
        under = d > 0 ? fewer_under : -f;
        over = d > 0 ? f : fewer_over;
        side = d > 0 ? 1 : -1;
    }
    int above = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) { above += k[i] > than ? 1 : 0; }
    int left = there > want ? want - row_sum(above) : 0; // how many of those that equal it
    int taken = 0;
    const int row = lane & 48;
    const uint32_t below = (1u << li) - 1u;
    const auto of_row = [&](bool v) { return static_cast<uint32_t>(__ballot(v) >> row) & 0xffffu; };
    if (!__any(left > 0)) { // no choice among equals
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool take = k[i] > than;
            const uint32_t all = of_row(take);
            if (take) { out[taken + __popc(all & below)] = first + 16 * i + li; }
            taken += __popc(all);
        }
        return min(there, want);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const bool equal = k[i] == than && k[i] != 0u;
        const uint32_t same = of_row(equal);
        const bool take = k[i] > than || (equal && static_cast<int>(__popc(same & below)) < left);
        const uint32_t all = of_row(take);
        if (take) { out[taken + __popc(all & below)] = first + 16 * i + li; }
        taken += __popc(all);
        left = max(0, left - static_cast<int>(__popc(same)));
    }
    return min(there, want);
}

// Up to as many keys as 64 registers a lane hold. A wave per token takes longer: 2,048 tokens at 40/8/128 over 60, 250, 500, 750 and 1,000
// blocks 17.6, 24.8, 35.4, 66.3 and 75.2 us so, 12.3, 19.7, 29.7, 49.9 and 64.4 us with rows.
constexpr int kRowKeys = 1024;

__device__ __forceinline__ int choose_rows(const uint32_t* of, int count, int most, int want, int first, int32_t* out, int lane) {
    const int r = (most + 15) / 16;
    if (r <= 4) { return choose_rows<4>(of, count, want, first, out, lane); }
    if (r <= 8) { return choose_rows<8>(of, count, want, first, out, lane); }
    if (r <= 12) { return choose_rows<12>(of, count, want, first, out, lane); }
    if (r <= 16) { return choose_rows<16>(of, count, want, first, out, lane); }
    if (r <= 20) { return choose_rows<20>(of, count, want, first, out, lane); }
    if (r <= 24) { return choose_rows<24>(of, count, want, first, out, lane); }
    if (r <= 32) { return choose_rows<32>(of, count, want, first, out, lane); }
    if (r <= 48) { return choose_rows<48>(of, count, want, first, out, lane); }
    return choose_rows<64>(of, count, want, first, out, lane);
}

// NW: 4 for tiles of 16 tokens (a wave chooses for four of them, or for one, of at most 2,048 keys), 8 for smaller ones (all waves for
// one). 32 single tokens over up to 2,001 blocks: 22.8 us, without the guess 23.2; with 16 waves 27.4 (barriers), with one wave choosing 39.7; 4,096 tokens
// over up to 320 blocks 37.5 us.
template <int D, int NW>
__global__ __launch_bounds__(64 * NW) void block_select_kernel(SelectArgs x) {
    constexpr int L = D / 8;
    constexpr int PAD = 16;
    extern __shared__ uint32_t keys[]; // [tile token][cap]
    __shared__ __attribute__((aligned(16))) char qcode[16 * (D + PAD)];
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % x.c.Hkv;
    const int bs = x.b.shift;
    const int tt = 1 << x.tile_shift;
    const Found f = find_unit(x.c.B, blockIdx.x / x.c.Hkv, lane, [&](int b) { return span_of(x.a.starts, x.a.history, b, x.a.tokens); }, [&](const Span& s) {
        // a sequence outside the envelope takes no part
        return s.tokens <= x.a.max_new && static_cast<int64_t>(s.history) + s.tokens <= x.a.max_keys ? (s.tokens + tt - 1) >> x.tile_shift : 0;
    });
    if (f.b < 0) { return; }
    const int t0 = f.at << x.tile_shift;
    const int tokens = min(tt, f.s.tokens - t0);
    const int pos0 = f.s.history + t0;
    const int first = x.a.first, local = x.a.local;
    // candidates of the tile's last token: blocks first .. last
    const int last = ((pos0 + tokens - 1) >> bs) - local;

    // ---- the first blocks' codes, on their way while the query's are made
    const int c = lane & 15, g = lane >> 4;
    const int per = x.c.page_shift - bs; // log2(blocks of a page)
    const int32_t* table = x.c.table + f.b * x.c.table_row;
    const int from = first & ~15;
    constexpr int AHEAD = NW == 4 ? 2 : 4; // sets of 16 blocks on their way
    constexpr int STEP = 16 * NW * AHEAD;
    struct Pages {
        int32_t page[AHEAD];
    };
    struct Codes {
        int32_t page[AHEAD];
        i4 k[AHEAD][D / 64];
        float scale[AHEAD];
    };
    const auto load_pages = [&](int b0, Pages& p) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int blk = b0 + 16 * NW * u + c;
            p.page[u] = -1;
            if (blk >= first && blk <= last && (blk >> per) < x.c.max_pages) { p.page[u] = table[blk >> per]; }
        }
    };
    const auto load_codes = [&](int b0, const Pages& p, Codes& y) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int blk = b0 + 16 * NW * u + c;
            const int32_t page = p.page[u] >= 0 && p.page[u] < x.c.pages ? p.page[u] : -1;
            const int64_t slot = (static_cast<int64_t>(h) << per) + (blk & ((1 << per) - 1));
            y.page[u] = page;
            y.scale[u] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) { y.k[u][i] = i4{0, 0, 0, 0}; }
            if (page >= 0) {
                const char* src = x.b.codes + page * x.b.code_page + slot * D + 16 * g;
#pragma unroll
                for (int i = 0; i < D / 64; ++i) { y.k[u][i] = *reinterpret_cast<const i4*>(src + 64 * i); }
                y.scale[u] = *reinterpret_cast<const float*>(x.b.scales + page * x.b.scale_page + slot * 4);
            }
        }
    };
    int b0 = from + 16 * wave;
    Pages ids;
    Codes now, then;
    load_pages(b0, ids);
    load_codes(b0, ids, now);
    load_pages(b0 + STEP, ids);

    // ---- query codes
    for (int i = threadIdx.x; i < 16 * (D + PAD) / 16; i += 64 * NW) { reinterpret_cast<u4*>(qcode)[i] = u4{0u, 0u, 0u, 0u}; }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * L; i += 64 * NW) {
        const int t = i / L, li = i & (L - 1);
        const char* src = x.a.q.data + static_cast<int64_t>(f.s.start + t0 + t) * x.a.q.token_stride + (h * x.G * D + 8 * li) * 2;
        double sum[8] = {};
        for (int g0 = 0; g0 < x.G; g0 += 8) {
            i4 raw[8]; // eight heads on their way
#pragma unroll
            for (int g = 0; g < 8; ++g) { raw[g] = g0 + g < x.G ? *reinterpret_cast<const i4*>(src + (g0 + g) * (D * 2)) : i4{0, 0, 0, 0}; }
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                if (g0 + g >= x.G) { break; }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t w = static_cast<uint32_t>(raw[g][e >> 1]);
                    sum[e] += __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
                }
            }
        }
        const double amax = head_amax<D>(sum);
        *reinterpret_cast<i2*>(qcode + t * (D + PAD) + 8 * li) = codes_of(sum, amax, amax * kStep);
    }
    __syncthreads();

    // ---- scores
    i4 q[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) { q[i] = *reinterpret_cast<const i4*>(qcode + c * (D + PAD) + 64 * i + 16 * g); }
    constexpr bool FULL = NW == 4; // tiles of 16 tokens
    int lasts[4];                  // of tokens 4 g .. 4 g + 3: the last block to choose
    uint32_t* to = keys + 4 * g * x.cap + c - from;
#pragma unroll
    for (int r = 0; r < 4; ++r) { lasts[r] = ((pos0 + 4 * g + r) >> bs) - local; }
#pragma unroll 1
    for (; b0 <= last; b0 += STEP) {
        load_codes(b0 + STEP, ids, then);
        load_pages(b0 + 2 * STEP, ids);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int blk = b0 + 16 * NW * u + c;
            if (blk - c > last) { continue; }
            i4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < D / 64; ++i) { acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[i], now.k[u][i], acc, 0, 0, 0); }
#pragma unroll
            for (int r = 0; r < 4; ++r) { // token 4 g + r, block c
                const float score = now.scale[u] * static_cast<float>(acc[r]);
                const uint32_t key = now.scale[u] == INFINITY ? 0xff800000u : ordered(score);
                if (FULL || 4 * g + r < tt) { to[r * x.cap + blk - c] = now.page[u] >= 0 && blk <= lasts[r] ? key : 0u; }
            }
        }
        now = then;
    }
    __syncthreads();

    // ---- lists
    const int S = first + local + x.a.top;
    constexpr int TOGETHER = NW == 4 ? 1 : NW; // waves of a token
    const auto ends = [&](int32_t* out, int own, int heads, int tail, int taken, int at, int lanes) {
        for (int i = at; i < heads; i += lanes) { out[i] = i; }
        for (int i = tail + at; i <= own; i += lanes) { out[taken + i - tail] = i; }
        for (int i = taken + own - tail + 1 + at; i < S; i += lanes) { out[i] = -1; }
    };
    if constexpr (NW == 4) {
        const int most = last - first + 1;
        if (most <= kRowKeys) {
            const int t = 4 * wave + (lane >> 4);
            const bool there = t < tokens;
            const int own = there ? (pos0 + t) >> bs : -1; // no block, no candidate
            int32_t* out = x.a.selected + (static_cast<int64_t>(f.s.start + t0 + (there ? t : 0)) * x.c.Hkv + h) * S;
            const int heads = min(first, own + 1);
            const int tail = max(heads, own - local + 1);
            const int count = there && x.a.top > 0 ? max(0, own - local - first + 1) : 0;
            const int taken = heads + choose_rows(keys + t * x.cap + (first - from), count, most, x.a.top, first, out + heads, lane);
            if (there) { ends(out, own, heads, tail, taken, lane & 15, 16); }
            return;
        }
    }
    for (int t = NW == 4 ? wave : 0; t < tokens; t += NW / TOGETHER) {
        const int own = (pos0 + t) >> bs;
        const int64_t token = f.s.start + t0 + t;
        int32_t* out = x.a.selected + (token * x.c.Hkv + h) * S;
        const int part = TOGETHER == 1 ? 0 : wave;
        const int heads = min(first, own + 1);        // the first blocks
        const int tail = max(heads, own - local + 1); // the last ones: tail .. own
        const int count = own - local - first + 1;    // blocks between
        int taken = heads;
        if (x.a.top > 0 && count > 0) {
            taken += choose<TOGETHER>(keys + t * x.cap + (first - from), count, x.a.top, first, out + heads, lane, part, sh);
        }
        if (part == 0) { ends(out, own, heads, tail, taken, lane, 64); }
    }
}

template <int D>
void select(const SelectArgs& x, int64_t tiles, hipStream_t stream) {
    const size_t lds = (static_cast<size_t>(x.cap) << x.tile_shift) * 4;
    const int64_t grid = tiles * x.c.Hkv;
    if (grid > 0x3FFFFF) { throw Unsupported("paged block selection: more than 2^22 workgroups are not built"); }
    if (x.tile_shift == 4) {
        hipLaunchKernelGGL((block_select_kernel<D, 4>), dim3(static_cast<uint32_t>(grid)), dim3(256), lds, stream, x);
    } else {
        hipLaunchKernelGGL((block_select_kernel<D, 8>), dim3(static_cast<uint32_t>(grid)), dim3(512), lds, stream, x);
    }
    check_launch("block_select_kernel");
}

} // namespace

void launch_block_update(int64_t tokens, const int32_t* starts, const int32_t* history, const PagedRef& c, const BlocksRef& b, hipStream_t stream) {
    // a sequence's new rows touch at most tokens / rows + 2 blocks
    const int64_t units = ((tokens >> b.shift) + 2 * static_cast<int64_t>(c.B)) * c.Hkv;
    const UpdateArgs x{tokens, starts, history, c, b, units};
    const int64_t grid = (units + 3) / 4;
    if (grid > 0x7FFFFF) { throw Unsupported("paged block update: more than 2^23 workgroups are not built"); }
    const dim3 blocks(static_cast<uint32_t>(grid));
    if (c.D == 128 && c.bf16) {
        hipLaunchKernelGGL((block_update_kernel<128, true>), blocks, dim3(256), 0, stream, x);
    } else if (c.D == 128) {
        hipLaunchKernelGGL((block_update_kernel<128, false>), blocks, dim3(256), 0, stream, x);
    } else if (c.bf16) {
        hipLaunchKernelGGL((block_update_kernel<256, true>), blocks, dim3(256), 0, stream, x);
    } else {
        hipLaunchKernelGGL((block_update_kernel<256, false>), blocks, dim3(256), 0, stream, x);
    }
    check_launch("block_update_kernel");
}

// The scores of a tile fit the LDS, so the call needs none.
size_t block_select_bytes(int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

void launch_block_select(const BlockSelect& a, const PagedRef& c, const BlocksRef& b, void*, hipStream_t stream) {
    SelectArgs x{};
    x.a = a;
    x.c = c;
    x.b = b;
    x.G = a.Hq / c.Hkv;
    const int32_t blocks = ((a.max_keys + (1 << b.shift) - 1) >> b.shift);
    x.cap = (blocks + 31) & ~15; // a tile's keys begin at a multiple of 16
    // as many tokens of a tile as its keys leave room for in 128 KiB, no more than a sequence may have
    x.tile_shift = 4;
    while (x.tile_shift > 0 && ((static_cast<int64_t>(x.cap) << x.tile_shift) > 32768 || (1 << (x.tile_shift - 1)) >= a.max_new)) { --x.tile_shift; }
    const int64_t tiles = std::min<int64_t>(a.tokens, (a.tokens >> x.tile_shift) + c.B);
    c.D == 128 ? select<128>(x, tiles, stream) : select<256>(x, tiles, stream);
}

} // namespace nmi
