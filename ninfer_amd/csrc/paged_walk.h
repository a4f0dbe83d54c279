// What the kernels over a paged KV cache share: the call's arguments, and a wave's walk over 32 keys at a time straight
// from the cache (scores, probabilities with a running maximum and sum, products with the values) for 16 or 32 query rows.
// The mathematics and its roundings stand in paged_attention.hip.
#pragma once

#include "attn_math.h"
#include "common.h"
#include "device_utils.h"
#include "lds_dma.h"
#include "paged_internal.h"

#include <type_traits>

namespace nmi {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct PagedAttnArgs {
    PagedAttention a;
    PagedRef c;
    int32_t G;
    float scale_log2;
    int32_t few_rows;  // sequences with at most this many rows (tokens x G) are the few-row kernel's
    int32_t slots;     // its workgroups per KV head
    float* part_o;     // FP32 O [partial row][D] and (log2-domain maximum, sum) [partial row][2]
    float* part_ml;
    int32_t* seq_table; // per sequence: first slot, parts
    int32_t many_parts; // parts that the many-row workgroups' splits may have (0: none), and those as above
    float* many_o;
    float* many_ml;
};

// Sequence b's tokens and history, checked against the call's bounds: a sequence outside them takes no part.
struct Seq {
    int32_t start;
    int32_t tokens;
    int32_t history;
};

__device__ __forceinline__ Seq checked(const PagedAttnArgs& x, int32_t start, int32_t end, int32_t history) {
    const bool ok = start >= 0 && end >= start && end <= x.a.tokens && end - start <= x.a.max_new && history >= 0 &&
                    static_cast<int64_t>(history) + (end - start) <= x.a.max_keys;
    return Seq{start, ok ? end - start : 0, history};
}

__device__ __forceinline__ Seq sequence(const PagedAttnArgs& x, int b) { return checked(x, x.a.starts[b], x.a.starts[b + 1], x.a.history[b]); }

// Lane `at`'s sequence, for the whole wave.
__device__ __forceinline__ Seq lane_seq(const Seq& s, int at) {
    return Seq{__builtin_amdgcn_readlane(s.start, at), __builtin_amdgcn_readlane(s.tokens, at), __builtin_amdgcn_readlane(s.history, at)};
}

// The tiles (of 2^lg keys) that tokens at positions p0 .. p1 need: [0, sink) and [first, end) of the sequence's tiles,
// numbered on without the gap.
struct Tiles {
    int32_t sink;
    int32_t first;
    int32_t count;
    __device__ __forceinline__ int32_t tile(int32_t i) const { return i < sink ? i : i - sink + first; }
};

__device__ __forceinline__ Tiles tiles_of(const PagedAttnArgs& x, int32_t p0, int32_t p1, int lg) {
    const int32_t first = max(0, p0 + 1 - x.a.window);
    Tiles t{(min(x.a.sinks, first) + (1 << lg) - 1) >> lg, first >> lg, 0};
    if (t.sink >= t.first) { t.sink = t.first = 0; }
    t.count = t.sink + (p1 >> lg) + 1 - t.first;
    return t;
}

// The weights of two parts of a row, log2-domain maxima and sums M, L and m, l, in their merge. A part that saw nothing
// weighs nothing, one whose sum is NaN stays NaN.
struct Weights {
    float M, a, b;
};

__device__ __forceinline__ Weights weights(float M, float L, float m, float l) {
    Weights w;
    w.M = fmaxf(M, m);
    w.a = M == -INFINITY ? (L == L ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(M - w.M);
    w.b = m == -INFINITY ? (l == l ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - w.M);
    return w;
}

// Four outputs O / L as BF16, zero where the sum is.
__device__ __forceinline__ u2 out_pair(f4 O, float L) {
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { y[e] = f32_to_bf16_bits(L == 0.0f ? 0.0f : O[e] * inv); }
    return u2{y[0] | (y[1] << 16), y[2] | (y[3] << 16)};
}

// ---- one wave: 16 NT query rows against 32 keys straight from the cache -------------------------
//
// S^T = K Q^T and O^T = V^T P^T on 16x16x32 MFMAs. Lane (c, g) = (lane & 15, lane >> 4) loads row c of each half
// tile's K in 16-byte pieces (piece i of a quarter g: the MFMA steps run over the dims in the order the pieces leave
// them, and Q follows), and four bytes (INT8; BF16: sixteen) of the V rows 4g .. 4g + 3 of both halves, the keys
// whose scores the S^T accumulator leaves in this lane; so P needs no exchange between lanes, and V is transposed
// by byte selects alone. No LDS in the loop.
//
// What bounds it: HBM (31 flop a byte with INT8 rows and one row tile); the VALU converts and weighs 60% of the
// time. Measured on MI355X: 32 single tokens over 535,000 ragged rows at 40/8/128 INT8 208 us (5.4 TB/s), 4 tokens over
// 131,004 rows at 24/4/256 BF16 99 us (5.4 TB/s).

template <int D, bool BF>
struct Chunk {
    static constexpr int KP = BF ? D / 32 : D / 64; // K pieces of a lane and half
    static constexpr int VP = BF ? D / 128 : D / 64; // V pieces of a lane and key
    static constexpr int VW = BF ? 4 : 1;            // words of a V piece
    static constexpr int SW = BF ? 1 : D / 128;      // 16-byte words of four keys' scales
};

template <int D, bool BF>
struct ChunkK {
    u4 k[2][Chunk<D, BF>::KP];
    u4 ks[2][Chunk<D, BF>::SW];
};

template <int D, bool BF>
struct ChunkV {
    uint32_t v[8][Chunk<D, BF>::VP][Chunk<D, BF>::VW];
    u4 vs[2][Chunk<D, BF>::SW];
};

// What a chunk's loads are aimed at: the 16-row halves' pages (-1: none).
struct Halves {
    int32_t page[2];
};

// One plane's rows of a half tile as a buffer; an absent half is a buffer of no bytes, whose loads give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t half_rows(const PagedAttnArgs& x, const char* plane, int64_t page_stride, int bytes, int h, int tile,
                                                           int kt, Halves hv) {
    const bool there = hv.page[kt] >= 0;
    const int64_t page = there ? hv.page[kt] : 0;
    const int64_t row = (static_cast<int64_t>(h) << x.c.page_shift) + ((32 * tile + 16 * kt) & ((1 << x.c.page_shift) - 1));
    return raw_buffer(plane + page * page_stride + row * bytes, there ? 16 * bytes : 0);
}

constexpr int kOnce = 2; // cache policy of rows that a call reads once (non-temporal)

template <int D, bool BF>
__device__ __forceinline__ void load_keys(const PagedAttnArgs& x, int h, int tile, Halves hv, int c, int g, ChunkK<D, BF>& r) {
    using CK = Chunk<D, BF>;
    constexpr int kRow = BF ? 2 * D : D;
    constexpr int kScaleRow = D / 32; // bytes of a row's scales
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        const __amdgpu_buffer_rsrc_t kb = half_rows(x, x.c.k, x.c.k_page, kRow, h, tile, kt, hv);
#pragma unroll
        for (int i = 0; i < CK::KP; ++i) {
            r.k[kt][i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(kb, c * kRow + 64 * i + 16 * g, 0, kOnce));
        }
        if constexpr (!BF) {
            const __amdgpu_buffer_rsrc_t ksb = half_rows(x, x.c.ks, x.c.ks_page, kScaleRow, h, tile, kt, hv);
#pragma unroll
            for (int w = 0; w < CK::SW; ++w) {
                r.ks[kt][w] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(ksb, 4 * g * kScaleRow + 16 * w, 0, 0));
            }
        }
    }
}

template <int D, bool BF>
__device__ __forceinline__ void load_values(const PagedAttnArgs& x, int h, int tile, Halves hv, int c, int g, ChunkV<D, BF>& r) {
    using CK = Chunk<D, BF>;
    constexpr int kRow = BF ? 2 * D : D;
    constexpr int kScaleRow = D / 32;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        if constexpr (!BF) {
            const __amdgpu_buffer_rsrc_t vsb = half_rows(x, x.c.vs, x.c.vs_page, kScaleRow, h, tile, kt, hv);
#pragma unroll
            for (int w = 0; w < CK::SW; ++w) {
                r.vs[kt][w] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vsb, 4 * g * kScaleRow + 16 * w, 0, 0));
            }
        }
        const __amdgpu_buffer_rsrc_t vb = half_rows(x, x.c.v, x.c.v_page, kRow, h, tile, kt, hv);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < CK::VP; ++i) {
                if constexpr (BF) {
                    const u4 w = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vb, (4 * g + j) * kRow + 256 * i + 16 * c, 0, kOnce));
#pragma unroll
                    for (int e = 0; e < 4; ++e) { r.v[4 * kt + j][i][e] = w[e]; }
                } else {
                    r.v[4 * kt + j][i][0] = __builtin_amdgcn_raw_buffer_load_b32(vb, (4 * g + j) * kRow + 64 * i + 4 * c, 0, kOnce);
                }
            }
        }
    }
}

// Two INT8 codes, bytes B0 of `lo` and B1 of `hi`, as exact FP16 values: 0x6400 | (code + 128) is 1152 + code.
template <int B0, int B1>
__device__ __forceinline__ uint32_t codes2(uint32_t lo, uint32_t hi) {
    const uint32_t x = __builtin_amdgcn_perm(hi, lo, 0x0c000c00u | (static_cast<uint32_t>(4 + B1) << 16) | static_cast<uint32_t>(B0));
    const h2 y = __builtin_bit_cast(h2, x ^ 0x64806480u) - h2{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    return __builtin_bit_cast(uint32_t, y);
}

__device__ __forceinline__ h8 codes8(uint32_t a, uint32_t b) {
    const u4 w = {codes2<0, 1>(a, a), codes2<2, 3>(a, a), codes2<0, 1>(b, b), codes2<2, 3>(b, b)};
    return __builtin_bit_cast(h8, w);
}

// The FP16 scale of key e (0..3) of a half's four, group i, from its loaded words.
template <int D>
__device__ __forceinline__ float scale_of(const u4 (&w)[D / 128], int e, int i) {
    const int half = e * (D / 64) + i;
    const uint32_t x = w[half >> 3][(half >> 1) & 3];
    return f16_bits_to_f32(static_cast<uint16_t>((half & 1) ? x >> 16 : x & 0xffffu));
}

constexpr float kLargest = 3.4028234663852886e38f;

// Online-softmax state of a wave's rows 16 nt + c.
template <int D, bool BF, int NT>
struct Rows {
    u4 q[NT][D / 32];  // B operand of Q^T, dims in the K pieces' order
    float rowmul[NT];  // raw score -> log2 domain
    int pos[NT];       // the row's position (-1: no row)
    float m[NT];       // running maximum of the raw scores
    float l[NT];       // this lane's part of the sum
    f4 O[NT][D / 16];  // O^T tile t, entry e' of lane (c, g): dim out_dim(t, 4 g + e') of row 16 nt + c
    int lo, hi;        // first and last position of the wave's rows
};

// MFMA row m of O^T tile t is this dim.
template <bool BF>
__device__ __forceinline__ constexpr int out_dim(int t, int m) {
    return BF ? 128 * (t >> 3) + 8 * m + (t & 7) : 64 * (t >> 2) + 4 * m + (t & 3);
}

// Row tile nt's row of the lane: its query from `src` (a row without one: zeros) and its empty state.
template <int D, bool BF, int NT>
__device__ __forceinline__ void init_row(const PagedAttnArgs& x, const uint16_t* src, bool valid, int nt, int g, Rows<D, BF, NT>& r) {
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
        // INT8: step 2 i + j holds dims 64 i + 16 g + 8 j ..; BF16: step i dims 32 i + 8 g ..
        const int dim = BF ? 32 * k + 8 * g : 64 * (k >> 1) + 16 * g + 8 * (k & 1);
        r.q[nt][k] = valid ? *reinterpret_cast<const u4*>(src + dim) : u4{0u, 0u, 0u, 0u};
    }
    if constexpr (BF) {
        r.rowmul[nt] = x.scale_log2;
    } else {
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(r.q[nt][k][w] << 16)), fabsf(__uint_as_float(r.q[nt][k][w] & 0xffff0000u))));
            }
        }
        amax = group4_max(amax);
        int fexp = 0; // amax * 2^fexp in [2^14, 2^15): what FP16 then rounds is below 2^-39 of amax
        if (amax > 0.0f && amax < INFINITY) { fexp = 14 - max(static_cast<int>((__float_as_uint(amax) >> 23) & 0xff) - 127, -46); }
        const float factor = ldexpf(1.0f, fexp);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t y = r.q[nt][k][w];
                const h2 p = {static_cast<_Float16>(__uint_as_float(y << 16) * factor),
                              static_cast<_Float16>(__uint_as_float(y & 0xffff0000u) * factor)};
                r.q[nt][k][w] = __builtin_bit_cast(uint32_t, p);
            }
        }
        r.rowmul[nt] = fminf(ldexpf(x.scale_log2, -fexp), kLargest); // finite: a score of zero stays one
    }
    r.m[nt] = -INFINITY;
    r.l[nt] = 0.0f;
#pragma unroll
    for (int t16 = 0; t16 < D / 16; ++t16) { r.O[nt][t16] = f4{0.f, 0.f, 0.f, 0.f}; }
}

// Rows row0 .. of the sequence's, token after token.
template <int D, bool BF, int NT>
__device__ __forceinline__ void init_rows(const PagedAttnArgs& x, const Seq& s, int h, int row0, int c, int g, Rows<D, BF, NT>& r) {
    const int rows = s.tokens * x.G;
    r.lo = 0x7fffffff;
    r.hi = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + 16 * nt + c;
        const bool valid = row < rows;
        const int t = valid ? row / x.G : 0;
        const int head = h * x.G + (valid ? row - t * x.G : 0);
        r.pos[nt] = valid ? s.history + t : -1;
        init_row<D, BF, NT>(x, reinterpret_cast<const uint16_t*>(x.a.q.data + (s.start + t) * x.a.q.token_stride) + head * D, valid, nt, g, r);
    }
    if (row0 < rows) {
        r.lo = s.history + row0 / x.G;
        r.hi = s.history + (min(row0 + 16 * NT, rows) - 1) / x.G;
    }
}

// Whether a token at `pos` sees row `key` of page `page`: no row of an absent page (negative), nor from pos -1.
__device__ __forceinline__ bool sees(const PagedAttnArgs& x, int pos, int key, int page) {
    return (key <= (pos | (page >> 31))) & ((pos - key < x.a.window) | (key < x.a.sinks));
}

// Whether every row of the wave sees all 32 keys of the tile.
__device__ __forceinline__ bool all_seen(const PagedAttnArgs& x, int lo, int hi, int tile, Halves hv) {
    const int k0 = 32 * tile, k1 = k0 + 31;
    return (hv.page[0] | hv.page[1]) >= 0 && k1 <= lo && (hi - k0 < x.a.window || k1 < x.a.sinks);
}

// An infinite or NaN BF16 in either half of a word: that half's sign bit (of the result) set.
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// A chunk's probabilities (times 2^kPOffset), and which of its keys a lane's rows see.
template <int NT>
struct Probs {
    float p[NT][8];
    uint32_t seen[NT]; // bit i: row nt's lane sees key i
    bool whole;        // every row sees every key
};

template <int D, bool BF, int NT>
__device__ __forceinline__ void chunk_probs(const PagedAttnArgs& x, int tile, Halves hv, int g, const ChunkK<D, BF>& r, Rows<D, BF, NT>& s, Probs<NT>& y) {
    using CK = Chunk<D, BF>;
    const bool whole = all_seen(x, s.lo, s.hi, tile, hv);
    float sv[NT][8];
    // ---- scores
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if constexpr (BF) {
                f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < CK::KP; ++i) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, r.k[kt][i]), __builtin_bit_cast(bf8, s.q[nt][i]), acc, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) { sv[nt][4 * kt + e] = acc[e]; }
            } else {
#pragma unroll
                for (int i = 0; i < CK::KP; ++i) {
                    const u4 w = r.k[kt][i];
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(w[0], w[1]), __builtin_bit_cast(h8, s.q[nt][2 * i]), acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(w[2], w[3]), __builtin_bit_cast(h8, s.q[nt][2 * i + 1]), acc, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float sc = scale_of<D>(r.ks[kt], e, i);
                        sv[nt][4 * kt + e] = i == 0 ? acc[e] * sc : fmaf(acc[e], sc, sv[nt][4 * kt + e]);
                    }
                }
            }
        }
    }
    y.whole = whole;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { y.seen[nt] = 0xffu; }
    if (!whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            y.seen[nt] = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool ok = sees(x, s.pos[nt], 32 * tile + 16 * (i >> 2) + 4 * g + (i & 3), hv.page[i >> 2]);
                y.seen[nt] |= ok ? 1u << i : 0u;
                sv[nt][i] = ok ? sv[nt][i] : -INFINITY;
            }
        }
    }
    // ---- running maximum (it moves only when a score tops it by 2^kLazyTau), probabilities, sums
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float cmax = score_max(sv[nt]);
        const bool need = (cmax - s.m[nt]) * s.rowmul[nt] > kLazyTau;
        if (__any(need)) {
            const float mn = need ? cmax : s.m[nt];
            const float alpha = need ? __builtin_amdgcn_exp2f((s.m[nt] - mn) * s.rowmul[nt]) : 1.0f;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) { s.O[nt][t] *= alpha; }
            s.l[nt] *= alpha;
            s.m[nt] = mn;
        }
        const float ref = s.m[nt] == -INFINITY ? 0.0f : s.m[nt];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // the difference first: -m * rowmul rounded would move every p by up to 2^(score 2^-25)
            y.p[nt][i] = __builtin_amdgcn_exp2f(fmaf(sv[nt][i] - ref, s.rowmul[nt], kPOffset));
        }
        const float(&p)[8] = y.p[nt];
        s.l[nt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    }
}

// The careful products' weights are p * down. A sum of 2^23 weights, each up to 2^15, times values below 2^80 stays finite; where
// there are larger ones `down` is 2^-40, which keeps sums of BF16's largest value finite (values below 2^-78 lose bits that way,
// so not everywhere).
constexpr uint32_t kCareTop = static_cast<uint32_t>(127 + 80) << 23; // 2^80
constexpr float kCareDown = 0x1p-40f;

// The (log2-domain maximum, sum) of a state whose outputs were made by the lower weights.
__device__ __forceinline__ void care_units(float& M, float& L) {
    M += 40.0f;
    L *= kCareDown;
}

// Tile `tile`'s pages; rows past `last` need none.
__device__ __forceinline__ Halves halves_of(const PagedAttnArgs& x, const int32_t* table, int tile, int last) {
    Halves hv;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        const int key = 32 * tile + 16 * kt;
        const int pg = key <= last ? table[key >> x.c.page_shift] : -1;
        hv.page[kt] = __builtin_amdgcn_readfirstlane(pg >= 0 && pg < x.c.pages ? pg : -1);
    }
    return hv;
}

// A word of two BF16 values with zeros for infinite and NaN ones, and the bits of the larger one's magnitude.
__device__ __forceinline__ uint32_t finite_word(uint32_t x) { return x & ~((nonfinite_bits(x) >> 15) * 0xffffu); }
__device__ __forceinline__ uint32_t larger_bits(uint32_t x) { return max(x & 0x7fff0000u, (x << 16) & 0x7fff0000u); }

// O^T += V^T P^T. CARE (BF16): infinite and NaN values reach only the rows that see them, finite ones overflow no sum; without
// it they may make any row of the wave NaN. `large`: the bits of the largest finite value so far (CARE).
template <int D, bool BF, int NT, bool CARE>
__device__ __forceinline__ void chunk_values(int tile, Halves hv, int g, const Probs<NT>& y, ChunkV<D, BF>& r, Rows<D, BF, NT>& s, float down, uint32_t& large) {
    using CK = Chunk<D, BF>;
    const float(&p)[NT][8] = y.p;
    if (!y.whole) {
        if constexpr (BF) {
            // keys that no row of the wave may see: whatever their rows hold is taken out
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool dead = 32 * tile + 16 * (i >> 2) + 4 * g + (i & 3) > (s.hi | (hv.page[i >> 2] >> 31));
#pragma unroll
                for (int w = 0; w < CK::VP; ++w) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) { r.v[i][w][e] = dead ? 0u : r.v[i][w][e]; }
                }
            }
        }
    }
    if constexpr (!BF) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            float sc[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) { sc[k] = scale_of<D>(r.vs[k >> 2], k & 3, i); }
            h8 w[NT];
            float up[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float z[8];
                float top = 0.0f; // the row's largest weight of the chunk in group i
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    z[k] = p[nt][k] * sc[k];
                    if (!y.whole) { z[k] = ((y.seen[nt] >> k) & 1u) ? z[k] : 0.0f; } // an unseen row's scale may be anything
                    top = fmaxf(top, fabsf(z[k]));
                }
                top = group4_max(top);
                // 2^E > top; next to an infinite scale 2^31, which tops every finite weight (p <= 2^15, FP16 scales)
                const int E = max(-100, min(31, static_cast<int>(__float_as_uint(top) >> 23) - 126));
                const float down = __uint_as_float(static_cast<uint32_t>(127 + 15 - E) << 23);
                up[nt] = __uint_as_float(static_cast<uint32_t>(127 - 15 + E) << 23);
#pragma unroll
                for (int k = 0; k < 8; ++k) { w[nt][k] = static_cast<_Float16>(z[k] * down); }
            }
            const auto tile4 = [&](auto byte) {
                constexpr int Bt = decltype(byte)::value;
                uint32_t va[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) { va[q] = codes2<Bt, Bt>(r.v[2 * q][i][0], r.v[2 * q + 1][i][0]); }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const f4 o = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, va), w[nt], f4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { s.O[nt][4 * i + Bt][e] = fmaf(o[e], up[nt], s.O[nt][4 * i + Bt][e]); }
                }
            };
            tile4(std::integral_constant<int, 0>{});
            tile4(std::integral_constant<int, 1>{});
            tile4(std::integral_constant<int, 2>{});
            tile4(std::integral_constant<int, 3>{});
        }
    } else {
        bf8 hi[NT], lo[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float z = CARE ? p[nt][k] * down : p[nt][k];
                hi[nt][k] = static_cast<__bf16>(z);
                lo[nt][k] = static_cast<__bf16>(z - static_cast<float>(hi[nt][k]));
            }
        }
        if constexpr (CARE) {
            // infinite and NaN values: counted apart (+: infinity or NaN, -: the same with the other sign) for the
            // rows that see them, and left out of the products
            h8 one[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int k = 0; k < 8; ++k) { one[nt][k] = ((y.seen[nt] >> k) & 1u) ? static_cast<_Float16>(1.0f) : static_cast<_Float16>(0.0f); }
            }
#pragma unroll
            for (int i = 0; i < CK::VP; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    __builtin_amdgcn_sched_barrier(0); // one at a time: the registers are full
                    h8 up, dn;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t z = ((e & 1) ? r.v[k][i][e >> 1] >> 16 : r.v[k][i][e >> 1]) & 0xffffu;
                        const bool nan = (z & 0x7fffu) > 0x7f80u;
                        up[k] = nan || z == 0x7f80u ? static_cast<_Float16>(1.0f) : static_cast<_Float16>(0.0f);
                        dn[k] = nan || z == 0xff80u ? static_cast<_Float16>(1.0f) : static_cast<_Float16>(0.0f);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const f4 z = {0.f, 0.f, 0.f, 0.f};
                        const f4 a = __builtin_amdgcn_mfma_f32_16x16x32_f16(up, one[nt], z, 0, 0, 0);
                        const f4 b = __builtin_amdgcn_mfma_f32_16x16x32_f16(dn, one[nt], z, 0, 0, 0);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            if (a[q] > 0.0f) { s.O[nt][8 * i + e][q] += INFINITY; }
                            if (b[q] > 0.0f) { s.O[nt][8 * i + e][q] -= INFINITY; }
                        }
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int i = 0; i < CK::VP; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        r.v[k][i][e] = finite_word(r.v[k][i][e]);
                        large = max(large, larger_bits(r.v[k][i][e]));
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < CK::VP; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                u4 va;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    va[q] = __builtin_amdgcn_perm(r.v[2 * q + 1][i][e >> 1], r.v[2 * q][i][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    f4& o = s.O[nt][8 * i + e];
                    o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, va), hi[nt], o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, va), lo[nt], o, 0, 0, 0);
                }
            }
        }
    }
}

// The states of a workgroup's NW waves into wave 0's: the upper half into the lower one, again and again. M, L: a row's log2-domain
// maximum and sum.
template <int D, bool BF, int NT, int NW>
__device__ __forceinline__ void join_waves(Rows<D, BF, NT>& r, float (&M)[NT], float (&L)[NT], int wave, int lane, f4 (&xo)[NW / 2][NT * (D / 16) * 64],
                                           float2 (&xm)[NW / 2][NT * 64]) {
    const auto halve = [&](int half) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) { xo[wave - half][(nt * (D / 16) + t) * 64 + lane] = r.O[nt][t]; }
                xm[wave - half][nt * 64 + lane] = float2{M[nt], L[nt]};
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float2 o = xm[wave][nt * 64 + lane];
                const Weights wt = weights(M[nt], L[nt], o.x, o.y);
                L[nt] = L[nt] * wt.a + o.y * wt.b;
                M[nt] = wt.M;
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    const f4 y = xo[wave][(nt * (D / 16) + t) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // a part without weight adds nothing, whatever it holds
                        r.O[nt][t][e] = (wt.a == 0.0f ? 0.0f : r.O[nt][t][e] * wt.a) + (wt.b == 0.0f ? 0.0f : y[e] * wt.b);
                    }
                }
            }
        }
    };
    if constexpr (NW == 8) {
        halve(4);
        __syncthreads();
    }
    halve(2);
    __syncthreads();
    halve(1);
}

// Row tile nt's row of the lane (16 nt + c) as part `at` of the workspace.
template <int D, bool BF, int NT>
__device__ __forceinline__ void store_part(const PagedAttnArgs& x, const Rows<D, BF, NT>& r, int nt, float M, float L, int64_t at, int g) {
    constexpr int RUN = BF ? 8 : 4; // consecutive dims of a lane
#pragma unroll
    for (int i = 0; i < D / (16 * RUN); ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float* dst = x.part_o + at * D + out_dim<BF>(RUN * i, 4 * g + e);
#pragma unroll
            for (int k = 0; k < RUN; k += 4) {
                *reinterpret_cast<f4*>(dst + k) = f4{r.O[nt][RUN * i + k][e], r.O[nt][RUN * i + k + 1][e], r.O[nt][RUN * i + k + 2][e], r.O[nt][RUN * i + k + 3][e]};
            }
        }
    }
    if (g == 0) { *reinterpret_cast<float2*>(x.part_ml + 2 * at) = float2{M, L}; }
}

// The same as token `token`'s head `head` of the group in the output.
template <int D, bool BF, int NT>
__device__ __forceinline__ void store_out(const PagedAttnArgs& x, int token, int h, int head, const Rows<D, BF, NT>& r, int nt, float L, int g) {
    constexpr int RUN = BF ? 8 : 4;
    uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + token * x.a.out.token_stride) + (h * x.G + head) * D;
#pragma unroll
    for (int i = 0; i < D / (16 * RUN); ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint16_t* dst = out + out_dim<BF>(RUN * i, 4 * g + e);
#pragma unroll
            for (int k = 0; k < RUN; k += 4) {
                const f4 o = {r.O[nt][RUN * i + k][e], r.O[nt][RUN * i + k + 1][e], r.O[nt][RUN * i + k + 2][e], r.O[nt][RUN * i + k + 3][e]};
                *reinterpret_cast<u2*>(dst + k) = out_pair(o, L);
            }
        }
    }
}

// Parts of a row, joined one after another.
struct Merge {
    float M = -INFINITY, L = 0.0f;
    f4 O = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void add(float m, float l, f4 o) {
        const Weights w = weights(M, L, m, l);
        L = L * w.a + l * w.b;
#pragma unroll
        for (int e = 0; e < 4; ++e) { O[e] = (w.a == 0.0f ? 0.0f : O[e] * w.a) + (w.b == 0.0f ? 0.0f : o[e] * w.b); }
        M = w.M;
    }
};

} // namespace
} // namespace nmi
