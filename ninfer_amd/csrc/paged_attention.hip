// Attention of packed new tokens over a paged KV cache on gfx950.
//
// Mathematics: token i of sequence b stands at position p = history[b] + i and sees the rows j <= p of its
// sequence with p - j < window or j < sinks (every j <= p without a window) whose page exists;
// out = sum_j softmax_j(scale * q . K_j) V_j in one pass with a running maximum and sum, zero where no row is seen.
// The query heads of a KV head are rows of one problem (row r of a sequence: token r / G, head r % G), so each
// cached row is fetched once for all of them.
//
// Numbers: an INT8 code is exact in FP16, and Q is BF16 made FP16 by a power of two per row, so q . code is exact
// up to the FP32 sum; the scale of a key's 64-value group multiplies that sum in FP32. The probabilities take the
// V scales in the same way: w = p * s * 2^-E in FP16 (off by 2^-11 of itself, 2^-39 of the largest at least), times codes,
// times 2^E in FP32. 2^E is the row's own: it tops w of the 32 keys at hand, so no scale is too large or too small,
// and keys that the row does not see or that weigh nothing take no bits from the others. BF16 caches multiply stored
// values; p goes in as two BF16 terms (16 bits). Maxima, sums (of p as it is, before either rounding) and accumulators
// are FP32. The many-row kernel rounds more, to keep the matrix cores fed; what it rounds stands there.
#include "attn_math.h"
#include "common.h"
#include "device_utils.h"
#include "lds_dma.h"
#include "paged_internal.h"

#include <algorithm>
#include <cmath>
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

__device__ __forceinline__ Seq sequence(const PagedAttnArgs& x, int b) {
    Seq s{x.a.starts[b], 0, x.a.history[b]};
    const int32_t end = x.a.starts[b + 1];
    const bool ok = s.start >= 0 && end >= s.start && end <= x.a.tokens && end - s.start <= x.a.max_new && s.history >= 0 &&
                    static_cast<int64_t>(s.history) + (end - s.start) <= x.a.max_keys;
    s.tokens = ok ? end - s.start : 0;
    return s;
}

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
        const uint16_t* src = reinterpret_cast<const uint16_t*>(x.a.q.data + (s.start + t) * x.a.q.token_stride) + head * D;
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

// ---- few rows: splits of the keys over workgroups and waves --------------------------------------

constexpr int kUnit = 4; // tiles of a unit: one for each wave

// The units of sequence b's keys that the few-row kernel walks (0: not its sequence).
__device__ __forceinline__ int few_units(const PagedAttnArgs& x, int b, Seq& s) {
    s = sequence(x, b);
    if (s.tokens == 0 || s.tokens * x.G > x.few_rows) { return 0; }
    const Tiles t = tiles_of(x, s.history, s.history + s.tokens - 1, 5);
    return (t.count + kUnit - 1) / kUnit;
}

// The batch's units in a row, sequence after sequence, are cut into `shares` equal runs, one for a workgroup: no workgroup
// has more than one unit above another, whatever the lengths. A run may end one sequence and begin another: its part of a
// sequence goes to the slot (share + rank of the sequence among those that have units), a number that no other part has.
struct FewPlan {
    int total;  // units
    int shares;
    __device__ __forceinline__ int begin(int share) const { return static_cast<int>(static_cast<int64_t>(share) * total / shares); }
    __device__ __forceinline__ int share_of(int unit) const { return static_cast<int>((static_cast<int64_t>(unit + 1) * shares - 1) / total); }
};

// A sequence and its place among the units.
struct FewSeq {
    int b;     // -1: none
    int rank;
    int first; // its first unit
    int units;
    Seq s;
};

// The sequences 64 at a time, spread over the lanes of a wave: units and their inclusive sums.
struct FewLanes {
    int units;
    int end;
    Seq s;
};

__device__ __forceinline__ FewLanes few_lanes(const PagedAttnArgs& x, int base, int sum, int lane) {
    FewLanes f{};
    if (base + lane < x.c.B) { f.units = few_units(x, base + lane, f.s); }
    f.end = sum + wave_inclusive_scan(f.units);
    return f;
}

__device__ __forceinline__ FewPlan few_plan(const PagedAttnArgs& x, int lane, FewLanes& f) {
    FewPlan p{0, 1};
    for (int base = 0; base < x.c.B; base += 64) {
        f = few_lanes(x, base, p.total, lane);
        p.total = __builtin_amdgcn_readlane(f.end, 63);
    }
    p.shares = max(1, min(x.slots, p.total));
    return p;
}

// The sequence that holds `unit`. `f`: the lanes of the only 64 sequences where there are no more.
__device__ __forceinline__ FewSeq few_find(const PagedAttnArgs& x, int unit, int lane, FewLanes f) {
    FewSeq q{-1, 0, 0, 0, {}};
    int sum = 0;
    for (int base = 0; base < x.c.B; base += 64) {
        if (x.c.B > 64) { f = few_lanes(x, base, sum, lane); }
        const uint64_t some = __ballot(f.units > 0);
        const uint64_t past = __ballot(f.units > 0 && f.end > unit);
        if (past != 0u) {
            const int at = __ffsll(static_cast<long long>(past)) - 1;
            q.b = base + at;
            q.rank += __popcll(some & ((uint64_t{1} << at) - 1));
            q.units = __builtin_amdgcn_readlane(f.units, at);
            q.first = __builtin_amdgcn_readlane(f.end, at) - q.units;
            q.s = lane_seq(f.s, at);
            return q;
        }
        q.rank += __popcll(some);
        sum = __builtin_amdgcn_readlane(f.end, 63);
    }
    return q;
}

// Waves per SIMD: one where two would not hold a chunk and the accumulators.
constexpr int few_waves(int D) { return D == 128 ? 2 : 1; }

// A wave's tiles [j0, j1) of a sequence: the state of its rows.
template <int D, bool BF, int NT, bool CARE>
__device__ __forceinline__ void few_walk(const PagedAttnArgs& x, int h, const Seq& s, const Tiles& tiles, const int32_t* table, int j0, int j1, int c, int g,
                                         Rows<D, BF, NT>& r, float down) {
    const int lane = threadIdx.x & 63;
    const int end = s.history + s.tokens;
    // pages of 64 halves (32 tiles) at a time, one per lane, the next 64 fetched ahead
    const auto pages_from = [&](int j) {
        const int v = j + (lane >> 1);
        const int key = 32 * tiles.tile(v) + 16 * (lane & 1);
        int page = -1;
        if (v < j1 && key < end) { page = table[key >> x.c.page_shift]; }
        return page >= 0 && page < x.c.pages ? page : -1;
    };
    int ids = pages_from(j0), next_ids = pages_from(j0 + 32);
    // at even tiles: past the 32nd of a fetch the other one is refilled for tiles j + 34 ..
    const auto refill = [&](int j) {
        if (((j - j0) & 63) == 30) { ids = pages_from(j + 34); }
        if (((j - j0) & 63) == 62) { next_ids = pages_from(j + 34); }
    };
    const auto halves = [&](int j) { // of tile j in [j0, ...): past the end no page
        const int i = 2 * (j - j0);
        const int from = (i & 127) < 64 ? 0 : 1; // this or the next 64
        Halves hv;
        hv.page[0] = __builtin_amdgcn_readlane(from ? next_ids : ids, i & 63);
        hv.page[1] = __builtin_amdgcn_readlane(from ? next_ids : ids, (i & 63) + 1);
        return hv;
    };
    Probs<NT> pr;
    uint32_t large = 0u; // known already
    // registers for one chunk: its keys make room for the next ones' as soon as the scores are there, then its values
    ChunkK<D, BF> ka;
    ChunkV<D, BF> va;
    Halves ha = halves(j0);
    load_keys<D, BF>(x, h, tiles.tile(j0), ha, c, g, ka);
    load_values<D, BF>(x, h, tiles.tile(j0), ha, c, g, va);
    init_rows<D, BF, NT>(x, s, h, 0, c, g, r);
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
        chunk_probs<D, BF, NT>(x, tiles.tile(j), ha, g, ka, r, pr);
        const Halves hb = halves(j + 1); // before the refill: tile 31 of a fetch is still in it
        if (((j - j0) & 1) == 0) { refill(j); }
        __builtin_amdgcn_sched_barrier(0);
        load_keys<D, BF>(x, h, tiles.tile(j + 1), hb, c, g, ka);
        __builtin_amdgcn_sched_barrier(0);
        chunk_values<D, BF, NT, CARE>(tiles.tile(j), ha, g, pr, va, r, down, large);
        __builtin_amdgcn_sched_barrier(0);
        load_values<D, BF>(x, h, tiles.tile(j + 1), hb, c, g, va);
        ha = hb;
    }
}

// Units [u0, u1) of sequence q: the part goes to its slot, or, where it is the whole sequence, to the output.
template <int D, bool BF, int NT, int NW>
__device__ __forceinline__ void few_part(const PagedAttnArgs& x, int h, const FewSeq& q, const FewPlan& plan, int share, int u0, int u1,
                                         f4 (&xo)[NW / 2][NT * (D / 16) * 64], float2 (&xm)[NW / 2][NT * 64]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const Seq s = q.s;
    const Tiles tiles = tiles_of(x, s.history, s.history + s.tokens - 1, 5);
    const int t0 = min(u0 * kUnit, tiles.count), t1 = min(u1 * kUnit, tiles.count);
    const int each = (t1 - t0 + NW - 1) / NW;
    const int j0 = min(t0 + wave * each, t1), j1 = min(j0 + each, t1);
    const int rows = s.tokens * x.G;
    const int head = plan.share_of(q.first), splits = plan.share_of(q.first + q.units - 1) - head + 1;
    if (x.seq_table != nullptr && u0 == 0 && h == 0 && threadIdx.x == 0) {
        x.seq_table[2 * q.b] = head + q.rank;
        x.seq_table[2 * q.b + 1] = splits;
    }
    Rows<D, BF, NT> r;
    const int32_t* table = x.c.table + q.b * x.c.table_row;
    few_walk<D, BF, NT, false>(x, h, s, tiles, table, j0, j1, c, g, r, 1.0f);
    bool lower = false; // by the lower weights
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
        // sums from 2^100 up (no sum of parts may overflow either), infinite ones or NaN
        if (__builtin_expect(__any(top >= static_cast<uint32_t>(127 + 100) << 24), 0)) {
            uint32_t large = 0u;
#pragma unroll 1
            for (int j = j0; j < j1; ++j) {
                const int tile = tiles.tile(j);
                ChunkV<D, BF> cv;
                load_values<D, BF>(x, h, tile, halves_of(x, table, tile, s.history + s.tokens - 1), c, g, cv);
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
            few_walk<D, BF, NT, true>(x, h, s, tiles, table, j0, j1, c, g, r, lower ? kCareDown : 1.0f);
        }
    }
    // ---- the waves' states into wave 0's: the upper half into the lower one, again and again
    float M[NT], L[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        M[nt] = r.m[nt] == -INFINITY ? -INFINITY : r.m[nt] * r.rowmul[nt];
        L[nt] = group4_sum(r.l[nt]);
        if (lower) { care_units(M[nt], L[nt]); }
    }
    __syncthreads(); // the last part's states are read
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
    if (wave != 0) { return; }
    constexpr int RUN = BF ? 8 : 4; // consecutive dims of a lane
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = 16 * nt + c;
        if (row >= rows) { continue; }
        if (splits > 1) {
            const int64_t at = (static_cast<int64_t>(share + q.rank) * x.c.Hkv + h) * (16 * NT) + row;
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
            if (g == 0) { *reinterpret_cast<float2*>(x.part_ml + 2 * at) = float2{M[nt], L[nt]}; }
        } else {
            const int t = row / x.G;
            uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + (s.start + t) * x.a.out.token_stride) + (h * x.G + row - t * x.G) * D;
#pragma unroll
            for (int i = 0; i < D / (16 * RUN); ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint16_t* dst = out + out_dim<BF>(RUN * i, 4 * g + e);
#pragma unroll
                    for (int k = 0; k < RUN; k += 4) {
                        const f4 o = {r.O[nt][RUN * i + k][e], r.O[nt][RUN * i + k + 1][e], r.O[nt][RUN * i + k + 2][e], r.O[nt][RUN * i + k + 3][e]};
                        *reinterpret_cast<u2*>(dst + k) = out_pair(o, L[nt]);
                    }
                }
            }
        }
    }
}

// WHOLE: a workgroup per sequence and KV head instead of a share.
template <int D, bool BF, int NT, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW == 8 ? 2 : few_waves(D), NW == 8 ? 2 : few_waves(D)))) void
paged_attn_few_kernel(PagedAttnArgs x) {
    // half of the waves' O and (m, l) at a time
    __shared__ f4 xo[NW / 2][NT * (D / 16) * 64];
    __shared__ float2 xm[NW / 2][NT * 64];
    const int lane = threadIdx.x & 63;
    if constexpr (WHOLE) {
        FewSeq q{static_cast<int>(blockIdx.x) / x.c.Hkv, 0, 0, 0, {}};
        q.units = few_units(x, q.b, q.s);
        if (q.units > 0) { few_part<D, BF, NT, NW>(x, blockIdx.x % x.c.Hkv, q, FewPlan{q.units, 1}, 0, 0, q.units, xo, xm); }
        return;
    }
    const int h = blockIdx.x % x.c.Hkv;
    FewLanes fl;
    const FewPlan plan = few_plan(x, lane, fl);
    const int share = blockIdx.x / x.c.Hkv;
    if (plan.total == 0 || share >= plan.shares) { return; }
    const int stop = plan.begin(share + 1);
#pragma unroll 1
    for (int u = plan.begin(share); u < stop;) {
        const FewSeq q = few_find(x, u, lane, fl);
        const int next = min(stop, q.first + q.units);
        few_part<D, BF, NT, NW>(x, h, q, plan, share, u - q.first, next - q.first, xo, xm);
        u = next;
    }
}
// ---- many rows: tiles of query rows over key tiles that a workgroup decodes once ------------------
//
// A workgroup of 8 waves owns a tile of query rows of one (sequence, KV head): WR row waves of 16 NT rows, each
// times WK waves that take different 32-key chunks (short prompts). It walks the keys in tiles of 16,384 values per
// plane: the rows of tile j + 2 are on their way to registers while tile j + 1 is decoded into the spare half of a
// double LDS buffer and tile j is multiplied, one barrier per tile. A wave stages 16 (head_dim 256: 8) whole rows of
// a tile, so its page is a scalar. K and V keep their row order in LDS: K pieces are swizzled for the 16-byte operand
// reads, V in 32-byte segments for the transposing reads (ds_read_b64_tr_b16), which deliver V^T operands in the key
// order that the S^T accumulator leaves P in.
// Operands are FP16 (K and Q of BF16 caches stay BF16): K' = code * scale and V' = code * scale or value, times a
// power of two that the workgroup takes from its first tile with a value (three bits of room above its largest scale or
// value), rounded once (2^-11); BF16 values down to 2^-29 of the top are exact, smaller ones off by at most 2^-19 of the
// largest of their unit of eight. A tile with a larger, infinite or NaN value, or with an INT8 scale or a BF16 unit below
// 2^-18 of the top (other than zero) is left out, and its chunks are walked as the few-row kernel does it afterwards, which
// has no such range but decodes each key in every wave (with every tile 2,370 instead of 790 us, as below; BF16 4,490).
// P is FP16, off by 2^-11 of itself and 2^-33 of the row's largest, and its sum is that of the same rounded numbers.
//
// What bounds it: neither matrix cores (40% busy) nor VALU (57%) alone; a SIMD's two waves hardly overlap them, and the
// registers (256 each) leave no room for more work of one wave in flight. Measured on MI355X, 8,192 first tokens at
// 40/8/128: INT8 790 us (870 TFLOP/s), BF16 785 us; at 24/4/256 1,167 and 1,097 us; a large library product reaches 1,318.

constexpr int kManyThreads = 512;
constexpr int kManyMarks = 131072;          // key tiles of a workgroup, at most
static_assert(kPagedMaxKeys <= 64 * kManyMarks);

template <int D, int WK>
struct ManyGeo {
    static constexpr int NT = D == 128 ? 2 : 1;
    static constexpr int WR = 8 / WK;
    static constexpr int BM = 16 * NT * WR; // query rows of a workgroup
    static constexpr int KT = 16384 / D;    // keys of a tile
    static constexpr int LG = D == 128 ? 7 : 6;
    static constexpr int NCH = KT / 32;
    static constexpr int RW = KT / 8;       // rows that a wave stages
    static constexpr int kPlane = 32768;
    static constexpr int kBuf = 2 * kPlane;
    static_assert(NCH % WK == 0, "every wave takes whole chunks");
};

// A wave's rows of a tile on their way.
template <int D, bool BF>
struct StageRegs {
    static constexpr int U = BF ? 4 : 2; // 16-byte units of a lane and plane
    u4 k[U], v[U];
    uint32_t ks[BF ? 1 : U], vs[BF ? 1 : U];
};

template <int D, bool BF>
__device__ __forceinline__ void stage_load(const PagedAttnArgs& x, int h, int key0, int page, int lane, StageRegs<D, BF>& r) {
    constexpr int kRow = BF ? 2 * D : D;
    constexpr int PR = kRow / 16; // units of a row
    constexpr int RW = ManyGeo<D, 1>::RW;
    const bool there = page >= 0;
    const int64_t pg = there ? page : 0;
    const int64_t row = (static_cast<int64_t>(h) << x.c.page_shift) + (key0 & ((1 << x.c.page_shift) - 1));
    const __amdgpu_buffer_rsrc_t kb = raw_buffer(x.c.k + pg * x.c.k_page + row * kRow, there ? RW * kRow : 0);
    const __amdgpu_buffer_rsrc_t vb = raw_buffer(x.c.v + pg * x.c.v_page + row * kRow, there ? RW * kRow : 0);
#pragma unroll
    for (int i = 0; i < StageRegs<D, BF>::U; ++i) {
        r.k[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(kb, 16 * (lane + 64 * i), 0, 0));
        r.v[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vb, 16 * (lane + 64 * i), 0, 0));
    }
    if constexpr (!BF) {
        constexpr int kScaleRow = D / 32;
        const __amdgpu_buffer_rsrc_t ksb = raw_buffer(x.c.ks + pg * x.c.ks_page + row * kScaleRow, there ? RW * kScaleRow : 0);
        const __amdgpu_buffer_rsrc_t vsb = raw_buffer(x.c.vs + pg * x.c.vs_page + row * kScaleRow, there ? RW * kScaleRow : 0);
#pragma unroll
        for (int i = 0; i < StageRegs<D, BF>::U; ++i) {
            const int u = lane + 64 * i;
            const int off = (u / PR) * kScaleRow + 2 * ((u % PR) / 4);
            r.ks[i] = __builtin_amdgcn_raw_buffer_load_b16(ksb, off, 0, 0) & 0xffffu;
            r.vs[i] = __builtin_amdgcn_raw_buffer_load_b16(vsb, off, 0, 0) & 0xffffu;
        }
    }
}

// Rows at or past `live` (of the wave's RW) belong to no visible key: their scales and values become zero.
template <int D, bool BF>
__device__ __forceinline__ void stage_trim(StageRegs<D, BF>& r, int live, int lane) {
    constexpr int PR = (BF ? 2 * D : D) / 16;
#pragma unroll
    for (int i = 0; i < StageRegs<D, BF>::U; ++i) {
        const bool dead = (lane + 64 * i) / PR >= live;
        if constexpr (BF) {
            r.v[i] = dead ? u4{0u, 0u, 0u, 0u} : r.v[i];
        } else {
            r.ks[i] = dead ? 0u : r.ks[i];
            r.vs[i] = dead ? 0u : r.vs[i];
        }
    }
}

// The largest magnitudes of a thread's part, NaN kept: K's and V's scales, or (BF16) V's values. `least` (BF16): the smallest
// of its units' largest values, zeros aside, as bits less one.
struct StageSize {
    float k, v;
    uint32_t least;
};

template <int D, bool BF>
__device__ __forceinline__ StageSize stage_size(const StageRegs<D, BF>& r) {
    StageSize z{0.0f, 0.0f, 0xffffffffu};
#pragma unroll
    for (int i = 0; i < StageRegs<D, BF>::U; ++i) {
        if constexpr (BF) {
            float m = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) { m = fmax_ieee(m, fmax_ieee(fabsf(__uint_as_float(r.v[i][w] << 16)), fabsf(__uint_as_float(r.v[i][w] & 0xffff0000u)))); }
            z.v = fmax_ieee(z.v, m);
            z.least = min(z.least, __float_as_uint(m) - 1u);
        } else {
            z.k = fmax_ieee(z.k, fabsf(f16_bits_to_f32(static_cast<uint16_t>(r.ks[i]))));
            z.v = fmax_ieee(z.v, fabsf(f16_bits_to_f32(static_cast<uint16_t>(r.vs[i]))));
        }
    }
    return z;
}

// The workgroup's powers of two and the bounds of what they can hold.
struct ManyScale {
    float k, v;       // factors of K' and V'
    float klim, vlim; // a tile with a larger scale (BF16: value) needs care
    uint32_t vleast;  // BF16: so does one with a smaller, but not zero, unit, as StageSize::least has it
};

// INT8: |code| <= 128, so scales below 2^E give K' below 2^15; BF16: values below 2^E.
__device__ __forceinline__ void pick(float top, int shift, float& factor, float& lim) {
    const uint32_t b = __float_as_uint(top) >> 23;
    // no finite top (or none): factor one
    const int E = top > 0.0f && b < 255u ? max(-100, min(60, static_cast<int>(b) - 126 + 3)) : shift; // sums stay below 2^100
    factor = __uint_as_float(static_cast<uint32_t>(127 + shift - E) << 23);
    lim = __uint_as_float(static_cast<uint32_t>(127 + E) << 23);
}

// Decodes a thread's part into a tile; returns whether it holds what the FP16 operands cannot.
template <int D, bool BF>
__device__ __forceinline__ bool stage_store(const StageRegs<D, BF>& r, const ManyScale& sc, char* buf, int row0, int lane) {
    constexpr int kRow = BF ? 2 * D : D;
    constexpr int PR = kRow / 16;
    char* vp = buf + ManyGeo<D, 1>::kPlane;
    const StageSize z = stage_size<D, BF>(r);
    bool small = BF && z.least < sc.vleast; // an INT8 scale, or a unit of BF16 values, that FP16 would round
#pragma unroll
    for (int i = 0; i < StageRegs<D, BF>::U; ++i) {
        const int u = lane + 64 * i;
        const int row = row0 + u / PR;
        const int at = row * 2 * D;
        const int k7 = row & 7;
        if constexpr (BF) {
            const int p = u % PR; // piece of eight dims
            *reinterpret_cast<u4*>(buf + at + 16 * (p ^ (row & 15))) = r.k[i];
            u4 y;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const h2 z = {static_cast<_Float16>(__uint_as_float(r.v[i][w] << 16) * sc.v),
                              static_cast<_Float16>(__uint_as_float(r.v[i][w] & 0xffff0000u) * sc.v)};
                y[w] = __builtin_bit_cast(uint32_t, z);
            }
            *reinterpret_cast<u4*>(vp + at + 32 * ((p >> 1) ^ k7) + 16 * (p & 1)) = y;
        } else {
            const int p = 2 * (u % PR); // two pieces of eight dims
            const _Float16 k1 = static_cast<_Float16>(f16_bits_to_f32(static_cast<uint16_t>(r.ks[i])) * sc.k);
            const _Float16 v1 = static_cast<_Float16>(f16_bits_to_f32(static_cast<uint16_t>(r.vs[i])) * sc.v);
            const h2 k2 = {k1, k1}, v2 = {v1, v1};
            small |= (r.ks[i] != 0u && fabsf(static_cast<float>(k1)) < 0x1p-14f) || (r.vs[i] != 0u && fabsf(static_cast<float>(v1)) < 0x1p-14f);
            *reinterpret_cast<h8*>(buf + at + 16 * (p ^ (row & 15))) = scale_h8(codes8(r.k[i][0], r.k[i][1]), k2);
            *reinterpret_cast<h8*>(buf + at + 16 * ((p + 1) ^ (row & 15))) = scale_h8(codes8(r.k[i][2], r.k[i][3]), k2);
            char* vr = vp + at + 32 * ((p >> 1) ^ k7);
            *reinterpret_cast<h8*>(vr) = scale_h8(codes8(r.v[i][0], r.v[i][1]), v2);
            *reinterpret_cast<h8*>(vr + 16) = scale_h8(codes8(r.v[i][2], r.v[i][3]), v2);
        }
    }
    return small || !(z.k <= sc.klim && z.v <= sc.vlim); // NaN: care
}

constexpr int kCus = 256;

// What the choices below weigh, in us on MI355X: a key tile with WK = 1, 2, 4 waves per row tile (8,192 tokens, every WK
// forced: 802, 1,054 and 1,574 us at head_dim 128, 1,161 and 1,614 us at 256, INT8), and a workgroup besides its tiles
// (the batch's plan, the first page, the epilogue). Half empty row tiles of one sequence's verify round fit too: 5 to 8 tokens
// over 45,000 and 131,000 rows reckoned 49, 103, 65, 151 and 149 us, took 45, 90, 70, 160 and 136.
__host__ __device__ constexpr float tile_us(int D, int wk) {
    return D == 128 ? (wk == 1 ? 4.9f : wk == 2 ? 3.2f : 2.6f) : (wk == 1 ? 2.95f : 2.05f);
}
constexpr float kWorkgroupUs = 8.0f;

// The last `rem` row tiles x heads that do not fill the chip: key splits of each, and the time they take. Parts are
// written and read at 4 TB/s and cost a launch. Measured at 40/8/128 INT8: 200 tokens over 2,000 rows 39.9 us with
// two waves per row tile and four splits, 38.2 and 48.0 us with one and four waves; 700 over 300 rows 41.0 (two waves,
// no splits), 51.8 and 58.5 us.
struct Tail {
    int splits;
    float us;
};

constexpr int kMaxSplits = 32;

// The time with `ns` splits; infinite where they are not possible.
__host__ __device__ inline float tail_us(int rem, int ns, int longest, float us_tile, int elements, int parts) {
    if (ns == 1) { return kWorkgroupUs + static_cast<float>(longest) * us_tile; }
    if (ns * rem > parts || ns > longest) { return INFINITY; }
    const int rounds = (rem * ns + kCus - 1) / kCus;
    return static_cast<float>(rounds) * (kWorkgroupUs + static_cast<float>((longest + ns - 1) / ns) * us_tile) + 8.0f +
           static_cast<float>(rem * ns) * static_cast<float>(elements) * 2.0e-6f;
}

// On the host one after another, on the device a lane each (with a loop there 200 tokens over 2,000 rows took 38.8 us
// instead of 34.2).
inline Tail tail_of(int rem, int longest, float us_tile, int elements, int parts) {
    Tail best{1, rem > 0 ? tail_us(rem, 1, longest, us_tile, elements, parts) : 0.0f};
    for (int ns = 2; rem > 0 && ns <= kMaxSplits; ++ns) {
        const float us = tail_us(rem, ns, longest, us_tile, elements, parts);
        if (us < best.us) { best = Tail{ns, us}; }
    }
    return best;
}

__device__ __forceinline__ int tail_splits(int rem, int longest, float us_tile, int elements, int parts, int lane) {
    const float us = lane < kMaxSplits ? tail_us(rem, lane + 1, longest, us_tile, elements, parts) : INFINITY;
    const uint64_t best = __ballot(us == -wave_max(-us));
    return __ffsll(static_cast<long long>(best));
}

// The row tiles of 64 sequences, spread over the lanes of a wave: their numbers and inclusive sums.
struct ManyLanes {
    int n;
    int end;
    Seq s;
};

__device__ __forceinline__ ManyLanes many_lanes(const PagedAttnArgs& x, int base, int sum, int bm, int lane) {
    ManyLanes f{};
    if (base + lane < x.c.B) {
        f.s = sequence(x, base + lane);
        const int rows = f.s.tokens * x.G;
        f.n = rows > x.few_rows ? (rows + bm - 1) / bm : 0;
    }
    f.end = sum + wave_inclusive_scan(f.n);
    return f;
}

// Row tiles x heads of the batch: the first `full` fill the chip's rounds, each of the others has `splits` workgroups.
struct ManyPlan {
    int units;
    int full;
    int splits;
};

template <int D, int WK>
__device__ __forceinline__ ManyPlan many_plan(const PagedAttnArgs& x, int lane, ManyLanes& f) {
    constexpr int BM = ManyGeo<D, WK>::BM;
    int total = 0, longest = 0;
    for (int base = 0; base < x.c.B; base += 64) {
        f = many_lanes(x, base, total, BM, lane);
        int len = 0;
        if (f.n > 0) {
            const int last = f.s.history + f.s.tokens - 1;
            len = tiles_of(x, max(f.s.history, last - (BM - 1) / x.G), last, ManyGeo<D, WK>::LG).count;
        }
        total = __builtin_amdgcn_readlane(f.end, 63);
        longest = max(longest, static_cast<int>(wave_max(static_cast<float>(len))));
    }
    ManyPlan p{total * x.c.Hkv, 0, 1};
    p.full = p.units / kCus * kCus;
    if (p.units > p.full) { p.splits = tail_splits(p.units - p.full, longest, tile_us(D, WK), BM * D, x.many_parts, lane); }
    if (p.splits == 1) { p.full = p.units; }
    return p;
}

struct ManyWork {
    int b; // -1: none
    int tile;
    Seq s;
};

// The sequences' row tiles in order; `slot` counts them over the batch. `f`: the lanes of the only 64 sequences where
// there are no more.
__device__ __forceinline__ ManyWork many_work(const PagedAttnArgs& x, int slot, int bm, int lane, ManyLanes f) {
    ManyWork w{-1, 0, {}};
    int sum = 0;
    for (int base = 0; base < x.c.B; base += 64) {
        if (x.c.B > 64) { f = many_lanes(x, base, sum, bm, lane); }
        const uint64_t mine = __ballot(f.n > 0 && slot >= f.end - f.n && slot < f.end);
        if (mine != 0u) {
            const int at = __ffsll(static_cast<long long>(mine)) - 1;
            w.b = base + at;
            // the last tokens see the most keys: their tiles first
            w.tile = __builtin_amdgcn_readlane(f.end, at) - 1 - slot;
            w.s = lane_seq(f.s, at);
            return w;
        }
        sum = __builtin_amdgcn_readlane(f.end, 63);
    }
    return w;
}

typedef short s4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u2 read_tr(const char* p) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((NMI_AS3 s4*)(p)));
}

template <int D, bool BF, int WK>
__global__ __launch_bounds__(kManyThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_many_kernel(PagedAttnArgs x) {
    using MG = ManyGeo<D, WK>;
    constexpr int NT = MG::NT, KT = MG::KT;
    constexpr int VF = D == 128 ? 8 : 4; // V^T operands in flight
    __shared__ __attribute__((aligned(256))) char smem[2 * MG::kBuf];
    __shared__ uint32_t marks[kManyMarks / 32]; // tiles that need care
    __shared__ uint32_t state[2][8];            // per buffer and wave: bit 0 its page exists, bit 1 care
    __shared__ float tops[2][8];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int wr = wave / WK, wk = wave % WK;
    ManyLanes lanes;
    const ManyPlan plan = many_plan<D, WK>(x, lane, lanes);
    const int id = blockIdx.x;
    const int unit = id < plan.full ? id : plan.full + (id - plan.full) / plan.splits;
    const int splits = id < plan.full ? 1 : plan.splits;
    const int split = id < plan.full ? 0 : (id - plan.full) % plan.splits;
    if (unit >= plan.units) { return; }
    const int h = unit % x.c.Hkv;
    const ManyWork w = many_work(x, unit / x.c.Hkv, MG::BM, lane, lanes);
    if (w.b < 0) { return; }
    const Seq s = w.s;
    const int rows = s.tokens * x.G;
    const int r0 = w.tile * MG::BM;
    const int p0 = s.history + r0 / x.G, p1 = s.history + (min(r0 + MG::BM, rows) - 1) / x.G;
    const Tiles tiles = tiles_of(x, p0, p1, MG::LG);
    const int per = (tiles.count + splits - 1) / splits;
    const int j0 = min(split * per, tiles.count), j1 = min(j0 + per, tiles.count);

    // pages of the wave's rows, 64 tiles at a time
    const int32_t* table = x.c.table + w.b * x.c.table_row;
    const auto pages_from = [&](int j) {
        const int key = tiles.tile(j + lane) * KT + wave * MG::RW;
        int page = -1;
        if (j + lane < j1 && key <= p1) { page = table[key >> x.c.page_shift]; }
        return page >= 0 && page < x.c.pages ? page : -1;
    };
    int ids = pages_from(j0), next_ids = pages_from(j0 + 64);
    StageRegs<D, BF> sr;
    int page = -1; // of the rows in `sr`
    const auto fetch = [&](int j) {
        const int i = j - j0;
        if ((i & 63) == 0 && i > 0) { // a new 64: they were fetched 64 tiles ago
            ids = next_ids;
            next_ids = pages_from(j + 64);
        }
        page = __builtin_amdgcn_readlane(ids, i & 63);
        stage_load<D, BF>(x, h, tiles.tile(j) * KT + wave * MG::RW, page, lane, sr);
    };
    ManyScale sc{1.0f, 1.0f, INFINITY, INFINITY, 0u};
    const auto trim = [&](int j) {
        const int live = p1 + 1 - (tiles.tile(j) * KT + wave * MG::RW);
        if (live < MG::RW) { stage_trim<D, BF>(sr, live, lane); }
    };
    const auto put = [&](int j) {
        trim(j);
        const bool care = stage_store<D, BF>(sr, sc, smem + ((j - j0) & 1) * MG::kBuf, wave * MG::RW, lane);
        const uint32_t st = (page >= 0 ? 1u : 0u) | (__any(care) ? 2u : 0u);
        if (lane == 0) { state[(j - j0) & 1][wave] = st; }
    };

    if (j0 < j1) { fetch(j0); }
    Rows<D, BF, NT> r;
    const int row0 = r0 + 16 * NT * wr;
    init_rows<D, BF, NT>(x, s, h, row0, c, g, r);
    f4 l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { l[nt] = f4{0.f, 0.f, 0.f, 0.f}; }
    bool cared = false;
    if (j0 < j1) {
        for (int i = threadIdx.x; 32 * i < j1 - j0; i += kManyThreads) { marks[i] = 0u; }
        // the first tile that holds a value tells how large they are: absent pages and zero rows say nothing
        float kt = 0.0f, vt = 0.0f;
        int js = j0;
        for (;; ++js) {
            if (js > j0) { stage_load<D, BF>(x, h, tiles.tile(js) * KT + wave * MG::RW, __builtin_amdgcn_readfirstlane(pages_from(js)), lane, sr); }
            trim(js);
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
            if (__any(vt > 0.0f) || js + 1 == j1) { break; }
            __syncthreads(); // the tops are read
        }
        if (js > j0) { fetch(j0); }
        pick(kt, 8, sc.k, sc.klim);
        pick(vt, BF ? 15 : 8, sc.v, sc.vlim);
        sc.vleast = __float_as_uint(0x1p-6f / sc.v) - 1u;
        put(j0);
        if (j0 + 1 < j1) { fetch(j0 + 1); }
        __syncthreads();
    }
    float mul[NT]; // raw score of the FP16 K' -> log2 domain
    // The products start from the running maximum's negative: scores come out less it (rounded with it, -m * mul would move
    // every p by up to 2^(score 2^-25)). BF16 rows of 128 have no registers left for that: there it is added afterwards (8,192
    // tokens 785 us, 816 with eight registers spilled). `lim`: what moves the maximum; -infinity before the first score.
    constexpr bool kFromRef = !(BF && D == 128);
    std::conditional_t<kFromRef, f4, float> ref[NT];
    float lim[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        mul[nt] = BF ? r.rowmul[nt] : fminf(r.rowmul[nt] / sc.k, kLargest);
        ref[nt] = {};
        lim[nt] = -INFINITY;
    }
    // the wave's V^T reads: lane (c, g) addresses key 4 g + (c >> 2), dims 4 (c & 3) .. of a 16-dim segment
    const int vkey = 4 * g + (c >> 2);
    const int voff = vkey * 2 * D + 32 * (vkey & 7) + 8 * (c & 3);
    // waves w and w + 4 share a SIMD: one decodes the next tile before its products, one after them
    const bool early = wave < 4;
    const int low = min(r.lo, kPagedMaxKeys) + 1 - x.a.window; // the wave sees nothing below it but sinks
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
        const char* buf = smem + ((j - j0) & 1) * MG::kBuf;
        const uint32_t st = lane < 8 ? state[(j - j0) & 1][lane] : 0u;
        const uint32_t here = static_cast<uint32_t>(__ballot((st & 1u) != 0u));
        const bool care = __any((st & 2u) != 0u);
        const int key0 = tiles.tile(j) * KT;
        const auto stage = [&] {
            if (j + 1 < j1) {
                put(j + 1);
                if (j + 2 < j1) { fetch(j + 2); }
            }
        };
        if (early) { stage(); }
        if (care) {
            cared = true;
            if (threadIdx.x == 0) { marks[(j - j0) >> 5] |= 1u << ((j - j0) & 31); }
        } else {
            u4 kf[2][D / 32];
            const auto read_k = [&](const char* from, int chunk) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const char* krow = from + (32 * chunk + 16 * kt + c) * 2 * D;
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
                        const int piece = BF ? 4 * k + g : 8 * (k >> 1) + 2 * g + (k & 1);
                        kf[kt][k] = *reinterpret_cast<const u4*>(krow + 16 * (piece ^ c));
                    }
                }
            };
#pragma unroll 1
            for (int cw = 0; cw < MG::NCH / WK; ++cw) {
                const int ci = cw * WK + wk;
                const int c0 = key0 + 32 * ci;
                // the halves' pages: two waves' rows each at head_dim 256
                const uint32_t bits = D == 128 ? here >> (2 * ci) : (here >> (4 * ci) & 1u) | (here >> (4 * ci + 1) & 2u);
                // by arithmetic: hipcc 7.2 inverted a select on a bit of a scalar here (s_bitcmp0 for s_bitcmp1)
                const Halves hv{{static_cast<int>(bits & 1u) - 1, static_cast<int>((bits >> 1) & 1u) - 1}};
                if (c0 > r.hi || (c0 + 31 < low && c0 >= x.a.sinks) || (hv.page[0] & hv.page[1]) < 0) {
                    continue;
                }
                read_k(buf, ci);
                f4 sacc[2][NT];
                __builtin_amdgcn_s_setprio(1); // products first: the SIMD's other wave fills in with its softmax
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            f4 acc = {0.f, 0.f, 0.f, 0.f};
                            if constexpr (kFromRef) { acc = ref[nt]; }
                            if (k > 0) { acc = sacc[kt][nt]; }
                            if constexpr (BF) {
                                sacc[kt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, kf[kt][k]), __builtin_bit_cast(bf8, r.q[nt][k]), acc, 0, 0, 0);
                            } else {
                                sacc[kt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, kf[kt][k]), __builtin_bit_cast(h8, r.q[nt][k]), acc, 0, 0, 0);
                            }
                        }
                    }
                }
                // the V^T operands are on their way while the softmax is worked out
                const char* vp = buf + MG::kPlane + 32 * ci * 2 * D;
                u4 vf[VF];
                const auto read_v = [&](int t) {
                    const int at = (voff ^ (32 * (t & 7))) + 256 * (t >> 3);
                    const u2 a = read_tr(vp + at), b = read_tr(vp + at + 16 * 2 * D);
                    return u4{a[0], a[1], b[0], b[1]};
                };
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < VF; ++t) { vf[t] = read_v(t); }
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                float sv[NT][8];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        sv[nt][i] = sacc[i >> 2][nt][i & 3];
                        if constexpr (!kFromRef) { sv[nt][i] += ref[nt]; }
                    }
                }
                if (!all_seen(x, r.lo, r.hi, c0 >> 5, hv)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const bool ok = sees(x, r.pos[nt], c0 + 16 * (i >> 2) + 4 * g + (i & 3), hv.page[i >> 2]);
                            sv[nt][i] = ok ? sv[nt][i] : -INFINITY;
                        }
                    }
                }
                float cmax[NT];
                bool any = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    cmax[nt] = score_max(sv[nt]);
                    any |= cmax[nt] > lim[nt];
                }
                if (__any(any)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const bool need = cmax[nt] > lim[nt];
                        const float up = need ? cmax[nt] : 0.0f;
                        const float alpha = lim[nt] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-up * mul[nt]);
#pragma unroll
                        for (int t = 0; t < D / 16; ++t) { r.O[nt][t] *= alpha; }
                        l[nt] *= alpha;
                        ref[nt] -= up;
#pragma unroll
                        for (int i = 0; i < 8; ++i) { sv[nt][i] -= up; }
                        lim[nt] = need ? kLazyTau / mul[nt] : lim[nt];
                    }
                }
                h8 p[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) { p[nt][i] = static_cast<_Float16>(__builtin_amdgcn_exp2f(fmaf(sv[nt][i], mul[nt], kPOffset))); }
                }
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    const u4 va = vf[t % VF];
                    if (t + VF < D / 16) { vf[t % VF] = read_v(t + VF); }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        r.O[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, va), p[nt], r.O[nt][t], 0, 0, 0);
                    }
                }
                const h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) { l[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[nt], l[nt], 0, 0, 0); }
                __builtin_amdgcn_s_setprio(0);
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
        if constexpr (kFromRef) { neg = ref[nt][0]; } else { neg = ref[nt]; }
        M[nt] = lim[nt] == -INFINITY ? -INFINITY : -neg * mul[nt];
        L[nt] = l[nt][0];
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
            for (int base = 0; base < j1 - j0; base += 32) {
                uint32_t bits = __builtin_amdgcn_readfirstlane(marks[base >> 5]);
#pragma unroll 1
                for (; bits != 0u; bits &= bits - 1u) {
                    const int key0 = tiles.tile(j0 + base + __builtin_ctz(bits)) * KT;
#pragma unroll 1
                    for (int cw = 0; cw < MG::NCH / WK; ++cw) {
                        const int tile = (key0 >> 5) + cw * WK + wk;
                        if (32 * tile > r.hi) { continue; }
                        const Halves hv = halves_of(x, table, tile, p1);
                        Probs<NT> pr;
                        {
                            ChunkK<D, BF> ck;
                            load_keys<D, BF>(x, h, tile, hv, c, g, ck);
                            chunk_probs<D, BF, NT>(x, tile, hv, g, ck, r, pr);
                        }
                        __builtin_amdgcn_sched_barrier(0); // the registers hold one plane's rows at a time
                        ChunkV<D, BF> cv;
                        load_values<D, BF>(x, h, tile, hv, c, g, cv);
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
            const Weights q = weights(M[nt], L[nt], m2, l2);
            L[nt] = L[nt] * q.a + l2 * q.b;
            M[nt] = q.M;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
                f4 o; // back in the first walk's order of dims, so that what follows is the same
#pragma unroll
                for (int e = 0; e < 4; ++e) { o[e] = q.b == 0.0f ? 0.0f : r.O[nt][t][e] * q.b; }
                r.O[nt][t] = o;
            }
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float* y = keep + (16 * nt + c) * D + out_dim<BF>(t, 4 * g + e);
                    *y = (q.a == 0.0f ? 0.0f : *y * q.a) + r.O[nt][t][e];
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
                const Weights q = weights(M[nt], L[nt], o.x, o.y);
                L[nt] = L[nt] * q.a + o.y * q.b;
                M[nt] = q.M;
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    const f4 y = xo[at * kPer + (nt * (D / 16) + t) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) { r.O[nt][t][e] = (q.a == 0.0f ? 0.0f : r.O[nt][t][e] * q.a) + (q.b == 0.0f ? 0.0f : y[e] * q.b); }
                }
            }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int rr = 16 * (NT * wr + nt) + c; // of the workgroup's rows
        const int row = r0 + rr;
        if (row >= rows) { continue; }
        if (splits > 1) {
            const int64_t at = static_cast<int64_t>(id - plan.full) * MG::BM + rr;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) { *reinterpret_cast<f4*>(x.many_o + at * D + 16 * t + 4 * g) = r.O[nt][t]; }
            if (g == 0) { *reinterpret_cast<float2*>(x.many_ml + 2 * at) = float2{M[nt], L[nt]}; }
        } else {
            const int t1 = row / x.G;
            uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + (s.start + t1) * x.a.out.token_stride) + (h * x.G + row - t1 * x.G) * D + 4 * g;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) { *reinterpret_cast<u2*>(out + 16 * t) = out_pair(r.O[nt][t], L[nt]); }
        }
    }
}

// ---- the parts of a row, one after another in the workspace ----------------------------------------
//
// One launch for both kernels' parts. Few rows: a workgroup per row and sequence, groups of D / 4 threads taking every
// group-th part, joined through LDS. Many rows: D / 4 threads per row of a split row tile.

template <int D>
__device__ __forceinline__ void store_row(const PagedAttnArgs& x, const Seq& s, int h, int row, int d, f4 O, float L) {
    const int t = row / x.G;
    uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + (s.start + t) * x.a.out.token_stride) + (h * x.G + row - t * x.G) * D + d;
    *reinterpret_cast<u2*>(out) = out_pair(O, L);
}

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

template <int D>
__device__ __forceinline__ void merge_few(const PagedAttnArgs& x, int block) {
    constexpr int TPR = D / 4, GRP = 256 / TPR;
    __shared__ f4 xo[GRP][TPR];
    __shared__ float2 xm[GRP];
    const int h = block % x.c.Hkv;
    const int row = block / x.c.Hkv % x.few_rows;
    const int b = block / x.c.Hkv / x.few_rows;
    const int first = x.seq_table[2 * b], splits = x.seq_table[2 * b + 1]; // of a sequence of the kernel's only
    const Seq s = sequence(x, b);
    const int rows = s.tokens * x.G;
    if (rows > x.few_rows || row >= rows || splits == 1) { return; } // one part is written already
    const int grp = threadIdx.x / TPR, d = 4 * (threadIdx.x % TPR);
    Merge m;
#pragma unroll 4
    for (int k = grp; k < splits; k += GRP) {
        const int64_t at = (static_cast<int64_t>(first + k) * x.c.Hkv + h) * x.few_rows + row;
        const float2 ml = *reinterpret_cast<const float2*>(x.part_ml + 2 * at);
        m.add(ml.x, ml.y, *reinterpret_cast<const f4*>(x.part_o + at * D + d));
    }
    xo[grp][threadIdx.x % TPR] = m.O;
    if (threadIdx.x % TPR == 0) { xm[grp] = float2{m.M, m.L}; }
    __syncthreads();
    if (grp != 0) { return; }
#pragma unroll
    for (int k = 1; k < GRP; ++k) { m.add(xm[k].x, xm[k].y, xo[k][threadIdx.x]); }
    store_row<D>(x, s, h, row, d, m.O, m.L);
}

template <int D, int WK>
__device__ __forceinline__ void merge_many(const PagedAttnArgs& x, int block) {
    constexpr int TPR = D / 4, RPB = 256 / TPR, BM = ManyGeo<D, WK>::BM;
    const int lane = threadIdx.x & 63;
    ManyLanes lanes;
    const ManyPlan plan = many_plan<D, WK>(x, lane, lanes);
    const int tail = block / (BM / RPB);
    const int unit = plan.full + tail;
    if (unit >= plan.units) { return; }
    const int h = unit % x.c.Hkv;
    const int rr = block % (BM / RPB) * RPB + threadIdx.x / TPR;
    const ManyWork w = many_work(x, unit / x.c.Hkv, BM, lane, lanes);
    if (w.b < 0) { return; }
    const int row = w.tile * BM + rr;
    if (row >= w.s.tokens * x.G) { return; }
    const int d = 4 * (threadIdx.x % TPR);
    const int64_t first = static_cast<int64_t>(tail) * plan.splits * BM + rr;
    Merge m;
#pragma unroll 4
    for (int k = 0; k < plan.splits; ++k) {
        const int64_t at = first + static_cast<int64_t>(k) * BM;
        const float2 ml = *reinterpret_cast<const float2*>(x.many_ml + 2 * at);
        m.add(ml.x, ml.y, *reinterpret_cast<const f4*>(x.many_o + at * D + d));
    }
    store_row<D>(x, w.s, h, row, d, m.O, m.L);
}

// The first `few` workgroups merge the few-row kernel's parts, the others the many-row kernel's.
template <int D, int WK>
__global__ __launch_bounds__(256) void paged_attn_merge_kernel(PagedAttnArgs x, int few) {
    if (static_cast<int>(blockIdx.x) < few) {
        merge_few<D>(x, blockIdx.x);
    } else {
        merge_many<D, WK>(x, blockIdx.x - few);
    }
}

} // namespace

namespace {

// How a call is cut.
struct PagedPlan {
    int32_t nt = 1;        // 16-row tiles of a few-row workgroup
    int32_t few_rows = 0;
    int32_t slots = 0;     // 0: no sequence of few rows is possible
    bool whole = false;    // a workgroup per few-row sequence
    bool merge = false;
    int32_t wk = 1;        // many rows: waves of a row tile over the keys
    int32_t tiles = 0;     // row tiles of the batch, at most (0: no sequence of many rows is possible)
    int32_t parts = 0;     // of the split row tiles
    size_t ml_offset = 0;
    size_t table_offset = 0;
    size_t many_offset = 0;
    size_t many_ml_offset = 0;
    size_t bytes = 0;
};

size_t align_up(size_t v) { return (v + 255) & ~size_t{255}; }

PagedPlan plan_paged(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t max_new, int32_t max_keys, int32_t window,
                     int32_t sinks) {
    const int32_t G = Hq / Hkv;
    PagedPlan p;
    // next to sequences of many rows, those of 17 to 32 are theirs: two row tiles cost the single tokens more
    p.nt = static_cast<int64_t>(max_new) * G <= 16 || static_cast<int64_t>(max_new) * G > 32 ? 1 : 2;
    p.few_rows = 16 * p.nt;
    const int64_t most_rows = std::min<int64_t>(max_new, tokens) * G; // of a sequence
    // one sequence of many rows: the many-row kernel serves it, whatever its rows turn out to be (no launches for none)
    if (B == 1 && most_rows > p.few_rows) { p.few_rows = 0; }
    // the most keys that `n` tokens see
    const auto seen = [&](int64_t n) {
        if (window == 0) { return static_cast<int64_t>(max_keys); }
        return std::min<int64_t>(max_keys, static_cast<int64_t>(window) + n + 126 + (static_cast<int64_t>(sinks) + 127) / 128 * 128);
    };
    size_t at = 0;
    if (p.few_rows > 0) {
        const int64_t units = (seen(std::min<int64_t>(max_new, p.few_rows)) + 127) / 128;
        // Where the sequences' heads are about as many as the CUs and short, a workgroup of eight waves each needs no merge
        // launch: 32 sequences at 40/8/128 INT8 of 200 rows 17.0 -> 11.1 us, of 500 20.2 -> 14.2, of 1,000 25.4 -> 19.6; 64 at
        // 24/4/256 of 500 28.6 -> 25.7. Fewer leave CUs idle (16 of 1,000 at 24/4/256 20.3 -> 34.5), more or longer ones gain
        // nothing or lose by their lengths' differences (200 of 300 rows 78 -> 84).
        const int64_t heads = static_cast<int64_t>(B) * Hkv;
        p.whole = p.nt == 1 && units <= 8 && heads > kCus * 3 / 4 && heads <= kCus;
        p.slots = p.whole ? B : static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(kCus * few_waves(D) / Hkv, B * units)));
        p.merge = !p.whole && p.slots > 1;
        if (p.merge) {
            const size_t rows = static_cast<size_t>(p.slots + B) * Hkv * p.few_rows;
            p.ml_offset = align_up(rows * D * sizeof(float));
            at = align_up(p.ml_offset + rows * 2 * sizeof(float));
        }
        if (p.merge) {
            p.table_offset = at;
            at = align_up(at + static_cast<size_t>(B) * 2 * sizeof(int32_t));
        }
    }
    if (most_rows > p.few_rows) {
        const int64_t rows = tokens * G;
        const int64_t seqs = std::min<int64_t>(B, rows / (p.few_rows + 1));
        const int64_t keys = seen(max_new);
        const int32_t kt = 16384 / D;
        const int32_t longest = static_cast<int32_t>((keys + kt - 1) / kt);
        const double mean = std::max(1.0, (static_cast<double>(keys) - (window == 0 ? 0.5 * std::min<double>(static_cast<double>(keys), max_new) : 0.0)) / kt);
        double best = 1e30;
        for (int32_t wk = 1; wk <= (D == 128 ? 4 : 2); wk *= 2) {
            const int32_t bm = (D == 128 ? 256 : 128) / wk;
            const int64_t tiles = rows / bm + seqs;
            const int32_t parts = static_cast<int32_t>(std::min<int64_t>((1 << 23) / (bm * D), longest > 1 ? tiles * Hkv * 32 : 0));
            const int64_t units = (rows + bm - 1) / bm * Hkv; // as if one sequence had them
            const double us = static_cast<double>(units / kCus) * (kWorkgroupUs + mean * tile_us(D, wk)) +
                              tail_of(static_cast<int>(units % kCus), longest, tile_us(D, wk), bm * D, parts).us;
            if (us < best) {
                best = us;
                p.wk = wk;
                p.parts = parts;
                p.tiles = static_cast<int32_t>(tiles);
            }
        }
        if (p.parts > 0) {
            const size_t part_rows = static_cast<size_t>(p.parts) * ((D == 128 ? 256 : 128) / p.wk);
            p.many_offset = at;
            p.many_ml_offset = align_up(at + part_rows * D * sizeof(float));
            at = align_up(p.many_ml_offset + part_rows * 2 * sizeof(float));
        }
    }
    p.bytes = at;
    return p;
}

template <int D, bool BF, int WK>
void launch(const PagedAttnArgs& x, const PagedPlan& p, hipStream_t stream) {
    uint32_t few = 0, tails = 0; // workgroups of the merge
    if (p.slots > 0) {
        const uint32_t grid = static_cast<uint32_t>(p.slots) * x.c.Hkv;
        if (p.whole) {
            hipLaunchKernelGGL((paged_attn_few_kernel<D, BF, 1, 8, true>), dim3(grid), dim3(512), 0, stream, x);
        } else if (p.nt == 1) {
            hipLaunchKernelGGL((paged_attn_few_kernel<D, BF, 1, 4, false>), dim3(grid), dim3(256), 0, stream, x);
        } else {
            hipLaunchKernelGGL((paged_attn_few_kernel<D, BF, 2, 4, false>), dim3(grid), dim3(256), 0, stream, x);
        }
        check_launch("paged_attn_few_kernel");
        if (p.merge) { few = static_cast<uint32_t>(p.few_rows) * x.c.Hkv * x.c.B; }
    }
    if (p.tiles > 0) {
        const int64_t blocks = static_cast<int64_t>(p.tiles) * x.c.Hkv;
        if (blocks > 0x7FFFFF) { throw Unsupported("paged attention: more than 2^23 workgroups are not built"); }
        hipLaunchKernelGGL((paged_attn_many_kernel<D, BF, WK>), dim3(static_cast<uint32_t>(blocks) + p.parts), dim3(kManyThreads), 0, stream, x);
        check_launch("paged_attn_many_kernel");
        // the row tiles that may be split
        if (p.parts > 0) { tails = static_cast<uint32_t>(std::min<int64_t>(blocks, kCus - 1)) * (ManyGeo<D, WK>::BM / (1024 / D)); }
    }
    if (few + tails == 0) { return; }
    hipLaunchKernelGGL((paged_attn_merge_kernel<D, WK>), dim3(few + tails), dim3(256), 0, stream, x, static_cast<int>(few));
    check_launch("paged_attn_merge_kernel");
}

template <int D, bool BF>
void launch(const PagedAttnArgs& x, const PagedPlan& p, hipStream_t stream) {
    if (p.wk == 1) {
        launch<D, BF, 1>(x, p, stream);
    } else if (p.wk == 2) {
        launch<D, BF, 2>(x, p, stream);
    } else if constexpr (D == 128) {
        launch<D, BF, 4>(x, p, stream);
    }
}

} // namespace

size_t paged_attention_bytes(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t max_new, int32_t max_keys,
                             int32_t window, int32_t sinks) {
    return plan_paged(Hq, Hkv, D, tokens, B, max_new, max_keys, window, sinks).bytes;
}

void launch_paged_attention(const PagedAttention& a, const PagedRef& c, void* workspace, hipStream_t stream) {
    const PagedPlan p = plan_paged(a.Hq, c.Hkv, c.D, a.tokens, c.B, a.max_new, a.max_keys, a.window, a.sinks);
    PagedAttnArgs x{};
    x.a = a;
    if (a.window == 0) { x.a.window = 0x7FFFFFFF; } // every row of at most kPagedMaxKeys
    x.c = c;
    x.G = a.Hq / c.Hkv;
    x.scale_log2 = a.scale * 1.4426950408889634f;
    x.few_rows = p.few_rows;
    x.slots = p.slots;
    x.many_parts = p.parts;
    char* ws = static_cast<char*>(workspace);
    x.part_o = reinterpret_cast<float*>(ws);
    x.part_ml = reinterpret_cast<float*>(ws + p.ml_offset);
    x.seq_table = p.merge ? reinterpret_cast<int32_t*>(ws + p.table_offset) : nullptr;
    x.many_o = reinterpret_cast<float*>(ws + p.many_offset);
    x.many_ml = reinterpret_cast<float*>(ws + p.many_ml_offset);
    if (c.D == 128 && !c.bf16) {
        launch<128, false>(x, p, stream);
    } else if (c.D == 128) {
        launch<128, true>(x, p, stream);
    } else if (!c.bf16) {
        launch<256, false>(x, p, stream);
    } else {
        launch<256, true>(x, p, stream);
    }
}

} // namespace nmi
