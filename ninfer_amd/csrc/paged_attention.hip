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
// V scales in the same way: w = p * s * 2^-E in FP16 (off by 2^-11 of itself; 2^E tops the scales of the 32 keys
// at hand, so w neither overflows nor, next to them, vanishes), times codes, times 2^E in FP32. No scale is too
// large or too small for that. BF16 caches multiply stored values; p goes in as two BF16 terms (16 bits).
// Maxima, sums and accumulators are FP32.
#include "attn_math.h"
#include "common.h"
#include "device_utils.h"
#include "lds_dma.h"
#include "paged_internal.h"

#include <algorithm>
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
    int32_t slots;     // its key splits per KV head
    int32_t min_units; // its shortest split, in units of 128 keys
    float* part_o;     // FP32 O [partial row][D] and (log2-domain maximum, sum) [partial row][2]
    float* part_ml;
    int32_t* seq_table; // per sequence: first slot, splits
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

// The 32-key tiles that tokens at positions p0 .. p1 need: [0, sink) and [first, end) of the sequence's tiles,
// numbered on without the gap.
struct Tiles {
    int32_t sink;
    int32_t first;
    int32_t count;
    __device__ __forceinline__ int32_t tile(int32_t i) const { return i < sink ? i : i - sink + first; }
};

__device__ __forceinline__ Tiles tiles_of(const PagedAttnArgs& x, int32_t p0, int32_t p1) {
    const int32_t first = x.a.window > 0 ? max(0, p0 + 1 - x.a.window) : 0;
    Tiles t{(min(x.a.sinks, first) + 31) >> 5, first >> 5, 0};
    if (t.sink >= t.first) { t.sink = t.first = 0; }
    t.count = t.sink + ((p1 + 32) >> 5) - t.first;
    return t;
}

// ---- one wave: 16 NT query rows against 32 keys straight from the cache -------------------------
//
// S^T = K Q^T and O^T = V^T P^T on 16x16x32 MFMAs. Lane (c, g) = (lane & 15, lane >> 4) loads row c of each half
// tile's K in 16-byte pieces (piece i of a quarter g: the MFMA steps run over the dims in the order the pieces leave
// them, and Q follows), and four bytes (INT8; BF16: sixteen) of the V rows 4g .. 4g + 3 of both halves, the keys
// whose scores the S^T accumulator leaves in this lane; so P needs no exchange between lanes, and V is transposed
// by byte selects alone. No LDS in the loop.

template <int D, bool BF>
struct Chunk {
    static constexpr int KP = BF ? D / 32 : D / 64; // K pieces of a lane and half
    static constexpr int VP = BF ? D / 128 : D / 64; // V pieces of a lane and key
    static constexpr int VW = BF ? 4 : 1;            // words of a V piece
    static constexpr int SW = BF ? 1 : D / 128;      // 16-byte words of four keys' scales
    u4 k[2][KP];
    uint32_t v[8][VP][VW];
    u4 ks[2][SW];
    u4 vs[2][SW];
};

// What a chunk's loads are aimed at: the 16-row halves' pages (-1: none).
struct Halves {
    int32_t page[2];
};

template <int D, bool BF>
__device__ __forceinline__ void load_chunk(const PagedAttnArgs& x, int h, int tile, Halves hv, int c, int g, Chunk<D, BF>& r) {
    using CK = Chunk<D, BF>;
    constexpr int kRow = BF ? 2 * D : D;
    constexpr int kScaleRow = D / 32; // bytes of a row's scales
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        // an absent half loads nothing (a buffer of no bytes): zeros
        const bool there = hv.page[kt] >= 0;
        const int64_t page = there ? hv.page[kt] : 0;
        const int64_t row = (static_cast<int64_t>(h) << x.c.page_shift) + ((32 * tile + 16 * kt) & ((1 << x.c.page_shift) - 1));
        const __amdgpu_buffer_rsrc_t kb = raw_buffer(x.c.k + page * x.c.k_page + row * kRow, there ? 16 * kRow : 0);
        const __amdgpu_buffer_rsrc_t vb = raw_buffer(x.c.v + page * x.c.v_page + row * kRow, there ? 16 * kRow : 0);
#pragma unroll
        for (int i = 0; i < CK::KP; ++i) {
            r.k[kt][i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(kb, c * kRow + 64 * i + 16 * g, 0, 2));
        }
        if constexpr (!BF) {
            const __amdgpu_buffer_rsrc_t ksb = raw_buffer(x.c.ks + page * x.c.ks_page + row * kScaleRow, there ? 16 * kScaleRow : 0);
            const __amdgpu_buffer_rsrc_t vsb = raw_buffer(x.c.vs + page * x.c.vs_page + row * kScaleRow, there ? 16 * kScaleRow : 0);
#pragma unroll
            for (int w = 0; w < CK::SW; ++w) {
                r.ks[kt][w] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(ksb, 4 * g * kScaleRow + 16 * w, 0, 0));
                r.vs[kt][w] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vsb, 4 * g * kScaleRow + 16 * w, 0, 0));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < CK::VP; ++i) {
                if constexpr (BF) {
                    const u4 w = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vb, (4 * g + j) * kRow + 256 * i + 16 * c, 0, 2));
#pragma unroll
                    for (int e = 0; e < 4; ++e) { r.v[4 * kt + j][i][e] = w[e]; }
                } else {
                    r.v[4 * kt + j][i][0] = __builtin_amdgcn_raw_buffer_load_b32(vb, (4 * g + j) * kRow + 64 * i + 4 * c, 0, 2);
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
            r.rowmul[nt] = ldexpf(x.scale_log2, -fexp);
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

// Whether a token at `pos` sees row `key` (of an existing page).
__device__ __forceinline__ bool sees(const PagedAttnArgs& x, int pos, int key) {
    return key <= pos && (x.a.window == 0 || pos - key < x.a.window || key < x.a.sinks);
}

// Whether every row of the wave sees all 32 keys of the tile.
__device__ __forceinline__ bool all_seen(const PagedAttnArgs& x, int lo, int hi, int tile, Halves hv) {
    const int k0 = 32 * tile, k1 = k0 + 31;
    return hv.page[0] >= 0 && hv.page[1] >= 0 && k1 <= lo && (x.a.window == 0 || hi - k0 < x.a.window || k1 < x.a.sinks);
}

// An infinite or NaN BF16 in either half of a word: that half's sign bit (of the result) set.
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

template <int D, bool BF, int NT>
__device__ __forceinline__ void attend_chunk(const PagedAttnArgs& x, int tile, Halves hv, int c, int g, Chunk<D, BF>& r, Rows<D, BF, NT>& s) {
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
    uint32_t seen[NT]; // bit i: row nt's lane sees key i (masked chunks)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { seen[nt] = 0xffu; }
    if (!whole) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            seen[nt] = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool ok = hv.page[i >> 2] >= 0 && sees(x, s.pos[nt], 32 * tile + 16 * (i >> 2) + 4 * g + (i & 3));
                seen[nt] |= ok ? 1u << i : 0u;
                sv[nt][i] = ok ? sv[nt][i] : -INFINITY;
            }
        }
        // keys that no row of the wave may see: whatever their rows hold is taken out
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool dead = hv.page[i >> 2] < 0 || 32 * tile + 16 * (i >> 2) + 4 * g + (i & 3) > s.hi;
            if constexpr (BF) {
#pragma unroll
                for (int w = 0; w < CK::VP; ++w) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) { r.v[i][w][e] = dead ? 0u : r.v[i][w][e]; }
                }
            } else {
#pragma unroll
                for (int w = 0; w < D / 128; ++w) {
                    if constexpr (D == 128) {
                        r.vs[i >> 2][0][i & 3] = dead ? 0u : r.vs[i >> 2][0][i & 3];
                    } else {
                        r.vs[i >> 2][(i & 3) >> 1][2 * (i & 1) + w] = dead ? 0u : r.vs[i >> 2][(i & 3) >> 1][2 * (i & 1) + w];
                    }
                }
            }
        }
    }
    // ---- running maximum (it moves only when a score tops it by 2^kLazyTau), probabilities, sums
    float p[NT][8];
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
        const float bias = s.m[nt] == -INFINITY ? 0.0f : fmaf(-s.m[nt], s.rowmul[nt], kPOffset);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[nt][i] = __builtin_amdgcn_exp2f(fmaf(sv[nt][i], s.rowmul[nt], bias));
        }
        s.l[nt] += ((p[nt][0] + p[nt][1]) + (p[nt][2] + p[nt][3])) + ((p[nt][4] + p[nt][5]) + (p[nt][6] + p[nt][7]));
    }
    // ---- values
    if constexpr (!BF) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            float sc[8];
            float top = 0.0f; // the largest finite scale of the chunk's keys, in group i
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                sc[k] = scale_of<D>(r.vs[k >> 2], k & 3, i);
                const float a = fabsf(sc[k]);
                top = fmaxf(top, a < INFINITY ? a : 0.0f);
            }
            top = group4_max(top);
            // 2^E > top; FP16 scales have exponents of -24 to 15
            const int E = static_cast<int>(__float_as_uint(top) >> 23) - 126;
            const float down = top > 0.0f ? __uint_as_float(static_cast<uint32_t>(127 - E) << 23) : 1.0f;
            const float up = top > 0.0f ? __uint_as_float(static_cast<uint32_t>(127 + E) << 23) : 1.0f;
            h8 w[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float y = p[nt][k] * (sc[k] * down);
                    if (!whole) { y = ((seen[nt] >> k) & 1u) ? y : 0.0f; } // an unseen row's scale may be anything
                    w[nt][k] = static_cast<_Float16>(y);
                }
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
                    for (int e = 0; e < 4; ++e) { s.O[nt][4 * i + Bt][e] = fmaf(o[e], up, s.O[nt][4 * i + Bt][e]); }
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
                hi[nt][k] = static_cast<__bf16>(p[nt][k]);
                lo[nt][k] = static_cast<__bf16>(p[nt][k] - static_cast<float>(hi[nt][k]));
            }
        }
        uint32_t odd = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
#pragma unroll
            for (int i = 0; i < CK::VP; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) { odd |= nonfinite_bits(r.v[k][i][e]); }
            }
        }
        const bool care = __any(odd != 0u);
        if (__builtin_expect(care, 0)) {
            // infinite and NaN values: counted apart (+: infinity or NaN, -: the same with the other sign) for the
            // rows that see them, and left out of the products
            h8 one[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int k = 0; k < 8; ++k) { one[nt][k] = ((seen[nt] >> k) & 1u) ? static_cast<_Float16>(1.0f) : static_cast<_Float16>(0.0f); }
            }
#pragma unroll
            for (int i = 0; i < CK::VP; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h8 up, dn;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t y = r.v[k][i][e >> 1];
                        const uint32_t z = ((e & 1) ? y >> 16 : y) & 0xffffu;
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
                    for (int e = 0; e < 4; ++e) { r.v[k][i][e] &= ~((nonfinite_bits(r.v[k][i][e]) >> 15) * 0xffffu); }
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

constexpr int kFewWaves = 4;
constexpr int kFewThreads = 64 * kFewWaves;
constexpr int kUnit = 4; // tiles of a split's unit: one for each wave

// The units of sequence b's keys that the few-row kernel walks (0: not its sequence).
__device__ __forceinline__ int few_units(const PagedAttnArgs& x, int b, Seq& s, Tiles& t) {
    s = sequence(x, b);
    if (s.tokens == 0 || s.tokens * x.G > x.few_rows) { return 0; }
    t = tiles_of(x, s.history, s.history + s.tokens - 1);
    return (t.count + kUnit - 1) / kUnit;
}

struct FewWork {
    int b;      // -1: none
    int first;  // the sequence's first slot
    int split;
    int splits;
    int units;  // of the sequence
};

// The split of `slot`: the shortest split length u (in units) for which all sequences' splits, ceil(units / u) of each,
// fit the slots. Every wave works it out alone (64 sequences and 64 candidates at a time).
__device__ __forceinline__ FewWork few_work(const PagedAttnArgs& x, int slot, int lane) {
    const int B = x.c.B;
    Seq s;
    Tiles t;
    int total = 0, active = 0;
    int units = 0; // of sequence `lane` of the last 64
    for (int base = 0; base < B; base += 64) {
        units = base + lane < B ? few_units(x, base + lane, s, t) : 0;
        total += __builtin_amdgcn_readlane(wave_inclusive_scan(units), 63);
        active += __popcll(__ballot(units > 0));
    }
    FewWork w{-1, 0, 0, 0, 0};
    if (active == 0) { return w; }
    const int lo = max(x.min_units, (total + x.slots - 1) / x.slots);
    const int spare = x.slots - active; // the host gives more slots than sequences
    const int hi = max(lo, (total + spare - 1) / spare);
    int u = lo;
    if (hi > lo && active > 1) {
        const int step = (hi - lo + 62) / 63;
        const int mine = lo + lane * step;
        const float inv = 1.0f / static_cast<float>(mine);
        int need = 0;
        for (int base = 0; base < B; base += 64) {
            if (B > 64) { units = base + lane < B ? few_units(x, base + lane, s, t) : 0; }
            const int n = min(64, B - base);
            for (int i = 0; i < n; ++i) {
                const int v = __builtin_amdgcn_readlane(units, i);
                need += static_cast<int>((static_cast<float>(v + mine - 1) + 0.5f) * inv);
            }
        }
        const uint64_t fits = __ballot(need <= x.slots);
        u = fits ? lo + (__ffsll(static_cast<long long>(fits)) - 1) * step : hi;
    }
    // the prefix sums of the sequences' splits; should the estimate above have been one off, `hi` fits for certain
    for (;;) {
        int sum = 0;
        w.b = -1;
        for (int base = 0; base < B; base += 64) {
            if (B > 64) { units = base + lane < B ? few_units(x, base + lane, s, t) : 0; }
            const int n = (units + u - 1) / u;
            const int end = sum + wave_inclusive_scan(n);
            const uint64_t mine = __ballot(n > 0 && slot >= end - n && slot < end);
            if (mine != 0u) {
                const int at = __ffsll(static_cast<long long>(mine)) - 1;
                w.b = base + at;
                w.splits = __builtin_amdgcn_readlane(n, at);
                w.first = __builtin_amdgcn_readlane(end, at) - w.splits;
                w.split = slot - w.first;
                w.units = __builtin_amdgcn_readlane(units, at);
            }
            sum = __builtin_amdgcn_readlane(end, 63);
        }
        if (sum <= x.slots || u >= hi) { break; }
        u = hi;
    }
    return w;
}

// Waves per SIMD: one where two would not hold the chunk in flight, the chunk at hand and the accumulators.
constexpr int few_waves(int D, bool, int NT) { return D == 128 && NT == 1 ? 2 : 1; }

template <int D, bool BF, int NT>
__global__ __launch_bounds__(kFewThreads) __attribute__((amdgpu_waves_per_eu(few_waves(D, BF, NT), few_waves(D, BF, NT)))) void paged_attn_few_kernel(PagedAttnArgs x) {
    // two waves' O and (m, l) at a time
    __shared__ f4 xo[2][NT * (D / 16) * 64];
    __shared__ float2 xm[2][NT * 64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int h = blockIdx.x % x.c.Hkv;
    const FewWork w = few_work(x, blockIdx.x / x.c.Hkv, lane);
    if (w.b < 0) { return; }
    const Seq s = sequence(x, w.b);
    const Tiles tiles = tiles_of(x, s.history, s.history + s.tokens - 1);
    const int per = (w.units + w.splits - 1) / w.splits * kUnit; // tiles of a split
    const int t0 = min(w.split * per, tiles.count), t1 = min(t0 + per, tiles.count);
    const int each = (t1 - t0 + kFewWaves - 1) / kFewWaves;
    const int j0 = min(t0 + wave * each, t1), j1 = min(j0 + each, t1);
    const int rows = s.tokens * x.G;
    const int end = s.history + s.tokens;
    if (w.split == 0 && h == 0 && threadIdx.x == 0) {
        x.seq_table[2 * w.b] = w.first;
        x.seq_table[2 * w.b + 1] = w.splits;
    }
    Rows<D, BF, NT> r;
    // pages of 64 halves (32 tiles) at a time, one per lane, the next 64 fetched ahead
    const int32_t* table = x.c.table + w.b * x.c.table_row;
    const auto pages_from = [&](int j) {
        const int v = j + (lane >> 1);
        const int key = 32 * tiles.tile(v) + 16 * (lane & 1);
        int page = -1;
        if (v < j1 && key < end) { page = table[key >> x.c.page_shift]; }
        return page >= 0 && page < x.c.pages ? page : -1;
    };
    int ids = pages_from(j0), next_ids = pages_from(j0 + 32);
    const auto halves = [&](int j) { // of tile j in [j0, ...): past the end no page
        const int i = 2 * (j - j0);
        const int from = (i & 127) < 64 ? 0 : 1; // this or the next 64 (see the turn below)
        Halves hv;
        hv.page[0] = __builtin_amdgcn_readlane(from ? next_ids : ids, i & 63);
        hv.page[1] = __builtin_amdgcn_readlane(from ? next_ids : ids, (i & 63) + 1);
        return hv;
    };
    Chunk<D, BF> ca, cb;
    Halves ha = halves(j0), hb;
    load_chunk<D, BF>(x, h, tiles.tile(j0), ha, c, g, ca);
    init_rows<D, BF, NT>(x, s, h, 0, c, g, r);
#pragma unroll 1
    for (int j = j0; j < j1; j += 2) {
        const int in = (j - j0) & 63; // 0 .. 62: two fetches of 32 tiles
        hb = halves(j + 1);
        load_chunk<D, BF>(x, h, tiles.tile(j + 1), hb, c, g, cb);
        attend_chunk<D, BF, NT>(x, tiles.tile(j), ha, c, g, ca, r);
        // tiles j + 2 .. : past the 32nd of this fetch the other one is refilled
        if (in == 30) { ids = pages_from(j + 34); }
        if (in == 62) { next_ids = pages_from(j + 34); }
        ha = halves(j + 2);
        load_chunk<D, BF>(x, h, tiles.tile(j + 2), ha, c, g, ca);
        if (j + 1 < j1) { attend_chunk<D, BF, NT>(x, tiles.tile(j + 1), hb, c, g, cb, r); }
    }
    // ---- the four waves' states into wave 0's: 2 and 3 into 0 and 1, then 1 into 0
    float M[NT], L[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        M[nt] = r.m[nt] == -INFINITY ? -INFINITY : r.m[nt] * r.rowmul[nt];
        L[nt] = group4_sum(r.l[nt]);
    }
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
                const float Mx = fmaxf(M[nt], o.x);
                const float a = M[nt] == -INFINITY ? (L[nt] == L[nt] ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(M[nt] - Mx);
                const float b = o.x == -INFINITY ? (o.y == o.y ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(o.x - Mx);
                L[nt] = L[nt] * a + o.y * b;
                M[nt] = Mx;
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    const f4 y = xo[wave][(nt * (D / 16) + t) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // a part without weight adds nothing, whatever it holds
                        r.O[nt][t][e] = (a == 0.0f ? 0.0f : r.O[nt][t][e] * a) + (b == 0.0f ? 0.0f : y[e] * b);
                    }
                }
            }
        }
    };
    halve(2);
    __syncthreads();
    halve(1);
    if (wave != 0) { return; }
    constexpr int RUN = BF ? 8 : 4; // consecutive dims of a lane
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = 16 * nt + c;
        if (row >= rows) { continue; }
        if (w.splits > 1) {
            const int64_t at = (static_cast<int64_t>(w.first + w.split) * x.c.Hkv + h) * (16 * NT) + row;
#pragma unroll
            for (int i = 0; i < D / (16 * RUN); ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float* dst = x.part_o + at * D + out_dim<BF>(RUN * i, 4 * g + e);
#pragma unroll
                    for (int q = 0; q < RUN; q += 4) {
                        *reinterpret_cast<f4*>(dst + q) = f4{r.O[nt][RUN * i + q][e], r.O[nt][RUN * i + q + 1][e], r.O[nt][RUN * i + q + 2][e], r.O[nt][RUN * i + q + 3][e]};
                    }
                }
            }
            if (g == 0) { *reinterpret_cast<float2*>(x.part_ml + 2 * at) = float2{M[nt], L[nt]}; }
        } else {
            const int t = row / x.G;
            const float inv = L[nt] == 0.0f ? 0.0f : 1.0f / L[nt];
            uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + (s.start + t) * x.a.out.token_stride) + (h * x.G + row - t * x.G) * D;
#pragma unroll
            for (int i = 0; i < D / (16 * RUN); ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t y[RUN / 2];
#pragma unroll
                    for (int q = 0; q < RUN / 2; ++q) {
                        const float o0 = L[nt] == 0.0f ? 0.0f : r.O[nt][RUN * i + 2 * q][e] * inv;
                        const float o1 = L[nt] == 0.0f ? 0.0f : r.O[nt][RUN * i + 2 * q + 1][e] * inv;
                        y[q] = static_cast<uint32_t>(f32_to_bf16_bits(o0)) | (static_cast<uint32_t>(f32_to_bf16_bits(o1)) << 16);
                    }
                    __builtin_memcpy(__builtin_assume_aligned(out + out_dim<BF>(RUN * i, 4 * g + e), RUN * 2), y, sizeof(y));
                }
            }
        }
    }
}

// Log-sum-exp merge of a row's splits: a workgroup per row, groups of D / 4 threads taking every group-th split.
template <int D>
__global__ __launch_bounds__(256) void paged_attn_merge_kernel(PagedAttnArgs x, int slot_rows) {
    constexpr int TPR = D / 4, GRP = 256 / TPR;
    __shared__ f4 xo[GRP][TPR];
    __shared__ float2 xm[GRP];
    const int b = blockIdx.y;
    const int row = blockIdx.x / x.c.Hkv;
    const int h = blockIdx.x % x.c.Hkv;
    const Seq s = sequence(x, b);
    const int rows = s.tokens * x.G;
    if (rows > x.few_rows || row >= rows) { return; }
    const int first = x.seq_table[2 * b], splits = x.seq_table[2 * b + 1];
    if (splits == 1) { return; } // written already
    const int grp = threadIdx.x / TPR, d = 4 * (threadIdx.x % TPR);
    float M = -INFINITY, L = 0.0f;
    f4 O = {0.f, 0.f, 0.f, 0.f};
    const auto add = [&](float m, float l, f4 o) {
        const float Mx = fmaxf(M, m);
        const float a = M == -INFINITY ? (L == L ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(M - Mx);
        const float q = m == -INFINITY ? (l == l ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - Mx);
        L = L * a + l * q;
#pragma unroll
        for (int e = 0; e < 4; ++e) { O[e] = (a == 0.0f ? 0.0f : O[e] * a) + (q == 0.0f ? 0.0f : o[e] * q); }
        M = Mx;
    };
#pragma unroll 4
    for (int k = grp; k < splits; k += GRP) {
        const int64_t at = (static_cast<int64_t>(first + k) * x.c.Hkv + h) * slot_rows + row;
        const float2 ml = *reinterpret_cast<const float2*>(x.part_ml + 2 * at);
        add(ml.x, ml.y, *reinterpret_cast<const f4*>(x.part_o + at * D + d));
    }
    xo[grp][threadIdx.x % TPR] = O;
    if (threadIdx.x % TPR == 0) { xm[grp] = float2{M, L}; }
    __syncthreads();
    if (grp != 0) { return; }
#pragma unroll
    for (int k = 1; k < GRP; ++k) { add(xm[k].x, xm[k].y, xo[k][threadIdx.x]); }
    const int t = row / x.G;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint16_t* out = reinterpret_cast<uint16_t*>(x.a.out.data + (s.start + t) * x.a.out.token_stride) + (h * x.G + row - t * x.G) * D + d;
    uint32_t y[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const float o0 = L == 0.0f ? 0.0f : O[2 * q] * inv;
        const float o1 = L == 0.0f ? 0.0f : O[2 * q + 1] * inv;
        y[q] = static_cast<uint32_t>(f32_to_bf16_bits(o0)) | (static_cast<uint32_t>(f32_to_bf16_bits(o1)) << 16);
    }
    *reinterpret_cast<u2*>(out) = u2{y[0], y[1]};
}

// One workgroup per (token, query head).
template <int D, bool BF>
__global__ __launch_bounds__(256) void paged_attn_row_kernel(PagedAttnArgs x) {
    __shared__ float xq[D], xp[256], xr[8], xv[256 / (D / 4)][D];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t n = blockIdx.x / x.a.Hq;
    const int qh = static_cast<int>(blockIdx.x % x.a.Hq);
    const int h = qh / x.G;
    int lo = 0, hi = x.c.B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (x.a.starts[mid] <= n) { lo = mid; } else { hi = mid; }
    }
    const Seq s = sequence(x, lo);
    if (n < s.start || n >= s.start + s.tokens || s.tokens * x.G <= x.few_rows) { return; }
    const int p = s.history + static_cast<int>(n - s.start);
    const int first = x.a.window > 0 ? max(0, p + 1 - x.a.window) : 0;
    const int nsink = min(x.a.sinks, first);
    const int keys = nsink + p + 1 - first;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(x.a.q.data + n * x.a.q.token_stride) + qh * D;
    if (tid < D) { xq[tid] = bf16_to_f32(q[tid]) * x.scale_log2; }
    __syncthreads();
    const int32_t* table = x.c.table + lo * x.c.table_row;
    const int mask = (1 << x.c.page_shift) - 1;
    const auto where = [&](int i, int& page) {
        const int key = i < nsink ? i : first + i - nsink;
        const int slot = key >> x.c.page_shift;
        page = slot < x.c.max_pages ? table[slot] : -1;
        page = page >= 0 && page < x.c.pages ? page : -1;
        return (h << x.c.page_shift) + (key & mask);
    };
    float M = -INFINITY, L = 0.0f;
    f4 O = {0.f, 0.f, 0.f, 0.f};
    constexpr int TPR = D / 4, PARTS = 256 / TPR;
    const int d4 = 4 * (tid % TPR), part = tid / TPR;
    for (int base = 0; base < keys; base += 256) {
        float sc = -INFINITY;
        int page;
        if (base + tid < keys) {
            const int64_t row = where(base + tid, page);
            if (page >= 0) {
                sc = 0.0f;
                const char* kp = x.c.k + page * x.c.k_page + row * D * (BF ? 2 : 1);
                for (int d = 0; d < D; ++d) {
                    float k;
                    if constexpr (BF) {
                        k = bf16_to_f32(reinterpret_cast<const uint16_t*>(kp)[d]);
                    } else {
                        k = static_cast<float>(reinterpret_cast<const int8_t*>(kp)[d]) *
                            f16_bits_to_f32(reinterpret_cast<const uint16_t*>(x.c.ks + page * x.c.ks_page)[row * (D / 64) + d / 64]);
                    }
                    sc = fmaf(xq[d], k, sc);
                }
            }
        }
        const float wm = wave_max(sc);
        if (lane == 0) { xr[wave] = wm; }
        __syncthreads();
        float Mn = M;
        for (int w = 0; w < 4; ++w) { Mn = fmaxf(Mn, xr[w]); }
        const float alpha = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
        const float pr = sc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sc - Mn);
        xp[tid] = pr;
        const float ws = wave_sum(pr);
        if (lane == 0) { xr[4 + wave] = ws; }
        __syncthreads();
        L = fmaf(L, alpha, xr[4] + xr[5] + xr[6] + xr[7]);
        O *= alpha;
        for (int i = part; i < 256; i += PARTS) {
            if (base + i >= keys) { break; }
            const int64_t row = where(base + i, page);
            if (page < 0) { continue; }
            const char* vp = x.c.v + page * x.c.v_page + row * D * (BF ? 2 : 1);
            float s8 = 1.0f;
            if constexpr (!BF) { s8 = f16_bits_to_f32(reinterpret_cast<const uint16_t*>(x.c.vs + page * x.c.vs_page)[row * (D / 64) + d4 / 64]); }
            for (int e = 0; e < 4; ++e) {
                const float v = BF ? bf16_to_f32(reinterpret_cast<const uint16_t*>(vp)[d4 + e])
                                   : static_cast<float>(reinterpret_cast<const int8_t*>(vp)[d4 + e]) * s8;
                O[e] = fmaf(xp[i], v, O[e]);
            }
        }
        M = Mn;
        __syncthreads();
    }
    *reinterpret_cast<f4*>(&xv[part][d4]) = O;
    __syncthreads();
    if (tid < D) {
        float o = 0.0f;
        for (int w = 0; w < PARTS; ++w) { o += xv[w][tid]; }
        o = L > 0.0f || L != L ? o / L : 0.0f;
        (reinterpret_cast<uint16_t*>(x.a.out.data + n * x.a.out.token_stride) + qh * D)[tid] = f32_to_bf16_bits(o);
    }
}

} // namespace

namespace {

// How a call is cut. Few-row slots: two workgroups of the kernel fill a CU.
struct PagedPlan {
    int32_t nt = 1;        // 16-row tiles of a few-row workgroup
    int32_t few_rows = 0;
    int32_t slots = 0;
    int32_t min_units = 2;
    bool merge = false;
    size_t ml_offset = 0;
    size_t table_offset = 0;
    size_t bytes = 0;
};

PagedPlan plan_paged(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t max_new, int32_t max_keys, int32_t window,
                     int32_t sinks) {
    const int32_t G = Hq / Hkv;
    PagedPlan p;
    p.nt = static_cast<int64_t>(max_new) * G <= 16 ? 1 : 2;
    p.few_rows = 16 * p.nt;
    // the most tiles that a few-row sequence walks
    int64_t keys = max_keys;
    if (window > 0) {
        const int64_t most = static_cast<int64_t>(window) + std::min<int64_t>(max_new, p.few_rows) + 62 + (static_cast<int64_t>(sinks) + 31) / 32 * 32;
        keys = std::min(keys, most);
    }
    const int64_t units = (keys + 127) / 128;
    if (units <= p.min_units) {
        p.slots = B + 1;
    } else {
        p.slots = static_cast<int32_t>(std::max<int64_t>(std::min<int64_t>(512 / Hkv, B * ((units + p.min_units - 1) / p.min_units)), 2 * B));
        p.merge = true;
    }
    size_t at = 0;
    if (p.merge) {
        const size_t rows = static_cast<size_t>(p.slots) * Hkv * p.few_rows;
        at = rows * D * sizeof(float);
        p.ml_offset = at;
        at += rows * 2 * sizeof(float);
    }
    p.table_offset = at;
    p.bytes = at + static_cast<size_t>(B) * 2 * sizeof(int32_t);
    return p;
}

template <int D, bool BF>
void launch(PagedAttnArgs& x, const PagedPlan& p, hipStream_t stream) {
    const uint32_t grid = static_cast<uint32_t>(p.slots) * x.c.Hkv;
    if (p.nt == 1) {
        hipLaunchKernelGGL((paged_attn_few_kernel<D, BF, 1>), dim3(grid), dim3(kFewThreads), 0, stream, x);
    } else {
        hipLaunchKernelGGL((paged_attn_few_kernel<D, BF, 2>), dim3(grid), dim3(kFewThreads), 0, stream, x);
    }
    check_launch("paged_attn_few_kernel");
    if (p.merge) {
        hipLaunchKernelGGL((paged_attn_merge_kernel<D>), dim3(p.few_rows * x.c.Hkv, x.c.B), dim3(256), 0, stream, x, p.few_rows);
        check_launch("paged_attn_merge_kernel");
    }
    if (static_cast<int64_t>(x.a.max_new) * x.G > p.few_rows) {
        const int64_t blocks = x.a.tokens * x.a.Hq;
        if (blocks > 0x7FFFFFFF) { throw Unsupported("paged attention: more than 2^31 query rows are not built"); }
        hipLaunchKernelGGL((paged_attn_row_kernel<D, BF>), dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream, x);
        check_launch("paged_attn_row_kernel");
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
    x.c = c;
    x.G = a.Hq / c.Hkv;
    x.scale_log2 = a.scale * 1.4426950408889634f;
    x.few_rows = p.few_rows;
    x.slots = p.slots;
    x.min_units = p.min_units;
    char* ws = static_cast<char*>(workspace);
    x.part_o = reinterpret_cast<float*>(ws);
    x.part_ml = reinterpret_cast<float*>(ws + p.ml_offset);
    x.seq_table = reinterpret_cast<int32_t*>(ws + p.table_offset);
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
