// What the kernels share that decode key tiles of a paged KV cache once for a workgroup of eight waves: a tile of 16,384
// values per plane in a double LDS buffer, and a wave's products over 32 of its keys. The mathematics and its roundings stand in
// paged_attention.hip.
#pragma once

#include "paged_walk.h"

#include <algorithm>
#include <type_traits>

namespace nmi {
namespace {

constexpr int kManyThreads = 512;

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

typedef short s4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u2 read_tr(const char* p) {
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((NMI_AS3 s4*)(p)));
}

// The products start from the running maximum's negative: scores come out less it (rounded with it, -m * mul would move
// every p by up to 2^(score 2^-25)). BF16 rows of 128 have no registers left for that: there it is added afterwards (8,192
// tokens 785 us, 816 with eight registers spilled).
template <int D, bool BF>
constexpr bool kFromRef = !(BF && D == 128);

// Online-softmax state of a wave's rows over decoded tiles, next to Rows' outputs. `lim`: what moves the maximum; -infinity
// before the first score.
template <int D, bool BF, int NT>
struct ManyState {
    float mul[NT]; // raw score of the FP16 K' -> log2 domain
    std::conditional_t<kFromRef<D, BF>, f4, float> ref[NT];
    float lim[NT];
    f4 l[NT];
};

// Chunk ci of the tile in `buf`: 32 keys from key c0 on, their halves' pages in hv. voff: the lane's place in V.
template <int D, bool BF, int NT>
__device__ __forceinline__ void many_chunk(const PagedAttnArgs& x, const char* buf, int ci, int c0, Halves hv, int c, int g, int voff, Rows<D, BF, NT>& r,
                                           ManyState<D, BF, NT>& s) {
    constexpr int VF = D == 128 ? 8 : 4; // V^T operands in flight
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
                if constexpr (kFromRef<D, BF>) { acc = s.ref[nt]; }
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
    const char* vp = buf + ManyGeo<D, 1>::kPlane + 32 * ci * 2 * D;
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
            if constexpr (!kFromRef<D, BF>) { sv[nt][i] += s.ref[nt]; }
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
        any |= cmax[nt] > s.lim[nt];
    }
    if (__any(any)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const bool need = cmax[nt] > s.lim[nt];
            const float up = need ? cmax[nt] : 0.0f;
            const float alpha = s.lim[nt] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-up * s.mul[nt]);
#pragma unroll
            for (int t = 0; t < D / 16; ++t) { r.O[nt][t] *= alpha; }
            s.l[nt] *= alpha;
            s.ref[nt] -= up;
#pragma unroll
            for (int i = 0; i < 8; ++i) { sv[nt][i] -= up; }
            s.lim[nt] = need ? kLazyTau / s.mul[nt] : s.lim[nt];
        }
    }
    h8 p[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 8; ++i) { p[nt][i] = static_cast<_Float16>(__builtin_amdgcn_exp2f(fmaf(sv[nt][i], s.mul[nt], kPOffset))); }
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
    for (int nt = 0; nt < NT; ++nt) { s.l[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[nt], s.l[nt], 0, 0, 0); }
    __builtin_amdgcn_s_setprio(0);
}

} // namespace
} // namespace nmi
