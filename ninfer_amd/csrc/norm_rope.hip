// Head norms of queries and keys with the rotation by position in the same pass on gfx950; on its way into a paged KV
// cache, the keys (and the values) are appended in that pass too.
//
// Mathematics: for every head x of a token at position p, y = x / sqrt(mean(x^2) + eps) * (weight + offset); pair i of the
// rotated dims, (a, b) = (y[i], y[i + half]) or interleaved (y[2i], y[2i + 1]), becomes (a cos t - b sin t, b cos t + a sin t)
// with t = p * inv_freq[i]; one rounding to BF16 at the end. The append is that of paged_cache.hip, to the bit.
//
// Numbers: t in turns is p * (inv_freq / 2 pi) in 64 bits, less its nearest whole number, so a far position loses nothing (in
// 32 bits a position of 2^23 would be half a radian off); sine and cosine of what is left are FP32, the sum of squares too,
// scaled down first where it passes FP32's range.
//
// What bounds it: HBM for prompts (8,192 tokens at 24/4/256 54 us, 4.3 TB/s; 4,187 tokens of five prompts into a BF16 cache 29 us,
// 4.7 TB/s), with the VALU busy 79% of the time; launch and the chain token -> sequence -> page for decode steps (16 tokens 6 us).
#include "common.h"
#include "device_utils.h"
#include "kv_codec.h"
#include "paged_internal.h"

#include <algorithm>

namespace nmi {
namespace {

struct NormRopeArgs {
    NormRope a;
    PagedRef c;
};

// The sum over the D / 8 lanes of a head, in every one of them.
template <int D>
__device__ __forceinline__ float head_sum(float v) {
    v += dpp_from<0xB1, 0xf>(v, 0.0f);  // lane ^ 1
    v += dpp_from<0x4E, 0xf>(v, 0.0f);  // lane ^ 2
    v += dpp_from<0x141, 0xf>(v, 0.0f); // the other four of eight
    v += dpp_from<0x140, 0xf>(v, 0.0f); // the other eight of sixteen
    if constexpr (D == 256) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

__device__ __forceinline__ float bf16_of(i4 raw, int e) {
    const uint32_t w = static_cast<uint32_t>(raw[e >> 1]);
    return __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
}

// Eight weights from dim d on, the offset added.
__device__ __forceinline__ void load_weights(const void* w, bool f32, float offset, int d, float (&y)[8]) {
    if (w == nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { y[e] = 1.0f + offset; }
    } else if (f32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { y[e] = static_cast<const float*>(w)[d + e] + offset; }
    } else {
        const i4 raw = *reinterpret_cast<const i4*>(static_cast<const uint16_t*>(w) + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) { y[e] = bf16_of(raw, e) + offset; }
    }
}

// Two FP32 values rounded to BF16, the first in the low half (v_cvt_pk_bf16_f32).
__device__ __forceinline__ int bf16_pair(float lo, float hi) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(int, b2{static_cast<__bf16>(lo), static_cast<__bf16>(hi)});
}

// What a lane's eight dims of a head become: x own + y other, x its normalised values and y its partners' (its own ones, times
// zero, where nothing is rotated).
struct Turn {
    float own[8];
    float other[8];
};

// A workgroup per token (and share of its heads): D / 8 lanes a head, eight dims a lane, so a wave holds HEADS heads. Queries, keys
// and values are dealt out in runs of HEADS, so that a wave's heads are of one kind and their weights (times sines and cosines, once
// per token) come from registers without a choice per value.
//
// Two waves a workgroup: more waves wait for the token's sines and cosines together (8,192 tokens at 24/4/256 with one, two, four and
// eight waves 65.8, 56.5, 61.9 and 72.2 us).
constexpr int kWaves = 2;
constexpr int kThreads = 64 * kWaves;

template <bool STREAM, typename T>
__device__ __forceinline__ void put(char* to, T v) {
    if constexpr (STREAM) {
        __builtin_nontemporal_store(v, reinterpret_cast<T*>(to));
    } else {
        *reinterpret_cast<T*>(to) = v;
    }
}

template <int D, bool APPEND, bool STREAM>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs x) {
    constexpr int L = D / 8;      // lanes of a head
    constexpr int HEADS = 64 / L; // heads of a wave
    __shared__ float2 turn[D / 2];
    const NormRope& a = x.a;
    const int64_t n = blockIdx.x;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & (L - 1);
    const int q_runs = (a.Hq + HEADS - 1) / HEADS, kv_runs = (a.Hkv + HEADS - 1) / HEADS;
    const int runs = q_runs + kv_runs * (APPEND ? 2 : 1);
    const int step = kWaves * gridDim.y;
    // run i: its tensor, the lane's head there and whether there is one
    struct Run {
        int kind; // 0 queries, 1 keys, 2 values
        int head;
        bool live;
    };
    const auto run_of = [&](int i) {
        const int kind = i < q_runs ? 0 : i < q_runs + kv_runs ? 1 : 2;
        const int head = (i - (kind == 0 ? 0 : kind == 1 ? q_runs : q_runs + kv_runs)) * HEADS + lane / L;
        return Run{kind, head, i < runs && head < (kind == 0 ? a.Hq : a.Hkv)};
    };
    const auto load = [&](const Run& r) {
        const PackedRef& src = r.kind == 0 ? a.q : r.kind == 1 ? a.k : a.v;
        return r.live ? *reinterpret_cast<const i4*>(src.data + n * src.token_stride + (r.head * D + 8 * li) * 2) : i4{0, 0, 0, 0};
    };
    int at = blockIdx.y * kWaves + wave;
    Run run = run_of(at);
    i4 raw = load(run);

    int64_t pos;
    int32_t page = -1, row = 0;
    if constexpr (APPEND) {
        // the last sequence that starts at or before the token
        int count = 0;
        for (int i = threadIdx.x; i - static_cast<int>(threadIdx.x) < x.c.B; i += kThreads) { count += __syncthreads_count(i < x.c.B && a.starts[i] <= n); }
        if (count == 0) { return; }
        const int b = count - 1;
        const int32_t start = a.starts[b], end = a.starts[b + 1], history = a.history[b];
        if (start < 0 || n < start || n >= end || history < 0) { return; } // of no sequence
        pos = static_cast<int64_t>(history) + (n - start);
        if ((pos >> x.c.page_shift) < x.c.max_pages) {
            page = x.c.table[b * x.c.table_row + (pos >> x.c.page_shift)];
            page = page >= 0 && page < x.c.pages ? page : -1;
            row = static_cast<int32_t>(pos & ((int64_t{1} << x.c.page_shift) - 1));
        }
    } else {
        pos = a.positions[n];
    }
    for (int i = threadIdx.x; i < a.half; i += kThreads) {
        double t = static_cast<double>(pos) * (static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577);
        t -= rint(t);
        float s, c;
        sincospif(static_cast<float>(2.0 * t), &s, &c);
        turn[i] = float2{c, s};
    }
    // the lane's dims and its partner's
    const int lanes = a.half / 8; // lanes of half a rotated part
    const bool rotated = 8 * li < 2 * a.half;
    const bool upper = !a.interleaved && li >= lanes; // b of its pairs
    const int partner = !rotated || a.interleaved ? li : upper ? li - lanes : li + lanes;
    const int from = 4 * ((lane & ~(L - 1)) + partner);
    Turn q, k;
    load_weights(a.q_weight, a.q_weight_f32, a.offset, 8 * li, q.own);
    load_weights(a.k_weight, a.k_weight_f32, a.offset, 8 * li, k.own);
    load_weights(a.q_weight, a.q_weight_f32, a.offset, 8 * partner, q.other);
    load_weights(a.k_weight, a.k_weight_f32, a.offset, 8 * partner, k.other);
    __syncthreads();
    if (a.interleaved) { // a dim's partner stands next to it
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            q.other[e] = q.own[e + 1];
            q.other[e + 1] = q.own[e];
            k.other[e] = k.own[e + 1];
            k.other[e + 1] = k.own[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float c = 1.0f, s = 0.0f;
        if (rotated) {
            const float2 z = turn[a.interleaved ? 4 * li + (e >> 1) : 8 * (upper ? li - lanes : li) + e];
            c = z.x;
            s = (a.interleaved ? (e & 1) != 0 : upper) ? z.y : -z.y;
        }
        q.own[e] *= c;
        k.own[e] *= c;
        // (an infinite weight times zero would be no number)
        q.other[e] = rotated ? q.other[e] * s : 0.0f;
        k.other[e] = rotated ? k.other[e] * s : 0.0f;
    }

    while (at < runs) {
        at += step;
        const Run after = run_of(at);
        const i4 next = load(after);
        i4 out = raw;
        if (run.kind < 2) {
            float v[8];
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = bf16_of(raw, e);
                ss = fmaf(v[e], v[e], ss);
            }
            ss = head_sum<D>(ss);
            float r = __builtin_amdgcn_rsqf(fmaf(ss, 1.0f / D, a.eps));
            const bool huge = __any(ss > 0x1p120f);
            if (__builtin_expect(huge, 0)) { // beyond FP32's squares: 2^-70 of the values, eps is nothing next to them
                float s2 = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) { s2 = fmaf(v[e] * 0x1p-70f, v[e] * 0x1p-70f, s2); }
                s2 = head_sum<D>(s2);
                if (ss > 0x1p120f) { r = 0x1p-70f * __builtin_amdgcn_rsqf(s2 * (1.0f / D)); }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[e] *= r; }
            float z[8];
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; ++e) { z[e] = v[e ^ 1]; }
            } else {
                i4 other;
#pragma unroll
                for (int w = 0; w < 4; ++w) { other[w] = __builtin_amdgcn_ds_bpermute(from, raw[w]); }
#pragma unroll
                for (int e = 0; e < 8; ++e) { z[e] = bf16_of(other, e) * r; }
            }
            const auto apply = [&](const Turn& t) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) { y[e] = fmaf(v[e], t.own[e], z[e] * t.other[e]); }
#pragma unroll
                for (int w = 0; w < 4; ++w) { out[w] = bf16_pair(y[2 * w], y[2 * w + 1]); }
            };
            if (run.kind == 0) {
                apply(q);
            } else {
                apply(k);
            }
            if (__builtin_expect(huge && a.interleaved, 0)) { // an infinite value stays out of the dims next to it that do not turn with it
                const Turn& t = run.kind == 0 ? q : k;
#pragma unroll
                for (int w = 0; w < 4; ++w) { out[w] = rotated ? out[w] : bf16_pair(v[2 * w] * t.own[2 * w], v[2 * w + 1] * t.own[2 * w + 1]); }
            }
        }
        if (run.kind == 0) {
            if (run.live) { put<STREAM>(a.q_out.data + n * a.q_out.token_stride + (run.head * D + 8 * li) * 2, out); }
        } else if constexpr (!APPEND) {
            if (run.live) { put<STREAM>(a.k_out.data + n * a.k_out.token_stride + (run.head * D + 8 * li) * 2, out); }
        } else if (page >= 0) {
            const bool value = run.kind == 2;
            const int64_t to = (static_cast<int64_t>(run.head) << x.c.page_shift) + row;
            char* dst = value ? x.c.v + page * x.c.v_page : x.c.k + page * x.c.k_page;
            if (x.c.bf16) {
                if (run.live) { put<STREAM>(dst + (to * D + 8 * li) * 2, out); }
            } else {
                uint16_t scale;
                const i2 code = quantize_g64(out, scale);
                if (run.live) {
                    put<STREAM>(dst + to * D + 8 * li, code);
                    if ((li & 7) == 0) {
                        char* sdst = value ? x.c.vs + page * x.c.vs_page : x.c.ks + page * x.c.ks_page;
                        *reinterpret_cast<uint16_t*>(sdst + (to * (D / 64) + (li >> 3)) * 2) = scale;
                    }
                }
            }
        }
        run = after;
        raw = next;
    }
}

// Outputs of more than 64 MiB are written past the caches: together with a kernel that reads the queries right after, 8,192 tokens at
// 24/4/256 (112 MiB) take 91.7 us so and 99.7 us through the caches, 4,096 (56 MiB) 51.6 and 47.9, 1,024 (14 MiB) 16.8 and 16.1.
constexpr int64_t kCached = 64 << 20;

template <int D, bool APPEND>
void launch(const NormRopeArgs& x, hipStream_t stream) {
    constexpr int HEADS = 512 / D;
    const int runs = (x.a.Hq + HEADS - 1) / HEADS + (x.a.Hkv + HEADS - 1) / HEADS * (APPEND ? 2 : 1);
    // one token's heads over several workgroups where the tokens alone leave CUs idle
    const int shares = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((runs + kWaves - 1) / kWaves, 1024 / x.a.tokens)));
    const dim3 grid(static_cast<uint32_t>(x.a.tokens), shares);
    if (x.a.tokens * (x.a.Hq + (APPEND ? 2 : 1) * x.a.Hkv) * D * 2 > kCached) {
        hipLaunchKernelGGL((norm_rope_kernel<D, APPEND, true>), grid, dim3(kThreads), 0, stream, x);
    } else {
        hipLaunchKernelGGL((norm_rope_kernel<D, APPEND, false>), grid, dim3(kThreads), 0, stream, x);
    }
    check_launch("norm_rope_kernel");
}

} // namespace

void launch_norm_rope(const NormRope& a, const PagedRef* cache, hipStream_t stream) {
    NormRopeArgs x{};
    x.a = a;
    if (cache != nullptr) {
        x.c = *cache;
        a.D == 128 ? launch<128, true>(x, stream) : launch<256, true>(x, stream);
    } else {
        a.D == 128 ? launch<128, false>(x, stream) : launch<256, false>(x, stream);
    }
}

} // namespace nmi
