// Attention of packed new tokens over a paged KV cache on gfx950.
//
// Mathematics: token i of sequence b stands at position p = history[b] + i and sees the rows j <= p of its
// sequence with p - j < window or j < sinks (every j <= p without a window) whose page exists;
// out = sum_j softmax_j(scale * q . K_j) V_j in one pass with a running maximum and sum, zero where no row is seen.
#include "attn_math.h"
#include "common.h"
#include "device_utils.h"
#include "paged_internal.h"

#include <algorithm>

namespace nmi {
namespace {

struct PagedAttnArgs {
    PagedAttention a;
    PagedRef c;
    int32_t G;
    float scale_log2;
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
    if (n < s.start || n >= s.start + s.tokens) { return; }
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

size_t paged_attention_bytes(int32_t, int32_t, int32_t, int64_t, int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

void launch_paged_attention(const PagedAttention& a, const PagedRef& c, void*, hipStream_t stream) {
    PagedAttnArgs x{};
    x.a = a;
    x.c = c;
    x.G = a.Hq / c.Hkv;
    x.scale_log2 = a.scale * 1.4426950408889634f;
    const int64_t blocks = a.tokens * a.Hq;
    if (blocks > 0x7FFFFFFF) { throw Unsupported("paged attention: more than 2^31 query rows are not built"); }
    const dim3 grid(static_cast<uint32_t>(blocks));
    if (c.D == 128 && !c.bf16) {
        hipLaunchKernelGGL((paged_attn_row_kernel<128, false>), grid, dim3(256), 0, stream, x);
    } else if (c.D == 128) {
        hipLaunchKernelGGL((paged_attn_row_kernel<128, true>), grid, dim3(256), 0, stream, x);
    } else if (!c.bf16) {
        hipLaunchKernelGGL((paged_attn_row_kernel<256, false>), grid, dim3(256), 0, stream, x);
    } else {
        hipLaunchKernelGGL((paged_attn_row_kernel<256, true>), grid, dim3(256), 0, stream, x);
    }
    check_launch("paged_attn_row_kernel");
}

} // namespace nmi
