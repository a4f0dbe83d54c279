// Rows of a paged KV cache on gfx950: written as they arrive (INT8-G64 quantised, or BF16 copied) and read
// back as values.
//
// Mathematics: the codec of kv_codec.h on the way in; value = FP32(code) * FP32(scale), rounded once to the
// output's type, on the way out. No row depends on another one.
// What bounds it: HBM for prompts (an INT8 append of N tokens at 8 KV heads of 128 reads 4,096 B and writes
// 2,112 B a token), launch and dependent-load latency for decode steps: token -> sequence -> page -> row.
// So a lane holds eight values (16-byte loads of the new rows, issued before the walk through the table), the
// sequences' first tokens are fetched once per workgroup into LDS and searched there, and neighbouring lanes
// take neighbouring pieces of a row.
#include "common.h"
#include "device_utils.h"
#include "kv_codec.h"
#include "paged_internal.h"

namespace nmi {
namespace {

struct PagedRowArgs {
    PackedRef k;
    PackedRef v;
    const int32_t* starts;
    const int32_t* history;
    PagedRef c;
    int64_t units; // 8-value pieces of all tokens of one plane
    int32_t per_token;
};

// Where packed token n lies: page -1 where its row has none; seq -1 where no sequence has the token.
struct Place {
    int32_t seq;
    int32_t page;
    int32_t row;
};

__device__ __forceinline__ Place place_of(int64_t n, const int32_t* starts, const int32_t* history, const PagedRef& c) {
    int lo = 0, hi = c.B; // the last sequence that starts at or before n
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= n) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    Place p{-1, -1, 0};
    if (starts[lo] < 0 || n < starts[lo] || n >= starts[lo + 1]) { return p; }
    p.seq = lo;
    const int64_t pos = static_cast<int64_t>(history[lo]) + (n - starts[lo]);
    if (history[lo] < 0 || (pos >> c.page_shift) >= c.max_pages) { return p; }
    const int32_t page = c.table[lo * c.table_row + (pos >> c.page_shift)];
    p.page = page >= 0 && page < c.pages ? page : -1;
    p.row = static_cast<int32_t>(pos & ((int64_t{1} << c.page_shift) - 1));
    return p;
}

// starts [B + 1] and history [B] into LDS.
__device__ __forceinline__ void fetch_sequences(const PagedRowArgs& a, int32_t* smem) {
    for (int i = threadIdx.x; i <= a.c.B; i += 256) { smem[i] = a.starts[i]; }
    for (int i = threadIdx.x; i < a.c.B; i += 256) { smem[a.c.B + 1 + i] = a.history[i]; }
    __syncthreads();
}

template <bool BF>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedRowArgs a) {
    __shared__ int32_t smem[2 * kPagedMaxBatch + 1];
    const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const bool live = u < a.units; // units is a multiple of 8: whole groups stay together
    const int64_t n = live ? u / a.per_token : 0;
    const int32_t piece = static_cast<int32_t>(live ? u - n * a.per_token : 0);
    const PackedRef& src = blockIdx.y ? a.v : a.k;
    i4 raw = {0, 0, 0, 0};
    if (live) { raw = *reinterpret_cast<const i4*>(src.data + n * src.token_stride + static_cast<int64_t>(piece) * 16); }
    fetch_sequences(a, smem);
    uint16_t sbits = 0;
    i2 code = {0, 0};
    if constexpr (!BF) { code = quantize_g64(raw, sbits); }
    if (!live) { return; }
    const Place p = place_of(n, smem, smem + a.c.B + 1, a.c);
    if (p.page < 0) { return; }
    const int32_t pr = a.c.D / 8; // pieces of a row
    const int32_t h = piece / pr;
    const int64_t row = (static_cast<int64_t>(h) << a.c.page_shift) + p.row;
    char* dst = blockIdx.y ? a.c.v + p.page * a.c.v_page : a.c.k + p.page * a.c.k_page;
    if constexpr (BF) {
        *reinterpret_cast<i4*>(dst + (row * pr + (piece - h * pr)) * 16) = raw;
    } else {
        *reinterpret_cast<i2*>(dst + (row * pr + (piece - h * pr)) * 8) = code;
        if ((piece & 7) == 0) {
            char* sdst = blockIdx.y ? a.c.vs + p.page * a.c.vs_page : a.c.ks + p.page * a.c.ks_page;
            *reinterpret_cast<uint16_t*>(sdst + (row * (pr / 8) + (piece - h * pr) / 8) * 2) = sbits;
        }
    }
}

template <bool BF, bool F32>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedRowArgs a) {
    __shared__ int32_t smem[2 * kPagedMaxBatch + 1];
    fetch_sequences(a, smem);
    const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (u >= a.units) { return; }
    const int64_t n = u / a.per_token;
    const int32_t piece = static_cast<int32_t>(u - n * a.per_token);
    const Place p = place_of(n, smem, smem + a.c.B + 1, a.c);
    if (p.seq < 0) { return; }
    const int32_t pr = a.c.D / 8;
    const int32_t h = piece / pr;
    const int64_t row = (static_cast<int64_t>(h) << a.c.page_shift) + p.row;
    i4 raw = {0, 0, 0, 0};
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; // the rows of an absent page read as zero
    if (p.page >= 0) {
        const char* src = blockIdx.y ? a.c.v + p.page * a.c.v_page : a.c.k + p.page * a.c.k_page;
        if constexpr (BF) {
            raw = *reinterpret_cast<const i4*>(src + (row * pr + (piece - h * pr)) * 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t w = static_cast<uint32_t>(raw[e >> 1]);
                x[e] = __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
            }
        } else {
            const i2 code = *reinterpret_cast<const i2*>(src + (row * pr + (piece - h * pr)) * 8);
            const char* ssrc = blockIdx.y ? a.c.vs + p.page * a.c.vs_page : a.c.ks + p.page * a.c.ks_page;
            const float s = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(ssrc + (row * (pr / 8) + (piece - h * pr) / 8) * 2));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = static_cast<float>(static_cast<int8_t>(static_cast<uint32_t>(code[e >> 2]) >> (8 * (e & 3)))) * s;
            }
        }
    }
    const PackedRef& out = blockIdx.y ? a.v : a.k;
    char* dst = out.data + n * out.token_stride + static_cast<int64_t>(piece) * (F32 ? 32 : 16);
    if constexpr (F32) {
        *reinterpret_cast<f4*>(dst) = f4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f4*>(dst + 16) = f4{x[4], x[5], x[6], x[7]};
    } else if constexpr (BF) {
        *reinterpret_cast<i4*>(dst) = raw;
    } else {
        i4 o;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            o[w] = static_cast<int>(static_cast<uint32_t>(f32_to_bf16_bits(x[2 * w])) | (static_cast<uint32_t>(f32_to_bf16_bits(x[2 * w + 1])) << 16));
        }
        *reinterpret_cast<i4*>(dst) = o;
    }
}

PagedRowArgs row_args(PackedRef k, PackedRef v, int64_t tokens, const int32_t* starts, const int32_t* history, const PagedRef& c) {
    PagedRowArgs a{};
    a.k = k;
    a.v = v;
    a.starts = starts;
    a.history = history;
    a.c = c;
    a.per_token = c.Hkv * (c.D / 8);
    a.units = tokens * a.per_token;
    return a;
}

dim3 row_grid(const PagedRowArgs& a) {
    const int64_t blocks = (a.units + 255) / 256;
    if (blocks > 0x7FFFFFFF) { throw Unsupported("paged KV rows: more than 2^39 values in one call are not built"); }
    return dim3(static_cast<uint32_t>(blocks), 2);
}

} // namespace

void launch_paged_append(PackedRef k, PackedRef v, int64_t tokens, const int32_t* starts, const int32_t* history,
                         const PagedRef& c, hipStream_t stream) {
    const PagedRowArgs a = row_args(k, v, tokens, starts, history, c);
    if (c.bf16) {
        hipLaunchKernelGGL(paged_append_kernel<true>, row_grid(a), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL(paged_append_kernel<false>, row_grid(a), dim3(256), 0, stream, a);
    }
    check_launch("paged_append_kernel");
}

void launch_paged_read(PackedRef k, PackedRef v, bool f32, int64_t tokens, const int32_t* starts, const int32_t* first,
                       const PagedRef& c, hipStream_t stream) {
    const PagedRowArgs a = row_args(k, v, tokens, starts, first, c);
    if (c.bf16 && f32) {
        hipLaunchKernelGGL((paged_read_kernel<true, true>), row_grid(a), dim3(256), 0, stream, a);
    } else if (c.bf16) {
        hipLaunchKernelGGL((paged_read_kernel<true, false>), row_grid(a), dim3(256), 0, stream, a);
    } else if (f32) {
        hipLaunchKernelGGL((paged_read_kernel<false, true>), row_grid(a), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((paged_read_kernel<false, false>), row_grid(a), dim3(256), 0, stream, a);
    }
    check_launch("paged_read_kernel");
}

} // namespace nmi
