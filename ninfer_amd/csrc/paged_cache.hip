// Rows of a paged KV cache on gfx950: written as they arrive (INT8-G64 quantised, or BF16 copied) and read
// back as values.
//
// Mathematics: the codec of kv_codec.h on the way in; value = FP32(code) * FP32(scale), rounded once to the
// output's type, on the way out. No row depends on another one.
// What bounds it: HBM for prompts (an INT8 append of N tokens at 8 KV heads of 128 reads 4,096 B and writes
// 2,112 B a token), launch and dependent-load latency for decode steps: token -> sequence -> page -> row.
// So a lane holds eight values (16-byte loads of the new rows, issued before the walk through the table), the
// sequences' first tokens are fetched once per workgroup into LDS, a token's place is searched there once for all its
// pieces (searching per lane was most of the time of long calls), and neighbouring lanes take neighbouring pieces.
#include "common.h"
#include "device_utils.h"
#include "kv_codec.h"
#include "paged_internal.h"
#include "paged_place.h"

namespace nmi {
namespace {

struct PagedRowArgs {
    PackedRef k;
    PackedRef v;
    const int32_t* starts;
    const int32_t* history;
    PagedRef c;
    int64_t units; // pieces of all tokens of one plane
    int32_t per_token;
    uint32_t magic; // ceil(2^32 / per_token)
};

// What a workgroup's threads share: the sequences, and the places of its tokens, looked up once for all their pieces.
template <int ITER>
struct RowShared {
    static constexpr int kTokens = 256 * ITER / 16 + 2; // a token has at least 16 pieces
    int32_t starts[kPagedMaxBatch + 1];
    int32_t history[kPagedMaxBatch];
    Place places[kTokens];
};

// The workgroup's first piece: token n0 and the piece of it.
struct First {
    int64_t unit;
    int64_t n0;
    uint32_t rest;
};

template <int ITER>
__device__ __forceinline__ First first_of(const PagedRowArgs& a) {
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (256 * ITER);
    const int64_t n0 = unit / a.per_token;
    return First{unit, n0, static_cast<uint32_t>(unit - n0 * a.per_token)};
}

// A lane's i-th piece: token n0 + t. The multiplication divides exactly (its operands' product is below 2^32).
struct Unit {
    uint32_t t;
    uint32_t piece;
    bool live;
};

template <int ITER>
__device__ __forceinline__ Unit unit_of(const PagedRowArgs& a, const First& f, int i) {
    const uint32_t r = f.rest + 256 * i + threadIdx.x;
    const uint32_t t = __umulhi(r, a.magic);
    return Unit{t, r - t * a.per_token, f.unit + 256 * i + threadIdx.x < a.units};
}

template <int ITER>
__device__ __forceinline__ void fetch_places(const PagedRowArgs& a, const First& f, RowShared<ITER>& sh) {
    for (int i = threadIdx.x; i <= a.c.B; i += 256) { sh.starts[i] = a.starts[i]; }
    for (int i = threadIdx.x; i < a.c.B; i += 256) { sh.history[i] = a.history[i]; }
    __syncthreads();
    if (threadIdx.x < RowShared<ITER>::kTokens) { sh.places[threadIdx.x] = place_of(f.n0 + threadIdx.x, sh.starts, sh.history, a.c); }
    __syncthreads();
}

// ITER pieces of eight values per lane: all loads of a lane are in flight together.
template <bool BF, int ITER>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedRowArgs a) {
    __shared__ RowShared<ITER> sh;
    const PackedRef& src = blockIdx.y ? a.v : a.k;
    const First f = first_of<ITER>(a);
    const char* from = src.data + f.n0 * src.token_stride;
    Unit u[ITER];
    i4 raw[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        u[i] = unit_of<ITER>(a, f, i); // units is a multiple of 8: whole groups stay together
        raw[i] = i4{0, 0, 0, 0};
        if (u[i].live) { raw[i] = *reinterpret_cast<const i4*>(from + static_cast<int64_t>(u[i].t) * src.token_stride + u[i].piece * 16); }
    }
    fetch_places(a, f, sh);
    const int32_t lg = a.c.D == 128 ? 4 : 5; // log2 of a row's pieces
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        uint16_t sbits = 0;
        i2 code = {0, 0};
        if constexpr (!BF) { code = quantize_g64(raw[i], sbits); }
        if (!u[i].live) { continue; }
        const Place p = sh.places[u[i].t];
        if (p.page < 0) { continue; }
        const uint32_t at = u[i].piece & ((1 << lg) - 1);
        const uint32_t row = ((u[i].piece >> lg) << a.c.page_shift) + p.row; // a page is below 2^31 bytes
        char* dst = blockIdx.y ? a.c.v + p.page * a.c.v_page : a.c.k + p.page * a.c.k_page;
        if constexpr (BF) {
            *reinterpret_cast<i4*>(dst + ((row << lg) + at) * 16) = raw[i];
        } else {
            *reinterpret_cast<i2*>(dst + ((row << lg) + at) * 8) = code;
            if ((at & 7) == 0) {
                char* sdst = blockIdx.y ? a.c.vs + p.page * a.c.vs_page : a.c.ks + p.page * a.c.ks_page;
                *reinterpret_cast<uint16_t*>(sdst + ((row << (lg - 3)) + (at >> 3)) * 2) = sbits;
            }
        }
    }
}

template <bool BF, bool F32, int ITER>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedRowArgs a) {
    __shared__ RowShared<ITER> sh;
    const First f = first_of<ITER>(a);
    fetch_places(a, f, sh);
    Unit u[ITER];
    bool mine[ITER]; // of a sequence
    const int32_t lg = a.c.D == 128 ? 4 : 5;
    i4 raw[ITER];
    uint16_t sbits[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        raw[i] = i4{0, 0, 0, 0}; // the rows of an absent page read as zero
        sbits[i] = 0;
        u[i] = unit_of<ITER>(a, f, i);
        mine[i] = false;
        if (!u[i].live) { continue; }
        const Place p = sh.places[u[i].t];
        mine[i] = p.seq >= 0;
        if (p.page < 0) { continue; }
        const uint32_t at = u[i].piece & ((1 << lg) - 1);
        const uint32_t row = ((u[i].piece >> lg) << a.c.page_shift) + p.row;
        const char* src = blockIdx.y ? a.c.v + p.page * a.c.v_page : a.c.k + p.page * a.c.k_page;
        if constexpr (BF) {
            raw[i] = *reinterpret_cast<const i4*>(src + ((row << lg) + at) * 16);
        } else {
            const i2 code = *reinterpret_cast<const i2*>(src + ((row << lg) + at) * 8);
            raw[i][0] = code[0];
            raw[i][1] = code[1];
            const char* ssrc = blockIdx.y ? a.c.vs + p.page * a.c.vs_page : a.c.ks + p.page * a.c.ks_page;
            sbits[i] = *reinterpret_cast<const uint16_t*>(ssrc + ((row << (lg - 3)) + (at >> 3)) * 2);
        }
    }
    const PackedRef& out = blockIdx.y ? a.v : a.k;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if (!mine[i]) { continue; }
        char* dst = out.data + (f.n0 + u[i].t) * out.token_stride + u[i].piece * (F32 ? 32 : 16);
        if constexpr (BF && !F32) {
            *reinterpret_cast<i4*>(dst) = raw[i];
        } else {
            float x[8];
            const float s = f16_bits_to_f32(sbits[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (BF) {
                    const uint32_t w = static_cast<uint32_t>(raw[i][e >> 1]);
                    x[e] = __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
                } else {
                    x[e] = static_cast<float>(static_cast<int8_t>(static_cast<uint32_t>(raw[i][e >> 2]) >> (8 * (e & 3)))) * s;
                }
            }
            if constexpr (F32) {
                *reinterpret_cast<f4*>(dst) = f4{x[0], x[1], x[2], x[3]};
                *reinterpret_cast<f4*>(dst + 16) = f4{x[4], x[5], x[6], x[7]};
            } else {
                i4 o;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    o[w] = static_cast<int>(static_cast<uint32_t>(f32_to_bf16_bits(x[2 * w])) | (static_cast<uint32_t>(f32_to_bf16_bits(x[2 * w + 1])) << 16));
                }
                *reinterpret_cast<i4*>(dst) = o;
            }
        }
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
    a.magic = static_cast<uint32_t>((int64_t{1} << 32) / a.per_token + 1);
    return a;
}

// Pieces per lane: four where that still leaves every CU several workgroups.
constexpr int kIter = 4;
bool deep(const PagedRowArgs& a) { return a.units >= 256 * kIter * 1024; }

dim3 row_grid(const PagedRowArgs& a) {
    const int64_t per = 256 * (deep(a) ? kIter : 1);
    const int64_t blocks = (a.units + per - 1) / per;
    if (blocks > 0x7FFFFF) { throw Unsupported("paged KV rows: more than 2^36 values in one call are not built"); }
    return dim3(static_cast<uint32_t>(blocks), 2);
}

template <bool BF>
void append(const PagedRowArgs& a, hipStream_t stream) {
    if (deep(a)) {
        hipLaunchKernelGGL((paged_append_kernel<BF, kIter>), row_grid(a), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((paged_append_kernel<BF, 1>), row_grid(a), dim3(256), 0, stream, a);
    }
    check_launch("paged_append_kernel");
}

template <bool BF, bool F32>
void read(const PagedRowArgs& a, hipStream_t stream) {
    if (deep(a)) {
        hipLaunchKernelGGL((paged_read_kernel<BF, F32, kIter>), row_grid(a), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((paged_read_kernel<BF, F32, 1>), row_grid(a), dim3(256), 0, stream, a);
    }
    check_launch("paged_read_kernel");
}

} // namespace

void launch_paged_append(PackedRef k, PackedRef v, int64_t tokens, const int32_t* starts, const int32_t* history,
                         const PagedRef& c, hipStream_t stream) {
    const PagedRowArgs a = row_args(k, v, tokens, starts, history, c);
    c.bf16 ? append<true>(a, stream) : append<false>(a, stream);
}

void launch_paged_read(PackedRef k, PackedRef v, bool f32, int64_t tokens, const int32_t* starts, const int32_t* first,
                       const PagedRef& c, hipStream_t stream) {
    const PagedRowArgs a = row_args(k, v, tokens, starts, first, c);
    if (c.bf16) {
        f32 ? read<true, true>(a, stream) : read<true, false>(a, stream);
    } else {
        f32 ? read<false, true>(a, stream) : read<false, false>(a, stream);
    }
}

} // namespace nmi
