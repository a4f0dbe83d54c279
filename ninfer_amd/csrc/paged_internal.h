// Host-side launch interfaces of the paged KV cache between its C ABI (capi_paged.cpp) and its kernels
// (paged_cache.hip, paged_attention.hip).
#pragma once

#include "common.h"

namespace nmi {

// Sequences of one call: the kernels keep their first tokens in LDS or spread them over a wave.
inline constexpr int32_t kPagedMaxBatch = 1024;

// Rows of a sequence in an attention call: a workgroup marks key tiles of 64 rows in a bit field in LDS.
inline constexpr int32_t kPagedMaxKeys = 1 << 23;

// A validated paged cache view. Row r of a page: plane + page * page_stride + (h * page_size + r) * row bytes.
struct PagedRef {
    char* k = nullptr; // I8 codes or BF16 values
    char* v = nullptr;
    char* ks = nullptr; // FP16 scales (INT8-G64 only)
    char* vs = nullptr;
    int64_t k_page = 0; // bytes between pages of each plane
    int64_t v_page = 0;
    int64_t ks_page = 0;
    int64_t vs_page = 0;
    const int32_t* table = nullptr; // [sequence][page of the sequence]
    int64_t table_row = 0;          // entries between sequences
    int32_t max_pages = 0;          // entries of a sequence
    int32_t pages = 0;              // pages of the pool; an entry outside [0, pages) is an absent page
    int32_t page_shift = 0;         // log2(page_size)
    int32_t Hkv = 0;
    int32_t D = 0;
    int32_t B = 0;
    bool bf16 = false;
};

// Packed tokens: token n of head h at data + n * token_stride + h * head bytes.
struct PackedRef {
    char* data = nullptr;
    int64_t token_stride = 0; // bytes
};

void launch_paged_append(PackedRef k, PackedRef v, int64_t tokens, const int32_t* starts, const int32_t* history,
                         const PagedRef& cache, hipStream_t stream);

void launch_paged_read(PackedRef k, PackedRef v, bool f32, int64_t tokens, const int32_t* starts, const int32_t* first,
                       const PagedRef& cache, hipStream_t stream);

struct PagedAttention {
    PackedRef q;
    PackedRef out;
    int64_t tokens = 0;
    const int32_t* starts = nullptr;
    const int32_t* history = nullptr;
    int32_t Hq = 0;
    int32_t max_new = 0;  // most new tokens of a sequence
    int32_t max_keys = 0; // most rows of a sequence, new ones included
    int32_t window = 0;   // 0: every row
    int32_t sinks = 0;
    float scale = 0.0f;
};

// Transient storage of launch_paged_attention (0: none).
size_t paged_attention_bytes(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t max_new, int32_t max_keys,
                             int32_t window, int32_t sinks);

void launch_paged_attention(const PagedAttention& a, const PagedRef& cache, void* workspace, hipStream_t stream);

} // namespace nmi
