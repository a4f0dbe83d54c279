// Host-side launch interfaces of the paged KV cache between its C ABI (capi_paged.cpp, capi_paged_blocks.cpp,
// capi_paged_pages.cpp, capi_norm_rope.cpp) and its kernels.
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

// ---- head norms and rotation (norm_rope.hip) ---------------------------------------------------

struct NormRope {
    PackedRef q;
    PackedRef k;
    PackedRef v; // of the form that appends
    PackedRef q_out;
    PackedRef k_out; // of the form that does not
    const void* q_weight = nullptr; // [D] FP32 or BF16, null: ones
    const void* k_weight = nullptr;
    const int32_t* positions = nullptr; // of the form that does not append
    const int32_t* starts = nullptr;    // of the form that does
    const int32_t* history = nullptr;
    const float* inv_freq = nullptr; // [half]
    int32_t half = 0;                // rotated pairs of a head
    int32_t Hq = 0;
    int32_t Hkv = 0;
    int32_t D = 0;
    int64_t tokens = 0;
    float eps = 0.0f;
    float offset = 0.0f;
    bool q_weight_f32 = false;
    bool k_weight_f32 = false;
    bool interleaved = false;
};

// `cache`: null for the form that writes k_out.
void launch_norm_rope(const NormRope& a, const PagedRef* cache, hipStream_t stream);

// ---- blocks of keys (paged_blocks.hip, paged_sparse.hip) ---------------------------------------

// Blocks of a sequence in one selection: a token's scores lie in LDS, four bytes each.
inline constexpr int32_t kPagedMaxBlocks = 32768;
// Blocks that a token selects.
inline constexpr int32_t kPagedMaxSelected = 1024;

// Means of blocks: codes [D, blocks of a page, Hkv, pages], scales [blocks of a page, Hkv, pages].
struct BlocksRef {
    char* codes = nullptr;
    char* scales = nullptr;
    int64_t code_page = 0; // bytes between pages
    int64_t scale_page = 0;
    int32_t shift = 0; // log2(rows of a block)
};

void launch_block_update(int64_t tokens, const int32_t* starts, const int32_t* history, const PagedRef& cache, const BlocksRef& blocks,
                         hipStream_t stream);

struct BlockSelect {
    PackedRef q;
    int64_t tokens = 0;
    const int32_t* starts = nullptr;
    const int32_t* history = nullptr;
    int32_t* selected = nullptr; // [token][KV head][first + local + top]
    int32_t Hq = 0;
    int32_t first = 0;
    int32_t local = 0;
    int32_t top = 0;
    int32_t max_new = 0;
    int32_t max_keys = 0;
};

size_t block_select_bytes(int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t max_new, int32_t max_keys, int32_t block_shift);
void launch_block_select(const BlockSelect& a, const PagedRef& cache, const BlocksRef& blocks, void* workspace, hipStream_t stream);

size_t sparse_attention_bytes(int32_t Hq, int32_t Hkv, int32_t D, int64_t tokens, int32_t B, int32_t selected, int32_t block_shift);
void launch_sparse_attention(const PagedAttention& a, const int32_t* selected, int32_t count, int32_t block_shift, const PagedRef& cache,
                             void* workspace, hipStream_t stream);

// ---- pages (paged_pages.hip) --------------------------------------------------------------------

// Pages of a pool in the calls that hand them out: a bit for each in the LDS of one workgroup.
inline constexpr int32_t kPagedMaxPool = 1 << 19;

// One plane's pages: `bytes` each, a multiple of 4; data, stride and bytes of 16 where `wide`.
struct PagePlane {
    char* data = nullptr;
    int64_t stride = 0;
    int64_t bytes = 0;
    bool wide = true;
};

void launch_copy_pages(const PagePlane* planes, int32_t count, const int32_t* src, const int32_t* dst, int32_t n, int32_t pages, hipStream_t stream);

// A table that a call changes, and the counts of its pages.
struct PageTable {
    int32_t* table = nullptr;
    int64_t row = 0; // entries between sequences
    int32_t max_pages = 0;
    int32_t B = 0;
    int32_t* refs = nullptr;
    int32_t pages = 0;
    int32_t shift = 0; // log2(page_size)
};

void launch_pages_reserve(const PageTable& t, const int32_t* starts, const int32_t* history, int32_t* granted, hipStream_t stream);
void launch_pages_release(const PageTable& t, const int32_t* sequences, const int32_t* keep, int32_t n, hipStream_t stream);
void launch_pages_fork(const PageTable& t, const int32_t* parents, const int32_t* children, int32_t n, int32_t* history, int32_t* src, int32_t* dst,
                       hipStream_t stream);
void launch_pages_compact(const PageTable& t, int32_t* src, int32_t* dst, int32_t n, int32_t* moved, hipStream_t stream);

} // namespace nmi
