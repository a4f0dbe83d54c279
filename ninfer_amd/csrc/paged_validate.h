// Host checks that the paged cache's entry points share (capi_paged*.cpp): views, packed tokens, index vectors, envelopes.
#pragma once

#include "common.h"
#include "paged_internal.h"

#include <limits>
#include <string>

namespace nmi {
namespace {

void require(bool ok, const std::string& op, const std::string& what) {
    if (!ok) { throw InvalidArgument(op + ": " + what); }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A pool plane [row, page_size, Hkv, pages]: whole pages are contiguous, the page stride is free.
int64_t plane_stride(const nmi_tensor& t, int32_t dtype, int32_t row, int32_t page_size, int32_t kv_heads, int32_t pages,
                     const std::string& op, const std::string& name) {
    require(t.dtype == dtype, op, "invalid dtype for " + name);
    require(t.ne[0] == row && t.ne[1] == page_size && t.ne[2] == kv_heads && t.ne[3] == pages, op, "invalid shape for " + name);
    require(t.data != nullptr, op, name + " data must be non-null");
    const int64_t elem = static_cast<int64_t>(dtype_size(dtype));
    const int64_t page = elem * row * page_size * kv_heads;
    require(t.nb[0] == elem && t.nb[1] == elem * row && (kv_heads == 1 || t.nb[2] == elem * row * page_size), op,
            "a page of " + name + " must be contiguous");
    const int64_t stride = pages > 1 ? t.nb[3] : page;
    require(stride >= page && stride % 16 == 0, op, "invalid page stride of " + name);
    require(aligned16(t.data), op, name + " must be 16-byte aligned");
    return stride;
}

// The page table I32 [max_pages, B] of sequences in pages of `page_size` rows.
void validate_table(const nmi_tensor* table, int32_t page_size, const std::string& op, PagedRef& r) {
    require(table != nullptr, op, "page_table must be non-null");
    const nmi_tensor& t = *table;
    require(t.dtype == NMI_I32, op, "page_table must be I32");
    require(t.ne[0] > 0 && t.ne[1] > 0 && t.ne[2] == 1 && t.ne[3] == 1, op, "invalid shape for page_table");
    require(t.data != nullptr, op, "page_table data must be non-null");
    r.max_pages = t.ne[0];
    r.B = t.ne[1];
    require(t.nb[0] == 4 && (r.B == 1 || (t.nb[1] >= 4 * static_cast<int64_t>(r.max_pages) && t.nb[1] % 4 == 0)), op,
            "invalid strides of page_table");
    r.table = static_cast<const int32_t*>(t.data);
    r.table_row = r.B > 1 ? t.nb[1] / 4 : r.max_pages;
    if (r.B > kPagedMaxBatch) { throw Unsupported(op + ": more than 1024 sequences in one call are not built"); }
    if (static_cast<int64_t>(r.max_pages) * page_size > std::numeric_limits<int32_t>::max()) {
        throw Overflow(op + ": the pages of a sequence hold more rows than int32 counts");
    }
}

PagedRef validate_cache(const nmi_paged_kv_layer_view* cache, const std::string& op) {
    require(cache != nullptr, op, "cache must be non-null");
    require(cache->dtype == NMI_I8 || cache->dtype == NMI_BF16, op, "invalid paged KV cache dtype");
    require(cache->num_kv_heads > 0, op, "invalid paged KV cache geometry");
    require(cache->head_dim > 0 && cache->head_dim % kQuantGroup == 0, op, "invalid paged KV cache head_dim");
    require(cache->quant_group == (cache->dtype == NMI_I8 ? kQuantGroup : 0), op,
            "an I8 paged KV cache must use quant_group 64, a BF16 one none");
    const int32_t ps = cache->page_size;
    require(ps >= 16 && ps <= 4096 && (ps & (ps - 1)) == 0, op, "page_size must be a power of two in [16, 4096]");
    if (cache->head_dim != 128 && cache->head_dim != 256) { throw Unsupported(op + ": head_dim 128 and 256 kernels are built"); }
    PagedRef r;
    r.bf16 = cache->dtype == NMI_BF16;
    r.Hkv = cache->num_kv_heads;
    r.D = cache->head_dim;
    r.pages = cache->k.ne[3];
    require(r.pages > 0, op, "a paged KV cache needs a page");
    if (r.Hkv > 1024) { throw Unsupported(op + ": more than 1024 KV heads are not built"); }
    if (static_cast<int64_t>(r.Hkv) * ps * r.D * 2 >= (int64_t{1} << 31)) {
        throw Unsupported(op + ": a page of 2^31 bytes or more is not built");
    }
    while ((1 << r.page_shift) < ps) { ++r.page_shift; }
    r.k_page = plane_stride(cache->k, cache->dtype, r.D, ps, r.Hkv, r.pages, op, "cache k");
    r.v_page = plane_stride(cache->v, cache->dtype, r.D, ps, r.Hkv, r.pages, op, "cache v");
    r.k = static_cast<char*>(cache->k.data);
    r.v = static_cast<char*>(cache->v.data);
    if (r.bf16) {
        require(cache->k_scale.data == nullptr && cache->v_scale.data == nullptr, op, "BF16 KV cache must not have scales");
    } else {
        r.ks_page = plane_stride(cache->k_scale, NMI_FP16, r.D / kQuantGroup, ps, r.Hkv, r.pages, op, "cache k scale");
        r.vs_page = plane_stride(cache->v_scale, NMI_FP16, r.D / kQuantGroup, ps, r.Hkv, r.pages, op, "cache v scale");
        r.ks = static_cast<char*>(cache->k_scale.data);
        r.vs = static_cast<char*>(cache->v_scale.data);
    }
    validate_table(&cache->page_table, ps, op, r);
    return r;
}

// Packed tokens [D, heads, N]: a token's heads are contiguous, the token stride is free.
PackedRef validate_packed(const nmi_tensor* t, int32_t dtype, int32_t D, int32_t heads, int32_t tokens, const std::string& op,
                          const std::string& name) {
    require(t != nullptr, op, name + " must be non-null");
    require(t->dtype == dtype, op, "invalid dtype for " + name);
    require(t->ne[0] == D && t->ne[1] == heads && t->ne[2] == tokens && t->ne[3] == 1, op, "invalid shape for " + name);
    require(t->data != nullptr, op, name + " data must be non-null");
    const int64_t elem = static_cast<int64_t>(dtype_size(dtype));
    const int64_t token = elem * D * heads;
    require(t->nb[0] == elem && (heads == 1 || t->nb[1] == elem * D), op, "the heads of a token of " + name + " must be contiguous");
    PackedRef r;
    r.data = static_cast<char*>(t->data);
    r.token_stride = tokens > 1 ? t->nb[2] : token;
    require(r.token_stride >= token && r.token_stride % 16 == 0, op, "invalid token stride of " + name);
    require(aligned16(t->data), op, name + " must be 16-byte aligned");
    return r;
}

const int32_t* validate_index(const nmi_tensor* t, int32_t n, const std::string& op, const std::string& name) {
    require(t != nullptr, op, name + " must be non-null");
    require(t->dtype == NMI_I32, op, name + " must be I32");
    require(t->ne[0] == n && t->ne[1] == 1 && t->ne[2] == 1 && t->ne[3] == 1, op, "invalid shape for " + name);
    require(is_contiguous(*t) && t->data != nullptr, op, name + " must be contiguous and non-null");
    return static_cast<const int32_t*>(t->data);
}

int32_t packed_tokens(const nmi_tensor* t, const std::string& op, const std::string& name) {
    require(t != nullptr, op, name + " must be non-null");
    require(t->ne[2] > 0, op, "the number of tokens must be positive");
    return t->ne[2];
}

// The bounds that the launch is sized for: most new tokens and most rows of a sequence.
void validate_envelope(nmi_paged_envelope e, nmi_attention_window w, const std::string& op) {
    constexpr uint32_t top = static_cast<uint32_t>(std::numeric_limits<int32_t>::max());
    if (e.max_new_tokens > top || e.max_visible_keys > top || w.size > top || w.sinks > top) {
        throw Overflow(op + ": the envelope or the window exceeds int32");
    }
    require(e.max_new_tokens > 0 && e.max_new_tokens <= e.max_visible_keys, op, "invalid execution envelope");
    require(w.size > 0 || w.sinks == 0, op, "sinks need a window");
}

int32_t log2_of(int32_t v) {
    int32_t s = 0;
    while ((1 << s) < v) { ++s; }
    return s;
}

bool power_of_two(int32_t v) { return v > 0 && (v & (v - 1)) == 0; }

// Means of blocks of a pool: whole blocks of a page, whole pages contiguous.
BlocksRef validate_blocks(const nmi_paged_block_view* b, int32_t D, int32_t Hkv, int32_t pages, int32_t page_size, const std::string& op) {
    require(b != nullptr, op, "blocks must be non-null");
    require(power_of_two(b->block_size) && b->block_size >= 32 && b->block_size <= page_size, op,
            "block_size must be a power of two from 32 to page_size");
    const int32_t per = page_size / b->block_size;
    BlocksRef r;
    r.shift = log2_of(b->block_size);
    r.code_page = plane_stride(b->codes, NMI_I8, D, per, Hkv, pages, op, "block codes");
    r.codes = static_cast<char*>(b->codes.data);
    const nmi_tensor& s = b->scales;
    require(s.dtype == NMI_FP32, op, "block scales must be FP32");
    require(s.ne[0] == per && s.ne[1] == Hkv && s.ne[2] == pages && s.ne[3] == 1, op, "invalid shape for block scales");
    require(s.data != nullptr && (reinterpret_cast<uintptr_t>(s.data) & 3u) == 0, op, "block scales must be non-null and 4-byte aligned");
    const int64_t page = 4 * static_cast<int64_t>(per) * Hkv;
    require(s.nb[0] == 4 && (Hkv == 1 || s.nb[1] == 4 * static_cast<int64_t>(per)), op, "a page of the block scales must be contiguous");
    r.scale_page = pages > 1 ? s.nb[2] : page;
    require(r.scale_page >= page && r.scale_page % 4 == 0, op, "invalid page stride of the block scales");
    r.scales = static_cast<char*>(s.data);
    return r;
}

} // namespace
} // namespace nmi
