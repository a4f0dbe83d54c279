// C ABI of the paged KV cache: host validation, then dispatch to paged_cache.hip and paged_attention.hip.
#include "common.h"
#include "paged_internal.h"

#include <cmath>
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
    const nmi_tensor& t = cache->page_table;
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
    if (static_cast<int64_t>(r.max_pages) * ps > std::numeric_limits<int32_t>::max()) {
        throw Overflow(op + ": the pages of a sequence hold more rows than int32 counts");
    }
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

} // namespace
} // namespace nmi

using namespace nmi;

extern "C" {

int nmi_paged_kv_append(const nmi_tensor* k, const nmi_tensor* v, const nmi_tensor* starts, const nmi_tensor* history,
                        const nmi_paged_kv_layer_view* cache, nmi_stream_t stream) {
    const std::string op = "paged_kv_append";
    return guarded([&] {
        const PagedRef c = validate_cache(cache, op);
        const int32_t n = packed_tokens(k, op, "k");
        const PackedRef rk = validate_packed(k, NMI_BF16, c.D, c.Hkv, n, op, "k");
        const PackedRef rv = validate_packed(v, NMI_BF16, c.D, c.Hkv, n, op, "v");
        const int32_t* ps = validate_index(starts, c.B + 1, op, "starts");
        const int32_t* ph = validate_index(history, c.B, op, "history");
        launch_paged_append(rk, rv, n, ps, ph, c, reinterpret_cast<hipStream_t>(stream));
    });
}

int nmi_paged_kv_read(const nmi_paged_kv_layer_view* cache, const nmi_tensor* starts, const nmi_tensor* first, nmi_tensor* k_out,
                      nmi_tensor* v_out, nmi_stream_t stream) {
    const std::string op = "paged_kv_read";
    return guarded([&] {
        const PagedRef c = validate_cache(cache, op);
        const int32_t n = packed_tokens(k_out, op, "k_out");
        require(k_out->dtype == NMI_BF16 || k_out->dtype == NMI_FP32, op, "k_out/v_out must be BF16 or FP32");
        const PackedRef rk = validate_packed(k_out, k_out->dtype, c.D, c.Hkv, n, op, "k_out");
        const PackedRef rv = validate_packed(v_out, k_out->dtype, c.D, c.Hkv, n, op, "v_out");
        const int32_t* ps = validate_index(starts, c.B + 1, op, "starts");
        const int32_t* pf = validate_index(first, c.B, op, "first");
        launch_paged_read(rk, rv, k_out->dtype == NMI_FP32, n, ps, pf, c, reinterpret_cast<hipStream_t>(stream));
    });
}

size_t nmi_paged_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t tokens, int32_t batch,
                                           nmi_paged_envelope envelope, nmi_attention_window window) {
    constexpr uint32_t top = static_cast<uint32_t>(std::numeric_limits<int32_t>::max());
    // 0 for what the op itself refuses
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0 || (head_dim != 128 && head_dim != 256) || tokens <= 0 || batch <= 0 ||
        batch > kPagedMaxBatch || envelope.max_new_tokens == 0 || envelope.max_new_tokens > envelope.max_visible_keys ||
        envelope.max_visible_keys > static_cast<uint32_t>(kPagedMaxKeys) || window.size > top || window.sinks > top ||
        static_cast<int64_t>(tokens) * q_heads > (int64_t{1} << 30)) {
        return 0;
    }
    return paged_attention_bytes(q_heads, kv_heads, head_dim, tokens, batch, static_cast<int32_t>(envelope.max_new_tokens),
                                 static_cast<int32_t>(envelope.max_visible_keys), static_cast<int32_t>(window.size),
                                 static_cast<int32_t>(window.sinks));
}

int nmi_paged_attention(const nmi_tensor* q, const nmi_tensor* starts, const nmi_tensor* history, float scale,
                        nmi_attention_window window, const nmi_paged_kv_layer_view* cache, nmi_paged_envelope envelope, void* workspace,
                        size_t workspace_bytes, nmi_tensor* out, nmi_stream_t stream) {
    const std::string op = "paged_attention";
    return guarded([&] {
        const PagedRef c = validate_cache(cache, op);
        const int32_t n = packed_tokens(q, op, "q");
        PagedAttention a;
        a.tokens = n;
        a.Hq = q->ne[1];
        require(a.Hq > 0 && a.Hq % c.Hkv == 0, op, "unsupported Q/KV head geometry");
        a.q = validate_packed(q, NMI_BF16, c.D, a.Hq, n, op, "q");
        a.out = validate_packed(out, NMI_BF16, c.D, a.Hq, n, op, "out");
        a.starts = validate_index(starts, c.B + 1, op, "starts");
        a.history = validate_index(history, c.B, op, "history");
        require(scale >= 0x1p-40f && scale <= 0x1p40f, op, "scale must be positive, from 2^-40 to 2^40");
        a.scale = scale;
        validate_envelope(envelope, window, op);
        require(static_cast<int64_t>(envelope.max_visible_keys) <= (static_cast<int64_t>(c.max_pages) << c.page_shift), op,
                "the execution envelope exceeds the page table");
        if (envelope.max_visible_keys > static_cast<uint32_t>(kPagedMaxKeys)) {
            throw Unsupported(op + ": more than 2^23 rows of a sequence are not built");
        }
        if (static_cast<int64_t>(n) * a.Hq > (int64_t{1} << 30)) { throw Unsupported(op + ": more than 2^30 query rows in one call are not built"); }
        a.max_new = static_cast<int32_t>(envelope.max_new_tokens);
        a.max_keys = static_cast<int32_t>(envelope.max_visible_keys);
        a.window = static_cast<int32_t>(window.size);
        a.sinks = static_cast<int32_t>(window.sinks);
        const size_t need = paged_attention_bytes(a.Hq, c.Hkv, c.D, n, c.B, a.max_new, a.max_keys, a.window, a.sinks);
        require(workspace_bytes >= need, op, "workspace is smaller than the size query");
        require(workspace != nullptr || need == 0, op, "workspace must be non-null");
        require((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, op, "workspace must be 256-byte aligned");
        launch_paged_attention(a, c, workspace, reinterpret_cast<hipStream_t>(stream));
    });
}

} // extern "C"
