// C ABI of the paged KV cache: host validation, then dispatch to paged_cache.hip and paged_attention.hip.
#include "paged_validate.h"

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
