// C ABI of the blocks of a paged KV cache: means, selection, attention over selected blocks.
#include "paged_validate.h"

namespace nmi {
namespace {

void validate_bounds(nmi_paged_envelope e, const PagedRef& c, const std::string& op) {
    validate_envelope(e, nmi_attention_window{0, 0}, op);
    require(static_cast<int64_t>(e.max_visible_keys) <= (static_cast<int64_t>(c.max_pages) << c.page_shift), op,
            "the execution envelope exceeds the page table");
    if (e.max_visible_keys > static_cast<uint32_t>(kPagedMaxKeys)) { throw Unsupported(op + ": more than 2^23 rows of a sequence are not built"); }
}

// The lists of a call: [count, Hkv, N].
int32_t* validate_lists(const nmi_tensor* t, int32_t count, int32_t Hkv, int32_t tokens, const std::string& op) {
    require(t != nullptr, op, "selected must be non-null");
    require(t->dtype == NMI_I32, op, "selected must be I32");
    require(t->ne[0] == count && t->ne[1] == Hkv && t->ne[2] == tokens && t->ne[3] == 1, op, "invalid shape for selected");
    require(is_contiguous(*t) && t->data != nullptr, op, "selected must be contiguous and non-null");
    return static_cast<int32_t*>(t->data);
}

void validate_workspace(const void* workspace, size_t bytes, size_t need, const std::string& op) {
    require(bytes >= need, op, "workspace is smaller than the size query");
    require(workspace != nullptr || need == 0, op, "workspace must be non-null");
    require((reinterpret_cast<uintptr_t>(workspace) & 255u) == 0, op, "workspace must be 256-byte aligned");
}

} // namespace
} // namespace nmi

using namespace nmi;

extern "C" {

int nmi_paged_block_update(const nmi_paged_kv_layer_view* cache, const nmi_tensor* starts, const nmi_tensor* history, int32_t tokens,
                           const nmi_paged_block_view* blocks, nmi_stream_t stream) {
    const std::string op = "paged_block_update";
    return guarded([&] {
        const PagedRef c = validate_cache(cache, op);
        const BlocksRef b = validate_blocks(blocks, c.D, c.Hkv, c.pages, 1 << c.page_shift, op);
        require(tokens > 0, op, "the number of tokens must be positive");
        const int32_t* ps = validate_index(starts, c.B + 1, op, "starts");
        const int32_t* ph = validate_index(history, c.B, op, "history");
        launch_block_update(tokens, ps, ph, c, b, reinterpret_cast<hipStream_t>(stream));
    });
}

size_t nmi_paged_block_select_workspace_bytes(int32_t kv_heads, int32_t head_dim, int32_t tokens, int32_t batch, nmi_paged_envelope envelope,
                                              int32_t block_size) {
    if (kv_heads <= 0 || kv_heads > 1024 || (head_dim != 128 && head_dim != 256) || tokens <= 0 || batch <= 0 || batch > kPagedMaxBatch ||
        envelope.max_new_tokens == 0 || envelope.max_new_tokens > envelope.max_visible_keys ||
        envelope.max_visible_keys > static_cast<uint32_t>(kPagedMaxKeys) || !power_of_two(block_size) || block_size < 32 || block_size > 4096) {
        return 0; // what the op itself refuses
    }
    return block_select_bytes(kv_heads, head_dim, tokens, batch, static_cast<int32_t>(envelope.max_new_tokens),
                              static_cast<int32_t>(envelope.max_visible_keys), log2_of(block_size));
}

int nmi_paged_block_select(const nmi_tensor* q, const nmi_tensor* starts, const nmi_tensor* history, const nmi_tensor* page_table,
                           int32_t page_size, const nmi_paged_block_view* blocks, nmi_block_selection selection, nmi_paged_envelope envelope,
                           void* workspace, size_t workspace_bytes, nmi_tensor* selected, nmi_stream_t stream) {
    const std::string op = "paged_block_select";
    return guarded([&] {
        require(blocks != nullptr, op, "blocks must be non-null");
        require(power_of_two(page_size) && page_size >= 32 && page_size <= 4096, op, "page_size must be a power of two in [32, 4096]");
        PagedRef c;
        c.page_shift = log2_of(page_size);
        c.D = blocks->codes.ne[0];
        c.Hkv = blocks->codes.ne[2];
        c.pages = blocks->codes.ne[3];
        require(c.D > 0 && c.D % kQuantGroup == 0 && c.Hkv > 0 && c.pages > 0, op, "invalid shape for block codes");
        if (c.D != 128 && c.D != 256) { throw Unsupported(op + ": head_dim 128 and 256 kernels are built"); }
        if (c.Hkv > 1024) { throw Unsupported(op + ": more than 1024 KV heads are not built"); }
        const BlocksRef b = validate_blocks(blocks, c.D, c.Hkv, c.pages, page_size, op);
        validate_table(page_table, page_size, op, c);
        BlockSelect a;
        const int32_t n = packed_tokens(q, op, "q");
        a.tokens = n;
        a.Hq = q->ne[1];
        require(a.Hq > 0 && a.Hq % c.Hkv == 0, op, "unsupported Q/KV head geometry");
        a.q = validate_packed(q, NMI_BF16, c.D, a.Hq, n, op, "q");
        a.starts = validate_index(starts, c.B + 1, op, "starts");
        a.history = validate_index(history, c.B, op, "history");
        require(selection.first >= 0 && selection.local >= 1 && selection.top >= 0, op, "a selection has first >= 0, local >= 1 and top >= 0 blocks");
        const int64_t count = static_cast<int64_t>(selection.first) + selection.local + selection.top;
        if (count > kPagedMaxSelected) { throw Unsupported(op + ": more than 1024 selected blocks are not built"); }
        a.first = selection.first;
        a.local = selection.local;
        a.top = selection.top;
        validate_bounds(envelope, c, op);
        a.max_new = static_cast<int32_t>(envelope.max_new_tokens);
        a.max_keys = static_cast<int32_t>(envelope.max_visible_keys);
        if (((a.max_keys - 1) >> b.shift) + 1 > kPagedMaxBlocks) { throw Unsupported(op + ": more than 32768 blocks of a sequence are not built"); }
        a.selected = validate_lists(selected, static_cast<int32_t>(count), c.Hkv, n, op);
        validate_workspace(workspace, workspace_bytes, block_select_bytes(c.Hkv, c.D, n, c.B, a.max_new, a.max_keys, b.shift), op);
        launch_block_select(a, c, b, workspace, reinterpret_cast<hipStream_t>(stream));
    });
}

size_t nmi_paged_sparse_attention_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t tokens, int32_t batch,
                                                  int32_t selected_blocks, int32_t block_size) {
    if (kv_heads <= 0 || kv_heads > 1024 || q_heads <= 0 || q_heads % kv_heads != 0 || (head_dim != 128 && head_dim != 256) || tokens <= 0 ||
        batch <= 0 || batch > kPagedMaxBatch || selected_blocks <= 0 || selected_blocks > kPagedMaxSelected || !power_of_two(block_size) ||
        block_size < 32 || block_size > 4096 || static_cast<int64_t>(tokens) * q_heads > (int64_t{1} << 30)) {
        return 0; // what the op itself refuses
    }
    return sparse_attention_bytes(q_heads, kv_heads, head_dim, tokens, batch, selected_blocks, log2_of(block_size));
}

int nmi_paged_sparse_attention(const nmi_tensor* q, const nmi_tensor* starts, const nmi_tensor* history, float scale, const nmi_tensor* selected,
                               int32_t block_size, const nmi_paged_kv_layer_view* cache, nmi_paged_envelope envelope, void* workspace,
                               size_t workspace_bytes, nmi_tensor* out, nmi_stream_t stream) {
    const std::string op = "paged_sparse_attention";
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
        require(power_of_two(block_size) && block_size >= 32 && block_size <= 4096, op, "block_size must be a power of two in [32, 4096]");
        require(selected != nullptr && selected->ne[0] > 0, op, "selected must hold a block");
        if (selected->ne[0] > kPagedMaxSelected) { throw Unsupported(op + ": more than 1024 selected blocks are not built"); }
        const int32_t count = selected->ne[0];
        const int32_t* lists = validate_lists(selected, count, c.Hkv, n, op);
        validate_bounds(envelope, c, op);
        if (static_cast<int64_t>(n) * a.Hq > (int64_t{1} << 30)) { throw Unsupported(op + ": more than 2^30 query rows in one call are not built"); }
        a.max_new = static_cast<int32_t>(envelope.max_new_tokens);
        a.max_keys = static_cast<int32_t>(envelope.max_visible_keys);
        const int32_t shift = log2_of(block_size);
        validate_workspace(workspace, workspace_bytes, sparse_attention_bytes(a.Hq, c.Hkv, c.D, n, c.B, count, shift), op);
        launch_sparse_attention(a, lists, count, shift, c, workspace, reinterpret_cast<hipStream_t>(stream));
    });
}

} // extern "C"
