// C ABI of the pages of a paged KV cache: host validation, then dispatch to paged_pages.hip.
#include "paged_validate.h"

namespace nmi {
namespace {

// A table and the counts of its pages, for calls that change them.
PageTable validate_pages(const nmi_tensor* table, const nmi_tensor* refs, int32_t page_size, const std::string& op) {
    require(page_size >= 16 && page_size <= 4096 && (page_size & (page_size - 1)) == 0, op, "page_size must be a power of two in [16, 4096]");
    PagedRef c;
    validate_table(table, page_size, op, c);
    PageTable t;
    t.table = static_cast<int32_t*>(table->data);
    t.row = c.table_row;
    t.max_pages = c.max_pages;
    t.B = c.B;
    while ((1 << t.shift) < page_size) { ++t.shift; }
    require(refs != nullptr, op, "refs must be non-null");
    t.pages = refs->ne[0];
    require(t.pages > 0, op, "a pool needs a page");
    t.refs = const_cast<int32_t*>(validate_index(refs, t.pages, op, "refs"));
    if (t.pages > kPagedMaxPool) { throw Unsupported(op + ": more than 2^19 pages are not built"); }
    return t;
}

int32_t* validate_output(const nmi_tensor* t, int32_t n, const std::string& op, const std::string& name) {
    return const_cast<int32_t*>(validate_index(t, n, op, name));
}

// A list of up to `most` entries.
int32_t list_length(const nmi_tensor* t, int32_t most, const std::string& op, const std::string& name) {
    require(t != nullptr && t->ne[0] > 0, op, name + " must hold an entry");
    if (t->ne[0] > most) { throw Unsupported(op + ": more than " + std::to_string(most) + " entries of " + name + " are not built"); }
    return t->ne[0];
}

bool wide(const PagePlane& p) { return (reinterpret_cast<uintptr_t>(p.data) & 15u) == 0 && p.stride % 16 == 0 && p.bytes % 16 == 0; }

} // namespace
} // namespace nmi

using namespace nmi;

extern "C" {

int nmi_paged_kv_copy_pages(const nmi_paged_kv_layer_view* cache, const nmi_paged_block_view* blocks, const nmi_tensor* src, const nmi_tensor* dst,
                            nmi_stream_t stream) {
    const std::string op = "paged_kv_copy_pages";
    return guarded([&] {
        const PagedRef c = validate_cache(cache, op);
        PagePlane planes[6];
        int32_t count = 0;
        const int64_t rows = static_cast<int64_t>(c.Hkv) << c.page_shift;
        const auto add = [&](char* data, int64_t stride, int64_t bytes) {
            planes[count] = PagePlane{data, stride, bytes, true};
            planes[count].wide = wide(planes[count]);
            ++count;
        };
        add(c.k, c.k_page, rows * c.D * (c.bf16 ? 2 : 1));
        add(c.v, c.v_page, rows * c.D * (c.bf16 ? 2 : 1));
        if (!c.bf16) {
            add(c.ks, c.ks_page, rows * (c.D / kQuantGroup) * 2);
            add(c.vs, c.vs_page, rows * (c.D / kQuantGroup) * 2);
        }
        if (blocks != nullptr) {
            const BlocksRef b = validate_blocks(blocks, c.D, c.Hkv, c.pages, 1 << c.page_shift, op);
            const int64_t each = rows >> b.shift;
            add(b.codes, b.code_page, each * c.D);
            add(b.scales, b.scale_page, each * 4);
        }
        require(src != nullptr && src->ne[0] > 0, op, "src must hold an entry");
        const int32_t n = src->ne[0];
        const int32_t* from = validate_index(src, n, op, "src");
        const int32_t* to = validate_index(dst, n, op, "dst");
        launch_copy_pages(planes, count, from, to, n, c.pages, reinterpret_cast<hipStream_t>(stream));
    });
}

int nmi_paged_pages_reserve(nmi_tensor* page_table, nmi_tensor* refs, const nmi_tensor* starts, const nmi_tensor* history, int32_t page_size,
                            nmi_tensor* granted, nmi_stream_t stream) {
    const std::string op = "paged_pages_reserve";
    return guarded([&] {
        const PageTable t = validate_pages(page_table, refs, page_size, op);
        const int32_t* ps = validate_index(starts, t.B + 1, op, "starts");
        const int32_t* ph = validate_index(history, t.B, op, "history");
        launch_pages_reserve(t, ps, ph, validate_output(granted, t.B, op, "granted"), reinterpret_cast<hipStream_t>(stream));
    });
}

int nmi_paged_pages_release(nmi_tensor* page_table, nmi_tensor* refs, const nmi_tensor* sequences, const nmi_tensor* keep_rows, int32_t page_size,
                            nmi_stream_t stream) {
    const std::string op = "paged_pages_release";
    return guarded([&] {
        const PageTable t = validate_pages(page_table, refs, page_size, op);
        const int32_t n = list_length(sequences, 65536, op, "sequences");
        const int32_t* s = validate_index(sequences, n, op, "sequences");
        const int32_t* k = validate_index(keep_rows, n, op, "keep_rows");
        launch_pages_release(t, s, k, n, reinterpret_cast<hipStream_t>(stream));
    });
}

int nmi_paged_pages_fork(nmi_tensor* page_table, nmi_tensor* refs, const nmi_tensor* parents, const nmi_tensor* children, nmi_tensor* history,
                         int32_t page_size, nmi_tensor* src, nmi_tensor* dst, nmi_stream_t stream) {
    const std::string op = "paged_pages_fork";
    return guarded([&] {
        const PageTable t = validate_pages(page_table, refs, page_size, op);
        const int32_t n = list_length(parents, kPagedMaxBatch, op, "parents");
        const int32_t* p = validate_index(parents, n, op, "parents");
        const int32_t* c = validate_index(children, n, op, "children");
        int32_t* h = validate_output(history, t.B, op, "history");
        int32_t* from = validate_output(src, n, op, "src");
        int32_t* to = validate_output(dst, n, op, "dst");
        launch_pages_fork(t, p, c, n, h, from, to, reinterpret_cast<hipStream_t>(stream));
    });
}

int nmi_paged_pages_compact(nmi_tensor* page_table, nmi_tensor* refs, nmi_tensor* src, nmi_tensor* dst, nmi_tensor* moved, nmi_stream_t stream) {
    const std::string op = "paged_pages_compact";
    return guarded([&] {
        const PageTable t = validate_pages(page_table, refs, 16, op);
        const int32_t n = list_length(src, kPagedMaxPool, op, "src");
        int32_t* from = validate_output(src, n, op, "src");
        int32_t* to = validate_output(dst, n, op, "dst");
        launch_pages_compact(t, from, to, n, validate_output(moved, 1, op, "moved"), reinterpret_cast<hipStream_t>(stream));
    });
}

} // extern "C"
