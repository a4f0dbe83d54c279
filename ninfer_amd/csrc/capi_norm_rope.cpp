// C ABI of the head norms with rotation: host validation, then dispatch to norm_rope.hip.
#include "paged_validate.h"

#include <cmath>

namespace nmi {
namespace {

constexpr int64_t kMostTokens = int64_t{1} << 23; // a workgroup per token

// A weight [D] in BF16 or FP32; null: ones.
void validate_weight(const nmi_tensor* w, int32_t D, const std::string& op, const std::string& name, const void*& data, bool& f32) {
    data = nullptr;
    f32 = false;
    if (w == nullptr) { return; }
    require(w->dtype == NMI_BF16 || w->dtype == NMI_FP32, op, name + " must be BF16 or FP32");
    require(w->ne[0] == D && w->ne[1] == 1 && w->ne[2] == 1 && w->ne[3] == 1, op, "invalid shape for " + name);
    require(is_contiguous(*w) && w->data != nullptr && aligned16(w->data), op, name + " must be contiguous, non-null and 16-byte aligned");
    data = w->data;
    f32 = w->dtype == NMI_FP32;
}

// What both forms check. A tensor may be written in place, token by token.
NormRope validate_norm_rope(const nmi_tensor* q, const nmi_tensor* k, const nmi_tensor* q_weight, const nmi_tensor* k_weight,
                            const nmi_tensor* inv_freq, nmi_norm_rope norm, const nmi_tensor* q_out, const std::string& op) {
    NormRope a;
    const int32_t n = packed_tokens(q, op, "q");
    require(k != nullptr, op, "k must be non-null");
    a.tokens = n;
    a.D = q->ne[0];
    a.Hq = q->ne[1];
    a.Hkv = k->ne[1];
    require(a.D > 0 && a.D % kQuantGroup == 0, op, "invalid head_dim");
    require(a.Hq > 0 && a.Hkv > 0, op, "invalid number of heads");
    if (a.D != 128 && a.D != 256) { throw Unsupported(op + ": head_dim 128 and 256 kernels are built"); }
    if (a.Hq > 65536 || a.Hkv > 1024) { throw Unsupported(op + ": more than 65536 query or 1024 KV heads are not built"); }
    if (n > kMostTokens) { throw Unsupported(op + ": more than 2^23 tokens in one call are not built"); }
    a.q = validate_packed(q, NMI_BF16, a.D, a.Hq, n, op, "q");
    a.k = validate_packed(k, NMI_BF16, a.D, a.Hkv, n, op, "k");
    a.q_out = validate_packed(q_out, NMI_BF16, a.D, a.Hq, n, op, "q_out");
    require(a.q_out.data != a.q.data || a.q_out.token_stride == a.q.token_stride, op, "q_out in place of q must have its strides");
    validate_weight(q_weight, a.D, op, "q_weight", a.q_weight, a.q_weight_f32);
    validate_weight(k_weight, a.D, op, "k_weight", a.k_weight, a.k_weight_f32);
    if (inv_freq != nullptr) {
        const int32_t half = inv_freq->ne[0];
        require(half > 0 && half <= a.D / 2 && half % 8 == 0, op, "inv_freq must have a multiple of 8 entries, at most half of head_dim");
        require(inv_freq->dtype == NMI_FP32, op, "inv_freq must be FP32");
        require(inv_freq->ne[1] == 1 && inv_freq->ne[2] == 1 && inv_freq->ne[3] == 1 && is_contiguous(*inv_freq) && inv_freq->data != nullptr, op,
                "inv_freq must be a contiguous non-null vector");
        a.inv_freq = static_cast<const float*>(inv_freq->data);
        a.half = half;
    }
    require(norm.eps >= 0x1p-60f && norm.eps <= 1.0f, op, "eps must be from 2^-60 to 1");
    require(std::isfinite(norm.weight_offset), op, "weight_offset must be finite");
    require(norm.interleaved == 0 || norm.interleaved == 1, op, "interleaved must be 0 or 1");
    a.eps = norm.eps;
    a.offset = norm.weight_offset;
    a.interleaved = norm.interleaved != 0;
    return a;
}

} // namespace
} // namespace nmi

using namespace nmi;

extern "C" {

int nmi_qk_norm_rope(const nmi_tensor* q, const nmi_tensor* k, const nmi_tensor* q_weight, const nmi_tensor* k_weight,
                     const nmi_tensor* positions, const nmi_tensor* inv_freq, nmi_norm_rope norm, nmi_tensor* q_out, nmi_tensor* k_out,
                     nmi_stream_t stream) {
    const std::string op = "qk_norm_rope";
    return guarded([&] {
        NormRope a = validate_norm_rope(q, k, q_weight, k_weight, inv_freq, norm, q_out, op);
        const int32_t n = static_cast<int32_t>(a.tokens);
        a.positions = validate_index(positions, n, op, "positions");
        a.k_out = validate_packed(k_out, NMI_BF16, a.D, a.Hkv, n, op, "k_out");
        require(a.k_out.data != a.k.data || a.k_out.token_stride == a.k.token_stride, op, "k_out in place of k must have its strides");
        launch_norm_rope(a, nullptr, reinterpret_cast<hipStream_t>(stream));
    });
}

int nmi_paged_qk_norm_rope_append(const nmi_tensor* q, const nmi_tensor* k, const nmi_tensor* v, const nmi_tensor* q_weight,
                                  const nmi_tensor* k_weight, const nmi_tensor* starts, const nmi_tensor* history,
                                  const nmi_tensor* inv_freq, nmi_norm_rope norm, const nmi_paged_kv_layer_view* cache, nmi_tensor* q_out,
                                  nmi_stream_t stream) {
    const std::string op = "paged_qk_norm_rope_append";
    return guarded([&] {
        const PagedRef c = validate_cache(cache, op);
        NormRope a = validate_norm_rope(q, k, q_weight, k_weight, inv_freq, norm, q_out, op);
        require(a.D == c.D && a.Hkv == c.Hkv, op, "q and k must have the cache's geometry");
        a.v = validate_packed(v, NMI_BF16, c.D, c.Hkv, static_cast<int32_t>(a.tokens), op, "v");
        a.starts = validate_index(starts, c.B + 1, op, "starts");
        a.history = validate_index(history, c.B, op, "history");
        launch_norm_rope(a, &c, reinterpret_cast<hipStream_t>(stream));
    });
}

} // extern "C"
