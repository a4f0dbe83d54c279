"""Python mirror of the reference op surface for the verify step (ninfer::ops).

Same names, argument meaning and error behaviour as include/ninfer/ops/*.h: invalid shapes or
dtypes raise ValueError (std::invalid_argument), int32 overflow raises OverflowError
(std::overflow_error). Tensors are nmi_tensor views (see ninfer_amd.device.DeviceArray.tensor()),
streams are ninfer_amd.device.Stream or None, workspaces are DeviceBuffer regions sized by the
*_workspace_bytes queries. Every call launches hand-written gfx950 kernels through the C ABI.
"""
from __future__ import annotations

import ctypes as C

from . import _capi
from ._capi import AttentionWindow, BlockSelection, CommitEnvelope, GqaEnvelope, NormRope, PagedEnvelope, Tensor, check, lib


def _s(stream):
    return stream.handle if stream is not None else None


def _ws(workspace):
    if workspace is None:
        return None, 0
    return C.c_void_p(workspace.ptr), workspace.nbytes


def _p(t: Tensor | None):
    return C.byref(t) if t is not None else None


# ---- verify attention (include/ninfer/ops/gqa_attention.h) -------------------------------------

def gqa_attention_workspace_bytes(q_heads: int, kv_heads: int, head_dim: int, tokens: int,
                                  batch: int, max_visible_keys: int) -> int:
    return int(lib().nmi_gqa_attention_workspace_bytes(q_heads, kv_heads, head_dim, tokens, batch, max_visible_keys))


def gqa_attention_workspace_bound(q_heads: int, tokens: int) -> int:
    """gqa_attention_workspace_bytes(q_heads, tokens) with the reference signature
    (gqa_attention.h:50): enough for every envelope of one sequence."""
    n = C.c_size_t(0)
    check(lib().nmi_gqa_attention_workspace_bound(int(q_heads), int(tokens), C.byref(n)))
    return int(n.value)


def gqa_attention(q, k, v, positions, scale, cache, envelope, workspace, out, stream=None) -> None:
    """A1: quantize-append k/v at `positions`, then causal GQA (gqa_attention.h:71-73)."""
    ws, nb = _ws(workspace)
    check(lib().nmi_gqa_attention(_p(q), _p(k), _p(v), _p(positions), float(scale), C.byref(cache),
                                  GqaEnvelope(*envelope), ws, nb, _p(out), _s(stream)))


def gqa_attention_noalloc(q, k, v, positions, scale, cache, envelope, out, stream=None) -> None:
    """A1 with the split partials in the library's static per-device scratch: allocates nothing,
    takes no workspace (no reference counterpart; for callers that cannot allocate)."""
    check(lib().nmi_gqa_attention_noalloc(_p(q), _p(k), _p(v), _p(positions), float(scale), C.byref(cache),
                                          GqaEnvelope(*envelope), _p(out), _s(stream)))


def gqa_kv_append(k, v, positions, cache, stream=None) -> None:
    """A2 (gqa_attention.h:80-81)."""
    check(lib().nmi_gqa_kv_append(_p(k), _p(v), _p(positions), C.byref(cache), _s(stream)))


def gqa_attention_cached(q, positions, scale, cache, envelope, workspace, out, stream=None) -> None:
    """A3 (gqa_attention.h:89-91)."""
    ws, nb = _ws(workspace)
    check(lib().nmi_gqa_attention_cached(_p(q), _p(positions), float(scale), C.byref(cache),
                                         GqaEnvelope(*envelope), ws, nb, _p(out), _s(stream)))


def gqa_attention_tree(q, k, v, positions, parents, scale, cache, envelope, write_cache, workspace,
                       out, stream=None) -> None:
    """Tree verification attention with an ancestor mask (extension)."""
    ws, nb = _ws(workspace)
    check(lib().nmi_gqa_attention_tree(_p(q), _p(k), _p(v), _p(positions), _p(parents), float(scale),
                                       C.byref(cache), GqaEnvelope(*envelope), int(bool(write_cache)),
                                       ws, nb, _p(out), _s(stream)))


# ---- paged cache (extension) -------------------------------------------------------------------
#
# Packed tokens: sequence b has tokens starts[b] .. starts[b + 1] - 1, the first at position history[b]
# (both I32 on the device). `cache` is a PagedKVLayerView (ninfer_amd.kv_cache.PagedKVCacheLayer.view()).

def paged_kv_append(k, v, starts, history, cache, stream=None) -> None:
    """Token i of sequence b to row history[b] + i of its pages (INT8-G64 quantised, or BF16 copied)."""
    check(lib().nmi_paged_kv_append(_p(k), _p(v), _p(starts), _p(history), C.byref(cache), _s(stream)))


def paged_kv_read(cache, starts, first, k_out, v_out, stream=None) -> None:
    """Row first[b] + i of sequence b to token starts[b] + i of k_out/v_out (BF16 or FP32 values)."""
    check(lib().nmi_paged_kv_read(C.byref(cache), _p(starts), _p(first), _p(k_out), _p(v_out), _s(stream)))


def paged_attention_workspace_bytes(q_heads: int, kv_heads: int, head_dim: int, tokens: int, batch: int, envelope,
                                    window=(0, 0)) -> int:
    return int(lib().nmi_paged_attention_workspace_bytes(q_heads, kv_heads, head_dim, tokens, batch, PagedEnvelope(*envelope),
                                                         AttentionWindow(*window)))


def paged_attention(q, starts, history, scale, window, cache, envelope, workspace, out, stream=None) -> None:
    """Causal attention of the packed tokens over their pages, new rows included. `window` (size, sinks): the last
    `size` rows and the first `sinks` ones, (0, 0) for every row. `envelope`: (most new tokens, most rows) of a sequence."""
    ws, nb = _ws(workspace)
    check(lib().nmi_paged_attention(_p(q), _p(starts), _p(history), float(scale), AttentionWindow(*window), C.byref(cache),
                                    PagedEnvelope(*envelope), ws, nb, _p(out), _s(stream)))


# ---- head norms and rotation (extension) --------------------------------------------------------

def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, norm, q_out, k_out, stream=None) -> None:
    """Every head normalised, times its weight, and rotated by positions * inv_freq in one pass. `norm`: (eps, weight_offset,
    interleaved); a weight may be None (ones), inv_freq None (no rotation)."""
    check(lib().nmi_qk_norm_rope(_p(q), _p(k), _p(q_weight), _p(k_weight), _p(positions), _p(inv_freq), NormRope(norm[0], norm[1], int(norm[2])),
                                 _p(q_out), _p(k_out), _s(stream)))


def paged_qk_norm_rope_append(q, k, v, q_weight, k_weight, starts, history, inv_freq, norm, cache, q_out, stream=None) -> None:
    """qk_norm_rope at the tokens' positions and paged_kv_append of the keys and values, in one pass."""
    check(lib().nmi_paged_qk_norm_rope_append(_p(q), _p(k), _p(v), _p(q_weight), _p(k_weight), _p(starts), _p(history), _p(inv_freq),
                                              NormRope(norm[0], norm[1], int(norm[2])), C.byref(cache), _p(q_out), _s(stream)))


# ---- sparse attention over blocks of a paged cache (extension) ------------------------------------
#
# `blocks` is a PagedBlockView (PagedKVCacheLayer(..., block_size=...).blocks()).

def paged_block_update(cache, starts, history, tokens: int, blocks, stream=None) -> None:
    """The means of the key blocks that hold the rows of the `tokens` packed tokens, which are in the cache already."""
    check(lib().nmi_paged_block_update(C.byref(cache), _p(starts), _p(history), int(tokens), C.byref(blocks), _s(stream)))


def paged_block_select_workspace_bytes(kv_heads: int, head_dim: int, tokens: int, batch: int, envelope, block_size: int) -> int:
    return int(lib().nmi_paged_block_select_workspace_bytes(kv_heads, head_dim, tokens, batch, PagedEnvelope(*envelope), block_size))


def paged_block_select(q, starts, history, page_table, page_size: int, blocks, selection, envelope, workspace, selected, stream=None) -> None:
    """For every token and KV head the blocks of `selection` (first, local, top): ascending in `selected`, -1 behind them."""
    ws, nb = _ws(workspace)
    check(lib().nmi_paged_block_select(_p(q), _p(starts), _p(history), _p(page_table), int(page_size), C.byref(blocks), BlockSelection(*selection),
                                       PagedEnvelope(*envelope), ws, nb, _p(selected), _s(stream)))


def paged_sparse_attention_workspace_bytes(q_heads: int, kv_heads: int, head_dim: int, tokens: int, batch: int, selected_blocks: int,
                                           block_size: int) -> int:
    return int(lib().nmi_paged_sparse_attention_workspace_bytes(q_heads, kv_heads, head_dim, tokens, batch, selected_blocks, block_size))


def paged_sparse_attention(q, starts, history, scale, selected, block_size: int, cache, envelope, workspace, out, stream=None) -> None:
    """paged_attention over the rows of the blocks that each token's list holds for the KV head (I32 [S, Hkv, N], negative: none)."""
    ws, nb = _ws(workspace)
    check(lib().nmi_paged_sparse_attention(_p(q), _p(starts), _p(history), float(scale), _p(selected), int(block_size), C.byref(cache),
                                           PagedEnvelope(*envelope), ws, nb, _p(out), _s(stream)))


# ---- pages of a paged cache (extension) ------------------------------------------------------------
#
# `refs` counts the entries of the page table that hold each page (PagedKVCacheLayer.refs); a page without any is free.

def paged_kv_copy_pages(cache, blocks, src, dst, stream=None) -> None:
    """Page src[i] to page dst[i] (negative: none), with its block means where `blocks` is not None."""
    check(lib().nmi_paged_kv_copy_pages(C.byref(cache), C.byref(blocks) if blocks is not None else None, _p(src), _p(dst), _s(stream)))


def paged_pages_reserve(page_table, refs, starts, history, page_size: int, granted, stream=None) -> None:
    """Free pages (the lowest first) for the new rows that have none; granted[b]: the new tokens of b that have theirs."""
    check(lib().nmi_paged_pages_reserve(_p(page_table), _p(refs), _p(starts), _p(history), int(page_size), _p(granted), _s(stream)))


def paged_pages_release(page_table, refs, sequences, keep_rows, page_size: int, stream=None) -> None:
    """Sequence sequences[i] gives back the pages past its first keep_rows[i] rows."""
    check(lib().nmi_paged_pages_release(_p(page_table), _p(refs), _p(sequences), _p(keep_rows), int(page_size), _s(stream)))


def paged_pages_fork(page_table, refs, parents, children, history, page_size: int, src, dst, stream=None) -> None:
    """Sequence children[i] as a copy of parents[i]: whole pages shared, the rest in a page of its own that paged_kv_copy_pages(src,
    dst) fills."""
    check(lib().nmi_paged_pages_fork(_p(page_table), _p(refs), _p(parents), _p(children), _p(history), int(page_size), _p(src), _p(dst),
                                     _s(stream)))


def paged_pages_compact(page_table, refs, src, dst, moved, stream=None) -> None:
    """The highest pages in use to the lowest free ones: table and counts now, contents by paged_kv_copy_pages(src, dst)."""
    check(lib().nmi_paged_pages_compact(_p(page_table), _p(refs), _p(src), _p(dst), _p(moved), _s(stream)))


# ---- acceptance (argmax.h, sampling.h, speculative_round.h) ------------------------------------

def argmax(logits, out, valid_rows: int, stream=None) -> None:
    check(lib().nmi_argmax(_p(logits), _p(out), int(valid_rows), _s(stream)))


def sampling_workspace_bytes(token_domain: int, columns: int, batch: int = 1) -> int:
    return int(lib().nmi_sampling_workspace_bytes(token_domain, columns, batch))


def speculative_prepare_verify_inputs(token, drafts, length, verify_ids, positions, stream=None) -> None:
    check(lib().nmi_speculative_prepare_verify_inputs(_p(token), _p(drafts), _p(length), _p(verify_ids),
                                                      _p(positions), _s(stream)))


def speculative_accept_greedy_drafts(target_tokens, logits, drafts, length, token, sampled_out,
                                     num_sampled, accepted, stats, token_domain: int, config_ptr: int,
                                     workspace, stream=None) -> None:
    """Greedy or reference-stochastic acceptance; `config_ptr` addresses device SamplingConfig[B]."""
    ws, nb = _ws(workspace)
    check(lib().nmi_speculative_accept_greedy_drafts(
        _p(target_tokens), _p(logits), _p(drafts), _p(length), _p(token), _p(sampled_out),
        _p(num_sampled), _p(accepted), _p(stats), int(token_domain), C.c_void_p(config_ptr), ws, nb,
        _s(stream)))


def general_accept_workspace_bytes(token_domain: int, K: int, batch: int = 1) -> int:
    return int(lib().nmi_general_accept_workspace_bytes(token_domain, K, batch))


def speculative_accept_general(logits, draft_logits, drafts, u_accept, u_residual, length, token,
                               sampled_out, num_sampled, accepted, stats, token_domain: int,
                               config_ptr: int, workspace, stream=None) -> None:
    """min(1, p/q) acceptance with normalized max(0, p - q) resampling (extension)."""
    ws, nb = _ws(workspace)
    check(lib().nmi_speculative_accept_general(
        _p(logits), _p(draft_logits), _p(drafts), _p(u_accept), _p(u_residual), _p(length), _p(token),
        _p(sampled_out), _p(num_sampled), _p(accepted), _p(stats), int(token_domain),
        C.c_void_p(config_ptr), ws, nb, _s(stream)))


def speculative_select_accepted_hidden(hidden, accepted, out, stream=None) -> None:
    check(lib().nmi_speculative_select_accepted_hidden(_p(hidden), _p(accepted), _p(out), _s(stream)))


def mtp_prepare_alignment_ids(verify_ids, token, accepted, alignment_ids, stream=None) -> None:
    """include/ninfer/ops/mtp_round.h:19-20."""
    check(lib().nmi_mtp_prepare_alignment_ids(_p(verify_ids), _p(token), _p(accepted), _p(alignment_ids), _s(stream)))


def tree_accept_greedy(parents, node_tokens, target_tokens, path, path_len, length, token,
                       sampled_out, num_sampled, accepted, stats, stream=None) -> None:
    check(lib().nmi_tree_accept_greedy(_p(parents), _p(node_tokens), _p(target_tokens), _p(path),
                                       _p(path_len), _p(length), _p(token), _p(sampled_out),
                                       _p(num_sampled), _p(accepted), _p(stats), _s(stream)))


# ---- lm_head (linear.h + the fused linear -> argmax) ----------------------------------------------

def linear(x, weight, out, stream=None) -> None:
    """include/ninfer/ops/linear.h:27 (Q6G64_F16S RowSplit weights)."""
    check(lib().nmi_linear(_p(x), C.byref(weight), _p(out), _s(stream)))


def linear_argmax_workspace_bytes(tokens) -> int:
    return lib().nmi_linear_argmax_workspace_bytes(tokens)


def linear_argmax(x, weight, valid_rows, ws, out, stream=None) -> None:
    """Fused linear -> argmax (the reference's deferred FUT-F03 contract)."""
    check(lib().nmi_linear_argmax(_p(x), C.byref(weight), int(valid_rows), C.c_void_p(ws.ptr), ws.nbytes, _p(out),
                                  _s(stream)))


def speculative_accept_fused_head_workspace_bytes(K: int, batch: int = 1) -> int:
    return int(lib().nmi_speculative_accept_fused_head_workspace_bytes(K, batch))


def speculative_accept_fused_head(x, weight, drafts, length, token, sampled_out, num_sampled, accepted, stats,
                                  token_domain: int, config_ptr: int, workspace, stream=None) -> None:
    """lm_head (Q6G64 linear) + speculative_accept_greedy_drafts in one call, the logits never written:
    x BF16 [hidden, K+1, B]; `config_ptr` addresses device SamplingConfig[B]."""
    ws, nb = _ws(workspace)
    check(lib().nmi_speculative_accept_fused_head(
        _p(x), C.byref(weight), _p(drafts), _p(length), _p(token), _p(sampled_out), _p(num_sampled), _p(accepted),
        _p(stats), int(token_domain), C.c_void_p(config_ptr), ws, nb, _s(stream)))


# ---- recurrent state of the hybrid layers (gated_delta_rule.h, causal_conv1d_silu.h, scalar.h) --

def gated_delta_rule_workspace_bytes(head_dim, qk_heads, value_heads, tokens, normalize_qk) -> int:
    """include/ninfer/ops/gated_delta_rule.h:18-21 (raises ValueError on an invalid geometry)."""
    import ctypes as C
    n = C.c_size_t(0)
    check(lib().nmi_gated_delta_rule_workspace_bytes(head_dim, qk_heads, value_heads, tokens,
                                                     1 if normalize_qk else 0, C.byref(n)))
    return n.value


def gated_delta_rule(q, k, v, g, beta, scale, normalize_qk, ssm_state_in, ssm_state_out, out,
                     stream=None) -> None:
    """include/ninfer/ops/gated_delta_rule.h:41-55; pass the same tensor twice for the in-place form."""
    check(lib().nmi_gated_delta_rule(_p(q), _p(k), _p(v), _p(g), _p(beta), scale, 1 if normalize_qk else 0,
                                     _p(ssm_state_in), _p(ssm_state_out), _p(out), _s(stream)))


def gated_delta_rule_snapshot(q, k, v, g, beta, scale, normalize_qk, ssm_states, initial_slot, out,
                              stream=None) -> None:
    """include/ninfer/ops/gated_delta_rule.h:57-68."""
    check(lib().nmi_gated_delta_rule_snapshot(_p(q), _p(k), _p(v), _p(g), _p(beta), scale,
                                              1 if normalize_qk else 0, _p(ssm_states), _p(initial_slot),
                                              _p(out), _s(stream)))


def causal_conv1d_silu(x, weight, conv_state_in, conv_state_out, out, stream=None) -> None:
    """include/ninfer/ops/causal_conv1d_silu.h:23-31; pass the same tensor twice for the in-place form."""
    check(lib().nmi_causal_conv1d_silu(_p(x), _p(weight), _p(conv_state_in), _p(conv_state_out), _p(out),
                                       _s(stream)))


def causal_conv1d_silu_snapshot(x, weight, conv_states, initial_slot, out, stream=None) -> None:
    """include/ninfer/ops/causal_conv1d_silu.h:33-40."""
    check(lib().nmi_causal_conv1d_silu_snapshot(_p(x), _p(weight), _p(conv_states), _p(initial_slot), _p(out),
                                                _s(stream)))


def set_i32_scalar(destination, value, stream=None) -> None:
    check(lib().nmi_set_i32_scalar(_p(destination), value, _s(stream)))


def assign_i32_scalar(source, destination, stream=None) -> None:
    check(lib().nmi_assign_i32_scalar(_p(source), _p(destination), _s(stream)))


def increment_i32_scalar(scalar, stream=None) -> None:
    check(lib().nmi_increment_i32_scalar(_p(scalar), _s(stream)))


def increment_i64_scalar(scalar, stream=None) -> None:
    check(lib().nmi_increment_i64_scalar(_p(scalar), _s(stream)))


# ---- commit / rollback (kv_cache_append_prefix.h + extensions) ----------------------------------

def kv_cache_append_prefix(k, v, positions, commit_count, envelope, cache, stream=None) -> None:
    check(lib().nmi_kv_cache_append_prefix(_p(k), _p(v), _p(positions), _p(commit_count),
                                           CommitEnvelope(*envelope), C.byref(cache), _s(stream)))


def kv_cache_append_prefix_cyclic(k, v, positions, commit_count, envelope, cache, stream=None) -> None:
    """The cyclic overload (kv_cache_append_prefix.h:40-51): row = position % capacity."""
    check(lib().nmi_kv_cache_append_prefix_cyclic(_p(k), _p(v), _p(positions), _p(commit_count),
                                                  CommitEnvelope(*envelope), C.byref(cache), _s(stream)))


def kv_cache_rollback(positions, keep_count, cache, stream=None) -> None:
    check(lib().nmi_kv_cache_rollback(_p(positions), _p(keep_count), C.byref(cache), _s(stream)))


def kv_cache_compact_path(base_position, path, path_len, cache, stream=None) -> None:
    check(lib().nmi_kv_cache_compact_path(_p(base_position), _p(path), _p(path_len), C.byref(cache),
                                          _s(stream)))
