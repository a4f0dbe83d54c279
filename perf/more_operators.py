"""Operators around a paged KV cache, as measurable cases: what stands between a projection and the cache, sparse
attention over blocks of the cache, and the pages themselves.

A serving program with many sequences takes the projections of the new tokens, normalises every head of the queries and
keys and rotates them by position (and appends the keys and values to the cache in the same pass); keeps a mean of every
block of keys, selects for each new token and KV head the blocks whose means its queries score highest, next to a few
first and last ones, and attends over those alone; forks sequences (several answers to one prompt), gives pages back,
closes the gaps that this leaves in the pool and hands pages out again.

Layout: a pool plane is [pages, KV heads, page, D]; INT8 planes have FP16 scales [pages, KV heads, page, D / 64]; block
means are INT8 codes [pages, KV heads, page / block, D] with an FP32 scale each; the table is [sequences, pages]; `refs`
counts the table entries of each page. Tokens of all sequences are packed: sequence b has tokens starts[b] ..
starts[b + 1] - 1, and its first one stands at position history[b]. Sizes come from the package's benchmark and tests (its
head geometries) or are generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
# (query heads, KV heads, head_dim) of the package's attention
GEOMETRIES = ((40, 8, 128), (24, 4, 256), (16, 2, 256))
EPS = 1e-6
PAGE_KINDS = ("fork", "turnover")


# ---- the cases -------------------------------------------------------------------------------

def _case(**kw):
    c = dict(kind="rope", q_heads=40, kv_heads=8, head_dim=128, cache="int8", page=64, block=64, batch=1, tokens=1, tokens_min=0,
             history=0, history_min=0, rotary=128, interleaved=False, offset=0.0, first=1, local=2, top=13, forks=0, pages=0)
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of 16 conversations: queries and keys as slices of the fused projection
        _case(name="rope_step", batch=16, history=30000, history_min=100),
        # a long prompt deep in a document, a quarter of each head rotated, weights stored around zero
        _case(name="rope_prompt", q_heads=24, kv_heads=4, head_dim=256, tokens=8192, history=900000, rotary=64, offset=1.0),
        # one decode step of 32 conversations, straight into the INT8 cache
        _case(name="rope_append_step", kind="rope_append", batch=32, history=8000, history_min=100),
        # several prompts of odd lengths into a BF16 cache, neighbouring dims rotated as pairs
        _case(name="rope_append_prompts", kind="rope_append", q_heads=24, kv_heads=4, head_dim=256, cache="bf16", batch=5, tokens=1301, tokens_min=437,
              history=2000, interleaved=True, rotary=256),
        # the block means of a long prompt
        _case(name="means_prompt", kind="means", batch=2, tokens=16000, tokens_min=9000, history=1000),
        # blocks for one decode step of 32 long conversations
        _case(name="select_decode", kind="select", batch=32, history=131072, history_min=20000, top=61),
        # blocks for every token of a prompt chunk over a long history, pages of two blocks
        _case(name="select_chunk", kind="select", page=128, tokens=4096, history=16384, top=29),
        # one token of one long document: launches and latency
        _case(name="attend_one", kind="attend", history=131000, top=29),
        # a decode step of 32 ragged conversations
        _case(name="attend_batch32", kind="attend", batch=32, history=65536, history_min=9000, top=61),
        # a prompt chunk over a BF16 cache at a head_dim-256 geometry, every token with blocks of its own
        _case(name="attend_chunk", kind="attend", q_heads=24, kv_heads=4, head_dim=256, cache="bf16", tokens=2048, history=12000, top=13),
        # 48 answers to four prompts: shared pages, a page of its own for each answer's unfinished one
        _case(name="fork_answers", kind="fork", cache="bf16", batch=64, forks=48, tokens=700, tokens_min=300, pages=4096),
        # half of the conversations end, the gaps close, the next prompts come in
        _case(name="turnover", kind="turnover", cache="bf16", page=32, batch=64, tokens=2000, tokens_min=300, pages=6144),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rope", "rope_append", "means", "select", "select", "attend", "attend", "attend", "fork", "turnover"))
    hq, hkv, d = rng.choice(GEOMETRIES)
    page = rng.choice((32, 64, 128))
    geo = dict(q_heads=hq, kv_heads=hkv, head_dim=d, cache=rng.choice(("int8", "bf16")), page=page, block=rng.choice([b for b in (32, 64, 128) if b <= page]))
    if kind in ("rope", "rope_append"):
        n = _log_int(rng, 1, 4000)
        return _case(**geo, kind=kind, batch=rng.randint(1, 2 if n > 500 else 16), tokens=n, tokens_min=max(1, n // 3),
                     history=_log_int(rng, 1, 100000) if kind == "rope" else _log_int(rng, 1, 4000), rotary=rng.choice((d, d // 2, 64)),
                     interleaved=rng.random() < 0.3, offset=rng.choice((0.0, 1.0)))
    if kind == "means":
        n = _log_int(rng, 1, 9000)
        return _case(**geo, kind=kind, batch=rng.randint(1, 3), tokens=n, tokens_min=max(1, n // 3), history=rng.randint(0, 3000))
    pick = dict(first=rng.choice((0, 1, 2)), local=rng.choice((1, 2, 3)), top=rng.randint(1, 40))
    if kind in ("select", "attend") and rng.random() < 0.6:  # single tokens, or the tokens of a verify round
        high = _log_int(rng, 2000, 60000)
        return _case(**geo, kind=kind, batch=_log_int(rng, 1, 24), tokens=rng.choice((1, 1, 1, 4)), history=high, history_min=max(1, high // 8), **pick)
    if kind == "select":
        return _case(**geo, kind=kind, tokens=_log_int(rng, 20, 3000), history=_log_int(rng, 100, 16000), **pick)
    if kind == "attend":
        pick["top"] = rng.randint(1, 10)
        return _case(**geo, kind=kind, tokens=_log_int(rng, 20, 1000), history=_log_int(rng, 100, 12000), **pick)
    geo.update(cache="bf16", kind=kind)
    if kind == "fork":
        batch = rng.randint(4, 64)
        n = _log_int(rng, 40, 900)
        return _case(**geo, batch=batch, forks=rng.randint(1, batch * 3 // 4), tokens=n, tokens_min=max(1, n // 3), pages=4000)
    n = _log_int(rng, 40, 1500)
    return _case(**geo, batch=rng.randint(2, 48), tokens=n, tokens_min=max(1, n // 3), pages=5000)


def _sequences(c):
    """(new tokens, rows before them) of every sequence: part of the case, the same for every seed."""
    r = random.Random(c["tokens"] * 7919 + c["history"] * 31 + c["batch"])
    return [(r.randint(c["tokens_min"], c["tokens"]) if c["tokens_min"] else c["tokens"],
             r.randint(c["history_min"], c["history"]) if c["history_min"] else c["history"]) for _ in range(c["batch"])]


def _blocks_of(c):
    return c["first"] + c["local"] + c["top"]


def _parents(c):
    """Fork: the first sequences hold prompts, the last ones become the answers, dealt out evenly."""
    prompts = max(1, (c["batch"] - c["forks"]) // 4)
    return [i % prompts for i in range(c["forks"])], list(range(c["batch"] - c["forks"], c["batch"]))


def _ceil(a, b):
    return -(-a // b)


def work(c):
    H, D, Hq, ps, bs = c["kv_heads"], c["head_dim"], c["q_heads"], c["page"], c["block"]
    seqs = _sequences(c)
    n = sum(t for t, _ in seqs)
    row = H * 2 * (D + D // 32) if c["cache"] == "int8" else H * 4 * D  # bytes of K and V of one cache row
    if c["kind"] == "rope":
        return {"bytes": n * (Hq + H) * D * 4, "flops": 10.0 * n * (Hq + H) * D}
    if c["kind"] == "rope_append":
        back = n * (row + 4 * H * D) if c["cache"] == "int8" else 0
        return {"bytes": n * (Hq * D * 4 + 4 * H * D + row) + back, "flops": n * (10.0 * (Hq + H) + 4.0 * H) * D}
    if c["kind"] == "means":
        rows = sum(h + t - h // bs * bs for t, h in seqs)
        blocks = sum(_ceil(h + t, bs) - h // bs for t, h in seqs)
        return {"bytes": rows * row // 2 + blocks * H * (D + 4) + blocks * H * D * 4, "flops": 2.0 * rows * H * D}
    if c["kind"] == "select":
        means = sum(_ceil(h + t, bs) for t, h in seqs) * H * (D + 4)
        return {"bytes": means + n * (Hq * D * 2 + H * _blocks_of(c) * 4), "flops": 2.0 * D * H * sum(t * _ceil(h + t, bs) for t, h in seqs)}
    if c["kind"] == "attend":
        S = _blocks_of(c)
        # a row that several tokens take is read once at least, one that a token takes at most once for it
        rows = sum(min(h + t, t * S * bs) for t, h in seqs)
        pairs = sum(min(h + i + 1, S * bs) for t, h in seqs for i in range(t))
        return {"bytes": rows * row + n * (Hq * D * 4 + H * S * 4), "flops": 4.0 * D * Hq * pairs}
    page = ps * H * 4 * D
    if c["kind"] == "fork":
        moved = sum(1 for p in _parents(c)[0] if seqs[p][0] % ps)
        return {"bytes": 2 * moved * page + 8 * c["forks"] * _ceil(c["tokens"], ps) + 4 * c["pages"], "flops": 1.0}
    moved = sum(_ceil(t, ps) for t, _ in seqs) / 4  # about half of what stays lies above the new end
    return {"bytes": 2 * moved * page + 8 * sum(_ceil(t, ps) for t, _ in seqs) + 4 * c["pages"], "flops": 1.0}


# ---- inputs ----------------------------------------------------------------------------------

def _quantize(x):
    """Codes and FP16 scales of rows [..., D]: s = FP16(amax / 127), code = clamp(rne(x * FP32(1 / s)), +-127)."""
    xf = x.float().unflatten(-1, (-1, 64))
    s = (xf.abs().amax(-1) / 127.0).half()
    inv = torch.where(s > 0, 1.0 / s.float(), 0.0)
    return (xf * inv[..., None]).round_().clamp_(-127, 127).to(torch.int8).flatten(-2), s


def _rows(g, shape, gain):
    """Keys or values as a layer leaves them: normal, with one dimension in 32 larger than the others."""
    x = torch.randn(shape, generator=g, device=DEV)
    x[..., ::32] *= gain
    return x.to(torch.bfloat16)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    H, D, ps, bs, Hq = c["kv_heads"], c["head_dim"], c["page"], c["block"], c["q_heads"]
    seqs = _sequences(c)
    s = dict(case=c, seqs=seqs, n=sum(t for t, _ in seqs))
    s["lengths"] = torch.tensor([t for t, _ in seqs], device=DEV, dtype=torch.int32)
    s["history"] = torch.tensor([h for _, h in seqs], device=DEV, dtype=torch.int32)
    s["starts"] = torch.nn.functional.pad(s["lengths"].cumsum(0), (1, 0)).to(torch.int32)
    if c["kind"] in ("rope", "rope_append"):
        qkv = torch.randn((s["n"], Hq + 2 * H, D), generator=g, device=DEV)
        qkv[..., ::32] *= 4.0
        qkv = qkv.to(torch.bfloat16)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
        s["q_weight"], s["k_weight"] = ((1.0 - c["offset"] + 0.2 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16) for _ in range(2))
        base = 1e4 if c["rotary"] < 128 else 1e6
        s["inv_freq"] = (base ** (-torch.arange(0, c["rotary"], 2, device=DEV, dtype=torch.float64) / c["rotary"])).float()
        if c["kind"] == "rope":
            token = torch.arange(s["n"], device=DEV)
            b = torch.searchsorted(s["starts"], token.int(), right=True) - 1
            s["positions"] = (s["history"][b] + token - s["starts"][b]).to(torch.int32)
            if own:
                s.update(_handle(s))
            torch.cuda.synchronize()
            return s
    if c["kind"] in PAGE_KINDS:
        _prepare_pages(s, g)
    else:
        need = [_ceil(t + h, ps) for t, h in seqs]
        pages = sum(need)
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)  # a pool in use hands out pages in any order
        table = torch.full((len(seqs), max(need)), -1, device=DEV, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            table[b, :k] = order[at:at + k]
            at += k
        s["table"] = table
        q8 = c["cache"] == "int8"
        shape = (pages, H, ps, D)
        if c["kind"] != "select":
            s["pool"] = [torch.zeros(shape, device=DEV, dtype=torch.int8 if q8 else torch.bfloat16) for _ in range(2)]
            if q8:
                s["pool"] += [torch.zeros((*shape[:3], D // 64), device=DEV, dtype=torch.float16) for _ in range(2)]
        step = max(1, (1 << 26) // (H * ps * D))
        for i in range(0, pages if c["kind"] in ("means", "attend") else 0, step):
            k = min(step, pages - i)
            for plane in range(2):
                x = _rows(g, (k, *shape[1:]), 4.0 if plane == 0 else 2.0)
                if q8:
                    s["pool"][plane][i:i + k], s["pool"][2 + plane][i:i + k] = _quantize(x)
                else:
                    s["pool"][plane][i:i + k] = x
    if c["kind"] in ("means", "select"):
        shape = (s["table"].amax().item() + 1, H, ps // bs)
        s["codes"] = torch.zeros((*shape, D), device=DEV, dtype=torch.int8)
        s["scales"] = torch.zeros(shape, device=DEV)
    if c["kind"] == "select":  # means of keys: the average over the blocks stands out in a few dimensions
        mean = torch.randn((*s["codes"].shape,), generator=g, device=DEV).mul_(1.0 / math.sqrt(bs))
        mean[..., ::32] += 2.0 * torch.randn((H, 1, D // 32), generator=g, device=DEV)
        s["codes"], s["scales"] = _mean_codes(mean.double(), 1)
        s["q"] = torch.randn((s["n"], Hq, D), generator=g, device=DEV).to(torch.bfloat16)
    if c["kind"] == "attend":
        s["q"] = torch.randn((s["n"], Hq, D), generator=g, device=DEV).to(torch.bfloat16)
        # blocks as a selection leaves them: neighbouring tokens mostly agree
        blocks = max(_ceil(t + h, bs) for t, h in seqs)
        b, pos = _tokens(s)
        like = torch.randn((len(seqs), H, blocks), generator=g, device=DEV)[b] + 0.5 * torch.randn((s["n"], H, blocks), generator=g, device=DEV)
        s["selected"] = _choose(like, torch.ones_like(like, dtype=torch.bool), (pos // bs)[:, None], c)
    if own:
        s.update(_handle(s))
    torch.cuda.synchronize()
    return s


def _prepare_pages(s, g):
    """A pool in use: every sequence (the answers aside) holds a prompt in random pages; a fork's lists, a turnover's groups."""
    c, seqs = s["case"], s["seqs"]
    ps, B = c["page"], c["batch"]
    holds = [0 if c["kind"] == "fork" and b >= B - c["forks"] else _ceil(t, ps) for b, (t, _) in enumerate(seqs)]
    order = torch.randperm(c["pages"], generator=g, device=DEV).to(torch.int32)
    width = _ceil(c["tokens"], ps) + 1
    first = [sum(holds[:b]) for b in range(B)]
    at = torch.arange(width, device=DEV)[None]
    first, holds = (torch.tensor(x, device=DEV)[:, None] for x in (first, holds))
    s["table"] = torch.where(at < holds, order[(first + at).clamp(max=c["pages"] - 1)], -1).to(torch.int32)
    s["refs"] = torch.zeros(c["pages"], device=DEV, dtype=torch.int32)
    _count(s, s["table"], 1)
    s["pool"] = [_rows(g, (c["pages"], c["kv_heads"], ps, c["head_dim"]), 2.0) for _ in range(2)]
    if c["kind"] == "fork":
        s["parents"], s["children"] = (torch.tensor(x, device=DEV, dtype=torch.int32) for x in _parents(c))
        s["history"] = torch.where(holds[:, 0] > 0, s["lengths"], 0).to(torch.int32)
        s["src"], s["dst"] = (torch.zeros(c["forks"], device=DEV, dtype=torch.int32) for _ in range(2))
        return
    # turnover: two groups of sequences take turns at ending; the group that ended comes back with prompts of the same lengths
    s["turn"] = 0
    odd = torch.arange(B, device=DEV) % 2
    s["groups"], s["group_starts"], s["entries"] = [], [], []
    s["keep"] = torch.zeros(_ceil(B, 2), device=DEV, dtype=torch.int32)
    for k in range(2):
        s["groups"].append(torch.arange(k, B, 2, device=DEV, dtype=torch.int32))
        s["group_starts"].append(torch.nn.functional.pad(torch.where(odd == k, s["lengths"], 0).cumsum(0), (1, 0)).to(torch.int32))
        s["entries"].append(sum(_ceil(t, ps) for t, _ in seqs[k::2]))
    s["history"] = torch.zeros(B, device=DEV, dtype=torch.int32)
    s["src"], s["dst"] = (torch.zeros(c["pages"] // 2, device=DEV, dtype=torch.int32) for _ in range(2))
    s["moved"] = torch.zeros(1, device=DEV, dtype=torch.int32)
    s["granted"] = torch.zeros(B, device=DEV, dtype=torch.int32)


def _handle(s):
    """The views, buffers and workspaces that a program keeps for these calls."""
    import ninfer_amd as na
    from ninfer_amd import ops
    from ninfer_amd.device import DeviceBuffer

    kinds = {torch.bfloat16: na.BF16, torch.float32: na.FP32, torch.int32: na.I32, torch.int8: na.I8, torch.float16: na.FP16}

    def view(t):
        v = na.Tensor.make(t.data_ptr(), kinds[t.dtype], tuple(reversed(t.shape)))
        v.nb[t.dim() - 1] = t.stride(0) * t.element_size()  # a slice of a projection: tokens further apart
        return v

    c = s["case"]
    H, D, ps, bs, n, B = c["kv_heads"], c["head_dim"], c["page"], c["block"], s["n"], c["batch"]
    h = dict(ops=ops)
    if c["kind"] in ("rope", "rope_append"):
        h["norm"] = (EPS, c["offset"], c["interleaved"])
        h["q_out"] = torch.zeros((n, c["q_heads"], D), device=DEV, dtype=torch.bfloat16)
        if c["kind"] == "rope" or c["cache"] == "int8":
            h["k_out"], h["v_out"] = (torch.zeros((n, H, D), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    if "pool" in s or "codes" in s:
        cache = na.PagedKVLayerView()
        if "pool" in s:
            cache.k, cache.v = view(s["pool"][0]), view(s["pool"][1])
            if c["cache"] == "int8":
                cache.k_scale, cache.v_scale = view(s["pool"][2]), view(s["pool"][3])
            cache.dtype, cache.quant_group = (na.I8, 64) if c["cache"] == "int8" else (na.BF16, 0)
        cache.page_table = view(s["table"])
        cache.page_size, cache.num_kv_heads, cache.head_dim = ps, H, D
        h["cache"] = cache
    h["envelope"] = (max(1, max(t for t, _ in s["seqs"])), max(1, max(t + r for t, r in s["seqs"])))
    if "codes" in s:
        blocks = na.PagedBlockView()
        blocks.codes, blocks.scales, blocks.block_size = view(s["codes"]), view(s["scales"]), bs
        h["blocks"] = blocks
    if c["kind"] == "select":
        h["selected"] = torch.full((n, H, _blocks_of(c)), -1, device=DEV, dtype=torch.int32)
        need = ops.paged_block_select_workspace_bytes(H, D, n, B, h["envelope"], bs)
        h["ws"] = DeviceBuffer(max(256, need))
    if c["kind"] == "attend":
        h["out"] = torch.zeros_like(s["q"])
        need = ops.paged_sparse_attention_workspace_bytes(c["q_heads"], H, D, n, B, _blocks_of(c), bs)
        h["ws"] = DeviceBuffer(max(256, need))
    both = {**s, **h}
    names = ("q", "k", "v", "q_weight", "k_weight", "inv_freq", "positions", "starts", "history", "q_out", "k_out", "v_out", "selected", "out", "table",
             "refs", "parents", "children", "src", "dst", "keep", "moved", "granted")
    h["views"] = {k: view(both[k]) for k in names if k in both}
    if c["kind"] == "turnover":
        h["group_views"] = [(view(a), view(s["keep"][:a.numel()]), view(b)) for a, b in zip(s["groups"], s["group_starts"])]
    return h


# ---- one pass --------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "rope":
        return _norm_rope(s["q"], s["q_weight"], s["positions"], s), _norm_rope(s["k"], s["k_weight"], s["positions"], s)
    if c["kind"] == "rope_append":
        return _rope_append(s, c)
    if c["kind"] == "means":
        return _means(s, c)
    if c["kind"] == "select":
        return _select(s, c)
    if c["kind"] == "attend":
        return _attend(s, c)
    return _fork(s, c) if c["kind"] == "fork" else _turnover(s, c)


def _run_own(s, c):
    ops, v = s["ops"], s["views"]
    if c["kind"] == "rope":
        ops.qk_norm_rope(v["q"], v["k"], v["q_weight"], v["k_weight"], v["positions"], v["inv_freq"], s["norm"], v["q_out"], v["k_out"])
        return s["q_out"], s["k_out"]
    if c["kind"] == "rope_append":
        ops.paged_qk_norm_rope_append(v["q"], v["k"], v["v"], v["q_weight"], v["k_weight"], v["starts"], v["history"], v["inv_freq"], s["norm"],
                                      s["cache"], v["q_out"])
        if c["cache"] == "bf16":
            return s["q_out"], *s["pool"]
        ops.paged_kv_read(s["cache"], v["starts"], v["history"], v["k_out"], v["v_out"])
        return s["q_out"], s["k_out"], s["v_out"]
    if c["kind"] == "means":
        ops.paged_block_update(s["cache"], v["starts"], v["history"], s["n"], s["blocks"])
        return s["codes"] * s["scales"][..., None]
    if c["kind"] == "select":
        ops.paged_block_select(v["q"], v["starts"], v["history"], v["table"], c["page"], s["blocks"], (c["first"], c["local"], c["top"]), s["envelope"],
                               s["ws"], v["selected"])
        return s["selected"]
    if c["kind"] == "attend":
        ops.paged_sparse_attention(v["q"], v["starts"], v["history"], 1.0 / math.sqrt(c["head_dim"]), v["selected"], c["block"], s["cache"],
                                   s["envelope"], s["ws"], v["out"])
        return s["out"]
    if c["kind"] == "fork":
        ops.paged_pages_fork(v["table"], v["refs"], v["parents"], v["children"], v["history"], c["page"], v["src"], v["dst"])
        ops.paged_kv_copy_pages(s["cache"], None, v["src"], v["dst"])
        return s["table"], s["refs"], s["history"], s["src"], s["dst"], *s["pool"]
    gone, keep, starts = s["group_views"][s["turn"]]
    s["turn"] ^= 1
    ops.paged_pages_release(v["table"], v["refs"], gone, keep, c["page"])
    ops.paged_pages_compact(v["table"], v["refs"], v["src"], v["dst"], v["moved"])
    ops.paged_kv_copy_pages(s["cache"], None, v["src"], v["dst"])
    ops.paged_pages_reserve(v["table"], v["refs"], starts, v["history"], c["page"], v["granted"])
    return s["table"], s["refs"], s["src"], s["dst"], s["moved"], s["granted"], *s["pool"]


# The plain form: torch operations in 32 bits (64 for angles and for what a selection hangs on).

def _tokens(s):
    """(sequence, position) of every packed token."""
    token = torch.arange(s["n"], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["starts"], token, right=True) - 1
    return b, s["history"][b] + token - s["starts"][b]


def _norm_rope(x, weight, positions, s):
    c = s["case"]
    R = c["rotary"]
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * (weight.float() + c["offset"])
    angle = positions.double()[:, None, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if c["interleaved"] else (y[..., :R // 2], y[..., R // 2:R])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., R:]), -1).to(torch.bfloat16)


def _rope_append(s, c):
    b, pos = _tokens(s)
    q = _norm_rope(s["q"], s["q_weight"], pos, s)
    k = _norm_rope(s["k"], s["k_weight"], pos, s)
    page, row = s["table"][b, pos // c["page"]].long(), pos % c["page"]
    if c["cache"] == "bf16":
        s["pool"][0][page, :, row] = k
        s["pool"][1][page, :, row] = s["v"]
        return q, *s["pool"]
    s["pool"][0][page, :, row], s["pool"][2][page, :, row] = _quantize(k)
    s["pool"][1][page, :, row], s["pool"][3][page, :, row] = _quantize(s["v"])
    return q, _read(s, 0, page, row), _read(s, 1, page, row)


def _read(s, plane, page, row):
    x = s["pool"][plane][page, :, row].float().unflatten(-1, (-1, 64))
    return (x * s["pool"][2 + plane][page, :, row].float()[..., None]).flatten(-2).to(torch.bfloat16)


def _mean_codes(total, n):
    """INT8 codes and an FP32 scale of means total / n, 64-bit totals [..., D]: step = amax / 127, code = rne(total * (1 / step))."""
    step = total.abs().amax(-1) / 127.0
    return (total * (1.0 / step)[..., None]).round().clamp(-127, 127).to(torch.int8), (step / n).float()


def _means(s, c):
    ps, bs, B = c["page"], c["block"], c["batch"]
    per, H, D = ps // bs, c["kv_heads"], c["head_dim"]
    end = s["history"] + s["lengths"]
    first = s["history"] // bs
    count = (end + bs - 1) // bs - first
    total = sum(_ceil(h + t, bs) - h // bs for t, h in s["seqs"])
    b = torch.repeat_interleave(torch.arange(B, device=DEV), count, output_size=total)
    block = first[b] + torch.arange(total, device=DEV) - (count.cumsum(0) - count)[b]
    page, slot = s["table"][b, block // per].long(), block % per
    x = s["pool"][0].view(-1, H, per, bs, D)[page, :, slot].float()
    if c["cache"] == "int8":
        x = (x.unflatten(-1, (-1, 64)) * s["pool"][2].view(-1, H, per, bs, D // 64)[page, :, slot].float()[..., None]).flatten(-2)
    rows = (end[b] - block * bs).clamp(max=bs)
    x = torch.where((torch.arange(bs, device=DEV) < rows[:, None])[:, None, :, None], x, 0.0)
    s["codes"][page, :, slot], s["scales"][page, :, slot] = _mean_codes(x.double().sum(2), rows[:, None])
    return s["codes"] * s["scales"][..., None]


def _choose(score, there, last, c):
    """Of blocks [.., blocks], those of a token whose own one is `last`: the first and the last ones and the `top` highest scores of
    the others that are there (the lower one of equals), in ascending order, -1 behind them."""
    S, blocks = _blocks_of(c), score.shape[-1]
    at = torch.arange(blocks, device=DEV)
    last = last[..., None]
    always = ((at < c["first"]) | (at > last - c["local"])) & (at <= last)
    open_ = there & (at >= c["first"]) & (at <= last - c["local"])
    order = torch.sort(torch.where(open_, score, -math.inf), dim=-1, descending=True, stable=True).indices[..., :c["top"]]
    chosen = (always | (open_ & torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order, True)))
    found = torch.where(chosen, at, blocks).sort(-1).values[..., :S]
    found = torch.nn.functional.pad(found, (0, S - found.shape[-1]), value=blocks)
    return torch.where(found < blocks, found, -1).to(torch.int32)


def _select(s, c):
    """Scores in whole numbers times a scale: the queries of a KV head summed, as INT8 codes, against the codes of the means."""
    ps, bs, H, D, B = c["page"], c["block"], c["kv_heads"], c["head_dim"], c["batch"]
    per, T = ps // bs, max(t for t, _ in s["seqs"])
    blocks = max(_ceil(t + h, bs) for t, h in s["seqs"])
    at = torch.arange(blocks, device=DEV)
    page = s["table"][:, at // per]
    there, page = page >= 0, page.clamp(min=0).long()
    mean = s["codes"][page, :, at % per].float().permute(0, 2, 3, 1)  # [B, H, D, blocks]
    scale = s["scales"][page, :, at % per].permute(0, 2, 1)
    token = s["starts"][:-1, None] + torch.arange(T, device=DEV)
    q = s["q"][token.clamp(max=s["n"] - 1)].double().unflatten(2, (H, -1)).sum(3)  # [B, T, H, D]
    q = _mean_codes(q, 1)[0].float().transpose(1, 2)
    score = torch.bmm(q.reshape(B * H, T, D), mean.reshape(B * H, D, blocks).contiguous()).view(B, H, T, blocks) * scale[:, :, None]
    last = (s["history"][:, None] + torch.arange(T, device=DEV)) // bs
    found = _choose(score, there[:, None, None], last[:, None], c).transpose(1, 2)  # [B, T, H, S]
    b, pos = _tokens(s)
    return found[b, (pos - s["history"][b]).long()].contiguous()


def _attend(s, c):
    H, D, ps, bs, n = c["kv_heads"], c["head_dim"], c["page"], c["block"], s["n"]
    b, pos = _tokens(s)
    row = (s["selected"].long()[..., None] * bs + torch.arange(bs, device=DEV)).flatten(-2)  # [n, H, rows]
    seen = (row >= 0) & (row <= pos[:, None, None])
    row = torch.where(seen, row, 0)
    page = s["table"][b[:, None, None], row // ps].long()
    at = (page, torch.arange(H, device=DEV)[None, :, None], row % ps)

    def values(plane):
        x = s["pool"][plane][at].float()
        if c["cache"] == "int8":
            x = x.unflatten(-1, (-1, 64)).mul_(s["pool"][2 + plane][at].float()[..., None]).flatten(-2)
        return x.view(n * H, -1, D)
    q = s["q"].float().view(n * H, -1, D)
    score = torch.bmm(values(0), q.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(D))  # [n H, rows, G]
    score.masked_fill_(~seen.view(n * H, -1, 1), -math.inf)
    p = (score - score.amax(1, keepdim=True)).exp_()
    p /= p.sum(1, keepdim=True)
    return torch.bmm(p.transpose(1, 2).contiguous(), values(1)).view(n, -1, D).to(torch.bfloat16)


def _count(s, entries, by):
    """Adds `by` to the count of every page among the entries."""
    s["refs"].index_add_(0, entries.clamp(min=0).flatten(), torch.where(entries >= 0, by, 0).to(torch.int32).flatten())


def _free_page(refs, k):
    """The k-th page (from 0) that nothing holds, the lowest first; the number of pages where there is none."""
    return torch.searchsorted((refs == 0).cumsum(0).to(torch.int32), (k + 1).to(torch.int32))


def _copy_pages(s):
    src, dst = s["src"], s["dst"]
    live = (src >= 0) & (dst >= 0)
    # a pair without pages copies a live pair's page again (where there is none, page 0 to itself)
    one = live.to(torch.uint8).argmax(0, keepdim=True)
    src, dst = (torch.where(live, x, x.index_select(0, one)).clamp(min=0).long() for x in (src, dst))
    s["pool"][0][dst] = s["pool"][0].index_select(0, src)
    s["pool"][1][dst] = s["pool"][1].index_select(0, src)


def _fork(s, c):
    ps, table, refs = c["page"], s["table"], s["refs"]
    parent, child = s["parents"].long(), s["children"].long()
    free = refs.clone()  # what the answers give back is not for use in the same call
    _count(s, table[child], -1)
    rows = s["history"][parent]
    at = torch.arange(table.shape[1], device=DEV)
    whole = (rows // ps)[:, None]
    entries = torch.where(at < whole, table[parent], -1)
    _count(s, entries, 1)
    part = rows % ps > 0
    page = _free_page(free, part.cumsum(0) - part.int())
    part = part & (page < refs.numel())
    entries = torch.where((at == whole) & part[:, None], page[:, None].to(torch.int32), entries)
    s["src"].copy_(torch.where(part, table[parent, (rows // ps).long()], -1))
    s["dst"].copy_(torch.where(part, page, -1))
    _count(s, s["dst"], 1)
    table[child] = entries
    s["history"][child] = torch.where(part, rows, rows // ps * ps)
    _copy_pages(s)
    return table, refs, s["history"], s["src"], s["dst"], *s["pool"]


def _turnover(s, c):
    ps, table, refs, B = c["page"], s["table"], s["refs"], c["batch"]
    gone, starts, total = (s[k][s["turn"]] for k in ("groups", "group_starts", "entries"))
    s["turn"] ^= 1
    # the group's pages are given back
    _count(s, table[gone.long()], -1)
    table[gone.long()] = -1
    # the highest pages in use move to the lowest free ones
    used = refs > 0
    k = torch.arange(s["src"].numel(), device=DEV)
    to = _free_page(refs, k)
    of = refs.numel() - 1 - torch.searchsorted(used.flip(0).cumsum(0).to(torch.int32), (k + 1).to(torch.int32))
    moves = (to < of) & (to < refs.numel())
    s["src"].copy_(torch.where(moves, of, -1))
    s["dst"].copy_(torch.where(moves, to, -1))
    s["moved"].copy_(moves.sum())
    spare = refs.numel()
    new = torch.arange(spare + 1, device=DEV, dtype=torch.int32)
    new[torch.where(moves, of, spare)] = torch.where(moves, to, spare).to(torch.int32)
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()], -1))
    count = torch.nn.functional.pad(refs, (0, 1))
    held = count[torch.where(moves, of, spare)]
    count[torch.where(moves, of, spare)] = 0
    count[torch.where(moves, to, spare)] = held
    refs.copy_(count[:spare])
    _copy_pages(s)
    # pages for the next prompts, the lowest free ones in the order of the sequences
    tokens = starts[1:] - starts[:-1]
    need = (tokens + ps - 1) // ps
    b = torch.repeat_interleave(torch.arange(B, device=DEV), need, output_size=total)
    k = torch.arange(total, device=DEV)
    page = _free_page(refs, k).to(torch.int32)
    page = torch.where(page < spare, page, -1)
    table[b, k - (need.cumsum(0) - need)[b]] = page
    _count(s, page, 1)
    got = torch.zeros_like(need).index_add_(0, b, (page >= 0).to(need.dtype))
    s["granted"].copy_(torch.minimum(got * ps, tokens))
    return table, refs, s["src"], s["dst"], s["moved"], s["granted"], *s["pool"]


# ---- the definition in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    c = case
    if c["kind"] == "attend" and work(c)["flops"] > 2e12:
        return None
    s = prepare(c, seed)
    H, D, ps, bs = c["kv_heads"], c["head_dim"], c["page"], c["block"]
    start = s["starts"].tolist()

    def turned(x, weight):
        """Heads [n, heads, D] of all tokens: unit mean square times the weight, pairs of dims as complex numbers times e^(i angle)."""
        where = torch.cat([torch.arange(h, h + t, dtype=torch.float64) for t, h in s["seqs"]]).to(DEV)
        z = x.double()
        z = z / (z.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * (weight.double() + c["offset"])
        half = c["rotary"] // 2
        pairs = z[..., :2 * half].unflatten(-1, (half, 2)) if c["interleaved"] else z[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), where[:, None, None] * s["inv_freq"].double())
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z[..., :2 * half] = pairs.flatten(-2) if c["interleaved"] else pairs.transpose(-1, -2).flatten(-2)
        return z

    if c["kind"] == "rope":
        return turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    if c["kind"] == "rope_append":
        q, k, v = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"]), s["v"].double()
        if c["cache"] == "bf16":
            planes = [torch.zeros(p.shape, dtype=torch.float64, device=DEV) for p in s["pool"]]
            table = s["table"].tolist()
            for plane, x in zip(planes, (k, v)):
                for b, (t, h) in enumerate(s["seqs"]):
                    for p0 in range(h // ps, _ceil(h + t, ps)):  # page by page
                        lo, hi = max(h, p0 * ps), min(h + t, (p0 + 1) * ps)
                        plane[table[b][p0], :, lo - p0 * ps:hi - p0 * ps] = x[start[b] + lo - h:start[b] + hi - h].transpose(0, 1)
            return q, *planes

        def stored(x):
            y = x.to(torch.bfloat16).double().unflatten(-1, (D // 64, 64))
            scale = (y.abs().amax(-1, keepdim=True) / 127).half()
            inverse = torch.where(scale > 0, scale.float().reciprocal(), torch.zeros_like(scale, dtype=torch.float32))
            return (torch.clamp(torch.round(y.float() * inverse), -127, 127).double() * scale.double()).flatten(-2)
        return q, stored(k), stored(v)
    if c["kind"] == "means":
        out = torch.zeros(s["codes"].shape, dtype=torch.float64, device=DEV)
        table = s["table"].tolist()
        for b, (t, h) in enumerate(s["seqs"]):
            for blk in range(h // bs, _ceil(h + t, bs)):
                page, r0 = table[b][blk * bs // ps], blk * bs % ps
                r1 = r0 + min(bs, h + t - blk * bs)
                x = s["pool"][0][page, :, r0:r1].double()
                if c["cache"] == "int8":
                    x = x * s["pool"][2][page, :, r0:r1].double().repeat_interleave(64, -1)
                mean = x.mean(1)
                step = mean.abs().amax(-1, keepdim=True) / 127
                out[page, :, r0 // bs] = torch.round(mean / step).clamp(-127, 127) * step
        return out
    if c["kind"] != "attend":
        return None  # whole numbers and copies
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    group, table = c["q_heads"] // H, s["table"].long()
    picked = s["selected"].long()
    for b, (t, h) in enumerate(s["seqs"]):
        rows = _ceil(h + t, ps) * ps
        for head in range(H):
            key, value = (s["pool"][i][table[b, :rows // ps], head].double().flatten(0, 1) for i in range(2))
            if c["cache"] == "int8":
                key, value = (x * s["pool"][2 + i][table[b, :rows // ps], head].double().flatten(0, 1).repeat_interleave(64, -1)
                              for i, x in enumerate((key, value)))
            for n0 in range(start[b], start[b] + t, 512):
                n1 = min(n0 + 512, start[b] + t)
                seen = torch.zeros((n1 - n0, _ceil(rows, bs) + 1), dtype=torch.bool, device=DEV)
                ids = picked[n0:n1, head]
                seen.scatter_(1, torch.where(ids >= 0, ids, seen.shape[1] - 1), True)
                seen = seen[:, :-1].repeat_interleave(bs, 1)[:, :rows]
                p = torch.arange(h + n0 - start[b], h + n1 - start[b], device=DEV)
                seen = seen & (torch.arange(rows, device=DEV)[None] <= p[:, None])
                q = s["q"][n0:n1, head * group:(head + 1) * group].double().reshape(-1, D)
                logit = (q @ key.t()).view(n1 - n0, group, rows) / D ** 0.5
                logit = torch.where(seen[:, None], logit, torch.full((), -math.inf, device=DEV, dtype=torch.float64))
                weight = torch.exp(logit - torch.logsumexp(logit, -1, keepdim=True))
                out[n0:n1, head * group:(head + 1) * group] = (weight.flatten(0, 1) @ value).view(n1 - n0, group, D)
    return out
