"""Operators over a paged KV cache, as measurable cases.

A serving program with many sequences keeps its keys and values in pages of a pool, one pool per layer,
and a table of pages per sequence. Per layer it appends the rows of the new tokens (quantised to INT8
with a scale per 64 values, or as BF16), attends over the cache (single tokens, chunks of a prompt, both
in one ragged batch; all rows or a sliding window with a few first tokens that stay visible) and, where a
sequence leaves the card or moves to another cache, reads rows back as values.

Layout: a pool plane is [pages, KV heads, page_size, D]; INT8 planes have FP16 scales [pages, KV heads,
page_size, D / 64]; the table is [sequences, pages]. Tokens of all sequences are packed: sequence b has
tokens starts[b] .. starts[b + 1] - 1, and its first one stands at position history[b]. Sizes come from
the package's benchmark and tests (its head geometries) or are generic.
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
# (query heads, KV heads, head_dim) of the package's attention
GEOMETRIES = ((40, 8, 128), (24, 4, 256), (16, 2, 256))


# ---- the cases -------------------------------------------------------------------------------

def _case(**kw):
    c = dict(kind="attention", q_heads=40, kv_heads=8, head_dim=128, cache="int8", page=64, batch=1, tokens=1, tokens_min=0,
             history=0, history_min=0, decodes=0, window=0, sinks=0, out="bf16")
    c.update(kw)
    return c


def listed():
    return [
        # one decode step's rows of 16 conversations, and the same rows read back (what a check of the cache does)
        _case(name="append_step", kind="append", batch=16, tokens=1, history=8192, history_min=100, out="fp32"),
        # several prompts of odd lengths into a BF16 cache at a head_dim-256 geometry
        _case(name="append_bf16", kind="append", q_heads=24, kv_heads=4, head_dim=256, cache="bf16", page=32, batch=5, tokens=901,
              tokens_min=37, history=2000),
        # the largest append: a batch of prompts, written as INT8 and read back as FP32
        _case(name="append_prompts", kind="append", batch=8, tokens=2500, tokens_min=1500, history=4000, out="fp32"),
        # one plain decode step of a short chat: launches and latency
        _case(name="decode_short", page=16, tokens=1, history=517),
        # a decode step of 32 ragged conversations
        _case(name="decode_batch32", batch=32, tokens=1, history=32768, history_min=1024),
        # a verify round of one long document over a BF16 cache at a head_dim-256 geometry
        _case(name="verify_long_bf16", q_heads=24, kv_heads=4, head_dim=256, cache="bf16", page=128, tokens=4, history=131000),
        # a prompt chunk of one conversation next to 16 that decode, in one batch
        _case(name="chunk_mixed", tokens=2048, history=4096, decodes=16),
        # three first prompts of odd lengths at a head_dim-256 geometry over a BF16 cache
        _case(name="prompts_d256", q_heads=24, kv_heads=4, head_dim=256, cache="bf16", page=32, batch=3, tokens=1300, tokens_min=500),
        # a decode step with a sliding window and four sinks, long conversations
        _case(name="window_decode16", batch=16, tokens=1, history=65536, history_min=2000, window=4096, sinks=4),
        # a long prompt under a short window with sinks, BF16 cache
        _case(name="window_prompt", cache="bf16", page=16, tokens=8192, history=1000, window=1024, sinks=4),
        # a short conversation read back as FP32
        _case(name="read_short", kind="read", page=16, tokens=517, out="fp32"),
        # eight conversations leave the card as BF16 rows
        _case(name="read_batch", kind="read", batch=8, tokens=16384, tokens_min=2000),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "read", "decode", "decode", "verify", "chunk", "chunk", "mixed", "window_decode", "window_chunk"))
    hq, hkv, d = rng.choice(GEOMETRIES)
    geo = dict(q_heads=hq, kv_heads=hkv, head_dim=d, cache=rng.choice(("int8", "bf16")), page=rng.choice((16, 32, 64, 128)))
    if kind == "append":
        n = _log_int(rng, 1, 2048)
        return _case(**geo, kind="append", batch=rng.randint(1, 8), tokens=n, tokens_min=max(1, n // 3), history=_log_int(rng, 1, 4000),
                     out="fp32")
    if kind == "read":
        n = _log_int(rng, 1, 12000)
        return _case(**geo, kind="read", batch=rng.randint(1, 8), tokens=n, tokens_min=max(1, n // 4), out=rng.choice(("bf16", "fp32")))
    if kind == "decode":
        top = _log_int(rng, 64, 12000)
        return _case(**geo, batch=_log_int(rng, 1, 32), tokens=1, history=top, history_min=max(1, top // 8))
    if kind == "verify":
        top = _log_int(rng, 256, 45000)
        return _case(**geo, batch=rng.randint(1, 4), tokens=rng.randint(2, 8), history=top, history_min=max(1, top // 2))
    if kind == "chunk":
        n = _log_int(rng, 17, 1024)
        return _case(**geo, batch=rng.randint(1, 2), tokens=n, tokens_min=max(1, n // 3), history=rng.choice((0, _log_int(rng, 1, 3000))))
    if kind == "mixed":
        return _case(**geo, tokens=_log_int(rng, 64, 1500), history=rng.randint(0, 4096), decodes=rng.randint(1, 16))
    window, sinks = _log_int(rng, 32, 2048), rng.choice((0, 1, 4, 16))
    if kind == "window_decode":
        top = _log_int(rng, 512, 60000)
        return _case(**geo, batch=_log_int(rng, 1, 16), tokens=rng.randint(1, 3), history=top, history_min=max(1, top // 8), window=window,
                     sinks=sinks)
    return _case(**geo, tokens=_log_int(rng, 33, 4000), history=rng.randint(0, 4000), window=window, sinks=sinks)


def _sequences(c):
    """(new tokens, rows before them) of every sequence: part of the case, the same for every seed."""
    r = random.Random(c["tokens"] * 7919 + c["history"] * 31 + c["batch"])
    seqs = []
    for _ in range(c["batch"]):
        t = r.randint(c["tokens_min"], c["tokens"]) if c["tokens_min"] else c["tokens"]
        h = r.randint(c["history_min"], c["history"]) if c["history_min"] else c["history"]
        seqs.append((t, h))
    for _ in range(c["decodes"]):  # next to a prompt chunk: conversations with one new token each
        seqs.append((1, r.randint(c["history"] // 8, 2 * c["history"])))
    return seqs


def _visible(c, t, h):
    """(rows that some token of the sequence sees, (token, row) pairs) for t new tokens after h rows."""
    w, s = c["window"] or (1 << 40), c["sinks"]
    lo = max(0, h + 1 - w)
    rows = h + t - lo + min(lo, s)
    pairs = 0
    for p in range(h, h + t):
        first = max(0, p + 1 - w)
        pairs += p + 1 - first + min(first, s)
    return rows, pairs


def work(c):
    H, D, Hq = c["kv_heads"], c["head_dim"], c["q_heads"]
    seqs = _sequences(c)
    n = sum(t for t, _ in seqs)
    row = H * 2 * (D + D // 32) if c["cache"] == "int8" else H * 4 * D  # bytes of K and V of one cache row
    out = 4 if c["out"] == "fp32" else 2
    if c["kind"] == "append":
        back = n * (row + 2 * H * D * out) if c["cache"] == "int8" else 0
        return {"bytes": n * (4 * H * D + row) + back, "flops": 4.0 * n * H * D}
    if c["kind"] == "read":
        return {"bytes": n * (row + 2 * H * D * out), "flops": 2.0 * n * H * D}
    seen = [_visible(c, t, h) for t, h in seqs]
    return {"bytes": sum(s[0] for s in seen) * row + n * Hq * D * 4, "flops": 4.0 * D * Hq * sum(s[1] for s in seen)}


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


def _pool(g, c, pages, fill):
    H, ps, D = c["kv_heads"], c["page"], c["head_dim"]
    q = c["cache"] == "int8"
    planes = [torch.zeros((pages, H, ps, D), device=DEV, dtype=torch.int8 if q else torch.bfloat16) for _ in range(2)]
    if q:
        planes += [torch.zeros((pages, H, ps, D // 64), device=DEV, dtype=torch.float16) for _ in range(2)]
    step = max(1, (1 << 26) // (H * ps * D))
    for i in range(0, pages if fill else 0, step):
        n = min(step, pages - i)
        for plane in range(2):
            x = _rows(g, (n, H, ps, D), 4.0 if plane == 0 else 2.0)
            if q:
                planes[plane][i:i + n], planes[2 + plane][i:i + n] = _quantize(x)
            else:
                planes[plane][i:i + n] = x
    return planes


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    H, D, ps, Hq = c["kv_heads"], c["head_dim"], c["page"], c["q_heads"]
    seqs = _sequences(c)
    n = sum(t for t, _ in seqs)
    need = [(t + h + ps - 1) // ps for t, h in seqs]
    pages = sum(need)
    s = dict(case=c, seqs=seqs, ps=ps)
    s["pool"] = _pool(g, c, pages, c["kind"] != "append")
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)  # a pool in use hands out pages in any order
    table = torch.full((len(seqs), max(need)), -1, device=DEV, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    if c["window"]:  # pages that no token sees any more have been given back
        for b, (t, h) in enumerate(seqs):
            first = max(0, h + 1 - c["window"]) // ps
            kept = (c["sinks"] + ps - 1) // ps
            if kept < first:
                table[b, kept:first] = -1
    s["table"] = table
    starts = [0]
    for t, _ in seqs:
        starts.append(starts[-1] + t)
    s["starts"] = torch.tensor(starts, device=DEV, dtype=torch.int32)
    s["history"] = torch.tensor([h for _, h in seqs], device=DEV, dtype=torch.int32)
    if c["kind"] == "append":
        s["k"], s["v"] = _rows(g, (n, H, D), 4.0), _rows(g, (n, H, D), 2.0)
    elif c["kind"] == "attention":
        s["q"] = torch.randn((n, Hq, D), generator=g, device=DEV).to(torch.bfloat16)
    if own:
        s.update(_handle(s, n))
    torch.cuda.synchronize()
    return s


def _handle(s, n):
    """The views, buffers and workspace that a program keeps for these calls."""
    import ninfer_amd as na
    from ninfer_amd import ops
    from ninfer_amd.device import DeviceBuffer

    kinds = {torch.bfloat16: na.BF16, torch.float32: na.FP32, torch.int32: na.I32, torch.int8: na.I8, torch.float16: na.FP16}

    def view(t):
        return na.Tensor.make(t.data_ptr(), kinds[t.dtype], tuple(reversed(t.shape)))

    c = s["case"]
    cache = na.PagedKVLayerView()
    cache.k, cache.v = view(s["pool"][0]), view(s["pool"][1])
    if c["cache"] == "int8":
        cache.k_scale, cache.v_scale = view(s["pool"][2]), view(s["pool"][3])
    cache.page_table = view(s["table"])
    cache.page_size, cache.num_kv_heads, cache.head_dim = c["page"], c["kv_heads"], c["head_dim"]
    cache.dtype, cache.quant_group = (na.I8, 64) if c["cache"] == "int8" else (na.BF16, 0)
    h = dict(ops=ops, cache=cache, views={k: view(s[k]) for k in ("starts", "history", "q", "k", "v") if k in s})
    kind = torch.float32 if c["out"] == "fp32" else torch.bfloat16
    if c["kind"] == "attention":
        h["out"] = torch.zeros_like(s["q"])
        h["views"]["out"] = view(h["out"])
        h["envelope"] = (max(t for t, _ in s["seqs"]), max(t + r for t, r in s["seqs"]))
        h["window"] = (c["window"], c["sinks"])
        need = ops.paged_attention_workspace_bytes(c["q_heads"], c["kv_heads"], c["head_dim"], n, len(s["seqs"]), h["envelope"], h["window"])
        h["ws"] = DeviceBuffer(max(256, need))
    elif c["kind"] == "read" or c["cache"] == "int8":
        h["back"] = [torch.zeros((n, c["kv_heads"], c["head_dim"]), device=DEV, dtype=kind) for _ in range(2)]
        h["views"]["k_out"], h["views"]["v_out"] = view(h["back"][0]), view(h["back"][1])
    return h


# ---- one pass --------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "attention":
        return _attention(s, c)
    if c["kind"] == "read":
        return _read(s, c)
    _append(s, c)
    return _read(s, c) if c["cache"] == "int8" else tuple(s["pool"])


def _run_own(s, c):
    ops, v = s["ops"], s["views"]
    if c["kind"] == "attention":
        ops.paged_attention(v["q"], v["starts"], v["history"], 1.0 / math.sqrt(c["head_dim"]), s["window"], s["cache"], s["envelope"], s["ws"],
                            v["out"])
        return s["out"]
    if c["kind"] == "append":
        ops.paged_kv_append(v["k"], v["v"], v["starts"], v["history"], s["cache"])
        if c["cache"] != "int8":
            return tuple(s["pool"])
    ops.paged_kv_read(s["cache"], v["starts"], v["history"], v["k_out"], v["v_out"])
    return tuple(s["back"])


# The plain form: torch operations in 32 bits.

def _places(s):
    """(page, row of the page) of every packed token."""
    token = torch.arange(sum(t for t, _ in s["seqs"]), device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["starts"], token, right=True) - 1
    pos = s["history"][b] + token - s["starts"][b]
    return s["table"][b, pos // s["ps"]].long(), pos % s["ps"]


def _append(s, c):
    page, row = _places(s)
    for plane, x in enumerate((s["k"], s["v"])):
        if c["cache"] == "int8":
            codes, scales = _quantize(x)
            s["pool"][plane][page, :, row] = codes
            s["pool"][2 + plane][page, :, row] = scales
        else:
            s["pool"][plane][page, :, row] = x


def _values(s, plane, page, row):
    """Cache rows [n, KV heads, D] in 32 bits."""
    x = s["pool"][plane][page, :, row].float()
    if len(s["pool"]) == 4:
        x = (x.unflatten(-1, (-1, 64)) * s["pool"][2 + plane][page, :, row].float()[..., None]).flatten(-2)
    return x


def _read(s, c):
    page, row = _places(s)
    kind = torch.float32 if c["out"] == "fp32" else torch.bfloat16
    return tuple(_values(s, plane, page, row).to(kind) for plane in range(2))


def _attention(s, c):
    H, D, Hq = c["kv_heads"], c["head_dim"], c["q_heads"]
    G, W, S = Hq // H, c["window"] or (1 << 30), c["sinks"]
    out = torch.empty_like(s["q"])
    at = 0
    for b, (tokens, h) in enumerate(s["seqs"]):
        for t0 in range(0, tokens, 1024):  # a prompt's scores a part at a time, so that they fit the memory
            t = min(1024, tokens - t0)
            pos = torch.arange(h + t0, h + t0 + t, device=DEV)
            lo = max(0, h + t0 + 1 - W)
            rows = torch.arange(lo, h + t0 + t, device=DEV)
            if lo > 0 and S > 0:
                rows = torch.cat((torch.arange(0, min(lo, S), device=DEV), rows))
            page = s["table"][b, rows // s["ps"]].long()
            k = _values(s, 0, page, rows % s["ps"]).transpose(0, 1).contiguous()  # [H, rows, D]
            v = _values(s, 1, page, rows % s["ps"]).transpose(0, 1).contiguous()
            q = s["q"][at + t0:at + t0 + t].float().view(t, H, G, D).permute(1, 0, 2, 3).reshape(H, t * G, D)
            score = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(1.0 / math.sqrt(D)).view(H, t, G, -1)
            hidden = (rows[None] > pos[:, None]) | ((pos[:, None] - rows[None] >= W) & (rows[None] >= S))
            score.masked_fill_(hidden[None, :, None], -math.inf)
            score = score.sub_(score.amax(-1, keepdim=True)).exp_()
            total = score.sum(-1, keepdim=True)
            o = torch.bmm(score.view(H, t * G, -1), v).view(H, t, G, D) / total
            out[at + t0:at + t0 + t] = o.permute(1, 0, 2, 3).reshape(t, Hq, D).to(torch.bfloat16)
        at += tokens
    return out


# ---- the definition in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    c = case
    if c["kind"] == "attention" and work(c)["flops"] > 2e12:
        return None
    s = prepare(c, seed)
    H, D, ps = c["kv_heads"], c["head_dim"], c["page"]
    table, pool = s["table"].cpu().tolist(), s["pool"]

    def stored(x):
        """What the cache holds of new rows x [n, H, D], in 64 bits."""
        if c["cache"] == "bf16":
            return x.double()
        y = x.double().view(*x.shape[:-1], D // 64, 64)
        scale = (y.abs().amax(-1, keepdim=True) / 127).half()
        inverse = torch.where(scale > 0, scale.float().reciprocal(), torch.zeros_like(scale, dtype=torch.float32))
        code = torch.clamp(torch.round((y.float() * inverse)), -127, 127)
        return (code.double() * scale.double()).view(x.shape)

    if c["kind"] == "append" and c["cache"] == "int8":
        return stored(s["k"]), stored(s["v"])
    if c["kind"] == "append":
        planes = [torch.zeros(p.shape, dtype=torch.float64, device=DEV) for p in pool]
        for plane, x in zip(planes, (s["k"], s["v"])):
            n = 0
            for b, (t, h) in enumerate(s["seqs"]):
                for p0 in range(h // ps, (h + t + ps - 1) // ps):  # page by page
                    lo, hi = max(h, p0 * ps), min(h + t, (p0 + 1) * ps)
                    plane[table[b][p0], :, lo - p0 * ps:hi - p0 * ps] = x[n + lo - h:n + hi - h].double().transpose(0, 1)
                n += t
        return tuple(planes)

    def history_of(b, plane, lo, hi):
        """Rows lo .. hi - 1 of sequence b, [H, hi - lo, D] in 64 bits, taken by whole pages."""
        ids = torch.tensor(table[b][lo // ps:(hi + ps - 1) // ps], device=DEV, dtype=torch.int64)
        x = pool[plane].index_select(0, ids).double()
        if c["cache"] == "int8":
            x *= pool[2 + plane].index_select(0, ids).double().repeat_interleave(64, -1)
        return x.movedim(1, 0).flatten(1, 2)[:, lo % ps:lo % ps + hi - lo]

    if c["kind"] == "read":
        return tuple(torch.cat([history_of(b, plane, h, h + t).movedim(0, 1) for b, (t, h) in enumerate(s["seqs"])]) for plane in range(2))

    parts = []
    group = c["q_heads"] // H
    n = 0
    for b, (tokens, h) in enumerate(s["seqs"]):
        for first in range(0, tokens, 256):
            last = min(tokens, first + 256)
            p = torch.arange(h + first, h + last, device=DEV)
            begin = max(0, h + first - c["window"] + 1) if c["window"] else 0
            spans = [(0, h + last)] if begin <= c["sinks"] else [x for x in ((0, c["sinks"]), (begin, h + last)) if x[1] > x[0]]
            place = torch.cat([torch.arange(x, y, device=DEV) for x, y in spans])
            seen = place[None] <= p[:, None]
            if c["window"]:
                seen &= (place[None] > p[:, None] - c["window"]) | (place[None] < c["sinks"])
            for head in range(H):
                key = torch.cat([history_of(b, 0, x, y)[head] for x, y in spans])
                value = torch.cat([history_of(b, 1, x, y)[head] for x, y in spans])
                q = s["q"][n + first:n + last, head * group:(head + 1) * group].double()  # [t, group, D]
                logit = (q.reshape(-1, D) @ key.t().contiguous()).view(last - first, group, -1) / D ** 0.5
                logit = torch.where(seen[:, None], logit, torch.full((), -math.inf, device=DEV, dtype=torch.float64))
                weight = torch.exp(logit - torch.logsumexp(logit, -1, keepdim=True))
                parts.append((n + first, head, (weight.view(-1, weight.shape[-1]) @ value).view(last - first, group, D)))
        n += tokens
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for at, head, o in parts:
        out[at:at + o.shape[0], head * group:(head + 1) * group] = o
    return out
