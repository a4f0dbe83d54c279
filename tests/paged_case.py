"""A paged-cache problem in numpy, its 64-bit results, and its run on the GPU."""
from __future__ import annotations

import numpy as np

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.device import DeviceArray, DeviceBuffer, synchronize


def bf16_bits(x):
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)


def bf16_values(bits):
    return (np.asarray(bits, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def quantize(bits):
    """INT8-G64 codes and FP16 scale bits of BF16 rows [..., D]."""
    x = bf16_values(bits).reshape(*bits.shape[:-1], -1, 64)
    s = (np.abs(x).max(-1) / np.float32(127)).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(s > 0, np.float32(1) / s.astype(np.float32), np.float32(0)).astype(np.float32)
        codes = np.clip(np.rint(x * inv[..., None]), -127, 127).astype(np.int8)
    return codes.reshape(bits.shape), s.view(np.uint16)


class PagedCase:
    """seqs: (new tokens, rows before them) per sequence. Pages are handed out in random order; rows that hold
    nothing are poison (INT8: NaN scales, BF16: NaN and infinities). `absent`: {(sequence, page of it)}; `lead` and
    `tail`: packed tokens before the first and after the last sequence; `pad`: bytes between tokens; `page_pad`: bytes
    between pages; `kgain`/`vgain`: (size of one dimension in 32)."""

    def __init__(self, seqs, Hq=40, Hkv=8, D=128, kv="i8", page=16, window=0, sinks=0, seed=0, absent=(), lead=0, tail=0, pad=0, page_pad=0,
                 spare=2, max_pages=None, scale=None, kgain=4.0, vgain=2.0, edit=None):
        self.seqs, self.Hq, self.Hkv, self.D, self.kv, self.page = list(seqs), Hq, Hkv, D, kv, page
        self.window, self.sinks, self.absent = window, sinks, set(absent)
        self.pad, self.page_pad = pad, page_pad
        self.scale = float(np.float32(scale if scale is not None else 1.0 / np.sqrt(D)))
        r = np.random.default_rng(seed)
        B = len(self.seqs)
        self.B = B
        need = [-(-(t + h) // page) for t, h in self.seqs]
        self.max_pages = max_pages or max(1, max(need))
        self.pages = sum(min(n, self.max_pages) for n in need) + spare
        order = r.permutation(self.pages)
        self.table = np.full((B, self.max_pages), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            n = min(n, self.max_pages)
            self.table[b, :n] = order[at:at + n]
            at += n
        for b, s in self.absent:
            self.table[b, s] = (-1, self.pages, 1 << 30)[(b + s) % 3]
        self.starts = np.cumsum([lead] + [t for t, _ in self.seqs]).astype(np.int32)
        self.history = np.array([h for _, h in self.seqs], np.int32)
        self.N = int(self.starts[-1]) + tail

        def rows(n, gain):
            x = r.standard_normal((n, Hkv, D), dtype=np.float32)
            x[..., ::32] *= gain
            return bf16_bits(x)

        # every row of every sequence, old and new
        self.k = [rows(t + h, kgain) for t, h in self.seqs]
        self.v = [rows(t + h, vgain) for t, h in self.seqs]
        self.q = bf16_bits(r.standard_normal((self.N, Hq, D), dtype=np.float32))
        self.k_new = rows(self.N, kgain)
        self.v_new = rows(self.N, vgain)
        if edit is not None:
            edit(self)
        for b, (t, h) in enumerate(self.seqs):
            n = self.starts[b]
            self.k_new[n:n + t] = self.k[b][h:]
            self.v_new[n:n + t] = self.v[b][h:]

    # ---- planes [page][h][row][d]
    def planes(self, new_rows=True):
        """The pool with the history (and the new rows) in place; everything else is poison."""
        shape = (self.pages, self.Hkv, self.page)
        if self.kv == "i8":
            out = [np.full((*shape, self.D), 77, np.int8) for _ in range(2)] + [np.full((*shape, self.D // 64), 0x7E00, np.uint16) for _ in range(2)]
        else:
            out = [np.full((*shape, self.D), p, np.uint16) for p in (0x7FC0, 0x7F80)]
        for b, (t, h) in enumerate(self.seqs):
            self.store(out, b, 0, h + (t if new_rows else 0))
        return out

    def store(self, planes, b, r0, r1):
        for plane, x in enumerate((self.k[b], self.v[b])):
            for s in range(r0 // self.page, -(-r1 // self.page)):
                if s >= self.max_pages or not 0 <= self.table[b, s] < self.pages:
                    continue
                lo, hi = max(r0, s * self.page), min(r1, (s + 1) * self.page)
                at = (self.table[b, s], slice(None), slice(lo - s * self.page, hi - s * self.page))
                y = x[lo:hi].transpose(1, 0, 2)
                if self.kv == "i8":
                    planes[plane][at], planes[2 + plane][at] = quantize(y)
                else:
                    planes[plane][at] = y

    def stored(self, b):
        """What the cache holds of sequence b's rows: 64-bit K and V [rows, Hkv, D]."""
        out = []
        for x in (self.k[b], self.v[b]):
            if self.kv == "i8":
                c, s = quantize(x)
                y = c.reshape(*c.shape[:-1], -1, 64).astype(np.float64) * s.view(np.float16).astype(np.float64)[..., None]
                out.append(y.reshape(c.shape))
            else:
                out.append(bf16_values(x).astype(np.float64))
        return out

    def present(self, b, rows):
        s = rows // self.page
        ok = s < self.max_pages
        e = self.table[b, np.minimum(s, self.max_pages - 1)]
        return ok & (e >= 0) & (e < self.pages)

    def oracle(self, only=None):
        """64-bit outputs [N, Hq, D] (NaN where no sequence has the token) and the largest errors that the operand
        roundings allow: FP16 operands and probabilities are off by at most 2^-11 of their value, so a score by 2^-11 of
        sum |q k| scale and, with the probabilities' and the values' own roundings, the output by
        (2 exp-error + 2^-10) sum p |v|; sums in 32 bits add 2^-20 of that, the BF16 result 2^-8 of itself."""
        out = np.full((self.N, self.Hq, self.D), np.nan)
        tol = np.zeros_like(out)
        G = self.Hq // self.Hkv
        for b, (t, h) in enumerate(self.seqs):
            if t == 0 or (only is not None and b not in only):
                continue
            K, V = self.stored(b)
            rows = np.arange(t + h)
            here = self.present(b, rows)
            n0 = int(self.starts[b])
            q = bf16_values(self.q[n0:n0 + t]).astype(np.float64).reshape(t, self.Hkv, G, self.D)
            for i0 in range(0, t, 64):
                i1 = min(t, i0 + 64)
                pos = h + np.arange(i0, i1)
                see = (rows[None] <= pos[:, None]) & here[None]
                if self.window:
                    see &= (pos[:, None] - rows[None] < self.window) | (rows[None] < self.sinks)
                used = np.flatnonzero(see.any(0))
                m = see[:, used]
                for hh in range(self.Hkv):
                    qq = q[i0:i1, hh]
                    k, v = K[used, hh], V[used, hh]
                    with np.errstate(invalid="ignore", over="ignore"):
                        sc = np.where(m[:, None], (qq @ k.T) * self.scale, -np.inf)
                        size = np.where(m[:, None], (np.abs(qq) @ np.abs(k).T) * self.scale, 0.0)
                        top = sc.max(-1, initial=-np.inf, keepdims=True)
                        p = np.where(m[:, None], np.exp(sc - np.where(np.isfinite(top), top, 0.0)), 0.0)
                        L = p.sum(-1, keepdims=True)
                        p = np.where(L > 0, p / np.where(L > 0, L, 1.0), 0.0)
                        o = p @ np.where(np.isfinite(v), v, 0.0)
                        for j in np.flatnonzero(~np.isfinite(v).all(-1)):  # only to the rows that see it
                            o += np.where(m[:, None, j, None] & ~np.isfinite(v[j]), v[j], 0.0)
                        A = p @ np.where(np.isfinite(v), np.abs(v), 0.0)
                        d = size.max(-1, initial=0.0, keepdims=True) * 2.0**-11
                        # a score error of d changes a probability by a factor of exp(2 d) at most; past 2 d = 50 that bounds nothing
                        # (a p of 1e-320 is 0 in `A` and may be 1), but any two weighted means of v lie within 2 max |v|
                        loose = 2.0 * np.where(m[:, :, None], np.where(np.isfinite(v), np.abs(v), 0.0)[None], 0.0).max(1, initial=0.0)[:, None]
                        e = np.where(2 * d > 50, loose, A * (2 * np.expm1(np.minimum(2 * d, 50.0)) + 2.0**-10 + 2.0**-20))
                        # FP16 holds p * 2^8 down to steps of 2^-24: every key's p is off by 2^-33 at least, and its V scale's share
                        # of the largest one by as much
                        floor = 2.0**-32 * m.sum(-1)[:, None, None] * np.where(np.isfinite(v), np.abs(v), 0.0).max(initial=0.0)
                        tol[n0 + i0:n0 + i1, hh * G:(hh + 1) * G] = 2.0**-8 * np.abs(o) + e + floor + 1e-30
                    out[n0 + i0:n0 + i1, hh * G:(hh + 1) * G] = o
        return out, tol

    # ---- the GPU
    def envelope(self):
        return (max(1, max(t for t, _ in self.seqs)), max(1, max(t + h for t, h in self.seqs)))

    def upload(self, planes=None):
        return Device(self, planes if planes is not None else self.planes())


class Strided:
    """Rows [n, bytes] in a buffer of their own with `pad` bytes after each, and the tensor over them."""

    def __init__(self, dtype, shape, pad, fill=0xCD):
        self.n, self.row = shape[-1], int(np.prod(shape[:-1])) * na._capi.DTYPE_SIZE[dtype]
        self.stride = self.row + pad
        self.buf = DeviceBuffer(self.n * self.stride)
        self.buf.fill(fill)
        self.t = na.Tensor.make(self.buf.ptr, dtype, shape)
        self.axis = len(shape) - 1
        self.t.nb[self.axis] = self.stride

    def upload(self, x):
        host = self.buf.download(np.uint8, self.n * self.stride).reshape(self.n, self.stride)
        host[:, :self.row] = np.ascontiguousarray(x).view(np.uint8).reshape(self.n, self.row)
        self.buf.upload(host)
        return self

    def numpy(self, dtype):
        host = self.buf.download(np.uint8, self.n * self.stride).reshape(self.n, self.stride)
        assert (host[:, self.row:] == 0xCD).all(), "bytes between rows were written"
        return np.ascontiguousarray(host[:, :self.row]).view(dtype)


class Device:
    """The case's tensors on the GPU."""

    def __init__(self, c: PagedCase, planes):
        self.c = c
        D, H = c.D, c.Hkv
        i8 = c.kv == "i8"
        kinds = [na.I8, na.I8, na.FP16, na.FP16] if i8 else [na.BF16, na.BF16]
        self.planes = [Strided(kd, (x.shape[-1], c.page, H, c.pages), c.page_pad).upload(x) for kd, x in zip(kinds, planes)]
        self.table = Strided(na.I32, (c.max_pages, c.B), 8).upload(c.table)
        self.table.t.ne[2] = self.table.t.ne[3] = 1
        self.starts = DeviceArray.from_numpy(na.I32, c.starts)
        self.history = DeviceArray.from_numpy(na.I32, c.history)
        self.q = Strided(na.BF16, (D, c.Hq, c.N), c.pad).upload(c.q)
        self.k = Strided(na.BF16, (D, H, c.N), c.pad).upload(c.k_new)
        self.v = Strided(na.BF16, (D, H, c.N), c.pad).upload(c.v_new)
        self.out = Strided(na.BF16, (D, c.Hq, c.N), c.pad)
        v = na.PagedKVLayerView()
        v.k, v.v = self.planes[0].t, self.planes[1].t
        if i8:
            v.k_scale, v.v_scale = self.planes[2].t, self.planes[3].t
        v.page_table = self.table.t
        v.page_size, v.num_kv_heads, v.head_dim, v.dtype, v.quant_group = c.page, H, D, na.I8 if i8 else na.BF16, 64 if i8 else 0
        self.view = v

    def workspace(self, envelope=None):
        c = self.c
        need = ops.paged_attention_workspace_bytes(c.Hq, c.Hkv, c.D, c.N, c.B, envelope or c.envelope(), (c.window, c.sinks))
        ws = DeviceBuffer(max(256, need))
        ws.fill(0xFF)  # NaN bit patterns: nothing may depend on what scratch held before
        return ws

    def append(self, stream=None):
        ops.paged_kv_append(self.k.t, self.v.t, self.starts.tensor(), self.history.tensor(), self.view, stream)

    def attend(self, envelope=None, ws=None, stream=None):
        c = self.c
        self.ws = ws or self.workspace(envelope)
        ops.paged_attention(self.q.t, self.starts.tensor(), self.history.tensor(), c.scale, (c.window, c.sinks), self.view,
                            envelope or c.envelope(), self.ws, self.out.t, stream)

    def read(self, first, dtype=na.FP32, stream=None):
        c = self.c
        outs = [Strided(dtype, (c.D, c.Hkv, c.N), c.pad) for _ in range(2)]
        f = DeviceArray.from_numpy(na.I32, np.asarray(first, np.int32))
        ops.paged_kv_read(self.view, self.starts.tensor(), f.tensor(), outs[0].t, outs[1].t, stream)
        synchronize()
        return [o.numpy(np.float32 if dtype == na.FP32 else np.uint16).reshape(c.N, c.Hkv, c.D) for o in outs]

    def pool(self):
        c = self.c
        G = c.D // 64
        if c.kv == "i8":
            return [p.numpy(t).reshape(c.pages, c.Hkv, c.page, n) for p, t, n in zip(self.planes, (np.int8, np.int8, np.uint16, np.uint16), (c.D, c.D, G, G))]
        return [p.numpy(np.uint16).reshape(c.pages, c.Hkv, c.page, c.D) for p in self.planes]

    def result(self):
        synchronize()
        return self.out.numpy(np.uint16).reshape(self.c.N, self.c.Hq, self.c.D)


def check_attention(case, bits, only=None):
    """Every served token within its tolerance, every other one untouched."""
    ref, tol = case.oracle(only)
    served = ~np.isnan(ref).all((1, 2))
    for b, (t, _) in enumerate(case.seqs):  # a served row may be NaN by its values
        if only is None or b in only:
            served[case.starts[b]:case.starts[b] + t] = True
    assert (bits[~served] == 0xCDCD).all(), "rows of no sequence were written"
    got = bf16_values(bits[served]).astype(np.float64)
    ref, tol = ref[served], tol[served]
    fine = np.isfinite(ref)
    same = np.where(np.isnan(ref), np.isnan(got), got == ref)
    assert same[~fine].all(), "infinite and NaN results differ"
    err = np.abs(got - ref)[fine]
    bad = ~(err <= tol[fine])
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, worst {np.nanmax(err / tol[fine]):.3g} of its tolerance, finite {np.isfinite(got[fine]).all()}"
    return float((err / tol[fine]).max()) if err.size else 0.0
