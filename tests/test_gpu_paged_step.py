"""The operators around a paged cache as a serving program calls them: prompts, answers that share them, decode steps over selected blocks,
pages that come and go, in two layers that share a table."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.device import DeviceArray, DeviceBuffer, synchronize
from ninfer_amd.kv_cache import PagedKVCacheLayer
from paged_case import bf16_bits, bf16_values

pytestmark = pytest.mark.gpu


HELD = []  # the arrays of a test: a view alone does not keep its memory


def dev(x):
    HELD.append(DeviceArray.from_numpy(na.I32, np.asarray(x, np.int32)))
    return HELD[-1]


@pytest.fixture(autouse=True)
def release_arrays():
    yield
    synchronize()
    HELD.clear()


class Program:
    Hq, Hkv, D, page, block, B, width, pages = 8, 2, 128, 64, 32, 6, 12, 40
    pick = (1, 2, 3)

    def __init__(self, kv):
        self.r = np.random.default_rng(1)
        kind = na.I8 if kv == "i8" else na.BF16
        first = PagedKVCacheLayer(self.pages, self.page, self.Hkv, self.D, self.B, self.width, kind, self.block)
        self.layers = [first, PagedKVCacheLayer(self.pages, self.page, self.Hkv, self.D, self.B, self.width, kind, self.block, table_of=first)]
        self.table, self.refs = first.page_table.tensor(), first.refs.tensor()
        self.history = np.zeros(self.B, np.int32)
        self.d_history = dev(self.history)
        self.rows = [[np.zeros((0, 2, self.Hkv, self.D), np.float32) for _ in range(self.B)] for _ in self.layers]  # rotated K and V as they were given
        w = self.r.standard_normal((2, self.D)).astype(np.float32)
        self.w = [DeviceArray.from_numpy(na.FP32, x) for x in w]
        self.freq = DeviceArray.from_numpy(na.FP32, (1e4 ** (-np.arange(32) / 32)).astype(np.float32))

    def step(self, tokens):
        """The sequences' next tokens through both layers; returns every layer's (sparse, dense where the lists hold all) output."""
        tokens = np.asarray(tokens)
        starts = np.concatenate(([0], np.cumsum(tokens))).astype(np.int32)
        n = int(starts[-1])
        d_starts, granted = dev(starts), dev([0] * self.B)
        ops.paged_pages_reserve(self.table, self.refs, d_starts.tensor(), self.d_history.tensor(), self.page, granted.tensor())
        assert (granted.numpy() == tokens).all()
        env = (int(tokens.max()), int((self.history + tokens).max()))
        outs = []
        for i, c in enumerate(self.layers):
            qkv = bf16_bits(self.r.standard_normal((n, self.Hq + 2 * self.Hkv, self.D), dtype=np.float32))
            fused = DeviceArray.from_numpy(na.BF16, qkv)
            part = lambda lo, heads: self.slice(fused, lo, heads, n)  # noqa: E731
            q, k, v = part(0, self.Hq), part(self.Hq, self.Hkv), part(self.Hq + self.Hkv, self.Hkv)
            args = (self.w[0].tensor(), self.w[1].tensor())
            norm = (1e-6, 0.0, False)
            ops.paged_qk_norm_rope_append(q, k, v, *args, d_starts.tensor(), self.d_history.tensor(), self.freq.tensor(), norm, c.view(), q)
            ops.paged_block_update(c.view(), d_starts.tensor(), self.d_history.tensor(), n, c.blocks())
            S = sum(self.pick)
            lists = dev(np.full((n, self.Hkv, S), -1))
            need = ops.paged_block_select_workspace_bytes(self.Hkv, self.D, n, self.B, env, self.block)
            ws = DeviceBuffer(max(256, need))
            ops.paged_block_select(q, d_starts.tensor(), self.d_history.tensor(), self.table, self.page, c.blocks(), self.pick, env, ws, lists.tensor())
            need = ops.paged_sparse_attention_workspace_bytes(self.Hq, self.Hkv, self.D, n, self.B, S, self.block)
            ws2, out = DeviceBuffer(max(256, need)), DeviceArray(na.BF16, (self.D, self.Hq, n))
            ops.paged_sparse_attention(q, d_starts.tensor(), self.d_history.tensor(), 0.1, lists.tensor(), self.block, c.view(), env, ws2, out.tensor())
            synchronize()
            whole = fused.numpy().reshape(n, -1, self.D)
            outs.append((whole[:, :self.Hq], lists.numpy().reshape(n, self.Hkv, S), out.numpy().reshape(n, self.Hq, self.D)))
        self.check(outs, starts)
        self.history = self.history + tokens.astype(np.int32)
        self.d_history.upload(self.history)
        return outs

    def slice(self, fused, lo, heads, n):
        t = na.Tensor.make(fused.ptr + lo * self.D * 2, na.BF16, (self.D, heads, n))
        t.nb[2] = (self.Hq + 2 * self.Hkv) * self.D * 2
        return t

    def values(self, c, b, rows):
        """Rows of sequence b read back as FP32 K and V [rows, Hkv, D]."""
        starts = np.zeros(self.B + 1, np.int32)
        starts[b + 1:] = rows
        outs = [DeviceArray(na.FP32, (self.D, self.Hkv, rows)) for _ in range(2)]
        ops.paged_kv_read(c.view(), dev(starts).tensor(), dev([0] * self.B).tensor(), outs[0].tensor(), outs[1].tensor())
        return [o.numpy().reshape(rows, self.Hkv, self.D).astype(np.float64) for o in outs]

    def check(self, outs, starts):
        """Every output against its lists and the cache's rows: FP16 operands of INT8 rows and FP16 probabilities move a score by 2^-11 of its
        terms and a weight by 2^-11, the result is rounded to BF16."""
        G = self.Hq // self.Hkv
        for c, (q, lists, out) in zip(self.layers, outs):
            for b in range(self.B):
                for n in range(starts[b], starts[b + 1]):
                    if n not in (starts[b], starts[b + 1] - 1):
                        continue
                    pos = int(self.history[b]) + n - int(starts[b])
                    K, V = self.values(c, b, pos + 1)
                    for h in range(self.Hkv):
                        own = pos // self.block
                        listed = lists[n, h][lists[n, h] >= 0]
                        assert len(listed) == min(own + 1, sum(self.pick)) and own in listed and 0 in listed
                        rows = np.flatnonzero(np.isin(np.arange(pos + 1) // self.block, listed))
                        x = bf16_values(q[n, h * G:(h + 1) * G]).astype(np.float64)
                        s = x @ K[rows, h].T * np.float64(np.float32(0.1))
                        d = 2.0**-10 * (np.abs(x) @ np.abs(K[rows, h]).T * 0.1).max(-1, keepdims=True) + 2.0**-9
                        p = np.exp(s - s.max(-1, keepdims=True))
                        p /= p.sum(-1, keepdims=True)
                        o = p @ V[rows, h]
                        tol = 2.0**-8 * np.abs(o) + np.expm1(2 * d) * (p @ np.abs(V[rows, h])) + 2.0**-20
                        assert (np.abs(bf16_values(out[n, h * G:(h + 1) * G]) - o) <= tol).all()

    def fork(self, parents, children):
        src, dst = dev([0] * len(parents)), dev([0] * len(parents))
        ops.paged_pages_fork(self.table, self.refs, dev(parents).tensor(), dev(children).tensor(), self.d_history.tensor(), self.page, src.tensor(), dst.tensor())
        self.move(src, dst)
        self.history = self.d_history.numpy()

    def move(self, src, dst):
        for c in self.layers:
            ops.paged_kv_copy_pages(c.view(), c.blocks(), src.tensor(), dst.tensor())

    def end(self, sequences):
        ops.paged_pages_release(self.table, self.refs, dev(sequences).tensor(), dev([0] * len(sequences)).tensor(), self.page)
        src, dst, moved = dev([0] * 20), dev([0] * 20), dev([0])
        ops.paged_pages_compact(self.table, self.refs, src.tensor(), dst.tensor(), moved.tensor())
        self.move(src, dst)
        self.history[sequences] = 0
        self.d_history.upload(self.history)
        return int(moved.numpy()[0])


@pytest.mark.parametrize("kv", ["i8", "bf16"])
def test_a_program(gpu, kv):
    p = Program(kv)
    p.step([150, 70, 0, 0, 0, 33])  # prompts
    before = [p.values(c, 0, 150) for c in p.layers]
    p.fork([0, 0, 1], [2, 3, 4])    # answers
    assert list(p.history) == [150, 70, 150, 150, 70, 33]
    for c, x in zip(p.layers, before):
        for b in (2, 3):
            assert all((a == y).all() for a, y in zip(p.values(c, b, 150), x))
    for _ in range(3):
        p.step([1, 1, 1, 1, 1, 1])
    kept = [p.values(c, 3, 153) for c in p.layers]
    assert p.end([0, 4, 5]) > 0     # pages move; the answers keep what they share
    for c, x in zip(p.layers, kept):
        assert all((a == y).all() for a, y in zip(p.values(c, 3, 153), x))
    p.step([200, 1, 2, 1, 0, 90])   # new prompts next to decode steps
    p.step([1, 1, 1, 1, 0, 1])
    held = p.layers[0].page_table.numpy()
    assert (np.bincount(held[held >= 0], minlength=p.pages) == p.layers[0].refs.numpy()).all()
