"""Head norms with rotation against a plain 64-bit form, every element within a derived tolerance; the form that appends against the two
calls that it stands for, bit by bit."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.device import DeviceArray, Graph, Stream, synchronize
from paged_blocks_case import norm_rope
from paged_case import PagedCase, Strided, bf16_bits, bf16_values

pytestmark = pytest.mark.gpu

GEO = {"40-8-128": (40, 8, 128), "24-4-256": (24, 4, 256), "16-2-256": (16, 2, 256), "1-1-128": (1, 1, 128), "5-5-256": (5, 5, 256)}


def _freq(half, base=1e4):
    return (base ** (-np.arange(half) / max(half, 1))).astype(np.float32)


class RopeCase:
    """q and k of n tokens as slices of a fused projection (`pad` bytes between tokens)."""

    def __init__(self, n, Hq, Hkv, D, half, positions, weight="bf16", offset=0.0, interleaved=False, eps=1e-6, pad=64, seed=0, edit=None):
        r = np.random.default_rng(seed)
        self.n, self.Hq, self.Hkv, self.D, self.half = n, Hq, Hkv, D, half
        self.positions = np.asarray(positions, np.int32)
        self.q, self.k = (bf16_bits(r.standard_normal((n, h, D), dtype=np.float32) * np.float32(3)) for h in (Hq, Hkv))
        if edit is not None:
            edit(self)
        self.norm = (eps, offset, interleaved)
        self.freq = _freq(half) if half else None
        self.weights = [None, None]
        if weight is not None:
            self.weights = [(1 - offset + 0.3 * r.standard_normal(D)).astype(np.float32) for _ in range(2)]
        if weight == "bf16":
            self.weights = [bf16_values(bf16_bits(w)) for w in self.weights]
        self.d_weights = [None if w is None else DeviceArray.from_numpy(na.FP32, w) if weight == "fp32" else DeviceArray.from_numpy(na.BF16, bf16_bits(w))
                          for w in self.weights]
        self.d_freq = DeviceArray.from_numpy(na.FP32, self.freq) if half else None
        self.d_q, self.d_k = (Strided(na.BF16, (D, x.shape[1], n), pad).upload(x) for x in (self.q, self.k))
        self.d_pos = DeviceArray.from_numpy(na.I32, self.positions)
        self.outs = [Strided(na.BF16, (D, h, n), pad) for h in (Hq, Hkv)]

    def args(self):
        w = [None if x is None else x.tensor() for x in self.d_weights]
        return w[0], w[1], self.d_pos.tensor(), None if self.d_freq is None else self.d_freq.tensor(), self.norm

    def call(self, outs=None, stream=None):
        outs = outs or self.outs
        ops.qk_norm_rope(self.d_q.t, self.d_k.t, *self.args(), outs[0].t, outs[1].t, stream)

    def check(self, outs=None):
        synchronize()
        for x, w, o in zip((self.q, self.k), self.weights, outs or self.outs):
            ref, tol = norm_rope(x, w, self.positions, self.freq, *self.norm)
            got = bf16_values(o.numpy(np.uint16).reshape(x.shape)).astype(np.float64)
            err = np.abs(got - ref)
            bad = ~(err <= tol)
            assert not bad.any(), f"{bad.sum()} of {bad.size} outside, worst {np.nanmax(err / tol):.3g} of the tolerance"


@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("n", [1, 2, 17, 130])
@pytest.mark.parametrize("part", [1.0, 0.5, 0.125])
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(gpu, geo, n, part, interleaved):
    Hq, Hkv, D = GEO[geo]
    c = RopeCase(n, Hq, Hkv, D, int(D * part) // 2, np.arange(n) * 7 + 3, interleaved=interleaved, seed=n)
    c.call()
    c.check()


@pytest.mark.parametrize("weight", [None, "bf16", "fp32"])
@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("half", [0, 8, 24, 40, 64])
def test_weights_and_odd_rotations(gpu, weight, offset, half):
    """Halves that are no power of two, no rotation, no weight."""
    c = RopeCase(9, 6, 2, 128, half, np.arange(9) * 1000, weight=weight, offset=offset, seed=half)
    c.call()
    c.check()


@pytest.mark.parametrize("position", [0, -5, (1 << 23) - 1, 2**31 - 1, -(2**31)])
def test_far_positions(gpu, position):
    c = RopeCase(3, 4, 2, 256, 128, [position, max(position - 1, -(2**31)), position // 2], seed=1)
    c.call()
    c.check()


@pytest.mark.parametrize("value", [0.0, 1e-30, 1e-41, 1e15, 1e20, 3e38])
@pytest.mark.parametrize("eps", [2.0**-60, 1e-6, 1.0])
def test_size_of_the_values(gpu, value, eps):
    """Rows of zeros, of tiny values next to eps, of values whose squares FP32 does not hold; ordinary rows beside them."""
    def edit(c):
        c.q[1, 2] = bf16_bits(bf16_values(c.q[1, 2]) * np.float32(value / 8))
        c.k[0, 1] = bf16_bits(np.full(c.D, value, np.float32))
    c = RopeCase(2, 5, 2, 128, 32, [5, 6], eps=eps, edit=edit, seed=2)
    c.call()
    c.check()


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_infinite_and_nan_values_stay_in_their_head(gpu, value):
    def edit(c):
        c.q[1, 2, 40] = bf16_bits(np.full(1, value, np.float32))[0]
    c, d = RopeCase(2, 5, 2, 128, 32, [5, 6], edit=edit, seed=3), RopeCase(2, 5, 2, 128, 32, [5, 6], seed=3)
    c.call()
    d.call()
    synchronize()
    got, ref = (bf16_values(x.outs[0].numpy(np.uint16).reshape(x.q.shape)) for x in (c, d))
    keep = np.ones((2, 5), bool)
    keep[1, 2] = False
    assert (got[keep] == ref[keep]).all()
    assert np.isnan(got[1, 2, 40]).any() and (c.outs[1].numpy(np.uint16) == d.outs[1].numpy(np.uint16)).all()
    if not np.isnan(value):  # everything else over an infinite root
        row = np.delete(got[1, 2], [8, 40])
        assert (row[~np.isnan(row)] == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("half", [0, 16])
def test_an_infinite_value_outside_the_rotated_part(gpu, half, interleaved):
    def edit(c):
        c.q[1, 2, 41] = 0x7F80
    c = RopeCase(2, 5, 2, 128, half, [5, 6], interleaved=interleaved, edit=edit, seed=3)
    c.call()
    synchronize()
    row = bf16_values(c.outs[0].numpy(np.uint16).reshape(c.q.shape))[1, 2]
    assert np.isnan(row[41]) and (np.delete(row, 41) == 0).all()


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("half", [0, 16])
def test_a_weight_without_a_number_outside_the_rotated_part(gpu, half, interleaved, kind, value):
    """It is the factor of its own dim alone: an infinite one gives an infinity, and every other dim keeps its bits."""
    c, d = (RopeCase(2, 5, 2, 128, half, [5, 6], weight=kind, interleaved=interleaved, seed=3) for _ in range(2))
    for i, w in enumerate(c.weights):
        w[41] = value
        c.d_weights[i] = DeviceArray.from_numpy(na.FP32, w) if kind == "fp32" else DeviceArray.from_numpy(na.BF16, bf16_bits(w))
    c.call()
    d.call()
    synchronize()
    for x, o, p in zip((c.q, c.k), c.outs, d.outs):
        got, ref = (y.numpy(np.uint16).reshape(x.shape) for y in (o, p))
        assert (np.delete(got, 41, -1) == np.delete(ref, 41, -1)).all()
        want = np.copysign(np.float32(1), bf16_values(x[..., 41])) * np.float32(value)
        assert np.array_equal(bf16_values(got[..., 41]), want, equal_nan=True)
    # on the way into a cache: the same bits
    p = PagedCase([(2, 5)], Hq=5, Hkv=2, kv="bf16", page=16, seed=3)
    one, two = p.upload(p.planes(new_rows=False)), p.upload(p.planes(new_rows=False))
    two.k = c.outs[1]
    two.append()
    q_out = Strided(na.BF16, (128, 5, 2), 64)
    qw, kw, _, freq, norm = c.args()
    ops.paged_qk_norm_rope_append(c.d_q.t, c.d_k.t, one.v.t, qw, kw, one.starts.tensor(), one.history.tensor(), freq, norm, one.view, q_out.t)
    synchronize()
    for a, b in zip(one.pool(), two.pool()):
        assert (a == b).all()
    assert (q_out.numpy(np.uint16) == c.outs[0].numpy(np.uint16)).all()


def test_in_place(gpu):
    c, d = RopeCase(40, 8, 2, 128, 64, np.arange(40), seed=4), RopeCase(40, 8, 2, 128, 64, np.arange(40), seed=4)
    c.call()
    d.call(outs=[d.d_q, d.d_k])
    synchronize()
    for a, b in zip(c.outs, (d.d_q, d.d_k)):
        assert (a.numpy(np.uint16) == b.numpy(np.uint16)).all()


def test_stream_and_graph(gpu):
    c = RopeCase(33, 8, 2, 256, 32, np.arange(33), seed=5)
    s = Stream()
    with Graph(s) as g:
        c.call(stream=s)
    for step in range(3):
        c.positions = np.arange(33, dtype=np.int32) * (step + 2)
        c.d_pos.upload(c.positions)
        for o in c.outs:
            o.buf.fill(0xCD)
        synchronize()
        g.launch()
        s.synchronize()
        c.check()


@pytest.mark.parametrize("kv", ["i8", "bf16"])
@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256", "5-5-256"])
@pytest.mark.parametrize("name,seqs", [("step", [(1, 40), (1, 0), (0, 9), (1, 700)]), ("prompts", [(70, 0), (33, 5), (1, 15), (200, 130)]), ("one", [(1, 0)])])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_is_the_two_calls(gpu, kv, geo, name, seqs, interleaved):
    """Ragged batches with an absent page, rows past the table, tokens before the first and after the last sequence."""
    Hq, Hkv, D = GEO[geo]
    for absent, max_pages in (((), None), ({(0, 0)}, None), ((), 3)):
        c = PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=7, lead=2, tail=3, pad=32, page_pad=64, absent=absent, max_pages=max_pages)
        r = RopeCase(c.N, Hq, Hkv, D, D // 4, np.zeros(c.N), interleaved=interleaved, offset=1.0, seed=8)
        position = np.zeros(c.N, np.int32)
        for b, (t, h) in enumerate(seqs):
            position[c.starts[b]:c.starts[b] + t] = h + np.arange(t)
        r.d_pos.upload(position)
        one, two = c.upload(c.planes(new_rows=False)), c.upload(c.planes(new_rows=False))
        r.call()
        two.k = r.outs[1]
        two.append()
        q_out = Strided(na.BF16, (D, Hq, c.N), 64)
        qw, kw, _, freq, norm = r.args()
        ops.paged_qk_norm_rope_append(r.d_q.t, r.d_k.t, one.v.t, qw, kw, one.starts.tensor(), one.history.tensor(), freq, norm, one.view, q_out.t)
        synchronize()
        for a, b in zip(one.pool(), two.pool()):
            assert (a == b).all()
        got, ref = (x.numpy(np.uint16).reshape(c.N, -1) for x in (q_out, r.outs[0]))
        mine = slice(int(c.starts[0]), int(c.starts[-1]))
        assert (got[mine] == ref[mine]).all()
        assert (got[:mine.start] == 0xCDCD).all() and (got[mine.stop:] == 0xCDCD).all(), "tokens of no sequence were written"


def test_append_of_a_large_batch(gpu):
    """1,024 sequences, the last of them found behind many that start at the same token."""
    seqs = [(b % 3 == 0, b % 50) for b in range(1024)]
    seqs = [(int(t), h) for t, h in seqs]
    c = PagedCase(seqs, Hq=2, Hkv=1, D=128, kv="i8", page=16, seed=9)
    r = RopeCase(c.N, 2, 1, 128, 64, np.concatenate([np.arange(h, h + t) for t, h in seqs]), seed=9)
    one, two = c.upload(c.planes(new_rows=False)), c.upload(c.planes(new_rows=False))
    r.call()
    two.k = r.outs[1]
    two.append()
    q_out = Strided(na.BF16, (128, 2, c.N), 64)
    qw, kw, _, freq, norm = r.args()
    ops.paged_qk_norm_rope_append(r.d_q.t, r.d_k.t, one.v.t, qw, kw, one.starts.tensor(), one.history.tensor(), freq, norm, one.view, q_out.t)
    synchronize()
    for a, b in zip(one.pool(), two.pool()):
        assert (a == b).all()
    assert (q_out.numpy(np.uint16) == r.outs[0].numpy(np.uint16)).all()


def test_large_outputs_are_the_small_ones(gpu):
    """More than 64 MiB of heads in one call: the same bits as two calls with half the tokens each."""
    c = RopeCase(1900, 64, 8, 256, 32, np.arange(1900) + 5, seed=10)
    c.call()
    synchronize()
    whole = [o.numpy(np.uint16).reshape(1900, -1).copy() for o in c.outs]
    for lo, hi in ((0, 950), (950, 1900)):
        h = RopeCase(1900, 64, 8, 256, 32, np.arange(1900) + 5, seed=10)
        qw, kw, _, freq, norm = h.args()
        h.d_q, h.d_k = (Strided(na.BF16, (256, x.shape[1], hi - lo), 64).upload(x[lo:hi]) for x in (c.q, c.k))
        h.d_pos = DeviceArray.from_numpy(na.I32, c.positions[lo:hi])
        h.outs = [Strided(na.BF16, (256, n, hi - lo), 64) for n in (64, 8)]
        h.call()
        synchronize()
        for o, w in zip(h.outs, whole):
            assert (o.numpy(np.uint16).reshape(hi - lo, -1) == w[lo:hi]).all()


@pytest.mark.parametrize("kv", ["i8", "bf16"])
def test_large_append_is_the_two_calls(gpu, kv):
    seqs = [(1001, 30), (800, 0), (1, 99)]
    c = PagedCase(seqs, Hq=64, Hkv=8, D=256, kv=kv, page=64, seed=11, absent={(1, 2)})
    r = RopeCase(c.N, 64, 8, 256, 128, np.concatenate([np.arange(h, h + t) for t, h in seqs]), interleaved=True, seed=12)
    one, two = c.upload(c.planes(new_rows=False)), c.upload(c.planes(new_rows=False))
    r.call()
    two.k = r.outs[1]
    two.append()
    q_out = Strided(na.BF16, (256, 64, c.N), 64)
    qw, kw, _, freq, norm = r.args()
    ops.paged_qk_norm_rope_append(r.d_q.t, r.d_k.t, one.v.t, qw, kw, one.starts.tensor(), one.history.tensor(), freq, norm, one.view, q_out.t)
    synchronize()
    for a, b in zip(one.pool(), two.pool()):
        assert (a == b).all()
    assert (q_out.numpy(np.uint16) == r.outs[0].numpy(np.uint16)).all()
