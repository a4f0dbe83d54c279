"""Attention over selected blocks of a paged cache against a 64-bit plain form, every element within a derived tolerance."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.device import DeviceArray, DeviceBuffer, Graph, Stream, synchronize
from paged_bound import bound, needles
from paged_case import PagedCase, bf16_bits, bf16_values

pytestmark = pytest.mark.gpu

GEO = {"40-8-128": (40, 8, 128), "24-4-256": (24, 4, 256), "16-2-256": (16, 2, 256), "3-3-128": (3, 3, 128), "17-1-128": (17, 1, 128), "40-1-256": (40, 1, 256)}
CACHES = ["i8", "bf16"]
# tokens of a sequence and geometries: single tokens, a wave or more each; prompts, whose lists a workgroup merges
SHAPES = {"one": (1, 8, 2, 128), "few": (40, 8, 2, 128), "prompt": (300, 40, 8, 128), "prompt256": (300, 24, 4, 256), "prompt1": (700, 8, 8, 128)}


def lists(c, S, block, seed=0, fill=1.0):
    """Random blocks for every token and KV head, ascending, -1 behind them; `fill`: how many of those there are."""
    r = np.random.default_rng(seed)
    out = np.full((c.N, c.Hkv, S), -1, np.int32)
    for b, (t, h) in enumerate(c.seqs):
        for i in range(t):
            blocks = (h + i) // block + 1
            for hh in range(c.Hkv):
                k = min(S, max(1, int(blocks * fill)))
                pick = np.sort(r.permutation(blocks)[:k])
                out[c.starts[b] + i, hh, :k] = pick
    return out


class Sparse:
    def __init__(self, c, selected, block, envelope=None):
        self.c, self.selected, self.block, self.env = c, selected, block, envelope or c.envelope()
        self.d = c.upload()
        self.lists = DeviceArray.from_numpy(na.I32, selected)
        need = ops.paged_sparse_attention_workspace_bytes(c.Hq, c.Hkv, c.D, c.N, c.B, selected.shape[-1], block)
        self.ws = DeviceBuffer(max(256, need))
        self.ws.fill(0xFF)

    def call(self, stream=None):
        c, d = self.c, self.d
        ops.paged_sparse_attention(d.q.t, d.starts.tensor(), d.history.tensor(), c.scale, self.lists.tensor(), self.block, d.view, self.env, self.ws, d.out.t,
                                   stream)
        return self

    def check(self, tokens=None, only=None):
        c, bits = self.c, self.d.result()
        stored = {}
        plain = c.stored
        c.stored = lambda b: stored.setdefault(b, plain(b))
        G = c.Hq // c.Hkv
        got = bf16_values(bits).astype(np.float64)
        worst = 0.0
        served = np.zeros(c.N, bool)
        for b, (t, h) in enumerate(c.seqs):
            if only is not None and b not in only:
                continue
            served[c.starts[b]:c.starts[b] + t] = True
            for i in range(t):
                n = int(c.starts[b]) + i
                if tokens is not None and n not in tokens:
                    continue
                for hh in range(c.Hkv):
                    blocks = self.selected[n, hh]
                    rows = np.arange(h + i + 1)
                    out_of = rows[~np.isin(rows // self.block, blocks)]
                    for _, _, o, tol in bound(c, [n], [hh], dropped=out_of):
                        err = np.abs(got[n, hh * G:(hh + 1) * G] - o)
                        bad = ~(err <= tol)
                        assert not bad.any(), f"token {n}, KV head {hh}: {bad.sum()} of {bad.size} outside, worst {(err / np.maximum(tol, 1e-300)).max():.3g}"
                        worst = max(worst, float((err / np.maximum(tol, 1e-300)).max()))
        c.stored = plain
        assert (bits[~served] == 0xCDCD).all(), "rows of no sequence were written"
        print(f"worst {worst:.3f} of the bound", flush=True)
        return self


def _run(c, S, block, fill=1.0, **kw):
    return Sparse(c, lists(c, S, block, seed=S, fill=fill), block, **kw).call().check()


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("rows", [1, 31, 32, 33, 517, 3000])
def test_one_token(gpu, geo, kv, rows):
    Hq, Hkv, D = GEO[geo]
    _run(PagedCase([(1, rows - 1)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=64 if rows % 2 else 16, seed=rows), 12, 32)


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256"])
@pytest.mark.parametrize("S", [1, 2, 3, 7, 40, 100])
@pytest.mark.parametrize("block", [32, 64, 256])
def test_lists(gpu, geo, kv, S, block):
    """From one tile of 32 keys to long lists: a wave, four, several workgroups."""
    Hq, Hkv, D = GEO[geo]
    _run(PagedCase([(1, 5000), (2, 700), (1, 3)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=S), S, block)


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256", "17-1-128"])
@pytest.mark.parametrize("seqs", [[(1, 900), (0, 40), (1, 0), (3, 333), (0, 0)], [(70, 300), (1, 64), (33, 0)]], ids=["step", "mixed"])
def test_ragged(gpu, geo, kv, seqs):
    Hq, Hkv, D = GEO[geo]
    _run(PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=len(seqs), lead=1, tail=3, pad=32, page_pad=64), 5, 32)


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256", "16-2-256"])
def test_prompt(gpu, geo, kv):
    """Two prompts, lists merged; blocks of neighbours that differ and agree."""
    Hq, Hkv, D = GEO[geo]
    c = PagedCase([(700, 900), (400, 0)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=64, seed=1)
    r = np.random.default_rng(2)
    Sparse(c, lists(c, 6, 64, seed=3), 64).call().check(tokens=set(r.integers(0, c.N, 60).tolist()) | {0, 699, 700, c.N - 1})


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_all_blocks_is_dense_attention(gpu, kv, shape):
    tokens, Hq, Hkv, D = SHAPES[shape]
    c = PagedCase([(tokens, 250)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=5)
    s = Sparse(c, lists(c, (249 + tokens) // 32 + 1, 32), 32).call().check(tokens={0, tokens - 1})
    a = bf16_values(s.d.result()).astype(np.float64)
    s.d.attend()
    b = bf16_values(s.d.result()).astype(np.float64)
    assert np.abs(a - b).max() <= 2.0**-6 * np.abs(b).max()  # 2 BF16 roundings and the two kernels' own, of values up to the largest


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_lists_of_any_kind(gpu, kv, shape):
    """Any order, gaps, entries past the token's own block or far beyond the table, negative ones: no blocks. Only such: zeros."""
    tokens, Hq, Hkv, D = SHAPES[shape]
    c = PagedCase([(tokens, 300), (1, 77)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=6)
    sel = lists(c, 9, 32, seed=1, fill=0.5)
    r = np.random.default_rng(2)
    for n in range(c.N):
        for hh in range(Hkv):
            r.shuffle(sel[n, hh])
    sel[:, :, 3] = np.array([1000, 2**31 - 1, -(2**31), 40])[np.arange(c.N) % 4][:, None]
    sel[0, 1] = -1
    sel[c.N - 1, 0] = 2**26
    s = Sparse(c, sel, 32).call().check(tokens={0, 1, tokens // 2, tokens - 1, c.N - 1})
    bits = s.d.result()
    assert (bits[0, Hq // Hkv:2 * Hq // Hkv] & 0x7FFF == 0).all() and (bits[c.N - 1, :Hq // Hkv] & 0x7FFF == 0).all()


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_a_block_that_stands_twice_counts_once(gpu, kv, shape):
    """Next to each other, apart, behind an entry that is none, many times over."""
    tokens, Hq, Hkv, D = SHAPES[shape]
    c = PagedCase([(tokens, 2300)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=7)
    sel = np.full((c.N, Hkv, 70), -1, np.int32)
    sel[:, :, :8] = [5, 5, 2, -1, 2, 60, 7, 5]
    sel[:, :, 64:] = [7, 9, 60, 2, 9, 1000]
    sel[::3, :, 8:60] = 2
    Sparse(c, sel, 32).call().check(tokens={0, 1, tokens // 2, tokens - 1})


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("tokens", [1, 3])
def test_the_longest_list_in_any_order(gpu, kv, tokens):
    """1,024 entries, shuffled, a third of them repeats of others, some no block."""
    c = PagedCase([(tokens, 40000)], Hq=8, Hkv=2, kv=kv, page=64, seed=21)
    sel = lists(c, 1024, 32, seed=2)
    r = np.random.default_rng(3)
    for n in range(tokens):
        for hh in range(c.Hkv):
            sel[n, hh, 680:] = r.choice(sel[n, hh, :680], 344)
            r.shuffle(sel[n, hh])
    sel[:, :, 5::97] = -1
    Sparse(c, sel, 32).call().check()


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_absent_pages(gpu, kv, shape):
    gone = {(0, p) for p in (0, 3, 4, 5, 9, 20)}
    tokens, Hq, Hkv, D = SHAPES[shape]
    c = PagedCase([(tokens, 340), (2, 60)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=8, absent=gone | {(1, p) for p in range(4)}, max_pages=66)
    s = Sparse(c, lists(c, 12, 32, seed=1), 32).call().check(tokens={0, 1, tokens - 1, tokens, tokens + 1})
    assert (s.d.result()[tokens:tokens + 2] & 0x7FFF == 0).all()


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_of_other_blocks_hold_anything(gpu, kv, shape):
    """Infinite and NaN keys and values in blocks that are not listed, and past the tokens' positions, change nothing."""
    def edit(c):
        c.v[0][64:96, :, 3] = 0x7F80
        c.k[0][70, :, 5] = 0x7FC0
        c.v[0][75, :, 9] = 0x7FC0
    tokens, Hq, Hkv, D = SHAPES[shape]
    kw = dict(Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=9)
    a, b = PagedCase([(tokens, 200)], edit=edit, **kw), PagedCase([(tokens, 200)], **kw)
    sel = lists(b, 20, 32)
    sel[sel == 2] = -1
    x, y = Sparse(a, sel, 32).call(), Sparse(b, sel, 32).call().check(tokens={0, tokens - 1})
    assert (x.d.result() == y.d.result()).all()


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", ["few", "prompt", "prompt256", "prompt1"])
def test_infinite_and_nan_values_reach_only_rows_that_see_them(gpu, kv, shape):
    """The last but one token's V is infinite, the last one's NaN: earlier tokens of the same block do not see them."""
    tokens, Hq, Hkv, D = SHAPES[shape]
    G = Hq // Hkv
    bad = tokens - 2

    def edit(c):
        c.v[0][300 + bad, 0, 3] = 0x7F80
        c.v[0][300 + bad + 1, 1, 71] = 0x7FC0
    kw = dict(Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=10)
    a, b = PagedCase([(tokens, 300)], edit=edit, **kw), PagedCase([(tokens, 300)], **kw)
    sel = lists(b, 40, 32)
    x, y = Sparse(a, sel, 32).call(), Sparse(b, sel, 32).call().check(tokens={0, bad - 1})
    p, q = bf16_values(x.d.result()), bf16_values(y.d.result())
    assert np.isfinite(p[:bad]).all()
    y.d.out = x.d.out  # the tokens before: within the bounds of the case without
    y.check(tokens=set(range(max(0, bad - 40), bad)))
    assert not np.isfinite(p[bad, 0:G, 3]).any() and np.isfinite(p[bad, G:]).all()
    assert np.isnan(p[bad + 1, G:2 * G, 71]).all()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("value", [1e30, 3e38])
def test_bf16_values_up_to_the_largest(gpu, shape, value):
    """Weighted means of finite values are finite: the largest is at most the largest value."""
    def edit(c):
        c.v[0][32:200, 0, ::3] = bf16_bits(np.float32(value))
    tokens, Hq, Hkv, D = SHAPES[shape]
    c = PagedCase([(tokens, 300)], Hq=Hq, Hkv=Hkv, D=D, kv="bf16", page=32, seed=11, edit=edit)
    Sparse(c, lists(c, 12, 32), 32).call().check(tokens={0, tokens - 1, tokens // 2})


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_needles(gpu, kv, shape):
    """Every listed key counts: a few keys hold all the weight, at the borders of blocks and pages."""
    h = 1000
    tokens, Hq, Hkv, D = SHAPES[shape]
    c = PagedCase([(tokens, h)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=64, seed=12, edit=lambda c: needles(c, 0, [0, 31, 32, 63, 64, 127, 128, 500, 511, 512, h - 1, h]))
    Sparse(c, lists(c, 20, 64, fill=0.9), 64).call().check(tokens={0, tokens - 1, tokens // 2})


@pytest.mark.parametrize("scale", [2.0**-40, 1.0, 2.0**10])
def test_scale(gpu, scale):
    _run(PagedCase([(1, 500), (5, 40)], Hq=4, Hkv=2, kv="bf16", page=32, seed=13, scale=scale), 8, 32)


@pytest.mark.parametrize("kv", CACHES)
def test_outside_the_envelope(gpu, kv):
    c = PagedCase([(3, 400), (1, 900), (9, 10), (1, 100)], Hq=4, Hkv=2, kv=kv, page=32, seed=14)
    Sparse(c, lists(c, 6, 32), 32, envelope=(4, 500)).call().check(only={0, 3})


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_runs_repeat_and_graphs_replay(gpu, kv, shape):
    tokens, Hq, Hkv, D = SHAPES[shape]
    c = PagedCase([(tokens, 2000), (tokens, 500)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=15)
    s = Sparse(c, lists(c, 33, 32), 32).call().check(tokens={0, tokens - 1})
    first = s.d.result()
    st = Stream()
    with Graph(st) as g:
        s.call(st)
    for _ in range(3):
        s.d.out.buf.fill(0xCD)
        s.ws.fill(0xFF)
        synchronize()
        g.launch()
        st.synchronize()
        assert (s.d.result() == first).all()


def test_two_graphs_share_a_workspace(gpu):
    a, b = (Sparse(c, lists(c, 40, 32), 32) for c in (PagedCase([(1, 3000)], Hq=40, Hkv=8, page=32, seed=16), PagedCase([(2, 2000)], Hq=24, Hkv=4, D=256, page=32, seed=17)))
    ws = a.ws if a.ws.nbytes >= b.ws.nbytes else b.ws
    a.ws = b.ws = ws
    st = Stream()
    graphs = []
    for s in (a, b):
        with Graph(st) as g:
            s.call(st)
        graphs.append(g)
    for _ in range(2):
        for s, g in zip((a, b), graphs):
            s.d.out.buf.fill(0xCD)
            synchronize()
            g.launch()
        st.synchronize()
        a.check()
        b.check()


@pytest.mark.parametrize("batch", [65, 300])
def test_many_sequences(gpu, batch):
    r = np.random.default_rng(batch)
    seqs = [(int(r.integers(0, 3)), int(r.integers(0, 200))) for _ in range(batch)]
    c = PagedCase(seqs, Hq=4, Hkv=2, page=32, seed=batch)
    Sparse(c, lists(c, 4, 32), 32).call().check(tokens=set(r.integers(0, c.N, 40).tolist()))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_sizes_far_apart(gpu, kv, shape):
    """Blocks whose keys and values are larger or smaller by far than the others': what FP16 operands do not hold next to each other."""
    tokens, Hq, Hkv, D = SHAPES[shape]

    def edit(c):
        for b, (k, v) in enumerate([(1, 1), (1e-5, 1e4), (3, 1e-6), (1, 0), (1e-3, 1), (2, 300)]):
            rows = slice(32 * b, 32 * b + 32)
            c.k[0][rows] = bf16_bits(bf16_values(c.k[0][rows]) * np.float32(k))
            c.v[0][rows] = bf16_bits(bf16_values(c.v[0][rows]) * np.float32(v))
    c = PagedCase([(tokens, 300)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=18, edit=edit)
    Sparse(c, lists(c, 8, 32, fill=0.8), 32).call().check(tokens={0, 1, tokens // 2, tokens - 1})


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_a_table_that_ends_inside_a_tile(gpu, kv, shape):
    """An odd number of pages of 16 rows, the last of them with values far larger than the others'."""
    tokens, Hq, Hkv, D = SHAPES[shape]
    h = 96 + (-(tokens - 1) % 32 + 9) % 32  # the last row is the tenth of a tile

    def edit(c):
        rows = slice(h + tokens - 10, h + tokens)
        c.v[0][rows] = bf16_bits(bf16_values(c.v[0][rows]) * np.float32(1e4))
    c = PagedCase([(tokens, h)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=20, edit=edit)
    assert c.max_pages % 2 == 1
    Sparse(c, lists(c, (h + tokens - 1) // 32 + 1, 32), 32).call().check(tokens={0, tokens // 2, tokens - 2, tokens - 1})


@pytest.mark.parametrize("block", [32, 128, 256, 512])
@pytest.mark.parametrize("S", [3, 150])
def test_prompts_of_many_blocks(gpu, block, S):
    """Long lists over long histories: more blocks than a workgroup's list holds stay with single tokens."""
    c = PagedCase([(150, 9000)], Hq=8, Hkv=2, kv="i8", page=64, seed=19)
    Sparse(c, lists(c, S, block, seed=1), block).call().check(tokens={0, 77, 149})
