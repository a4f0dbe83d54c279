"""Attention over a paged cache against a 64-bit plain implementation, every element within a derived tolerance."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.device import DeviceArray, DeviceBuffer, Graph, Stream, synchronize
from paged_case import PagedCase, bf16_bits, bf16_values, check_attention

pytestmark = pytest.mark.gpu

GEO = {"40-8-128": (40, 8, 128), "24-4-256": (24, 4, 256), "16-2-256": (16, 2, 256), "4-4-128": (4, 4, 128), "33-1-128": (33, 1, 128)}
CACHES = ["i8", "bf16"]


def _run(c, **kw):
    d = c.upload()
    d.attend(**kw)
    worst = check_attention(c, d.result())
    print(f"worst {worst:.3f} of the tolerance", flush=True)
    return d


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("rows", [1, 15, 16, 17, 100, 517, 3000])
def test_one_token(gpu, geo, kv, rows):
    Hq, Hkv, D = GEO[geo]
    _run(PagedCase([(1, rows - 1)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16 if rows % 2 else 64, seed=rows))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [2, 3, 6, 7, 13, 33, 64, 150, 301])
def test_chunk_of_one_sequence(gpu, geo, kv, tokens):
    Hq, Hkv, D = GEO[geo]
    history = (0, 1, 130, 700)[tokens % 4]
    _run(PagedCase([(tokens, history)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=tokens, pad=16, tail=2))


RAGGED = {
    "decode": [(1, 40), (1, 900), (1, 0), (1, 2100), (1, 333)],
    "verify": [(4, 1000), (3, 17), (1, 0), (4, 400)],
    "empty": [(0, 100), (1, 50), (0, 0), (2, 0), (0, 7)],
    "mixed": [(1, 700), (200, 300), (1, 64), (0, 9), (33, 0), (7, 1200)],
    "prompts": [(130, 0), (257, 0), (64, 1000)],
}


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("name", RAGGED)
def test_ragged_batch(gpu, geo, kv, name):
    Hq, Hkv, D = GEO[geo]
    _run(PagedCase(RAGGED[name], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=len(name), lead=1, tail=3, page_pad=64))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("Hq,Hkv,D,batch", [(40, 8, 128, 32), (40, 8, 128, 25), (24, 4, 256, 64), (8, 1, 128, 250)])
@pytest.mark.parametrize("rows", [1, 40, 1000])
@pytest.mark.parametrize("window", [0, 50])
def test_as_many_short_sequences_as_compute_units(gpu, kv, Hq, Hkv, D, batch, rows, window):
    """One token each: a workgroup per sequence and head; some sequences without a token, one without pages."""
    r = np.random.default_rng(batch + rows)
    seqs = [(int(r.random() < 0.9), int(r.integers(0, rows))) for _ in range(batch)]
    seqs[3] = (1, rows - 1)
    seqs[7] = (1, 20)
    _run(PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=batch, absent={(7, 0), (7, 1)}, window=window, sinks=2 if window else 0))


@pytest.mark.parametrize("batch", [65, 200])
def test_many_sequences(gpu, batch):
    r = np.random.default_rng(batch)
    seqs = [(int(r.integers(0, 4)), int(r.integers(0, 300))) for _ in range(batch)]
    seqs[batch // 2] = (40, 100)
    _run(PagedCase(seqs, Hq=4, Hkv=2, page=32, seed=batch))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (16, 0), (37, 5), (100, 33), (128, 16), (4000, 4)])
@pytest.mark.parametrize("seqs", [[(1, 1500), (1, 20), (1, 0)], [(3, 500)], [(150, 333)], [(70, 0), (1, 800)]], ids=["decode", "verify", "chunk", "mixed"])
def test_window_and_sinks(gpu, geo, kv, window, sinks, seqs):
    Hq, Hkv, D = GEO[geo]
    _run(PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, window=window, sinks=sinks, seed=window))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("tokens", [1, 60])
def test_pages_that_left_the_window(gpu, kv, tokens):
    """Pages between the sinks and the window may be gone; so may pages that a token would see (those rows are not there)."""
    h, w, s = 1000, 100, 4
    gone = {(0, p) for p in range(1, (h + 1 - w) // 16)}
    _run(PagedCase([(tokens, h)], Hq=8, Hkv=2, kv=kv, window=w, sinks=s, absent=gone, seed=1))
    _run(PagedCase([(tokens, h)], Hq=8, Hkv=2, kv=kv, window=w, sinks=s, absent=gone | {(0, 59), (0, 0)}, seed=2))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("tokens,history", [(1, 100), (70, 0), (3, 5)])
def test_no_visible_row(gpu, kv, tokens, history):
    """All pages of a sequence absent: its rows are zero; its neighbour's are not touched by that."""
    pages = -(-(tokens + history) // 16)
    c = PagedCase([(tokens, history), (2, 30)], Hq=8, Hkv=2, kv=kv, absent={(0, p) for p in range(pages)}, seed=4)
    d = _run(c)
    assert (d.result()[:tokens] & 0x7FFF == 0).all()


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("tokens", [4, 100])
def test_infinite_and_nan_values_reach_only_rows_that_see_them(gpu, kv, tokens):
    """A new token's V is infinite (NaN for another): earlier tokens of the chunk do not see it."""
    bad = tokens - 2

    def edit(c):
        c.v[0][300 + bad, 0, 3] = 0x7F80
        c.v[0][300 + bad, 1, 70] = 0xFF80
        c.v[0][300 + bad + 1, 1, 71] = 0x7FC0
        c.k[0][300 + bad + 1, 0, 0] = 0x7F80 if c.kv == "bf16" else c.k[0][300 + bad + 1, 0, 0]
    c = PagedCase([(tokens, 300), (2, 40)], Hq=4, Hkv=2, kv=kv, seed=6, edit=edit)
    d = c.upload()
    d.attend()
    got = d.result()
    # rows before the values: as without them
    ref, tol = PagedCase([(tokens, 300), (2, 40)], Hq=4, Hkv=2, kv=kv, seed=6).oracle()
    g = bf16_values(got).astype(np.float64)
    keep = [i for i in range(tokens + 2) if i < bad or i >= tokens]
    assert (np.abs(g[keep] - ref[keep]) <= tol[keep]).all()
    # the row that sees the infinite value: not finite in that dimension (INT8: in its group)
    assert not np.isfinite(g[bad, 0:2, 3]).any() and not np.isfinite(g[bad, 2:4, 70]).any()
    assert np.isfinite(g[bad, 0:2, 64:]).all()


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("tokens", [1, 3, 90])
def test_rows_behind_the_window_hold_anything(gpu, kv, tokens):
    """Rows between the sinks and the window, and new rows that their own token no longer counts for: infinite and NaN
    keys and values there change nothing for the tokens that do not see them."""
    h, w, s = 700, 64, 5

    def edit(c):
        for r, bits in ((5, 0x7F80), (40, 0x7FC0), (h + 1 - w - 1, 0xFF80), (h + 1 - w - 20, 0x7FC0)):
            c.k[0][r] = bits
            c.v[0][r] = bits
    c = PagedCase([(tokens, h)], Hq=8, Hkv=2, kv=kv, window=w, sinks=s, seed=22, edit=edit)
    d = c.upload()
    d.attend()
    ref, tol = PagedCase([(tokens, h)], Hq=8, Hkv=2, kv=kv, window=w, sinks=s, seed=22).oracle()
    g = bf16_values(d.result()).astype(np.float64)
    assert (np.abs(g - ref) <= tol).all()


@pytest.mark.parametrize("kv", CACHES)
def test_graphs_that_share_a_workspace(gpu, kv):
    """Two captured calls of different batches with one workspace, replayed in turn on one stream, eager calls between."""
    cases = [PagedCase([(1, 1500), (1, 300), (4, 900)], Hq=40, Hkv=8, kv=kv, seed=23), PagedCase([(100, 700), (1, 2000)], Hq=40, Hkv=8, kv=kv, seed=24)]
    devs = [c.upload() for c in cases]
    stream = Stream()
    need = max(ops.paged_attention_workspace_bytes(c.Hq, c.Hkv, c.D, c.N, c.B, c.envelope()) for c in cases)
    ws = DeviceBuffer(need)
    ws.fill(0xFF)
    graphs = []
    for d in devs:
        with Graph(stream) as g:
            d.attend(ws=ws, stream=stream)
        graphs.append(g)
    first = []
    for turn in range(3):
        for i, (c, d, g) in enumerate(zip(cases, devs, graphs)):
            d.out.buf.fill(0xCD)
            synchronize()
            g.launch()
            stream.synchronize()
            got = d.result()
            if turn == 0:
                check_attention(c, got)
                first.append(got)
            assert np.array_equal(got, first[i])
            d.attend(ws=ws, stream=stream)
            stream.synchronize()
            assert np.array_equal(d.result(), first[i])


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3, 3e4, 2e5])
def test_range_of_values(gpu, kv, tokens, size):
    """V from 1e-6 to past what FP16 holds (an INT8 scale of 512 is a value of 65,024), keys alike."""
    def edit(c):
        for x in c.v:
            f = (x.astype(np.uint32) << 16).view(np.float32) * np.float32(size)
            x[:] = bf16_bits(f)
        if size > 1:
            for x in c.k:
                x[5] = bf16_bits((x[5].astype(np.uint32) << 16).view(np.float32) * np.float32(size))
    _run(PagedCase([(tokens, 400)], Hq=10, Hkv=2, kv=kv, seed=7, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("tokens", [1, 90])
def test_small_values_next_to_large_ones(gpu, kv, tokens):
    """A key that hardly counts has a V of 1e5 to 1e6 times the others' size."""
    def edit(c):
        c.q[:, :, 1] = bf16_bits(np.float32(8.0))
        c.k[0][7, :, 1] = bf16_bits(np.float32(-60.0))
        c.v[0][7] = bf16_bits(np.full(c.v[0][7].shape, 2e5, np.float32))
    _run(PagedCase([(tokens, 100)], Hq=10, Hkv=2, kv=kv, seed=7, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256"])
@pytest.mark.parametrize("tokens,window", [(13, 0), (90, 0), (300, 0), (300, 200)])
def test_large_values_in_later_tiles(gpu, geo, kv, tokens, window):
    """Keys and values that outgrow what the first key tile led to expect: a V of 1,000 times the size that counts, one of
    1e5 times that hardly does, a K of 300 times, in tiles of their own and among new tokens."""
    Hq, Hkv, D = GEO[geo]

    def grow(x, f):
        x[:] = bf16_bits((x.astype(np.uint32) << 16).view(np.float32) * np.float32(f))

    def edit(c):
        grow(c.v[0][310], 1e3)
        grow(c.k[0][450, 0], 300.0)
        grow(c.v[0][600 + tokens // 2, Hkv - 1], 3e3)
        c.q[:, :, 1] = bf16_bits(np.float32(8.0))
        c.k[0][590, :, 1] = bf16_bits(np.float32(-60.0))
        grow(c.v[0][590], 1e5)
    _run(PagedCase([(tokens, 600)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=21, window=window, sinks=3 if window else 0, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("scale", [1e-4, 1.0, 3.0])
def test_scale(gpu, kv, scale):
    _run(PagedCase([(1, 300), (70, 30)], Hq=8, Hkv=2, kv=kv, seed=11, scale=scale))


@pytest.mark.parametrize("kv", CACHES)
def test_growing_scores(gpu, kv):
    """Keys that grow along the history: the running maximum moves again and again."""
    def edit(c):
        for x in c.k:
            g = np.linspace(0.05, 6.0, x.shape[0], dtype=np.float32)[:, None, None]
            x[:] = bf16_bits((x.astype(np.uint32) << 16).view(np.float32) * g)
    _run(PagedCase([(1, 3000), (80, 900)], Hq=8, Hkv=2, kv=kv, seed=12, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("Hq,Hkv,D,tokens,rows", [(64, 64, 128, 1, 72000), (40, 8, 128, 1, 400000), (24, 4, 256, 1, 300000), (48, 8, 256, 4, 300000),
                                                  (40, 8, 128, 100, 600000), (24, 4, 256, 60, 500000)])
def test_long_walks_over_shared_pages(gpu, kv, Hq, Hkv, D, tokens, rows):
    """Every workgroup walks more tiles than one fetch of the page table holds. The history is a few pages that appear
    again and again in the table (a row of them counts as often), so the 64-bit result needs those rows only. One page
    appears once, at a hundred places in turn, and most of the weight is on it."""
    page, shared = 64, 13
    n = rows // page

    def edit(c):
        c.q[:, :, 1] = bf16_bits(np.float32(8.0))
        c.k[0][:, :, 1] = bf16_bits(np.float32(0.0))
        c.k[0][(shared - 1) * page:shared * page, :, 1] = bf16_bits(np.float32(18.0))  # scores 9 to 13 above the others
    c = PagedCase([(tokens, shared * page + 37)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=page, seed=25, spare=0, edit=edit)
    r = np.random.default_rng(26)
    order = np.concatenate([np.arange(shared), r.integers(0, shared - 1, n - shared)])
    own = c.table[0, shared:].copy()  # the last pages: some history, the new rows
    names = c.table[0, :shared].copy()
    planes = c.planes()
    K, V = c.stored(0)
    h = c.seqs[0][1]
    c.table, c.max_pages = np.concatenate([names[order], own])[None].astype(np.int32), n + len(own)
    d = c.upload(planes)
    d.history.upload(np.array([h + (n - shared) * page], np.int32))
    env = (tokens, c.max_pages * page)
    ws = d.workspace(env)
    G = Hq // Hkv
    q = bf16_values(c.q).astype(np.float64).reshape(tokens, Hkv, G, D)
    see = np.arange(h + tokens)[None] <= (h + np.arange(tokens))[:, None]
    heads = (0, Hkv - 1)
    sc = [np.where(see[:, None], (q[:, hh] @ K[:, hh].T) * c.scale, -np.inf) for hh in heads]
    size = [np.where(see[:, None], np.abs(q[:, hh]) @ np.abs(K[:, hh]).T * c.scale, 0.0).max(-1, keepdims=True) * 2.0**-11 for hh in heads]
    for place in r.integers(0, n, 100):
        at = order.copy()
        at[at == shared - 1] = 0
        at[place] = shared - 1
        d.table.upload(np.concatenate([names[at], own])[None].astype(np.int32))
        d.attend(envelope=env, ws=ws)
        got = bf16_values(d.result()).astype(np.float64)
        weight = np.ones(h + tokens)
        weight[:shared * page] = np.repeat(np.bincount(at, minlength=shared), page)
        for hh, s, e in zip(heads, sc, size):
            p = np.exp(s - s.max(-1, keepdims=True)) * weight
            p /= p.sum(-1, keepdims=True)
            o, A = p @ V[:, hh], p @ np.abs(V[:, hh])
            # as in PagedCase.oracle; the sums of this many rows in 32 bits add 2^-16 of the terms
            tol = 2.0**-8 * np.abs(o) + A * (2 * np.expm1(2 * e) + 2.0**-10 + 2.0**-16)
            assert (np.abs(got[:, hh * G:(hh + 1) * G] - o) <= tol).all(), f"the page at place {place} of {n}"


def test_sequences_outside_the_envelope_are_left_out(gpu):
    c = PagedCase([(1, 40), (5, 100), (1, 600), (2, 30)], Hq=8, Hkv=2, seed=13)
    d = c.upload()
    d.attend(envelope=(4, 200))  # the second has too many tokens, the third too many rows
    check_attention(c, d.result(), only=[0, 3])
    d = c.upload()
    d.history.upload(np.array([40, 100, -1, 30], np.int32))
    d.attend()
    check_attention(c, d.result(), only=[0, 1, 3])
    d = c.upload()
    d.starts.upload(np.array([0, 1, 6, 7, 2000], np.int32))
    d.attend()
    check_attention(c, d.result(), only=[0, 1, 2])


def test_wide_envelope_changes_nothing_but_the_split(gpu):
    c = PagedCase([(1, 200), (3, 90)], Hq=40, Hkv=8, seed=14, max_pages=4096)
    d = c.upload()
    d.attend(envelope=(512, 65536))
    check_attention(c, d.result())


def test_page_offsets_past_32_bits(gpu):
    """Pages 70 MB apart (a pool that many layers share): the last ones lie past 4 GiB."""
    c = PagedCase([(1, 900), (40, 100)], Hq=8, Hkv=2, seed=15, page=16, spare=0)
    assert c.pages > 64
    big = 70 << 20
    d = c.upload()
    bufs = []
    for i, (s, name) in enumerate(zip(d.planes, ("k", "v", "k_scale", "v_scale"))):
        step = big if i < 2 else 1 << 20
        buf = DeviceBuffer(c.pages * step)
        host = s.buf.download(np.uint8, s.n * s.stride).reshape(s.n, s.stride)
        for p in range(c.pages):
            buf.upload(np.ascontiguousarray(host[p, :s.row]), p * step)
        t = getattr(d.view, name)
        t.data = buf.ptr
        t.nb[3] = step
        bufs.append(buf)
    d.append()
    d.attend()
    check_attention(c, d.result())
    got = d.read(c.history)
    assert np.array_equal(got[0][0], c.stored(0)[0][900].astype(np.float32))


@pytest.mark.parametrize("kv", CACHES)
def test_steps_together_in_a_graph(gpu, kv):
    """Prompt, then decode steps: append, attention and read back on one stream, eagerly and as a graph that is
    replayed with the history advanced on the device; every replay is checked against the eager step and the oracle."""
    H, Hq, D, page, steps = 2, 8, 128, 16, 4
    full = PagedCase([(0, 90 + steps), (0, 37 + steps), (0, steps)], Hq=Hq, Hkv=H, D=D, kv=kv, page=page, seed=16, spare=1)
    B = full.B
    stream = Stream()

    def step_case(i):
        c = PagedCase([(1, h - steps + i) for _, h in full.seqs], Hq=Hq, Hkv=H, D=D, kv=kv, page=page, seed=100 + i)
        c.table, c.pages, c.max_pages = full.table, full.pages, full.max_pages
        c.k = [x[:h + 1] for x, (_, h) in zip(full.k, c.seqs)]
        c.v = [x[:h + 1] for x, (_, h) in zip(full.v, c.seqs)]
        for b, (_, h) in enumerate(c.seqs):
            c.k_new[b], c.v_new[b] = full.k[b][h], full.v[b][h]
        return c

    # the prompt: every sequence's rows but the last `steps`, appended and attended in one ragged batch
    p = PagedCase([(h - steps, 0) for _, h in full.seqs], Hq=Hq, Hkv=H, D=D, kv=kv, page=page, seed=17)
    p.table, p.pages, p.max_pages = full.table, full.pages, full.max_pages
    for b, (t, _) in enumerate(p.seqs):
        p.k[b], p.v[b] = full.k[b][:t], full.v[b][:t]
        p.k_new[p.starts[b]:p.starts[b] + t], p.v_new[p.starts[b]:p.starts[b] + t] = p.k[b], p.v[b]
    d = p.upload([np.full_like(x, 0x77) for x in full.planes()])
    d.append(stream)
    d.attend(stream=stream)
    stream.synchronize()
    check_attention(p, d.result())

    # decode steps: eager on a twin of the cache, and a captured graph
    env = (1, max(h for _, h in full.seqs))
    twins = []
    for _ in range(2):
        c0 = step_case(0)
        t = c0.upload(d.pool())
        t.work = t.workspace(env)
        t.back = [DeviceArray(na.FP32, (D, H, B)) for _ in range(2)]
        twins.append(t)

    def calls(t):
        t.append(stream)
        t.attend(envelope=env, ws=t.work, stream=stream)
        ops.paged_kv_read(t.view, t.starts.tensor(), t.history.tensor(), t.back[0].tensor(), t.back[1].tensor(), stream)
        for b in range(B):
            ops.increment_i32_scalar(na.Tensor.make(t.history.ptr + 4 * b, na.I32, (1,)), stream)

    with Graph(stream) as graph:
        calls(twins[0])
    for i in range(steps):
        c = step_case(i)
        for t in twins:
            t.q.upload(c.q)
            t.k.upload(c.k_new)
            t.v.upload(c.v_new)
        graph.launch()
        stream.synchronize()
        calls(twins[1])
        stream.synchronize()
        a, b = (t.result() for t in twins)
        assert np.array_equal(a, b)
        check_attention(c, a)
        for plane in range(2):
            assert np.array_equal(twins[0].back[plane].numpy(), twins[1].back[plane].numpy())
            want = np.stack([c.stored(s)[plane][h] for s, (_, h) in enumerate(c.seqs)]).astype(np.float32)
            assert np.array_equal(twins[0].back[plane].numpy().reshape(B, H, D), want)
    for x, y, w in zip(twins[0].pool(), twins[1].pool(), full.planes()):
        assert np.array_equal(x, y)


def test_two_streams_at_once(gpu):
    """Calls that overlap, each with its own workspace, and one graph replayed against another."""
    cases = [PagedCase([(1, 2500), (1, 300)], Hq=40, Hkv=8, seed=18), PagedCase([(120, 400)], Hq=24, Hkv=4, D=256, kv="bf16", seed=19)]
    devs = [c.upload() for c in cases]
    streams = [Stream(), Stream()]
    graphs = []
    for d, s in zip(devs, streams):
        d.work = d.workspace()
        with Graph(s) as g:
            d.attend(ws=d.work, stream=s)
        graphs.append(g)
    first = None
    for _ in range(4):
        for d, s, g in zip(devs, streams, graphs):
            g.launch()
            d.attend(ws=d.work, stream=s)
        synchronize()
        got = [d.result() for d in devs]
        if first is None:
            first = got
            for c, x in zip(cases, got):
                check_attention(c, x)
        for x, y in zip(first, got):
            assert np.array_equal(x, y)


@pytest.mark.parametrize("kv", CACHES)
def test_agrees_with_the_linear_cache(gpu, kv):
    """The same rows in a linear cache and in pages: gqa_attention_cached and paged_attention give the same within
    twice the tolerance of one of them."""
    from ninfer_amd.kv_cache import KVCacheLayer
    c = PagedCase([(4, 700)], Hq=40, Hkv=8, kv=kv, seed=20)
    d = _run(c)
    lin = KVCacheLayer(704, 8, 128, dtype=na.I8 if kv == "i8" else na.BF16)
    planes = c.planes()
    rows = []
    for x in planes:
        y = np.zeros((8, lin.padded_context, x.shape[-1]), x.dtype)
        for s in range(c.max_pages):
            y[:, s * 16:(s + 1) * 16] = x[c.table[0, s]]
        y[:, 704:] = 0
        rows.append(y)
    lin.upload(*rows)
    q = DeviceArray.from_numpy(na.BF16, c.q, (128, 40, 4))
    pos = DeviceArray.from_numpy(na.I32, np.arange(700, 704, dtype=np.int32))
    out = DeviceArray(na.BF16, (128, 40, 4))
    ws = DeviceBuffer(max(256, ops.gqa_attention_workspace_bytes(40, 8, 128, 4, 1, 704)))
    ops.gqa_attention_cached(q.tensor(), pos.tensor(), c.scale, lin.view(), (704, 704), ws, out.tensor())
    synchronize()
    _, tol = c.oracle()
    a = (out.numpy().astype(np.uint32) << 16).view(np.float32).reshape(4, 40, 128).astype(np.float64)
    b = (d.result().astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    assert (np.abs(a - b) <= 2 * tol).all()
