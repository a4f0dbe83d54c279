"""Paged attention and paged rows at the sizes that take the forms for long calls, against 64 bits: chosen tokens with most of
their weight on a few keys, so that a lost key, page or split shows."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd.device import synchronize
from paged_bound import borders, check_bound, needles
from paged_case import PagedCase, bf16_bits, bf16_values

pytestmark = pytest.mark.gpu

CACHES = ["i8", "bf16"]


def _tokens(c, r, each=6):
    """Packed tokens of every sequence: the first and last, the borders of row tiles, and some others."""
    out = set()
    for b, (t, _) in enumerate(c.seqs):
        if t:
            some = {0, 1, t // 2, t - 2, t - 1, 25, 26, 51, 52, *r.integers(0, t, each).tolist()}
            out |= {int(c.starts[b]) + i for i in some if 0 <= i < t}
    return sorted(out)


LARGE = {  # row tiles x heads past one round of the compute units, the rest split over the keys
    "40-8-128": (40, 8, 128, [(1700, 500), (1, 900), (0, 5), (70, 30), (1, 33)], {}),
    "40-8-128 one": (40, 8, 128, [(1800, 1500)], {}),
    "40-8-128 window": (40, 8, 128, [(1800, 900), (1, 2000)], dict(window=400, sinks=5)),
    "24-4-256": (24, 4, 256, [(1500, 600), (1, 700), (150, 30), (0, 4)], {}),
    "24-4-256 one": (24, 4, 256, [(1480, 2000)], {}),
    "24-4-256 window": (24, 4, 256, [(1500, 900), (1, 2000)], dict(window=400, sinks=5)),
    "16-2-256": (16, 2, 256, [(2300, 200), (3, 400)], {}),
}


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("name", LARGE)
@pytest.mark.parametrize("what", ["plain", "absent pages", "outgrown values"])
def test_more_row_tiles_than_compute_units(gpu, kv, name, what):
    Hq, Hkv, D, seqs, kw = LARGE[name]
    gone = {(0, p) for p in (3, 5, 20)} if what == "absent pages" else set()

    def edit(c):
        for b, (t, h) in enumerate(c.seqs):
            rows = borders(t, h) + ([h + 400, h + 800, h + 1200] if t > 1000 else [])
            if c.window:  # some in every token's window
                rows = [0, 3, 4] + list(range(70, t + h, 97))
            needles(c, b, rows)
        if what == "outgrown values":  # of one key tile, and of one new row
            for r in (300, 1300):
                c.v[0][r] = bf16_bits(bf16_values(c.v[0][r]) * np.float32(1e4))
    c = PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=32, seed=40, lead=1, tail=2, absent=gone, edit=edit, **kw)
    d = c.upload()
    d.attend()
    r = np.random.default_rng(41)
    check_bound(c, d.result(), _tokens(c, r), kv_heads=sorted({0, int(r.integers(1, Hkv))}))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("Hq,Hkv,D", [(40, 8, 128), (24, 4, 256), (16, 2, 256)])
@pytest.mark.parametrize("seqs", [[(1, 2999)], [(1, 9000), (1, 20), (0, 3), (1, 3000), (1, 777)], [(2, 5000), (1, 900)]], ids=["one", "ragged", "verify"])
def test_every_key_of_a_long_history_counts(gpu, kv, Hq, Hkv, D, seqs):
    """Most weight on keys at the borders of chunks and shares and on the newest rows, a third of them in turn."""
    for turn in range(3):
        def edit(c):
            r = np.random.default_rng(50)
            for b, (t, h) in enumerate(c.seqs):
                rows = [x for x in dict.fromkeys(borders(t, h) + r.integers(0, max(1, t + h), 12).tolist()) if 0 <= x < t + h]
                needles(c, b, rows[turn::3])
        c = PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, seed=42, edit=edit)
        d = c.upload()
        d.attend()
        check_bound(c, d.result())


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("batch", [65, 150])
def test_many_chunks(gpu, kv, batch):
    """More sequences of many rows than a wave has lanes, single tokens and empty ones among them."""
    r = np.random.default_rng(batch)
    seqs = [(int(r.integers(20, 60)) if i % 3 else int(r.integers(0, 2)), int(r.integers(1, 300))) for i in range(batch)]

    def edit(c):
        for b, (t, h) in enumerate(c.seqs):
            needles(c, b, [0, h // 2, h - 1, h, h + t - 1])
    c = PagedCase(seqs, Hq=8, Hkv=2, kv=kv, page=16, seed=43, lead=1, tail=1, edit=edit)
    d = c.upload()
    d.attend()
    check_bound(c, d.result(), _tokens(c, r, each=1))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", [(10, 2, 128), (12, 2, 256)])
@pytest.mark.parametrize("page", [128, 1024, 4096])
@pytest.mark.parametrize("tokens", [1, 100])
def test_large_pages(gpu, kv, geo, page, tokens):
    Hq, Hkv, D = geo

    def edit(c):
        for b, (t, h) in enumerate(c.seqs):
            needles(c, b, borders(t, h) + [1023, 1024, 4095, 4096])
    c = PagedCase([(tokens, 4500), (1, 1100), (tokens, 0)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=page, seed=44, edit=edit)
    d = c.upload()
    d.attend()
    check_bound(c, d.result(), _tokens(c, np.random.default_rng(45), each=3))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", [(10, 2, 128), (12, 2, 256)])
@pytest.mark.parametrize("window,sinks", [(1, 300), (50, 129), (200, 1000), (64, 64), (3000, 1)])
@pytest.mark.parametrize("tokens", [1, 4, 120])
def test_many_sinks(gpu, kv, geo, window, sinks, tokens):
    """Sinks over several key tiles, as long as the window or longer, up to and past the new tokens."""
    Hq, Hkv, D = geo

    def edit(c):
        for b, (t, h) in enumerate(c.seqs):
            needles(c, b, [0, 31, 63, 64, 127, 128, 129, 299, 300, h - window, h - 1, h, h + t - 2, h + t - 1])
    c = PagedCase([(tokens, 900), (tokens, 40)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=16, window=window, sinks=sinks, seed=46, edit=edit)
    d = c.upload()
    d.attend()
    check_bound(c, d.result(), _tokens(c, np.random.default_rng(47), each=6))


# ---- rows

SHAPES = [  # (KV heads, head_dim, sequences): more than 2^20 pieces of eight values
    (8, 128, [(5000, 40), (0, 9), (1, 0), (3300, 17), (77, 2000), (0, 1), (101, 128)]),
    (4, 256, [(8000, 3), (300, 60), (1, 1), (0, 7), (95, 0)]),
    (3, 128, [(21000, 100), (0, 2), (900, 31), (1, 127)]),
]


def _planes_equal(got, want):
    for g, w in zip(got, want, strict=True):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_long_append_and_read(gpu, kv, i):
    Hkv, D, seqs = SHAPES[i]
    c = PagedCase(seqs, Hq=Hkv, Hkv=Hkv, D=D, kv=kv, page=128, seed=60 + i, absent={(0, 2), (0, 30)}, lead=3, tail=5, pad=32, page_pad=64)
    assert c.N * Hkv * D // 8 > 1 << 20 and c.N * Hkv * D // 8 % 1024
    d = c.upload(c.planes(new_rows=False))
    d.append()
    synchronize()
    _planes_equal(d.pool(), c.planes())
    first = [max(0, h - 2) for _, h in seqs]
    for dtype in (na.BF16, na.FP32):
        got = d.read(first, dtype)
        for plane in range(2):
            want = np.full((c.N, Hkv, D), 0xCDCDCDCD, np.uint32) if dtype == na.FP32 else np.full((c.N, Hkv, D), 0xCDCD, np.uint16)
            for b, (t, _) in enumerate(seqs):
                rows = first[b] + np.arange(t)
                vals = c.stored(b)[plane][rows].astype(np.float32)
                vals[~c.present(b, rows)] = 0
                want[c.starts[b]:c.starts[b] + t] = vals.view(np.uint32) if dtype == na.FP32 else bf16_bits(vals)
            assert np.array_equal(got[plane].view(want.dtype), want)


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("batch", [300, 1024])
def test_rows_of_many_sequences(gpu, kv, batch):
    r = np.random.default_rng(batch)
    seqs = [(int(r.integers(0, 5)), int(r.integers(1, 40))) for _ in range(batch)]
    c = PagedCase(seqs, Hq=2, Hkv=2, kv=kv, page=16, seed=61, lead=2, tail=1)
    d = c.upload(c.planes(new_rows=False))
    d.append()
    got = d.read(c.history)
    _planes_equal(d.pool(), c.planes())
    for plane in range(2):
        want = np.concatenate([c.stored(b)[plane][h:] for b, (t, h) in enumerate(seqs)]).astype(np.float32)
        assert np.array_equal(got[plane][c.starts[0]:c.starts[-1]], want)
