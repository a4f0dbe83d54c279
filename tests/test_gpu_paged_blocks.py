"""Block means and block selection against plain 64-bit forms, bit by bit."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.device import DeviceArray, DeviceBuffer, Graph, Stream, synchronize
from paged_blocks_case import block_means, select
from paged_case import PagedCase, Strided, bf16_bits, bf16_values

pytestmark = pytest.mark.gpu

GEO = {"40-8-128": (40, 8, 128), "24-4-256": (24, 4, 256), "3-3-128": (3, 3, 128)}


class Blocks:
    """Means next to a case's pages, poison at first; `pad`: bytes between pages of the codes."""

    def __init__(self, c, block, pad=0):
        self.c, self.block, self.per = c, block, c.page // block
        self.codes = Strided(na.I8, (c.D, self.per, c.Hkv, c.pages), pad)
        self.scales = Strided(na.FP32, (self.per, c.Hkv, c.pages), 4 if pad else 0)
        self.scales.t.ne[3] = 1
        self.view = na.PagedBlockView()
        self.view.codes, self.view.scales, self.view.block_size = self.codes.t, self.scales.t, block

    def numpy(self):
        c = self.c
        return (self.codes.numpy(np.int8).reshape(c.pages, c.Hkv, self.per, c.D), self.scales.numpy(np.float32).reshape(c.pages, c.Hkv, self.per))

    def upload(self, codes, scales):
        self.codes.upload(codes)
        self.scales.upload(scales)
        return self


def _update(c, block, pad=0):
    d, b = c.upload(), Blocks(c, block, pad)
    ops.paged_block_update(d.view, d.starts.tensor(), d.history.tensor(), c.N, b.view)
    synchronize()
    codes, scales = b.numpy()
    ref = block_means(c, block)
    touched = np.zeros(scales.shape, bool)
    for (s, blk), (rc, rs) in ref.items():
        page, slot = c.table[s, blk * block // c.page], blk % b.per
        assert (codes[page, :, slot] == rc).all(), (s, blk)
        assert (scales[page, :, slot] == rs).all(), (s, blk, scales[page, :, slot], rs)
        touched[page, :, slot] = True
    assert (codes[~touched] == np.int8(-51)).all() and (scales.view(np.uint32)[~touched] == 0xCDCDCDCD).all(), "other blocks were written"
    return b


@pytest.mark.parametrize("kv", ["i8", "bf16"])
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("page,block", [(32, 32), (64, 32), (256, 64), (128, 128)])
@pytest.mark.parametrize("seqs", [[(1, 0)], [(1, 31), (1, 32), (0, 40), (1, 700)], [(500, 0), (3, 62), (129, 255)]], ids=["first", "step", "prompts"])
def test_means(gpu, kv, geo, page, block, seqs):
    Hq, Hkv, D = GEO[geo]
    _update(PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=page, seed=page + block, lead=1, tail=2, page_pad=32), block, pad=16)


@pytest.mark.parametrize("kv", ["i8", "bf16"])
def test_means_of_absent_pages_and_past_the_table(gpu, kv):
    _update(PagedCase([(200, 10), (90, 100)], Hq=4, Hkv=2, kv=kv, page=32, seed=1, absent={(0, 1), (1, 4)}, max_pages=5), 32)


def test_means_of_any_value(gpu):
    """Zeros, the type's largest and smallest values, infinite and NaN keys: each in a block of its own."""
    def edit(c):
        c.k[0][0:64] = 0
        c.k[0][64:128, 0] = bf16_bits(np.float32(3.3e38))
        c.k[0][130, 0, 5] = 0x7F80
        c.k[0][200, 1, 6] = 0x7FC0
        c.k[0][256:320, 0] = 1  # the smallest subnormal
        c.k[0][320:352, 1] = bf16_bits(np.float32(1e30))
    _update(PagedCase([(400, 0)], Hq=4, Hkv=2, kv="bf16", page=64, seed=2, edit=edit), 64)


@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256"])
def test_means_of_rows_of_any_scale(gpu, geo):
    """INT8 rows 2^20 apart in one block, rows of zeros, and one whose scale is infinite."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        r = np.random.default_rng(3)
        rows = bf16_values(c.k[0]) * np.float32(2.0) ** r.integers(-10, 9, (len(c.k[0]), 1, 1)).astype(np.float32)
        rows[40:70] = 0
        rows[300, 1, 7] = 3e38
        c.k[0] = bf16_bits(rows)
    with np.errstate(over="ignore", invalid="ignore"):
        _update(PagedCase([(700, 0)], Hq=Hq, Hkv=Hkv, D=D, kv="i8", page=128, seed=3, edit=edit), 128)


@pytest.mark.parametrize("kv", ["i8", "bf16"])
@pytest.mark.parametrize("geo", ["40-8-128", "24-4-256"])
@pytest.mark.parametrize("page,block,spread", [(512, 256, 9), (1024, 1024, 8), (4096, 4096, 7)])
def test_means_of_large_blocks(gpu, kv, geo, page, block, spread):
    """Up to the largest block, whole and partly filled, rows of sizes far apart. INT8: a lane adds at most rows / 2 products
    (code + 4224) * scale, each below 2^12.1 times the largest scale and a multiple of 2^-11 of the smallest: in 53 bits while scales lie
    within 2^30 / rows. BF16: `rows` values of 8 bits, in 53 bits while those that are not zero lie within 2^45 / rows. Here the rows'
    sizes lie within 2^(2 spread - 1), their scales within 2^4 more and their values, none below 2^-10, within 2^15 more."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        r = np.random.default_rng(block)
        for k in c.k:
            x = bf16_values(k)
            k[:] = bf16_bits(np.where(np.abs(x) < 2.0**-10, 0, x) * np.float32(2.0) ** r.integers(-spread, spread, (len(k), 1, 1)).astype(np.float32))
        c.k[0][block // 2:block // 2 + 30] = 0
    _update(PagedCase([(2 * block + 100, 0), (3, block - 2), (1, 0)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, page=page, seed=block, edit=edit), block, pad=16)


@pytest.mark.parametrize("batch", [65, 1024])
def test_means_of_many_sequences(gpu, batch):
    r = np.random.default_rng(batch)
    seqs = [(int(r.integers(0, 3)), int(r.integers(0, 90))) for _ in range(batch)]
    seqs[batch // 2] = (150, 40)
    _update(PagedCase(seqs, Hq=1, Hkv=1, page=32, seed=batch), 32)


def _select(c, block, pick, seed=0, envelope=None, absent_means=None, edit=None, stream=None, only=None):
    """Selection over random means (as a step over many blocks has them), every list compared."""
    r = np.random.default_rng(seed)
    b = Blocks(c, block, 16)
    codes = r.integers(-127, 128, (c.pages, c.Hkv, b.per, c.D)).astype(np.int8)
    scales = (0.01 + r.random((c.pages, c.Hkv, b.per))).astype(np.float32)
    if edit is not None:
        edit(c, codes, scales)
    b.upload(codes, scales)
    q = Strided(na.BF16, (c.D, c.Hq, c.N), c.pad).upload(c.q)
    starts, history = DeviceArray.from_numpy(na.I32, c.starts), DeviceArray.from_numpy(na.I32, c.history)
    table = Strided(na.I32, (c.max_pages, c.B), 8).upload(c.table)
    S = sum(pick)
    out = DeviceArray(na.I32, (S, c.Hkv, c.N))
    out.upload(np.full((c.N, c.Hkv, S), -77, np.int32))
    env = envelope or c.envelope()
    need = ops.paged_block_select_workspace_bytes(c.Hkv, c.D, c.N, c.B, env, block)
    ws = DeviceBuffer(max(256, need))
    ws.fill(0xFF)

    def call(stream=None):
        ops.paged_block_select(q.t, starts.tensor(), history.tensor(), table.t, c.page, b.view, pick, env, ws, out.tensor(), stream)

    def check():
        synchronize()
        got = out.numpy().reshape(c.N, c.Hkv, S)
        served = np.zeros(c.N, bool)
        G = c.Hq // c.Hkv
        for s, (t, h) in enumerate(c.seqs):
            if only is not None and s not in only:
                continue
            blocks = np.arange(-(-(t + h) // block))
            if t == 0:
                continue
            there = c.present(s, blocks * block)
            page = np.where(there, c.table[s, np.minimum(blocks * block // c.page, c.max_pages - 1)], 0)
            for i in range(t):
                n = int(c.starts[s]) + i
                served[n] = True
                qq = bf16_values(c.q[n]).astype(np.float64).reshape(c.Hkv, G, c.D)
                for hh in range(c.Hkv):
                    ref = select(qq[hh], codes[page, hh, blocks % b.per], scales[page, hh, blocks % b.per], there, h + i, block, *pick)
                    assert (got[n, hh] == ref).all(), (n, hh, got[n, hh], ref)
        assert (got[~served] == -77).all(), "lists of no sequence were written"
    call(stream)
    check()
    return call, check, out


@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("pick", [(0, 1, 0), (1, 2, 5), (0, 1, 1), (2, 3, 40), (5, 1, 16)])
@pytest.mark.parametrize("seqs", [[(1, 0)], [(1, 5000), (1, 31), (0, 9), (1, 2900)], [(70, 3000), (1, 64), (33, 0)]], ids=["first", "step", "mixed"])
def test_selection(gpu, geo, pick, seqs):
    Hq, Hkv, D = GEO[geo]
    _select(PagedCase(seqs, Hq=Hq, Hkv=Hkv, D=D, kv="i8", page=64, seed=len(seqs), lead=1, tail=2, pad=16), 32, pick, seed=sum(pick))


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 9, 16, 17, 31])
@pytest.mark.parametrize("page,block", [(32, 32), (256, 128)])
def test_selection_of_tiles(gpu, tokens, page, block):
    _select(PagedCase([(tokens, 2500), (tokens, 77)], Hq=6, Hkv=2, page=page, seed=tokens), block, (1, 1, 6), seed=tokens)


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("rows", [66000, 300000, 1048576 - 8])
def test_selection_of_many_blocks(gpu, tokens, rows):
    """Up to 32,768 blocks of a sequence: fewer tokens to a tile, down to one."""
    c = _long(tokens, rows, 1 << 12)
    _select(c, 32, (1, 2, 61), seed=rows)


@pytest.mark.parametrize("blocks", [3, 40, 65, 129, 193, 256, 300, 321, 385, 512, 520, 769, 1020, 1027, 1030, 1300, 2000])
@pytest.mark.parametrize("pick", [(1, 2, 29), (0, 1, 400)])
def test_selection_of_a_tile_of_sixteen(gpu, blocks, pick):
    """As many candidates as the forms of the choice take, with scores all over, a few values, and one value but for a few."""
    def some(c, codes, scales):
        scales[:] = 1.0
        codes[:] = 0
        codes[..., 5] = np.random.default_rng(4).integers(-2, 3, codes.shape[:-1])

    def one(c, codes, scales):
        scales[:] = np.where(np.random.default_rng(5).random(scales.shape) < 0.02, np.float32(3.0), np.float32(1.0))
        codes[:] = codes[0, :1, :1]
    for edit in (None, some, one):
        _select(_long(18, 32 * blocks + 7, 1 << 12), 32, pick, seed=blocks, edit=edit)


def _long(tokens, rows, page):
    """A sequence of many rows of which only the pages matter."""
    c = PagedCase([(tokens, 10)], Hq=4, Hkv=1, page=page, seed=tokens)
    h = rows - tokens
    c.seqs, c.history = [(tokens, h)], np.array([h], np.int32)
    c.max_pages = -(-rows // page)
    c.pages = c.max_pages + 2
    c.table = np.random.default_rng(rows).permutation(c.pages)[:c.max_pages].reshape(1, -1).astype(np.int32)
    return c


@pytest.mark.parametrize("tokens", [1, 20])
def test_equal_scores_take_the_lowest_blocks(gpu, tokens):
    def edit(c, codes, scales):
        codes[:] = codes[0, :1, :1]
        scales[:] = 0.5
    _select(PagedCase([(tokens, 4000)], Hq=4, Hkv=2, page=32, seed=3), 32, (2, 2, 9), edit=edit)

    def some(c, codes, scales):  # a few values, many of each
        codes[:] = 0
        codes[..., 0] = np.random.default_rng(4).integers(-1, 2, codes.shape[:-1])
        scales[:] = np.float32(2.0) ** np.random.default_rng(5).integers(-2, 2, scales.shape)
    _select(PagedCase([(tokens, 4000)], Hq=4, Hkv=2, page=32, seed=4), 32, (2, 2, 30), edit=some)


@pytest.mark.parametrize("tokens", [1, 20])
def test_scores_of_any_size(gpu, tokens):
    """Scales of zero (a score of zero, whatever its sign), subnormal, huge and infinite ones."""
    def edit(c, codes, scales):
        r = np.random.default_rng(6)
        scales[:] = r.choice(np.array([0.0, 1e-44, 1e-38, 1.0, 1e30, 2.6e36, np.inf], np.float32), scales.shape)
    _select(PagedCase([(tokens, 4000)], Hq=4, Hkv=2, page=32, seed=5), 32, (0, 1, 70), edit=edit)

    def queries(c, codes, scales):  # a query of zeros, one with an infinite and one with a NaN value
        c.q[0, 0:2] = 0
        c.q[-1, 0, 3] = 0x7F80
        c.q[-1, 2, 3] = 0x7FC0
    _select(PagedCase([(tokens, 4000)], Hq=4, Hkv=2, page=32, seed=6), 32, (1, 2, 10), edit=queries)


@pytest.mark.parametrize("tokens", [1, 40])
def test_codes_at_ties(gpu, tokens):
    """Queries with values at half, quarter and odd 254ths of the largest: which way a code rounds is part of the definition."""
    def queries(c, codes, scales):
        r = np.random.default_rng(8)
        top = np.float32(2.0) ** r.integers(-3, 4, (c.N, c.Hq, 1)).astype(np.float32) * r.integers(1, 255, (c.N, 1, 1)).astype(np.float32)
        c.q[:] = bf16_bits(np.where(r.random(c.q.shape) < 0.5, top / 2, top * r.choice(np.array([1, 0.25, 0.5, 0.75], np.float32), c.q.shape)))
        scales[:] = 1.0
    _select(PagedCase([(tokens, 4000)], Hq=4, Hkv=2, page=32, seed=12), 32, (0, 1, 12), edit=queries)


@pytest.mark.parametrize("tokens", [1, 40])
def test_selection_leaves_absent_pages_out(gpu, tokens):
    _select(PagedCase([(tokens, 900), (1, 500)], Hq=4, Hkv=2, page=32, seed=7, absent={(0, p) for p in range(3, 20)} | {(1, 2)}), 32, (1, 1, 12))


def test_selection_outside_the_envelope(gpu):
    c = PagedCase([(3, 400), (1, 900), (9, 10), (1, 100)], Hq=4, Hkv=2, page=32, seed=8)
    _select(c, 32, (1, 1, 4), envelope=(4, 500), only={0, 3})


def test_selection_graph(gpu):
    c = PagedCase([(1, 4000), (1, 900)], Hq=4, Hkv=2, page=32, seed=9)
    call, check, out = _select(c, 32, (1, 1, 8))
    s = Stream()
    with Graph(s) as g:
        call(s)
    for _ in range(3):
        out.upload(np.full((c.N, c.Hkv, 10), -77, np.int32))
        g.launch()
        s.synchronize()
        check()


@pytest.mark.parametrize("seqs", [[(1, 300)] * 5 + [(40, 100)] + [(0, 3)] * 60 + [(2, 64)] * 20])
def test_selection_of_many_sequences(gpu, seqs):
    _select(PagedCase(seqs, Hq=2, Hkv=1, page=32, seed=10), 32, (1, 1, 3))
