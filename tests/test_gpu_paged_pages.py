"""The pages of a paged cache: copies, handing out, giving back, sharing and moving together, against a table kept entry by entry."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.device import DeviceArray, Graph, Stream, synchronize
from paged_blocks_case import Pages
from paged_case import PagedCase, Strided

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


class Pool:
    """A table of B sequences whose lengths are given, in random pages; the same on the GPU."""

    def __init__(self, pages, page, B, width, lengths, seed=0, pad=8):
        r = np.random.default_rng(seed)
        self.page = page
        table = np.full((B, width), -1, np.int32)
        order = r.permutation(pages)
        at = 0
        for b, n in enumerate(lengths):
            k = min(-(-n // page), width)
            table[b, :k] = order[at:at + k]
            at += k
        refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
        self.ref = Pages(table, refs, page)
        self.history = np.array(list(lengths) + [0] * (B - len(lengths)), np.int32)
        self.d_table = Strided(na.I32, (width, B), pad).upload(table)
        self.d_refs = dev(refs)
        self.d_history = dev(self.history)
        self.args = (self.d_table.t, self.d_refs.tensor())

    def check(self):
        synchronize()
        table = self.d_table.numpy(np.int32).reshape(self.ref.table.shape)
        assert (table == self.ref.table).all()
        refs = self.d_refs.numpy()
        assert (refs == self.ref.refs).all()
        held = table[(table >= 0) & (table < len(refs))]
        assert (np.bincount(held, minlength=len(refs)) == refs).all(), "counts that are not the table's"

    def reserve(self, tokens, history=None):
        starts = np.concatenate(([0], np.cumsum(tokens))).astype(np.int32)
        h = self.history if history is None else np.asarray(history, np.int32)
        out = dev(np.full(len(h), -7))
        ops.paged_pages_reserve(*self.args, dev(starts).tensor(), dev(h).tensor(), self.page, out.tensor())
        got = out.numpy()
        want = self.ref.reserve(starts, h)
        assert (got == want).all(), (got, want)
        self.check()
        return got

    def release(self, sequences, keep):
        ops.paged_pages_release(*self.args, dev(sequences).tensor(), dev(keep).tensor(), self.page)
        self.ref.release(sequences, keep)
        self.check()

    def fork(self, parents, children):
        src, dst = dev(np.full(len(parents), -7)), dev(np.full(len(parents), -7))
        self.d_history.upload(self.history)
        ops.paged_pages_fork(*self.args, dev(parents).tensor(), dev(children).tensor(), self.d_history.tensor(), self.page, src.tensor(), dst.tensor())
        self.history, s, d = self.ref.fork(list(parents), list(children), self.history)
        assert (src.numpy() == s).all() and (dst.numpy() == d).all()
        assert (self.d_history.numpy() == self.history).all()
        self.check()
        return s, d

    def compact(self, n):
        src, dst, moved = dev(np.full(n, -7)), dev(np.full(n, -7)), dev([-7])
        ops.paged_pages_compact(*self.args, src.tensor(), dst.tensor(), moved.tensor())
        s, d, m = self.ref.compact(n)
        assert (src.numpy() == s).all() and (dst.numpy() == d).all() and moved.numpy()[0] == m
        self.check()
        return m


@pytest.mark.parametrize("pages,page,B,width", [(40, 16, 5, 9), (64, 32, 3, 20), (1000, 16, 33, 31), (4097, 64, 64, 70), (70000, 16, 1024, 60)])
def test_reserve(gpu, pages, page, B, width):
    """Single tokens, prompts of odd lengths, sequences without tokens, until the pool ends."""
    r = np.random.default_rng(pages)
    p = Pool(pages, page, B, width, r.integers(0, min(3 * page, pages * page // B // 2), B), seed=pages)
    for step in range(6):
        tokens = r.integers(0, 2 if step % 2 == 0 else width * page // 4, B)
        got = p.reserve(tokens)
        p.history = p.history + got
    p.reserve(np.full(B, width * page))  # past the table and the pool


def test_reserve_from_any_history(gpu):
    """Negative histories, histories past the table, holes in the table (pages that left a window) that stay holes."""
    p = Pool(50, 16, 6, 8, [128, 40, 0, 100, 5, 0], seed=1)
    p.release([0], [0])
    p.reserve([1, 20, 0, 3, 16, 1], history=[40, 40, 7, -1, 500, 127])
    p.reserve([1] * 6, history=[2**31 - 1, 60, 0, 103, 128, 128])


def test_reserve_refuses_no_entry_outside(gpu):
    """starts that descend or promise more tokens than there are: what they name is left out or cut at the table's end."""
    p = Pool(30, 16, 4, 6, [20, 0, 50, 16], seed=2)
    out = dev(np.zeros(4))
    starts, h = np.array([5, 3, 2**30, 2**30 + 9, 2**31 - 1], np.int32), np.array([20, 0, 50, 16], np.int32)
    ops.paged_pages_reserve(*p.args, dev(starts).tensor(), dev(h).tensor(), 16, out.tensor())
    assert (out.numpy() == p.ref.reserve(starts, h)).all()
    p.check()


@pytest.mark.parametrize("pages,page,B,width", [(40, 16, 5, 9), (4097, 64, 64, 70), (524288, 16, 1000, 500)])
def test_release(gpu, pages, page, B, width):
    r = np.random.default_rng(B)
    p = Pool(pages, page, B, width, r.integers(0, min(width * page, pages * page // B), B), seed=3)
    some = r.permutation(B)[:B // 2]
    p.release(some, r.integers(0, width * page, len(some)))
    p.release(some, np.zeros(len(some)))
    p.release([0, 0, B - 1, B, -1, 2, 2**31 - 1, 1], [17, 40, 0, 0, 0, -5, 0, 2**31 - 1])


@pytest.mark.parametrize("pages,page,B,width", [(40, 16, 6, 9), (4097, 64, 64, 70), (300000, 16, 1024, 64)])
def test_fork(gpu, pages, page, B, width):
    """Whole and unfinished last pages, answers that held something before, until no page is left."""
    r = np.random.default_rng(pages)
    lengths = np.concatenate((r.integers(0, min(width * page, pages * page // B), B // 2), np.zeros(B - B // 2, np.int64)))
    lengths[0], lengths[1] = 2 * page, 0
    p = Pool(pages, page, B, width, lengths, seed=4)
    for step in range(3):
        n = B - B // 2
        p.fork(r.integers(0, B // 2, n), B // 2 + r.permutation(n))
    p.release(np.arange(B // 2), np.zeros(B // 2))  # the answers keep their pages
    p.compact(pages)


def test_fork_of_pairs_that_do_not_fit(gpu):
    """A child that is a parent, one that two pairs name, sequences outside the table, a pair of one sequence."""
    p = Pool(60, 16, 8, 6, [20, 33, 16, 7, 90, 1], seed=5)
    p.fork([0, 1, 0, 4, 3, 3, 9, 0, -1, 2], [6, 0, 6, 7, 3, 5, 5, 8, 5, -3])
    p.fork([4], [0])
    small = Pool(6, 16, 6, 6, [20, 33], seed=6)  # one page is free
    small.fork([0, 1, 0], [2, 3, 4])
    assert list(small.history[2:5]) == [20, 32, 16]


@pytest.mark.parametrize("pages,B,width", [(40, 5, 9), (64, 8, 8), (4097, 64, 70), (524288, 1000, 500)])
@pytest.mark.parametrize("most", [1, 7, None])
def test_compact(gpu, pages, B, width, most):
    r = np.random.default_rng(pages)
    p = Pool(pages, 16, B, width, r.integers(0, min(width * 16, pages * 16 // B), B), seed=7)
    p.fork([0] * (B // 5), list(range(B - B // 5, B)))
    p.release(np.arange(1, B - B // 5, 2), np.zeros(len(np.arange(1, B - B // 5, 2))))
    p.compact(most or pages)
    if most is None:
        used = np.flatnonzero(p.ref.refs)
        assert len(used) == 0 or used[-1] == len(used) - 1
        assert p.compact(pages) == 0


def test_compact_of_none_and_all(gpu):
    p = Pool(64, 16, 4, 16, [], seed=8)
    assert p.compact(64) == 0
    p = Pool(64, 16, 4, 16, [256, 256, 256, 256], seed=8)
    assert p.compact(64) == 0
    p = Pool(130, 16, 1, 1, [3], seed=11)
    p.compact(5)


GEO = {"8-128": (8, 128), "2-256": (2, 256), "1-128": (1, 128), "3-128": (3, 128)}


@pytest.mark.parametrize("kv", ["i8", "bf16"])
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("page,block", [(16, 0), (32, 32), (128, 64), (256, 32)])
def test_copy(gpu, kv, geo, page, block):
    """Pages with strides of their own, their block means, pairs of no page; everything else stays."""
    Hkv, D = GEO[geo]
    c = PagedCase([(3, 9 * page)], Hq=Hkv, Hkv=Hkv, D=D, kv=kv, page=page, seed=page, page_pad=48, spare=6)
    d = c.upload()
    before = d.pool()
    r = np.random.default_rng(block)
    src, dst = np.array([0, 4, 9, -1, 2, 3, 2**31 - 1, 7, 5, -(2**31)]), np.array([1, 2, 3, 8, -1, c.pages, 8, 7, 6, 8])
    blocks = None
    if block:
        codes, scales = Strided(na.I8, (D, page // block, Hkv, c.pages), 32), Strided(na.FP32, (page // block, Hkv, c.pages), 4)
        scales.t.ne[3] = 1
        hc, hs = r.integers(-127, 128, (c.pages, Hkv, page // block, D)).astype(np.int8), r.random((c.pages, Hkv, page // block)).astype(np.float32)
        codes.upload(hc)
        scales.upload(hs)
        blocks = na.PagedBlockView()
        blocks.codes, blocks.scales, blocks.block_size = codes.t, scales.t, block
        before = [*before, hc, hs]
    # page 2 is written from 4, so it is not read
    ops.paged_kv_copy_pages(d.view, blocks, dev(src).tensor(), dev(dst).tensor())
    synchronize()
    after = d.pool()
    if block:
        after = [*after, codes.numpy(np.int8).reshape(hc.shape), scales.numpy(np.float32).reshape(hs.shape)]
    for x, y in zip(before, after):
        want = x.copy()
        for a, b in ((0, 1), (4, 2), (9, 3), (5, 6)):
            want[b] = x[a]
        assert (want.view(np.uint8) == y.view(np.uint8)).all()


def test_copy_of_many_pages(gpu):
    c = PagedCase([(1, 20000)], Hq=8, Hkv=8, kv="i8", page=16, seed=1, spare=1300)
    d = c.upload()
    before = d.pool()
    used = c.table[0, :1250]
    spare = np.setdiff1d(np.arange(c.pages), c.table[0])[:1250]
    ops.paged_kv_copy_pages(d.view, None, dev(used).tensor(), dev(spare).tensor())
    synchronize()
    for x, y in zip(before, d.pool()):
        assert (y[spare] == x[used]).all() and (np.delete(y, spare, 0) == np.delete(x, spare, 0)).all()


def test_a_scheduler_step_as_a_graph(gpu):
    """Give back, move together, hand out: captured once, replayed on new lists."""
    r = np.random.default_rng(9)
    p = Pool(500, 16, 12, 30, r.integers(20, 400, 12), seed=9)
    gone, keep, starts, hist = dev([0] * 4), dev([0] * 4), dev([0] * 13), dev([0] * 12)
    src, dst, moved, granted = dev([0] * 250), dev([0] * 250), dev([0]), dev([0] * 12)

    def step(stream):
        ops.paged_pages_release(*p.args, gone.tensor(), keep.tensor(), 16, stream)
        ops.paged_pages_compact(*p.args, src.tensor(), dst.tensor(), moved.tensor(), stream)
        ops.paged_pages_reserve(*p.args, starts.tensor(), hist.tensor(), 16, granted.tensor(), stream)
    s = Stream()
    with Graph(s) as g:
        step(s)
    for _ in range(4):
        ends = r.permutation(12)[:4]
        tokens = np.zeros(12, np.int64)
        tokens[ends] = r.integers(1, 400, 4)
        gone.upload(ends.astype(np.int32))
        starts.upload(np.concatenate(([0], np.cumsum(tokens))).astype(np.int32))
        synchronize()
        g.launch()
        s.synchronize()
        p.ref.release(ends, [0] * 4)
        a, b, m = p.ref.compact(250)
        assert (src.numpy() == a).all() and (dst.numpy() == b).all() and moved.numpy()[0] == m
        assert (granted.numpy() == p.ref.reserve(np.concatenate(([0], np.cumsum(tokens))), np.zeros(12))).all()
        p.check()
