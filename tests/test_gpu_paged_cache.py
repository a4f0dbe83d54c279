"""Rows of a paged cache: append and read back, bit for bit against the codec in numpy."""
import numpy as np
import pytest

import ninfer_amd as na
from ninfer_amd.device import synchronize
from paged_case import PagedCase, bf16_bits, quantize

pytestmark = pytest.mark.gpu

GEO = [(8, 128), (4, 256), (2, 256), (1, 128), (3, 128)]
SEQS = [[(1, 0)], [(1, 517)], [(5, 30), (0, 40), (17, 0), (1, 15), (33, 16)], [(0, 3), (200, 100)]]


def _same(got, want):
    for g, w in zip(got, want, strict=True):
        assert np.array_equal(g, w)


@pytest.mark.parametrize("kv", ["i8", "bf16"])
@pytest.mark.parametrize("Hkv,D", GEO)
@pytest.mark.parametrize("i", range(len(SEQS)))
def test_append(gpu, kv, Hkv, D, i):
    c = PagedCase(SEQS[i], Hq=Hkv, Hkv=Hkv, D=D, kv=kv, page=16 << (i % 3), seed=i, lead=i % 2, tail=3, pad=32 * (i % 2), page_pad=48 * (i % 2))
    d = c.upload(c.planes(new_rows=False))
    d.append()
    synchronize()
    _same(d.pool(), c.planes())


@pytest.mark.parametrize("kv", ["i8", "bf16"])
def test_append_drops_rows_without_a_page(gpu, kv):
    # absent pages in the middle, and rows past the table's end
    c = PagedCase([(40, 10), (30, 40)], Hq=2, Hkv=2, kv=kv, page=16, seed=3, absent={(0, 1), (1, 3)}, max_pages=4, tail=1)
    d = c.upload(c.planes(new_rows=False))
    d.append()
    synchronize()
    _same(d.pool(), c.planes())


def test_append_of_extreme_values(gpu):
    """Zeros, signed zeros, one large value, tiny and huge ones, and a group whose scale overflows FP16."""
    def edit(c):
        x = c.k[0][20:]
        x[0] = 0
        x[1] = 0x8000
        x[2, :, 5] = bf16_bits(np.float32(3e4))
        x[3] = bf16_bits(np.float32(1e-8))
        x[4] = bf16_bits(np.float32(8.2e6))
        x[5, 0, :64] = bf16_bits(np.float32(1e9))
    c = PagedCase([(6, 20)], Hq=2, Hkv=2, seed=9, edit=edit)
    d = c.upload(c.planes(new_rows=False))
    d.append()
    synchronize()
    got, want = d.pool(), c.planes()
    _same(got[1:], want[1:])
    s = want[2].view(np.float16)
    fine = np.repeat(np.isfinite(s), 64, -1)
    assert np.array_equal(got[0][fine], want[0][fine])
    assert (got[0][np.repeat(np.isinf(s), 64, -1)] == 0).all()


@pytest.mark.parametrize("dtype", [na.BF16, na.FP32])
@pytest.mark.parametrize("kv", ["i8", "bf16"])
@pytest.mark.parametrize("Hkv,D", GEO)
def test_read(gpu, kv, Hkv, D, dtype):
    c = PagedCase([(7, 60), (0, 9), (90, 40), (1, 0)], Hq=Hkv, Hkv=Hkv, D=D, kv=kv, page=32, seed=5, absent={(2, 2)}, lead=2, tail=2, pad=16)
    first = [3, 0, 17, 0]
    got = c.upload().read(first, dtype)
    for plane in range(2):
        want = np.full((c.N, Hkv, D), np.float32(0)).astype(np.float32)
        raw = np.full(want.shape, 0xCDCDCDCD, np.uint32).view(np.float32) if dtype == na.FP32 else np.full(want.shape, 0xCDCD, np.uint16)
        for b, (t, _) in enumerate(c.seqs):
            rows = first[b] + np.arange(t)
            x = c.stored(b)[plane].astype(np.float32)
            ok = c.present(b, rows)
            vals = np.zeros((t, Hkv, D), np.float32)
            vals[ok] = x[rows[ok]]
            raw[c.starts[b]:c.starts[b] + t] = vals if dtype == na.FP32 else bf16_bits(vals)
        g, w = (got[plane].view(np.uint32), raw.view(np.uint32)) if dtype == na.FP32 else (got[plane], raw)
        assert np.array_equal(g, w)


def test_written_rows_read_back(gpu):
    c = PagedCase([(300, 77), (1, 5)], Hq=4, Hkv=4, D=256, page=64, seed=8)
    d = c.upload(c.planes(new_rows=False))
    d.append()
    got = d.read(c.history)
    for plane, x in enumerate((c.k_new, c.v_new)):
        codes, s = quantize(x)
        want = codes.reshape(*codes.shape[:-1], -1, 64).astype(np.float32) * s.view(np.float16).astype(np.float32)[..., None]
        assert np.array_equal(got[plane], want.reshape(codes.shape))


def test_sequences_outside_the_batch_rules(gpu):
    """Device scalars that make no sense write nothing: a negative history, starts that fall, tokens past N."""
    c = PagedCase([(4, 20), (4, 20), (4, 20)], Hq=1, Hkv=1, seed=2)
    before = c.planes(new_rows=False)
    d = c.upload(before)
    d.history.upload(np.array([-5, 20, 2**31 - 1], np.int32))
    d.starts.upload(np.array([0, 4, 2, 2**31 - 1], np.int32))
    d.append()
    synchronize()
    got = d.pool()
    for b in (0, 2):
        for s in c.table[b]:
            if 0 <= s < c.pages:
                for g, w in zip(got, before):
                    assert np.array_equal(g[s], w[s])
