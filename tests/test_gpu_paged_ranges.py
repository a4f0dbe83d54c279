"""Paged attention where rows differ by many orders of magnitude: keys that a token does not see, or that hardly count,
cost the others no bits."""
import numpy as np
import pytest

from paged_bound import check_bound
from paged_case import PagedCase, bf16_bits, bf16_values

pytestmark = pytest.mark.gpu

CACHES = ["i8", "bf16"]
GEO = {"10-2-128": (10, 2, 128), "12-2-256": (12, 2, 256)}


def _grow(x, f):
    x[:] = bf16_bits(bf16_values(x) * np.float32(f))


def _run(c):
    d = c.upload()
    d.attend()
    check_bound(c, d.result())


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("size", [1e-4, 1e-6, 1e-7, 1e-8])
@pytest.mark.parametrize("first", ["absent pages", "zero rows", "zero rows of both signs"])
def test_small_values_behind_an_empty_tile(gpu, kv, geo, tokens, size, first):
    """The first key tile of a workgroup holds no value that could tell how large the others are."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        for x in c.v:
            _grow(x, size * (100 if kv == "i8" else 1))  # an INT8 value is at least its FP16 scale's smallest step
        if first == "zero rows":
            c.v[0][:256] = 0
        if first == "zero rows of both signs":
            c.v[0][:256] &= 0x8000
    absent = {(0, p) for p in range(16)} if first == "absent pages" else ()
    _run(PagedCase([(tokens, 400), (tokens, 30)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=30, absent=absent, edit=edit))


def _small_before_large(kv, geo, small):
    """First tokens see small values only; the tile that tells the size of the values holds ones of 1e3 too."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        _grow(c.v[0][:8], small)
        _grow(c.v[0][8:], 1e3)
    _run(PagedCase([(100, 0)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=31, edit=edit))


@pytest.mark.parametrize("geo", GEO)
def test_small_bf16_values_before_large_ones(gpu, geo):
    _small_before_large("bf16", geo, 1e-7)


@pytest.mark.parametrize("geo", GEO)
def test_small_int8_values_before_large_ones(gpu, geo):
    _small_before_large("i8", geo, 1e-4)


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 3, 90])
@pytest.mark.parametrize("small", [1.0, 1e-3, 1e-5])
def test_large_values_that_left_the_window(gpu, kv, geo, tokens, small):
    """Rows right before the window, in the window's first key chunk, hold values of 3e6; those that are seen are small."""
    Hq, Hkv, D = GEO[geo]
    h, w = 700, 50

    def edit(c):
        _grow(c.v[0], small)
        for r in (h - w, h - w - 1, h - w - 9):
            c.v[0][r] = bf16_bits(np.full(c.v[0][r].shape, 3e6, np.float32))
    _run(PagedCase([(tokens, h)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, window=w, sinks=3, seed=32, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [3, 90])
def test_large_values_of_later_tokens(gpu, kv, geo, tokens):
    """A later token of the chunk brings values of 3e6: earlier ones, whose values are 1e-3, do not see it."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        _grow(c.v[0], 1e-3)
        c.v[0][300 + tokens - 1] = bf16_bits(np.full(c.v[0][0].shape, 3e6, np.float32))
    _run(PagedCase([(tokens, 300)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=33, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 90])
def test_large_values_without_weight(gpu, kv, geo, tokens):
    """A key that is seen, but counts for less than 1e-20, has values of 3e6; the others have 1e-3."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        _grow(c.v[0], 1e-3)
        c.q[:, :, 1] = bf16_bits(np.float32(8.0))
        c.k[0][:, :, 1] = 0
        c.k[0][70, :, 1] = bf16_bits(np.float32(-100.0))
        c.v[0][70] = bf16_bits(np.full(c.v[0][70].shape, 3e6, np.float32))
    _run(PagedCase([(tokens, 100)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=34, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 3, 90])
def test_large_keys_that_left_the_window(gpu, kv, geo, tokens):
    """As for values: keys of 6e6 that are not seen, next to keys of 1e-3 under queries of 1e3."""
    Hq, Hkv, D = GEO[geo]
    h, w = 700, 50

    def edit(c):
        _grow(c.k[0], 1e-3)
        _grow(c.q, 1e3)
        for r in (h - w, h - w - 1, h - w - 9):
            c.k[0][r] = bf16_bits(np.full(c.k[0][r].shape, 6e6, np.float32))
    _run(PagedCase([(tokens, h)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, window=w, seed=35, edit=edit))


@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 3, 90])
@pytest.mark.parametrize("size", [1e33, 1e36, 5e37])
@pytest.mark.parametrize("rows", ["all", "late"])
def test_values_near_the_top_of_bf16(gpu, geo, tokens, size, rows):
    """Weighted means of finite values are finite."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        x = bf16_values(c.v[0]).astype(np.float64)
        x = np.clip(x * (size / 2), -3e38, 3e38)  # a normal value times 2 in one dimension of 32
        part = slice(0 if rows == "all" else 350, None)
        c.v[0][part] = bf16_bits(x[part].astype(np.float32))
    _run(PagedCase([(tokens, 500), (2, 20)], Hq=Hq, Hkv=Hkv, D=D, kv="bf16", seed=36, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("size", [1e-4, 1e3, 3e4, 2e5])
def test_size_of_values(gpu, kv, geo, tokens, size):
    Hq, Hkv, D = GEO[geo]
    _run(PagedCase([(tokens, 400)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=37, edit=lambda c: _grow(c.v[0], size)))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 90])
@pytest.mark.parametrize("size", [1e3, 2e5])
@pytest.mark.parametrize("sign", [1, -1])
def test_one_key_outgrows_the_others(gpu, kv, geo, tokens, size, sign):
    """A key of `size` times the others takes all the weight (or none) of the tokens that see it."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        c.q[:, :, 1] = bf16_bits(np.float32(16.0 * sign))
        c.k[0][390] = bf16_bits(np.float32(0.01) * bf16_values(c.k[0][390]))
        c.k[0][390, :, 1] = bf16_bits(np.float32(1.0))
        _grow(c.k[0][390], size)
    _run(PagedCase([(tokens, 400)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=38, edit=edit))


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 3, 90])
@pytest.mark.parametrize("size", [1e5, 1e6, 1e7, 1e9])
def test_large_scores(gpu, kv, geo, tokens, size):
    """Scores of about `size`: one key takes all the weight, and its values are the result."""
    Hq, Hkv, D = GEO[geo]

    def edit(c):
        _grow(c.q, size / 1e3)
        _grow(c.k[0], 1e3)
    _run(PagedCase([(tokens, 400)], Hq=Hq, Hkv=Hkv, D=D, kv=kv, seed=39, edit=edit))


@pytest.mark.parametrize("geo", GEO)
@pytest.mark.parametrize("tokens", [1, 3, 90])
@pytest.mark.parametrize("infinite", [False, True])
def test_values_near_the_bottom_of_bf16(gpu, geo, tokens, infinite):
    """Values of 1e-33 behind larger ones in tiles of their own, with and without an infinite one that no token sees."""
    Hq, Hkv, D = GEO[geo]
    h, w = 700, 190

    def edit(c):
        _grow(c.v[0], 1e-33)
        _grow(c.v[0][:520], 1e20)
        if infinite:
            c.v[0][h - w] = 0x7F80
    _run(PagedCase([(tokens, h), (2, 20)], Hq=Hq, Hkv=Hkv, D=D, kv="bf16", window=w, seed=29, edit=edit))
