"""The error bounds of the paged-attention tests are tight enough to see a mistake: zeros, doubled values, a lost
key and a lost page planted in the 64-bit results fall outside (no GPU)."""
import numpy as np
import pytest

from paged_bound import borders, bound, needles
from paged_case import PagedCase, bf16_bits, bf16_values

CACHES = ["i8", "bf16"]


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("size", [1e-7, 1.0, 2e5])
@pytest.mark.parametrize("tokens", [1, 3])
def test_zeros_are_outside(kv, size, tokens):
    def edit(c):
        c.v[0][:] = bf16_bits(bf16_values(c.v[0]) * np.float32(size * (100 if kv == "i8" and size < 1 else 1)))
    c = PagedCase([(tokens, 400)], Hq=4, Hkv=2, kv=kv, seed=1, edit=edit)
    for _, _, o, tol in bound(c):
        assert (np.abs(o) > tol).mean() > 0.9 and (np.abs(2 * o) > tol).mean() > 0.9


@pytest.mark.parametrize("kv", CACHES)
@pytest.mark.parametrize("D", [128, 256])
def test_a_lost_key_is_outside(kv, D):
    """Every needle of a long history, dropped by itself; and the page of one."""
    t, h = 2, 2998
    rows = [x for x in dict.fromkeys(borders(t, h)) if 0 <= x < t + h][1::4]
    c = PagedCase([(t, h)], Hq=4, Hkv=2, D=D, kv=kv, seed=2, edit=lambda c: needles(c, 0, rows))
    whole = {(n, hh): (o, tol) for n, hh, o, tol in bound(c)}
    for lost in [[x] for x in rows] + [range(rows[0] // 16 * 16, rows[0] // 16 * 16 + 16)]:
        for n, hh, o, _ in bound(c, dropped=lost):
            if min(lost) <= h + n:
                ref, tol = whole[n, hh]
                assert (np.abs(o - ref) > tol).any(), (list(lost), n, hh)
