"""Refusals of the paged-cache ops: host validation only, no launch."""
import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.kv_cache import PagedKVCacheLayer

FAKE = 0x10000


def T(dtype, *shape, data=FAKE, nb=None):
    t = na.Tensor.make(data, dtype, shape)
    for i, b in (nb or {}).items():
        t.nb[i] = b
    return t


class Ws:
    def __init__(self, ptr=FAKE, nbytes=1 << 40):
        self.ptr, self.nbytes = ptr, nbytes


def view(D=128, page=16, H=2, pages=8, B=3, max_pages=4, kv="i8", **kw):
    v = na.PagedKVLayerView()
    code = na.I8 if kv == "i8" else na.BF16
    v.k, v.v = T(code, D, page, H, pages), T(code, D, page, H, pages)
    if kv == "i8":
        v.k_scale, v.v_scale = T(na.FP16, D // 64, page, H, pages), T(na.FP16, D // 64, page, H, pages)
    v.page_table = T(na.I32, max_pages, B)
    v.page_size, v.num_kv_heads, v.head_dim, v.dtype, v.quant_group = page, H, D, code, 64 if kv == "i8" else 0
    for k, x in kw.items():
        setattr(v, k, x)
    return v


BAD_VIEWS = {
    "dtype": (dict(dtype=na.FP16), ValueError),
    "group": (dict(quant_group=32), ValueError),
    "page size": (dict(page=24), ValueError),
    "small page": (dict(page=8), ValueError),
    "large page": (dict(page=8192), ValueError),
    "page size of the planes": (dict(page_size=32), ValueError),
    "heads of the planes": (dict(num_kv_heads=4), ValueError),
    "head_dim 64": (dict(D=64), NotImplementedError),
    "head_dim 100": (dict(head_dim=100), ValueError),
    "k dtype": (dict(k=T(na.BF16, 128, 16, 2, 8)), ValueError),
    "v pages": (dict(v=T(na.I8, 128, 16, 2, 9)), ValueError),
    "k null": (dict(k=T(na.I8, 128, 16, 2, 8, data=0)), ValueError),
    "k alignment": (dict(k=T(na.I8, 128, 16, 2, 8, data=FAKE + 8)), ValueError),
    "scale dtype": (dict(k_scale=T(na.BF16, 2, 16, 2, 8)), ValueError),
    "scale null": (dict(v_scale=T(na.FP16, 2, 16, 2, 8, data=0)), ValueError),
    "row stride": (dict(k=T(na.I8, 128, 16, 2, 8, nb={1: 256})), ValueError),
    "head stride": (dict(k=T(na.I8, 128, 16, 2, 8, nb={2: 4096})), ValueError),
    "page stride too small": (dict(k=T(na.I8, 128, 16, 2, 8, nb={3: 4080})), ValueError),
    "page stride odd": (dict(k=T(na.I8, 128, 16, 2, 8, nb={3: 4104})), ValueError),
    "table dtype": (dict(page_table=T(na.I64, 4, 3)), ValueError),
    "table shape": (dict(page_table=T(na.I32, 4, 3, 2)), ValueError),
    "table null": (dict(page_table=T(na.I32, 4, 3, data=0)), ValueError),
    "table stride": (dict(page_table=T(na.I32, 4, 3, nb={1: 12})), ValueError),
    "table too long": (dict(max_pages=1 << 28), OverflowError),
    "batch": (dict(B=1025), NotImplementedError),
    "heads": (dict(H=1025), NotImplementedError),
    "page of 2 GiB": (dict(H=1024, page=4096, D=256), NotImplementedError),
    "bf16 with scales": (dict(kv="bf16", k_scale=T(na.FP16, 2, 16, 2, 8)), ValueError),
    "bf16 with a group": (dict(kv="bf16", quant_group=64), ValueError),
}


def _ops(v, B=None):
    """Every op on an otherwise right call (N = 5 packed tokens)."""
    B = v.page_table.ne[1] if B is None else B
    H, D = 2, v.head_dim if v.head_dim in (128, 256) else 128
    k, f = T(na.BF16, D, H, 5), T(na.FP32, D, H, 5)
    starts, hist = T(na.I32, B + 1), T(na.I32, B)
    yield lambda: ops.paged_kv_append(k, k, starts, hist, v)
    yield lambda: ops.paged_kv_read(v, starts, hist, f, f)
    yield lambda: ops.paged_attention(T(na.BF16, D, 8, 5), starts, hist, 0.1, (0, 0), v, (5, 32), Ws(), T(na.BF16, D, 8, 5))


@pytest.mark.parametrize("name", BAD_VIEWS)
def test_views(name):
    kw, error = BAD_VIEWS[name]
    for call in _ops(view(**kw)):
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("what,t", [
    ("k", T(na.FP16, 128, 2, 5)), ("k", T(na.BF16, 128, 3, 5)), ("k", T(na.BF16, 256, 2, 5)), ("k", T(na.BF16, 128, 2, 0)),
    ("k", T(na.BF16, 128, 2, 5, data=0)), ("k", T(na.BF16, 128, 2, 5, data=FAKE + 2)), ("k", T(na.BF16, 128, 2, 5, nb={2: 256})),
    ("k", T(na.BF16, 128, 2, 5, nb={2: 520})), ("k", T(na.BF16, 128, 2, 5, nb={1: 512})), ("k", T(na.BF16, 128, 2, 5, 2)), ("k", None),
    ("v", T(na.BF16, 128, 2, 4)), ("v", None),
    ("starts", T(na.I32, 3)), ("starts", T(na.I64, 4)), ("starts", T(na.I32, 4, data=0)), ("starts", None),
    ("history", T(na.I32, 4)), ("history", T(na.FP32, 3)), ("history", T(na.I32, 3, 2)), ("history", None),
])
def test_append_arguments(what, t):
    a = dict(k=T(na.BF16, 128, 2, 5), v=T(na.BF16, 128, 2, 5), starts=T(na.I32, 4), history=T(na.I32, 3))
    a[what] = t
    with pytest.raises(ValueError):
        ops.paged_kv_append(a["k"], a["v"], a["starts"], a["history"], view())
    if what in ("k", "v"):  # the same rules for the tensors that are read into
        if what == "k" and t is not None and t.dtype == na.FP16:
            t.dtype = na.I32
        with pytest.raises(ValueError):
            ops.paged_kv_read(view(), a["starts"], a["history"], a["k"], a["v"])


def test_read_types_agree():
    with pytest.raises(ValueError):
        ops.paged_kv_read(view(), T(na.I32, 4), T(na.I32, 3), T(na.BF16, 128, 2, 5), T(na.FP32, 128, 2, 5))


Q = T(na.BF16, 128, 8, 5)


@pytest.mark.parametrize("kw,error", [
    (dict(q=T(na.FP32, 128, 8, 5)), ValueError), (dict(q=T(na.BF16, 128, 7, 5)), ValueError), (dict(q=T(na.BF16, 256, 8, 5)), ValueError),
    (dict(q=None), ValueError), (dict(out=None), ValueError), (dict(out=T(na.FP32, 128, 8, 5)), ValueError),
    (dict(out=T(na.BF16, 128, 8, 4)), ValueError), (dict(out=T(na.BF16, 128, 8, 5, nb={2: 2056})), ValueError),
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=float("nan")), ValueError), (dict(scale=float("inf")), ValueError), (dict(scale=2.0**-41), ValueError), (dict(scale=2.0**41), ValueError),
    (dict(envelope=(0, 32)), ValueError), (dict(envelope=(33, 32)), ValueError), (dict(envelope=(5, 65)), ValueError),
    (dict(envelope=(5, (1 << 23) + 1)), NotImplementedError), (dict(envelope=(5, 1 << 31)), OverflowError), (dict(window=(1 << 31, 0)), OverflowError), (dict(window=(0, 4)), ValueError),
    (dict(ws=Ws(nbytes=0)), ValueError), (dict(ws=Ws(ptr=FAKE + 16)), ValueError), (dict(ws=None), ValueError),
])
def test_attention_arguments(kw, error):
    a = dict(q=Q, out=T(na.BF16, 128, 8, 5), scale=0.1, envelope=(5, 64), window=(0, 0), ws=Ws())
    a.update(kw)
    v = view()
    if "ws" in kw:  # a plan that needs a workspace
        v = view(max_pages=4096, pages=4096)
        a["envelope"] = (5, 65536)
    if error is NotImplementedError:
        v = view(max_pages=1 << 20)
    with pytest.raises(error):
        ops.paged_attention(a["q"], T(na.I32, 4), T(na.I32, 3), a["scale"], a["window"], v, a["envelope"], a["ws"], a["out"])


def test_workspace_query():
    q = ops.paged_attention_workspace_bytes
    assert q(40, 8, 128, 1, 1, (1, 65536)) > 0
    # what the op refuses needs none
    for bad in [(40, 7, 128, 1, 1, (1, 64)), (0, 8, 128, 1, 1, (1, 64)), (40, 8, 64, 1, 1, (1, 64)), (40, 8, 128, 0, 1, (1, 64)),
                (40, 8, 128, 1, 0, (1, 64)), (40, 8, 128, 1, 1025, (1, 64)), (40, 8, 128, 1, 1, (0, 64)), (40, 8, 128, 1, 1, (65, 64)),
                (40, 8, 128, 1, 1, (1, 1 << 31)), (40, 8, 128, 1, 1, (1, (1 << 23) + 1)), (40, 8, 128, 1 << 27, 1, (1, 64))]:
        assert q(*bad) == 0
    # a window bounds the rows that are split
    assert q(40, 8, 128, 1, 1, (1, 1 << 20), (64, 4)) <= q(40, 8, 128, 1, 1, (1, 1 << 20))


@pytest.mark.parametrize("kw", [dict(page_size=24), dict(page_size=8), dict(pages=0), dict(batch=0), dict(max_pages=0), dict(num_kv_heads=0),
                                dict(head_dim=100), dict(dtype=na.FP16)])
def test_owner_refuses(kw):
    a = dict(pages=4, page_size=16, num_kv_heads=2, head_dim=128, batch=1, max_pages=2, dtype=na.I8)
    a.update(kw)
    with pytest.raises(ValueError):
        PagedKVCacheLayer(**a)
