"""Refusals of the operators around a paged cache (head norms with rotation, blocks, pages), on the host; their C++ layer."""
import shutil
import subprocess
from pathlib import Path

import pytest

import ninfer_amd as na
from ninfer_amd import ops
from ninfer_amd.kv_cache import PagedKVCacheLayer
from test_paged_cpu import BAD_VIEWS, FAKE, T, Ws, view

ROOT = Path(__file__).resolve().parent.parent


def blocks(D=128, per=2, H=2, pages=8, size=32, **kw):
    b = na.PagedBlockView()
    b.codes, b.scales, b.block_size = T(na.I8, D, per, H, pages), T(na.FP32, per, H, pages), size
    for k, x in kw.items():
        setattr(b, k, x)
    return b


# ---- calls that are right but for what a test changes (N = 5 packed tokens, B = 3, pages of 64 rows, blocks of 32)

def rope(**kw):
    a = dict(q=T(na.BF16, 128, 8, 5), k=T(na.BF16, 128, 2, 5), qw=T(na.BF16, 128), kw=T(na.FP32, 128), pos=T(na.I32, 5), freq=T(na.FP32, 64),
             norm=(1e-6, 0.0, False), qo=T(na.BF16, 128, 8, 5, data=2 * FAKE), ko=T(na.BF16, 128, 2, 5, data=3 * FAKE))
    a.update(kw)
    ops.qk_norm_rope(a["q"], a["k"], a["qw"], a["kw"], a["pos"], a["freq"], a["norm"], a["qo"], a["ko"])


def rope_append(**kw):
    a = dict(q=T(na.BF16, 128, 8, 5), k=T(na.BF16, 128, 2, 5), v=T(na.BF16, 128, 2, 5), qw=T(na.BF16, 128), kw=T(na.FP32, 128), starts=T(na.I32, 4),
             history=T(na.I32, 3), freq=T(na.FP32, 64), norm=(1e-6, 0.0, False), cache=view(page=64), qo=T(na.BF16, 128, 8, 5, data=2 * FAKE))
    a.update(kw)
    ops.paged_qk_norm_rope_append(a["q"], a["k"], a["v"], a["qw"], a["kw"], a["starts"], a["history"], a["freq"], a["norm"], a["cache"], a["qo"])


def update(**kw):
    a = dict(cache=view(page=64), starts=T(na.I32, 4), history=T(na.I32, 3), tokens=5, blocks=blocks())
    a.update(kw)
    ops.paged_block_update(a["cache"], a["starts"], a["history"], a["tokens"], a["blocks"])


def select(**kw):
    a = dict(q=T(na.BF16, 128, 8, 5), starts=T(na.I32, 4), history=T(na.I32, 3), table=T(na.I32, 4, 3), page=64, blocks=blocks(), pick=(1, 2, 3),
             env=(5, 256), ws=Ws(), out=T(na.I32, 6, 2, 5))
    a.update(kw)
    ops.paged_block_select(a["q"], a["starts"], a["history"], a["table"], a["page"], a["blocks"], a["pick"], a["env"], a["ws"], a["out"])


def attend(**kw):
    a = dict(q=T(na.BF16, 128, 8, 5), starts=T(na.I32, 4), history=T(na.I32, 3), scale=0.1, lists=T(na.I32, 6, 2, 5), size=32, cache=view(page=64),
             env=(5, 256), ws=Ws(), out=T(na.BF16, 128, 8, 5))
    a.update(kw)
    ops.paged_sparse_attention(a["q"], a["starts"], a["history"], a["scale"], a["lists"], a["size"], a["cache"], a["env"], a["ws"], a["out"])


def copy(**kw):
    a = dict(cache=view(page=64), blocks=blocks(), src=T(na.I32, 7), dst=T(na.I32, 7))
    a.update(kw)
    ops.paged_kv_copy_pages(a["cache"], a["blocks"], a["src"], a["dst"])


TABLE = dict(table=T(na.I32, 4, 3), refs=T(na.I32, 8), page=64)


def reserve(**kw):
    a = dict(TABLE, starts=T(na.I32, 4), history=T(na.I32, 3), granted=T(na.I32, 3))
    a.update(kw)
    ops.paged_pages_reserve(a["table"], a["refs"], a["starts"], a["history"], a["page"], a["granted"])


def release(**kw):
    a = dict(TABLE, sequences=T(na.I32, 2), keep=T(na.I32, 2))
    a.update(kw)
    ops.paged_pages_release(a["table"], a["refs"], a["sequences"], a["keep"], a["page"])


def fork(**kw):
    a = dict(TABLE, parents=T(na.I32, 2), children=T(na.I32, 2), history=T(na.I32, 3), src=T(na.I32, 2), dst=T(na.I32, 2))
    a.update(kw)
    ops.paged_pages_fork(a["table"], a["refs"], a["parents"], a["children"], a["history"], a["page"], a["src"], a["dst"])


def compact(**kw):
    a = dict(TABLE, src=T(na.I32, 4), dst=T(na.I32, 4), moved=T(na.I32, 1))
    a.update(kw)
    ops.paged_pages_compact(a["table"], a["refs"], a["src"], a["dst"], a["moved"])


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("call", [rope, rope_append])
@pytest.mark.parametrize("kw,error", [
    (dict(q=None), ValueError), (dict(k=None), ValueError), (dict(qo=None), ValueError), (dict(q=T(na.FP32, 128, 8, 5)), ValueError),
    (dict(q=T(na.BF16, 128, 8, 0)), ValueError), (dict(q=T(na.BF16, 128, 8, 5, data=FAKE + 2)), ValueError), (dict(q=T(na.BF16, 128, 8, 5, nb={2: 8})), ValueError),
    (dict(q=T(na.BF16, 128, 8, 5, nb={1: 512})), ValueError), (dict(k=T(na.BF16, 128, 2, 4)), ValueError), (dict(k=T(na.BF16, 256, 2, 5)), ValueError),
    (dict(k=T(na.BF16, 128, 0, 5)), ValueError), (dict(qo=T(na.BF16, 128, 7, 5)), ValueError), (dict(qo=T(na.FP32, 128, 8, 5)), ValueError),
    (dict(qo=T(na.BF16, 128, 8, 5, nb={2: 4096})), ValueError),  # in place of q, other strides
    (dict(qw=T(na.FP16, 128)), ValueError), (dict(qw=T(na.BF16, 64)), ValueError), (dict(kw=T(na.FP32, 128, 2)), ValueError), (dict(kw=T(na.FP32, 128, data=0)), ValueError),
    (dict(kw=T(na.FP32, 128, data=FAKE + 4)), ValueError), (dict(freq=T(na.BF16, 64)), ValueError), (dict(freq=T(na.FP32, 72)), ValueError),
    (dict(freq=T(na.FP32, 12)), ValueError), (dict(freq=T(na.FP32, 0)), ValueError), (dict(freq=T(na.FP32, 64, data=0)), ValueError), (dict(freq=T(na.FP32, 8, 8)), ValueError),
    (dict(norm=(0.0, 0.0, 0)), ValueError), (dict(norm=(-1e-6, 0.0, 0)), ValueError), (dict(norm=(NAN, 0.0, 0)), ValueError), (dict(norm=(2.0, 0.0, 0)), ValueError),
    (dict(norm=(1e-6, INF, 0)), ValueError), (dict(norm=(1e-6, NAN, 0)), ValueError), (dict(norm=(1e-6, 0.0, 2)), ValueError),
])
def test_norm_rope(call, kw, error):
    with pytest.raises(error):
        call(**kw)


def test_norm_rope_forms():
    for kw in (dict(pos=None), dict(pos=T(na.I64, 5)), dict(pos=T(na.I32, 4)), dict(ko=None), dict(ko=T(na.BF16, 128, 1, 5)),
               dict(ko=T(na.BF16, 128, 2, 5, nb={2: 1024}))):
        with pytest.raises(ValueError):
            rope(**kw)
    for kw in (dict(v=None), dict(v=T(na.BF16, 128, 3, 5)), dict(starts=T(na.I32, 3)), dict(starts=None), dict(history=T(na.I32, 4)),
               dict(cache=view(D=256, page=64)), dict(cache=view(page=64, H=4))):
        with pytest.raises(ValueError):
            rope_append(**kw)
    d64 = dict(q=T(na.BF16, 64, 8, 5), k=T(na.BF16, 64, 2, 5), qw=None, kw=None, freq=None, qo=T(na.BF16, 64, 8, 5, data=2 * FAKE), ko=T(na.BF16, 64, 2, 5, data=3 * FAKE))
    with pytest.raises(NotImplementedError):
        rope(**d64)
    n = (1 << 23) + 1
    with pytest.raises(NotImplementedError):
        rope(q=T(na.BF16, 128, 8, n), k=T(na.BF16, 128, 2, n), qo=T(na.BF16, 128, 8, n, data=2 * FAKE), ko=T(na.BF16, 128, 2, n, data=3 * FAKE), pos=T(na.I32, n))
    with pytest.raises(NotImplementedError):
        rope(k=T(na.BF16, 128, 1025, 5), ko=T(na.BF16, 128, 1025, 5, data=3 * FAKE))


@pytest.mark.parametrize("name", [n for n in BAD_VIEWS if "page" not in n or "of the planes" in n])
def test_views(name):
    kw, error = BAD_VIEWS[name]
    kw = dict(dict(page=64), **kw)
    for call in (rope_append, update, attend, copy):
        with pytest.raises((error, ValueError)):  # planes for pages of 16 rows are of a wrong shape before anything else
            call(cache=view(**kw))


BAD_BLOCKS = [dict(size=16), dict(size=48), dict(size=128), dict(size=0), dict(codes=T(na.I8, 128, 1, 2, 8)), dict(codes=T(na.U8, 128, 2, 2, 8)),
              dict(codes=T(na.I8, 128, 2, 2, 8, data=0)), dict(codes=T(na.I8, 128, 2, 2, 8, data=FAKE + 8)), dict(codes=T(na.I8, 128, 2, 2, 8, nb={1: 256})),
              dict(codes=T(na.I8, 128, 2, 2, 8, nb={3: 496})), dict(scales=T(na.FP16, 2, 2, 8)), dict(scales=T(na.FP32, 1, 2, 8)),
              dict(scales=T(na.FP32, 2, 2, 9)), dict(scales=T(na.FP32, 2, 2, 8, data=0)), dict(scales=T(na.FP32, 2, 2, 8, data=FAKE + 2)),
              dict(scales=T(na.FP32, 2, 2, 8, nb={1: 16})), dict(scales=T(na.FP32, 2, 2, 8, nb={2: 12})), dict(scales=T(na.FP32, 2, 2, 8, 2))]


@pytest.mark.parametrize("kw", BAD_BLOCKS)
def test_blocks(kw):
    for call in (update, select, copy):
        with pytest.raises(ValueError):
            call(blocks=blocks(**kw))
    b = blocks(codes=T(na.I8, 128, 2, 2, 9), scales=T(na.FP32, 2, 2, 9))
    for call in (update, copy):  # of another pool
        with pytest.raises(ValueError):
            call(blocks=b)


def test_update_arguments():
    for kw in (dict(tokens=0), dict(tokens=-1), dict(starts=None), dict(starts=T(na.I32, 3)), dict(history=T(na.FP32, 3))):
        with pytest.raises(ValueError):
            update(**kw)


@pytest.mark.parametrize("kw,error", [
    (dict(q=None), ValueError), (dict(q=T(na.BF16, 128, 7, 5)), ValueError), (dict(q=T(na.BF16, 256, 8, 5)), ValueError), (dict(starts=T(na.I32, 5)), ValueError),
    (dict(history=None), ValueError), (dict(table=None), ValueError), (dict(table=T(na.I64, 4, 3)), ValueError), (dict(page=16), ValueError), (dict(page=96), ValueError),
    (dict(page=32), ValueError), (dict(pick=(-1, 2, 3)), ValueError), (dict(pick=(1, 0, 3)), ValueError), (dict(pick=(1, 2, -1)), ValueError),
    (dict(pick=(1, 1000, 24)), NotImplementedError), (dict(pick=(2**31 - 1, 2**31 - 1, 2**31 - 1)), NotImplementedError), (dict(env=(0, 64)), ValueError),
    (dict(env=(65, 64)), ValueError), (dict(env=(5, 257)), ValueError), (dict(env=(5, 1 << 31)), OverflowError), (dict(out=None), ValueError),
    (dict(out=T(na.I32, 5, 2, 5)), ValueError), (dict(out=T(na.I64, 6, 2, 5)), ValueError), (dict(out=T(na.I32, 6, 2, 5, nb={1: 32})), ValueError),
    (dict(ws=Ws(ptr=FAKE + 16)), ValueError), (dict(blocks=blocks(D=64)), NotImplementedError),
    (dict(table=T(na.I32, 1 << 18, 3), env=(5, (1 << 23) + 1)), NotImplementedError), (dict(table=T(na.I32, 1 << 18, 3), env=(5, (1 << 20) + 1)), NotImplementedError),
])
def test_select_arguments(kw, error):
    with pytest.raises(error):
        select(**kw)


@pytest.mark.parametrize("kw,error", [
    (dict(q=None), ValueError), (dict(q=T(na.BF16, 128, 7, 5)), ValueError), (dict(out=T(na.BF16, 128, 8, 4)), ValueError), (dict(out=None), ValueError),
    (dict(scale=0.0), ValueError), (dict(scale=NAN), ValueError), (dict(scale=2.0**41), ValueError), (dict(lists=None), ValueError),
    (dict(lists=T(na.I32, 6, 1, 5)), ValueError), (dict(lists=T(na.FP32, 6, 2, 5)), ValueError), (dict(lists=T(na.I32, 0, 2, 5)), ValueError),
    (dict(lists=T(na.I32, 1025, 2, 5)), NotImplementedError), (dict(size=16), ValueError), (dict(size=48), ValueError), (dict(size=8192), ValueError),
    (dict(size=0), ValueError), (dict(env=(5, 257)), ValueError), (dict(env=(0, 1)), ValueError), (dict(ws=Ws(ptr=FAKE + 16)), ValueError),
    (dict(starts=T(na.I32, 3)), ValueError), (dict(history=T(na.I32, 2)), ValueError),
])
def test_attention_arguments(kw, error):
    with pytest.raises(error):
        attend(**kw)


def test_attention_workspace():
    q = ops.paged_sparse_attention_workspace_bytes
    need = q(8, 2, 128, 5, 3, 200, 64)
    assert need > 0
    for ws in (Ws(nbytes=need - 1), Ws(nbytes=0), None):
        with pytest.raises(ValueError):
            attend(lists=T(na.I32, 200, 2, 5), size=64, ws=ws)
    for bad in [(8, 3, 128, 5, 3, 6, 64), (8, 2, 64, 5, 3, 6, 64), (8, 2, 128, 0, 3, 6, 64), (8, 2, 128, 5, 0, 6, 64), (8, 2, 128, 5, 1025, 6, 64),
                (8, 2, 128, 5, 3, 0, 64), (8, 2, 128, 5, 3, 1025, 64), (8, 2, 128, 5, 3, 6, 16), (8, 2, 128, 5, 3, 6, 96), (8, 2, 128, 1 << 28, 3, 6, 64)]:
        assert q(*bad) == 0
    for bad in [(0, 128, 5, 3, (5, 64), 32), (2, 64, 5, 3, (5, 64), 32), (2, 128, 0, 3, (5, 64), 32), (2, 128, 5, 0, (5, 64), 32), (2, 128, 5, 3, (0, 64), 32),
                (2, 128, 5, 3, (65, 64), 32), (2, 128, 5, 3, (5, (1 << 23) + 1), 32), (2, 128, 5, 3, (5, 64), 33)]:
        assert ops.paged_block_select_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("call", [reserve, release, fork, compact])
@pytest.mark.parametrize("kw,error", [
    (dict(table=None), ValueError), (dict(table=T(na.I64, 4, 3)), ValueError), (dict(table=T(na.I32, 4, 3, 2)), ValueError), (dict(table=T(na.I32, 4, 3, data=0)), ValueError),
    (dict(table=T(na.I32, 4, 3, nb={1: 12})), ValueError), (dict(table=T(na.I32, 4, 1025)), NotImplementedError), (dict(refs=None), ValueError),
    (dict(refs=T(na.I64, 8)), ValueError), (dict(refs=T(na.I32, 8, 2)), ValueError), (dict(refs=T(na.I32, 0)), ValueError), (dict(refs=T(na.I32, 8, data=0)), ValueError),
    (dict(refs=T(na.I32, (1 << 19) + 1)), NotImplementedError), (dict(table=T(na.I32, 1 << 28, 3)), OverflowError),
])
def test_tables(call, kw, error):
    with pytest.raises(error):
        call(**kw)


@pytest.mark.parametrize("call,kw,error", [
    (reserve, dict(page=24), ValueError), (release, dict(page=8), ValueError), (fork, dict(page=8192), ValueError),
    (reserve, dict(starts=T(na.I32, 3)), ValueError), (reserve, dict(history=None), ValueError), (reserve, dict(granted=T(na.I32, 4)), ValueError),
    (reserve, dict(granted=None), ValueError), (release, dict(sequences=None), ValueError), (release, dict(sequences=T(na.I32, 0)), ValueError),
    (release, dict(keep=T(na.I32, 3)), ValueError), (release, dict(sequences=T(na.I32, 65537), keep=T(na.I32, 65537)), NotImplementedError),
    (fork, dict(parents=None), ValueError), (fork, dict(children=T(na.I32, 3)), ValueError), (fork, dict(history=T(na.I32, 2)), ValueError),
    (fork, dict(src=T(na.I32, 3)), ValueError), (fork, dict(dst=None), ValueError), (fork, dict(parents=T(na.I32, 1025)), NotImplementedError),
    (compact, dict(src=None), ValueError), (compact, dict(dst=T(na.I32, 3)), ValueError), (compact, dict(moved=T(na.I32, 2)), ValueError),
    (compact, dict(moved=T(na.I64, 1)), ValueError), (copy, dict(src=None), ValueError), (copy, dict(src=T(na.I32, 0)), ValueError),
    (copy, dict(dst=T(na.I32, 6)), ValueError), (copy, dict(src=T(na.I64, 7)), ValueError), (copy, dict(src=T(na.I32, 1 << 24), dst=T(na.I32, 1 << 24)), NotImplementedError),
])
def test_page_arguments(call, kw, error):
    with pytest.raises(error):
        call(**kw)


@pytest.mark.parametrize("kw", [dict(block_size=16), dict(block_size=48), dict(block_size=128)])
def test_owner_refuses(kw):
    with pytest.raises(ValueError):
        PagedKVCacheLayer(pages=4, page_size=64, num_kv_heads=2, head_dim=128, batch=1, max_pages=2, **kw)


SOURCE = r"""
#include "ninfer_amd/ops.hpp"
#include <cstdio>
using namespace ninfer_amd;
static void* fake(int i = 1) { return reinterpret_cast<void*>(0x10000 * static_cast<size_t>(i)); }
int main() {
    PagedKVCacheLayerView c;
    c.k = c.v = Tensor(fake(), DType::I8, {128, 64, 2, 8});
    c.k_scale = c.v_scale = Tensor(fake(), DType::FP16, {2, 64, 2, 8});
    c.page_table = Tensor(fake(), DType::I32, {4, 3});
    c.page_size = 64; c.num_kv_heads = 2; c.head_dim = 128; c.dtype = DType::I8; c.quant_group = 64;
    PagedBlockView b;
    b.codes = Tensor(fake(), DType::I8, {128, 2, 2, 8});
    b.scales = Tensor(fake(), DType::FP32, {2, 2, 8});
    b.block_size = 32;
    Tensor q(fake(), DType::BF16, {128, 8, 5}), k(fake(), DType::BF16, {128, 2, 5}), qo(fake(2), DType::BF16, {128, 8, 5}), ko(fake(3), DType::BF16, {128, 2, 5});
    Tensor w(fake(), DType::BF16, {128}), freq(fake(), DType::FP32, {64}), pos(fake(), DType::I32, {5}), lists(fake(), DType::I32, {6, 2, 5});
    Tensor starts(fake(), DType::I32, {4}), history(fake(), DType::I32, {3}), few(fake(), DType::I32, {2}), refs(fake(), DType::I32, {8}), one(fake(), DType::I32, {1});
    Tensor table = c.page_table;
    WorkspaceArena arena(fake(), 1 << 30), none(fake(), 0);
    int bad = 0;
    const auto refuses = [&](auto f) { try { f(); ++bad; } catch (const std::invalid_argument& e) { std::printf("%s\n", e.what()); } };
    refuses([&] { ops::qk_norm_rope(q, k, &w, nullptr, starts, &freq, {1e-6f, 0.0f, 0}, qo, ko, nullptr); });
    refuses([&] { ops::qk_norm_rope(q, k, nullptr, nullptr, pos, nullptr, {0.0f, 0.0f, 0}, qo, ko, nullptr); });
    refuses([&] { ops::paged_qk_norm_rope_append(q, k, k, &w, &w, few, history, &freq, {1e-6f, 0.0f, 0}, c, qo, nullptr); });
    refuses([&] { ops::paged_block_update(c, starts, history, 0, b, nullptr); });
    refuses([&] { ops::paged_block_select(q, starts, history, table, 64, b, {1, 0, 5}, {5, 64}, arena, lists, nullptr); });
    refuses([&] { ops::paged_sparse_attention(q, starts, history, 0.0f, lists, 32, c, {5, 64}, arena, qo, nullptr); });
    refuses([&] { ops::paged_kv_copy_pages(c, &b, few, one, nullptr); });
    refuses([&] { ops::paged_pages_reserve(table, refs, starts, few, 64, history, nullptr); });
    refuses([&] { ops::paged_pages_release(table, refs, few, one, 64, nullptr); });
    refuses([&] { ops::paged_pages_fork(table, refs, few, few, history, 24, few, few, nullptr); });
    refuses([&] { ops::paged_pages_compact(table, refs, few, few, few, nullptr); });
    const PagedExecutionEnvelope wide{5, 1u << 31};
    try { ops::paged_sparse_attention(q, starts, history, 0.1f, lists, 32, c, wide, arena, qo, nullptr); ++bad; } catch (const std::overflow_error&) {}
    if (ops::paged_sparse_attention_workspace_bytes(40, 8, 128, 1, 1, 64, 64) == 0) { ++bad; }
    return bad;
}
"""


def test_ops_hpp(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None or not Path("/opt/rocm/include/hip/hip_runtime_api.h").exists():
        pytest.skip("no host compiler or HIP headers")
    src = tmp_path / "blocks.cpp"
    src.write_text(SOURCE)
    lib = ROOT / "ninfer_amd"
    cmd = [gxx, "-std=c++20", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT}/include", "-I/opt/rocm/include", str(src), "-o", str(tmp_path / "blocks"),
           f"-L{lib}", "-lninfer_amd", "-L/opt/rocm/lib", f"-Wl,-rpath,{lib}:/opt/rocm/lib"]
    subprocess.run(cmd, check=True, timeout=100)
    run = subprocess.run([str(tmp_path / "blocks")], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "paged_pages_fork: page_size" in run.stdout
