"""The C++ layer's paged ops: compiled against the header and the library, host checks as exceptions (no GPU)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SOURCE = r"""
#include "ninfer_amd/ops.hpp"
#include <cstdio>
using namespace ninfer_amd;
static void* fake() { return reinterpret_cast<void*>(0x10000); }
int main() {
    PagedKVCacheLayerView c;
    c.k = c.v = Tensor(fake(), DType::I8, {128, 16, 2, 8});
    c.k_scale = c.v_scale = Tensor(fake(), DType::FP16, {2, 16, 2, 8});
    c.page_table = Tensor(fake(), DType::I32, {4, 3});
    c.page_size = 16; c.num_kv_heads = 2; c.head_dim = 128; c.dtype = DType::I8; c.quant_group = 64;
    Tensor q(fake(), DType::BF16, {128, 8, 5}), k(fake(), DType::BF16, {128, 2, 5}), f(fake(), DType::FP32, {128, 2, 5});
    Tensor starts(fake(), DType::I32, {4}), history(fake(), DType::I32, {3}), few(fake(), DType::I32, {2});
    WorkspaceArena arena(fake(), 1 << 30), none(fake(), 0);
    int bad = 0;
    const auto refuses = [&](auto f) { try { f(); ++bad; } catch (const std::invalid_argument& e) { std::printf("%s\n", e.what()); } };
    refuses([&] { ops::paged_kv_append(k, k, few, history, c, nullptr); });
    refuses([&] { ops::paged_kv_read(c, starts, few, f, f, nullptr); });
    refuses([&] { ops::paged_attention(q, starts, history, 0.0f, {0, 0}, c, {5, 64}, arena, q, nullptr); });
    refuses([&] { ops::paged_attention(q, starts, history, 0.1f, {0, 0}, c, {5, 64}, none, q, nullptr); });
    try { ops::paged_attention(q, starts, history, 0.1f, {0, 0}, c, {5, 1u << 31}, arena, q, nullptr); ++bad; } catch (const std::overflow_error&) {}
    c.head_dim = 192;
    try { ops::paged_kv_append(k, k, starts, history, c, nullptr); ++bad; } catch (const std::runtime_error&) {}
    if (ops::paged_attention_workspace_bytes(40, 8, 128, 1, 1, {1, 65536}, {0, 0}) == 0) { ++bad; }
    return bad;
}
"""


def test_ops_hpp(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None or not Path("/opt/rocm/include/hip/hip_runtime_api.h").exists():
        pytest.skip("no host compiler or HIP headers")
    src = tmp_path / "paged.cpp"
    src.write_text(SOURCE)
    lib = ROOT / "ninfer_amd"
    cmd = [gxx, "-std=c++20", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT}/include", "-I/opt/rocm/include", str(src), "-o", str(tmp_path / "paged"),
           f"-L{lib}", "-lninfer_amd", "-L/opt/rocm/lib", f"-Wl,-rpath,{lib}:/opt/rocm/lib"]
    subprocess.run(cmd, check=True, timeout=100)
    run = subprocess.run([str(tmp_path / "paged")], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "invalid shape for starts" in run.stdout
