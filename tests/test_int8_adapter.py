"""The paged int8 cache behind the config switch and the C++ adapter (CPU)."""
import importlib
import os
import shutil
import subprocess
from pathlib import Path

import pytest

CF = importlib.import_module("truellm-engine_b200.config")
ROOT = Path(__file__).resolve().parents[1]
PKG = ROOT / "truellm-engine_b200"
CUDA_INC = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"

PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <stdexcept>
#include "truellm_kivi.hpp"

namespace kb = truellm::kivi_b200;
#define CHECK(x) do { if (!(x)) { std::printf("FAIL %d %s\n", __LINE__, #x); return 1; } } while (0)
template <class F>
bool refused(F f) {
  try { f(); } catch (const std::invalid_argument&) { return true; }
  return false;
}

int main() {
  CHECK(kb::PagedInt8Cache::page_bytes(128) == 4224 && kb::PagedInt8Cache::page_bytes(96) == 0);
  CHECK(refused([] { kb::PagedInt8Cache(nullptr, 4, 8, 96); }));
  kb::PagedInt8Cache cache(nullptr, 4, 2, 128);
  CHECK(cache.c().num_pages == 4 && cache.c().n_kv_heads == 2 && cache.c().head_dim == 128);
  CHECK(cache.workspace_bytes(2, 8, 1, 64) > 0 && cache.workspace_bytes(2, 7, 1, 64) == 0);
  const int64_t st[8] = {1024, 128, 1024, 128, 1024, 128, 1024, 128};
  alignas(16) static char x[64];
  int32_t idx[4] = {0, 1, 1, 1};
  // a null pool is refused before any CUDA call
  CHECK(refused([&] { cache.append(x, x, TKV_F16, st, idx, idx, idx, 1, 1, 1, 1, nullptr, nullptr); }));
  CHECK(refused([&] { cache.read(x, x, TKV_F16, idx, 1, idx, idx, 1, 1, 1, nullptr, nullptr); }));
  CHECK(refused([&] { cache.attend(x, TKV_F16, st, x, TKV_F16, idx, idx, 1, idx, 1, 8, 1, 1, 16, 0, 0.1f, x,
                                   sizeof x, nullptr, nullptr); }));
  const int32_t sec[3] = {16, 24, 24}, bad[3] = {16, 24, 25};
  kb::RopeAxes rope(128, 10000.0, sec, 3, TKV_ROPE_BLOCKS, TKV_ROPE_HALVES);
  CHECK(rope.plan().axis[15] == 0 && rope.plan().axis[16] == 1 && rope.plan().axis[40] == 2);
  CHECK(std::fabs(rope.plan().turns[0] * 2 * 3.14159265358979 - 1) < 1e-12);
  CHECK(refused([&] { kb::RopeAxes(128, 10000.0, bad, 3, TKV_ROPE_BLOCKS, TKV_ROPE_HALVES); }));
  CHECK(refused([&] { rope.apply(nullptr, nullptr, x, nullptr, TKV_F16, 8, 0, 128, 1, st, idx, 1, false, nullptr); }));
  std::printf("ok\n");
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_cpp_adapter(tmp_path):
    assert (PKG / "libtruellm_kivi.so").exists(), "build the library first (truellm-engine_b200/build.py)"
    src, exe = tmp_path / "int8.cpp", tmp_path / "int8"
    src.write_text(PROGRAM)
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT / 'include'}",
                          f"-I{CUDA_INC}", str(src), f"-L{PKG}", "-ltruellm_kivi",
                          f"-Wl,-rpath,{PKG}", "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


def config(**kw):
    c = dict(backend="cuda", kv_cache=dict(type_k="int8", type_v="int8"))
    c.update(kw)
    return CF.parse({"inference": c})


def test_the_config_switch_selects_the_cache():
    cfg = config()
    assert CF.validate(cfg) is None and cfg.paged_int8 and not cfg.paged_kivi
    assert cfg.kivi_path is None and not cfg.compression_pass and not cfg.pass_runs
    other = CF.parse({"inference": dict(backend="cuda")})
    assert not other.paged_int8


@pytest.mark.parametrize("kw, word", [
    (dict(kv_cache=dict(type_k="int8", type_v="f16")), "both"),
    (dict(kv_cache=dict(type_k="f16", type_v="int8")), "both"),
    (dict(kv_cache=dict(type_k="int8", type_v="kivi4")), "both"),
    (dict(kv_cache=dict(type_k="kivi4", type_v="int8")), "both"),
    (dict(backend="cpu"), "backend"),
    (dict(cuda_engine=dict(paged_kv_block_size=32)), "16"),
    (dict(cuda_engine=dict(use_megakernel=True)), "use_megakernel"),
    (dict(compression=dict(kv_kivi=dict(enabled=True))), "kv_kivi"),
])
def test_what_the_switch_does_not_go_with(kw, word):
    assert word in CF.validate(config(**kw))
