"""The C++ adapter of the paged int8 cache and of the rotary step hands every argument to
the C entry point in its place: linked with stand-ins that write down what they get
(CPU)."""
import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CUDA_INC = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "include"

PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <stdexcept>
#include <vector>
#include "truellm_kivi.hpp"

namespace kb = truellm::kivi_b200;
// what the last call got, pointers and numbers alike, in the order of the C declaration
static std::vector<double> got;
static int answer = TKV_OK;
template <class T> static double num(T* p) { return static_cast<double>(reinterpret_cast<intptr_t>(p)); }
template <class T> static double num(T x) { return static_cast<double>(x); }
template <class... A> static int note(A... a) { got = {num(a)...}; return answer; }

extern "C" {
int64_t tkv_int8_page_bytes(int d) { return d == 128 ? 4224 : 0; }
int tkv_int8_append(const tkv_int8_cache_t* c, const void* k, const void* v, int dt, const int64_t* st,
                    const int32_t* cu, const int32_t* old, const int32_t* bt, int mb, int n, int t, int mx,
                    int* err, void* s) {
  return note(c->pool, c->num_pages, c->n_kv_heads, c->head_dim, k, v, dt, st, cu, old, bt, mb, n, t, mx, err, s);
}
int tkv_int8_read(const tkv_int8_cache_t* c, void* k, void* v, int dt, const int32_t* bt, int mb,
                  const int32_t* st, const int32_t* cu, int n, int t, int mx, int* err, void* s) {
  return note(c->pool, c->num_pages, c->n_kv_heads, c->head_dim, k, v, dt, bt, mb, st, cu, n, t, mx, err, s);
}
size_t tkv_int8_attend_workspace_bytes(int a, int b, int c, int d, int e, int f) {
  note(a, b, c, d, e, f);
  return 77;
}
int tkv_int8_attend(const tkv_int8_cache_t* c, const void* q, int qd, const int64_t* st, void* o, int od,
                    const int32_t* cu, const int32_t* bt, int mb, const int32_t* lens, int n, int hq, int t,
                    int mq, int ml, int w, float sc, void* ws, size_t wb, int* err, void* s) {
  return note(c->pool, c->num_pages, c->n_kv_heads, c->head_dim, q, qd, st, o, od, cu, bt, mb, lens, n, hq, t, mq,
              ml, w, sc, ws, wb, err, s);
}
int tkv_rope_plan_init(tkv_rope_plan_t* p, int rd, double theta, const int32_t* sec, int n, int order, int pairing) {
  std::memset(p, 0, sizeof *p);
  p->rotary_dim = rd;
  return note(rd, theta, sec, n, order, pairing);
}
int tkv_rope_axes(const tkv_rope_plan_t* p, const void* q, const void* k, void* qo, void* ko, int dt, int hq, int hk,
                  int d, int t, const int64_t* st, const int32_t* pos, int64_t ax, int inv, void* s) {
  return note(p->rotary_dim, q, k, qo, ko, dt, hq, hk, d, t, st, pos, ax, inv, s);
}
const char* tkv_status_string(int) { return "told to"; }
}

template <class T> static T* at(int n) { return reinterpret_cast<T*>(static_cast<intptr_t>(n)); }
#define GOT(...) do { const std::vector<double> want = {__VA_ARGS__}; \
  if (got != want) { std::printf("FAIL %d\n", __LINE__); \
    for (size_t i = 0; i < got.size() || i < want.size(); ++i) \
      std::printf("%g %g\n", i < got.size() ? got[i] : -1, i < want.size() ? want[i] : -1); \
    return 1; } } while (0)
template <class F, class E> static bool throws(F f, E*) {
  try { f(); } catch (const E&) { return true; }
  return false;
}

int main() {
  kb::PagedInt8Cache cache(at<void>(1), 2, 3, 128);
  auto stream = reinterpret_cast<cudaStream_t>(at<void>(99));
  auto append = [&] { cache.append(at<void>(10), at<void>(11), 12, at<int64_t>(13), at<int32_t>(14), at<int32_t>(15),
                                   at<int32_t>(16), 17, 18, 19, 20, at<int>(21), stream); };
  append();
  GOT(1, 2, 3, 128, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21, 99);
  cache.read(at<void>(10), at<void>(11), 12, at<int32_t>(13), 14, at<int32_t>(15), at<int32_t>(16), 17, 18, 19,
             at<int>(20), stream);
  GOT(1, 2, 3, 128, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 99);
  if (cache.workspace_bytes(10, 11, 12, 13) != 77) return 1;
  GOT(10, 11, 3, 128, 12, 13);
  cache.attend(at<void>(10), 11, at<int64_t>(12), at<void>(13), 14, at<int32_t>(15), at<int32_t>(16), 17,
               at<int32_t>(18), 19, 20, 21, 22, 23, 24, 0.25f, at<void>(25), 26, at<int>(27), stream);
  GOT(1, 2, 3, 128, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21, 22, 23, 24, 0.25, 25, 26, 27, 99);
  kb::RopeAxes rope(10, 11.5, at<int32_t>(12), 13, 14, 15);
  GOT(10, 11.5, 12, 13, 14, 15);
  auto turn = [&](bool inverse) {
    rope.apply(at<void>(10), at<void>(11), at<void>(12), at<void>(13), 14, 15, 16, 17, 18, at<int64_t>(19),
               at<int32_t>(20), 21, inverse, stream);
  };
  turn(true);
  GOT(10, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21, 1, 99);
  turn(false);
  GOT(10, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21, 0, 99);
  // every other answer is an exception
  for (int status : {TKV_INVALID_ARGUMENT, TKV_NOT_IMPLEMENTED, TKV_BACKEND_ERROR}) {
    answer = status;
    if (!throws(append, static_cast<std::exception*>(nullptr)) ||
        !throws([&] { turn(true); }, static_cast<std::exception*>(nullptr))) return 2;
  }
  std::printf("ok\n");
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_arguments_arrive_in_their_places(tmp_path):
    src, exe = tmp_path / "calls.cpp", tmp_path / "calls"
    src.write_text(PROGRAM)
    res = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT / 'include'}",
                          f"-I{CUDA_INC}", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
