"""Calls of the int8 cache and the rotary step that the C ABI allows: one of two outputs,
frequencies of the caller's, the widest heads, very many sequences, chunks at once."""
import ctypes as C
import importlib
import math

import numpy as np
import pytest
import torch

from int8_helpers import HALF_STEP, f64
from test_gpu_int8 import DT, Batch, err_word, t32

pytestmark = pytest.mark.gpu
L = importlib.import_module("truellm-engine_b200._lib")
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
def test_one_of_the_two_is_read(ops, cuda, D, which):
    b = Batch(ops, cuda, [0, 0], [45, 7], 3, D, BF16)
    b.fill()
    z, cu, T = t32([0, 0], cuda), t32(b.cu_all, cuda), 52
    want = dict(zip("kv", ops.int8_read(b.cache, b.bt_t, z, cu, T, dtype=BF16)))
    out = torch.zeros(T, 3, D, device=cuda, dtype=BF16)
    p = {which: out.data_ptr()}
    err = err_word(cuda)
    st = L.lib().tkv_int8_read(C.byref(b.cache.c_struct()), p.get("k"), p.get("v"), L.TKV_BF16,
                               b.bt_t.data_ptr(), b.bt_t.shape[1], z.data_ptr(), cu.data_ptr(), 2, T, 45,
                               err.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert st == L.TKV_OK and torch.equal(out, want[which]) and err.item() == 0


@pytest.mark.parametrize("D,rotary", [(512, 256), (264, 16), (136, 128), (16, 16)])
@pytest.mark.parametrize("pairing", [L.TKV_ROPE_HALVES, L.TKV_ROPE_ADJACENT])
def test_frequencies_of_the_callers(cuda, D, rotary, pairing):
    """A plan whose turns were changed (as scaled frequencies do), heads up to 512."""
    T, Hq, Hk, half = 70, 3, 1, rotary // 2
    plan = L.TkvRopePlan()
    lib = L.lib()
    assert lib.tkv_rope_plan_init(C.byref(plan), rotary, 1e4, (C.c_int32 * 1)(half), 1, 0,
                                  pairing) == L.TKV_OK
    rng = np.random.default_rng(D)
    for i in range(half):
        plan.turns[i] *= float(rng.uniform(0.1, 3))
    turns = np.array(plan.turns[:half])
    q, k = (torch.randn(T, h, D, device=cuda, dtype=F16) for h in (Hq, Hk))
    pos = torch.randint(-5, 100000, (1, T), device=cuda, dtype=torch.int32)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    st = (C.c_int64 * 8)(Hq * D, D, Hk * D, D, Hq * D, D, Hk * D, D)
    assert lib.tkv_rope_axes(C.byref(plan), q.data_ptr(), k.data_ptr(), qo.data_ptr(), ko.data_ptr(),
                             L.TKV_F16, Hq, Hk, D, T, st, pos.data_ptr(), T, 0,
                             torch.cuda.current_stream().cuda_stream) == L.TKV_OK
    # the positions times turns is exact to 2^-53, of at most 2^16 turns
    w = 2 * math.pi * np.mod(f64(pos)[0][:, None] * turns, 1.0)
    c, s = np.cos(w)[:, None], np.sin(w)[:, None]
    for x, got in ((q, qo), (k, ko)):
        want, x = f64(x), f64(x)
        a = slice(0, half) if pairing == L.TKV_ROPE_HALVES else slice(0, rotary, 2)
        b = slice(half, rotary) if pairing == L.TKV_ROPE_HALVES else slice(1, rotary, 2)
        want[..., a], want[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size = np.zeros_like(x)
        size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
        lim = HALF_STEP[F16] * np.abs(want) + size * 2.0 ** -21 + 2.0 ** -25
        assert (np.abs(f64(got) - want) <= lim).all()


def test_very_many_sequences(ops, cuda):
    """20000 sequences of up to 40 tokens, most without a new one, bounds left to their
    defaults, against calls of parts of them."""
    B, H, Hq, D = 20000, 1, 8, 64
    rng = np.random.default_rng(0)
    new = (rng.random(B) < 0.3) * rng.integers(1, 4, B)
    b = Batch(ops, cuda, rng.integers(0, 37, B), new, H, D, F16, seed=1)
    b.fill()
    q, lens, cu = b.query(Hq), t32(b.lens, cuda), t32(b.cu, cuda)
    err = err_word(cuda)
    out = ops.int8_attend(b.cache, q, cu, b.bt_t, lens, max_q_tokens=3, err=err)
    assert err.item() == 0
    for at in (0, 7000, B - 300):
        r = slice(int(b.cu[at]), int(b.cu[at + 300]))
        part = ops.int8_attend(b.cache, q[r], t32(b.cu[at:at + 301] - b.cu[at], cuda),
                               b.bt_t[at:at + 300].contiguous(), lens[at:at + 300].contiguous(),
                               max_q_tokens=3)
        off = (out[r].double() - part.double()).abs()
        # contexts are cut elsewhere: each side is off by its output's rounding and the
        # weights', 2^-11 of a mean of |v| (and a thousandth of that for scores and sums)
        most = float(b.v.abs().max())
        assert (off <= part.double().abs() * 2.0 ** -10 + most * 2.0 ** -10 * 1.01 + 2.0 ** -24).all()
    keep = np.arange(0, 60)
    b.lens, b.old, b.new, b.cu = b.lens[keep], b.old[keep], b.new[keep], b.cu[:61]
    b.check(q[:b.cu[60]], out[:b.cu[60]])


@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16")])
def test_chunk_calls_at_once(ops, cuda, D, dt):
    """Calls with chunks and split contexts on two streams, each with its workspace."""
    bs = [Batch(ops, cuda, [3000, 40], [50, 1], 2, D, DT[dt], seed=i) for i in (1, 2)]
    for b in bs:
        b.fill()
    qs = [b.query(8) for b in bs]
    want = [b.attend(q) for b, q in zip(bs, qs)]
    ws = [ops.int8_workspace(2, 8, 2, D, 50, 3050) for _ in bs]
    args = [(b.cache, q, t32(b.cu, cuda), b.bt_t, t32(b.lens, cuda), 50, 3050) for b, q in zip(bs, qs)]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            got[i].append(ops.int8_attend(*args[i], workspace=ws[i], stream=streams[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in got[i])
