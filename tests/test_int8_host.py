"""The paged int8 cache and the rotary step without a GPU: sizes, the rotary
plan, and refusals, which answer before any CUDA call."""
import ctypes as C
import importlib
import math

import pytest
import torch

L = importlib.import_module("truellm-engine_b200._lib")
from int8_helpers import axis_of_pair  # noqa: E402

BAD, NOT = L.TKV_INVALID_ARGUMENT, L.TKV_NOT_IMPLEMENTED
P = 1 << 20  # an aligned address that no refused call touches


def test_page_bytes():
    lib = L.lib()
    assert [lib.tkv_int8_page_bytes(d) for d in (64, 128, 96, 0, -1)] == [2176, 4224, 0, 0, 0]


@pytest.mark.parametrize("sections", [(64,), (16, 24, 24), (0, 40, 24), (22, 21, 21), (1, 1, 62)])
@pytest.mark.parametrize("order", ["blocks", "round_robin"])
def test_plan_gives_every_pair_its_axis_and_frequency(sections, order):
    lib, p = L.lib(), L.TkvRopePlan()
    st = lib.tkv_rope_plan_init(C.byref(p), 128, 10000.0, (C.c_int32 * len(sections))(*sections),
                                len(sections), int(order == "round_robin"), L.TKV_ROPE_ADJACENT)
    assert st == L.TKV_OK and (p.rotary_dim, p.n_axes, p.pairing) == (128, len(sections), 1)
    assert list(p.axis[:64]) == axis_of_pair(sections, order)
    for i in range(64):
        assert math.isclose(p.turns[i] * 2 * math.pi, 10000.0 ** (-2 * i / 128), rel_tol=1e-14)


def test_plan_refusals():
    lib, p = L.lib(), L.TkvRopePlan()

    def init(rd=128, theta=1e4, sec=(64,), order=0, pairing=0, n=None):
        return lib.tkv_rope_plan_init(C.byref(p), rd, theta, (C.c_int32 * 16)(*sec),
                                      len(sec) if n is None else n, order, pairing)
    assert init() == L.TKV_OK
    for rd in (0, 8, 120, 272, -16):
        assert init(rd=rd) == NOT
    assert init(sec=(63,)) == init(sec=(65,)) == init(sec=(-1, 65)) == init(sec=(32, 31)) == BAD
    assert init(theta=0.0) == init(theta=-1.0) == init(theta=math.inf) == init(theta=math.nan) == BAD
    assert init(n=0) == init(n=9) == init(order=2) == init(pairing=2) == BAD
    assert lib.tkv_rope_plan_init(None, 128, 1e4, (C.c_int32 * 1)(64), 1, 0, 0) == BAD
    assert lib.tkv_rope_plan_init(C.byref(p), 128, 1e4, None, 1, 0, 0) == BAD


def test_rope_refusals():
    lib, p = L.lib(), L.TkvRopePlan()
    lib.tkv_rope_plan_init(C.byref(p), 128, 1e4, (C.c_int32 * 1)(64), 1, 0, 0)
    ok = dict(plan=C.byref(p), q=P, k=P, qo=P, ko=P, dt=L.TKV_BF16, hq=8, hk=2, d=128, t=0,
              st=(1024, 128) * 4, pos=P, ax=0)

    def call(**kw):
        a = {**ok, **kw}
        st = None if a["st"] is None else (C.c_int64 * 8)(*a["st"])
        return lib.tkv_rope_axes(a["plan"], a["q"], a["k"], a["qo"], a["ko"], a["dt"], a["hq"],
                                 a["hk"], a["d"], a["t"], st, a["pos"], a["ax"], 0, None)
    assert call() == L.TKV_OK  # no tokens: nothing to launch
    assert call(t=5, hq=0, hk=0) == L.TKV_OK
    assert call(t=-1) == call(d=64) == call(d=132) == call(hq=-1) == call(hk=-1) == BAD
    assert call(plan=None) == call(st=None) == BAD
    assert call(dt=L.TKV_F32) == call(d=520) == NOT
    for kw in (dict(q=None), dict(qo=None), dict(k=None), dict(ko=None), dict(pos=None),
               dict(q=P + 2), dict(ko=P + 8), dict(st=(1024, 128, 4, 128) * 2),
               dict(st=(-8, 128) * 4), dict(ax=-1)):
        assert call(t=5, **kw) == BAD, kw
    p.axis[63] = 1
    assert call(t=5) == BAD
    p.axis[63] = 0
    p.turns[3] = math.nan
    assert call(t=5) == BAD


def _cache(**kw):
    return L.TkvInt8Cache(**{**dict(pool=P, num_pages=4, n_kv_heads=2, head_dim=128), **kw})


BAD_CACHES = [dict(pool=None), dict(pool=P + 8), dict(num_pages=0), dict(n_kv_heads=0),
              dict(head_dim=96)]


def test_append_refusals():
    lib = L.lib()
    ok = dict(c=_cache(), k=P, v=P, dt=L.TKV_F16, st=(256, 128, 256, 128), cu=P, lens=P, bt=P, mb=4,
              b=2, t=0, mx=4)

    def call(**kw):
        a = {**ok, **kw}
        st = None if a["st"] is None else (C.c_int64 * 4)(*a["st"])
        return lib.tkv_int8_append(C.byref(a["c"]), a["k"], a["v"], a["dt"], st, a["cu"], a["lens"],
                                   a["bt"], a["mb"], a["b"], a["t"], a["mx"], None, None)
    assert call() == call(b=0, t=4) == call(mx=0, t=4) == L.TKV_OK
    for c in BAD_CACHES:
        assert call(c=_cache(**c)) == BAD, c
    assert lib.tkv_int8_append(None, P, P, 1, None, P, P, P, 4, 2, 0, 4, None, None) == BAD
    assert call(dt=L.TKV_F32) == NOT
    assert call(b=-1) == call(t=-1) == call(mx=-1) == call(mb=0) == BAD
    for kw in (dict(k=None), dict(v=None), dict(st=None), dict(cu=None), dict(lens=None),
               dict(bt=None), dict(k=P + 2), dict(v=P + 8), dict(st=(256, 128, 256, 4)),
               dict(st=(-256, 128, 256, 128))):
        assert call(t=4, **kw) == BAD, kw
    # more CTAs than one grid has
    assert call(t=2 ** 31 - 1, c=_cache(n_kv_heads=256)) == BAD


def test_read_refusals():
    lib = L.lib()
    ok = dict(c=_cache(), k=P, v=P, dt=L.TKV_F32, bt=P, mb=4, st=P, cu=P, b=2, t=0, mx=4)

    def call(**kw):
        a = {**ok, **kw}
        return lib.tkv_int8_read(C.byref(a["c"]), a["k"], a["v"], a["dt"], a["bt"], a["mb"],
                                 a["st"], a["cu"], a["b"], a["t"], a["mx"], None, None)
    assert call() == call(b=0, t=4) == call(mx=0, t=4) == L.TKV_OK
    for c in BAD_CACHES:
        assert call(c=_cache(**c)) == BAD, c
    assert call(dt=L.TKV_I32 if hasattr(L, "TKV_I32") else 3) == NOT
    assert call(b=-1) == call(t=-1) == call(mx=-1) == call(mb=0) == BAD
    for kw in (dict(k=None, v=None), dict(bt=None), dict(st=None), dict(cu=None), dict(k=P + 8),
               dict(v=P + 2)):
        assert call(t=4, **kw) == BAD, kw


def test_attend_refusals():
    lib = L.lib()
    need = lib.tkv_int8_attend_workspace_bytes(2, 8, 2, 128, 4, 64)
    assert need > 0
    ok = dict(c=_cache(), q=P, qd=L.TKV_BF16, st=(1024, 128), o=P, od=L.TKV_BF16, cu=P, bt=P, mb=4,
              lens=P, b=2, hq=8, t=0, mq=4, ml=64, w=0, sc=0.1, ws=P, wb=need)

    def call(**kw):
        a = {**ok, **kw}
        st = None if a["st"] is None else (C.c_int64 * 2)(*a["st"])
        return lib.tkv_int8_attend(C.byref(a["c"]), a["q"], a["qd"], st, a["o"], a["od"], a["cu"],
                                   a["bt"], a["mb"], a["lens"], a["b"], a["hq"], a["t"], a["mq"],
                                   a["ml"], a["w"], a["sc"], a["ws"], a["wb"], None, None)
    assert call() == call(b=0, t=4) == call(mq=0, t=4) == L.TKV_OK
    for c in BAD_CACHES:
        assert call(c=_cache(**c)) == BAD, c
    assert call(qd=L.TKV_F32) == call(od=L.TKV_F32) == NOT
    for kw in (dict(hq=7), dict(hq=0), dict(b=-1), dict(b=65536), dict(t=-1), dict(mq=-1),
               dict(ml=-1), dict(mb=0), dict(w=-1), dict(sc=0.0), dict(sc=-1.0), dict(sc=math.inf),
               dict(sc=math.nan)):
        assert call(**kw) == BAD, kw
    for kw in (dict(q=None), dict(st=None), dict(o=None), dict(cu=None), dict(bt=None),
               dict(lens=None), dict(ws=None), dict(q=P + 2), dict(o=P + 8), dict(ws=P + 4),
               dict(st=(1024, 4)), dict(st=(-1024, 128)), dict(wb=need - 1), dict(wb=0)):
        assert call(t=4, **kw) == BAD, kw
    # more CTAs than one grid has, refused before anything is launched
    for hq in (2, 8):
        assert call(t=4, b=65535, hq=hq, mq=1 << 27, mb=1 << 27, ml=1 << 27, wb=1 << 62) == BAD, hq


def test_workspace_sizes():
    lib = L.lib()
    ws = lib.tkv_int8_attend_workspace_bytes
    assert ws(2, 7, 2, 128, 1, 64) == ws(-1, 8, 2, 128, 1, 64) == ws(2, 8, 2, 96, 1, 64) == 0
    assert ws(2, 8, 2, 128, 1, -1) == ws(2, 8, 2, 128, 1, 2 ** 31 - 1) == 0
    assert ws(2, 8, 2, 128, 2 ** 28, 64) == 0  # 2^30 query rows of a kv head
    # serving sizes stay small beside a cache
    assert 0 < ws(64, 32, 8, 128, 1, 8192) < 64 << 20
    assert 0 < ws(1, 64, 8, 128, 1, 1 << 20) < 64 << 20
    assert 0 < ws(8, 32, 8, 128, 512, 8192) < 256 << 20


def test_tensor_checks(ops):
    """The Python entry points refuse CPU tensors and wrong shapes."""
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_axes(q, None, torch.zeros(1, 4, dtype=torch.int32), (64,))
    with pytest.raises(ValueError):
        ops.Int8PagedCache(8, 96, 4, device="cpu")
    with pytest.raises(ValueError):
        ops.Int8PagedCache(8, 128, device="cpu")
    c = ops.Int8PagedCache(8, 128, 4, device="cpu")
    assert c.pool.shape == (4, 8, 4224)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_append(c, q, q, i, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_read(c, i, i, i, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_attend(c, q, i, i, i)
    with pytest.raises(ValueError):
        ops.int8_workspace(2, 7, 2, 128, 1, 64, device="cpu")
    assert ops.int8_workspace(2, 8, 2, 128, 1, 64, device="cpu").sum() == 0
