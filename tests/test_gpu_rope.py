"""Rotary positions with several axes on the GPU, against 64 bits."""
import numpy as np
import pytest
import torch

from int8_helpers import HALF_STEP, f64, rope

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def positions(rng, axes, T, far, dev):
    return torch.tensor(rng.integers(0, far, (axes, T)), dtype=torch.int32, device=dev)


def bound(want, size, dt):
    """The output's rounding; sine, cosine (2 ulp each) and two products and a
    sum in 32 bits."""
    return HALF_STEP[dt] * np.abs(want) + size * 2.0 ** -21 + (2.0 ** -25 if dt == torch.float16 else 0)


CASES = [  # T, Hq, Hk, D, sections, far
    (1, 32, 8, 128, (16, 24, 24), 100), (5, 8, 8, 64, (32,), 1 << 20), (64, 4, 1, 128, (64,), 4096),
    (130, 3, 2, 128, (10, 11, 11), 131072), (33, 2, 2, 80, (40,), 5000), (7, 5, 1, 96, (8, 8), 100),
    (9, 2, 1, 256, (64, 64), 1000), (17, 1, 1, 72, (24, 8), 77), (3, 40, 8, 16, (8,), 2 ** 31 - 1),
    (700, 8, 2, 128, (0, 40, 24), 1 << 30)]


@pytest.mark.parametrize("T,Hq,Hk,D,sections,far", CASES)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("order,pairing", [("blocks", "halves"), ("round_robin", "adjacent"),
                                           ("round_robin", "halves"), ("blocks", "adjacent")])
def test_rotation(ops, cuda, T, Hq, Hk, D, sections, far, dt, order, pairing):
    rng = np.random.default_rng(T + D)
    pos = positions(rng, len(sections), T, far, cuda)
    q = torch.randn(T, Hq, D, device=cuda).to(DT[dt])
    k = torch.randn(T, Hk, D, device=cuda).to(DT[dt])
    how = dict(theta=500000.0, order=order, pairing=pairing)
    qo, ko = ops.rope_axes(q, k, pos, sections, **how)
    for x, y in ((q, qo), (k, ko)):
        want, size = rope(f64(x), pos.cpu().numpy(), sections, 500000.0, order, pairing)
        off = np.abs(f64(y) - want)
        assert (off <= bound(want, size, DT[dt])).all()
        r = 2 * sum(sections)
        assert torch.equal(x[..., r:], y[..., r:])
    # in place, keys left out, and turned back
    q2, k2 = q.clone(), k.clone()
    assert ops.rope_axes(q2, k2, pos, sections, q_out=q2, k_out=k2, **how)[0] is q2
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    alone, none = ops.rope_axes(q, None, pos, sections, **how)
    assert none is None and torch.equal(alone, qo)
    back, _ = ops.rope_axes(qo, None, pos, sections, inverse=True, **how)
    want, size = rope(f64(qo), pos.cpu().numpy(), sections, 500000.0, order, pairing, inverse=True)
    assert (np.abs(f64(back) - want) <= bound(want, size, DT[dt])).all()


def test_negative_positions_and_zero(ops, cuda):
    q = torch.randn(4, 2, 64, device=cuda, dtype=torch.float16)
    zero = torch.zeros(1, 4, dtype=torch.int32, device=cuda)
    assert torch.equal(ops.rope_axes(q, None, zero, (32,))[0], q)
    pos = torch.tensor([[1, -5, 100, -70000]], dtype=torch.int32, device=cuda)
    a = ops.rope_axes(q, None, pos, (32,))[0]
    assert torch.equal(a, ops.rope_axes(q, None, -pos, (32,), inverse=True)[0])
    want, size = rope(f64(q), pos.cpu().numpy(), (32,), 1e4, "blocks", "halves")
    assert (np.abs(f64(a) - want) <= bound(want, size, torch.float16)).all()


def test_strides(ops, cuda):
    """Slices of a fused projection, heads outermost, vectors that 16-byte loads
    cannot take; position rows of a wider tensor."""
    T, D = 21, 128
    qkv = torch.randn(T, 12 * D, device=cuda, dtype=torch.bfloat16)
    q, k = qkv[:, :8 * D].unflatten(1, (8, D)), qkv[:, 8 * D:10 * D].unflatten(1, (2, D))
    wide = torch.randint(0, 9999, (3, T + 11), device=cuda, dtype=torch.int32)
    pos = wide[:, 4:4 + T]
    qo, ko = ops.rope_axes(q.contiguous(), k.contiguous(), pos.contiguous(), (16, 24, 24))
    for qq, kk in ((q, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k)):
        a, b = ops.rope_axes(qq, kk, pos, (16, 24, 24))
        assert torch.equal(a, qo) and torch.equal(b, ko)
    odd = torch.zeros(T, 8, D + 3, device=cuda, dtype=torch.bfloat16)[..., 3:]
    odd.copy_(q)
    assert torch.equal(ops.rope_axes(odd, None, pos, (16, 24, 24))[0], qo)
    keep = qkv.clone()
    ops.rope_axes(q, k, pos, (16, 24, 24), q_out=q, k_out=k)  # in place in the projection
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(qkv[:, 10 * D:], keep[:, 10 * D:])


def test_gradient(ops, cuda):
    """Against the formula's (the rotation back) and against differences."""
    rng = np.random.default_rng(3)
    T, D, sections = 19, 64, (8, 12, 12)
    pos = positions(rng, 3, T, 3000, cuda)
    q = torch.randn(T, 4, D, device=cuda, dtype=torch.float16).requires_grad_()
    k = torch.randn(T, 2, D, device=cuda, dtype=torch.float16).requires_grad_()
    wq, wk = torch.randn_like(q), torch.randn_like(k)
    qo, ko = ops.rope_axes(q, k, pos, sections, order="round_robin")
    torch.autograd.backward([qo, ko], [wq, wk])
    for x, w in ((q, wq), (k, wk)):
        want, size = rope(f64(w), pos.cpu().numpy(), sections, 1e4, "round_robin", "halves", True)
        assert (np.abs(f64(x.grad) - want) <= bound(want, size, torch.float16)).all()
    # differences: the map is linear, so a step of any size gives the slope; each
    # of the two outputs is off by half a step of at most |a| + |b| < 16
    d = torch.randn_like(q).detach()
    with torch.no_grad():
        up = ops.rope_axes(q + d, None, pos, sections, order="round_robin")[0]
    step = f64((q + d).detach()) - f64(q)
    slope = float(((f64(up) - f64(qo)) * f64(wq)).sum())
    inner = float((f64(q.grad) * step).sum())
    lim = np.abs(f64(wq)).sum() * 2 * 16 * 2.0 ** -11 + np.abs(step).sum() * 16 * 2.0 ** -11
    assert abs(slope - inner) <= lim
    with pytest.raises(ValueError):
        ops.rope_axes(q, k, pos, sections, q_out=torch.empty_like(q))
    alone, _ = ops.rope_axes(q, None, pos, sections)
    alone.sum().backward()


def test_refusals(ops, cuda):
    q = torch.randn(4, 2, 64, device=cuda, dtype=torch.float16)
    pos = torch.zeros(1, 4, dtype=torch.int32, device=cuda)
    for bad in (pos.long(), pos[:, :3], pos[0], torch.zeros(2, 4, dtype=torch.int32, device=cuda),
                torch.zeros(1, 8, dtype=torch.int32, device=cuda)[:, ::2]):
        with pytest.raises(ValueError):
            ops.rope_axes(q, None, bad, (32,))
    with pytest.raises(ValueError):
        ops.rope_axes(q.float(), None, pos, (32,))
    with pytest.raises(ValueError):
        ops.rope_axes(q, q.to(torch.bfloat16), pos, (32,))
    with pytest.raises(ValueError):
        ops.rope_axes(q, q[:3], pos, (32,))
    with pytest.raises(ValueError):
        ops.rope_axes(q, None, pos, (32,), order="zigzag")
    with pytest.raises(ValueError):
        ops.rope_axes(q, None, pos, (32,), q_out=torch.empty(4, 2, 64, device=cuda))
    with pytest.raises(ValueError):
        ops.rope_axes(q, None, pos, (32,), q_out=torch.empty_like(q), k_out=torch.empty_like(q))
    with pytest.raises(RuntimeError):
        ops.rope_axes(q, None, pos, (33,))  # 66 channels
    with pytest.raises(RuntimeError):
        ops.rope_axes(q, None, pos, (64,))  # more channels than the head has
    empty = torch.empty(0, 2, 64, device=cuda, dtype=torch.float16)
    assert ops.rope_axes(empty, empty, pos[:, :0], (32,))[1].shape == empty.shape


def test_captured_and_on_another_stream(ops, cuda):
    q = torch.randn(40, 8, 128, device=cuda, dtype=torch.bfloat16)
    k = torch.randn(40, 2, 128, device=cuda, dtype=torch.bfloat16)
    pos = torch.randint(0, 5000, (3, 40), device=cuda, dtype=torch.int32)
    want = ops.rope_axes(q, k, pos, (16, 24, 24))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = ops.rope_axes(q, k, pos, (16, 24, 24), stream=s)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.rope_axes(q, k, pos, (16, 24, 24))
    q.copy_(torch.randn_like(q))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], ops.rope_axes(q, k, pos, (16, 24, 24))[0])


@pytest.mark.parametrize("T", [1023, 1024, 1025, 4099])
def test_long_calls_turn_as_short_ones_do(ops, cuda, T):
    """Calls long enough for several tokens a CTA, against calls of 100 tokens."""
    rng = np.random.default_rng(T)
    q = torch.randn(T, 5, 72, device=cuda, dtype=torch.bfloat16)
    k = torch.randn(T, 2, 72, device=cuda, dtype=torch.bfloat16)
    pos = positions(rng, 2, T, 1 << 20, cuda)
    got = ops.rope_axes(q, k, pos, (20, 12))
    for at in range(0, T, 100):
        s = slice(at, min(T, at + 100))
        want = ops.rope_axes(q[s], k[s], pos[:, s].contiguous(), (20, 12))
        assert torch.equal(got[0][s], want[0]) and torch.equal(got[1][s], want[1])


def test_second_derivative(ops, cuda):
    """The gradient is linear in what comes back: its own gradient turns forwards."""
    rng = np.random.default_rng(8)
    pos = positions(rng, 2, 21, 5000, cuda)
    q = torch.randn(21, 3, 64, device=cuda, dtype=torch.float16).requires_grad_()
    v = torch.randn_like(q).requires_grad_()
    u = torch.randn_like(q)
    (g,) = torch.autograd.grad(ops.rope_axes(q, None, pos, (20, 12))[0], q, v, create_graph=True)
    (h,) = torch.autograd.grad(g, v, u)
    assert torch.equal(h, ops.rope_axes(u, None, pos, (20, 12))[0])


@pytest.mark.parametrize("T", [1, 3])
def test_rows_at_odd_strides_and_addresses(ops, cuda, T):
    """Rows that 16-byte vectors cannot address are copied, one token's too (whose
    token stride counts for nothing)."""
    raw = torch.randn(T, 2 * 64 + 3, device=cuda, dtype=torch.bfloat16)
    pos = torch.arange(7, 7 + T, device=cuda, dtype=torch.int32)[None]
    for off in (0, 1):
        q = raw[:, off:off + 128].unflatten(1, (2, 64))
        same = q.new_empty(q.shape).copy_(q)
        assert torch.equal(ops.rope_axes(q, q, pos, (32,))[1], ops.rope_axes(same, None, pos, (32,))[0])
