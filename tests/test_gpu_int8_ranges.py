"""int8 attention where value rows differ in size by far more than fp16 holds: a row's
precision is that of the tokens it attends to, whatever others hold."""
import math

import numpy as np
import pytest
import torch

from int8_helpers import HALF_STEP, f64, scale_of, unpack
from test_gpu_int8 import Batch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def attend64(q, k, v, pos, scale, window):
    """One sequence in 64 bits: out, A = sum p |v|, S = scale * max over seen tokens of
    sum |q_c k_c| [n, Hq, D or 1], and the most that the weights' absolute error can
    make, per unit: N = (tokens seen) * max over them of p max_c |v|."""
    n, Hq, D = q.shape
    grp = Hq // k.shape[1]
    out, A = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    S, N = np.zeros((n, Hq, 1)), np.zeros((n, Hq, 1))
    for i in range(n):
        t = np.arange(max(0, pos[i] - window + 1) if window else 0, pos[i] + 1)
        for h in range(Hq):
            kk, vv = k[t, h // grp], v[t, h // grp]
            x = kk @ q[i, h] * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h], A[i, h] = p @ vv, p @ np.abs(vv)
            S[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
            N[i, h] = len(t) * (p * np.abs(vv).max(1)).max()
    return out, A, S, N


def bound(out, A, S, N, D, dt):
    """The output's own rounding; each weight's rounding to fp16 (2^-11 of it) and the
    error e of its score, as of every 32-bit sum of D + 8 terms and of queries held to
    2^-25 of their largest; 2^-15 for exponentials, whose arguments are sums of three
    numbers below 2^8 (each off by 2^-17 at most), and for scales and sums.  Weights
    below fp16's normal range are off by half a step of 2^-24 at most.  A weight is p s
    2^(5 - e) with s the token's scale and 2^e at most 2^5 times the row's largest p s so
    far, so 2^-25 of a weight is 2^-25 of that p s at most, and with codes up to 127, for
    each token that is seen, N 2^-25.  Outputs below the type's normal range are off by
    half its last step: 2^-25 for fp16, 2^-134 for bf16."""
    e = S * ((D + 8) * 2.0 ** -23 + D * 2.0 ** -25)
    tiny = 2.0 ** -25 if dt == F16 else 2.0 ** -134
    return (HALF_STEP[dt] * np.abs(out) + A * (2.0 ** -11 + 2 * e + 2.0 ** -15) * 1.01 +
            N * 2.0 ** -25 * 1.01 + tiny)


def check(b, q, out, window=0, rows=None):
    qn, got = f64(q), f64(out)
    assert np.isfinite(got).all()
    values = unpack(b.pool.cpu().numpy(), b.D)
    for s in range(len(b.lens)):
        n, o, r0 = int(b.new[s]), int(b.old[s]), int(b.cu[s])
        pick = np.arange(n) if rows is None or n <= rows else np.unique(
            np.r_[0, 1, n - 1, np.random.default_rng(n).integers(0, n, rows)])
        k, v = b.dense(s, values)
        want = attend64(qn[r0 + pick], k, v, o + pick, scale_of(b.D), window)
        off, lim = np.abs(got[r0 + pick] - want[0]), bound(*want, b.D, out.dtype)
        assert (off <= lim).all(), (s, float((off / lim).max()))


def batch(ops, cuda, old, new, D, dt, loud, seed=3, H=1):
    """`loud`: (position, power of two that its value row is multiplied by) of every
    sequence."""
    b = Batch(ops, cuda, old, new, H, D, dt, seed=seed)
    for s in range(len(old)):
        for p, e in loud:
            if p < b.lens[s]:
                at = int(b.cu_all[s]) + p
                b.v[at] = (b.v[at].double() * 2.0 ** e).to(dt)
    b.fill()
    return b


@pytest.mark.parametrize("new", [1, 2, 4, 80, 200])
@pytest.mark.parametrize("window", [0, 10, 90])
@pytest.mark.parametrize("e", [5, 16, 24, 30, 60, 100, 120])
def test_a_loud_value_costs_only_the_rows_that_weigh_it(ops, cuda, new, window, e):
    """One value row 2^e times its neighbours, in the chunk or before it: rows that do
    not see it, rows whose window has passed it, and rows that see it."""
    b = batch(ops, cuda, [20, 300], [new, new], 128, BF16, [(70, e)])
    q = b.query(4, mult=0.5)
    check(b, q, b.attend(q, window), window, rows=12)


@pytest.mark.parametrize("new", [1, 3, 60])
@pytest.mark.parametrize("e", [10, 14, -9, -14])
def test_loud_and_quiet_values_in_fp16(ops, cuda, new, e):
    b = batch(ops, cuda, [400], [new], 64, F16, [(0, e if e < 0 else 0), (130, e), (391, e)])
    q = b.query(8)
    check(b, q, b.attend(q), rows=12)


@pytest.mark.parametrize("new", [1, 3, 60, 140])
@pytest.mark.parametrize("e", [20, 40, 90, 140, 200])
def test_a_loud_value_of_hardly_any_weight(ops, cuda, new, e):
    """Rows see a token 2^e louder than the rest whose score is about e powers of two
    below the others': its product with the value is as large as theirs."""
    b = Batch(ops, cuda, [500], [new], 1, 128, BF16, seed=5)
    up = min(e, 110)
    b.v[:] = (b.v.double() * 2.0 ** (up - e)).to(BF16)
    b.v[77] = (torch.randn(128, device=cuda).double() * 2.0 ** up).to(BF16)
    # queries near one direction, the loud token's key against it
    d = torch.zeros(128, device=cuda)
    d[::2] = 1.0
    x = e * math.log(2.0) / scale_of(128) / 64
    b.k[77, 0] = (-x / 2 * d).to(BF16)
    b.fill()
    q = (b.query(4).float() * 0.05 + 2 * d).to(BF16)
    check(b, q, b.attend(q), rows=10)


@pytest.mark.parametrize("new", [1, 4, 70])
def test_values_that_grow_along_the_context(ops, cuda, new):
    """Every 16 tokens louder by 2^3 than the 16 before (a new power of two in most
    tiles), and the other way round; scores that fall and rise the other way."""
    for sign in (1, -1):
        b = Batch(ops, cuda, [560], [new], 1, 64, BF16, seed=7)
        n = int(b.lens[0])
        step = torch.arange(n, device=cuda) // 16 * 3.0 - 60.0
        b.v[:] = (b.v.double() * 2.0 ** (sign * step)[:, None, None]).to(BF16)
        ramp = -sign * step * math.log(2.0) / scale_of(64) / 64 * 0.7
        b.k[:] = (ramp[:, None, None] * torch.ones(64, device=cuda)).to(BF16)
        b.fill()
        q = (torch.ones(new, 4, 64, device=cuda) + 0.01 * b.query(4).float()).to(BF16)
        check(b, q, b.attend(q), rows=8)


@pytest.mark.parametrize("new", [1, 40])
def test_spread_rows_over_split_contexts(ops, cuda, new):
    """Long contexts in many parts, rows from 2^-40 to 2^40 times the ordinary size."""
    b = Batch(ops, cuda, [6000, 50], [new, new], 1, 128, BF16, seed=9, wild=2.0 ** 40)
    b.fill()
    q = b.query(8, mult=0.2)
    out = b.attend(q)
    check(b, q, out, rows=4)
    assert torch.equal(out, b.attend(q))


@pytest.mark.parametrize("new", [1, 30])
def test_rows_that_see_only_zeros_at_first(ops, cuda, new):
    b = Batch(ops, cuda, [300], [new], 1, 128, BF16, seed=12)
    b.v[:200] = 0
    b.v[210] = (b.v[210].double() * 2.0 ** 50).to(BF16)
    b.k[210] = (b.k[210].double() * 3).to(BF16)
    b.fill()
    q = b.query(4, mult=0.5)
    for window in (0, 40, 95):
        check(b, q, b.attend(q, window), window)


@pytest.mark.parametrize("new", [1, 3, 40, 150])
@pytest.mark.parametrize("size,scale", [(2.0 ** -120, 2.0 ** -60), (2.0 ** -30, 2.0 ** -100),
                                        (2.0 ** -120, 1.0), (2.0 ** -60, 2.0 ** -120)])
def test_scores_too_small_for_32_bits(ops, cuda, new, size, scale):
    """Queries and scales whose product is below the smallest float: all weights are
    equal, and masked tokens stay masked."""
    b = Batch(ops, cuda, [130], [new], 1, 128, BF16, seed=2)
    b.fill()
    q = b.query(4, mult=size)
    for window in (0, 50):
        out = b.attend(q, window, scale=scale)
        values = unpack(b.pool.cpu().numpy(), 128)
        k, v = b.dense(0, values)
        want = attend64(f64(q), k, v, 130 + np.arange(new), scale, window)
        off, lim = np.abs(f64(out) - want[0]), bound(*want, 128, BF16)
        assert (off <= lim).all()


@pytest.mark.parametrize("new", [1, 3, 40, 150])
@pytest.mark.parametrize("size", [2.0 ** -133, 2.0 ** -130, 2.0 ** -127])
def test_queries_below_the_normal_range(ops, cuda, new, size):
    """bf16 queries of subnormal size are no zeros: keys and a scale that bring them back."""
    b = Batch(ops, cuda, [130], [new], 1, 128, BF16, seed=4)
    b.k = (b.k.double() * 2.0 ** 60).to(BF16)
    b.fill()
    q = (torch.randint(-3, 4, (new, 4, 128), device=cuda).double() * size).to(BF16)
    scale = 2.0 ** -62 / size / 8
    out = b.attend(q, scale=scale)
    k, v = b.dense(0, unpack(b.pool.cpu().numpy(), 128))
    want = attend64(f64(q), k, v, 130 + np.arange(new), scale, 0)
    off, lim = np.abs(f64(out) - want[0]), bound(*want, 128, BF16)
    assert (off <= lim).all()


@pytest.mark.parametrize("new", [1, 3, 40, 150])
@pytest.mark.parametrize("e,small", [(100, 0), (115, 0), (126, 0), (126, 30), (-106, 0), (-116, 0),
                                     (-100, -100), (-110, -120)])
def test_keys_near_the_ends_of_the_type(ops, cuda, new, e, small):
    """Keys near 2^e in one direction with the queries, whose product passes 32 bits
    before the scale brings it back; queries of
    2^-small."""
    b = Batch(ops, cuda, [130], [new], 1, 128, BF16, seed=6)
    b.k = ((1 + 0.25 * b.k.float().clamp(-3, 3)).double() * 2.0 ** e).to(BF16)
    b.fill()
    q = ((1 + 0.1 * b.query(4).float()).double() * 2.0 ** -small).to(BF16)
    scale = 2.0 ** (small - e) / 64
    out = b.attend(q, scale=scale)
    k, v = b.dense(0, unpack(b.pool.cpu().numpy(), 128))
    want = attend64(f64(q), k, v, 130 + np.arange(new), scale, 0)
    off, lim = np.abs(f64(out) - want[0]), bound(*want, 128, BF16)
    assert (off <= lim).all()


@pytest.mark.parametrize("new,old,block", [(1, 300, 32), (4, 300, 32), (1, 5000, 600), (3, 5000, 600),
                                           (40, 5000, 700), (150, 1000, 256)])
@pytest.mark.parametrize("D", [64, 128])
def test_parts_whose_scores_and_values_are_far_apart(ops, cuda, new, old, block, D):
    """Blocks of tokens in turn 2^80 louder and quieter, with scores as far the other way,
    so that every block counts for as much: within a warp's share, between the warps of
    a CTA and between the parts of a context."""
    b = Batch(ops, cuda, [old], [new], 1, D, BF16, seed=8)
    n = int(b.lens[0])
    e = torch.where(torch.arange(n, device=cuda) // block % 2 == 0, 80.0, -80.0).double()
    b.v[:] = (b.v.double() * (2.0 ** e)[:, None, None]).to(BF16)
    x = -e * math.log(2.0) / scale_of(D) / D
    b.k[:] = (x[:, None, None] * torch.ones(D, device=cuda)).to(BF16)
    b.fill()
    q = (torch.ones(new, 4, D, device=cuda) + 0.001 * b.query(4).float()).to(BF16)
    for window in (0, 2 * block + 50):
        check(b, q, b.attend(q, window), window, rows=5)
