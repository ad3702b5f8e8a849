"""The paged int8 cache on the GPU: bytes, read-back and attention against 64
bits, refusals of bad tables and lengths, streams, graphs and strides."""
import importlib

import numpy as np
import pytest
import torch

from int8_helpers import (HALF_STEP, PAGE, attention, attention_bound, block_bytes, f64, pages_of,
                          quantise, scale_of, unpack)

pytestmark = pytest.mark.gpu
L = importlib.import_module("truellm-engine_b200._lib")
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DT = {"f16": F16, "bf16": BF16}


def t32(a, dev):
    return torch.tensor(np.asarray(a, np.int32), device=dev)


def err_word(dev):
    return torch.zeros(1, dtype=torch.int32, device=dev)


class Batch:
    """Sequences of `old` tokens, of which the last `new` are the chunk, in a
    pool whose unwritten bytes are 0xff (a NaN as a scale)."""

    def __init__(self, ops, dev, old, new, H, D, dt, seed=0, wild=1.0):
        rng = np.random.default_rng(seed)
        self.ops, self.dev, self.H, self.D, self.dt = ops, dev, H, D, dt
        self.old, self.new = np.asarray(old), np.asarray(new)
        self.lens = self.old + self.new
        self.bt, self.pages = pages_of(self.lens, rng)
        self.bt_t = t32(self.bt, dev)
        self.pool = torch.full((self.pages, H, block_bytes(D)), 255, dtype=torch.uint8, device=dev)
        self.cache = ops.Int8PagedCache(H, D, pool=self.pool)
        self.cu = np.concatenate([[0], np.cumsum(self.new)])
        self.cu_all = np.concatenate([[0], np.cumsum(self.lens)])
        T = int(self.lens.sum())
        # keys with loud channels, values whose rows differ in size by `wild`
        k = rng.standard_normal((T, H, D)) * np.where(np.arange(D) % 37 == 5, 8, 1)
        v = rng.standard_normal((T, H, D)) * wild ** rng.uniform(-1, 1, (T, H, 1))
        self.k = torch.tensor(k, dtype=torch.float32, device=dev).to(dt)
        self.v = torch.tensor(v, dtype=torch.float32, device=dev).to(dt)
        self.rng = rng

    def fill(self):
        z = t32(np.zeros(len(self.lens)), self.dev)
        self.ops.int8_append(self.cache, self.k, self.v, t32(self.cu_all, self.dev), z, self.bt_t)

    def dense(self, b, values=None):
        """Sequence b's dequantised keys and values [L, H, D], 64 bits."""
        kc, vc, s = values or unpack(self.pool.cpu().numpy(), self.D)
        n = int(self.lens[b])
        p = self.bt[b, :(n + PAGE - 1) // PAGE]
        k = kc[p] * s[p][..., :1].astype(np.float64)
        v = vc[p] * s[p][..., 1:].astype(np.float64)
        flat = lambda x: x.transpose(0, 2, 1, 3).reshape(-1, self.H, self.D)[:n]  # noqa: E731
        return flat(k), flat(v)

    def query(self, Hq, dt=None, mult=1.0):
        q = self.rng.standard_normal((int(self.new.sum()), Hq, self.D)) * mult
        return torch.tensor(q, dtype=torch.float32, device=self.dev).to(dt or self.dt)

    def attend(self, q, window=0, err=None, **kw):
        return self.ops.int8_attend(
            self.cache, q, t32(self.cu, self.dev), self.bt_t, t32(self.lens, self.dev),
            max_q_tokens=int(self.new.max()), max_context_len=int(self.lens.max()), window=window,
            err=err, **kw)

    def check(self, q, out, window=0, rows=None):
        qn, got = f64(q), f64(out)
        assert np.isfinite(got).all()
        values = unpack(self.pool.cpu().numpy(), self.D)
        for b in range(len(self.lens)):
            n, o, r0 = int(self.new[b]), int(self.old[b]), int(self.cu[b])
            pick = np.arange(n) if rows is None or n <= rows else np.unique(
                np.r_[0, 1, n - 1, self.rng.integers(0, n, rows)])
            if n == 0:
                continue
            k, v = self.dense(b, values)
            want, A, S, M = attention(qn[r0 + pick], k, v, o + pick, scale_of(self.D), window)
            off = np.abs(got[r0 + pick] - want)
            lim = attention_bound(want, A, S, M, self.D, out.dtype)
            assert (off <= lim).all(), (b, float((off / lim).max()))


# --------------------------------------------------------------------------
# bytes
# --------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("H", [1, 3])
def test_append_writes_the_formats_bytes_however_it_is_split(ops, cuda, D, dt, H):
    lens = [0, 1, 15, 16, 17, 33, 100]
    b = Batch(ops, cuda, [0] * len(lens), lens, H, D, DT[dt], seed=D + H)
    err = err_word(cuda)
    done = np.zeros(len(lens), int)
    step = 0
    while (done < lens).any():  # chunks of 1, 2, 5, 16 and 40 tokens
        n = np.minimum([(1, 2, 5, 16, 40)[(step + i) % 5] for i in range(len(lens))], lens - done)
        pick = np.concatenate([b.cu[i] + done[i] + np.arange(n[i]) for i in range(len(lens))])
        at = torch.tensor(pick, device=cuda, dtype=torch.long)
        ops.int8_append(b.cache, b.k[at], b.v[at], t32(np.r_[0, np.cumsum(n)], cuda),
                        t32(done, cuda), b.bt_t, max_new_tokens=int(n.max()), err=err)
        done += n
        step += 1
    split = b.pool.clone()
    b.pool.fill_(255)
    b.fill()
    assert torch.equal(split, b.pool) and err.item() == 0
    kc, vc, s = unpack(b.pool.cpu().numpy(), D)
    used = np.zeros((b.pages, PAGE), bool)
    for i, n in enumerate(lens):
        for p in range(n):
            page, slot = b.bt[i, p // PAGE], p % PAGE
            used[page, slot] = True
            for x, codes, w in ((b.k, kc, 0), (b.v, vc, 1)):
                want, d = quantise(f64(x[b.cu[i] + p]))
                assert np.array_equal(s[page, :, slot, w], d[:, 0])
                assert np.array_equal(codes[page, :, slot], want)
    free = ~used  # what no token owns is as it was
    assert (kc[free.nonzero()[0], :, free.nonzero()[1]] == 127).all()
    assert (vc[free.nonzero()[0], :, free.nonzero()[1]] == 127).all()
    assert np.isnan(s[free.nonzero()[0], :, free.nonzero()[1]]).all()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_append_of_special_rows(ops, cuda, dt):
    """Ties, zeros, the type's largest and smallest values, NaN and infinities."""
    D, H = 64, 1
    rows = []
    base = np.arange(D) * 2.0 - 63.0                      # odd numbers: ties at a scale of 2
    rows.append(np.where(np.arange(D) == 0, 254.0, base))   # scale exactly 2: x / 2 = k + 1/2
    rows.append(np.where(np.arange(D) == 1, -254.0, base))
    rows.append(np.zeros(D))
    rows.append(-np.zeros(D))
    big = float(torch.finfo(DT[dt]).max)
    rows.append(np.linspace(-1, 1, D) * big)
    rows.append(np.full(D, big))
    tiny = 2.0 ** -24 if dt == "f16" else 2.0 ** -100
    rows.append(np.arange(D) * tiny)
    rows.append(np.where(np.arange(D) == 3, tiny, 0.0))
    for bad in (np.nan, np.inf, -np.inf):
        rows.append(np.where(np.arange(D) == 7, bad, base))
    if dt == "bf16":
        rows.append(np.arange(D) * 2.0 ** -130)            # its scale is below the normal range
    x = torch.tensor(np.array(rows), dtype=torch.float32, device=cuda).to(DT[dt])[:, None, :]
    n = len(rows)
    cache = ops.Int8PagedCache(H, D, 1)
    z, cu = t32([0], cuda), t32([0, n], cuda)
    ops.int8_append(cache, x, x.flip(0), cu, z, t32([[0]], cuda))
    kc, vc, s = unpack(cache.pool.cpu().numpy(), D)
    want, d = quantise(f64(x))
    assert np.array_equal(s[0, 0, :n, 0], d[:, 0, 0], equal_nan=True)
    assert np.array_equal(s[0, 0, :n, 1], d[::-1, 0, 0], equal_nan=True)
    assert np.array_equal(kc[0, 0, :n], want[:, 0]) and np.array_equal(vc[0, 0, :n], want[::-1, 0])
    k, v = ops.int8_read(cache, t32([[0]], cuda), z, cu, n, dtype=F32)
    dd = np.where(np.isnan(d), np.nan, d).astype(np.float64)
    assert np.array_equal(f64(k), (want * dd).astype(np.float32).astype(np.float64), equal_nan=True)
    assert torch.equal(v.isnan(), k.flip(0).isnan())


def test_append_ties_everywhere(ops, cuda):
    """Scales that are powers of two and all their quotients in halves."""
    D = 128
    q = np.arange(-127, 127.5, 0.5)
    rows = []
    for e in (-6, 0, 3):
        for i in range(0, len(q), D - 1):
            r = np.zeros(D)
            r[0] = 127.0
            r[1:1 + len(q[i:i + D - 1])] = q[i:i + D - 1]
            rows.append(r * 2.0 ** e)
    x = torch.tensor(np.array(rows), dtype=F16, device=cuda)[:, None]
    n = len(rows)
    cache = ops.Int8PagedCache(1, D, 1 + n // PAGE)
    bt = t32([list(range(1 + n // PAGE))], cuda)
    ops.int8_append(cache, x, x, t32([0, n], cuda), t32([0], cuda), bt)
    kc, vc, s = unpack(cache.pool.cpu().numpy(), D)
    want, d = quantise(f64(x))
    assert np.array_equal(kc.transpose(0, 2, 1, 3).reshape(-1, D)[:n], want[:, 0])
    assert np.array_equal(vc.transpose(0, 2, 1, 3).reshape(-1, D)[:n], want[:, 0])


@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16")])
@pytest.mark.parametrize("out", [F16, BF16, F32])
def test_read_back(ops, cuda, D, dt, out):
    lens = [40, 0, 7, 129, 64]
    b = Batch(ops, cuda, [0] * 5, lens, 2, D, DT[dt], seed=3)
    b.fill()
    starts = np.array([3, 0, 0, 16, 63])
    n = np.array([30, 0, 7, 113, 1])
    cu = np.r_[2, 2 + np.cumsum(n)]
    T = int(cu[-1]) + 3
    err = err_word(cuda)
    ko = torch.full((T, 2, D), 7.0, dtype=out, device=cuda)
    vo = ko.clone()
    got = ops.int8_read(b.cache, b.bt_t, t32(starts, cuda), t32(cu, cuda), T, k_out=ko, v_out=vo,
                        err=err)
    assert got[0] is ko and got[1] is vo and err.item() == 0
    values = unpack(b.pool.cpu().numpy(), D)
    for i in range(5):
        for g, w in zip((ko, vo), b.dense(i, values)):
            w = w[starts[i]:starts[i] + n[i]]
            off = np.abs(f64(g[cu[i]:cu[i + 1]]) - w)
            assert (off <= np.abs(w) * (HALF_STEP[out] + 2.0 ** -23) + 2.0 ** -25).all()
    for g in (ko, vo):  # rows of no sequence
        assert (g[:2] == 7).all() and (g[-3:] == 7).all()
    k2, v2 = ops.int8_read(b.cache, b.bt_t, t32(starts, cuda), t32(cu, cuda), T, dtype=out)
    assert torch.equal(k2[2:-3], ko[2:-3]) and torch.equal(v2[2:-3], vo[2:-3])


def test_append_reads_strided_rows_where_they_lie(ops, cuda):
    B, H, D = 5, 2, 128
    lens = [3, 20, 1, 0, 40]
    T = sum(lens)
    qkv = torch.randn(T, 8 * D + 2 * H * D, device=cuda, dtype=BF16)
    k = qkv[:, 8 * D:8 * D + H * D].unflatten(1, (H, D))
    v = qkv[:, 8 * D + H * D:].unflatten(1, (H, D))
    bt, pages = pages_of(lens, np.random.default_rng(0))
    a, c, e = (ops.Int8PagedCache(H, D, pages) for _ in range(3))
    cu, z, bt = t32(np.r_[0, np.cumsum(lens)], cuda), t32([0] * B, cuda), t32(bt, cuda)
    ops.int8_append(a, k, v, cu, z, bt)
    ops.int8_append(c, k.contiguous(), v.contiguous(), cu, z, bt)
    # heads outermost, and strides that 16-byte vectors cannot take (copied)
    odd = torch.empty(T, H, D + 1, device=cuda, dtype=BF16)[..., 1:]
    odd.copy_(v)
    ops.int8_append(e, k.transpose(0, 1).contiguous().transpose(0, 1), odd, cu, z, bt)
    assert torch.equal(a.pool, c.pool) and torch.equal(a.pool, e.pool)


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------
SHAPES = {  # (tokens before, new tokens) of each sequence
    "decode": [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (30, 1), (31, 1), (127, 1), (511, 1),
               (1000, 1)],
    "drafts": [(0, 2), (3, 4), (15, 2), (100, 3), (14, 4), (513, 4)],
    "chunk": [(0, 1), (0, 33), (17, 64), (100, 129), (0, 0), (63, 65), (64, 17)],
    "mixed": [(700, 1), (0, 140), (33, 0), (5, 1), (259, 31), (90, 2)],
}


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("Hq,H,D,dt", [(8, 8, 64, "f16"), (8, 2, 128, "bf16"), (14, 2, 128, "f16"),
                                       (16, 2, 64, "bf16"), (17, 1, 128, "bf16"), (40, 1, 64, "f16")])
@pytest.mark.parametrize("window", [0, 1, 19, 300])
def test_attention(ops, cuda, shape, Hq, H, D, dt, window):
    b = Batch(ops, cuda, *zip(*SHAPES[shape]), H, D, DT[dt], seed=len(shape) + Hq + window)
    b.fill()
    err = err_word(cuda)
    q = b.query(Hq)
    out = b.attend(q, window, err)
    assert err.item() == 0 and out.dtype == DT[dt]
    b.check(q, out, window, rows=6)
    assert torch.equal(out, b.attend(q, window, err))  # the same bits again


@pytest.mark.parametrize("old,new,H,Hq", [([5000], [1], 1, 4), ([20000, 3, 9000], [1, 1, 1], 2, 8),
                                          ([6001], [40], 2, 8), ([9000, 100], [33, 1], 1, 8),
                                          ([700] * 40, [1] * 40, 8, 32), ([40], [700], 1, 8)])
@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16")])
def test_attention_over_long_contexts(ops, cuda, old, new, H, Hq, D, dt):
    b = Batch(ops, cuda, old, new, H, D, DT[dt], seed=1)
    b.fill()
    q = b.query(Hq)
    out = b.attend(q)
    b.check(q, out, rows=3)
    assert torch.equal(out, b.attend(q))


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("wild", [100.0, 2.0 ** 9])
def test_value_rows_of_very_different_sizes(ops, cuda, new, wild):
    """Rows from 1/wild to wild times the ordinary size."""
    b = Batch(ops, cuda, [300, 77], [new, new], 2, 128, BF16, seed=9, wild=wild)
    b.fill()
    q = b.query(8, mult=0.3)
    b.check(q, b.attend(q), rows=8)


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -14, 2.0 ** 14, 2.0 ** 60])
def test_values_far_from_one(ops, cuda, new, size):
    """All values tiny or huge: bf16 holds them, fp16 weights must not flush."""
    b = Batch(ops, cuda, [200], [new], 1, 128, BF16, seed=11)
    b.v = (b.v.float() * size).to(BF16)
    b.fill()
    q = b.query(4)
    b.check(q, b.attend(q), rows=8)


@pytest.mark.parametrize("new", [1, 50])
def test_large_and_small_queries(ops, cuda, new):
    """bf16 queries outside the range of fp16, keys that bring them back."""
    for size in (2.0 ** 40, 2.0 ** -40):
        b = Batch(ops, cuda, [200], [new], 1, 128, BF16, seed=12)
        b.k = (b.k.float() / size).to(BF16)
        b.fill()
        q = b.query(4, mult=size)
        b.check(q, b.attend(q), rows=8)


@pytest.mark.parametrize("new", [1, 3, 60])
def test_rising_scores_and_zero_rows(ops, cuda, new):
    """Every score larger than the last (each tile moves the maximum); zero keys
    and values among them."""
    b = Batch(ops, cuda, [400], [new], 1, 64, F16, seed=13)
    n = int(b.lens[0])
    ramp = torch.linspace(0.0, 3.0, n, device=cuda)
    b.k = (torch.ones_like(b.k) * ramp[:, None, None]).to(F16)
    b.v[::7] = 0
    b.k[5::11] = 0
    b.fill()
    q = torch.full((new, 4, 64), 1.5, device=cuda, dtype=F16)
    b.check(q, b.attend(q), rows=8)


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_values_reach_only_the_rows_that_see_them(ops, cuda, what, bad):
    """A key or value that is no number, at position 70 of 100: rows before it
    and rows whose window has passed it are untouched."""
    def outs(window, spoil):
        b = Batch(ops, cuda, [20], [80], 1, 128, BF16, seed=4)
        if spoil:
            getattr(b, what)[70, 0, 3] = bad
        b.fill()
        b.rng = np.random.default_rng(5)
        return b.attend(b.query(4), window)
    for window in (0, 10):
        good, got = outs(window, False), outs(window, True)
        seen = torch.zeros(80, dtype=torch.bool, device=cuda)
        seen[50:] = True  # positions 70 ..
        if window:
            seen[60:] = False  # 70 left the window of position 80
        assert torch.equal(got[~seen], good[~seen])
        assert got[seen].isnan().all()


def test_one_token_sequences_return_their_value(ops, cuda):
    """The one weight is its row's scale rounded to fp16, 2^-11 of it at most, so
    the output is the value within that and its own rounding; every q head of a
    kv head gets the same bits."""
    b = Batch(ops, cuda, [0] * 9, [1] * 9, 2, 128, F16, seed=6)
    b.fill()
    q = b.query(8)
    out = b.attend(q)
    b.check(q, out)
    _, v = ops.int8_read(b.cache, b.bt_t, t32([0] * 9, cuda), t32(range(10), cuda), 9, dtype=F32)
    want = f64(v.repeat_interleave(4, 1))
    assert (np.abs(f64(out) - want) <= np.abs(want) * 2.0 ** -10 * 1.01 + 2.0 ** -25).all()
    assert torch.equal(out[:, ::4].repeat_interleave(4, 1), out)


def test_rows_of_no_sequence_stay(ops, cuda):
    b = Batch(ops, cuda, [5, 40, 9], [3, 0, 20], 1, 64, BF16, seed=7)
    b.fill()
    q = torch.cat([b.query(4), torch.full((6, 4, 64), float("nan"), device=cuda, dtype=BF16)])
    out = torch.full_like(q, 3.0)
    b.attend(q, out=out)
    b.check(q[:23], out[:23])
    assert (out[23:] == 3).all()


@pytest.mark.parametrize("new", [1, 3, 40])
def test_pages_that_the_window_has_passed_may_be_gone(ops, cuda, new):
    b = Batch(ops, cuda, [700, 333], [new, new], 1, 128, BF16, seed=14)
    b.fill()
    q = b.query(8)
    want = b.attend(q, 50)
    for s in (0, 1):
        b.bt[s, :(b.old[s] - 50 + 1) // PAGE] = -1
    b.bt_t = t32(b.bt, cuda)
    err = err_word(cuda)
    assert torch.equal(b.attend(q, 50, err), want) and err.item() == 0


def test_strided_queries_and_output_types(ops, cuda):
    b = Batch(ops, cuda, [50, 3], [1, 30], 2, 128, BF16, seed=8)
    b.fill()
    q = b.query(8)
    want = b.attend(q)
    wide = torch.zeros(31, 12, 128, device=cuda, dtype=BF16)
    wide[:, 2:10] = q
    assert torch.equal(b.attend(wide[:, 2:10]), want)
    assert torch.equal(b.attend(q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    odd = torch.zeros(31, 8, 132, device=cuda, dtype=BF16)[..., 4:]
    odd.copy_(q)
    assert torch.equal(b.attend(odd), want)
    half = b.attend(q, out_dtype=F16)
    b.check(q, half)
    q16 = q.to(F16)
    b.check(q16, b.attend(q16, out_dtype=BF16))


def test_bad_lengths_and_tables_are_flagged(ops, cuda):
    old, new = [40, 17, 100, 33], [2, 17, 30, 1]
    b = Batch(ops, cuda, old, new, 1, 64, F16, seed=10)
    b.fill()
    q = b.query(4)
    good = b.attend(q)

    def run(lens=None, cu=None, bt=None, mq=30, ml=130, mb=None):
        err = err_word(cuda)
        out = torch.full_like(q, 9.0)
        ops.int8_attend(b.cache, q, t32(b.cu if cu is None else cu, cuda),
                        b.bt_t if bt is None else t32(bt, cuda),
                        t32(b.lens if lens is None else lens, cuda), max_q_tokens=mq,
                        max_context_len=ml, out=out, err=err)
        return out, err.item()

    same = lambda out, rows: all(  # noqa: E731
        torch.equal(out[b.cu[s]:b.cu[s + 1]], good[b.cu[s]:b.cu[s + 1]]) for s in rows)
    kept = lambda out, s: bool((out[b.cu[s]:b.cu[s + 1]] == 9).all())  # noqa: E731
    out, e = run()
    assert e == 0 and torch.equal(out, good)
    for bad in (16, -5, 2 ** 31 - 1, 131):  # shorter than its chunk, negative, past the bounds
        out, e = run(lens=[42, bad, 130, 34])
        assert e == L.TKV_ERR_BAD_LENGTH and kept(out, 1) and same(out, (0, 2, 3))
    out, e = run(mq=29)
    assert e == L.TKV_ERR_BAD_LENGTH and kept(out, 2) and same(out, (0, 1, 3))
    out, e = run(cu=[0, 2, 19, 49, 51])  # past the last row
    assert e == L.TKV_ERR_BAD_LENGTH and kept(out, 3) and same(out, (0, 1, 2))
    out, e = run(bt=b.bt[:, :8], ml=144)
    assert e == L.TKV_ERR_BAD_LENGTH and kept(out, 2) and same(out, (0, 1, 3))
    for bad in (-1, b.pages, 2 ** 31 - 1, -2 ** 31):
        bt = b.bt.copy()
        bt[2, 3] = bad
        out, e = run(bt=bt)
        assert e == L.TKV_ERR_BAD_PAGE and same(out, (0, 1, 3))
        # append: its token is not written, the others are
        err = err_word(cuda)
        c = ops.Int8PagedCache(1, 64, b.pages)
        ops.int8_append(c, b.k, b.v, t32(b.cu_all, cuda), t32([0] * 4, cuda), t32(bt, cuda), err=err)
        assert err.item() == L.TKV_ERR_BAD_PAGE
        missing = torch.zeros(b.pages, dtype=torch.bool)
        missing[int(b.bt[2, 3])] = True
        missing[[p for p in range(b.pages) if p not in b.bt]] = True
        assert not c.pool[missing.to(cuda)].any()
        written = b.bt[b.bt >= 0]
        full = [int(p) for p in written if p not in (b.bt[0, 2], b.bt[1, 2], b.bt[2, 8], b.bt[3, 2])
                and p != b.bt[2, 3]]
        assert torch.equal(c.pool[full], b.pool[full])
        err = err_word(cuda)
        k, v = ops.int8_read(c, t32(bt, cuda), t32([0] * 4, cuda), t32(b.cu_all, cuda),
                             int(b.cu_all[-1]), err=err)
        at = int(b.cu_all[2]) + 48
        assert err.item() == L.TKV_ERR_BAD_PAGE and not k[at:at + 16].any() and not v[at:at + 16].any()
        assert k[at - 1].any() and k[at + 16].any()
    # append and read: lengths
    for cu, old_, t in (([0, 5, 3], [0, 0], 8), ([0, 4, 9], [0, 0], 8), ([0, 4, 8], [-1, 0], 8),
                        ([0, 4, 8], [125, 0], 8), ([-1, 4, 8], [0, 0], 8)):
        c = ops.Int8PagedCache(1, 64, 20)
        err = err_word(cuda)
        bt = t32(np.arange(16).reshape(2, 8), cuda)
        ops.int8_append(c, b.k[:t], b.v[:t], t32(cu, cuda), t32(old_, cuda), bt, err=err)
        assert err.item() == L.TKV_ERR_BAD_LENGTH
        assert not c.pool[16:].any()
        err = err_word(cuda)
        ops.int8_read(c, bt, t32(old_, cuda), t32(cu, cuda), t, err=err)
        assert err.item() == L.TKV_ERR_BAD_LENGTH


def test_wrapper_refusals(ops, cuda):
    b = Batch(ops, cuda, [4], [2], 2, 64, F16)
    q = b.query(4)
    i, z = t32([0, 2], cuda), t32([4], cuda)
    with pytest.raises(ValueError):
        b.attend(q.float())
    with pytest.raises(ValueError):
        b.attend(q[..., :32])
    with pytest.raises(ValueError):
        b.attend(q, out=torch.empty(2, 4, 64, device=cuda))
    with pytest.raises(ValueError):
        b.attend(q, out=torch.empty(3, 4, 64, device=cuda, dtype=F16))
    with pytest.raises(ValueError):
        ops.int8_attend(b.cache, q, i.long(), b.bt_t, z)
    with pytest.raises(ValueError):
        ops.int8_attend(b.cache, q, i, b.bt_t, t32([4, 4], cuda))
    with pytest.raises(ValueError, match="gradient"):
        b.attend(q.clone().requires_grad_())
    with pytest.raises(ValueError):
        b.attend(q[:, :3])
    with pytest.raises(L.TkvError):
        b.attend(q, workspace=torch.zeros(16, dtype=torch.uint8, device=cuda))
    with pytest.raises(ValueError):
        ops.int8_append(b.cache, b.k, b.v[:, :1], i, z, b.bt_t)
    with pytest.raises(ValueError):
        ops.int8_append(b.cache, b.k, b.v.to(BF16), i, z, b.bt_t)
    with pytest.raises(ValueError):
        ops.int8_read(b.cache, b.bt_t, z, i, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.Int8PagedCache(2, 64, pool=b.pool[:, :, :-1])


# --------------------------------------------------------------------------
# the set together
# --------------------------------------------------------------------------
@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16")])
def test_prefill_then_decode_steps(ops, cuda, D, dt):
    """Rotate, append, attend: a ragged prefill, then steps of one token on
    captured graphs; every step against dense attention in 64 bits."""
    H, Hq, steps = 2, 8, 5
    new = np.array([37, 1, 130, 16])
    B = len(new)
    rng = np.random.default_rng(0)
    bt, pages = pages_of(new + steps + 1, rng)
    bt_t = t32(bt, cuda)
    cache = ops.Int8PagedCache(H, D, pages)
    sections = (D // 8, D // 8, D // 4)
    ws = ops.int8_workspace(B, Hq, H, D, int(new.max()), 200)
    b = Batch(ops, cuda, [0] * B, new, H, D, DT[dt])  # only its check()
    b.cache, b.pool, b.bt, b.bt_t = cache, cache.pool, bt, bt_t

    def tokens(n):
        mk = lambda h: torch.tensor(rng.standard_normal((n, h, D)), dtype=torch.float32,  # noqa: E731
                                    device=cuda).to(DT[dt])
        return mk(Hq), mk(H), mk(H)

    def step(q, k, v, pos, cu, old, lens, mq):
        qr, kr = ops.rope_axes(q, k, pos, sections, theta=500000.0)
        ops.int8_append(cache, kr, v, cu, old, bt_t, max_new_tokens=mq)
        return qr, kr, ops.int8_attend(cache, qr, cu, bt_t, lens, max_q_tokens=mq,
                                       max_context_len=200, workspace=ws)

    T = int(new.sum())
    pos = np.concatenate([np.arange(n) for n in new])
    q, k, v = tokens(T)
    qr, kr, out = step(q, k, v, t32(np.tile(pos, (3, 1)), cuda), t32(np.r_[0, np.cumsum(new)], cuda),
                       t32([0] * B, cuda), t32(new, cuda), int(new.max()))
    b.old, b.new, b.lens, b.cu = np.zeros(B, int), new, new, np.r_[0, np.cumsum(new)]
    b.check(qr, out, rows=8)
    rb, _ = ops.int8_read(cache, bt_t, t32([0] * B, cuda), t32(b.cu, cuda), T, dtype=F32)
    want, d = quantise(f64(kr))
    assert np.array_equal(f64(rb), (want * d.astype(np.float64)).astype(np.float32).astype(np.float64))

    # one decode step, captured once and replayed
    q, k, v = (x.clone() for x in tokens(B))
    pos_t, old_t, len_t = t32(np.tile(new, (3, 1)), cuda), t32(new, cuda), t32(new + 1, cuda)
    cu = t32(range(B + 1), cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, v, pos_t, cu, old_t, len_t, 1)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        qr, kr, out = step(q, k, v, pos_t, cu, old_t, len_t, 1)
    for s in range(steps):
        for dst, src in zip((q, k, v), tokens(B)):
            dst.copy_(src)
        pos_t.copy_(t32(np.tile(new + s, (3, 1)), cuda))
        old_t.copy_(t32(new + s, cuda))
        len_t.copy_(t32(new + s + 1, cuda))
        g.replay()
        b.old, b.new, b.lens, b.cu = new + s, np.ones(B, int), new + s + 1, np.arange(B + 1)
        b.check(qr, out)
    eager = ops.int8_attend(cache, qr, cu, bt_t, len_t, max_q_tokens=1, max_context_len=200)
    assert torch.equal(eager, out)


def test_calls_on_other_streams(ops, cuda):
    """A stream handed to the call (as a torch stream and as its address), with
    inputs that the wrappers copy first."""
    b = Batch(ops, cuda, [300, 20, 7], [1, 60, 1], 2, 128, BF16, seed=2)
    b.fill()
    q = b.query(8)
    want = b.attend(q)
    k0, v0 = ops.int8_read(b.cache, b.bt_t, t32([0] * 3, cuda), t32(b.cu_all, cuda), int(b.cu_all[-1]))
    s = torch.cuda.Stream()
    odd = torch.zeros(62, 8, 130, device=cuda, dtype=BF16)[..., 1:-1]
    odd.copy_(q)
    for stream in (s, s.cuda_stream):
        s.wait_stream(torch.cuda.current_stream())
        c = ops.Int8PagedCache(2, 128, b.pages)
        s.wait_stream(torch.cuda.current_stream())
        cu, z = t32(b.cu_all, cuda), t32([0] * 3, cuda)
        lens, cuq = t32(b.lens, cuda), t32(b.cu, cuda)
        s.wait_stream(torch.cuda.current_stream())
        ops.int8_append(c, b.k, b.v, cu, z, b.bt_t, stream=stream)
        k, v = ops.int8_read(c, b.bt_t, z, cu, int(b.cu_all[-1]), stream=stream)
        out = ops.int8_attend(c, odd, cuq, b.bt_t, lens, max_q_tokens=60, max_context_len=301,
                              stream=stream)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(k, k0) and torch.equal(v, v0)


def test_two_calls_at_once(ops, cuda):
    """Decode calls on two streams, each with its workspace, many times over."""
    bs = [Batch(ops, cuda, [4000, 700], [1, 1], 2, 128, BF16, seed=i) for i in (1, 2)]
    for b in bs:
        b.fill()
    qs = [b.query(8) for b in bs]
    want = [b.attend(q) for b, q in zip(bs, qs)]
    ws = [ops.int8_workspace(2, 8, 2, 128, 1, 4001) for _ in bs]
    args = [(b.cache, q, t32(b.cu, cuda), b.bt_t, t32(b.lens, cuda), 1, 4001)
            for b, q in zip(bs, qs)]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            got[i].append(ops.int8_attend(*args[i], workspace=ws[i], stream=streams[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_one_workspace_serves_smaller_calls(ops, cuda):
    """A workspace sized for the largest call, for calls of other shapes one
    after the other."""
    shapes = [([2500, 9], [1, 1]), ([100, 60], [20, 1]), ([1999, 3], [40, 40]), ([2500, 9], [1, 1])]
    ws = ops.int8_workspace(2, 8, 2, 128, 64, 2600)
    for i, (old, new) in enumerate(shapes):
        b = Batch(ops, cuda, old, new, 2, 128, BF16, seed=i)
        b.fill()
        q = b.query(8)
        out = ops.int8_attend(b.cache, q, t32(b.cu, cuda), b.bt_t, t32(b.lens, cuda),
                              max_q_tokens=64, max_context_len=2600, workspace=ws)
        b.check(q, out, rows=4)


def test_a_workspace_shared_by_calls_of_very_different_sizes(ops, cuda):
    """Few pairs with many runs, many pairs with few, chunks: in turn, twice."""
    shapes = [([20000], [1], 1, 8), ([600] * 40, [1] * 40, 4, 8), ([900, 40], [50, 3], 1, 4),
              ([9, 3000], [1, 1], 2, 32)]
    bs, need = [], 0
    for i, (old, new, H, Hq) in enumerate(shapes):
        b = Batch(ops, cuda, old, new, H, 64, BF16, seed=i)
        b.fill()
        bs.append((b, b.query(Hq)))
        need = max(need, ops.int8_workspace_bytes(len(old), Hq, H, 64, max(new), int(b.lens.max())))
    ws = torch.zeros(need, dtype=torch.uint8, device=cuda)
    for _ in range(2):
        for b, q in bs:
            assert torch.equal(b.attend(q, workspace=ws), b.attend(q))


def test_no_tokens(ops, cuda):
    b = Batch(ops, cuda, [4, 0], [0, 0], 1, 64, F16)
    q = torch.empty(0, 4, 64, device=cuda, dtype=F16)
    assert ops.int8_attend(b.cache, q, t32([0, 0, 0], cuda), b.bt_t, t32([4, 0], cuda)).shape == q.shape
    ops.int8_append(b.cache, q[:, :1], q[:, :1], t32([0, 0, 0], cuda), t32([4, 0], cuda), b.bt_t)
    k, v = ops.int8_read(b.cache, b.bt_t, t32([0, 0], cuda), t32([0, 0, 0], cuda), 0)
    assert k.shape == v.shape == (0, 1, 64)


def test_a_pool_past_4_gib(ops, cuda):
    """Pages whose byte offsets pass 32 bits."""
    H, D = 8, 128
    pages = (1 << 32) // (H * block_bytes(D)) + 40
    cache = ops.Int8PagedCache(H, D, pool=torch.full((pages, H, block_bytes(D)), 255,
                                                     dtype=torch.uint8, device=cuda))
    bt = np.array([[pages - 1, 0, pages - 2]])
    n = 40
    k = torch.randn(n, H, D, device=cuda, dtype=BF16)
    v = torch.randn(n, H, D, device=cuda, dtype=BF16)
    cu, z, bt_t = t32([0, n], cuda), t32([0], cuda), t32(bt, cuda)
    ops.int8_append(cache, k, v, cu, z, bt_t)
    small = ops.Int8PagedCache(H, D, 3)
    ops.int8_append(small, k, v, cu, z, t32([[0, 1, 2]], cuda))
    assert torch.equal(cache.pool[[pages - 1, 0]], small.pool[:2])
    for got, want in zip(ops.int8_read(cache, bt_t, z, cu, n),
                         ops.int8_read(small, t32([[0, 1, 2]], cuda), z, cu, n)):
        assert torch.equal(got, want)
    q = torch.randn(n, 32, D, device=cuda, dtype=BF16)
    for r in (slice(0, n), slice(n - 1, n)):
        m = q[r].shape[0]
        a = ops.int8_attend(cache, q[r], t32([0, m], cuda), bt_t, t32([n], cuda))
        c = ops.int8_attend(small, q[r], t32([0, m], cuda), t32([[0, 1, 2]], cuda), t32([n], cuda))
        assert torch.equal(a, c)


# --------------------------------------------------------------------------
# how work is shared out
# --------------------------------------------------------------------------
@pytest.mark.parametrize("H", [5, 8, 20])
@pytest.mark.parametrize("D,dt", [(64, "f16"), (128, "bf16")])
def test_several_heads_a_cta(ops, cuda, H, D, dt):
    """Long calls, in which a CTA takes several kv heads one after another (and a
    last CTA fewer), leave the bytes and values of short ones."""
    lens = [0, 4093, 1, 2500, 16, 31]
    b = Batch(ops, cuda, [0] * len(lens), lens, H, D, DT[dt], seed=H)
    b.fill()
    whole = b.pool.clone()
    b.pool.fill_(255)
    for i, n in enumerate(lens):
        for at in range(0, n, 60):
            m = min(60, n - at)
            rows = slice(int(b.cu_all[i]) + at, int(b.cu_all[i]) + at + m)
            ops.int8_append(b.cache, b.k[rows], b.v[rows], t32([0, m], cuda), t32([at], cuda),
                            b.bt_t[i:i + 1])
    assert torch.equal(whole, b.pool)
    T, z = sum(lens), t32([0] * len(lens), cuda)
    ko, vo = ops.int8_read(b.cache, b.bt_t, z, t32(b.cu_all, cuda), T, dtype=BF16)
    # outputs that start 16 bytes off a sector
    raw = [torch.zeros(T * H * D + 8, dtype=BF16, device=cuda) for _ in range(2)]
    k1, v1 = (x[8:].view(T, H, D) for x in raw)
    ops.int8_read(b.cache, b.bt_t, z, t32(b.cu_all, cuda), T, k_out=k1, v_out=v1)
    assert torch.equal(k1, ko) and torch.equal(v1, vo)
    for i, n in enumerate(lens):
        for at in range(0, n, 999):
            m = min(60, n - at)
            rows = slice(int(b.cu_all[i]) + at, int(b.cu_all[i]) + at + m)
            kk, vv = ops.int8_read(b.cache, b.bt_t[i:i + 1], t32([at], cuda), t32([0, m], cuda), m,
                                   dtype=BF16)
            assert torch.equal(kk, ko[rows]) and torch.equal(vv, vo[rows])


def test_one_token_of_many_sequences(ops, cuda):
    """A decode step's append and read-back: more sequences than tokens / 16."""
    B, H, D = 700, 2, 64
    rng = np.random.default_rng(5)
    old = rng.integers(0, 40, B)
    new = (rng.random(B) < 0.8).astype(int)
    b = Batch(ops, cuda, old, new, H, D, BF16, seed=5)
    b.fill()
    want = b.pool.clone()
    last = torch.tensor(b.cu_all[1:][new > 0] - 1, device=cuda, dtype=torch.long)
    pages, slots = b.bt[np.arange(B), np.maximum(b.lens - 1, 0) // PAGE], (b.lens - 1) % PAGE
    kc, vc, s = unpack(want.cpu().numpy(), D)
    for other in (True, False):  # another token's rows first
        k, v = (x[last].flip(-1) * 3 if other else x[last] for x in (b.k, b.v))
        ops.int8_append(b.cache, k, v, t32(b.cu, cuda), t32(old, cuda), b.bt_t, max_new_tokens=1)
        assert torch.equal(b.pool, want) != other
    ko, vo = ops.int8_read(b.cache, b.bt_t, t32(old, cuda), t32(b.cu, cuda), int(new.sum()),
                           max_tokens=1, dtype=F32)
    for j, i in enumerate(np.flatnonzero(new)):
        p, t = pages[i], slots[i]
        for h in range(H):
            assert np.array_equal(f64(ko[j, h]), np.float64(np.float32(kc[p, h, t]) * s[p, h, t, 0]))
            assert np.array_equal(f64(vo[j, h]), np.float64(np.float32(vc[p, h, t]) * s[p, h, t, 1]))


@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16")])
@pytest.mark.parametrize("window", [0, 200])
def test_decode_ranges_across_sequences(ops, cuda, D, dt, window):
    """CTAs whose range of the steps begins and ends inside contexts and spans short
    ones, sequences without tokens and, more than 32 in a row, chunks."""
    rng = np.random.default_rng(11)
    old = np.r_[rng.integers(0, 700, 60), [0] * 40, [9000, 1, 0, 2500], rng.integers(0, 300, 100)]
    new = np.r_[np.ones(60, int), [17] * 40, [1, 0, 1, 1], rng.integers(0, 2, 100)]
    b = Batch(ops, cuda, old, new, 2, D, DT[dt], seed=9)
    b.fill()
    q = b.query(8)
    err = err_word(cuda)
    out = b.attend(q, window=window, err=err)
    b.check(q, out, window=window, rows=3)
    assert err.item() == 0
    assert torch.equal(out, b.attend(q, window=window))


@pytest.mark.parametrize("n", [1, 3])
def test_rows_at_odd_strides_and_addresses(ops, cuda, n):
    """Rows that 16-byte vectors cannot address are copied, a single token's too."""
    H, D, old = 2, 64, 20
    b = Batch(ops, cuda, [old], [n], H, D, F16, seed=n)
    b.fill()
    want = b.pool.clone()
    q = b.query(4)
    out = b.attend(q)
    for off in (0, 1):
        raw = torch.zeros(n, 4 * D + 3, dtype=F16, device=cuda)
        at = lambda x: raw[:, off:off + x[0].numel()].unflatten(1, x.shape[1:]).copy_(x)  # noqa: E731
        assert torch.equal(b.attend(at(q)), out)
        b.pool.copy_(want)
        k, v = at(b.k[old:]), b.v[old:]
        b.pool[b.bt[0, old // PAGE]] = 3  # the page of the last tokens, but for its first ones
        ops.int8_append(b.cache, b.k[16:old], b.v[16:old], t32([0, old - 16], cuda), t32([16], cuda),
                        b.bt_t)
        ops.int8_append(b.cache, k, v, t32([0, n], cuda), t32([old], cuda), b.bt_t)
        kc, vc, s = unpack(b.pool.cpu().numpy(), D)
        kw, vw, sw = unpack(want.cpu().numpy(), D)
        p, t = b.bt[0, old // PAGE], slice(0, old - 16 + n)
        for x, y in ((kc, kw), (vc, vw), (s, sw)):
            assert np.array_equal(x[p][:, t], y[p][:, t])


@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16")])
def test_graphs_that_share_a_workspace_and_change_lengths(ops, cuda, D, dt):
    """A decode call and a call that mixes chunks and decodes, captured on one
    workspace, replayed in turn with other lengths and shares of the rows."""
    B, H, Hq = 5, 2, 8
    b = Batch(ops, cuda, [900, 300, 2000, 64, 1500], [80] * B, H, D, DT[dt], seed=2)
    b.fill()
    ws = ops.int8_workspace(B, Hq, H, D, 80, 2100)
    q1, q2 = (torch.randn(n, Hq, D, device=cuda).to(DT[dt]) for n in (B, 120))
    lens, cu1, cu2 = t32(b.lens, cuda), t32(range(B + 1), cuda), t32([0, 80, 81, 85, 118, 120], cuda)
    call = lambda q, cu, n, w: ops.int8_attend(b.cache, q, cu, b.bt_t, lens, max_q_tokens=n,  # noqa: E731
                                               max_context_len=2100, workspace=w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(q1, cu1, 1, ws), call(q2, cu2, 80, ws)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for q, cu, n in ((q1, cu1, 1), (q2, cu2, 80)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(q, cu, n, ws)
        graphs.append((g, out, q, cu, n))
    for length, share in (([980, 380, 2080, 144, 1580], [0, 80, 81, 85, 118, 120]),
                          ([90, 91, 2080, 100, 82], [0, 1, 2, 79, 80, 120]),
                          ([980, 17, 1, 144, 700], [0, 80, 97, 98, 119, 120])):
        lens.copy_(t32(length, cuda))
        cu2.copy_(t32(share, cuda))
        for g, out, q, cu, n in graphs * 2:
            out.fill_(3)
            g.replay()
            assert torch.equal(out, call(q, cu, n, None))
        b.lens, b.cu = np.array(length), np.array(share)
        b.new = np.diff(b.cu)
        b.old = b.lens - b.new
        b.check(q2, graphs[1][1], rows=5)


def test_append_at_the_smallest_scales(ops, cuda):
    """bf16 rows whose scale is the smallest normal float and a little more (or
    below it, which counts as none), every mantissa of the largest value."""
    D, n = 64, 4 * 128
    rng = np.random.default_rng(6)
    x = rng.integers(-255, 256, (n, D)) * 2.0 ** rng.integers(-7, 1, (n, D))
    x[:, 0] = np.repeat(np.arange(128, 256), 4)
    x *= 2.0 ** np.tile([-126, -127, -125, -128], 128)[:, None]
    t = torch.tensor(x, dtype=torch.float64, device=cuda).to(BF16)[:, None]
    cache = ops.Int8PagedCache(1, D, n // PAGE)
    ops.int8_append(cache, t, t.flip(0), t32([0, n], cuda), t32([0], cuda),
                    t32([list(range(n // PAGE))], cuda))
    kc, vc, s = unpack(cache.pool.cpu().numpy(), D)
    want, d = quantise(f64(t))
    assert (d == 0).any() and (d > 0).any()
    flat = lambda c: c.transpose(0, 2, 1, 3).reshape(n, -1)  # noqa: E731
    assert np.array_equal(flat(kc), want[:, 0]) and np.array_equal(flat(vc)[::-1], want[:, 0])
    assert np.array_equal(flat(s)[:, :1], d[:, 0])
