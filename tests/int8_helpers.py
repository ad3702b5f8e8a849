"""The paged int8 cache and the rotary step in numpy, 64 bits: what the GPU
tests compare with."""
import math

import numpy as np
import torch

PAGE = 16
# off by at most half a step: a rounding to this type, relative to the value
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def quantise(x: np.ndarray):
    """Codes and scales of [..., D] values that fp16 / bf16 hold."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = (np.abs(x).max(-1, keepdims=True) / 127).astype(np.float32)
        d[np.abs(d) < np.finfo(np.float32).tiny] = 0
        d[~np.isfinite(np.abs(x).max(-1, keepdims=True))] = np.nan
        q = x / d.astype(np.float64)
        code = np.where((d > 0) & np.isfinite(d), np.rint(q), 0)
    return code.astype(np.int64), d


def block_bytes(D: int) -> int:
    return 32 * D + 128


def unpack(pool: np.ndarray, D: int):
    """K codes, V codes [pages, H, 16, D] and scales [pages, H, 16, 2] of a pool."""
    n, H, _ = pool.shape
    k = np.zeros((n, H, PAGE, D), np.int64)
    v = np.zeros((n, H, PAGE, D), np.int64)
    for t in range(PAGE):
        for c in range(D):
            ch = c // 16
            k[:, :, t, c] = pool[:, :, ch * 256 + (t ^ (2 * (ch % 4))) * 16 + c % 16]
            u, g, j = c // 32, c % 32 // 4, c % 4
            v[:, :, t, c] = pool[:, :, 16 * D + ((u * 8 + g) * 4 + t // 4) * 16 + 4 * j + t % 4]
    s = np.ascontiguousarray(pool[:, :, 32 * D:]).view(np.float32).reshape(n, H, PAGE, 2)
    return k - 128, v - 128, s


def pages_of(lengths, rng, spare=3):
    """Block tables of sequences of these lengths in a shuffled pool; pages in all."""
    need = [(n + PAGE - 1) // PAGE for n in lengths]
    pages = sum(need) + spare
    order = rng.permutation(pages).astype(np.int32)
    bt = np.full((len(lengths), max(1, max(need, default=1))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n]
        at += n
    return bt, pages


def attention(q, k, v, pos, scale, window):
    """out, and the sizes its error bound needs, of one sequence in 64 bits: q
    [n, Hq, D] at positions pos [n], k, v [L, H, D]; also A = sum p |v| / l, S =
    scale * max over seen tokens of sum |q_c k_c|, and M = tokens * max |v|."""
    n, Hq, D = q.shape
    L, H, _ = k.shape
    grp = Hq // H
    out = np.zeros((n, Hq, D))
    A = np.zeros((n, Hq, D))
    S = np.zeros((n, Hq, 1))
    M = np.abs(v).max() * L
    for i in range(n):
        lo = max(0, pos[i] - window + 1) if window else 0
        t = np.arange(lo, pos[i] + 1)
        for h in range(Hq):
            kk, vv = k[t, h // grp], v[t, h // grp]
            x = kk @ q[i, h] * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h] = p @ vv
            A[i, h] = p @ np.abs(vv)
            S[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return out, A, S, M


def attention_bound(out, A, S, M, D, out_dtype):
    """How far the kernels may be: the output's own rounding; the weights'
    rounding to fp16 (half a step of each, so of A); the scores' 32-bit sums of
    D + 8 terms, twice for truncating adders, and queries rounded to 2^-25 of
    their largest (an error e of a score is a factor 1 + e of its weight, and of
    the sum's); and 2^-20 for the exponentials, scales and sums.  Below the
    normal range fp16 has steps of 2^-24, so half a step is 2^-25 absolute: for
    an fp16 output directly; for a weight, which is held times 2^5 and times its
    row's scale over at most twice the largest scale, it is 2^-25 2^-5 2 max|v|
    of the output, for each token at most: M 2^-29."""
    e = S * ((D + 8) * 2.0 ** -23 + D * 2.0 ** -25)
    return HALF_STEP[out_dtype] * np.abs(out) + A * (2.0 ** -11 + 2 * e + 2.0 ** -20) * 1.01 + (
        M * 2.0 ** -29 + (2.0 ** -25 if out_dtype == torch.float16 else 0) + 1e-30)


def axis_of_pair(sections, order):
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    got, left = [], list(sections)
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def rope(x, positions, sections, theta, order, pairing, inverse=False):
    """x [T, H, D] turned, in 64 bits, and |a| + |b| of each output's pair."""
    y, size = np.array(x, np.float64), np.abs(np.array(x, np.float64))
    r = 2 * sum(sections)
    for p, a in enumerate(axis_of_pair(sections, order)):
        w = positions[a].astype(np.float64) * theta ** (-2.0 * p / r)
        c, s = np.cos(w)[:, None], np.sin(w)[:, None] * (-1 if inverse else 1)
        i, j = (p, p + r // 2) if pairing == "halves" else (2 * p, 2 * p + 1)
        y[..., i] = x[..., i] * c - x[..., j] * s
        y[..., j] = x[..., j] * c + x[..., i] * s
        size[..., i] = size[..., j] = np.abs(x[..., i]) + np.abs(x[..., j])
    return y, size


def scale_of(D):
    return 1.0 / math.sqrt(D)
