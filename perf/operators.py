"""The int8 paged cache, the attention over it and the rotary positions before
it, as measured work: cases, inputs, a plain form, and the library's calls.

Operators (importable as truellm-engine_b200.ops):
  rope_axes    rotary positions with several axes (time, height, width) on q and k
  int8_append  quantises new K/V as they are written into 16-token pages
  int8_read    reads a range of tokens back as dense K/V
  int8_attend  attention of each sequence's last tokens (one or many) over its pages

One (page, kv head) block of the cache, with D channels, is
  K codes  [D/16 chunks][16 slots][16 channels] u8, token t of chunk c in slot t ^ (2 (c % 4))
  V codes  [D/32][8][4][4][4] u8: channel 32 u + 4 g + j of token 4 t + i at [u][g][t][j][i]
  scales   [16 tokens][2] f32 (key, value)
A code u stands for (u - 128) * scale; the scale of a token's D values x is
max|x| / 127 and the codes are round(x / scale), halves to even.
"""
import math
import random

import torch

own = False

PAGE = 16


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # the rotary step of one decode step: one token of 64 sequences
        dict(name="rope-decode", op="rope", T=64, Hq=32, Hkv=8, D=128, rotary=128, axes=3,
             order="blocks", pairing="halves", theta=500000.0, far=8192, dtype="bf16", pick=1),
        # the rotary step of a long image-and-text prefill, an odd number of tokens
        dict(name="rope-prefill", op="rope", T=32771, Hq=32, Hkv=8, D=128, rotary=128, axes=3,
             order="round_robin", pairing="halves", theta=1000000.0, far=131072, dtype="bf16", pick=2),
        # a decode step's 64 new tokens written to 64 sequences, and read back
        dict(name="append-decode", op="append", B=64, nmin=1, nmax=1, lmin=1024, lmax=8192, Hkv=8,
             D=128, dtype="bf16", pick=3),
        # 64 chunks of 2048 tokens written (the chunk of the bulk-append benchmark), and read back
        dict(name="append-chunk", op="append", B=64, nmin=2048, nmax=2048, lmin=0, lmax=100, Hkv=8,
             D=128, dtype="bf16", pick=4),
        # one short prefix brought back to dense fp16, 64-channel heads
        dict(name="read-short", op="read", B=1, nmin=333, nmax=333, lmin=5, lmax=5, Hkv=8, D=64,
             dtype="f16", pick=5),
        # ragged prefixes of 16 sequences brought back to bf16 (moving a cache to another format)
        dict(name="read-prefixes", op="read", B=16, nmin=500, nmax=8192, lmin=0, lmax=64, Hkv=8,
             D=128, dtype="bf16", pick=6),
        # the smallest attention: one token, one sequence, 512 tokens, 8 heads of 64 channels
        dict(name="decode-small", op="attend", B=1, nmin=1, nmax=1, lmin=511, lmax=511, Hq=8, Hkv=8,
             D=64, window=0, dtype="f16", pick=7),
        # a serving step: 64 sequences of 1024 to 8192 tokens, 4 q heads a kv head
        dict(name="decode-batch", op="attend", B=64, nmin=1, nmax=1, lmin=1023, lmax=8191, Hq=32,
             Hkv=8, D=128, window=0, dtype="bf16", pick=8),
        # long contexts: 4 sequences of 131072 tokens, 8 q heads a kv head
        dict(name="decode-long", op="attend", B=4, nmin=1, nmax=1, lmin=131071, lmax=131071, Hq=64,
             Hkv=8, D=128, window=0, dtype="bf16", pick=9),
        # chunked prefill: 8 chunks of 512 tokens, each behind 4096 cached ones
        dict(name="chunk-512", op="attend", B=8, nmin=512, nmax=512, lmin=4096, lmax=4096, Hq=32,
             Hkv=8, D=128, window=0, dtype="bf16", pick=10),
        # a mixed step: decodes, short and long ragged chunks together, a sliding window, fp16
        dict(name="mixed-window", op="attend", B=20, nmin=1, nmax=641, lmin=0, lmax=6000, Hq=32,
             Hkv=8, D=128, window=1000, dtype="f16", pick=11),
        # few rows over a long context: 33 draft tokens checked behind about 60000 cached ones
        dict(name="chunk-few-rows", op="attend", B=2, nmin=33, nmax=33, lmin=50001, lmax=61111, Hq=32,
             Hkv=8, D=128, window=0, dtype="bf16", pick=12),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8, 8])
    pick = rng.randrange(1 << 20)
    if op == "rope":
        rotary = rng.choice([D, D, D // 2])
        return dict(op=op, T=_log(rng, 1, 32768), Hq=Hkv * rng.choice([1, 4, 8]), Hkv=Hkv, D=D,
                    rotary=rotary, axes=rng.choice([1, 2, 3, 3]),
                    order=rng.choice(["blocks", "round_robin"]),
                    pairing=rng.choice(["halves", "adjacent"]),
                    theta=rng.choice([10000.0, 500000.0, 1000000.0]), far=_log(rng, 64, 1 << 20),
                    dtype=dtype, pick=pick)
    if op in ("append", "read"):
        B = _log(rng, 1, 64)
        nmax = _log(rng, 1, max(1, 120000 // B))
        return dict(op=op, B=B, nmin=rng.choice([1, nmax]), nmax=nmax, lmin=0, lmax=_log(rng, 1, 8192),
                    Hkv=Hkv, D=D, dtype=dtype, pick=pick)
    kind = rng.choice(["decode", "decode", "chunk", "mixed"])
    grp = rng.choice([1, 2, 4, 4, 7, 8])
    window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
    if kind == "decode":
        B = _log(rng, 1, 96)
        lmax = _log(rng, 1, min(131071, 300000 // B))
        nmax = rng.choice([1, 1, 1, 2, 4])
        return dict(op=op, B=B, nmin=1, nmax=nmax, lmin=rng.choice([0, lmax // 4, lmax]), lmax=lmax,
                    Hq=Hkv * grp, Hkv=Hkv, D=D, window=window, dtype=dtype, pick=pick)
    B = _log(rng, 1, 12)
    nmax = _log(rng, 2, max(2, 4096 // B))
    lmax = _log(rng, 1, max(2, min(60000, (30 << 20) // (B * nmax))))
    return dict(op=op, B=B, nmin=nmax if kind == "chunk" else 1, nmax=nmax, lmin=lmax // 2, lmax=lmax,
                Hq=Hkv * grp, Hkv=Hkv, D=D, window=window, dtype=dtype, pick=pick)


# --------------------------------------------------------------------------
# shapes of a case (the same for every seed)
# --------------------------------------------------------------------------
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _lengths(case):
    """(tokens already there, new tokens) of every sequence."""
    rng = random.Random(case["pick"])
    old = [rng.randint(case["lmin"], case["lmax"]) for _ in range(case["B"])]
    new = [rng.randint(case["nmin"], case["nmax"]) for _ in range(case["B"])]
    if case["nmin"] == 1 and case["nmax"] > 8:  # a mixed step: half of them decodes
        new = [1 if i % 2 else n for i, n in enumerate(new)]
        new[0] = case["nmax"]
    return old, new


def _sections(rotary, axes):
    """Frequency pairs of each axis: a quarter to the first, the rest shared, as the sum of all pairs."""
    n = rotary // 2
    if axes == 1:
        return (n,)
    if axes == 2:
        return (n // 2, n - n // 2)
    a = n // 4
    return (a, (n - a) // 2, n - a - (n - a) // 2)


def _axis_of_pair(sections, order):
    """Which axis turns each frequency pair: runs of pairs, or the axes in turn while they have pairs left."""
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, got = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def _visible(case):
    """(pairs of a query and a key that it sees, cached tokens that some query sees)."""
    w, pairs, seen = case["window"], 0, 0
    for o, n in zip(*_lengths(case)):
        L = o + n
        if w and w < L:
            pairs += sum(min(w, o + i + 1) for i in range(n))
            seen += min(L, w + n - 1)
        else:
            pairs += n * o + n * (n + 1) // 2
            seen += L
    return pairs, seen


def work(case):
    D = case["D"]
    if case["op"] == "rope":
        rows = case["T"] * (case["Hq"] + case["Hkv"])
        return {"bytes": rows * D * 4 + case["T"] * case["axes"] * 4, "flops": rows * case["rotary"] * 3}
    old, new = _lengths(case)
    T, H = sum(new), case["Hkv"]
    if case["op"] == "append":  # dense read, codes and scales written; then codes read, dense written
        return {"bytes": T * H * 2 * (2 * D + (D + 4) + (D + 4) + 2 * D), "flops": T * H * 2 * D * 6}
    if case["op"] == "read":
        return {"bytes": T * H * 2 * ((D + 4) + 2 * D), "flops": T * H * 2 * D * 2}
    pairs, seen = _visible(case)
    return {"bytes": seen * H * 2 * (D + 4) + 2 * T * case["Hq"] * D * 2 + 4 * (seen // PAGE),
            "flops": 4 * D * case["Hq"] * pairs}


# --------------------------------------------------------------------------
# the cache's layout, in plain torch
# --------------------------------------------------------------------------
def _layout(D, device):
    """Byte of token t, channel c in the K codes and in the V codes of a block: [16, D] each."""
    t = torch.arange(PAGE, device=device)[:, None]
    c = torch.arange(D, device=device)[None, :]
    chunk = c // 16
    k = chunk * 256 + (t ^ (2 * (chunk % 4))) * 16 + c % 16
    v = ((c // 32) * 32 + (c % 32 // 4) * 4 + t // 4) * 16 + (c % 4) * 4 + t % 4
    return k, v


def _quantise(x):
    """Codes (1 .. 255 around 128) and 32-bit scales of [..., D] values."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()
    code = torch.where(scale > 0, torch.round(x / scale.clamp_min(1e-300)), torch.zeros_like(x))
    return (code.clamp(-127, 127) + 128).to(torch.uint8), scale.float()


def _pack(k, v):
    """Blocks [n, H, bytes] of pages of dense tokens [n, 16, H, D]."""
    n, _, H, D = k.shape
    block = torch.empty(n, H, 2 * PAGE * D + PAGE * 8, dtype=torch.uint8, device=k.device)
    ki, vi = _layout(D, k.device)
    kc, ks = _quantise(k)
    vc, vs = _quantise(v)
    block[:, :, ki.reshape(-1)] = kc.transpose(1, 2).reshape(n, H, PAGE * D)
    block[:, :, PAGE * D + vi.reshape(-1)] = vc.transpose(1, 2).reshape(n, H, PAGE * D)
    scales = torch.cat([ks, vs], -1).transpose(1, 2).contiguous()  # [n, H, 16, 2]
    block[:, :, 2 * PAGE * D:] = scales.view(torch.uint8).reshape(n, H, PAGE * 8)
    return block


def _values(block, D):
    """Keys and values [..., 16, D] in 32 bits of blocks [..., bytes]."""
    ki, vi = _layout(D, block.device)
    lead = block.shape[:-1]
    scales = block[..., 2 * PAGE * D:].contiguous().view(torch.float32).reshape(*lead, PAGE, 2)
    k = block[..., ki.reshape(-1)].reshape(*lead, PAGE, D).float() - 128
    v = block[..., PAGE * D + vi.reshape(-1)].reshape(*lead, PAGE, D).float() - 128
    return k * scales[..., 0:1], v * scales[..., 1:2]


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt = torch.device("cuda"), _DT[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    if case["op"] == "rope":
        T, n = case["T"], case["axes"]
        # runs of text (every axis the same) and of image patches (a grid), somewhere in the context
        t = torch.arange(T, device=dev)
        base = torch.randint(0, max(1, case["far"] - T), (1,), generator=g, device=dev)
        image = (t // 256) % 2 == 1
        pos = torch.stack([base + t, base + torch.where(image, t % 256 // 16, t),
                           base + torch.where(image, t % 16, t)][:n]).to(torch.int32)
        return {"case": case, "q": normal(T, case["Hq"], case["D"]), "k": normal(T, case["Hkv"], case["D"]),
                "positions": pos.contiguous(), "sections": _sections(case["rotary"], n)}

    old, new = _lengths(case)
    H, D, B, T = case["Hkv"], case["D"], case["B"], sum(new)
    total = [o + n for o, n in zip(old, new)]
    blocks = [(n + PAGE - 1) // PAGE for n in total]
    width, used = max(blocks), sum(blocks)
    pages = used + used // 10 + 1
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    starts = torch.tensor([0] + blocks, device=dev).cumsum(0)
    j = torch.arange(width, device=dev)[None, :]
    have = j < torch.tensor(blocks, device=dev)[:, None]
    at = (starts[:-1, None] + j).clamp_max(pages - 1)
    tables = torch.where(have, order[at], torch.full_like(order[at], -1)).contiguous()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = {"case": case, "tables": tables, "old": i32(old), "lens": i32(total), "total": T,
         "max_new": max(new), "max_len": max(total),
         "cu": i32([0] + [sum(new[:i + 1]) for i in range(B)])}

    # keys have a few loud channels, as a model's keys have
    loud = torch.ones(D, device=dev)
    loud[torch.randperm(D, generator=g, device=dev)[: max(1, D // 50)]] = 8.0
    if case["op"] == "append":
        s["pool"] = torch.full((pages, H, 2 * PAGE * D + PAGE * 8), 128, dtype=torch.uint8, device=dev)
        s["k"] = (normal(T, H, D, dtype=torch.float32) * loud).to(dt)
        s["v"] = normal(T, H, D)
        return s
    pool = torch.empty(pages, H, 2 * PAGE * D + PAGE * 8, dtype=torch.uint8, device=dev)
    for i in range(0, pages, 4096):
        n = min(4096, pages - i)
        pool[i:i + n] = _pack(normal(n, PAGE, H, D, dtype=torch.float32) * loud,
                              normal(n, PAGE, H, D, dtype=torch.float32))
    s["pool"] = pool
    if case["op"] == "attend":
        s["q"] = normal(T, case["Hq"], D)
        s["scale"] = 1.0 / math.sqrt(D)
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"rope": _rope, "append": _append, "read": _read, "attend": _attend}[state["case"]["op"]](state)


def _run_own(s):
    import importlib
    ops = importlib.import_module("truellm-engine_b200.ops")
    c = s["case"]
    if c["op"] == "rope":
        return ops.rope_axes(s["q"], s["k"], s["positions"], s["sections"], theta=c["theta"],
                             order=c["order"], pairing=c["pairing"])
    if "cache" not in s:
        s["cache"] = ops.Int8PagedCache(c["Hkv"], c["D"], pool=s["pool"])
    if c["op"] == "append":
        ops.int8_append(s["cache"], s["k"], s["v"], s["cu"], s["old"], s["tables"],
                        max_new_tokens=s["max_new"])
    if c["op"] in ("append", "read"):
        return ops.int8_read(s["cache"], s["tables"], s["old"], s["cu"], s["total"],
                             max_tokens=s["max_new"], dtype=_DT[c["dtype"]])
    if "workspace" not in s:
        s["workspace"] = ops.int8_workspace(c["B"], c["Hq"], c["Hkv"], c["D"], s["max_new"],
                                            s["max_len"], device=s["q"].device)
    return ops.int8_attend(s["cache"], s["q"], s["cu"], s["tables"], s["lens"],
                           max_q_tokens=s["max_new"], max_context_len=s["max_len"],
                           scale=s["scale"], window=c["window"], workspace=s["workspace"])


def _rope(s):
    c = s["case"]
    half, dev = c["rotary"] // 2, s["q"].device
    i = torch.arange(half, device=dev, dtype=torch.float64)
    freq = c["theta"] ** (-2 * i / c["rotary"])
    axis = torch.tensor(_axis_of_pair(s["sections"], c["order"]), device=dev)
    angle = s["positions"].double()[axis].T * freq  # [T, pairs]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        r, keep = x[..., : c["rotary"]].float(), x[..., c["rotary"]:].float()
        if c["pairing"] == "halves":
            a, b = r[..., :half], r[..., half:]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([y, keep], -1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _where(s):
    """Page and slot of every new token: [T] each."""
    T, cu = s["total"], s["cu"].long()
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    pos = s["old"].long()[b] + t - cu[b]
    return s["tables"][b, pos // PAGE].long(), pos % PAGE


def _append(s):
    D = s["case"]["D"]
    page, slot = _where(s)
    ki, vi = _layout(D, page.device)
    pool, H = s["pool"], s["case"]["Hkv"]
    h = torch.arange(H, device=page.device)[None, :, None]
    kc, ks = _quantise(s["k"])
    vc, vs = _quantise(s["v"])
    pool[page[:, None, None], h, ki[slot][:, None]] = kc
    pool[page[:, None, None], h, PAGE * D + vi[slot][:, None]] = vc
    scales = torch.cat([ks, vs], -1).view(torch.uint8).reshape(-1, H, 8)
    byte = 2 * PAGE * D + slot[:, None, None] * 8 + torch.arange(8, device=page.device)
    pool[page[:, None, None], h, byte] = scales
    return _read(s)


def _read(s):
    D, dt = s["case"]["D"], _DT[s["case"]["dtype"]]
    page, slot = _where(s)
    ki, vi = _layout(D, page.device)
    pool, H = s["pool"], s["case"]["Hkv"]
    h = torch.arange(H, device=page.device)[None, :, None]
    byte = 2 * PAGE * D + slot[:, None, None] * 8 + torch.arange(8, device=page.device)
    scales = pool[page[:, None, None], h, byte].view(torch.float32)  # [T, H, 2]
    k = (pool[page[:, None, None], h, ki[slot][:, None]].float() - 128) * scales[..., 0:1]
    v = (pool[page[:, None, None], h, PAGE * D + vi[slot][:, None]].float() - 128) * scales[..., 1:2]
    return k.to(dt), v.to(dt)


def _attend(s):
    c = s["case"]
    B, H, D, grp, n, T = c["B"], c["Hkv"], c["D"], c["Hq"] // c["Hkv"], s["max_new"], s["total"]
    dev = s["q"].device
    k, v = _values(s["pool"][s["tables"].clamp_min(0).long()], D)  # [B, blocks, H, 16, D]
    k = k.permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
    v = v.permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(s["cu"].long()[1:], t, right=True)
    i = t - s["cu"].long()[b]
    q = torch.zeros(B, n, H, grp, D, device=dev)
    q[b, i] = s["q"].float().reshape(T, H, grp, D)
    q = q.permute(0, 2, 1, 3, 4).reshape(B, H, n * grp, D)
    x = (q @ k.transpose(-1, -2)) * s["scale"]
    at = (s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long())[:, None] + torch.arange(n, device=dev)
    key = torch.arange(k.shape[2], device=dev)
    hide = key > at[..., None]
    if c["window"]:
        hide = hide | (key <= at[..., None] - c["window"])
    x = x.view(B, H, n, grp, -1).masked_fill_(hide[:, None, :, None], -math.inf).view(B, H, n * grp, -1)
    x = torch.exp(x.sub_(x.amax(-1, keepdim=True)))
    o = (x @ v) / x.sum(-1, keepdim=True)
    o = o.view(B, H, n, grp, D).permute(0, 2, 1, 3, 4)[b, i]
    return o.reshape(T, c["Hq"], D).to(s["q"].dtype)


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    D, H = case["D"], case["Hkv"]
    if case["op"] == "rope":
        r = case["rotary"]
        axis, left, turn = [], list(s["sections"]), 0
        for _ in range(r // 2):
            if case["order"] == "blocks":
                turn = next(a for a in range(len(left)) if left[a])
            else:
                while not left[turn % len(left)]:
                    turn += 1
                turn %= len(left)
            left[turn] -= 1
            axis.append(turn)
            turn += case["order"] != "blocks"
        out = []
        for x in (s["q"], s["k"]):
            y = x.double()
            z = y.clone()
            for p in range(r // 2):
                w = s["positions"][axis[p]].double()[:, None] / case["theta"] ** (2 * p / r)
                a, b = (p, p + r // 2) if case["pairing"] == "halves" else (2 * p, 2 * p + 1)
                z[..., a] = y[..., a] * torch.cos(w) - y[..., b] * torch.sin(w)
                z[..., b] = y[..., b] * torch.cos(w) + y[..., a] * torch.sin(w)
            out.append(z)
        return tuple(out)

    if case["op"] == "append":
        out = []
        for x in (s["k"].double(), s["v"].double()):
            d = (x.abs().max(-1, keepdim=True).values / 127).to(torch.float32).double()
            out.append(torch.round(x / d) * d)
        return tuple(out)

    def dense(seq, lo, hi):
        """Keys and values [H, hi - lo, D] of one sequence's tokens, in 64 bits."""
        p0, p1 = lo // PAGE, (hi + PAGE - 1) // PAGE
        blk = s["pool"][s["tables"][seq, p0:p1].long()]
        n = p1 - p0
        sc = blk[:, :, 2 * PAGE * D:].contiguous().view(torch.float32).view(n, H, PAGE, 2).double()
        kb = blk[:, :, : PAGE * D].reshape(n, H, D // 16, PAGE, 16)
        tok = torch.arange(PAGE, device=blk.device)
        ks = torch.stack([kb[:, :, u][:, :, tok ^ (2 * (u % 4))] for u in range(D // 16)], 3)
        kd = (ks.reshape(n, H, PAGE, D).double() - 128) * sc[..., :1]
        vb = blk[:, :, PAGE * D: 2 * PAGE * D].reshape(n, H, D // 32, 8, 4, 4, 4)  # u g t j i
        vd = (vb.permute(0, 1, 4, 6, 2, 3, 5).reshape(n, H, PAGE, D).double() - 128) * sc[..., 1:]
        cut = slice(lo - p0 * PAGE, hi - p0 * PAGE)
        return (kd.transpose(0, 1).reshape(H, n * PAGE, D)[:, cut],
                vd.transpose(0, 1).reshape(H, n * PAGE, D)[:, cut])

    old, new = _lengths(case)
    if case["op"] == "read":
        got = [dense(b, o, o + n) for b, (o, n) in enumerate(zip(old, new))]
        return tuple(torch.cat([g[i].transpose(0, 1) for g in got]) for i in (0, 1))

    out, row, grp = [], 0, case["Hq"] // H
    for b, (o, n) in enumerate(zip(old, new)):
        L = o + n
        lo = max(0, o + 1 - case["window"]) if case["window"] else 0
        k, v = dense(b, lo, L)
        q = s["q"][row: row + n].double().reshape(n, H, grp, D)
        row += n
        got = torch.empty(n, H, grp, D, dtype=torch.float64, device=q.device)
        key = torch.arange(lo, L, device=q.device)
        for i in range(0, n, 256):
            at = torch.arange(o + i, o + min(n, i + 256), device=q.device)[:, None]
            ok = key[None] <= at
            if case["window"]:
                ok &= key[None] > at - case["window"]
            x = torch.einsum("nhgd,hld->hgnl", q[i:i + 256], k) * s["scale"]
            p = torch.softmax(x.masked_fill(~ok, -math.inf), -1)
            got[i:i + 256] = torch.einsum("hgnl,hld->nhgd", p, v)
        out.append(got.reshape(n, case["Hq"], D))
    return torch.cat(out)
