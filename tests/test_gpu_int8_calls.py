"""The int8 cache as an engine calls it: one workspace for batches of all sizes, numbers
out of range, a sequence that forks."""
import numpy as np
import pytest
import torch

from test_gpu_int8 import Batch, DT, t32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dt", [(128, "bf16"), (64, "f16")])
def test_a_workspace_of_the_largest_sizes_serves_smaller_batches(ops, cuda, D, dt):
    """Fewer sequences, shorter chunks and contexts, fewer q heads than the workspace
    was made for, each call with its own bounds; nothing behind it is written."""
    H, Hq, most = 2, 8, (40, 200, 3000)
    n = ops.int8_workspace_bytes(most[0], Hq, H, D, *most[1:])
    raw = torch.zeros(n + 4096, dtype=torch.uint8, device=cuda)
    raw[n:] = 0x5a
    ws = raw[:n]
    shapes = [([100] * 40, [200] + [1] * 39, 8), ([2800], [200], 8), ([2900], [9], 8),
              ([2900, 40, 2500], [33, 1, 64], 8), ([2999], [1], 8), ([700] * 5, [130] * 5, 4),
              ([60] * 39, [1] * 39, 8), ([1500] * 37, [5] * 37, 8)]
    for i, (old, new, hq) in enumerate(shapes):
        b = Batch(ops, cuda, old, new, H, D, DT[dt], seed=i)
        b.fill()
        q = b.query(hq)
        out = b.attend(q, workspace=ws)
        b.check(q, out, rows=2)
        assert torch.equal(out, b.attend(q))
    assert (raw[n:] == 0x5a).all()


def test_numbers_past_32_bits_are_refused(ops, cuda):
    """A window of 2^32 is not "no window", a bound of 2^32 not 0."""
    b = Batch(ops, cuda, [100], [4], 2, 64, DT["f16"])
    b.fill()
    q, z, cu = b.query(4), t32([0], cuda), t32([0, 4], cuda)
    lens = t32(b.lens, cuda)
    want = b.attend(q)
    assert torch.equal(b.attend(q, window=2 ** 31 - 1), want)
    for call in (lambda n: b.attend(q, window=n),
                 lambda n: ops.int8_attend(b.cache, q, cu, b.bt_t, lens, max_q_tokens=n),
                 lambda n: ops.int8_attend(b.cache, q, cu, b.bt_t, lens, max_context_len=n),
                 lambda n: ops.int8_append(b.cache, b.k[:4], b.v[:4], cu, z, b.bt_t, max_new_tokens=n),
                 lambda n: ops.int8_read(b.cache, b.bt_t, z, cu, 4, max_tokens=n),
                 lambda n: ops.int8_read(b.cache, b.bt_t, z, cu, n)):
        for n in (2 ** 31, 2 ** 32, 2 ** 32 + 200, -2 ** 32):
            with pytest.raises(ValueError, match="32 bits"):
                call(n)


@pytest.mark.parametrize("through_host", [False, True])
def test_a_sequence_that_forks_inside_a_page(ops, cuda, through_host):
    """Two sequences share 21 tokens; the partly filled page is copied (or brought back
    from the host), then both append and attend."""
    H, Hq, D, old, new = 2, 8, 128, 21, 5
    b = Batch(ops, cuda, [old, old], [new, new], H, D, DT["bf16"], seed=1)
    whole = t32([0, old], cuda)
    ops.int8_append(b.cache, b.k[:old], b.v[:old], whole, t32([0], cuda), b.bt_t[:1])
    first, last, fresh = int(b.bt[0, 0]), int(b.bt[0, 1]), int(b.bt[1, 1])
    b.pool[fresh] = b.pool[last].cpu().to(cuda) if through_host else b.pool[last]
    b.bt[1, 0] = first
    b.bt_t = t32(b.bt, cuda)
    rows = torch.cat([torch.arange(old, old + new), torch.arange(2 * old + new, 2 * (old + new))])
    at = rows.to(cuda)
    ops.int8_append(b.cache, b.k[at], b.v[at], t32(b.cu, cuda), t32(b.old, cuda), b.bt_t)
    q = b.query(Hq)
    b.check(q, b.attend(q))
    alone = ops.Int8PagedCache(H, D, 2)  # the second sequence's tokens without sharing
    k, v = (torch.cat([x[:old], x[at[new:]]]) for x in (b.k, b.v))
    ops.int8_append(alone, k, v, t32([0, old + new], cuda), t32([0], cuda), t32([[0, 1]], cuda))
    assert torch.equal(
        ops.int8_attend(alone, q[new:], t32([0, new], cuda), t32([[0, 1]], cuda), t32([26], cuda)),
        ops.int8_attend(b.cache, q[new:], t32([0, new], cuda), b.bt_t[1:].contiguous(), t32([26], cuda)))
