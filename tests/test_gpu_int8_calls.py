"""int8 attention as an engine calls it: one workspace for batches of all sizes."""
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
