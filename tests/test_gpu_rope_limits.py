"""The rotary step at the most tokens that a call takes, 2^31 - 1."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_most_tokens(ops, cuda):
    """One row for all tokens (a stride of 0), positions 0 but at both ends."""
    T = 2 ** 31 - 1
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("77 GB are needed")
    q = torch.randn(1, 1, 16, device=cuda, dtype=torch.float16)
    pos = torch.zeros(1, T, dtype=torch.int32, device=cuda)
    pos[0, 0], pos[0, T - 1], pos[0, T - 2], pos[0, T - 6] = 9, 5, -3, 70000
    out = ops.rope_axes(q.expand(T, 1, 16), None, pos, (8,))[0]
    for at in (slice(0, 3), slice(T // 2, T // 2 + 5), slice(T - 9, T)):
        n = pos[0, at].numel()
        want = ops.rope_axes(q.expand(n, 1, 16).contiguous(), None, pos[:, at].contiguous(), (8,))[0]
        assert torch.equal(out[at], want)
    del out, pos
    torch.cuda.empty_cache()
