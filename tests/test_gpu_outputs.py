"""Outputs that the caller gives to the rotary step and the int8 cache: in place, side by
side with inputs, refused where memory is shared, and known to autograd."""
import pytest
import torch

from test_gpu_int8 import Batch, t32

pytestmark = pytest.mark.gpu
F16 = torch.float16


def rope(ops, q, k, pos, **kw):
    return ops.rope_axes(q, k, pos, (16, 24, 24), **kw)


def tokens(dev, T=37):
    q, k = (torch.randn(T, h, 128, device=dev, dtype=F16) for h in (8, 2))
    return q, k, torch.randint(0, 5000, (3, T), device=dev, dtype=torch.int32)


@pytest.mark.parametrize("T", [1, 37])
def test_rotary_outputs_beside_their_inputs(ops, cuda, T):
    q, k, pos = tokens(cuda, T)
    qo, ko = rope(ops, q, k, pos)
    # one buffer: q, k, and room for both results in the same rows; then heads outermost
    wide = torch.zeros(T, 20, 128, device=cuda, dtype=F16)
    deep = torch.zeros(20, T, 128, device=cuda, dtype=F16).transpose(0, 1)
    for buf in (wide, deep):
        q1, k1, q2, k2 = buf[:, :8], buf[:, 8:10], buf[:, 10:18], buf[:, 18:]
        q1.copy_(q), k1.copy_(k)
        rope(ops, q1, k1, pos, q_out=q2, k_out=k2)
        assert torch.equal(q2, qo) and torch.equal(k2, ko) and torch.equal(q1, q)
        rope(ops, q1, k1, pos, q_out=q1, k_out=k2)  # one of them in place
        assert torch.equal(q1, qo) and torch.equal(k2, ko)


def test_rotary_outputs_that_share_memory_are_refused(ops, cuda):
    q, k, pos = tokens(cuda)
    buf = torch.zeros(40, 10, 128, device=cuda, dtype=F16)
    inside = buf[:37, :8]
    for call in (lambda: rope(ops, inside, k, pos, q_out=buf[1:38, :8]),
                 lambda: rope(ops, inside, k, pos, q_out=buf[:37, 1:9]),
                 lambda: rope(ops, q, k, pos, q_out=q[:, :1].expand(37, 8, 128)),
                 lambda: rope(ops, q, k, pos, q_out=q[:1].expand(37, 8, 128)),
                 lambda: rope(ops, inside, buf[:37, 8:], pos, q_out=buf[:37, 2:]),
                 lambda: rope(ops, q, k, pos, q_out=inside, k_out=buf[:37, 7:9]),
                 lambda: rope(ops, q, q, pos, q_out=q, k_out=q),
                 lambda: rope(ops, q, q, pos, q_out=q, k_out=torch.empty_like(q))):
        with pytest.raises(ValueError, match="overlap|share memory"):
            call()


def test_attention_over_its_queries_and_beside_them(ops, cuda):
    for old, new in (([3000, 40], [1, 1]), ([500, 2000], [60, 3])):
        b = Batch(ops, cuda, old, new, 2, 128, F16, seed=3)
        b.fill()
        q = b.query(8)
        want = b.attend(q)
        for _ in range(3):
            same = q.clone()
            assert b.attend(same, out=same) is same and torch.equal(same, want)
        n = q.shape[0]
        buf = torch.zeros(2 * n + 1, 8, 128, device=cuda, dtype=F16)
        buf[:n] = q
        assert torch.equal(b.attend(buf[:n], out=buf[n:2 * n]), want)
        for out in (buf[1:n + 1], buf[n - 1:2 * n - 1]):
            with pytest.raises(ValueError, match="overlap"):
                b.attend(buf[:n], out=out)
        with pytest.raises(ValueError, match="overlap"):  # queries inside a wider buffer
            b.attend(buf.view(-1)[:n * 12 * 128].view(n, 12, 128)[:, :8], out=buf[:n])


def test_read_outputs_that_share_memory_are_refused(ops, cuda):
    b = Batch(ops, cuda, [0], [20], 2, 64, F16)
    b.fill()
    buf = torch.zeros(41, 2, 64, device=cuda, dtype=F16)
    args = (b.cache, b.bt_t, t32([0], cuda), t32([0, 20], cuda), 20)
    ops.int8_read(*args, k_out=buf[:20], v_out=buf[20:40])
    for v in (buf[:20], buf[19:39]):
        with pytest.raises(ValueError, match="overlap"):
            ops.int8_read(*args, k_out=buf[:20], v_out=v)


def test_autograd_knows_of_written_outputs(ops, cuda):
    """What a backward pass has kept and a call then writes is an error in that pass;
    tensors that require a gradient are no outputs."""
    q, k, pos = tokens(cuda)
    b = Batch(ops, cuda, [50], [37], 2, 128, F16)
    b.fill()
    read = (b.cache, b.bt_t, t32([0], cuda), t32([0, 37], cuda), 37)
    for write, shape in ((lambda t: rope(ops, t, None, pos, q_out=t), q.shape),
                         (lambda t: rope(ops, k, q, pos, k_out=t), q.shape),
                         (lambda t: b.attend(q, out=t), q.shape),
                         (lambda t: ops.int8_read(*read, k_out=t), k.shape),
                         (lambda t: ops.int8_read(*read, v_out=t), k.shape)):
        w = torch.randn(shape, device=cuda, dtype=F16, requires_grad=True)
        kept = torch.randn(shape, device=cuda, dtype=F16)
        loss = (w * kept).sum()
        write(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()
        with pytest.raises(ValueError, match="gradient"):
            write(w)
        with torch.no_grad():
            write(w)
        with torch.inference_mode():
            write(torch.randn(shape, device=cuda, dtype=F16))
