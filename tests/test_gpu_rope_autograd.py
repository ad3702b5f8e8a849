"""rope_axes and autograd: streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SECTIONS = (16, 24, 24)


def inputs(dev, T=3000):
    g = torch.Generator(device=dev).manual_seed(T)
    mk = lambda h: torch.randn(T, h, 128, generator=g, device=dev, dtype=torch.float32).half()  # noqa: E731
    pos = torch.randint(0, 5000, (3, T), generator=g, device=dev, dtype=torch.int32)
    return mk(8), mk(2), pos, mk(8), mk(2)


@pytest.mark.parametrize("form", ["stream", "address"])
def test_a_gradient_on_a_given_stream_waits_and_is_waited_for(ops, cuda, form):
    """The gradient that comes back is late (a long sleep before it on the current
    stream), and what the call returns is used there at once."""
    q, k, pos, wq, wk = inputs(cuda)
    want = [ops.rope_axes(w, None, pos, SECTIONS, inverse=True)[0] for w in (wq, wk)]
    side = torch.cuda.Stream()
    for _ in range(3):
        ql, kl = q.clone().requires_grad_(), k.clone().requires_grad_()
        side.wait_stream(torch.cuda.current_stream())
        qo, ko = ops.rope_axes(ql * 1, kl * 1, pos, SECTIONS,
                               stream=side if form == "stream" else side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        late = torch.zeros_like(wq)
        torch.cuda._sleep(20_000_000)  # about 10 ms
        late.copy_(wq)
        gq, gk = torch.autograd.grad([qo, ko], [ql, kl], [late, wk.clone()])
        late.zero_()
        assert torch.equal(gq, want[0]) and torch.equal(gk, want[1])


def test_a_backward_pass_of_a_given_stream_is_captured(ops, cuda):
    """Forward and backward in one graph, the call on a stream that joins the capture."""
    q, k, pos, wq, wk = inputs(cuda, T=64)
    side = torch.cuda.Stream()
    ql, kl = q.clone().requires_grad_(), k.clone().requires_grad_()

    def step():
        side.wait_stream(torch.cuda.current_stream())
        qo, ko = ops.rope_axes(ql, kl, pos, SECTIONS, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        return torch.autograd.grad([qo, ko], [ql, kl], [wq, wk])
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gq, gk = step()
    wq.copy_(torch.randn_like(wq))
    g.replay()
    assert torch.equal(gq, ops.rope_axes(wq, None, pos, SECTIONS, inverse=True)[0])
    assert torch.equal(gk, ops.rope_axes(wk, None, pos, SECTIONS, inverse=True)[0])
