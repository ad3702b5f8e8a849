"""rope_axes and autograd: streams and tangents."""
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


def test_a_tangent_turns_as_its_input_does(ops, cuda):
    """Forward mode: of both inputs, of one, and of a call that turns back."""
    fwd = torch.autograd.forward_ad
    q, k, pos, tq, tk = inputs(cuda, T=33)
    how = dict(order="round_robin", pairing="adjacent")
    turned = lambda t, **kw: ops.rope_axes(t, None, pos, SECTIONS, **how, **kw)[0]  # noqa: E731
    with fwd.dual_level():
        dq, dk = fwd.make_dual(q, tq), fwd.make_dual(k, tk)
        for a, b in ((dq, dk), (dq, k), (q, dk), (dq, None)):
            got = ops.rope_axes(a, b, pos, SECTIONS, **how)
            for x, y, t, dual in ((got[0], q, tq, a is dq), (got[1], k, tk, b is dk)):
                if x is None:
                    continue
                p, tangent = fwd.unpack_dual(x)
                assert torch.equal(p, turned(y))
                if dual:
                    assert torch.equal(tangent, turned(t))
                else:
                    assert tangent is None or not tangent.any()
        back = ops.rope_axes(dq, None, pos, SECTIONS, inverse=True, **how)[0]
        assert torch.equal(fwd.unpack_dual(back).tangent, turned(tq, inverse=True))
        with torch.no_grad():  # stops gradients, not tangents
            out = ops.rope_axes(dq, None, pos, SECTIONS, **how)[0]
        assert torch.equal(fwd.unpack_dual(out).tangent, turned(tq))
        with pytest.raises(ValueError, match="gradient"):
            ops.rope_axes(dq, None, pos, SECTIONS, q_out=torch.empty_like(q))


def test_functional_transforms_are_refused(ops, cuda):
    """torch.func hides tensors' memory: an error, and no lost derivative."""
    q, k, pos, wq, wk = inputs(cuda, T=17)
    f = lambda a, b: ops.rope_axes(a, b, pos, SECTIONS)  # noqa: E731
    for call in (lambda: torch.func.vjp(f, q, k), lambda: torch.func.jvp(f, (q, k), (wq, wk)),
                 lambda: torch.func.grad(lambda a: f(a, k)[0].sum())(q)):
        with pytest.raises(RuntimeError):
            call()


def test_what_has_no_derivative_refuses_a_tangent(ops, cuda):
    fwd = torch.autograd.forward_ad
    cache = ops.Int8PagedCache(2, 128, 2)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    k, q = (torch.randn(5, h, 128, device=cuda, dtype=torch.float16) for h in (2, 8))
    cu, old, bt = i32([0, 5]), i32([0]), i32([[0, 1]])
    with fwd.dual_level(), torch.no_grad():
        with pytest.raises(ValueError, match="tangent"):
            ops.int8_append(cache, fwd.make_dual(k, k), k, cu, old, bt)
        with pytest.raises(ValueError, match="tangent"):
            ops.int8_attend(cache, fwd.make_dual(q, q), cu, bt, i32([5]))
        ops.int8_append(cache, k, k, cu, old, bt)
        ops.int8_attend(cache, q, cu, bt, i32([5]))
