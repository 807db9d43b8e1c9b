"""Forward and backward pass of the clipped policy loss in different captures, or only one of them captured: each replay of a
backward pass gives that pass's gradients, to the bit those of an eager call."""
import gc

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_garbage():
    """(a HIP graph that the garbage collector frees while another one is captured ends the process)"""
    gc.collect()
    yield
    gc.collect()


def _make(torch, N=3000, dtype="float32"):
    g = torch.Generator(device="cuda").manual_seed(3)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dt = getattr(torch, dtype)
    return [(0.3 * rn(N, 2)).to(dt).requires_grad_(), torch.zeros(2, device="cuda", dtype=dt).requires_grad_(), rn(N, 2), rn(N), rn(N)]


def _loss(c):
    from marl_amd.policy_loss import clipped_policy_loss
    return clipped_policy_loss(*c, kl_coef=0.1, entropy_coef=0.01)[0]


def _grads(torch, c, loss, up, **kw):
    return torch.autograd.grad(loss, c[:2], up, **kw)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("forward", ["eager", "own graph", "same graph"])
def test_a_captured_backward_pass_may_be_replayed(torch_cuda, no_garbage, forward, dtype):
    torch = torch_cuda
    c, up = _make(torch, dtype=dtype), torch.tensor(0.5, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in _grads(torch, c, _loss(c), up)]
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    if forward == "eager":
        with torch.cuda.stream(side):
            loss = _loss(c)
        side.synchronize()
    elif forward == "own graph":
        with torch.cuda.graph(first, stream=side):
            loss = _loss(c)
    with torch.cuda.graph(second, stream=side):
        if forward == "same graph":
            loss = _loss(c)
        got = _grads(torch, c, loss, up)
    if forward == "own graph":
        first.replay()
    for k in range(3):
        second.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_an_eager_backward_pass_of_a_captured_loss_keeps_its_gradients(torch_cuda, no_garbage):
    """What an eager backward pass handed out is not written by the next replay of the forward pass."""
    torch = torch_cuda
    c, up = _make(torch), torch.tensor(0.5, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in _grads(torch, c, _loss(c), up)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = _loss(c)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = _grads(torch, c, loss, up, retain_graph=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,B,D", [(600, 3, 20), (20, 7, 64), (20, 1200, 256)])
def test_the_memorys_backward_pass_captured_alone(torch_cuda, no_garbage, T, B, D, dtype):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    L = [torch.randn(T, B, D, device="cuda").to(getattr(torch, dtype)).requires_grad_() for _ in range(2)]
    dh = torch.randn(T, B, D, device="cuda").to(getattr(torch, dtype))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h, last = gated_scan(*L)
        want = [t.clone() for t in torch.autograd.grad(h, L, dh, retain_graph=True)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(h, L, dh)
    for k in range(3):
        for t in got:
            t.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
