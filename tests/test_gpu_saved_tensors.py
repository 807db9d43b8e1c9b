"""The gated memory under saved-tensor hooks: what a backward pass gets back has another alignment and other strides than what
the forward pass was given.  Bounds: seq_oracle.scan's."""
import pytest

import seq_oracle as so
from test_gpu_recurrence_states import _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,B,D", [(11, 1200, 256), (24, 1200, 256), (19, 500, 12)])
def test_saved_tensors_may_come_back_dense(torch_cuda, T, B, D, dtype):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    both = torch.randn(T, B, 2 * D + 3, device="cuda").to(getattr(torch, dtype))
    for lo in (0, 1, 2):
        gate, x = both[..., lo:lo + D], both[..., D + lo:2 * D + lo]
        leaves = [gate.detach().requires_grad_(), x.detach().requires_grad_()]
        # (memory that later allocations are likely to get: states that were never written are NaN)
        fill = [torch.full(((T + 7) // 8 * B * D,), float("nan"), device="cuda") for _ in range(8)]
        del fill
        with torch.autograd.graph.save_on_cpu():
            h, last = gated_scan(*leaves)
        dh, dl = torch.randn_like(h), torch.randn_like(last)
        grads = torch.autograd.grad((h, last), leaves, (dh, dl))
        want = _want(gate, x, None, None, None, False, dh, dl)
        for name, got in zip(("h", "last", "dgate", "dx"), (h, last) + grads):
            so.within(got, *want[name], f"offset {lo} {name}")


def test_saved_tensors_may_come_back_transposed(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    T, B, D = 9, 4, 6
    leaves = [torch.randn(T, B, D, device="cuda", requires_grad=True) for _ in range(2)]
    turned = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() == 3 else t  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(turned, lambda t: t):
        h, last = gated_scan(*leaves)
    dh, dl = torch.randn_like(h), torch.randn_like(last)
    got = torch.autograd.grad((h, last), leaves, (dh, dl))
    want = torch.autograd.grad(gated_scan(*leaves), leaves, (dh, dl))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_every_saved_tensor_may_come_back_strided(torch_cuda, dtype):
    """States, lengths, resets and advantage moments too; the loss reads its saved tensors in a second backward pass."""
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    from marl_amd.recurrence import gated_scan
    T, B, D = 9, 4, 6

    def spread(t):                                                      # twice as far apart along every axis, something else between
        wide = torch.full([2 * n for n in t.shape], 7, device=t.device).to(t.dtype)
        out = wide[tuple(slice(0, None, 2) for _ in t.shape)]
        out.copy_(t)
        return out

    dt = getattr(torch, dtype)
    leaves = [torch.randn(T, B, D, device="cuda").to(dt).requires_grad_(), torch.randn(T, B, D, device="cuda").to(dt).requires_grad_(),
              torch.randn(B, D, device="cuda", requires_grad=True)]
    kw = dict(resets=torch.rand(T, B, device="cuda") < 0.2, lengths=torch.tensor([9, 0, 4, 7], device="cuda", dtype=torch.int32))
    dh, dl = torch.randn(T, B, D, device="cuda").to(dt), torch.randn(B, D, device="cuda")
    want = torch.autograd.grad(gated_scan(*leaves, **kw), leaves, (dh, dl))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        out = gated_scan(*leaves, **kw)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, (dh, dl)), want))
    rows = [torch.randn(50, 2, device="cuda", requires_grad=True), torch.zeros(2, device="cuda", requires_grad=True), torch.randn(50, 2, device="cuda"),
            torch.randn(50, device="cuda"), torch.randn(50, device="cuda")]
    kw = dict(adv_moments=torch.tensor([0.3, 1.7], device="cuda"), mask=torch.rand(50, device="cuda") < 0.7, kl_coef=0.1)
    want = torch.autograd.grad(clipped_policy_loss(*rows, **kw)[0], rows[:2])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
        loss, _ = clipped_policy_loss(*rows, **kw)
    for _ in range(2):
        got = torch.autograd.grad(loss, rows[:2], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
