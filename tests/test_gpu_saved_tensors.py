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
