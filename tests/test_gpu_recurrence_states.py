"""The state that a backward pass works from: float32 whatever the outputs' type, at every size and alignment.

Bounds: bfloat16 values are float32 values, so seq_oracle.scan's float32 bounds hold for what is computed from them, and the
only rounding to fewer bits is each output's own, half a step of bfloat16 (2^-8) of the result."""
import pytest

import seq_oracle as so
from test_gpu_recurrence import SHAPES, _make

pytestmark = pytest.mark.gpu


def _want(gate, x, h0, r, n, bf, dh, dl):
    want = so.scan(gate.float(), x.float(), h0, r, n, bf, dh.float(), dl)
    half = so.HALF[gate.dtype] if gate.element_size() == 2 else 0.0
    return {k: (v, e + half * (v.abs() + e) if k in ("h", "dgate", "dx") else e) for k, (v, e) in want.items()}


def _check(torch, gate, x, h0, r, n, bf, what):
    from marl_amd.recurrence import gated_scan
    leaves = [t.detach().requires_grad_() for t in (gate, x)] + ([] if h0 is None else [h0.detach().requires_grad_()])
    h, last = gated_scan(leaves[0], leaves[1], leaves[2] if h0 is not None else None, resets=r, lengths=n, batch_first=bf)
    g = torch.Generator(device="cuda").manual_seed(5)
    dh = torch.randn(h.shape, device="cuda", generator=g).to(h.dtype)
    dl = torch.randn(last.shape, device="cuda", generator=g)
    grads = torch.autograd.grad((h, last), leaves, (dh, dl))
    want = _want(gate, x, h0, r, n, bf, dh, dl)
    for name, got in zip(("h", "last", "dgate", "dx", "dh0"), (h, last) + grads):
        so.within(got, *want[name], f"{what} {name}")


@pytest.mark.parametrize("settled", [False, True])
@pytest.mark.parametrize("marks", ["none", "all"])
@pytest.mark.parametrize("T,B,D", SHAPES + [(7, 5, 8), (8, 5, 8), (16, 900, 64), (57, 900, 64), (330, 3, 64), (1000, 70, 9)])
def test_the_gates_gradient_comes_from_a_float32_state(torch_cuda, T, B, D, marks, settled):
    """settled: a memory near its input, h - x a small part of either: half a step of h in bfloat16 is as large as it."""
    torch = torch_cuda
    bf = (T + B + D) % 2 == 0
    gate, x, h0, r, n = _make(torch, T, B, D, torch.bfloat16, bf, T + D + 1, marks == "all", marks == "all", True)
    if settled:
        x, h0 = (5.0 + 0.02 * x.float()).to(torch.bfloat16), 5.0 + 0.02 * h0
    _check(torch, gate, x, h0, r, n, bf, f"{T}x{B}x{D} {marks} {settled}")


def test_the_gates_gradient_of_strided_tensors(torch_cuda):
    torch = torch_cuda
    for T, B, D in ((50, 6, 24), (20, 300, 256), (11, 1200, 256)):
        both = (5.0 + 0.05 * torch.randn(T, B, 2 * D + 4, device="cuda")).to(torch.bfloat16)
        for a, b, what in ((both[..., :D], both[..., D:2 * D], "aligned cut"), (both[..., 1:D + 1], both[..., D + 2:2 * D + 2], "odd offset"),
                           (both[..., 2:D + 2], both[..., D + 2:2 * D + 2], "two values aligned")):
            _check(torch, a, b, None, None, None, False, what)
