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


def _through_c(torch, gate, x, r, dh, flip, keep):
    """Forward and backward pass through the C entries, time-major; flip: every tensor is walked backwards along that axis."""
    from marl_amd import _lib
    lib, dt = _lib.load(), _lib.SEQ_BF16
    T, B, D = gate.shape
    h, dgate, dx = (torch.zeros_like(gate) for _ in range(3))

    def at(t):
        s = list(t.stride()[:2])
        p = t.data_ptr()
        if flip is not None:
            p += (t.shape[flip] - 1) * s[flip] * t.element_size()
            s[flip] = -s[flip]
        return (p, *s)
    st = torch.cuda.current_stream().cuda_stream
    need, size = lib.asm_gated_scan_workspace(dt, T, B, D), lib.asm_gated_scan_kept(dt, T, B, D)
    assert size == (T + 7) // 8 * B * D * 4
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    kept = torch.full((size // 4,), float("nan"), device="cuda") if keep else None
    pk = kept.data_ptr() if keep else None
    _lib.check(lib.asm_gated_scan_forward(dt, T, B, D, *at(gate), *at(x), None, *at(r), None, *at(h), None, pk, ws.data_ptr(), need, st), "forward")
    _lib.check(lib.asm_gated_scan_backward(dt, T, B, D, *at(gate), *at(x), *at(h), None, *at(r), None, *at(dh), None, *at(dgate), *at(dx), None, pk, ws.data_ptr(), need,
                                           st), "backward")
    return h, dgate, dx


@pytest.mark.parametrize("flip", [None, 0, 1])
@pytest.mark.parametrize("T,B,D", [(19, 500, 64), (19, 500, 256), (19, 1000, 256), (13, 7, 9), (350, 3, 30)])
def test_c_entries_with_and_without_kept_states(torch_cuda, T, B, D, flip):
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(T + D)
    gate, x, dh = (torch.randn(T, B, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(3))
    r = (torch.rand(T, B, device="cuda", generator=g) < 0.1).to(torch.uint8)
    turned = lambda t: t if flip is None else t.flip(flip)  # noqa: E731
    for keep in (True, False):
        got = [turned(t) for t in _through_c(torch, gate, x, r, dh, flip, keep)]
        if keep:
            want = _want(turned(gate), turned(x), None, turned(r) != 0, None, False, turned(dh), torch.zeros(B, D))
        else:                                                           # (the states are h as stored: seq_oracle's own bound)
            want = so.scan(turned(gate), turned(x), resets=turned(r) != 0, dh=turned(dh))
        for name, t in zip(("h", "dgate", "dx"), got):
            so.within(t, *want[name], f"flip {flip} kept {keep} {name}")
