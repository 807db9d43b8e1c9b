"""Outputs in the same buffer as inputs: refused where they overlap, computed where they lie between."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("B,D", [(1, 8), (6, 8), (37, 61)])
def test_step(torch_cuda, B, D, dtype):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan_step
    dt = getattr(torch, dtype)
    buf = torch.randn(B, 4 * D, device="cuda").to(dt)
    gate, x = buf[:, :D], buf[:, D:2 * D]
    want = gated_scan_step(gate.clone(), x.clone(), torch.zeros(B, D, device="cuda"))
    for out in (buf[:, 2 * D:3 * D], buf[:, 3 * D:], gate, x):          # pieces of one projection, then gate and x themselves
        b2 = buf.clone()
        at = lambda t: b2.as_strided(t.shape, t.stride(), t.storage_offset())  # noqa: E731
        got = gated_scan_step(at(gate), at(x), torch.zeros(B, D, device="cuda"), out=at(out))
        assert torch.equal(got, want) and torch.equal(at(out), want)
    keep, state = buf.clone(), torch.zeros(B, D, device="cuda")
    reset = buf.view(torch.uint8)[:, 0]
    for out, r in ((buf[:, 1:D + 1], None), (buf[:, D - 1:2 * D - 1], None), (buf[:, 2 * D - 1:3 * D - 1], None), (buf[:, :D], reset)):
        with pytest.raises(RuntimeError, match="share memory"):
            gated_scan_step(gate, x, state, reset=r, out=out)
    assert torch.equal(buf, keep) and not bool(state.any())
