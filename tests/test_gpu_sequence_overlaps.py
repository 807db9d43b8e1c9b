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


def test_actions(torch_cuda):
    torch = torch_cuda
    from marl_amd.policy_loss import gaussian_act, gaussian_log_pi
    E, n, A = 5, 30, 2
    buf = torch.randn(E, n, 4 * A + 1, device="cuda")
    mean, std, noise, lp = buf[..., :A], buf[..., A:2 * A], buf[..., 2 * A:3 * A], buf[..., 4 * A]
    want, wl = gaussian_act(mean.clone(), std.clone(), noise.clone())
    for act in (buf[..., 3 * A:4 * A], noise, mean, std):               # a head's output and its actions in one buffer, then in place
        b2 = buf.clone()
        at = lambda t: b2.as_strided(t.shape, t.stride(), t.storage_offset())  # noqa: E731
        got, gl = gaussian_act(at(mean), at(std), at(noise), actions=at(act), log_pi=at(lp))
        assert torch.equal(got, want) and torch.equal(at(act), want) and torch.equal(gl, wl) and torch.equal(at(lp), wl)
    ring = torch.zeros(3, E, A, n, device="cuda")                       # the replay's layout
    gaussian_act(mean, std, noise, actions=ring[1].transpose(-1, -2), log_pi=ring[2, :, 0])
    assert torch.equal(ring[1].transpose(-1, -2), want) and torch.equal(ring[2, :, 0], wl) and not bool(ring[0].any()) and not bool(ring[2, :, 1].any())
    keep = buf.clone()
    for kw in (dict(actions=buf[..., 1:A + 1]), dict(actions=buf[..., 2 * A + 1:3 * A + 1]), dict(log_pi=buf[..., 0]), dict(log_pi=buf[..., 3 * A - 1]),
               dict(actions=buf[..., 3 * A:4 * A], log_pi=buf[..., 4 * A - 1])):
        with pytest.raises(RuntimeError, match="share memory"):
            gaussian_act(mean, std, noise, **kw)
    with pytest.raises(RuntimeError, match="share memory"):
        gaussian_log_pi(mean, std, noise, log_pi=buf[..., 2 * A])
    with pytest.raises(RuntimeError, match="share memory"):             # rows of one output that lie in each other
        gaussian_act(mean, std, noise, actions=torch.zeros(400, device="cuda").as_strided((E, n, A), (30, 1, 1)))
    assert torch.equal(buf, keep)
