"""Dual tensors (forward-mode differentiation) are refused, not computed without their tangent."""
import pytest

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused(torch_cuda):
    torch = torch_cuda
    import torch.autograd.forward_ad as fw
    from marl_amd.policy_loss import clipped_policy_loss
    from marl_amd.recurrence import gated_scan
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    gate, x, h0 = r(4, 2, 8), r(4, 2, 8), r(2, 8)
    rows = [r(6, 2), r(2), r(6, 2), r(6), r(6)]
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for k in range(3):
                    args = [gate, x, h0]
                    args[k] = dual(args[k])
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        gated_scan(*args)
                for k in range(5):
                    args = list(rows)
                    args[k] = dual(args[k])
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        clipped_policy_loss(*args)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    clipped_policy_loss(*rows, log_pi_ref=dual(r(6)))
        inside = gated_scan(gate, x, h0)[0]                              # tensors without a tangent are
    assert torch.equal(inside, gated_scan(gate, x, h0)[0])
