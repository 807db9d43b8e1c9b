"""Outputs that the sequence operators refuse to write.  Runs on the CPU: refused before any device is asked for."""
import pytest
import torch

from marl_amd.policy_loss import gaussian_act, gaussian_log_pi

f = torch.zeros
M, S, N = f(5, 2), f(2), f(5)


def _grad(*shape):
    return f(*shape, requires_grad=True)


@pytest.mark.parametrize("call", [
    lambda: gaussian_act(M, S, M, actions=_grad(5, 2)),
    lambda: gaussian_act(M, S, M, actions=2 * _grad(5, 2)),
    lambda: gaussian_act(M, S, M, log_pi=_grad(5)),
    lambda: gaussian_log_pi(M, S, M, log_pi=_grad(5)),
])
def test_outputs_that_require_a_gradient(call):
    with pytest.raises(ValueError, match="cannot require a gradient"):
        call()
    with torch.no_grad(), pytest.raises(ValueError, match="HIP device"):
        call()


def test_given_actions_may_require_one():
    with pytest.raises(ValueError, match="HIP device"):
        gaussian_log_pi(_grad(5, 2), S, _grad(5, 2))


def test_no_noise_and_no_actions():
    """(an uninitialised tensor was taken in their place)"""
    with pytest.raises(ValueError, match="noise"):
        gaussian_act(M, S, None)
    with pytest.raises(ValueError, match="noise"):
        gaussian_act(M, S, None, actions=f(5, 2))
    with pytest.raises(ValueError, match="actions"):
        gaussian_log_pi(M, S, None)
