"""What the sequence operators refuse, at the Python entry points (before any device is asked for) and at the C ABI
(before anything is launched).  Runs on the CPU."""
import struct

import pytest
import torch

from marl_amd import _lib
from marl_amd.policy_loss import clipped_policy_loss, gaussian_act, gaussian_log_pi
from marl_amd.recurrence import advantages, gated_scan, gated_scan_step

f = torch.zeros
T, B, D = 4, 3, 8
G = f(T, B, D)
BF = torch.bfloat16


@pytest.mark.parametrize("args,kw,msg", [
    ((f(T, B), f(T, B)), {}, "three axes"),
    ((G, f(T, B, D + 1)), {}, "one shape"),
    ((G, G.to(BF)), {}, "both be float32"),
    ((G.half(), G.half()), {}, "both be float32"),
    ((G.double(), G.double()), {}, "both be float32"),
    ((G, G, f(B, D + 1)), {}, "h0"),
    ((G, G, f(1, D)), {}, "h0"),
    ((G, G, f(B, D).to(BF)), {}, "h0"),
    ((G, G), dict(resets=f(T, B)), "resets"),
    ((G, G), dict(resets=f(B, T, dtype=torch.bool)), "resets"),
    ((G, G), dict(resets=f(T, B, dtype=torch.bool), batch_first=True, lengths=None), "HIP device"),
    ((G, G), dict(lengths=f(B, dtype=torch.int64)), "lengths"),
    ((G, G), dict(lengths=f(T, dtype=torch.int32)), "lengths"),
    ((G, G), {}, "HIP device"),
])
def test_scan(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        gated_scan(*args, **kw)


@pytest.mark.parametrize("args,kw,msg", [
    ((f(B, D), f(B, D), f(B, D + 1)), {}, "one shape"),
    ((f(B, D), f(B, D), f(B, D).to(BF)), {}, "state"),
    ((f(B, D), f(B, D), f(D, B).t()), {}, "contiguous"),
    ((f(B, D), f(B, D), f(B, D, requires_grad=True)), {}, "gradient"),
    ((f(B, D), f(B, D).to(BF), f(B, D)), {}, "both be float32"),
    ((f(B, D), f(B, D), f(B, D)), dict(reset=f(B)), "reset"),
    ((f(B, D), f(B, D), f(B, D)), dict(out=f(B, D).to(BF)), "out"),
    ((f(B, D), f(B, D), f(B, D)), dict(out=f(D).expand(B, D)), "out"),
    ((f(B, D), f(B, D), f(B, D)), dict(out=f(D, B).t()), "out"),
    ((f(B, D), f(B, D), f(B, D)), {}, "HIP device"),
])
def test_step(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        gated_scan_step(*args, **kw)


@pytest.mark.parametrize("args,kw,msg", [
    ((f(T), f(T + 1)), {}, "non-empty"),
    ((f(0, B), f(1, B)), {}, "non-empty"),
    ((f(T, 0), f(T + 1, 0)), {}, "non-empty"),
    ((f(T, B), f(T, B)), {}, "values"),
    ((f(T, B), f(T + 1, B).double()), {}, "float32"),
    ((f(T, B), f(T + 1, B)), dict(dones=f(T, B)), "dones"),
    ((f(T, B), f(T + 1, B)), dict(lengths=f(T, dtype=torch.int32)), "lengths"),
    ((f(T, B), f(T + 1, B)), dict(gamma=1.5), "gamma"),
    ((f(T, B), f(T + 1, B)), dict(lam=float("nan")), "gamma"),
    ((f(T, B), f(T + 1, B)), {}, "HIP device"),
])
def test_advantages(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        advantages(*args, **kw)


M, S, N = f(5, 2), f(2), f(5)


@pytest.mark.parametrize("args,kw,msg", [
    ((f(5, 33), f(33), f(5, 33), N, N), {}, "1 to 32"),
    ((f(5, 0), f(0), f(5, 0), N, N), {}, "1 to 32"),
    ((M.half(), S.half(), M, N, N), {}, "float32 or bfloat16"),
    ((M, S.to(BF), M, N, N), {}, "float32 or bfloat16"),
    ((M, f(1), M, N, N), {}, "log_std"),
    ((M, f(5, 1), M, N, N), {}, "log_std"),
    ((M, S, f(2, 5), N, N), {}, "actions"),
    ((M, S, M.to(BF), N, N), {}, "actions"),
    ((M, S, M, f(5, 1), N), {}, "log_pi_old"),
    ((M, S, M, N, f(4)), {}, "adv"),
    ((M, S, M, N, N), dict(log_pi_ref=f(4)), "log_pi_ref"),
    ((M, S, M, N, N), dict(mask=N), "mask"),
    ((M, S, M, N, N), dict(adv_moments=f(3)), "adv_moments"),
    ((M, S, M, N, N), dict(clip=0.0), "clip"),
    ((M, S, M, N, N), dict(clip=float("inf")), "clip"),
    ((M, S, M, N, N), dict(kl_coef=float("nan")), "finite"),
    ((M, S, M, f(5, requires_grad=True), N), {}, "detached"),
    ((M, S, M, N, f(5, requires_grad=True)), {}, "detached"),
    ((M, S, M, N, N), {}, "HIP device"),
])
def test_loss(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        clipped_policy_loss(*args, **kw)


def test_act():
    for args, kw, msg in (((M, S, f(5, 3)), {}, "noise"), ((M, S, M), dict(log_pi=f(5, 1)), "log_pi"), ((M, S, M), dict(actions=f(2, 5)), "actions"), ((M, S, M), {}, "HIP device")):
        with pytest.raises(ValueError, match=msg):
            gaussian_act(*args, **kw)
    with pytest.raises(ValueError, match="HIP device"):
        gaussian_log_pi(M, S, M)


def _msg(lib):
    return lib.asm_last_error().decode()


def test_c_abi_refuses_before_it_launches():
    """Made-up addresses: a call that got as far as a launch would fail differently."""
    lib = _lib.load()
    p = 1 << 20
    fwd = lambda dt=0, T=T, B=B, D=D, gate=p, x=p, h=p, ws=None, n=0, kept=None: lib.asm_gated_scan_forward(  # noqa: E731
        dt, T, B, D, gate, 0, 0, x, 0, 0, None, None, 0, 0, None, h, 0, 0, None, kept, ws, n, None)
    for kw, msg in ((dict(dt=7), "dtype"), (dict(T=-1), "negative"), (dict(B=1 << 31), "too large"), (dict(B=1 << 29, D=2), "too large"), (dict(B=1 << 20, D=1 << 20), "too large"),
                    (dict(T=1 << 31), "too large"), (dict(gate=None), "NULL"), (dict(x=None), "NULL"), (dict(h=None), "NULL"),
                    (dict(T=100000), "workspace"), (dict(T=100000, ws=p, n=8), "workspace"), (dict(T=100000, ws=p + 8, n=1 << 40), "aligned"), (dict(kept=p + 4), "kept")):
        assert fwd(**kw) != 0 and msg in _msg(lib), (kw, _msg(lib))
    assert fwd(B=0, gate=None, x=None, h=None) == 0                     # nothing to do
    assert lib.asm_gated_scan_workspace(0, 100000, B, D) > 0 and lib.asm_gated_scan_workspace(0, -1, B, D) < 0
    assert lib.asm_gated_scan_kept(0, 20, B, D) == 0 and lib.asm_gated_scan_kept(0, 20, 600, 256) == 3 * 600 * 256 * 4 and lib.asm_gated_scan_kept(5, 20, B, D) < 0
    bwd = lambda T=T, dgate=p, h=p: lib.asm_gated_scan_backward(0, T, B, D, p, 0, 0, p, 0, 0, h, 0, 0, None, None, 0, 0, None, None, 0, 0, None,  # noqa: E731
                                                                dgate, 0, 0, p, 0, 0, None, None, None, 0, None)
    assert bwd(dgate=None) != 0 and "NULL" in _msg(lib)
    assert bwd(h=None) != 0 and "NULL" in _msg(lib)
    assert bwd(T=100000) != 0 and "workspace" in _msg(lib)
    assert lib.asm_gated_scan_step(0, B, D, p, D, p, D, None, None, 0, p, D, None) != 0 and "NULL" in _msg(lib)
    adv = lambda T=T, g=0.9, r=p, ws=None, n=0: lib.asm_advantages_f32(T, B, D, r, 0, p, 0, None, 0, None, g, 0.9, p, p, None, ws, n, None)  # noqa: E731
    for kw, msg in ((dict(T=0), "no steps"), (dict(g=1.5), "gamma"), (dict(g=float("nan")), "gamma"), (dict(r=None), "NULL"), (dict(T=100000), "workspace")):
        assert adv(ws=None, **kw) != 0 and msg in _msg(lib), (kw, _msg(lib))
    R = lambda *ptrs: struct.pack(f"{4 * len(ptrs)}q", *(v for q in ptrs for v in (q, 0, 0, 0)))  # noqa: E731
    loss = lambda B=1, n=5, A=2, mean=p, std=p, clip=0.2, dm=p, nb=0: lib.asm_policy_loss(  # noqa: E731
        0, B, n, A, 1, R(mean, std, p, p, 0, p, 0), None, clip, 0.0, 0.0, p, p, dm, p, None, nb, None)
    for kw, msg in ((dict(A=0), "A = 0"), (dict(A=33), "A = 33"), (dict(mean=0), "NULL"), (dict(std=0), "NULL"), (dict(dm=None), "NULL"),
                    (dict(clip=-1.0), "clip"), (dict(clip=float("nan")), "clip"), (dict(n=1 << 20), "workspace"), (dict(B=1 << 20, n=1 << 20), "too large")):
        assert loss(**kw) != 0 and msg in _msg(lib), (kw, _msg(lib))
    assert lib.asm_policy_loss_scale(0, None, 4, p, 0, None, None) != 0
    assert lib.asm_policy_loss(0, 1, 5, 2, 1, None, None, 0.2, 0.0, 0.0, p, p, p, p, None, 0, None) != 0 and "NULL" in _msg(lib)
    assert lib.asm_gaussian_act(0, 1, 5, 2, R(p, p, p, 0, p), None) != 0 and "NULL" in _msg(lib)
    assert lib.asm_gaussian_act(0, 1, 5, 2, None, None) != 0 and "NULL" in _msg(lib)
    assert lib.asm_gaussian_act(3, 1, 5, 2, R(p, p, p, p, p), None) != 0 and "dtype" in _msg(lib)
