"""A diagonal Gaussian policy's clipped loss with its KL and entropy terms and its gradients, and the sampling of its
actions, on the device (include/marl_amd_env.h, group D).

Rows are agents at steps: mean is (..., A) with any leading axes, everything with one value per row has those leading axes.
Tensors may be strided views -- an action ring (T, E, A, n) of DeviceReplay is passed as ring.transpose(-1, -2) -- and
are read where they are when their leading axes but the last can be walked with one stride (otherwise they are copied).
mean and log_std are float32 or bfloat16, everything else float32.  No CPU fallback."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .recurrence import _DTYPES, _guard_leaves, _need, _on_device, _ptr, _workspace

STATS_FIELDS = ("gain", "kl", "entropy", "clipped", "ratio", "rows")


def _walk(t: torch.Tensor, lead: int) -> Optional[Tuple[int, int]]:
    """Strides (sb, sn) that walk t's first `lead` axes as (all but the last, the last); None if there are none."""
    shape, st = t.shape, t.stride()
    sn = st[lead - 1] if lead else 0
    sb, span = 0, None
    for k in range(lead - 2, -1, -1):
        if shape[k] == 1:
            continue
        if span is None:
            sb, span = st[k], st[k] * shape[k]
        elif st[k] != span:
            return None
        else:
            span = st[k] * shape[k]
    return sb, sn


def _rows(t: Optional[torch.Tensor], lead: int, axis: bool):
    """(struct asm_rows, the tensor it points into) of an input."""
    if t is None:
        return _lib.AsmRows(None, 0, 0, 0), None
    w = _walk(t, lead)
    if w is None:
        t = t.contiguous()
        w = _walk(t, lead)
    return _lib.AsmRows(t.data_ptr(), w[0], w[1], t.stride(-1) if axis else 0), t


def _rows_out(t: torch.Tensor, lead: int, axis: bool, what: str):
    w = _walk(t, lead)
    _need(w is not None, f"{what} must be a tensor whose leading axes but the last can be walked with one stride")
    _need(all(s != 0 for n, s in zip(t.shape, t.stride()) if n > 1), f"{what} must not be an expanded tensor")
    return _lib.AsmRows(t.data_ptr(), w[0], w[1], t.stride(-1) if axis else 0)


def _dims(lead) -> Tuple[int, int]:
    return (math.prod(lead[:-1]), lead[-1]) if lead else (1, 1)


def _check_policy(fn, mean, log_std, rows_of):
    _need(mean.dim() >= 1 and 1 <= mean.shape[-1] <= 32, f"{fn}: mean must be (..., A) with 1 to 32 action components, got {tuple(mean.shape)}")
    _need(mean.dtype in _DTYPES and log_std.dtype == mean.dtype, f"{fn}: mean and log_std must both be float32 or bfloat16, got {mean.dtype} and {log_std.dtype}")
    shared = log_std.shape == mean.shape[-1:]
    _need(shared or log_std.shape == mean.shape, f"{fn}: log_std must have the shape {tuple(mean.shape[-1:])} or {tuple(mean.shape)}")
    for name, (t, axis) in rows_of.items():
        want = mean.shape if axis else mean.shape[:-1]
        _need(t is None or (t.shape == want and t.dtype == torch.float32), f"{fn}: {name} must be a float32 tensor of shape {tuple(want)}")
    return shared


class _ClippedLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, mean, log_std, actions, old, ref, adv, mask, moments, shared, clip, kl_coef, entropy_coef):
        ctx.set_materialize_grads(False)
        loss, stats, dmean, dstd = _loss(mean, log_std, actions, old, ref, adv, mask, moments, shared, clip, kl_coef, entropy_coef)
        ctx.grads, ctx.args = (dmean, dstd), (shared, clip, kl_coef, entropy_coef)
        ctx.save_for_backward(mean, log_std, actions, old, ref, adv, mask, moments)
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        none = (None,) * 10
        if g is None:
            return (None, None) + none
        # the gradients of the forward pass are handed out once; a second backward pass over a retained graph makes its own
        tensors = ctx.saved_tensors                                     # (notices inputs overwritten since)
        grads, ctx.grads = ctx.grads, None
        dmean, dstd = grads if grads is not None else _loss(*tensors, *ctx.args)[2:]
        with torch.cuda.device(dmean.device):
            rc = _lib.load().asm_policy_loss_scale(_DTYPES[dmean.dtype], g.data_ptr(), dmean.numel(), dmean.data_ptr(), dstd.numel(), dstd.data_ptr(),
                                                   torch.cuda.current_stream(dmean.device).cuda_stream)
        _lib.check(rc, "asm_policy_loss_scale")
        return (dmean, dstd) + none


def _loss(mean, log_std, actions, old, ref, adv, mask, moments, shared, clip, kl_coef, entropy_coef):
    lib, dev = _lib.load(), mean.device
    lead, A = mean.dim() - 1, mean.shape[-1]
    B, n = _dims(mean.shape[:-1])
    out = torch.empty(7, dtype=torch.float32, device=dev)
    loss, stats = out[0], out[1:]
    dmean = torch.empty(mean.shape, dtype=mean.dtype, device=dev)
    dstd = torch.empty(log_std.shape, dtype=mean.dtype, device=dev)
    need = lib.asm_policy_loss_workspace(B * n, A)
    ws = _workspace(need, dev)
    r_std = (_lib.AsmRows(log_std.data_ptr(), 0, 0, log_std.stride(0)), log_std) if shared else _rows(log_std, lead, True)
    held = [_rows(mean, lead, True), r_std, _rows(actions, lead, True), _rows(old, lead, False), _rows(ref, lead, False),
            _rows(adv, lead, False), _rows(mask, lead, False)]
    with torch.cuda.device(dev):
        rc = lib.asm_policy_loss(_DTYPES[mean.dtype], B, n, A, int(shared), *[h[0] for h in held], _ptr(moments), clip, kl_coef, entropy_coef,
                                 loss.data_ptr(), stats.data_ptr(), dmean.data_ptr(), dstd.data_ptr(), _ptr(ws), max(need, 0),
                                 torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, "asm_policy_loss")
    return loss, stats, dmean, dstd


def clipped_policy_loss(mean: torch.Tensor, log_std: torch.Tensor, actions: torch.Tensor, log_pi_old: torch.Tensor, adv: torch.Tensor, *,
                        log_pi_ref: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                        adv_moments: Optional[torch.Tensor] = None, clip: float = 0.2, kl_coef: float = 0.0,
                        entropy_coef: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, stats) of a Gaussian policy on recorded actions.  With the ratio q = exp(log_pi - log_pi_old) and D = log_pi_ref - log_pi
    (without log_pi_ref the old policy is the reference), per row

        -min(q A, clip(q, 1 - clip, 1 + clip) A) + kl_coef (e^D - 1 - D) - entropy_coef H

    and loss (float32 scalar) is the mean over the rows whose mask (bool or uint8) is set; 0 with zero gradients if there are
    none.  What a masked row holds does not matter.  Differentiable (once) in mean and log_std; the gradients are computed in
    the same pass.  log_std: mean's shape, or (A,) for all rows.  adv_moments: the (mean, 1 / deviation) that
    advantages(..., moments=True) returns; A = (adv - mean) / deviation then, else A = adv.
    stats: 6 floats, STATS_FIELDS (means over the valid rows of min(..), e^D - 1 - D, H, rows cut off, q; the rows)."""
    fn = "clipped_policy_loss"
    shared = _check_policy(fn, mean, log_std, dict(actions=(actions, True), log_pi_old=(log_pi_old, False), log_pi_ref=(log_pi_ref, False), adv=(adv, False)))
    _need(mask is None or (mask.shape == mean.shape[:-1] and mask.dtype in (torch.bool, torch.uint8)), f"{fn}: mask must be a bool or uint8 tensor of shape {tuple(mean.shape[:-1])}")
    _need(adv_moments is None or (adv_moments.shape == (2,) and adv_moments.dtype == torch.float32), f"{fn}: adv_moments must be two float32 numbers")
    _need(0.0 < clip < math.inf and math.isfinite(kl_coef) and math.isfinite(entropy_coef), f"{fn}: clip must be positive, the coefficients finite")
    for name, t in (("actions", actions), ("log_pi_old", log_pi_old), ("log_pi_ref", log_pi_ref), ("adv", adv), ("adv_moments", adv_moments)):
        _need(t is None or not (t.requires_grad and torch.is_grad_enabled()), f"{fn}: no gradient for {name}: pass it detached")
    _on_device(fn, mean.device, log_std, actions, log_pi_old, log_pi_ref, adv, mask, adv_moments)
    adv_moments = None if adv_moments is None else adv_moments.contiguous()
    loss, stats = _ClippedLoss.apply(mean, log_std, actions, log_pi_old, log_pi_ref, adv, mask, adv_moments, shared, float(clip), float(kl_coef), float(entropy_coef))
    return (_guard_leaves(loss, mean.device) if loss.requires_grad else loss), stats


@torch.no_grad()
def gaussian_act(mean: torch.Tensor, log_std: torch.Tensor, noise: torch.Tensor, *, actions: Optional[torch.Tensor] = None,
                 log_pi: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A rollout's actions, without gradients: (actions, log_pi) with actions = mean + e^log_std noise and log_pi the
    log-probability of the actions as they are stored in float32, so that a ratio taken from it later starts at 1.
    noise: standard normal draws of mean's shape (torch.randn); log_std: mean's shape, or (A,) for all rows.  actions, log_pi: where to write
    (strided views are fine: DeviceReplay.action_slot().transpose(-1, -2))."""
    return _act("gaussian_act", mean, log_std, noise, actions, log_pi)


@torch.no_grad()
def gaussian_log_pi(mean: torch.Tensor, log_std: torch.Tensor, actions: torch.Tensor, *, log_pi: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Log-probabilities of given actions, without gradients: what a reference policy says of a recorded episode."""
    return _act("gaussian_log_pi", mean, log_std, None, actions, log_pi)[1]


def _act(fn, mean, log_std, noise, actions, log_pi):
    shared = _check_policy(fn, mean, log_std, dict(noise=(noise, True), actions=(actions, True), log_pi=(log_pi, False)))
    dev, lead, A = mean.device, mean.dim() - 1, mean.shape[-1]
    _on_device(fn, dev, log_std, noise, actions, log_pi)
    B, n = _dims(mean.shape[:-1])
    if actions is None:
        actions = torch.empty(mean.shape, dtype=torch.float32, device=dev)
    if log_pi is None:
        log_pi = torch.empty(mean.shape[:-1], dtype=torch.float32, device=dev)
    if noise is not None:
        r_act = _rows_out(actions, lead, True, f"{fn}: actions")
    else:
        r_act, held_act = _rows(actions, lead, True)
    r_lp = _rows_out(log_pi, lead, False, f"{fn}: log_pi")
    r_std = (_lib.AsmRows(log_std.data_ptr(), 0, 0, log_std.stride(0)), log_std) if shared else _rows(log_std, lead, True)
    r_mean, r_noise = _rows(mean, lead, True), _rows(noise, lead, True)
    with torch.cuda.device(dev):
        rc = _lib.load().asm_gaussian_act(_DTYPES[mean.dtype], B, n, A, r_mean[0], r_std[0], r_noise[0], r_act, r_lp, torch.cuda.current_stream(dev).cuda_stream)
    _lib.check(rc, "asm_gaussian_act")
    torch.autograd.graph.increment_version([log_pi] if noise is None else [actions, log_pi])
    return actions, log_pi
