"""A diagonal Gaussian policy's clipped loss with its KL and entropy terms and its gradients, and the sampling of its
actions, on the device (include/marl_amd_env.h, group D).

Rows are agents at steps: mean is (..., A) with any leading axes, everything with one value per row has those leading axes.
Tensors may be strided views -- an action ring (T, E, A, n) of DeviceReplay is passed as ring.transpose(-1, -2) -- and
are read where they are when their leading axes but the last can be walked with one stride (otherwise they are copied).
mean and log_std are float32 or bfloat16, everything else float32.  No CPU fallback."""
from __future__ import annotations

import math
import struct
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from .recurrence import _DTYPES, _FLAGS, _call, _capture, _guard_leaves, _need, _no_tangents, _on_device, _once, _ptr, _workspace

STATS_FIELDS = ("gain", "kl", "entropy", "clipped", "ratio", "rows")
_NO_ROWS = (0, 0, 0, 0)
_pack_loss = struct.Struct("28q").pack                                  # struct asm_loss_rows
_pack_act = struct.Struct("20q").pack                                   # struct asm_act_rows


def _walk(shape, st, lead: int) -> Optional[Tuple[int, int]]:
    """Strides (sb, sn) that walk a tensor's first `lead` axes as (all but the last, the last); None if there are none."""
    if lead < 2:
        return (0, st[0]) if lead else (0, 0)
    if lead == 2:
        return st[0], st[1]
    sb, span = 0, None
    for k in range(lead - 2, -1, -1):
        if shape[k] == 1:
            continue
        if span is None:
            sb = st[k]
        elif st[k] != span:
            return None
        span = st[k] * shape[k]
    return sb, st[lead - 1]


def _rows(t: torch.Tensor, lead: int, axis: bool):
    """One struct asm_rows (as four numbers) of an input, and the tensor it points into."""
    st = t.stride()
    w = _walk(t.shape, st, lead)
    if w is None:
        t = t.contiguous()
        st = t.stride()
        w = _walk(t.shape, st, lead)
    return (t.data_ptr(), w[0], w[1], st[-1] if axis else 0), t


def _rows_std(t: torch.Tensor, lead: int, shared: bool):
    return ((t.data_ptr(), 0, 0, t.stride(0)), t) if shared else _rows(t, lead, True)


def _rows_out(t: torch.Tensor, lead: int, axis: bool, what: str):
    shape, st = t.shape, t.stride()
    w = _walk(shape, st, lead)
    if w is None or 0 in st:
        _need(w is not None, f"{what} must be a tensor whose leading axes but the last can be walked with one stride")
        _need(all(s != 0 for n, s in zip(shape, st) if n > 1), f"{what} must not be an expanded tensor")
    return t.data_ptr(), w[0], w[1], st[-1] if axis else 0


def _dims(lead) -> Tuple[int, int]:
    return (lead[:-1].numel(), lead[-1]) if lead else (1, 1)


def _policy_ok(mean, log_std, full, per_row) -> bool:
    """Shapes, types and devices of a policy operator's tensors: full ones like mean, per_row ones without its last axis."""
    shape, dt, dev = mean.shape, mean.dtype, mean.device
    if not (shape and 1 <= shape[-1] <= 32 and dt in _DTYPES and log_std.dtype == dt and log_std.device == dev and dev.type == "cuda" and
            (log_std.shape == shape[-1:] or log_std.shape == shape)):
        return False
    for t in full:
        if t is not None and not (t.shape == shape and t.dtype == torch.float32 and t.device == dev):
            return False
    lead = shape[:-1]
    for t in per_row:
        if t is not None and not (t.shape == lead and t.dtype == torch.float32 and t.device == dev):
            return False
    return True


def _explain_policy(fn, mean, log_std, full, per_row):
    _need(mean.dim() >= 1 and 1 <= mean.shape[-1] <= 32, f"{fn}: mean must be (..., A) with 1 to 32 action components, got {tuple(mean.shape)}")
    _need(mean.dtype in _DTYPES and log_std.dtype == mean.dtype, f"{fn}: mean and log_std must both be float32 or bfloat16, got {mean.dtype} and {log_std.dtype}")
    _need(log_std.shape == mean.shape[-1:] or log_std.shape == mean.shape, f"{fn}: log_std must have the shape {tuple(mean.shape[-1:])} or {tuple(mean.shape)}")
    for names, want in ((full, mean.shape), (per_row, mean.shape[:-1])):
        for name, t in names.items():
            _need(t is None or (t.shape == want and t.dtype == torch.float32), f"{fn}: {name} must be a float32 tensor of shape {tuple(want)}")


class _ClippedLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, mean, log_std, fixed, options):                    # fixed: the tensors without a gradient
        ctx.set_materialize_grads(False)
        loss, stats, dmean, dstd = _loss(mean, log_std, *fixed, *options)
        ctx.grads, ctx.options, ctx.capture = (dmean, dstd), options, _capture(mean.device)
        ctx.save_for_backward(mean, log_std, *fixed)
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    def backward(ctx, g, _):
        if g is None:
            return None, None, None, None
        _once("clipped_policy_loss")
        # the gradients of the forward pass are handed out once, scaled where they are; a second backward pass over a retained graph
        # makes its own, and so does one that is captured apart from the forward pass: its replays would scale them again
        tensors = ctx.saved_tensors                                     # (notices inputs overwritten since)
        grads = None
        if ctx.capture == _capture(g.device):
            grads, ctx.grads = ctx.grads, None
        dmean, dstd = grads if grads is not None else _loss(*tensors, *ctx.options)[2:]
        _call("asm_policy_loss_scale", dmean.device, _DTYPES[dmean.dtype], g.data_ptr(), dmean.numel(), dmean.data_ptr(), dstd.numel(), dstd.data_ptr())
        return dmean, dstd, None, None


@lru_cache(maxsize=1024)
def _loss_workspace(rows: int, A: int) -> int:
    return _lib.load().asm_policy_loss_workspace(rows, A)


def _loss(mean, log_std, actions, old, ref, adv, mask, moments, shared, clip, kl_coef, entropy_coef):
    dev, shape, dt = mean.device, mean.shape, mean.dtype
    lead, A = len(shape) - 1, shape[-1]
    B, n = _dims(shape[:-1])
    loss = torch.empty((), dtype=torch.float32, device=dev)
    stats = torch.empty(6, dtype=torch.float32, device=dev)
    dmean = torch.empty(shape, dtype=dt, device=dev)
    dstd = torch.empty(log_std.shape, dtype=dt, device=dev)
    need = _loss_workspace(B * n, A)
    ws = _workspace(need, dev)
    moments = None if moments is None else moments.contiguous()
    r0, k0 = _rows(mean, lead, True)                                    # (k: the tensors a copy may have been made of)
    r1, k1 = _rows_std(log_std, lead, shared)
    r2, k2 = _rows(actions, lead, True)
    r3, k3 = _rows(old, lead, False)
    r4, k4 = _rows(ref, lead, False) if ref is not None else (_NO_ROWS, None)
    r5, k5 = _rows(adv, lead, False)
    r6, k6 = _rows(mask, lead, False) if mask is not None else (_NO_ROWS, None)
    _call("asm_policy_loss", dev, _DTYPES[dt], B, n, A, shared, _pack_loss(*r0, *r1, *r2, *r3, *r4, *r5, *r6), _ptr(moments), clip, kl_coef,
          entropy_coef, loss.data_ptr(), stats.data_ptr(), dmean.data_ptr(), dstd.data_ptr(), _ptr(ws), need)
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
    stats: 6 floats, STATS_FIELDS (means over the valid rows of min(..), e^D - 1 - D, H, rows cut off, q; the rows).  The mean of
    e^D - 1 - D estimates KL(pi || pi_ref) without bias for actions drawn from pi itself: near the first update after the rollout.
    For actions of an older policy, and with that policy as the reference, it is a distance (0 where the two agree) but no such estimate.
    A row is computed in double and rounded once; with kl_coef = 0 that term takes no part, however far off a row is.
    Without gradients enabled they are computed all the same."""
    dev, lead = mean.device, mean.shape[:-1]
    if not (_policy_ok(mean, log_std, (actions,), (log_pi_old, log_pi_ref, adv)) and
            (mask is None or (mask.shape == lead and mask.dtype in _FLAGS and mask.device == dev)) and
            (adv_moments is None or (adv_moments.shape == (2,) and adv_moments.dtype == torch.float32 and adv_moments.device == dev)) and
            0.0 < clip < math.inf and math.isfinite(kl_coef) and math.isfinite(entropy_coef) and
            not (torch.is_grad_enabled() and (actions.requires_grad or log_pi_old.requires_grad or adv.requires_grad or
                                              (log_pi_ref is not None and log_pi_ref.requires_grad) or
                                              (adv_moments is not None and adv_moments.requires_grad)))):
        _explain_loss(mean, log_std, actions, log_pi_old, adv, log_pi_ref, mask, adv_moments, clip, kl_coef, entropy_coef)
    _no_tangents("clipped_policy_loss", mean, log_std, actions, log_pi_old, adv, log_pi_ref, adv_moments)
    shared = int(log_std.shape == mean.shape[-1:])
    loss, stats = _ClippedLoss.apply(mean, log_std, (actions, log_pi_old, log_pi_ref, adv, mask, adv_moments),
                                     (shared, float(clip), float(kl_coef), float(entropy_coef)))
    return (_guard_leaves(loss, mean.device) if loss.requires_grad else loss), stats


def _explain_loss(mean, log_std, actions, log_pi_old, adv, log_pi_ref, mask, adv_moments, clip, kl_coef, entropy_coef):
    fn = "clipped_policy_loss"
    _explain_policy(fn, mean, log_std, dict(actions=actions), dict(log_pi_old=log_pi_old, log_pi_ref=log_pi_ref, adv=adv))
    _need(mask is None or (mask.shape == mean.shape[:-1] and mask.dtype in _FLAGS), f"{fn}: mask must be a bool or uint8 tensor of shape {tuple(mean.shape[:-1])}")
    _need(adv_moments is None or (adv_moments.shape == (2,) and adv_moments.dtype == torch.float32), f"{fn}: adv_moments must be two float32 numbers")
    _need(0.0 < clip < math.inf and math.isfinite(kl_coef) and math.isfinite(entropy_coef), f"{fn}: clip must be positive, the coefficients finite")
    for name, t in (("actions", actions), ("log_pi_old", log_pi_old), ("log_pi_ref", log_pi_ref), ("adv", adv), ("adv_moments", adv_moments)):
        _need(t is None or not (t.requires_grad and torch.is_grad_enabled()), f"{fn}: no gradient for {name}: pass it detached")
    _on_device(fn, mean.device, log_std, actions, log_pi_old, log_pi_ref, adv, mask, adv_moments)
    raise ValueError(f"{fn}: bad arguments")


def gaussian_act(mean: torch.Tensor, log_std: torch.Tensor, noise: torch.Tensor, *, actions: Optional[torch.Tensor] = None,
                 log_pi: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A rollout's actions, without gradients: (actions, log_pi) with actions = mean + e^log_std noise and log_pi the
    log-probability of the actions as they are stored in float32, so that a ratio taken from it later starts at 1.
    noise: standard normal draws of mean's shape (torch.randn); log_std: mean's shape, or (A,) for all rows.  actions, log_pi: where to write
    (strided views are fine: DeviceReplay.action_slot().transpose(-1, -2); actions may be noise, mean or log_std itself; outputs that
    overlap an input otherwise, each other or themselves are refused)."""
    _need(noise is not None, "gaussian_act: noise must be a float32 tensor of mean's shape")
    return _act("gaussian_act", mean, log_std, noise, actions, log_pi)


def gaussian_log_pi(mean: torch.Tensor, log_std: torch.Tensor, actions: torch.Tensor, *, log_pi: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Log-probabilities of given actions, without gradients: what a reference policy says of a recorded episode."""
    _need(actions is not None, "gaussian_log_pi: actions must be a float32 tensor of mean's shape")
    return _act("gaussian_log_pi", mean, log_std, None, actions, log_pi)[1]


def _act(fn, mean, log_std, noise, actions, log_pi):
    for name, t in (("actions", None if noise is None else actions), ("log_pi", log_pi)):
        _need(t is None or not (t.requires_grad and torch.is_grad_enabled()), f"{fn}: {name} is written in place and cannot require a gradient")
    if not _policy_ok(mean, log_std, (noise, actions), (log_pi,)):
        _explain_policy(fn, mean, log_std, dict(noise=noise, actions=actions), dict(log_pi=log_pi))
        _on_device(fn, mean.device, log_std, noise, actions, log_pi)
        raise ValueError(f"{fn}: bad arguments")
    dev, shape, dt = mean.device, mean.shape, mean.dtype
    lead, A = len(shape) - 1, shape[-1]
    B, n = _dims(shape[:-1])
    if actions is None:
        actions = torch.empty(shape, dtype=torch.float32, device=dev)
    if log_pi is None:
        log_pi = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    if noise is not None:
        r_act, k_act = _rows_out(actions, lead, True, "actions"), None
        r_noise, k_noise = _rows(noise, lead, True)
    else:
        r_act, k_act = _rows(actions, lead, True)
        r_noise, k_noise = _NO_ROWS, None
    r_mean, k_mean = _rows(mean, lead, True)
    r_std, k_std = _rows_std(log_std, lead, log_std.shape == shape[-1:])
    _call("asm_gaussian_act", dev, _DTYPES[dt], B, n, A, _pack_act(*r_mean, *r_std, *r_noise, *r_act, *_rows_out(log_pi, lead, False, "log_pi")))
    torch.autograd.graph.increment_version((log_pi,) if noise is None else (actions, log_pi))
    return actions, log_pi
