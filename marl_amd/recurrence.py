"""First-order recurrences over time on the device (include/marl_amd_env.h, group D): the gated memory of a policy that
sees only its neighbourhood, over whole sequences with its gradients (gated_scan) and one rollout step at a time
(gated_scan_step), and the advantages and returns of an episode (advantages).

    a = sigmoid(gate_t),   h_t = a h_{t-1} + (1 - a) x_t

float32 or bfloat16 inputs and outputs, the state itself always float32.  Time-major tensors (T, B, D) are what the rings
of DeviceReplay hold; batch_first=True takes (B, T, D).  Tensors may be strided as long as their last axis is contiguous
(others are copied).  No CPU fallback."""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.SEQ_F32, torch.bfloat16: _lib.SEQ_BF16}
_FLAGS = (torch.bool, torch.uint8)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _on_device(fn: str, dev: torch.device, *tensors) -> None:
    _need(dev.type == "cuda", f"{fn}: the tensors are on {dev}: it runs on a HIP device only")
    for t in tensors:
        _need(t is None or t.device == dev, f"{fn}: tensors on different devices")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _tb(t: Optional[torch.Tensor], batch_first: bool) -> Tuple[Optional[int], int, int]:
    """(pointer, stride of time, stride of the batch)"""
    if t is None:
        return None, 0, 0
    s = t.stride()
    return (t.data_ptr(), s[1], s[0]) if batch_first else (t.data_ptr(), s[0], s[1])


def _workspace(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def _call(name: str, dev: torch.device, *args) -> None:
    """One entry point of the library on dev's current stream (its last argument).  A small call is bound by what Python does
    around it: the device is only switched when it is not the current one, and the stream's handle is asked for
    as a number (2.5 us less than through a torch.cuda.Stream object)."""
    fn, index = getattr(_lib.load(), name), dev.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _no_tangents(fn: str, *tensors) -> None:
    """(an operator that is not entered through its autograd function would drop a dual tensor's tangent without a word)"""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{fn} has no forward-mode derivative: its inputs may not be dual tensors")


def _once(fn: str) -> None:
    """(what torch.autograd.function.once_differentiable makes sure of, at a twentieth of its price a call)"""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{fn} is differentiable once: no create_graph=True through it")


def _capture(dev: torch.device) -> int:
    """The capture into a HIP graph that dev's current stream is part of, 0 for none."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _capture(dev)
    return _lib.load().asm_capture_id(_raw_stream(dev.index)) if torch.cuda.is_current_stream_capturing() else 0


def _guard_leaves(out: torch.Tensor, device) -> torch.Tensor:
    """A leaf's accumulation node belongs to the stream it was first used on and lives as long as any graph that uses the
    leaf; a backward pass captured into a HIP graph would have to join that other stream, which ends the process.
    The node remembers its stream (in its own metadata, gone with the node), and such a capture is refused."""
    stream = _raw_stream(device.index)
    for node, _ in out.grad_fn.next_functions:
        if type(node).__name__ == "AccumulateGrad":
            first = node.metadata.setdefault("marl_amd_stream", stream)
            if first != stream and _capture(device):
                raise RuntimeError("captured into a HIP graph while an autograd graph of the same leaf tensor, made on another stream, is alive: "
                                   "drop it (its loss and outputs) before capturing")
    return out


def _explain_scan(gate, x, h0, resets, lengths, B, D):
    fn = "gated_scan"
    _need(gate.dim() == 3 and gate.shape == x.shape, f"{fn}: gate and x must have one shape of three axes, got {tuple(gate.shape)} and {tuple(x.shape)}")
    _need(gate.dtype in _DTYPES and x.dtype == gate.dtype, f"{fn}: gate and x must both be float32 or bfloat16, got {gate.dtype} and {x.dtype}")
    _need(h0 is None or (h0.shape == (B, D) and h0.dtype == torch.float32), f"{fn}: h0 must be a float32 tensor of shape {(B, D)}")
    _need(resets is None or (resets.shape == gate.shape[:2] and resets.dtype in _FLAGS),
          f"{fn}: resets must be a bool or uint8 tensor of shape {tuple(gate.shape[:2])}")
    _need(lengths is None or (lengths.shape == (B,) and lengths.dtype == torch.int32), f"{fn}: lengths must be an int32 tensor of shape {(B,)}")
    _on_device(fn, gate.device, x, h0, resets, lengths)


@lru_cache(maxsize=1024)
def _scan_sizes(dt: int, T: int, B: int, D: int) -> Tuple[int, int]:
    """(workspace, kept states) in bytes: functions of the sizes alone."""
    lib = _lib.load()
    return lib.asm_gated_scan_workspace(dt, T, B, D), lib.asm_gated_scan_kept(dt, T, B, D)


def _scan_forward(gate, x, h0, resets, lengths, batch_first, T, B, D, keep=False):
    dev, dt = gate.device, _DTYPES[gate.dtype]
    h = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
    last = torch.empty((B, D), dtype=torch.float32, device=dev)
    need, states = _scan_sizes(dt, T, B, D)
    ws = _workspace(need, dev)
    kept = _workspace(states, dev) if keep else None
    _call("asm_gated_scan_forward", dev, dt, T, B, D, *_tb(gate, batch_first), *_tb(x, batch_first), _ptr(h0), *_tb(resets, batch_first),
          _ptr(lengths), *_tb(h, batch_first), last.data_ptr(), _ptr(kept), _ptr(ws), need)
    return h, last, kept


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, x, h0, marks, batch_first, dims):
        ctx.set_materialize_grads(False)
        h, last, kept = _scan_forward(gate, x, h0, *marks, batch_first, *dims, keep=True)
        ctx.save_for_backward(gate, x, h, h0, *marks, kept)
        ctx.batch_first, ctx.dims = batch_first, dims
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        _once("gated_scan")
        gate, x, h, h0, resets, lengths, kept = ctx.saved_tensors
        gate, x, h = _dense(gate), _dense(x), _dense(h)                  # (saved-tensor hooks may hand back other strides)
        h0, lengths, kept = (None if t is None else t.contiguous() for t in (h0, lengths, kept))
        T, B, D = ctx.dims
        bf, dev, dt = ctx.batch_first, gate.device, _DTYPES[gate.dtype]
        dh = None if dh is None else _dense(dh)
        dlast = None if dlast is None else dlast.contiguous()
        dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
        dx = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
        dh0 = torch.empty((B, D), dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        need = _scan_sizes(dt, T, B, D)[0]
        ws = _workspace(need, dev)
        _call("asm_gated_scan_backward", dev, dt, T, B, D, *_tb(gate, bf), *_tb(x, bf), *_tb(h, bf), _ptr(h0), *_tb(resets, bf), _ptr(lengths),
              *_tb(dh, bf), _ptr(dlast), *_tb(dgate, bf), *_tb(dx, bf), _ptr(dh0), _ptr(kept), _ptr(ws), need)
        return dgate, dx, dh0, None, None, None


def gated_scan(gate: torch.Tensor, x: torch.Tensor, h0: Optional[torch.Tensor] = None, *, resets: Optional[torch.Tensor] = None,
               lengths: Optional[torch.Tensor] = None, batch_first: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The memory over a sequence: (h, h_last), h of gate's shape and type, h_last (B, D) float32, the state behind the
    last step.  Differentiable (once) in gate, x and h0.

    gate, x: (T, B, D), or (B, T, D) with batch_first; float32 or bfloat16, both the same.  h0: (B, D) float32, the state in
    front of the first step (None: zeros).  resets: bool or uint8 of gate's first two axes; where set, the state counts as
    zero in front of that step, whatever it holds, and no gradient passes.  lengths: (B,) int32, clamped to 0..T: steps from
    there on are no part of the sequence; h and the gradients are zero there, and what gate and x hold does not matter.
    Sequences may be of length 0.  The backward pass works from float32 states: those in front of every eighth step are kept for it
    (T B D / 2 bytes; float32 with less than 480 KB a step takes them from h)."""
    shape, dev = gate.shape, gate.device
    T, B, D = shape if len(shape) == 3 and not batch_first else (shape[1], shape[0], shape[2]) if len(shape) == 3 else (0, 0, 0)
    if not (len(shape) == 3 and x.shape == shape and gate.dtype in _DTYPES and x.dtype == gate.dtype and dev.type == "cuda" and x.device == dev and
            (h0 is None or (h0.shape == (B, D) and h0.dtype == torch.float32 and h0.device == dev)) and
            (resets is None or (resets.shape == shape[:2] and resets.dtype in _FLAGS and resets.device == dev)) and
            (lengths is None or (lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.device == dev))):
        _explain_scan(gate, x, h0, resets, lengths, B, D)
    _no_tangents("gated_scan", gate, x, h0)
    gate, x = _dense(gate), _dense(x)
    h0 = None if h0 is None else h0.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    if torch.is_grad_enabled() and (gate.requires_grad or x.requires_grad or (h0 is not None and h0.requires_grad)):
        h, last = _GatedScan.apply(gate, x, h0, (resets, lengths), batch_first, (T, B, D))
        return _guard_leaves(h, h.device), last
    return _scan_forward(gate, x, h0, resets, lengths, batch_first, T, B, D)[:2]


def gated_scan_step(gate: torch.Tensor, x: torch.Tensor, state: torch.Tensor, *, reset: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step of the memory in a rollout, without gradients: state (B, D) float32, contiguous, is updated in place, the
    new state is returned in gate's type (in `out` if given; it may be gate or x itself, not the state, and may not overlap the
    state, reset or, shifted, gate or x: refused).  reset: (B,) bool or uint8; where set, the state counts as zero first."""
    shape, dt, dev = gate.shape, gate.dtype, gate.device
    D = shape[-1] if shape else 0
    if out is None and dev.type == "cuda":
        out = torch.empty(shape, dtype=dt, device=dev)
    if not (len(shape) == 2 and x.shape == shape and state.shape == shape and dt in _DTYPES and x.dtype == dt and state.dtype == torch.float32 and
            state.is_contiguous() and not ((state.requires_grad or (out is not None and out.requires_grad)) and torch.is_grad_enabled()) and
            (reset is None or (reset.shape == shape[:1] and reset.dtype in _FLAGS and reset.device == dev)) and dev.type == "cuda" and
            x.device == dev and state.device == dev and out.device == dev and out.shape == shape and out.dtype == dt and
            (D <= 1 or out.stride(1) == 1) and (shape[0] <= 1 or out.stride(0) >= D) and _apart(state, out)):
        _explain_step(gate, x, state, reset, out)
    gate, x = _dense(gate), _dense(x)
    _call("asm_gated_scan_step", dev, _DTYPES[dt], shape[0], D, gate.data_ptr(), gate.stride(0), x.data_ptr(), x.stride(0), state.data_ptr(),
          _ptr(reset), 0 if reset is None else reset.stride(0), out.data_ptr(), out.stride(0))
    torch.autograd.graph.increment_version((state, out))                # (written behind autograd's back)
    return out


def _apart(state, out) -> bool:
    """Whether a contiguous state and the rows of out lie in different memory (with the rows' gaps)."""
    s, o = state.data_ptr(), out.data_ptr()
    B, D = out.shape
    return o >= s + state.nbytes or o + ((B - 1) * out.stride(0) + D) * out.element_size() <= s or B * D == 0


def _explain_step(gate, x, state, reset, out):
    fn = "gated_scan_step"
    _need(gate.dim() == 2 and gate.shape == x.shape == state.shape, f"{fn}: gate, x and state must have one shape of two axes")
    _need(gate.dtype in _DTYPES and x.dtype == gate.dtype, f"{fn}: gate and x must both be float32 or bfloat16, got {gate.dtype} and {x.dtype}")
    _need(state.dtype == torch.float32 and state.is_contiguous(), f"{fn}: state must be a contiguous float32 tensor")
    _need(not (state.requires_grad and torch.is_grad_enabled()), f"{fn}: the state is updated in place and cannot require a gradient")
    B, D = gate.shape
    _need(reset is None or (reset.shape == (B,) and reset.dtype in _FLAGS), f"{fn}: reset must be a bool or uint8 tensor of shape {(B,)}")
    _need(out is None or (out.shape == gate.shape and out.dtype == gate.dtype and (D <= 1 or out.stride(1) == 1) and (B <= 1 or out.stride(0) >= D)
                          and not (out.requires_grad and torch.is_grad_enabled())),
          f"{fn}: out must be a tensor of gate's shape and type with contiguous rows that do not overlap")
    _on_device(fn, gate.device, x, state, reset, out)
    raise ValueError(f"{fn}: out and state must not share memory")


def _time_rows(t: torch.Tensor) -> torch.Tensor:
    """t with every time step contiguous (steps may lie any distance apart)."""
    return t if t.is_contiguous() or t[0].is_contiguous() else t.contiguous()


def advantages(rewards: torch.Tensor, values: torch.Tensor, *, dones: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
               gamma: float = 0.95, lam: float = 0.95, moments: bool = False):
    """Advantages and returns of an episode, without gradients: (adv, ret), or (adv, ret, moments).

        delta_t = r_t + gamma (1 - done_t) V_{t+1} - V_t,   adv_t = delta_t + gamma lam (1 - done_t) adv_{t+1},   ret_t = adv_t + V_t

    rewards: (T, E, ...) float32, T >= 1, for instance DeviceReplay.rew_ring[slot]; values: (T + 1, E, ...) float32, the last
    one behind the last step; dones: bool or uint8 of rewards' shape: where set, nothing behind that step counts, whatever it holds.
    lengths: (E,) int32, clamped to 0..T: environment e ends after lengths[e] steps, values[lengths[e]] behind its last one;
    beyond it both results are zero.  moments=True also returns the two numbers clipped_policy_loss normalises with:
    mean and 1 / (standard deviation + 1e-8) of the advantages of all steps (population deviation), as a float32 tensor."""
    shape, dev = rewards.shape, rewards.device
    if not (len(shape) >= 2 and shape.numel() > 0 and values.shape == (shape[0] + 1,) + shape[1:] and rewards.dtype == torch.float32 and
            values.dtype == torch.float32 and (dones is None or (dones.shape == shape and dones.dtype in _FLAGS and dones.device == dev)) and
            (lengths is None or (lengths.shape == shape[1:2] and lengths.dtype == torch.int32 and lengths.device == dev)) and
            0.0 <= gamma <= 1.0 and 0.0 <= lam <= 1.0 and dev.type == "cuda" and values.device == dev):
        _explain_advantages(rewards, values, dones, lengths, gamma, lam)
    T, E = shape[0], shape[1]
    D = shape.numel() // (T * E)
    rewards, values = _time_rows(rewards), _time_rows(values)
    dones = None if dones is None else _time_rows(dones)
    lengths = None if lengths is None else lengths.contiguous()
    adv = torch.empty(shape, dtype=torch.float32, device=dev)
    ret = torch.empty(shape, dtype=torch.float32, device=dev)
    mom = torch.empty(2, dtype=torch.float32, device=dev) if moments else None
    need = _lib.load().asm_advantages_workspace(T, E, D)
    ws = _workspace(need, dev)
    _call("asm_advantages_f32", dev, T, E, D, rewards.data_ptr(), rewards.stride(0), values.data_ptr(), values.stride(0), _ptr(dones),
          0 if dones is None else dones.stride(0), _ptr(lengths), gamma, lam, adv.data_ptr(), ret.data_ptr(), _ptr(mom), _ptr(ws), need)
    return (adv, ret, mom) if moments else (adv, ret)


def _explain_advantages(rewards, values, dones, lengths, gamma, lam):
    fn = "advantages"
    _need(rewards.dim() >= 2 and rewards.numel() > 0, f"{fn}: rewards must be a non-empty (T, E, ...) tensor")
    T, E = rewards.shape[0], rewards.shape[1]
    _need(tuple(values.shape) == (T + 1,) + tuple(rewards.shape[1:]), f"{fn}: values must have the shape {(T + 1,) + tuple(rewards.shape[1:])}")
    _need(rewards.dtype == torch.float32 and values.dtype == torch.float32, f"{fn}: rewards and values must be float32")
    _need(dones is None or (dones.shape == rewards.shape and dones.dtype in _FLAGS), f"{fn}: dones must be a bool or uint8 tensor of rewards' shape")
    _need(lengths is None or (lengths.shape == (E,) and lengths.dtype == torch.int32), f"{fn}: lengths must be an int32 tensor of shape {(E,)}")
    _need(0.0 <= gamma <= 1.0 and 0.0 <= lam <= 1.0, f"{fn}: gamma and lam must lie in [0, 1]")
    _on_device(fn, rewards.device, values, dones, lengths)
