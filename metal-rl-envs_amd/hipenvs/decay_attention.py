"""Linear attention with a decay for each head, for policies with a memory: over collected
trajectories (``sequence``, with gradients) and for one step of every environment (``step``).
The reference has no counterpart; its policies see the current observation only.

A head of a row keeps a state S (dk, dv) in float32, with lambda = exp(log_decay[h]):

    S_t = lambda S_{t-1} + k_t v_t^T          o_t = scale * S_t^T q_t

and lambda S_{t-1} is left out where ``reset`` marks token t as the first of an episode (the
``done`` of the environment step before it). ``scale`` defaults to 1 / sqrt(dk). Acting costs
the same at every step, whatever the episode's length: the state is the whole memory.
``sequence`` over a trajectory and ``step`` token by token compute the same thing.

q, k, v are float32 or bfloat16 of one type, of any strides (views of one projection, rows
collected time-major and transposed); a tensor whose last axis is not contiguous is copied.
States, sums and log_decay are float32. Everything is asynchronous on the current stream, new
tensors are returned and inputs are not written, except where ``next_state`` names one.
"""

import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib

MAX_DIM = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _tensor(x, name):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(x).__name__}")
    return x


def _check(x, name, dtype, device, shape):
    """A tensor of that type, shape and device (a GPU's index), its last axis contiguous."""
    if _tensor(x, name).dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
    if x.get_device() != device:
        raise ValueError(f"{name} is on {x.device}, q is on GPU {device}")
    return x if x.stride(-1) == 1 or shape[-1] == 1 else x.contiguous()


def _check_qkv(q, k, v, axes):
    """(q, k, v, the GPU's index, lead, h, dk, dv) of tensors (*lead, h, d) with `axes` axes in all."""
    dtype = _tensor(q, "q").dtype
    if dtype not in _DTYPES:
        raise TypeError(f"q must be float32 or bfloat16, got {dtype}")
    device = q.get_device()
    if not q.is_cuda:
        raise ValueError(f"q must be on a ROCm GPU, got device {q.device}")
    shape = tuple(q.shape)
    if len(shape) != axes:
        raise ValueError(f"q must have {axes} axes, got shape {shape}")
    if _tensor(v, "v").dim() != axes:
        raise ValueError(f"v must have {axes} axes, got shape {tuple(v.shape)}")
    lead, h, dk, dv = shape[:-2], shape[-2], shape[-1], v.shape[-1]
    if not (1 <= dk <= MAX_DIM and 1 <= dv <= MAX_DIM):
        raise ValueError(f"dk and dv must be in 1..{MAX_DIM}, got {dk} and {dv}")
    if not 1 <= h <= 65536:
        raise ValueError(f"there must be 1 to 65536 heads, got {h}")
    if q.stride(-1) != 1 and dk != 1:
        q = q.contiguous()
    k = _check(k, "k", dtype, device, shape)
    v = _check(v, "v", dtype, device, (*lead, h, dv))
    return q, k, v, device, lead, h, dk, dv


def _check_f32(x, name, shape, device):
    if _tensor(x, name).dtype is not torch.float32:
        raise TypeError(f"{name} must be float32, got {x.dtype}")
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(x.shape)}")
    if x.get_device() != device:
        raise ValueError(f"{name} is on {x.device}, q is on GPU {device}")
    return x.contiguous()


def _check_decay(log_decay, h, device):
    log_decay = _check_f32(log_decay, "log_decay", (h,), device)
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant of each head and has no gradient: pass it detached")
    return log_decay


def _check_reset(reset, shape, device):
    if reset is None:
        return None
    if _tensor(reset, "reset").dtype is not torch.bool:
        raise TypeError(f"reset must be bool, got {reset.dtype}")
    if reset.shape != shape:
        raise ValueError(f"reset must have shape {shape}, got {tuple(reset.shape)}")
    if reset.get_device() != device:
        raise ValueError(f"reset is on {reset.device}, q is on GPU {device}")
    return reset


def _refuse_tangents(name, *tensors):
    """Forward-mode derivatives are not there, and outputs without one would read as a derivative of
    zero. Outside every dual level, which torch counts from 0, there is nothing to look for."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    if any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise ValueError(f"{name} has no forward-mode derivative: pass it tensors without tangents")


_STRIDES = {n: ctypes.c_int64 * n for n in (11, 14)}


def _strides(rows, reset):
    """The host array of strides: b, t, h of each tensor, then b, t of reset."""
    flat = [s for x in rows for s in x.stride()[:3]]
    flat += reset.stride() if reset is not None else (0, 0)
    return _STRIDES[len(flat)](*flat)


def _scale(scale, dk):
    return 1.0 / math.sqrt(dk) if scale is None else float(scale)


def _workspace(dtype, b, t, h, dk, dv, device):
    """(address, bytes, tensor) of the workspace of a sequence's calls."""
    nbytes = _lib.lib().hipenvs_decay_attention_workspace_bytes(dtype, b, t, h, dk, dv)
    if nbytes < 0:
        raise _lib.HipEnvsError(f"hipenvs_decay_attention: unsupported sequence ({b}, {t}, {h}, {dk}, {dv})")
    held = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    return _lib.ptr(held), nbytes, held


def _forward(q, k, v, log_decay, state, reset, scale):
    """(out, final_state, workspace): the workspace holds the states between a long row's parts."""
    b, t, h, dk = q.shape
    dv = v.shape[-1]
    out = torch.empty((b, t, h, dv), dtype=q.dtype, device=q.device)
    final = torch.empty((b, h, dk, dv), dtype=torch.float32, device=q.device)
    with _lib.on(q.device):
        at, nbytes, workspace = _workspace(_DTYPES[q.dtype], b, t, h, dk, dv, q.device)
        _lib.call("hipenvs_decay_attention", _DTYPES[q.dtype], _lib.ptr(q), _lib.ptr(k), _lib.ptr(v),
                  _strides((q, k, v), reset), _lib.ptr(log_decay), _lib.ptr(state), _lib.ptr(reset), scale,
                  _lib.ptr(out), _lib.ptr(final), b, t, h, dk, dv, at, nbytes, _lib.stream_of(q.device))
    return out, final, workspace


class _Sequence(torch.autograd.Function):
    # The backward runs in the engine's own thread, where Python costs several times what it does here:
    # what it can be given ready, the forward makes. Not the layout of what is saved: hooks on saved
    # tensors may hand back others of the same values (a copy on the host and back packs a view).
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, reset, scale):
        ctx.set_materialize_grads(False)
        out, final, workspace = _forward(q, k, v, log_decay, state, reset, scale)
        ctx.save_for_backward(q, k, v, log_decay, state, reset, workspace)
        b, t, h, dk = q.shape
        ctx.ready = (_DTYPES[q.dtype], q.dtype, q.device, q.get_device(), b, t, h, dk, v.shape[-1], scale,
                     workspace.numel() if workspace is not None else 0)
        return out, final

    @staticmethod
    def backward(ctx, dout, dfinal):
        if torch.is_grad_enabled():
            return _backward_once(ctx, dout, dfinal)
        return _backward(ctx, dout, dfinal)


def _backward(ctx, dout, dfinal):
    q, k, v, log_decay, state, reset, states = ctx.saved_tensors
    code, dtype, device, index, b, t, h, dk, dv, scale, nbytes = ctx.ready
    q = _check(q, "the saved q", dtype, index, (b, t, h, dk))
    k = _check(k, "the saved k", dtype, index, (b, t, h, dk))
    v = _check(v, "the saved v", dtype, index, (b, t, h, dv))
    log_decay = _check_f32(log_decay, "the saved log_decay", (h,), index)
    reset = _check_reset(reset, (b, t), index)
    if state is not None:
        state = _check_f32(state, "the saved state", (b, h, dk, dv), index)
    if states is not None:
        states = _check(states, "the saved workspace", torch.uint8, index, (nbytes,))
    _refuse_tangents("the gradient of sequence", dout, dfinal)
    if dout is None:
        dout = torch.zeros((b, t, h, dv), dtype=dtype, device=device)
    elif dout.stride(-1) != 1 and dv != 1:
        dout = dout.contiguous()
    if dfinal is not None:
        dfinal = dfinal.contiguous()
    dq = torch.empty((b, t, h, dk), dtype=dtype, device=device)
    dk_ = torch.empty((b, t, h, dk), dtype=dtype, device=device)
    dv_ = torch.empty((b, t, h, dv), dtype=dtype, device=device)
    dstate = torch.empty((b, h, dk, dv), dtype=torch.float32, device=device)
    held = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    with _lib.on(device):
        _lib.call("hipenvs_decay_attention_backward", code, q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(),
                  _strides((q, k, v, dout), reset), log_decay.data_ptr(), _lib.ptr(state),
                  _lib.ptr(reset), _lib.ptr(dfinal), _lib.ptr(states), scale, dq.data_ptr(), dk_.data_ptr(),
                  dv_.data_ptr(), dstate.data_ptr(), b, t, h, dk, dv, _lib.ptr(held), nbytes, _lib.stream_of(device))
    return dq, dk_, dv_, None, dstate if state is not None else None, None, None


# where a graph of the gradient is asked for: the gradients are without one, and say so when used
_backward_once = torch.autograd.function.once_differentiable(_backward)


def sequence(q, k, v, log_decay, state=None, reset=None, scale=None):
    """Whole trajectories: q, k (b, t, h, dk), v (b, t, h, dv), log_decay (h,) float32, state
    (b, h, dk, dv) float32 before the first token (None: zeros), reset (b, t) bool, True where
    an episode begins at that token (None: nowhere). Returns (out (b, t, h, dv) of q's type,
    final_state (b, h, dk, dv) float32), differentiable once in q, k, v and state, in reverse mode."""
    q, k, v, device, (b, t), h, dk, dv = _check_qkv(q, k, v, 4)
    log_decay = _check_decay(log_decay, h, device)
    reset = _check_reset(reset, (b, t), device)
    if state is not None:
        state = _check_f32(state, "state", (b, h, dk, dv), device)
    _refuse_tangents("sequence", q, k, v, log_decay, state)
    scale = _scale(scale, dk)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (state is not None and state.requires_grad)):
        return _Sequence.apply(q, k, v, log_decay, state, reset, scale)
    return _forward(q, k, v, log_decay, state, reset, scale)[:2]


def step(q, k, v, log_decay, state, reset=None, scale=None, next_state=None):
    """One token of every environment: q, k (n, h, dk), v (n, h, dv), state (n, h, dk, dv) float32
    contiguous, reset (n,) bool, True where this token begins an episode. Returns
    (out (n, h, dv) of q's type, next_state). ``next_state`` receives the new states and may be
    ``state`` itself. Not differentiable: training goes through ``sequence``."""
    q, k, v, device, (n,), h, dk, dv = _check_qkv(q, k, v, 3)
    log_decay = _check_decay(log_decay, h, device)
    reset = _check_reset(reset, (n,), device)
    state = _check_f32(state, "state", (n, h, dk, dv), device)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise ValueError("step has no gradient: call it under torch.no_grad(), or use sequence")
    if next_state is not None and _check_f32(next_state, "next_state", (n, h, dk, dv), device) is not next_state:
        raise ValueError("next_state must be contiguous")
    _refuse_tangents("step", q, k, v, log_decay, state, next_state)
    if next_state is None:
        next_state = torch.empty_like(state)
    else:
        torch.autograd.graph.increment_version(next_state)
    on = q.device
    out = torch.empty((n, h, dv), dtype=q.dtype, device=on)
    with _lib.on(on):
        _lib.call("hipenvs_decay_attention_step", _DTYPES[q.dtype], q.data_ptr(), q.stride(0), q.stride(1),
                  k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                  log_decay.data_ptr(), state.data_ptr(), _lib.ptr(reset), reset.stride(0) if reset is not None else 0,
                  _scale(scale, dk), out.data_ptr(), next_state.data_ptr(), n, h, dk, dv, _lib.stream_of(on))
    return out, next_state
