"""The short causal convolution of a token's channels with those of the tokens just before it, the
usual companion of ``selective_scan``: over collected trajectories (``sequence``, with gradients) and
for one step of every environment (``step``). The reference has no counterpart.

    pre_t[c] = bias[c] + sum_{j < w} weight[c, j] x_{t-w+1+j}[c]        out = silu(pre), or pre

Taps that reach before the first token of t's episode (``reset``) are left out; those before a row's
first token come from ``state``, the w - 1 values before it. ``sequence`` over a trajectory and
``step`` token by token compute the same thing.

x is float32 or bfloat16 of any strides; a tensor whose last axis is not contiguous is copied. weight,
bias, states and sums are float32. Everything is asynchronous on the current stream, new tensors are
returned and inputs are not written, except where ``next_state`` names one.
"""

import ctypes

import torch

from . import _checks, _lib

MAX_TAPS = 4
MAX_CHANNELS = 65536
_STRIDES = {n: ctypes.c_int64 * n for n in (4, 6)}


def _check(x, weight, bias, state, reset, axes):
    """The checked inputs, the GPU's index, d, w."""
    device = _checks.first(x, "x", axes)
    shape = tuple(x.shape)
    d = shape[-1]
    if not 1 <= d <= MAX_CHANNELS:
        raise ValueError(f"there must be 1 to {MAX_CHANNELS} channels, got {d}")
    if _checks.tensor(weight, "weight").dim() != 2 or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError(f"weight must have shape ({d}, 1..{MAX_TAPS}), got {tuple(weight.shape)}")
    w = weight.shape[1]
    x = _checks.rows(x, "x", x.dtype, shape, device)
    weight = _checks.f32(weight, "weight", (d, w), device)
    bias = _checks.f32(bias, "bias", (d,), device)
    state = _checks.f32(state, "state", (shape[0], w - 1, d), device)
    reset = _checks.resets(reset, shape[:-1], device)
    return x, weight, bias, state, reset, device, d, w


def _strides(x, reset, dout=None):
    """The host array of strides: b, t of x, of reset (and of dout)."""
    flat = (*x.stride()[:2], *(reset.stride() if reset is not None else (0, 0)))
    if dout is not None:
        flat += dout.stride()[:2]
    return _STRIDES[len(flat)](*flat)


def _forward(x, weight, bias, state, reset, silu):
    b, t, d = x.shape
    w = weight.shape[1]
    ptr = _lib.ptr
    out = torch.empty((b, t, d), dtype=x.dtype, device=x.device)
    final = torch.empty((b, w - 1, d), dtype=torch.float32, device=x.device)
    with _lib.on(x.device):
        _lib.call("hipenvs_causal_conv", _checks.DTYPES[x.dtype], x.data_ptr(), weight.data_ptr(), ptr(bias),
                  ptr(state), ptr(reset), _strides(x, reset), silu, out.data_ptr(), final.data_ptr(), b, t, d, w,
                  _lib.stream_of(x.device))
    return out, final


def _backward(ctx, dout, dfinal):
    x, weight, bias, state, reset = ctx.saved_tensors
    dtype, (b, t, d, w), index, silu = ctx.ready
    if x.dtype is not dtype or x.shape != (b, t, d) or x.stride(2) != 1 or x.get_device() != index:
        x = _checks.saved(x, dtype, (b, t, d), index)
    weight = _checks.saved(weight, torch.float32, (d, w), index)
    bias = _checks.saved(bias, torch.float32, (d,), index)
    state = _checks.saved(state, torch.float32, (b, w - 1, d), index)
    if reset is not None:
        reset = _checks.resets(reset, (b, t), index)
    _checks.refuse_tangents("the gradient of sequence", dout, dfinal)
    device, ptr = x.device, _lib.ptr
    if dout is None:
        dout = torch.zeros((b, t, d), dtype=dtype, device=device)
    elif dout.dtype is not dtype or dout.shape != (b, t, d) or dout.stride(2) != 1 or dout.get_device() != index:
        dout = _checks.saved(dout, dtype, (b, t, d), index)
    dfinal = _checks.saved(dfinal, torch.float32, (b, w - 1, d), index)
    dx = torch.empty((b, t, d), dtype=dtype, device=device)
    dparams = torch.empty(d * (w + 1), dtype=torch.float32, device=device)
    dstate = torch.empty((b, w - 1, d), dtype=torch.float32, device=device)
    with _lib.on(device):
        nbytes = _lib.lib().hipenvs_causal_conv_workspace_bytes(b, t, d, w)
        if nbytes < 0:
            raise _lib.HipEnvsError(f"hipenvs_causal_conv: unsupported sequence ({b}, {t}, {d}, {w})")
        held = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _lib.call("hipenvs_causal_conv_backward", _checks.DTYPES[dtype], x.data_ptr(), weight.data_ptr(), ptr(bias),
                  ptr(state), ptr(reset), dout.data_ptr(), ptr(dfinal), _strides(x, reset, dout), silu, dx.data_ptr(),
                  dparams.data_ptr(), dstate.data_ptr(), b, t, d, w, ptr(held), nbytes, _lib.stream_of(device))
    dweight, dbias = torch.split(dparams, (d * w, d))
    return (dx, dweight.view(d, w), dbias if bias is not None else None, dstate if state is not None else None, None,
            None)


class _Sequence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, reset, silu):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, reset)
        ctx.ready = (x.dtype, (*x.shape, weight.shape[1]), x.get_device(), silu)
        return _forward(x, weight, bias, state, reset, silu)

    backward = _checks.once(_backward)


def sequence(x, weight, bias=None, state=None, reset=None, silu=True):
    """Whole trajectories: x (b, t, d), weight (d, w) float32 with w of 1 to 4, the last column that of
    the token itself, bias (d,) float32, state (b, w - 1, d) float32, the values before the first token
    in their order (None: zeros), reset (b, t) bool, True where an episode begins at that token (None:
    nowhere). Returns (out (b, t, d) of x's type, final_state (b, w - 1, d) float32, zeros where a tap
    would reach before the last episode's first token), differentiable once in x, weight, bias and
    state, in reverse mode."""
    x, weight, bias, state, reset, _, _, _ = _check(x, weight, bias, state, reset, 3)
    _checks.refuse_tangents("sequence", x, weight, bias, state)
    if _checks.wants_grad(x, weight, bias, state):
        return _Sequence.apply(x, weight, bias, state, reset, bool(silu))
    return _forward(x, weight, bias, state, reset, bool(silu))


def step(x, weight, bias=None, state=None, reset=None, silu=True, next_state=None):
    """One token of every environment: x (n, d), state (n, w - 1, d) float32 contiguous (None: zeros),
    reset (n,) bool, True where this token begins an episode. Returns (out (n, d) of x's type,
    next_state). ``next_state`` receives the new values and may be ``state`` itself. Not differentiable:
    training goes through ``sequence``."""
    x, weight, bias, state, reset, device, d, w = _check(x, weight, bias, state, reset, 2)
    if _checks.wants_grad(x, weight, bias, state):
        raise ValueError("step has no gradient: call it under torch.no_grad(), or use sequence")
    _checks.refuse_tangents("step", x, weight, bias, state, next_state)
    n, on, ptr = x.shape[0], x.device, _lib.ptr
    if state is None:
        state = torch.zeros((n, w - 1, d), dtype=torch.float32, device=on)
    if next_state is None:
        next_state = torch.empty_like(state)
    else:
        _checks.target(next_state, "next_state", (n, w - 1, d), device)
    out = torch.empty((n, d), dtype=x.dtype, device=on)
    with _lib.on(on):
        _lib.call("hipenvs_causal_conv_step", _checks.DTYPES[x.dtype], x.data_ptr(), x.stride(0), weight.data_ptr(),
                  ptr(bias), ptr(state), ptr(reset), reset.stride(0) if reset is not None else 0, bool(silu),
                  out.data_ptr(), next_state.data_ptr(), n, d, w, _lib.stream_of(on))
    return out, next_state
