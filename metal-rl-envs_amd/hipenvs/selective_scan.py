"""The selective state space scan, a memory whose decay and input each token chooses: over collected
trajectories (``sequence``, with gradients) and for one step of every environment (``step``). Stands
beside ``decay_attention``, whose decays are constants. The reference has no counterpart; its policies
see the current observation only.

Each channel of a row keeps n states in float32:

    delta = softplus(dt_t + dt_bias)
    h_t[n] = exp(delta rate[n]) h_{t-1}[n] + delta x_t write_t[n]
    out_t  = (sum_n read_t[n] h_t[n] + skip x_t) silu(gate_t)

and h_{t-1} is left out where ``reset`` marks token t as the first of an episode (the ``done`` of
the environment step before it). ``rate`` is below zero for a state that decays. Channels share
``write`` and ``read``: all of them, or each of g equal groups of neighbouring channels its own.
Without ``skip``, ``gate`` or ``dt_bias`` that term is left out. ``sequence`` over a trajectory and
``step`` token by token compute the same thing.

x, dt, write, read and gate are float32 or bfloat16 of one type, of any strides (parts of one
projection, rows collected time-major and transposed); a tensor whose last axis is not contiguous
is copied. rate, skip, dt_bias, states and sums are float32. Everything is asynchronous on the current
stream, new tensors are returned and inputs are not written, except where ``next_state`` names one.
"""

import ctypes

import torch

from . import _checks, _lib

MAX_STATES = 64
MAX_CHANNELS = 65536
_STRIDES = {n: ctypes.c_int64 * n for n in (8, 14, 16)}


def _check(x, dt, rate, write, read, skip, gate, dt_bias, reset, axes):
    """The checked inputs, write and read with an axis of groups; the GPU's index, d, n, g."""
    device = _checks.first(x, "x", axes)
    dtype, shape, lead = x.dtype, tuple(x.shape), tuple(x.shape[:-1])
    d = shape[-1]
    if not 1 <= d <= MAX_CHANNELS:
        raise ValueError(f"there must be 1 to {MAX_CHANNELS} channels, got {d}")
    if _checks.tensor(rate, "rate").dim() != 2 or not 1 <= rate.shape[1] <= MAX_STATES:
        raise ValueError(f"rate must have shape ({d}, 1..{MAX_STATES}), got {tuple(rate.shape)}")
    n = rate.shape[1]
    if _checks.tensor(write, "write").dim() == axes:
        write = write.unsqueeze(-2)
    if _checks.tensor(read, "read").dim() == axes:
        read = read.unsqueeze(-2)
    g = write.shape[-2] if write.dim() == axes + 1 else 0
    if g < 1 or d % g:
        raise ValueError(f"write must have shape {(*lead, 'groups', n)} or {(*lead, n)}, the groups a divisor of {d}; "
                         f"got {tuple(write.shape)}")
    x = _checks.rows(x, "x", dtype, shape, device)
    dt = _checks.rows(dt, "dt", dtype, shape, device)
    write = _checks.rows(write, "write", dtype, (*lead, g, n), device)
    read = _checks.rows(read, "read", dtype, (*lead, g, n), device)
    if gate is not None:
        gate = _checks.rows(gate, "gate", dtype, shape, device)
    rate = _checks.f32(rate, "rate", (d, n), device)
    skip = _checks.f32(skip, "skip", (d,), device)
    dt_bias = _checks.f32(dt_bias, "dt_bias", (d,), device)
    reset = _checks.resets(reset, lead, device)
    return x, dt, rate, write, read, skip, gate, dt_bias, reset, device, d, n, g


def _strides(x, dt, write, read, gate, reset, dout=None):
    """The host array of strides: b, t of x, dt, gate, then b, t, g of write, read, then b, t of reset
    (and of dout)."""
    flat = (*x.stride()[:2], *dt.stride()[:2], *(gate.stride()[:2] if gate is not None else (0, 0)),
            *write.stride()[:3], *read.stride()[:3], *(reset.stride() if reset is not None else (0, 0)))
    if dout is not None:
        flat += dout.stride()[:2]
    return _STRIDES[len(flat)](*flat)


def _near(x):
    """x, copied where its tokens lie further apart than the kernels' offsets reach. A clone: a row of one
    token is contiguous whatever its stride, and contiguous() would leave that as it is."""
    if x is None or -0x80000000 < x.stride(1) < 0x80000000:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _laid(x, dtype, shape, device):
    """A tensor of the backward pass whose tokens the kernels reach: any strides, a contiguous last axis."""
    if x is None or (x.dtype is dtype and x.shape == shape and x.stride(-1) == 1 and x.get_device() == device
                     and -0x80000000 < x.stride(1) < 0x80000000):
        return x
    return _near(_checks.saved(x, dtype, shape, device).contiguous())


def _workspace(which, b, t, d, n, g, device):
    """(address, bytes, tensor): the workspace of a pass (0 forward, 2 backward), or the states that the
    backward pass starts from (1)."""
    nbytes = _lib.lib().hipenvs_selective_scan_workspace_bytes(which, b, t, d, n, g)
    if nbytes < 0:
        raise _lib.HipEnvsError(f"hipenvs_selective_scan: unsupported sequence ({b}, {t}, {d}, {n}, {g})")
    held = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    return _lib.ptr(held), nbytes, held


def _forward(x, dt, rate, write, read, skip, gate, dt_bias, state, reset, train):
    b, t, d = x.shape
    g, n = write.shape[2:]
    ptr = _lib.ptr
    x, dt, write, read, gate, reset = (_near(y) for y in (x, dt, write, read, gate, reset))
    out = torch.empty((b, t, d), dtype=x.dtype, device=x.device)
    final = torch.empty((b, d, n), dtype=torch.float32, device=x.device)
    with _lib.on(x.device):
        at, nbytes, held = _workspace(0, b, t, d, n, g, x.device)
        checks = _workspace(1, b, t, d, n, g, x.device)[2] if train else None
        _lib.call("hipenvs_selective_scan", _checks.DTYPES[x.dtype], x.data_ptr(), dt.data_ptr(), rate.data_ptr(),
                  write.data_ptr(), read.data_ptr(), ptr(skip), ptr(gate), ptr(dt_bias), ptr(state), ptr(reset),
                  _strides(x, dt, write, read, gate, reset), out.data_ptr(), final.data_ptr(), ptr(checks), b, t, d, n,
                  g, at, nbytes, _lib.stream_of(x.device))
    return out, final, checks


def _backward(ctx, dout, dfinal):
    x, dt, rate, write, read, skip, gate, dt_bias, reset, checks = ctx.saved_tensors
    dtype, (b, t, d, n, g), index, nchecks, has_state = ctx.ready
    shape, mixed = (b, t, d), (b, t, g, n)
    x, dt, gate = _laid(x, dtype, shape, index), _laid(dt, dtype, shape, index), _laid(gate, dtype, shape, index)
    write, read = _laid(write, dtype, mixed, index), _laid(read, dtype, mixed, index)
    rate = _checks.saved(rate, torch.float32, (d, n), index)
    skip, dt_bias = _checks.saved(skip, torch.float32, (d,), index), _checks.saved(dt_bias, torch.float32, (d,), index)
    if reset is not None:
        reset = _near(_checks.resets(reset, (b, t), index))
    checks = _checks.saved(checks, torch.uint8, (nchecks,), index)
    _checks.refuse_tangents("the gradient of sequence", dout, dfinal)
    device, ptr = x.device, _lib.ptr
    dout = torch.zeros(shape, dtype=dtype, device=device) if dout is None else _laid(dout, dtype, shape, index)
    dfinal = _checks.saved(dfinal, torch.float32, (b, d, n), index)
    dx, ddt = (torch.empty((b, t, d), dtype=dtype, device=device) for _ in range(2))
    dgate = torch.empty((b, t, d), dtype=dtype, device=device) if gate is not None else None
    dwrite, dread = (torch.empty((b, t, g, n), dtype=dtype, device=device) for _ in range(2))
    dparams = torch.empty(d * (n + 2), dtype=torch.float32, device=device)
    dstate = torch.empty((b, d, n), dtype=torch.float32, device=device)
    with _lib.on(device):
        at, nbytes, held = _workspace(2, b, t, d, n, g, device)
        _lib.call("hipenvs_selective_scan_backward", _checks.DTYPES[dtype], x.data_ptr(), dt.data_ptr(),
                  rate.data_ptr(), write.data_ptr(), read.data_ptr(), ptr(skip), ptr(gate), ptr(dt_bias), ptr(reset),
                  dout.data_ptr(), ptr(dfinal), ptr(checks), _strides(x, dt, write, read, gate, reset, dout),
                  dx.data_ptr(), ddt.data_ptr(), dwrite.data_ptr(), dread.data_ptr(), ptr(dgate), dparams.data_ptr(),
                  dstate.data_ptr(), b, t, d, n, g, at, nbytes, _lib.stream_of(device))
    drate, dskip, dbias = torch.split(dparams, (d * n, d, d))
    return (dx, ddt, drate.view(d, n), dwrite, dread, dskip if skip is not None else None, dgate,
            dbias if dt_bias is not None else None, dstate if has_state else None, None)


class _Sequence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, rate, write, read, skip, gate, dt_bias, state, reset):
        ctx.set_materialize_grads(False)
        out, final, checks = _forward(x, dt, rate, write, read, skip, gate, dt_bias, state, reset, True)
        ctx.save_for_backward(x, dt, rate, write, read, skip, gate, dt_bias, reset, checks)
        ctx.ready = (x.dtype, (*x.shape, *rate.shape[1:], write.shape[2]), x.get_device(),
                     checks.numel() if checks is not None else 0, state is not None)
        return out, final

    backward = _checks.once(_backward)


def sequence(x, dt, rate, write, read, skip=None, gate=None, dt_bias=None, state=None, reset=None):
    """Whole trajectories: x, dt, gate (b, t, d), rate (d, n) float32, write, read (b, t, n) or
    (b, t, g, n), skip, dt_bias (d,) float32, state (b, d, n) float32 before the first token (None:
    zeros), reset (b, t) bool, True where an episode begins at that token (None: nowhere). Returns
    (out (b, t, d) of x's type, final_state (b, d, n) float32), differentiable once in every input but
    reset, in reverse mode."""
    x, dt, rate, write, read, skip, gate, dt_bias, reset, device, d, n, _ = _check(
        x, dt, rate, write, read, skip, gate, dt_bias, reset, 3)
    state = _checks.f32(state, "state", (x.shape[0], d, n), device)
    given = (x, dt, rate, write, read, skip, gate, dt_bias, state)
    _checks.refuse_tangents("sequence", *given)
    if _checks.wants_grad(*given):
        return _Sequence.apply(*given, reset)
    return _forward(*given, reset, False)[:2]


def step(x, dt, rate, write, read, skip=None, gate=None, dt_bias=None, state=None, reset=None, next_state=None):
    """One token of every environment: x, dt, gate (n_envs, d), write, read (n_envs, n) or
    (n_envs, g, n), state (n_envs, d, n) float32 contiguous (None: zeros), reset (n_envs,) bool, True
    where this token begins an episode. Returns (out (n_envs, d) of x's type, next_state).
    ``next_state`` receives the new states and may be ``state`` itself. Not differentiable: training
    goes through ``sequence``."""
    x, dt, rate, write, read, skip, gate, dt_bias, reset, device, d, n, g = _check(
        x, dt, rate, write, read, skip, gate, dt_bias, reset, 2)
    count, on, ptr = x.shape[0], x.device, _lib.ptr
    if state is None:
        state = torch.zeros((count, d, n), dtype=torch.float32, device=on)
    state = _checks.f32(state, "state", (count, d, n), device)
    given = (x, dt, rate, write, read, skip, gate, dt_bias, state)
    if _checks.wants_grad(*given):
        raise ValueError("step has no gradient: call it under torch.no_grad(), or use sequence")
    _checks.refuse_tangents("step", *given, next_state)
    if next_state is None:
        next_state = torch.empty_like(state)
    else:
        _checks.target(next_state, "next_state", (count, d, n), device)
    out = torch.empty((count, d), dtype=x.dtype, device=on)
    strides = _STRIDES[8](x.stride(0), dt.stride(0), gate.stride(0) if gate is not None else 0, *write.stride()[:2],
                          *read.stride()[:2], reset.stride(0) if reset is not None else 0)
    with _lib.on(on):
        _lib.call("hipenvs_selective_scan_step", _checks.DTYPES[x.dtype], x.data_ptr(), dt.data_ptr(), rate.data_ptr(),
                  write.data_ptr(), read.data_ptr(), ptr(skip), ptr(gate), ptr(dt_bias), ptr(state), ptr(reset),
                  strides, out.data_ptr(), next_state.data_ptr(), count, d, n, g, _lib.stream_of(on))
    return out, next_state
