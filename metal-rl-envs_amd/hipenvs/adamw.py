"""AdamW over all tensors of a policy, one launch for every 64 of them, moments in 32 bits or in
8 bits with a scale for every 256 values. The reference has no counterpart: its gradient learners call
their array library's optimizer.

    m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

``step`` is the operator: parameters, gradients and flat moments, updated in place.
``AdamW`` keeps the moments and counts each tensor's steps around it. Parameters and gradients
are float32 or bfloat16 in any mix; the arithmetic is float32, each operation rounded on its
own, and no sum's order varies, so a step gives the same bits every time.

The moments of all tensors lie one after another, each tensor beginning at a multiple of 256
values: ``(m, v)`` float32, or in 8 bits ``(m_codes int8, v_codes uint8, m_scales, v_scales)``
where a code c stands for scale * t|t|, t = c / 127 (m), or scale * t^4, t = c / 255 (v).
Asynchronous on the current stream.
"""

import math
import operator
from array import array

import torch

from . import _lib

BLOCK = 256
_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_OF_GRAD = {torch.float32: 0, torch.bfloat16: 2}
_dtype, _shape, _add = operator.attrgetter("dtype"), operator.attrgetter("shape"), operator.add
_device, _contiguous = torch.Tensor.get_device, torch.Tensor.is_contiguous
_address, _numel = torch.Tensor.data_ptr, torch.Tensor.numel


def _is_tensor(x):
    return x is not None


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def init(params, bits=32):
    """Zero moments for `params`: (m, v), or (m_codes, v_codes, m_scales, v_scales) for bits=8."""
    if bits not in (32, 8):
        raise ValueError(f"bits must be 32 or 8, got {bits}")
    params = list(params)
    if not params:
        raise ValueError("no parameters")
    device, n = params[0].device, sum(_padded(p.numel()) for p in params)
    if bits == 32:
        return tuple(torch.zeros(n, dtype=torch.float32, device=device) for _ in range(2))
    scales = tuple(torch.zeros(n // BLOCK, dtype=torch.float32, device=device) for _ in range(2))
    return (torch.zeros(n, dtype=torch.int8, device=device), torch.zeros(n, dtype=torch.uint8, device=device), *scales)


def _check_moments(moments, n, device):
    """The bits of `moments`, whose tensors must hold n values."""
    if len(moments) == 2:
        wanted = ((torch.float32, n),) * 2
    elif len(moments) == 4:
        wanted = ((torch.int8, n), (torch.uint8, n), (torch.float32, n // BLOCK), (torch.float32, n // BLOCK))
    else:
        raise ValueError(f"moments must be (m, v) or (m_codes, v_codes, m_scales, v_scales), got {len(moments)} tensors")
    for x, (dtype, size) in zip(moments, wanted):
        if not isinstance(x, torch.Tensor) or x.dtype != dtype:
            raise TypeError(f"moments must be tensors of {', '.join(str(d) for d, _ in wanted)}")
        if x.shape != (size,) or not x.is_contiguous() or x.device != device:
            raise ValueError(f"moments must be contiguous, of shapes {[s for _, s in wanted]}, on {device}")
    return 32 if len(moments) == 2 else 8


def _corrections(t, lr, beta1, beta2):
    """(lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t))."""
    return lr / (1.0 - beta1 ** t), 1.0 / math.sqrt(1.0 - beta2 ** t)


def _refused_param(params, device):
    for i, p in enumerate(params):
        if p.dtype not in _TYPES:
            return TypeError(f"params[{i}] must be float32 or bfloat16, got {p.dtype}")
        if p.device != device:
            return ValueError(f"params[{i}] is on {p.device}, params[0] is on {device}")
        if not p.is_contiguous():
            return ValueError(f"params[{i}] must be contiguous")


def _refused_grad(params, grads, device):
    for i, (p, g) in enumerate(zip(params, grads)):
        if g is None:
            continue
        if g.dtype not in _OF_GRAD:
            return TypeError(f"grads[{i}] must be float32 or bfloat16, got {g.dtype}")
        if g.device != device:
            return ValueError(f"grads[{i}] is on {g.device}, params[0] is on {device}")
        if g.shape != p.shape:
            return ValueError(f"grads[{i}] must have shape {tuple(p.shape)}, got {tuple(g.shape)}")


def step(params, grads, moments, t, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01):
    """One step in place: params and moments change, grads do not. `grads` holds a tensor for each
    parameter, or None where it has none (that parameter and its moments stay). `t` is the
    step's number, from 1, for all of them or a sequence with one for each."""
    params, grads = list(params), list(grads)
    count = len(params)
    if len(grads) != count:
        raise ValueError(f"{count} parameters and {len(grads)} gradients")
    if count == 0:
        return
    beta1, beta2 = float(betas[0]), float(betas[1])
    lr, eps, weight_decay = float(lr), float(eps), float(weight_decay)
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"betas must be in [0, 1), got {betas}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    device = params[0].device
    if device.type != "cuda":
        raise ValueError(f"params must be on a ROCm GPU, got device {device}")
    # one pass of a C function over the list for each property: a loop over the tensors in Python
    # costs twice as much, and more than the launch at a few dozen tensors
    index = params[0].get_device()
    types = list(map(_TYPES.get, map(_dtype, params)))
    if None in types or set(map(_device, params)) != {index} or not all(map(_contiguous, params)):
        raise _refused_param(params, device)
    given = grads if all(map(_is_tensor, grads)) else [g for g in grads if g is not None]
    of_grads = list(map(_OF_GRAD.get, map(_dtype, given)))
    whole = len(given) == count
    if (None in of_grads or (given and set(map(_device, given)) != {index})
            or list(map(_shape, given)) != list(map(_shape, params if whole else
                                                    [p for p, g in zip(params, grads) if g is not None]))):
        raise _refused_grad(params, grads, device)
    if not all(map(_contiguous, given)):   # the copies live until the launch: their memory may go to the next tensor then
        given = [g.contiguous() for g in given]
    grad_ptrs = list(map(_address, given))
    if not whole:
        ptr_of, kind_of = iter(grad_ptrs), iter(of_grads)
        grad_ptrs = [0 if g is None else next(ptr_of) for g in grads]
        of_grads = [0 if g is None else next(kind_of) for g in grads]
    types = list(map(_add, types, of_grads))
    ptrs, sizes = list(map(_address, params)), list(map(_numel, params))
    flat = sum(-(-n // BLOCK) for n in sizes) * BLOCK
    if len(set(ptrs)) != count and len({a for a, n in zip(ptrs, sizes) if n}) != sum(n > 0 for n in sizes):
        raise ValueError("a parameter is listed twice")
    bits = _check_moments(moments, flat, device)
    if isinstance(t, int):
        if t < 1:
            raise ValueError(f"t must be a step number from 1, got {t}")
        rate, root = _corrections(t, lr, beta1, beta2)
        rates, roots = array("d", [rate]) * count, array("d", [root]) * count
    else:
        steps = [int(x) for x in t]
        if len(steps) != count or min(steps) < 1:
            raise ValueError("t must be a step number from 1, or one for each parameter")
        of_step = {n: _corrections(n, lr, beta1, beta2) for n in set(steps)}
        rates = array("d", [of_step[n][0] for n in steps])
        roots = array("d", [of_step[n][1] for n in steps])
    m, v, *scales = (x.data_ptr() for x in moments)
    m_scales, v_scales = scales if scales else (None, None)
    arrays = (array("Q", ptrs), array("Q", grad_ptrs), array("q", sizes), array("i", types), rates, roots)
    with _lib.on(device):
        _lib.call("hipenvs_adamw_step", bits, count, *(a.buffer_info()[0] for a in arrays), beta1, beta2, eps,
                  1.0 - lr * weight_decay, m, v, m_scales, v_scales, _lib.stream_of(device))
    changed = params if whole else [p for p, g in zip(params, grads) if g is not None]
    if changed:   # the others are as they were: a graph that holds them stays good
        torch.autograd.graph.increment_version((*changed, *moments))


def decode(moments):
    """(m, v) float32 of any moments: themselves in 32 bits, what the codes stand for in 8."""
    if len(moments) == 2:
        return tuple(moments)
    m_codes, v_codes, m_scales, v_scales = moments
    n, device = m_codes.numel(), m_codes.device
    _check_moments(moments, n, device)
    if device.type != "cuda":
        raise ValueError(f"moments must be on a ROCm GPU, got device {device}")
    if n % BLOCK:
        raise ValueError(f"moments must hold whole blocks of {BLOCK} values, got {n}")
    m, v = (torch.empty(n, dtype=torch.float32, device=device) for _ in range(2))
    with _lib.on(device):
        _lib.call("hipenvs_adamw_decode", _lib.ptr(m_codes), _lib.ptr(v_codes), _lib.ptr(m_scales),
                  _lib.ptr(v_scales), n // BLOCK, _lib.ptr(m), _lib.ptr(v), _lib.stream_of(device))
    return m, v


class AdamW:
    """The optimizer of a set of tensors: their moments and each one's step count. ``step()`` takes
    the tensors' ``.grad``, or the gradients it is given."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, bits=32):
        self.params = list(params)
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.moments = init(self.params, bits)
        self.steps = [0] * len(self.params)

    def step(self, grads=None):
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(self.params)} parameters and {len(grads)} gradients")
        if torch.cuda.is_current_stream_capturing():
            raise _lib.HipEnvsError("AdamW.step counts on the host: a captured step would repeat one step's "
                                    "bias corrections at every replay")
        steps = [n + (g is not None) for n, g in zip(self.steps, grads)]
        with torch.no_grad():
            step(self.params, grads, self.moments, [max(n, 1) for n in steps], self.lr, self.betas, self.eps,
                 self.weight_decay)
        self.steps = steps

    def zero_grad(self):
        for p in self.params:
            p.grad = None
