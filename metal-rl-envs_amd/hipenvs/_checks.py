"""Checks of arguments shared by the operators of policies over tokens. `device` is the index of
the GPU that the call's first tensor is on, `first` that tensor's name."""

import torch
from torch.autograd import forward_ad

DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def tensor(x, name):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(x).__name__}")
    return x


def first(x, name, axes):
    """The call's first tensor: float32 or bfloat16, on a GPU, `axes` axes (None: one at least); its GPU."""
    if tensor(x, name).dtype not in DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on a ROCm GPU, got device {x.device}")
    if x.dim() != axes if axes is not None else x.dim() < 1:
        raise ValueError(f"{name} must have {axes or 'one or more'} axes, got shape {tuple(x.shape)}")
    return x.get_device()


def rows(x, name, dtype, shape, device, first="x"):
    """A tensor of that type, shape and GPU; copied where its last axis is not contiguous."""
    if (isinstance(x, torch.Tensor) and x.dtype is dtype and x.shape == shape and x.get_device() == device
            and x.stride(-1) == 1):
        return x
    if tensor(x, name).dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.get_device() != device:
        raise ValueError(f"{name} is on {x.device}, {first} is on GPU {device}")
    return x if x.stride(-1) == 1 or shape[-1] == 1 else x.contiguous()


def f32(x, name, shape, device, first="x"):
    """A float32 tensor of that shape and GPU; copied where it is not contiguous. None stays None."""
    if x is None or (isinstance(x, torch.Tensor) and x.dtype is torch.float32 and x.shape == shape
                     and x.get_device() == device and x.is_contiguous()):
        return x
    return rows(x, name, torch.float32, shape, device, first).contiguous()


def saved(x, dtype, shape, device):
    """A tensor that autograd hands back, or a gradient: contiguous, of the type, shape and GPU that the
    call works with. Hooks on saved tensors may hand back others of the same values, laid out in their own
    way; anything else is refused. In the engine's thread each call costs several times what it does in the
    caller's, so there is one for the ordinary case. None stays None."""
    if x is None or (x.dtype is dtype and x.shape == shape and x.is_contiguous() and x.get_device() == device):
        return x
    return rows(x, "a tensor of the backward pass", dtype, shape, device, "the forward pass").contiguous()


def resets(reset, shape, device, first="x"):
    if reset is None:
        return None
    if tensor(reset, "reset").dtype is not torch.bool:
        raise TypeError(f"reset must be bool, got {reset.dtype}")
    if reset.shape != shape:
        raise ValueError(f"reset must have shape {tuple(shape)}, got {tuple(reset.shape)}")
    if reset.get_device() != device:
        raise ValueError(f"reset is on {reset.device}, {first} is on GPU {device}")
    return reset


def refuse_tangents(name, *tensors):
    """Forward-mode derivatives are not there, and outputs without one would read as a derivative of
    zero. Outside every dual level, which torch counts from 0, there is nothing to look for."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    if any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise ValueError(f"{name} has no forward-mode derivative: pass it tensors without tangents")


def wants_grad(*tensors):
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors)


def target(x, name, shape, device, first="x"):
    """A contiguous float32 tensor that a call writes, marked as changed."""
    if f32(x, name, shape, device, first) is not x:
        raise ValueError(f"{name} must be contiguous")
    torch.autograd.graph.increment_version(x)
    return x


def once(backward):
    """A backward whose gradients have no graph, and say so when one is asked for and used."""
    marked = torch.autograd.function.once_differentiable(backward)

    def either(ctx, *grads):
        return (marked if torch.is_grad_enabled() else backward)(ctx, *grads)

    return staticmethod(either)
