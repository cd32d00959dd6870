"""The differentiable decay attention's host side without a GPU (CPU): the native calls are replaced by
the oracle on the memory that the arguments name, every access checked against the tensors that
are there."""

import contextlib
import gc

import numpy as np
import pytest
import torch

from oracle import decay_attention as oda


def memory_at(ptr, shape, strides, dtype):
    """The values at an address, in a tensor that is alive and holds all of them."""
    last = sum((n - 1) * s for n, s in zip(shape, strides))
    size = torch.empty(0, dtype=dtype).element_size()
    for x in gc.get_objects():
        if type(x) is torch.Tensor and x.dtype == dtype and x.numel():
            store = x.untyped_storage()
            at = ptr - store.data_ptr()
            if 0 <= at and at + (last + 1) * size <= store.nbytes():
                return x.detach().as_strided(shape, strides, at // size)
    raise AssertionError(f"no tensor holds {shape} of strides {strides} at its address")


class Native:
    """hipenvs' entry points of a sequence, on CPU memory."""

    def __init__(self):
        self.strides = None

    def __call__(self, name, dtype, q, k, v, *args):
        backward = name == "hipenvs_decay_attention_backward"
        assert backward or name == "hipenvs_decay_attention"
        if backward:
            dout, strides, log_decay, state, reset, dfinal, states, scale, *outs = args[:12]
            b, t, h, dk, dv, work, nbytes = args[12:19]
        else:
            strides, log_decay, state, reset, scale, *outs = args[:7]
            b, t, h, dk, dv, work, nbytes = args[7:14]
        self.strides = st = list(strides)
        assert dtype == 0 and nbytes == 64   # as if in parts
        memory_at(work, (64,), (1,), torch.uint8)

        def rows(ptr, i, d):
            return memory_at(ptr, (b, t, h, d), (*st[3 * i:3 * i + 3], 1), torch.float32).numpy()

        def whole(ptr):
            return None if ptr is None else memory_at(ptr, (b, h, dk, dv), (h * dk * dv, dk * dv, dv, 1), torch.float32).numpy()

        args = [rows(q, 0, dk), rows(k, 1, dk), rows(v, 2, dv), memory_at(log_decay, (h,), (1,), torch.float32).numpy(),
                whole(state), None if reset is None else memory_at(reset, (b, t), st[-2:], torch.bool).numpy(), scale]
        if backward:
            assert memory_at(states, (64,), (1,), torch.uint8).tolist() == list(range(64))
            got = oda.gradients(*args, rows(dout, 3, dv), whole(dfinal))
            shapes = [(b, t, h, dk), (b, t, h, dk), (b, t, h, dv), (b, h, dk, dv)]
        else:
            memory_at(work, (64,), (1,), torch.uint8).copy_(torch.arange(64))
            got = oda.sequence(*args)
            shapes = [(b, t, h, dv), (b, h, dk, dv)]
        for ptr, shape, x in zip(outs, shapes, got):
            memory_at(ptr, shape, torch.empty(shape, device="meta").stride(), torch.float32).copy_(torch.from_numpy(x))


@pytest.fixture
def native(monkeypatch):
    from hipenvs import _lib, decay_attention

    made = Native()
    monkeypatch.setattr(_lib, "call", made)
    monkeypatch.setattr(_lib, "on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)

    def workspace(*args):
        held = torch.empty(64, dtype=torch.uint8)
        return held.data_ptr(), 64, held

    monkeypatch.setattr(decay_attention, "_workspace", workspace)
    return made


B, T, H, DK, DV = 2, 6, 3, 5, 4


def inputs(layout):
    gen = torch.Generator().manual_seed(1)
    rows = torch.randn(*((T, B) if layout == "time" else (B, T)), H * (2 * DK + DV), generator=gen)
    if layout == "time":
        rows = rows.transpose(0, 1)
    q, k, v = (x.unflatten(-1, (H, -1)) for x in torch.split(rows, (H * DK, H * DK, H * DV), -1))
    state = torch.randn(B, H, DK, DV, generator=gen)
    reset = torch.rand(T, B, generator=gen).t() < 0.3
    leaves = [x.detach().requires_grad_() for x in (q, k, v, state)]
    return leaves, torch.tensor([-0.1, -0.5, 0.0]), reset, torch.randn(B, T, H, DV, generator=gen)


def gradients(layout, hooks=contextlib.nullcontext()):
    from hipenvs import decay_attention

    leaves, log_decay, reset, dout = inputs(layout)
    with hooks:
        out, final = decay_attention._Sequence.apply(*leaves[:3], log_decay, leaves[3], reset, 0.5)
    return torch.autograd.grad((out, final), leaves, (dout, torch.ones_like(final)))


def on_another_layout(x):
    """The same values, every axis' stride another one."""
    return x.permute(*reversed(range(x.dim()))).contiguous().permute(*reversed(range(x.dim())))


def on_every_other(x):
    if x.dim() == 1 and x.dtype == torch.uint8:
        return x.clone()   # the library's own workspace
    wide = torch.empty(*x.shape[:-1], 2 * x.shape[-1], dtype=x.dtype)
    wide[..., ::2] = x
    return wide[..., ::2]


@pytest.mark.parametrize("layout", ["fused", "time"])
@pytest.mark.parametrize("change", [torch.clone, on_another_layout, on_every_other, lambda x: x.clone().contiguous()])
def test_saved_tensors_that_hooks_hand_back_in_another_layout(native, layout, change):
    """Cloned, transposed, spread: the strides that go with an address are those of what lies there."""
    want = gradients(layout)
    got = gradients(layout, torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: change(x.detach())))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    packed = gradients(layout, torch.autograd.graph.saved_tensors_hooks(lambda x: change(x.detach()), lambda x: x))
    assert all(torch.equal(x, y) for x, y in zip(packed, want))


@pytest.mark.parametrize("change, error", [
    (lambda x: x.double() if x.is_floating_point() else x, TypeError),
    (lambda x: x[:1] if x.dim() == 4 else x, ValueError),
    (lambda x: x.int() if x.dtype == torch.bool else x, TypeError),
    (lambda x: x[:, :-1] if x.dtype == torch.bool else x, ValueError),
    (lambda x: x[:-1] if x.dtype == torch.uint8 else x, ValueError),
    (lambda x: x.float() if x.dtype == torch.uint8 else x, TypeError),
])
def test_saved_tensors_that_hooks_hand_back_as_others_are_refused(native, change, error):
    """Another type, shape or device: no native call sees them."""
    with pytest.raises(error):
        gradients("fused", torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: change(x.detach())))


def test_c_abi_refuses_states_that_floats_do_not_lie_in():
    import ctypes

    from hipenvs import _lib

    a, strides = ctypes.c_void_p(4096), (ctypes.c_int64 * 14)()
    assert _lib.lib().hipenvs_decay_attention_backward(0, a, a, a, a, strides, a, None, None, None, ctypes.c_void_p(4098), 1.0,
                                                       a, a, a, a, 2, 3, 2, 8, 4, None, 0, None) == _lib.E_ARG


def test_tangents_are_found():
    from torch.autograd import forward_ad

    from hipenvs import decay_attention

    x = torch.ones(3)
    decay_attention._refuse_tangents("it", x, None)
    with forward_ad.dual_level():
        decay_attention._refuse_tangents("it", x, None)
        dual = forward_ad.make_dual(x, x)
        with pytest.raises(ValueError, match="it has no forward-mode derivative"):
            decay_attention._refuse_tangents("it", x, None, dual[1:])
