"""Decay attention and AdamW without a GPU: what the C ABI and the Python wrappers refuse before
any launch, and the oracles' own identities (CPU)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw as oad
from oracle import decay_attention as oda


def test_c_abi_checks_attention_arguments():
    from hipenvs import _lib

    l, a = _lib.lib(), ctypes.c_void_p(4096)
    strides = (ctypes.c_int64 * 14)()

    def forward(dtype=0, q=a, out=a, final=a, b=2, t=3, h=2, dk=8, dv=4):
        return l.hipenvs_decay_attention(dtype, q, a, a, strides, a, None, None, 1.0, out, final, b, t, h, dk, dv, None, 0, None)

    for bad in (dict(dtype=2), dict(dtype=-1), dict(q=None), dict(out=None), dict(final=None), dict(b=-1), dict(t=-1),
                dict(h=0), dict(dk=0), dict(dk=129), dict(dv=129), dict(dv=0), dict(b=1 << 31), dict(b=1 << 30, h=4),
                dict(t=1 << 31)):
        assert forward(**bad) == _lib.E_ARG, bad
    assert forward(b=0) == _lib.OK
    assert l.hipenvs_decay_attention_backward(0, a, a, a, None, strides, a, None, None, None, None, 1.0, a, a, a, a, 2, 3, 2, 8,
                                              4, None, 0, None) == _lib.E_ARG
    assert l.hipenvs_decay_attention_backward(0, a, a, a, a, strides, a, None, None, None, None, 1.0, a, a, a, None, 2, 3, 2, 8,
                                              4, None, 0, None) == _lib.E_ARG
    step = l.hipenvs_decay_attention_step
    assert step(0, a, 1, 1, a, 1, 1, a, 1, 1, a, None, None, 0, 1.0, a, a, 4, 2, 8, 4, None) == _lib.E_ARG
    assert step(0, a, 1, 1, a, 1, 1, a, 1, 1, a, a, None, 0, 1.0, a, a, 4, 2, 200, 4, None) == _lib.E_ARG
    assert step(0, a, 1, 1, a, 1, 1, a, 1, 1, a, a, None, 0, 1.0, a, a, 1 << 30, 4, 8, 4, None) == _lib.E_ARG
    assert step(0, a, 1, 1, a, 1, 1, a, 1, 1, a, a, None, 0, 1.0, a, a, 0, 2, 8, 4, None) == _lib.OK


def test_c_abi_checks_adamw_arguments():
    from hipenvs import _lib

    l, a = _lib.lib(), ctypes.c_void_p(4096)
    one_p, one_i = (ctypes.c_void_p * 1)(4096), (ctypes.c_int64 * 1)(10)
    kind, num = (ctypes.c_int32 * 1)(0), (ctypes.c_double * 1)(1.0)

    def step(bits=32, count=1, params=one_p, sizes=one_i, types=kind, m=a, scales=None):
        return l.hipenvs_adamw_step(bits, count, params, one_p, sizes, types, num, num, 0.9, 0.9, 0.0, 1.0, m, a, scales,
                                    scales, None)

    for bad in (dict(bits=16), dict(count=-1), dict(params=None), dict(sizes=None), dict(m=None), dict(bits=8),
                dict(types=(ctypes.c_int32 * 1)(4)), dict(sizes=(ctypes.c_int64 * 1)(-1)),
                dict(params=(ctypes.c_void_p * 1)(None)), dict(m=ctypes.c_void_p(4098))):
        assert step(**bad) == _lib.E_ARG, bad
    assert step(count=0) == _lib.OK
    assert step(sizes=(ctypes.c_int64 * 1)(0)) == _lib.OK
    assert l.hipenvs_adamw_decode(a, a, a, a, -1, a, a, None) == _lib.E_ARG
    assert l.hipenvs_adamw_decode(a, a, a, None, 1, a, a, None) == _lib.E_ARG
    assert l.hipenvs_adamw_decode(a, a, a, a, 1, ctypes.c_void_p(4100), a, None) == _lib.E_ARG
    assert l.hipenvs_adamw_decode(a, a, a, a, 0, a, a, None) == _lib.OK


def test_wrappers_want_a_gpu():
    from hipenvs import adamw, decay_attention

    q = torch.zeros(2, 3, 1, 4)
    with pytest.raises(ValueError):
        decay_attention.sequence(q, q, q, torch.zeros(1))
    with pytest.raises(ValueError):
        decay_attention.step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(1), torch.zeros(2, 1, 4, 4))
    with pytest.raises(TypeError):
        decay_attention.sequence(np.zeros((2, 3, 1, 4)), q, q, torch.zeros(1))
    p = [torch.zeros(4)]
    with pytest.raises(ValueError):
        adamw.step(p, p, adamw.init(p), 1)
    with pytest.raises(ValueError):
        adamw.init([])


def test_moments_are_laid_out_in_blocks():
    from hipenvs import adamw

    m = adamw.init([torch.zeros(1), torch.zeros(256), torch.zeros(0), torch.zeros(257)], 8)
    assert [x.shape[0] for x in m] == [1024, 1024, 4, 4]
    assert [x.dtype for x in m] == [torch.int8, torch.uint8, torch.float32, torch.float32]


def test_oracle_gradients_are_the_sequence_s_differences():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((2, 9, 2, d)) for d in (3, 3, 4))
    state, ld = rng.standard_normal((2, 2, 3, 4)), np.array([-0.1, -1.0])
    reset = rng.random((2, 9)) < 0.3
    out, final = oda.sequence(q, k, v, ld, state, reset, 0.5)
    dout, dfinal = rng.standard_normal(out.shape), rng.standard_normal(final.shape)
    grads = oda.gradients(q, k, v, ld, state, reset, 0.5, dout, dfinal)

    def value(*x):
        o, f = oda.sequence(x[0], x[1], x[2], ld, x[3], reset, 0.5)
        return (o * dout).sum() + (f * dfinal).sum()

    xs = [q, k, v, state]
    for i, g in enumerate(grads):
        for _ in range(5):
            u = rng.standard_normal(xs[i].shape)
            up, down = ([x + s * 1e-5 * u if j == i else x for j, x in enumerate(xs)] for s in (1, -1))
            assert abs((value(*up) - value(*down)) / 2e-5 - (g * u).sum()) < 1e-7


def test_oracle_codes_read_back_as_their_nearest():
    x = np.linspace(-3, 3, 256, dtype=np.float32)[None]
    code, scale = oad.encode_m(x)
    assert code.min() == -127 and code.max() == 127 and scale[0] == 3
    assert np.array_equal(oad.encode_m(oad.decode_m(code, scale))[0], code)
    v = (x * x).astype(np.float32)
    code, scale = oad.encode_v(v)
    assert np.array_equal(oad.encode_v(oad.decode_v(code, scale))[0], code) and (code > 0).all()
    tiny = np.zeros((1, 256), np.float32)
    tiny[0, 0], tiny[0, 1] = 1.0, 1e-30
    assert oad.encode_v(tiny)[0][0, :3].tolist() == [255, 1, 0]
