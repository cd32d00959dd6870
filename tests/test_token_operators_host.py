"""The scan, the convolution, the lookup and the log probabilities without a GPU: what the C ABI and the
Python wrappers refuse before any launch, and the oracles' gradients against differences (CPU)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import categorical as oca
from oracle import causal_conv as occ
from oracle import selective_scan as oss

A, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4100)


def test_c_abi_checks_scan_arguments():
    from hipenvs import _lib

    l, st = _lib.lib(), (ctypes.c_int64 * 16)()

    def forward(dtype=0, x=A, rate=A, out=A, final=A, b=2, t=3, d=4, n=5, g=2, strides=st):
        return l.hipenvs_selective_scan(dtype, x, A, rate, A, A, None, None, None, None, None, strides, out, final, None, b,
                                        t, d, n, g, None, 0, None)

    for bad in (dict(dtype=2), dict(dtype=-1), dict(x=None), dict(rate=None), dict(out=None), dict(final=None),
                dict(strides=None), dict(b=-1), dict(t=-1), dict(d=0), dict(d=65537), dict(n=0), dict(n=65), dict(g=0),
                dict(g=3), dict(g=8), dict(b=1 << 31), dict(b=1 << 30, d=4), dict(t=1 << 31)):
        assert forward(**bad) == _lib.E_ARG, bad
    assert forward(b=0) == _lib.OK

    def backward(checks=A, dout=A, dx=A, gate=None, dgate=None, dparams=A, dstate=A, n=5):
        return l.hipenvs_selective_scan_backward(0, A, A, A, A, A, None, gate, None, None, dout, None, checks, st, dx, A, A, A,
                                                 dgate, dparams, dstate, 2, 3, 4, n, 2, None, 0, None)

    for bad in (dict(checks=None), dict(dout=None), dict(dx=None), dict(gate=A), dict(dparams=None), dict(dstate=None),
                dict(n=65)):
        assert backward(**bad) == _lib.E_ARG, bad

    def step(state=A, out=A, count=2, d=4, n=5, g=2):
        return l.hipenvs_selective_scan_step(0, A, A, A, A, A, None, None, None, state, None, st, out, A, count, d, n, g, None)

    for bad in (dict(state=None), dict(out=None), dict(count=-1), dict(n=65), dict(g=3), dict(count=1 << 30)):
        assert step(**bad) == _lib.E_ARG, bad
    assert step(count=0) == _lib.OK
    size = l.hipenvs_selective_scan_workspace_bytes
    assert size(1, 2, 33, 10, 6, 1) == 2 * 3 * 10 * 6 * 4
    assert size(3, 2, 33, 10, 6, 1) == -1 and size(0, 2, 33, 10, 65, 1) == -1 and size(0, 0, 33, 10, 6, 1) == 0


def test_c_abi_checks_conv_arguments():
    from hipenvs import _lib

    l, st = _lib.lib(), (ctypes.c_int64 * 6)()

    def forward(dtype=0, x=A, weight=A, out=A, final=A, b=2, t=3, d=4, w=4):
        return l.hipenvs_causal_conv(dtype, x, weight, None, None, None, st, 1, out, final, b, t, d, w, None)

    for bad in (dict(dtype=2), dict(x=None), dict(weight=None), dict(out=None), dict(final=None), dict(b=-1), dict(t=-1),
                dict(d=0), dict(d=65537), dict(w=0), dict(w=5), dict(b=1 << 30)):
        assert forward(**bad) == _lib.E_ARG, bad
    assert forward(b=0) == _lib.OK
    assert l.hipenvs_causal_conv_backward(0, A, A, None, None, None, None, None, st, 1, A, A, A, 2, 3, 4, 4, A, 1 << 30,
                                          None) == _lib.E_ARG
    assert l.hipenvs_causal_conv_backward(0, A, A, None, None, None, A, None, st, 1, A, None, A, 2, 3, 4, 4, A, 1 << 30,
                                          None) == _lib.E_ARG
    step = l.hipenvs_causal_conv_step
    assert step(0, A, 4, A, None, None, None, 0, 1, A, A, 2, 4, 4, None) == _lib.E_ARG
    assert step(0, A, 4, A, None, A, None, 0, 1, A, A, 2, 4, 5, None) == _lib.E_ARG
    assert step(0, A, 4, A, None, A, None, 0, 1, A, A, 0, 4, 4, None) == _lib.OK


def test_c_abi_checks_lookup_and_log_probs_arguments():
    from hipenvs import _lib

    l = _lib.lib()

    def lookup(dtype=0, tokens=A, size=8, table=A, out=A, count=3, v=4, d=5):
        return l.hipenvs_embedding(dtype, tokens, size, table, 5, 1.0, out, count, v, d, None)

    for bad in (dict(dtype=2), dict(tokens=None), dict(size=2), dict(table=None), dict(out=None), dict(count=-1),
                dict(count=1 << 31), dict(v=0), dict(v=1 << 31), dict(d=0), dict(d=65537)):
        assert lookup(**bad) == _lib.E_ARG, bad
    assert lookup(count=0) == _lib.OK
    need = l.hipenvs_embedding_workspace_bytes(1000, 50, 8)
    assert need > 0 and l.hipenvs_embedding_workspace_bytes(1000, 0, 8) == -1

    def lookup_back(dout=A, dtable=A, work=A, nbytes=need):
        return l.hipenvs_embedding_backward(0, A, 8, dout, 8, 1.0, dtable, 1000, 50, 8, work, nbytes, None)

    for bad in (dict(dout=None), dict(dtable=None), dict(work=None), dict(work=ODD), dict(nbytes=need - 1)):
        assert lookup_back(**bad) == _lib.E_ARG, bad

    def log_probs(dtype=0, logits=A, tokens=A, entropy=A, top=0, best=A, index=A, rows=3, v=9):
        return l.hipenvs_log_probs(dtype, logits, v, tokens, A, entropy, None, top, best, index, rows, v, None, 0, None)

    for bad in (dict(dtype=2), dict(logits=None), dict(tokens=None), dict(entropy=None), dict(top=-1), dict(top=65),
                dict(top=10), dict(top=3, best=None), dict(top=3, index=None), dict(rows=-1), dict(v=0), dict(v=1 << 31)):
        assert log_probs(**bad) == _lib.E_ARG, bad
    assert log_probs(rows=0) == _lib.OK
    back = l.hipenvs_log_probs_backward
    assert back(0, A, 9, A, None, A, A, A, A, 3, 9, None) == _lib.E_ARG
    assert back(0, A, 9, A, A, A, A, A, None, 3, 9, None) == _lib.E_ARG
    assert back(0, A, 9, A, A, A, A, A, A, 0, 9, None) == _lib.OK
    assert l.hipenvs_log_probs_workspace_bytes(3, 9, 10) == -1


def test_wrappers_want_a_gpu():
    from hipenvs import categorical, causal_conv, embedding, selective_scan

    x, mix, rate = torch.zeros(2, 3, 4), torch.zeros(2, 3, 5), torch.zeros(4, 5)
    for call in (lambda: selective_scan.sequence(x, x, rate, mix, mix),
                 lambda: selective_scan.step(x[:, 0], x[:, 0], rate, mix[:, 0], mix[:, 0]),
                 lambda: causal_conv.sequence(x, rate[:, :3]), lambda: causal_conv.step(x[:, 0], rate[:, :3]),
                 lambda: embedding.lookup(torch.zeros(3, dtype=torch.int64), rate),
                 lambda: categorical.log_probs(rate, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: selective_scan.sequence(x.numpy(), x, rate, mix, mix), lambda: causal_conv.sequence(x.half(), rate),
                 lambda: embedding.lookup(x, "table"), lambda: categorical.log_probs(rate.double(), x)):
        with pytest.raises(TypeError):
            call()


def differences(value, inputs, grads, rng):
    """Directional differences of `value` in each input against the gradients."""
    for i, g in enumerate(grads):
        if g is None:
            continue
        for _ in range(4):
            u = rng.standard_normal(inputs[i].shape)
            up, down = (value(*[x + s * 1e-5 * u if j == i else x for j, x in enumerate(inputs)]) for s in (1, -1))
            assert abs((up - down) / 2e-5 - (g * u).sum()) < 1e-7 * (1 + abs((g * u).sum())), i


def test_scan_oracle_gradients_are_differences():
    rng = np.random.default_rng(0)
    b, t, d, n, g = 2, 7, 6, 3, 2
    x, dt, gate = (rng.standard_normal((b, t, d)) for _ in range(3))
    rate, skip, bias = -np.exp(rng.standard_normal((d, n))), rng.standard_normal(d), rng.standard_normal(d)
    write, read = (rng.standard_normal((b, t, g, n)) for _ in range(2))
    state, reset = rng.standard_normal((b, d, n)), rng.random((b, t)) < 0.3
    inputs = [x, dt, rate, write, read, skip, gate, bias, state]
    out, final = oss.sequence(*inputs, reset)
    dout, dfinal = rng.standard_normal(out.shape), rng.standard_normal(final.shape)

    def value(*a):
        o, f = oss.sequence(*a, reset)
        return (o * dout).sum() + (f * dfinal).sum()

    differences(value, inputs, oss.gradients(*inputs, reset, dout, dfinal), rng)
    got = oss.magnitudes(*inputs, reset, dout, dfinal)
    assert all((m >= np.abs(w) - 1e-12).all() for m, w in zip(got, (out, final, *oss.gradients(*inputs, reset, dout, dfinal))))


def test_conv_oracle_gradients_are_differences():
    rng = np.random.default_rng(1)
    for b, t, d, w, silu in ((2, 9, 3, 4, True), (1, 2, 2, 3, False), (2, 3, 2, 1, True), (1, 0, 2, 3, True)):
        x, weight, bias = rng.standard_normal((b, t, d)), rng.standard_normal((d, w)), rng.standard_normal(d)
        state, reset = rng.standard_normal((b, w - 1, d)), rng.random((b, t)) < 0.3
        inputs = [x, weight, bias, state]
        out, final = occ.sequence(*inputs, reset, silu)
        dout, dfinal = rng.standard_normal(out.shape), rng.standard_normal(final.shape)

        def value(*a):
            o, f = occ.sequence(*a, reset, silu)
            return (o * dout).sum() + (f * dfinal).sum()

        differences(value, inputs, occ.gradients(*inputs, reset, silu, dout, dfinal), rng)


def test_log_probs_oracle_gradients_are_differences():
    rng = np.random.default_rng(2)
    x, tokens = rng.standard_normal((5, 7)), np.array([0, 6, -1, 3, 2])
    x[3, [0, 5]] = -np.inf
    a, b = rng.standard_normal(5), rng.standard_normal(5)

    def value(y):
        lp, h = oca.log_probs(y, tokens)
        return (lp * a).sum() + (h * b).sum()

    differences(value, [x], [oca.gradient(x, tokens, a, b)], rng)
    x[1] = -np.inf
    assert (oca.gradient(x, tokens, a, b)[1] == 0).all() and oca.log_probs(x, tokens)[1][1] == 0
