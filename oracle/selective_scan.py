"""The selective state space scan and its gradients in float64, token by token, from the definition.

    delta = softplus(dt + dt_bias)   h_t[n] = exp(delta rate[n]) h_{t-1}[n] + delta x write[n]
    out = (sum_n read[n] h_t[n] + skip x) silu(gate)

x, dt, gate (b, t, d); rate (d, n); write, read (b, t, g, n); skip, dt_bias (d); state (b, d, n);
reset (b, t) bool: h_{t-1} is left out. skip, gate, dt_bias, state and reset may be None.
"""

import numpy as np


def sigmoid(x):
    return np.where(x >= 0, 1.0 / (1.0 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1.0 + np.exp(-np.abs(x))))


def softplus(x):
    return np.maximum(x, 0.0) + np.log1p(np.exp(-np.abs(x)))


def _spread(m, d):
    """(b, t, g, n) -> (b, t, d, n)."""
    return np.repeat(m, d // m.shape[2], axis=2)


def _given(x, dt, rate, write, read, skip, gate, dt_bias, state, reset):
    (b, t, d), n = x.shape, rate.shape[1]
    raw = dt + (0.0 if dt_bias is None else dt_bias)
    delta = softplus(raw)
    keep = np.exp(delta[..., None] * rate)
    begins = np.zeros((b, t), bool) if reset is None else reset
    return {"raw": raw, "delta": delta, "keep": keep, "begins": begins, "skip": np.zeros(d) if skip is None else skip,
            "state": np.zeros((b, d, n)) if state is None else state, "write": _spread(write, d), "read": _spread(read, d)}


def _walk(x, f):
    """States (b, t, d, n) after each token, and what of the state before reached each."""
    h, states, before = f["state"], [], []
    for t in range(x.shape[1]):
        prev = np.where(f["begins"][:, t, None, None], 0.0, f["keep"][:, t] * h)
        h = prev + (f["delta"][:, t] * x[:, t])[..., None] * f["write"][:, t]
        states.append(h)
        before.append(prev)
    shape = f["write"].shape
    return np.stack(states, 1) if states else np.zeros(shape), np.stack(before, 1) if states else np.zeros(shape)


def sequence(x, dt, rate, write, read, skip=None, gate=None, dt_bias=None, state=None, reset=None):
    """(out (b, t, d), final state (b, d, n))."""
    f = _given(x, dt, rate, write, read, skip, gate, dt_bias, state, reset)
    states, _ = _walk(x, f)
    y = (states * f["read"]).sum(-1) + f["skip"] * x
    if gate is not None:
        y = y * gate * sigmoid(gate)
    return y, states[:, -1] if x.shape[1] else f["state"]


def gradients(x, dt, rate, write, read, skip, gate, dt_bias, state, reset, dout, dfinal):
    """Gradients of x, dt, rate, write, read, skip, gate, dt_bias, state."""
    f = _given(x, dt, rate, write, read, skip, gate, dt_bias, state, reset)
    z = gate if gate is not None else None
    open_ = z * sigmoid(z) if z is not None else np.ones_like(x)
    slope = sigmoid(z) * (1.0 + z * (1.0 - sigmoid(z))) if z is not None else np.zeros_like(x)
    return _gradients(x, rate, f, sigmoid(f["raw"]), open_, slope, write.shape[2], dout, dfinal)


def _gradients(x, rate, f, one, open_, slope, g, dout, dfinal):
    (b, t, d), n = x.shape, rate.shape[1]
    states, before = _walk(x, f)
    y = (states * f["read"]).sum(-1) + f["skip"] * x
    dy = dout * open_
    G = dfinal.copy()
    dx, ddt = np.zeros_like(x), np.zeros_like(x)
    dwrite, dread, drate = np.zeros((b, t, d, n)), np.zeros((b, t, d, n)), np.zeros((d, n))
    for i in reversed(range(t)):
        G = G + f["read"][:, i] * dy[:, i, :, None]
        dread[:, i] = states[:, i] * dy[:, i, :, None]
        dwrite[:, i] = G * (f["delta"][:, i] * x[:, i])[..., None]
        into = (G * f["write"][:, i]).sum(-1)
        begins = f["begins"][:, i, None, None]   # the state before owes nothing, to an infinite G or delta neither
        through = np.where(begins, 0.0, G * before[:, i])
        drate += np.where(begins, 0.0, through * f["delta"][:, i, :, None]).sum(0)
        ddt[:, i] = ((through * rate).sum(-1) + into * x[:, i]) * one[:, i]
        dx[:, i] = f["skip"] * dy[:, i] + f["delta"][:, i] * into
        G = np.where(f["begins"][:, i, None, None], 0.0, G * f["keep"][:, i])
    dwrite, dread = (m.reshape(b, t, g, d // g, n).sum(3) for m in (dwrite, dread))
    return (dx, ddt, drate, dwrite, dread, (dy * x).sum((0, 1)), dout * y * slope, ddt.sum((0, 1)), G)


def magnitudes(x, dt, rate, write, read, skip, gate, dt_bias, state, reset, dout, dfinal):
    """The same sums over the magnitudes of their terms: out, final state, then the gradients."""
    f = _given(x, dt, rate, write, read, skip, gate, dt_bias, state, reset)
    f.update({k: np.abs(f[k]) for k in ("skip", "state", "write", "read")})
    a = np.abs(x)
    states, _ = _walk(a, f)
    open_, slope = np.ones_like(x), np.zeros_like(x)
    if gate is not None:
        one = sigmoid(gate)
        open_, slope = np.abs(gate) * one, one * (1.0 + np.abs(gate) * (1.0 - one))
    out = ((states * f["read"]).sum(-1) + f["skip"] * a) * open_
    return (out, states[:, -1] if x.shape[1] else f["state"],
            *_gradients(a, np.abs(rate), f, sigmoid(f["raw"]), open_, slope, write.shape[2], np.abs(dout), np.abs(dfinal)))
