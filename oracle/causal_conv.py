"""The short causal convolution and its gradients in float64, token by token, from the definition.

x (b, t, d), weight (d, w), bias (d) or None, state (b, w - 1, d) or None (zeros), reset (b, t) bool or
None. pre_t = bias + sum_j weight[:, j] x_{t-w+1+j} within t's episode; out = silu(pre) or pre.
"""

import numpy as np

from .selective_scan import sigmoid


def _windows(x, w, state, reset):
    """(b, t, w, d): the values that each token's taps meet; and the values left after the row."""
    (b, t, d) = x.shape
    held = np.zeros((b, w - 1, d)) if state is None else state
    out = np.zeros((b, t, w, d))
    for i in range(t):
        if reset is not None:
            held = np.where(reset[:, i, None, None], 0.0, held)
        out[:, i] = np.concatenate([held, x[:, i:i + 1]], 1)
        held = out[:, i, 1:]
    return out, held


def sequence(x, weight, bias=None, state=None, reset=None, silu=True):
    windows, final = _windows(x, weight.shape[1], state, reset)
    pre = (windows * weight.T).sum(2) + (0.0 if bias is None else bias)
    return pre * sigmoid(pre) if silu else pre, final


def gradients(x, weight, bias, state, reset, silu, dout, dfinal):
    """Gradients of x, weight, bias, state."""
    windows, _ = _windows(x, weight.shape[1], state, reset)
    pre = (windows * weight.T).sum(2) + (0.0 if bias is None else bias)
    one = sigmoid(pre)
    dpre = dout * (one * (1.0 + pre * (1.0 - one)) if silu else 1.0)
    return back(weight, reset, windows, dpre, dfinal)


def back(weight, reset, windows, dpre, dfinal):
    b, t, w, d = windows.shape
    carry, dx = dfinal, np.zeros((b, t, d))
    for i in reversed(range(t)):
        into = weight.T * dpre[:, i, None, :]
        into[:, 1:] += carry
        dx[:, i] = into[:, -1]
        carry = into[:, :-1] if reset is None else np.where(reset[:, i, None, None], 0.0, into[:, :-1])
    return dx, (windows * dpre[:, :, None, :]).sum((0, 1)).T, dpre.sum((0, 1)), carry


def magnitudes(x, weight, bias, state, reset, dout, dfinal):
    """|pre|'s terms summed, and the gradients' sums over the magnitudes of their terms, with silu's
    slope (at most 1.1) taken as 1.1 and dpre's error per unit of |dout|."""
    held = None if state is None else np.abs(state)
    windows, _ = _windows(np.abs(x), weight.shape[1], held, reset)
    pre = (windows * np.abs(weight).T).sum(2) + (0.0 if bias is None else np.abs(bias))
    grads = back(np.abs(weight), reset, windows, 1.1 * np.abs(dout) * (1.0 + pre), np.abs(dfinal))
    return pre, grads
