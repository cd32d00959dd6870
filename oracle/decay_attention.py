"""Decay attention from its definition, token by token in float64 (see
``hipenvs.decay_attention``): outputs, states and gradients, and for error bounds the same sums
over the terms' magnitudes."""

import numpy as np


def _keep(log_decay, reset, t):
    """(b, h, 1, 1): what is left of the state before token t; None where nothing resets."""
    lam = np.exp(np.asarray(log_decay, np.float64))[None, :, None, None]
    return lam if reset is None else np.where(reset[:, t, None, None, None], 0.0, lam)


def _decayed(S, log_decay, reset, t):
    out = S * _keep(log_decay, None, t)
    if reset is not None:   # left out, not multiplied by zero: what it holds does not matter
        out[reset[:, t]] = 0.0
    return out


def sequence(q, k, v, log_decay, state, reset, scale):
    """(out (b, t, h, dv), final state) in float64; state None: zeros."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    b, t_max, h, dk = q.shape
    S = np.zeros((b, h, dk, v.shape[-1])) if state is None else np.array(state, np.float64)
    out = np.empty((b, t_max, h, v.shape[-1]))
    for t in range(t_max):
        S = _decayed(S, log_decay, reset, t) + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * np.einsum("bhkv,bhk->bhv", S, q[:, t])
    return out, S


def gradients(q, k, v, log_decay, state, reset, scale, dout, dfinal):
    """(dq, dk, dv, dstate) in float64; state and dfinal None: zeros."""
    q, k, v, dout = (np.asarray(x, np.float64) for x in (q, k, v, dout))
    b, t_max, h, dk = q.shape
    dv = v.shape[-1]
    S = np.zeros((b, h, dk, dv)) if state is None else np.array(state, np.float64)
    G = np.zeros((b, h, dk, dv)) if dfinal is None else np.array(dfinal, np.float64)
    d_q, d_k, d_v = np.empty_like(q), np.empty_like(k), np.empty_like(v)
    for t in range(t_max):
        S = _decayed(S, log_decay, reset, t) + k[:, t, :, :, None] * v[:, t, :, None, :]
        d_q[:, t] = scale * np.einsum("bhkv,bhv->bhk", S, dout[:, t])
    for t in reversed(range(t_max)):
        G = G + scale * q[:, t, :, :, None] * dout[:, t, :, None, :]
        d_k[:, t] = np.einsum("bhkv,bhv->bhk", G, v[:, t])
        d_v[:, t] = np.einsum("bhkv,bhk->bhv", G, k[:, t])
        G = _decayed(G, log_decay, reset, t)
    return d_q, d_k, d_v, G


def magnitudes(q, k, v, log_decay, state, reset, scale, dout=None, dfinal=None):
    """The same sums over the magnitudes of their terms: what rounding errors scale with."""
    a = [None if x is None else np.abs(np.asarray(x, np.float64)) for x in (q, k, v, state, dout, dfinal)]
    q, k, v, state, dout, dfinal = a
    both = sequence(q, k, v, log_decay, state, reset, abs(scale))
    if dout is None:
        return both
    return (*both, *gradients(q, k, v, log_decay, state, reset, abs(scale), dout, dfinal))
