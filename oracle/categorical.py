"""Log probabilities, entropies, the most likely tokens and the gradient of the logits in float64."""

import numpy as np


def log_softmax(x):
    """(rows, v); -inf is a token that is not allowed, a row of nothing else is -inf throughout."""
    m = x.max(1, keepdims=True)
    m = np.where(np.isneginf(m), 0.0, m)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        return (x - m) - np.log(np.exp(x - m).sum(1, keepdims=True)) if x.size else x


def log_probs(x, tokens):
    """(log_prob, entropy) of rows of finite or -inf logits."""
    with np.errstate(invalid="ignore"):
        empty = np.isneginf(x).all(1)
        lp = np.where(empty[:, None], -np.inf, log_softmax(x))
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0).sum(1)
    chosen = lp[np.arange(len(tokens)), np.maximum(tokens, 0)]
    return np.where(tokens < 0, 0.0, chosen), entropy


def gradient(x, tokens, dlog_prob, dentropy):
    with np.errstate(invalid="ignore"):
        empty = np.isneginf(x).all(1)
        lp = np.where(empty[:, None], -np.inf, log_softmax(x))
    p = np.exp(lp)
    _, entropy = log_probs(x, tokens)
    dlp = np.where((tokens < 0) | empty, 0.0, dlog_prob)
    finite = np.where(p > 0, lp, 0.0)
    dx = -p * (dlp[:, None] + dentropy[:, None] * (finite + entropy[:, None]))
    there = np.flatnonzero(tokens >= 0)
    dx[there, tokens[there]] += dlp[there]
    return dx


def top(x, k):
    """(values' places, in order): the largest first, of equals the lowest place."""
    return np.argsort(-x, axis=1, kind="stable")[:, :k]
