"""AdamW from its formula in float64, and the 8-bit moments' codes in numpy float32, operation by
operation as ``hipenvs.adamw`` rounds them."""

import numpy as np

BLOCK = 256
F = np.float32


def step64(p, g, m, v, t, lr, betas, eps, weight_decay):
    """(p, m, v) after a step, float64."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    root = np.sqrt(v / (1 - betas[1] ** t)) + eps
    return p * (1 - lr * weight_decay) - lr * (m / (1 - betas[0] ** t)) / root, m, v


def moved(g, m, v, betas):
    """The moments after gradient g, float32 operation by operation."""
    b1, b2, r1, r2 = F(betas[0]), F(betas[1]), F(1 - betas[0]), F(1 - betas[1])
    return m * b1 + g * r1, v * b2 + (g * g) * r2


def updated(p, m, v, t, lr, betas, eps, weight_decay):
    """The parameters after moments m, v, float32 operation by operation."""
    rate, root = F(lr / (1 - betas[0] ** t)), F(1 / np.sqrt(1 - betas[1] ** t))
    return p * F(1 - lr * weight_decay) - (m * rate) / (np.sqrt(v) * root + F(eps))


def _scales(x):
    a = np.abs(x).max(axis=1)
    return np.where((a > 0) & (a < F(2.0 ** -126)), F(2.0 ** -126), a).astype(np.float32)


def _of_largest(x, scale):
    with np.errstate(divide="ignore"):
        return np.abs(x) * np.where(scale > 0, F(1) / scale, F(0)).astype(np.float32)[:, None]


def encode_m(x):
    """(codes int8, scales float32) of blocks (n, 256) of finite float32."""
    scale = _scales(x)
    code = np.rint(np.sqrt(_of_largest(x, scale)) * F(127))
    return (np.minimum(code, 127) * np.sign(x)).astype(np.int8), scale


def encode_v(x):
    """(codes uint8, scales float32) of blocks (n, 256) of finite float32, none below zero."""
    scale = _scales(x)
    code = np.minimum(np.rint(np.sqrt(np.sqrt(_of_largest(x, scale))) * F(255)), 255)
    return np.where(x > 0, np.maximum(code, 1), 0).astype(np.uint8), scale


def decode_m(code, scale):
    t = code.astype(np.float32) * F(1.0 / 127.0)
    return (t * np.abs(t)) * scale[:, None]


def decode_v(code, scale):
    t = code.astype(np.float32) * F(1.0 / 255.0)
    t = t * t
    return (t * t) * scale[:, None]
