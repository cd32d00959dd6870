"""Decay attention (GPU) with bfloat16 rows: every operand of its products carries float32's 24 bits.

Two kinds of test. On whole numbers without decay every product and sum is a whole number, and
where the sum of the terms' magnitudes stays within 2^24 every order of float32 sums gives it
exactly: the result is that number, rounded once to bfloat16, and the tolerance is zero. The
values are arranged so that large operands (weights q.k, states, scaled rows, of 18 to 20 bits)
cancel in the results: an operand held in fewer bits shows in full.

On random values the bound is float32's own, as for float32 rows (a term meets at most
t + dk + dv + 256 roundings of 2^-24, twice that for the matrix instructions; an operand's three
bfloat16 parts leave less than one such rounding), and one rounding of the result to bfloat16:
2^-8 of it.
"""

import numpy as np
import pytest
import torch

from oracle import decay_attention as oda
from test_gpu_decay_attention import BF16, F32, SHAPES, case, gamma, to_np

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "log_decay", "state", "reset")


def results(c, scale, dout, dfinal):
    """(out, final state, dq, dk, dv, dstate) of the kernels."""
    from hipenvs import decay_attention

    leaves = [c[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
    out, final = decay_attention.sequence(*leaves[:3], c["log_decay"], leaves[3], c["reset"], scale=scale)
    return out.detach(), final.detach(), *torch.autograd.grad((out, final), leaves, (dout, dfinal))


def once(want):
    """float64 values that float32 holds exactly, rounded once to bfloat16."""
    assert np.array_equal(want, want.astype(np.float32))
    return torch.from_numpy(want.astype(np.float32)).to(BF16)


def exact(dev, c, scale, dout, dfinal, large):
    """The results on whole numbers, bit for bit. `large`: results whose operands are large."""
    c, dout, dfinal = ({n: torch.from_numpy(x) for n, x in c.items()}, torch.from_numpy(dout), torch.from_numpy(dfinal))
    for n in ("q", "k", "v"):
        assert torch.equal(c[n].to(BF16).double(), c[n])
        c[n] = c[n].to(BF16).to(dev)
    assert torch.equal(dout.to(BF16).double(), dout)
    c["log_decay"] = torch.zeros(c["q"].shape[2], device=dev)
    c["state"], c["reset"] = c["state"].float().to(dev), c["reset"].to(dev)
    dout, dfinal = dout.to(BF16).to(dev), dfinal.float().to(dev)
    args = [to_np(c[n]) for n in NAMES]
    grads = (to_np(dout), to_np(dfinal))
    want = (*oda.sequence(*args, scale), *oda.gradients(*args, scale, *grads))
    size = oda.magnitudes(*args, scale, *grads)
    for x in size:
        assert x.max() <= 2.0 ** 24   # else the sums' order matters
    for i in large:   # terms of at least 18 bits
        assert size[i].max() >= 2.0 ** 21
    got = results(c, scale, dout, dfinal)
    for name, x, w in zip(("out", "final", "dq", "dk", "dv", "dstate"), got, want):
        y = torch.from_numpy(w.astype(np.float32)) if x.dtype == F32 else once(w)
        off = (x.cpu().double() - y.double()).abs()
        assert torch.equal(x.cpu().double(), y.double()), f"{name}: {int((off > 0).sum())} of {off.numel()} off, by up to {off.max()}"


def signs(rng, *shape):
    return rng.choice((-1.0, 1.0), size=shape)


def pairs(rng, large, *shape):
    """(b, t, h, d) values of `large` magnitude: tokens 2 m and 2 m + 1 equal but for one column in
    one pair of four."""
    x = np.rint(rng.uniform(0.8, 1.2, size=shape) * large)
    b, t, h, d = shape
    x[:, 1::2] = x[:, 0:t - 1:2]
    x[:, 1::8, :, rng.integers(d)] += 1.0
    return x


def alternating(rng, *shape):
    """(b, t, h, d) of -1 and 1, each value at 2 m + 1 the negative of that at 2 m."""
    x = signs(rng, *shape)
    x[:, 1::2] = -x[:, 0:shape[1] - 1:2]
    return x


EXACT = [(2, 150, 2, 32, 32), (1, 150, 2, 16, 16), (1, 130, 2, 64, 64), (1, 131, 1, 96, 80), (1, 130, 1, 128, 128),
         (1, 150, 2, 64, 16), (1, 150, 2, 16, 64), (1, 6000, 1, 32, 32)]


@pytest.mark.parametrize("shape", EXACT)
def test_weights_of_19_bits(dev, shape):
    """q.k about 280,000 with values of alternating sign (outputs and dv), then dout.v of that
    size with keys and queries of alternating sign (dq and dk). Episodes of 40 tokens."""
    b, t, h, dk, dv = shape
    print("weights", shape, flush=True)
    rng = np.random.default_rng(1)
    reset = np.zeros((b, t), bool)
    reset[:, 24::40] = True
    zeros = np.zeros((b, h, dk, dv))
    big = 280000.0
    c = {"q": pairs(rng, (big / dk) ** 0.5, b, t, h, dk), "k": pairs(rng, (big / dk) ** 0.5, b, t, h, dk),
         "v": alternating(rng, b, t, h, dv), "state": zeros, "reset": reset}
    exact(dev, c, 1.0, alternating(rng, b, t, h, dv), zeros, (0, 4))
    c = {"q": alternating(rng, b, t, h, dk), "k": alternating(rng, b, t, h, dk),
         "v": pairs(rng, (big / dv) ** 0.5, b, t, h, dv), "state": zeros, "reset": reset}
    exact(dev, c, 1.0, pairs(rng, (big / dv) ** 0.5, b, t, h, dv), zeros, (2, 3))


@pytest.mark.parametrize("shape", EXACT)
def test_states_of_18_bits(dev, shape):
    """States and their gradients about 200,000 with signs like a chess board's, read by rows of
    ones: of S, what is left are differences of a few units."""
    b, t, h, dk, dv = shape
    print("states", shape, flush=True)
    rng = np.random.default_rng(2)

    def board():
        x = np.rint(200003 + rng.uniform(-40, 40, size=(b, h, dk, dv)))
        return x * np.where((np.arange(dk)[:, None] + np.arange(dv)) % 2, -1.0, 1.0)

    def few(d):   # 16 of the columns are one, pairs of neighbours of unlike sign in the board
        x = np.zeros((b, t, h, d))
        for i in range(b):
            for j in range(t):
                at = 2 * rng.choice(d // 2, size=8, replace=False)
                x[i, j, :, at] = x[i, j, :, at + 1] = 1.0
        return x

    def sparse(d, n):   # one column of n tokens in a row: little beside the state
        x = np.zeros((b, t, h, d))
        at = rng.integers(t, size=n)
        x[:, at, :, rng.integers(d, size=n)] = 1.0
        return x

    reset = np.zeros((b, t), bool)
    reset[:, t // 2] = True   # the state reaches the tokens before, its gradient those from there on
    c = {"q": few(dk), "k": sparse(dk, 5), "v": sparse(dv, 5), "state": board(), "reset": reset}
    exact(dev, c, 1.0, few(dv), np.zeros((b, h, dk, dv)), (0, 2))
    c = {"q": sparse(dk, 5), "k": few(dk), "v": few(dv), "state": np.zeros((b, h, dk, dv)), "reset": reset}
    exact(dev, c, 1.0, sparse(dv, 5), board(), (3, 4))


@pytest.mark.parametrize("shape", EXACT)
def test_scaled_rows_of_20_bits(dev, shape):
    """What enters the states' gradients is scale * dout, here 200,003 times 3, -1 and -2 in turn,
    whose sums over an episode of 21 tokens cancel: dk and dv where an episode crosses chunks."""
    b, t, h, dk, dv = shape
    print("scaled rows", shape, flush=True)
    rng = np.random.default_rng(3)
    scale = 200003.0
    reset = np.zeros((b, t), bool)
    reset[:, 11::21] = True   # chunks begin at 64 n: inside episodes
    begin = np.maximum.accumulate(np.where(reset[0], np.arange(t), 0))
    turn = np.array([3.0, -1.0, -2.0])[(np.arange(t) - begin) % 3]
    row, column = rng.integers(dk), rng.integers(dv)   # one column of each row counts
    q, k, v, dout = (np.zeros((b, t, h, d)) for d in (dk, dk, dv, dv))
    q[..., row] = k[..., row] = v[..., column] = 1.0
    dout[..., column] = turn[None, :, None]
    zeros = np.zeros((b, h, dk, dv))
    exact(dev, {"q": q, "k": k, "v": v, "state": zeros, "reset": reset}, scale, dout, zeros, (3, 4))


def bound(size, want, dtype, t, dk, dv):
    b = gamma(t, dk, dv) * size
    return b + 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -6) if dtype == BF16 else b


def within(got, want, size, t, dk, dv, name):
    off = np.abs(to_np(got) - want) - bound(size, want, got.dtype, t, dk, dv)
    assert np.all(off <= 1e-37), f"{name}: {off.max()} over the bound"


@pytest.mark.parametrize("shape", SHAPES)
def test_random_rows_at_float32_s_bound(dev, shape):
    b, t, h, dk, dv = shape
    print("float32's bound", shape, flush=True)
    for seed, episode in ((50, 0), (51, 40)):
        c = case(dev, seed, *shape, BF16, "fused", episode)
        gen = torch.Generator().manual_seed(seed)
        dout = torch.randn(b, t, h, dv, generator=gen).to(BF16).to(dev)
        dfinal = torch.randn(b, h, dk, dv, generator=gen).to(dev)
        args, scale = [to_np(c[n]) for n in NAMES], dk ** -0.5
        grads = (to_np(dout), to_np(dfinal))
        want = (*oda.sequence(*args, scale), *oda.gradients(*args, scale, *grads))
        size = oda.magnitudes(*args, scale, *grads)
        got = results(c, scale, dout, dfinal)
        for name, x, w, s in zip(("out", "final", "dq", "dk", "dv", "dstate"), got, want, size):
            within(x, w, s, t, dk, dv, name)


@pytest.mark.parametrize("shape", [(3, 2, 5, 3), (64, 4, 32, 32), (7, 3, 48, 80), (5, 2, 128, 128), (9, 1, 31, 127)])
def test_a_step_at_float32_s_bound(dev, shape):
    from hipenvs import decay_attention

    n, h, dk, dv = shape
    c = case(dev, 52, n, 1, h, dk, dv, BF16, "fused", 2)
    args = [to_np(c[x]) for x in NAMES]
    want, size = oda.sequence(*args, dk ** -0.5), oda.magnitudes(*args, dk ** -0.5)
    out, state = decay_attention.step(*(c[x][:, 0] for x in "qkv"), c["log_decay"], c["state"], c["reset"][:, 0])
    within(out, want[0][:, 0], size[0][:, 0], 1, dk, dv, "out")
    within(state, want[1], size[1], 1, dk, dv, "state")
