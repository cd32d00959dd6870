"""Log probabilities, entropies, the most likely tokens and the gradient of logits (GPU) against the
definition in float64.

Error bounds, in units of 2^-24. Of s = sum exp(x - m): a term's exponent r = m - x carries 2 r units (its
product with log2 e and its difference), which its size exp(-r) keeps below 1; exp2 adds 2; running sums
over v / 64 values a lane and 70 lanes, waves and parts, each perhaps rescaled (3 more), add that
many: UNITS(v). log s has those and 4 of itself. So a log probability is off by UNITS + 4 |log s| + 2 |x - m|,
an entropy, whose sum w has |w| / s as its size, by UNITS (1 + w / s) + 4 log s + 2 H, and a probability by
UNITS + 4 (|log p| + |log s|) of itself. A bfloat16 gradient is rounded once, by 2^-8 of itself.
"""

import numpy as np
import pytest
import torch

from oracle import categorical as oca

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
UNIT = 2.0 ** -24


def units(v):
    return 4.0 * (v / 64 + 70) + 16


def make(dev, seed, rows, v, dtype=F32, masked=0.0, spread=3.0, layout="apart"):
    gen = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(rows, v, generator=gen)).to(dtype)
    tokens = torch.randint(0, v, (rows,), generator=gen)
    if masked:
        out = torch.rand(rows, v, generator=gen) < masked
        out[torch.arange(rows), tokens] = False
        x[out] = -float("inf")
    tokens[torch.rand(rows, generator=gen) < 0.1] = -1
    if layout == "odd":
        flat = torch.empty(rows * (v + 5) + 3, dtype=dtype, device=dev)
        held = flat[3:].view(rows, v + 5)[:, 1:v + 1]
        held.copy_(x)
        x = held
    elif layout == "columns":
        x = x.t().contiguous().to(dev).t()
    return x.to(dev), tokens.to(dev)


def check(x, tokens, top=0, seed=0):
    from hipenvs import categorical

    rows, v = x.shape
    dtype, dev = x.dtype, x.device
    leaf = x.detach().requires_grad_()
    found = categorical.log_probs(leaf, tokens, top=top)
    with torch.no_grad():
        again = categorical.log_probs(x, tokens, top=top)
    assert all(torch.equal(a, b) for a, b in zip(found, again)) and len(found) == (4 if top else 2)
    f64, t = x.double().cpu().numpy(), tokens.cpu().numpy()
    lp, h = oca.log_probs(f64, t)
    lp = np.where(lp < -float(torch.finfo(F32).max), -np.inf, lp)   # a difference past float32's range
    with np.errstate(invalid="ignore"):
        m = f64.max(1)
        m0 = np.where(np.isneginf(m), 0.0, m)
        s = np.exp(f64 - m0[:, None]).sum(1)
        empty = np.isneginf(m)
        log_s = np.where(empty, 0.0, np.log(np.where(empty, 1.0, s)))
    mean = np.maximum(log_s - h, 0) + np.abs(h)   # |w| / s and more
    got = found[0].detach().double().cpu().numpy()
    fin = np.isfinite(lp)
    assert np.array_equal(got[~fin], lp[~fin])
    away = np.abs(np.where(fin, lp, 0.0) + log_s)
    assert np.all(np.abs(got[fin] - lp[fin]) <= (UNIT * (units(v) + 4 * log_s + 2 * away + 2))[fin])
    bound_h = UNIT * (units(v) * (1 + mean) + 4 * log_s + 2 * h + 2)
    assert np.all(np.abs(found[1].detach().double().cpu().numpy() - h) <= bound_h)
    if top:
        order = oca.top(f64, top)
        assert np.array_equal(found[3].cpu().numpy(), order)
        with np.errstate(invalid="ignore"):
            all_lp = np.where(empty[:, None], -np.inf, oca.log_softmax(f64))
        want = np.take_along_axis(all_lp, order, 1)
        want = np.where(want < -float(torch.finfo(F32).max), -np.inf, want)
        got = found[2].double().cpu().numpy()
        fin = np.isfinite(want)
        assert np.array_equal(got[~fin], want[~fin])
        wide = np.abs(np.where(fin, want, 0.0) + log_s[:, None])
        bound = UNIT * (units(v) + 4 * log_s[:, None] + 2 * wide + 2)
        assert np.all(np.abs(got[fin] - want[fin]) <= bound[fin])
    gen = torch.Generator().manual_seed(seed)
    da, db = (torch.randn(rows, generator=gen).to(dev) for _ in range(2))
    grad, = torch.autograd.grad(found[:2], leaf, (da, db))
    a, b = (y.double().cpu().numpy() for y in (da, db))
    want = oca.gradient(f64, t, a, b)
    with np.errstate(invalid="ignore"):
        all_lp = np.where(empty[:, None], -np.inf, oca.log_softmax(f64))
    p = np.exp(all_lp)
    flp = np.where(p > 0, np.abs(np.where(p > 0, all_lp, 0.0)), 0.0)
    size = p * (np.abs(a)[:, None] + np.abs(b)[:, None] * (flp + np.abs(h)[:, None]))
    unit = UNIT * (units(v) + 4 * (flp + log_s[:, None]) + 8)
    bound = unit * size + p * np.abs(b)[:, None] * (bound_h + UNIT * (units(v) + 4 * flp + 4 * log_s[:, None]
                                                                     ).max(1))[:, None]
    # exp2 gives 0 below 2^-126, the least normal number, where |log p| is at least 87
    tiny = 2.0 ** -126 * (np.abs(a)[:, None] + np.abs(b)[:, None] * (np.maximum(flp, 88) + np.abs(h)[:, None]))
    bound = bound + 2 * UNIT * np.abs(want) + tiny + 1e-37
    if dtype == BF16:
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
    off = np.abs(grad.double().cpu().numpy() - want) - bound
    assert grad.dtype == dtype and np.all(off <= 0), off.max()
    return found, grad


SHAPES = [(1, 1), (7, 2), (1000, 3), (300, 4), (65, 5), (33, 16), (50, 17), (20, 64), (9, 65), (13, 256), (5, 257),
          (6, 1000), (3, 1024), (3, 1025), (1, 4097), (2, 40009), (300, 1500), (700, 1100)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_log_probs_and_gradients_match_the_definition(dev, shape, dtype):
    rows, v = shape
    for k, (layout, masked, spread) in enumerate((("apart", 0.0, 3.0), ("odd", 0.4, 1.0), ("columns", 0.9, 20.0))):
        for top in (0, min(v, 1), min(v, 23)):
            print("log_probs", shape, dtype, layout, top, flush=True)
            check(*make(dev, k, rows, v, dtype, masked, spread, layout), top)
    check(*make(dev, 9, rows, v, dtype), min(v, 64))


@pytest.mark.parametrize("v", [6, 8, 9, 24, 32, 33, 66, 128, 129, 255, 400, 512, 513])
def test_rows_of_every_number_of_lanes(dev, v):
    for k, dtype in enumerate((F32, BF16)):
        print("log_probs", v, dtype, flush=True)
        check(*make(dev, 20 + k, 300, v, dtype, 0.3, 2.0, "odd"), min(v, 5))


@pytest.mark.parametrize("v", [3, 100, 900, 5000, 20000])
def test_rows_that_leave_nothing_and_extreme_masks(dev, v):
    """Rows of -inf alone, masks of the type's lowest value, one token left, the given token not allowed."""
    for dtype in (F32, BF16):
        x, tokens = make(dev, 4, 9, v, dtype)
        low = torch.finfo(dtype).min
        x[0] = -float("inf")
        x[1] = low                                   # all alike: uniform
        x[2, 1:] = low
        x[3, :-1] = -float("inf")
        x[4, 0] = torch.finfo(dtype).max
        x[5, 0], x[5, 1] = torch.finfo(dtype).max, low
        tokens[:] = torch.tensor([0, 1, 0, v - 1, 0, 0, -1, 2, 1])
        x[7, 2] = -float("inf")
        (lp, h, best, index), grad = check(x, tokens, min(v, 5))
        assert lp[0] == -float("inf") and h[0] == 0 and (grad[0] == 0).all()
        assert index[0].tolist() == list(range(min(v, 5)))
        assert lp[7] == -float("inf") and lp[6] == 0


@pytest.mark.parametrize("v", [3, 900, 5000])
def test_a_row_that_is_no_number(dev, v):
    from hipenvs import categorical

    x, tokens = make(dev, 4, 6, v)
    tokens[:] = 1
    tokens[4] = v                                    # past the row
    x[1, 2], x[2, 0] = float("nan"), float("inf")
    x.requires_grad_()
    lp, h, best, index = categorical.log_probs(x, tokens, top=2)
    assert torch.isnan(lp).tolist() == [False, True, True, False, True, False]
    assert torch.isnan(h).tolist() == [False, True, True, False, False, False]
    assert index[1, 0] == 2 and index[2, 0] == 0     # NaN first, as the largest
    grad, = torch.autograd.grad(lp[:4].sum() + h[:4].sum(), x)
    assert torch.isnan(grad[1]).all() and torch.isnan(grad[2]).all() and torch.isfinite(grad[[0, 3, 5]]).all()


def test_ties_go_to_the_lowest_index(dev):
    from hipenvs import categorical

    for v in (7, 300, 1000, 9000, 50000):
        gen = torch.Generator().manual_seed(v)
        x = torch.randint(-2, 3, (5, v), generator=gen).float()
        x[1] = 0.0
        x[2] = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)
        x[3] = torch.arange(v).float()               # every one the largest so far
        k = min(v, 64)
        _, _, _, index = categorical.log_probs(x.to(dev), torch.zeros(5, dtype=torch.int32, device=dev), top=k)
        assert np.array_equal(index.cpu().numpy(), oca.top(x.double().numpy() + 0.0, k))


def test_leading_axes_and_gradients_that_are_missing(dev):
    from hipenvs import categorical

    x, tokens = make(dev, 2, 24, 11)
    flat = categorical.log_probs(x, tokens, top=3)
    shaped = categorical.log_probs(x.view(2, 3, 4, 11), tokens.view(2, 3, 4), top=3)
    assert all(torch.equal(a.view(b.shape), b) and b.shape[:3] == (2, 3, 4) for a, b in zip(flat, shaped))
    turned = categorical.log_probs(x.view(4, 6, 11).transpose(0, 1), tokens.view(4, 6).t(), top=3)
    assert all(torch.equal(a.view(4, 6, *a.shape[1:]).transpose(0, 1), b) for a, b in zip(flat, turned))
    one = categorical.log_probs(x[0], tokens[0], top=3)
    assert all(torch.equal(a[0], b) for a, b in zip(flat, one))
    leaf = x.detach().requires_grad_()
    f64, t = x.double().cpu().numpy(), tokens.cpu().numpy()
    for which, pair in ((0, (1.0, 0.0)), (1, (0.0, 1.0))):
        out = categorical.log_probs(leaf, tokens)[which]
        grad, = torch.autograd.grad(out.mean(), leaf)
        want = oca.gradient(f64, t, *(np.full(24, y / 24) for y in pair))
        assert np.allclose(grad.double().cpu().numpy(), want, rtol=1e-4, atol=1e-7)
    a, b, c, d = categorical.log_probs(leaf, tokens, top=2)
    assert a.requires_grad and b.requires_grad and not c.requires_grad and not d.requires_grad


def test_empty(dev):
    from hipenvs import categorical

    x = torch.zeros(0, 5, device=dev, requires_grad=True)
    found = categorical.log_probs(x, torch.zeros(0, dtype=torch.int64, device=dev), top=2)
    assert [tuple(y.shape) for y in found] == [(0,), (0,), (0, 2), (0, 2)]
    (found[0].sum() + found[1].sum()).backward()
    assert x.grad.shape == (0, 5)
    found = categorical.log_probs(torch.zeros(3, 0, 5, device=dev), torch.zeros(3, 0, dtype=torch.int64, device=dev))
    assert found[0].shape == (3, 0)


@pytest.mark.parametrize("shape", [(50, 3), (20, 900), (2, 20000)])
def test_captured_training_replays(dev, shape):
    from hipenvs import categorical

    given = [make(dev, 40 + k, *shape) for k in range(4)]
    x, tokens = (y.clone() for y in given[0])

    def train():
        leaf = x.detach().requires_grad_()
        found = categorical.log_probs(leaf, tokens, top=3)
        grad, = torch.autograd.grad(found[:2], leaf, (x[:, 0], x[:, 1]))
        return (*(y.detach() for y in found), grad)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        train()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = train()
    for c in given[1:] + given[:2]:
        x.copy_(c[0])
        tokens.copy_(c[1])
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in captured]
        assert all(torch.equal(a, e) for a, e in zip(got, train()))


def test_rows_past_32_bit_offsets(dev):
    from hipenvs import categorical

    v = 40009
    rows = (1 << 31) // v + 20
    x = torch.zeros(rows, v, dtype=BF16, device=dev)
    x[-5:] = torch.randn(5, v, device=dev).to(BF16)
    tokens = torch.randint(0, v, (rows,), device=dev)
    x.requires_grad_()
    lp, h = categorical.log_probs(x, tokens)
    grad, = torch.autograd.grad(lp.sum() + h.sum(), x)
    y = x.detach()[-5:].clone().requires_grad_()
    lp5, h5 = categorical.log_probs(y, tokens[-5:])
    grad5, = torch.autograd.grad(lp5.sum() + h5.sum(), y)
    # other parts of the rows: other roundings
    assert torch.allclose(lp[-5:], lp5, rtol=1e-5) and torch.allclose(h[-5:], h5, rtol=1e-5)
    assert torch.allclose(grad[-5:].float(), grad5.float(), rtol=2.0 ** -7, atol=1e-9)
    assert torch.allclose(lp[0], torch.tensor(-np.log(v), dtype=F32, device=dev), rtol=1e-5)


def test_refusals(dev):
    from hipenvs import categorical

    x, tokens = torch.zeros(3, 5, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for bad in (dict(logits=x.half()), dict(tokens=tokens.float()), dict(tokens=[0, 0, 0]), dict(logits="x")):
        with pytest.raises(TypeError):
            categorical.log_probs(**{"logits": x, "tokens": tokens, **bad})
    for bad in (dict(logits=x[:, :0]), dict(tokens=tokens[:2]), dict(tokens=tokens.cpu()), dict(top=6), dict(top=-1),
                dict(logits=x.cpu()), dict(logits=torch.tensor(1.0, device=dev), tokens=tokens[0])):
        with pytest.raises(ValueError):
            categorical.log_probs(**{"logits": x, "tokens": tokens, **bad})
    with pytest.raises(ValueError):
        categorical.log_probs(torch.zeros(1, 100, device=dev), tokens[:1], top=65)
