"""The short causal convolution (GPU): outputs, states and gradients against the definition in float64.

Error bounds, in units of 2^-24 of the sums of magnitudes. pre has W + 1 roundings; silu adds its
sigmoid's units, 8, and one product, and passes pre's error on with a slope of at most 1.1; its own
slope's error is at most half of pre's and 16 units. A gradient of a value sums W of those; one of a
weight runs over at most 64 tokens of a run and then over the runs. Twice that for second-order terms. A
bfloat16 result is rounded once, by 2^-8 of itself.
"""

import numpy as np
import pytest
import torch

from oracle import causal_conv as occ

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
UNIT = 2.0 ** -24
NAMES = ("x", "weight", "bias", "state")


def make(dev, seed, b, t, d, w, dtype=F32, layout="apart", episode=5, without=()):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(b, t, d, generator=gen).to(dtype)
    if layout == "time":
        x = x.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
    elif layout == "odd":
        flat = torch.empty(b * t * (d + 3) + 1, dtype=dtype, device=dev)
        rows = flat[1:].view(b, t, d + 3)[..., 2:d + 2]
        rows.copy_(x)
        x = rows
    elif layout == "columns":
        x = x.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    c = {"x": x.to(dev), "weight": torch.randn(d, w, generator=gen).to(dev), "bias": torch.randn(d, generator=gen).to(dev),
         "state": torch.randn(b, w - 1, d, generator=gen).to(dev),
         "reset": (torch.rand(b, t, generator=gen) < 1.0 / episode).to(dev) if episode else None}
    c.update({name: None for name in without})
    return c


def to_np(x):
    return None if x is None else x.detach().cpu().numpy() if x.dtype == torch.bool else x.detach().double().cpu().numpy()


def close(got, want, bound, dtype=F32):
    got = to_np(got)
    assert got.shape == want.shape
    if dtype == BF16:
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
    off = np.abs(got - want) - bound
    assert np.all(off <= 1e-37), f"{off.max()} over the bound, worst {np.abs(got - want).max()}"


def check(dev, c, silu=True):
    from hipenvs import causal_conv

    (b, t, d), w, dtype = c["x"].shape, c["weight"].shape[1], c["x"].dtype
    leaves = {k: c[k].detach().requires_grad_() for k in NAMES if c[k] is not None}
    out, final = causal_conv.sequence(**{**c, **leaves}, silu=silu)
    with torch.no_grad():
        plain = causal_conv.sequence(**c, silu=silu)
    assert torch.equal(out, plain[0]) and torch.equal(final, plain[1])
    f64 = [to_np(c[k]) for k in (*NAMES, "reset")]
    dout, dfinal = torch.randn(b, t, d, device=dev).to(dtype), torch.randn(b, w - 1, d, device=dev)
    back = (to_np(dout), to_np(dfinal))
    want = occ.sequence(*f64, silu)
    size, sizes = occ.magnitudes(*f64, *back)
    close(out, want[0], 2 * UNIT * (1.1 * (w + 1) * size + 10 * np.abs(want[0])), dtype)
    assert np.array_equal(to_np(final), want[1])   # copies
    grads = torch.autograd.grad((out, final), list(leaves.values()), (dout, dfinal))
    expect = dict(zip(NAMES, occ.gradients(*f64, silu, *back)))
    bounds = dict(zip(NAMES, sizes))
    for (name, leaf), g in zip(leaves.items(), grads):
        length = 64 + b * (t + 7) // 8 if name in ("weight", "bias") else w
        close(g, expect[name], 2 * UNIT * (length + w + 24) * bounds[name], leaf.dtype)


SHAPES = [(1, 1, 1, 4), (2, 2, 3, 4), (3, 5, 4, 3), (2, 64, 64, 4), (1, 65, 129, 2), (5, 33, 7, 1), (2, 130, 30, 4),
          (40, 9, 12, 3), (1, 1000, 6, 4)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequence_and_gradients_match_the_definition(dev, shape, dtype):
    for k, (layout, episode, silu) in enumerate((("apart", 5, True), ("time", 0, True), ("odd", 2, False),
                                                 ("columns", 20, True))):
        print("conv", shape, dtype, layout, flush=True)
        check(dev, make(dev, k, *shape, dtype, layout, episode), silu)


@pytest.mark.parametrize("without", [("bias",), ("state",), ("bias", "state", "reset")])
def test_terms_left_out(dev, without):
    check(dev, make(dev, 3, 2, 37, 70, 4, without=without))


def test_what_a_reset_leaves_out(dev):
    from hipenvs import causal_conv

    c = make(dev, 1, 2, 30, 10, 4, episode=0)
    reset = torch.zeros(2, 30, dtype=torch.bool, device=dev)
    reset[:, 15] = True
    runs = []
    for bad in (False, True):
        x, state = c["x"].clone(), c["state"].clone()
        if bad:
            x[:, 12:15], state[:] = float("nan"), float("inf")
        x.requires_grad_()
        out, final = causal_conv.sequence(x, c["weight"], c["bias"], state, reset)
        runs.append((out.detach()[:, 15:], final.detach(), torch.autograd.grad(out[:, 15:].sum(), x)[0][:, 15:]))
    assert all(torch.isfinite(a).all() and torch.equal(a, e) for a, e in zip(*runs))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("w,d", [(4, 20), (1, 7), (2, 129), (3, 64)])
def test_step_by_step_is_the_sequence(dev, dtype, w, d):
    from hipenvs import causal_conv

    c = make(dev, 6, 9, 12, d, w, dtype, "time", 4)
    out, final = causal_conv.sequence(**c)
    state = c["state"].clone()
    for i in range(12):
        o, s = causal_conv.step(c["x"][:, i], c["weight"], c["bias"], state, c["reset"][:, i], next_state=state)
        assert s is state and torch.equal(o, out[:, i])
    assert torch.equal(state, final)
    before = c["state"].clone()
    _, s = causal_conv.step(c["x"][:, 0], c["weight"], c["bias"], c["state"], c["reset"][:, 0])
    assert torch.equal(before, c["state"]) and (w == 1 or s.data_ptr() != c["state"].data_ptr())


def test_empty(dev):
    from hipenvs import causal_conv

    for b, t in ((0, 5), (2, 0)):
        c = make(dev, 1, b, t, 6, 4)
        leaves = {k: v.detach().requires_grad_() if k in NAMES else v for k, v in c.items()}
        out, final = causal_conv.sequence(**leaves)
        assert out.shape == (b, t, 6) and torch.equal(final, c["state"])
        (out.sum() + final.sum()).backward()
        assert (leaves["weight"].grad == 0).all() and (leaves["state"].grad == 1).all()


def test_captured_training_and_steps_replay(dev):
    from hipenvs import causal_conv

    given = [make(dev, 20 + k, 3, 70, 30, 4) for k in range(4)]
    static = {k: v.clone() for k, v in given[0].items()}

    def train():
        leaves = {k: v.detach().requires_grad_() if k in NAMES else v for k, v in static.items()}
        out, final = causal_conv.sequence(**leaves)
        grads = torch.autograd.grad((out, final), [leaves[k] for k in NAMES], (static["x"], static["state"]))
        step = causal_conv.step(static["x"][:, 0], static["weight"], static["bias"], static["state"], static["reset"][:, 0])
        return (out.detach(), final.detach(), *grads, *step)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        train()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = train()
    for c in given[1:] + given[:2]:
        for k, v in static.items():
            v.copy_(c[k])
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        assert all(torch.equal(a, e) for a, e in zip(got, train()))


def test_rows_past_32_bit_offsets(dev):
    from hipenvs import causal_conv

    t, d, last = 33000, 65536, 9
    x = torch.zeros(1, t, d, dtype=BF16, device=dev)
    x[:, -last:] = torch.randn(1, last, d, device=dev).to(BF16)
    weight = torch.randn(d, 4, device=dev)
    out, final = causal_conv.sequence(x, weight)
    short, short_final = causal_conv.sequence(x[:, -last:], weight)
    assert torch.equal(out[:, -last:], short) and torch.equal(final, short_final)
    assert (out[:, :-last] == 0).all()


def test_refusals(dev):
    from hipenvs import causal_conv

    c = make(dev, 1, 2, 5, 6, 4)

    def refused(error, **changes):
        with pytest.raises(error):
            causal_conv.sequence(**{**c, **changes})

    refused(TypeError, x=c["x"].half())
    refused(TypeError, weight=c["weight"].to(BF16))
    refused(TypeError, reset=c["reset"].int())
    refused(ValueError, x=c["x"][0])
    refused(ValueError, weight=torch.zeros(6, 5, device=dev))
    refused(ValueError, weight=torch.zeros(5, 4, device=dev))
    refused(ValueError, bias=c["bias"][:5])
    refused(ValueError, state=c["state"][:, :2])
    refused(ValueError, state=c["state"].cpu())
    refused(ValueError, reset=c["reset"][:, :3])
    with pytest.raises(ValueError):
        causal_conv.step(c["x"][:, 0].detach().requires_grad_(), c["weight"])
    with pytest.raises(ValueError):
        causal_conv.step(c["x"][:, 0], c["weight"], next_state=torch.zeros(2, 6, 3, device=dev).transpose(1, 2))
