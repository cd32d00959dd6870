"""The selective scan (GPU): outputs, states and gradients against the definition in float64.

Error bounds. A is the same sum over the magnitudes of its terms. A term of a state of T tokens meets at
most T roundings of the running state, and T decays whose exponents delta rate carry the roundings of delta
(within SOFTPLUS units of 2^-24 of its own size), of rate log2(e) and of the two products: together
(SOFTPLUS + 4) units of the exponents' sum, which is at most 104 before the decay is zero, and 2 more
units a decay. What is read or summed from states adds the sum's length. A gradient has two such terms
as factors. UNITS below counts all of it, twice for safety of second-order terms; SOFTPLUS is itself
tested. A gate adds the units of a sigmoid, SIGMOID, of its size. A bfloat16 result is rounded once,
by 2^-8 of itself.
"""

import numpy as np
import pytest
import torch

from oracle import selective_scan as oss

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SOFTPLUS, SIGMOID = 8, 8
NAMES = ("x", "dt", "rate", "write", "read", "skip", "gate", "dt_bias", "state")


def make(dev, seed, b, t, d, n, g, dtype=F32, layout="apart", episode=7, without=(), fast=False):
    gen = torch.Generator().manual_seed(seed)

    def rows(*widths):
        if layout == "fused":     # parts of one projection's rows
            parts = torch.split(torch.randn(b, t, sum(widths), generator=gen).to(dtype).to(dev), widths, -1)
        elif layout == "time":    # collected time-major
            parts = torch.split(torch.randn(t, b, sum(widths), generator=gen).to(dtype).to(dev).transpose(0, 1), widths, -1)
        elif layout == "odd":     # one element past every alignment
            parts = []
            for w in widths:
                flat = torch.empty(b * t * w + 1, dtype=dtype, device=dev)
                flat[1:] = torch.randn(b * t * w, generator=gen).to(dtype).to(dev)
                parts.append(flat[1:].view(b, t, w))
        elif layout == "columns":   # last axis not contiguous
            parts = [torch.randn(b, w, t, generator=gen).to(dtype).to(dev).transpose(1, 2) for w in widths]
        else:
            parts = [torch.randn(b, t, w, generator=gen).to(dtype).to(dev) for w in widths]
        return parts

    x, gate = rows(d, d)
    dt, write, read = rows(d, g * n, g * n)
    if g == 1 and seed % 2:
        mix = [write, read]
    else:
        mix = [m.unflatten(-1, (g, n)) if m.stride(-1) == 1 or g * n == 1 else m.reshape(b, t, g, n) for m in (write, read)]
    c = {"x": x, "dt": dt, "rate": -torch.exp(torch.randn(d, n, generator=gen)).to(dev) * (30.0 if fast else 1.0),
         "write": mix[0], "read": mix[1], "skip": torch.randn(d, generator=gen).to(dev), "gate": gate,
         "dt_bias": (torch.randn(d, generator=gen) - 2.0).to(dev), "state": torch.randn(b, d, n, generator=gen).to(dev),
         "reset": (torch.rand(b, t, generator=gen) < 1.0 / episode).to(dev) if episode else None}
    c.update({name: None for name in without})
    return c


def to_np(c):
    out = {}
    for k, v in c.items():
        out[k] = None if v is None else v.detach().cpu().numpy() if v.dtype == torch.bool else v.detach().double().cpu().numpy()
    for k in ("write", "read"):
        if out[k].ndim == 3:
            out[k] = out[k][:, :, None]
    return out


def units(t, d, n):
    return 2.0 * 2.0 ** -24 * (5 * t + (SOFTPLUS + 4) * 104 + n + d + 64)


def close(got, want, size, dtype, unit):
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape, (got.shape, want.shape)
    bound = unit * size + 1e-37
    if dtype == BF16:
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
    off = np.abs(got - want) - bound
    assert np.all(off <= 0), f"{off.max()} over the bound, worst {np.abs(got - want).max()} of {np.abs(want).max()}"


def check(dev, c, train=True, use_out=True, use_final=True):
    from hipenvs import selective_scan

    (b, t, d), n, dtype = c["x"].shape, c["rate"].shape[1], c["x"].dtype
    with torch.no_grad():
        out, final = selective_scan.sequence(**c)
    assert out.dtype == dtype and final.dtype == F32 and out.is_contiguous() and final.is_contiguous()
    f64 = to_np(c)
    dout = torch.randn(b, t, d, device=dev).to(dtype)
    dfinal = torch.randn(b, d, n, device=dev)
    back = [g.double().cpu().numpy() * on for g, on in ((dout, use_out), (dfinal, use_final))]
    size = oss.magnitudes(*f64.values(), *back)
    unit = units(t, d, n)
    want = oss.sequence(**f64)
    close(out, want[0], size[0], dtype, unit)
    close(final, want[1], size[1], F32, unit)
    if not train:
        return out, final
    leaves = {k: c[k].detach().requires_grad_() for k in NAMES if c[k] is not None}
    out2, final2 = selective_scan.sequence(**{**c, **leaves})
    assert torch.equal(out2, out) and torch.equal(final2, final)
    pairs = [(o, g) for o, g, on in ((out2, dout, use_out), (final2, dfinal, use_final)) if on]
    got = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs], allow_unused=True)
    grads = dict(zip(NAMES, oss.gradients(*f64.values(), *back)))
    sizes = dict(zip(NAMES, size[2:]))
    for (name, leaf), g in zip(leaves.items(), got):
        if g is None:   # what only the outputs read, where only the states are used
            assert name in ("read", "skip", "gate") and not use_out
            continue
        w, s = (x.reshape(leaf.shape) for x in (grads[name], sizes[name]))
        # parameters are summed over all rows and tokens
        extra = b * t if name in ("rate", "skip", "dt_bias") else 0
        close(g, w, s, leaf.dtype, 2 * unit + 2.0 ** -23 * extra)
    return out, final


SHAPES = [  # b, t, d, n, g
    (1, 1, 1, 1, 1), (2, 3, 5, 3, 1), (2, 15, 64, 4, 1), (1, 16, 65, 5, 5), (3, 17, 130, 16, 2), (2, 33, 100, 16, 4),
    (1, 100, 64, 64, 1), (2, 50, 40, 33, 2), (1, 70, 96, 20, 3), (40, 9, 12, 8, 1), (2, 31, 3, 2, 3), (1, 40, 257, 7, 1),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequence_and_gradients_match_the_definition(dev, shape, dtype):
    for k, (layout, episode) in enumerate((("fused", 7), ("time", 0), ("odd", 90), ("columns", 2))):
        print("scan", shape, dtype, layout, flush=True)
        check(dev, make(dev, k, *shape, dtype, layout, episode))


# groups of few channels and of more, at every number of lanes, with all of their states and without
@pytest.mark.parametrize("n", [6, 8, 13, 16, 27, 32, 61, 64])
@pytest.mark.parametrize("d,g", [(1, 1), (16, 1), (31, 1), (32, 1), (33, 1), (65, 1), (96, 3), (68, 2)])
def test_groups_of_every_width(dev, d, g, n):
    for k, dtype in enumerate((F32, BF16)):
        print("scan", d, g, n, dtype, flush=True)
        check(dev, make(dev, 30 + k, 2, 19, d, n, g, dtype, ("fused", "odd")[k], 11))


@pytest.mark.parametrize("without", [("skip",), ("gate",), ("dt_bias",), ("state",), ("skip", "gate", "dt_bias", "state")])
def test_terms_left_out(dev, without):
    check(dev, make(dev, 3, 2, 37, 70, 16, 1, without=without))


def test_gradients_of_one_output(dev):
    c = make(dev, 4, 2, 37, 70, 6, 2)
    check(dev, c, use_final=False)
    check(dev, c, use_out=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [3, 8, 16, 30, 50])
def test_few_long_rows(dev, dtype, n):
    """Rows walked in parts, with and without episodes, slow and fast decays."""
    for episode, fast in ((0, False), (300, True), (5, False)):
        print("long", n, dtype, episode, flush=True)
        check(dev, make(dev, 5, 2, 709, 24, n, 2, dtype, "fused", episode, fast=fast))
    check(dev, make(dev, 6, 1, 128, 8, n, 1, dtype, "fused", 0))


@pytest.mark.parametrize("n", [3, 8, 16, 30, 32, 50, 64])
def test_few_long_rows_of_wide_groups(dev, n):
    for k, (b, d, g) in enumerate(((2, 80, 1), (1, 140, 2))):
        print("long", n, d, g, flush=True)
        check(dev, make(dev, 40 + k, b, 517, d, n, g, (F32, BF16)[k], "fused", (0, 200)[k]))


def test_softplus_and_sigmoid_units(dev):
    """delta from one token of a zero state: within SOFTPLUS units and the four of products; and silu."""
    from hipenvs import selective_scan

    d = 60000
    dt = torch.linspace(-60.0, 40.0, d, device=dev)[None]
    one, ones = torch.ones(1, d, device=dev), torch.ones(1, 1, device=dev)
    rate = torch.full((d, 1), -1.0, device=dev)
    out, _ = selective_scan.step(one, dt, rate, ones, ones)
    want = oss.softplus(dt.double().cpu().numpy())
    off = np.abs(out.double().cpu().numpy() / want - 1)
    print("softplus units", off.max() * 2 ** 24, flush=True)
    assert off.max() <= (SOFTPLUS + 1) * 2.0 ** -24
    out, _ = selective_scan.step(one, torch.full_like(dt, 1.0), rate, ones, ones, gate=dt)
    z = dt.double().cpu().numpy()
    want = np.log1p(np.e) * z * oss.sigmoid(z)
    big = np.abs(want) > 1e-30
    off = np.abs(out.double().cpu().numpy() - want)[big] / np.abs(want)[big]
    print("silu units", off.max() * 2 ** 24, flush=True)
    assert off.max() <= (SOFTPLUS + SIGMOID + 3) * 2.0 ** -24


def test_extreme_steps(dev):
    """dt far out on both sides: no decay and nothing added, or all of the state gone."""
    from hipenvs import selective_scan

    x, mix = torch.ones(1, 3, 4, device=dev), torch.ones(1, 3, 2, device=dev)
    dt = torch.tensor([-300.0, -float("inf"), -104.5, 1e30], device=dev).expand(1, 3, 4).contiguous()
    rate = torch.full((4, 2), -1.0, device=dev)
    state = torch.full((1, 4, 2), 3.0, device=dev)
    out, final = selective_scan.sequence(x, dt, rate, mix, mix, state=state)
    assert torch.equal(out[0, :, :3], torch.full((3, 3), 6.0, device=dev)) and torch.equal(final[0, :3], state[0, :3])
    assert torch.equal(final[0, 3], torch.full((2,), 1e30, device=dev))


@pytest.mark.parametrize("t", [40, 900])
def test_what_a_reset_leaves_out(dev, t):
    """A NaN or an infinity before an episode's first token, in the state too, does not reach it."""
    from hipenvs import selective_scan

    b, d, n = 2, 20, 16
    c = make(dev, 8, b, t, d, n, 1, without=("reset",))
    reset = torch.zeros(b, t, dtype=torch.bool, device=dev)
    at = t // 2 + 3
    reset[:, at] = True
    good = {k: v for k, v in c.items()}
    bad = dict(good)
    bad["state"] = torch.full_like(c["state"], float("nan"))
    bad["x"] = c["x"].clone()
    bad["x"][:, 5] = float("inf")
    bad["write"] = c["write"].clone()
    bad["write"][:, 7] = float("nan")
    bad["reset"] = good["reset"] = reset
    leaves = []
    for given in (good, bad):
        given = {k: v.detach().requires_grad_() if v is not None and k in NAMES else v for k, v in given.items()}
        out, final = selective_scan.sequence(**given)
        grads = torch.autograd.grad((out[:, at:].sum(), final.sum()), [given[k] for k in ("x", "write", "read", "dt")])
        leaves.append((out.detach()[:, at:], final.detach(), *(g[:, at:] for g in grads)))
    for a, e in zip(*leaves):
        assert torch.isfinite(a).all() and torch.equal(a, e)


@pytest.mark.parametrize("n", [3, 5, 8, 12, 16, 24, 40, 64])
def test_infinities_reach_what_they_should(dev, n):
    """An infinite x of one channel: its outputs and states are infinite until the episode ends, and no other
    channel's or later token's is touched; an infinite dt decays all of a state, past n too."""
    from hipenvs import selective_scan

    b, t, d = 1, 40, 6
    x, dt = torch.ones(b, t, d, device=dev), torch.zeros(b, t, d, device=dev)
    mix = torch.ones(b, t, n, device=dev)
    rate = -torch.full((d, n), 0.01, device=dev)
    reset = torch.zeros(b, t, dtype=torch.bool, device=dev)
    reset[0, 30] = True
    clean, _ = selective_scan.sequence(x, dt, rate, mix, mix, reset=reset)
    x[0, 3, 2] = float("inf")
    out, final = selective_scan.sequence(x, dt, rate, mix, mix, reset=reset)
    assert torch.isinf(out[0, 3:30, 2]).all() and torch.isfinite(final).all()
    keep = torch.ones(b, t, d, dtype=torch.bool, device=dev)
    keep[0, 3:30, 2] = False
    assert torch.equal(out[keep], clean[keep])
    state = torch.zeros(1, d, n, device=dev)
    acted = []
    for i in range(t):
        o, _ = selective_scan.step(x[:, i], dt[:, i], rate, mix[:, i], mix[:, i], state=state, reset=reset[:, i],
                                   next_state=state)
        acted.append(o)
    acted = torch.stack(acted, 1)
    assert torch.equal(torch.isinf(acted), ~keep) and torch.isfinite(state).all()
    # the gradients of a clean window before and behind it, an infinite dout of one token among them
    x = torch.ones(b, t, d, device=dev, requires_grad=True)
    dout = torch.ones(b, t, d, device=dev)
    dout[0, 35, 1] = float("inf")
    out, _ = selective_scan.sequence(x, dt, rate, mix, mix, reset=reset)
    dx, = torch.autograd.grad(out, x, dout)
    assert torch.isinf(dx[0, 30:36, 1]).all() and torch.isfinite(dx[0, :30]).all() and torch.isfinite(dx[0, 36:]).all()
    # an infinite dt: the state before is gone, the token's own is infinite
    dt = dt.clone()
    dt[0, 5, 4] = float("inf")
    out, _ = selective_scan.sequence(x.detach(), dt, rate, mix, mix, reset=reset)
    assert torch.isinf(out[0, 5:30, 4]).all() and torch.isfinite(out[0, 30:]).all() and torch.isfinite(out[0, :5]).all()


def test_infinite_and_zero_states_pass_parts(dev):
    """An infinite state stays infinite and a zero one zero over parts whose decay leaves float32's
    range, as token by token."""
    from hipenvs import selective_scan

    t, d, n = 1024, 2, 16
    x = torch.zeros(1, t, d, device=dev)
    dt = torch.full((1, t, d), 1.0, device=dev)
    mix = torch.ones(1, t, n, device=dev)
    rate = torch.tensor([-1.0, 1.0], device=dev)[:, None].expand(d, n).contiguous()
    state = torch.stack([torch.full((n,), float("inf")), torch.zeros(n)])[None].to(dev)
    _, final = selective_scan.sequence(x, dt, rate, mix, mix, state=state)
    assert torch.equal(final, state)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,g", [(16, 1), (5, 2), (64, 1), (1, 1), (24, 4)])
def test_step_by_step_is_the_sequence(dev, dtype, n, g):
    """step over the tokens, the state updated in place, against the definition and the sequence."""
    from hipenvs import selective_scan

    b, t, d = 9, 12, 20
    c = make(dev, 9 + 2 * g, b, t, d, n, g, dtype, "fused", 4)
    out, final = selective_scan.sequence(**c)
    state = c["state"].clone()
    steps = []
    for i in range(t):
        one = {k: (v[:, i] if k in ("x", "dt", "write", "read", "gate", "reset") else v) for k, v in c.items()}
        o, s = selective_scan.step(**{**one, "state": state}, next_state=state)
        assert s is state
        steps.append(o)
    f64 = to_np(c)
    want = oss.sequence(**f64)
    size = oss.magnitudes(*f64.values(), np.zeros(out.shape), np.zeros(final.shape))
    close(torch.stack(steps, 1), want[0], size[0], dtype, units(t, d, n))
    close(state, want[1], size[1], F32, units(t, d, n))


def test_step_makes_new_states(dev):
    from hipenvs import selective_scan

    c = make(dev, 2, 6, 1, 10, 16, 1)
    one = {k: (v[:, 0] if k in ("x", "dt", "write", "read", "gate", "reset") else v) for k, v in c.items()}
    before = one["state"].clone()
    _, s = selective_scan.step(**one)
    assert torch.equal(one["state"], before) and s.data_ptr() != before.data_ptr()
    fresh, _ = selective_scan.step(**{**one, "state": None})
    zero, _ = selective_scan.step(**{**one, "state": torch.zeros_like(before)})
    assert torch.equal(fresh, zero)
    version = before._version
    selective_scan.step(**{**one, "state": before}, next_state=before)
    assert before._version > version


def test_empty(dev):
    from hipenvs import selective_scan

    c = make(dev, 1, 0, 5, 6, 3, 1)
    leaves = {k: v.requires_grad_() if k in NAMES else v for k, v in c.items()}
    out, final = selective_scan.sequence(**leaves)
    assert out.shape == (0, 5, 6) and final.shape == (0, 6, 3)
    (out.sum() + final.sum()).backward()
    assert all((leaves[k].grad == 0).all() for k in ("rate", "skip", "dt_bias"))
    c = make(dev, 1, 2, 0, 6, 3, 1)
    leaves = {k: v.detach().requires_grad_() if k in NAMES else v for k, v in c.items()}
    out, final = selective_scan.sequence(**leaves)
    assert out.shape == (2, 0, 6) and torch.equal(final, c["state"])
    final.sum().backward()
    assert (leaves["state"].grad == 1).all() and (leaves["rate"].grad == 0).all()
    one = {k: (v[:0, 0] if k in ("x", "dt", "write", "read", "gate", "reset") else v)
           for k, v in make(dev, 1, 2, 1, 6, 3, 1).items()}
    out, s = selective_scan.step(**{**one, "state": torch.zeros(0, 6, 3, device=dev)})
    assert out.shape == (0, 6) and s.shape == (0, 6, 3)


def test_the_same_bits_on_every_run(dev):
    from hipenvs import selective_scan

    for shape in ((300, 40, 130, 16, 1), (1, 2000, 24, 12, 2)):
        c = make(dev, 6, *shape)
        runs = []
        for _ in range(2):
            leaves = {k: v.detach().requires_grad_() if k in NAMES else v for k, v in c.items()}
            out, final = selective_scan.sequence(**leaves)
            runs.append((out, final, *torch.autograd.grad(out.sum() + final.sum(), [leaves[k] for k in NAMES])))
        assert all(torch.equal(a, e) for a, e in zip(*runs))


@pytest.mark.parametrize("shape", [(3, 40, 70, 16, 2), (1, 1000, 24, 12, 1)])
def test_captured_training_and_steps_replay(dev, shape):
    """A graph of forward and backward, and of steps, replayed with new inputs and eager work between."""
    from hipenvs import selective_scan

    given = [make(dev, 20 + 2 * k, *shape) for k in range(4)]
    static = {k: v.clone() if v is not None else None for k, v in given[0].items()}

    def train():
        leaves = {k: v.detach().requires_grad_() if k in NAMES else v for k, v in static.items()}
        out, final = selective_scan.sequence(**leaves)
        grads = torch.autograd.grad((out, final), [leaves[k] for k in NAMES], (static["x"], static["state"]))
        one = {k: (v[:, 0] if k in ("x", "dt", "write", "read", "gate", "reset") else v) for k, v in static.items()}
        return (out.detach(), final.detach(), *grads, *selective_scan.step(**one))

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
        want = train()
        assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_two_streams(dev):
    from hipenvs import selective_scan

    cases = [make(dev, k, 2, 600, 40, 16, 1) for k in range(2)]
    want = [selective_scan.sequence(**c) for c in cases]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in cases]
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            got.append(selective_scan.sequence(**c))
    torch.cuda.synchronize()
    for (a, b), (e, f) in zip(got, want):
        assert torch.equal(a, e) and torch.equal(b, f)


def test_saved_tensors_may_come_back_laid_out_anew(dev):
    from hipenvs import selective_scan

    c = make(dev, 2, 2, 30, 20, 16, 1, layout="time")
    grads = []
    for hooks in (False, True):
        leaves = {k: v.detach().requires_grad_() if k in NAMES else v for k, v in c.items()}
        if hooks:
            with torch.autograd.graph.save_on_cpu():
                out, final = selective_scan.sequence(**leaves)
        else:
            out, final = selective_scan.sequence(**leaves)
        grads.append(torch.autograd.grad(out.sum() + final.sum(), [leaves[k] for k in NAMES]))
    assert all(torch.equal(a, e) for a, e in zip(*grads))


def test_rows_past_32_bit_offsets(dev):
    """2^31 values and more: the last tokens of a long row, after an episode's beginning, are those of
    the short row."""
    from hipenvs import selective_scan

    t, d, last = 33000, 65536, 37
    x = torch.zeros(1, t, d, dtype=BF16, device=dev)
    x[:, -last:] = torch.randn(1, last, d, device=dev).to(BF16)
    mix = torch.randn(1, t, 4, device=dev).to(BF16)
    reset = torch.zeros(1, t, dtype=torch.bool, device=dev)
    reset[0, -last] = True
    rate = -torch.ones(d, 4, device=dev)
    out, final = selective_scan.sequence(x, x, rate, mix, mix, gate=x, reset=reset)
    short, short_final = selective_scan.sequence(*(y[:, -last:] for y in (x, x)), rate, mix[:, -last:], mix[:, -last:],
                                                 gate=x[:, -last:], reset=reset[:, -last:])
    assert torch.equal(out[:, -last:], short) and torch.equal(final, short_final)


def test_refusals(dev):
    from hipenvs import selective_scan

    c = make(dev, 1, 2, 5, 6, 4, 2)

    def refused(error, call=selective_scan.sequence, **changes):
        with pytest.raises(error):
            call(**{**c, **changes})

    refused(TypeError, x=c["x"].half())
    refused(TypeError, x=c["x"].to(BF16))
    refused(TypeError, write=c["write"].to(BF16))
    refused(TypeError, rate=c["rate"].double())
    refused(TypeError, reset=c["reset"].int())
    refused(TypeError, state="zeros")
    refused(ValueError, dt=c["dt"][:, :4])
    refused(ValueError, x=c["x"][0])
    refused(ValueError, rate=c["rate"][:, :3])
    refused(ValueError, rate=c["rate"][:5])
    refused(ValueError, rate=torch.zeros(6, 65, device=dev))
    refused(ValueError, write=torch.zeros(2, 5, 4, 4, device=dev), read=torch.zeros(2, 5, 4, 4, device=dev))
    refused(ValueError, read=c["read"][:, :, :1])
    refused(ValueError, skip=c["skip"][:5])
    refused(ValueError, state=c["state"][:1])
    refused(ValueError, state=c["state"].cpu())
    refused(ValueError, reset=c["reset"][:, :3])
    one = {k: (v[:, 0] if k in ("x", "dt", "write", "read", "gate", "reset") else v) for k, v in c.items()}
    with pytest.raises(ValueError):
        selective_scan.step(**{**one, "x": one["x"].detach().requires_grad_()})
    with pytest.raises(ValueError):
        selective_scan.step(**one, next_state=torch.zeros(2, 4, 6, device=dev).transpose(1, 2))
    out, _ = selective_scan.sequence(**{**c, "x": c["x"].detach().requires_grad_()})
    grad, = torch.autograd.grad(out.sum(), [out.grad_fn.next_functions[0][0].variable], create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(c["x"], torch.ones_like(c["x"]))
        refused(ValueError, x=dual)


@pytest.mark.parametrize("count,d,n,g", [(4099, 256, 16, 2), (3001, 200, 5, 1), (8190, 64, 40, 4)])
def test_steps_of_many_environments(dev, count, d, n, g):
    """Several environments a thread, the last group not whole, against the definition."""
    from hipenvs import selective_scan

    for dtype in (F32, BF16):
        c = make(dev, 2 * g, count, 1, d, n, g, dtype, "fused", 3)
        one = {k: (v[:, 0] if k in ("x", "dt", "write", "read", "gate", "reset") else v) for k, v in c.items()}
        out, state = selective_scan.step(**one)
        f64 = to_np(c)
        want = oss.sequence(**f64)
        size = oss.magnitudes(*f64.values(), np.zeros((count, 1, d)), np.zeros((count, d, n)))
        close(out[:, None], want[0], size[0], dtype, units(1, d, n))
        close(state, want[1], size[1], F32, units(1, d, n))
        again, same = selective_scan.step(**one, next_state=one["state"])
        assert torch.equal(again, out) and torch.equal(same, state)
