"""Infinities where an operator over tokens has left something out (GPU): an episode's first token leaves out the
state and the taps before it, a logit of -inf its token. What is left out owes nothing to an infinite gradient or
decay on the other side, where zero times an infinity would be no number."""

import numpy as np
import pytest
import torch

from oracle import categorical as oca
from oracle import causal_conv as occ
from oracle import selective_scan as oss

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def to_np(x):
    return x.detach().cpu().numpy() if x.dtype == torch.bool else x.detach().double().cpu().numpy()


# n: two to sixteen lanes, with all of their states and without; t: in one part, and in several
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [3, 8, 12, 16, 27, 64])
@pytest.mark.parametrize("t", [40, 900])
def test_scan_infinite_gradient_of_an_episodes_first_token(dev, n, t, dtype):
    """The state before is left out: rate's gradient, and all others but that token's own, are those with a
    gradient of zero there; and the token's own are the definition's."""
    from hipenvs import selective_scan

    gen = torch.Generator().manual_seed(n)
    b, d, at = 2, 40, t // 2 + 3
    reset = torch.zeros(b, t, dtype=torch.bool)
    reset[0, at] = True
    rows = [torch.rand(b, t, w, generator=gen).add(0.1).to(dtype) for w in (d, d, n, n)]
    given = {"x": rows[0], "dt": rows[1], "rate": -torch.rand(d, n, generator=gen) - 0.1, "write": rows[2], "read": rows[3]}
    given = {k: v.to(dev) for k, v in given.items()}
    grads = []
    for first in (0.0, INF):
        dout = torch.ones(b, t, d, dtype=dtype, device=dev)
        dout[0, at, 5] = first
        leaves = {k: v.detach().requires_grad_() for k, v in given.items()}
        out, _ = selective_scan.sequence(**leaves, reset=reset.to(dev))
        grads.append(dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dout))))
    zero, inf = grads
    assert torch.isfinite(inf["rate"]).all() and torch.equal(inf["rate"], zero["rate"])
    for name in ("x", "dt"):
        elsewhere = torch.ones(b, t, d, dtype=torch.bool, device=dev)
        elsewhere[0, at, 5] = False
        assert torch.equal(inf[name][elsewhere], zero[name][elsewhere])
        assert inf[name][0, at, 5] == INF   # x, write, read and the slope of softplus are above zero
    for name in ("write", "read"):
        others = torch.arange(t, device=dev) != at
        assert torch.equal(inf[name][:, others], zero[name][:, others]) and (inf[name][0, at] == INF).all()
    f64 = [to_np(given[k]) for k in ("x", "dt", "rate")] + [to_np(given[k])[:, :, None] for k in ("write", "read")]
    with np.errstate(invalid="ignore"):   # the token's own sums
        want = oss.gradients(*f64, None, None, None, None, to_np(reset), to_np(dout), np.zeros((b, d, n)))
    assert np.isfinite(want[2]).all() and want[1][0, at, 5] == INF


@pytest.mark.parametrize("n", [3, 8, 12, 16, 64])
@pytest.mark.parametrize("t", [40, 900])
def test_scan_infinite_delta_of_an_episode_of_one_token(dev, n, t):
    """Its state is infinite and ends with it: rate's gradient is what it is with a finite delta there."""
    from hipenvs import selective_scan

    gen = torch.Generator().manual_seed(n)
    b, d, at = 1, 40, t // 2 + 3
    reset = torch.zeros(b, t, dtype=torch.bool)
    reset[0, at:at + 2] = True
    x, dt, write, read = (torch.rand(b, t, w, generator=gen).add(0.1) for w in (d, d, n, n))
    rate = -torch.rand(d, n, generator=gen) - 0.1
    drates = []
    for first in (0.5, INF):
        dt[0, at, 5] = first
        leaf = rate.to(dev).requires_grad_()
        out, _ = selective_scan.sequence(x.to(dev), dt.to(dev), leaf, write.to(dev), read.to(dev), reset=reset.to(dev))
        drates.append(torch.autograd.grad(out, leaf, torch.ones_like(out))[0])
    assert torch.isfinite(drates[1]).all() and torch.equal(*drates)
    with np.errstate(invalid="ignore"):   # a gate of one at an infinite output
        want = oss.gradients(*(to_np(y) for y in (x, dt, rate)), to_np(write)[:, :, None], to_np(read)[:, :, None], None,
                             None, None, None, to_np(reset), np.ones((b, t, d)), np.zeros((b, d, n)))
    assert np.isfinite(want[2]).all()


@pytest.mark.parametrize("n", [3, 8, 12, 16, 64])
@pytest.mark.parametrize("t", [40, 900])
def test_scan_infinite_decay_at_an_episodes_first_token(dev, n, t):
    """A rate above zero and a large delta: the decay of an episode's first token is infinite, and meets no state."""
    from hipenvs import selective_scan

    b, d, at = 2, 6, t // 2 + 3
    x, dt, mix = torch.ones(b, t, d), torch.full((b, t, d), -30.0), torch.ones(b, t, n)
    dt[:, at, 1] = 200.0
    reset = torch.zeros(b, t, dtype=torch.bool)
    reset[:, at] = True
    rate, state = torch.ones(d, n), torch.ones(b, d, n)
    given = [y.to(dev) for y in (x, dt, rate, mix, mix)]
    out, final = selective_scan.sequence(*given, state=state.to(dev), reset=reset.to(dev))
    f64 = {k: to_np(y) for k, y in (("x", x), ("dt", dt), ("rate", rate), ("state", state), ("reset", reset))}
    want = oss.sequence(**f64, write=to_np(mix)[:, :, None], read=to_np(mix)[:, :, None])
    # all terms are above zero. A state sums at most t of them and meets t decays, each within two units of
    # 2^-24 (their exponents are below 1e-12); delta is within 8 units and its product; an output sums n states
    assert np.isfinite(want[0]).all()
    assert np.all(np.abs(to_np(out) - want[0]) <= (3 * t + n + 16) * 2.0 ** -24 * np.abs(want[0]))
    assert np.all(np.abs(to_np(final) - want[1]) <= (3 * t + n + 16) * 2.0 ** -24 * np.abs(want[1]))
    one = [y[:, at].contiguous() if y.dim() == 3 else y for y in given]
    o, s = selective_scan.step(*one, state=state.to(dev), reset=torch.ones(b, dtype=torch.bool, device=dev))
    assert torch.isfinite(s).all()
    assert ((o - out[:, at]).abs() <= 2 * (n + 16) * 2.0 ** -24 * out[:, at]).all()   # the same sums, in either order


@pytest.mark.parametrize("n", [3, 16])
@pytest.mark.parametrize("t", [40, 900])
def test_scan_infinite_rates(dev, n, t):
    """A rate of -inf keeps nothing of the state before, and all of it where delta is zero; walked whole, in parts
    and step by step."""
    from hipenvs import selective_scan

    b, d = 1, 4
    x, mix, state = torch.ones(b, t, d, device=dev), torch.ones(b, t, n, device=dev), torch.full((b, d, n), 2.0, device=dev)
    rate = torch.full((d, n), -INF, device=dev)
    reset = torch.zeros(b, t, dtype=torch.bool, device=dev)
    reset[0, t // 2] = True
    for value, want in ((-300.0, 0.0), (3.0, float(np.log1p(np.exp(3.0))))):
        dt = torch.full((b, t, d), value, device=dev)
        kept = value < 0
        for begins in (None, reset):
            out, final = selective_scan.sequence(x, dt, rate, mix, mix, state=state, reset=begins)
            last = state if kept and begins is None else torch.full_like(state, want)
            # one token's delta, within 8 units of 2^-24, and its product; sums of n of them
            assert ((final - last).abs() <= 9 * 2.0 ** -24 * last).all()
            held = state.clone()
            for i in range(t):
                o, _ = selective_scan.step(x[:, i], dt[:, i], rate, mix[:, i], mix[:, i], state=held,
                                           reset=None if begins is None else begins[:, i], next_state=held)
                assert ((o - out[:, i]).abs() <= 2 * n * 2.0 ** -24 * out[:, i]).all()
            assert torch.equal(held, final)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("w", [2, 3, 4])
def test_conv_infinite_gradient_next_to_an_episodes_first_tokens(dev, w, dtype):
    """Every place of an episode's beginning and of an infinite gradient just behind it: the weights of the taps
    that are left out have the gradient that they have without it."""
    from hipenvs import causal_conv

    gen = torch.Generator().manual_seed(w)
    b, t, d = 1, 70, 6
    x = torch.rand(b, t, d, generator=gen).add(0.1).to(dtype).to(dev)
    weight = torch.rand(d, w, generator=gen).add(0.1).to(dev)
    for begin in (0, 1, 5, 7, 8, 15, 16, 30, 31, 32, 62, 63, 64, 66):
        reset = torch.zeros(b, t, dtype=torch.bool, device=dev)
        reset[0, begin] = True
        for behind in range(w - 1):
            grads = []
            for value in (0.0, INF):
                dout = torch.ones(b, t, d, dtype=dtype, device=dev)
                dout[0, begin + behind, 2] = value
                leaf = weight.detach().requires_grad_()
                out, _ = causal_conv.sequence(x, leaf, reset=reset, silu=False)
                grads.append(torch.autograd.grad(out, leaf, dout)[0])
            zero, inf = grads
            hit = torch.zeros(d, w, dtype=torch.bool, device=dev)
            hit[2, w - 1 - behind:] = True   # the taps within the episode
            assert torch.equal(inf[~hit], zero[~hit]), (begin, behind)
            assert (inf[hit] == INF).all(), (begin, behind)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [2, 3, 7, 16, 30, 64, 100, 200, 500, 1000, 1024, 1025, 5000])
def test_log_probs_infinite_gradients_leave_masked_tokens_at_zero(dev, v, dtype):
    """Tokens that are not allowed, in rows with others and in rows of nothing else."""
    from hipenvs import categorical

    gen = torch.Generator().manual_seed(v)
    x = torch.randn(6, v, generator=gen).to(dtype)
    x[:, ::2] = -INF
    x[2:4] = -INF
    tokens = torch.tensor([1, 1, 1, -1, 1, 1])
    leaf = x.to(dev).requires_grad_()
    log_prob, entropy = categorical.log_probs(leaf, tokens.to(dev))
    for given in ((INF, 1.0), (1.0, INF), (-INF, -INF), (float("nan"), 1.0)):
        dlog_prob, dentropy = (torch.full((6,), y, device=dev) for y in given)
        grad, = torch.autograd.grad((log_prob, entropy), leaf, (dlog_prob, dentropy), retain_graph=True)
        assert (grad[:, ::2] == 0).all() and (grad[2:4] == 0).all()
    # finite ones: a p is within 32 units of 2^-24 of itself (its exponent is below 20), the bracket below
    # 1 + 2 log 5000 < 19 within 64 of its size: below 1e-5
    grad, = torch.autograd.grad((log_prob, entropy), leaf, (torch.ones(6, device=dev), torch.ones(6, device=dev)))
    want = oca.gradient(x.double().numpy(), tokens.numpy(), np.ones(6), np.ones(6))
    off = np.abs(to_np(grad) - want)
    assert off.max() <= 1e-5 + (2.0 ** -8 if dtype == BF16 else 0.0) * np.abs(want).max()


def test_rows_of_tokens_far_apart(dev):
    """Tokens 2^31 values apart, whose offsets from each other do not fit 32 bits: as they are for the
    convolution, copied for the scan, in every input and in the gradient that comes back."""
    from hipenvs import causal_conv, selective_scan

    gen = torch.Generator().manual_seed(1)
    d, n, t, far = 24, 4, 3, (1 << 31) + 7
    whole = torch.empty((t - 1) * far + 6 * d, dtype=BF16, device=dev)
    marks = torch.zeros((t - 1) * far + 2, dtype=torch.bool, device=dev)

    def apart(values, at):
        y = whole.as_strided((1, t, values.shape[-1]), (1, far, 1), at)
        y.copy_(values)
        return y

    x, dt, gate, mix, dout = (torch.randn(1, t, w, generator=gen).to(BF16).to(dev) for w in (d, d, d, 2 * n, d))
    reset = torch.tensor([[False, False, True]], device=dev)
    begins = marks.as_strided((1, t), (1, far), 1)
    begins.copy_(reset)
    spread = [apart(y, k * d) for k, y in enumerate((x, dt, gate, mix[..., :n], mix[..., n:], dout))]
    rate, weight = -torch.ones(d, n, device=dev), torch.randn(d, 4, generator=gen).to(dev)
    near = (x, dt, gate, mix[..., :n].contiguous(), mix[..., n:].contiguous(), dout)
    results = []
    for given, r in ((near, reset), (spread, begins)):
        a, b, c, w, o = (y.detach().requires_grad_() for y in given[:5])
        out, final = selective_scan.sequence(a, b, rate, w, o, gate=c, reset=r)
        conv, held = causal_conv.sequence(a, weight, reset=r)
        grads = torch.autograd.grad((out, conv), (a, b, c, w, o), (given[5], given[5]))
        results.append((out.detach(), final.detach(), conv.detach(), held.detach(), *grads))
    assert all(torch.equal(a, e) for a, e in zip(*results))


def test_rows_of_one_token_far_apart(dev):
    """A row of one token has no next one: its stride of t may be anything."""
    from hipenvs import selective_scan

    gen = torch.Generator().manual_seed(1)
    d, n, far = 10, 4, 1 << 33
    x, dt, gate = (torch.randn(2, 1, d, generator=gen).to(dev) for _ in range(3))
    write, read = (torch.randn(2, 1, 1, n, generator=gen).to(dev) for _ in range(2))
    reset = torch.ones(2, 1, dtype=torch.bool, device=dev)
    rate = -torch.ones(d, n, device=dev)
    results = []
    for apart in (False, True):
        leaves = [y.detach().clone() for y in (x, dt, write, read, gate)]
        begins, dout = reset, torch.ones(2, 1, d, device=dev)
        if apart:
            leaves = [y.as_strided(y.shape, (y.stride(0), far, *y.stride()[2:])) for y in leaves]
            begins, dout = (y.as_strided(y.shape, (y.stride(0), far, *y.stride()[2:])) for y in (begins, dout))
        leaves = [y.requires_grad_() for y in leaves]
        out, final = selective_scan.sequence(leaves[0], leaves[1], rate, leaves[2], leaves[3], gate=leaves[4], reset=begins)
        results.append((out.detach(), final.detach(), *torch.autograd.grad(out, leaves, dout)))
    assert all(torch.equal(a, e) for a, e in zip(*results))
