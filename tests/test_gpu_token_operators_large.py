"""Gradients of the scan and the convolution past 2^31 values (GPU): the last tokens of the last row, behind an
episode's beginning, have those that they have by themselves, and the zeros before them zeros. 1,024 blocks of channels, so
that the scan's sums over blocks lie past 2^31 bytes too."""

import numpy as np
import pytest
import torch

from oracle import selective_scan as oss

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
B, T, D, LAST = 2, 16500, 65536, 37


def late(dev, gen, width, dtype=BF16):
    """Values above zero in the last tokens of the last row, zeros before."""
    x = torch.zeros(B, T, width, dtype=dtype, device=dev)
    x[-1, -LAST:] = torch.rand(LAST, width, generator=gen, device=dev).add(0.1).to(dtype)
    return x


def end(x):
    return x[-1:, -LAST:]


@pytest.fixture()
def given(dev):
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    reset = torch.zeros(B, T, dtype=torch.bool, device=dev)
    reset[-1, -LAST] = True
    return gen, late(dev, gen, D), late(dev, gen, D), reset


def test_scan(dev, given):
    """Against the definition in float64, within the bounds of the scan's own tests; the short row's bits differ, as
    a tile's states are computed again from those before it, and its tiles begin at other tokens."""
    from hipenvs import selective_scan

    gen, x, dout, reset = given
    mix = torch.rand(B, T, 8, generator=gen, device=dev).to(BF16)
    rate = -torch.rand(D, 4, generator=gen, device=dev)
    leaves = [y.detach().requires_grad_() for y in (x, x, rate, mix[..., :4], mix[..., 4:], x)]
    out, _ = selective_scan.sequence(*leaves[:5], gate=leaves[5], reset=reset)
    got = torch.autograd.grad(out, leaves, dout)
    a, r, w, o = (y.detach().double().cpu().numpy() for y in (end(x), rate, end(mix)[..., None, :4], end(mix)[..., None, 4:]))
    f64 = (a, a, r, w, o, None, a, None, None, end(reset[..., None])[..., 0].cpu().numpy(), end(dout).double().cpu().numpy(),
           np.zeros((1, D, 4)))
    want, size = oss.gradients(*f64), oss.magnitudes(*f64)[2:]
    # sums over tokens and states, and over channels where write and read are shared
    for g, k, over in zip(got, (0, 1, 2, 3, 4, 6), (4, 4, LAST, D, D, 4)):
        e, bound = want[k], 4 * 2.0 ** -24 * (5 * LAST + 12 * 104 + over + 64) * size[k]
        if g.dtype == BF16:
            assert not g[:-1].any() and not g[-1, :-LAST].any()
            bound, g = bound + 2.0 ** -8 * (np.abs(e) + bound), end(g)
        off = np.abs(g.double().cpu().numpy().reshape(e.shape) - e) - bound
        assert off.max() <= 0 and e.any(), (k, off.max())


def test_conv(dev, given):
    from hipenvs import causal_conv

    gen, x, dout, reset = given
    weight = torch.rand(D, 4, generator=gen, device=dev) + 0.1
    grads = []
    for of in (lambda y: y, end):
        leaves = [of(x).detach().requires_grad_(), weight.detach().requires_grad_()]
        out, _ = causal_conv.sequence(*leaves, reset=of(reset), silu=False)
        grads.append(torch.autograd.grad(out, leaves, of(dout)))
    whole, short = grads
    assert torch.equal(end(whole[0]), short[0]) and not whole[0][:-1].any() and not whole[0][-1, :-LAST].any()
    # sums of LAST terms above zero, in runs of their own: a rounding a term on both sides
    assert ((whole[1] - short[1]).abs() <= 2 * (LAST + 1) * 2.0 ** -24 * short[1]).all() and (short[1] > 0).all()
