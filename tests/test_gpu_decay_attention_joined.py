"""Rows walked in parts (GPU): a part's decay, lambda^n over all its tokens, may underflow or overflow
where no token's does. What the definition holds on to is held on to: an infinity under decay, a
zero under growth."""

import numpy as np
import pytest
import torch

from oracle import decay_attention as oda
from test_gpu_decay_attention import BF16, F32, gamma

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("t", [300, 6000])
def test_an_infinite_state_stays_under_any_decay(dev, t, dtype):
    """e^-1 and e^-0.05 a token; the columns without the infinity are the definition's, the one with it
    is infinite at every token (its queries are positive), until the second row's reset."""
    from hipenvs import decay_attention

    b, h, dk, dv = 2, 2, 8, 4
    gen = torch.Generator().manual_seed(70)
    q = (torch.rand(b, t, h, dk, generator=gen) + 0.5).to(dtype)
    k, v = (torch.randn(b, t, h, d, generator=gen).to(dtype) for d in (dk, dv))
    log_decay = torch.tensor([-1.0, -0.05])
    state = torch.randn(b, h, dk, dv, generator=gen)
    state[:, :, 3, 2] = float("inf")
    reset = torch.zeros(b, t, dtype=torch.bool)
    reset[1, t // 2] = True
    out, final = decay_attention.sequence(*(x.to(dev) for x in (q, k, v, log_decay, state, reset)))
    infinite = torch.zeros(b, t, h, dv, dtype=torch.bool)
    infinite[0, :, :, 2] = infinite[1, :t // 2, :, 2] = True
    assert torch.equal(torch.isposinf(out.cpu().float()), infinite)
    stays = torch.zeros(b, h, dk, dv, dtype=torch.bool)
    stays[0, :, 3, 2] = True
    assert torch.equal(torch.isposinf(final.cpu()), stays)

    state[:, :, 3, 2] = 0.0
    args = [x.double().numpy() if x.dtype != torch.bool else x.numpy() for x in (q, k, v, log_decay, state, reset)]
    want, size = oda.sequence(*args, dk ** -0.5), oda.magnitudes(*args, dk ** -0.5)
    for x, w, s, left in ((out, want[0], size[0], ~infinite), (final, want[1], size[1], ~stays)):
        bound = gamma(t, dk, dv) * s + (2.0 ** -8 * np.abs(w) * (1 + 2.0 ** -6) if x.dtype == BF16 else 0.0)
        x, left = x.cpu().double().numpy(), left.numpy()
        assert np.all(np.abs(x - w)[left] <= bound[left] + 1e-37)


@pytest.mark.parametrize("backwards", [False, True])
def test_zeros_stay_under_any_growth(dev, backwards):
    """Growth by e^0.2 a token over 6,000 tokens of which the last 90 (for gradients, the first 90)
    hold anything: e^18 at the most."""
    from hipenvs import decay_attention

    b, t, h, dk, dv = 1, 6000, 1, 8, 4
    gen = torch.Generator().manual_seed(71)
    q, k, v = (torch.randn(b, t, h, d, generator=gen) for d in (dk, dk, dv))
    dout = torch.randn(b, t, h, dv, generator=gen)
    if backwards:
        q[:, 90:] = dout[:, 90:] = k[:, 90:] = 0.0
        v[:, 90:] = 0.0
        reset = torch.zeros(b, t, dtype=torch.bool)
        reset[:, 90] = True   # the states end here, as no growth of theirs is meant
    else:
        k[:, :-90] = 0.0
        dout[:] = 0.0
        reset = None
    log_decay = torch.tensor([0.2])
    leaves = [x.to(dev).requires_grad_() for x in (q, k, v)]
    out, final = decay_attention.sequence(*leaves, log_decay.to(dev), None, None if reset is None else reset.to(dev), 0.5)
    grads = torch.autograd.grad(out, leaves, dout.to(dev))
    args = [x.double().numpy() for x in (q, k, v, log_decay)] + [None, None if reset is None else reset.numpy(), 0.5]
    want = (*oda.sequence(*args), *oda.gradients(*args, dout.double().numpy(), None))
    size = oda.magnitudes(*args, dout.double().numpy(), None)
    for x, w, s in zip((out, final, *grads), want, size):
        assert np.all(np.abs(x.detach().cpu().double().numpy() - w) <= gamma(t, dk, dv) * s + 1e-37)
