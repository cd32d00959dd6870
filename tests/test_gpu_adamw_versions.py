"""What AdamW (GPU) tells autograd: parameters and moments that a step changed are changed in place,
those it left alone are not."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_only_what_changes_counts_as_changed(dev, bits):
    from hipenvs import adamw

    gen = torch.Generator(device=dev)
    gen.manual_seed(4)
    w = [torch.randn(300, generator=gen, device=dev).requires_grad_() for _ in range(3)]
    g = torch.randn(300, generator=gen, device=dev)
    moments = adamw.init(w, bits)
    held = [(x * x).sum() for x in w]   # each keeps its tensor for its gradient
    before = [x.detach().clone() for x in w]

    adamw.step(w, [None, None, None], moments, 1)
    assert [x._version for x in (*w, *moments)] == [0] * (3 + len(moments))
    adamw.step(w, [None, g, None], moments, 1)
    assert [x._version for x in w] == [0, 1, 0] and [x._version for x in moments] == [1] * len(moments)
    assert torch.equal(w[0], before[0]) and torch.equal(w[2], before[2]) and not torch.equal(w[1], before[1])
    for i in (0, 2):
        assert torch.equal(torch.autograd.grad(held[i], w[i])[0], 2 * before[i])
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(held[1], w[1])

    optimizer = adamw.AdamW(w, bits=bits)
    again = [(x * x).sum() for x in w]
    optimizer.step([None, None, g])
    assert torch.equal(torch.autograd.grad(again[0], w[0])[0], 2 * w[0].detach())
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(again[2], w[2])
