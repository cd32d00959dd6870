"""What the lookup's backward pass refuses before any launch (CPU)."""

from types import SimpleNamespace

import pytest
import torch


def test_lookup_refuses_saved_tokens_of_another_shape():
    """Hooks on saved tensors may hand back others: as many rows are read of the gradient as there are tokens,
    so more of them would be read past its end."""
    from hipenvs import embedding

    here = SimpleNamespace(index=torch.zeros(1).get_device())   # a tensor of the host passes for one of this device
    dout = torch.zeros(3, 2, 5)
    for tokens in (torch.zeros(3, 3, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int64),
                   torch.zeros(7, dtype=torch.int32), torch.zeros(0, dtype=torch.int64)):
        ctx = SimpleNamespace(saved_tensors=(tokens,), ready=(torch.float32, (4, 5), (3, 2), here, 1.0))
        with pytest.raises(ValueError, match="shape"):
            embedding._backward(ctx, dout)


@pytest.mark.parametrize("clip", [-0.1, -2.0, float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("epochs", [1, 2])
def test_learner_refuses_a_clip_whose_bounds_cross(clip, epochs):
    """clamp(1 - clip, 1 + clip) of a clip below zero is a constant, without a gradient."""
    from hipenvs import recurrent

    with pytest.raises(ValueError, match="clip"):
        recurrent.Learner(recurrent.Config(clip=clip, epochs=epochs))


def test_policy_refuses_an_unknown_memory():
    """It would be given decay attention."""
    from hipenvs import recurrent

    for memory in ("scam", None, "Scan"):
        with pytest.raises(ValueError, match="memory"):
            recurrent.Policy(2, 3, 8, 2, 1, torch.Generator(), memory=memory)
    for memory, count in (("decay", 5), ("scan", 11)):
        assert len(recurrent.Policy(2, 3, 8, 2, 1, torch.Generator(), memory=memory, states=4).parameters()) == count
