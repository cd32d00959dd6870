"""One update of the memory policy's learner (GPU) runs without the host waiting for the device."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("task", ["cartpole", "acrobot"])
def test_an_update_waits_for_nothing(dev, task):
    """torch raises at every call that would wait, an upload from pageable memory among them."""
    from hipenvs import recurrent

    learner = recurrent.Learner(recurrent.Config(task=task, envs=64, horizon=8))
    learner.update()   # what is made once, is made
    torch.cuda.synchronize()
    seen = learner.env.state[list(recurrent.TASKS[task][1])].T.clone()
    torch.cuda.set_sync_debug_mode("error")
    try:
        (obs, *_), _ = learner.collect()
        lasted = learner.update()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(obs[:, 0], seen)
    assert torch.isfinite(lasted) and lasted >= 1
