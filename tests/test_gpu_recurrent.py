"""The memory policy's learner (GPU): acting step by step and over whole trajectories is one
policy, its gradients are those of float64 autograd, and it learns CartPole without velocities."""

import numpy as np
import pytest
import torch

from oracle import decay_attention as oda

pytestmark = pytest.mark.gpu


def test_acting_and_training_see_one_policy(dev):
    """Logits from acting (states updated in place over 40 steps, episodes ending inside) and from
    the whole trajectory, against the policy in float64: every product of width 32 and the
    attention of 40 steps, at 400 roundings of 2^-24 through two layers whose gains are below 4."""
    from hipenvs import recurrent

    gen = torch.Generator(device=dev)
    gen.manual_seed(3)
    policy = recurrent.Policy(2, 3, 32, 2, 2, gen)
    obs = torch.randn(17, 40, 2, generator=gen, device=dev)
    begins = torch.rand(17, 40, generator=gen, device=dev) < 0.1
    state = policy.initial_state(17)
    acted = torch.stack([policy.act(obs[:, t], state, begins[:, t]) for t in range(40)], 1)
    whole = policy.logits(obs, policy.initial_state(17), begins).detach()

    f64 = [w.detach().double().cpu().numpy() for w in policy.parameters()]
    x = np.tanh(obs.double().cpu().numpy() @ f64[0] + f64[1])
    ld, r = policy.log_decay.double().cpu().numpy(), begins.cpu().numpy()
    for project, mix in ((f64[2], f64[3]), (f64[4], f64[5])):
        q, k, v = np.split((x @ project).reshape(17, 40, 6, 16), 3, axis=2)
        out, _ = oda.sequence(q, k, v, ld, None, r, 0.25)
        x = x + np.tanh(out.reshape(17, 40, 32)) @ mix
    want = x @ f64[6]
    bound = 400 * 2.0 ** -24 * 16 * np.abs(want).max()
    assert np.abs(acted.double().cpu().numpy() - want).max() <= bound
    assert np.abs(whole.double().cpu().numpy() - want).max() <= bound


@pytest.mark.parametrize("bits", [32, 8])
def test_learns_cartpole_from_positions_alone(dev, bits):
    """Episodes last about 25 steps under a random policy; after 60 updates of 512 environments at
    least twice that, with either form of the optimizer's moments."""
    from hipenvs import recurrent

    lasted = []
    cfg = recurrent.Config(envs=512, seed=1, bits=bits)
    learner = recurrent.train(cfg, 60, lambda i, n: lasted.append(n))
    print("steps an episode", [round(x, 1) for x in lasted[::10]], flush=True)
    assert lasted[0] < 40 and np.mean(lasted[-5:]) > 2 * lasted[0]
    assert all(torch.isfinite(p).all() for p in learner.policy.parameters())


def test_learner_refusals(dev):
    from hipenvs import recurrent

    with pytest.raises(ValueError):
        recurrent.Learner(recurrent.Config(task="nothing"))
    with pytest.raises(ValueError):
        recurrent.Learner(recurrent.Config(width=30, heads=4))


def test_discounted_returns_end_with_episodes():
    from hipenvs import recurrent

    reward = torch.ones(1, 4)
    done = torch.tensor([[False, True, False, False]])
    assert recurrent.discounted(reward, done, 0.5).tolist() == [[1.5, 1.0, 1.5, 1.0]]
