"""The learner with a selective scan, the action before and clipped ratios (GPU): the operators together
as they are used. Acting step by step and over whole trajectories is one policy, its loss has the
gradients of float64 autograd over the definitions, and an update waits for nothing."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def make_policy(dev, seed=3, width=32, layers=2, actions=3):
    from hipenvs import recurrent

    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    return recurrent.Policy(2, actions, width, 2, layers, gen, memory="scan", states=6, previous_action=True), gen


def f64_logits(policy, weights, obs, previous, begins):
    """The policy's logits from the definitions in float64, token by token, differentiable in `weights`."""
    encoder, bias, *rest = weights
    table, head = rest.pop(), rest.pop()
    there = (previous >= 0)[..., None]
    x = torch.tanh(obs @ encoder + bias + torch.where(there, table[previous.clamp(min=0)], 0.0))
    n, t, width = x.shape
    for i in range(len(policy.blocks)):
        project, weight, cbias, choose, log_rate, skip, dt_bias, mix = rest[8 * i:8 * i + 8]
        u, gate = (x @ project).chunk(2, -1)
        hist, outs = torch.zeros(n, 3, width, dtype=x.dtype), []
        h = torch.zeros(n, width, log_rate.shape[1], dtype=x.dtype)
        for j in range(t):
            fresh = begins[:, j, None, None]
            window = torch.cat([torch.where(fresh, 0.0, hist), u[:, j:j + 1]], 1)
            hist = window[:, 1:]
            pre = (window * weight.t()).sum(1) + cbias
            c = pre * torch.sigmoid(pre)
            dt, write, read = torch.split(c @ choose, (width, log_rate.shape[1], log_rate.shape[1]), -1)
            delta = torch.nn.functional.softplus(dt + dt_bias)
            keep = torch.exp(delta[..., None] * -torch.exp(log_rate))
            h = torch.where(fresh, 0.0, keep * h) + (delta * c)[..., None] * write[:, None]
            y = (h * read[:, None]).sum(-1) + skip * c
            outs.append(y * gate[:, j] * torch.sigmoid(gate[:, j]))
        x = x + torch.stack(outs, 1) @ mix
    return x @ head


def inputs(dev, gen, n, t, actions=3):
    obs = torch.randn(n, t, 2, generator=gen, device=dev)
    begins = torch.rand(n, t, generator=gen, device=dev) < 0.1
    action = torch.randint(0, actions, (n, t), generator=gen, device=dev)
    previous = torch.where(begins, -1, torch.roll(action, 1, 1))
    previous[:, 0] = -1
    return obs, begins, action, previous


def test_acting_and_training_see_one_policy(dev):
    """Within 4,000 roundings of 2^-24 of the largest logit: two layers of products of width 32, 4 taps and
    states of 40 steps, whose gains multiply to below 8 and whose softplus and decays take 104 units more
    for each (the scan's own bound)."""
    policy, gen = make_policy(dev)
    obs, begins, _, previous = inputs(dev, gen, 17, 40)
    state = policy.initial_state(17)
    acted = torch.stack([policy.act(obs[:, t], state, begins[:, t], previous[:, t]) for t in range(40)], 1)
    whole = policy.logits(obs, policy.initial_state(17), begins, previous).detach()
    weights = [w.detach().double().cpu() for w in policy.parameters()]
    want = f64_logits(policy, weights, obs.double().cpu(), previous.cpu(), begins.cpu())
    bound = 4000 * 2.0 ** -24 * want.abs().max()
    assert (acted.double().cpu() - want).abs().max() <= bound
    assert (whole.double().cpu() - want).abs().max() <= bound


def test_gradients_of_the_clipped_loss(dev):
    """The learner's loss with clip and entropy against float64 autograd over the definitions, each gradient
    within 2^-12 of its own norm: some 10,000 roundings of sums over 12 x 30 tokens, against a wrong
    term's order of one."""
    from hipenvs import recurrent

    policy, gen = make_policy(dev, 5)
    obs, begins, action, previous = inputs(dev, gen, 12, 30)
    advantage = torch.randn(12, 30, generator=gen, device=dev)
    learner = recurrent.Learner.__new__(recurrent.Learner)
    learner.cfg, learner.policy = recurrent.Config(clip=0.2, epochs=2, entropy=0.05), policy
    before = policy.initial_state(12)
    acted = torch.log_softmax(policy.logits(obs, before, begins, previous), -1).gather(-1, action[..., None])[..., 0].detach()
    acted = acted + 0.3 * torch.randn(12, 30, generator=gen, device=dev)   # some ratios are clipped
    batch = (obs, begins, action, None, None, previous, acted)
    params = policy.parameters()
    got = torch.autograd.grad(learner._loss(batch, before, advantage), params)

    weights = [w.detach().double().cpu().requires_grad_() for w in params]
    logits = f64_logits(policy, weights, obs.double().cpu(), previous.cpu(), begins.cpu())
    log_p = torch.log_softmax(logits, -1)
    chosen = log_p.gather(-1, action.cpu()[..., None])[..., 0]
    entropy = -(log_p.exp() * log_p).sum(-1)
    ratio = torch.exp(chosen - acted.double().cpu())
    a = advantage.double().cpu()
    gain = torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
    # no ratio next to its border, where the two would take different sides
    assert ((ratio.detach() - 0.8).abs() > 1e-4).all() and ((ratio.detach() - 1.2).abs() > 1e-4).all()
    want = torch.autograd.grad(-(gain + 0.05 * entropy).mean(), weights)
    for g, w in zip(got, want):
        assert (g.double().cpu() - w).norm() <= 2.0 ** -12 * w.norm() + 1e-12


CONFIGS = [dict(memory="scan"), dict(memory="scan", previous_action=True, clip=0.2, epochs=3, entropy=0.01, layers=2),
           dict(previous_action=True), dict(clip=0.1), dict(entropy=0.01, bits=8), dict(memory="scan", width=30, states=5)]


@pytest.mark.parametrize("config", CONFIGS)
def test_an_update_runs_and_waits_for_nothing(dev, config):
    """torch raises at every call that would wait, an upload from pageable memory among them."""
    from hipenvs import recurrent

    learner = recurrent.Learner(recurrent.Config(task="acrobot", envs=64, horizon=8, **config))
    learner.update()   # what is made once, is made
    torch.cuda.synchronize()
    start = [p.detach().clone() for p in learner.policy.parameters()]
    torch.cuda.set_sync_debug_mode("error")
    try:
        lasted = learner.update()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.isfinite(lasted) and lasted >= 1
    params = learner.policy.parameters()
    assert all(torch.isfinite(p).all() for p in params) and all(not torch.equal(a, b) for a, b in zip(start, params))


def test_the_first_ratio_is_one(dev):
    """The log probabilities kept while acting are those that training finds before it moves the policy."""
    from hipenvs import recurrent, categorical

    learner = recurrent.Learner(recurrent.Config(envs=128, horizon=32, memory="scan", previous_action=True, clip=0.2))
    learner.update()
    (obs, begins, action, _, _, previous, acted), before = learner._collect()
    assert (previous[:, 1:][begins[:, 1:]] == -1).all() and (previous >= -1).all()
    kept = ~begins[:, 1:]
    assert torch.equal(previous[:, 1:][kept], action[:, :-1][kept])
    now, _ = categorical.log_probs(learner.policy.logits(obs, before, begins, previous), action)
    assert (now - acted).abs().max() < 1e-4


def test_command_line_runs(dev, capsys):
    from hipenvs import recurrent

    learner = recurrent.main(["--envs", "64", "--horizon", "8", "--updates", "2", "--memory", "scan", "--states", "4",
                              "--previous-action", "--clip", "0.2", "--epochs", "2", "--entropy", "0.01"])
    assert capsys.readouterr().out.count("update") == 2 and learner.cfg.memory == "scan"


def test_refusals(dev):
    from hipenvs import recurrent

    for bad in (dict(memory="none"), dict(epochs=2), dict(epochs=0, clip=0.1), dict(width=30, heads=4)):
        with pytest.raises(ValueError):
            recurrent.Learner(recurrent.Config(envs=8, **bad))
