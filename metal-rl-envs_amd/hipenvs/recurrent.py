"""A policy with a memory, trained by policy gradients on device-resident environments: the
operators of ``decay_attention`` and ``adamw`` as a learner uses them. The reference's gradient
learners (``ppo.py:84-95`` for the environment they step) see the whole state and keep no
memory; here some of the state can be hidden, and the policy has to remember.

``Policy`` acts one step at a time (``act``: ``decay_attention.step``, its state the whole
memory) and is evaluated over whole trajectories with gradients (``logits``:
``decay_attention.sequence``), episodes ending inside them. ``Learner`` collects `horizon`
steps of every environment, takes the gradient of the discounted returns' advantage over
their mean (REINFORCE), and steps ``adamw.AdamW``. Nothing in an update reads the device from the
host.

    python -m hipenvs.recurrent --envs 1024 --updates 100
"""

import argparse
import math
from dataclasses import dataclass

import torch

from . import _lib, acrobot, adamw, adapter, cartpole, decay_attention

# body, the rows of its state that the policy sees, actions. The angles and positions alone:
# velocities have to be inferred from the steps before.
TASKS = {"cartpole": (cartpole, (0, 2), 2), "acrobot": (acrobot, (0, 1), 3)}


@dataclass(frozen=True)
class Config:
    task: str = "cartpole"
    envs: int = 1024
    horizon: int = 64
    width: int = 64
    heads: int = 4
    layers: int = 1
    gamma: float = 0.99
    lr: float = 3e-3
    weight_decay: float = 0.0
    bits: int = 32          # of the optimizer's moments
    seed: int = 0


class Policy:
    """An encoder, ``layers`` blocks of decay attention, a head of logits; float32."""

    def __init__(self, obs_dim, actions, width, heads, layers, generator):
        if width % heads:
            raise ValueError(f"width {width} must be a multiple of heads {heads}")
        device = generator.device

        def normal(rows, columns, gain=1.0):
            x = torch.randn(rows, columns, generator=generator, device=device) * (gain / math.sqrt(rows))
            return x.requires_grad_()

        self.heads, self.width = heads, width
        self.encoder = normal(obs_dim, width)
        self.bias = torch.zeros(width, device=device, requires_grad=True)
        self.blocks = [(normal(width, 3 * width), normal(width, width, 0.5)) for _ in range(layers)]
        self.head = normal(width, actions, 0.1)
        # memories of 2, 4, 8, ... steps
        self.log_decay = torch.log1p(-(2.0 ** -torch.arange(1.0, heads + 1.0, device=device)))

    def parameters(self):
        return [self.encoder, self.bias, *(w for block in self.blocks for w in block), self.head]

    def initial_state(self, n):
        d = self.width // self.heads
        return [torch.zeros(n, self.heads, d, d, device=self.head.device) for _ in self.blocks]

    def _through(self, obs, attend):
        """The logits of observations (..., obs_dim); attend(layer, q, k, v) -> outputs like v."""
        x = torch.tanh(obs @ self.encoder + self.bias)
        for i, (project, mix) in enumerate(self.blocks):
            q, k, v = ((x @ project).unflatten(-1, (3 * self.heads, -1))).chunk(3, dim=-2)
            x = x + torch.tanh(attend(i, q, k, v).flatten(-2)) @ mix
        return x @ self.head

    @torch.no_grad()
    def act(self, obs, state, reset):
        """Logits (n, actions) for obs (n, obs_dim); state, the list of initial_state, is updated in
        place. reset (n,) bool: this observation is an episode's first."""
        return self._through(obs, lambda i, q, k, v: decay_attention.step(
            q, k, v, self.log_decay, state[i], reset, next_state=state[i])[0])

    def logits(self, obs, state, reset):
        """Logits (n, t, actions) for trajectories obs (n, t, obs_dim) from the states before them."""
        return self._through(obs, lambda i, q, k, v: decay_attention.sequence(
            q, k, v, self.log_decay, state[i], reset)[0])


def discounted(reward, done, gamma):
    """Returns (n, t) to the end of each episode or of the trajectory."""
    total, out = torch.zeros_like(reward[:, 0]), torch.empty_like(reward)
    for t in reversed(range(reward.shape[1])):
        total = reward[:, t] + gamma * torch.where(done[:, t], 0.0, total)
        out[:, t] = total
    return out


class Learner:
    def __init__(self, cfg, device=None):
        if cfg.task not in TASKS:
            raise ValueError(f"task must be one of {sorted(TASKS)}, got {cfg.task}")
        self.cfg = cfg
        device = torch.device(device) if device is not None else _lib.default_device()
        body, seen, actions = TASKS[cfg.task]
        self.seen = torch.tensor(seen, device=device)   # a list would be uploaded, and waited for, at every step
        body.reseed(cfg.seed)
        self.env = adapter.DeviceEnv(body, cfg.envs, seed=cfg.seed + 1, device=device)
        self.generator = torch.Generator(device=device)
        self.generator.manual_seed(cfg.seed)
        self.policy = Policy(len(seen), actions, cfg.width, cfg.heads, cfg.layers, self.generator)
        self.optimizer = adamw.AdamW(self.policy.parameters(), lr=cfg.lr, weight_decay=cfg.weight_decay, bits=cfg.bits)
        self.memory = self.policy.initial_state(cfg.envs)
        self.begins = torch.ones(cfg.envs, dtype=torch.bool, device=device)

    def collect(self):
        """One trajectory of every environment: (obs, begins, action, reward, done), each (envs,
        horizon, ...), collected time-major; and the memory before it."""
        before = [s.clone() for s in self.memory]
        steps = []
        for _ in range(self.cfg.horizon):
            obs = self.env.obs().index_select(1, self.seen)
            logits = self.policy.act(obs, self.memory, self.begins)
            noise = torch.rand(logits.shape, generator=self.generator, device=logits.device)
            action = (logits - torch.log(-torch.log(noise.clamp(1e-12, 1 - 1e-7)))).argmax(-1)   # Gumbel's maximum
            begins = self.begins
            reward, self.begins = self.env.step(action.to(torch.int32))
            steps.append((obs, begins, action, reward, self.begins))
        return tuple(torch.stack(x).transpose(0, 1) for x in zip(*steps)), before

    def update(self):
        """Collects, and moves the policy once; the steps an episode lasted on average (a device
        scalar: environment steps over episodes that ended)."""
        (obs, begins, action, reward, done), before = self.collect()
        returns = discounted(reward, done, self.cfg.gamma)
        advantage = returns - returns.mean()
        advantage = advantage / (advantage.std() + 1e-6)
        chosen = torch.log_softmax(self.policy.logits(obs, before, begins), -1).gather(-1, action[..., None])[..., 0]
        loss = -(chosen * advantage).mean()
        grads = torch.autograd.grad(loss, self.optimizer.params)
        self.optimizer.step(grads)
        return done.numel() / done.sum().clamp(min=1)


def train(cfg, updates, log=None):
    """`updates` updates; log(update, steps an episode lasts) after each. Returns the learner."""
    learner = Learner(cfg)
    for i in range(updates):
        lasted = learner.update()
        if log is not None:
            log(i + 1, float(lasted))
    return learner


def main(argv=None):
    p = argparse.ArgumentParser(prog="python -m hipenvs.recurrent", description=__doc__,
                                formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--task", choices=sorted(TASKS), default="cartpole")
    p.add_argument("--envs", type=int, default=1024)
    p.add_argument("--horizon", type=int, default=64)
    p.add_argument("--width", type=int, default=64)
    p.add_argument("--heads", type=int, default=4)
    p.add_argument("--layers", type=int, default=1)
    p.add_argument("--lr", type=float, default=3e-3)
    p.add_argument("--bits", type=int, choices=(8, 32), default=32)
    p.add_argument("--updates", type=int, default=100)
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args(argv)
    cfg = Config(task=a.task, envs=a.envs, horizon=a.horizon, width=a.width, heads=a.heads, layers=a.layers, lr=a.lr,
                 bits=a.bits, seed=a.seed)
    return train(cfg, a.updates, lambda i, lasted: print(f"update {i:4d}  steps an episode {lasted:7.1f}", flush=True))


if __name__ == "__main__":
    main()
