"""A policy with a memory, trained by policy gradients on device-resident environments: the
operators of ``decay_attention`` or ``selective_scan`` with ``causal_conv``, ``embedding``,
``categorical`` and ``adamw`` as a learner uses them. The reference's gradient
learners (``ppo.py:84-95`` for the environment they step) see the whole state and keep no
memory; here some of the state can be hidden, and the policy has to remember.

``Policy`` acts one step at a time (``act``: the ``step`` of its memory, whose state is all that
it remembers) and is evaluated over whole trajectories with gradients (``logits``: the
memory's ``sequence``), episodes ending inside them. Its memory is decay attention
(``memory="decay"``) or a selective scan behind a convolution of four steps (``memory="scan"``); it
may see the action before (``previous_action``). ``Learner`` collects `horizon`
steps of every environment, takes the gradient of the discounted returns' advantage over
their mean (REINFORCE; with ``clip``, `epochs` times that of the clipped ratio to the policy that
acted; with ``entropy``, that of the policy's entropy too), and steps ``adamw.AdamW``. Nothing in
an update reads the device from the host.

    python -m hipenvs.recurrent --envs 1024 --updates 100
    python -m hipenvs.recurrent --memory scan --previous-action --clip 0.2 --epochs 4 --entropy 0.01
"""

import argparse
import math
from dataclasses import dataclass

import torch

from . import _lib, acrobot, adamw, adapter, cartpole
from . import categorical, causal_conv, decay_attention, embedding, selective_scan

# body, the rows of its state that the policy sees, actions. The angles and positions alone:
# velocities have to be inferred from the steps before.
TASKS = {"cartpole": (cartpole, (0, 2), 2), "acrobot": (acrobot, (0, 1), 3)}
MEMORIES = ("decay", "scan")


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
    memory: str = "decay"   # or "scan"
    states: int = 16        # a channel's, of a scan
    previous_action: bool = False
    clip: float = 0.0       # of the ratio to the policy that acted; 0: the plain gradient
    epochs: int = 1         # gradients of each collected batch, with clip
    entropy: float = 0.0    # the weight of the policy's entropy


class ScanBlock:
    """The convolution, the scan and its gate; the state of `n` environments is two tensors."""

    taps = 4

    def __init__(self, width, states, normal):
        self.width, self.states = width, states
        self.project, self.mix = normal(width, 2 * width), normal(width, width, 0.5)
        device = self.mix.device
        self.weight = normal(width, self.taps, math.sqrt(width / self.taps))
        self.bias = torch.zeros(width, device=device, requires_grad=True)
        self.choose = normal(width, width + 2 * states)
        # decays of 1, 2, 3, ... a unit of delta, which starts between 0.01 and 1 a step
        self.log_rate = torch.log(torch.arange(1.0, states + 1.0, device=device)).repeat(width, 1).requires_grad_()
        self.skip = torch.ones(width, device=device, requires_grad=True)
        delta = torch.logspace(-2.0, 0.0, width, device=device)
        self.dt_bias = torch.log(torch.expm1(delta)).requires_grad_()

    def parameters(self):
        return [self.project, self.weight, self.bias, self.choose, self.log_rate, self.skip, self.dt_bias, self.mix]

    def initial_state(self, n):
        device = self.mix.device
        return [torch.zeros(n, self.taps - 1, self.width, device=device),
                torch.zeros(n, self.width, self.states, device=device)]

    def through(self, x, convolve, scan):
        """The block's output for x (..., width); convolve(u) and scan(u, dt, rate, write, read, gate) are the
        operators over whole trajectories or for one step."""
        u, gate = (x @ self.project).chunk(2, dim=-1)
        u = convolve(u)
        dt, write, read = torch.split(u @ self.choose, (self.width, self.states, self.states), dim=-1)
        return scan(u, dt, -torch.exp(self.log_rate), write, read, gate) @ self.mix

    def sequence(self, x, state, reset):
        return self.through(
            x, lambda u: causal_conv.sequence(u, self.weight, self.bias, state[0], reset)[0],
            lambda u, dt, rate, write, read, gate: selective_scan.sequence(
                u, dt, rate, write, read, self.skip, gate, self.dt_bias, state[1], reset)[0])

    def step(self, x, state, reset):
        return self.through(
            x, lambda u: causal_conv.step(u, self.weight, self.bias, state[0], reset, next_state=state[0])[0],
            lambda u, dt, rate, write, read, gate: selective_scan.step(
                u, dt, rate, write, read, self.skip, gate, self.dt_bias, state[1], reset, next_state=state[1])[0])


class DecayBlock:
    """Decay attention; the state of `n` environments is one tensor."""

    def __init__(self, width, heads, normal, log_decay):
        self.width, self.heads, self.log_decay = width, heads, log_decay
        self.project, self.mix = normal(width, 3 * width), normal(width, width, 0.5)

    def parameters(self):
        return [self.project, self.mix]

    def initial_state(self, n):
        d = self.width // self.heads
        return [torch.zeros(n, self.heads, d, d, device=self.mix.device)]

    def through(self, x, attend):
        q, k, v = ((x @ self.project).unflatten(-1, (3 * self.heads, -1))).chunk(3, dim=-2)
        return torch.tanh(attend(q, k, v).flatten(-2)) @ self.mix

    def sequence(self, x, state, reset):
        return self.through(x, lambda q, k, v: decay_attention.sequence(q, k, v, self.log_decay, state[0], reset)[0])

    def step(self, x, state, reset):
        return self.through(x, lambda q, k, v: decay_attention.step(
            q, k, v, self.log_decay, state[0], reset, next_state=state[0])[0])


class Policy:
    """An encoder, ``layers`` blocks with a memory, a head of logits; float32."""

    def __init__(self, obs_dim, actions, width, heads, layers, generator, memory="decay", states=16,
                 previous_action=False):
        if memory not in MEMORIES:
            raise ValueError(f"memory must be {' or '.join(MEMORIES)}, got {memory}")
        if memory == "decay" and width % heads:
            raise ValueError(f"width {width} must be a multiple of heads {heads}")
        device = generator.device

        def normal(rows, columns, gain=1.0):
            x = torch.randn(rows, columns, generator=generator, device=device) * (gain / math.sqrt(rows))
            return x.requires_grad_()

        self.heads, self.width = heads, width
        self.encoder = normal(obs_dim, width)
        self.bias = torch.zeros(width, device=device, requires_grad=True)
        # memories of 2, 4, 8, ... steps
        self.log_decay = torch.log1p(-(2.0 ** -torch.arange(1.0, heads + 1.0, device=device)))
        self.blocks = [ScanBlock(width, states, normal) if memory == "scan"
                       else DecayBlock(width, heads, normal, self.log_decay) for _ in range(layers)]
        self.head = normal(width, actions, 0.1)
        self.table = normal(actions, width, math.sqrt(actions)) if previous_action else None

    def parameters(self):
        return [self.encoder, self.bias, *(w for block in self.blocks for w in block.parameters()), self.head,
                *([self.table] if self.table is not None else [])]

    def initial_state(self, n):
        return [s for block in self.blocks for s in block.initial_state(n)]

    def _through(self, obs, previous, state, remember):
        """The logits of observations (..., obs_dim); remember(block, x, its part of state) -> its output."""
        x = obs @ self.encoder + self.bias
        if self.table is not None:
            x = x + embedding.lookup(previous, self.table)
        x = torch.tanh(x)
        each = len(state) // len(self.blocks) if self.blocks else 0
        for i, block in enumerate(self.blocks):
            x = x + remember(block, x, state[i * each:(i + 1) * each])
        return x @ self.head

    @torch.no_grad()
    def act(self, obs, state, reset, previous=None):
        """Logits (n, actions) for obs (n, obs_dim); state, the list of initial_state, is updated in
        place. reset (n,) bool: this observation is an episode's first. previous (n,): the action before
        it, -1 for none, where the policy sees it."""
        return self._through(obs, previous, state, lambda block, x, s: block.step(x, s, reset))

    def logits(self, obs, state, reset, previous=None):
        """Logits (n, t, actions) for trajectories obs (n, t, obs_dim) from the states before them."""
        return self._through(obs, previous, state, lambda block, x, s: block.sequence(x, s, reset))


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
        if cfg.memory not in MEMORIES:
            raise ValueError(f"memory must be {' or '.join(MEMORIES)}, got {cfg.memory}")
        if not 0.0 <= cfg.clip < math.inf:
            raise ValueError(f"clip must be 0 or above and finite, got {cfg.clip}")
        if cfg.epochs < 1 or (cfg.epochs > 1 and not cfg.clip > 0):
            raise ValueError(f"epochs must be 1, or more with a clip above 0, got {cfg.epochs} with clip {cfg.clip}")
        self.cfg = cfg
        device = torch.device(device) if device is not None else _lib.default_device()
        body, seen, actions = TASKS[cfg.task]
        self.seen = torch.tensor(seen, device=device)   # a list would be uploaded, and waited for, at every step
        body.reseed(cfg.seed)
        self.env = adapter.DeviceEnv(body, cfg.envs, seed=cfg.seed + 1, device=device)
        self.generator = torch.Generator(device=device)
        self.generator.manual_seed(cfg.seed)
        self.policy = Policy(len(seen), actions, cfg.width, cfg.heads, cfg.layers, self.generator, cfg.memory,
                             cfg.states, cfg.previous_action)
        self.optimizer = adamw.AdamW(self.policy.parameters(), lr=cfg.lr, weight_decay=cfg.weight_decay, bits=cfg.bits)
        self.memory = self.policy.initial_state(cfg.envs)
        self.begins = torch.ones(cfg.envs, dtype=torch.bool, device=device)
        self.previous = torch.full((cfg.envs,), -1, dtype=torch.int64, device=device) if cfg.previous_action else None

    def collect(self):
        """One trajectory of every environment: (obs, begins, action, reward, done), each (envs,
        horizon, ...), collected time-major; and the memory before it."""
        batch, before = self._collect()
        return batch[:5], before

    def _collect(self):
        """What collect returns, and where the policy sees it the action before each (-1 for none), and
        where a ratio to it is taken the log probability of each action under the policy that acted; None
        otherwise."""
        before = [s.clone() for s in self.memory]
        steps, previous, acted = [], [], []
        for _ in range(self.cfg.horizon):
            obs = self.env.obs().index_select(1, self.seen)
            logits = self.policy.act(obs, self.memory, self.begins, self.previous)
            noise = torch.rand(logits.shape, generator=self.generator, device=logits.device)
            action = (logits - torch.log(-torch.log(noise.clamp(1e-12, 1 - 1e-7)))).argmax(-1)   # Gumbel's maximum
            begins = self.begins
            reward, self.begins = self.env.step(action.to(torch.int32))
            steps.append((obs, begins, action, reward, self.begins))
            if self.previous is not None:
                previous.append(self.previous)
                self.previous = torch.where(self.begins, -1, action)
            if self.cfg.clip:
                acted.append(categorical.log_probs(logits, action)[0])
        extra = (torch.stack(x).transpose(0, 1) if x else None for x in (previous, acted))
        return (*(torch.stack(x).transpose(0, 1) for x in zip(*steps)), *extra), before

    def _loss(self, batch, before, advantage):
        obs, begins, action, _, _, previous, acted = batch
        logits = self.policy.logits(obs, before, begins, previous)
        if not self.cfg.clip and not self.cfg.entropy:
            chosen = torch.log_softmax(logits, -1).gather(-1, action[..., None])[..., 0]
            return -(chosen * advantage).mean()
        log_prob, entropy = categorical.log_probs(logits, action)
        gain = log_prob * advantage
        if self.cfg.clip:
            ratio = torch.exp(log_prob - acted)
            near = ratio.clamp(1.0 - self.cfg.clip, 1.0 + self.cfg.clip)
            gain = torch.minimum(ratio * advantage, near * advantage)
        return -(gain + self.cfg.entropy * entropy).mean()

    def update(self):
        """Collects, and moves the policy once (``epochs`` times); the steps an episode lasted on average (a
        device scalar: environment steps over episodes that ended)."""
        batch, before = self._collect()
        reward, done = batch[3:5]
        returns = discounted(reward, done, self.cfg.gamma)
        advantage = returns - returns.mean()
        advantage = advantage / (advantage.std() + 1e-6)
        for _ in range(self.cfg.epochs):
            grads = torch.autograd.grad(self._loss(batch, before, advantage), self.optimizer.params)
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
    p.add_argument("--memory", choices=MEMORIES, default="decay")
    p.add_argument("--states", type=int, default=16)
    p.add_argument("--previous-action", action="store_true")
    p.add_argument("--clip", type=float, default=0.0)
    p.add_argument("--epochs", type=int, default=1)
    p.add_argument("--entropy", type=float, default=0.0)
    a = p.parse_args(argv)
    cfg = Config(task=a.task, envs=a.envs, horizon=a.horizon, width=a.width, heads=a.heads, layers=a.layers, lr=a.lr,
                 bits=a.bits, seed=a.seed, memory=a.memory, states=a.states, previous_action=a.previous_action,
                 clip=a.clip, epochs=a.epochs, entropy=a.entropy)
    return train(cfg, a.updates, lambda i, lasted: print(f"update {i:4d}  steps an episode {lasted:7.1f}", flush=True))


if __name__ == "__main__":
    main()
