"""The operators of a policy over tokens, as measurable cases: the selective scan and its short
convolution (a policy's memory), the lookup of action tokens, and the log probabilities of chosen
actions.

Eight kinds of call:

* ``scan``: the selective scan over whole trajectories, outputs and final states;
* ``scan_train``: the same with its backward pass, gradients of every input;
* ``scan_step``: one token of every environment, from the state before it to the state after it;
* ``conv_train``: the short causal convolution over trajectories, with gradients of every input;
* ``conv_step``: one token of every environment through the convolution;
* ``lookup_train``: rows of a table for tokens, and the gradient of the table;
* ``log_probs``: log probabilities of given tokens, entropies and the most likely tokens;
* ``log_probs_train``: log probabilities and entropies with the gradient of the logits.

A channel's state is h_t[n] = exp(delta rate[n]) h_{t-1}[n] + delta x write_t[n] with delta =
softplus(dt + dt_bias), and its output (sum_n read_t[n] h_t[n] + skip x) silu(gate). h_{t-1}, and
the convolution's taps before t, are left out where an episode begins at t (``reset``). Where
``own`` is false, ``run`` computes that in elementary torch operations in float32; where it is
true, it makes the calls of ``hipenvs.selective_scan``, ``causal_conv``, ``embedding`` and
``categorical``.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
BLOCK = 64            # tokens whose decays the plain form computes at once
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _package():
    """hipenvs' modules; asked for only where ``own`` is true."""
    path = os.path.join(os.getcwd(), "metal-rl-envs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from hipenvs import categorical, causal_conv, embedding, selective_scan

    return selective_scan, causal_conv, embedding, categorical


# ---- the cases ----------------------------------------------------------------------------

def listed():
    return [
        # the window of a few environments re-read after a policy change: latency
        {"name": "scan_short", "kind": "scan", "b": 16, "t": 33, "d": 64, "n": 16, "g": 1, "dtype": "f32",
         "layout": "fused", "gate": True, "episode": 20},
        # one long recording: few rows, a long axis
        {"name": "scan_long", "kind": "scan", "b": 1, "t": 16381, "d": 512, "n": 16, "g": 1, "dtype": "bf16",
         "layout": "fused", "gate": True, "episode": 0},
        # the update of a learner with 4,096 CartPole environments, 128 steps each, several episodes in each row
        {"name": "scan_train_many_envs", "kind": "scan_train", "b": 4096, "t": 128, "d": 128, "n": 16, "g": 1,
         "dtype": "f32", "layout": "time", "gate": True, "episode": 40},
        # whole legged episodes, a state width that is no power of two, two groups of channels
        {"name": "scan_train_episodes", "kind": "scan_train", "b": 64, "t": 1000, "d": 500, "n": 12, "g": 2,
         "dtype": "bf16", "layout": "apart", "gate": False, "episode": 500},
        # acting in the populations' 4,096 environments
        {"name": "scan_step", "kind": "scan_step", "b": 4096, "d": 512, "n": 16, "g": 1, "dtype": "bf16",
         "layout": "fused", "gate": True, "episode": 500},
        # the convolution before the scan of whole legged episodes, uneven channels
        {"name": "conv_train", "kind": "conv_train", "b": 64, "t": 1000, "d": 501, "w": 4, "dtype": "bf16",
         "layout": "fused", "episode": 500},
        # acting in a thousand environments: latency and the host path
        {"name": "conv_step", "kind": "conv_step", "b": 1021, "d": 128, "w": 4, "dtype": "f32", "layout": "fused",
         "episode": 100},
        # the previous action of Acrobot's three as an input: every token at every place, few rows
        {"name": "lookup_actions", "kind": "lookup_train", "shape": "4096x128", "v": 3, "d": 64, "dtype": "f32",
         "skew": 0.0, "absent": 0.03},
        # a vocabulary of tokens, most of them rare
        {"name": "lookup_vocabulary", "kind": "lookup_train", "shape": "64x1000", "v": 40009, "d": 512,
         "dtype": "bf16", "skew": 3.0, "absent": 0.0},
        # the chosen actions of that learner's batch
        {"name": "log_probs_actions", "kind": "log_probs_train", "rows": 524288, "v": 3, "dtype": "f32", "masked": 0.0},
        # a head over the vocabulary, some tokens not allowed
        {"name": "log_probs_vocabulary", "kind": "log_probs_train", "rows": 4093, "v": 40009, "dtype": "bf16",
         "masked": 0.2},
        # one answer of a few streams: the chosen token and its 20 alternatives
        {"name": "log_probs_top", "kind": "log_probs", "rows": 16, "v": 131071, "dtype": "bf16", "masked": 0.0,
         "top": 20},
    ]


def _size(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi], odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rows(rng, kind, d, each):
    """(b, t) of `each` values a token and channel, below the largest listed case's."""
    t = _size(rng, 1, 16384)
    return _size(rng, 1, max(1, min(8192, (1 << 29) // (t * d * each), (1 << 19) // t))), t


def draw(rng):
    kind = rng.choice(("scan", "scan_train", "scan_train", "scan_step", "conv_train", "conv_step", "lookup_train",
                       "log_probs", "log_probs_train"))
    dtype = rng.choice(("f32", "bf16"))
    if kind == "lookup_train":
        v, d = _size(rng, 2, 1 << 17), _size(rng, 4, 1024)
        v = min(v, (1 << 25) // d)
        return {"kind": kind, "shape": str(_size(rng, 1, min(1 << 19, (1 << 25) // d))), "v": v, "d": d, "dtype": dtype,
                "skew": rng.choice((0.0, 1.0, 3.0)), "absent": rng.choice((0.0, 0.1))}
    if kind in ("log_probs", "log_probs_train"):
        v = _size(rng, 2, 1 << 17)
        case = {"kind": kind, "rows": _size(rng, 1, min(1 << 19, (1 << 27) // v)), "v": v, "dtype": dtype,
                "masked": rng.choice((0.0, 0.3))}
        if kind == "log_probs":
            case["top"] = rng.choice((0, 1, rng.randint(1, min(v, 32))))
        return case
    d = rng.choice((64, 128, 256, 512, _size(rng, 1, 1024)))
    case = {"kind": kind, "d": d, "dtype": dtype, "layout": rng.choice(("fused", "time", "apart")),
            "episode": rng.choice((0, 10, 100, 1000))}
    if kind.startswith("conv"):
        case["w"] = rng.choice((4, 4, 3, 2))
    else:
        case["n"] = rng.choice((16, 16, 8, rng.randint(1, 64)))
        case["g"] = rng.choice([g for g in (1, 1, 2, 4) if d % g == 0])
        case["gate"] = rng.choice((True, False))
    if kind.endswith("_step"):
        case["layout"] = rng.choice(("fused", "apart"))
        case["b"] = _size(rng, 1, max(1, min(8192, (1 << 25) // (d * case.get("n", 1)))))
    else:
        case["b"], case["t"] = _draw_rows(rng, kind, d, case.get("n", 4))
    return case


# ---- inputs -------------------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32)


def _rows(gen, case, lead, widths, gain=1.0):
    """Tensors (*lead, width): parts of one projection's rows ("fused"), of one that was collected
    time-major ("time"), or tensors of their own ("apart")."""
    dtype = DTYPES[case["dtype"]]
    if case["layout"] == "apart":
        return [(_normal(gen, *lead, w) * gain).to(dtype) for w in widths]
    rows = (_normal(gen, *(reversed(lead) if case["layout"] == "time" else lead), sum(widths)) * gain).to(dtype)
    if case["layout"] == "time":
        rows = rows.transpose(0, 1)
    return list(torch.split(rows, widths, dim=-1))


def _begins(gen, shape, episode):
    """Where an episode begins: each token with probability 1 / episode, none for episode 0."""
    draws = torch.rand(*shape, generator=gen, device=DEVICE)
    return draws < (1.0 / episode if episode else 0.0)


def _prepare_scan(case, gen, lead):
    d, n, g = case["d"], case["n"], case["g"]
    x, gate = _rows(gen, case, lead, [d, d])
    dt, write, read = _rows(gen, case, lead, [d, g * n, g * n])
    steps = 0.001 * 100.0 ** torch.rand(d, generator=gen, device=DEVICE)   # steps between 0.001 and 0.1
    s = {"x": x, "dt": dt, "rate": -(torch.arange(n, device=DEVICE) + 1.0).repeat(d, 1)
         * torch.exp(0.1 * _normal(gen, d, n)),
         "write": write.unflatten(-1, (g, n)), "read": read.unflatten(-1, (g, n)), "skip": 1.0 + 0.1 * _normal(gen, d),
         "gate": gate if case["gate"] else None, "dt_bias": torch.log(torch.expm1(steps)),
         "state": _normal(gen, lead[0], d, n), "reset": _begins(gen, lead, case["episode"])}
    if case["kind"] == "scan_train":
        s["dout"] = _normal(gen, *lead, d).to(x.dtype)
        s["dfinal"] = _normal(gen, lead[0], d, n)
    return s


def _prepare_conv(case, gen, lead):
    d, w = case["d"], case["w"]
    x = _rows(gen, case, lead, [d, d])[0]
    s = {"x": x, "weight": _normal(gen, d, w) / math.sqrt(w), "bias": 0.1 * _normal(gen, d),
         "state": _normal(gen, lead[0], w - 1, d), "reset": _begins(gen, lead, case["episode"])}
    if case["kind"] == "conv_train":
        s["dout"] = _normal(gen, *lead, d).to(x.dtype)
        s["dfinal"] = _normal(gen, lead[0], w - 1, d)
    return s


def _prepare_lookup(case, gen):
    shape = [int(n) for n in case["shape"].split("x")]
    dtype, v = DTYPES[case["dtype"]], case["v"]
    # skew 0: all tokens alike; above: the lower ones more often
    token = (v * torch.rand(*shape, generator=gen, device=DEVICE, dtype=torch.float64) ** (1.0 + case["skew"])).long()
    token = token.clamp(max=v - 1)
    token = torch.where(torch.rand(*shape, generator=gen, device=DEVICE) < case["absent"], -1, token)
    return {"tokens": token, "table": _normal(gen, v, case["d"]).to(dtype), "scale": math.sqrt(case["d"]),
            "dout": _normal(gen, *shape, case["d"]).to(dtype)}


def _prepare_log_probs(case, gen):
    rows, v = case["rows"], case["v"]
    logits = (2.0 * _normal(gen, rows, v)).to(DTYPES[case["dtype"]])
    tokens = torch.randint(0, v, (rows,), generator=gen, device=DEVICE)
    if case["masked"]:
        out = torch.rand(rows, v, generator=gen, device=DEVICE) < case["masked"]
        logits = logits.masked_fill_(out.scatter_(1, tokens[:, None], False), -math.inf)
    return {"logits": logits, "tokens": tokens, "top": case.get("top", 0), "dlog_prob": _normal(gen, rows),
            "dentropy": _normal(gen, rows)}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    kind = case["kind"]
    if kind == "lookup_train":
        s = _prepare_lookup(case, gen)
    elif kind.startswith("log_probs"):
        s = _prepare_log_probs(case, gen)
    else:
        lead = (case["b"],) if kind.endswith("_step") else (case["b"], case["t"])
        s = (_prepare_conv if kind.startswith("conv") else _prepare_scan)(case, gen, lead)
    return {"kind": kind, **s}


# ---- plain forms --------------------------------------------------------------------------

def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _spread(x, d):
    """(b, t, g, n) -> (b, t, g, d / g, n), one row for every channel of its group."""
    return x.float()[:, :, :, None, :].expand(-1, -1, -1, d // x.shape[2], -1)


def _plain_scan(x, dt, rate, write, read, skip, gate, dt_bias, state, reset):
    """The recurrence token by token, the decays and what enters a state for 64 tokens at once."""
    (b, t, d), g, dtype = x.shape, write.shape[2], x.dtype
    x, delta = x.float().unflatten(2, (g, -1)), _softplus(dt.float() + dt_bias).unflatten(2, (g, -1))
    rate, h = rate.unflatten(0, (g, -1)), state.unflatten(1, (g, -1))
    write, read = _spread(write, d), _spread(read, d)
    outs = []
    for at in range(0, t, BLOCK):
        part = slice(at, min(at + BLOCK, t))
        keep = torch.exp(delta[:, part, ..., None] * rate)
        keep = torch.where(reset[:, part, None, None, None], 0.0, keep)
        add = (delta[:, part] * x[:, part])[..., None] * write[:, part]
        states = []
        for k, a in zip(keep.unbind(1), add.unbind(1)):
            h = torch.addcmul(a, k, h)
            states.append(h)
        outs.append((torch.stack(states, 1) * read[:, part]).sum(-1))
    y = (torch.cat(outs, 1) + skip.unflatten(0, (g, -1)) * x).flatten(2)
    if gate is not None:
        y = y * _silu(gate.float())
    return y.to(dtype), h.flatten(1, 2)


def _plain_conv(x, weight, bias, state, reset):
    (b, t, d), w = x.shape, weight.shape[1]
    begun = torch.nn.functional.pad(reset.to(torch.int64).cumsum(1), (w - 1, 0))
    held = torch.cat([state, x.float()], 1)                            # token i at i + w - 1
    out = bias.expand(b, t, d)
    for j in range(w):   # the tap at t - (w - 1) + j
        same = begun[:, j:j + t] == begun[:, w - 1:]
        out = out + weight[:, j] * torch.where(same[:, :, None], held[:, j:j + t], 0.0)
    last = begun[:, t:] == begun[:, -1:]
    return _silu(out).to(x.dtype), torch.where(last[:, :w - 1, None], held[:, t:], 0.0)


def _with_gradients(call, s, names):
    """The outputs of call(inputs by name), and the gradients of those in `names` that are there."""
    leaves = {n: s[n].detach().requires_grad_() for n in names if s[n] is not None}
    out, final = call(**{n: leaves.get(n, s[n]) for n in (*names, "reset")})
    return (out.detach(), final.detach(),
            *torch.autograd.grad((out, final), list(leaves.values()), (s["dout"], s["dfinal"])))


SCAN = ("x", "dt", "rate", "write", "read", "skip", "gate", "dt_bias", "state")
CONV = ("x", "weight", "bias", "state")


def _plain_step(call, s, names, tokens):
    """One token by the plain form of whole rows."""
    given = {n: s[n].unsqueeze(1) if n in tokens and s[n] is not None else s[n] for n in (*names, "reset")}
    out, final = call(**given)
    return out.squeeze(1), final


def _plain_lookup(s):
    tokens, table = s["tokens"].flatten(), s["table"]
    there = tokens >= 0
    out = table[tokens.clamp(min=0)].float() * s["scale"]
    out = torch.where(there[:, None], out, 0.0).to(table.dtype).view(*s["tokens"].shape, -1)
    # a row may gather every token: the sum in 64 bits, and of a small table as a product
    dout = s["dout"].flatten(0, -2).double()
    if table.shape[0] <= 64:
        grad = (torch.arange(table.shape[0], device=table.device)[:, None] == tokens).double() @ dout
    else:
        grad = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
        grad.index_add_(0, tokens[there], dout[there])
    return out, (grad * s["scale"]).to(table.dtype)


def _plain_log_probs(s):
    logits, tokens = s["logits"], s["tokens"]
    x = logits.float()
    m = x.amax(1, keepdim=True)
    shifted = x - m
    e = torch.exp(shifted)
    total = e.sum(1, keepdim=True)
    p = e / total
    log_p = shifted - torch.log(total)
    term = torch.where(p > 0, p * log_p, 0.0)
    entropy = -term.sum(1)
    out = [log_p.gather(1, tokens[:, None])[:, 0], entropy]
    if s["kind"] == "log_probs_train":
        chosen = torch.arange(x.shape[1], device=x.device) == tokens[:, None]
        grad = s["dlog_prob"][:, None] * (chosen.float() - p) - s["dentropy"][:, None] * (term + p * entropy[:, None])
        out.append(grad.to(logits.dtype))
    elif s["top"]:
        _, index = torch.sort(x, dim=1, descending=True, stable=True)
        index = index[:, :s["top"]]
        out += [log_p.gather(1, index), index]
    return out


# ---- one pass -----------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    kind = s["kind"]
    if kind == "scan":
        return _plain_scan(*(s[n] for n in (*SCAN, "reset")))
    if kind == "scan_train":
        return _with_gradients(_plain_scan, s, SCAN)
    if kind == "scan_step":
        return _plain_step(_plain_scan, s, SCAN, ("x", "dt", "write", "read", "gate", "reset"))
    if kind == "conv_train":
        return _with_gradients(_plain_conv, s, CONV)
    if kind == "conv_step":
        return _plain_step(_plain_conv, s, CONV, ("x", "reset"))
    return (_plain_lookup if kind == "lookup_train" else _plain_log_probs)(s)


def _own(s):
    scan, conv, embedding, categorical = _package()
    kind = s["kind"]
    if kind == "scan":
        return scan.sequence(*(s[n] for n in (*SCAN, "reset")))
    if kind == "scan_train":
        return _with_gradients(scan.sequence, s, SCAN)
    if kind == "scan_step":
        return scan.step(*(s[n] for n in (*SCAN, "reset")))
    if kind == "conv_train":
        return _with_gradients(conv.sequence, s, CONV)
    if kind == "conv_step":
        return conv.step(*(s[n] for n in (*CONV, "reset")))
    if kind == "lookup_train":
        table = s["table"].detach().requires_grad_()
        out = embedding.lookup(s["tokens"], table, scale=s["scale"])
        return (out.detach(), *torch.autograd.grad(out, table, s["dout"]))
    if kind == "log_probs":
        return categorical.log_probs(s["logits"], s["tokens"], top=s["top"])
    logits = s["logits"].detach().requires_grad_()
    log_prob, entropy = categorical.log_probs(logits, s["tokens"])
    return (log_prob.detach(), entropy.detach(),
            *torch.autograd.grad((log_prob, entropy), logits, (s["dlog_prob"], s["dentropy"])))


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    e, kind = 4 if case["dtype"] == "f32" else 2, case["kind"]
    if kind == "lookup_train":
        rows = math.prod(int(n) for n in case["shape"].split("x"))
        v, d = case["v"], case["d"]
        # tokens and rows of the output and its gradient, the table's rows that are met and its gradient
        return {"bytes": 8 * rows + 2 * e * rows * d + e * d * (v + min(v, rows)), "flops": 2 * rows * d}
    if kind.startswith("log_probs"):
        rows, v = case["rows"], case["v"]
        once = e * rows * v + 16 * rows
        if kind == "log_probs":
            return {"bytes": once + 12 * rows * case["top"], "flops": 6 * rows * v}
        return {"bytes": once + 8 * rows + e * rows * v, "flops": 12 * rows * v}
    b, d = case["b"], case["d"]
    tokens = b * case.get("t", 1)
    if kind.startswith("conv"):
        w = case["w"]
        once = {"bytes": tokens * d * 2 * e + tokens + 8 * b * (w - 1) * d, "flops": (2 * w + 5) * tokens * d}
        if kind == "conv_step":
            return once
        return {"bytes": once["bytes"] + tokens * d * 2 * e + 8 * b * (w - 1) * d, "flops": 3 * once["flops"]}
    n, g = case["n"], case["g"]
    wide = 3 + case["gate"]   # x, dt, out and the gate
    once = {"bytes": tokens * e * (wide * d + 2 * g * n) + tokens + 8 * b * d * n + 4 * d * n,
            "flops": tokens * d * (7 * n + 20)}
    if kind != "scan_train":
        return once
    # backward: dout in, the gradients of x, dt, write, read and the gate out, the states' gradients
    return {"bytes": once["bytes"] + tokens * e * (wide * d + 2 * g * n) + 8 * b * d * n + 4 * d * n,
            "flops": 3.5 * once["flops"]}


# ---- the definition in 64 bits --------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "lookup_train":
        return _exact_lookup(s)
    if kind.startswith("log_probs"):
        return _exact_log_probs(s)
    if kind.endswith("_step"):
        for n in ("x", "dt", "write", "read", "gate", "reset"):
            if s.get(n) is not None:
                s[n] = s[n].unsqueeze(1)
        out, final = (_exact_conv if kind.startswith("conv") else _exact_scan)(s)
        return out.squeeze(1), final
    return (_exact_conv if kind.startswith("conv") else _exact_scan)(s)


def _exact_scan(s):
    x, rate, h = s["x"].double(), s["rate"].double(), s["state"].double()
    raw = s["dt"].double() + s["dt_bias"].double()
    delta = torch.nn.functional.softplus(raw)
    (b, t, d), n, g = x.shape, rate.shape[1], s["write"].shape[2]

    def per_channel(name, i):  # (b, d, n)
        return s[name][:, i].double().repeat_interleave(d // g, dim=1)

    def keep(i):
        return torch.exp(delta[:, i, :, None] * rate) * (~s["reset"][:, i]).double()[:, None, None]

    y, before = torch.empty_like(x), []
    train = s["kind"] == "scan_train"
    for i in range(t):
        if train:
            before.append(h)
        h = keep(i) * h + (delta[:, i] * x[:, i])[..., None] * per_channel("write", i)
        y[:, i] = (h * per_channel("read", i)).sum(-1) + s["skip"].double() * x[:, i]
    z = s["gate"].double() if s["gate"] is not None else None
    gate = z * torch.sigmoid(z) if z is not None else torch.ones_like(x)
    if not train:
        return y * gate, h
    dout, G = s["dout"].double(), s["dfinal"].double()
    dy = dout * gate
    drate, ddelta, dx = torch.zeros_like(rate), torch.empty_like(x), torch.empty_like(x)
    dwrite, dread = (torch.empty(b, t, g, n, dtype=torch.float64, device=x.device) for _ in range(2))
    after = h
    for i in reversed(range(t)):
        write, a = per_channel("write", i), keep(i)
        dread[:, i] = (after * dy[:, i, :, None]).unflatten(1, (g, -1)).sum(2)
        G = G + per_channel("read", i) * dy[:, i, :, None]
        dwrite[:, i] = (G * (delta[:, i] * x[:, i])[..., None]).unflatten(1, (g, -1)).sum(2)
        through = G * a * before[i]
        into = (G * write).sum(-1)
        drate += (through * delta[:, i, :, None]).sum(0)
        ddelta[:, i] = (through * rate).sum(-1) + into * x[:, i]
        dx[:, i] = s["skip"].double() * dy[:, i] + into * delta[:, i]
        G, after = G * a, before[i]
    ddt = ddelta * torch.sigmoid(raw)
    grads = [dx, ddt, drate, dwrite, dread, (dy * x).sum((0, 1))]
    if z is not None:
        one = torch.sigmoid(z)
        grads.append(dout * y * one * (1.0 + z * (1.0 - one)))
    return (y * gate, h, *grads, ddt.sum((0, 1)), G)


def _exact_conv(s):
    x, weight, hist = s["x"].double(), s["weight"].double(), s["state"].double()
    t, w = x.shape[1], weight.shape[1]
    pre, windows = torch.empty_like(x), []
    for i in range(t):
        hist = torch.where(s["reset"][:, i, None, None], 0.0, hist)
        window = torch.cat([hist, x[:, i:i + 1]], 1)                   # (b, w, d)
        pre[:, i] = s["bias"].double() + (window * weight.t()).sum(1)
        windows.append(window)
        hist = window[:, 1:]
    one = torch.sigmoid(pre)
    if s["kind"] != "conv_train":
        return pre * one, hist
    dpre = s["dout"].double() * one * (1.0 + pre * (1.0 - one))
    carry, dx, dweight = s["dfinal"].double(), torch.empty_like(x), torch.zeros_like(weight)
    for i in reversed(range(t)):
        into = weight.t() * dpre[:, i, None, :]                        # of each of the w values
        into = torch.cat([into[:, :1], into[:, 1:] + carry], 1)
        dweight += (windows[i] * dpre[:, i, None, :]).sum(0).t()
        dx[:, i] = into[:, -1]
        carry = torch.where(s["reset"][:, i, None, None], 0.0, into[:, :-1])
    return pre * one, hist, dx, dweight, dpre.sum((0, 1)), carry


def _exact_lookup(s):
    tokens, table, dout = s["tokens"].flatten(), s["table"].double(), s["dout"].double().flatten(0, -2)
    padded = torch.cat([table, torch.zeros_like(table[:1])])           # the last row: no token
    out = padded[tokens] * s["scale"]
    order = torch.argsort(tokens, stable=True)
    upto = torch.nn.functional.pad(dout[order].cumsum(0), (0, 0, 1, 0))
    ends = torch.bincount(tokens + 1, minlength=table.shape[0] + 1).cumsum(0)
    return out.view(*s["tokens"].shape, -1), (upto[ends[1:]] - upto[ends[:-1]]) * s["scale"]


def _exact_log_probs(s):
    x, tokens = s["logits"].double(), s["tokens"]
    lse = torch.logsumexp(x, 1, keepdim=True)
    log_p = x - lse
    p = torch.exp(log_p)
    entropy = torch.special.entr(p).sum(1)
    out = [log_p[torch.arange(len(tokens), device=x.device), tokens], entropy]
    if s["kind"] == "log_probs_train":
        finite = torch.where(torch.isinf(log_p), 0.0, log_p)
        grad = -p * (s["dlog_prob"].double()[:, None] + s["dentropy"].double()[:, None] * (finite + entropy[:, None]))
        grad[torch.arange(len(tokens), device=x.device), tokens] += s["dlog_prob"].double()
        out.append(grad)
    elif s["top"]:
        k = s["top"]
        index = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
        out += [torch.take_along_dim(log_p, index, 1), index]
    return out
