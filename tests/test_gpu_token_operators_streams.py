"""The operators over tokens on two streams at once, with their gradients (GPU): each call's workspace is its own."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def conv(gen, dev):
    from hipenvs import causal_conv

    x, weight, bias = (torch.randn(*s, generator=gen, device=dev) for s in ((8, 3000, 130), (130, 4), (130,)))
    return lambda: causal_conv.sequence(x, weight, bias), (x, weight, bias)


def lookup(gen, dev, rows=20000):
    from hipenvs import embedding

    tokens = torch.randint(-1, rows, (60000,), generator=gen, device=dev)
    table = torch.randn(rows, 64, generator=gen, device=dev)
    return lambda: (embedding.lookup(tokens, table),), (table,)


def log_probs(gen, dev):
    from hipenvs import categorical

    logits = torch.randn(20, 70000, generator=gen, device=dev)
    tokens = torch.randint(0, 70000, (20,), generator=gen, device=dev)
    return lambda: categorical.log_probs(logits, tokens, top=9)[:2], (logits,)


def scan(gen, dev):
    from hipenvs import selective_scan

    x, dt, write, read = (torch.randn(2, 3000, w, generator=gen, device=dev) for w in (40, 40, 12, 12))
    rate = -torch.rand(40, 12, generator=gen, device=dev)
    return lambda: selective_scan.sequence(x, dt, rate, write, read), (x, dt, rate, write, read)


@pytest.mark.parametrize("case", [conv, lookup, lambda gen, dev: lookup(gen, dev, 7), log_probs, scan],
                         ids=["conv", "lookup", "lookup_small", "log_probs", "scan"])
def test_two_streams(dev, case):
    calls = []
    for seed in range(2):
        gen = torch.Generator(device=dev)
        gen.manual_seed(seed)
        call, leaves = case(gen, dev)
        for x in leaves:
            x.requires_grad_()
        calls.append((call, leaves))

    def run(call, leaves):
        outs = call()
        return [x.detach() for x in outs] + list(torch.autograd.grad(outs, leaves, [torch.ones_like(x) for x in outs]))

    want = [run(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(*calls[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for g, w in zip(got, want) for a, e in zip(g, w))
