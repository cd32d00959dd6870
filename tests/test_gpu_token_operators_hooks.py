"""Convolution, lookup and log probabilities (GPU) under hooks on saved tensors and in forward mode: the bits are
those without hooks whatever the layout that a hook hands back, what is not the saved tensor's type, shape or GPU
is refused, and so are tensors with tangents."""

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
hooks = torch.autograd.graph.saved_tensors_hooks


def conv_case(dev, dtype=F32):
    from hipenvs import causal_conv

    gen = torch.Generator().manual_seed(1)
    x = torch.randn(40, 3, 21, generator=gen).to(dtype).to(dev).transpose(0, 1)
    weight, bias, state = (torch.randn(*s, generator=gen).to(dev) for s in ((21, 4), (21,), (3, 3, 21)))
    reset = (torch.rand(40, 3, generator=gen) < 0.1).to(dev).t()
    return (lambda *leaves: causal_conv.sequence(*leaves, reset)), (x, weight, bias, state)


def lookup_case(dev, dtype=F32, rows=300):
    from hipenvs import embedding

    gen = torch.Generator().manual_seed(2)
    tokens = torch.randint(-1, rows, (30, 7), generator=gen).to(dev).t()
    return (lambda table: (embedding.lookup(tokens, table, scale=0.5),)), (torch.randn(rows, 21, generator=gen).to(dtype).to(dev),)


def log_probs_case(dev, dtype=F32, v=33):
    from hipenvs import categorical

    gen = torch.Generator().manual_seed(3)
    logits = torch.randn(17, v + 2, generator=gen).to(dtype).to(dev)[:, 1:v + 1]
    tokens = torch.randint(-1, v, (17,), generator=gen).to(dev)
    return (lambda x: categorical.log_probs(x, tokens, top=2)[:2]), (logits,)


CASES = {"conv": conv_case, "lookup": lookup_case, "lookup_small": lambda dev, dtype=F32: lookup_case(dev, dtype, 5),
         "log_probs": log_probs_case, "log_probs_long": lambda dev, dtype=F32: log_probs_case(dev, dtype, 2000)}


def gradients(call, inputs, under=None):
    leaves = [x.detach().requires_grad_() for x in inputs]
    if under is None:
        outs = call(*leaves)
    else:
        with under:
            outs = call(*leaves)
    gen = torch.Generator(device=inputs[0].device)
    gen.manual_seed(4)
    given = [torch.randn(x.shape, generator=gen, device=x.device).to(x.dtype) for x in outs]
    return torch.autograd.grad(outs, leaves, given)


def turned(x):
    return x.detach().permute(*reversed(range(x.dim()))).contiguous().permute(*reversed(range(x.dim())))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", CASES)
def test_gradients_under_hooks(dev, name, dtype):
    print("hooks", name, dtype, flush=True)
    call, inputs = CASES[name](dev, dtype)
    want = gradients(call, inputs)
    for under in (hooks(lambda x: x.detach().clone(), lambda x: x), hooks(lambda x: x, turned),
                  torch.autograd.graph.save_on_cpu()):
        assert all(torch.equal(x, y) for x, y in zip(gradients(call, inputs, under), want))


@pytest.mark.parametrize("name", CASES)
def test_other_saved_tensors_are_refused(dev, name):
    """Every saved tensor in turn comes back left on the host, of another type, with a row less or more."""
    call, inputs = CASES[name](dev)
    kept = []
    with hooks(lambda x: kept.append(x) or x, lambda x: x):
        call(*(x.detach().requires_grad_() for x in inputs))
    assert kept
    for i in range(len(kept)):
        for change, error in ((lambda x: x.cpu(), ValueError), (lambda x: x[1:], ValueError),
                              (lambda x: torch.cat([x, x[:1]]), ValueError), (lambda x: x.half(), TypeError)):
            count = iter(range(len(kept)))
            print("refused", name, i, flush=True)
            with pytest.raises(error):
                gradients(call, inputs, hooks(lambda x: (next(count), x),
                                              lambda pair: change(pair[1].detach()) if pair[0] == i else pair[1]))


@pytest.mark.parametrize("name", CASES)
def test_forward_mode_derivatives_are_refused(dev, name):
    """A level without dual tensors changes nothing; a tangent of any differentiable input, or of a gradient
    that comes back, is refused."""
    call, inputs = CASES[name](dev)
    want = call(*inputs)
    with forward_ad.dual_level():
        assert all(torch.equal(x, y) for x, y in zip(call(*inputs), want))
        for i in range(len(inputs)):
            given = [forward_ad.make_dual(x, torch.ones_like(x)) if k == i else x for k, x in enumerate(inputs)]
            with pytest.raises(ValueError, match="forward-mode"):
                call(*given)
            given = [x.detach().requires_grad_() if k != i else given[i] for k, x in enumerate(inputs)]
            with pytest.raises(ValueError, match="forward-mode"):
                call(*given)
        leaf = inputs[0].detach().requires_grad_()
        out = call(leaf, *inputs[1:])[0]
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out, leaf, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_steps_refuse_tangents(dev):
    from hipenvs import causal_conv

    x, weight, bias, state = (torch.ones(*s, device=dev) for s in ((5, 6), (6, 4), (6,), (5, 3, 6)))
    with forward_ad.dual_level():
        for i in range(4):
            given = [forward_ad.make_dual(y, torch.ones_like(y)) if k == i else y for k, y in enumerate((x, weight, bias, state))]
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                causal_conv.step(*given)
        into = forward_ad.make_dual(state.clone(), torch.ones_like(state))
        version = into._version
        with pytest.raises(ValueError, match="forward-mode"):
            causal_conv.step(x, weight, bias, state, next_state=into)
        assert into._version == version
