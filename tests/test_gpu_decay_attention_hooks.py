"""Decay attention's gradients (GPU) under hooks on saved tensors: the bits are those without hooks,
whatever the layout that a hook hands back, and what is no longer on the GPU is refused."""

import pytest
import torch

from test_gpu_decay_attention import BF16, F32, case

pytestmark = pytest.mark.gpu


def gradients(c, hooks=None):
    from hipenvs import decay_attention

    leaves = {n: c[n].detach().requires_grad_() for n in ("q", "k", "v", "state")}
    gen = torch.Generator(device=c["q"].device)
    gen.manual_seed(1)
    if hooks is None:
        out, final = decay_attention.sequence(**{**c, **leaves})
    else:
        with hooks:
            out, final = decay_attention.sequence(**{**c, **leaves})
    given = [torch.randn(x.shape, generator=gen, device=x.device).to(x.dtype) for x in (out, final)]
    return torch.autograd.grad((out, final), list(leaves.values()), given)


def turned(x):
    return x.detach().permute(*reversed(range(x.dim()))).contiguous().permute(*reversed(range(x.dim())))


SHAPES = [(3, 70, 2, 32, 32), (2, 130, 3, 20, 12), (1, 2500, 2, 32, 48)]   # the last one walked in parts


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["fused", "time"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_under_hooks(dev, shape, layout, dtype):
    print("hooks", shape, layout, dtype, flush=True)
    c = case(dev, 60, *shape, dtype, layout, 30)
    c["reset"] = c["reset"].t().contiguous().t()
    want = gradients(c)
    hooks = torch.autograd.graph.saved_tensors_hooks
    for under in (hooks(lambda x: x.detach().clone(), lambda x: x), hooks(lambda x: x, turned),
                  torch.autograd.graph.save_on_cpu()):
        assert all(torch.equal(x, y) for x, y in zip(gradients(c, under), want))


def test_saved_tensors_left_on_the_host_are_refused(dev):
    c = case(dev, 61, 2, 40, 2, 16, 16, F32, "fused", 10)
    for which in (lambda x: x.dim() == 4, lambda x: x.dim() == 1, lambda x: x.dtype == torch.bool):
        def unpack(x):
            return x.detach().cpu() if which(x) else x

        with pytest.raises(ValueError):
            gradients(c, torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack))
    long = case(dev, 62, 1, 2500, 1, 16, 16, F32, "fused", 0)
    with pytest.raises(ValueError):
        gradients(long, torch.autograd.graph.saved_tensors_hooks(
            lambda x: x, lambda x: x.cpu() if x.dtype == torch.uint8 else x))


def test_forward_mode_derivatives_are_refused(dev):
    """A dual tensor asks for a derivative along its tangent, which nothing here gives; a level without
    dual tensors changes nothing."""
    from torch.autograd import forward_ad

    from hipenvs import decay_attention

    c = case(dev, 63, 2, 9, 2, 8, 4, F32, "apart", 3)
    want = decay_attention.sequence(**c)
    one = [c[n][:, 0].contiguous() for n in ("q", "k", "v")] + [c["log_decay"], c["state"].clone()]
    stepped = decay_attention.step(*one)
    with forward_ad.dual_level():
        assert all(torch.equal(x, y) for x, y in zip(decay_attention.sequence(**c), want))
        assert all(torch.equal(x, y) for x, y in zip(decay_attention.step(*one), stepped))
        for n in ("q", "k", "v", "log_decay", "state"):
            dual = forward_ad.make_dual(c[n], torch.ones_like(c[n]))
            with pytest.raises(ValueError, match="forward-mode"):
                decay_attention.sequence(**{**c, n: dual})
            leaf = c["q"].detach().requires_grad_()
            if n != "q":
                with pytest.raises(ValueError, match="forward-mode"):
                    decay_attention.sequence(**{**c, "q": leaf, n: dual})
        for i in range(5):
            dual = forward_ad.make_dual(one[i], torch.ones_like(one[i]))
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                decay_attention.step(*one[:i], dual, *one[i + 1:])
        into = forward_ad.make_dual(one[4].clone(), torch.ones_like(one[4]))
        version = into._version
        with pytest.raises(ValueError, match="forward-mode"):
            decay_attention.step(*one, next_state=into)
        assert into._version == version
        leaf = c["q"].detach().requires_grad_()
        out, _ = decay_attention.sequence(**{**c, "q": leaf})
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out, leaf, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))
