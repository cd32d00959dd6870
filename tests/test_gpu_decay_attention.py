"""Decay attention (GPU): outputs, states and gradients against the definition in float64.

Error bounds. A is the same sum over the magnitudes of its terms. In float32 a term meets at
most T + dk + dv roundings of a running sum, product or decay, and its decay lambda^n carries
the rounding of n * log_decay, at most 104 units before lambda^n is zero: GAMMA below, twice
that for the matrix instructions, which need not round to nearest. With bfloat16 inputs a term
of an output or a gradient is rounded to bfloat16 twice at most (a weight or a state, 2^-8
each: 8 significant bits) and the result once; states and their gradients are float32 results throughout.
"""

import numpy as np
import pytest
import torch

from oracle import decay_attention as oda

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def gamma(t, dk, dv):
    return 2.0 * (t + dk + dv + 256) * 2.0 ** -24


def close(got, want, size, dtype, t, dk, dv):
    """got within the bound of `want` for terms of summed magnitude `size`, everywhere."""
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape
    bound = gamma(t, dk, dv) * size
    if dtype == BF16:
        bound = bound + 2.0 ** -7 * size + 2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -6)
    off = np.abs(got - want) - bound
    assert np.all(off <= 1e-37), f"{off.max()} over the bound, worst {np.abs(got - want).max()} of {np.abs(want).max()}"


def case(dev, seed, b, t, h, dk, dv, dtype, layout="apart", episode=7, state=True):
    gen = torch.Generator().manual_seed(seed)

    def rows(d):
        return torch.randn(b, t, h, d, generator=gen).to(dtype)

    q, k, v = rows(dk), rows(dk), rows(dv)
    if layout == "time":
        q, k, v = (x.transpose(0, 1).contiguous().to(dev).transpose(0, 1) for x in (q, k, v))
    elif layout == "fused":
        both = torch.cat([x.flatten(2) for x in (q, k, v)], -1).to(dev)
        q, k, v = (x.unflatten(-1, (h, -1)) for x in torch.split(both, (h * dk, h * dk, h * dv), -1))
    elif layout == "odd":   # one element past every alignment
        def shifted(x):
            flat = torch.empty(x.numel() + 1, dtype=dtype, device=dev)
            flat[1:] = x.reshape(-1).to(dev)
            return flat[1:].view(x.shape)
        q, k, v = shifted(q), shifted(k), shifted(v)
    else:
        q, k, v = q.to(dev), k.to(dev), v.to(dev)
    log_decay = torch.log1p(-(2.0 ** -torch.linspace(1.0, 8.0, h)))
    reset = (torch.rand(b, t, generator=gen) < 1.0 / episode) if episode else None
    s = torch.randn(b, h, dk, dv, generator=gen) if state else None
    return {"q": q, "k": k, "v": v, "log_decay": log_decay.to(dev), "state": s.to(dev) if state else None,
            "reset": reset.to(dev) if episode else None}


def to_np(x):
    return None if x is None else x.detach().cpu().numpy() if x.dtype == torch.bool else x.detach().double().cpu().numpy()


def check_forward(c, scale=None):
    from hipenvs import decay_attention

    b, t, h, dk = c["q"].shape
    dv = c["v"].shape[-1]
    out, final = decay_attention.sequence(**c, scale=scale)
    assert out.dtype == c["q"].dtype and final.dtype == F32 and out.is_contiguous() and final.is_contiguous()
    args = [to_np(c[n]) for n in ("q", "k", "v", "log_decay", "state", "reset")]
    s = dk ** -0.5 if scale is None else scale
    want, size = oda.sequence(*args, s), oda.magnitudes(*args, s)
    close(out, want[0], size[0], c["q"].dtype, t, dk, dv)
    close(final, want[1], size[1], F32, t, dk, dv)
    return out, final


def check_backward(c, seed=5, use_out=True, use_final=True):
    from hipenvs import decay_attention

    b, t, h, dk = c["q"].shape
    dv, dtype = c["v"].shape[-1], c["q"].dtype
    gen = torch.Generator().manual_seed(seed)
    dout = torch.randn(b, t, h, dv, generator=gen).to(dtype).to(c["q"].device)
    dfinal = torch.randn(b, h, dk, dv, generator=gen).to(c["q"].device)
    leaves = {n: c[n].detach().requires_grad_() for n in ("q", "k", "v", "state") if c[n] is not None}
    out, final = decay_attention.sequence(**{**c, **leaves})
    pairs = [(x, g) for x, g, on in ((out, dout, use_out), (final, dfinal, use_final)) if on]
    got = torch.autograd.grad([x for x, _ in pairs], list(leaves.values()), [g for _, g in pairs])
    args = [to_np(c[n]) for n in ("q", "k", "v", "log_decay", "state", "reset")]
    grads = (to_np(dout) * use_out, to_np(dfinal) * use_final)
    want = oda.gradients(*args, dk ** -0.5, *grads)
    size = oda.magnitudes(*args, dk ** -0.5, *grads)[2:]
    for x, n, w, s in zip(got, leaves, want, size):
        assert x.dtype == leaves[n].dtype and x.shape == leaves[n].shape
        close(x, w, s, F32 if n == "state" else dtype, t, dk, dv)
    return dict(zip(leaves, got)), grads


SHAPES = [  # b, t, h, dk, dv
    (1, 1, 1, 1, 1), (3, 2, 2, 5, 3), (2, 63, 3, 32, 32), (2, 64, 1, 16, 64), (1, 65, 2, 64, 16), (5, 127, 2, 33, 31),
    (2, 200, 3, 48, 80), (1, 129, 2, 128, 128), (2, 130, 1, 127, 65), (1, 700, 4, 64, 64), (40, 17, 2, 32, 32),
    (1, 1500, 1, 20, 128),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sequence_and_gradients_match_the_definition(dev, shape, dtype):
    print("decay attention", shape, dtype, flush=True)
    for k, (layout, episode, state) in enumerate((("fused", 7, True), ("time", 0, False), ("odd", 90, True))):
        c = case(dev, k, *shape, dtype, layout, episode, state)
        check_forward(c)
        check_backward(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_rows_and_few_heads(dev, dtype):
    """Rows long enough to be split over the axis, with and without episodes."""
    for episode in (0, 300):
        c = case(dev, 3, 1, 5003, 2, 32, 48, dtype, "fused", episode)
        check_forward(c)
        check_backward(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_short_rows(dev, dtype):
    c = case(dev, 4, 700, 9, 3, 16, 16, dtype, "time", 4)
    check_forward(c)
    check_backward(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dk, dv", [(9, 16), (16, 8), (40, 16), (96, 1), (128, 16), (16, 100)])
def test_a_narrow_side(dev, dk, dv, dtype):
    """Keys or values of at most 16 columns, whose walks have blocks of one wave: short, with a
    ragged end, and long enough for parts."""
    for b, t, episode in ((3, 95, 0), (2, 161, 11), (1, 2500, 400)):
        c = case(dev, 12, b, t, 2, dk, dv, dtype, "fused", episode)
        check_forward(c)
        check_backward(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bad_values_of_narrow_heads(dev, dtype):
    """A NaN in a value row stays within its episode and its column; nothing before it changes."""
    from hipenvs import decay_attention

    c = case(dev, 13, 2, 200, 2, 32, 16, dtype, "apart", 0)
    c["reset"] = torch.zeros(2, 200, dtype=torch.bool, device=dev)
    c["reset"][:, 90] = c["reset"][:, 150] = True
    spoilt = {**c, "v": c["v"].clone()}
    spoilt["v"][0, 100, 1, 5] = float("nan")
    out, final = decay_attention.sequence(**spoilt)
    touched = torch.zeros(2, 200, 2, 16, dtype=torch.bool, device=dev)
    touched[0, 100:150, 1, 5] = True
    assert torch.isnan(out[touched]).all()
    args = [to_np(c[n]) for n in ("q", "k", "v", "log_decay", "state", "reset")]
    want, size = oda.sequence(*args, 32 ** -0.5), oda.magnitudes(*args, 32 ** -0.5)
    mask = touched.cpu().numpy()
    close(out[~touched], want[0][~mask], size[0][~mask], dtype, 200, 32, 16)
    close(final, want[1], size[1], F32, 200, 32, 16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_only_one_of_the_results_is_used(dev, dtype):
    c = case(dev, 6, 2, 100, 2, 32, 32, dtype, "apart", 30)
    check_backward(c, use_final=False)
    check_backward(c, use_out=False)


@pytest.mark.parametrize("pattern", ["all", "first", "last", "borders", "beyond"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_reset_patterns(dev, pattern, dtype):
    """Every token its own episode; a reset on the first or last token; on every border of 16 and 64."""
    c = case(dev, 7, 2, 193, 2, 32, 24, dtype, "apart", 7)
    r = torch.zeros(2, 193, dtype=torch.bool)
    if pattern == "all":
        r[:] = True
    elif pattern == "first":
        r[:, 0] = True
    elif pattern == "last":
        r[:, -1] = True
    elif pattern == "borders":
        r[0, ::64] = True
        r[1, 16::16] = True
    else:
        r[:, 1::64] = True
        r[:, 63::64] = True
    c["reset"] = r.to(dev)
    check_forward(c)
    check_backward(c)


@pytest.mark.parametrize("decays", [[0.0, -1e-6], [-float("inf"), -200.0], [-5.0, -0.693147], [0.001, -0.01]])
def test_extreme_decays(dev, decays):
    """No decay at all, one that leaves only the token itself, very fast ones, a slow growth."""
    for dtype in (F32, BF16):
        c = case(dev, 8, 2, 150, 2, 16, 16, dtype, "apart", 40)
        c["log_decay"] = torch.tensor(decays, device=dev)
        check_forward(c)
        check_backward(c)


def test_scale_and_reset_views(dev):
    c = case(dev, 9, 3, 70, 2, 16, 32, F32)
    c["reset"] = c["reset"].t().contiguous().t()
    check_forward(c, scale=-0.3)
    c["reset"] = torch.zeros(3, 1, dtype=torch.bool, device=dev).expand(3, 70)
    check_forward(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_an_earlier_episode_or_a_later_token_holds_does_not_reach(dev, dtype, bad):
    """A row's bad values at one token: outputs before it, and after the next reset, are those of
    the row without them, within the rounding of a sum in another order; likewise its gradients."""
    from hipenvs import decay_attention

    for name in ("q", "k", "v", "dout"):
        c = case(dev, 10, 2, 200, 2, 32, 32, dtype, "apart", 0)
        r = torch.zeros(2, 200, dtype=torch.bool, device=dev)
        r[:, 40] = r[:, 90] = r[:, 150] = True
        c["reset"] = r
        dout = torch.randn(2, 200, 2, 32, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
        at = 100   # in the episode of tokens 90 .. 149

        def grads(cc, d):
            leaves = {n: cc[n].detach().requires_grad_() for n in ("q", "k", "v", "state")}
            out, final = decay_attention.sequence(**{**cc, **leaves})
            return out.detach(), final.detach(), *torch.autograd.grad(out, list(leaves.values()), d)

        clean = grads(c, dout)
        spoilt, d = dict(c), dout
        if name == "dout":
            d = dout.clone()
            d[0, at, 1, 5] = bad
        else:
            spoilt[name] = c[name].clone()
            spoilt[name][0, at, 1, 5] = bad
        got = grads(spoilt, d)
        for x, y in zip(got[2:5] + got[:1], clean[2:5] + clean[:1]):
            inside = torch.zeros_like(y, dtype=torch.bool)
            inside[0, 90:150, 1] = True
            assert torch.isfinite(x[~inside]).all(), name
            tol = 2.0 ** -7 if dtype == BF16 else 1e-4
            assert torch.allclose(x[~inside].float(), y[~inside].float(), rtol=tol, atol=tol), name
        assert torch.isfinite(got[1]).all() and torch.isfinite(got[5]).all(), name
        before = got[0][0, 90:at, 1]
        if name in ("q", "k", "v"):   # causal: outputs of the same episode before the token
            assert torch.isfinite(before).all(), name
        if name in ("k", "v"):
            assert not torch.isfinite(got[0][0, at, 1]).all(), name
        if name == "q":
            assert not torch.isfinite(got[0][0, at, 1]).all()
            assert torch.isfinite(got[0][0, at + 1:150, 1]).all()
            assert torch.isfinite(got[3][0, at + 1:150, 1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bad_values_in_rows_walked_in_parts(dev, dtype):
    """A long row: a NaN in its value rows inside one part, an infinity in another, each ended by a
    reset: everything after the resets, and every other head and row, is as without them."""
    from hipenvs import decay_attention

    c = case(dev, 30, 2, 3000, 2, 32, 48, dtype, "apart", 0)
    c["reset"] = torch.zeros(2, 3000, dtype=torch.bool, device=dev)
    c["reset"][0, 700] = c["reset"][0, 1500] = c["reset"][0, 2200] = True
    clean = decay_attention.sequence(**c)
    spoilt = {**c, "v": c["v"].clone(), "k": c["k"].clone()}
    spoilt["v"][0, 650, 1, 3] = float("nan")
    spoilt["k"][0, 1490, 1, 5] = float("inf")
    got = decay_attention.sequence(**spoilt)
    touched = torch.zeros(2, 3000, 2, dtype=torch.bool, device=dev)
    touched[0, 650:700, 1] = touched[0, 1490:1500, 1] = True
    assert not torch.isfinite(got[0][touched].float()).all()
    args = [to_np(c[n]) for n in ("q", "k", "v", "log_decay", "state", "reset")]
    want, size = oda.sequence(*args, 32 ** -0.5), oda.magnitudes(*args, 32 ** -0.5)
    mask = touched.cpu().numpy()
    for x in (got, clean):
        close(x[0][~touched], want[0][~mask], size[0][~mask], dtype, 3000, 32, 48)
        close(x[1], want[1], size[1], F32, 3000, 32, 48)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_backward_with_and_without_the_forward_s_states(dev, dtype):
    """The C entry point computes the states between parts again where it is given none."""
    import ctypes

    from hipenvs import _lib, decay_attention

    b, t, h, dk, dv = 2, 3000, 2, 32, 48
    c = case(dev, 31, b, t, h, dk, dv, dtype, "fused", 700)
    code = decay_attention._DTYPES[dtype]
    need = _lib.lib().hipenvs_decay_attention_workspace_bytes(code, b, t, h, dk, dv)
    assert need > 0
    gen = torch.Generator().manual_seed(2)
    dout = torch.randn(b, t, h, dv, generator=gen).to(dtype).to(dev)
    out, final, states = decay_attention._forward(c["q"], c["k"], c["v"], c["log_decay"], c["state"], c["reset"], 0.2)
    assert states.numel() == need
    args = [to_np(c[n]) for n in ("q", "k", "v", "log_decay", "state", "reset")]
    want = oda.gradients(*args, 0.2, to_np(dout), None)
    size = oda.magnitudes(*args, 0.2, to_np(dout), None)[2:]
    for given in (states, None):
        grads = [torch.empty(b, t, h, d, dtype=dtype, device=dev) for d in (dk, dk, dv)]
        dstate = torch.empty(b, h, dk, dv, device=dev)
        work = torch.empty(need, dtype=torch.uint8, device=dev)
        strides = decay_attention._strides((c["q"], c["k"], c["v"], dout), c["reset"])
        _lib.call("hipenvs_decay_attention_backward", code, *(_lib.ptr(c[n]) for n in "qkv"), _lib.ptr(dout), strides,
                  _lib.ptr(c["log_decay"]), _lib.ptr(c["state"]), _lib.ptr(c["reset"]), None, _lib.ptr(given), 0.2,
                  *(_lib.ptr(g) for g in grads), _lib.ptr(dstate), b, t, h, dk, dv, _lib.ptr(work), need,
                  _lib.stream_of(dev))
        for x, w, s in zip((*grads, dstate), want, size):
            close(x, w, s, x.dtype, t, dk, dv)
    rc = _lib.lib().hipenvs_decay_attention(code, *(_lib.ptr(c[n]) for n in "qkv"), strides, _lib.ptr(c["log_decay"]),
                                            None, None, 0.2, _lib.ptr(out), _lib.ptr(final), b, t, h, dk, dv,
                                            _lib.ptr(states), need - 1, None)
    assert rc == _lib.E_ARG   # a workspace too small


def test_a_captured_sequence(dev):
    """A long row's three launches in a graph, replayed with the program's own work between."""
    from hipenvs import decay_attention

    c = case(dev, 32, 1, 2500, 2, 32, 32, BF16, "apart", 300)
    decay_attention.sequence(**c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, final = decay_attention.sequence(**c)
    for seed in range(4):
        other = case(dev, 33 + seed, 1, 2500, 2, 32, 32, BF16, "apart", 300)
        for n in ("q", "k", "v", "state", "reset"):
            c[n].copy_(other[n])
        graph.replay()
        torch.cuda.synchronize()
        want = decay_attention.sequence(**other)
        assert torch.equal(out, want[0]) and torch.equal(final, want[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_state_that_is_not_finite_ends_at_the_reset(dev, dtype):
    c = case(dev, 11, 2, 90, 2, 16, 16, dtype, "apart", 0)
    c["state"][0, 1] = float("nan")
    c["reset"] = torch.zeros(2, 90, dtype=torch.bool, device=dev)
    c["reset"][:, 30] = True
    from hipenvs import decay_attention

    out, final = decay_attention.sequence(**c)
    assert torch.isnan(out[0, :30, 1]).all() and torch.isfinite(out[0, 30:, 1]).all()
    assert torch.isfinite(out[0, :, 0]).all() and torch.isfinite(out[1]).all() and torch.isfinite(final).all()


def test_empty_batches_and_sequences(dev):
    from hipenvs import decay_attention

    for b, t in ((0, 5), (3, 0), (0, 0)):
        c = case(dev, 12, b, t, 2, 8, 4, F32, "apart", 7)
        out, final = decay_attention.sequence(**c)
        assert out.shape == (b, t, 2, 4)
        assert torch.equal(final, c["state"])
        check_backward(c)
        c["state"] = None
        assert not decay_attention.sequence(**c)[1].any()
    s = torch.zeros(0, 2, 8, 4, device=dev)
    out, nxt = decay_attention.step(torch.zeros(0, 2, 8, device=dev), torch.zeros(0, 2, 8, device=dev),
                                    torch.zeros(0, 2, 4, device=dev), torch.zeros(2, device=dev), s)
    assert out.shape == (0, 2, 4) and nxt.shape == s.shape


def test_shared_keys_and_values(dev):
    """One key and value head for all queries (stride 0): its gradient is the heads' sum."""
    from hipenvs import decay_attention

    c = case(dev, 13, 2, 80, 4, 16, 24, F32, "apart", 20)
    one_k, one_v = (c[n][:, :, :1].detach().clone().requires_grad_() for n in ("k", "v"))
    out, _ = decay_attention.sequence(c["q"], one_k.expand(-1, -1, 4, -1), one_v.expand(-1, -1, 4, -1), c["log_decay"],
                                      c["state"], c["reset"])
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).to(dev)
    gk, gv = torch.autograd.grad(out, (one_k, one_v), dout)
    args = [to_np(x) for x in (c["q"], one_k.expand(-1, -1, 4, -1), one_v.expand(-1, -1, 4, -1), c["log_decay"],
                               c["state"], c["reset"])]
    want = oda.gradients(*args, 0.25, to_np(dout), None)
    size = oda.magnitudes(*args, 0.25, to_np(dout), None)[2:]
    close(gk, want[1].sum(2, keepdims=True), size[1].sum(2, keepdims=True), F32, 80, 16, 24)
    close(gv, want[2].sum(2, keepdims=True), size[2].sum(2, keepdims=True), F32, 80, 16, 24)


def test_an_expanded_output_gradient(dev):
    """The gradient of out.sum() is one value with strides 0."""
    from hipenvs import decay_attention

    c = case(dev, 14, 2, 70, 2, 16, 16, F32, "apart", 20)
    q = c["q"].detach().requires_grad_()
    out, _ = decay_attention.sequence(**{**c, "q": q})
    got, = torch.autograd.grad(out.sum(), q)
    args = [to_np(c[n]) for n in ("q", "k", "v", "log_decay", "state", "reset")]
    ones = np.ones((2, 70, 2, 16))
    close(got, oda.gradients(*args, 0.25, ones, None)[0], oda.magnitudes(*args, 0.25, ones, None)[2], F32, 70, 16, 16)


def test_gradients_match_differences(dev):
    """Along random directions, against central differences of the definition in float64."""
    c = case(dev, 15, 2, 90, 2, 12, 20, F32, "apart", 30)
    got, (dout, dfinal) = check_backward(c)
    x = {n: to_np(c[n]) for n in ("q", "k", "v", "log_decay", "state", "reset")}
    rng = np.random.default_rng(0)

    def value(y):
        out, final = oda.sequence(y["q"], y["k"], y["v"], y["log_decay"], y["state"], y["reset"], 12 ** -0.5)
        return (out * dout).sum() + (final * dfinal).sum()

    for n in ("q", "k", "v", "state"):
        u = rng.standard_normal(x[n].shape)
        e = 1e-4   # the sums are at most quadratic in q, k, v, state apart: central differences are exact to rounding
        d = (value({**x, n: x[n] + e * u}) - value({**x, n: x[n] - e * u})) / (2 * e)
        inner = (to_np(got[n]) * u).sum()
        bound = gamma(90, 12, 20) * (np.abs(to_np(got[n])) * np.abs(u)).sum() * 4 + 1e-6 * abs(d)
        assert abs(inner - d) <= bound, (n, inner, d)


def test_the_same_bits_every_time(dev):
    from hipenvs import decay_attention

    for dtype in (F32, BF16):
        c = case(dev, 16, 3, 1100, 2, 64, 64, dtype, "fused", 200)
        first = decay_attention.sequence(**c)
        for _ in range(3):
            again = decay_attention.sequence(**c)
            assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_strides_past_32_bits(dev):
    """Rows 2^32 elements apart."""
    from hipenvs import decay_attention

    far = torch.empty((1 << 32) + 4096, dtype=BF16, device=dev)
    gen = torch.Generator().manual_seed(17)
    near = torch.randn(2, 16, 2, 16, generator=gen).to(BF16).to(dev)
    q = far.as_strided((2, 16, 2, 16), (1 << 32, 32, 16, 1))
    q.copy_(near)
    ld = torch.tensor([-0.1, -0.01], device=dev)
    assert all(torch.equal(x, y) for x, y in zip(decay_attention.sequence(q, q, q, ld),
                                                 decay_attention.sequence(near, near, near, ld)))
    state = torch.zeros(2, 2, 16, 16, device=dev)
    assert torch.equal(decay_attention.step(q[:, 3], q[:, 4], q[:, 5], ld, state)[0],
                       decay_attention.step(near[:, 3], near[:, 4], near[:, 5], ld, state)[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 2, 5, 3), (64, 4, 32, 32), (7, 3, 48, 80), (5, 2, 128, 128),
                                   (9, 1, 31, 127), (300, 2, 64, 64), (4, 3, 100, 4)])
def test_step_matches_the_definition(dev, shape, dtype):
    from hipenvs import decay_attention

    n, h, dk, dv = shape
    print("decay attention step", shape, dtype, flush=True)
    for layout in ("fused", "odd"):
        c = case(dev, 20, n, 1, h, dk, dv, dtype, layout, 2)
        args = [to_np(c[x]) for x in ("q", "k", "v", "log_decay", "state", "reset")]
        want, size = oda.sequence(*args, dk ** -0.5), oda.magnitudes(*args, dk ** -0.5)
        one = (c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"])
        before = c["state"].clone()
        out, nxt = decay_attention.step(*one, c["state"], c["reset"][:, 0])
        assert torch.equal(c["state"], before)
        close(out, want[0][:, 0], size[0][:, 0], dtype, 1, dk, dv)
        close(nxt, want[1], size[1], F32, 1, dk, dv)
        out2, same = decay_attention.step(*one, c["state"], c["reset"][:, 0], next_state=c["state"])
        assert same is c["state"] and torch.equal(same, nxt) and torch.equal(out2, out)


def test_steps_follow_the_sequence(dev):
    """Acting token by token, states in place and not, and over the whole trajectory."""
    from hipenvs import decay_attention

    c = case(dev, 21, 6, 75, 2, 32, 32, F32, "apart", 20)
    args = [to_np(c[x]) for x in ("q", "k", "v", "log_decay", "state", "reset")]
    want, size = oda.sequence(*args, 32 ** -0.5), oda.magnitudes(*args, 32 ** -0.5)
    state = c["state"].clone()
    for t in range(75):
        into = state if t % 2 else None
        out, state = decay_attention.step(c["q"][:, t], c["k"][:, t], c["v"][:, t], c["log_decay"], state,
                                          c["reset"][:, t], next_state=into)
        close(out, want[0][:, t], size[0][:, t], F32, 75, 32, 32)
    close(state, want[1], size[1], F32, 75, 32, 32)


def test_step_leaves_out_what_a_reset_state_holds(dev):
    from hipenvs import decay_attention

    c = case(dev, 22, 4, 1, 2, 16, 16, F32, "apart", 0)
    c["state"][1] = float("nan")
    c["state"][2] = float("inf")
    reset = torch.tensor([False, True, True, True], device=dev)
    out, nxt = decay_attention.step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], c["state"], reset)
    assert torch.isfinite(out).all() and torch.isfinite(nxt).all()
    outer = c["k"][1:, 0, :, :, None] * c["v"][1:, 0, :, None, :]
    assert torch.equal(nxt[1:], outer)


def test_other_streams_and_graphs(dev):
    """A side stream, and a captured acting step replayed with the program's own work between."""
    from hipenvs import decay_attention

    c = case(dev, 23, 8, 40, 2, 32, 32, F32, "apart", 10)
    want = decay_attention.sequence(**c)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = decay_attention.sequence(**c)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))

    q, k, v, r = (c[n][:, 0].clone() for n in ("q", "k", "v", "reset"))
    state = c["state"].clone()
    graph = torch.cuda.CUDAGraph()
    decay_attention.step(q, k, v, c["log_decay"], state, r)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, _ = decay_attention.step(q, k, v, c["log_decay"], state, r, next_state=state)
    state.copy_(c["state"])
    eager = c["state"].clone()
    for t in range(6):
        for x, n in ((q, "q"), (k, "k"), (v, "v"), (r, "reset")):
            x.copy_(c[n][:, t])
        graph.replay()
        torch.cuda.synchronize()
        o, eager = decay_attention.step(c["q"][:, t], c["k"][:, t], c["v"][:, t], c["log_decay"], eager, c["reset"][:, t])
        assert torch.equal(out, o) and torch.equal(state, eager), t


def test_refusals_on_the_device(dev):
    from hipenvs import decay_attention

    c = case(dev, 24, 2, 6, 2, 8, 4, F32)
    ok = [c[n] for n in ("q", "k", "v", "log_decay", "state", "reset")]

    def but(i, x):
        return [*ok[:i], x, *ok[i + 1:]]

    for args, err in ((but(1, ok[1].double()), TypeError), (but(1, ok[1][:, :5]), ValueError),
                      (but(2, ok[2][..., 0]), ValueError), (but(3, ok[3].double()), TypeError),
                      (but(3, ok[3][:1]), ValueError), (but(3, ok[3].clone().requires_grad_()), ValueError),
                      (but(4, ok[4][:1]), ValueError), (but(4, ok[4].bfloat16()), TypeError),
                      (but(5, ok[5].int()), TypeError), (but(5, ok[5][:, :3]), ValueError),
                      (but(1, ok[1].cpu()), ValueError), (but(0, ok[0].half()), TypeError)):
        with pytest.raises(err):
            decay_attention.sequence(*args)
    wide = torch.zeros(1, 2, 1, 129, device=dev)
    with pytest.raises(ValueError):
        decay_attention.sequence(wide, wide, wide, torch.zeros(1, device=dev))
    one = [x[:, 0] for x in ok[:3]]
    with pytest.raises(ValueError):
        decay_attention.step(*one, ok[3], ok[4], next_state=torch.zeros(2, 2, 4, 8, device=dev).transpose(2, 3))
    with pytest.raises(ValueError):
        decay_attention.step(one[0].clone().requires_grad_(), *one[1:], ok[3], ok[4])
    with pytest.raises(TypeError):
        decay_attention.step(*one, ok[3], None)


def test_a_second_derivative_is_refused(dev):
    """create_graph gives the gradient; differentiating that raises."""
    from hipenvs import decay_attention

    c = case(dev, 40, 1, 9, 1, 4, 4, F32, "apart", 0)
    q = c["q"].detach().requires_grad_()
    out, _ = decay_attention.sequence(**{**c, "q": q})
    once, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    plain, = torch.autograd.grad(decay_attention.sequence(**{**c, "q": q})[0].square().sum(), q)
    assert torch.equal(once.detach(), plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(once.sum(), q)


def test_more_states_than_a_launch_takes(dev):
    """17 million states of 1 x 1 a step, and 34 million rows of one token with their gradients: more
    threads than one grid holds. o = q (lambda s + k v), and the products' derivatives."""
    from hipenvs import decay_attention

    n = 17_000_011
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)

    def draw(count, *shape):
        return torch.randn(count, *shape, generator=gen, device=dev)

    ld = torch.zeros(1, device=dev)
    q, k, v, s = draw(n, 1, 1), draw(n, 1, 1), draw(n, 1, 1), draw(n, 1, 1, 1)
    out, nxt = decay_attention.step(q, k, v, ld, s, scale=1.0)
    want = s.flatten() + k.flatten() * v.flatten()
    assert torch.allclose(nxt.flatten(), want, rtol=1e-6, atol=1e-6)
    assert torch.allclose(out.flatten(), q.flatten() * want, rtol=1e-5, atol=1e-5)

    n = 34_000_003
    q, k, v = (draw(n, 1, 1, 1).requires_grad_() for _ in range(3))
    s = draw(n, 1, 1, 1).requires_grad_()
    out, final = decay_attention.sequence(q, k, v, ld, s, scale=1.0)
    do = draw(n, 1, 1, 1)
    grads = torch.autograd.grad(out, (q, k, v, s), do)
    with torch.no_grad():
        state = s + k * v
        for x, y in zip((out, final, *grads), (q * state, state, do * state, do * q * v, do * q * k, do * q)):
            assert torch.allclose(x, y, rtol=1e-5, atol=1e-5)
