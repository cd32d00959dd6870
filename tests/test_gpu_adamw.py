"""AdamW over many tensors (GPU): 32-bit moments against the formula in float64, every code of
8-bit moments against numpy float32, operation by operation.

Bounds of the 32-bit form: m and v are sums of two products, 3 units of 2^-24 of the sum of
their magnitudes; a parameter is keep p (2 units) minus an update whose value carries the
relative error of m (in units of its magnitudes), of sqrt(v) and of six operations.
"""

import numpy as np
import pytest
import torch

from oracle import adamw as oad

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
HYPER = {"lr": 3e-3, "betas": (0.9, 0.99), "eps": 1e-7, "weight_decay": 0.05}
SHAPES = [(1,), (3, 5), (256,), (257,), (0, 4), (1023,), (64, 65), (4, 1024), (7, 11, 13), (40000,)]


def tensors(dev, seed, shapes=SHAPES, p_type=F32, g_type=F32):
    gen = torch.Generator().manual_seed(seed)
    params = [torch.randn(s, generator=gen).to(p_type).to(dev) for s in shapes]
    grads = [(torch.randn(s, generator=gen) * 10.0 ** -(i % 4)).to(g_type).to(dev) for i, s in enumerate(shapes)]
    return params, grads


def offsets(params):
    at = [0]
    for p in params:
        at.append(at[-1] + -(-p.numel() // 256) * 256)
    return at


def f64(x):
    return x.detach().double().cpu().numpy().reshape(-1)


def f32(x):
    return x.detach().float().cpu().numpy().reshape(-1)


def check32(params, grads, before, moments, old, t):
    """params and moments after one step against the formula on what was before."""
    at = offsets(params)
    b1, b2 = HYPER["betas"]
    for i, (p, g, q) in enumerate(zip(params, grads, before)):
        part = slice(at[i], at[i] + p.numel())
        m0, v0 = f64(old[0][part]), f64(old[1][part])
        want_p, want_m, want_v = oad.step64(f64(q), f64(g), m0, v0, t, **HYPER)
        size_m = b1 * np.abs(m0) + (1 - b1) * np.abs(f64(g))
        assert np.all(np.abs(f64(moments[0][part]) - want_m) <= 4 * U * size_m + 1e-45)
        assert np.all(np.abs(f64(moments[1][part]) - want_v) <= 5 * U * want_v + 1e-44)
        root = np.sqrt(want_v / (1 - b2 ** t)) + HYPER["eps"]
        update = HYPER["lr"] / (1 - b1 ** t) * size_m / root
        bound = 4 * U * np.abs(f64(q)) + 16 * U * update + U * np.abs(want_p)
        if p.dtype == BF16:
            bound = bound + 2.0 ** -8 * np.abs(want_p) * (1 + 2.0 ** -6)   # 8 significant bits
        assert np.all(np.abs(f64(p) - want_p) <= bound + 1e-44), i
        assert not f64(moments[0][at[i] + p.numel():at[i + 1]]).any()


@pytest.mark.parametrize("p_type", [F32, BF16])
@pytest.mark.parametrize("g_type", [F32, BF16])
def test_steps_match_the_formula(dev, p_type, g_type):
    from hipenvs import adamw

    params, grads = tensors(dev, 1, p_type=p_type, g_type=g_type)
    moments = adamw.init(params)
    for t in range(1, 5):
        before, old = [p.clone() for p in params], [x.clone() for x in moments]
        kept = [g.clone() for g in grads]
        adamw.step(params, grads, moments, t, **HYPER)
        check32(params, grads, before, moments, old, t)
        assert all(torch.equal(g, k) for g, k in zip(grads, kept))
        grads = [g * (-0.7) for g in grads]


def test_mixed_types_and_alignments(dev):
    """Tensors that start one element past every alignment, of all four mixes of types."""
    from hipenvs import adamw

    def shifted(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=dev)
        flat[1:] = x.reshape(-1)
        return flat[1:].view(x.shape)

    params, grads = tensors(dev, 2)
    kinds = [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)]
    params = [p.to(kinds[i % 4][0]) for i, p in enumerate(params)]
    grads = [g.to(kinds[i % 4][1]) for i, g in enumerate(grads)]
    for bits in (32, 8):
        straight = [p.clone() for p in params]
        odd = [shifted(p) for p in params]
        a, b = adamw.init(params, bits), adamw.init(params, bits)
        for t in (1, 2):
            adamw.step(straight, grads, a, t, **HYPER)
            adamw.step(odd, [shifted(g) for g in grads], b, t, **HYPER)
        assert all(torch.equal(x, y) for x, y in zip(straight, odd))
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    flat = torch.zeros(offsets(params)[-1] + 1, device=dev)   # 32-bit moments off their 16 bytes
    c = (flat[1:].clone(), torch.zeros_like(flat)[1:])
    odd, straight = [p.clone() for p in params], [p.clone() for p in params]
    adamw.step(odd, grads, c, 1, **HYPER)
    a = adamw.init(params)
    adamw.step(straight, grads, a, 1, **HYPER)
    assert all(torch.equal(x, y) for x, y in zip((*odd, *c), (*straight, *a)))


def test_more_tensors_than_a_launch_takes(dev):
    """200 tensors of odd sizes equal 200 steps of one tensor each."""
    from hipenvs import adamw

    shapes = [(1 + 37 * i % 900,) for i in range(200)]
    for bits in (32, 8):
        params, grads = tensors(dev, 3, shapes)
        alone = [p.clone() for p in params]
        moments = adamw.init(params, bits)
        adamw.step(params, grads, moments, 3, **HYPER)
        for i, p in enumerate(alone):
            own = adamw.init([p], bits)
            adamw.step([p], [grads[i]], own, 3, **HYPER)
            assert torch.equal(p, params[i]), i


def test_tensors_without_a_gradient_stay(dev):
    from hipenvs import adamw

    for bits in (32, 8):
        params, grads = tensors(dev, 4)
        opt = adamw.AdamW(params, lr=1e-2, bits=bits)
        opt.step(grads)
        kept, old = [p.clone() for p in params], [x.clone() for x in adamw.decode(opt.moments)]
        some = [g if i % 2 else None for i, g in enumerate(grads)]
        opt.step(some)
        assert opt.steps == [1 + i % 2 for i in range(len(params))]
        at, now = offsets(params), adamw.decode(opt.moments)
        for i, (p, k) in enumerate(zip(params, kept)):
            part = slice(at[i], at[i + 1])
            same = torch.equal(p, k) and all(torch.equal(x[part], y[part]) for x, y in zip(now, old))
            assert same == (i % 2 == 0 or p.numel() == 0), i


def test_step_numbers_of_their_own(dev):
    from hipenvs import adamw

    params, grads = tensors(dev, 5)
    alone, moments = [p.clone() for p in params], adamw.init(params)
    adamw.step(params, grads, moments, [1 + 3 * i for i in range(len(params))], **HYPER)
    for i, p in enumerate(alone):
        adamw.step([p], [grads[i]], adamw.init([p]), 1 + 3 * i, **HYPER)
        assert torch.equal(p, params[i])


def reference8(codes, g, betas):
    """Codes and scales after gradient g (blocks, 256), and the moments before rounding, in numpy float32."""
    m, v = oad.moved(g, oad.decode_m(codes[0], codes[2]), oad.decode_v(codes[1], codes[3]), betas)
    (mc, ms), (vc, vs) = oad.encode_m(m), oad.encode_v(v)
    return (mc, vc, ms, vs), m, v


@pytest.mark.parametrize("p_type,g_type", [(F32, F32), (BF16, BF16)])
def test_codes_of_8_bit_moments(dev, p_type, g_type):
    """Several steps: every code and scale as numpy float32 gives it, parameters within the
    rounding of their update, and the read-back moments."""
    from hipenvs import adamw

    params, grads = tensors(dev, 6, [(5000,), (3,), (256, 3), (70001,)], p_type, g_type)
    moments = adamw.init(params, 8)
    at = offsets(params)
    blocks = at[-1] // 256
    codes = (np.zeros((blocks, 256), np.int8), np.zeros((blocks, 256), np.uint8), np.zeros(blocks, np.float32),
             np.zeros(blocks, np.float32))
    for t in range(1, 6):
        flat = np.zeros(at[-1], np.float32)
        for i, g in enumerate(grads):
            flat[at[i]:at[i] + g.numel()] = f32(g)
        before = [f32(p) for p in params]
        adamw.step(params, grads, moments, t, **HYPER)
        codes, m, v = reference8(codes, flat.reshape(-1, 256), HYPER["betas"])
        for got, want in zip(moments, codes):
            assert np.array_equal(got.cpu().numpy().reshape(want.shape), want), t
        back = adamw.decode(moments)
        assert np.array_equal(f32(back[0]).reshape(-1, 256), oad.decode_m(codes[0], codes[2]))
        assert np.array_equal(f32(back[1]).reshape(-1, 256), oad.decode_v(codes[1], codes[3]))
        for i, p in enumerate(params):
            part = slice(at[i], at[i] + p.numel())
            want = oad.updated(before[i], m.reshape(-1)[part], v.reshape(-1)[part], t, **HYPER)
            got = torch.from_numpy(want).to(p_type).float().numpy()
            assert np.array_equal(f32(p), got), (t, i)
        grads = [g * (0.5 + 0.3 * t) * (-1) ** t for g in grads]


def test_8_bit_moments_hold_their_values(dev):
    """A value reads back within half a step of its code's root: |root error| <= 0.5 / 127 (m, whose
    root is |m / A|^(1/2)) and 0.5 / 255 (v, (v / A)^(1/4)), except what v's smallest code raises."""
    from hipenvs import adamw

    params, grads = tensors(dev, 7, [(100000,)])
    a, b = adamw.init(params, 32), adamw.init(params, 8)
    twin = [p.clone() for p in params]
    adamw.step(params, grads, a, 1, **HYPER)
    adamw.step(twin, grads, b, 1, **HYPER)
    assert torch.equal(params[0], twin[0])   # from the moments before they are rounded
    (m, v), (m8, v8) = ([f64(x).reshape(-1, 256) for x in y] for y in (a, adamw.decode(b)))
    top_m, top_v = np.abs(m).max(1, keepdims=True), v.max(1, keepdims=True)
    assert np.all(np.abs(np.sqrt(np.abs(m8) / top_m) - np.sqrt(np.abs(m) / top_m)) <= 0.5 / 127 + 1e-6)
    quart = (v8 / top_v) ** 0.25, (v / top_v) ** 0.25
    raised = np.where(v > 0, np.maximum(quart[1], 1 / 255), 0)
    assert np.all(np.abs(quart[0] - raised) <= 0.5 / 255 + 1e-6)
    assert np.all((v8 > 0) == (v > 0))


def test_values_that_are_not_finite_stay_in_their_place(dev):
    """32 bits: in their element. 8 bits: in their block's moments; parameters elsewhere in the
    block still get this step's update. Zero and subnormal blocks read back as they are held."""
    from hipenvs import adamw

    for bad in (float("nan"), float("inf"), -float("inf")):
        params, grads = tensors(dev, 8, [(1000,)])
        grads[0][300] = bad
        for bits in (32, 8):
            p = [params[0].clone()]
            moments = adamw.init(p, bits)
            adamw.step(p, grads, moments, 1, **HYPER)
            rest = torch.arange(1000, device=dev) != 300
            assert torch.isfinite(p[0][rest]).all() and not torch.isfinite(p[0][~rest]).any()
            m, v = adamw.decode(moments)
            inside = torch.zeros(m.numel(), dtype=torch.bool, device=dev)
            if bits == 32:
                inside[300] = True
            else:
                inside[256:512] = True
            for x in (m, v):
                assert torch.isfinite(x[~inside]).all() and not torch.isfinite(x[inside]).any()
    p, g = [torch.ones(600, device=dev)], [torch.zeros(600, device=dev)]
    moments = adamw.init(p, 8)
    adamw.step(p, g, moments, 1, **HYPER)
    assert all(not x.any() for x in moments) and torch.isfinite(p[0]).all()
    g[0][:] = 1e-38   # m below the normal numbers, v zero
    adamw.step(p, g, moments, 2, **HYPER)
    m, v = adamw.decode(moments)
    assert torch.isfinite(m).all() and not v.any()
    assert m[:600].min() > 0.9e-39 and m[:600].max() < 1.1e-39


def test_betas_and_weight_decay_at_their_ends(dev):
    from hipenvs import adamw

    params, grads = tensors(dev, 9)
    for betas, wd in (((0.0, 0.0), 0.0), ((0.0, 0.999), 1.0)):
        hyper = {"lr": 1e-2, "betas": betas, "eps": 1e-8, "weight_decay": wd}
        p, moments = [x.clone() for x in params], adamw.init(params)
        adamw.step(p, grads, moments, 1, **hyper)
        for x, y, g in zip(p, params, grads):
            want = oad.step64(f64(y), f64(g), 0.0 * f64(g), 0.0 * f64(g), 1, **hyper)[0]
            assert np.all(np.abs(f64(x) - want) <= 20 * U * (np.abs(f64(y)) + 1e-2 + np.abs(want)))


def test_strided_gradients_and_repeated_runs(dev):
    from hipenvs import adamw

    p = [torch.randn(30, 40, generator=torch.Generator().manual_seed(1)).to(dev)]
    g = torch.randn(40, 30, generator=torch.Generator().manual_seed(2)).to(dev)
    a, b = [p[0].clone()], [p[0].clone()]
    adamw.step(a, [g.t()], adamw.init(a), 1)
    adamw.step(b, [g.t().contiguous()], adamw.init(b), 1)
    assert torch.equal(a[0], b[0])
    c = [p[0].clone()]
    adamw.step(c, [torch.ones(1, device=dev).expand(30, 40)], adamw.init(c), 1)
    assert torch.isfinite(c[0]).all() and not torch.equal(c[0], p[0])


def test_class_follows_the_function_and_marks_what_it_writes(dev):
    from hipenvs import _lib, adamw

    w = torch.randn(8, 8, generator=torch.Generator().manual_seed(1)).to(dev).requires_grad_()
    x = torch.randn(5, 8, generator=torch.Generator().manual_seed(2)).to(dev)
    twin, moments = [w.detach().clone()], adamw.init([w])
    opt = adamw.AdamW([w], lr=1e-2)
    for t in (1, 2, 3):
        ((x @ w).tanh().square().sum()).backward()
        adamw.step(twin, [w.grad], moments, t, lr=1e-2)
        opt.step()
        opt.zero_grad()
        assert torch.equal(w.detach(), twin[0])
    late = (w * w).sum()
    opt.step([torch.ones_like(w)])
    with pytest.raises(RuntimeError):   # the product's saved factor has changed since
        late.backward()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.HipEnvsError):
        with torch.cuda.graph(graph):
            opt.step([torch.ones_like(w)])


def test_a_tensor_past_32_bits(dev):
    """2^32 + 1025 parameters in bfloat16 with 8-bit moments: its first and last values move as a
    short tensor's do."""
    from hipenvs import adamw

    n = (1 << 32) + 1025
    p, g = torch.ones(n, dtype=BF16, device=dev), torch.zeros(n, dtype=BF16, device=dev)
    moments = adamw.init([p], 8)
    short_p, short_g = torch.ones(1025, dtype=BF16, device=dev), torch.linspace(-1, 1, 1025, device=dev).to(BF16)
    g[:1025] = short_g
    g[-1025:] = short_g
    adamw.step([p], [g], moments, 1, lr=0.1)
    adamw.step([short_p], [short_g], adamw.init([short_p], 8), 1, lr=0.1)
    assert torch.equal(p[:1025], short_p) and torch.equal(p[-1025:], short_p)
    assert int(moments[0][1 << 20]) == 0 and float(p[1 << 31]) == float(p[1 << 22])
    m, v = adamw.decode(moments)
    short = adamw.init([short_p], 8)
    adamw.step([short_p], [short_g], short, 1, lr=0.1)
    for x, y in zip((m, v), adamw.decode(short)):   # the last 1025 values share their blocks' scale with zeros
        assert torch.equal(x[:1025], y[:1025]) and torch.equal(x[-1280:][:1025], x[n - 1025:n])
    assert m[n - 1025:n].abs().max() == m[:1025].abs().max() and not m[1 << 31:(1 << 31) + 4096].any()


def test_refusals_on_the_device(dev):
    from hipenvs import adamw

    p, g = tensors(dev, 10, [(10,), (4, 4)])
    m = adamw.init(p)
    for bad in (lambda: adamw.step(p, g[:1], m, 1), lambda: adamw.step(p, g, m, 0),
                lambda: adamw.step(p, g, m, [1]), lambda: adamw.step(p, [g[0], g[0]], m, 1),
                lambda: adamw.step(p, [g[0].cpu(), g[1]], m, 1), lambda: adamw.step([p[0], p[1].t()[:, :2]], g, m, 1),
                lambda: adamw.step(p, g, (m[0][:256], m[1]), 1), lambda: adamw.step(p, g, m, 1, betas=(1.0, 0.9)),
                lambda: adamw.step(p, g, m, 1, eps=-1.0), lambda: adamw.step([p[0], p[0]], [g[0], g[0]], m, 1),
                lambda: adamw.step(p, g, m[:1], 1), lambda: adamw.init(p, 4)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: adamw.step([p[0].double(), p[1]], g, m, 1), lambda: adamw.step(p, [g[0].half(), g[1]], m, 1),
                lambda: adamw.step(p, g, (m[0].double(), m[1]), 1)):
        with pytest.raises(TypeError):
            bad()
    adamw.step([], [], (), 1)


def test_a_captured_step(dev):
    """adamw.step in a graph (its step number the captured one), replayed with new gradients and the
    program's own work between, against the same calls made eagerly."""
    from hipenvs import adamw

    for bits in (32, 8):
        params, grads = tensors(dev, 11)
        twin = [p.clone() for p in params]
        a, b = adamw.init(params, bits), adamw.init(params, bits)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            adamw.step(params, grads, a, 7, **HYPER)
        for k in range(4):
            for g in grads:
                g.mul_(-0.8 - 0.1 * k)
            graph.replay()
            torch.cuda.synchronize()
            adamw.step(twin, grads, b, 7, **HYPER)
            assert all(torch.equal(x, y) for x, y in zip((*params, *a), (*twin, *b))), (bits, k)
