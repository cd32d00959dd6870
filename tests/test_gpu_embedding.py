"""The lookup of tokens and its gradient (GPU) against the definition in float64.

An output is one product, rounded once more to bfloat16: half a unit of its type. A row of the
gradient is a float32 sum of as many terms as its token has places, in any order: that many units of
2^-24 of the sum of magnitudes, one for the scale, and half a unit of its type.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def half(dtype):
    return torch.finfo(dtype).eps / 2


def check(tokens, table, scale, dout):
    from hipenvs import embedding

    dtype, (v, d) = table.dtype, table.shape
    leaf = table.detach().requires_grad_()
    out = embedding.lookup(tokens, leaf, scale=scale)
    assert out.shape == (*tokens.shape, d) and out.dtype == dtype
    flat, rows = tokens.flatten().cpu().numpy().astype(np.int64), table.detach().double().cpu().numpy()
    there = (flat >= 0) & (flat < v)
    want = np.zeros((len(flat), d))
    want[there] = rows[flat[there]] * float(np.float32(scale))
    got = out.detach().double().cpu().numpy().reshape(-1, d)
    assert np.isnan(got[flat >= v]).all()
    keep = flat < v
    assert np.all(np.abs(got - want)[keep] <= (2.0 ** -24 + half(dtype) * (dtype == BF16)) * 1.01 * np.abs(want)[keep])
    grad, = torch.autograd.grad(out, leaf, dout)
    assert grad.shape == table.shape and grad.dtype == dtype
    g = dout.double().cpu().numpy().reshape(-1, d)
    sums, size, count = np.zeros((v, d)), np.zeros((v, d)), np.bincount(flat[there], minlength=v)[:, None]
    np.add.at(sums, flat[there], g[there])
    np.add.at(size, flat[there], np.abs(g[there]))
    sums, size = sums * float(np.float32(scale)), size * abs(scale)
    bound = (count + 2) * 2.0 ** -24 * size * 1.01
    bound = bound + (half(dtype) * (np.abs(sums) + bound) if dtype == BF16 else 0.0)
    off = np.abs(grad.double().cpu().numpy() - sums) - bound
    assert np.all(off <= 0), off.max()
    return out.detach(), grad


def make(dev, seed, count, v, d, dtype, wide=True, past=0, absent=0.1, skew=1.0):
    gen = torch.Generator().manual_seed(seed)
    tokens = (v * torch.rand(count, generator=gen, dtype=torch.float64) ** skew).long().clamp(max=v - 1)
    tokens[torch.rand(count, generator=gen) < absent] = -1
    if past and count:
        tokens[::past] = v + torch.arange(len(tokens[::past]))
    return (tokens.to(torch.int64 if wide else torch.int32).to(dev), torch.randn(v, d, generator=gen).to(dtype).to(dev),
            torch.randn(count, d, generator=gen).to(dtype).to(dev))


CASES = [  # tokens, rows of the table, width
    (1, 1, 1), (5, 3, 4), (3000, 16, 300), (3000, 17, 300), (63, 2, 64), (64, 3, 65), (65, 1, 7), (1000, 3, 64), (4097, 255, 3), (5000, 256, 130),
    (9000, 257, 32), (20000, 70000, 12), (3000, 65535, 8), (700, 5, 513), (129, 17000000, 1), (70000, 2, 5), (30000, 65536, 2),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", CASES)
def test_rows_and_their_gradient_match_the_definition(dev, case, dtype):
    for k, (wide, skew, absent) in enumerate(((True, 1.0, 0.1), (False, 4.0, 0.0))):
        print("lookup", case, dtype, wide, flush=True)
        tokens, table, dout = make(dev, k, *case, dtype, wide, skew=skew, absent=absent)
        check(tokens, table, 1.0 if k else 3.3, dout)


def test_tokens_past_the_table_and_none(dev):
    tokens, table, dout = make(dev, 3, 500, 20, 9, F32, past=7)
    check(tokens, table, 2.0, dout)
    check(torch.full_like(tokens, -5), table, 2.0, dout)
    check(torch.full_like(tokens, 20), table, 2.0, dout)
    check(torch.full_like(tokens, 7), table, 2.0, dout)
    check(torch.full_like(tokens, -(1 << 40)), table, 2.0, dout)
    check(torch.full_like(tokens, 1 << 40), table, 2.0, dout)


def test_whole_numbers_are_exact(dev):
    """Sums of whole numbers below 2^24 in any order: every place is added exactly once."""
    from hipenvs import embedding

    gen = torch.Generator().manual_seed(1)
    for count, v, d in ((100000, 5, 16), (100000, 3001, 16), (100000, 100, 64)):
        tokens = torch.randint(-1, v, (count,), generator=gen)
        dout = torch.randint(-30, 31, (count, d), generator=gen).float()
        table = torch.zeros(v, d, device=dev, requires_grad=True)
        grad, = torch.autograd.grad(embedding.lookup(tokens.to(dev), table), table, dout.to(dev))
        want = torch.zeros(v, d, dtype=torch.int64).index_add_(0, tokens[tokens >= 0], dout[tokens >= 0].long())
        assert torch.equal(grad.cpu().long(), want)


def test_layouts(dev):
    """A table that is part of another, tokens and gradients of any strides, a mean's expanded gradient."""
    from hipenvs import embedding

    gen = torch.Generator().manual_seed(5)
    whole = torch.randn(30, 24, generator=gen).to(dev)
    tokens = torch.randint(-1, 30, (11, 17), generator=gen).to(dev)
    for table in (whole[:, 3:16], whole.t()[:, :9], whole[::2]):
        t = tokens.t() % table.shape[0]
        dout = torch.randn(11, table.shape[1], 17, generator=gen).to(dev).permute(2, 0, 1)
        check(t, table, 0.5, dout)
    table = whole.clone().requires_grad_()
    embedding.lookup(tokens, table).mean().backward()
    count = torch.bincount(tokens[tokens >= 0].flatten(), minlength=30).double()
    want = (count / (tokens.numel() * 24))[:, None].expand(30, 24)
    assert torch.allclose(table.grad.double(), want, rtol=1e-5, atol=0)


def test_infinities_and_nan_stay_in_their_rows(dev):
    from hipenvs import embedding

    tokens = torch.tensor([0, 1, 1, 2, -1, 3], device=dev)
    dout = torch.ones(6, 8, device=dev)
    dout[1] = float("inf")
    dout[4] = float("nan")
    table = torch.zeros(5, 8, device=dev, requires_grad=True)
    grad, = torch.autograd.grad(embedding.lookup(tokens, table), table, dout)
    assert torch.equal(grad[:, 0].cpu(), torch.tensor([1.0, float("inf"), 1.0, 1.0, 0.0]))


def test_the_same_bits_on_every_run(dev):
    for case in ((50000, 7, 64), (50000, 40009, 64)):
        tokens, table, dout = make(dev, 2, *case, F32, skew=3.0)
        first, second = check(tokens, table, 1.0, dout), check(tokens, table, 1.0, dout)
        assert torch.equal(first[1], second[1])


def test_empty(dev):
    from hipenvs import embedding

    table = torch.ones(4, 6, device=dev, requires_grad=True)
    out = embedding.lookup(torch.zeros(3, 0, dtype=torch.int64, device=dev), table)
    assert out.shape == (3, 0, 6)
    out.sum().backward()
    assert (table.grad == 0).all()
    scalar = embedding.lookup(torch.tensor(2, device=dev), table)
    assert torch.equal(scalar, table[2])


@pytest.mark.parametrize("v", [3, 5000])
def test_captured_training_replays(dev, v):
    from hipenvs import embedding

    given = [make(dev, 30 + k, 6000, v, 48, F32) for k in range(4)]
    static = [x.clone() for x in given[0]]

    def train():
        table = static[1].detach().requires_grad_()
        out = embedding.lookup(static[0], table, scale=2.0)
        return out.detach(), torch.autograd.grad(out, table, static[2])[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        train()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = train()
    for c in given[1:] + given[:2]:
        for to, of in zip(static, c):
            to.copy_(of)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        assert all(torch.equal(a, e) for a, e in zip(got, train()))


def test_rows_past_32_bit_offsets(dev):
    from hipenvs import embedding

    count, d = (1 << 31) // 1024 + 100, 1024
    tokens = torch.zeros(count, dtype=torch.int32, device=dev)
    tokens[-50:] = torch.arange(50, device=dev) % 7 + 1
    table = torch.randn(8, d, device=dev).to(BF16).requires_grad_()
    out = embedding.lookup(tokens, table)
    assert torch.equal(out[-50:], table.detach()[tokens[-50:].long()])
    dout = torch.zeros_like(out)
    dout[-50:] = 1.0
    grad, = torch.autograd.grad(out, table, dout)
    want = torch.bincount(tokens[-50:].long(), minlength=8).float()
    assert torch.equal(grad.float(), want.to(dev)[:, None].expand(8, d))


def test_refusals(dev):
    from hipenvs import embedding

    table, tokens = torch.zeros(4, 6, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for bad in (dict(table=table.half()), dict(tokens=tokens.float()), dict(tokens=[1, 2]), dict(tokens=tokens.to(torch.int16))):
        with pytest.raises(TypeError):
            embedding.lookup(**{"tokens": tokens, "table": table, **bad})
    for bad in (dict(table=table[0]), dict(table=table[:0]), dict(table=table[:, :0]), dict(tokens=tokens.cpu()),
                dict(table=table.cpu())):
        with pytest.raises(ValueError):
            embedding.lookup(**{"tokens": tokens, "table": table, **bad})
