"""Seeded dropout: what stays, what it becomes, and its gradient."""
import numpy as np
import pytest
import torch

import polyrl_amd.ops as ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def philox(counters, seed):
    """Four 32-bit words for every counter, in whole numbers of any length."""
    out = []
    for n in counters:
        c = [n & 0xffffffff, n >> 32, 0, 0]
        k = [seed & 0xffffffff, seed >> 32 & 0xffffffff]
        for _ in range(10):
            p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [q >> 32 ^ c[1] ^ k[0], q & 0xffffffff,
                 p >> 32 ^ c[3] ^ k[1], p & 0xffffffff]
            k = [k[0] + 0x9E3779B9 & 0xffffffff, k[1] + 0xBB67AE85 & 0xffffffff]
        out.append(c)
    return out


def stays(first, n, drop, seed):
    """Of elements first .. first + n."""
    lo, hi = first // 8, (first + n + 7) // 8
    bits = [w >> s & 0xffff for c in philox(range(lo, hi), seed) for w in c
            for s in (0, 16)]
    return torch.tensor(bits[first - lo * 8:][:n]) >= drop


def test_generator_is_the_published_one():
    # the method's authors' answer for counter 0 and key 0
    assert philox([0], 0) == [[0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(0,), (1,), (7,), (8,), (9,), (3, 5, 11),
                                   (1, 2048), (33, 127)])
@pytest.mark.parametrize("p,seed", [(0.0, 1), (0.1, -3), (0.5, 1 << 62), (1.0, 0)])
def test_values_and_gradient(dev, dtype, shape, p, seed):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(shape, generator=g).to(dtype).to(dev).requires_grad_()
    dy = torch.randn(shape, generator=g).to(dtype).to(dev)
    key = torch.tensor([seed], device=dev)
    y = ops.dropout_train(x, p, key)
    dx, = torch.autograd.grad(y, x, dy)
    drop = round(p * 65536)
    keep = stays(0, x.numel(), drop, seed % (1 << 64)).view(shape)
    # one product in 32 bits with a scale of 24 bits, one rounding
    off = torch.finfo(dtype).eps / 2 + 2.0 ** -22
    for got, t in ((y, x), (dx, dy)):
        assert got.dtype == dtype
        got, t = got.detach().double().cpu(), t.detach().double().cpu()
        want = torch.where(keep, t * 65536 / max(65536 - drop, 1), 0.0)
        assert ((got - want).abs() <= off * want.abs()).all()
        assert torch.equal(got == 0, (~keep | (t == 0)))


@pytest.mark.parametrize("dev", DEVICES)
def test_gradient_against_differences(dev):
    g = torch.Generator().manual_seed(1)
    x, u, dy = (torch.randn(40, 9, generator=g).to(dev) for _ in range(3))
    seed = torch.tensor([11], device=dev)
    x.requires_grad_()
    dx, = torch.autograd.grad(ops.dropout_train(x, 0.3, seed), x, dy)
    f = lambda t: (ops.dropout_train(t.detach(), 0.3, seed).double() * dy).sum()
    step = 2.0 ** -3
    slope = (f(x + step * u) - f(x - step * u)) / (2 * step)
    # linear in x: only roundings of x + step u and of y, 2^-24 of at most 8 each, 360
    # elements times |dy| <= 5, over 2 step
    assert abs(slope - (dx.double() * u).sum()) < 360 * 5 * 16 * 2.0 ** -24 / (2 * step)


@pytest.mark.parametrize("dev", DEVICES)
def test_places(dev):
    """An element's place is that in the rows one after the other, however they lie."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(24, 50, generator=g).to(dev)
    seed = torch.tensor([7], device=dev)
    want = ops.dropout_train(x, 0.25, seed)
    wide = torch.zeros(24, 61, device=dev)
    wide[:, 3:53] = x
    flat = torch.zeros(1201, device=dev)
    flat[1:] = x.flatten()
    for same in (wide[:, 3:53], x.t().contiguous().t(), flat[1:].view(24, 50)):
        assert torch.equal(ops.dropout_train(same, 0.25, seed), want)
    # gradients that come as a broadcast number or transposed
    leaf = x.clone().requires_grad_()
    ops.dropout_train(leaf, 0.25, seed).sum().backward()
    assert torch.equal(leaf.grad != 0, want != 0)
    leaf.grad = None
    ops.dropout_train(leaf, 0.25, seed).t().contiguous().sum().backward()
    assert torch.equal(leaf.grad != 0, want != 0)


@pytest.mark.parametrize("dev", DEVICES)
def test_dropped_places_are_zero_whatever_they_held(dev):
    x = torch.tensor([float("nan"), float("inf"), -float("inf")] * 40).to(dev)
    y = ops.dropout_train(x, 0.5, torch.tensor([3], device=dev))
    keep = stays(0, 120, 32768, 3).to(dev)
    assert (y[~keep] == 0).all() and not y[keep].isfinite().any()


@pytest.mark.parametrize("dev", DEVICES)
def test_rate_and_seeds(dev):
    x = torch.ones(100003, device=dev)
    a, b = (ops.dropout_train(x, 0.1, torch.tensor([s], device=dev)) for s in (1, 2))
    for y in (a, b):                       # six standard deviations
        assert abs((y == 0).double().mean() - 0.1) < 6 * (0.09 / 100003) ** 0.5
    both = ((a == 0) & (b == 0)).double().mean()
    assert abs(both - 0.01) < 6 * (0.01 / 100003) ** 0.5
    assert torch.equal(a, ops.dropout_train(x, 0.1, torch.tensor([1], device=dev)))


@pytest.mark.gpu
def test_same_on_both_devices():
    x = torch.randn(513, 77)
    seed = torch.tensor([-99])
    assert torch.equal(ops.dropout_train(x, 0.2, seed),
                       ops.dropout_train(x.cuda(), 0.2, seed.cuda()).cpu())


@pytest.mark.gpu
def test_more_elements_than_31_bits():
    n = (1 << 31) + 13
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout_train(x, 0.5, torch.tensor([5], device="cuda"))
    for first in (0, (1 << 31) - 9, n - 21):
        m = min(30, n - first)
        assert torch.equal(y[first:first + m].cpu() != 0,
                           stays(first, m, 32768, 5))


@pytest.mark.gpu
def test_captured():
    """Forward and backward in a graph whose seed moves on."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(64, 100, generator=g).cuda().requires_grad_()
    seed = torch.tensor([100], device="cuda")

    def step():
        y = ops.dropout_train(x, 0.3, seed.clone())
        dx, = torch.autograd.grad((y * y).sum(-1), x, torch.ones(64, device="cuda"))
        return y.detach(), dx
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
        seed.add_(1)
    for i in range(4):
        seed.fill_(100 + i)
        graph.replay()
        got = y.clone(), dx.clone()
        torch.cuda.synchronize()
        assert int(seed) == 101 + i
        seed.fill_(100 + i)
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    x = torch.ones(4, device=dev)
    seed = torch.tensor([1], device=dev)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout_train(x, p, seed)
    for bad in (seed.int(), torch.tensor([1, 2], device=dev)):
        with pytest.raises(ValueError):
            ops.dropout_train(x, 0.1, bad)
    for bad in (x.double(), x.long()):
        with pytest.raises(ValueError):
            ops.dropout_train(bad, 0.1, seed)
    if dev == "cuda":
        with pytest.raises(ValueError):
            ops.dropout_train(x, 0.1, seed.cpu())
