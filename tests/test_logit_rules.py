"""Penalties, biases and allowed tokens on logits, against 64 bits."""
import math
import warnings

import numpy as np
import pytest
import torch

import polyrl_amd.ops as ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, F32 = torch.bfloat16, torch.float32


def expected(logits, rules, rows):
    """The result and the sum of the magnitudes that it is made of."""
    x = logits.double().cpu().numpy().copy()
    size = np.abs(np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0))
    V = x.shape[1]
    get = {k: v.cpu().numpy() for k, v in vars(rules).items()
           if isinstance(v, torch.Tensor)}
    for i, s in enumerate(rows.tolist()):
        if not 0 <= s < rules.slots:
            continue
        prompt, total = get["prompt_len"][s], get["total_len"][s]
        words = get["history"][s, :total]
        rep, freq, pres = (float(get[k][s]) for k in (
            "repetition", "frequency", "presence"))
        for t in set(words.tolist()):
            if 0 <= t < V:
                x[i, t] = x[i, t] / rep if x[i, t] > 0 else x[i, t] * rep
                size[i, t] *= max(rep, 1 / rep)
                c = int((words[prompt:] == t).sum())
                if c:
                    x[i, t] -= freq * c + pres
                    size[i, t] += abs(freq * c) + abs(pres)
        last = {t: v for t, v in zip(get["bias_tokens"][s].tolist(),
                                     get["bias_values"][s].tolist()) if 0 <= t < V}
        for t, v in last.items():
            x[i, t] += v
            size[i, t] += abs(v) if math.isfinite(v) else 0
        if get["masked"][s]:
            for t in range(V):
                if not get["mask"][s, t // 32] >> (t % 32) & 1:
                    x[i, t] = -np.inf
    # the lowest number doubled is -2^129: infinite in 32 bits, whose numbers end
    # half a step below 2^128
    x = np.where(np.abs(x) >= 2.0 ** 128 * (1 - 2.0 ** -25), np.sign(x) * np.inf, x)
    return torch.from_numpy(x), torch.from_numpy(size)


def compared(got, want, size):
    """Four operations in 32 bits, each off by 2^-24 of what it is made of (doubled for
    what comes after), then one rounding."""
    got = got.double().cpu()
    fine = want.isfinite()
    assert torch.equal(fine, got.isfinite())
    assert torch.equal(want.isnan(), got.isnan())
    edge = ~fine & ~want.isnan()
    assert torch.equal(got[edge], want[edge])
    inner = 8 * 2.0 ** -24 * size
    return got, fine, inner


def check(got, want, size):
    eps = torch.finfo(got.dtype).eps / 2
    g, fine, inner = compared(got, want, size)
    diff = (g - want).abs()[fine]
    assert (diff <= (eps * (want.abs() + inner) + inner)[fine]).all(), diff.max()


def make(dev, V, slots, cap, biases=0, seed=0):
    """Rules of all kinds, one slot of each, and tokens that repeat."""
    g = torch.Generator().manual_seed(seed)
    rules = ops.LogitRules(slots, V, cap, dev, biases=biases)
    for s in range(slots):
        n = int(torch.randint(0, cap + 1, (1,), generator=g)) if s % 3 else cap
        words = ((torch.rand(n, generator=g) ** 3) * V).int().tolist()
        cut = n * (s % 4) // 4
        kind = s % 6
        bias = {}
        if biases and kind in (2, 4, 5):
            bias = {int(t): float(v) for t, v in zip(
                torch.randint(0, V, (biases,), generator=g),
                torch.randn(biases, generator=g) * 5)}
        allowed = None
        if kind in (3, 4):
            allowed = torch.randperm(V, generator=g)[:max(V // 3, 1)].tolist()
        rules.set(s, words[:cut], words[cut:],
                  repetition=1.25 if kind in (1, 4, 5) else 1.0,
                  frequency=0.3 if kind in (0, 4) else 0.0,
                  presence=-0.4 if kind in (0, 5) else 0.0,
                  bias=bias, allowed=allowed)
    return rules


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V,cap,biases", [
    (1, 0, 0), (7, 5, 3), (33, 64, 1), (1000, 31, 0), (1024, 300, 7),
    (8192, 40, 2), (8193, 1000, 300), (50257, 77, 5)])
def test_against_64_bits(dev, dtype, V, cap, biases):
    slots = 7
    rules = make(dev, V, slots, cap, biases)
    g = torch.Generator().manual_seed(1)
    logits = (torch.randn(9, V, generator=g) * 4).to(dtype).to(dev)
    rows = torch.tensor([3, 6, -1, 0, 1, 2, 5, 4, 7], dtype=torch.int32, device=dev)
    keep = logits.clone()
    got = ops.adjust_logits(logits, rules, rows)
    assert torch.equal(logits, keep)
    check(got, *expected(logits, rules, rows))
    assert torch.equal(got[2], logits[2]) and torch.equal(got[8], logits[8])
    assert ops.adjust_logits(logits, rules, rows, out=logits) is logits
    assert torch.equal(logits, got)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pad,shift,opad,oshift", [
    (8, 0, 0, 0), (3, 1, 3, 1), (5, 2, 1, 0), (0, 1, 8, 9)])
def test_strides_and_addresses(dev, dtype, pad, shift, opad, oshift):
    V, N = 3001, 6

    def rows_of(pad, shift):
        g = torch.Generator().manual_seed(pad)
        full = torch.randn(N * (V + pad) + shift, generator=g).to(dtype).to(dev)
        return full, full[shift:].view(N, V + pad)[:, :V]
    rules = make(dev, V, N, 100, 4)
    rows = torch.arange(N, dtype=torch.int32, device=dev).flip(0)
    _, logits = rows_of(pad, shift)
    around, out = rows_of(opad, oshift)
    before = around.clone()
    ops.adjust_logits(logits, rules, rows, out=out)
    check(out, *expected(logits, rules, rows))
    mask = torch.ones_like(around, dtype=torch.bool)
    mask[oshift:].view(N, -1)[:, :V] = False
    assert torch.equal(around[mask], before[mask])
    want = out.clone()
    ops.adjust_logits(logits, rules, rows, out=logits)
    assert torch.equal(logits, want)


@pytest.mark.parametrize("dev", DEVICES)
def test_edges(dev):
    """No allowed token, infinities and undefined numbers, one slot for two rows, tokens that
    are none, a token said thousands of times, one bias twice."""
    V, cap = 300, 6000
    rules = ops.LogitRules(4, V, cap, dev, biases=4)
    inf, nan = float("inf"), float("nan")
    logits = torch.linspace(-3, 3, V).repeat(5, 1)
    logits[:, 10], logits[:, 11], logits[:, 12] = nan, inf, -inf
    logits[:, 0] = torch.finfo(F32).min
    logits = logits.to(dev)
    rules.set(0, [10, 11, 12], [13] * 5000 + [10, 11, 12, 14], repetition=1.5,
              frequency=0.001, presence=0.5, allowed=range(13, 200))
    rules.set(1, allowed=[])
    rules.set(2, [10, 11, 12], [299, 0], repetition=2.0, frequency=1.0)
    rules.history[2, 5:8] = torch.tensor([-5, V, 2 ** 31 - 1], dtype=torch.int32)
    rules.total_len[2] = 8
    rules.set(3, bias=[(5, 1.0), (7, -inf), (5, 2.0), (299, inf)])
    rows = torch.tensor([0, 1, 2, 3, 0], dtype=torch.int32, device=dev)
    got = ops.adjust_logits(logits, rules, rows)
    check(got, *expected(logits, rules, rows))
    assert (got[1] == -inf).all()
    assert torch.equal(got[0].isnan(), torch.zeros(V, dtype=torch.bool, device=dev))
    assert got[3, 5] == logits[3, 5] + 2.0 and got[3, 7] == -inf and got[3, 299] == inf
    assert torch.equal(got[4], got[0])


@pytest.mark.parametrize("dev", DEVICES)
def test_lengths_outside_of_the_history(dev):
    """Lengths that a program wrote wrongly stay within the history."""
    rules = ops.LogitRules(3, 50, 4, dev)
    rules.history.copy_(torch.arange(12).view(3, 4))
    rules.repetition.fill_(2.0)
    rules.frequency.fill_(1.0)
    rules.total_len.copy_(torch.tensor([9, -3, 2]))
    rules.prompt_len.copy_(torch.tensor([-1, 5, 7]))
    logits = torch.ones(3, 50, device=dev)
    rows = torch.arange(3, dtype=torch.int32, device=dev)
    got = ops.adjust_logits(logits, rules, rows).cpu()
    want = torch.ones(3, 50)
    want[0, :4] = -0.5
    want[2, 8:10] = 0.5
    assert torch.equal(got, want)


@pytest.mark.parametrize("dev", DEVICES)
def test_append(dev):
    """Tokens follow each other in their slots, two of one slot in their order."""
    rules = ops.LogitRules(4, 100, 5, dev)
    rules.set(2, [1, 2], [3])
    rows = torch.tensor([2, 0, -1, 2, 4, 2, 0], dtype=torch.int32, device=dev)
    tokens = torch.tensor([10, 11, 12, 13, 14, 15, -1], device=dev)
    ops.append_tokens(rules, rows, tokens)
    assert rules.total_len.tolist() == [2, 0, 5, 0]
    assert rules.history[2].tolist() == [1, 2, 3, 10, 13]       # full
    assert rules.history[0].tolist() == [11, -1, -1, -1, -1]
    assert rules.history[3].tolist() == [-1] * 5
    many = torch.arange(700, device=dev).int() % 2 + 1
    rules = ops.LogitRules(4, 1000, 400, dev)
    ops.append_tokens(rules, many, torch.arange(700, device=dev))
    assert rules.total_len.tolist() == [0, 350, 350, 0]
    assert rules.history[1, :350].tolist() == list(range(0, 700, 2))
    assert rules.history[2, :350].tolist() == list(range(1, 700, 2))


@pytest.mark.parametrize("dev", DEVICES)
def test_append_to_lengths_outside_of_the_history(dev):
    """A full history stays as it is, its length too, whatever a program wrote there; a
    negative length is an empty history."""
    rules = ops.LogitRules(5, 40, 3, dev)
    rules.total_len.copy_(torch.tensor([3, 9, -4, 2, 7], dtype=torch.int32))
    rows = torch.tensor([0, 1, 2, 3, 3, 1, 3], dtype=torch.int32, device=dev)
    ops.append_tokens(rules, rows, torch.arange(10, 17, device=dev))
    assert rules.total_len.tolist() == [3, 9, 1, 3, 7]
    assert rules.history.tolist() == [[-1] * 3, [-1] * 3, [12, -1, -1], [-1, -1, 13],
                                      [-1] * 3]
    with pytest.raises((ValueError, RuntimeError)):
        ops.append_tokens(rules, torch.zeros(16385, dtype=torch.int32, device=dev),
                          torch.zeros(16385, dtype=torch.int64, device=dev))


@pytest.mark.gpu
def test_captured():
    """A decode step with rules: logits, token, history; replayed as it runs."""
    V, N = 5000, 5

    def program(rules, logits, rows, step):
        adjusted = ops.adjust_logits(logits, rules, rows)
        token = adjusted.argmax(-1)
        ops.append_tokens(rules, rows, token)
        step.copy_(token)
    g = torch.Generator().manual_seed(2)
    inputs = [(torch.randn(N, V, generator=g) * 0.1).cuda() for _ in range(6)]
    runs = []
    for captured in (False, True):
        rules = make("cuda", V, 8, 60, 3)
        rules.total_len.clamp_(max=20)
        rules.frequency.fill_(0.5)
        rows = torch.tensor([1, 7, 3, -1, 0], dtype=torch.int32, device="cuda")
        logits, step = inputs[0].clone(), torch.zeros(N, dtype=torch.int64,
                                                      device="cuda")
        if captured:
            lens = rules.total_len.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                program(rules, logits, rows, step)
            torch.cuda.current_stream().wait_stream(side)
            rules.total_len.copy_(lens)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                program(rules, logits, rows, step)
        seen = []
        for x in inputs:
            logits.copy_(x)
            graph.replay() if captured else program(rules, logits, rows, step)
            seen.append(step.tolist())
        runs.append((seen, rules.history.tolist(), rules.total_len.tolist()))
    # (beyond its length a history holds what the capture's first run left)
    assert runs[0][0] == runs[1][0] and runs[0][2] == runs[1][2]
    for a, b, n in zip(runs[0][1], runs[1][1], runs[0][2]):
        assert a[:n] == b[:n]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_outputs_on_top_of_logits(dev, dtype):
    """A view of the logits' memory that is not the logits is refused where it shares
    a number with them, and a place like others where it does not."""
    N, V = 5, 40
    pool = torch.randn(2048, generator=torch.Generator().manual_seed(0)).to(dtype).to(dev)
    at = lambda first, pitch=96: pool.as_strided((N, V), (pitch, 1), first)
    logits, rules = at(256), ops.LogitRules(2, V, 6, dev)
    rules.set(0, prompt=[3], output=[4, 4], repetition=1.5, frequency=0.5)
    rules.set(1, allowed=range(7))
    rows = torch.tensor([0, 1, -1, 0, 1], dtype=torch.int32, device=dev)
    keep = pool.clone()
    for out in (at(256 + 96), at(256 - 96), at(256 + 8), at(256 - 39), at(256, 48),
                at(256, 104), at(300, 47)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.adjust_logits(logits, rules, rows, out=out)
    assert torch.equal(pool, keep)
    want = ops.adjust_logits(logits, rules, rows)
    for first in (256 + 40, 256 - 40, 256 + 51, 256 + 5 * 96, 256):
        pool.copy_(keep)
        out = at(first)
        assert ops.adjust_logits(logits, rules, rows, out=out) is out
        assert torch.equal(out, want), first


@pytest.mark.parametrize("dev", DEVICES)
def test_outputs_that_autograd_knows(dev):
    """An output with a gradient of its own is refused; one that a backward pass still needs
    is found changed there, as with any operator in place."""
    rules = ops.LogitRules(1, 40, 6, dev)
    rules.set(0, allowed=[3])
    rows = torch.zeros(2, dtype=torch.int32, device=dev)
    logits = torch.zeros(2, 40, device=dev)
    leaf = torch.zeros(2, 40, device=dev, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(RuntimeError):
            ops.adjust_logits(logits, rules, rows, out=out)
        with torch.no_grad():
            ops.adjust_logits(logits, rules, rows, out=out)
    w = torch.ones(40, 3, device=dev, requires_grad=True)
    for out in (torch.zeros_like(logits), logits):
        loss = (out @ w).sum()
        ops.adjust_logits(logits, rules, rows, out=out)
        with pytest.raises(RuntimeError):
            loss.backward()
    with torch.inference_mode():
        z = logits.clone()
    ops.adjust_logits(z, rules, rows)
    with torch.inference_mode():
        ops.adjust_logits(z, rules, rows, out=z)


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    rules = ops.LogitRules(2, 40, 6, dev, biases=1)
    for kw in (dict(repetition=0.0), dict(repetition=-1.0),
               dict(frequency=float("nan")), dict(presence=float("inf")),
               dict(bias={40: 1.0}), dict(bias={-1: 1.0}),
               dict(bias={1: 1.0, 2: 2.0}), dict(bias={1: float("nan")}),
               dict(prompt=[1] * 7), dict(allowed=[40]), dict(allowed=[-1]),
               dict(allowed=np.zeros(3, np.int32))):
        with pytest.raises(ValueError):
            rules.set(0, **kw)
    assert rules.masked.tolist() == [0, 0]
    for slot in (-1, 2):
        with pytest.raises(ValueError):
            rules.set(slot)
    for args in ((0, 4, 4), (1, 0, 4), (1, 4, 1 << 19), (1, 4, -1), (1, 4, 4, 4096)):
        with pytest.raises(ValueError):
            ops.LogitRules(*args[:3], dev, *args[3:])
    rows = torch.zeros(3, dtype=torch.int32, device=dev)
    logits = torch.zeros(3, 40, device=dev)
    error = (ValueError, RuntimeError)
    for bad in (logits[:, :39], logits[0], logits[:2]):
        with pytest.raises(error):
            ops.adjust_logits(bad, rules, rows)
    with pytest.raises(error):
        ops.adjust_logits(logits, rules, rows.long())
    with pytest.raises(error):
        ops.adjust_logits(logits.clone().requires_grad_(), rules, rows)
    with pytest.raises(error):                    # rows on top of each other
        ops.adjust_logits(logits, rules, rows, out=logits[0].expand(3, 40)
                          if dev == "cuda" else logits[:2])
    with pytest.raises(error):
        ops.append_tokens(rules, rows, torch.zeros(2, dtype=torch.int64, device=dev))
    with pytest.raises(error):
        ops.append_tokens(rules, rows, torch.zeros(3, device=dev))
    if dev == "cuda":
        with pytest.raises(error):
            ops.adjust_logits(logits.half(), rules, rows)
        with pytest.raises(error):
            ops.adjust_logits(logits, rules, rows, out=logits.bfloat16())
        with pytest.raises(error):
            ops.adjust_logits(logits, rules, rows.cpu())
        with pytest.raises(error):
            ops.adjust_logits(torch.zeros(40, 3, device=dev).t(), rules, rows)


@pytest.mark.parametrize("dev", DEVICES)
def test_numbers_that_32_bits_do_not_hold(dev):
    """A rule is what its 32 bits say: a repetition of 1e-60 would be a division by 0."""
    rules = ops.LogitRules(1, 40, 6, dev, biases=2)
    for kw in (dict(repetition=1e-60), dict(repetition=1e60),
               dict(frequency=-1e60), dict(presence=1e60)):
        with pytest.raises(ValueError):
            rules.set(0, **kw)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        rules.set(0, bias={1: -1e60, 2: 5.0})
    assert rules.bias_values[0].tolist() == [-math.inf, 5.0]
