"""Low-rank adapters of many requests beside a shared projection, against 64 bits."""
import pytest
import torch

import polyrl_amd.ops as ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, F32 = torch.bfloat16, torch.float32


def make(dev, dtype, T, K, widths, r, S, seed=0, pad=0, shift=0):
    """y, x, a, b, scale; rows ``pad`` numbers longer than they are and ``shift``
    numbers into their memory."""
    g = torch.Generator().manual_seed(seed)

    def rows(n, width):
        full = torch.randn(n * (width + pad) + shift, generator=g).to(dtype).to(dev)
        return full[shift:].view(n, width + pad)[:, :width]
    N = sum(widths)
    a = (torch.randn(S, len(widths), r, K, generator=g) * K ** -0.5).to(dtype).to(dev)
    b = torch.randn(S, N, r, generator=g).to(dtype).to(dev)
    scale = (torch.rand(S, generator=g) + 0.5).to(dev)
    return rows(T, N), rows(T, K), a, b, scale


def expected(y, x, a, b, scale, index, widths, ranks=None):
    """The result and how far off it may be.

    h = A x is a sum of K products in 32 bits, then split into two bf16 numbers for
    bf16 (2^-8 of what 2^-8 leaves); B h a sum of r products in 32 bits, of hi and lo
    apart; y is added in 32 bits and the sum rounded once."""
    y, x, a, b = (t.double().cpu() for t in (y, x, a, b))
    S, P, r, K = a.shape
    want, size = y.clone(), torch.zeros_like(y)
    for t, s in enumerate(index.tolist()):
        if not 0 <= s < S:
            continue
        n = r if ranks is None else int(ranks[s])
        at = 0
        for p, w in enumerate(widths):
            A, B = a[s, p, :n], b[s, at:at + w, :n]
            want[t, at:at + w] += float(scale[s]) * (B @ (A @ x[t]))
            size[t, at:at + w] += float(scale[s]) * (B.abs() @ (A.abs() @ x[t].abs()))
            at += w
    return want, size


def close(got, want, size, y, K, r):
    eps = torch.finfo(got.dtype).eps / 2
    lost = 2.0 ** -16 if got.dtype == BF16 else 0.0
    inner = size * ((K + 2 * r + 32) * 2.0 ** -24 + lost)
    inner = inner + 2.0 ** -23 * (y.double().cpu().abs() + size)
    diff = (got.double().cpu() - want).abs()
    bad = diff > eps * (want.abs() + inner) + inner
    assert not bad.any(), (diff.max(), bad.nonzero()[:5])


SIZES = [
    # T, K, widths, r, S
    (1, 64, (16,), 1, 1),
    (1, 1024, (1024, 256, 256), 8, 4),
    (5, 33, (7,), 5, 3),
    (16, 128, (48, 16, 7), 16, 2),
    (17, 100, (64, 64), 33, 5),
    (57, 256, (300,), 64, 70),
    (257, 192, (256, 64, 64), 20, 3),
    (300, 520, (130,), 100, 7),
    (64, 4096, (32,), 16, 2),
    (3, 1, (1,), 1, 1),
    # both sides of the rows from which blocks are larger, ranks that need more than one
    # round, several parts whose ranks fall into several groups
    (1024, 136, (130, 30), 48, 2),
    (1025, 136, (130, 30), 48, 2),
    (1100, 4096, (256, 64, 64), 96, 2),
    (40, 2050, (20, 20, 20), 130, 3),
    (130, 600, (8, 8, 8, 8, 8, 8, 8, 8), 256, 2),
    (258, 300, (70, 0, 5), 256, 4),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size", SIZES)
def test_against_64_bits(dev, dtype, size):
    T, K, widths, r, S = size
    y, x, a, b, scale = make(dev, dtype, T, K, widths, r, S)
    g = torch.Generator().manual_seed(1)
    index = torch.randint(-1, S + 1, (T,), generator=g, dtype=torch.int32)
    index[0] = 0
    plan = ops.adapter_plan(index.to(dev), S)
    keep = y.clone()
    got = ops.adapter_add(y, x, a, b, scale, plan, widths)
    assert torch.equal(y, keep)
    want, size = expected(y, x, a, b, scale, index, widths)
    close(got, want, size, y, K, r)
    none = (index < 0) | (index >= S)
    assert torch.equal(got[none.to(dev)], y[none.to(dev)])
    # in place: the same bits
    assert ops.adapter_add(y, x, a, b, scale, plan, widths, out=y) is y
    assert torch.equal(y, got)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1), (5, 3)])
@pytest.mark.parametrize("T", [9, 260])
def test_strides_and_addresses(dev, dtype, pad, shift, T):
    K, widths, r, S = 72, (40, 24), 16, 3
    y, x, a, b, scale = make(dev, dtype, T, K, widths, r, S, pad=pad, shift=shift)
    index = (torch.arange(T, dtype=torch.int32) % 4) - 1
    around = y._base.clone()
    plan = ops.adapter_plan(index.to(dev), S)
    got = ops.adapter_add(y, x, a, b, scale, plan, widths)
    want, size = expected(y, x, a, b, scale, index, widths)
    close(got, want, size, y, K, r)
    ops.adapter_add(y, x, a, b, scale, plan, widths, out=y)
    assert torch.equal(y, got)
    # what lies between and before the rows is as it was
    after = y._base.clone()
    mask = torch.ones_like(after, dtype=torch.bool)
    mask[shift:].view(T, -1)[:, :sum(widths)] = False
    assert torch.equal(after[mask], around[mask])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [40, 300])
def test_ranks(dev, dtype, T):
    """Smaller ranks in a pool: what lies beyond them is not read; rank 0 is none."""
    K, widths, r, S = 128, (64, 32), 40, 6
    y, x, a, b, scale = make(dev, dtype, T, K, widths, r, S)
    ranks = torch.tensor([40, 0, 1, 16, 33, 7], dtype=torch.int32)
    for s in range(S):
        a[s, :, ranks[s]:] = float("nan")
        b[s, :, ranks[s]:] = float("nan")
    index = torch.arange(T, dtype=torch.int32) % S
    plan = ops.adapter_plan(index.to(dev), S)
    got = ops.adapter_add(y, x, a, b, scale, plan, widths, ranks=ranks.to(dev))
    want, size = expected(y, x, a, b, scale, index, widths, ranks)
    close(got, want, size, y, K, r)
    assert torch.equal(got[index == 1], y[index == 1])
    out = y.clone()
    ops.adapter_add(out, x, a, b, scale, plan, widths, ranks=ranks.to(dev), out=out)
    assert torch.equal(out, got)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_do_not_touch_each_other(dev, dtype):
    """An infinite or undefined row stays its own, an infinite h stays infinite."""
    T, K, r, S = 33, 64, 8, 2
    y, x, a, b, scale = make(dev, dtype, T, K, (32,), r, S)
    index = torch.arange(T, dtype=torch.int32) % S
    plan = ops.adapter_plan(index.to(dev), S)
    clean = ops.adapter_add(y, x, a, b, scale, plan)
    x[4] = float("nan")
    a[0, 0, 0], b[0, :, 0] = 1.0, 1.0
    a[0, 0, 1:] = 0.0
    clean0 = ops.adapter_add(y, x, a, b, scale, plan)
    x[6] = torch.finfo(dtype).max               # sums to infinity
    got = ops.adapter_add(y, x, a, b, scale, plan)
    assert got[4].isnan().all()
    assert (got[6] == float("inf")).all()
    for t in range(T):
        if t not in (4, 6):
            assert torch.equal(got[t], (clean if index[t] else clean0)[t])


@pytest.mark.parametrize("dev", DEVICES)
def test_none_and_empty(dev):
    y, x, a, b, scale = make(dev, BF16, 20, 32, (16,), 8, 2)
    for v in (-1, -7, 2, 99):
        plan = ops.adapter_plan(torch.full((20,), v, dtype=torch.int32, device=dev), 2)
        assert torch.equal(ops.adapter_add(y, x, a, b, scale, plan), y)
    plan = ops.adapter_plan(torch.zeros(0, dtype=torch.int32, device=dev), 2)
    assert ops.adapter_add(y[:0], x[:0], a, b, scale, plan).shape == (0, 16)


@pytest.mark.gpu
def test_many_rows_and_slots():
    """Plans of many rows and of the most adapters, in any order."""
    S, K, N, r = 4095, 64, 32, 4
    y, x, a, b, scale = make("cuda", F32, 20000, K, (N,), r, S)
    g = torch.Generator().manual_seed(3)
    index = torch.randint(-1, S, (20000,), generator=g, dtype=torch.int32)
    index[:9000] = 17
    plan = ops.adapter_plan(index.cuda(), S)
    got = ops.adapter_add(y, x, a, b, scale, plan)
    i = index.clamp(min=0).long().cuda()
    h = (a[i, 0].double() @ x.double().unsqueeze(-1))
    d = (b[i].double() @ h).squeeze(-1) * scale[i].double().unsqueeze(1)
    d[(index < 0).cuda()] = 0
    h = (a[i, 0].double().abs() @ x.double().abs().unsqueeze(-1))
    size = (b[i].double().abs() @ h).squeeze(-1) * scale[i].double().unsqueeze(1)
    close(got, (y.double() + d).cpu(), size.cpu(), y, K, r)


@pytest.mark.gpu
def test_work_space_is_the_rows():
    """Of many adapters most tiles are of few rows: what lies between the two products
    takes rows * parts * rank numbers of 32 bits, up to four shares of them, and not the
    places of tiles."""
    T, K, widths, r, S = 2000, 8, (8, 8, 8), 256, 4095
    y, x, a, b, scale = make("cuda", BF16, T, K, widths, r, S)
    index = torch.randperm(S, generator=torch.Generator().manual_seed(3))[:T].int()
    plan = ops.adapter_plan(index.cuda(), S)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = ops.adapter_add(y, x, a, b, scale, plan, widths)
    most = torch.cuda.max_memory_allocated() - before
    assert most <= 4 * T * len(widths) * r * 4 + 2 * y.numel() * 2 + (1 << 21)
    want, size = expected(y, x, a, b, scale, index, widths)
    close(got, want, size, y, K, r)


@pytest.mark.gpu
def test_result_does_not_hang_on_the_order_of_rows():
    T, K, widths, r, S = 600, 512, (96,), 24, 4
    y, x, a, b, scale = make("cuda", BF16, T, K, widths, r, S)
    g = torch.Generator().manual_seed(4)
    index = torch.randint(-1, S, (T,), generator=g, dtype=torch.int32).cuda()
    want = ops.adapter_add(y, x, a, b, scale, ops.adapter_plan(index, S))
    for seed in range(3):
        p = torch.randperm(T, generator=g).cuda()
        got = ops.adapter_add(y[p], x[p], a, b, scale,
                              ops.adapter_plan(index[p], S))
        assert torch.equal(got, want[p])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,r", [(3, 4), (40, 70), (300, 4), (300, 70)])
def test_inner_sums_keep_32_bits(dev, dtype, T, r):
    """Whole numbers whose every sum is below 2^24: 32 bits hold them all, so that the
    result is the exact one, rounded once.  y is the negative of the rounded product, which
    leaves the places that 16 bits of h would lose."""
    K, widths, S = 64, (40, 24), 2
    g = torch.Generator().manual_seed(11)
    x = torch.randint(128, 256, (T, K), generator=g).double()
    a = torch.randint(128, 256, (S, len(widths), r, K), generator=g).double()
    b = torch.zeros(S, sum(widths), r, dtype=torch.double)
    at = torch.rand(b.shape, generator=g).topk(4, -1).indices
    b.scatter_(2, at, 1.0)                       # 4 * 64 * 255 * 255 < 2^24
    index = torch.arange(T, dtype=torch.int32) % S
    h = torch.einsum("tprk,tk->tpr", a[index.long()], x)
    h = h.repeat_interleave(torch.tensor(widths), 1)
    total = (b[index.long()] * h).sum(-1)
    assert total.max() < 1 << 24
    y = -total.to(BF16).double()
    want = (y + total).to(dtype)
    y, x, a, b = (t.to(dtype).to(dev) for t in (y, x, a, b))
    got = ops.adapter_add(y, x, a, b, torch.ones(S, device=dev),
                          ops.adapter_plan(index.to(dev), S), widths)
    assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [6, 400])
def test_captured(T):
    """A captured step goes by the adapters of its replay."""
    K, widths, r, S = 256, (64, 32), 16, 3
    y, x, a, b, scale = make("cuda", BF16, T, K, widths, r, S)
    index = torch.zeros(T, dtype=torch.int32, device="cuda")

    def step():
        plan = ops.adapter_plan(index, S)
        return ops.adapter_add(y, x, a, b, scale, plan, widths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    g = torch.Generator().manual_seed(5)
    for _ in range(4):
        index.copy_(torch.randint(-1, S + 1, (T,), generator=g))
        x.copy_(torch.randn(T, K, generator=g))
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(replayed, step())


def test_which_views_share_memory():
    """Both forms of the rule against the sets of addresses, over views of one buffer."""
    from polyrl_amd.ops import ref
    buf = torch.zeros(64)
    at = torch.arange(64)
    g = torch.Generator().manual_seed(0)
    pick = lambda low, high: int(torch.randint(low, high + 1, (1,), generator=g))
    seen = [0, 0]
    for _ in range(4000):
        views = []
        for _ in range(2):
            n, width, pitch = pick(0, 4), pick(0, 5), pick(0, 9)
            first = pick(0, 63 - 3 * 9 - 5)
            views.append(((n, width), (pitch, 1), first))
        a, b = (buf.as_strided(*v) for v in views)
        one, two = (set(at.as_strided(*v).flatten().tolist()) for v in views)
        want = bool(one & two)
        seen[want] += 1
        assert ref.rows_overlap(a, b) is want, views
        if ops.extension_loaded():
            assert ops._EXT.rows_overlap(a, b) is want, views
    assert min(seen) > 500
    flat = buf[:24].view(2, 3, 4)                 # contiguous tensors of any rank
    for off, want in ((20, True), (24, False)):
        assert ref.rows_overlap(buf[off:off + 8].view(2, 4), flat) is want


@pytest.mark.parametrize("dev", DEVICES)
def test_outputs_on_top_of_operands(dev):
    """Shifted by rows or columns, or over x or the adapters: refused.  Rows between y's,
    columns beside them and y itself are places like others."""
    T, N, K, r, S = 6, 16, 32, 8, 2
    g = torch.Generator().manual_seed(0)
    pool = torch.randn(4096, generator=g).to(dev)
    y = pool[64:].as_strided((T, N), (40, 1))
    x = pool[1024:1024 + T * K].view(T, K)
    a = pool[2048:2048 + S * r * K].view(S, 1, r, K)
    b = pool[3200:3200 + S * N * r].view(S, N, r)
    scale = torch.ones(S, device=dev)
    index = torch.arange(T, dtype=torch.int32) % (S + 1) - 1
    plan = ops.adapter_plan(index.to(dev), S)
    keep = pool.clone()
    at = lambda first, pitch=40: pool.as_strided((T, N), (pitch, 1), first)
    for out in (at(64 + 40), at(64 - 40), at(64 + 15), at(64 - 1), at(64, 41), at(66, 16),
                at(1024, N), at(1024 + T * K - 1), at(2048, N), at(3200 + 5, 33)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.adapter_add(y, x, a, b, scale, plan, out=out)
    assert torch.equal(pool, keep)                # refused before anything is written
    want = ops.adapter_add(y, x, a, b, scale, plan)
    for first in (64 + 16, 64 - 16, 64 + 24, 64 + T * 40, 1024 + T * K, 64):
        pool.copy_(keep)
        out = at(first)
        assert ops.adapter_add(y, x, a, b, scale, plan, out=out) is out
        assert torch.equal(out, want), first


@pytest.mark.parametrize("dev", DEVICES)
def test_outputs_that_autograd_knows(dev):
    """An output with a gradient of its own is refused; one that a backward pass still needs
    is found changed there, as with any operator in place."""
    y, x, a, b, scale = make(dev, F32, 6, 32, (16,), 8, 2)
    plan = ops.adapter_plan(torch.zeros(6, dtype=torch.int32, device=dev), 2)
    leaf = torch.zeros(6, 16, device=dev, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(RuntimeError):
            ops.adapter_add(y, x, a, b, scale, plan, out=out)
        with torch.no_grad():
            ops.adapter_add(y, x, a, b, scale, plan, out=out)
    w = torch.ones(16, 3, device=dev, requires_grad=True)
    for out in (torch.zeros_like(y), y):
        loss = (out @ w).sum()
        ops.adapter_add(y, x, a, b, scale, plan, out=out)
        with pytest.raises(RuntimeError):
            loss.backward()
    with torch.inference_mode():
        z = y.clone()
    ops.adapter_add(z, x, a, b, scale, plan) # (tensors of inference have no versions)
    with torch.inference_mode():
        ops.adapter_add(z, x, a, b, scale, plan, out=z)


@pytest.mark.parametrize("dev", DEVICES)
def test_refusals(dev):
    y, x, a, b, scale = make(dev, BF16, 6, 32, (16,), 8, 2)
    index = torch.zeros(6, dtype=torch.int32, device=dev)
    plan = ops.adapter_plan(index, 2)
    error = (ValueError, RuntimeError)
    for bad in (index.long(), index.view(2, 3)):
        with pytest.raises(error):
            ops.adapter_plan(bad, 2)
    for slots in (0, 4096):
        with pytest.raises(error):
            ops.adapter_plan(index, slots)
    with pytest.raises(error):                              # another number of rows
        ops.adapter_add(y[:5], x[:5], a, b, scale, plan)
    with pytest.raises(error):
        ops.adapter_add(y, x[:5], a, b, scale, plan)
    for widths in ((8, 8), (8,), (16, 0)):
        with pytest.raises(error):
            ops.adapter_add(y, x, a, b, scale, plan, widths)
    with pytest.raises(error):
        ops.adapter_add(y, x[:, :31], a, b, scale, plan)
    with pytest.raises(error):
        ops.adapter_add(y, x, a, b[:, :15], scale, plan)
    with pytest.raises(error):
        ops.adapter_add(y, x, a.clone().requires_grad_(), b, scale, plan)
    with pytest.raises(error):                              # ranks beyond 256
        ops.adapter_add(y, x, a.new_zeros(2, 1, 257, 32), b.new_zeros(2, 16, 257),
                        scale, plan)
    with pytest.raises(error):                              # nine parts
        ops.adapter_add(y, x, a.new_zeros(2, 9, 8, 32), b, scale, plan,
                        [8] + [1] * 8)
    with pytest.raises(error):                              # other adapters
        ops.adapter_add(y, x, a[:1].contiguous(), b[:1].contiguous(), scale[:1],
                        plan)
    with pytest.raises(error):                              # rows on top of each other
        ops.adapter_add(y, x, a, b, scale, plan,
                        out=y[:1].expand(6, 16) if dev == "cuda" else y[:5])
    if dev == "cuda":
        # a plan of fewer rows whose table is as long
        many = ops.adapter_plan(torch.zeros(224, dtype=torch.int32, device=dev), 2)
        big = [t.new_zeros(230, t.shape[1]) for t in (y, x)]
        assert many.table.numel() == ops.adapter_plan(
            torch.zeros(230, dtype=torch.int32, device=dev), 2).table.numel()
        with pytest.raises(error):
            ops.adapter_add(*big, a, b, scale, many)
        with pytest.raises(error):
            ops.adapter_add(y, x, a, b, scale, ops.adapter_plan(index.cpu(), 2))
        for bad in (x.float(), x.half()):
            with pytest.raises(error):
                ops.adapter_add(y, bad, a, b, scale, plan)
        with pytest.raises(error):
            ops.adapter_add(y.half(), x.half(), a.half(), b.half(), scale, plan)
        with pytest.raises(error):
            ops.adapter_add(y, x, a, b, scale.double(), plan)
        with pytest.raises(error):
            ops.adapter_add(y, x, a.cpu(), b, scale, plan)
        with pytest.raises(error):
            ops.adapter_add(y, x, a.transpose(2, 3), b, scale, plan)
