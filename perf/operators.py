"""Adapters of many requests, rules on logits and seeded dropout, as measurable cases.

``own`` False: the operators in elementary torch operations, in 32 bits, rounded
once.  True: the public entry points (``polyrl_amd.ops``).

kind "adapters"  The adapters' part of one decoder layer: y + scale * B (A x) beside the
                 four shared projections (q/k/v, output, gate/up, down), every row by
                 the adapter of its request or by none.  Widths are those of the
                 model registry.
kind "rules"     Logits of one decode step under their requests' rules: penalties for
                 tokens of the history, biases, sets of allowed tokens.
kind "dropout"   Seeded dropout of a training step, forward and backward; the mask is
                 a function of (seed, place) and kept by nobody.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
# hidden size, (q, k, v) widths, feed-forward width of the registry's decoders
MODELS = {
    "llama-400m": (1024, (1024, 256, 256), 4096),
    "qwen2.5-1.5b": (1536, (1536, 256, 256), 8960),
    "qwen2.5-7b": (3584, (3584, 512, 512), 18944),
    "llama3-8b": (4096, (4096, 1024, 1024), 14336),
}
VOCABS = (32000, 50257, 128256, 151936, 152064)


def listed():
    return [
        # one request with an adapter on a small model: latency of the smallest call
        dict(name="adapter-one", kind="adapters", model="llama-400m", rows=1,
             low=1, high=1, slots=4, rank=8, mixed=False, f32=False),
        # the benchmark's decode batch, 128 samples, a few adapters of usual rank
        dict(name="adapter-batch", kind="adapters", model="llama3-8b", rows=128,
             low=1, high=1, slots=8, rank=16, mixed=False, f32=False),
        # serving: every request its own adapter, large and small ranks
        dict(name="adapter-many", kind="adapters", model="qwen2.5-7b", rows=57,
             low=1, high=1, slots=64, rank=64, mixed=True, f32=False),
        # ragged prompts in full precision, a rank that fills no tile
        dict(name="adapter-exact", kind="adapters", model="qwen2.5-1.5b", rows=5,
             low=37, high=211, slots=3, rank=20, mixed=True, f32=True),
        # an engine step over whole prompts: 8 of up to 1024 tokens
        dict(name="adapter-prompts", kind="adapters", model="llama3-8b", rows=8,
             low=600, high=1024, slots=4, rank=32, mixed=False, f32=False),
        # one request of a small vocabulary, some words of history
        dict(name="rules-one", kind="rules", rows=1, vocab=32000, low=37, high=37,
             biases=0, masked=False, f32=False),
        # the benchmark's decode batch: 256 + 256 tokens of history, some biases
        dict(name="rules-batch", kind="rules", rows=128, vocab=128256, low=257,
             high=512, biases=16, masked=False, f32=False),
        # grammars: every request its set of allowed tokens
        dict(name="rules-grammar", kind="rules", rows=64, vocab=151936, low=20,
             high=700, biases=0, masked=True, f32=True),
        # long chains of thought: few rows, ten thousands of tokens, all rules
        dict(name="rules-long", kind="rules", rows=33, vocab=152064, low=9000,
             high=32768, biases=300, masked=True, f32=False),
        # the input of one adapter in a trainer's micro-batch
        dict(name="dropout-train", kind="dropout", rows=8192, cols=4096, p=0.05,
             dtype="bfloat16"),
        # ... of a small model, a micro-batch of odd length, full precision
        dict(name="dropout-small", kind="dropout", rows=37, cols=1023, p=0.1,
             dtype="float32"),
        # ... of the widest layer
        dict(name="dropout-wide", kind="dropout", rows=8192, cols=14336, p=0.1,
             dtype="bfloat16"),
    ]


def _log(rng, low, high):
    """A whole number in [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(
        rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(("adapters", "rules", "dropout"))
    if kind == "adapters":
        model = rng.choice(sorted(MODELS))
        f32 = rng.random() < 0.2
        case = dict(kind=kind, model=model, slots=_log(rng, 1, 64),
                    rank=rng.choice((4, 8, 12, 16, 20, 32, 33) if f32 else
                                    (4, 8, 12, 16, 20, 32, 33, 64)),
                    mixed=rng.random() < 0.5, f32=f32)
        if rng.random() < 0.5:                       # a decode step
            return dict(case, rows=_log(rng, 1, 256), low=1, high=1)
        high = _log(rng, 2, 1024)
        rows = _log(rng, 1, max(1, (1200 if f32 else 5000) // high))
        return dict(case, rows=rows, low=rng.randint(high // 4 + 1, high),
                    high=high, rank=min(case["rank"], 32))
    if kind == "rules":
        high = _log(rng, 1, 32768)
        return dict(kind=kind, rows=_log(rng, 1, max(1, min(
                        128, 33 * 32768 // high))),
                    vocab=rng.choice(VOCABS), low=rng.randint(high // 4, high),
                    high=high, biases=rng.choice((0, 0, _log(rng, 1, 300))),
                    masked=rng.random() < 0.4, f32=rng.random() < 0.25)
    cols = rng.choice((1023, 1024, 1536, 3584, 4096, 8960, 14336))
    return dict(kind=kind, rows=_log(rng, 1, 8192), cols=cols,
                p=rng.choice((0.05, 0.1, 0.2, 0.5)),
                dtype=rng.choice(("bfloat16", "bfloat16", "float32", "float16")))


# ------------------------------------------------------------------ sizes


def _lens(case):
    """Lengths spread evenly from low to high."""
    n, lo, hi = case["rows"], case["low"], case["high"]
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _has_adapter(case):
    """One request in eight, if there are as many, has none."""
    return [i % 8 != 7 for i in range(case["rows"])]


def _ranks(case):
    r = case["rank"]
    return [max(r // 2, 1) if case["mixed"] and s % 2 else r
            for s in range(case["slots"])]


def _layers(case):
    """(inner width, widths of the parts) of a layer's four projections."""
    h, qkv, ff = MODELS[case["model"]]
    return [(h, qkv), (qkv[0], (h,)), (h, (ff, ff)), (ff, (h,))]


def work(case):
    if case["kind"] == "dropout":
        n = case["rows"] * case["cols"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 4 * n * size, "flops": 4 * n}
    if case["kind"] == "rules":
        n, v = case["rows"], case["vocab"]
        size = 4 if case["f32"] else 2
        return {"bytes": n * v * 2 * size + 4 * sum(_lens(case))
                + (n * ((v + 31) // 32) * 4 if case["masked"] else 0)
                + 8 * n * case["biases"],
                "flops": 5 * sum(_lens(case))}
    size = 4 if case["f32"] else 2
    lens, has, ranks = _lens(case), _has_adapter(case), _ranks(case)
    rows = sum(lens)
    served = sum(n for n, h in zip(lens, has) if h)
    # requests with an adapter take the slots in turn
    used = [0] * case["slots"]
    at = 0
    for n, h in zip(lens, has):
        if h:
            used[at % case["slots"]] += n
            at += 1
    bytes_, flops = 0, 0
    for k, widths in _layers(case):
        n, p = sum(widths), len(widths)
        bytes_ += size * (served * k + 2 * rows * n)
        for tokens, r in zip(used, ranks):
            if tokens:
                bytes_ += size * r * (p * k + n)
                flops += 2 * tokens * r * (p * k + n)
    return {"bytes": bytes_, "flops": flops}


# ----------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    if case["kind"] == "adapters":
        return _prepare_adapters(case, g, host)
    if case["kind"] == "rules":
        return _prepare_rules(case, g, host)
    dt = getattr(torch, case["dtype"])
    shape = (case["rows"], case["cols"])
    return {"case": case,
            "x": torch.randn(shape, generator=g, device=DEV).to(dt),
            "dy": torch.randn(shape, generator=g, device=DEV).to(dt),
            "seed": torch.randint(-1 << 62, 1 << 62, (1,), generator=g,
                                  device=DEV)}


def _prepare_adapters(case, g, host):
    dt = torch.float32 if case["f32"] else torch.bfloat16
    slots, rank = case["slots"], case["rank"]
    lens, has, ranks = _lens(case), _has_adapter(case), _ranks(case)
    # slots in any order, but of full and half rank in turn, as work() counts them
    names = torch.randperm(slots, generator=host).tolist()
    evens = [s for s in names if s % 2 == 0]
    odds = [s for s in names if s % 2]
    turn = [(odds if i % 2 else evens)[i // 2] for i in range(slots)]
    slot, at = [], 0
    for h in has:
        slot.append(turn[at % slots] if h else -1)
        at += h
    # requests in any order; (slot, its rows) as the program that packed them knows
    order = torch.randperm(case["rows"], generator=host).tolist()
    index, rows = [], {}
    for i in order:
        rows.setdefault(slot[i], []).extend(
            range(len(index), len(index) + lens[i]))
        index.extend([slot[i]] * lens[i])
    t = len(index)

    def rand(*shape, scale=1.0):
        x = torch.empty(shape, dtype=dt, device=DEV)
        for part in x.split(max(1, (1 << 26) // max(x[0].numel(), 1))):
            part.copy_(torch.randn(part.shape, generator=g, device=DEV) * scale)
        return x
    past = torch.arange(rank, device=DEV) >= torch.tensor(
        ranks, device=DEV).unsqueeze(1)
    layers = []
    for k, widths in _layers(case):
        a = rand(slots, len(widths), rank, k, scale=k ** -0.5)
        b = rand(slots, sum(widths), rank, scale=0.1)
        # a pool of one rank: what an adapter of a smaller one leaves is zero
        a.masked_fill_(past[:, None, :, None], 0)
        b.masked_fill_(past[:, None, :], 0)
        layers.append(dict(x=rand(t, k), y=rand(t, sum(widths)), a=a, b=b,
                           widths=widths))
    ii = dict(dtype=torch.int32, device=DEV)
    return {"case": case, "layers": layers, "index": torch.tensor(index, **ii),
            "scale": torch.full((slots,), 2.0, device=DEV),
            "ranks": torch.tensor(ranks, **ii),
            "rows": {s: torch.tensor(r, device=DEV) for s, r in rows.items()}}


def _prepare_rules(case, g, host):
    n, v = case["rows"], case["vocab"]
    dt = torch.float32 if case["f32"] else torch.bfloat16
    slots = n + n // 3 + 1
    lens = _lens(case)
    cap = max(max(lens), 1)
    rows = torch.randperm(slots, generator=host)[:n]
    total = torch.zeros(slots, dtype=torch.int32)
    total[rows] = torch.tensor(lens, dtype=torch.int32)
    # prompts are up to half of the history; words repeat as words do
    prompt = (total.double() * torch.rand(slots, generator=host) / 2).int()
    history = (torch.rand(slots, cap, generator=g, device=DEV) ** 6 * v).int()
    history.clamp_(max=v - 1)

    def spread(low, high):
        x = torch.rand(slots, generator=g, device=DEV) * (high - low) + low
        return x
    state = {"case": case,
             "logits": (torch.randn(n, v, generator=g, device=DEV) * 4).to(dt),
             "rows": rows.to(DEV).int(), "history": history,
             "prompt_len": prompt.to(DEV), "total_len": total.to(DEV),
             "repetition": spread(1.0, 1.3), "frequency": spread(0.0, 0.5),
             "presence": spread(0.0, 0.5), "bias_tokens": None,
             "bias_values": None, "mask": None}
    if case["biases"]:
        nb = case["biases"]
        step = v // nb                       # no token twice
        first = torch.randint(0, step, (slots, nb), generator=g, device=DEV)
        state["bias_tokens"] = (first + torch.arange(nb, device=DEV) * step).int()
        state["bias_values"] = torch.randn(slots, nb, generator=g, device=DEV) * 5
    if case["masked"]:
        w = (v + 31) // 32
        words = torch.randint(-1 << 31, 1 << 31, (2, slots, w), generator=g,
                              device=DEV)
        state["mask"] = (words[0] & words[1]).int()     # a token in four
    if own:
        import polyrl_amd.ops as ops
        rules = ops.LogitRules(slots, v, cap, DEV, biases=case["biases"])
        for name in ("history", "prompt_len", "total_len", "repetition",
                     "frequency", "presence"):
            getattr(rules, name).copy_(state[name])
        if case["biases"]:
            rules.bias_tokens.copy_(state["bias_tokens"])
            rules.bias_values.copy_(state["bias_values"])
        if case["masked"]:
            rules.mask.copy_(state["mask"])
            rules.masked.fill_(1)
        state["rules"] = rules
    return state


# ------------------------------------------------------------------ passes


def run(state):
    kind = state["case"]["kind"]
    if own:
        import polyrl_amd.ops as ops
        if kind == "adapters":
            plan = ops.adapter_plan(state["index"], state["case"]["slots"])
            return [ops.adapter_add(p["y"], p["x"], p["a"], p["b"], state["scale"],
                                    plan, widths=p["widths"], ranks=state["ranks"])
                    for p in state["layers"]]
        if kind == "rules":
            return ops.adjust_logits(state["logits"], state["rules"],
                                     state["rows"])
        x = state["x"].detach().requires_grad_()
        y = ops.dropout_train(x, state["case"]["p"], state["seed"])
        dx, = torch.autograd.grad(y, x, state["dy"])
        return [y.detach(), dx]
    if kind == "adapters":
        return [_adapters_plain(state, p) for p in state["layers"]]
    if kind == "rules":
        return _rules_plain(state)
    keep, scale = _keep(state["x"].numel(), state["case"]["p"], state["seed"])
    keep = keep.view_as(state["x"])
    return [torch.where(keep, t.float() * scale, 0.0).to(t.dtype)
            for t in (state["x"], state["dy"])]


def _adapters_plain(state, p):
    x, y, a, b = p["x"], p["y"], p["a"], p["b"]
    if state["case"]["high"] == 1:
        # single tokens: every row's own matrices, gathered
        index = state["index"]
        slot = index.clamp(min=0).long()
        scale = torch.where(index < 0, 0.0, state["scale"][slot])
        h = torch.matmul(a[slot].flatten(1, 2).float(),
                         x.float().unsqueeze(-1)).squeeze(-1)
        h = h.view(len(x), a.shape[1], -1) * scale[:, None, None]
        out = y.float()
        at = 0
        for i, n in enumerate(p["widths"]):
            out[:, at:at + n] += torch.matmul(
                b[:, at:at + n][slot].float(), h[:, i].unsqueeze(-1)).squeeze(-1)
            at += n
        return out.to(y.dtype)
    out = y.clone()
    for s, rows in state["rows"].items():
        if s < 0:
            continue
        xs = x.index_select(0, rows).float()
        total = y.index_select(0, rows).float()
        at = 0
        for i, n in enumerate(p["widths"]):
            h = (xs @ a[s, i].float().t()) * state["scale"][s]
            total[:, at:at + n] += h @ b[s, at:at + n].float().t()
            at += n
        out.index_copy_(0, rows, total.to(y.dtype))
    return out


def _rules_plain(state):
    logits, rows = state["logits"], state["rows"].long()
    n, v = logits.shape
    history = state["history"][rows].long()
    place = torch.arange(history.shape[1], device=DEV)
    prompt = state["prompt_len"][rows].unsqueeze(1)
    total = state["total_len"][rows].unsqueeze(1)
    said = ((place >= prompt) & (place < total)).float()
    asked = (place < prompt).float()
    count = torch.zeros(n, v, device=DEV).scatter_add_(1, history, said)
    seen = torch.zeros(n, v, device=DEV).scatter_add_(1, history, asked)
    seen = (seen + count) > 0
    x = logits.float()
    rep = state["repetition"][rows].unsqueeze(1)
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - state["frequency"][rows].unsqueeze(1) * count
    x = x - torch.where(count > 0, state["presence"][rows].unsqueeze(1), 0.0)
    if state["bias_tokens"] is not None:
        x = x.scatter_add(1, state["bias_tokens"][rows].long(),
                          state["bias_values"][rows])
    if state["mask"] is not None:
        bits = torch.arange(32, dtype=torch.int32, device=DEV)
        allowed = (state["mask"][rows].unsqueeze(-1) >> bits) & 1
        x = torch.where(allowed.flatten(1)[:, :v] != 0, x, -math.inf)
    return x.to(logits.dtype)


# Philox4x32-10: Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
# 1, 2, 3", SC 2011
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)


def _steps(p):
    return int(round(p * 65536))


def _keep(numel, p, seed):
    """Whether each element stays, and what it is multiplied by."""
    low = (1 << 32) - 1
    block = torch.arange((numel + 7) // 8, device=DEV)
    c = [block & low, block >> 32, torch.zeros_like(block),
         torch.zeros_like(block)]
    key = [seed & low, (seed >> 32) & low]
    for i in range(10):
        p0, p1 = c[0] * PHILOX_M[0], c[2] * PHILOX_M[1]
        c = [((p1 >> 32) & low) ^ c[1] ^ key[0], p1 & low,
             ((p0 >> 32) & low) ^ c[3] ^ key[1], p0 & low]
        key = [(key[0] + PHILOX_W[0]) & low, (key[1] + PHILOX_W[1]) & low]
    words = torch.stack(c, -1)
    bits = torch.stack([words & 0xffff, words >> 16], -1).flatten()[:numel]
    n = _steps(p)
    return bits >= n, 65536.0 / (65536 - n)


# ------------------------------------------------------------------- exact


def exact(case, seed):
    if case["kind"] == "dropout":
        return _exact_dropout(case, prepare(case, seed))
    if case["kind"] == "rules":
        return _exact_rules(case, prepare(case, seed))
    state = prepare(case, seed)
    index = state["index"].tolist()
    outs = []
    for p in state["layers"]:
        out = p["y"].double()
        starts = [sum(p["widths"][:i]) for i in range(len(p["widths"]) + 1)]
        for s in sorted(set(index)):
            if s < 0:
                continue
            rows = torch.tensor([t for t, i in enumerate(index) if i == s],
                                device=DEV)
            xs = p["x"][rows].double()
            r = _ranks(case)[s]
            for i, (lo, hi) in enumerate(zip(starts, starts[1:])):
                h = xs @ p["a"][s, i, :r].double().t()
                out[rows, lo:hi] += float(state["scale"][s]) * (
                    h @ p["b"][s, lo:hi, :r].double().t())
        outs.append(out)
    return outs


def _exact_rules(case, state):
    out = state["logits"].double().cpu().numpy()
    get = {k: v.cpu().numpy() for k, v in state.items()
           if isinstance(v, torch.Tensor) and k != "logits"}
    for i, s in enumerate(get["rows"]):
        words = get["history"][s]
        prompt, total = get["prompt_len"][s], get["total_len"][s]
        seen = np.unique(words[:total])
        said, count = np.unique(words[prompt:total], return_counts=True)
        rep = float(get["repetition"][s])
        x = out[i]
        x[seen] = np.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
        x[said] -= float(get["frequency"][s]) * count + float(get["presence"][s])
        if case["biases"]:
            np.add.at(x, get["bias_tokens"][s],
                      get["bias_values"][s].astype(np.float64))
        if case["masked"]:
            bits = np.unpackbits(get["mask"][s].view(np.uint8),
                                 bitorder="little")[:case["vocab"]]
            x[bits == 0] = -np.inf
    return torch.from_numpy(out)


def _exact_dropout(case, state):
    numel = case["rows"] * case["cols"]
    seed = int(state["seed"]) & ((1 << 64) - 1)
    blocks = np.arange((numel + 7) // 8, dtype=np.uint64)
    u32, mask = np.uint64(32), np.uint64(0xffffffff)
    x0, x1 = blocks & mask, blocks >> u32
    x2, x3 = np.zeros_like(blocks), np.zeros_like(blocks)
    k0, k1 = seed & 0xffffffff, seed >> 32
    for _ in range(10):
        m0, m1 = x0 * np.uint64(PHILOX_M[0]), x2 * np.uint64(PHILOX_M[1])
        x0, x1, x2, x3 = ((m1 >> u32) ^ x1 ^ np.uint64(k0), m1 & mask,
                          (m0 >> u32) ^ x3 ^ np.uint64(k1), m0 & mask)
        k0 = (k0 + PHILOX_W[0]) & 0xffffffff
        k1 = (k1 + PHILOX_W[1]) & 0xffffffff
    words = np.stack([x0, x1, x2, x3], -1).astype(np.uint32)
    bits = words.view(np.uint16).reshape(-1)[:numel]
    dropped = torch.from_numpy(bits.astype(np.int32) < _steps(case["p"])).to(
        DEV).view(case["rows"], case["cols"])
    part = 1 - _steps(case["p"]) / 65536
    return [(t.double() / part).masked_fill_(dropped, 0)
            for t in (state["x"], state["dy"])]
