"""Requests of one batch with adapters and rules of their own, through the engine, its
HTTP facade and from a trained adapter to a served one."""
import asyncio
import contextlib
import dataclasses
import gc
import math
import os
import subprocess
import sys
import weakref
from unittest import mock

import numpy as np
import pytest
import torch

from conftest import free_port, retry_run
from polyrl_amd.models import create_model, get_model_config
from polyrl_amd.models.lora import (LoRALinear, SeededDropout, apply_lora,
                                    export_adapter, merged_state_dict)
from polyrl_amd.rollout.engine import Engine, SamplingParams

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CFG = "llama-debug-cpu"


def trained(seed, r=4, targets=None, name=CFG):
    """(model with an adapter that does something, base weights)"""
    torch.manual_seed(7)
    m = create_model(get_model_config(name), kind="actor", dtype="float32",
                     device="cpu")
    base = {k: v.clone() for k, v in m.state_dict().items()}
    kw = {} if targets is None else {"targets": targets}
    apply_lora(m, r=r, alpha=2.0 * r, **kw)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for mod in m.modules():
            if isinstance(mod, LoRALinear):
                mod.lora_A.copy_(torch.randn(mod.lora_A.shape, generator=g)
                                 / mod.lora_A.shape[1] ** 0.5)
                mod.lora_B.copy_(torch.randn(mod.lora_B.shape, generator=g) * 0.08)
    return m, base


@pytest.fixture(scope="module")
def models():
    return [trained(1), trained(2, r=3, targets=("q_proj", "up_proj", "down_proj"))]


def engine(sd, name=CFG, **kw):
    e = Engine(get_model_config(name), device="cpu", dtype=torch.float32,
               kv_bytes_budget=8 << 20,
               **{"max_num_batched_tokens": 64, "max_running_requests": 8, **kw})
    e.model.load_state_dict(sd)
    return e


def serving(models, **kw):
    e = engine(models[0][1], **kw)
    for name, (m, _) in zip(("one", "two"), models):
        e.load_adapter(name, *export_adapter(m))
    return e


def run(e, jobs):
    """[(prompt, sampling)] -> outputs, all in the engine at once"""
    for i, (p, sp) in enumerate(jobs):
        e.add_request(f"r{i}", p, sp)
    outs = {}
    while e.has_work():
        for o in e.step():
            outs[o.rid] = o
    return [outs[f"r{i}"] for i in range(len(jobs))]


def greedy(n=8, **kw):
    return SamplingParams(temperature=0.0, max_new_tokens=n, **kw)


PROMPTS = [[5, 9, 2, 7], [11, 3], list(range(20, 90)), [5, 9, 2, 7]]


def test_adapters_of_one_batch_are_the_merged_models(models):
    """Base and two adapters side by side, prompts in portions: every request as from an
    engine of its own merged weights."""
    want = []
    for sd in (models[0][1], *(merged_state_dict(m) for m, _ in models)):
        want.append(run(engine(sd), [(p, greedy()) for p in PROMPTS]))
    e = serving(models)
    names = ("", "one", "two")
    jobs = [(p, greedy(adapter=a)) for p in PROMPTS for a in names]
    outs = run(e, jobs[:8]) + run(e, jobs[8:])
    for i, o in enumerate(outs):
        w = want[i % 3][i // 3]
        assert o.output_ids == w.output_ids
        assert np.allclose(o.output_logprobs, w.output_logprobs, atol=2e-4)
    assert want[0][0].output_ids != want[1][0].output_ids


def test_long_prompt_steps_of_any_order(models):
    """Steps of many rows put requests without adapter first: every request gets its own
    result, cached histories and forced tokens included."""
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist()
               for n in (300, 7, 150, 90, 1, 260, 40)]
    names = ("one", "", "two", "", "two", "", "one")
    want = {}
    for name, sd in (("", models[0][1]), ("one", merged_state_dict(models[0][0])),
                     ("two", merged_state_dict(models[1][0]))):
        want[name] = run(engine(sd, max_num_batched_tokens=2048),
                         [(p, greedy(4)) for p in prompts])
    for tokens in (2048, 600):                    # at once, and in portions
        e = serving(models, max_num_batched_tokens=tokens, max_running_requests=16)
        outs = run(e, [(p, greedy(4, adapter=a)) for p, a in zip(prompts, names)])
        for i, (o, a) in enumerate(zip(outs, names)):
            assert o.output_ids == want[a][i].output_ids
            assert np.allclose(o.output_logprobs, want[a][i].output_logprobs, atol=2e-4)


def test_groups_and_prefix_cache_keep_adapters_apart(models):
    e = serving(models, enable_radix_cache=True)
    prompt = list(range(40, 75))                  # two whole pages
    plain = serving(models)
    want = {a: run(plain, [(prompt, greedy(adapter=a))])[0].output_ids
            for a in ("", "one", "two")}
    for a in ("", "one", "", "two", "one"):
        assert run(e, [(prompt, greedy(adapter=a))])[0].output_ids == want[a]
    e.add_request_group("g", prompt, greedy(adapter="two"), 3)
    outs = []
    while e.has_work():
        outs += e.step()
    assert len(outs) == 3 and all(o.output_ids == want["two"] for o in outs)


def test_adapters_come_and_go(models):
    e = serving(models, max_adapters=2)
    assert e.adapters == ["one", "two"]
    sd, scaling = export_adapter(models[0][0])
    base = run(engine(models[0][1]), [(PROMPTS[0], greedy())])[0].output_ids
    one = run(e, [(PROMPTS[0], greedy(adapter="one"))])[0].output_ids
    with pytest.raises(RuntimeError):             # no slot left
        e.load_adapter("three", sd, scaling)
    e.unload_adapter("two")
    e.load_adapter("three", sd, scaling)          # in the slot of a smaller one
    assert run(e, [(PROMPTS[0], greedy(adapter="three"))])[0].output_ids == one
    e.load_adapter("one", sd, 0.0)                # replaced
    assert run(e, [(PROMPTS[0], greedy(adapter="one"))])[0].output_ids == base
    e.add_request("busy", PROMPTS[0], greedy(adapter="three"))
    for call in (lambda: e.unload_adapter("three"),
                 lambda: e.load_adapter("three", sd, scaling)):
        with pytest.raises(RuntimeError):
            call()
    while e.has_work():
        e.step()
    e.unload_adapter("three")
    with pytest.raises(ValueError):
        e.unload_adapter("three")
    with pytest.raises(ValueError):
        e.add_request("x", [1], greedy(adapter="three"))
    with pytest.raises(ValueError):
        e.add_request_group("x", [1], greedy(adapter="three"), 2)
    assert not e.has_work()


def test_adapters_that_do_not_fit(models):
    e = serving(models, max_adapter_rank=4)
    sd, scaling = export_adapter(models[0][0])
    key = "model.layers.0.self_attn.q_proj.lora_"
    A, B = sd[key + "A"], sd[key + "B"]
    for bad in ({}, {key + "A": A}, {key + "A": A, key + "B": B[:-1]},
                {key + "A": A[:, :-1], key + "B": B},
                {key + "A": A[:3], key + "B": B},
                {key + "A": torch.cat([A, A]), key + "B": torch.cat([B, B], 1)},
                {key.replace("0", "9") + "A": A, key.replace("0", "9") + "B": B},
                {key.replace("q_", "x_") + "A": A},
                {key + "A": A, key + "A.weight": A, key + "B": B}):
        with pytest.raises(ValueError):
            e.load_adapter("bad", bad, scaling)
    with pytest.raises(ValueError):
        e.load_adapter("bad", sd, float("nan"))
    assert e.adapters == ["one", "two"]
    # names of other programs' files
    e.unload_adapter("two")
    e.load_adapter("two", {"base_model.model." + k + ".weight": v
                           for k, v in sd.items()}, scaling)
    assert run(e, [(PROMPTS[0], greedy(adapter="two"))])[0].output_ids == \
        run(e, [(PROMPTS[0], greedy(adapter="one"))])[0].output_ids
    for name in ("gpt2-debug", "kuforax-debug"):
        other = Engine(get_model_config(name), device="cpu", dtype=torch.float32,
                       kv_token_capacity=256, max_running_requests=2)
        with pytest.raises(ValueError):
            other.load_adapter("one", sd, scaling)
        with pytest.raises(ValueError):
            other.add_request("x", [1], greedy(adapter="one"))


# ------------------------------------------------------------------- rules


def test_refused_replacements_leave_what_was_there(models):
    """A scaling that 32 bits do not hold, tensors that do not convert: the adapter of that name answers as before."""
    e = serving(models)
    job = [(PROMPTS[0], greedy(adapter="one"))]
    want, = run(e, job)
    sd, _ = export_adapter(models[1][0])
    held = [t.clone() for layer in e.model.adapters.layers for p in layer.values()
            for t in p]
    for scaling in (1e39, -1e60, math.inf, math.nan):
        with pytest.raises(ValueError):
            e.load_adapter("one", sd, scaling)
    with pytest.raises(ValueError):               # of a new name: no slot is taken
        e.load_adapter("three", sd, 1e39)
    last = list(sd)[-1]
    with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
        e.load_adapter("one", {**sd, last: sd[last].to("meta")}, 1.0)
    assert e.adapters == ["one", "two"]
    now = [t for layer in e.model.adapters.layers for p in layer.values() for t in p]
    assert all(torch.equal(a, b) for a, b in zip(now, held))
    got, = run(e, job)
    assert got.output_ids == want.output_ids
    assert got.output_logprobs == want.output_logprobs


def rolled(models, prompt, sp, adapter=""):
    """Greedy tokens under rules and the model's own log-probabilities, token by token
    from the trainer's model."""
    sd = {"": models[0][1]}.get(adapter) or merged_state_dict(
        models[("one", "two").index(adapter)][0])
    m = create_model(get_model_config(CFG), kind="actor", dtype="float32",
                     device="cpu")
    m.load_state_dict(sd)
    ids, out, lps = list(prompt), [], []
    for _ in range(sp.max_new_tokens):
        with torch.no_grad():
            x = m(torch.tensor([ids]))[0, -1].float()
        lp = torch.log_softmax(x, -1)
        for t in set(ids):
            if sp.repetition_penalty != 1.0:
                x[t] = x[t] / sp.repetition_penalty if x[t] > 0 \
                    else x[t] * sp.repetition_penalty
        for t in set(out):
            x[t] -= sp.frequency_penalty * out.count(t) + sp.presence_penalty
        for t, v in dict(sp.logit_bias).items():
            x[t] += v
        if sp.allowed_token_ids:
            keep = torch.zeros(len(x), dtype=torch.bool)
            keep[list(sp.allowed_token_ids)] = True
            x[~keep] = -math.inf
        t = int(x.argmax())
        out.append(t)
        lps.append(float(lp[t]))
        ids.append(t)
    return out, lps


RULES = [dict(), dict(repetition_penalty=1.4), dict(frequency_penalty=3.0),
         dict(presence_penalty=2.0, logit_bias=((17, 4.0), (300, -1.0))),
         dict(allowed_token_ids=tuple(range(100, 140)), frequency_penalty=0.5),
         dict(logit_bias={5: -math.inf, 9: 3.0}, repetition_penalty=0.8)]


def test_rules_of_one_batch(models):
    """Six requests with rules, some with adapters, in chunks of decode steps; their
    log-probabilities are the model's."""
    e = serving(models)
    jobs = [(PROMPTS[i % 4], greedy(20, adapter=("", "one", "two")[i % 3], **kw))
            for i, kw in enumerate(RULES)]
    for (p, sp), o in zip(jobs, run(e, jobs)):
        ids, lps = rolled(models, p, sp, sp.adapter)
        assert o.output_ids == ids
        assert np.allclose(o.output_logprobs, lps, atol=2e-4)
        assert o.finish_reason == "length"


def test_penalties_reach_what_they_say(models):
    e = engine(models[0][1])
    base, distinct, banned = run(e, [
        (PROMPTS[0], greedy(30)), (PROMPTS[0], greedy(30, frequency_penalty=1e4)),
        (PROMPTS[0], greedy(30, logit_bias={t: -math.inf for t in range(400)}))])
    assert len(set(distinct.output_ids)) == 30
    assert min(banned.output_ids) >= 400
    assert distinct.output_ids[0] == base.output_ids[0]


def test_grammar(models):
    """A mask for every token, as ids or as words; where nothing may follow the
    request ends."""
    from polyrl_amd.ops import token_words
    calls = []

    def spell(out):
        calls.append(list(out))
        word = [7, 300, 12]
        return [word[len(out)], 511] if len(out) < 2 else \
            token_words([word[2]], 512) if len(out) == 2 else []
    e = engine(models[0][1], enable_radix_cache=True)
    bias = {511: -math.inf}
    a, b, c = run(e, [(list(range(40)), greedy(9, token_mask=spell, logit_bias=bias)),
                      (PROMPTS[1], greedy(9)),
                      (PROMPTS[0], greedy(5, token_mask=lambda out: None))])
    assert a.output_ids == [7, 300, 12] and a.finish_reason == "stop"
    assert b.output_ids == run(engine(models[0][1]),
                               [(PROMPTS[1], greedy(9))])[0].output_ids
    assert c.output_ids == run(engine(models[0][1]),
                               [(PROMPTS[0], greedy(5))])[0].output_ids
    assert [7, 300] in calls
    # pages and slots are back, and what the cache kept is right
    assert run(e, [(list(range(40)), greedy(9))])[0].output_ids == run(
        engine(models[0][1]), [(list(range(40)), greedy(9))])[0].output_ids
    with pytest.raises(ValueError):               # nothing from the start
        e.add_request("x", [1], greedy(3, token_mask=lambda out: []))
    # a function that fails ends its own request
    d, f = run(e, [(PROMPTS[0], greedy(5, token_mask=lambda out: [9, 8][:2 // (2 - len(out))])),
                   (PROMPTS[1], greedy(9))])
    assert len(d.output_ids) == 2 and d.finish_reason == "abort"
    assert f.output_ids == b.output_ids


def test_masks_of_one_buffer(models):
    """A grammar that fills the same words again for every call: each request goes by what
    the words were when it was asked."""
    words = np.zeros(16, np.int32)

    def mask(ids):
        def f(out):
            words[:] = 0
            t = ids[len(out)]
            words.view(np.uint32)[t // 32] = 1 << t % 32
            return words
        return f
    ways = [[10, 11, 12], [100, 101, 102], [511, 31, 32]]
    e = engine(models[0][1])
    for o, ids in zip(run(e, [(PROMPTS[0], greedy(3, token_mask=mask(ids)))
                              for ids in ways]), ways):
        assert o.output_ids == ids
    e.add_request_group("g", PROMPTS[0], greedy(3, token_mask=mask(ways[0])), 2)
    e.add_request("x", PROMPTS[1], greedy(3, token_mask=mask(ways[1])))
    outs = {}
    while e.has_work():
        outs.update((o.rid, o.output_ids) for o in e.step())
    assert outs == {"g-s0": ways[0], "g-s1": ways[0], "x": ways[1]}


def test_more_requests_than_slots(models):
    """Groups that fork past the running limit, and biases that outgrow the table."""
    e = engine(models[0][1], max_running_requests=2)
    sp = SamplingParams(temperature=1.0, max_new_tokens=12, frequency_penalty=1e4)
    e.add_request_group("g", PROMPTS[0], sp, 7)
    outs = []
    while e.has_work():
        outs += e.step()
    assert len(outs) == 7
    assert all(len(set(o.output_ids)) == 12 for o in outs)
    jobs = [(PROMPTS[0], greedy(6, logit_bias={t: -math.inf for t in range(n)}))
            for n in (0, 3, 50, 400)]
    for (p, sp), o in zip(jobs, run(e, jobs)):
        assert o.output_ids == rolled(models, p, sp)[0]
    assert not e.rules._slots


def test_captured_steps_go_with_their_table(models):
    """When the rules' tables are made larger the old ones are let go, with every step that
    was captured over them; the other steps stay."""
    e = engine(models[0][1])
    run(e, [(PROMPTS[0], greedy(3, logit_bias={5: 1.0}))])
    old = weakref.ref(e.rules.table)
    with no_collector():
        e._graphs = {4: {"rules": None}, (4, True, False): {"rules": old()},
                     (2, True, True): {"rules": old()}, (2, False, True): {"rules": None}}
        e._graph_pool = (0, 1)
        run(e, [(PROMPTS[0], greedy(3, logit_bias={6: 1.0}))])
        assert old() is e.rules.table and len(e._graphs) == 4
        run(e, [(PROMPTS[0], greedy(3, logit_bias={t: 1.0 for t in range(9)}))])
        assert list(e._graphs) == [4, (2, False, True)] and e._graph_pool == (0, 1)
        assert old() is None
        # a pool that no captured step holds any more cannot be taken again
        e._graphs = {(4, True, False): {"rules": e.rules.table}}
        run(e, [(PROMPTS[0], greedy(3, logit_bias={t: 1.0 for t in range(99)}))])
        assert e._graphs == {} and e._graph_pool is None


def test_rules_that_cannot_hold(models):
    e = engine(models[0][1])
    inf = math.inf
    for kw in (dict(repetition_penalty=0.0), dict(repetition_penalty=inf),
               dict(frequency_penalty=math.nan), dict(presence_penalty=inf),
               dict(logit_bias={512: 1.0}), dict(logit_bias={-1: 1.0}),
               dict(logit_bias={1: math.nan}), dict(logit_bias={1: inf}),
               dict(allowed_token_ids=(512,)), dict(allowed_token_ids=(-1,)),
               dict(allowed_token_ids=(3, 4), logit_bias={3: -inf, 4: -inf}),
               dict(logit_bias={t: -inf for t in range(512)})):
        with pytest.raises(ValueError):
            e.add_request("x", [1, 2], greedy(**kw))
    with pytest.raises(ValueError):               # longer than a history
        e.add_request("x", [1] * 1026, greedy(presence_penalty=1.0))
    assert not e.has_work()


def test_rules_that_32_bits_do_not_hold(models):
    """1e60 is infinite to the kernels: refused like infinities, and a ban below."""
    e = engine(models[0][1])
    v = e.cfg.vocab_size
    for kw in (dict(repetition_penalty=1e-60), dict(repetition_penalty=1e60),
               dict(frequency_penalty=1e60), dict(presence_penalty=-1e60),
               dict(logit_bias={3: 1e60}), dict(logit_bias={t: -1e60 for t in range(v)}),
               dict(logit_bias={3: -1e60}, allowed_token_ids=(3,))):
        with pytest.raises(ValueError):
            e.add_request("r", PROMPTS[0], greedy(4, **kw))
    assert not e.has_work()
    out, = run(e, [(PROMPTS[0], greedy(4, logit_bias={3: -1e60},
                                       allowed_token_ids=(3, 5)))])
    assert out.output_ids == [5] * 4


@pytest.mark.parametrize("sharing", [True, False])
@pytest.mark.parametrize("n", [1, 3])
def test_groups_are_admitted_whole(models, sharing, n):
    """One question to a token_mask decides on all samples of a group: none is left behind
    by a refusal of another."""
    e = engine(models[0][1])
    e.enable_prefix_sharing = sharing
    asked = []

    def mask(out):
        asked.append(list(out))
        if len(asked) > 1 and not out:
            raise KeyError("asked twice")
        return [7]
    e.add_request_group("g", PROMPTS[0], greedy(2, token_mask=mask), n)
    assert asked == [[]]
    outs = []
    while e.has_work():
        outs += e.step()
    assert sorted(o.rid for o in outs) == [f"g-s{i}" for i in range(n)]
    assert all(o.output_ids == [7, 7] for o in outs)


def test_numbers_that_no_table_holds(models):
    """Token ids beyond 64 bits, numbers beyond floats, a mask that fails at once: the
    request is refused as others are."""
    from polyrl_amd.ops import LogitRules, token_words
    e = engine(models[0][1])

    def fails(out):
        raise KeyError("state")
    for kw in (dict(allowed_token_ids=(2 ** 70,)), dict(allowed_token_ids=(-2 ** 70, 3)),
               dict(logit_bias={3: 10 ** 400}), dict(logit_bias={2 ** 70: 1.0}),
               dict(frequency_penalty=10 ** 400), dict(presence_penalty=-10 ** 400),
               dict(repetition_penalty=10 ** 400), dict(token_mask=fails),
               dict(token_mask=lambda out: [2 ** 70])):
        with pytest.raises(ValueError):
            e.add_request("x", [1, 2], greedy(**kw))
        with pytest.raises(ValueError):
            e.add_request_group("g", [1, 2], greedy(**kw), 2)
    assert not e.has_work()
    out, = run(e, [(PROMPTS[0], greedy(3, logit_bias={3: -10 ** 400},
                                       allowed_token_ids=(3, 5)))])
    assert out.output_ids == [5] * 3              # a ban, as any below 32 bits
    with pytest.raises(ValueError):
        token_words([2 ** 70], 512)
    rules = LogitRules(1, 8, 4, "cpu", biases=1)
    for kw in (dict(frequency=10 ** 400), dict(allowed=[2 ** 70]),
               dict(bias={2 ** 70: 1.0})):
        with pytest.raises(ValueError):
            rules.set(0, **kw)
    rules.set(0, bias={1: -10 ** 400})
    assert rules.bias_values[0, 0] == -math.inf
    with pytest.raises(ValueError):
        e.load_adapter("x", export_adapter(models[0][0])[0], 10 ** 400)


def test_rules_on_hybrid_decoders():
    e = Engine(get_model_config("kuforax-debug"), device="cpu", dtype=torch.float32,
               kv_token_capacity=512, max_running_requests=4)
    e.model.init_random(0)
    outs = run(e, [([1, 2, 3], greedy(10, frequency_penalty=1e4)),
                   ([4, 5], greedy(10)),
                   ([4, 5], greedy(10, allowed_token_ids=(8, 9)))])
    assert len(set(outs[0].output_ids)) == 10
    assert set(outs[2].output_ids) <= {8, 9}


# -------------------------------------------------------------------- HTTP


def test_http(models, tmp_path):
    import httpx
    from safetensors.torch import save, save_file

    from polyrl_amd.rollout.runner import EngineRunner
    from polyrl_amd.server import create_app
    e = engine(models[0][1])
    runner = EngineRunner(e)
    app = create_app(e, runner)
    sd, scaling = export_adapter(models[0][0])
    save_file(sd, str(tmp_path / "a.safetensors"))

    async def go():
        async with httpx.AsyncClient(transport=httpx.ASGITransport(app=app),
                                     base_url="http://t") as c:
            async def gen(**sp):
                return await c.post("/generate", json={
                    "input_ids": PROMPTS[0], "return_logprob": True,
                    "sampling_params": {"max_new_tokens": 8, "temperature": 0.0, **sp}})
            r = await gen(adapter="one")
            assert r.status_code == 400 and "one" in r.json()["message"]
            r = await c.post("/load_adapter", content=save(sd), headers={
                "x-adapter-name": "one", "x-adapter-scaling": str(scaling)})
            assert r.json() == {"success": True, "adapters": ["one"]}
            r = await c.post("/load_adapter", json={
                "name": "file", "path": str(tmp_path / "a.safetensors"),
                "scaling": scaling})
            assert r.json()["adapters"] == ["one", "file"]
            r = await c.post("/load_adapter", json={"name": "x", "path": "/no/file"})
            assert r.status_code == 400
            a = (await gen(adapter="one")).json()[0]["output_ids"]
            assert a == (await gen(adapter="file")).json()[0]["output_ids"]
            assert a == run(engine(merged_state_dict(models[0][0])),
                            [(PROMPTS[0], greedy())])[0].output_ids
            b = (await gen(frequency_penalty=1e4)).json()[0]["output_ids"]
            assert len(set(b)) == 8
            r = await gen(allowed_token_ids=[6, 7], logit_bias={"6": "-inf"})
            assert r.json()[0]["output_ids"] == [7] * 8
            r = await gen(n=2, repetition_penalty=-1.0)
            assert r.status_code == 400
            r = await c.post("/unload_adapter", json={"name": "file"})
            assert r.json()["adapters"] == ["one"]
            r = await c.post("/unload_adapter", json={"name": "file"})
            assert r.status_code == 400
        assert not runner._futures
    asyncio.run(go())
    runner.stop()


def test_refused_requests_leave_no_future(models, monkeypatch):
    """Whatever the engine raises when it is asked, nobody is left waiting."""
    from polyrl_amd.rollout.runner import EngineRunner
    e = engine(models[0][1])
    runner = EngineRunner(e)

    async def go():
        for error in (OverflowError, KeyError, TypeError, AssertionError):
            def refuse(*a):
                raise error
            for name in ("add_request", "add_request_group"):
                monkeypatch.setattr(e, name, refuse)
            with pytest.raises(error):
                runner.submit([1], greedy())
            with pytest.raises(error):
                runner.submit_group([1], greedy(), 3)
            assert not runner._futures
    asyncio.run(go())
    runner.stop()


def test_http_numbers_and_bodies_of_any_kind(models):
    httpx = pytest.importorskip("httpx")
    from polyrl_amd.rollout.runner import EngineRunner
    from polyrl_amd.server.engine_server import create_app
    e = engine(models[0][1])
    runner = EngineRunner(e)
    app = create_app(e, runner)
    big = "1" + "0" * 400

    async def go():
        async with httpx.AsyncClient(transport=httpx.ASGITransport(
                app=app, raise_app_exceptions=False), base_url="http://t") as c:
            kind = {"content-type": "application/json"}
            for sp in ('"allowed_token_ids": [%s]' % big, '"logit_bias": {"3": %s}' % big,
                       '"logit_bias": {"%s": 1}' % big, '"allowed_token_ids": [Infinity]',
                       '"frequency_penalty": %s' % big, '"top_k": Infinity',
                       '"allowed_token_ids": [%d]' % 2 ** 70):
                r = await c.post("/generate", headers=kind, content=
                                 '{"input_ids": [1, 2], "sampling_params": {%s}}' % sp)
                assert r.status_code == 400, sp
            for body in ("[]", "5", "null", '"a"', "{", "",
                         '{"name": "a", "path": "/no", "scaling": %s}' % big):
                for where in ("/load_adapter", "/unload_adapter"):
                    r = await c.post(where, headers=kind, content=body)
                    assert r.status_code == 400, (where, body)
                    assert r.json()["success"] is False
        assert not runner._futures and not e.has_work() and not e.adapters
    asyncio.run(go())
    runner.stop()


# ---------------------------------------------------- from training to serving


def test_trained_with_dropout_and_served(models):
    """Adapter training with seeded dropout, the same gradients when activations are
    computed again, and the adapter served beside the base model."""
    torch.manual_seed(3)
    m = create_model(get_model_config(CFG), kind="actor", dtype="float32",
                     device="cpu")
    base = {k: v.clone() for k, v in m.state_dict().items()}
    apply_lora(m, r=4, alpha=8.0, seeded_dropout=0.25)
    assert sum(isinstance(x, SeededDropout) for x in m.modules()) == 14
    ids = torch.randint(0, 512, (2, 24))
    params = [p for p in m.parameters() if p.requires_grad]
    with torch.no_grad():
        for p in params:
            p.normal_(0, 0.05)

    def grads(again):
        torch.manual_seed(11)
        m.train()
        call = (lambda: torch.utils.checkpoint.checkpoint(
            m, ids, use_reentrant=False)) if again else (lambda: m(ids))
        loss = torch.nn.functional.cross_entropy(
            call()[:, :-1].flatten(0, 1).float(), ids[:, 1:].flatten())
        return torch.autograd.grad(loss, params)
    a, b = grads(False), grads(True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    torch.manual_seed(12)
    m.train()
    other = m(ids)
    m.eval()
    assert not torch.allclose(other, m(ids))      # dropout acts in training alone
    assert torch.equal(m(ids), m(ids))
    with torch.no_grad():
        for p, g in zip(params, a):
            p -= 0.5 * g
    e = engine(base)
    e.load_adapter("mine", *export_adapter(m))
    got, plain = run(e, [(PROMPTS[0], greedy(adapter="mine")),
                         (PROMPTS[0], greedy())])
    assert got.output_ids == run(engine(merged_state_dict(m)),
                                 [(PROMPTS[0], greedy())])[0].output_ids
    assert plain.output_ids == run(engine(base),
                                   [(PROMPTS[0], greedy())])[0].output_ids


def test_dropout_of_lora_refusals():
    lin = torch.nn.Linear(4, 4)
    for kw in (dict(seeded_dropout=1.5), dict(dropout=0.1, seeded_dropout=0.1)):
        with pytest.raises(ValueError):
            LoRALinear(lin, 2, **kw)
    with pytest.raises(ValueError):
        export_adapter(lin)


def test_dropout_rates_that_are_none():
    """A negative rate or none at all is refused before the layer is changed."""
    for p in (-0.1, 1.5, float("nan")):
        lin = torch.nn.Linear(4, 4)
        with pytest.raises(ValueError):
            LoRALinear(lin, 2, seeded_dropout=p)
        assert lin.weight.requires_grad
    assert isinstance(LoRALinear(lin, 2, seeded_dropout=0.0).dropout,
                      torch.nn.Identity)


TP_WORKER = r"""
import sys; sys.path.insert(0, "tests")
import torch, torch.distributed as dist
dist.init_process_group("gloo")
from test_request_engine import *
from polyrl_amd.parallel.tp import TPContext
models = [trained(1), trained(2, r=3, targets=("q_proj", "up_proj", "down_proj"))]
jobs = [(p, greedy(adapter=a, frequency_penalty=f)) for p in PROMPTS[:2]
        for a in ("", "one", "two") for f in (0.0, 1.0)]
want = run(serving(models, max_running_requests=12), jobs)
got = run(serving(models, max_running_requests=12,
                  tp_ctx=TPContext(dist.group.WORLD)), jobs)
for a, b in zip(got, want):
    assert a.output_ids == b.output_ids, (a.output_ids, b.output_ids)
print("TP OK")
"""


def test_tensor_parallel_adapters(tmp_path):
    f = tmp_path / "w.py"
    f.write_text(TP_WORKER)
    env = dict(os.environ, PYTHONPATH=REPO + os.pathsep + os.environ.get("PYTHONPATH", ""))
    r = retry_run(lambda: subprocess.run(
        [sys.executable, "-m", "torch.distributed.run", "--nnodes=1",
         "--nproc-per-node", "2", "--master-addr", "127.0.0.1", "--master-port",
         free_port(), str(f)], capture_output=True, text=True, timeout=240, env=env,
        cwd=REPO))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]


# --------------------------------------------------------------------- GPU


def gpu_engine(models, graphs, **kw):
    e = Engine(get_model_config("llama-tiny"), device="cuda", dtype=torch.bfloat16,
               kv_token_capacity=1 << 15, max_running_requests=32, **kw)
    e.enable_hip_graphs = graphs
    e.model.load_state_dict(models[0][1])
    for name, (m, _) in zip(("one", "two"), models):
        e.load_adapter(name, *export_adapter(m))
    return e


@pytest.fixture(scope="module")
def tiny():
    return [trained(1, r=16, name="llama-tiny"),
            trained(2, r=5, name="llama-tiny",
                    targets=("q_proj", "v_proj", "gate_proj", "down_proj"))]


def mixed_jobs(n):
    g = torch.Generator().manual_seed(n)
    jobs = []
    for i in range(n):
        length = int(torch.randint(1, 200, (1,), generator=g))
        kw = (dict(), dict(frequency_penalty=0.7, presence_penalty=0.3),
              dict(repetition_penalty=1.3, logit_bias={3: 2.0, 900: -math.inf}),
              dict(allowed_token_ids=tuple(range(64, 512))))[i % 4]
        jobs.append((torch.randint(0, 1024, (length,), generator=g).tolist(),
                     greedy(40, adapter=("", "one", "two")[i % 3], **kw)))
    return jobs


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 13])
def test_captured_decode_is_the_eager_one(tiny, n):
    """Decode steps with adapters and rules, replayed from graphs (whose histories and
    adapters move on between replays) and issued one by one: the same tokens."""
    jobs = mixed_jobs(n)[-1:] if n == 1 else mixed_jobs(n)
    # (the products' algorithms are searched for by their first calls, whose results
    # come from others)
    run(gpu_engine(tiny, False), jobs)
    eager = gpu_engine(tiny, False)
    # attention cuts a row by the width of the page table: as wide as the captured one
    own = eager.kv.page_table

    def wide(ids):
        t = own(ids)
        return torch.nn.functional.pad(t, (0, eager._graph_max_pages - t.shape[1]))
    eager.kv.page_table = wide
    want = run(eager, jobs)
    e = gpu_engine(tiny, True)
    for again in range(2):                        # the second time by older graphs
        got = run(e, jobs)
        assert e.enable_hip_graphs and e._graphs
        for a, b in zip(got, want):
            assert a.output_ids == b.output_ids
            assert a.output_logprobs == b.output_logprobs
    allowed = [o for (p, sp), o in zip(jobs, got) if sp.allowed_token_ids]
    assert all(64 <= t < 512 for o in allowed for t in o.output_ids)


@contextlib.contextmanager
def no_collector():
    gc.collect()
    gc.disable()
    try:
        yield
    finally:
        gc.enable()


@pytest.mark.parametrize("name", ["llama-debug-cpu", "kuforax-debug"])
def test_engines_go_at_once(name):
    """An engine that is let go goes with its last reference: its captured steps are not
    left to a collector that may run while another engine captures."""
    with no_collector():
        e = Engine(get_model_config(name), device="cpu", dtype=torch.float32,
                   kv_token_capacity=512, max_running_requests=4)
        gone = [weakref.ref(t) for t in (e, e.model, e.kv)]
        assert gone[1]()._engine_owner() is e
        del e
        assert [r() for r in gone] == [None] * 3


@pytest.mark.parametrize("on", [True, False])
def test_no_collection_while_a_step_is_captured(monkeypatch, on):
    from polyrl_amd.rollout import engine as module

    @contextlib.contextmanager
    def graph(g, pool=None):
        assert not gc.isenabled()
        yield
        assert not gc.isenabled()
    monkeypatch.setattr(torch.cuda, "graph", graph)
    try:
        (gc.enable if on else gc.disable)()
        with module._captured(None):
            pass
        assert gc.isenabled() == on
        with pytest.raises(KeyError):
            with module._captured(None, 1):
                raise KeyError
        assert gc.isenabled() == on
    finally:
        gc.enable()


@pytest.mark.parametrize("on", [True, False])
def test_no_collection_while_another_thread_captures(monkeypatch, on):
    """Two engines that capture at once: the collector is off until both are done."""
    import threading

    from polyrl_amd.rollout import engine as module
    monkeypatch.setattr(torch.cuda, "graph",
                        lambda g, pool=None: contextlib.nullcontext())
    inside, leave, seen = threading.Event(), threading.Event(), []

    def second():
        with module._captured(None):
            inside.set()
            assert leave.wait(30)
            seen.append(gc.isenabled())
    thread = threading.Thread(target=second)
    try:
        (gc.enable if on else gc.disable)()
        with module._captured(None):
            thread.start()
            assert inside.wait(30)
        assert not gc.isenabled()                 # the other one goes on
        leave.set()
        thread.join(30)
        assert seen == [False] and gc.isenabled() == on
    finally:
        leave.set()
        gc.enable()


@pytest.mark.gpu
def test_captured_steps_go_with_their_engine(tiny):
    with no_collector():
        e = gpu_engine(tiny, True)
        run(e, mixed_jobs(4))
        assert e._graphs
        gone = [weakref.ref(e)] + [weakref.ref(t["tokens"]) for t in e._graphs.values()]
        del e
        assert not any(r() is not None for r in gone)


@pytest.mark.gpu
def test_steps_are_captured_anew_for_a_larger_table(tiny):
    jobs = [(p, greedy(20, logit_bias={3: 2.0})) for p, _ in mixed_jobs(3)]
    more = [(p, greedy(20, logit_bias={t: 2.0 for t in range(40)})) for p, _ in jobs]
    want = [run(gpu_engine(tiny, True), j) for j in (jobs, more)]
    for plain in (False, True):                   # with a step that stays, and without
        e = gpu_engine(tiny, True)
        if plain:
            run(e, [(p, greedy(20)) for p, _ in jobs])
        for _ in range(2):
            assert [o.output_ids for o in run(e, jobs)] == \
                [o.output_ids for o in want[0]]
        for _ in range(2):
            assert [o.output_ids for o in run(e, more)] == \
                [o.output_ids for o in want[1]]
        assert e.enable_hip_graphs and e._graphs
        assert all(st["rules"] in (None, e.rules.table) for st in e._graphs.values())


@pytest.mark.gpu
def test_plain_requests_keep_their_results_beside_others(tiny):
    """The kernels' other rows: logits of requests without adapter or rules, in a batch
    with and without ones that have them, are the same bits."""
    jobs = mixed_jobs(12)
    plain = [(p, greedy(24)) for p, _ in jobs]
    want = run(gpu_engine(tiny, True), plain)
    got = run(gpu_engine(tiny, True),
              [(p, greedy(24, frequency_penalty=0.5) if i % 3 == 0 else greedy(24))
               for i, (p, _) in enumerate(jobs)])
    for i, (a, b) in enumerate(zip(got, want)):
        if i % 3:
            assert a.output_ids == b.output_ids
            assert a.output_logprobs == b.output_logprobs


@pytest.fixture(scope="module")
def whole():
    """(an engine's maker, models) of llama-tiny with feed-forward rows in whole tiles, which
    prompts take in one kernel with the activation"""
    cfg = dataclasses.replace(get_model_config("llama-tiny"), intermediate_size=768)

    def here(f):
        def call(*args, **kw):
            with mock.patch.object(sys.modules[__name__], "get_model_config",
                                   lambda name: cfg):
                return f(*args, **kw)
        return call
    models = [here(trained)(1, r=16),
              here(trained)(2, r=5, targets=("q_proj", "v_proj", "gate_proj",
                                             "down_proj"))]
    return lambda: here(gpu_engine)(models, False)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [(300, 700, 90), (513, 20), (900, 4, 1200, 300)])
def test_plain_prompts_keep_their_results_beside_adapters(whole, lens):
    """A prompt without adapter in a step of many rows has the bits that it has beside
    prompts that name none: its gate and up stay in 32 bits until the activation."""
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in lens]
    want = run(whole(), [(p, greedy(1)) for p in prompts])
    for names in (("", "one", "two", ""), ("two", "", "one", "two"),
                  ("", "", "one", "")):
        got = run(whole(), [(p, greedy(1, adapter=a))
                            for p, a in zip(prompts, names)])
        for a, o, w in zip(names, got, want):
            if a == "":
                assert o.output_ids == w.output_ids
                assert o.output_logprobs == w.output_logprobs
            else:
                assert o.output_logprobs != w.output_logprobs


@pytest.mark.gpu
@pytest.mark.parametrize("T", [520, 1300])
def test_gate_and_up_of_adapters_beside_plain_rows(whole, T):
    """The three ways through the first half of the MLP: rows without adapter first, last or
    between, every one as among its like."""
    from polyrl_amd.rollout.engine import _gate_up
    e = whole()
    w = e.model.layers[0].w_gate_up
    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, w.shape[1], generator=g).bfloat16().cuda()
    index = torch.randint(-1, 2, (T,), generator=g, dtype=torch.int32).cuda()
    full = _gate_up(x, w)
    own = e.model.gate_up_adapted(0, x, index, e.model.adapters.plan(index), 0)
    some = e.model.gate_up_adapted(0, x, index, e.model.adapters.plan(index), None)
    has = index >= 0
    assert torch.equal(some[~has], full[~has]) and torch.equal(some[has], own[has])
    assert not torch.equal(own[~has], full[~has])
    order = torch.argsort(has.int(), stable=True)
    plain = int((~has).sum())
    x, index = x[order].contiguous(), index[order].contiguous()
    first = e.model.gate_up_adapted(0, x, index, e.model.adapters.plan(index), plain,
                                    e.model.adapters.plan(index[plain:]))
    assert torch.equal(first[:plain], full[order][:plain])
    # (the product of fewer rows may be another kernel's: a rounding of gate or up, 2^-9 of
    # them, and one of the result)
    a, b = first[plain:].float(), own[order][plain:].float()
    assert ((a - b).abs() <= 0.05 * (b.abs() + 0.1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [(5, 40), (300, 700, 90), (1500, 1200, 900, 600)])
def test_prompt_steps_against_merged_weights(tiny, lens):
    """Log-probabilities of prompts of few and many rows, adapters beside each other, are
    those of merged fp32 models: 16-bit layers round at 2^-8, in two layers of some ten
    roundings each; an adapter moves them by far more."""
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in lens]
    names = ["", "one", "two", "one"][:len(lens)]
    e = gpu_engine(tiny, False)
    got = run(e, [(p, greedy(1, adapter=a)) for p, a in zip(prompts, names)])
    states = {"": tiny[0][1], "one": merged_state_dict(tiny[0][0]),
              "two": merged_state_dict(tiny[1][0])}
    m = create_model(get_model_config("llama-tiny"), kind="actor", dtype="float32",
                     device="cpu")
    moved = []
    for p, a, o in zip(prompts, names, got):
        lp = {}
        for which in {a, ""}:
            m.load_state_dict(states[which])
            with torch.no_grad():
                lp[which] = torch.log_softmax(m(torch.tensor([p]))[0, -1].float(), -1)
        t = o.output_ids[0]
        assert abs(o.output_logprobs[0] - float(lp[a][t])) < 0.06
        if a:
            moved.append(float((lp[a] - lp[""]).abs().mean()))
    assert min(moved) > 0.2


def test_http_requests_that_say_nothing(models, tmp_path):
    """Fields of other types and files that are none are the caller's: 400."""
    httpx = pytest.importorskip("httpx")
    from polyrl_amd.rollout.runner import EngineRunner
    from polyrl_amd.server.engine_server import create_app
    e = engine(models[0][1])
    runner = EngineRunner(e)
    app = create_app(e, runner)
    (tmp_path / "none").write_bytes(b"no tensors")

    async def go():
        async with httpx.AsyncClient(transport=httpx.ASGITransport(app=app),
                                     base_url="http://t") as c:
            for sp in (dict(logit_bias={"a": 1.0}), dict(logit_bias=[1, 2]),
                       dict(repetition_penalty="high"), dict(frequency_penalty=None),
                       dict(allowed_token_ids=5), dict(allowed_token_ids=["x"])):
                r = await c.post("/generate", json={
                    "input_ids": PROMPTS[0], "sampling_params": sp})
                assert r.status_code == 400, sp
            for body in (dict(name="a", path=str(tmp_path / "none")),
                         dict(path=str(tmp_path / "none")), dict(name="a"),
                         dict(name="a", path=str(tmp_path / "none"), scaling="x")):
                r = await c.post("/load_adapter", json=body)
                assert r.status_code == 400, body
            r = await c.post("/load_adapter", content=b"no tensors",
                             headers={"x-adapter-name": "a"})
            assert r.status_code == 400
            r = await c.post("/load_adapter", content=b"", headers={
                "x-adapter-name": "a", "x-adapter-scaling": "x"})
            assert r.status_code == 400
            r = await c.post("/unload_adapter", json={})
            assert r.status_code == 400
        assert not runner._futures and not e.adapters
    asyncio.run(go())
