"""Whole models over the 8-bit cache against a plain implementation in 64 bits that attends over the rows which the engine's own cache
held: what is left between the two is a bfloat16 run's rounding, so a moderate mistake in a sum, a scale or a position shows."""
import pytest
import torch

import plain_e4m3_model as M
import test_cache_e4m3_engine_gpu as E
import traces as T
from tiny_configs import random_tokens

pytestmark = pytest.mark.gpu

TRACES = {
    "whole": lambda reqs: T.whole(reqs),
    "one by one": lambda reqs: T.tail_one_by_one(reqs, 20),
    "batches": lambda reqs: T.batched(reqs, 3, [5, 17, 1, 30]),
    "pieces": lambda reqs: T.chunked(reqs, [1, 40, 7, 64, 100]),
}


def _check_trace(eng, name, mixed, trace):
    reqs = E.requests(name)
    steps = TRACES[trace](reqs)
    order = list(dict.fromkeys(e["id"] for st in steps for e in st["entries"]))       # (slots are taken in this order)
    with M.Recorder(eng) as rec:
        got = T.collect(steps, T.run_in_process(eng, steps), reqs)
    assert len(rec.taken) == len(order)
    for rid, held in zip(order, rec.taken):
        faults = M.faults(name, reqs[rid], M.rows_of(held, len(reqs[rid])), got[rid], mixed)
        assert not faults, (rid, len(reqs[rid]), faults)


@pytest.mark.parametrize("trace", list(TRACES))
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(E.SIZES))
def test_logits_and_rows(name, mixed, trace):
    _check_trace(E.engine(name, True, mixed), name, mixed, trace)


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(E.SIZES))
def test_logits_and_rows_without_graphs_and_part_by_part(name, mixed, monkeypatch):
    eng = E.engine(name, False, mixed)
    _check_trace(eng, name, mixed, "one by one")
    monkeypatch.setattr(eng.model, "prompt_runs", {})
    _check_trace(eng, name, mixed, "pieces")


@pytest.mark.parametrize("how", ["greedy", "greedy step by step", "sampled", "sampled step by step"])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(E.SIZES))
def test_generation(name, mixed, how):
    """Tokens that the generation loop feeds back: every row that a decode step stored belongs to its token and position, and every
    greedy token is the plain model's best one, or as near to it as twice the error that its logits are allowed."""
    from dlgo_b200.api import LLM
    V = E.SIZES[name][6]
    prompts = [random_tokens(n, V, n) for n in (3, 70, 200)]
    options = dict(greedy=True) if "greedy" in how else dict(temperature=0.8, seed=3)
    with M.Recorder(E.engine(name, "step" not in how, mixed)) as rec:
        outs = LLM(E.engine(name, "step" not in how, mixed)).generate(prompts, max_tokens=24, ignore_eos=True, **options)
    assert len(rec.taken) == len(prompts) and all(len(o) == 24 for o in outs)
    for prompt, out, held in zip(prompts, outs, rec.taken):
        tokens = prompt + out[:-1]
        rows = M.rows_of(held, len(tokens))
        faults = M.faults(name, tokens, rows, None, mixed)
        assert not faults, (len(prompt), faults)
        if "greedy" in how:
            ref = M.run(name, tuple(tokens), mixed, rows)[0][len(prompt) - 1:]
            behind = ref.amax(1) - ref[torch.arange(24), torch.tensor(out)]
            assert (behind <= 2 * 3e-2 * ref.abs().amax()).all(), (len(prompt), behind.tolist())


OTHERS = {   # hidden, layers, ffn, heads, kv heads, head size, vocab
    "inputs no multiple of eight": (100, 2, 260, 4, 2, 64, 300),
    "sixteen query heads to one key head": (192, 2, 320, 16, 1, 64, 300),
    "a key head each, a narrow model": (64, 2, 96, 5, 5, 128, 200),
}


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(OTHERS))
def test_other_sizes(name, mixed, monkeypatch):
    """Contractions that run on the fp32 pipes, groups beyond one block's, prompts and single tokens in one step."""
    from dlgo_b200.engine.engine import Engine
    monkeypatch.setitem(E.SIZES, name, OTHERS[name])
    spec = E.mixed_spec(name) if mixed else E.config(name).architecture_spec()
    eng = Engine(spec=spec, tensors=dict(E.tensors(name)), max_tokens=1536, cache_dtype="e4m3")
    eng.cache.poison()
    _check_trace(eng, name, mixed, "batches")
    _check_trace(eng, name, mixed, "pieces")
