"""Whole models over the 8-bit cache against a plain implementation in 64 bits whose keys and values go through the cache's
definition, under every way of cutting the work."""
import dataclasses
import functools

import pytest
import torch

import plain_e4m3 as P
import traces as T
from tiny_configs import random_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

SIZES = {   # hidden, layers, ffn, heads, kv heads, head size, vocab
    "H64": (256, 2, 512, 6, 2, 64, 512),
    "H128": (192, 2, 320, 9, 1, 128, 300),
}
LENGTHS = [1, 9, 64, 65, 130, 300]


def config(name):
    from dlgo_b200.config import config_from_dict
    d, n, f, hq, hkv, hd, v = SIZES[name]
    return config_from_dict(dict(
        architectures=["LlamaForCausalLM"], hidden_size=d, num_hidden_layers=n, intermediate_size=f, num_attention_heads=hq,
        num_key_value_heads=hkv, head_dim=hd, vocab_size=v, rope_theta=10000.0, rope_scaling=None, rms_norm_eps=1e-5,
        max_position_embeddings=640, tie_word_embeddings=False, eos_token_id=None))


@functools.lru_cache(maxsize=None)
def tensors(name, sharpen=8.0):
    """Random weights; queries and keys x8, so that attention is far from uniform and a wrong key moves the logits."""
    from dlgo_b200.engine.model import CausalLM
    g = torch.Generator().manual_seed(len(name))
    out = {}
    for key, ps in sorted(CausalLM(config(name).architecture_spec()).expected_tensors().items()):
        x = torch.randn(ps.shape, generator=g) * 0.02 + (1.0 if ps.init == "one_plus_normal" else 0.0)
        out[key] = (x * (sharpen if "q_proj" in key or "k_proj" in key else 1.0)).to(torch.bfloat16)
    return out


def mixed_spec(name):
    """Layers that differ: a window in one, half of each head rotated in neighbouring pairs in the other; run twice, the last
    entry reading the second's cache."""
    from dlgo_b200.config.spec import PartSpec, RunEntry
    spec = config(name).architecture_spec()
    hd = SIZES[name][5]
    l0, l1 = spec.layers
    l0 = dataclasses.replace(l0, mixer=PartSpec("gqa_attention", {**l0.mixer.params, "window": 70, "cache_group": "win"}))
    l1 = dataclasses.replace(l1, mixer=PartSpec("gqa_attention", {**l1.mixer.params, "position_encoding": "part"}))
    rope = spec.position_encodings["rope"]
    part = PartSpec(rope.kind, {**rope.params, "rotary_dim": hd // 2, "pairing": "interleaved"})
    return dataclasses.replace(spec, layers=[l0, l1], order=[RunEntry(0), RunEntry(1), RunEntry(0), RunEntry(1, cache_of=1)],
                               position_encodings={"rope": rope, "part": part})


def rotate(x, rot, inter, theta=10000.0):
    """x [T, heads, hd] in 64 bits at positions 0 .. T - 1."""
    ang = torch.outer(torch.arange(x.shape[0]).double(), theta ** (-torch.arange(rot // 2).double() / (rot // 2)))
    c, s = ang.cos().unsqueeze(1), ang.sin().unsqueeze(1)
    out = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return out


@functools.lru_cache(maxsize=None)
def plain(name, tokens, mixed=False, quantised=True):
    """Logits [T, vocab] in 64 bits; keys and values as the 8-bit cache holds them (or as they are)."""
    d, _, _, hq, hkv, hd, _ = SIZES[name]
    w = {k: v.double() for k, v in tensors(name).items()}
    order = [(0, 70, hd, False, None), (1, None, hd // 2, True, None), (0, 70, hd, False, None), (1, None, hd // 2, True, 1)] if mixed \
        else [(0, None, hd, False, None), (1, None, hd, False, None)]
    norm = lambda x, g: x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * g  # noqa: E731
    n = len(tokens)
    x = w["model.embed_tokens.weight"][list(tokens)]
    kept = []
    i, j = torch.arange(n).view(-1, 1), torch.arange(n).view(1, -1)
    for layer, window, rot, inter, cache_of in order:
        p = f"model.layers.{layer}."
        h = norm(x, w[p + "input_layernorm.weight"])
        q, k, v = ((h @ w[p + f"self_attn.{c}_proj.weight"].T).view(n, -1, hd) for c in "qkv")
        q, k = rotate(q, rot, inter), rotate(k, rot, inter)
        if quantised:
            k, v = (s * P.two_to(b.long() - 127).unsqueeze(-1) for s, b in (P.quantised(k), P.quantised(v)))
        if cache_of is not None:
            k, v = kept[cache_of]
        kept.append((k, v))
        kh, vh = (y.repeat_interleave(hq // hkv, dim=1) for y in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, kh) * hd ** -0.5
        s = s.masked_fill((j > i) | ((j <= i - window) if window else torch.zeros_like(j > i)), float("-inf"))
        a = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), vh).reshape(n, -1)
        x = x + a @ w[p + "self_attn.o_proj.weight"].T
        h = norm(x, w[p + "post_attention_layernorm.weight"])
        g = h @ w[p + "mlp.gate_proj.weight"].T
        x = x + (g * torch.sigmoid(g) * (h @ w[p + "mlp.up_proj.weight"].T)) @ w[p + "mlp.down_proj.weight"].T
    return norm(x, w["model.norm.weight"]) @ w["lm_head.weight"].T


def requests(name):
    return {f"r{i}": random_tokens(n, SIZES[name][6], 40 + i) for i, n in enumerate(LENGTHS)}


_engines = {}


def engine(name, graphs=True, mixed=False, e4m3=True):
    from dlgo_b200.engine.engine import Engine
    key = (name, graphs, mixed, e4m3)
    if key not in _engines:
        spec = mixed_spec(name) if mixed else config(name).architecture_spec()
        eng = Engine(spec=spec, tensors=dict(tensors(name)), max_tokens=1536, cuda_graphs=graphs, cache_dtype="e4m3" if e4m3 else None)
        eng.cache.poison()              # whatever was never written, or was given back, reads as NaN
        _engines[key] = eng
    return _engines[key]


def check(name, steps, outs, reqs, mixed=False):
    """A bfloat16 run's keys and values are off by up to half a step of 2^-8, so where the plain ones lie near a border between
    two e4m3 numbers (2^-4 apart at least) they fall on its other side: one in sixteen at most, each off by a whole step
    instead of the half step at most that the rounding itself moves it.  Errors that fall independently add up by their squares:
    (1/16) step^2 against the rounding's step^2 / 12, no more than the rounding's own effect, which is what the plain run
    with and without it differs by.  Beside it the 3e-2 of the logits' size that bfloat16 runs are held to throughout."""
    got = T.collect(steps, outs, reqs)
    for rid, toks in reqs.items():
        ref = plain(name, tuple(toks), mixed)
        effect = float((ref - plain(name, tuple(toks), mixed, False)).abs().max())
        off = float((got[rid].double() - ref).abs().max())
        assert torch.isfinite(got[rid]).all(), rid
        assert off <= 3e-2 * float(ref.abs().max()) + effect, (rid, len(toks), off, effect, float(ref.abs().max()))


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(SIZES))
def test_whole_requests(name, mixed):
    reqs = requests(name)
    steps = T.whole(reqs)
    eng = engine(name, mixed=mixed)
    check(name, steps, T.run_in_process(eng, steps), reqs, mixed)
    eng.cache.book.check()
    assert eng.cache.book.live_slots() == []


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(SIZES))
def test_last_tokens_one_by_one(name, mixed, graphs):
    reqs = requests(name)
    steps = T.tail_one_by_one(reqs, 20)
    check(name, steps, T.run_in_process(engine(name, graphs, mixed), steps), reqs, mixed)


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(SIZES))
def test_unequal_batches_with_slots_used_again(name, mixed):
    reqs = requests(name)
    steps = T.batched(reqs, 3, [5, 17, 1, 30])
    check(name, steps, T.run_in_process(engine(name, True, mixed), steps), reqs, mixed)


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(SIZES))
def test_requests_in_pieces_and_single_tokens_among_prompts(name, mixed):
    reqs = requests(name)
    steps = T.chunked(reqs, [1, 40, 7, 64, 100])
    check(name, steps, T.run_in_process(engine(name, True, mixed), steps), reqs, mixed)


@pytest.mark.parametrize("name", list(SIZES))
def test_prompts_part_by_part(name, monkeypatch):
    """The other tests' prompts go through the native loop over the layers; here every part runs by itself.  (Two runs of either
    kind may differ by twice what each is off: their few-token products add their slices in any order, and a key that lies near a
    border between two e4m3 numbers then falls on its other side.)"""
    eng = engine(name)
    assert eng.model.prompt_runs
    reqs = requests(name)
    monkeypatch.setattr(eng.model, "prompt_runs", {})
    for steps in (T.whole(reqs), T.chunked(reqs, [30, 70, 200])):
        check(name, steps, T.run_in_process(eng, steps), reqs)


def test_ordered_sums_run_too(tmp_path):
    """K-slices kept apart (a setting of the process): the projection then comes finished, not as a sum to be cleared."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", os.path.join(root, "tests", "test_cache_e4m3_engine_gpu.py"), "-m", "gpu",
                        "-k", "one_by_one and H64 and True"], cwd=root, env={**os.environ, "DLGO_ORDERED_SUMS": "1"}, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-3000:]


def test_greedy_runs_give_the_same_tokens_as_single_steps_and_repeat():
    from dlgo_b200.api import LLM
    prompts = [random_tokens(n, 512, n) for n in (3, 70, 200)]
    outs = [LLM(engine("H64", graphs)).generate(prompts, max_tokens=24, greedy=True, ignore_eos=True) for graphs in (True, True, False)]
    # (graphs and single launches cut the few-token products alike; both add their K-slices in any order, so a token that was
    # nearly tied may differ: the first ones agree)
    assert outs[0] == outs[1] or [o[:1] for o in outs[0]] == [o[:1] for o in outs[1]]
    assert [o[:1] for o in outs[0]] == [o[:1] for o in outs[2]]
    assert all(len(o) == 24 for o in outs[0])
    sampled = LLM(engine("H64")).generate(prompts, max_tokens=8, temperature=0.8, seed=3, ignore_eos=True)
    assert all(len(o) == 8 for o in sampled)


def test_the_cache_takes_half_the_bytes():
    for name in SIZES:
        hd = SIZES[name][5]
        assert engine(name).cache.bytes() * 2 * hd == engine(name, e4m3=False).cache.bytes() * (hd + 1)


def test_what_cannot_keep_8_bits_is_refused(tmp_path, model_dirs):
    from dlgo_b200.api import load_llm
    from dlgo_b200.engine.engine import Engine
    with pytest.raises(ValueError, match="bfloat16 runs"):
        Engine(model_dirs["A"], dtype="float32", cache_dtype="e4m3")
    with pytest.raises(ValueError, match="heads of 16"):
        load_llm(model_dirs["A"], cache_dtype="e4m3")
    for bad in ("int8", "float32", 5):
        with pytest.raises(ValueError, match="cache_dtype"):
            Engine(model_dirs["A"], cache_dtype=bad)
    assert Engine(model_dirs["A"], max_tokens=64, cache_dtype="bfloat16").cache.e4m3 is False
    # a mixer that appends by a kernel of its own
    from dlgo_b200.config.spec import PartSpec
    spec = config("H64").architecture_spec()
    l0, l1 = spec.layers
    keys = {k: v for k, v in l0.mixer.params.items() if k not in ("position_encoding",)}
    other = dataclasses.replace(l0, mixer=PartSpec("keys_as_values_attention", keys))
    with pytest.raises(ValueError, match="KeysAsValuesAttention"):
        Engine(spec=dataclasses.replace(spec, layers=[other, l1]), tensors=dict(tensors("H64")), max_tokens=64, cache_dtype="e4m3")


def test_command_line_and_trace_program_take_the_option(tmp_path):
    import json
    import os
    import subprocess
    import sys
    from dlgo_b200.weights import write_random_model
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    write_random_model(config("H64"), 5, str(tmp_path / "m"))
    run = subprocess.run([sys.executable, "-m", "dlgo_b200", "generate", str(tmp_path / "m"), "--prompt-ids", "1,2,3", "--max-tokens", "5",
                          "--greedy", "--ignore-eos", "--cache-dtype", "e4m3"], cwd=root, capture_output=True, text=True)
    assert run.returncode == 0 and len(run.stdout.split()) == 5, run.stderr[-2000:]
    line = json.dumps({"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3], "want": [0, 2]}], "end": ["a"]}) + "\n"
    run = subprocess.run([sys.executable, os.path.join(root, "bin", "trace_run"), "--model", str(tmp_path / "m"), "--dtype", "bfloat16", "--out",
                          str(tmp_path / "o"), "--max-tokens", "64", "--cache-dtype", "e4m3"], input=line, capture_output=True, text=True)
    assert run.returncode == 0 and "done 0" in run.stdout, run.stderr[-2000:]
    assert os.path.getsize(tmp_path / "o" / "0.f32") == 2 * 512 * 4
