"""The 8-bit cache's functions without a GPU: what their sources have to say, and calls that the other files leave out."""
import os
import re

import pytest
import torch

import dlgo_b200.csrc

CSRC = os.path.dirname(os.path.abspath(dlgo_b200.csrc.__file__))


@pytest.mark.parametrize("name", ["attention_decode_e4m3.cu", "cache_e4m3.cu", "e4m3.cuh", "tcgen05.cuh"])
def test_what_a_whole_warp_executes_stays_where_it_stands(name):
    """An ``asm`` that is not volatile may be moved into a branch that only some lanes take, or left out: that is not for
    instructions that name the lanes which execute them, nor for those that reach memory or a barrier."""
    text = open(os.path.join(CSRC, name)).read()
    found = re.findall(r'\basm\s*\(((?:[^;"]|"[^"]*")*);', text)
    assert name == "tcgen05.cuh" or name == "cache_e4m3.cu" or found
    for body in found:
        code = " ".join(re.findall(r'"([^"]*)"', body))
        assert not re.search(r"\.sync\b|\.aligned\b|\bbar\.|mbarrier|tcgen05|fence|\b(ld|st|atom|red|cp)\.", code), code


@pytest.mark.parametrize("kinds", [(False, True, False), (True, False, True)])
def test_a_model_with_caches_of_both_kinds_hands_the_native_loop_what_each_needs(kinds, monkeypatch):
    """Entry points belong to a cache's kind, not to whichever cache the model's run of layers saw first."""
    from types import SimpleNamespace as NS

    from dlgo_b200.csrc import kernels as K
    from dlgo_b200.engine import prompt_run
    from dlgo_b200.parts import tensor_core
    d, hq, hkv, hd, f, tokens = 256, 4, 2, 64, 1024, 200
    monkeypatch.setattr(tensor_core, "sm_count", lambda device=None: 148)
    monkeypatch.setattr(K, "prompt_entry_points", lambda e4m3=False: f"entry points {e4m3}")
    seen = []
    monkeypatch.setattr(K, "prompt_layers", lambda entry, shape, layers, step: seen.append((entry, bool(step.n_seen))))
    shapes = dict(wqkv=((hq + 2 * hkv) * hd, d), wo=(d, hq * hd), w_gate_up=(2 * f, d), w_down=(d, f))
    linear = {n: NS(_tc=tensor_core.TensorCorePlan(torch.empty(s, dtype=torch.bfloat16), swiglu=n == "w_gate_up")) for n, s in shapes.items()}
    mixer = NS(wqkv=linear["wqkv"], wo=linear["wo"], fuses_prompt_rope=lambda *a: False)
    model = NS(blocks={0: NS(mixer=mixer, ffn=NS(w_gate_up=linear["w_gate_up"], w_down=linear["w_down"]))}, order=[NS(layer=0)],
               positions={"rope": NS(cos=torch.empty(1, hd // 2), sin=torch.empty(1, hd // 2))})
    run = prompt_run.PromptRun(0, 1, (d, hq, hkv, hd, f, 1.0, 0, "rope", hd, False, "full"))
    run._descriptors = lambda *a: (None, None)
    some = torch.ones(1, 3, dtype=torch.int32)
    ctx = NS(decode=False, n_tokens=tokens, tiles=lambda *a, **k: (some, 1, 1), token_pos=some, token_seq=some, seq_slot=some,
             scratch=lambda name, n, dt: torch.empty(n, dtype=dt), zeros=lambda name, n, dt: torch.zeros(n, dtype=dt),
             pages_in_sight=lambda span, page: (some, some, some))
    for e4m3 in kinds:
        view = NS(page_table=torch.empty(1, 4, dtype=torch.int32), page_size=64, keys=torch.empty(1, dtype=torch.bfloat16),
                  key_scales=torch.empty(1, dtype=torch.uint8) if e4m3 else None)
        run.run(model, torch.empty(tokens, d), ctx, NS(view=lambda i: view))
    assert seen == [(f"entry points {e}", e) for e in kinds]


def _cache(hkv=2, hd=64, pages=3):
    kp = torch.zeros(pages, hkv, 64, hd, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = torch.zeros(pages, hkv, 64, dtype=torch.uint8)
    return [kp, kp.clone(), sc, sc.clone(), torch.zeros(2, 4, dtype=torch.int32)]


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_decode_refuses_an_output_that_meets_the_queries_or_itself():
    from dlgo_b200.csrc import kernels as K
    cols = 256
    buf = torch.zeros(4 * 3 * cols + 64, dtype=torch.bfloat16)

    def rows(first, stride, n=3):
        return buf.as_strided((n, cols), (stride, 1), first)

    def decode(q, out):
        return K.attention_decode_e4m3(q, *_cache(), _ints(*range(q.shape[0])), _ints(*[0] * q.shape[0]), 4, 2, 64, 1.0, out=out)

    for q, out in ((rows(0, cols), rows(0, cols)), (rows(0, cols), rows(8, cols)), (rows(8, cols), rows(0, cols)),
                   (rows(0, cols), rows(2 * cols, cols)), (rows(0, 2 * cols), rows(cols - 4, 2 * cols)),
                   (rows(0, 2 * cols), rows(cols + 4, 2 * cols)), (rows(cols, 2 * cols), rows(0, cols)),
                   (rows(0, cols, 1), rows(cols - 4, cols, 1)), (rows(0, 0), rows(0, cols))):
        with pytest.raises(K.KernelError, match="another tensor"):
            decode(q, out)
    other = torch.zeros(3 * cols, dtype=torch.bfloat16)
    for stride in (0, 4, cols - 4):
        with pytest.raises(K.KernelError, match="overlap one another"):
            decode(rows(0, cols), other.as_strided((3, cols), (stride, 1)))
    # columns of one buffer, rows behind one another, more rows than sequences, one row: as before
    for q, out in ((rows(0, 2 * cols), rows(cols, 2 * cols)), (rows(cols, 2 * cols), rows(0, 2 * cols)), (rows(0, cols), rows(3 * cols, cols)),
                   (rows(3 * cols, cols, 2), rows(cols, cols, 4)[:3]), (rows(0, cols, 1), rows(cols, 0, 1)), (rows(0, 0), rows(cols, cols))):
        with pytest.raises(K.KernelError, match="GPU"):
            decode(q, out)


def test_the_c_entry_refuses_rows_that_meet():
    import struct

    from dlgo_b200.csrc import kernels as K
    fn = K._lib("attention_decode_e4m3").dlgo_attention_decode_e4m3_record

    def call(B, ldq, ldo):        # (pointers are looked at for their alignment alone before the sizes are; B = 0 launches nothing)
        p = 4096
        return fn(struct.pack("=19qd4q", p, B, ldq, p, p, p, p, 3, p, 2, 4, p, p, p, ldo, 4, 2, 64, 0, 1.0, 0, p, p, 0))

    assert K._STATUS[call(2, 256, 252)] == K._STATUS[call(2, 256, 0)] == K._STATUS[call(2, -256, 256)] == K._STATUS[call(2, 256, -256)]
    assert "size" in K._STATUS[call(2, 256, 252)] and call(0, 256, 0) == 0


def test_reading_into_one_buffer_and_writing_into_shared_pages_are_refused():
    from dlgo_b200.csrc import kernels as K
    cache = _cache()
    buf = torch.zeros(2 * 2 * 64 * 64 + 8, dtype=torch.bfloat16)
    one = lambda at: buf[at:at + 2 * 64 * 64].view(1, 2, 64, 64)  # noqa: E731
    pages = torch.zeros(1, 3, dtype=torch.int32)
    for a, b in ((0, 0), (0, 8), (8, 0), (0, 2 * 64 * 64 - 8)):
        with pytest.raises(K.KernelError, match="in common"):
            K.read_pages_e4m3(*cache, pages, one(a), one(b))
    with pytest.raises(K.KernelError, match="GPU"):
        K.read_pages_e4m3(*cache, pages, one(0), one(2 * 64 * 64))

    def write(cache, **more):
        cos = torch.zeros(10, 32)
        return K.rope_append_e4m3(torch.zeros(1, 8 * 64), cos, cos, _ints(0), _ints(0), _ints(0), *cache, 4, 2, 64, 64, **more)

    for i in (1, 3):
        shared = list(cache)
        shared[i] = shared[i - 1]
        with pytest.raises(K.KernelError, match="in common"):
            write(shared)
        with pytest.raises(K.KernelError, match="GPU"):
            write(shared, write_cache=False)
    with pytest.raises(K.KernelError, match="GPU"):
        write(cache)


def test_a_mixer_that_keeps_16_bits_of_its_weights_keeps_its_cache_too():
    from dlgo_b200.parts.attention import GQAAttention
    for heads in (4, 16):
        mixer = GQAAttention(256, heads, 2, 64, 0.125)
        assert mixer.takes_e4m3_cache()
        mixer.split_weights = True
        assert not mixer.takes_e4m3_cache()
    assert not GQAAttention(256, 4, 2, 96, 0.125).takes_e4m3_cache()


def test_without_a_rotation_the_tables_are_not_looked_at():
    from dlgo_b200.csrc import kernels as K

    def write(cos, sin, rot):
        return K.rope_append_e4m3(torch.zeros(1, 8 * 64), cos, sin, _ints(0), _ints(0), _ints(0), *_cache(), 4, 2, 64, rot)

    for cos in (None, torch.zeros(0), torch.zeros(3, dtype=torch.float64)):
        with pytest.raises(K.KernelError, match="GPU"):
            write(cos, cos, 0)
    for cos, sin in ((None, None), (torch.zeros(10, 32), None), (None, torch.zeros(10, 32)), (torch.zeros(32), torch.zeros(32))):
        with pytest.raises(K.KernelError, match="cos and sin"):
            write(cos, sin, 64)


def test_overlap_of_rows_agrees_with_a_count_of_their_numbers():
    import random

    from dlgo_b200.csrc import kernels as K
    rng = random.Random(0)
    buf = torch.zeros(400, dtype=torch.bfloat16)
    seen = [0, 0]
    for _ in range(4000):
        rows, cols = rng.randint(1, 5), rng.randint(1, 12)
        a, b = (dict(first=rng.randint(0, 90), stride=rng.choice([0, cols, rng.randint(0, 60), 24])) for _ in range(2))
        if rng.random() < 0.5:
            b["stride"] = a["stride"]
        numbers = [{t["first"] + r * t["stride"] + c for r in range(rows) for c in range(cols)} for t in (a, b)]
        want = bool(numbers[0] & numbers[1])
        x, y = (buf.as_strided((rows, cols), (t["stride"], 1), t["first"]) for t in (a, b))
        assert K._rows_overlap(x, y, rows, cols) == K._rows_overlap(y, x, rows, cols) == want, (rows, cols, a, b)
        seen[want] += 1
    assert min(seen) > 500
