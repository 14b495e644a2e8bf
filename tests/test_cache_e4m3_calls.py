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
