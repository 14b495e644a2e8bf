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
