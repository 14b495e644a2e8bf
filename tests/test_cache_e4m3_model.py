"""What the whole-model tests over the 8-bit cache would notice: mistakes planted in the plain implementation (no GPU)."""
import pytest
import torch

import plain_e4m3_model as M
import test_cache_e4m3_engine_gpu as E


def _softmax(s, v, factor=1.0):
    return torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v) * factor


def _without(back):
    """The key ``back`` positions before a query is not seen (by queries that have one)."""
    def attend(s, v):
        s, i = s.clone(), torch.arange(s.shape[1])
        s[:, i[max(back, 1):], i[max(back, 1) - back:len(i) - back]] = float("-inf")
        return _softmax(s, v)
    return attend


def _run(name, tokens, mixed, **spoiled):
    """A bfloat16 run, spoiled: (its logits, the rows that its cache would hold)."""
    logits, made, read = M.run(name, tokens, mixed, rounded="token", **spoiled)
    return logits, [None if m is None else r for m, r in zip(made, read)]


@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("name", list(E.SIZES))
@pytest.mark.parametrize("n", [9, 64, 130])
def test_a_right_run_passes_and_spoiled_ones_do_not(name, mixed, n):
    tokens = E.random_tokens(n, E.SIZES[name][6], 7 * n)
    logits, rows = _run(name, tokens, mixed)
    assert M.faults(name, tokens, rows, logits, mixed) == []
    for spoil in (lambda s, v: _softmax(s, v, 1.125), lambda s, v: _softmax(s * 1.25, v), _without(0), _without(1)):
        logits, rows = _run(name, tokens, mixed, attend=spoil)
        assert M.faults(name, tokens, rows, logits, mixed), spoil
    # rows in 8 bits, attention over unrounded ones; rows of a position too far; another token fed back
    logits, rows = _run(name, tokens, mixed)
    assert M.faults(name, tokens, rows, M.run(name, tokens, mixed, quantised=False, rounded="token")[0], mixed)
    shifted = [None if r is None else tuple(x.roll(1, 0) for x in r) for r in rows]
    assert M.faults(name, tokens, shifted, None, mixed)
    other = list(tokens)
    other[n // 2] = (other[n // 2] + 1) % E.SIZES[name][6]
    assert M.faults(name, other, rows, None, mixed)
