"""A whole model in 64 bits that attends over given keys and values: those that an engine's 8-bit cache holds.

With the engine's own rows a key near a border between two e4m3 numbers lies on the same side in both, so what is left between
the two runs is the bfloat16 run's rounding alone."""
import torch

import plain_e4m3 as P
import test_cache_e4m3_engine_gpu as E

# (layer, window, rotated numbers of a head of hd, neighbouring pairs, the run entry whose cache it reads) of each run entry
ORDERS = {False: [(0, None, 1, False, None), (1, None, 1, False, None)],
          True: [(0, 70, 1, False, None), (1, None, 2, True, None), (0, 70, 1, False, None), (1, None, 2, True, 1)]}


def _bf16(x):
    return x.to(torch.bfloat16).double()


def run(name, tokens, mixed=False, rows=None, quantised=True, rounded=None, attend=None):
    """(logits [n, vocab], [(keys, values) [n, kv heads, hd] as the projections make them, None where another entry's are read],
    [the keys and values that attention read]).

    ``rows[i]``: the keys and values that run entry i's attention reads; without them the entry's own, as the 8-bit cache would hold
    them (``quantised``) or as they are.  ``rounded``: to bfloat16 wherever a bfloat16 run rounds, 64 bits between: normed rows,
    queries, the softmax's weights, attention's result, the feed-forward's inner numbers, and ("prompt", not "token") the projection
    itself.  ``attend(scores [heads, n, n], values)`` stands in for the softmax and the sum, for tests of the tests."""
    d, _, _, hq, hkv, hd, _ = E.SIZES[name]
    w = {k: v.double() for k, v in E.tensors(name).items()}
    r = _bf16 if rounded else lambda x: x
    norm = lambda x, g: r(x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * g)  # noqa: E731
    n = len(tokens)
    x = w["model.embed_tokens.weight"][list(tokens)]
    made, read = [], []
    i, j = torch.arange(n).view(-1, 1), torch.arange(n).view(1, -1)
    for entry, (layer, window, part, inter, cache_of) in enumerate(ORDERS[mixed]):
        p = f"model.layers.{layer}."
        h = norm(x, w[p + "input_layernorm.weight"])
        q, k, v = ((h @ w[p + f"self_attn.{c}_proj.weight"].T).view(n, -1, hd) for c in "qkv")
        if rounded == "prompt":
            q, k, v = r(q), r(k), r(v)
        q, k = r(E.rotate(q, hd // part, inter)), E.rotate(k, hd // part, inter)
        made.append((k, v) if cache_of is None else None)
        if cache_of is not None:
            k, v = read[cache_of]
        elif rows is not None:
            k, v = rows[entry]
        elif quantised:
            k, v = (s * P.two_to(b.long() - 127).unsqueeze(-1) for s, b in (P.quantised(k), P.quantised(v)))
        read.append((k, v))
        kh, vh = (y.repeat_interleave(hq // hkv, dim=1) for y in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, kh) * hd ** -0.5
        s = s.masked_fill((j > i) | ((j <= i - window) if window else torch.zeros_like(j > i)), float("-inf"))
        if attend is None:
            e = (s - s.amax(-1, keepdim=True)).exp()
            a = torch.einsum("hij,jhd->ihd", r(e), vh) / e.sum(-1).T.unsqueeze(-1)
        else:
            a = attend(s, vh)
        x = x + r(a).reshape(n, -1) @ w[p + "self_attn.o_proj.weight"].T
        h = norm(x, w[p + "post_attention_layernorm.weight"])
        g = h @ w[p + "mlp.gate_proj.weight"].T
        x = x + r(g * torch.sigmoid(g) * (h @ w[p + "mlp.up_proj.weight"].T)) @ w[p + "mlp.down_proj.weight"].T
    return norm(x, w["model.norm.weight"]) @ w["lm_head.weight"].T, made, read


def _rms(x, dim=None):
    return x.pow(2).mean().sqrt() if dim is None else x.pow(2).mean(dim).sqrt()


def faults(name, tokens, rows, logits, mixed=False):
    """What is wrong with a bfloat16 run whose cache held ``rows`` and which gave ``logits`` [n, vocab] (None: not looked at), as a
    list of sentences.

    The tolerances are what roundings to bfloat16 at the run's own places do to the same tokens, simulated in 64 bits, in both forms
    of a step: a whole request's error is an average over many roundings, so twice the simulated one; a single position's varies more
    (two simulations of a position differ by up to 7 times, by less where the request's median is the least taken), so eight times; the
    largest error of a key or a value four times, beside the half step that its own rounding to 8 bits moves it."""
    tokens = tuple(tokens)
    ref, made, _ = run(name, tokens, mixed, rows)
    noise, off = [], [None if m is None else [0.0, 0.0] for m in made]
    for form in ("prompt", "token"):
        got, kv, read = run(name, tokens, mixed, rounded=form)
        want, kv_want, _ = run(name, tokens, mixed, [None if m is None else y for m, y in zip(kv, read)])
        noise.append(_rms(got - want, 1))
        for o, a, b in zip(off, kv, kv_want):
            for side in range(2 if o is not None else 0):
                o[side] = max(o[side], float((a[side] - b[side]).abs().max()))
    noise = torch.maximum(*noise)
    out = []
    for e, (m, stored) in enumerate(zip(made, rows)):
        for side, what in enumerate(("keys", "values") if m is not None else ()):
            x, y = m[side], stored[side]
            left = (y - x).abs() - 2.0 ** -4 * x.abs() - 4 * (1 + 2.0 ** -4) * off[e][side]
            if not (left <= 0).all():
                out.append(f"entry {e}: {what} off by {float((y - x).abs().max())}, at positions {(~(left <= 0)).flatten(1).any(1).nonzero().flatten().tolist()[:8]}")
    if logits is None:
        return out
    logits = logits.double()
    err = _rms(logits - ref, 1)
    if not _rms(err) <= 2 * _rms(noise):
        out.append(f"logits off by {float(_rms(err)):.2e}, {float(_rms(err) / _rms(noise)):.1f} times what rounding does")
    far = ~(err <= 8 * noise.clamp_min(float(noise.median())))
    if far.any():
        out.append(f"logits of positions {far.nonzero().flatten().tolist()[:8]} off by up to {float((err / noise.clamp_min(float(noise.median()))).max()):.1f} times "
                   "what rounding does")
    # (simulated: 0.03 to 0.09 of the distance to a run whose keys and values are not in 8 bits)
    plain = run(name, tokens, mixed, quantised=False)[0]
    if not _rms(logits - ref) < 0.25 * _rms(logits - plain):
        out.append("logits as near to a run without 8-bit rows")
    return out


class Recorder:
    """What an engine's 8-bit cache held: for every slot taken while it is on, in that order, [(keys, values) per run entry (None
    where another entry's are read)] in 64 bits.  Rows are read before pages are given back."""

    def __init__(self, engine):
        self.cache, self.entries = engine.cache, len(engine.model.order)
        self.taken, self.slots = [], {}

    def __enter__(self):
        c = self.cache
        self.plain = c.take_slot, c.reserve, c.free_slot
        c.take_slot, c.reserve, c.free_slot = self.take_slot, self.reserve, self.free_slot
        return self

    def __exit__(self, *exc):
        del self.cache.take_slot, self.cache.reserve, self.cache.free_slot

    def take_slot(self):
        slot = self.plain[0]()
        n = self.cache.max_seq_len
        rows = []
        for e in range(self.entries):
            view = self.cache.view(e)
            shape = (n, view.keys.shape[1], view.keys.shape[3])
            rows.append(tuple(torch.full(shape, float("nan"), dtype=torch.float64) for _ in range(2)) if view.writes else None)
        self.slots[slot] = dict(rows=rows, upto=0)
        self.taken.append(self.slots[slot])
        return slot

    def look(self, slot):
        rec, n = self.slots[slot], self.cache.length(slot)
        for e, rows in enumerate(rec["rows"]):
            if rows is None:
                continue
            view = self.cache.view(e)
            table = view.page_table[slot].tolist()
            for p in range(rec["upto"] // 64, -(-n // 64)):
                if table[p] < 0:
                    continue
                lo, hi = 64 * p, min(n, 64 * p + 64)
                for out, pages, scales in zip(rows, (view.keys, view.values), (view.key_scales, view.value_scales)):
                    out[lo:hi] = P.values(pages[table[p]], scales[table[p]]).transpose(0, 1)[:hi - lo]
        rec["upto"] = n

    def reserve(self, slots, n_new):
        for s in slots:
            self.look(s)
        return self.plain[1](slots, n_new)

    def free_slot(self, slot):
        self.look(slot)
        self.slots.pop(slot)
        return self.plain[2](slot)


def rows_of(record, n):
    """The first n positions of what a slot held."""
    assert record["upto"] == n, (record["upto"], n)
    return [None if r is None else tuple(x[:n] for x in r) for r in record["rows"]]
