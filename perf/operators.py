"""What the 8-bit cache's operators are measured on.

The cache keeps a key's or a value's row of one head as e4m3 numbers (``torch.float8_e4m3fn``) with one power of two per
row, in pages of 64 positions that a table finds:

    e = the smallest whole number with max |x| <= 448 * 2^e, kept within [-119, 119];  byte = e + 127
    stored = x / 2^e, clamped to +-448, to the nearest e4m3 number (ties to even);  value = stored * 2^e

A value needs no more than 4 bits of mantissa, so bfloat16 holds it exactly.  Three operators:

* ``write``   queries and keys of a step's tokens rotated at their positions, keys and values into the cache; what the
              touched pages then hold is read back as bfloat16 (rows that no token has reached read as zeros).
* ``read``    whole sequences' pages back as bfloat16 pages, for the attention of a prompt's next part.
* ``decode``  attention of one new token per sequence over what the cache holds, its own key and value included.
"""
import math
import random

import torch

own = False

PAGE = 64
NAN_BYTE, DEAD_SCALE = 0x7F, 255          # what lies in rows that no token has reached

# query heads, key heads, head size: Llama 3.2 1B and 3B, 3.1 8B; then groups of 1, 5 and 16 heads
HEADS = {"1b": (32, 8, 64), "3b": (24, 8, 128), "8b": (32, 8, 128), "one": (6, 6, 64), "five": (20, 4, 128), "sixteen": (32, 2, 128)}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a small batch's generation step: one token each behind about a thousand
        dict(name="write-8x1-1b", op="write", heads="1b", batch=8, new=1, low=300, high=1700, f32=True, spread=False),
        # a full batch's generation step
        dict(name="write-64x1-3b", op="write", heads="3b", batch=64, new=1, low=64, high=4000, f32=True, spread=False),
        # a few short prompts of unequal length at once, behind what earlier turns left
        dict(name="write-3x700-1b", op="write", heads="1b", batch=3, new=700, low=0, high=500, f32=False, spread=True),
        # long prompts, four at a time
        dict(name="write-4x4096-8b", op="write", heads="8b", batch=4, new=4096, low=0, high=1000, f32=False, spread=False),
        # the second part of a short prompt reads the first
        dict(name="read-1x300-1b", op="read", heads="1b", batch=1, low=300, high=300),
        # long prompts that go on in parts
        dict(name="read-8x16k-8b", op="read", heads="8b", batch=8, low=2000, high=16384),
        # one request, just begun
        dict(name="decode-1x57-1b", op="decode", heads="1b", batch=1, low=57, high=57, window=0, sink=False),
        # a small batch of chats
        dict(name="decode-8x1k-1b", op="decode", heads="1b", batch=8, low=300, high=1700, window=0, sink=False),
        # a full batch of unequal lengths
        dict(name="decode-64x4k-1b", op="decode", heads="1b", batch=64, low=128, high=4096, window=0, sink=False),
        dict(name="decode-32x4k-8b", op="decode", heads="8b", batch=32, low=256, high=4096, window=0, sink=False),
        # one long document
        dict(name="decode-1x128k-8b", op="decode", heads="8b", batch=1, low=131072, high=131072, window=0, sink=False),
        # a layer with a window and sinks, five heads to a key head
        dict(name="decode-16x8k-five", op="decode", heads="five", batch=16, low=64, high=8192, window=1024, sink=True),
    ]


def _between(rng, low, high):
    """A whole number, its logarithm spread evenly."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode"])
    heads = rng.choice(sorted(HEADS))
    if op == "write":
        if rng.random() < 0.5:
            batch, new = _between(rng, 1, 200), 1
        else:
            new = _between(rng, 2, 4096)
            batch = _between(rng, 1, min(32, max(1, 16384 // new)))
        low = _between(rng, 1, 2000) - 1
        return dict(op=op, heads=heads, batch=batch, new=new, low=low, high=low + _between(rng, 1, 2000), f32=rng.random() < 0.5,
                    spread=rng.random() < 0.5)
    if op == "read":
        batch = _between(rng, 1, 16)
        high = _between(rng, 1, 131072 // batch)
        return dict(op=op, heads=heads, batch=batch, low=_between(rng, 1, high), high=high)
    batch = _between(rng, 1, 200)
    high = _between(rng, 1, 131072 // batch)
    return dict(op=op, heads=heads, batch=batch, low=_between(rng, 1, high), high=high,
                window=rng.choice([0, 0, 0, _between(rng, 1, 4096)]), sink=rng.random() < 0.3)


def _lengths(case):
    """(positions that lie in the cache before the step, new tokens) of every sequence."""
    rng = random.Random(f"{case['op']} {case['batch']} {case['low']} {case['high']}")
    n = case["batch"]
    before = [rng.randint(case["low"], case["high"]) for _ in range(n)]
    if n > 1:
        before[rng.randrange(n)] = case["high"]
    if case["op"] != "write":
        return before, [0] * n
    new = [max(1, rng.randint(case["new"] // 2, case["new"])) if case["spread"] else case["new"] for _ in range(n)]
    return before, new


# ------------------------------------------------------------------ inputs
def _power(scales):
    """2^(byte - 127) in 32 bits (bytes of rows that no token has reached: anything)."""
    return (scales.to(torch.int32) << 23).view(torch.float32)


def _quantised(x):
    """e4m3 numbers and scale bytes of rows ``x`` [..., head size] in 32 bits."""
    most = x.abs().amax(dim=-1)
    half, power = torch.frexp(most)               # most = half * 2^power, 0.5 <= half < 1; 448 = 0.875 * 2^9
    e = (power - 9 + (half > 0.875).to(power.dtype)).clamp(-119, 119)
    e = torch.where(most == 0, torch.full_like(e, -119), e)
    stored = (x * _power(127 - e).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return stored, (e + 127).to(torch.uint8)


def _rows(shape, gen, device):
    """Rows as a model's projections make them: a few channels of every head are an order of magnitude larger."""
    x = torch.randn(shape, generator=gen, device=device)
    loud = torch.rand(shape[-2:], generator=gen, device=device) < 0.03
    return x * torch.where(loud, 8.0, 1.0)


def _cache(case, lengths, room, gen, device):
    """Pages with ``lengths`` positions of every sequence written and room for ``room``, the rest NaN."""
    _, hkv, hd = HEADS[case["heads"]]
    need = [-(-r // PAGE) for r in room]
    order = list(range(sum(need) + 3))
    rng = random.Random(sum(need))
    rng.shuffle(order)
    slots = list(range(len(need) + 2))
    rng.shuffle(slots)
    table = torch.full((len(slots), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[slots[i], :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    state = dict(table=table.to(device), slots=torch.tensor(slots[:len(need)], dtype=torch.int32, device=device))
    where = torch.tensor([order[j] for j in range(at)], dtype=torch.int64, device=device)
    left = torch.tensor([min(PAGE, max(0, lengths[i] - PAGE * p)) for i, n in enumerate(need) for p in range(n)], device=device)
    live = torch.arange(PAGE, device=device).view(1, 1, PAGE) < left.view(-1, 1, 1)
    live = live.expand(-1, hkv, -1)
    for name in ("keys", "values"):
        pages = torch.full((len(order), hkv, PAGE, hd), NAN_BYTE, dtype=torch.uint8, device=device)
        scales = torch.full((len(order), hkv, PAGE), DEAD_SCALE, dtype=torch.uint8, device=device)
        for lo in range(0, at, 512):              # (as bfloat16 rows would have been written, 32,768 positions at a time)
            w, ok = where[lo:lo + 512], live[lo:lo + 512]
            rows = _rows((w.numel(), PAGE, hkv, hd), gen, device).transpose(1, 2)
            q, s = _quantised(rows.to(torch.bfloat16).float())
            pages[w] = torch.where(ok.unsqueeze(-1), q.view(torch.uint8), pages[w])
            scales[w] = torch.where(ok, s, scales[w])
        state[name], state[name + "_scales"] = pages.view(torch.float8_e4m3fn), scales
    return state


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    hq, hkv, hd = HEADS[case["heads"]]
    before, new = _lengths(case)
    after = [b + n for b, n in zip(before, new)]
    state = _cache(case, before, after, gen, device)
    state.update(op=case["op"], shape=(hq, hkv, hd))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    if case["op"] == "write":
        pos = [p for b, n in zip(before, new) for p in range(b, b + n)]
        seq = [i for i, n in enumerate(new) for _ in range(n)]
        state.update(token_pos=ints(pos), token_seq=ints(seq))
        x = _rows((len(pos), hq + 2 * hkv, hd), gen, device).reshape(len(pos), -1)
        state["qkv"] = x if case["f32"] else x.to(torch.bfloat16)
        freq = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=device) / hd)
        angle = torch.arange(max(after), dtype=torch.float64, device=device).unsqueeze(1) * freq
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        slots = state["slots"].tolist()
        state["pages"] = ints([[slots[i], p, min(PAGE, after[i] - PAGE * p)] for i in range(len(new))
                               for p in range(before[i] // PAGE, -(-after[i] // PAGE))])
    elif case["op"] == "read":
        slots = state["slots"].tolist()
        state["pages"] = ints([[slots[i], p, min(PAGE, n - PAGE * p)] for i, n in enumerate(before) for p in range(-(-n // PAGE))])
    else:
        state.update(token_pos=ints([n - 1 for n in before]), window=case["window"], scale=1.0 / math.sqrt(hd))
        state["q"] = _rows((len(before), hq, hd), gen, device).to(torch.bfloat16).reshape(len(before), hq * hd)
        state["sink"] = torch.randn(hq, generator=gen, device=device) if case["sink"] else None
        state["longest"] = max(before)
        state["tickets"] = torch.zeros(len(before) * hq, dtype=torch.int32, device=device)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    hq, hkv, hd = state["shape"]
    if own:
        from dlgo_b200.csrc import kernels as K
        cache = (state["keys"], state["values"], state["keys_scales"], state["values_scales"], state["table"])
        if state["op"] == "write":
            q = K.rope_append_e4m3(state["qkv"], state["cos"], state["sin"], state["token_pos"], state["token_seq"], state["slots"],
                                   *cache, hq, hkv, hd, hd)
            keys, values = K.read_pages_e4m3(*cache, state["pages"])
            return {"q": q, "keys": keys, "values": values}
        if state["op"] == "read":
            keys, values = K.read_pages_e4m3(*cache, state["pages"])
            return {"keys": keys, "values": values}
        return {"out": K.attention_decode_e4m3(state["q"], *cache, state["slots"], state["token_pos"], hq, hkv, hd, state["scale"],
                                               window=state["window"], sink=state["sink"], tickets=state["tickets"])}
    if state["op"] == "write":
        q = _plain_write(state)
        keys, values = _plain_read(state)
        return {"q": q, "keys": keys, "values": values}
    if state["op"] == "read":
        keys, values = _plain_read(state)
        return {"keys": keys, "values": values}
    return {"out": _plain_decode(state)}


def _plain_write(state):
    hq, hkv, hd = state["shape"]
    T = state["qkv"].shape[0]
    x = state["qkv"].float().view(T, hq + 2 * hkv, hd)
    pos = state["token_pos"].long()
    c, s = state["cos"][pos].unsqueeze(1), state["sin"][pos].unsqueeze(1)
    a, b = x[:, :hq + hkv, :hd // 2], x[:, :hq + hkv, hd // 2:]
    turned = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    page = state["table"][state["slots"][state["token_seq"].long()].long(), pos // PAGE].long()
    for name, rows in (("keys", turned[:, hq:]), ("values", x[:, hq + hkv:])):
        stored, scale = _quantised(rows)
        state[name].view(torch.uint8)[page, :, pos % PAGE] = stored.view(torch.uint8)
        state[name + "_scales"][page, :, pos % PAGE] = scale
    return turned[:, :hq].reshape(T, hq * hd).to(torch.bfloat16)


def _plain_read(state):
    slot, index, live = state["pages"].long().unbind(1)
    page = state["table"][slot, index].long()
    dead = torch.arange(PAGE, device=page.device).view(1, 1, PAGE, 1) >= live.view(-1, 1, 1, 1)
    out = []
    for name in ("keys", "values"):
        rows = state[name].view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * _power(state[name + "_scales"][page]).unsqueeze(-1)
        out.append(rows.masked_fill(dead, 0.0).to(torch.bfloat16))
    return out


def _plain_decode(state):
    hq, hkv, hd = state["shape"]
    pos, window = state["token_pos"].long(), state["window"]
    B, pages = pos.numel(), -(-state["longest"] // PAGE)
    page = state["table"][state["slots"].long(), :pages].long().clamp_min(0)
    t = torch.arange(pages * PAGE, device=page.device).view(1, 1, 1, -1)
    p = pos.view(B, 1, 1, 1)
    seen = (t <= p) & (t > p - window) if window else t <= p

    def rows(name):                                # [sequences, key heads, positions, head size], unreached rows zero
        x = state[name].view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * _power(state[name + "_scales"][page]).unsqueeze(-1)
        x = x.transpose(1, 2).reshape(B, hkv, pages * PAGE, hd)
        return x.masked_fill_(~seen.transpose(2, 3), 0.0)

    q = state["q"].float().view(B, hkv, hq // hkv, hd)
    s = ((q @ rows("keys").transpose(2, 3)) * state["scale"]).masked_fill(~seen, float("-inf"))
    most = s.amax(dim=-1, keepdim=True)
    if state["sink"] is not None:
        sink = state["sink"].view(1, hkv, hq // hkv, 1)
        most = torch.maximum(most, sink)
    w = (s - most).exp()
    total = w.sum(dim=-1, keepdim=True)
    if state["sink"] is not None:
        total = total + (sink - most).exp()
    return ((w @ rows("values")) / total).reshape(B, hq * hd).to(torch.bfloat16)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    hq, hkv, hd = HEADS[case["heads"]]
    before, new = _lengths(case)
    row = 2 * hkv * (hd + 1)                      # a position's key and value with their scales
    if case["op"] == "write":
        T = sum(new)
        touched = sum(-(-(b + n) // PAGE) - b // PAGE for b, n in zip(before, new))
        old = sum(b % PAGE for b in before)       # rows of the touched pages that were there
        size = 4 if case["f32"] else 2
        moved = T * ((hq + 2 * hkv) * hd * size + hd * 4 + hq * hd * 2 + row) + old * row + touched * PAGE * 2 * hkv * hd * 2
        return {"bytes": moved, "flops": T * (hq + hkv) * hd * 3}
    if case["op"] == "read":
        pages = sum(-(-n // PAGE) for n in before)
        return {"bytes": sum(before) * row + pages * PAGE * 2 * hkv * hd * 2, "flops": 0}
    seen = sum(min(n, case["window"]) if case["window"] else n for n in before)
    return {"bytes": seen * row + len(before) * hq * hd * 4, "flops": seen * hq * hd * 4}


# ------------------------------------------------------------------ the definition in 64 bits
def _two_to(k):
    """2^k in 64 bits, without a rounding (the GPU's pow has one)."""
    return (k.to(torch.int64) + 1023 << 52).view(torch.float64)


def _e4m3_nearest(x):
    """The e4m3 number nearest to each |x| <= 448 (64 bits): steps of 2^(k - 3) from 2^k on, of 2^-9 below 2^-6."""
    _, k = torch.frexp(x)
    step = _two_to((k - 1).clamp_min(-6) - 3)
    return torch.round(x / step) * step           # (torch.round takes halves to even)


def _e4m3_value(bits):
    bits = bits.to(torch.int64)
    sign, k, m = 1 - 2 * (bits >> 7), (bits >> 3) & 15, (bits & 7).double()
    return sign * torch.where(k > 0, (8 + m) * _two_to(k - 10), m / 512)


def exact(case, seed):
    state = prepare(case, seed)
    hq, hkv, hd = state["shape"]
    before, new = _lengths(case)
    slots = state["slots"].tolist()
    table = state["table"]

    def held(name, i, n):                         # the first n positions of sequence i: [key heads, n, head size]
        page = table[slots[i], :-(-n // PAGE)].long()
        x = _e4m3_value(state[name].view(torch.uint8)[page]) * _two_to(state[name + "_scales"][page].long() - 127).unsqueeze(-1)
        return x.transpose(0, 1).reshape(hkv, -1, hd)[:, :n]

    def pages_of(rows, first):                    # rows from a page's first position on -> zero-padded pages
        n = rows.shape[1]
        full = torch.zeros(hkv, -(-n // PAGE) * PAGE, hd, dtype=torch.float64, device=rows.device)
        full[:, :n] = rows
        return full.view(hkv, -1, PAGE, hd).transpose(0, 1)[first:]

    if case["op"] == "read":
        return {name: torch.cat([pages_of(held(name, i, n), 0) for i, n in enumerate(before)]) for name in ("keys", "values")}
    if case["op"] == "decode":
        out = []
        for i, n in enumerate(before):
            lo = max(0, n - case["window"]) if case["window"] else 0
            k, v = held("keys", i, n)[:, lo:], held("values", i, n)[:, lo:]
            s = state["q"][i].double().view(hkv, -1, hd) @ k.transpose(1, 2) * state["scale"]
            if state["sink"] is not None:
                s = torch.cat([s, state["sink"].double().view(hkv, -1, 1)], dim=-1)
            w = torch.softmax(s, dim=-1)[:, :, :n - lo]
            out.append((w @ v).reshape(-1))
        return {"out": torch.stack(out)}
    x = state["qkv"].double().view(-1, hq + 2 * hkv, hd)
    at = torch.complex(state["cos"].double(), state["sin"].double())[state["token_pos"].long()].unsqueeze(1)
    z = torch.complex(x[:, :hq + hkv, :hd // 2], x[:, :hq + hkv, hd // 2:]) * at
    turned = torch.cat([z.real, z.imag], dim=-1)
    out = {"q": turned[:, :hq].reshape(-1, hq * hd)}
    for name, rows in (("keys", turned[:, hq:]), ("values", x[:, hq + hkv:])):
        most = rows.abs().amax(dim=-1, keepdim=True)
        half, k = torch.frexp(most / 448)         # in (2^(k - 1), 2^k), or 2^(k - 1) itself
        unit = _two_to((k - (half == 0.5).to(k.dtype)).clamp(-119, 119))
        rows = (_e4m3_nearest((rows / unit).clamp(-448, 448)) * unit).transpose(0, 1)
        got, lo = [], 0
        for i, n in enumerate(new):
            whole = torch.cat([held(name, i, before[i]), rows[:, lo:lo + n]], dim=1) if before[i] else rows[:, lo:lo + n]
            got.append(pages_of(whole, before[i] // PAGE))
            lo += n
        out[name] = torch.cat(got)
    return out
