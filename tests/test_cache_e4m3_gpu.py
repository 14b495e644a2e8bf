"""The 8-bit cache's kernels against their definition in 64 bits.

Tolerances are derived, not tuned.  A rounding is off by at most half a step relative to the value: bf16 2^-8, fp16 2^-11, fp32
2^-24, e4m3 2^-4 (2^-10 of the row's power among its subnormal numbers)."""
import pytest
import torch

import plain_e4m3 as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64


def K():
    from dlgo_b200.csrc import kernels
    return kernels


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Cache:
    """Pages in a scrambled order, slots in falling order, NaN wherever nothing was written."""

    def __init__(self, lens, hkv, hd, room=None, spare=3):
        room = room or lens
        need = [-(-max(r, 1) // PAGE) for r in room]
        n = sum(need) + spare
        g = torch.Generator().manual_seed(n * 7 + hd)
        order = torch.randperm(n, generator=g).tolist()
        self.keys, self.values = (torch.full((n, hkv, PAGE, hd), 0x7F, dtype=torch.uint8) for _ in range(2))
        self.kscales, self.vscales = (torch.full((n, hkv, PAGE), 255, dtype=torch.uint8) for _ in range(2))
        self.slots = [len(lens) + 1 - i for i in range(len(lens))]
        self.table = torch.full((len(lens) + 2, max(need) + 1), -1, dtype=torch.int32)
        for i, k in enumerate(need):
            for p in range(k):
                self.table[self.slots[i], p] = order.pop()

    def put(self, i, rows, values, first=0):
        """Write rows [n, hkv, hd] as positions first .. of sequence i; returns what they then stand for."""
        back = []
        t = torch.arange(first, first + rows.shape[0])
        page = self.table[self.slots[i], t // PAGE].long()
        for pages, scales, x in ((self.keys, self.kscales, rows), (self.values, self.vscales, values)):
            stored, s = P.quantised(x)
            pages[page, :, t % PAGE] = stored.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
            scales[page, :, t % PAGE] = s
            back.append(stored * P.two_to(s.long() - 127).unsqueeze(-1))
        return back

    def device(self):
        f8 = torch.float8_e4m3fn
        return (self.keys.to(DEV).view(f8), self.values.to(DEV).view(f8), self.kscales.to(DEV), self.vscales.to(DEV), self.table.to(DEV))


# ------------------------------------------------------------------ writing
def _write_case(dtype, hq, hkv, hd, rot, inter, seqs, rows=None, **more):
    """seqs: (first position, tokens) per sequence.  Returns (q, cache tensors, Cache, x in 64 bits, positions, sequences, qkv)."""
    torch.manual_seed(hq * 100 + hd + rot)
    cache = Cache([s for s, _ in seqs], hkv, hd, room=[s + n for s, n in seqs])
    pos = [p for s, n in seqs for p in range(s, s + n)]
    seq = [i for i, (_, n) in enumerate(seqs) for _ in range(n)]
    x = torch.randn(len(pos), hq + 2 * hkv, hd) * torch.exp(torch.randn(hd)) if rows is None else rows(len(pos))
    x = x.to(dtype)
    angle = torch.outer(torch.arange(max(pos) + 1).double(), 10000.0 ** (-torch.arange(rot // 2).double() / max(rot // 2, 1)))
    cos, sin = angle.cos().float(), angle.sin().float()
    if rot == 0:
        cos = sin = torch.zeros(1, 1)
    qkv = x.reshape(len(pos), -1).to(DEV)
    dev = cache.device()
    q = K().rope_append_e4m3(qkv, cos.to(DEV), sin.to(DEV), ints(pos), ints(seq), ints(cache.slots), *dev, hq, hkv, hd, rot, inter, **more)
    y = x.double().clone()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        c, s = cos[pos, i].double().view(-1, 1), sin[pos, i].double().view(-1, 1)
        h = slice(0, hq + hkv)
        y[:, h, a], y[:, h, b] = (x[:, h, a].double() * c - x[:, h, b].double() * s, x[:, h, a].double() * s + x[:, h, b].double() * c)
    return q, dev, cache, x, y, pos, seq, qkv


def _check_write(q, dev, cache, x, y, pos, seq, hq, hkv, hd, written=True):
    # the rotation: two products and a sum in fp32, each off by half a step of no more than |a| + |b| of the pair's numbers
    turn = 3 * 2.0 ** -24 * x.double().abs().amax(dim=-1, keepdim=True) * 2
    assert ((q.cpu().double().view(len(pos), hq, hd) - y[:, :hq]).abs() <= 2.0 ** -8 * y[:, :hq].abs() + turn[:, :hq]).all()
    touched = torch.zeros(dev[0].shape[:3], dtype=torch.bool)
    for what, pages, scales, h0 in (("k", dev[0], dev[2], hq), ("v", dev[1], dev[3], hq + hkv)):
        held, bytes_ = P.values(pages, scales), scales.cpu()
        for r, p in enumerate(pos):
            page = int(cache.table[cache.slots[seq[r]], p // PAGE])
            if not written:
                continue
            touched[page, :, p % PAGE] = True
            want, got = y[r, h0:h0 + hkv], held[page, :, p % PAGE]
            stored, s = P.quantised(want)
            if what == "v":                         # not computed: the definition to the bit
                assert torch.equal(bytes_[page, :, p % PAGE], s)
                assert torch.equal(got, stored * P.two_to(s.long() - 127).unsqueeze(-1))
            else:
                unit = P.two_to(bytes_[page, :, p % PAGE].long() - 127).unsqueeze(-1)
                assert ((got - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * unit) + turn[r, h0:h0 + hkv] * 1.0625).all()
                for e in (-1, 1):                   # the byte is that of the maximum, give or take the rotation's rounding
                    assert (e * (bytes_[page, :, p % PAGE].long() -
                                 P.scale_bytes(want.abs().amax(-1, keepdim=True) + e * turn[r, h0:h0 + hkv]).long()) <= 0).all()
        rest = ~touched if written else torch.ones_like(touched)
        assert (pages.cpu().view(torch.uint8)[rest] == 0x7F).all() and (bytes_[rest] == 255).all(), "written outside its positions"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,hd,rot,inter", [(4, 2, 64, 64, False), (3, 1, 128, 128, False), (5, 5, 64, 32, False), (2, 1, 128, 128, True),
                                                 (16, 1, 128, 96, True), (1, 1, 64, 0, False), (24, 8, 128, 128, False)])
def test_write(dtype, hq, hkv, hd, rot, inter):
    seqs = [(62, 5), (130, 1), (0, 3), (63, 1)]
    q, dev, cache, x, y, pos, seq, _ = _write_case(dtype, hq, hkv, hd, rot, inter, seqs)
    _check_write(q, dev, cache, x, y, pos, seq, hq, hkv, hd)
    K().check_device_errors()


@pytest.mark.parametrize("rot,inter", [(64, False), (32, True)])
@pytest.mark.parametrize("write_cache", [True, False])
def test_write_clears_the_sum_and_a_borrower_writes_nothing(rot, inter, write_cache):
    q, dev, cache, x, y, pos, seq, qkv = _write_case(torch.float32, 6, 2, 64, rot, inter, [(3, 2), (64, 1)], write_cache=write_cache, clear=True)
    _check_write(q, dev, cache, x, y, pos, seq, 6, 2, 64, written=write_cache)
    assert (qkv == 0).all()


def test_write_many_tokens():
    """As many tokens as give each a warp of its own, and a step of several rounds a warp."""
    for dtype in (torch.float32, torch.bfloat16):
        case = _write_case(dtype, 8, 4, 64, 64, False, [(1, 3000), (500, 2100)])
        _check_write(*case[:7], 8, 4, 64)


def test_write_strided_rows():
    """qkv as columns of a wider tensor."""
    hq, hkv, hd = 4, 2, 64
    cache = Cache([0], hkv, hd, room=[3])
    wide = torch.randn(3, (hq + 2 * hkv) * hd + 24, device=DEV)
    cos, sin = torch.ones(3, 32, device=DEV), torch.zeros(3, 32, device=DEV)
    outs = []
    for x in (wide[:, :(hq + 2 * hkv) * hd], wide[:, :(hq + 2 * hkv) * hd].contiguous()):
        dev = cache.device()
        q = K().rope_append_e4m3(x, cos, sin, ints([0, 1, 2]), ints([0, 0, 0]), ints(cache.slots), *dev, hq, hkv, hd, hd)
        outs.append((q, dev[0].view(torch.uint8), dev[1].view(torch.uint8), dev[2], dev[3]))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("rot", [64, 0])
def test_write_zeros_infinities_nan_and_the_ends_of_the_range(rot):
    """Through both kernels (without positions: cosines of 1, or no rotation)."""
    hd = 64
    special = torch.zeros(9, hd)
    special[1, 3] = 1e-42
    special[2, :2] = torch.tensor([448 * 2.0 ** -119, 1e-38])
    special[3, 5], special[3, 6] = 3.4e38, -3e38
    special[4, 7], special[4, 8] = float("inf"), 2.0
    special[5, 9], special[5, 10] = float("nan"), -7.3
    special[6, 11], special[6, 40] = -float("inf"), 1e30
    special[7] = 448.0
    special[8] = torch.linspace(-449, 449, hd)
    x = torch.stack([torch.ones(9, hd), special, -special], dim=1)
    cache = Cache([0], 1, hd, room=[9])
    dev = cache.device()
    cos, sin = torch.ones(9, 32, device=DEV), torch.zeros(9, 32, device=DEV)
    qkv = x.reshape(9, -1).to(DEV)
    if rot:                                         # inf * 0 in the rotation is NaN, as it is in the formula: the values only
        qkv[:, hd:2 * hd] = 0
    K().rope_append_e4m3(qkv, cos, sin, ints(range(9)), ints([0] * 9), ints(cache.slots), *dev, 1, 1, hd, rot)
    page = int(cache.table[cache.slots[0], 0])
    for pages, scales, rows in ((dev[0], dev[2], special), (dev[1], dev[3], -special))[1 if rot else 0:]:
        stored, s = P.quantised(rows)
        assert torch.equal(scales[page, 0, :9].cpu(), s)
        got = P.values(pages, torch.full_like(scales, 127))[page, 0, :9]
        assert torch.equal(torch.nan_to_num(got, nan=-999.0), torch.nan_to_num(stored, nan=-999.0))


def test_write_without_a_page_or_a_position_stores_nothing_and_says_so():
    hq, hkv, hd = 2, 1, 64
    x = torch.randn(1, (hq + 2 * hkv) * hd, device=DEV)
    cos, sin = torch.ones(200, 32, device=DEV), torch.zeros(200, 32, device=DEV)
    for pos, slot, rot in ((70, 0, 64), (70, 0, 32), (-1, 1, 64), (199, 1, 64), (200, 1, 64), (5, 2, 64), (5, -1, 32), (127, 1, 64)):
        cache = Cache([0], hkv, hd, room=[64])
        dev = cache.device()
        table = torch.tensor([[0, -1], [0, 99]], dtype=torch.int32, device=DEV)      # (a page number beyond the cache, too)
        t = (cos, sin) if rot == 64 else (cos[:, :16].contiguous(), sin[:, :16].contiguous())
        q = K().rope_append_e4m3(x, *t, ints([pos]), ints([0]), ints([slot]), *dev[:4], table, hq, hkv, hd, rot)
        assert (dev[0].view(torch.uint8) == 0x7F).all() and (dev[2] == 255).all()
        assert torch.equal(q, x[:, :hq * hd].to(torch.bfloat16))
        with pytest.raises(K().KernelError, match="no page"):
            K().check_device_errors()
        K().check_device_errors()


# ------------------------------------------------------------------ reading back
@pytest.mark.parametrize("hkv,hd", [(1, 64), (2, 128), (7, 64), (8, 128)])
def test_read(hkv, hd):
    torch.manual_seed(hd)
    lens = [1, 64, 65, 200, 128]
    cache = Cache(lens, hkv, hd)
    want = []
    for i, n in enumerate(lens):
        k, v = (torch.randn(n, hkv, hd) * torch.exp(20 * torch.randn(n, hkv, 1)) for _ in range(2))
        want.append(cache.put(i, k, v))
    dev = cache.device()
    order = [(3, 3), (0, 0), (1, 0), (2, 1), (2, 0), (3, 0), (4, 1), (3, 3)]           # any order, a page twice
    pages = ints([[cache.slots[i], p, min(PAGE, lens[i] - PAGE * p)] for i, p in order])
    got = K().read_pages_e4m3(*dev, pages)
    for side in range(2):
        assert got[side].shape == (len(order), hkv, PAGE, hd) and got[side].dtype == torch.bfloat16
        for j, (i, p) in enumerate(order):
            rows = want[i][side][PAGE * p:PAGE * p + PAGE]
            assert torch.equal(got[side][j, :, :rows.shape[0]].cpu().double(), rows.transpose(0, 1))
            assert (got[side][j, :, rows.shape[0]:] == 0).all()
    # given buffers, and fewer rows than there are
    k2, v2 = (torch.full((2, hkv, PAGE, hd), 5.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    K().read_pages_e4m3(*dev, ints([[cache.slots[1], 0, 10], [cache.slots[1], 0, 0]]), k2, v2)
    assert torch.equal(k2[0, :, :10].cpu().double(), want[1][0][:10].transpose(0, 1)) and (k2[0, :, 10:] == 0).all() and (v2[1] == 0).all()


def test_read_of_pages_that_are_not_there_gives_zeros():
    cache = Cache([64], 2, 64)
    cache.put(0, torch.randn(64, 2, 64), torch.randn(64, 2, 64))
    dev = list(cache.device())
    dev[4] = torch.tensor([[-1, 99, 0]], dtype=torch.int32, device=DEV)
    for entry in ([0, 0, 64], [0, 1, 64], [0, 3, 64], [0, -1, 64], [1, 0, 64], [-1, 0, 64], [0, 2, -3]):
        k, v = K().read_pages_e4m3(*dev, ints([entry]))
        assert (k == 0).all() and (v == 0).all()
    k, v = K().read_pages_e4m3(*dev, torch.zeros(0, 3, dtype=torch.int32, device=DEV))
    assert k.shape == (0, 2, 64, 64) and v.shape == (0, 2, 64, 64)


def test_read_gives_back_nan():
    cache = Cache([3], 1, 64)
    x = torch.randn(3, 1, 64)
    x[1, 0, 5] = float("nan")
    cache.put(0, x, x)
    k, _ = K().read_pages_e4m3(*cache.device(), ints([[cache.slots[0], 0, 3]]))
    assert torch.isnan(k[0, 0, 1, 5]) and torch.isnan(k).sum() == 1


# ------------------------------------------------------------------ attention of single tokens
def _visible(pos, span):
    return max(0, pos - span + 1) if span > 0 else (pos - pos % -span if span < 0 else 0)


def _decode_case(hq, hkv, hd, lens, span=0, sink=False, shape=None, dead_pages=False):
    """A cache of sequences of ``lens`` positions; returns (call arguments, [what P.attend gives] per sequence)."""
    torch.manual_seed(hq * 10 + hkv + hd + len(lens) + lens[0])
    cache = Cache(lens, hkv, hd)
    q = (torch.randn(len(lens), hq, hd) * 2).to(torch.bfloat16)
    scale = hd ** -0.5
    sinks = torch.randn(hq) if sink else None
    want = []
    for i, n in enumerate(lens):
        k, v = torch.randn(n, hkv, hd), torch.randn(n, hkv, hd)
        if shape:
            shape(i, q[i], k, v)
        k, v = cache.put(i, k, v)
        lo = _visible(n - 1, span)
        want.append(P.attend(q[i], k[lo:], v[lo:], scale, sinks))
        if dead_pages:
            cache.table[cache.slots[i], :lo // PAGE] = -1
    args = [q.reshape(len(lens), -1).to(DEV), *cache.device(), ints(cache.slots), ints([n - 1 for n in lens]), hq, hkv, hd, scale]
    return args, dict(window=span, sink=None if sinks is None else sinks.to(DEV)), want


def _check_decode(out, want, hd, group):
    """Weights: kept as two e4m3 terms, each off by 2^-4 of what it takes (2^-8 of the weight), or three where a block has four
    heads at most (2^-12, behind a rounding to fp16: 2^-11 in all); below the terms' smallest number, off by 2^-22 (2^-26) of the
    largest weight of their 128 keys, 128 times that in all: 2^-15.  Exponentials within 2^-21, their arguments within what fp32 sums of hd products lose, 2 (hd + 8) 2^-24 of the
    sum of |q k|, and what queries lose below 2^-22 of a row's largest number, hd 2^-22 of the largest product (no more than the
    sum of |q k| again, times 2^-22 hd); the sum over the keys likewise in fp32 (folded into 2^-20); the result to bf16, whose
    smallest number is 2^-133 (half a step: 2^-134).  A weight is an fp32 number relative to the row's largest: one below 2^-126
    may count as zero, so a result may lack 2^-126 of every row's values (which matters where a row of zeros holds all of the
    softmax's weight: in 64 bits the others then come to 2^-650 or so, which no type here holds)."""
    for i, (o, pv, mass, most) in enumerate(want):
        got = out[i].cpu().double().view(o.shape)
        weight = 2.0 ** -11 if group <= 4 else 2.0 ** -8
        tol = 2.0 ** -8 * o.abs() + (weight + 2.0 ** -15 + 2.0 ** -20 + (2 * (hd + 8) * 2.0 ** -24 + hd * 2.0 ** -22) * 1.5 * mass) * pv
        tol = tol + 2.0 ** -134 + 2.0 ** -126 * most
        assert torch.isfinite(got).all(), i
        assert ((got - o).abs() <= tol).all(), (i, float(((got - o).abs() / tol.clamp_min(1e-300)).max()))


HEADS = [(4, 4, 64), (8, 2, 64), (8, 1, 128), (6, 2, 128), (10, 2, 128), (9, 1, 64), (16, 1, 128), (32, 2, 64)]


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [65, 1, 64, 63, 128], [700, 3, 129, 64, 1500], [257]])
def test_decode(hq, hkv, hd, lens):
    args, more, want = _decode_case(hq, hkv, hd, lens)
    _check_decode(K().attention_decode_e4m3(*args, **more), want, hd, hq // hkv)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 64), (10, 2, 128)])
@pytest.mark.parametrize("span", [1, 31, 32, 33, 64, 500, -1, -32, -50, -100000])
@pytest.mark.parametrize("sink", [False, True])
def test_decode_windows_chunks_and_sinks(hq, hkv, hd, span, sink):
    """Pages in front of the window or the chunk have been given back."""
    args, more, want = _decode_case(hq, hkv, hd, [1, 32, 100, 333, 64, 1000], span, sink, dead_pages=True)
    _check_decode(K().attention_decode_e4m3(*args, **more), want, hd, hq // hkv)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 8, 64), (8, 2, 128)])
def test_decode_of_many_sequences(hq, hkv, hd):
    """More sequences than a head has blocks, and than a round's; every length from 1 on."""
    g = torch.Generator().manual_seed(hd)
    lens = [1 + int(x) for x in torch.randint(0, 150, (260,), generator=g)]
    lens[7] = 3000
    args, more, want = _decode_case(hq, hkv, hd, lens)
    _check_decode(K().attention_decode_e4m3(*args, **more), want, hd, hq // hkv)


def test_decode_of_more_sequences_than_a_launch_takes():
    lens = [1 + i % 3 for i in range(2050)]
    args, more, want = _decode_case(2, 1, 64, lens)
    _check_decode(K().attention_decode_e4m3(*args, **more), want, 64, 2)


@pytest.mark.parametrize("hd", [64, 128])
def test_decode_of_one_long_sequence(hd):
    args, more, want = _decode_case(8, 2, hd, [9001])
    _check_decode(K().attention_decode_e4m3(*args, **more), want, hd, 4)


def _tiny_and_huge(i, q, k, v):
    """Values of powers far apart, the small ones under the largest weights, and rows of zeros."""
    v *= 2.0 ** torch.randint(-60, 60, (v.shape[0], 1, 1))
    top = torch.randint(0, v.shape[0], (1,))
    k[top] = 40 * q.float().view(k.shape[1], -1, k.shape[2])[:, 0].sign()
    v[top] *= 2.0 ** -50
    if i == 1:
        v[top] = 0
    if i == 2:
        k.zero_()


def _sharp(i, q, k, v):
    q *= 30.0
    k *= 2.0 ** torch.randint(-4, 4, (k.shape[0], 1, 1))


def _small_queries(i, q, k, v):
    q *= 2.0 ** -100
    k *= 2.0 ** 100
    if i == 0:
        q.zero_()


def _one_value(i, q, k, v):
    v.fill_(-3.0)


def _one_key_and_a_tail(i, q, k, v):
    """The first key holds most of the softmax's weight, all others together the rest, a 2^-16 each."""
    k[1:] = 0
    heads = q.float().view(k.shape[1], -1, k.shape[2])
    k[0] = heads[:, 0] * (16 * 0.6931 * k.shape[2] ** 0.5 / (heads[:, 0] ** 2).sum(-1, keepdim=True))
    q.copy_(heads[:, :1].expand_as(heads).reshape_as(q))


@pytest.mark.parametrize("shape", [_tiny_and_huge, _sharp, _small_queries, _one_value, _one_key_and_a_tail])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 64), (12, 3, 128)])
def test_decode_of_extreme_rows(shape, hq, hkv, hd):
    args, more, want = _decode_case(hq, hkv, hd, [100, 20000 if shape is _one_key_and_a_tail else 2000, 45, 700], shape=shape)
    _check_decode(K().attention_decode_e4m3(*args, **more), want, hd, hq // hkv)


def test_decode_of_nothing_and_of_nan():
    hq, hkv, hd = 8, 2, 64
    for sink in (False, True):
        args, more, want = _decode_case(hq, hkv, hd, [100, 400, 70], sink=sink)
        args[7] = ints([99, -1, 69])
        out = K().attention_decode_e4m3(*args, **more)
        assert (out[1] == 0).all()                          # nothing is visible: zeros
        _check_decode(out[[0, 2]], [want[0], want[2]], hd, hq // hkv)
    # a NaN among the values reaches the heads and the number that it belongs to, and nothing else
    args, more, want = _decode_case(hq, hkv, hd, [100, 400, 70])
    page = int(args[5][int(args[6][1]), 4])
    args[2].view(torch.uint8)[page, 1, 17, 9] = 0x7F        # position 273, key head 1, number 9
    out = K().attention_decode_e4m3(*args, **more)
    bad = torch.isnan(out.view(3, hq, hd))
    assert bad[1, 4:, 9].all() and bad.sum() == 4
    _check_decode(out[[0, 2]], [want[0], want[2]], hd, hq // hkv)
    assert K().attention_decode_e4m3(args[0][:0], *args[1:], **more).shape == (0, hq * hd)


def test_decode_keeps_to_its_rows_and_takes_strides():
    hq, hkv, hd = 8, 2, 64
    args, more, want = _decode_case(hq, hkv, hd, [100, 400, 70])
    plain = K().attention_decode_e4m3(*args, **more)
    wide = torch.full((3, hq * hd + 16), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[:, :hq * hd] = args[0]
    out = torch.full((5, hq * hd + 4), 9.0, dtype=torch.bfloat16, device=DEV)
    K().attention_decode_e4m3(wide[:, :hq * hd], *args[1:], out=out, **more)
    assert torch.equal(out[:3, :hq * hd], plain)
    assert (out[3:] == 9).all() and (out[:, hq * hd:] == 9).all()


def test_decode_repeats_its_bits_and_leaves_its_tickets_zero():
    hq, hkv, hd = 8, 2, 128
    args, more, _ = _decode_case(hq, hkv, hd, [1000, 4000, 70, 2500])
    tickets = torch.zeros(4 * hkv, dtype=torch.int32, device=DEV)
    scratch = torch.empty(K().attention_decode_e4m3_scratch(hq, hkv, hd), device=DEV)
    one = K().attention_decode_e4m3(*args, **more)
    for _ in range(5):
        scratch.fill_(float("nan"))
        assert torch.equal(K().attention_decode_e4m3(*args, scratch=scratch, tickets=tickets, **more), one)
        assert (tickets == 0).all()
    for short in (dict(scratch=scratch[:-1], tickets=tickets), dict(scratch=scratch, tickets=tickets[:-1])):
        with pytest.raises(K().KernelError, match="needed"):
            K().attention_decode_e4m3(*args, **short)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 64), (12, 4, 128)])
def test_a_sequence_grows_token_by_token_through_a_captured_step(hq, hkv, hd):
    """Write, then attend, captured once and replayed with other positions; two sequences on a stream that is not the default
    one.  Every step's result is that of the rows written so far, read back."""
    torch.manual_seed(0)
    cache = Cache([0, 0], hkv, hd, room=[140, 140])
    dev = cache.device()
    slots, seq = ints(cache.slots), ints([0, 1])
    cols = (hq + 2 * hkv) * hd
    angle = torch.outer(torch.arange(140.0), 10000.0 ** (-torch.arange(hd // 2) / (hd // 2)))
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    qkv, pos = torch.zeros(2, cols, device=DEV), ints([0, 0])
    tickets = torch.zeros(2 * hkv, dtype=torch.int32, device=DEV)
    scratch = torch.empty(K().attention_decode_e4m3_scratch(hq, hkv, hd), device=DEV)

    def step():
        q = K().rope_append_e4m3(qkv, cos, sin, pos, seq, slots, *dev, hq, hkv, hd, hd, clear=True)
        return q, K().attention_decode_e4m3(q, *dev, slots, pos, hq, hkv, hd, hd ** -0.5, scratch=scratch, tickets=tickets)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            q, out = step()
        for t in range(130):
            qkv.copy_(torch.randn(2, cols))
            pos.copy_(ints([t, max(0, t - 65)]))
            graph.replay()
            if t in (0, 31, 63, 64, 65, 129):
                lens = [t + 1, max(0, t - 65) + 1]
                pages = ints([[cache.slots[i], p, min(PAGE, n - PAGE * p)] for i, n in enumerate(lens) for p in range(-(-n // PAGE))])
                k, v = K().read_pages_e4m3(*dev, pages)
                stream.synchronize()
                assert (qkv == 0).all()
                want, at = [], 0
                for i, n in enumerate(lens):
                    m = -(-n // PAGE)
                    kk, vv = (x[at:at + m].transpose(1, 2).reshape(m * PAGE, hkv, hd)[:n].cpu() for x in (k, v))
                    want.append(P.attend(q[i].cpu().view(hq, hd), kk.double(), vv.double(), hd ** -0.5))
                    at += m
                _check_decode(out, want, hd, hq // hkv)
    torch.cuda.current_stream().wait_stream(stream)
    K().check_device_errors()


# ------------------------------------------------------------------ calls that users may make
def test_decode_on_two_streams_at_once():
    """Two launches with workspaces of their own, on two streams, many times over."""
    cases = [_decode_case(8, 2, 64, [3000, 700, 64, 1]), _decode_case(16, 2, 128, [2500, 1, 130])]
    want = [K().attention_decode_e4m3(*a, **m).clone() for a, m, _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(30):
        for i, (a, m, _) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                outs[i].append(K().attention_decode_e4m3(*a, **m))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    K().check_device_errors()


def test_decode_launches_one_behind_another_share_their_workspaces():
    """Launches of other lengths and sizes with the same scratch and tickets, without a pause in between."""
    cases = [_decode_case(8, 2, 128, lens) for lens in ([4000], [1, 2, 3], [700] * 9, [64, 2000])]
    want = [K().attention_decode_e4m3(*a, **m).clone() for a, m, _ in cases]
    scratch = torch.empty(K().attention_decode_e4m3_scratch(8, 2, 128), device=DEV)
    tickets = torch.zeros(9 * 2, dtype=torch.int32, device=DEV)
    outs = [[K().attention_decode_e4m3(*a, scratch=scratch, tickets=tickets, **m) for a, m, _ in cases] for _ in range(10)]
    torch.cuda.synchronize()
    for row in outs:
        assert all(torch.equal(o, w) for o, w in zip(row, want))
    assert (tickets == 0).all()


def test_decode_of_one_sequence_several_times_and_of_pages_that_two_share():
    hq, hkv, hd = 8, 2, 64
    args, more, want = _decode_case(hq, hkv, hd, [300])
    q = args[0].repeat(5, 1)
    pos = [299, 0, 63, 64, 299]
    cut = list(args)
    cut[0], cut[6], cut[7] = q, args[6].repeat(5), ints(pos)
    out = K().attention_decode_e4m3(*cut, **more)
    assert torch.equal(out[0], out[4])
    _check_decode(out[[0]], want, hd, hq // hkv)
    k, v = (P.values(args[i], args[i + 2])[args[5][int(args[6][0]), :5].cpu().long()].transpose(1, 2).reshape(-1, hkv, hd) for i in (1, 2))
    for j, p in enumerate(pos):
        _check_decode(out[[j]], [P.attend(args[0][0].cpu().view(hq, hd), k[:p + 1], v[:p + 1], hd ** -0.5)], hd, hq // hkv)
    # two sequences whose first pages are the same ones
    table = args[5].clone()
    other = int(args[6][0]) - 1
    table[other] = table[int(args[6][0])]
    cut = list(args)
    cut[0], cut[5], cut[6], cut[7] = q[:2], table, ints([int(args[6][0]), other]), ints([299, 200])
    out = K().attention_decode_e4m3(*cut, **more)
    _check_decode(out, want + [P.attend(args[0][0].cpu().view(hq, hd), k[:201], v[:201], hd ** -0.5)], hd, hq // hkv)


def test_numbers_outside_the_tables_reach_no_other_row():
    """Slots, positions and page numbers that the tables do not have: kept within them; the other sequences' results stay."""
    hq, hkv, hd = 8, 2, 64
    args, more, want = _decode_case(hq, hkv, hd, [100, 400, 70])
    for slot, pos in ((77, 50), (-3, 50), (int(args[6][1]), 1 << 30), (int(args[6][1]), -(1 << 30))):
        cut = list(args)
        cut[6], cut[7] = ints([int(args[6][0]), slot, int(args[6][2])]), ints([99, pos, 69])
        out = K().attention_decode_e4m3(*cut, **more)
        _check_decode(out[[0, 2]], [want[0], want[2]], hd, hq // hkv)
    cut = list(args)
    cut[5] = args[5].clone()
    cut[5][int(args[6][1])] = torch.tensor([1 << 30, -5, 9999, -1] + [0] * 9, dtype=torch.int32)[:args[5].shape[1]]
    out = K().attention_decode_e4m3(*cut, **more)
    _check_decode(out[[0, 2]], [want[0], want[2]], hd, hq // hkv)
    K().check_device_errors()


def test_alignment_is_asked_for():
    hq, hkv, hd = 8, 2, 64
    args, more, _ = _decode_case(hq, hkv, hd, [100, 40])
    odd = torch.zeros(2, hq * hd + 2, dtype=torch.bfloat16, device=DEV)
    for q, out in ((odd[:, 1:hq * hd + 1], None), (odd[:, :hq * hd], None), (args[0], odd[:, 1:hq * hd + 1])):
        with pytest.raises(K().KernelError, match="alignment"):
            K().attention_decode_e4m3(q, *args[1:], out=out, **more)
    buffer = torch.zeros(1 + args[1].numel(), dtype=torch.uint8, device=DEV)
    shifted = buffer[1:].view(torch.float8_e4m3fn).view(args[1].shape)
    with pytest.raises(K().KernelError, match="alignment"):
        K().attention_decode_e4m3(args[0], shifted, *args[2:], **more)
    with pytest.raises(K().KernelError, match="alignment"):
        K().read_pages_e4m3(shifted, *args[2:6], torch.zeros(1, 3, dtype=torch.int32, device=DEV))
    qkv = torch.zeros(2, (hq + 2 * hkv) * hd + 4, device=DEV)
    cos = torch.zeros(64, 32, device=DEV)
    with pytest.raises(K().KernelError, match="alignment"):
        K().rope_append_e4m3(qkv[:, :-4], cos, cos, ints([0, 1]), ints([0, 0]), args[6], *args[1:6], hq, hkv, hd, hd)


def test_nothing_to_do_is_done():
    hq, hkv, hd = 8, 2, 64
    args, _, _ = _decode_case(hq, hkv, hd, [100])
    cos = torch.zeros(64, 32, device=DEV)
    q = K().rope_append_e4m3(torch.zeros(0, (hq + 2 * hkv) * hd, device=DEV), cos, cos, ints([]), ints([]), args[6], *args[1:6], hq, hkv, hd, hd)
    assert q.shape == (0, hq * hd)


def test_a_query_head_with_an_infinity_gives_nan_and_the_others_their_numbers():
    for hq, hkv, hd in ((8, 2, 64), (8, 1, 128)):
        args, more, want = _decode_case(hq, hkv, hd, [100, 700, 70])
        q = args[0].view(3, hq, hd)
        q[1, 2, 5], q[1, 5, 40], q[0, 3, 7] = float("inf"), -float("inf"), float("nan")
        out = K().attention_decode_e4m3(*args, **more).view(3, hq, hd)
        for i, h in ((1, 2), (1, 5), (0, 3)):
            assert torch.isnan(out[i, h]).all()
            out[i, h] = want[i][0].reshape(hq, hd)[h].to(out)
        _check_decode(out.view(3, -1), want, hd, hq // hkv)


def test_keywords_alone_and_an_output_in_the_queries_place():
    hq, hkv, hd = 4, 2, 64
    args, more, want = _decode_case(hq, hkv, hd, [100, 7])
    names = ("q", "kpages", "vpages", "kscales", "vscales", "page_table", "seq_slot", "token_pos", "num_heads", "num_kv_heads", "head_dim", "scale")
    _check_decode(K().attention_decode_e4m3(**dict(zip(names, args)), **more), want, hd, hq // hkv)
    with pytest.raises(K().KernelError, match="another tensor"):
        K().attention_decode_e4m3(*args, **more, out=args[0])


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 64), (8, 1, 128), (32, 8, 128), (74, 37, 64)])
@pytest.mark.parametrize("lens", [[700], [513, 1], [5000, 300, 260, 1], [129] * 4 + [20000], [900 + 37 * i for i in range(9)],
                                  [200 * (1 + i % 7) for i in range(37)], [100] * 74 + [1500], [40] * 148, [64 * i + 1 for i in range(40)]])
def test_decode_where_blocks_keep_to_one_sequence_and_where_they_do_not(hq, hkv, hd, lens):
    """Numbers of sequences and heads about where a block for each part just is or is not there; sequences whole and cut."""
    args, more, want = _decode_case(hq, hkv, hd, lens)
    tickets = torch.zeros(len(lens) * hkv, dtype=torch.int32, device=DEV)
    out = K().attention_decode_e4m3(*args, **more, tickets=tickets)
    _check_decode(out, want, hd, hq // hkv)
    assert (tickets == 0).all() and torch.equal(out, K().attention_decode_e4m3(*args, **more, tickets=tickets))


@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 128), (8, 1, 64), (3, 1, 64), (16, 1, 128), (2, 2, 128)])
def test_decode_joins_more_parts_than_shared_memory_holds(hq, hkv, hd):
    """One long sequence, its blocks' parts joined in several goes; and a second behind it, of a few parts."""
    for lens in ([60000], [40000, 1500]):
        args, more, want = _decode_case(hq, hkv, hd, lens)
        _check_decode(K().attention_decode_e4m3(*args, **more), want, hd, hq // hkv)


@pytest.mark.parametrize("rot", [64, 32])
def test_write_for_a_sequence_that_is_not_there_stores_nothing_and_says_so(rot):
    hq, hkv, hd = 2, 1, 64
    x = torch.randn(3, (hq + 2 * hkv) * hd, device=DEV)
    cos, sin = torch.ones(4, rot // 2, device=DEV), torch.zeros(4, rot // 2, device=DEV)
    for seq in (2, -1, 2 ** 31 - 1, -2 ** 31):
        cache = Cache([3, 3], hkv, hd)
        dev = cache.device()
        q = K().rope_append_e4m3(x, cos, sin, ints([0, 1, 2]), ints([0, seq, 1]), ints(cache.slots), *dev, hq, hkv, hd, rot)
        assert torch.equal(q, x[:, :hq * hd].to(torch.bfloat16))
        written = torch.zeros(dev[2].shape, dtype=torch.bool)
        written[int(cache.table[cache.slots[0], 0]), :, 0] = written[int(cache.table[cache.slots[1], 0]), :, 2] = True
        assert torch.equal((dev[2] != 255).cpu(), written) and torch.equal((dev[0].view(torch.uint8) != 0x7F).any(-1).cpu(), written)
        with pytest.raises(K().KernelError, match="no page"):
            K().check_device_errors()


def test_more_tiles_than_32_bits_count_are_refused():
    args, more, want = _decode_case(2, 1, 64, [70])
    table = torch.full((1, 2 ** 21), -1, dtype=torch.int32, device=DEV)
    table[0, :2] = args[5][int(args[6][0]), :2]
    args[5], args[6] = table, ints([0])
    _check_decode(K().attention_decode_e4m3(*args, **more), want, 64, 2)
    args[0], args[6], args[7] = args[0].expand(1024, -1).contiguous(), ints([0] * 1024), ints([69] * 1024)
    with pytest.raises(K().KernelError, match="size"):
        K().attention_decode_e4m3(*args, **more)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes of keys, written, read and attended at its last pages; more than 2^31 numbers read back."""
    hq, hkv, hd = 16, 8, 128
    n = 2 ** 32 // (hkv * PAGE * hd) + 8
    kp, vp = (torch.zeros(n, hkv, PAGE, hd, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.full((n, hkv, PAGE), 127, dtype=torch.uint8, device=DEV) for _ in range(2))
    f8 = torch.float8_e4m3fn
    table = ints([[n - 1, n - 3], [-1, n - 2]])
    cache = (kp.view(f8), vp.view(f8), ks, vs, table)
    torch.manual_seed(1)
    x = torch.randn(100, hq + 2 * hkv, hd)
    cos, sin = torch.ones(100, hd // 2, device=DEV), torch.zeros(100, hd // 2, device=DEV)
    q = K().rope_append_e4m3(x.reshape(100, -1).to(DEV), cos, sin, ints(range(100)), ints([0] * 100), ints([0]), *cache, hq, hkv, hd, hd)
    K().check_device_errors()
    rows = []
    for h0, pages, scales in ((hq, kp, ks), (hq + hkv, vp, vs)):
        stored, s = P.quantised(x[:, h0:h0 + hkv])
        rows.append(stored * P.two_to(s.long() - 127).unsqueeze(-1))
        held = P.values(pages[[n - 1, n - 3]].view(f8), scales[[n - 1, n - 3]])
        assert torch.equal(held.transpose(1, 2).reshape(2 * PAGE, hkv, hd)[:100], rows[-1])
        assert not pages[:n - 8].any() and not pages[n - 2].any()
    out = K().attention_decode_e4m3(q[99:], *cache, ints([0]), ints([99]), hq, hkv, hd, hd ** -0.5)
    _check_decode(out, [P.attend(q[99].cpu().view(hq, hd), rows[0], rows[1], hd ** -0.5, None)], hd, hq // hkv)
    del kp, vp, pages
    many = 2 ** 31 // (hkv * PAGE * hd) + 3
    listed = torch.tensor([[1, 1, 0]], dtype=torch.int32).repeat(many, 1)
    listed[-2:] = torch.tensor([[0, 1, 36], [0, 0, 64]])
    for got, want in zip(K().read_pages_e4m3(*cache, listed.to(DEV)), rows):
        assert torch.equal(got[-1].transpose(0, 1).double().cpu(), want[:PAGE])
        assert torch.equal(got[-2].transpose(0, 1)[:36].double().cpu(), want[PAGE:]) and not got[-2, :, 36:].any() and not got[-3].any()
