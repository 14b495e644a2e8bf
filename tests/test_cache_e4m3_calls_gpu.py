"""The 8-bit cache's functions on the GPU: calls that the other files leave out."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def K():
    from dlgo_b200.csrc import kernels
    return kernels


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(hkv, hd, pages=4):
    kp, vp = (torch.full((pages, hkv, 64, hd), 0x7F, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((pages, hkv, 64), 255, dtype=torch.uint8, device=DEV) for _ in range(2))
    return kp, vp, ks, vs, ints(*range(pages)).view(1, pages)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_write_without_a_rotation_takes_no_tables(hd, dtype):
    """The same rows as with cosines of one, which the rotation leaves as they are, to the bit; positions beyond any table too."""
    hq, hkv = 4, 2
    torch.manual_seed(hd)
    x = torch.randn(5, (hq + 2 * hkv) * hd, device=DEV).to(dtype)
    pos = ints(0, 1, 63, 64, 255)
    got = []
    for cos, sin, rot in ((None, None, 0), (torch.ones(256, hd // 2, device=DEV), torch.zeros(256, hd // 2, device=DEV), hd)):
        cache = _cache(hkv, hd)
        q = K().rope_append_e4m3(x, cos, sin, pos, ints(0, 0, 0, 0, 0), ints(0), *cache, hq, hkv, hd, rot)
        got.append((q, *(c.view(torch.uint8) for c in cache[:4])))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert torch.equal(got[0][0], x[:, :hq * hd].to(torch.bfloat16)) and (got[0][3] != 255).sum() == 5 * hkv
    K().check_device_errors()


def test_decode_into_columns_beside_the_queries():
    """One buffer, queries left and outputs right: no memory in common, so it is taken."""
    hq, hkv, hd, B = 8, 2, 64, 3
    cache = _cache(hkv, hd)
    torch.manual_seed(0)
    cos, sin = torch.ones(100, hd // 2, device=DEV), torch.zeros(100, hd // 2, device=DEV)
    K().rope_append_e4m3(torch.randn(100, (hq + 2 * hkv) * hd, device=DEV), cos, sin, ints(*range(100)), ints(*[0] * 100), ints(0), *cache,
                         hq, hkv, hd, hd)
    buf = torch.randn(B, 2 * hq * hd, device=DEV).to(torch.bfloat16)
    q = buf[:, :hq * hd].clone()
    args = (*cache, ints(0, 0, 0), ints(99, 5, 64), hq, hkv, hd, hd ** -0.5)
    want = K().attention_decode_e4m3(q, *args)
    K().attention_decode_e4m3(buf[:, :hq * hd], *args, out=buf[:, hq * hd:])
    assert torch.equal(buf[:, hq * hd:], want) and torch.equal(buf[:, :hq * hd], q)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 8, 128), (7, 7, 128), (6, 6, 128), (36, 6, 128), (4, 4, 64), (3, 3, 64), (24, 3, 64), (42, 6, 64)])
def test_decode_joins_about_as_many_parts_as_one_go_holds(hq, hkv, hd):
    """One long sequence over all blocks of the device, 37 to 98 parts a kv head, around what shared memory holds at a time (45 to 91);
    against a plain softmax in 64 bits with the tolerance of the other tests."""
    import test_cache_e4m3_gpu as G
    args, more, want = G._decode_case(hq, hkv, hd, [24000])
    out = K().attention_decode_e4m3(*args, **more)
    G._check_decode(out, want, hd, hq // hkv)
    assert torch.equal(out, K().attention_decode_e4m3(*args, **more))
    K().check_device_errors()


def _off_by(args, more, lens, want, out, hd, group):
    """The largest error over its bound.  As in the other tests, with the bound of what is lost below the smallest term of a weight
    written out: 2^-22 of the largest weight of a tile (2^-26 with three terms), a weight being a softmax's times its value's power
    of two, for every number that the values hold.  It matters where the heaviest key's value is zero at a number and a key far
    lighter is all that is left there.  (Weights counted against the whole row's largest: no less than a tile's.)"""
    import plain_e4m3 as P
    hq, hkv, scale, worst = args[8], args[9], args[11], 0.0
    pages, table, slots = [a.cpu() for a in args[1:5]], args[5].cpu(), args[6].tolist()
    for i, (o, pv, mass, most) in enumerate(want):
        n = lens[i]
        at = table[slots[i], :-(-n // 64)].long()
        k, v = (P.values(pages[j][at], pages[j + 2][at]).transpose(1, 2).reshape(-1, hkv, hd)[:n] for j in (0, 1))
        power = P.two_to(pages[3][at].transpose(1, 2).reshape(-1, hkv)[:n].long() - 127)
        s = torch.einsum("hd,nhd->hn", args[0][i].cpu().double().view(hq, hd), k.repeat_interleave(group, 1)) * scale
        if more["sink"] is not None:
            s = torch.cat([s, more["sink"].cpu().double().view(-1, 1)], 1)
        p = torch.softmax(s, 1)[:, :n]
        weight, least = (2.0 ** -11, 2.0 ** -26) if group <= 4 else (2.0 ** -8, 2.0 ** -22)
        lost = least * (p * power.repeat_interleave(group, 1).T).amax(1, keepdim=True) * (v / power.unsqueeze(-1)).abs().sum(0).repeat_interleave(group, 0)
        tol = 2.0 ** -8 * o.abs() + (weight + 2.0 ** -20 + (2 * (hd + 8) * 2.0 ** -24 + hd * 2.0 ** -22) * 1.5 * mass) * pv
        tol = tol + lost * (1 + 2.0 ** -8) + 2.0 ** -134 + 2.0 ** -126 * most
        worst = max(worst, float(((out[i].cpu().double().view(o.shape) - o).abs() / tol).max()))
    return worst


@pytest.mark.parametrize("hq,hkv,hd", [(6, 2, 64), (16, 1, 128), (45, 5, 128), (24, 1, 64), (8, 8, 128)])
@pytest.mark.parametrize("lens", [[1 + i % 3 for i in range(40)], [6, 20, 2, 1, 27, 3], [1 + 7 * i % 31 for i in range(150)]])
@pytest.mark.parametrize("shape", ["_sharp", "_tiny_and_huge"])
def test_decode_of_few_keys_whose_weights_are_far_apart(hq, hkv, hd, lens, shape):
    import test_cache_e4m3_gpu as G
    for sink in (False, True):
        args, more, want = G._decode_case(hq, hkv, hd, lens, sink=sink, shape=getattr(G, shape))
        out = K().attention_decode_e4m3(*args, **more)
        assert _off_by(args, more, lens, want, out, hd, hq // hkv) <= 1
