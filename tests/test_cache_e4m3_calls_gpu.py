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
