"""The 8-bit cache without a GPU: its definition, and what its operators refuse."""
import pytest
import torch

import plain_e4m3 as P


def test_nearest_agrees_with_the_types_own_rounding():
    x = torch.cat([torch.linspace(-460, 460, 20011), torch.linspace(-0.05, 0.05, 4001), torch.arange(0, 449, dtype=torch.float32) / 512])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(P.nearest(x), want)
    assert torch.isnan(P.nearest(torch.tensor([float("nan")]))).all()
    assert P.nearest(torch.tensor([float("inf"), float("-inf")])).tolist() == [448.0, -448.0]


def test_values_agree_with_the_types_own_values():
    bits = torch.arange(256, dtype=torch.uint8)
    got = P.values(bits.view(1, 1, 1, 256), torch.full((1, 1, 1), 127, dtype=torch.uint8)).view(-1)
    want = bits.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(got, nan=-7.0), torch.nan_to_num(want, nan=-7.0))


def test_scale_bytes_at_their_borders():
    top = 448.0
    rows = torch.tensor([[0.0], [top], [top * (1 + 2.0 ** -23)], [1.75], [1.7500001], [1e-45], [3.4e38], [float("inf")], [float("nan")],
                         [top * 2.0 ** -119], [top * 2.0 ** 10]], dtype=torch.float32)
    assert P.scale_bytes(rows).tolist() == [8, 127, 128, 119, 120, 8, 246, 246, 8, 8, 137]


@pytest.mark.parametrize("hd", [64, 128])
def test_a_values_distance_from_its_row_is_half_a_step(hd):
    torch.manual_seed(hd)
    rows = torch.randn(200, hd) * torch.exp(4 * torch.randn(200, 1)) * torch.exp(torch.randn(hd))
    stored, s = P.quantised(rows)
    unit = P.two_to(s.long() - 127).unsqueeze(-1)
    off = (stored * unit - rows.double()).abs()
    assert (off <= torch.maximum(2.0 ** -4 * rows.double().abs(), 2.0 ** -10 * unit)).all()
    assert torch.equal((stored * unit).to(torch.bfloat16).double(), stored * unit), "bfloat16 holds every value"


def _tensors(hd=64, hkv=2, pages=3, page=64):
    kp = torch.zeros(pages, hkv, page, hd, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = torch.zeros(pages, hkv, page, dtype=torch.uint8)
    return kp, kp.clone(), sc, sc.clone(), torch.zeros(2, 4, dtype=torch.int32)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_operators_name_what_does_not_fit():
    from dlgo_b200.csrc import kernels as K
    kp, vp, ks, vs, pt = _tensors()
    cos = torch.zeros(10, 32)
    qkv = torch.zeros(3, 8 * 64)

    def write(qkv=qkv, cache=(kp, vp, ks, vs, pt), hq=4, hkv=2, hd=64, rot=64, cos=cos, pos=_ints(0, 1, 2), seq=_ints(0, 0, 0), **more):
        return K.rope_append_e4m3(qkv, cos, cos, pos, seq, _ints(0), *cache, hq, hkv, hd, rot, **more)

    def decode(q=torch.zeros(3, 256, dtype=torch.bfloat16), cache=(kp, vp, ks, vs, pt), hq=4, hkv=2, hd=64, slot=_ints(0, 1, 0), **more):
        return K.attention_decode_e4m3(q, *cache, slot, _ints(0, 0, 0), hq, hkv, hd, 1.0, **more)

    def read(cache=(kp, vp, ks, vs, pt), pages=torch.zeros(1, 3, dtype=torch.int32), **more):
        return K.read_pages_e4m3(*cache, pages, **more)

    for call in (write, decode, read):
        with pytest.raises(K.KernelError, match="GPU"):
            call()
        for cache, word in (((kp, vp[:2], ks, vs, pt), "keys and values"), ((kp, vp, ks[:, :1], vs, pt), "scale byte"),
                            ((kp, vp, ks, vs, pt[:0]), "page table"), (_tensors(hd=96), "64 or 128"), (_tensors(page=32), "64 or 128")):
            with pytest.raises(K.KernelError, match=word):
                call(cache=cache)
    for more, word in ((dict(hkv=1), "fit"), (dict(hd=128), "columns"), (dict(hq=0), "positive"), (dict(qkv=qkv[:, :300]), "columns"),
                       (dict(qkv=qkv.t()), "columns"), (dict(pos=_ints(0)), "per token"), (dict(rot=66), "rotary_dim"), (dict(rot=3), "rotary_dim"),
                       (dict(rot=32), "cos and sin"), (dict(cos=cos[:0]), "cos and sin"), (dict(qkv=qkv.half()), "float32 or bfloat16"),
                       (dict(qkv=qkv.bfloat16(), clear=True), "fp32")):
        with pytest.raises(K.KernelError, match=word):
            write(**more)
    for more, word in ((dict(hq=3), "multiple"), (dict(hkv=1), "fit"), (dict(q=torch.zeros(3, 200)), "columns"), (dict(slot=_ints(0)), "per sequence"),
                       (dict(sink=torch.zeros(3)), "sink"), (dict(out=torch.zeros(2, 256)), "rows")):
        with pytest.raises(K.KernelError, match=word):
            decode(**more)
    for more, word in ((dict(pages=torch.zeros(1, 2, dtype=torch.int32)), "slot, page"), (dict(keys=torch.zeros(2, 2, 64, 64)), "must be")):
        with pytest.raises(K.KernelError, match=word):
            read(**more)


def test_pages_in_sight_of_a_step():
    """The list of pages that a prompt step copies, and the table that finds them in the copy."""
    from dlgo_b200.engine.runtime import StepContext

    class Runtime:
        device = torch.device("cpu")

    def ctx():
        return StepContext(runtime=Runtime(), n_tokens=0, n_seqs=3, token_ids=None, token_pos=None, token_seq=None, seq_slot=None,
                           seq_slots_host=[7, 2, 5], seq_start_host=[0, 130, 63], seq_ntok_host=[3, 65, 1], decode=False, max_len=195)

    pages, table, at = ctx().pages_in_sight(0, 64)
    assert pages.tolist() == [[7, 0, 3], [2, 0, 64], [2, 1, 64], [2, 2, 64], [2, 3, 3], [5, 0, 64]]
    assert table.tolist() == [[0, -1, -1, -1], [1, 2, 3, 4], [5, -1, -1, -1]] and at.tolist() == [0, 1, 2]
    pages, table, _ = ctx().pages_in_sight(3, 64)           # a window of 3: the first query at 130 sees 128 on
    assert pages.tolist() == [[7, 0, 3], [2, 2, 64], [2, 3, 3], [5, 0, 64]] and table.tolist() == [[0, -1, -1, -1], [-1, -1, 1, 2], [3, -1, -1, -1]]
    pages, table, _ = ctx().pages_in_sight(4, 64)           # 127 on: a page more
    assert pages.tolist()[1] == [2, 1, 64] and table.tolist()[1] == [-1, 1, 2, 3]
    pages, table, _ = ctx().pages_in_sight(-100, 64)        # chunks of 100: from position 100 on
    assert pages.tolist() == [[7, 0, 3], [2, 1, 64], [2, 2, 64], [2, 3, 3], [5, 0, 64]]


def test_operators_take_their_arguments_by_name():
    from dlgo_b200.csrc import kernels as K
    kp, vp, ks, vs, pt = _tensors()
    with pytest.raises(K.KernelError, match="GPU"):
        K.read_pages_e4m3(kpages=kp, vpages=vp, kscales=ks, vscales=vs, page_table=pt, pages=torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(TypeError, match="kpages"):
        K.read_pages_e4m3(vpages=vp)
