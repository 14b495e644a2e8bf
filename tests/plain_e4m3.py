"""The 8-bit cache's definition in 64 bits, for tests: rows of e4m3 numbers with one power of two each."""
import torch


def two_to(k):
    """2^k in 64 bits (whole k within the exponents' range)."""
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def scale_bytes(rows):
    """e + 127 with e the smallest whole number such that max |x| <= 448 * 2^e, within [-119, 119] (NaN does not count)."""
    most = torch.nan_to_num(rows.double(), nan=0.0, posinf=1e300, neginf=-1e300).abs().amax(dim=-1)
    limits = 448 * two_to(torch.arange(-119, 119))          # by comparing, not by the bits: the limits that it is beyond
    e = torch.searchsorted(limits, most.contiguous()) - 119
    return (e + 127).to(torch.uint8)


def nearest(x):
    """The e4m3 number nearest to each x, ties to even, beyond 448 the largest (64 bits; NaN stays)."""
    grid = torch.tensor(sorted({m * 2.0 ** (max(k, 1) - 10) for k in range(16) for m in (range(8, 16) if k else range(8))} - {480.0}),
                        dtype=torch.float64)        # 0, the subnormal and normal numbers up to 448, in the order of their bits
    a = torch.nan_to_num(x.double(), nan=0.0, posinf=1e300, neginf=-1e300).abs().clamp_max(448.0)
    hi = torch.searchsorted(grid, a.contiguous()).clamp_max(grid.numel() - 1)
    lo = (hi - 1).clamp_min(0)
    up, down = grid[hi] - a, a - grid[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    out = torch.copysign(grid[pick], x.double())
    return torch.where(torch.isnan(x), torch.full_like(out, float("nan")), out)


def quantised(rows):
    """(stored numbers in 64 bits, scale bytes) of rows [..., head size]."""
    rows = rows.double()
    s = scale_bytes(rows)
    return nearest(rows / two_to(s.long() - 127).unsqueeze(-1)), s


def values(pages, scales):
    """The values that e4m3 pages and their scale bytes stand for, in 64 bits on the CPU."""
    bits = pages.cpu().view(torch.uint8).long()
    sign, k, m = 1 - 2 * (bits >> 7), (bits >> 3) & 15, bits & 7
    x = torch.where(k > 0, (8 + m).double() * two_to(k - 10), m.double() / 512)
    x = torch.where((bits & 127) == 127, torch.full_like(x, float("nan")), x) * sign
    return x * two_to(scales.cpu().long() - 127).unsqueeze(-1)


def attend(q, k, v, scale, sink=None):
    """softmax(q k^T scale) v for one query row per head: q [Hq, d], k and v [n, Hkv, d] -> ([Hq, d], the sum of p |v|, the
    largest sum of |q k| scale, the sum of the rows' largest |v|), in 64 bits; ``sink`` [Hq] joins the denominator."""
    hq, hkv = q.shape[0], k.shape[1]
    kh, vh = (x.double().repeat_interleave(hq // hkv, dim=1) for x in (k, v))
    s = torch.einsum("hd,nhd->hn", q.double(), kh) * scale
    mass = torch.einsum("hd,nhd->hn", q.double().abs(), kh.abs()).amax(dim=1, keepdim=True) * abs(scale)
    if sink is not None:
        s = torch.cat([s, sink.double().view(-1, 1)], dim=1)
    p = torch.softmax(s, dim=1)[:, :k.shape[0]]
    return torch.einsum("hn,nhd->hd", p, vh), torch.einsum("hn,nhd->hd", p, vh.abs()), mass, float(vh.abs().amax(dim=2).amax(dim=1).sum())
