"""Inputs and 64-bit references for the chunk attention and 8-bit cache tests (CPU torch, no kernels)."""
import math

import torch

# e4m3, by its definition: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f / 0xff are NaN
_B = torch.arange(256)
_E, _M = (_B >> 3) & 15, (_B & 7).double()
E4M3 = torch.where(_E == 0, _M / 8 * 2.0 ** -6, (1 + _M / 8) * 2.0 ** (_E - 7).double()) * (1 - 2.0 * (_B >> 7))
E4M3[127] = E4M3[255] = math.nan
_GRID = E4M3[:127]                                   # the non-negative values, ascending


def pages(lens, bs, gen, extra=2, first=0):
    """(block_table [R, MB], number of blocks): each session's blocks in shuffled physical order."""
    n = [-(-s // bs) for s in lens]
    order = torch.randperm(sum(n) + extra, generator=gen) + first
    table = torch.zeros(len(lens), max(max(n), 1), dtype=torch.int32)
    at = 0
    for r, k in enumerate(n):
        table[r, :k] = order[at:at + k].int()
        at += k
    return table, sum(n) + extra + first


def slots(table, r, first, last, bs):
    pos = torch.arange(first, last)
    return table[r].long()[pos // bs] * bs + pos % bs


def offsets(new):
    return torch.tensor([0] + list(new)).cumsum(0).int()


def attention_ref(q, off, k_of, v_of, lens, scale):
    """64-bit attention of the newest queries of every session.

    k_of(r) / v_of(r): [S, Hkv, D].  Returns out, lse, and the two magnitudes that the error bounds
    are made of: sum p |v| / l per output and max_t scale * sum |q_d k_d| per row."""
    T, hq, d = q.shape
    out, mag = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(T, hq, d, dtype=torch.float64)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64)
    size = torch.zeros(T, hq, dtype=torch.float64)
    for r, s in enumerate(lens):
        o0, o1 = int(off[r]), int(off[r + 1])
        if o1 == o0 or s == 0:
            continue
        k, v = k_of(r).double(), v_of(r).double()
        g = hq // k.shape[1]
        for t in range(o0, o1):
            seen = s - (o1 - t) + 1
            if seen <= 0:
                continue
            qq = q[t].double().view(-1, g, d)
            kk, vv = k[:seen], v[:seen]
            x = torch.einsum("hgd,shd->hgs", qq, kk) * scale
            m = x.amax(-1, keepdim=True)
            p = torch.exp(x - m)
            l = p.sum(-1, keepdim=True)
            out[t] = (torch.einsum("hgs,shd->hgd", p, vv) / l).view(hq, d)
            mag[t] = (torch.einsum("hgs,shd->hgd", p, vv.abs()) / l).view(hq, d)
            lse[t] = (m + l.log()).view(hq)
            size[t] = (torch.einsum("hgd,shd->hgs", qq.abs(), kk.abs()).amax(-1) * scale).view(hq)
    return out, lse, mag, size


def quantise_ref(x):
    """[..., D] -> (values, bytes, scale bytes) of the 8-bit row, in 64 bits from the definition."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    finite = torch.isfinite(g).all(-1)
    e = torch.full(top.shape, -127, dtype=torch.int64)
    for k in range(-127, 129):                        # the smallest exponent that fits, from below
        e = torch.where((e == k) & (top > 448.0 * 2.0 ** k) & finite, torch.tensor(k + 1), e)
    z = torch.where(finite.unsqueeze(-1), g * 2.0 ** (-e.double()).unsqueeze(-1), torch.zeros_like(g))
    a = z.abs().contiguous()
    hi = torch.searchsorted(_GRID, a).clamp(max=126)  # first grid value >= a
    lo = (hi - 1).clamp(min=0)
    up, down = _GRID[hi] - a, a - _GRID[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(a == _GRID[hi], hi, code)
    byte = code + 128 * torch.signbit(z).long()
    scale = torch.where(finite, e + 127, torch.tensor(255))
    val = E4M3[byte] * (2.0 ** (scale - 127).double()).unsqueeze(-1)
    val = torch.where((scale == 255).unsqueeze(-1), torch.tensor(math.nan, dtype=torch.float64), val)
    return val.flatten(-2), byte.flatten(-2).to(torch.uint8), scale.to(torch.uint8)


def pack_rows(x, row):
    """[N, Hkv, D] -> [N, row] uint8 rows of the 8-bit cache (padding 0xAB)."""
    n, hkv, d = x.shape
    _, byte, scale = quantise_ref(x)
    out = torch.full((n, row), 0xAB, dtype=torch.uint8)
    out[:, :hkv * d] = byte.reshape(n, hkv * d)
    out[:, hkv * d:hkv * (d + d // 32)] = scale.reshape(n, hkv * d // 32)
    return out


def unpack_rows(rows, hkv, d):
    """[N, row] uint8 -> [N, Hkv, D] in 64 bits."""
    scale = rows[:, hkv * d:hkv * (d + d // 32)].long()
    s = torch.where(scale == 255, torch.tensor(math.nan, dtype=torch.float64), 2.0 ** (scale - 127).double())
    val = E4M3[rows[:, :hkv * d].long()].unflatten(-1, (-1, 32)) * s.unsqueeze(-1)
    return val.reshape(-1, hkv, d)
