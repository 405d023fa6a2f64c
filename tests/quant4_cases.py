"""The 4-bit row and the position rotation from their definitions, in 64 bits (CPU torch, no kernels)."""
import math

import torch

import chunk_cases as C

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def place(d):
    """(byte of a head, half of it) of every dim."""
    dim = torch.arange(d)
    g, p, j = dim // 32, dim % 32 // 4, dim % 4
    return p * (d // 16) + 2 * g + j // 2, j % 2


def quantise_ref(x):
    """[..., D] -> (values, codes, scale bytes [..., D / 32]) of the 4-bit row."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    finite = torch.isfinite(g).all(-1)
    e = torch.full(top.shape, -127, dtype=torch.int64)
    for k in range(-127, 125):                        # the smallest exponent that fits, from below
        e = torch.where((e == k) & (top > 7.0 * 2.0 ** k) & finite, torch.tensor(k + 1), e)
    z = torch.where(finite.unsqueeze(-1), g * 2.0 ** (-e.double()).unsqueeze(-1), torch.zeros_like(g))
    a = z.abs()
    far = (a.unsqueeze(-1) - LEVELS).abs()
    near = far.amin(-1, keepdim=True)
    ties = far == near                                # one level, or two neighbours: then the even code
    code = torch.where(ties & (torch.arange(8) % 2 == 0), torch.arange(8), torch.where(ties, torch.arange(8) + 100, 1000))
    code = code.amin(-1) % 100
    scale = torch.where(finite, e + 127, torch.tensor(255))
    val = LEVELS[code] * torch.where(torch.signbit(z), -1.0, 1.0).double() * (2.0 ** (scale - 127).double()).unsqueeze(-1)
    val = torch.where((scale == 255).unsqueeze(-1), torch.tensor(math.nan, dtype=torch.float64), val)
    code = code + 8 * torch.signbit(z).long()
    return val.flatten(-2), code.flatten(-2).to(torch.uint8), scale.to(torch.uint8)


def pack_rows(x, row):
    """[N, Hkv, D] -> [N, row] uint8 rows of the 4-bit cache (padding 0xAB)."""
    n, hkv, d = x.shape
    _, code, scale = quantise_ref(x)
    byte, half = place(d)
    vals = torch.zeros(n, hkv, d // 2, dtype=torch.uint8)
    for dim in range(d):
        vals[:, :, byte[dim]] |= code[:, :, dim] << int(4 * half[dim])
    out = torch.full((n, row), 0xAB, dtype=torch.uint8)
    out[:, :hkv * d // 2] = vals.reshape(n, hkv * d // 2)
    out[:, hkv * d // 2:hkv * (d // 2 + d // 32)] = scale.reshape(n, hkv * d // 32)
    return out


def unpack_rows(rows, hkv, d):
    """[N, row] uint8 -> [N, Hkv, D] in 64 bits."""
    n = len(rows)
    byte, half = place(d)
    code = rows[:, :hkv * d // 2].reshape(n, hkv, d // 2)[:, :, byte].long() >> (4 * half) & 15
    scale = rows[:, hkv * d // 2:hkv * (d // 2 + d // 32)].long().reshape(n, hkv, d // 32)
    s = torch.where(scale >= 253, torch.tensor(math.nan, dtype=torch.float64), 2.0 ** (scale - 127).double())
    val = LEVELS[code & 7] * (1.0 - 2.0 * (code >> 3)) * s.repeat_interleave(32, -1)
    return val


def turn(x, positions, angles, pairs):
    """[L, T, H, D] rotated, in x's type (fp32: each product and sum rounded by itself; or fp64)."""
    rot = angles.shape[1]
    c = angles[positions.long(), None, :rot // 2].to(x.dtype)
    s = angles[positions.long(), None, rot // 2:].to(x.dtype)
    y = x.clone()
    if pairs:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def new_tokens(lens, new, hq, hkv, d, bs, layers, dtype, seed, rot=0, positions=5000):
    """Inputs of a call: block table, offsets, q, k, v and, with rot, positions and angles."""
    gen = torch.Generator().manual_seed(seed)
    table, nb = C.pages(lens, bs, gen)
    off = C.offsets(new)
    n = int(off[-1])
    k = (torch.randn(layers, n, hkv, d, generator=gen) * torch.exp(2 * torch.randn(layers, n, hkv, 1, generator=gen))).to(dtype)
    v = torch.randn(layers, n, hkv, d, generator=gen).to(dtype)
    q = torch.randn(layers, n, hq, d, generator=gen).to(dtype)
    pos = torch.randint(0, positions, (n,), generator=gen).int()
    return table, nb, off, q, k, v, pos


def written(table, off, lens, bs, layers):
    """(layer-independent) pairs of packed token and cache slot of a call's tokens."""
    tok, slot = [], []
    for r, s in enumerate(lens):
        o0, o1 = int(off[r]), int(off[r + 1])
        if o1 > o0:
            tok.append(torch.arange(o0, o1))
            slot.append(C.slots(table, r, s - (o1 - o0), s, bs))
    if not tok:
        return torch.zeros(0, dtype=torch.long), torch.zeros(0, dtype=torch.long)
    return torch.cat(tok), torch.cat(slot)
