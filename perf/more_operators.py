"""Operators that rotate, store in 4 bits and attend over 4 bits beside the eviction path, as cases to be
timed and compared:

  rotate  the position rotation of new queries and keys, with keys and values written into the paged
          16-bit cache on the way
  store   new keys and values (rotated or not) quantised into a paged 4-bit cache, and those tokens
          read back out of it
  attn    attention of each session's newest tokens (a chunk; a single token is a chunk of one) over
          the 4-bit cache, with its log-sum-exp

With ``own`` false, ``run`` computes them in plain torch; with it true, through actkv_open_b200.

The rotation: with c, s the cosine and sine of position * frequency i (an fp32 table [P, rot]: rot / 2
cosines, then as many sines), (x, y) becomes (x c - y s, y c + x s).  The pair i is dims (i, i + rot / 2)
("halves") or (2 i, 2 i + 1) ("pairs"); dims from rot on stay.  Positions are their own input: after
an eviction a token's position is not its place in the cache.

The 4-bit cache: ``rows`` [L, 2, NB, BS, row_bytes] uint8, a token's row of one plane being Hkv * D / 2
bytes of e2m1 values, then Hkv * D / 32 scale bytes (one per 32 values: the value is e2m1 * 2^(byte - 127);
from 253 on NaN), then padding.  The exponent is the smallest, up to byte 252, with
max|x| <= 7 * 2^(byte - 127).  Value 32 g + 4 p + j of a head (p < 8, j < 4) is in the head's byte
p * D / 16 + 2 g + j / 2, the low half for even j.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
GROUP = 32              # values that share a scale byte
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
POSITIONS = 65536       # positions of the rotation's table


def listed():
    heads = {"hq": 32, "hkv": 8, "d": 128, "bs": 16, "dtype": "bfloat16", "rot": 128, "pairs": False}
    return [
        # a decoding step's queries, keys and values of one layer: launch and latency
        {"name": "rotate step", "kind": "rotate", "r": 32, "s_lo": 1, "s_hi": 2000, "a_lo": 1, "a_hi": 1, "l": 1, **heads},
        # prompts of mixed lengths, half of each head rotated in neighbouring pairs, fp16
        {"name": "rotate partial fp16", "kind": "rotate", "r": 9, "s_lo": 701, "s_hi": 1500, "a_lo": 0, "a_hi": 700, "l": 2,
         "hq": 24, "hkv": 8, "d": 64, "bs": 32, "dtype": "float16", "rot": 32, "pairs": True},
        # one session's chunk of a long prompt, one layer
        {"name": "rotate chunk", "kind": "rotate", "r": 1, "s_lo": 6001, "s_hi": 6001, "a_lo": 2048, "a_hi": 2048, "l": 1, **heads},
        # an agent round's rows of several layers
        {"name": "rotate round", "kind": "rotate", "r": 8, "s_lo": 1088, "s_hi": 2500, "a_lo": 1088, "a_hi": 1088, "l": 8, **heads},
        # a decoding step of one layer into 4 bits
        {"name": "store step", "kind": "store", "r": 32, "s_lo": 1, "s_hi": 2000, "a_lo": 1, "a_hi": 1, "l": 1, **heads},
        # rows that were rotated before, an agent round's
        {"name": "store round unrotated", "kind": "store", "r": 8, "s_lo": 1088, "s_hi": 2500, "a_lo": 1088, "a_hi": 1088, "l": 8,
         **heads, "rot": 0},
        # prompts of mixed lengths with their rotation, fp16
        {"name": "store prompts fp16", "kind": "store", "r": 12, "s_lo": 901, "s_hi": 4000, "a_lo": 0, "a_hi": 901, "l": 4,
         "hq": 32, "hkv": 8, "d": 64, "bs": 32, "dtype": "float16", "rot": 64, "pairs": False},
        # one user's next token at a short context: the launch and latency end of decoding
        {"name": "attn one token", "kind": "attn", "r": 1, "s_lo": 2000, "s_hi": 2000, "a_lo": 1, "a_hi": 1, **heads},
        # a full decoding batch of ragged contexts: the cache is read once, bandwidth bound
        {"name": "attn decode batch", "kind": "attn", "r": 32, "s_lo": 4096, "s_hi": 32768, "a_lo": 1, "a_hi": 1, **heads},
        # a few drafted tokens per session, two query heads per KV head, fp16
        {"name": "attn drafted fp16", "kind": "attn", "r": 16, "s_lo": 1000, "s_hi": 9000, "a_lo": 2, "a_hi": 4,
         "hq": 16, "hkv": 8, "d": 64, "bs": 16, "dtype": "float16", "rot": 0, "pairs": False},
        # prompts, single tokens and idle sessions in one batch, three query heads per KV head
        {"name": "attn mixed", "kind": "attn", "r": 9, "s_lo": 701, "s_hi": 5001, "a_lo": 0, "a_hi": 700, **heads, "hq": 24},
        # observation chunks on top of long sessions
        {"name": "attn chunk", "kind": "attn", "r": 4, "s_lo": 4096, "s_hi": 16384, "a_lo": 512, "a_hi": 512, **heads},
    ]


def draw(rng):
    def spread(lo, hi):                       # whole numbers, evenly in their logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))

    kind = rng.choice(["rotate", "store", "attn", "attn"])
    hkv, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    d = rng.choice({"rotate": [64, 80, 96, 128, 128], "store": [64, 96, 128, 128], "attn": [64, 128, 128]}[kind])
    case = {"kind": kind, "hq": hkv * g, "hkv": hkv, "d": d, "bs": rng.choice([16, 16, 32]),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16"]), "rot": 0, "pairs": False}
    if kind != "attn":
        case["rot"] = rng.choice([d, d, d // 2, 32] if kind == "rotate" else [d, d, d // 2, 0])
        case["pairs"] = rng.random() < 0.3
        while True:
            r, layers, a_hi = spread(1, 32), spread(1, 36), spread(1, 20000)
            if r * layers * a_hi * (2 * hkv + hkv * g) <= 8 * 8 * 1088 * 48:
                break
        s_hi = a_hi + rng.randint(0, 500)
        a_lo = a_hi if rng.random() < 0.5 else rng.randint(0, a_hi)
        case.update(r=r, l=layers, a_lo=a_lo, a_hi=a_hi, s_hi=s_hi, s_lo=rng.randint(max(1, a_lo), s_hi))
        return case
    while True:
        r, a_hi, s_hi = spread(1, 32), rng.choice([1, spread(2, 16), spread(17, 2048)]), spread(16, 32768)
        a_hi = min(a_hi, s_hi)
        # the padded logits of the plain form, and the cache, stay below the listed cases'
        if r * hkv * g * a_hi * s_hi <= 1.0e9 and r * hkv * s_hi <= 32 * 8 * 24000:
            break
    a_lo = a_hi if rng.random() < 0.4 else rng.randint(0, a_hi)
    case.update(r=r, a_lo=a_lo, a_hi=a_hi, s_hi=s_hi, s_lo=rng.randint(max(a_hi, 1), s_hi))
    return case


def ragged(lo, hi, n, turn):
    """n whole numbers over [lo, hi], the two ends among them where n allows, in a mixed order."""
    if n == 1:
        return [hi]
    steps = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    mixed = sorted(range(n), key=lambda i: (i * 0.6180339887 + turn) % 1.0)
    return [steps[i] for i in mixed]


def lengths(case):
    """(tokens in each session's cache, the newest of them that the call is about)."""
    s = ragged(case["s_lo"], case["s_hi"], case["r"], 0.1)
    a = ragged(case["a_lo"], case["a_hi"], case["r"], 0.7)
    return s, [min(x, y) for x, y in zip(a, s)]


def row_bytes(hkv, d):
    return -(-hkv * (d // 2 + d // GROUP) // 32) * 32


# ------------------------------------------------------------------------------ a user's data

def normal(shape, gen, dtype, scale=None):
    x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    return x if scale is None else x.mul_(scale.to(dtype))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt = "cuda", DTYPES[case["dtype"]]
    hq, hkv, d, bs, layers, rot = case["hq"], case["hkv"], case["d"], case["bs"], case.get("l", 1), case["rot"]
    seq, new = lengths(case)
    r = len(seq)
    blocks = [-(-n // bs) for n in seq]
    nb, mb, total = max(1, sum(blocks)), max(1, max(blocks)), sum(new)
    # physical blocks in a shuffled order, as an allocator that has run for a while gives them
    order = torch.randperm(nb, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(r, mb, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    off = [0]
    for n in new:
        off.append(off[-1] + n)
    st = {"case": case, "table": table, "seq": torch.tensor(seq, dtype=torch.int32, device=dev),
          "off": torch.tensor(off, dtype=torch.int32, device=dev), "seq_max": max(seq), "new_max": max(new), "total": total}
    # keys with unequal channels, as models have them; values and queries of unit size
    chan = torch.rand(hkv, d, generator=gen, device=dev) * 1.5 + 0.5
    if case["kind"] == "attn":
        rows = torch.zeros(2, nb, bs, row_bytes(hkv, d), dtype=torch.uint8, device=dev)
        for p in range(2):
            x = normal((nb * bs, hkv, d), gen, dt, chan if p == 0 else None)
            rows[p].view(nb * bs, -1)[:, :hkv * (d // 2 + d // GROUP)] = plain_pack(x)
        st["rows"], st["q"] = rows, normal((total, hq, d), gen, dt)
        return st
    st["k"], st["v"] = normal((layers, total, hkv, d), gen, dt, chan), normal((layers, total, hkv, d), gen, dt)
    if case["kind"] == "rotate":
        st["kv"] = torch.zeros(layers, 2, nb, bs, hkv, d, dtype=dt, device=dev)
    else:
        st["rows"] = torch.zeros(layers, 2, nb, bs, row_bytes(hkv, d), dtype=torch.uint8, device=dev)
    if rot:
        st["q"] = normal((layers, total, hq, d), gen, dt)
        # every session has had tokens evicted: its newest ones stand further on than its length
        gone = torch.randint(0, POSITIONS - max(seq), (r,), generator=gen, device=dev, dtype=torch.int32)
        sess, pos = newest(st)
        st["pos"] = (pos + gone[sess]).to(torch.int32)
        angle = torch.arange(POSITIONS, device=dev, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
        st["angles"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    return st


# ------------------------------------------------------------------------------ the plain forms

def pow2(e):
    """2^e in 32 bits, exactly, for whole e in [-127, 127]."""
    bits = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22))
    return bits.to(torch.int32).view(torch.float32)


def plain_pack(x):
    """[N, Hkv, D] -> [N, Hkv * (D / 2 + D / 32)] uint8: the row of the 4-bit cache."""
    n, hkv, d = x.shape
    f = x.float().view(n, hkv * d // GROUP, GROUP)
    top = f.abs().amax(-1)
    mant, exp = torch.frexp(top)                                    # top = mant * 2^exp, mant in [0.5, 1)
    byte = torch.where(mant <= 0.875, exp - 3, exp - 2) + 127
    byte = torch.where(top > 0, byte.clamp(0, 252), torch.zeros_like(byte))
    bad = ~torch.isfinite(f).all(-1)
    small = f * pow2(127 - byte).unsqueeze(-1)                      # |.| <= 7, unless the byte is 252
    small = torch.where(bad.unsqueeze(-1), torch.zeros_like(small), small)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    a = small.abs()                                                 # to the nearest level, ties to the even code
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code += 8 * torch.signbit(small)
    code = code.view(n, hkv, d // GROUP, 8, 2, 2)                   # group, piece, byte of the piece, half of the byte
    both = (code[..., 0] + 16 * code[..., 1]).permute(0, 1, 3, 2, 4)
    return torch.cat([both.reshape(n, hkv * d // 2), byte.to(torch.uint8)], 1)


def plain_unpack(rows, hkv, d):
    """[..., row_bytes] uint8 -> [..., Hkv, D] in 32 bits."""
    both = rows[..., :hkv * d // 2].unflatten(-1, (hkv, 8, d // GROUP, 2)).transpose(-2, -3)
    code = torch.stack([both & 15, both >> 4], -1).flatten(-3)      # [..., Hkv, groups, 32]
    signed = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=rows.device)
    byte = rows[..., hkv * d // 2:hkv * (d // 2 + d // GROUP)].to(torch.int32)
    scale = pow2((byte - 127).clamp(max=125))
    scale = torch.where(byte >= 253, torch.full_like(scale, math.nan), scale).unflatten(-1, (hkv, d // GROUP))
    return (signed[code.to(torch.int32)] * scale.unsqueeze(-1)).flatten(-2)


def plain_rotate(x, pos, angles, pairs):
    """x [L, T, H, D] rotated, in 32 bits."""
    f = x.float()
    rot = angles.shape[1]
    c, s = angles[pos.long(), None, :rot // 2], angles[pos.long(), None, rot // 2:]
    if pairs:
        a, b = f[..., 0:rot:2], f[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = f[..., :rot // 2], f[..., rot // 2:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, f[..., rot:]], -1)


def newest(st):
    """(session, position in its cache) of every new token, in the packed order."""
    t = torch.arange(st["total"], device="cuda", dtype=torch.int32)
    sess = torch.bucketize(t, st["off"][1:], right=True)
    new = st["off"][1:] - st["off"][:-1]
    return sess, (st["seq"] - new)[sess] + t - st["off"][:-1][sess]


def slots(st):
    """The cache slot of every new token."""
    bs = st["case"]["bs"]
    sess, pos = newest(st)
    return st["table"][sess, (pos // bs).long()].long() * bs + pos % bs


def plain_attention(st, k, v):
    """k, v [R, S, Hkv, D] in 32 bits, padded to the longest session -> (out [T, Hq, D], lse [T, Hq])."""
    q, seq, off = st["q"], st["seq"].long(), st["off"].long()
    n, hq, d = q.shape
    r, s, hkv = k.shape[:3]
    a, g = st["new_max"], hq // hkv
    j = torch.arange(a, device="cuda")
    new = off[1:] - off[:-1]
    pick = (off[:-1, None] + j).clamp(max=n - 1)                    # [R, A]
    qp = q[pick].float().view(r, a, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, g * a, d)
    x = torch.matmul(qp, k.permute(0, 2, 3, 1)) * d ** -0.5         # [R, Hkv, G * A, S]
    seen = torch.arange(s, device="cuda") <= (seq - new)[:, None, None] + j[:, None]      # [R, A, S]
    x = x.view(r, hkv, g, a, s).masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    x = x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    valid = torch.arange(s, device="cuda") < seq[:, None]
    v = torch.where(valid[:, :, None, None], v, torch.zeros_like(v))
    o = torch.matmul(x.view(r, hkv, g * a, s), v.permute(0, 2, 1, 3)).view(r, hkv, g, a, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (m + total.log()).squeeze(-1)
    sess, pos = newest(st)
    t = (pos - (seq - new)[sess]).long()
    out = o.permute(0, 3, 1, 2, 4).reshape(r, a, hq, d)[sess, t]
    return out.to(q.dtype), lse.permute(0, 3, 1, 2).reshape(r, a, hq)[sess, t]


def run_plain(st):
    case = st["case"]
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    dt = DTYPES[case["dtype"]]
    if kind == "attn":
        at = st["table"].long()
        return plain_attention(st, *(plain_unpack(st["rows"][p][at].flatten(1, 2)[:, :st["seq_max"]], hkv, d) for p in range(2)))
    slot = slots(st)
    q, k = None, st["k"]
    if case["rot"]:
        q = plain_rotate(st["q"], st["pos"], st["angles"], case["pairs"]).to(dt)
        k = plain_rotate(k, st["pos"], st["angles"], case["pairs"])
    if kind == "rotate":
        flat = st["kv"].flatten(2, 3)
        flat[:, 0, slot], flat[:, 1, slot] = k.to(dt), st["v"]
        return q, st["kv"]
    flat = st["rows"].flatten(2, 3)                                 # [L, 2, NB * BS, row_bytes]
    for p, x in enumerate((k, st["v"])):
        packed = plain_pack(x.flatten(0, 1)).view(x.shape[0], x.shape[1], -1)
        flat[:, p, slot, :packed.shape[-1]] = packed
    back = plain_unpack(flat[:, :, slot], hkv, d).to(dt)
    return {"q": q, "k": back[:, 0], "v": back[:, 1]}


# ------------------------------------------------------------------------------ the framework's

def run_own(st):
    from actkv_open_b200.kernels import chunk_attn, quant_cache, rotary
    case = st["case"]
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    if kind == "attn":
        if "workspace" not in st:               # a serving loop keeps it from call to call
            st["workspace"] = chunk_attn.chunk_workspace("cuda")
        return quant_cache.paged_chunk_attention_quant(st["q"], st["off"], st["rows"], hkv, st["table"], st["seq"],
                                                       workspace=st["workspace"], bits=4)
    if kind == "rotate":
        q = rotary.rotate_write(st["q"], st["k"], st["v"], st["pos"], st["angles"], st["off"], st["kv"], st["table"],
                                st["seq"], interleaved=case["pairs"])
        return q, st["kv"]
    q = None
    if case["rot"]:
        q = rotary.rotate_write(st["q"], st["k"], st["v"], st["pos"], st["angles"], st["off"], st["rows"], st["table"],
                                st["seq"], interleaved=case["pairs"], bits=4)
    else:
        quant_cache.quantize_write(st["k"], st["v"], st["off"], st["rows"], st["table"], st["seq"], bits=4)
    k, v = quant_cache.dequantize_read(st["rows"], hkv, d, st["off"], st["table"], st["seq"], st["total"],
                                       dtype=DTYPES[case["dtype"]], bits=4)
    return {"q": q, "k": k, "v": v}


def run(st):
    return run_own(st) if own else run_plain(st)


# ------------------------------------------------------------------------------ floors and 64 bits

def work(case):
    seq, new = lengths(case)
    hq, hkv, d, layers, rot = case["hq"], case["hkv"], case["d"], case.get("l", 1), case["rot"]
    total = sum(new)
    packed = hkv * (d // 2 + d // GROUP)
    if case["kind"] == "attn":
        live = sum(s for s, a in zip(seq, new) if a)
        pairs = sum(a * (s - a) + a * (a + 1) // 2 for s, a in zip(seq, new))
        return {"bytes": 2 * live * packed + total * hq * (4 * d + 4), "flops": 4 * pairs * hq * d}
    moved = 2 * hkv * d * 4 if case["kind"] == "rotate" else 2 * (hkv * d * 4 + 2 * packed)
    turned = (hq * d * 4 if rot else 0, (hq + hkv) * rot * 3)
    return {"bytes": total * (layers * (moved + turned[0]) + 4 * rot), "flops": total * layers * (turned[1] + 2 * hkv * d)}


def exact_pow2(e):
    """2^e in 64 bits, exactly, for whole e of any type."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exact_rows(rows, hkv, d):
    """What the rows' bytes stand for, [N, Hkv * D] in 64 bits."""
    n = rows.shape[0]
    dim = torch.arange(d, device=rows.device)
    group, piece, j = dim // 32, dim % 32 // 4, dim % 4
    place = piece * (d // 16) + 2 * group + j // 2
    byte = rows[:, :hkv * d // 2].reshape(n, hkv, d // 2)[:, :, place].long()
    code = byte >> (4 * (j % 2)) & 15
    e, m = code >> 1 & 3, (code & 1).double()
    size = torch.where(e == 0, m / 2, (1 + m / 2) * exact_pow2(e - 1))
    scale = exact_pow2(rows[:, hkv * d // 2:hkv * (d // 2 + d // GROUP)].long() - 127).view(n, hkv, -1)
    return ((1.0 - 2.0 * (code >> 3)) * size * scale[:, :, group]).view(n, hkv * d)


def exact_turn(x, pos, angles, pairs):
    """x [T, H, D] rotated in 64 bits, as complex numbers."""
    rot = angles.shape[1]
    turn = torch.complex(angles[:, :rot // 2].double()[pos.long()], angles[:, rot // 2:].double()[pos.long()])[:, None]
    y = x.double().clone()
    first = y[..., :rot].unflatten(-1, (rot // 2, 2) if pairs else (2, rot // 2))
    z = torch.complex(*(first.unbind(-1) if pairs else first.unbind(-2))) * turn
    y[..., :rot] = torch.stack([z.real, z.imag], -1 if pairs else -2).flatten(-2)
    return y


def exact_stored(x):
    """[T, H, D] in 64 bits -> what the 4-bit cache holds of it."""
    y = x.flatten(1).unflatten(-1, (-1, GROUP))
    top = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 7.0))                     # settled below where log2 is near a whole number
    e = torch.where(top > 7.0 * exact_pow2(e), e + 1, e)
    e = torch.where(top <= 7.0 * exact_pow2(e - 1), e - 1, e).clamp(-127, 125)
    z = y * exact_pow2(-e)
    step = exact_pow2(torch.frexp(z.abs().clamp(min=1.0))[1] - 2)     # a half below 2, 1 below 4, 2 from there on
    return ((torch.round(z / step) * step).clamp(-6.0, 6.0) * exact_pow2(e)).view(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    seq, new = lengths(case)
    hq, hkv, d, bs, layers = case["hq"], case["hkv"], case["d"], case["bs"], case.get("l", 1)
    g = hq // hkv
    offs = st["off"].tolist()

    def places(i, first, last):
        pos = torch.arange(first, last, device="cuda")
        return st["table"][i].long()[pos // bs] * bs + pos % bs

    if case["kind"] == "attn":
        out = torch.zeros(st["total"], hq, d, dtype=torch.float64, device="cuda")
        lse = torch.zeros(st["total"], hq, dtype=torch.float64, device="cuda")
        src = st["rows"].view(2, -1, st["rows"].shape[-1])
        for i, (s, a) in enumerate(zip(seq, new)):
            if a == 0:
                continue
            both = [exact_rows(src[p][places(i, 0, s)], hkv, d).view(s, hkv, d) for p in range(2)]
            hidden = torch.arange(s, device="cuda")[None] > torch.arange(s - a, s, device="cuda")[:, None]
            for x in range(hq):
                logit = st["q"][offs[i]:offs[i + 1], x].double() @ both[0][:, x // g].T / math.sqrt(d)
                logit[hidden] = -math.inf
                one = torch.logsumexp(logit, -1)
                lse[offs[i]:offs[i + 1], x] = one
                out[offs[i]:offs[i + 1], x] = torch.exp(logit - one[:, None]) @ both[1][:, x // g]
        return out, lse
    turn = (lambda x: exact_turn(x, st["pos"], st["angles"], case["pairs"])) if case["rot"] else (lambda x: x.double())
    q = torch.stack([turn(x) for x in st["q"]]) if case["rot"] else None
    if case["kind"] == "store":
        return {"q": q, "k": torch.stack([exact_stored(turn(x)) for x in st["k"]]),
                "v": torch.stack([exact_stored(x.double()) for x in st["v"]])}
    nb = st["kv"].shape[2]
    kv = torch.zeros(layers, 2, nb * bs, hkv, d, dtype=torch.float64, device="cuda")
    for la in range(layers):
        k = turn(st["k"][la])
        for i, (s, a) in enumerate(zip(seq, new)):
            at = places(i, s - a, s)
            kv[la, 0, at], kv[la, 1, at] = k[offs[i]:offs[i + 1]], st["v"][la, offs[i]:offs[i + 1]].double()
    return q, kv.view(layers, 2, nb, bs, hkv, d)
