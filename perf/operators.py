"""The operators that attend and store beside the eviction path, as cases to be timed and compared:

  attn        attention of each session's newest tokens (a chunk; a single token is a chunk of one)
              over its paged cache, with the log-sum-exp that the scoring step consumes
  attn_quant  the same over a paged cache held in 8 bits
  write       quantising new K / V rows into that cache, every layer at once
  read        the newest tokens of each session read back out of it

With ``own`` false, ``run`` computes them in plain torch; with it true, through actkv_open_b200.

The 8-bit cache: ``rows`` [L, 2, NB, BS, row_bytes] uint8, a token's row of one plane being Hkv * D
e4m3 values, then Hkv * D / 32 scale bytes (one per 32 values: the value is e4m3 * 2^(byte - 127);
byte 255 is NaN), then padding.  The exponent is the smallest with max|x| <= 448 * 2^(byte - 127).
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
GROUP = 32              # values that share a scale byte
E4M3_MAX = 448.0


def listed():
    heads = {"hq": 32, "hkv": 8, "d": 128, "bs": 16, "dtype": "bfloat16"}
    return [
        # one user's next token at a short context: the launch and latency end of decoding
        {"name": "attn one token", "kind": "attn", "r": 1, "s_lo": 2000, "s_hi": 2000, "a_lo": 1, "a_hi": 1, **heads},
        # a full decoding batch of ragged contexts: the cache is read once, bandwidth bound
        {"name": "attn decode batch", "kind": "attn", "r": 32, "s_lo": 4096, "s_hi": 32768, "a_lo": 1, "a_hi": 1, **heads},
        # a few drafted tokens per session, to be verified in one pass
        {"name": "attn drafted", "kind": "attn", "r": 16, "s_lo": 1000, "s_hi": 9000, "a_lo": 3, "a_hi": 7, **heads},
        # prompts, single tokens and idle sessions in one batch: fp16, three query heads per KV head
        {"name": "attn mixed fp16", "kind": "attn", "r": 9, "s_lo": 701, "s_hi": 5001, "a_lo": 0, "a_hi": 700,
         "hq": 24, "hkv": 8, "d": 64, "bs": 32, "dtype": "float16"},
        # an agent round: 1024 observed and 64 action tokens per session on top of its cache
        {"name": "attn agent round", "kind": "attn", "r": 6, "s_lo": 2000, "s_hi": 10000, "a_lo": 1088, "a_hi": 1088, **heads},
        # a chunk of a long prompt at the end of a 32K context: the compute-bound end
        {"name": "attn long chunk", "kind": "attn", "r": 1, "s_lo": 32768, "s_hi": 32768, "a_lo": 2048, "a_hi": 2048, **heads},
        # the decoding batch over the 8-bit cache: half the bytes
        {"name": "attn_quant decode batch", "kind": "attn_quant", "r": 32, "s_lo": 4096, "s_hi": 32768, "a_lo": 1, "a_hi": 1, **heads},
        # observation chunks over the 8-bit cache
        {"name": "attn_quant chunk", "kind": "attn_quant", "r": 4, "s_lo": 4096, "s_hi": 16384, "a_lo": 512, "a_hi": 512, **heads},
        # a decoding step's rows of all layers
        {"name": "write step", "kind": "write", "r": 32, "s_lo": 1, "s_hi": 2000, "a_lo": 1, "a_hi": 1, "l": 36, **heads},
        # an agent round's rows of several layers
        {"name": "write round", "kind": "write", "r": 8, "s_lo": 1088, "s_hi": 2500, "a_lo": 1088, "a_hi": 1088, "l": 8, **heads},
        # the action region of every session and layer (a window at the end of each cache)
        {"name": "read window", "kind": "read", "r": 16, "s_lo": 128, "s_hi": 1500, "a_lo": 128, "a_hi": 128, "l": 4, **heads},
        # whole sessions of some layers, e.g. to score them in 16 bits
        {"name": "read sessions", "kind": "read", "r": 4, "s_lo": 3000, "s_hi": 20001, "a_lo": 20001, "a_hi": 20001, "l": 4, **heads},
    ]


def draw(rng):
    def spread(lo, hi):                       # whole numbers, evenly in their logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))

    kind = rng.choice(["attn", "attn", "attn", "attn_quant", "write", "read"])
    hkv = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 8]) if kind == "attn" else rng.choice([1, 2, 4, 8])
    case = {"kind": kind, "hq": hkv * g, "hkv": hkv, "d": rng.choice([64, 128, 128]), "bs": rng.choice([16, 16, 32]),
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16"])}
    if kind in ("attn", "attn_quant"):
        while True:
            r, a_hi, s_hi = spread(1, 32), rng.choice([1, spread(2, 16), spread(17, 2048)]), spread(16, 32768)
            a_hi = min(a_hi, s_hi)
            # the padded logits of the plain form, and the cache, stay below the listed cases'
            if r * hkv * g * a_hi * s_hi <= 2.0e9 and r * hkv * s_hi <= 32 * 8 * 24000:
                break
        a_lo = a_hi if rng.random() < 0.4 else rng.randint(0, a_hi)
        case.update(r=r, a_lo=a_lo, a_hi=a_hi, s_hi=s_hi, s_lo=rng.randint(max(a_hi, 1), s_hi))
    else:
        while True:
            r, layers, a_hi = spread(1, 32), spread(1, 36), spread(1, 20000)
            if r * layers * a_hi * hkv <= 8 * 8 * 1088 * 8:
                break
        s_hi = a_hi + rng.randint(0, 500)
        a_lo = a_hi if rng.random() < 0.5 else rng.randint(0, a_hi)
        case.update(r=r, l=layers, a_lo=a_lo, a_hi=a_hi, s_hi=s_hi, s_lo=rng.randint(max(1, a_lo), s_hi))
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
    return -(-hkv * (d + d // GROUP) // 64) * 64


# ------------------------------------------------------------------------------ a user's data

def normal(shape, gen, dtype, scale=None):
    x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    return x if scale is None else x.mul_(scale.to(dtype))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt = "cuda", DTYPES[case["dtype"]]
    hq, hkv, d, bs, layers = case["hq"], case["hkv"], case["d"], case["bs"], case.get("l", 1)
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
    kind = case["kind"]
    if kind == "attn":
        kv = normal((2, nb, bs, hkv, d), gen, dt)
        kv[0] *= chan.to(dt)
        st["kv"] = kv
    elif kind in ("attn_quant", "read"):
        rows = torch.zeros(layers, 2, nb, bs, row_bytes(hkv, d), dtype=torch.uint8, device=dev)
        for la in range(layers):
            for p in range(2):
                x = normal((nb * bs, hkv, d), gen, dt, chan if p == 0 else None)
                rows[la, p].view(nb * bs, -1)[:, :hkv * (d + d // GROUP)] = plain_pack(x)
        st["rows"] = rows[0] if kind == "attn_quant" else rows
    else:
        st["rows"] = torch.zeros(layers, 2, nb, bs, row_bytes(hkv, d), dtype=torch.uint8, device=dev)
        st["k"] = normal((layers, total, hkv, d), gen, dt, chan)
        st["v"] = normal((layers, total, hkv, d), gen, dt)
    if kind in ("attn", "attn_quant"):
        st["q"] = normal((total, hq, d), gen, dt)
    return st


# ------------------------------------------------------------------------------ the plain forms

def pow2(e):
    """2^e in 32 bits, exactly, for whole e in [-127, 127]."""
    bits = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22))
    return bits.to(torch.int32).view(torch.float32)


def plain_pack(x):
    """[N, Hkv, D] -> [N, Hkv * (D + D / 32)] uint8: the row of the 8-bit cache."""
    n, hkv, d = x.shape
    f = x.float().view(n, hkv * d // GROUP, GROUP)
    top = f.abs().amax(-1)
    mant, exp = torch.frexp(top)                                    # top = mant * 2^exp, mant in [0.5, 1)
    byte = torch.where(mant <= E4M3_MAX / 512, exp - 9, exp - 8) + 127
    byte = torch.where(top > 0, byte.clamp(0, 254), torch.zeros_like(byte))
    bad = ~torch.isfinite(f).all(-1)
    small = f * pow2(127 - byte).unsqueeze(-1)                      # |.| <= 448
    small = torch.where(bad.unsqueeze(-1), torch.zeros_like(small), small)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    return torch.cat([small.to(torch.float8_e4m3fn).view(torch.uint8).view(n, hkv * d), byte.to(torch.uint8)], 1)


def plain_unpack(rows, hkv, d):
    """[..., row_bytes] uint8 -> [..., Hkv, D] in 32 bits."""
    val = rows[..., :hkv * d].view(torch.float8_e4m3fn).float()
    byte = rows[..., hkv * d:hkv * (d + d // GROUP)].to(torch.int32)
    val = val.unflatten(-1, (-1, GROUP)) * pow2((byte - 127).clamp(max=127)).unsqueeze(-1)
    val = torch.where((byte == 255).unsqueeze(-1), torch.full_like(val, float("nan")), val)
    return val.flatten(-2).unflatten(-1, (hkv, d))


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
    kind, hkv, d, bs = case["kind"], case["hkv"], case["d"], case["bs"]
    if kind in ("attn", "attn_quant"):
        table = st["table"].long()
        planes = []
        for p in range(2):
            x = st["kv"][p] if kind == "attn" else st["rows"][p]
            x = x[table].flatten(1, 2)[:, :st["seq_max"]]
            planes.append(x.float() if kind == "attn" else plain_unpack(x, hkv, d))
        return plain_attention(st, *planes)
    slot = slots(st)
    rows = st["rows"]
    flat = rows.flatten(2, 3)                                       # [L, 2, NB * BS, row_bytes]
    if kind == "write":
        for p, x in enumerate((st["k"], st["v"])):
            packed = plain_pack(x.flatten(0, 1)).view(x.shape[0], x.shape[1], -1)
            flat[:, p, slot, :packed.shape[-1]] = packed
        return written(st)
    got = plain_unpack(flat[:, :, slot], hkv, d).to(DTYPES[case["dtype"]])
    return got[:, 0], got[:, 1]


def written(st):
    """The whole cache after a write, as the values that its bytes stand for (views)."""
    hkv, d = st["case"]["hkv"], st["case"]["d"]
    rows = st["rows"]
    return {"values": rows[..., :hkv * d].view(torch.float8_e4m3fn),
            "scales": rows[..., hkv * d:hkv * (d + d // GROUP)].view(torch.float8_e8m0fnu)}


# ------------------------------------------------------------------------------ the framework's

def run_own(st):
    from actkv_open_b200.kernels import chunk_attn, quant_cache
    case = st["case"]
    kind, hkv, d = case["kind"], case["hkv"], case["d"]
    if kind in ("attn", "attn_quant"):
        if "workspace" not in st:               # a serving loop keeps it from call to call
            st["workspace"] = chunk_attn.chunk_workspace("cuda")
        if kind == "attn":
            return chunk_attn.paged_chunk_attention(st["q"], st["off"], st["kv"], st["table"], st["seq"],
                                                    workspace=st["workspace"])
        return quant_cache.paged_chunk_attention_quant(st["q"], st["off"], st["rows"], hkv, st["table"], st["seq"],
                                                       workspace=st["workspace"])
    if kind == "write":
        quant_cache.quantize_write(st["k"], st["v"], st["off"], st["rows"], st["table"], st["seq"])
        return written(st)
    return quant_cache.dequantize_read(st["rows"], hkv, d, st["off"], st["table"], st["seq"], st["total"],
                                       dtype=DTYPES[case["dtype"]])


def run(st):
    return run_own(st) if own else run_plain(st)


# ------------------------------------------------------------------------------ floors and 64 bits

def work(case):
    seq, new = lengths(case)
    hq, hkv, d, layers = case["hq"], case["hkv"], case["d"], case.get("l", 1)
    total = sum(new)
    packed = hkv * (d + d // GROUP)
    if case["kind"] in ("write", "read"):
        return {"bytes": layers * 2 * total * (hkv * d * 2 + packed), "flops": layers * 2 * total * hkv * d * 2}
    token = packed if case["kind"] == "attn_quant" else hkv * d * 2
    live = sum(s for s, a in zip(seq, new) if a)
    pairs = sum(a * (s - a) + a * (a + 1) // 2 for s, a in zip(seq, new))
    return {"bytes": 2 * live * token + total * hq * (4 * d + 4), "flops": 4 * pairs * hq * d}


def exact_pow2(e):
    """2^e in 64 bits, exactly, for whole e of any type."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exact_e4m3(byte):
    """What e4m3 bytes stand for, in 64 bits."""
    b = torch.arange(256, device=byte.device)
    sign = 1.0 - 2.0 * (b >> 7).double()
    e, m = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * exact_pow2(e - 7))
    mag = torch.where((b & 127) == 127, torch.full_like(mag, math.nan), mag)
    return (sign * mag)[byte.long()]


def exact_rows(rows, hkv, d):
    scale = exact_pow2(rows[..., hkv * d:hkv * (d + d // GROUP)].long() - 127)
    return (exact_e4m3(rows[..., :hkv * d]).unflatten(-1, (-1, GROUP)) * scale.unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    seq, new = lengths(case)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    g = hq // hkv
    kind = case["kind"]
    offs = st["off"].tolist()

    def places(i, first, last):
        pos = torch.arange(first, last, device="cuda")
        return st["table"][i].long()[pos // bs] * bs + pos % bs

    if kind in ("attn", "attn_quant"):
        out = torch.zeros(st["total"], hq, d, dtype=torch.float64, device="cuda")
        lse = torch.zeros(st["total"], hq, dtype=torch.float64, device="cuda")
        src = st["kv"].view(2, -1, hkv, d) if kind == "attn" else st["rows"].view(2, -1, st["rows"].shape[-1])
        for i, (s, a) in enumerate(zip(seq, new)):
            if a == 0:
                continue
            at = places(i, 0, s)
            both = [src[p][at] for p in range(2)]
            both = [x.double() if kind == "attn" else exact_rows(x, hkv, d).view(s, hkv, d) for x in both]
            limit = torch.arange(s - a, s, device="cuda")
            hidden = torch.arange(s, device="cuda")[None] > limit[:, None]
            for h in range(hkv):
                for x in range(h * g, h * g + g):
                    logit = st["q"][offs[i]:offs[i + 1], x].double() @ both[0][:, h].T / math.sqrt(d)
                    logit[hidden] = -math.inf
                    one = torch.logsumexp(logit, -1)
                    lse[offs[i]:offs[i + 1], x] = one
                    out[offs[i]:offs[i + 1], x] = torch.exp(logit - one[:, None]) @ both[1][:, h]
        return out, lse
    if kind == "read":
        out = torch.zeros(2, case["l"], st["total"], hkv, d, dtype=torch.float64, device="cuda")
        for i, (s, a) in enumerate(zip(seq, new)):
            at = places(i, s - a, s)
            for la in range(case["l"]):
                for p in range(2):
                    out[p, la, offs[i]:offs[i + 1]] = exact_rows(st["rows"][la, p].flatten(0, 1)[at], hkv, d).view(a, hkv, d)
        return out[0], out[1]
    layers, _, nb = st["rows"].shape[:3]
    values = torch.zeros(layers, 2, nb * bs, hkv * d, dtype=torch.float64, device="cuda")
    scales = torch.full((layers, 2, nb * bs, hkv * d // GROUP), 2.0 ** -127, dtype=torch.float64, device="cuda")
    for i, (s, a) in enumerate(zip(seq, new)):
        at = places(i, s - a, s)
        for la in range(layers):
            for p, x in enumerate((st["k"], st["v"])):
                y = x[la, offs[i]:offs[i + 1]].double().view(a, -1, GROUP)
                top = y.abs().amax(-1, keepdim=True)
                e = torch.ceil(torch.log2(top / E4M3_MAX))            # settled below where log2 is near a whole number
                e = torch.where(top > E4M3_MAX * exact_pow2(e), e + 1, e)
                e = torch.where(top <= E4M3_MAX * exact_pow2(e - 1), e - 1, e).clamp(min=-127)
                z = y * exact_pow2(-e)
                step = exact_pow2(torch.frexp(z.abs().clamp(min=2.0 ** -6))[1] - 4)
                values[la, p, at] = (torch.round(z / step) * step).view(a, -1)
                scales[la, p, at] = exact_pow2(e).view(a, -1)
    return {"values": values.view(layers, 2, nb, bs, -1), "scales": scales.view(layers, 2, nb, bs, -1)}
