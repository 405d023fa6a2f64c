"""A paged KV cache in 8 or 4 bits: quantising rows as they are written, reading them back, and attention
over it.  (The reference has no counterpart; its cache is 16-bit, actkv/paged.py:54.)

``rows`` [L, 2, NB, BS, row_bytes] uint8 (one layer for attention: [2, NB, BS, row_bytes]).  A token's
row of one plane is Hkv * D e4m3 values, then Hkv * D / 32 scale bytes, one per 32 values along D
(value = e4m3 * 2^(byte - 127); byte 255 is NaN), then padding.  The scale is the smallest power of
two with max|x| <= 448 * scale, so values are exact in bf16 and err by at most 1/16 of themselves
(or 2^-10 of the scale's unit, for values that small).  Rows move as bytes: append, release and
compaction treat such a cache like any other (``engine.QuantPagedCache``).

With ``bits`` 4 a row is Hkv * D / 2 bytes of e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives), then the scale bytes (from 253 on: NaN), then padding.  The scale is the smallest power of
two, up to 2^125, with max|x| <= 7 * scale (between 6 and 7 the largest value becomes 6): values err by
at most 1 / 7 of the largest of their 32, about 0.11 of themselves in the mean square.  Value
32 g + 4 p + j of a head (p < 8, j < 4) is in the head's byte p * D / 16 + 2 g + j // 2, the low half for
even j.
"""
from __future__ import annotations

import torch

from .. import _native as N
from .chunk_attn import _PATHS, _check

QUANT_GROUP = 32


def _bits(bits) -> bool:
    """Whether it is the 4-bit cache."""
    if bits != 8 and bits != 4:
        raise ValueError(f"bits {bits}: the cache holds its rows in 8 or 4")
    return bits == 4


def quant_row_bytes(n_kv_heads: int, head_dim: int, bits: int = 8) -> int:
    """Bytes of a token's row of one plane: values and scales, padded to whole 64-byte pieces (so
    that every head's values start on one); in 4 bits, where a head of 64 has half of that, to 32-byte ones."""
    assert head_dim % QUANT_GROUP == 0, f"head_dim must be a multiple of {QUANT_GROUP}"
    pad = 32 if _bits(bits) else 64
    return -(-n_kv_heads * (head_dim * bits // 8 + head_dim // QUANT_GROUP) // pad) * pad


_I32, _U8 = torch.int32, torch.uint8
_pack_write, _pack_read, _pack_attend = (N.words("actkv_" + x) for x in ("quantize_write", "dequantize_read", "chunk_attention_quant"))


def _tables(dev, L, t_n, hkv, d, rows, tok_off, block_table, seq_used, bits):
    """The checks and the arguments that writing and reading share."""
    assert rows.dim() == 5 and rows.dtype is _U8, "rows is [L, 2, NB, BS, row_bytes] uint8"
    rl, _2, nb, bs, row = rows.shape
    assert _2 == 2 and rl == L, "rows and the tokens must have the same layers"
    assert row >= hkv * (d * bits // 8 + d // QUANT_GROUP), "rows are too short for these heads"
    s_l, s_kv, s_b, s_s, s_1 = rows.stride()
    assert s_1 == 1 and block_table.stride(1) == 1
    assert tok_off.dtype is _I32 and seq_used.dtype is _I32 and block_table.dtype is _I32
    assert tok_off.is_contiguous() and seq_used.is_contiguous()
    r_n, mb = block_table.shape
    assert tok_off.shape == (r_n + 1,) and seq_used.shape == (r_n,), "tok_off [R + 1], block_table [R, MB], seq_used [R]"
    return (tok_off.data_ptr(), t_n, rows.data_ptr(), s_l, s_kv, s_b, s_s, block_table.data_ptr(),
            block_table.stride(0), seq_used.data_ptr(), r_n, L, mb, nb, bs, hkv, d,
            N.status_word(dev).data_ptr(), N.stream_ptr(dev))


def quantize_write(k_new, v_new, tok_off, rows, block_table, seq_used, bits: int = 8):
    """Quantise new K / V rows into the cache, every layer in one launch.  In place; returns ``rows``.
    (``rotary.rotate_write`` does the same with the keys' position rotation on the way.)

    k_new / v_new [L, T, Hkv, D] (bf16, fp16 or fp32) hold the sessions' new tokens packed, session r
    owning tok_off[r]:tok_off[r+1] (int32 [R+1], T = tok_off[R]); they become the newest
    tok_off[r+1] - tok_off[r] of its seq_used[r] tokens, whose blocks block_table [R, MB] holds.
    """
    dev = k_new.device
    if not k_new.is_cuda or v_new.device != dev or tok_off.device != dev or rows.device != dev or \
            block_table.device != dev or seq_used.device != dev:
        N.require_cuda(k_new, v_new, tok_off, rows, block_table, seq_used)
    shape = k_new.shape
    assert len(shape) == 4 and shape == v_new.shape and k_new.dtype is v_new.dtype, \
        "k_new / v_new are [L, T, Hkv, D] of one dtype"
    k_l, k_t, k_h, k_1 = k_new.stride()
    v_l, v_t, v_h, v_1 = v_new.stride()
    assert k_1 == 1 and v_1 == 1
    _bits(bits)
    code = N.load().actkv_quantize_write_words(bits, _pack_write(
        k_new.data_ptr(), v_new.data_ptr(), N.dtype_code(k_new), k_l, k_t, k_h, v_l, v_t, v_h,
        *_tables(dev, *shape, rows, tok_off, block_table, seq_used, bits)))
    if code:
        N.check(code, "quantize_write")
    return rows


def dequantize_read(rows, n_kv_heads, head_dim, tok_off, block_table, seq_used, n_tokens, dtype=torch.bfloat16,
                    k_out=None, v_out=None, planes: str = "kv", bits: int = 8):
    """Read each session's newest tok_off[r+1] - tok_off[r] tokens back: (k, v) [L, n_tokens, Hkv, D],
    packed as ``quantize_write`` takes them (n_tokens = tok_off[R]), rounded to ``dtype`` (fp16:
    values past its range become its largest).

    ``planes`` "k" or "v" reads one of the two (the other comes back as None).
    """
    if planes not in ("kv", "k", "v"):
        raise ValueError(planes)
    dev = rows.device
    if not rows.is_cuda or tok_off.device != dev or block_table.device != dev or seq_used.device != dev or \
            k_out is not None or v_out is not None:
        N.require_cuda(rows, tok_off, block_table, seq_used, k_out, v_out)
    shape = (rows.shape[0], n_tokens, n_kv_heads, head_dim)
    if "k" not in planes:
        k_out = None
    elif k_out is None:
        k_out = rows.new_empty(shape, dtype=dtype)
    if "v" not in planes:
        v_out = None
    elif v_out is None:
        v_out = rows.new_empty(shape, dtype=dtype)
    some = k_out if k_out is not None else v_out
    strides = []
    for x in (k_out, v_out):
        if x is None:
            strides += (0, 0, 0)
            continue
        *three, one = x.stride()
        assert x.shape == shape and x.dtype is some.dtype and one == 1
        strides += three
    _bits(bits)
    code = N.load().actkv_dequantize_read_words(bits, _pack_read(
        N.ptr(k_out) or 0, N.ptr(v_out) or 0, N.dtype_code(some), *strides,
        *_tables(dev, *shape, rows, tok_off, block_table, seq_used, bits)))
    if code:
        N.check(code, "dequantize_read")
    return k_out, v_out


def paged_chunk_attention_quant(q, q_off, rows, n_kv_heads, block_table, seq_used, scale=None, out=None, lse=None,
                                workspace=None, path: str = "auto", bits: int = 8):
    """``paged_chunk_attention`` over one layer of the 8- or 4-bit cache, rows [2, NB, BS, row_bytes]:
    the keys and values are what ``dequantize_read`` gives in q's dtype, and each counts by its weight whatever its size
    (over 4 bits, sessions of few rows take longer where value scales differ by more than 2^7 within 32 tokens)."""
    _bits(bits)
    dev, r_n, out, lse, workspace = _check(q, q_off, rows, block_table, seq_used, out, lse, workspace)
    t_n, hq, d = q.shape
    _2, nb, bs, row = rows.shape
    assert _2 == 2 and rows.dtype is _U8, "rows is [2, NB, BS, row_bytes] uint8"
    assert hq % n_kv_heads == 0
    assert row >= n_kv_heads * (d * bits // 8 + d // QUANT_GROUP), "rows are too short for these heads"
    s_kv, s_b, s_s, s_1 = rows.stride()
    assert s_1 == 1
    q_t, q_h, _1 = q.stride()
    o_t, o_h, _1 = out.stride()
    code = N.load().actkv_chunk_attention_quant_words(bits, _pack_attend(
        q.data_ptr(), N.dtype_code(q), q_t, q_h, q_off.data_ptr(), t_n, rows.data_ptr(), s_kv, s_b, s_s,
        block_table.data_ptr(), block_table.stride(0), seq_used.data_ptr(), out.data_ptr(), o_t, o_h, lse.data_ptr(),
        lse.stride(0), r_n, block_table.size(1), nb, bs, hq, n_kv_heads, d,
        d ** -0.5 if scale is None else float(scale), _PATHS[path], workspace.data_ptr(), workspace.nbytes,
        N.status_word(dev).data_ptr(), N.stream_ptr(dev)))
    if code:
        N.check(code, "paged_chunk_attention_quant")
    return out, lse
