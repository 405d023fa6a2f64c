"""A paged KV cache in 8 bits: quantising rows as they are written, reading them back, and attention
over it.  (The reference has no counterpart; its cache is 16-bit, actkv/paged.py:54.)

``rows`` [L, 2, NB, BS, row_bytes] uint8 (one layer for attention: [2, NB, BS, row_bytes]).  A token's
row of one plane is Hkv * D e4m3 values, then Hkv * D / 32 scale bytes, one per 32 values along D
(value = e4m3 * 2^(byte - 127); byte 255 is NaN), then padding.  The scale is the smallest power of
two with max|x| <= 448 * scale, so values are exact in bf16 and err by at most 1/16 of themselves
(or 2^-10 of the scale's unit, for values that small).  Rows move as bytes: append, release and
compaction treat such a cache like any other (``engine.QuantPagedCache``).
"""
from __future__ import annotations

import torch

from .. import _native as N
from .chunk_attn import _PATHS, _check

QUANT_GROUP = 32


def quant_row_bytes(n_kv_heads: int, head_dim: int) -> int:
    """Bytes of a token's row of one plane: values and scales, padded to whole 64-byte pieces (so
    that every head's values start on one)."""
    assert head_dim % QUANT_GROUP == 0, f"head_dim must be a multiple of {QUANT_GROUP}"
    return -(-n_kv_heads * (head_dim + head_dim // QUANT_GROUP) // 64) * 64


def _move_args(x, rows, tok_off, block_table, seq_used):
    assert rows.dim() == 5 and rows.shape[1] == 2 and rows.dtype == torch.uint8, "rows is [L, 2, NB, BS, row_bytes] uint8"
    assert rows.stride(4) == 1 and block_table.stride(1) == 1
    assert tok_off.dtype == torch.int32 and seq_used.dtype == torch.int32 and block_table.dtype == torch.int32
    assert tok_off.is_contiguous() and seq_used.is_contiguous()
    r_n = seq_used.shape[0]
    assert tok_off.shape[0] == r_n + 1 and block_table.shape[0] == r_n, \
        "tok_off [R + 1], block_table [R, MB], seq_used [R]"
    L, t_n, hkv, d = x.shape
    assert rows.shape[0] == L, "rows and the tokens must have the same layers"
    assert rows.shape[4] >= hkv * (d + d // QUANT_GROUP), "rows are too short for these heads"
    s_l, s_kv, s_b, s_s, _ = rows.stride()
    return ((tok_off.data_ptr(), t_n, rows.data_ptr(), s_l, s_kv, s_b, s_s, block_table.data_ptr(),
             block_table.stride(0), seq_used.data_ptr(), r_n, L, block_table.shape[1], rows.shape[2], rows.shape[3],
             hkv, d))


def quantize_write(k_new, v_new, tok_off, rows, block_table, seq_used):
    """Quantise new K / V rows into the cache, every layer in one launch.  In place; returns ``rows``.

    k_new / v_new [L, T, Hkv, D] (bf16, fp16 or fp32) hold the sessions' new tokens packed, session r
    owning tok_off[r]:tok_off[r+1] (int32 [R+1], T = tok_off[R]); they become the newest
    tok_off[r+1] - tok_off[r] of its seq_used[r] tokens, whose blocks block_table [R, MB] holds.
    """
    dev = k_new.device
    if dev.type != "cuda" or not (v_new.device == tok_off.device == rows.device == block_table.device ==
                                  seq_used.device == dev):
        N.require_cuda(k_new, v_new, tok_off, rows, block_table, seq_used)
    assert k_new.dim() == 4 and k_new.shape == v_new.shape and k_new.dtype == v_new.dtype, \
        "k_new / v_new are [L, T, Hkv, D] of one dtype"
    ks, vs = k_new.stride(), v_new.stride()
    assert ks[3] == 1 and vs[3] == 1
    N.check(N.load().actkv_quantize_write(
        k_new.data_ptr(), v_new.data_ptr(), N.dtype_code(k_new), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        *_move_args(k_new, rows, tok_off, block_table, seq_used), N.status_word(dev).data_ptr(), N.stream_ptr(dev)),
        "quantize_write")
    return rows


def dequantize_read(rows, n_kv_heads, head_dim, tok_off, block_table, seq_used, n_tokens, dtype=torch.bfloat16,
                    k_out=None, v_out=None, planes: str = "kv"):
    """Read each session's newest tok_off[r+1] - tok_off[r] tokens back: (k, v) [L, n_tokens, Hkv, D],
    packed as ``quantize_write`` takes them (n_tokens = tok_off[R]), rounded to ``dtype`` (fp16:
    values past its range become its largest).

    ``planes`` "k" or "v" reads one of the two (the other comes back as None).
    """
    if planes not in ("kv", "k", "v"):
        raise ValueError(planes)
    dev = rows.device
    if dev.type != "cuda" or not (tok_off.device == block_table.device == seq_used.device == dev) or \
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
        if x is not None:
            assert tuple(x.shape) == shape and x.dtype == some.dtype and x.stride(3) == 1
        strides += [0, 0, 0] if x is None else x.stride()[:3]
    N.check(N.load().actkv_dequantize_read(
        N.ptr(k_out), N.ptr(v_out), N.dtype_code(some), *strides,
        *_move_args(some, rows, tok_off, block_table, seq_used), N.status_word(dev).data_ptr(), N.stream_ptr(dev)),
        "dequantize_read")
    return k_out, v_out


def paged_chunk_attention_quant(q, q_off, rows, n_kv_heads, block_table, seq_used, scale=None, out=None, lse=None,
                                workspace=None, path: str = "auto"):
    """``paged_chunk_attention`` over one layer of the 8-bit cache, rows [2, NB, BS, row_bytes]: the
    keys and values are what ``dequantize_read`` gives in q's dtype."""
    dev, out, lse, workspace = _check(q, q_off, rows, block_table, seq_used, out, lse, workspace)
    t_n, hq, d = q.shape
    assert rows.dim() == 4 and rows.shape[0] == 2 and rows.dtype == torch.uint8, "rows is [2, NB, BS, row_bytes] uint8"
    assert hq % n_kv_heads == 0
    assert rows.shape[3] >= n_kv_heads * (d + d // QUANT_GROUP), "rows are too short for these heads"
    s_kv, s_b, s_s, s_1 = rows.stride()
    assert s_1 == 1
    N.check(N.load().actkv_chunk_attention_quant(
        q.data_ptr(), N.dtype_code(q), q.stride(0), q.stride(1), q_off.data_ptr(), t_n, rows.data_ptr(), s_kv, s_b, s_s,
        block_table.data_ptr(), block_table.stride(0), seq_used.data_ptr(), out.data_ptr(), out.stride(0),
        out.stride(1), lse.data_ptr(), lse.stride(0), seq_used.shape[0], block_table.shape[1], rows.shape[1],
        rows.shape[2], hq, n_kv_heads, d, d ** -0.5 if scale is None else float(scale), _PATHS[path],
        workspace.data_ptr(), workspace.numel(), N.status_word(dev).data_ptr(), N.stream_ptr(dev)),
        "paged_chunk_attention_quant")
    return out, lse
