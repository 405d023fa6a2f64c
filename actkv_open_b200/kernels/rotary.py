"""The position rotation of new queries and keys on their way into a paged cache.  (The reference's caller
rotates before append, actkv/paged.py:67-85 copies keys as they come.)

A pair (x, y) of a head at position p becomes (x c - y s, y c + x s) with c, s the cosine and sine of
p * base^(-2 i / rot): dims (i, i + rot / 2), or (2 i, 2 i + 1) when ``interleaved``; dims from ``rot`` on
stay.  Positions are an input of their own: an evicted session is shorter than its next position, and its
cached keys keep the positions they came with.
"""
from __future__ import annotations

import torch

from .. import _native as N
from .quant_cache import QUANT_GROUP

_I32, _F32, _U8 = torch.int32, torch.float32, torch.uint8


def rotary_table(rot: int, max_positions: int, base: float = 10000.0, frequencies=None, device="cuda") -> torch.Tensor:
    """The angles of positions 0 .. max_positions - 1: fp32 [max_positions, rot], rot / 2 cosines, then as many
    sines, taken in 64 bits.  ``frequencies`` [rot / 2] replaces base^(-2 i / rot) (scaled or mixed ones)."""
    assert rot > 0 and rot % 2 == 0 and max_positions > 0, "rot is even; at least one position"
    if frequencies is None:
        frequencies = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    freq = torch.as_tensor(frequencies).to(device=device, dtype=torch.float64)
    assert freq.shape == (rot // 2,), "frequencies [rot / 2]"
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def rotate_write(q, k_new, v_new, positions, angles, tok_off, cache, block_table, seq_used, q_out=None,
                 interleaved: bool = False, bits: int | None = None):
    """Rotate new queries and keys, and write the keys and the values into the cache, every layer in one
    launch; returns the rotated queries (None without ``q``).

    q [L, T, Hq, D] (or None) and k_new / v_new [L, T, Hkv, D] of one dtype (bf16, fp16 or fp32) hold the
    sessions' new tokens packed, session r owning tok_off[r]:tok_off[r+1] (int32 [R+1], T = tok_off[R]);
    they become the newest tok_off[r+1] - tok_off[r] of its seq_used[r] tokens, whose blocks block_table
    [R, MB] holds.  positions int32 [T]; ``angles`` fp32 [P, rot] as ``rotary_table`` gives them.  ``cache`` is
    [L, 2, NB, BS, Hkv, D] of that dtype, or with ``bits`` 8 or 4 the rows [L, 2, NB, BS, row_bytes] of such a
    cache, quantised from the 32-bit results.  ``q_out`` may be q itself.

    A token whose position the angles do not have is left alone, one that the tables do not hold is not
    written into the cache (device status BAD_INDEX, both); so is a token of no session, unflagged.
    """
    dev = k_new.device
    N.require_cuda(k_new, v_new, q, positions, angles, tok_off, cache, block_table, seq_used, q_out)
    shape = k_new.shape
    assert len(shape) == 4 and shape == v_new.shape and k_new.dtype is v_new.dtype, \
        "k_new / v_new are [L, T, Hkv, D] of one dtype"
    L, t_n, hkv, d = shape
    k_l, k_t, k_h, k_1 = k_new.stride()
    v_l, v_t, v_h, v_1 = v_new.stride()
    assert k_1 == 1 and v_1 == 1
    hq = 0
    qs = os = (0, 0, 0)
    if q is not None:
        assert q.dim() == 4 and q.shape[0] == L and q.shape[1] == t_n and q.shape[3] == d and \
            q.dtype is k_new.dtype, "q is [L, T, Hq, D] of k_new's dtype"
        hq = q.shape[2]
        if q_out is None:
            q_out = q.new_empty(q.shape)
        assert q_out.shape == q.shape and q_out.dtype is q.dtype
        *qs, q_1 = q.stride()
        *os, o_1 = q_out.stride()
        assert q_1 == 1 and o_1 == 1
    else:
        assert q_out is None, "q_out without q"
    assert positions.dtype is _I32 and positions.shape == (t_n,) and positions.is_contiguous(), "positions int32 [T]"
    assert angles.dim() == 2 and angles.dtype is _F32 and angles.stride(1) == 1, "angles fp32 [P, rot]"
    places, rot = angles.shape
    assert 0 < rot <= d and rot % 2 == 0, "rot is even and at most D"
    if bits is None:
        assert cache.dim() == 6 and cache.dtype is k_new.dtype and cache.shape[0] == L and cache.shape[1] == 2 and \
            cache.shape[4] == hkv and cache.shape[5] == d and cache.stride(5) == 1, \
            "the cache is [L, 2, NB, BS, Hkv, D] of k_new's dtype"
        c_l, c_kv, c_b, c_s, c_h = cache.stride()[:5]
    else:
        if bits not in (8, 4):
            raise ValueError(f"bits {bits}: the cache holds its rows in 8 or 4")
        assert cache.dim() == 5 and cache.dtype is _U8 and cache.shape[0] == L and cache.shape[1] == 2 and \
            cache.stride(4) == 1, "rows is [L, 2, NB, BS, row_bytes] uint8"
        assert d % QUANT_GROUP == 0 and cache.shape[4] >= hkv * (d * bits // 8 + d // QUANT_GROUP), \
            "rows are too short for these heads"
        c_l, c_kv, c_b, c_s = cache.stride()[:4]
        c_h = 0
    nb, bs = cache.shape[2], cache.shape[3]
    assert tok_off.dtype is _I32 and seq_used.dtype is _I32 and block_table.dtype is _I32
    assert tok_off.is_contiguous() and seq_used.is_contiguous() and block_table.stride(1) == 1
    r_n = len(seq_used)
    assert len(tok_off) == r_n + 1 and len(block_table) == r_n, "tok_off [R + 1], block_table [R, MB], seq_used [R]"
    code = N.load().actkv_rotate_write(
        N.ptr(q), *qs, N.ptr(q_out), *os, k_new.data_ptr(), k_l, k_t, k_h, v_new.data_ptr(), v_l, v_t, v_h,
        N.dtype_code(k_new), positions.data_ptr(), angles.data_ptr(), angles.stride(0), places, rot, interleaved,
        tok_off.data_ptr(), t_n, cache.data_ptr(), bits or 0, c_l, c_kv, c_b, c_s, c_h, block_table.data_ptr(),
        block_table.stride(0), seq_used.data_ptr(), r_n, L, block_table.size(1), nb, bs, hq, hkv, d,
        N.status_word(dev).data_ptr(), N.stream_ptr(dev))
    if code:
        N.check(code, "rotate_write")
    return q_out
