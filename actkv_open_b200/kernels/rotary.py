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
_pack = N.words("actkv_rotate_write")


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
                 interleaved: bool = False, bits: int | None = None, fits=None):
    """Rotate new queries and keys, and write the keys and the values into the cache, every layer in one
    launch; returns the rotated queries (None without ``q``).

    q [L, T, Hq, D] (or None) and k_new / v_new [L, T, Hkv, D] of one dtype (bf16, fp16 or fp32) hold the
    sessions' new tokens packed, session r owning tok_off[r]:tok_off[r+1] (int32 [R+1], T = tok_off[R]);
    they become the newest tok_off[r+1] - tok_off[r] of its seq_used[r] tokens, whose blocks block_table
    [R, MB] holds.  positions int32 [T]; ``angles`` fp32 [P, rot] as ``rotary_table`` gives them.  ``cache`` is
    [L, 2, NB, BS, Hkv, D] of that dtype, or with ``bits`` 8 or 4 the rows [L, 2, NB, BS, row_bytes] of such a
    cache, quantised from the 32-bit results.  ``q_out`` may be q itself.  ``fits`` (int32 [R]): of sessions with 0
    nothing is written into the cache (those that an allocation had no room for).

    A token whose position the angles do not have is left alone, one that the tables do not hold is not
    written into the cache (device status BAD_INDEX, both); so is a token of no session, unflagged.
    """
    # (each look at a tensor costs a fraction of a microsecond, and a call of one token's rows little more than they do)
    dev = k_new.device
    if not k_new.is_cuda or v_new.device != dev or positions.device != dev or angles.device != dev or \
            tok_off.device != dev or cache.device != dev or block_table.device != dev or seq_used.device != dev or \
            q is not None and q.device != dev or q_out is not None and q_out.device != dev or \
            fits is not None and fits.device != dev:
        N.require_cuda(k_new, v_new, q, positions, angles, tok_off, cache, block_table, seq_used, q_out, fits)
    shape, dtype = k_new.shape, k_new.dtype
    assert len(shape) == 4 and shape == v_new.shape and dtype is v_new.dtype, "k_new / v_new are [L, T, Hkv, D] of one dtype"
    L, t_n, hkv, d = shape
    k_l, k_t, k_h, k_1 = k_new.stride()
    v_l, v_t, v_h, v_1 = v_new.stride()
    assert k_1 == 1 and v_1 == 1
    if q is None:
        assert q_out is None, "q_out without q"
        hq = q_p = o_p = 0
        q_l = q_t = q_h = o_l = o_t = o_h = 0
    else:
        q_shape = q.shape
        assert len(q_shape) == 4 and q.dtype is dtype, "q is [L, T, Hq, D] of k_new's dtype"
        q_n, q_tn, hq, q_d = q_shape
        assert q_n == L and q_tn == t_n and q_d == d, "q is [L, T, Hq, D] of k_new's dtype"
        q_l, q_t, q_h, q_1 = q.stride()
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            assert q_out.shape == q_shape and q_out.dtype is dtype
        o_l, o_t, o_h, o_1 = q_out.stride()
        assert q_1 == 1 and o_1 == 1
        q_p, o_p = q.data_ptr(), q_out.data_ptr()
    assert positions.dtype is _I32 and positions.shape == (t_n,) and positions.is_contiguous(), "positions int32 [T]"
    a_s, a_1 = angles.stride()
    assert angles.dtype is _F32 and a_1 == 1, "angles fp32 [P, rot]"
    places, rot = angles.shape
    assert 0 < rot <= d and rot % 2 == 0, "rot is even and at most D"
    if bits is None:
        c_shape = cache.shape
        assert len(c_shape) == 6 and cache.dtype is dtype, "the cache is [L, 2, NB, BS, Hkv, D] of k_new's dtype"
        c_n, c_2, nb, bs, c_hn, c_d = c_shape
        c_l, c_kv, c_b, c_s, c_h, c_1 = cache.stride()
        assert c_n == L and c_2 == 2 and c_hn == hkv and c_d == d and c_1 == 1, \
            "the cache is [L, 2, NB, BS, Hkv, D] of k_new's dtype"
    else:
        if bits not in (8, 4):
            raise ValueError(f"bits {bits}: the cache holds its rows in 8 or 4")
        c_shape = cache.shape
        assert len(c_shape) == 5 and cache.dtype is _U8, "rows is [L, 2, NB, BS, row_bytes] uint8"
        c_n, c_2, nb, bs, row = c_shape
        c_l, c_kv, c_b, c_s, c_1 = cache.stride()
        c_h = 0
        assert c_n == L and c_2 == 2 and c_1 == 1, "rows is [L, 2, NB, BS, row_bytes] uint8"
        assert d % QUANT_GROUP == 0 and row >= hkv * (d * bits // 8 + d // QUANT_GROUP), "rows are too short for these heads"
    assert tok_off.dtype is _I32 and seq_used.dtype is _I32 and block_table.dtype is _I32
    b_r, b_1 = block_table.stride()
    assert b_1 == 1 and tok_off.is_contiguous() and seq_used.is_contiguous()
    r_n, mb = block_table.shape
    assert tok_off.shape == (r_n + 1,) and seq_used.shape == (r_n,), "tok_off [R + 1], block_table [R, MB], seq_used [R]"
    assert fits is None or fits.dtype is _I32 and fits.shape == (r_n,) and fits.is_contiguous(), "fits int32 [R]"
    code = N.load().actkv_rotate_write_fits(N.ptr(fits), _pack(
        q_p, q_l, q_t, q_h, o_p, o_l, o_t, o_h, k_new.data_ptr(), k_l, k_t, k_h, v_new.data_ptr(), v_l, v_t, v_h,
        N.dtype_code(k_new), positions.data_ptr(), angles.data_ptr(), a_s, places, rot, interleaved, tok_off.data_ptr(),
        t_n, cache.data_ptr(), bits or 0, c_l, c_kv, c_b, c_s, c_h, block_table.data_ptr(), b_r, seq_used.data_ptr(),
        r_n, L, mb, nb, bs, hq, hkv, d, N.status_word(dev).data_ptr(), N.stream_ptr(dev)))
    if code:
        N.check(code, "rotate_write")
    return q_out
