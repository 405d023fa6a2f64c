"""Attention of each session's newest tokens over a paged KV cache, with its log-sum-exp: the step
before scoring in an agent loop (the reference leaves it to its attention backend and takes the lse,
actkv/kernels/lse_attn.py:42-60).

A session's chunk (an observation, a drafted run, a prompt piece, or a single token) is appended to
the cache first; its queries then attend over everything the session holds, causally within the
chunk.  bf16 / fp16 caches with head_dim 64 or 128 run on the tensor cores, the rest on CUDA cores.
"""
from __future__ import annotations

import torch

from .. import _native as N

_PATHS = {"auto": N.PATH_AUTO, "simt": N.PATH_SIMT, "tcgen05": N.PATH_TCGEN05}
_ws_bytes = {}


def chunk_workspace(device) -> torch.Tensor:
    """The workspace of the chunk attention calls on ``device``: any sizes, kept from call to call;
    calls that may overlap on the GPU (other streams) need one each."""
    dev = torch.device(device)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    if idx not in _ws_bytes:
        with torch.cuda.device(idx):
            _ws_bytes[idx] = int(N.load().actkv_chunk_workspace_bytes())
    return N.workspace(_ws_bytes[idx], torch.device("cuda", idx))


_I32, _F32 = torch.int32, torch.float32


def _check(q, q_off, cache, block_table, seq_used, out, lse, workspace):
    """Checks shared by the two caches; returns (device, sessions, out, lse, workspace)."""
    dev = q.device
    if not q.is_cuda or q_off.device != dev or cache.device != dev or block_table.device != dev or \
            seq_used.device != dev:
        N.require_cuda(q, q_off, cache, block_table, seq_used)
    assert q.dim() == 3 and q.stride(2) == 1, "q is [T, Hq, D] with contiguous rows"
    assert q_off.dtype is _I32 and seq_used.dtype is _I32 and block_table.dtype is _I32
    assert block_table.stride(1) == 1 and q_off.is_contiguous() and seq_used.is_contiguous()
    r_n = block_table.shape[0]
    assert q_off.shape == (r_n + 1,) and seq_used.shape == (r_n,), "q_off [R + 1], block_table [R, MB], seq_used [R]"
    if out is None:
        out = q.new_empty(q.shape)
    else:
        assert out.device == dev and out.shape == q.shape and out.dtype is q.dtype and out.stride(2) == 1
    if lse is None:
        lse = q.new_empty(q.shape[:2], dtype=_F32)
    else:
        assert lse.device == dev and lse.shape == q.shape[:2] and lse.dtype is _F32 and lse.stride(1) == 1
    if workspace is None:
        workspace = chunk_workspace(dev)
    else:
        assert workspace.device == dev and workspace.is_contiguous()
    return dev, r_n, out, lse, workspace


def paged_chunk_attention(q, q_off, kv, block_table, seq_used, scale=None, out=None, lse=None, workspace=None,
                          path: str = "auto"):
    """Attention of every session's newest tokens over its paged cache: (out [T, Hq, D] of q's dtype,
    lse [T, Hq] fp32).

    q [T, Hq, D] holds the sessions' queries packed, session r owning rows q_off[r]:q_off[r+1]
    (int32 [R+1], T = q_off[R]); kv [2, NB, BS, Hkv, D] is one layer's cache, of q's dtype;
    block_table [R, MB] and seq_used [R] int32.  The queries belong to the newest
    A = q_off[r+1] - q_off[r] of the seq_used[r] tokens, already in the cache: query j sees the
    first seq_used[r] - A + j + 1 of them.  A query that sees none gets out 0, lse -inf; a session
    may have no queries; one whose offsets leave the T rows is left alone (device status BAD_INDEX).
    ``scale`` defaults to D ** -0.5; ``workspace`` to a new
    ``chunk_workspace`` (a loop keeps one).  ``path``: "auto", or "tcgen05" / "simt" to force the
    tensor cores (NotImplementedError where they do not apply) or the CUDA cores.

    16-bit calls round the softmax's p and the result to the cache's type each.  For single tokens
    ``lse_attn.paged_decode_attention`` is the more exact (p in two 16-bit terms, out in fp32) where it applies (1, 2,
    4 or 8 query heads per KV head); this call takes any number of tokens, gives q's dtype and shares a batch with chunks.
    """
    dev, r_n, out, lse, workspace = _check(q, q_off, kv, block_table, seq_used, out, lse, workspace)
    t_n, hq, d = q.shape
    _2, nb, bs, hkv, kd = kv.shape
    assert _2 == 2 and kd == d, "kv is [2, NB, BS, Hkv, D]"
    assert kv.dtype is q.dtype, "q and the cache must share a dtype"
    assert hq % hkv == 0
    s_kv, s_b, s_s, s_h, s_d = kv.stride()
    assert s_d == 1
    q_t, q_h, _1 = q.stride()
    o_t, o_h, _1 = out.stride()
    code = N.load().actkv_chunk_attention(
        q.data_ptr(), N.dtype_code(q), q_t, q_h, q_off.data_ptr(), t_n, kv.data_ptr(), s_kv, s_b, s_s, s_h,
        block_table.data_ptr(), block_table.stride(0), seq_used.data_ptr(), out.data_ptr(), o_t, o_h, lse.data_ptr(),
        lse.stride(0), r_n, block_table.size(1), nb, bs, hq, hkv, d, d ** -0.5 if scale is None else float(scale),
        _PATHS[path], workspace.data_ptr(), workspace.nbytes, N.status_word(dev).data_ptr(), N.stream_ptr(dev))
    if code:
        N.check(code, "paged_chunk_attention")
    return out, lse
