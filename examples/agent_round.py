"""Rounds of an agent loop on a device-resident cache, as a serving engine would drive them: each
round appends an observation and an action to every session, attends the whole chunk over the cache
layer by layer (paged_chunk_attention: output for the model, lse for the eviction), and evicts each
session to its budget with that lse (EvictionPipeline.step).  With ``quant`` the cache is held in 8
bits (in 4 with ``bits`` 4): rows are quantised as they are appended, attention reads them as they are,
and the scoring reads its keys back.  With ``rotate`` queries and keys are rotated by their positions on
the way into the cache (write_rotated); positions go on counting where evicted sessions got shorter.

The model is stood in for by a random projection of the attention output, so that every layer's
queries, keys and values depend on the layer before.

    python examples/agent_round.py [--quant [--bits 4]] [--rotate] [--rounds N] [--sessions N] [--layers N]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from actkv_open_b200.config import EvictionConfig                                        # noqa: E402
from actkv_open_b200.engine import DevicePagedCache, EvictionPipeline, QuantPagedCache   # noqa: E402
from actkv_open_b200.kernels.quant_cache import quantize_write                           # noqa: E402
from actkv_open_b200.kernels.rotary import rotary_table                                  # noqa: E402


def run(quant=False, sessions=4, layers=4, hq=32, hkv=8, d=128, observe=256, act=32, rounds=3, budget=0.25,
        dtype=torch.bfloat16, seed=0, device="cuda", bits=8, rotate=False):
    """Runs the rounds; returns per round the model's last hidden state [T, Hq * D], the lse of the
    action tokens [L, sum(act), Hq] and the sessions' lengths after eviction."""
    gen = torch.Generator(device=device).manual_seed(seed)
    new = observe + act
    most = -(-(new * rounds + 16) // 16) * 16
    blocks = sessions * (most // 16) + 4
    kind = dict(dtype=dtype, device=device)
    cache = QuantPagedCache(blocks, 16, hkv, d, layers, sessions, most, bits=bits, **kind) if quant else \
        DevicePagedCache(blocks, 16, hkv, d, layers, sessions, most, **kind)
    cache.set_state([[] for _ in range(sessions)], [0] * sessions, list(range(blocks)), protected=4)
    pipe = EvictionPipeline(cache, EvictionConfig())
    off = torch.arange(sessions + 1, dtype=torch.int32, device=device) * new
    rows = sessions * new
    is_action = torch.zeros(sessions, new, dtype=torch.bool, device=device)
    is_action[:, observe:] = True
    is_action = is_action.flatten()
    w_q = torch.randn(hq * d, hq * d, generator=gen, device=device).to(dtype) / (hq * d) ** 0.5
    w_kv = torch.randn(hq * d, 2 * hkv * d, generator=gen, device=device).to(dtype) / (hq * d) ** 0.5
    results = []
    angles = rotary_table(d, rounds * new, device=device) if rotate else None
    for turn in range(rounds):
        x = torch.randn(rows, hq * d, generator=gen, device=device).to(dtype)
        # room for every session's new tokens in all layers; each layer's rows follow as it runs
        cache.reserve([new] * sessions)
        positions = (turn * new + torch.arange(new, dtype=torch.int32, device=device)).repeat(sessions)
        q_act = torch.empty(layers, sessions * act, hq, d, dtype=dtype, device=device)
        lse_act = torch.empty(layers, sessions * act, hq, device=device)
        for layer in range(layers):
            q = (x @ w_q).view(rows, hq, d)
            kv = (x @ w_kv).view(rows, 2, hkv, d)
            if rotate:
                q = cache.write_rotated(layer, q, kv[:, 0], kv[:, 1], positions, angles, off)
            else:
                write_rows(cache, layer, kv[:, 0], kv[:, 1], off)
            out, lse = cache.chunk_attention(layer, q, off)
            q_act[layer], lse_act[layer] = q[is_action], lse[is_action]
            x = x + out.view(rows, hq * d)
            x = x / x.float().pow(2).mean(-1, keepdim=True).sqrt().to(dtype)
        lens = cache.seq_used[:sessions].tolist()
        pipe.set_round([act] * sessions, [int(n * budget) for n in lens])
        pipe.step(q_act, lse_act)
        results.append((x, lse_act, cache.seq_used[:sessions].tolist()))
    return results


def write_rows(cache, layer, k, v, off):
    """One layer's new rows into the slots that were set aside (the newest tokens)."""
    R = off.shape[0] - 1
    table, seq = cache.block_table[:R], cache.seq_used[:R]
    if isinstance(cache, QuantPagedCache):
        quantize_write(k[None], v[None], off, cache.rows[layer:layer + 1], table, seq, bits=cache.bits)
        return
    new = off[1:] - off[:-1]
    t = torch.arange(k.shape[0], device=k.device, dtype=torch.int32)
    r = torch.bucketize(t, off[1:], right=True)
    pos = (seq - new)[r] + t - off[:-1][r]
    slot = table[r, (pos // cache.block_size).long()].long() * cache.block_size + pos % cache.block_size
    flat = cache.kv[layer].flatten(1, 2)
    flat[0, slot], flat[1, slot] = k, v


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--quant", action="store_true", help="hold the cache in 8 bits")
    ap.add_argument("--bits", type=int, default=8, choices=[8, 4], help="... or in 4")
    ap.add_argument("--rotate", action="store_true", help="rotate queries and keys by their positions")
    ap.add_argument("--rounds", type=int, default=3)
    ap.add_argument("--sessions", type=int, default=4)
    ap.add_argument("--layers", type=int, default=4)
    args = ap.parse_args()
    for i, (x, lse, lens) in enumerate(run(args.quant, args.sessions, args.layers, rounds=args.rounds, bits=args.bits,
                                               rotate=args.rotate)):
        print(f"round {i}: hidden rms {x.float().pow(2).mean().sqrt():.4f}, mean lse of the action tokens "
              f"{lse.mean():.4f}, sessions now {lens} tokens")


if __name__ == "__main__":
    main()
