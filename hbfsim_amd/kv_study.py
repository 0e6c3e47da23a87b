"""A decode over a paged 8-bit cache whose full blocks live on flash.

    python -m hbfsim_amd.kv_study --seqs 8 --tokens 8192 --steps 24 --count 64

Every step appends a token per sequence, attends to all visible blocks (the
dense step, which also accumulates the blocks' weights) and to the `count`
blocks that their key bounds select, and times what either form reads and
writes of the flash pools with the engine.  Half way the cache is cut down to
`keep` blocks a sequence by accumulated weight.  Keys and values are synthetic:
queries lean towards a few tokens of their sequence, as attention does.

Prints one JSON object: per form the flash accesses, the modeled makespan of a
step and the bytes; how far the selected form's outputs are from the dense
ones; the share of the dense step's attention that the selected blocks hold
before and after the eviction; and the blocks that left.
"""
from __future__ import annotations

import argparse
import json

import numpy as np
import torch

from . import kvcache, workloads
from .engine import Engine

KEY_BASE = 0x2000_0000_0000
PAGE = 16384


def flash_step(engine: Engine, cache: kvcache.KvCache, reads: np.ndarray,
               writes: np.ndarray) -> dict:
    """Modeled time of a step's flash accesses, from idle media."""
    head_bytes = cache.keys[0, 0].numel()
    pool = -(-cache.keys.numel() // PAGE) * PAGE
    base, first, op = workloads.kv_cache_spans(KEY_BASE, KEY_BASE + pool, head_bytes,
                                               cache.kv_heads, reads, writes)
    n = int(first[-1])
    if n == 0:
        return {"accesses": 0, "ms": 0.0, "bytes": 0}
    records = workloads.gpu_span_records(base, first, op, 128, 64_000, 256)
    done = torch.empty(n, dtype=torch.int64, device=records.device)
    engine.reset()
    report = engine.run(records, done)
    return {"accesses": n, "ms": report["makespan_ps"] / 1e9, "bytes": n * 128}


def on_flash(table: np.ndarray, lens: np.ndarray, block_tokens: int, chosen: np.ndarray | None,
             kv_heads: int) -> np.ndarray:
    """(block, kv head) pairs that a step reads from flash: the full blocks
    among `chosen` (logical, [seqs, kv_heads, count]), or all of them."""
    out = []
    for s, n in enumerate(lens):
        full = int(n) // block_tokens
        for h in range(kv_heads):
            picked = np.arange(full) if chosen is None else chosen[s, h]
            picked = picked[(picked >= 0) & (picked < full)]
            out.append(np.stack([table[s, picked], np.full(len(picked), h)], 1))
    return np.concatenate(out)


def run(seqs: int = 8, tokens: int = 8192, steps: int = 24, count: int = 64, keep: int = 256,
        heads: int = 32, kv_heads: int = 8, head_dim: int = 128, seed: int = 0) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    t = 16
    width = -(-(tokens + steps) // t)
    cache = kvcache.KvCache(seqs * width, kv_heads, head_dim, t, dev)
    table = torch.randperm(seqs * width, generator=gen, device=dev).to(torch.int32)
    table = table.view(seqs, width).contiguous()
    lens = torch.full((seqs,), tokens, dtype=torch.int32, device=dev)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    k, v = (normal(seqs * tokens, kv_heads, head_dim).bfloat16() for _ in range(2))
    first = torch.arange(seqs + 1, dtype=torch.int32, device=dev) * tokens
    cache.append(k, v, table, lens, first)
    # what each sequence's queries lean towards: four of its prompt's keys
    at = torch.randint(tokens, (4, seqs), generator=gen, device=dev)
    lean = k.view(seqs, tokens, kv_heads, head_dim)[torch.arange(seqs, device=dev), at].float()
    engine = Engine(str(workloads.PROFILES / "c3.json"))
    pool = -(-cache.keys.numel() // PAGE) * PAGE
    engine.register(KEY_BASE, pool)
    engine.register(KEY_BASE + pool, pool)

    flash = {"dense": [], "selected": []}
    error, held = [], {"before": [], "after": []}
    evicted = 0
    for step in range(steps):
        lens = lens + 1
        x = normal(seqs, kv_heads, head_dim).bfloat16()
        cache.append(x, normal(seqs, kv_heads, head_dim).bfloat16(), table, lens)
        q = normal(seqs, kv_heads, heads // kv_heads, head_dim) + 1.5 * lean[step % 4][:, :, None]
        q = q.view(seqs, heads, head_dim).bfloat16()
        chosen = cache.select(q, table, lens, count)
        some = cache.attend(q, table, lens, selected=chosen)
        before = cache.weights()
        full = cache.attend(q, table, lens, accumulate=True)
        gained = cache.weights() - before
        # how much of the dense attention the selected blocks hold
        ids = torch.gather(table.long()[:, None].expand(seqs, kv_heads, table.shape[1]), 2,
                           chosen.clamp(min=0).long())
        share = torch.gather(gained.t()[None].expand(seqs, kv_heads, cache.blocks), 2, ids)
        share = torch.where(chosen >= 0, share, 0.0).sum() / gained.sum()
        held["after" if evicted else "before"].append(float(share))
        error.append(float((some.float() - full.float()).norm() / full.float().norm()))
        n, rows = lens.cpu().numpy(), table.cpu().numpy()
        done = n // t
        writes = rows[np.arange(seqs), done - 1][n % t == 0]
        for form, pick in (("dense", None), ("selected", chosen.cpu().numpy())):
            flash[form].append(flash_step(engine, cache, on_flash(rows, n, t, pick, kv_heads),
                                          writes))
        if step == steps // 2 - 1:
            short, lens, freed, gone = cache.evict(table, lens, keep)
            evicted = int(gone.sum())
            # the freed blocks are the sequence's next ones to fill
            order = torch.arange(width, device=dev)[None]
            kept = (lens[:, None] + t - 1) // t
            moved = torch.gather(freed, 1, (order - kept).clamp(min=0))
            table = torch.where(order < kept, short, torch.where(order < kept + gone[:, None],
                                                                 moved, -1)).contiguous()
    engine.close()

    def mean(form, key, part):
        rows = flash[form][:steps // 2] if part == "before" else flash[form][steps // 2:]
        return float(np.mean([r[key] for r in rows])) if rows else 0.0

    out = {"seqs": seqs, "tokens": tokens, "steps": steps, "count": count, "keep": keep,
           "evicted_blocks": evicted, "output_error": float(np.mean(error)),
           "attention_held": {k: float(np.mean(x)) if x else None for k, x in held.items()}}
    for form in flash:
        out[form] = {part: {key: mean(form, key, part) for key in ("accesses", "ms", "bytes")}
                     for part in ("before", "after")}
    return out


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("seqs", 8), ("tokens", 8192), ("steps", 24), ("count", 64),
                        ("keep", 256), ("heads", 32), ("kv-heads", 8), ("head-dim", 128),
                        ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    print(json.dumps(run(**vars(ap.parse_args())), indent=1), flush=True)


if __name__ == "__main__":
    main()
