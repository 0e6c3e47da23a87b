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

    python -m hbfsim_amd.kv_study --seqs 8 --tokens 8192 --branches 4 --drafts 4

With `--branches` or `--drafts` the decode branches and drafts instead: every
prompt is continued by that many sequences that share its blocks, and every
step appends and attends to the drafted tokens as well, verifies them against
the target's probabilities (synthetic ones over `--vocab` tokens, of a draft
that knows the target's mind but for some noise) and gives back the blocks of
those that do not stay.  Half way every second branch ends and the blocks in
use move to the front of the pool.  Prints what a step gains and reads, with
the drafts and without, and the flash time before and after the compaction.
"""
from __future__ import annotations

import argparse
import json

import numpy as np
import torch

from . import drafts as drafted
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


def run_drafts(seqs: int = 8, tokens: int = 8192, steps: int = 24, branches: int = 4,
               drafts: int = 4, vocab: int = 32000, heads: int = 32, kv_heads: int = 8,
               head_dim: int = 128, seed: int = 0) -> dict:
    """A decode of `branches` sequences a prompt with `drafts` drafted tokens a step."""
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    t, m = 16, drafts + 1
    rows = seqs * branches
    width = -(-(tokens + (steps + 1) * m) // t)
    # every prompt once, and each branch's own blocks from its last prompt block on
    own = -(-((steps + 1) * m) // t) + 2
    cache = kvcache.KvCache(seqs * -(-tokens // t) + 2 * rows * own, kv_heads, head_dim, t, dev)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device=dev)
    lens = torch.full((seqs,), tokens, dtype=torch.int32, device=dev)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    first = torch.arange(seqs + 1, dtype=torch.int32, device=dev) * tokens
    lens, missing = cache.grow(table, lens, first, seqs * tokens)
    cache.append(normal(seqs * tokens, kv_heads, head_dim).bfloat16(),
                 normal(seqs * tokens, kv_heads, head_dim).bfloat16(), table, lens, first)
    parents = torch.arange(seqs, dtype=torch.int32, device=dev).repeat_interleave(branches)
    table, lens = cache.fork(table, lens, parents)
    engine = Engine(str(workloads.PROFILES / "c3.json"))
    pool = -(-cache.keys.numel() // PAGE) * PAGE
    engine.register(KEY_BASE, pool)
    engine.register(KEY_BASE + pool, pool)

    def reads(n: np.ndarray, ids: np.ndarray) -> np.ndarray:
        # a block that branches share is read once a step
        return np.unique(on_flash(ids, n, t, None, kv_heads), axis=0)

    parts = {"before": [], "after": []}
    gained = {"before": [], "after": []}
    result = {"seqs": seqs, "tokens": tokens, "steps": steps, "branches": branches,
              "drafts": drafts, "vocab": vocab, "missing": int((missing != 0).sum())}
    for step in range(steps):
        now = "before" if step < steps // 2 else "after"
        if step == steps // 2:
            keep = torch.arange(0, table.shape[0], 2, dtype=torch.int32, device=dev)
            table, lens = cache.fork(table, lens, keep)
            held, ids = lens.cpu().numpy(), table.cpu().numpy()
            spread = flash_step(engine, cache, reads(held, ids), np.zeros(0, np.int64))
            where = cache.compact(table)
            ids = table.cpu().numpy()
            packed = flash_step(engine, cache, reads(held, ids), np.zeros(0, np.int64))
            used = where >= 0
            at = torch.arange(cache.blocks, device=dev)
            result["compaction"] = {
                "blocks": int(used.sum()), "moved": int((used & (where != at)).sum()),
                "named_by_rows": int((table >= 0).sum()), "ms_before": spread["ms"],
                "ms_after": packed["ms"]}
            rows = table.shape[0]
        first = torch.arange(rows + 1, dtype=torch.int32, device=dev) * m
        want = rows * m
        step_lens, missing = cache.grow(table, lens + m, first, want)
        # a sequence that lacks blocks reads nothing
        n = torch.where(missing == 0, lens, 0).cpu().numpy()
        result["missing"] += int((missing != 0).sum())
        k, v = (normal(want, kv_heads, head_dim).bfloat16() for _ in range(2))
        cache.append(k, v, table, step_lens, first)
        cache.attend(normal(want, heads, head_dim).bfloat16(), table, step_lens, first)
        x = normal(want, vocab).mul_(3.5)
        target = torch.softmax(x, 1)
        draft = torch.softmax(x.add_(normal(want, vocab), alpha=0.8), 1)
        said = torch.zeros(want, dtype=torch.int32, device=dev)
        said[1:] = (draft / torch.empty_like(draft).exponential_(generator=gen)).argmax(1)[:-1]
        u = torch.rand((want,), generator=gen, device=dev)
        _, count, lens = drafted.verify(target, said, u, first, draft=draft, lens=step_lens,
                                        stored=lens)
        cache.release(table, lens)
        left, ids = torch.where(missing == 0, lens, 0).cpu().numpy(), table.cpu().numpy()
        done = [ids[s, n[s] // t:left[s] // t] for s in range(rows)]  # filled by this step
        parts[now].append(flash_step(engine, cache, reads(n, ids), np.concatenate(done)))
        gained[now].append(float(count.float().mean()))
    engine.close()
    for now, steps_of in parts.items():
        got = float(np.mean(gained[now])) if gained[now] else 0.0
        out = {key: float(np.mean([x[key] for x in steps_of])) if steps_of else 0.0
               for key in ("accesses", "ms", "bytes")}
        # a step without drafts reads the same and gains one token
        out |= {"gained": got, "ms_per_token": out["ms"] / got if got else 0.0}
        result[now] = out
    return result


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("seqs", 8), ("tokens", 8192), ("steps", 24), ("count", 64),
                        ("keep", 256), ("heads", 32), ("kv-heads", 8), ("head-dim", 128),
                        ("seed", 0), ("branches", 1), ("drafts", 0), ("vocab", 32000)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = vars(ap.parse_args())
    branching = args["branches"] != 1 or args["drafts"] != 0
    for name in ("count", "keep") if branching else ("branches", "drafts", "vocab"):
        del args[name]
    print(json.dumps((run_drafts if branching else run)(**args), indent=1), flush=True)


if __name__ == "__main__":
    main()
