"""What the operators of a branching, drafting decode over the paged cache are judged by.

Every case is one pass through an operator of `hbfsim_amd.kvcache` or `hbfsim_amd.drafts`. `refs`
(int32 [blocks]) counts the table entries that name a block; a block of no reference is free.

- `copy`: blocks of one pool become blocks of another (to and from a second tier);
- `fork`: the next batch's rows continue rows of this one, sharing their blocks (branches, beams);
- `release`: blocks past the sequences' lengths leave their rows (rejected drafts, ended sequences);
- `grow`: every sequence gets the blocks that the step's tokens go to, and a block of its own in
  place of one that it would write to and shares;
- `compact`: blocks in use move to the front of the pool, tables and references with them;
- `verify`: which of a step's drafted tokens stay, and the token that follows them, from the target's
  and the draft's probabilities and given random numbers.

Blocks are moved and never computed here, so their codes are compared as they are. The pool's arrays
are in the layout that perf/operators.py describes; a block is contiguous in each of them.
"""
import math
import random

import torch

own = False

UNIT = 2.0 ** 40  # a probability of one, in the whole numbers that are summed


def listed():
    return [
        # one conversation with four drafted tokens: latency is what it costs (a vocabulary of 32000)
        dict(name="verify_one", kind="verify", seqs=1, min_drafts=4, max_drafts=4, vocab=32000,
             dtype="f32", draft=True),
        # a decode step of 64 sequences, one to seven drafts each, over a large vocabulary
        dict(name="verify_step", kind="verify", seqs=64, min_drafts=1, max_drafts=7, vocab=151936,
             dtype="f32", draft=True),
        # eight beams of one answer take their next parents
        dict(name="fork_beams", kind="fork", seqs=8, rows=8, share=8, min_len=700, max_len=700,
             block=16, ended=False),
        # the paged-KV workload's batch, every sequence continued by four branches
        dict(name="fork_batch", kind="fork", seqs=64, rows=256, share=1, min_len=1024, max_len=32768,
             block=16, ended=False),
        # the blocks of rejected drafts are given back after a step
        dict(name="release_step", kind="release", seqs=64, share=1, min_len=1024, max_len=32768,
             most=7, block=16, ended=False),
        # branches end: 256 rows of shared prefixes, a third of them done
        dict(name="release_rows", kind="release", seqs=256, share=4, min_len=4000, max_len=20001,
             most=40, block=16, ended=True),
        # a decode step's blocks, one new token each, half of the groups of four just forked
        dict(name="grow_step", kind="grow", seqs=64, share=4, min_len=1024, max_len=16001, min_new=1,
             max_new=1, kv_heads=8, head_dim=128, block=16, free=4000),
        # ragged prompts taken in at once, wider blocks (TinyLlama's heads)
        dict(name="grow_prompts", kind="grow", seqs=17, share=1, min_len=1, max_len=3001, min_new=501,
             max_new=4001, kv_heads=4, head_dim=64, block=32, free=9000),
        # the blocks that a decode step's forks part with, copied by hand
        dict(name="copy_few", kind="copy", blocks=600, count=12, kv_heads=4, head_dim=64, block=16,
             two=False),
        # sequences swapped out to the other tier's pool
        dict(name="copy_pool", kind="copy", blocks=16001, count=8003, kv_heads=8, head_dim=128,
             block=16, two=True),
        # a small pool (one short conversation's blocks and what others left)
        dict(name="compact_few", kind="compact", seqs=3, share=1, min_len=500, max_len=2000, kv_heads=4,
             head_dim=64, block=16, free=150),
        # a pool of the paged-KV workload's heads, a third of it free in holes
        dict(name="compact_pool", kind="compact", seqs=64, share=4, min_len=4000, max_len=16384,
             kv_heads=8, head_dim=128, block=16, free=9001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "fork", "release", "grow", "grow", "copy", "compact"])
    if kind == "verify":
        c = dict(kind=kind, vocab=_log(rng, 900, 200_000), max_drafts=rng.choice([0, 1, 3, 5, 8, 17]),
                 dtype=rng.choice(["f32", "f32", "bf16", "f16"]), draft=rng.random() < 0.7)
        c["min_drafts"] = rng.choice([0, c["max_drafts"]])
        c["seqs"] = _log(rng, 1, max(2, min(300, 24_000_000 // (c["vocab"] * (c["max_drafts"] + 1)))))
        return c
    heads = dict(kv_heads=rng.choice([1, 2, 4, 5, 8]), head_dim=rng.choice([64, 80, 128, 128, 192, 256]))
    block = rng.choice([16, 16, 32, 64, 128])
    # the widest draws stay below the largest listed pools
    most = int(2.0e9 / (2 * block * heads["kv_heads"] * (-(-heads["head_dim"] // 64) * 64)))
    if kind == "copy":
        c = dict(kind=kind, **heads, block=block, blocks=_log(rng, 4, min(most // 2, 16000)),
                 two=rng.random() < 0.5)
        c["count"] = max(1, _log(rng, 1, max(2, c["blocks"] // 2 - 1)))
        return c
    c = dict(kind=kind, block=block, seqs=_log(rng, 1, 250), max_len=_log(rng, 20, 30_000))
    c["share"] = rng.choice([1, 1, 2, 4, c["seqs"]])
    while c["seqs"] > 1 and c["seqs"] * (c["max_len"] // block + 1) > min(most // 2, 60_000):
        c["seqs"] //= 2
    c["min_len"] = rng.choice([0, 1, max(1, c["max_len"] // 8), c["max_len"]])
    if kind == "fork":
        return c | dict(rows=_log(rng, 1, 300), ended=rng.random() < 0.5)
    if kind == "release":
        return c | dict(most=rng.choice([0, 1, 7, block, 5 * block]), ended=rng.random() < 0.5)
    c |= heads | dict(free=_log(rng, 1, min(8000, most // 2)))
    if kind == "grow":
        c["max_new"] = rng.choice([1, 1, 2, 5, 8, _log(rng, 8, 3000)])
        c["min_new"] = rng.choice([1, c["max_new"]])
        need = c["seqs"] * (c["max_new"] // block + 1)
        if rng.random() < 0.75:
            c["free"] = max(c["free"], min(2 * need, most // 2))
        else:  # the pool may run short
            c["free"] = _log(rng, 1, max(2, need // 2))
    return c


# ---- sizes ----------------------------------------------------------------


def _rows(case):
    """Per row of the batch: tokens stored, tokens of the step, the blocks that it shares with the
    first row of its group, and all of its blocks."""
    r = random.Random(str(sorted((k, v) for k, v in case.items() if k != "name")))
    t, out = case["block"], []
    share = max(1, min(case["share"], case["seqs"]))
    for at in range(0, case["seqs"], share):
        n = min(share, case["seqs"] - at)
        lens = [r.randint(case["min_len"], case["max_len"]) for _ in range(n)]
        if at == 0:
            lens[0] = case["max_len"]
        if n > 1 and case["kind"] in ("grow", "fork") and r.random() < 0.5:
            lens, common = [lens[0]] * n, -(-lens[0] // t)  # just forked
        else:
            common = min(lens) // (2 * t)
        for i, x in enumerate(lens):
            new = r.randint(case["min_new"], case["max_new"]) if case["kind"] == "grow" else 0
            out.append((x, new, common if i else 0, -(-x // t)))
    return out


def _block_bytes(case):
    dims = -(-case["head_dim"] // 64) * 64
    return case["kv_heads"] * (2 * case["block"] * dims + 2 * dims + 16)


def _pool(case):
    """(blocks in use, blocks of the pool)"""
    used = sum(nb - common for _, _, common, nb in _rows(case))
    if case["kind"] in ("fork", "release"):
        return used, used + used // 4 + 64
    return used, used + case["free"]


def _drafts(case):
    r = random.Random(str((case["seqs"], case["min_drafts"], case["max_drafts"])))
    return [r.randint(case["min_drafts"], case["max_drafts"]) for _ in range(case["seqs"])]


def work(case):
    if case["kind"] == "verify":
        size = 4 if case["dtype"] == "f32" else 2
        tables = 2 if case["draft"] and case["max_drafts"] else 1
        n, v = sum(_drafts(case)), case["vocab"]
        return {"bytes": case["seqs"] * (v * size * tables + 20) + n * (size * tables + 12),
                "flops": 2 * case["seqs"] * v * tables}
    if case["kind"] == "copy":
        return {"bytes": case["count"] * (2 * _block_bytes(case) + 8), "flops": case["count"]}
    rows, (used, total) = _rows(case), _pool(case)
    entries = sum(nb for _, _, _, nb in rows)
    width = max(nb for _, _, _, nb in rows) + 1
    if case["kind"] == "fork":
        return {"bytes": 4 * (entries + case["rows"] * width) + 8 * used + 12 * case["rows"],
                "flops": entries}
    if case["kind"] == "release":
        gone = entries if case["ended"] else case["seqs"] * (case["most"] // case["block"] + 1)
        return {"bytes": 4 * (entries + gone) + 8 * gone, "flops": gone}
    if case["kind"] == "grow":
        t = case["block"]
        need = sum(-(-(x + m) // t) - -(-x // t) for x, m, _, _ in rows)
        parted = sum(1 for x, m, common, nb in rows if common == nb and x % t)
        return {"bytes": 4 * need * max(1, total // max(1, case["free"])) + 8 * (need + parted)
                + 16 * case["seqs"] + parted * 2 * _block_bytes(case), "flops": need + case["seqs"]}
    moved = int(used * (1 - used / total))
    return {"bytes": 4 * (2 * total + 2 * entries) + moved * 2 * _block_bytes(case), "flops": total}


# ---- inputs ---------------------------------------------------------------


def _arrays(case, blocks, gen, dev):
    """A pool's arrays, every block filled."""
    kv, t, dims = case["kv_heads"], case["block"], -(-case["head_dim"] // 64) * 64
    shape = (blocks, kv, t // 16, dims // 64, 4, 16)

    def codes(*s):
        return torch.randint(-127, 128, s, generator=gen, device=dev, dtype=torch.int8)

    def scales():
        return torch.randn((blocks, kv), generator=gen, device=dev).mul_(0.3).exp_().div_(32)

    return [codes(*shape, 16), codes(*shape, 4, 4), scales(), scales(), codes(blocks, kv, 2, dims),
            torch.randint(0, 1 << 40, (blocks, kv), generator=gen, device=dev)]


ARRAYS = ("keys", "values", "key_scale", "value_scale", "bounds", "weight")


def _cache(arrays, case, refs=None):
    from hbfsim_amd.kvcache import KvCache
    return KvCache.from_tensors(*arrays, head_dim=case["head_dim"], refs=refs)


def _prepare_verify(case, gen, dev):
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[case["dtype"]]
    drafts, v = _drafts(case), case["vocab"]
    first = [0]
    for n in drafts:
        first.append(first[-1] + n + 1)
    rows = first[-1]
    target = torch.empty((rows, v), dtype=dtype, device=dev)
    draft = torch.empty((rows, v), dtype=dtype, device=dev) if case["draft"] else None
    tokens = torch.randint(0, v, (rows,), generator=gen, device=dev, dtype=torch.int32)
    step = max(1, (1 << 26) // v)
    for a in range(0, rows, step):
        n = min(step, rows - a)
        x = torch.randn((n, v), generator=gen, device=dev).mul_(3.5)
        target[a:a + n] = torch.softmax(x, 1).to(dtype)
        # the draft knows the target's mind, but for some noise; its token is drawn from it
        x.add_(torch.randn((n, v), generator=gen, device=dev).mul_(0.8))
        q = torch.softmax(x, 1)
        if draft is not None:
            draft[a:a + n] = q.to(dtype)
            drawn = (q / torch.empty_like(q).exponential_(generator=gen)).argmax(1)
        else:
            drawn = q.argmax(1)
        k = min(n, rows - a - 1)
        tokens[a + 1:a + 1 + k] = drawn[:k].to(torch.int32)
    u = torch.rand((rows,), generator=gen, device=dev)
    lens = torch.tensor([100 + 13 * i + n for i, n in enumerate(drafts)], dtype=torch.int32, device=dev)
    return {"target": target, "draft": draft, "tokens": tokens, "uniform": u, "lens": lens,
            "first": torch.tensor(first, dtype=torch.int32, device=dev) if case["max_drafts"] else None,
            "most": max(drafts) + 1}


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 2 + 1)
    st = {"case": dict(case)}
    if case["kind"] == "verify":
        return st | _prepare_verify(case, gen, dev)
    if case["kind"] == "copy":
        st["from"] = _arrays(case, case["blocks"], gen, dev)
        st["to"] = _arrays(case, case["blocks"], gen, dev) if case["two"] else st["from"]
        ids = torch.randperm(case["blocks"], generator=gen, device=dev).to(torch.int32)
        st["src"] = ids[:case["count"]].contiguous()
        st["dst"] = ids[case["blocks"] - case["count"]:].contiguous()
        if own:
            st["cache"] = _cache(st["from"], case)
            st["other"] = _cache(st["to"], case) if case["two"] else None
        return st
    rows, (used, total) = _rows(case), _pool(case)
    t = case["block"]
    new = [m for _, m, _, _ in rows]
    blocks = [nb for _, _, _, nb in rows]
    width = max(1, max(-(-(x + m) // t) for x, m, _, _ in rows)) + (case["kind"] != "grow")
    ids = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    # references and table side by side, as they start out and as the operators change them
    room = -(-total // 64) * 64
    start = torch.zeros(room + len(rows) * width, dtype=torch.int32, device=dev)
    refs, table = start[:total], start[room:].view(len(rows), width)
    table.fill_(-1)
    at, share = 0, max(1, min(case["share"], case["seqs"]))
    for i, (_, _, common, nb) in enumerate(rows):
        if common:
            table[i, :common] = table[i - i % share, :common]
        table[i, common:nb] = ids[at:at + nb - common]
        at += nb - common
    flat = table.reshape(-1).long()
    refs.index_add_(0, flat.clamp(min=0), (flat >= 0).to(torch.int32))
    st.update(start=start, live=start.clone(), room=room, total=total, width=width)
    st["refs"], st["table"] = st["live"][:total], st["live"][room:].view(len(rows), width)
    lens = torch.tensor([x + m for x, m, _, _ in rows], dtype=torch.int32, device=dev)
    if case["kind"] == "fork":
        # row i's parent is of the group that row i's branch belongs to
        n, groups = case["rows"], -(-len(rows) // share)
        of = torch.arange(n, device=dev) * groups // n
        one = torch.rand((n,), generator=gen, device=dev)
        size = (len(rows) - of * share).clamp(max=share)
        parents = of * share + (one * size).long().clamp(max=share - 1)
        if case["ended"]:
            gone = torch.rand((n,), generator=gen, device=dev) < 0.2
            parents = torch.where(gone, -1, parents)
        st["parents"] = parents.to(torch.int32)
    if case["kind"] == "release":
        drop = torch.randint(0, case["most"] + 1, (len(rows),), generator=gen, device=dev)
        kept = (lens - drop).clamp(min=0)
        if case["ended"]:
            kept = torch.where(torch.rand((len(rows),), generator=gen, device=dev) < 0.33, 0, kept)
        lens = kept.to(torch.int32)
    st["lens"] = lens
    if case["kind"] in ("grow", "compact"):
        st["pool"] = _arrays(case, total, gen, dev)
        if own:
            st["cache"] = _cache(st["pool"], case, st["refs"])
    if case["kind"] == "grow":
        # what one step writes at most, and the offsets of its rows where they are not one each
        st["most"] = max(-(-(x + m) // t) - x // t for x, m, _, _ in rows)
        st["tokens"], st["first"] = sum(new), None
        if case["max_new"] > 1:
            first = [0]
            for m in new:
                first.append(first[-1] + m)
            st["first"] = torch.tensor(first, dtype=torch.int32, device=dev)
    return st


# ---- the plain forms ------------------------------------------------------


def _start(st):
    """References and table as they are before the call."""
    return (st["start"][:st["total"]].clone(),
            st["start"][st["room"]:].view(-1, st["width"]).clone())


def _plain_copy(st):
    src, dst = st["src"].long(), st["dst"].long()
    for a, b in zip(st["from"], st["to"]):
        b[dst] = a[src]
    return dict(zip(ARRAYS, st["to"]))


def _plain_fork(st):
    refs, table = _start(st)
    seqs = table.shape[0]
    parents = st["parents"].long()
    there = (parents >= 0) & (parents < seqs)
    at = torch.where(there, parents, 0)
    out = torch.where(there[:, None], table[at], -1)
    lens = torch.where(there, st["lens"][at], 0)
    children = torch.zeros(seqs, dtype=torch.int32, device=table.device)
    children.index_add_(0, at, there.to(torch.int32))
    valid = (table >= 0) & (table < st["total"])
    change = torch.where(valid, (children - 1)[:, None], 0)
    refs.index_add_(0, torch.where(valid, table, 0).reshape(-1).long(), change.reshape(-1))
    return {"table": out, "lens": lens, "refs": refs}


def _plain_release(st):
    refs, table = _start(st)
    t = st["case"]["block"]
    keep = (st["lens"].long().clamp(min=0) + t - 1) // t
    leaves = torch.arange(table.shape[1], device=table.device) >= keep[:, None]
    gone = leaves & (table >= 0) & (table < st["total"])
    refs.index_add_(0, torch.where(gone, table, 0).reshape(-1).long(), -gone.to(torch.int32).reshape(-1))
    return {"table": torch.where(leaves, -1, table), "refs": refs}


def _plain_grow(st):
    refs, table = _start(st)
    t, most, total = st["case"]["block"], st["most"], st["total"]
    seqs, width = table.shape
    dev = table.device
    n = st["lens"].long()
    m = torch.ones_like(n) if st["first"] is None else (st["first"][1:] - st["first"][:-1]).long()
    come = n - m
    live = (m > 0) & (come >= 0)
    block = come[:, None].div(t, rounding_mode="floor") + torch.arange(most, device=dev)
    writes = live[:, None] & (block * t < n[:, None])
    outside = writes & (block >= width)
    short = outside.any(1)
    at = block.clamp(0, width - 1)
    e = torch.gather(table, 1, at).long()
    named = writes & ~short[:, None] & (e >= 0) & (e < total)
    e = torch.where(named, e, 0)
    count = refs[e]
    there = named & (count > 0)
    begun = block * t < come[:, None]
    # where all of a block's holders write to it, the last keeps it
    order = torch.arange(seqs * most, device=dev).view(seqs, most)
    writers = torch.zeros(total + 1, dtype=torch.int64, device=dev)
    last = torch.full((total + 1,), -1, dtype=torch.int64, device=dev)
    slot = torch.where(there, e, total).view(-1)
    writers.index_add_(0, slot, torch.ones_like(slot))
    last.scatter_reduce_(0, slot, order.view(-1), "amax")
    wanted = writes & ~short[:, None] & ~(begun & ~there)
    keeps = there & (writers[e] >= count) & (last[e] == order)
    free = (refs <= 0).cumsum(0)
    enough = (wanted & ~keeps).sum() <= free[-1]
    fresh = wanted & ~torch.where(enough, keeps, there & (count == 1))
    need = fresh.sum(1)
    granted = ~short & ((need == 0) | (need.cumsum(0) <= free[-1]))
    fresh &= granted[:, None]
    rank = fresh.view(-1).cumsum(0).view(seqs, most)
    new = torch.searchsorted(free, rank)
    stale = granted[:, None] & named & ~there & begun
    entry = torch.where(fresh, new, -1).to(torch.int32)
    entry = torch.where(fresh | stale, entry, torch.gather(table, 1, at))
    hit = torch.where(fresh | stale, at, width)
    wide = torch.cat([table, table[:, :1]], 1)
    wide.scatter_(1, hit, entry)
    parted = fresh & there
    refs.index_add_(0, torch.where(parted, e, 0).view(-1), -parted.to(torch.int32).view(-1))
    got = torch.where(fresh, new, 0).view(-1)
    refs.index_add_(0, got, torch.where(fresh.view(-1), 1 - refs[got], 0).to(torch.int32))
    moved = parted & begun
    src, dst = e[moved], new[moved]
    for a in st["pool"]:
        a[dst] = a[src]
    lacking = live & ~granted
    return {"lens": torch.where(lacking, 0, st["lens"]),
            "missing": torch.where(lacking, need + outside.sum(1), 0).to(torch.int32),
            "table": wide[:, :width].contiguous(), "refs": refs} | dict(zip(ARRAYS, st["pool"]))


def _plain_compact(st):
    refs, table = _start(st)
    used = refs > 0
    live = used.sum()
    i = torch.arange(st["total"], device=refs.device)
    src = torch.nonzero(used & (i >= live)).view(-1)
    dst = torch.nonzero(~used & (i < live)).view(-1)
    where = torch.where(used, i, -1)
    where[src] = dst
    for a in st["pool"]:
        a[dst] = a[src]
    valid = (table >= 0) & (table < st["total"])
    table = torch.where(valid, where[table.clamp(0, st["total"] - 1).long()], -1).to(torch.int32)
    moved = refs[src]
    refs = torch.where(i < live, refs, 0)
    refs[dst] = moved
    return {"where": where.to(torch.int32), "table": table, "refs": refs} | dict(zip(ARRAYS, st["pool"]))


def _plain_verify(st):
    p, q, u, tokens = st["target"], st["draft"], st["uniform"], st["tokens"].long()
    rows, vocab = p.shape
    seqs, dev = st["lens"].shape[0], p.device
    first = st["first"]
    first = torch.arange(seqs + 1, device=dev) if first is None else first.long()
    n = first[1:] - first[:-1]
    i = torch.arange(st["most"], device=dev)
    at = (first[:-1, None] + i).clamp(max=rows - 1)
    drafted = i < (n - 1)[:, None]
    x = tokens[(at + 1).clamp(max=rows - 1)]
    known = drafted & (x >= 0) & (x < vocab)
    x = torch.where(known, x, 0)

    def share(z):  # a probability, with what is none taken for the nearest
        return torch.nan_to_num(z.float(), nan=0.0).clamp(0.0, 1.0)

    def whole(z):
        return torch.round(share(z).double() * UNIT).long()

    px = share(p[at, x]).double()
    qx = share(q[at, x]).double() if q is not None else torch.ones_like(px)
    stays = known & (u[at].double() * qx < px)
    accepted = stays.long().cumprod(1).sum(1)
    live = n > 0
    row = (first[:-1] + accepted).clamp(max=rows - 1)
    refused = torch.gather(known, 1, accepted[:, None].clamp(max=st["most"] - 1))[:, 0] & (accepted < n - 1)
    weight = whole(p[row])
    less = weight
    if q is not None:
        less = (weight - whole(q[row])).clamp(min=0)
    else:
        token = torch.gather(x, 1, accepted[:, None].clamp(max=st["most"] - 1))
        less = torch.where(torch.arange(vocab, device=dev) == token, 0, weight)
    less = torch.where(refused[:, None], less, weight)
    less = torch.where(less.sum(1, keepdim=True) > 0, less, weight)
    run_sum = less.cumsum(1)
    sums = run_sum[:, -1]
    draw_at = torch.nan_to_num(u[(first[1:] - 1).clamp(min=0)].double(), nan=0.0).clamp(0.0, 1.0)
    k = (draw_at * 2.0 ** 31).long().clamp(max=2 ** 31 - 1)
    k = k * (sums >> 31) + ((k * (sums & (2 ** 31 - 1))) >> 31)
    last = torch.searchsorted(run_sum, k[:, None], right=True)[:, 0]
    last = torch.where(sums > 0, last, -1)
    given = torch.where(i < accepted[:, None], x, torch.where(i == accepted[:, None], last[:, None], -1))
    out = torch.full((rows + 1,), -1, dtype=torch.int32, device=dev)
    inside = live[:, None] & (i < n[:, None])
    out.scatter_(0, torch.where(inside, at, rows).view(-1), torch.where(inside, given, -1).view(-1).to(torch.int32))
    gained = torch.where(live, accepted + 1, 0)
    return {"out": out[:rows], "gained": gained.to(torch.int32),
            "lens": (st["lens"] - n + gained).to(torch.int32)}


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        return {"copy": _plain_copy, "fork": _plain_fork, "release": _plain_release, "grow": _plain_grow,
                "compact": _plain_compact, "verify": _plain_verify}[kind](state)
    if kind == "verify":
        from hbfsim_amd import drafts
        out, gained, lens = drafts.verify(state["target"], state["tokens"], state["uniform"],
                                          state["first"], draft=state["draft"], lens=state["lens"])
        return {"out": out, "gained": gained, "lens": lens}
    if kind == "copy":
        state["cache"].copy(state["src"], state["dst"], to=state["other"])
        return dict(zip(ARRAYS, state["to"]))
    state["live"].copy_(state["start"])  # the pass before changed them
    refs, table = state["refs"], state["table"]
    if kind in ("fork", "release"):
        from hbfsim_amd import kvcache
        if kind == "fork":
            out, lens = kvcache.fork(refs, table, state["lens"], state["parents"])
            return {"table": out, "lens": lens, "refs": refs}
        kvcache.release(refs, table, state["lens"], block_tokens=c["block"])
        return {"table": table, "refs": refs}
    cache = state["cache"]
    if kind == "grow":
        lens, missing = cache.grow(table, state["lens"], state["first"], tokens=state["tokens"])
        got = {"lens": lens, "missing": missing}
    else:
        got = {"where": cache.compact(table)}
    return got | {"table": table, "refs": refs} | dict(zip(ARRAYS, state["pool"]))


# ---- the definition in 64 bits --------------------------------------------


def exact(case, seed):
    if case["kind"] != "verify":
        return None  # block ids, counts and moved bytes: nothing is computed
    st = prepare(case, seed)
    p, q = st["target"], st["draft"]
    u, tokens, drafts = st["uniform"].tolist(), st["tokens"].tolist(), _drafts(case)
    out, gained, lens, at = [], [], [], 0
    for n, was in zip(drafts, st["lens"].tolist()):
        got, token, i = [], None, 0
        while i < n:
            x = tokens[at + i + 1]
            if not u[at + i] * (1.0 if q is None else float(q[at + i, x])) < float(p[at + i, x]):
                token = x
                break
            got.append(x)
            i += 1
        # sums of whole numbers below 2^53 are exact in float64
        full = torch.round(p[at + i].double() * 2 ** 40)
        part = full
        if token is not None and q is not None:
            part = torch.relu(full - torch.round(q[at + i].double() * 2 ** 40))
        elif token is not None:
            part = full.clone()
            part[token] = 0
        if not float(part.sum()):
            part = full
        run_sum = torch.cumsum(part, 0)
        k = (int(u[at + n] * 2 ** 31) * int(run_sum[-1])) >> 31
        got.append(int((run_sum <= k).sum()))
        out += got + [-1] * (n - i)
        gained.append(len(got))
        lens.append(was - n - 1 + len(got))
        at += n + 1
    dev = p.device
    return {"out": torch.tensor(out, device=dev, dtype=torch.int32),
            "gained": torch.tensor(gained, device=dev, dtype=torch.int32),
            "lens": torch.tensor(lens, device=dev, dtype=torch.int32)}
