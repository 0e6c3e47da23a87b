"""What the paged 8-bit key/value cache's operators are judged by.

Every case is one pass through an operator of `hbfsim_amd.kvcache` as a decode
or prompt step of a flash-tiered cache study calls it:

- `append`: new tokens' keys and values quantised into their blocks, and the
  blocks read back as the values they now stand for;
- `attend`: attention of a batch's query tokens over the cache (one token a
  sequence, or chunks of a prompt; every visible block, or a list of blocks
  for each query; with or without the accumulated weights);
- `select`: the blocks that a cheap score picks for each query;
- `evict`: the blocks that leave the cache, by accumulated weight.

The cache's tensors are in the layout that the library documents:

- keys int8 [blocks, kv_heads, tokens / 16, dims / 64, 4, 16, 16]: token of the
  tile next to last, dim = 64 chunk + 16 quarter + last;
- values int8 [blocks, kv_heads, tokens / 16, dims / 64, 4, 16, 4, 4]: token of
  the tile = 4 quarter + last, dim = 64 chunk + 16 (next to last) + 16-index;
- key_scale, value_scale float32 [blocks, kv_heads];
- bounds int8 [blocks, kv_heads, 2, dims]: lowest and highest key code of the
  block in each dim;
- weight int64 [blocks, kv_heads]: accumulated attention, in units of 2^-32.

`dims` is the head dimension rounded up to a multiple of 64, zeros beyond it.
"""
import math
import random

import torch

own = False

INV127 = 1.0 / 127.0
SCALE_MIN, SCALE_MAX = 2.0 ** -40, 2.0 ** 40
WEIGHT_UNIT = 2.0 ** -32


def listed():
    return [
        # a decode step's new tokens, one for each of 64 sequences (the paged-KV workload's shape)
        dict(name="append_step", kind="append", seqs=64, min_len=1024, max_len=32768, min_new=1,
             max_new=1, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # prompts of seven sequences taken in at once, ragged, blocks begun before among them
        dict(name="append_prompts", kind="append", seqs=7, min_len=4001, max_len=9001, min_new=3900,
             max_new=4001, heads=32, kv_heads=8, head_dim=128, block=16, dtype="f16"),
        # one short conversation, where the call's latency is what it costs (TinyLlama's heads)
        dict(name="attend_one_short", kind="attend", seqs=1, min_len=333, max_len=333, min_new=1,
             max_new=1, heads=32, kv_heads=4, head_dim=64, block=16, dtype="bf16"),
        # one long document: a single sequence has to fill the whole card
        dict(name="attend_one_long", kind="attend", seqs=1, min_len=262147, max_len=262147,
             min_new=1, max_new=1, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # the paged-KV workload's decode step, one layer: 64 sequences of 1024..32768 tokens
        dict(name="attend_step", kind="attend", seqs=64, min_len=1024, max_len=32768, min_new=1,
             max_new=1, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # the same step while a study accumulates weights for eviction, wider blocks and groups
        dict(name="attend_weigh", kind="attend", seqs=24, min_len=777, max_len=20001, min_new=1,
             max_new=1, heads=64, kv_heads=8, head_dim=128, block=32, dtype="bf16", accumulate=True),
        # the decode step over the 128 blocks that a selection left to each kv head
        dict(name="attend_selected", kind="attend", seqs=64, min_len=1024, max_len=32768, min_new=1,
             max_new=1, heads=32, kv_heads=8, head_dim=128, block=16, dtype="f16", count=128),
        # a chunk of two prompts over what is cached of them: bound by the matrix units
        dict(name="attend_prompt", kind="attend", seqs=2, min_len=12001, max_len=16384,
             min_new=2001, max_new=2049, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # the selection of a decode step
        dict(name="select_step", kind="select", seqs=64, min_len=1024, max_len=32768, min_new=1,
             max_new=1, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16", count=128),
        # the selection for every query of a prompt's chunk
        dict(name="select_prompt", kind="select", seqs=1, min_len=16001, max_len=16001, min_new=1001,
             max_new=1001, heads=32, kv_heads=4, head_dim=64, block=16, dtype="f16", count=64),
        # eviction down to a budget: a few sequences, and the whole batch
        dict(name="evict_few", kind="evict", seqs=3, min_len=900, max_len=5000, heads=32, kv_heads=4,
             head_dim=64, block=16, dtype="bf16", keep=48),
        dict(name="evict_batch", kind="evict", seqs=64, min_len=1024, max_len=32768, heads=32,
             kv_heads=8, head_dim=128, block=16, dtype="bf16", keep=500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "select", "evict"])
    kv = rng.choice([1, 2, 4, 5, 8])
    c = dict(kind=kind, kv_heads=kv, heads=kv * rng.choice([1, 2, 3, 4, 7, 8, 16]),
             head_dim=rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256]),
             block=rng.choice([16, 16, 32, 64, 128]), dtype=rng.choice(["bf16", "f16"]))
    longest = _log(rng, 20, 30_000)
    c.update(seqs=_log(rng, 1, 60), max_len=longest,
             min_len=rng.choice([0, 1, max(1, longest // 8), longest]))
    # the widest draws stay below the largest listed case's cache
    while c["seqs"] > 1 and c["seqs"] * longest * kv * c["head_dim"] > 64 * 16384 * 8 * 128:
        c["seqs"] //= 2
    blocks = -(-longest // c["block"])
    if kind == "evict":
        c["keep"] = max(2, _log(rng, 2, max(3, blocks)))
        return c
    chunk = rng.random() < 0.4 if kind != "append" else rng.random() < 0.6
    c.update(min_new=1, max_new=1)
    if chunk:
        most = max(1, min(longest, int(6e11 / (c["seqs"] * longest * c["heads"] * c["head_dim"])),
                          int(4e8 / (c["seqs"] * c["heads"] * longest)), 5000))
        c["max_new"] = _log(rng, 1, most) if most > 1 else 1
        c["min_new"] = rng.choice([1, c["max_new"]])
    c["min_len"] = max(c["min_len"], 0 if kind == "attend" else 1)
    if kind == "append":
        c["min_len"] = max(c["min_len"], c["max_new"])
    if kind == "select" or (kind == "attend" and rng.random() < 0.3):
        c["count"] = max(2, min(_log(rng, 2, 256), blocks + 3))
    if kind == "attend" and "count" not in c and rng.random() < 0.3:
        c["accumulate"] = True
    return c


# ---- sizes ----------------------------------------------------------------


def _dims(case):
    return -(-case["head_dim"] // 64) * 64


def _lengths(case):
    """(tokens in the cache after the step, tokens of the step) of each sequence."""
    r = random.Random(str((case["seqs"], case["min_len"], case["max_len"])))
    lens = [r.randint(case["min_len"], case["max_len"]) for _ in range(case["seqs"])]
    lens[-1] = case["max_len"]
    new = [r.randint(case.get("min_new", 1), case.get("max_new", 1)) for _ in lens]
    if case["kind"] in ("append", "select"):
        lens = [max(a, b) for a, b in zip(lens, new)]
    return lens, new


def _blocks(case):
    lens, _ = _lengths(case)
    return [-(-n // case["block"]) for n in lens]


def _seen(case):
    """Tokens of the cache that each query token attends to, summed over them, and the cache tokens
    that have to be read for them."""
    lens, new = _lengths(case)
    t, count = case["block"], case.get("count")
    pairs = read = 0
    for n, m in zip(lens, new):
        vis = [max(0, n - m + i + 1) for i in range(m)]
        if count:
            vis = [min(v, count * t) for v in vis]
            read += min(n, sum(vis))
        else:
            read += n
        pairs += sum(vis)
    return pairs, read


def work(case):
    h, kv, d, t = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    lens, new = _lengths(case)
    tokens, nblk = sum(new), sum(_blocks(case))
    if case["kind"] == "append":
        touched = len(_touched(case))
        # values in, codes out, the blocks' codes in, their values and bounds out
        moved = 2 * tokens * kv * d * (2 + 1) + touched * kv * (2 * t * d * (1 + 2) + 2 * d * (1 + 2))
        return {"bytes": moved, "flops": 6 * tokens * kv * d}
    if case["kind"] == "attend":
        pairs, read = _seen(case)
        b = read * kv * 2 * d + -(-read // t) * kv * 8 + 2 * 2 * tokens * h * d
        if case.get("accumulate"):
            b += nblk * kv * 16
        return {"bytes": b, "flops": 4.0 * pairs * h * d}
    if case["kind"] == "select":
        vis = sum(-(-(n - m + i + 1) // t) for n, m in zip(lens, new) for i in range(m))
        b = nblk * (kv * (2 * d + 4) + 4) + 2 * tokens * h * d + 4 * tokens * kv * case["count"]
        return {"bytes": b, "flops": 4.0 * vis * kv * d}
    return {"bytes": nblk * (8 * kv + 4 + 4), "flops": nblk * kv}


# ---- inputs ---------------------------------------------------------------


def _touched(case):
    """(sequence, logical block) of every block that the step's tokens go to."""
    lens, new = _lengths(case)
    t = case["block"]
    return [(s, b) for s, (n, m) in enumerate(zip(lens, new))
            for b in range((n - m) // t, -(-n // t))]


def _codes(shape, gen, dev):
    """Key codes: a direction of each block's own and the tokens' spread around it."""
    b, h, tiles, chunks = shape[:4]
    out = torch.empty(shape, dtype=torch.int8, device=dev)
    step = max(1, (1 << 27) // max(1, out[0].numel())) if b else 1
    for at in range(0, b, step):
        n = min(step, b - at)
        mean = torch.randn((n, h, 1, chunks, 4, 1, 16), generator=gen, device=dev)
        x = torch.randn((n, *shape[1:]), generator=gen, device=dev)
        out[at:at + n] = x.mul_(26).add_(mean, alpha=18).round_().clamp_(-127, 127).to(torch.int8)
    return out


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 2 + 1)
    h, kv, d, t, dims = case["heads"], case["kv_heads"], case["head_dim"], case["block"], _dims(case)
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16}[case["dtype"]]
    lens, new = _lengths(case)
    per_seq = _blocks(case)
    # the table is as wide as the longest sequence needs, the pool a little larger than what is used
    width, total = max(1, max(per_seq)), sum(per_seq) + 3
    perm = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(per_seq):
        table[s, :n] = perm[at:at + n]
        at += n
    st = {"case": dict(case), "table": table,
          "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "width": width,
          "weight": torch.zeros((total, kv), dtype=torch.int64, device=dev)}
    if case["kind"] == "evict":
        # weights of many steps: a few heavy blocks, many light ones, some equal
        x = torch.randn((total, kv), generator=gen, device=dev).mul_(2).exp_()
        st["weight"] = (x * 2.0 ** 10).to(torch.int64) << 24
        return st
    shape = (total, kv, t // 16, dims // 64, 4, 16, 16)
    st["keys"] = _codes(shape, gen, dev)
    values = torch.empty((*shape[:6], 4, 4), dtype=torch.int8, device=dev)
    step = max(1, (1 << 27) // values[0].numel())
    for a in range(0, total, step):
        n = min(step, total - a)
        x = torch.randn((n, *values.shape[1:]), generator=gen, device=dev)
        values[a:a + n] = x.mul_(32).round_().clamp_(-127, 127).to(torch.int8)
    st["values"] = values
    if d != dims:
        dim = torch.arange(dims, device=dev)
        st["keys"] *= (dim.view(dims // 64, 4, 1, 16) < d).to(torch.int8)
        live = (dim.view(dims // 64, 1, 4, 16, 1) < d).to(torch.int8)
        st["values"] *= live.permute(0, 1, 3, 2, 4)
    st["key_scale"] = torch.randn((total, kv), generator=gen, device=dev).mul_(0.2).exp_().div_(32)
    st["value_scale"] = torch.randn((total, kv), generator=gen, device=dev).mul_(0.3).exp_().div_(40)
    lo, hi = (f(st["keys"], dim=(2, 5)).reshape(total, kv, 1, dims)
              for f in (torch.amin, torch.amax))
    st["bounds"] = torch.cat([lo, hi], 2).contiguous()
    if case["max_new"] > 1:
        first = [0]
        for m in new:
            first.append(first[-1] + m)
        st["first"] = torch.tensor(first, dtype=torch.int32, device=dev)
    else:
        st["first"] = None
    # queries, keys and values are views of one projection's output
    tokens = sum(new)
    qkv = torch.randn((tokens, (h + 2 * kv) * d), generator=gen, device=dev).mul_(1.5).to(dtype)
    st["q"] = qkv[:, :h * d].view(tokens, h, d)
    st["k"] = qkv[:, h * d:(h + kv) * d].view(tokens, kv, d)
    st["v"] = qkv[:, (h + kv) * d:].view(tokens, kv, d)
    st["longest_new"] = max(new)
    st["scale"] = 1.0 / math.sqrt(d)
    if case["kind"] == "append":
        where = torch.tensor(_touched(case), device=dev)
        st["touched"] = table[where[:, 0], where[:, 1]].contiguous()
    if case["kind"] == "attend" and case.get("count"):
        # distinct blocks in ascending order for each query token and kv head, the last one in
        seq = torch.repeat_interleave(torch.arange(len(lens), device=dev),
                                      torch.tensor(new, device=dev))
        sees = _limits(st, seq)
        nb = (sees.clamp(min=0) + t - 1) // t
        key = torch.rand((tokens, kv, width), generator=gen, device=dev)
        idx = torch.arange(width, device=dev)
        key = torch.where(idx == nb[:, None, None] - 1, 2.0, key)
        key = torch.where(idx < nb[:, None, None], key, -1.0)
        k = min(case["count"], width)
        top, at = key.topk(k, dim=2)
        at = torch.where(top >= 0, at, width).sort(dim=2).values
        sel = torch.full((tokens, kv, case["count"]), -1, dtype=torch.int32, device=dev)
        sel[:, :, :k] = torch.where(at < width, at, -1).to(torch.int32)
        st["selected"] = sel
    if own:
        from hbfsim_amd.kvcache import KvCache
        st["cache"] = KvCache.from_tensors(st["keys"], st["values"], st["key_scale"],
                                           st["value_scale"], st["bounds"], st["weight"],
                                           head_dim=d)
    return st


# ---- the plain forms ------------------------------------------------------


def _key_codes(keys, d):
    """[n, kv, tiles, chunks, 4, 16, 16] -> float32 [n, kv, tokens, d]."""
    n, kv, tiles, chunks = keys.shape[:4]
    x = keys.permute(0, 1, 2, 5, 3, 4, 6).reshape(n, kv, tiles * 16, chunks * 64)
    return x[..., :d].float()


def _value_codes(values, d):
    n, kv, tiles, chunks = values.shape[:4]
    x = values.permute(0, 1, 2, 4, 7, 3, 6, 5).reshape(n, kv, tiles * 16, chunks * 64)
    return x[..., :d].float()


def _seq_of(st):
    """(sequence, tokens before it in the batch, its own tokens) of every token of the step."""
    n = st["q"].shape[0]
    i = torch.arange(n, device=st["q"].device)
    if st["first"] is None:
        return i, i, torch.ones_like(i)
    first = st["first"].long()
    seq = torch.searchsorted(first[1:].contiguous(), i, right=True)
    return seq, first[seq], first[seq + 1] - first[seq]


def _limits(st, seq=None):
    """How many tokens of its sequence each query token sees."""
    s, before, m = _seq_of(st)
    i = torch.arange(s.shape[0], device=s.device)
    return st["lens"].long()[s] - m + (i - before) + 1


def _quantise(x, inv):
    return torch.nan_to_num(torch.round(x * inv), nan=0.0).clamp(-127, 127)


def _plain_append(st):
    t, d, kv = st["case"]["block"], st["case"]["head_dim"], st["case"]["kv_heads"]
    touched = st["touched"].long()
    n, dev = touched.shape[0], touched.device
    seq, _, _ = _seq_of(st)
    pos = _limits(st) - 1
    phys = st["table"][seq, pos // t].long()
    row_of = torch.zeros(st["keys"].shape[0], dtype=torch.int64, device=dev)
    row_of[touched] = torch.arange(n, device=dev)
    row, slot = row_of[phys], pos % t
    is_new = torch.zeros((n, t), dtype=torch.bool, device=dev)
    is_new[row, slot] = True
    begun = is_new[:, 0].logical_not()  # the block held tokens before the step
    is_new = is_new[:, None, :, None]
    outs = []
    for x, pool, scales, codes_of in ((st["k"], st["keys"], st["key_scale"], _key_codes),
                                      (st["v"], st["values"], st["value_scale"], _value_codes)):
        fresh = torch.zeros((n, t, kv, d), device=dev)
        fresh[row, slot] = x.float()
        fresh = fresh.transpose(1, 2)
        s = fresh.abs().amax((2, 3)) * INV127
        s = torch.where(s <= SCALE_MAX, s.clamp(min=SCALE_MIN), math.nan)
        before = scales[touched]
        s = torch.where(begun[:, None], torch.maximum(before, s), s)
        ratio = torch.where(begun[:, None], before / s, 0.0)[:, :, None, None]
        old = _quantise(codes_of(pool[touched], d), ratio)
        code = torch.where(is_new, _quantise(fresh, torch.reciprocal(s)[:, :, None, None]), old)
        scales[touched] = s
        tiles, chunks = pool.shape[2:4]
        wide = torch.zeros((n, kv, t, chunks * 64), device=dev)
        wide[..., :d] = code
        wide = wide.to(torch.int8)
        if codes_of is _key_codes:
            pool[touched] = wide.view(n, kv, tiles, 16, chunks, 4, 16).permute(0, 1, 2, 4, 5, 3, 6)
            b = st["bounds"][touched].float()[..., :d]
            b = _quantise(b, ratio)
            lo = torch.where(is_new, code, 127.0).amin(2)
            hi = torch.where(is_new, code, -127.0).amax(2)
            lo = torch.where(begun[:, None, None], torch.minimum(b[:, :, 0], lo), lo)
            hi = torch.where(begun[:, None, None], torch.maximum(b[:, :, 1], hi), hi)
            kept = torch.zeros((n, kv, 2, chunks * 64), device=dev)
            kept[:, :, 0, :d], kept[:, :, 1, :d] = lo, hi
            st["bounds"][touched] = kept.to(torch.int8)
        else:
            pool[touched] = wide.view(n, kv, tiles, 4, 4, chunks, 4, 16).permute(0, 1, 2, 5, 3, 7, 6, 4)
        outs.append((code * s[:, :, None, None]).to(torch.bfloat16))
        if codes_of is _key_codes:
            ends = [(x * s[:, :, None]).to(torch.bfloat16) for x in (lo, hi)]
    return {"k": outs[0], "v": outs[1], "low": ends[0], "high": ends[1]}


def _plain_attend(st):
    c = st["case"]
    t, d, kv, h = c["block"], c["head_dim"], c["kv_heads"], c["heads"]
    g, dev = h // kv, st["q"].device
    seqs, width = st["table"].shape
    ids = st["table"].clamp(min=0).long()
    seq, before, _ = _seq_of(st)
    tokens, most = seq.shape[0], st["longest_new"]
    sees = _limits(st)
    row = torch.arange(tokens, device=dev) - before
    q = torch.zeros((seqs, most, h, d), device=dev)
    q[seq, row] = st["q"].float()
    q = q.view(seqs, most, kv, g, d).permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * g, d)
    limit = torch.zeros((seqs, most), dtype=torch.int64, device=dev)
    limit[seq, row] = sees
    k = _key_codes(st["keys"][ids.view(-1)], d).mul_(st["key_scale"][ids.view(-1)][:, :, None, None])
    k = k.view(seqs, width, kv, t, d).transpose(1, 2).reshape(seqs, kv, width * t, d)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(st["scale"]).view(seqs, kv, most, g, width * t)
    del k
    v = _value_codes(st["values"][ids.view(-1)], d)
    v = v.mul_(st["value_scale"][ids.view(-1)][:, :, None, None])
    v = v.view(seqs, width, kv, t, d).transpose(1, 2).reshape(seqs, kv, width * t, d)
    at = torch.arange(width * t, device=dev)
    ok = (at < limit[:, :, None])[:, None]  # [seqs, 1 or kv, most, tokens]
    if c.get("count"):
        sel = st["selected"].long()
        chosen = torch.zeros((tokens, kv, width + 1), dtype=torch.bool, device=dev)
        chosen.scatter_(2, torch.where(sel < 0, width, sel), True)
        wide = torch.zeros((seqs, most, kv, width), dtype=torch.bool, device=dev)
        wide[seq, row] = chosen[:, :, :width]
        wide = wide.transpose(1, 2)
        ok = ok & wide[..., None].expand(*wide.shape, t).reshape(seqs, kv, most, width * t)
    s = torch.where(ok[:, :, :, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    del s
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-37)
    out = torch.matmul(p.reshape(seqs, kv, most * g, width * t), v)
    out = out.view(seqs, kv, most, g, d).permute(0, 2, 1, 3, 4).reshape(seqs, most, h, d)[seq, row]
    out = {"out": out.to(st["q"].dtype)}
    if c.get("accumulate"):
        live = torch.zeros((seqs, most), device=dev)
        live[seq, row] = 1.0
        by_block = (p.sum(3) * live[:, None, :, None]).sum(2).view(seqs, kv, width, t).sum(3)
        by_block = torch.where(st["table"][:, None] >= 0, by_block, 0.0).transpose(1, 2)
        total = torch.zeros(st["weight"].shape, device=dev)
        total.index_add_(0, ids.view(-1), by_block.reshape(seqs * width, kv))
        st["weight"] = torch.round(total.double() / WEIGHT_UNIT).long()
        out["weight"] = total
    return out


def _plain_select(st):
    c = st["case"]
    t, d, kv, count = c["block"], c["head_dim"], c["kv_heads"], c["count"]
    seqs, width = st["table"].shape
    dev = st["q"].device
    seq, before, _ = _seq_of(st)
    tokens, most = seq.shape[0], st["longest_new"]
    sees = _limits(st)
    nb = ((sees.clamp(min=0) + t - 1) // t).clamp(max=width)[:, None, None]
    q = st["q"].float().view(tokens, kv, -1, d)
    s = (q.abs().amax((2, 3)) * INV127).clamp(min=2.0 ** -100)
    code = _quantise(q, torch.reciprocal(s)[:, :, None, None])
    code = torch.cat([code.clamp(max=0).sum(2), code.clamp(min=0).sum(2)], 2)  # with low, with high
    row = torch.arange(tokens, device=dev) - before
    qp = torch.zeros((seqs, most, kv, 2 * d), device=dev)
    qp[seq, row] = code
    ids = st["table"].clamp(min=0).long().view(-1)
    b = st["bounds"][ids][..., :d].float().reshape(seqs, width, kv, 2 * d).permute(0, 2, 3, 1)
    score = torch.matmul(qp.transpose(1, 2), b)  # whole numbers
    score = score.transpose(1, 2)[seq, row]
    score = score * st["key_scale"][ids].view(seqs, width, kv).transpose(1, 2)[seq]
    i = torch.arange(width, device=dev)
    forced = (i < 1) | (i >= nb - 1)
    score = torch.where(forced | torch.isnan(score), math.inf, score)
    score = torch.where((i < nb) & (st["table"][seq] >= 0)[:, None], score, -math.inf)
    score, at = torch.sort(score, dim=2, descending=True, stable=True)
    k = min(count, width)
    at = torch.where(score[:, :, :k] > -math.inf, at[:, :, :k], width).sort(dim=2).values
    out = torch.full((tokens, kv, count), -1, dtype=torch.int32, device=dev)
    out[:, :, :k] = torch.where(at < width, at, -1).to(torch.int32)
    return {"selected": out}


def _plain_evict(st):
    c = st["case"]
    t, keep = c["block"], c["keep"]
    table = st["table"]
    seqs, width = table.shape
    dev = table.device
    lens = st["lens"].long()
    nb = ((lens + t - 1) // t).clamp(max=width)[:, None]
    i = torch.arange(width, device=dev)
    score = st["weight"].sum(1)[table.clamp(min=0).long()]
    score = torch.where(table >= 0, score, -1)
    big = torch.iinfo(torch.int64).max
    score = torch.where((i < 1) | (i >= nb - 1), big, score)
    score = torch.where(i < nb, score, -2)
    order = torch.sort(score, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, i.expand(seqs, width).contiguous())
    inside = i < nb
    kept = inside & (rank < keep)
    freed = inside & ~kept

    def pack(mask):
        at = torch.where(mask, i, width).sort(dim=1).values
        got = torch.gather(table, 1, at.clamp(max=width - 1))
        return torch.where(at < width, got, -1)

    gone = freed.sum(1)
    return {"table": pack(kept), "lens": (lens - gone * t).to(torch.int32), "freed": pack(freed),
            "freed_count": gone.to(torch.int32)}


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select,
                "evict": _plain_evict}[kind](state)
    if kind == "evict":
        from hbfsim_amd import kvcache
        table, lens, freed, count = kvcache.evict(state["weight"], state["table"], state["lens"],
                                                  c["keep"], block_tokens=c["block"])
        return {"table": table, "lens": lens, "freed": freed, "freed_count": count}
    cache = state["cache"]
    if kind == "append":
        cache.append(state["k"], state["v"], state["table"], state["lens"], state["first"])
        k, v, low, high = cache.read(state["touched"], torch.bfloat16)
        return {"k": k, "v": v, "low": low, "high": high}
    if kind == "attend":
        if not c.get("accumulate"):
            return {"out": cache.attend(state["q"], state["table"], state["lens"], state["first"],
                                        selected=state.get("selected"))}
        cache.weight.zero_()  # this step's weights alone
        out = cache.attend(state["q"], state["table"], state["lens"], state["first"],
                           accumulate=True)
        return {"out": out, "weight": cache.weights()}
    return {"selected": cache.select(state["q"], state["table"], state["lens"], c["count"],
                                     state["first"])}


# ---- the definition in 64 bits --------------------------------------------


def _whole(pool, block, kv, d, values):
    """One sequence's codes [tokens, d] of one kv head, from its blocks' ids."""
    x = pool[block, kv]  # [n, tiles, chunks, 4, 16, ...]
    n, tiles, chunks = x.shape[:3]
    if values:
        x = x.permute(0, 1, 3, 6, 2, 5, 4)
    else:
        x = x.permute(0, 1, 4, 2, 3, 5)
    return x.reshape(n * tiles * 16, chunks * 64)[:, :d].double()


def exact(case, seed):
    if case["kind"] in ("select", "evict"):
        return None
    st = prepare(case, seed)
    lens, new = _lengths(case)
    t, d, kv, h = case["block"], case["head_dim"], case["kv_heads"], case["heads"]
    g, dev = h // kv, st["table"].device
    if case["kind"] == "append":
        outs = {"k": [], "v": [], "low": None, "high": None}
        slots = _touched(case)
        first = [0]
        for m in new:
            first.append(first[-1] + m)
        # where each touched block's slots come from: a token of the step, or -1
        src = torch.full((len(slots), t), -1, dtype=torch.int64)
        for r, (s, b) in enumerate(slots):
            lo, hi = max(b * t, lens[s] - new[s]), min((b + 1) * t, lens[s])
            src[r, lo - b * t:hi - b * t] = torch.arange(lo, hi) - (lens[s] - new[s]) + first[s]
        src = src.to(dev)
        isnew, begun = (src >= 0)[:, None, :, None], (src[:, 0] < 0)[:, None, None, None]
        ids = st["touched"].long()
        for name, x, pool, sc in (("k", st["k"], st["keys"], st["key_scale"]),
                                  ("v", st["v"], st["values"], st["value_scale"])):
            got = x.double()[src.clamp(min=0)].transpose(1, 2) * isnew  # [n, kv, t, d]
            s = got.abs().amax((2, 3), keepdim=True) / 127
            was = sc[ids].double()[:, :, None, None]
            s = torch.where(begun, torch.maximum(s, was), s)
            old = torch.stack([_whole(pool, ids, j, d, name == "v").view(-1, t, d)
                               for j in range(kv)], 1)
            old = torch.where(begun, torch.round(old * was / s), 0.0)
            code = torch.where(isnew, torch.round(got / s), old)
            outs[name] = code * s
            if name == "k":
                b = torch.round(st["bounds"][ids].double()[..., :d] * was / s)
                lo = torch.where(isnew, code, 1e3).amin(2)
                hi = torch.where(isnew, code, -1e3).amax(2)
                w = begun[:, :, 0]
                outs["low"] = torch.where(w, torch.minimum(lo, b[:, :, 0]), lo) * s[:, :, 0]
                outs["high"] = torch.where(w, torch.maximum(hi, b[:, :, 1]), hi) * s[:, :, 0]
        return outs
    out = torch.zeros((sum(new), h, d), dtype=torch.float64, device=dev)
    weight = torch.zeros(st["weight"].shape, dtype=torch.float64, device=dev)
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        nb = -(-n // t)
        ids = st["table"][s, :nb].long()
        sees = n - m + 1 + torch.arange(m, device=dev)
        for j in range(kv):
            if not nb:
                continue
            k = _whole(st["keys"], ids, j, d, False).view(nb, t, d)
            k = (k * st["key_scale"][ids, j].double()[:, None, None]).view(nb * t, d)
            v = _whole(st["values"], ids, j, d, True).view(nb, t, d)
            v = (v * st["value_scale"][ids, j].double()[:, None, None]).view(nb * t, d)
            ok = torch.arange(nb * t, device=dev)[None] < sees[:, None]
            if case.get("count"):
                pick = st["selected"][at:at + m, j].long()
                inlist = torch.zeros((m, nb + 1), dtype=torch.bool, device=dev)
                inlist.scatter_(1, torch.where(pick < 0, nb, pick), True)
                ok &= inlist[:, :nb].repeat_interleave(t, 1)
            for a in range(g):
                x = st["q"][at:at + m, j * g + a].double() @ k.T / math.sqrt(d)
                x = x.masked_fill(~ok, -math.inf)
                x = torch.nan_to_num(torch.softmax(x, 1), nan=0.0)
                out[at:at + m, j * g + a] = x @ v
                if case.get("accumulate"):
                    weight[:, j].index_add_(0, ids, x.sum(0).view(nb, t).sum(1))
        at += m
    if case.get("accumulate"):
        return {"out": out, "weight": weight}
    return {"out": out}
