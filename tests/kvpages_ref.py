"""The operators on a paged cache's blocks and the verification of drafted
tokens from their definitions, on the CPU: one entry, one block, one sequence at
a time, in whole numbers.
"""
from __future__ import annotations

import math
from fractions import Fraction

import numpy as np

ARRAYS = ("keys", "values", "key_scale", "value_scale", "bounds", "weight")


def inside(x, n):
    return 0 <= int(x) < n


def count(table, blocks):
    refs = np.zeros(blocks, np.int32)
    hold(refs, table)
    return refs


def hold(refs, table):
    for b in np.asarray(table).reshape(-1):
        if inside(b, len(refs)):
            refs[b] += 1


def fork(refs, table, lens, parents):
    """Changes refs; returns the next batch's table and lengths."""
    out = np.full((len(parents), table.shape[1]), -1, np.int32)
    out_lens = np.zeros(len(parents), np.int32)
    for i, p in enumerate(parents):
        if inside(p, len(table)):
            out[i], out_lens[i] = table[p], lens[p]
    for b in table.reshape(-1):
        if inside(b, len(refs)):
            refs[b] -= 1
    hold(refs, out)
    return out, out_lens


def release(refs, table, lens, t):
    """Changes refs and table."""
    for s in range(len(table)):
        n = 0 if lens is None else max(0, int(lens[s]))
        for i in range(-(-n // t), table.shape[1]):
            if inside(table[s, i], len(refs)):
                refs[table[s, i]] -= 1
            table[s, i] = -1


def grow(refs, table, lens, t, first=None, tokens=None):
    """Changes refs and table; returns (lens, missing, [(source, destination)])."""
    seqs, width = table.shape
    tokens = seqs if first is None else tokens
    first = list(range(seqs + 1)) if first is None else [int(x) for x in first]
    writes, outside = {}, {}  # by sequence: (place, begun); how many past the table
    for s in range(seqs):
        m, n = first[s + 1] - first[s], int(lens[s])
        if m <= 0 or first[s] < 0 or first[s] + m > tokens or n < m:
            continue
        places = range((n - m) // t, -(-n // t))
        outside[s] = sum(b >= width for b in places)
        writes[s] = [] if outside[s] else [(b, b * t < n - m) for b in places]

    def named(s, b):
        return inside(table[s, b], len(refs))

    def used(s, b):
        return named(s, b) and refs[table[s, b]] > 0

    writers = {}
    for s in sorted(writes):
        for b, _ in writes[s]:
            if used(s, b):
                writers.setdefault(int(table[s, b]), []).append((s, b))
    free = [b for b in range(len(refs)) if refs[b] <= 0]

    def needs(s, share):
        out = []
        for b, begun in writes[s]:
            if not used(s, b):
                if not begun:
                    out.append(b)
                continue
            e = int(table[s, b])
            last = share and len(writers[e]) >= refs[e] and writers[e][-1] == (s, b)
            if refs[e] > 1 and not last:
                out.append(b)
        return out

    share = sum(len(needs(s, True)) for s in writes) <= len(free)
    plan = {s: needs(s, share) for s in sorted(writes)}
    out_lens, missing = np.array(lens, np.int32), np.zeros(seqs, np.int32)
    asked, granted = 0, []
    for s in plan:
        asked += len(plan[s])
        if outside[s]:
            missing[s] = outside[s]
        elif plan[s] and asked > len(free):
            missing[s] = len(plan[s])
        else:
            granted.append(s)
        if missing[s]:
            out_lens[s] = 0
    pairs, at, changes = [], 0, []
    for s in plan:
        if s in granted:
            for b, begun in writes[s]:
                if begun and named(s, b) and not used(s, b):
                    changes.append((s, b, -1))
            for k, b in enumerate(plan[s]):
                changes.append((s, b, free[at + k]))
                if used(s, b) and dict(writes[s])[b]:
                    pairs.append((int(table[s, b]), free[at + k]))
        at += len(plan[s])
    was = {(s, b): used(s, b) for s, b, _ in changes}
    for s, b, new in changes:
        if was[s, b] and new >= 0:
            refs[table[s, b]] -= 1
        if new >= 0:
            refs[new] = 1
        table[s, b] = new
    return out_lens, missing, pairs


def compact(refs, table):
    """Changes refs and table; returns (where, [(source, destination)])."""
    live = [b for b in range(len(refs)) if refs[b] > 0]
    front = len(live)
    pairs = list(zip([b for b in live if b >= front],
                     [b for b in range(front) if refs[b] <= 0]))
    where = np.full(len(refs), -1, np.int32)
    where[live] = live
    for src, dst in pairs:
        where[src] = dst
    for s in range(len(table)):
        for i, b in enumerate(table[s]):
            table[s, i] = where[b] if inside(b, len(refs)) else -1
    for src, dst in pairs:
        refs[dst], refs[src] = refs[src], 0
    return where, pairs


def copy_pairs(src, dst, blocks, to_blocks, same):
    """The pairs of a copy that count."""
    pairs = [(int(a), int(b)) for a, b in zip(src, dst)
             if inside(a, blocks) and inside(b, to_blocks)]
    written = {b for _, b in pairs}
    out, seen = [], set()
    for a, b in pairs:
        if b not in seen:
            seen.add(b)
            if not (same and a in written):
                out.append((a, b))
    return out


def share(x):
    x = float(x)
    return 0.0 if math.isnan(x) else min(max(x, 0.0), 1.0)


def whole(x):
    """2^40 x to the nearest whole number, ties to even; x of 24 bits, so that
    the product is exact in float64."""
    x = np.clip(np.nan_to_num(np.asarray(x, np.float64), nan=0.0), 0.0, 1.0)
    return np.rint(x * 2.0 ** 40).astype(np.int64)


def verify(target, tokens, uniform, first=None, draft=None, lens=None):
    """target, draft float32 [rows, vocab] that hold the values of their type.
    Returns (out, gained, lens)."""
    rows, vocab = target.shape
    seqs = rows if first is None else len(first) - 1
    first = list(range(seqs + 1)) if first is None else [int(x) for x in first]
    out = np.full(rows, -1, np.int32)
    gained = np.zeros(seqs, np.int32)
    left = None if lens is None else np.array(lens, np.int32)
    for s in range(seqs):
        begin, n = first[s], first[s + 1] - first[s]
        if left is not None:
            left[s] -= n
        if n <= 0 or begin < 0 or begin + n > rows:
            continue
        stays, refused = 0, None
        while stays < n - 1:
            r, x = begin + stays, int(tokens[begin + stays + 1])
            if not inside(x, vocab):
                break
            q = 1.0 if draft is None else share(draft[r, x])
            u = float(uniform[r])
            if math.isnan(u) or not Fraction(u) * Fraction(q) < Fraction(share(target[r, x])):
                refused = x
                break
            stays += 1
        r = begin + stays
        full = whole(target[r])
        weight = full.copy()
        if refused is not None and draft is None:
            weight[refused] = 0
        elif refused is not None:
            weight = np.maximum(0, full - whole(draft[r]))
        if not weight.any():
            weight = full
        upto = np.cumsum(weight)  # below 2^63
        k = min(int(Fraction(share(uniform[begin + n - 1])) * 2 ** 31), 2 ** 31 - 1)
        k = k * int(upto[-1]) >> 31
        token = int(np.argmax(upto > k)) if upto[-1] else -1
        out[begin:begin + stays] = tokens[begin + 1:begin + 1 + stays]
        out[r] = token
        gained[s] = stays + 1
        if left is not None:
            left[s] += stays + 1
    return out, gained, left
