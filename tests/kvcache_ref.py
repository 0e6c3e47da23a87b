"""The paged 8-bit cache's operators from their definitions, on the CPU.

Codes, scales and selections follow the definition's own float32 steps one by
one (numpy rounds each operation as IEEE asks), so they are compared exactly;
attention is computed in float64 from the codes, with a bound on what the
kernels' float32 sums and 11-bit probabilities may differ by.
"""
from __future__ import annotations

import math

import numpy as np
import torch

F = np.float32
INV127 = F(1.0 / 127.0)


class RefCache:
    """Codes in natural order: keys and values [blocks, kv, tokens, dim]."""

    def __init__(self, blocks, kv, dim, tokens):
        self.shape = (blocks, kv, tokens, dim)
        self.codes = [np.zeros(self.shape, np.int8) for _ in range(2)]
        self.scale = [np.ones((blocks, kv), F) for _ in range(2)]
        self.bounds = np.zeros((blocks, kv, 2, dim), np.int8)
        self.weight = np.zeros((blocks, kv), np.int64)

    def append(self, k, v, table, lens, first=None):
        """k, v float32 [tokens, kv, dim]; loops over the definition."""
        blocks, kv, t, _ = self.shape
        width = table.shape[1]
        first = list(range(len(lens) + 1)) if first is None else first
        for s, n in enumerate(lens):
            m = first[s + 1] - first[s]
            if m <= 0 or n - m < 0:
                continue
            for b in range((n - m) // t, -(-n // t)):
                ident = table[s, b] if b < width else -1
                if not 0 <= ident < blocks:
                    continue
                lo, hi = max(n - m, b * t), min(n, (b + 1) * t)
                rows = slice(first[s] + lo - (n - m), first[s] + hi - (n - m))
                for h in range(kv):
                    for which, x in enumerate((k, v)):
                        self._store(ident, h, which, x[rows, h], lo - b * t, hi - b * t)

    def _store(self, ident, h, which, x, lo, hi):
        begun = lo > 0
        with np.errstate(all="ignore"):
            top = F(np.max(np.abs(x))) if np.isfinite(x).all() else F(np.nan)
            s = F(top * INV127)
            s = max(s, F(2.0 ** -40)) if s <= F(2.0 ** 40) else F(np.nan)
            ratio = F(0)
            if begun:
                was = self.scale[which][ident, h]
                s = F(np.nan) if np.isnan(was) or np.isnan(s) else max(was, s)
                ratio = F(was / s)
            inv = F(F(1) / s)
            self.scale[which][ident, h] = s
            code = self.codes[which][ident, h]
            code[:] = quantise(code.astype(F), ratio) if begun else 0
            new = quantise(x, inv)
            code[lo:hi] = new
            if which == 0:
                b = self.bounds[ident, h]
                low, high = new.min(0), new.max(0)
                if begun:
                    old = quantise(b.astype(F), ratio)
                    low, high = np.minimum(low, old[0]), np.maximum(high, old[1])
                else:
                    self.weight[ident, h] = 0
                b[0], b[1] = low, high

    def select(self, q, table, lens, count, first=None, keep_first=1, keep_last=1):
        blocks, kv, t, dim = self.shape
        tokens, heads, _ = q.shape
        g = heads // kv
        first = list(range(len(lens) + 1)) if first is None else first
        out = np.full((tokens, kv, count), -1, np.int32)
        for s, n in enumerate(lens):
            m = first[s + 1] - first[s]
            for i in range(m):
                seen = n - m + i + 1
                nb = min(-(-max(seen, 0) // t), table.shape[1])
                ids = table[s, :nb]
                live = (ids >= 0) & (ids < blocks)
                for h in range(kv):
                    x = np.nan_to_num(q[first[s] + i, h * g:(h + 1) * g], posinf=np.inf,
                                      neginf=-np.inf)
                    with np.errstate(all="ignore"):
                        sq = max(F(np.abs(x).max() * INV127), F(2.0 ** -100))
                        c = quantise(x, F(F(1) / sq)).astype(np.int64)
                    b = self.bounds[np.where(live, ids, 0), h].astype(np.int64)
                    whole = np.maximum(c[None] * b[:, None, 0], c[None] * b[:, None, 1]).sum((1, 2))
                    score = whole.astype(F) * self.scale[0][np.where(live, ids, 0), h]
                    score = np.where(np.isnan(score), np.inf, score)
                    at = np.arange(nb)
                    always = (at < keep_first) | (at + keep_last >= nb)
                    order = [j for j in sorted(at, key=lambda j: (not always[j], -score[j], j))
                             if live[j]]
                    got = sorted(order[:count])
                    out[first[s] + i, h, :len(got)] = got
        return out

    def attend(self, q, table, lens, first=None, selected=None, scale=None):
        """(out, bound on each output's error before its own rounding, weight
        [blocks, kv], bound on it), float64."""
        blocks, kv, t, dim = self.shape
        tokens, heads, _ = q.shape
        g = heads // kv
        scale = dim ** -0.5 if scale is None else scale
        first = list(range(len(lens) + 1)) if first is None else first
        out = np.zeros((tokens, heads, dim))
        bound = np.zeros((tokens, heads, dim))
        weight = np.zeros((blocks, kv))
        wbound = np.zeros((blocks, kv))
        q = q.astype(np.float64)
        for s, n in enumerate(lens):
            m = first[s + 1] - first[s]
            nb = min(-(-max(n, 0) // t), table.shape[1])
            ids = table[s, :nb].astype(np.int64)
            live = (ids >= 0) & (ids < blocks)
            for h in range(kv):
                at = np.where(live, ids, 0)
                with np.errstate(all="ignore"):
                    k, v = ((self.codes[w][at, h].astype(np.float64) *
                             self.scale[w][at, h].astype(np.float64)[:, None, None])
                            .reshape(nb * t, dim) for w in (0, 1))
                logv = np.abs(np.log2(np.where(live, self.scale[1][at, h], 1)))
                for i in range(m):
                    seen = n - m + i + 1
                    pos = np.arange(nb * t)
                    ok = (pos < seen) & np.repeat(live, t)
                    if selected is not None:
                        ok &= np.isin(pos // t, selected[first[s] + i, h])
                    if not ok.any():
                        continue
                    kk, vv = k[ok], v[ok]
                    for a in range(g):
                        x = q[first[s] + i, h * g + a]
                        z = scale * (kk @ x)
                        size = np.max(np.abs(scale) * (np.abs(kk) @ np.abs(x)))
                        p = np.exp(z - z.max())
                        p /= p.sum()
                        # f32 sums of dim products, the exponent's own rounding
                        # (scores and log2 of the value scales), exp2 and the sum
                        eps = 2 * (dim * 2.0 ** -24 * size +
                                   4 * 2.0 ** -24 * (1.45 * size + logv.max() + 16) +
                                   len(z) * 2.0 ** -24 + 2.0 ** -21)
                        mass = p @ np.abs(vv)
                        out[first[s] + i, h * g + a] = p @ vv
                        # 11 bits of each probability, and the smallest f16 below them
                        bound[first[s] + i, h * g + a] = (2.0 ** -11 + eps) * mass + \
                            len(z) * 2.0 ** -31 * np.abs(vv).max() + 1e-30
                        full = np.zeros(nb * t)
                        full[ok] = p
                        per = full.reshape(nb, t).sum(1)
                        np.add.at(weight, (at, h), per)
                        np.add.at(wbound, (at, h), per * 2 * eps + 2.0 ** -31)
        return out, bound, weight, wbound


def quantise(x, inv):
    with np.errstate(all="ignore"):
        r = np.rint((x * inv).astype(F))
    return np.clip(np.nan_to_num(r, nan=0.0), -127, 127).astype(np.int8)


def evict(weight, table, lens, keep, tokens, keep_first=1, keep_last=1):
    blocks = weight.shape[0]
    seqs, width = table.shape
    out, freed = np.full((2, seqs, width), -1, np.int32)
    left, count = np.zeros((2, seqs), np.int32)
    for s, n in enumerate(lens):
        nb = min(-(-max(int(n), 0) // tokens), width)
        ids = table[s, :nb]

        def key(i):
            if i < keep_first or i + keep_last >= nb:
                return math.inf
            return int(weight[ids[i]].sum()) + 1 if 0 <= ids[i] < blocks else 0

        kept = sorted(sorted(range(nb), key=lambda i: (-key(i), i))[:keep])
        gone = [i for i in range(nb) if i not in set(kept)]
        out[s, :len(kept)] = ids[kept]
        freed[s, :len(gone)] = ids[gone]
        left[s], count[s] = n - len(gone) * tokens, len(gone)
    return out, left, freed, count


def codes_of(cache):
    """A KvCache's keys and values in natural order, padding included."""
    k, v = cache.keys.cpu(), cache.values.cpu()
    n, kv, tiles, chunks = k.shape[:4]
    k = k.permute(0, 1, 2, 5, 3, 4, 6).reshape(n, kv, tiles * 16, chunks * 64)
    v = v.permute(0, 1, 2, 4, 7, 3, 6, 5).reshape(n, kv, tiles * 16, chunks * 64)
    return k.numpy(), v.numpy()


def fill(cache, ref, rng, blocks=None, spread=0.3):
    """Random codes, scales and bounds, the same in both."""
    n, kv, t, dim = ref.shape
    for w in (0, 1):
        ref.codes[w][:] = np.clip(np.rint(rng.normal(0, 34, ref.shape)), -127, 127)
        ref.scale[w][:] = (np.exp(rng.normal(0, spread, (n, kv))) / 36).astype(F)
    ref.bounds[:, :, 0], ref.bounds[:, :, 1] = ref.codes[0].min(2), ref.codes[0].max(2)
    upload(cache, ref)


def upload(cache, ref):
    n, kv, t, dim = ref.shape
    dims = -(-dim // 64) * 64
    wide = [np.zeros((n, kv, t, dims), np.int8) for _ in range(2)]
    for w in (0, 1):
        wide[w][..., :dim] = ref.codes[w]
    k, v = (torch.from_numpy(x) for x in wide)
    k = k.view(n, kv, t // 16, 16, dims // 64, 4, 16).permute(0, 1, 2, 4, 5, 3, 6)
    v = v.view(n, kv, t // 16, 4, 4, dims // 64, 4, 16).permute(0, 1, 2, 5, 3, 7, 6, 4)
    cache.keys.copy_(k)
    cache.values.copy_(v)
    b = np.zeros((n, kv, 2, dims), np.int8)
    b[..., :dim] = ref.bounds
    cache.bounds.copy_(torch.from_numpy(b))
    cache.key_scale.copy_(torch.from_numpy(ref.scale[0]))
    cache.value_scale.copy_(torch.from_numpy(ref.scale[1]))
    cache.weight.copy_(torch.from_numpy(ref.weight))


def make_table(rng, lens, tokens, blocks, width=None):
    need = [-(-max(n, 0) // tokens) for n in lens]
    width = max(1, max(need, default=1)) if width is None else width
    perm = rng.permutation(blocks)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    return table
