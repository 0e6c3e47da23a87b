"""Rows of a step that belong to no sequence: a batch padded to a captured
step's size, or one that starts behind other rows."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvcache_ref as kr
from test_gpu_kvcache import check_attend, ints, pair, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,g,dim,t,lens,new", [
    (2, 4, 128, 16, [300, 0, 77], [5, 0, 3]),      # few rows, one split
    (1, 3, 37, 16, [5000, 333], [2, 1]),           # several splits, odd dims
    (1, 40, 64, 32, [2000, 50], [1, 2]),           # several row tiles
    (2, 2, 80, 16, [400, 150], [300, 150]),        # many rows
    (1, 8, 256, 64, [3000], [12]),                 # many rows, several splits
    (1, 1, 64, 16, [0, 0], [0, 0])])               # no sequence has a token
@pytest.mark.parametrize("before,after", [(0, 40), (3, 0), (29, 1)])
def test_rows_of_no_sequence_are_zeros(kv, g, dim, t, lens, new, before, after):
    rng = np.random.default_rng(dim + before)
    blocks = sum(-(-n // t) for n in lens) + 1
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table = kr.make_table(rng, lens, t, blocks)
    first = before + np.concatenate([[0], np.cumsum(new)])
    tokens = int(first[-1]) + after
    if tokens == 0:
        return
    q, qn = rows(rng, (tokens, kv * g, dim), "bf16", 2.0)
    rest = np.ones(tokens, bool)
    rest[first[0]:first[-1]] = False
    chosen = cache.select(q, ints(table), ints(lens), 4, ints(first))
    assert (chosen.cpu().numpy()[rest] == -1).all()
    for kw in ({}, {"selected": chosen.cpu().numpy()}, {"accumulate": True}):
        out = torch.full((tokens, kv * g, dim), 9.0, dtype=torch.bfloat16, device="cuda")
        got, weight, wbound = check_attend(cache, ref, q, qn, table, lens, first, out=out, **kw)
        assert got is out and not out.cpu()[torch.from_numpy(rest)].any()
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= wbound + 2.0 ** -24 * weight).all()


def test_a_sequence_that_ends_past_the_step_s_rows():
    """Its rows and those of later ones come back as zeros, the others as ever."""
    rng = np.random.default_rng(71)
    kv, g, dim, t = 1, 4, 64, 16
    lens = [100, 200, 300]
    blocks = sum(-(-n // t) for n in lens)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table = kr.make_table(rng, lens, t, blocks)
    q, qn = rows(rng, (50, g, dim), "f16", 2.0)
    for first in ([0, 20, 45, 60], [0, 20, 60, 70], [0, 20, 51, 51]):
        out = torch.full((50, g, dim), 9.0, dtype=torch.float16, device="cuda")
        cache.attend(q, ints(table), ints(lens), ints(first), out=out)
        kept = max(f for f in first if f <= 50)
        n = first.index(kept)
        want = cache.attend(q[:kept], ints(table[:n]), ints(lens[:n]), ints(first[:n + 1]))
        assert torch.equal(out[:kept], want) and not out[kept:].any()


@pytest.mark.parametrize("at", [0, 7, 300])
def test_a_step_of_no_sequences(at):
    kv, g, dim = 2, 3, 80
    cache, _ = pair(kv, dim, 16, 4)
    q, _ = rows(np.random.default_rng(72), (300, kv * g, dim), "bf16")
    table = torch.zeros((0, 5), dtype=torch.int32, device="cuda")
    out = torch.full((300, kv * g, dim), 9.0, dtype=torch.bfloat16, device="cuda")
    for kw in ({}, {"accumulate": True}):
        assert not cache.attend(q, table, ints([]), ints([at]), out=out.fill_(9), **kw).any()
    assert (cache.select(q, table, ints([]), 3, ints([at])) == -1).all()
    assert not cache.weight.any()
