"""Accumulated block weights: what a query that is not finite leaves out does
not depend on how the kernels group its rows."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvcache_ref as kr
from test_gpu_kvcache import ints, pair, rows

pytestmark = pytest.mark.gpu


def gains(ref, qn, table, lens, first, without):
    """Weight of a step and its bound, less what the (row, kv head) pairs of
    `without` add."""
    _, _, weight, bound = ref.attend(qn, table, lens, first)
    for row, head in without:
        s = int(np.searchsorted(first, row, side="right")) - 1
        seen = lens[s] - (first[s + 1] - first[s]) + (row - first[s]) + 1
        _, _, own, _ = ref.attend(qn[row:row + 1], table[s:s + 1], [seen])
        weight[:, head] -= own[:, head]
    return weight, bound


@pytest.mark.parametrize("kv,g,dim,t,lens,new,bad", [
    # (row, query head) pairs that are not finite
    (2, 2, 64, 16, [300, 90], [1, 1], [(1, 0)]),
    (2, 2, 64, 32, [300, 90], [11, 5], [(3, 1), (12, 3)]),           # 8 tokens a unit
    (1, 20, 80, 16, [200, 100], [2, 1], [(1, 17)]),                  # two row tiles
    (2, 2, 128, 16, [350, 80], [150, 80], [(0, 0), (77, 1), (200, 2)]),  # many rows
    (1, 20, 64, 64, [300], [60], [(9, 3), (59, 19)]),                # and two row tiles again
    (1, 3, 256, 16, [200], [40], [(20, 2)])])
def test_a_token_that_is_not_a_number_adds_nothing(kv, g, dim, t, lens, new, bad):
    rng = np.random.default_rng(dim + g)
    first = np.concatenate([[0], np.cumsum(new)])
    blocks = sum(-(-n // t) for n in lens)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table = kr.make_table(rng, lens, t, blocks)
    q, qn = rows(rng, (int(first[-1]), kv * g, dim), "bf16", 1.0)
    for i, (row, head) in enumerate(bad):
        q[row, head, 1 + i] = (float("nan"), float("inf"))[i % 2]
    cache.attend(q, ints(table), ints(lens), ints(first), accumulate=True)
    weight, bound = gains(ref, qn, table, lens, first, {(r, h // g) for r, h in bad})
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= bound + 2.0 ** -24 * weight).all(), diff.max()


@pytest.mark.parametrize("new", [6, 100])
@pytest.mark.parametrize("which", ["key_scale", "value_scale"])
def test_tokens_that_see_a_block_of_nan_scale_add_nothing(new, which):
    rng = np.random.default_rng(new)
    kv, g, dim, t, n = 2, 2, 64, 16, 240
    cache, ref = pair(kv, dim, t, n // t)
    kr.fill(cache, ref, rng)
    table = kr.make_table(rng, [n], t, n // t)
    q, qn = rows(rng, (new, kv * g, dim), "f16", 1.0)
    at = n - new // 2 - 2  # a token that the step's first half does not see
    getattr(cache, which)[int(table[0, at // t]), 1] = float("nan")
    cache.attend(q, ints(table), ints([n]), ints([0, new]), accumulate=True)
    without = {(i, 1) for i in range(new) if n - new + i >= at // t * t}
    assert 0 < len(without) <= new and (new == 6 or len(without) < new)
    weight, bound = gains(ref, qn, table, [n], np.array([0, new]), without)
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= bound + 2.0 ** -24 * np.abs(weight)).all(), diff.max()


@pytest.mark.parametrize("kv,g,dim,t,dtype", [(2, 1, 64, 16, "f16"), (1, 3, 64, 128, "bf16"),
                                              (1, 20, 128, 16, "f16"), (2, 3, 100, 128, "bf16"),
                                              (1, 48, 192, 16, "bf16"), (2, 3, 170, 32, "f16"),
                                              (1, 1, 256, 128, "bf16"), (2, 20, 256, 16, "f16"),
                                              (1, 48, 230, 64, "bf16")])
def test_weights_of_many_rows(kv, g, dim, t, dtype):
    """The second pass over the keys: every count of dims, both types, groups
    of one, several and more than 16 heads, blocks of one tile and more, holes,
    a shared block, a sequence without tokens and a row that is not finite."""
    rng = np.random.default_rng(dim * g)
    room = 4 * (5 - -(-dim // 64)) * 16          # rows of a many-row workgroup
    m = -(-13 * room // (10 * g)) + 3
    assert 2 * m * g * 5 >= room * 3 * 4         # or the step takes the other form
    lens, new = [m + 2 * t + 45, m + 5, 0], [m, m, 0]
    first = np.concatenate([[0], np.cumsum(new)])
    blocks = sum(-(-n // t) for n in lens) + 1
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng, spread=1.0)
    table = kr.make_table(rng, lens, t, blocks)
    table[0, 1], table[1, 0] = -1, table[0, 0]
    q, qn = rows(rng, (2 * m, kv * g, dim), dtype, 1.5)
    q[m // 2, g - 1, 3] = float("nan")
    cache.attend(q, ints(table), ints(lens), ints(first), accumulate=True)
    weight, bound = gains(ref, qn, table, lens, first, {(m // 2, 0)})
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= bound + 2.0 ** -24 * weight).all(), diff.max()


@pytest.mark.parametrize("new", [1, 5, 90])
def test_output_in_place_of_the_queries(new):
    rng = np.random.default_rng(81)
    kv, g, dim, t, n = 2, 3, 128, 16, 900
    cache, ref = pair(kv, dim, t, -(-n // t))
    kr.fill(cache, ref, rng)
    table, lens = ints(kr.make_table(rng, [n], t, -(-n // t))), ints([n])
    first = None if new == 1 else ints([0, new])
    q, _ = rows(rng, (new, kv * g, dim), "bf16", 1.0)
    want = cache.attend(q, table, lens, first)
    x = q.clone()
    assert cache.attend(x, table, lens, first, out=x) is x and torch.equal(x, want)
    x = q.clone()
    if first is not None:
        with pytest.raises(ValueError):
            cache.attend(x, table, lens, first, accumulate=True, out=x)
        assert torch.equal(x, q) and not cache.weight.any()
        with pytest.raises(ValueError):
            cache.attend(x[1:], table, lens, ints([0, new - 1]), out=x[:-1])
    else:
        cache.attend(q, table, lens, accumulate=True)
        once = cache.weight.clone()
        assert torch.equal(cache.attend(x, table, lens, accumulate=True, out=x), want)
        assert torch.equal(cache.weight, 2 * once)
