"""The paged cache's operators where their sizes choose another form of the
work: many query rows, many splits, rows enough for a workgroup each, tables
too wide for LDS."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvcache_ref as kr
from hbfsim_amd import kvcache
from test_gpu_kvcache import check_attend, dev, ints, pair, rows

pytestmark = pytest.mark.gpu


def filled(rng, kv, dim, t, lens, spread=0.3, spare=1):
    blocks = sum(-(-n // t) for n in lens) + spare
    table = kr.make_table(rng, lens, t, blocks)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng, spread=spread)
    return cache, ref, table


@pytest.mark.parametrize("kv,g,dim,t,dtype", [(1, 4, 37, 16, "bf16"), (2, 3, 192, 32, "f16"),
                                              (1, 48, 128, 16, "bf16"), (1, 200, 64, 64, "f16"),
                                              (2, 1, 256, 128, "bf16"), (2, 2, 256, 32, "bf16"),
                                              (1, 130, 256, 16, "f16")])
def test_many_rows_of_odd_shapes(kv, g, dim, t, dtype):
    """Odd dims and groups that leave rows of a workgroup empty, or need one
    token each; a long and a short sequence, and one whose queries see less
    than they are."""
    rng = np.random.default_rng(dim + g)
    lens, new = [400, 75, 50], [150, 75, 60]
    first = np.concatenate([[0], np.cumsum(new)])
    cache, ref, table = filled(rng, kv, dim, t, lens)
    q, qn = rows(rng, (int(first[-1]), kv * g, dim), dtype, 2.0)
    got, _, _ = check_attend(cache, ref, q, qn, table, lens, first, dtype=dtype)
    assert not got[225:235].any() and got[235].any()


@pytest.mark.parametrize("scale", [0.0, -0.05, 3.0])
def test_many_rows_scale_arguments(scale):
    rng = np.random.default_rng(51)
    kv, g, dim, t = 1, 4, 128, 16
    lens, first = [500], [0, 130]
    cache, ref, table = filled(rng, kv, dim, t, lens, spread=4.0)
    q, qn = rows(rng, (130, g, dim), "bf16", 1.0)
    check_attend(cache, ref, q, qn, table, lens, first, scale=scale)


def test_many_rows_scores_that_rise_late():
    """References have to move up by far more than the f16 range, tile after
    tile, and down at once for rows whose first scores are far below zero."""
    rng = np.random.default_rng(52)
    kv, g, dim, t = 1, 2, 64, 16
    lens, first = [900], [0, 200]
    cache, ref, table = filled(rng, kv, dim, t, lens)
    order = table[0, :-(-900 // t)]
    ramp = np.linspace(0.05, 6.0, len(order)).astype(np.float32)
    ref.codes[0][order] = np.abs(ref.codes[0][order])
    ref.scale[0][order] = (ramp / 36)[:, None]
    kr.upload(cache, ref)
    for sign in (1, -1):
        q, qn = rows(rng, (200, g, dim), "bf16", 1.0)
        q, qn = sign * q.abs(), sign * np.abs(qn)
        check_attend(cache, ref, q, qn, table, lens, first, scale=0.5)
        # one token a sequence takes the other form through the same ramp
        check_attend(cache, ref, q[:1], qn[:1], table, lens, scale=0.5)


def test_many_rows_holes_and_nan_scales():
    rng = np.random.default_rng(53)
    kv, g, dim, t = 2, 2, 64, 32
    lens, first = [420], [0, 140]
    cache, ref, table = filled(rng, kv, dim, t, lens, spare=3)
    table[0, 2], table[0, 5] = -1, cache.blocks + 7
    q, qn = rows(rng, (140, kv * g, dim), "bf16", 2.0)
    got, _, _ = check_attend(cache, ref, q, qn, table, lens, first)
    # the block of tokens 352..383: queries 0..71 end before it, and tokens 280.. see it
    block = int(table[0, 11])
    for scales in (cache.key_scale, cache.value_scale):
        keep = scales[block, 1].clone()
        scales[block, 1] = float("nan")
        after = cache.attend(q, ints(table), ints(lens), ints(first))
        scales[block, 1] = keep
        assert torch.equal(after[:, :g], got[:, :g])
        assert torch.equal(after[:72], got[:72])
        assert torch.isnan(after[72:, g:]).all()
    # a query that is not finite spoils its own row alone
    q[17, 3, 0] = float("inf")
    after = cache.attend(q, ints(table), ints(lens), ints(first))
    assert torch.isnan(after[17, 3]).all()
    after[17, 3] = got[17, 3]
    assert torch.equal(after, got)


@pytest.mark.parametrize("kv,g,dim,t", [(1, 4, 64, 16), (1, 20, 192, 32), (2, 1, 128, 128)])
def test_many_splits_with_weights(kv, g, dim, t):
    rng = np.random.default_rng(54)
    lens = [9001, 0, 4500]
    cache, ref, table = filled(rng, kv, dim, t, lens, spread=1.0)
    q, qn = rows(rng, (3, kv * g, dim), "bf16", 2.0)
    _, weight, wbound = check_attend(cache, ref, q, qn, table, lens, accumulate=True)
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= wbound + 2.0 ** -24 * weight).all()
    # a few tokens each take 16-row units of several tokens
    lens, first = [9001, 0, 4500], [0, 3, 3, 5]
    q, qn = rows(rng, (5, kv * g, dim), "f16", 2.0)
    cache.weight.zero_()
    _, weight, wbound = check_attend(cache, ref, q, qn, table, lens, first, dtype="f16",
                                     accumulate=True)
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= wbound + 2.0 ** -24 * weight).all()


def test_weights_skip_holes_and_sums_that_are_not_numbers():
    rng = np.random.default_rng(55)
    kv, g, dim, t = 2, 2, 64, 16
    lens = [100, 90]
    cache, ref, table = filled(rng, kv, dim, t, lens)
    table[0, 3] = -1
    q, qn = rows(rng, (2, kv * g, dim), "bf16", 2.0)
    q[1, 0, 0] = float("nan")  # head 0 of sequence 1
    cache.attend(q, ints(table), ints(lens), accumulate=True)
    got = cache.weights()
    _, _, weight, wbound = ref.attend(np.nan_to_num(qn), table, lens)
    fine = np.abs(got.double().cpu().numpy() - weight) <= wbound + 2.0 ** -24 * weight
    spoiled = np.zeros_like(fine)
    spoiled[table[1, :6], 0] = True
    assert fine[~spoiled].all()
    assert not got.cpu().numpy()[table[1, :6], 0].any()


@pytest.mark.parametrize("kv,g,dim,t,seqs,dtype", [(8, 4, 128, 16, 20, "bf16"),
                                                   (2, 16, 64, 32, 64, "f16"),
                                                   (1, 3, 200, 16, 130, "bf16")])
def test_select_one_workgroup_a_row(kv, g, dim, t, seqs, dtype):
    rng = np.random.default_rng(seqs)
    lens = [int(x) for x in rng.integers(0, 700, seqs)]
    lens[0], lens[1] = 0, 1
    cache, ref, table = filled(rng, kv, dim, t, lens)
    table[5, :2] = -1
    q, qn = rows(rng, (seqs, kv * g, dim), dtype, 2.0)
    for count, keep in ((9, (1, 1)), (2, (1, 1)), (20, (0, 3)), (60, (2, 2))):
        got = cache.select(q, ints(table), ints(lens), count, None, *keep)
        np.testing.assert_array_equal(got.cpu().numpy(),
                                      ref.select(qn, table, lens, count, None, *keep))


@pytest.mark.parametrize("blocks", [3000, 40_000])
def test_select_over_wide_tables(blocks):
    """One sequence over a table whose keys fit LDS, and one whose do not."""
    rng = np.random.default_rng(blocks)
    kv, g, dim, t = 1, 2, 64, 16
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table = rng.permutation(blocks).astype(np.int32)[None]
    lens = [blocks * t - 5]
    q, qn = rows(rng, (1, g, dim), "bf16", 2.0)
    for count in (2, 77, blocks - 1, blocks):
        got = cache.select(q, ints(table), ints(lens), count)
        np.testing.assert_array_equal(got.cpu().numpy(), ref.select(qn, table, lens, count))


def test_select_tells_tokens_of_a_group_apart():
    """Eight query tokens share a pass over the bounds; their choices are
    those of each alone."""
    rng = np.random.default_rng(57)
    kv, g, dim, t = 2, 4, 128, 16
    lens, first = [2000, 333], [0, 21, 34]
    cache, ref, table = filled(rng, kv, dim, t, lens)
    q, qn = rows(rng, (34, kv * g, dim), "f16", 2.0)
    q[3] *= 100
    qn[3] *= 100
    qn = q.float().cpu().numpy()
    got = cache.select(q, ints(table), ints(lens), 13, ints(first))
    np.testing.assert_array_equal(got.cpu().numpy(), ref.select(qn, table, lens, 13, first))


def test_append_of_every_block_size_at_every_slot():
    """A token into each slot of a block that then has to grow its scale."""
    rng = np.random.default_rng(58)
    for t in (16, 32, 64, 128):
        kv, dim = 2, 80
        cache, ref = pair(kv, dim, t, t)
        table = np.arange(t, dtype=np.int32)[:, None]
        lens = np.arange(1, t + 1)
        first = np.concatenate([[0], np.cumsum(lens)])
        x, xn = rows(rng, (int(first[-1]), kv, dim), "f16")
        cache.append(x, x, ints(table), ints(lens), ints(first))
        ref.append(xn, xn, table, lens, first)
        keep = lens < t
        lens = lens + keep
        first = np.concatenate([[0], np.cumsum(keep)])
        x, xn = rows(rng, (int(first[-1]), kv, dim), "f16", 4.0)
        cache.append(x, x, ints(table), ints(lens), ints(first))
        ref.append(xn, xn, table, lens, first)
        for got, want in zip(kr.codes_of(cache), ref.codes):
            np.testing.assert_array_equal(got[..., :dim], want)
        np.testing.assert_array_equal(cache.key_scale.cpu().numpy(), ref.scale[0])
        np.testing.assert_array_equal(cache.bounds.cpu().numpy()[..., :dim], ref.bounds)


def test_evict_first_and_last_alone():
    """keep no larger than what is always kept: nothing competes."""
    rng = np.random.default_rng(59)
    weight = rng.integers(0, 9, (50, 2)).astype(np.int64)
    table = kr.make_table(rng, [400, 30], 16, 50)
    for keep, first, last in ((3, 1, 2), (1, 0, 1), (5, 2, 3)):
        got = kvcache.evict(dev(weight), ints(table), ints([400, 30]), keep, 16, first, last)
        want = kr.evict(weight, table, [400, 30], keep, 16, first, last)
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("new", [1, 300])
def test_weights_far_below_the_largest_still_count(dim, new):
    """One token 21.5 bits above 30,000 others, whose weights lie below the
    normal numbers of 16 bits: they are a hundredth of the denominator and all
    of the second half of the dims.  Their rounding is at most 2^-10 of them,
    the largest's and the output's 2^-11."""
    n, t = 30_000, 16
    k = torch.zeros((n + 1, 1, dim))
    v = torch.ones((n + 1, 1, dim))
    k[0, 0, 0] = 21.5 * np.log(2)
    v[0, 0, dim // 2:] = 0
    blocks = -(-(n + 1) // t)
    cache = kvcache.KvCache(blocks, 1, dim, t)
    table, lens = ints(np.arange(blocks)[None]), ints([n + 1])
    cache.append(k.cuda(), v.cuda(), table, lens, ints([0, n + 1]))
    q = torch.zeros((new, 1, dim), dtype=torch.float16)
    q[:, 0, 0] = 1
    got = cache.attend(q.cuda(), table, lens, ints([0, new]), scale=1.0)[-1, 0].double().cpu()
    rest = n * 2.0 ** -21.5
    want = torch.ones(dim, dtype=torch.float64)
    want[dim // 2:] = rest / (1 + rest)
    assert ((got - want).abs() <= 2.0 ** -8 * want).all(), (got - want).abs().max()
