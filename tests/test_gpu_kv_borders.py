"""The operators on a paged cache's blocks on both sides of where their forms
change, against the definitions (kvpages_ref): whole numbers or moved bytes,
equal or wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvpages_ref as pr
from hbfsim_amd import kvcache
from test_gpu_kvpages import batch, dev, filled, grow_both, moved, same
from test_gpu_verify import check, steps

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1023, 1024, 1025])
@pytest.mark.parametrize("two", [False, True])
def test_copy_of_pairs_around_one_launch(n, two):
    """Up to 1,024 pairs every workgroup looks through them itself."""
    rng = np.random.default_rng(n)
    cache, was = filled(1600, 2, 64, 16, 1)
    other, was_other = filled(900, 2, 64, 16, 2) if two else (cache, was)
    src, dst = rng.integers(-1, 1601, n), rng.integers(-1, other.blocks + 1, n)
    cache.copy(dev(src), dev(dst), to=other if two else None)
    same(other, moved(was_other, pr.copy_pairs(src, dst, 1600, other.blocks, not two), was))


@pytest.mark.parametrize("rows,width", [(1024, 7), (1025, 8), (1025, 9), (1152, 9), (1153, 9)])
def test_fork_around_both_ways_of_counting(rows, width):
    """Children are looked for up to 1,024 rows, or 128 a table entry."""
    rng = np.random.default_rng(rows + width)
    table, _ = batch(rng, 60, width, 600)
    lens, parents = rng.integers(0, 99, 60), rng.integers(-1, 61, rows)
    refs = pr.count(table, 600)
    got = dev(refs)
    out, out_lens = kvcache.fork(got, dev(table), dev(lens), dev(parents))
    want, want_lens = pr.fork(refs, table, lens, parents)
    np.testing.assert_array_equal(out.cpu(), want)
    np.testing.assert_array_equal(out_lens.cpu(), want_lens)
    np.testing.assert_array_equal(got.cpu(), refs)


@pytest.mark.parametrize("blocks", [4095, 4096, 4097, 8191, 8192, 8193, 65537])
@pytest.mark.parametrize("start", [0, 1])
@pytest.mark.parametrize("used", ["random", "back"])
def test_compact_around_one_workgroup(blocks, start, used):
    """One workgroup plans pools of up to 8,192 blocks, 4,096 in a round;
    counts at any address."""
    rng = np.random.default_rng(blocks)
    refs = rng.integers(-1, 3, blocks).astype(np.int32)
    if used == "back":
        refs[:] = 0
        refs[blocks // 2 + 3:] = 1
    cache, was = filled(blocks, 1, 64, 16, 7)
    buffer = torch.zeros(start + blocks, dtype=torch.int32, device="cuda")
    cache.refs = buffer[start:]
    cache.refs.copy_(dev(refs))
    table = rng.integers(-1, blocks + 1, (5, 300)).astype(np.int32)
    got = dev(table)
    where = cache.compact(got)
    want, pairs = pr.compact(refs, table)
    np.testing.assert_array_equal(where.cpu(), want)
    np.testing.assert_array_equal(got.cpu(), table)
    np.testing.assert_array_equal(cache.refs.cpu(), refs)
    same(cache, moved(was, pairs))


@pytest.mark.parametrize("blocks", [65535, 65536, 65537, 100_001])
@pytest.mark.parametrize("seqs", [200, 1024, 1025, 2500])
@pytest.mark.parametrize("enough", [True, False])
def test_grow_in_pools_around_the_counted_ones(blocks, seqs, enough):
    """Free blocks are counted by tiles of 8,192 in pools above 65,536, for a
    slot a thread and for more: free ones in several tiles, some tiles without
    one, rows that share blocks, enough blocks and too few."""
    rng = np.random.default_rng(blocks + seqs)
    table = np.full((seqs, 3), -1, np.int32)
    table[:, :2] = rng.permutation(blocks)[:2 * seqs].reshape(seqs, 2)
    table[1::3, :2] = table[0::3, :2][:len(table[1::3])]  # every third row shares the one before
    lens = rng.integers(16, 33, seqs)
    need = 2 * seqs
    refs = np.ones(blocks, np.int32)
    spread = np.concatenate([np.arange(8192), np.arange(3 * 8192, 5 * 8192),
                             np.arange(7 * 8192 + 5, blocks)])
    spread = spread[~np.isin(spread, table)]
    refs[rng.permutation(spread)[:need if enough else seqs // 4]] = rng.integers(-1, 1)
    held = pr.count(table, blocks)
    refs = np.where(held > 0, held, refs).astype(np.int32)
    cache = kvcache.KvCache(blocks, 1, 64)
    cache.refs.copy_(dev(refs))
    cache.weight.copy_(torch.arange(blocks, device="cuda")[:, None])
    got = dev(table)
    now, missing = cache.grow(got, dev(lens + 1))
    out, lacks, pairs = pr.grow(refs, table, lens + 1, 16)
    np.testing.assert_array_equal(now.cpu(), out)
    np.testing.assert_array_equal(missing.cpu(), lacks)
    np.testing.assert_array_equal(got.cpu(), table)
    np.testing.assert_array_equal(cache.refs.cpu(), refs)
    weight = np.arange(blocks)
    for a, b in pairs:
        weight[b] = a
    np.testing.assert_array_equal(cache.weight.cpu()[:, 0], weight)
    assert pairs and lacks.any() == (not enough)


@pytest.mark.parametrize("kv,dim,t,seqs", [(1, 64, 16, 9001), (8, 128, 16, 3000), (2, 64, 128, 2731)])
def test_grow_copies_more_parts_than_there_are_workgroups(kv, dim, t, seqs):
    """8,192 workgroups take the planned copies' parts in turn: of one part a
    block, and of three."""
    table = np.full((seqs, 2), -1, np.int32)
    table[:, 0] = np.arange(seqs) // 2
    blocks = (seqs + 1) // 2 + seqs // 2
    cache, was = filled(blocks, kv, dim, t, 3, pr.count(table, blocks))
    missing, pairs = grow_both(cache, was, table, np.full(seqs, 7))
    assert not missing.any() and len(pairs) == seqs // 2


@pytest.mark.parametrize("dtype,vocab", [("f32", 8191), ("f32", 8192), ("f32", 8193), ("bf16", 16_383),
                                         ("bf16", 16_384), ("bf16", 16_385), ("f16", 16_384),
                                         ("f16", 16_385), ("bf16", 16_388)])
def test_verify_around_one_workgroup(dtype, vocab):
    """Rows of up to 8,192 floats, or twice that of two bytes, are one
    workgroup's."""
    rng = np.random.default_rng(vocab)
    check(*steps(rng, [3, 1, 4, 2, 0, 5], vocab, dtype))


@pytest.mark.parametrize("dtype,vocab", [("f32", 20_480), ("bf16", 40_960), ("f32", 20_477)])
@pytest.mark.parametrize("seqs", [74, 75])
def test_verify_around_four_loads_a_wave(dtype, vocab, seqs):
    """A load a wave below 1,500 waves of four."""
    rng = np.random.default_rng(vocab + seqs)
    check(*steps(rng, rng.integers(1, 3, seqs), vocab, dtype))
