"""The operators on a paged cache's blocks on the GPU against their definitions
(kvpages_ref).  Everything is whole numbers or moved bytes: equal, or wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvpages_ref as pr
from hbfsim_amd import kvcache

pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.array(x, np.int32)).cuda()


def strided(x, extra=0):
    """The table as rows of a wider buffer of 77s."""
    wide = torch.full((x.shape[0], x.shape[1] + extra), 77, dtype=torch.int32, device="cuda")
    wide[:, :x.shape[1]] = dev(x)
    return wide[:, :x.shape[1]], wide


def filled(blocks, kv=2, dim=64, t=16, seed=0, refs=None):
    """A cache whose every byte is random, and its arrays on the host."""
    cache = kvcache.KvCache(blocks, kv, dim, t)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for name in pr.ARRAYS:
        x = getattr(cache, name)
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda") if x.is_floating_point() else
                torch.randint(-128, 127, x.shape, generator=gen, device="cuda"))
    if refs is not None:
        cache.refs.copy_(dev(refs))
    return cache, host(cache)


def host(cache):
    return {name: getattr(cache, name).cpu().numpy() for name in pr.ARRAYS}


def moved(was, pairs, source=None):
    """The arrays after the copies, all read before any is written."""
    want = {name: x.copy() for name, x in was.items()}
    for name, x in (source or was).items():
        for a, b in pairs:
            want[name][b] = x[a]
    return want


def same(cache, want):
    for name, x in host(cache).items():
        np.testing.assert_array_equal(x, want[name], err_msg=name)


def batch(rng, seqs, width, blocks, most=None, holes=True):
    """Rows that share prefixes and name each block as a batch may: some holes,
    some entries of no pool; (table, blocks per row)."""
    order = rng.permutation(blocks)[:most]
    table = np.full((seqs, width), -1, np.int32)
    n = rng.integers(0, width + 1, seqs)
    at = 0
    for s in range(seqs):
        common = 0
        if s and rng.random() < 0.5:
            p = rng.integers(0, s)
            common = int(min(n[p], n[s], rng.integers(0, width + 1)))
            table[s, :common] = table[p, :common]
        own = min(int(n[s]) - common, len(order) - at)
        table[s, common:common + own] = order[at:at + own]
        n[s] = common + own
        at += own
    if holes and seqs * width:
        for x in (-1, -7, blocks, 2 ** 31 - 1, -2 ** 31):
            table[rng.integers(0, seqs), rng.integers(0, width)] = x
    return table, n


# ---- hold, fork, release ------------------------------------------------------


@pytest.mark.parametrize("seqs,width,rows,extra", [(1, 1, 1, 0), (5, 40, 9, 3), (64, 130, 64, 0),
                                                   (3, 1025, 700, 1), (300, 7, 2, 0), (4, 2500, 5, 8),
                                                   (6, 9, 0, 0), (2, 0, 3, 0), (0, 4, 3, 0),
                                                   (1500, 2, 1600, 1), (40, 8, 1025, 0)])
def test_hold_and_fork(seqs, width, rows, extra):
    rng = np.random.default_rng(seqs * 7 + width)
    blocks = max(3, seqs * width)
    table, _ = batch(rng, seqs, width, blocks)
    lens = rng.integers(-3, 50, seqs).astype(np.int32)
    parents = rng.integers(-2, seqs + 2, rows).astype(np.int32)
    got_table, _ = strided(table, extra)
    refs, want = torch.zeros(blocks, dtype=torch.int32, device="cuda"), pr.count(table, blocks)
    kvcache.hold(refs, got_table)
    np.testing.assert_array_equal(refs.cpu(), want)
    out, out_lens = kvcache.fork(refs, got_table, dev(lens), dev(parents))
    want_table, want_lens = pr.fork(want, table, lens, parents)
    np.testing.assert_array_equal(out.cpu(), want_table)
    np.testing.assert_array_equal(out_lens.cpu(), want_lens)
    np.testing.assert_array_equal(refs.cpu(), want)
    np.testing.assert_array_equal(got_table.cpu(), table)  # the old table is only read
    np.testing.assert_array_equal(want, pr.count(want_table, blocks))


@pytest.mark.parametrize("t", [16, 128])
@pytest.mark.parametrize("seqs,width,extra", [(1, 1, 0), (7, 33, 5), (64, 1024, 0), (3, 2051, 2),
                                              (1, 0, 0), (0, 3, 0)])
def test_release(seqs, width, extra, t):
    rng = np.random.default_rng(seqs + width)
    blocks = max(3, seqs * width)
    table, n = batch(rng, seqs, width, blocks)
    lens = np.maximum(0, n * t - rng.integers(0, 3 * t, seqs)).astype(np.int32)
    lens[::5] = 0
    lens[1::5] = -9
    lens[2::7] = 2 ** 31 - 1
    refs = pr.count(table, blocks)
    got_refs = dev(refs)
    got_table, wide = strided(table, extra)
    kvcache.release(got_refs, got_table, dev(lens), block_tokens=t)
    pr.release(refs, table, lens, t)
    np.testing.assert_array_equal(got_table.cpu(), table)
    np.testing.assert_array_equal(got_refs.cpu(), refs)
    assert (wide[:, width:] == 77).all()
    kvcache.release(got_refs, got_table)
    assert not got_refs.any() and (got_table == -1).all() and (wide[:, width:] == 77).all()


def test_what_evict_frees_is_released():
    rng = np.random.default_rng(2)
    cache, _ = filled(200)
    cache.weight.random_(0, 1 << 40)
    table = dev(rng.permutation(200)[:180].reshape(6, 30))
    lens = dev([480, 479, 465, 1, 0, 300])
    cache.hold(table)
    kept, left, freed, gone = cache.evict(table, lens, keep=11)
    cache.release(freed)
    assert int((freed >= 0).sum()) == 0 and int(gone.sum()) > 0
    used = kept.cpu().numpy()
    cache_refs = cache.refs.cpu().numpy()
    # evict's table names the blocks of its lengths; those past them were never in it
    past = table.cpu().numpy().copy()
    for s, n in enumerate(lens.tolist()):
        past[s, :-(-n // 16)] = -1
    np.testing.assert_array_equal(cache_refs, pr.count(used, 200) + pr.count(past, 200))
    assert int(left.sum()) == int(lens.sum()) - 16 * int(gone.sum())


# ---- copy ---------------------------------------------------------------------


@pytest.mark.parametrize("kv,dim,t", [(2, 64, 16), (8, 128, 16), (1, 37, 128), (5, 192, 32),
                                      (3, 256, 64), (1024, 1, 16)])
@pytest.mark.parametrize("two", [False, True])
def test_copy(kv, dim, t, two):
    rng = np.random.default_rng(kv + dim)
    cache, was = filled(40, kv, dim, t, 1)
    other, was_other = filled(23, kv, dim, t, 2) if two else (cache, was)
    ids = rng.permutation(40)
    src, dst = ids[:13], (rng.permutation(23)[:13] if two else ids[20:33])
    cache.copy(dev(src), dev(dst), to=other if two else None)
    pairs = pr.copy_pairs(src, dst, 40, other.blocks, not two)
    assert len(pairs) == 13
    same(other, moved(was_other, pairs, was))
    if two:
        same(cache, was)


@pytest.mark.parametrize("n", [1, 2, 30, 700, 5000])
@pytest.mark.parametrize("two", [False, True])
def test_copy_of_ids_that_repeat_or_are_none(n, two):
    """The first of the pairs with one destination copies, a block that is
    written is no source, ids outside the pools count for nothing."""
    rng = np.random.default_rng(n)
    blocks = 2 * n + 5
    cache, was = filled(blocks, 1, 64, 16, 3)
    other, was_other = filled(n + 2, 1, 64, 16, 4) if two else (cache, was)
    src = rng.integers(-1, blocks + 1, n)
    dst = rng.integers(-1, other.blocks + 1, n)
    src[n // 2:n // 2 + 1], dst[-1:] = -2 ** 31, 2 ** 31 - 1
    for _ in range(2):  # whatever an earlier call left in the scratch memory
        cache.copy(dev(src), dev(dst), to=other if two else None)
    pairs = pr.copy_pairs(src, dst, blocks, other.blocks, not two)
    same(other, moved(was_other, pairs, was))
    cache.copy(dev([]), dev([]))
    same(other, moved(was_other, pairs, was))


def test_copy_onto_itself_and_in_a_ring():
    cache, was = filled(4, 1, 64, 16, 5)
    cache.copy(dev([0, 1, 2, 3]), dev([0, 2, 3, 1]))
    same(cache, was)  # every source is written


def test_copy_past_2_31_bytes():
    """Blocks whose bytes lie beyond 32-bit offsets, in a pool of 4.4 GB of codes."""
    blocks = 8500
    cache = kvcache.KvCache(blocks, 8, 256, 128)
    assert cache.keys.numel() > 2 ** 31
    for name in pr.ARRAYS:
        getattr(cache, name)[7] = 5
        getattr(cache, name)[blocks - 1] = 3
    cache.copy(dev([7, blocks - 1]), dev([blocks - 2, 1]))
    for name in pr.ARRAYS:
        x = getattr(cache, name)
        assert (x[blocks - 2] == 5).all() and (x[1] == 3).all() and (x[blocks - 1] == 3).all()
        assert (x[blocks - 3] == x[8]).all() and (x[2] == x[8]).all()


# ---- grow -----------------------------------------------------------------------


def grow_both(cache, was, table, lens, first=None, tokens=None, extra=0):
    t, refs = cache.block_tokens, cache.refs.cpu().numpy().copy()
    got_table, wide = strided(table, extra)
    width = table.shape[1]
    got = cache.grow(got_table, dev(lens), None if first is None else dev(first), tokens)
    out, missing, pairs = pr.grow(refs, table, lens, t, first, tokens)
    np.testing.assert_array_equal(got[0].cpu(), out)
    np.testing.assert_array_equal(got[1].cpu(), missing)
    np.testing.assert_array_equal(got_table.cpu(), table)
    np.testing.assert_array_equal(cache.refs.cpu(), refs)
    assert (wide[:, width:] == 77).all()
    same(cache, moved(was, pairs))
    return missing, pairs


@pytest.mark.parametrize("kv,dim,t", [(2, 64, 16), (1, 100, 128), (3, 128, 32)])
@pytest.mark.parametrize("seqs,width,new", [(1, 3, 1), (9, 6, 1), (70, 5, 9), (40, 12, 200),
                                            (1500, 3, 1), (2, 90, 1500), (600, 4, 40)])
@pytest.mark.parametrize("spare", [0.02, 0.4, 3.0])
def test_grow(kv, dim, t, seqs, width, new, spare):
    """One token and chunks of tokens each, rows that share prefixes, pools
    with too few, just enough and many free blocks."""
    rng = np.random.default_rng(seqs + width + new + int(10 * spare))
    used = seqs * width // 2 + 1
    blocks = used + max(1, int(spare * seqs * (new // t + 1)))
    table, n = batch(rng, seqs, width, blocks, used)
    stored = np.maximum(0, n * t - rng.integers(0, t, seqs)) * (rng.random(seqs) < 0.9)
    stored = np.where(rng.random(seqs) < 0.1, stored // 2, stored)  # behind its own blocks
    many = np.ones(seqs, np.int64) if new == 1 else rng.integers(0, new + 1, seqs)
    first = None if new == 1 else np.concatenate([[0], np.cumsum(many)])
    refs = pr.count(table, blocks)
    refs[rng.integers(0, blocks, 2)] *= rng.integers(0, 2)  # named, yet free
    refs[refs == 0] -= rng.integers(0, 2, int((refs == 0).sum()))
    cache, was = filled(blocks, kv, dim, t, 6, refs)
    lens = stored + many
    lens[rng.random(seqs) < 0.05] = 0  # fewer than the step's tokens
    missing, pairs = grow_both(cache, was, table, lens, first,
                               None if first is None else int(first[-1]), extra=3)
    if seqs == 1500:
        assert pairs and (missing.any() if spare < 0.1 else True)


def test_grow_after_a_fork_leaves_the_last_its_block():
    """Four branches of one sequence write to its last block: three copies, and
    with another holder that does not write four."""
    for others in (0, 1):
        rows = np.array([[3, 5, 9, -1]] * (4 + others), np.int32)
        cache, was = filled(20, refs=pr.count(rows, 20))
        lens = np.array([42] * 4 + [0] * others)  # of the last no token is stored
        first = np.array([0, 1, 2, 3, 4] + [4] * others)
        _, pairs = grow_both(cache, was, rows, lens, first, 4)
        assert [a for a, _ in pairs] == [9] * (3 + others)
        assert cache.refs[9] == 1 and (rows[3, 2] == 9) == (others == 0)


def test_grow_with_too_few_blocks_parts_with_nothing():
    """Two of three branches could be served if one kept the shared block, but
    who lacks a block still holds it."""
    rows = np.array([[0, 1], [0, 1], [0, 1]], np.int32)
    refs = pr.count(rows, 3)
    cache, was = filled(3, refs=refs)
    table = rows.copy()
    missing, pairs = grow_both(cache, was, table, np.array([20, 20, 20]))
    assert missing.tolist() == [0, 1, 1] and pairs == [(1, 2)]
    # what it lacked it gets once the first ends
    cache.refs.copy_(dev([3, 1, 1]))
    cache.refs[0] = 3
    table = np.array([[0, 2], [0, 1], [-1, -1]], np.int32)
    cache.refs.copy_(dev(pr.count(table, 3)))
    grow_both(cache, host(cache), table, np.array([20, 21, 0]), np.array([0, 1, 2, 2]), 2)


def test_grow_of_what_a_batch_may_not_say():
    """Offsets that go back or end past the rows, more tokens than are stored,
    places past the table: such sequences get nothing and take nothing."""
    table = np.full((7, 3), -1, np.int32)
    cache, was = filled(30)
    lens = np.array([48, 49, 3, 16, 20, 2 ** 31 - 1, -5])
    first = np.array([0, 48, 97, 101, 101, 100, 130, 140])
    grow_both(cache, was, table, lens, first, 120)
    grow_both(cache, host(cache), np.full((0, 3), -1, np.int32), np.zeros(0, int))
    table = np.full((3, 0), -1, np.int32)
    missing, _ = grow_both(cache, host(cache), table, np.array([1, 0, 40]))
    assert missing.tolist() == [1, 0, 1]


@pytest.mark.parametrize("seqs,start", [(1024, 0), (1025, 0), (512, 1), (513, 3), (2000, 1),
                                        (4096, 0), (4097, 0)])
def test_grow_on_both_sides_of_a_thread_a_slot(seqs, start):
    """One token each, and two each with offsets; counts at any address."""
    rng = np.random.default_rng(seqs)
    for new in (1, 2):
        blocks = 3 * seqs
        table, n = batch(rng, seqs, 3, blocks, 2 * seqs)
        cache, was = filled(blocks, 1, 64, 16, 6)
        buffer = torch.zeros(start + blocks, dtype=torch.int32, device="cuda")
        cache.refs = buffer[start:]
        cache.refs.copy_(dev(pr.count(table, blocks)))
        lens = np.minimum(np.maximum(0, n * 16 - rng.integers(0, 16, seqs)) + new, 48)
        first = None if new == 1 else 2 * np.arange(seqs + 1)
        _, pairs = grow_both(cache, was, table, lens, first, None if new == 1 else 2 * seqs)
        assert pairs


def test_grow_in_a_large_pool():
    """Free blocks far apart and behind many that are held."""
    rng = np.random.default_rng(8)
    blocks = 300_000
    refs = np.ones(blocks, np.int32)
    refs[rng.permutation(blocks)[:90]] = 0
    refs[-1] = 0
    cache = kvcache.KvCache(blocks, 1, 64)
    cache.refs.copy_(dev(refs))
    table = np.full((88, 4), -1, np.int32)
    got = dev(table)
    lens = np.full(88, 17)
    first = np.arange(89)
    lens[::2] = 1
    for step in range(2):
        n = lens.copy()
        n[1::2] = 1 if step == 0 else 17
        if step:
            n[::2] = 2
        out, missing, _ = pr.grow(refs, table, n, 16, first, 88)
        a, b = cache.grow(got, dev(n), dev(first), 88)
        np.testing.assert_array_equal(a.cpu(), out)
        np.testing.assert_array_equal(b.cpu(), missing)
        np.testing.assert_array_equal(got.cpu(), table)
        np.testing.assert_array_equal(cache.refs.cpu(), refs)
    assert missing.any() and not (refs == 0).any()


# ---- compact --------------------------------------------------------------------


@pytest.mark.parametrize("kv,dim,t", [(2, 64, 16), (1, 37, 128), (3, 192, 32)])
@pytest.mark.parametrize("blocks,seqs,width", [(1, 1, 1), (2, 1, 1), (50, 4, 9), (1024, 30, 30),
                                               (1025, 3, 20), (5000, 64, 60), (4097, 1, 1500),
                                               (700, 0, 0)])
def test_compact(kv, dim, t, blocks, seqs, width):
    rng = np.random.default_rng(blocks)
    table, _ = batch(rng, seqs, width, blocks, blocks - blocks // 4)
    refs = pr.count(table, blocks)
    refs[rng.integers(0, blocks, blocks // 20)] = rng.integers(-2, 3)  # other tables', and none's
    cache, was = filled(blocks, kv, dim, t, 7, refs)
    got_table, wide = strided(table, 2)
    where = cache.compact(got_table)
    want, pairs = pr.compact(refs, table)
    np.testing.assert_array_equal(where.cpu(), want)
    np.testing.assert_array_equal(got_table.cpu(), table)
    np.testing.assert_array_equal(cache.refs.cpu(), refs)
    assert (wide[:, width:] == 77).all()
    same(cache, moved(was, pairs))
    live = int((refs > 0).sum())
    assert (refs[:live] > 0).all()
    cache.compact(got_table)  # nothing is left to move
    np.testing.assert_array_equal(got_table.cpu(), table)
    same(cache, moved(was, pairs))


@pytest.mark.parametrize("blocks", [65536, 65537, 150_001])
@pytest.mark.parametrize("start", [0, 1])
def test_compact_of_large_pools(blocks, start):
    """On both sides of what one workgroup plans; counts at any address."""
    rng = np.random.default_rng(blocks)
    refs = rng.integers(-1, 3, blocks).astype(np.int32)
    cache = kvcache.KvCache(blocks, 1, 64)
    buffer = torch.zeros(start + blocks, dtype=torch.int32, device="cuda")
    cache.refs = buffer[start:]
    cache.refs.copy_(dev(refs))
    cache.weight.copy_(torch.arange(blocks, device="cuda")[:, None])
    cache.values.view(blocks, -1)[:] = (torch.arange(blocks, device="cuda")[:, None] % 127).to(torch.int8)
    weight = np.arange(blocks)
    table = rng.integers(-1, blocks + 1, (40, 700)).astype(np.int32)
    got = dev(table)
    where = cache.compact(got)
    want, pairs = pr.compact(refs, table)
    for src, dst in pairs:
        weight[dst] = src
    np.testing.assert_array_equal(where.cpu(), want)
    np.testing.assert_array_equal(got.cpu(), table)
    np.testing.assert_array_equal(cache.refs.cpu(), refs)
    np.testing.assert_array_equal(cache.weight.cpu()[:, 0], weight)
    values = cache.values.view(blocks, -1).cpu().numpy()
    assert (values == (weight % 127)[:, None]).all()


@pytest.mark.parametrize("used", ["none", "all", "front", "back", "every other"])
def test_compact_of_one_kind(used):
    blocks = 3000
    refs = np.zeros(blocks, np.int32)
    refs[{"none": slice(0, 0), "all": slice(None), "front": slice(0, 1024),
          "back": slice(1500, None), "every other": slice(1, None, 2)}[used]] = 2
    cache, was = filled(blocks, 1, 64, 16, 9, refs)
    table = np.arange(blocks, dtype=np.int32).reshape(3, 1000)
    got = dev(table)
    where = cache.compact(got)
    want, pairs = pr.compact(refs, table)
    np.testing.assert_array_equal(where.cpu(), want)
    np.testing.assert_array_equal(got.cpu(), table)
    np.testing.assert_array_equal(cache.refs.cpu(), refs)
    same(cache, moved(was, pairs))


# ---- lengths in place, two calls at once --------------------------------------


@pytest.mark.parametrize("seqs", [5, 1300])
def test_grow_writes_the_step_s_lengths_over_the_lengths(seqs):
    """As the C call may: both forms read every length before they write one."""
    import ctypes

    from hbfsim_amd import _native as nat

    rng = np.random.default_rng(seqs)
    blocks = 2 * seqs
    table, n = batch(rng, seqs, 4, blocks, blocks - 3)
    cache, _ = filled(blocks, refs=pr.count(table, blocks))
    refs = cache.refs.cpu().numpy().copy()
    lens = np.maximum(1, n * 16 - rng.integers(0, 16, seqs)) + rng.integers(0, 30, seqs)
    first = np.concatenate([[0], np.cumsum(rng.integers(0, 30, seqs))])
    got, at, offsets = dev(table), dev(lens), dev(first)
    need, missing = ctypes.c_size_t(), torch.empty(seqs, dtype=torch.int32, device="cuda")
    lib, tokens = nat.load(), int(first[-1])
    assert lib.hbfsim_amd_kv_grow_workspace(cache._ref, seqs, tokens, ctypes.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    assert lib.hbfsim_amd_kv_grow(
        cache._ref, cache.refs.data_ptr(), got.data_ptr(), at.data_ptr(), offsets.data_ptr(), seqs,
        tokens, 4, 4, at.data_ptr(), missing.data_ptr(), ws.data_ptr(), need.value,
        torch.cuda.current_stream().cuda_stream) == 0
    out, short, _ = pr.grow(refs, table, lens, 16, first, tokens)
    np.testing.assert_array_equal(at.cpu(), out)
    np.testing.assert_array_equal(missing.cpu(), short)
    np.testing.assert_array_equal(got.cpu(), table)
    np.testing.assert_array_equal(cache.refs.cpu(), refs)
    assert short.any() or seqs == 5  # of the five none lacks a block


def test_two_streams_at_once():
    """Calls on two caches side by side share nothing."""
    rng = np.random.default_rng(21)
    runs = []
    for i in range(2):
        table, n = batch(rng, 300, 20, 4000, 3500)
        cache, was = filled(4000, seed=30 + i, refs=pr.count(table, 4000))
        runs.append((cache, was, table, (n * 16 + 1).astype(np.int32), torch.cuda.Stream()))
    args = [(dev(t), dev(n), dev(rng.integers(-1, 300, 280)), dev(rng.permutation(4000)[:1500]))
            for _, _, t, n, _ in runs]
    torch.cuda.synchronize()
    got = []
    for (cache, _, _, _, s), (table, lens, parents, ids) in zip(runs, args):
        got.append((cache.grow(table, lens, stream=s)[0], cache.copy(ids, ids.flip(0), stream=s),
                    cache.fork(table, lens, parents, stream=s)))
    for (cache, _, _, _, s), (_, _, (table, _)) in zip(runs, got):
        cache.compact(table, stream=s)
    torch.cuda.synchronize()
    for (cache, was, table, lens, _), (_, _, parents, ids), (out, _, (new, _)) in zip(runs, args, got):
        refs = pr.count(table, 4000)
        want, _, pairs = pr.grow(refs, table, lens, 16)
        was = moved(was, pairs)
        ids = ids.cpu().numpy()
        was = moved(was, pr.copy_pairs(ids, ids[::-1], 4000, 4000, True))
        table, _ = pr.fork(refs, table, lens, parents.cpu().numpy())
        _, pairs = pr.compact(refs, table)
        np.testing.assert_array_equal(out.cpu(), want)
        np.testing.assert_array_equal(new.cpu(), table)
        np.testing.assert_array_equal(cache.refs.cpu(), refs)
        same(cache, moved(was, pairs))


@pytest.mark.parametrize("n", [40, 1500])
def test_a_captured_copy_replays(n):
    """With other ids each time, in one launch and in three."""
    rng = np.random.default_rng(n)
    cache, was = filled(2 * n, 1, 64, 16, 9)
    src, dst = dev([-1] * n), dev([-1] * n)
    cache.copy(src, dst)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.copy(src, dst)
    for _ in range(6):
        a, b = rng.integers(-1, 2 * n, n), rng.integers(0, 2 * n, n)
        src.copy_(dev(a)), dst.copy_(dev(b))
        graph.replay()
        torch.cuda.synchronize()
        was = moved(was, pr.copy_pairs(a, b, 2 * n, 2 * n, True))
        same(cache, was)


# ---- other devices' ways: streams and graphs ------------------------------------


def test_calls_on_another_stream():
    rng = np.random.default_rng(11)
    table, n = batch(rng, 8, 12, 200, 120, holes=False)
    lens = (n * 16).astype(np.int32)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for s in (stream, stream.cuda_stream):
        refs = pr.count(table, 200)
        cache, was = filled(200, refs=refs)
        got = dev(table)
        at = {"lens": dev(lens + 1), "parents": dev([7, 1, 1, -1, 3])}
        torch.cuda.synchronize()
        out, missing = cache.grow(got, at["lens"], stream=s)
        forked, left = cache.fork(got, out, at["parents"], stream=s)
        cache.release(forked, left, stream=s)
        where = cache.compact(forked, stream=s)
        torch.cuda.synchronize()
        t = table.copy()
        want, _, pairs = pr.grow(refs, t, lens + 1, 16)
        now = moved(was, pairs)
        t, want = pr.fork(refs, t, want, [7, 1, 1, -1, 3])
        pr.release(refs, t, want, 16)
        w, pairs = pr.compact(refs, t)
        np.testing.assert_array_equal(forked.cpu(), t)
        np.testing.assert_array_equal(left.cpu(), want)
        np.testing.assert_array_equal(where.cpu(), w)
        np.testing.assert_array_equal(cache.refs.cpu(), refs)
        same(cache, moved(now, pairs))


def test_captured_steps_replay():
    """grow, append, fork, release and compact in one graph, replayed with
    other lengths; eager work between the replays."""
    t, seqs, width, blocks = 16, 6, 5, 60
    rng = np.random.default_rng(12)
    cache, _ = filled(blocks)
    cache.refs.zero_()
    table = dev(np.full((seqs, width), -1))
    lens, parents, keep = dev([0] * seqs), dev([0] * seqs), dev([0] * seqs)
    k = torch.randn((seqs, 2, 64), device="cuda").bfloat16()
    first = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")

    def step():
        out, missing = cache.grow(table, lens, first, seqs)
        cache.append(k, k, table, out)
        new, left = cache.fork(table, out, parents)
        torch.minimum(left, keep, out=left)
        cache.release(new, left)
        where = cache.compact(new)
        table.copy_(new)
        return out, missing, left, where

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # lengths of 0: nothing comes of it
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    refs, want = np.zeros(blocks, np.int32), np.full((seqs, width), -1, np.int32)
    stored = np.zeros(seqs, np.int64)
    for i in range(40):
        new = np.minimum(stored + 1, width * t)
        who = rng.integers(-1, seqs, seqs) if i % 7 == 6 else np.arange(seqs)
        cut = np.full(seqs, 10 ** 6) if i % 5 else rng.integers(0, 40, seqs)
        lens.copy_(dev(new)), parents.copy_(dev(who)), keep.copy_(dev(cut))
        graph.replay()
        torch.cuda.synchronize()
        out, missing, _ = pr.grow(refs, want, new, t, np.arange(seqs + 1), seqs)
        want, left = pr.fork(refs, want, out, who)
        left = np.minimum(left, cut)
        pr.release(refs, want, left, t)
        w, _ = pr.compact(refs, want)
        for a, b in zip(got, (out, missing, left, w)):
            np.testing.assert_array_equal(a.cpu(), b)
        np.testing.assert_array_equal(table.cpu(), want)
        np.testing.assert_array_equal(cache.refs.cpu(), refs)
        stored = left.astype(np.int64)
    assert stored.max() > 16
