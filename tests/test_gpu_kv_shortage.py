"""Steps of drafts in which the pool runs short: a sequence that `grow` leaves
out gains nothing, keeps its row and its length, and is served once others
have given blocks back."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kvpages_ref as pr
from hbfsim_amd import _native as nat
from hbfsim_amd import drafts, kv_study, kvcache
from test_gpu_verify import dev, steps

pytestmark = pytest.mark.gpu


def verify(target, tokens, uniform, first, draft, lens, stored=None):
    """`kvpages_ref.verify`, with the sequences left out whose length is below
    their rows."""
    out, gained, left = pr.verify(target, tokens, uniform, first, draft, lens)
    first = range(len(lens) + 1) if first is None else [int(x) for x in first]
    for s, n in enumerate(lens):
        if first[s + 1] - first[s] > 0 and n < first[s + 1] - first[s]:
            out[max(0, first[s]):first[s + 1]] = -1
            gained[s], left[s] = 0, n if stored is None else stored[s]
    return out, gained, left


def case(vocab, dtype, sure, one_each, seqs=50):
    """A batch in which every length from none to all of the rows' occurs, some
    rows belong to no sequence and the last one's end past the batch."""
    rng = np.random.default_rng(vocab + seqs)
    counts = np.ones(seqs, int) if one_each else rng.integers(0, 6, seqs)
    p, q, tokens, u, first = steps(rng, counts, vocab, dtype, sure)
    if not one_each:
        first = first + 2
        first[-1] += 3
        counts[-1] += 3
        p, q = (None if x is None else torch.cat((x[-2:], x)) for x in (p, q))
        tokens, u = np.concatenate((tokens[-2:], tokens)), np.concatenate((u[-2:], u))
    stored = rng.integers(0, 900, seqs).astype(np.int32)
    lens = np.where(rng.random(seqs) < 0.4, rng.integers(-1, 6, seqs), stored + counts)
    lens[::7] = 0
    lens[3::7] = counts[3::7]
    return p, q, tokens, u, None if one_each else first, lens.astype(np.int32), stored


CASES = [(700, "f32", False, False), (8192, "bf16", False, False), (8192, "f32", True, False),
         (9001, "f32", False, True), (16_385, "f16", False, False), (40_001, "f32", False, False),
         (300, "bf16", True, True)]


@pytest.mark.parametrize("vocab,dtype,sure,one_each", CASES)
def test_verify_of_a_step_that_left_sequences_out(vocab, dtype, sure, one_each):
    p, q, tokens, u, first, lens, _ = case(vocab, dtype, sure, one_each)
    want = verify(p.float().numpy(), tokens, u, first, None if q is None else q.float().numpy(), lens)
    got = drafts.verify(p.cuda(), dev(tokens), dev(u, np.float32), None if first is None else dev(first),
                        draft=None if q is None else q.cuda(), lens=dev(lens))
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.cpu(), b)
    assert (want[1] == 0).sum() > 5 and (want[1] > 0).any()


@pytest.mark.parametrize("vocab,dtype,sure,one_each", CASES)
def test_verify_returns_the_lengths_before_the_step(vocab, dtype, sure, one_each):
    p, q, tokens, u, first, lens, stored = case(vocab, dtype, sure, one_each)
    want = verify(p.float().numpy(), tokens, u, first, None if q is None else q.float().numpy(), lens,
                  stored)
    args = (p.cuda(), dev(tokens), dev(u, np.float32), None if first is None else dev(first),
            None if q is None else q.cuda(), dev(lens))
    got = drafts.verify(*args, stored=dev(stored))
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.cpu(), b)


@pytest.mark.parametrize("over", ["lens", "stored"])
@pytest.mark.parametrize("vocab,dtype,sure,one_each", CASES)
def test_lengths_in_place(vocab, dtype, sure, one_each, over):
    """The C call may write over either kind of lengths: every wave of a
    sequence has read them before one is written."""
    p, q, tokens, u, first, lens, stored = case(vocab, dtype, sure, one_each,
                                                   700 if vocab < 9000 else 120)
    want = verify(p.float().numpy(), tokens, u, first, None if q is None else q.float().numpy(), lens,
                  stored)
    kind = {"f32": nat.KV_F32, "bf16": nat.KV_BF16, "f16": nat.KV_F16}[dtype]
    lib, need, seqs = nat.load(), ctypes.c_size_t(), len(lens)
    assert lib.hbfsim_amd_verify_workspace(seqs, vocab, kind, ctypes.byref(need)) == 0
    ws = torch.empty(max(16, need.value), dtype=torch.uint8, device="cuda")
    p, tokens, u = p.cuda(), dev(tokens), dev(u, np.float32)
    q, first = (None if x is None else y(x) for x, y in ((q, torch.Tensor.cuda), (first, dev)))
    for _ in range(3):
        at, before = dev(lens), dev(stored)
        out, gained = dev(np.full(len(p), 7)), dev(np.full(seqs, 7))
        left = at if over == "lens" else before
        assert lib.hbfsim_amd_verify_step(
            p.data_ptr(), None if q is None else q.data_ptr(), kind, vocab, vocab, vocab,
            tokens.data_ptr(), u.data_ptr(), None if first is None else first.data_ptr(), seqs, len(p),
            at.data_ptr(), before.data_ptr(), out.data_ptr(), gained.data_ptr(), left.data_ptr(),
            ws.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream) == 0
        for a, b in zip((out, gained, left), want):
            np.testing.assert_array_equal(a.cpu(), b)


@pytest.mark.parametrize("vocab,dtype,sure,one_each", CASES[2:6])
def test_left_out_on_another_stream_and_in_a_graph(vocab, dtype, sure, one_each):
    """One captured call serves steps that leave out other sequences each time."""
    p, q, tokens, u, first, lens, stored = case(vocab, dtype, sure, one_each)
    rng = np.random.default_rng(1)
    host = (p.float().numpy(), tokens, u, first, None if q is None else q.float().numpy())
    at, before = dev(lens), dev(stored)
    args = (p.cuda(), dev(tokens), dev(u, np.float32), None if first is None else dev(first),
            None if q is None else q.cuda(), at)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        drafts.verify(*args, stored=before)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = drafts.verify(*args, stored=before)
    for _ in range(5):
        n, m = np.where(rng.random(len(lens)) < 0.5, 0, lens), rng.integers(0, 99, len(lens))
        at.copy_(dev(n)), before.copy_(dev(m))
        torch.cuda.synchronize()
        graph.replay()
        eager = drafts.verify(*args, stored=before, stream=stream)
        torch.cuda.synchronize()
        for got in (captured, eager):
            for a, b in zip(got, verify(*host, n, m)):
                np.testing.assert_array_equal(a.cpu(), b)


def test_a_pool_that_runs_short():
    """Drafted steps of six sequences that share a prompt over a pool that
    cannot hold them all, beside a cache in which each has blocks of its own:
    what each attends to stays equal to the last bit, rows that lack blocks
    keep them, and go on when others have ended."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    rng = np.random.default_rng(3)
    kv, heads, dim, t, vocab, seqs, width, blocks = 2, 4, 64, 16, 50, 6, 9, 14
    cache = kvcache.KvCache(blocks, kv, dim, t)
    alone = kvcache.KvCache(seqs * width, kv, dim, t)
    own = torch.arange(seqs * width, dtype=torch.int32, device="cuda").view(seqs, width)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").bfloat16()

    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    k, v, one = normal(40, kv, dim), normal(40, kv, dim), dev([0, 40])
    lens, missing = cache.grow(table, dev([40]), one, 40)
    cache.append(k, v, table, lens, one)
    table, lens = cache.fork(table, lens, dev([0] * seqs))
    alone.append(k.repeat(seqs, 1, 1), v.repeat(seqs, 1, 1), own, lens, dev(40 * np.arange(seqs + 1)))
    starved, ended, had = np.zeros(seqs, bool), np.zeros(seqs, bool), None
    for step in range(38):
        counts = rng.integers(0, 7, seqs)
        if step == 30:  # of the six only those that were short of blocks go on
            ended, had = ~starved, lens.cpu().numpy()
            assert starved.any() and ended.any()
            table, lens = cache.fork(table, lens, dev(np.where(starved, np.arange(seqs), -1)))
        counts[ended] = 0
        first = np.concatenate([[0], np.cumsum(counts)])
        total, at = int(first[-1]), dev(first)
        refs, rows = cache.refs.cpu().numpy().copy(), table.cpu().numpy().copy()
        before, wanted = lens.cpu().numpy(), lens + dev(counts)
        now, missing = cache.grow(table, wanted, at, total)
        step_lens, lacks, _ = pr.grow(refs, rows, wanted.cpu().numpy(), t, first, total)
        np.testing.assert_array_equal(now.cpu(), step_lens)
        np.testing.assert_array_equal(missing.cpu(), lacks)
        k, v, q = normal(total, kv, dim), normal(total, kv, dim), normal(total, heads, dim)
        cache.append(k, v, table, now, at)
        alone.append(k, v, own, now, at)
        a, b = cache.attend(q, table, now, at), alone.attend(q, own, now, at)
        assert torch.equal(a, b) and torch.isfinite(a.float()).all()
        p = torch.softmax(torch.randn((total, vocab), generator=gen, device="cuda") * 3, 1)
        d = torch.softmax(torch.log(p) + torch.randn((total, vocab), generator=gen, device="cuda"), 1)
        said = d.argmax(1).roll(1).to(torch.int32)
        u = torch.rand((total,), generator=gen, device="cuda")
        got = drafts.verify(p, said, u, at, draft=d, lens=now, stored=lens)
        want = verify(p.cpu().numpy(), said.cpu().numpy(), u.cpu().numpy(), first, d.cpu().numpy(),
                      step_lens, before)
        for x, y in zip(got, want):
            np.testing.assert_array_equal(x.cpu(), y)
        _, gained, lens = got
        left = lens.cpu().numpy()
        assert (left[lacks != 0] == before[lacks != 0]).all() and not gained.cpu().numpy()[lacks != 0].any()
        assert (left >= before).all()
        if step < 30:
            starved |= lacks != 0
        cache.release(table, lens)
        pr.release(refs, rows, left, t)
        np.testing.assert_array_equal(table.cpu(), rows)
        np.testing.assert_array_equal(cache.refs.cpu(), refs)
        assert ((rows >= 0).sum(1) == -(-left // t)).all()
        if step % 3 == 2 and step < 30:  # the longest begins again as a branch of the shortest
            parents = np.arange(seqs)
            parents[left.argmax()] = left.argmin()
            table, lens = cache.fork(table, lens, dev(parents))
            whole = own[dev(parents).long()].clone()
            alone.copy(whole[left.argmax()], own[left.argmax()])
            starved[left.argmax()] = False
    assert (lens.cpu().numpy()[starved] > had[starved]).all() and not lens[dev(ended) != 0].any()


def test_a_study_whose_pool_runs_short(monkeypatch):
    """No row is lost: the prompts' 32 full blocks stay shared by the rows that
    go on (0, 2 and 4, the first two of one prompt)."""
    whole = kvcache.KvCache
    monkeypatch.setattr(kv_study.kvcache, "KvCache", lambda blocks, *a: whole(blocks - 58, *a))
    got = kv_study.run_drafts(seqs=2, tokens=520, steps=10, branches=3, drafts=3, vocab=500, heads=4,
                              kv_heads=2, head_dim=64, seed=1)
    assert got["missing"] > 0
    assert got["compaction"]["named_by_rows"] - got["compaction"]["blocks"] == 32


@pytest.mark.parametrize("blocks", [40, 9])
def test_branches_continue_what_the_step_appended(blocks):
    """Decode, branch, decode again, with room for all and without: the tokens
    of the step before the branch are attended to after it."""
    gen = torch.Generator(device="cuda").manual_seed(blocks)
    kv, heads, dim, seqs, width = 2, 4, 64, 3, 4
    cache, alone = kvcache.KvCache(blocks, kv, dim), kvcache.KvCache(2 * seqs * width, kv, dim)
    own = torch.arange(2 * seqs * width, dtype=torch.int32, device="cuda").view(2 * seqs, width)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").bfloat16()

    first = dev([0, 16, 31, 63])
    lens, missing = cache.grow(table, dev([16, 15, 32]), first, 63)
    assert not missing.any()
    k, v = normal(63, kv, dim), normal(63, kv, dim)
    cache.append(k, v, table, lens, first)
    alone.append(k, v, own[:seqs], lens, first)
    short = 0
    for step in range(9):
        now, missing = cache.grow(table, lens + 1)
        short += int((missing != 0).sum())
        n = len(table)
        k, v, q = normal(n, kv, dim), normal(n, kv, dim), normal(n, heads, dim)
        cache.append(k, v, table, now)
        alone.append(k, v, own[:n], now)
        assert torch.equal(cache.attend(q, table, now), alone.attend(q, own[:n], now))
        before, lens = lens, torch.where(missing == 0, now, lens)
        assert torch.equal(lens, before + (missing == 0))
        # all of it is there to be attended to
        assert torch.equal(cache.attend(q, table, lens), alone.attend(q, own[:n], lens))
        if step in (1, 4):
            parents = dev([2, 0, 1, 0, 2, 0][:6 if step == 1 else 4])
            held = lens
            table, lens = cache.fork(table, lens, parents)
            assert torch.equal(lens, held[parents.long()])
            extra = kvcache.KvCache(2 * seqs * width, kv, dim)
            alone.copy(own[parents.long()].reshape(-1), own[:len(parents)].reshape(-1), to=extra)
            alone = extra
    assert int(lens.max()) > 32 and (short == 0) == (blocks == 40)


def test_an_eviction_leaves_no_reference_behind():
    """Rows that name blocks past their lengths (grown for drafts that did not
    stay), some of them shared: released to the lengths, evicted, and what is
    freed released, they hold what they name and no block more."""
    rng = np.random.default_rng(9)
    blocks, seqs, width = 300, 8, 30
    cache = kvcache.KvCache(blocks, 2, 64)
    cache.weight.random_(0, 1 << 40)
    rows = rng.permutation(blocks)[:seqs * width].reshape(seqs, width).astype(np.int32)
    rows[1, :12] = rows[0, :12]
    table, lens = dev(rows), dev([480, 470, 465, 16, 0, 300, 177, 176])
    cache.hold(table)
    cache.release(table, lens)
    table, lens, freed, gone = cache.evict(table, lens, keep=11)
    assert int(gone.sum()) > 0
    cache.release(freed)
    np.testing.assert_array_equal(cache.refs.cpu(), pr.count(table.cpu().numpy(), blocks))
    assert (table >= 0).sum(1).tolist() == [11, 11, 11, 1, 0, 11, 11, 11]
    cache.release(table)
    assert not cache.refs.any()


def test_other_tables_follow_a_compaction():
    """As the guide has it: entries that name no block stay -1, also where the
    pool's last block is in use."""
    rng = np.random.default_rng(10)
    blocks = 90
    ids = rng.permutation(blocks - 1)[:36].astype(np.int32)
    ids[0] = blocks - 1
    one, two = np.full((3, 9), -1, np.int32), np.full((2, 11), -1, np.int32)
    one[:, :6], two[:, :9] = ids[:18].reshape(3, 6), ids[18:].reshape(2, 9)
    refs = pr.count(one, blocks)
    pr.hold(refs, two)
    cache = kvcache.KvCache(blocks, 1, 64)
    cache.refs.copy_(dev(refs))
    cache.weight.copy_(torch.arange(blocks, device="cuda")[:, None])
    table, other = dev(one), dev(two)
    where = cache.compact(table)
    other = torch.where(other >= 0, where[other.clamp(min=0).long()], -1)
    for got, was in ((table, one), (other, two)):
        assert torch.equal(got >= 0, dev(was) >= 0) and int(got.max()) < 36
        named = torch.where(got >= 0, cache.weight[got.clamp(min=0).long(), 0], -1)
        np.testing.assert_array_equal(named.cpu(), was)


@pytest.mark.parametrize("vocab,seqs", [(151_936, 64), (40_000, 3), (500, 64)])
def test_what_verify_returns_keeps_no_scratch_alive(vocab, seqs):
    """A program that collects each step's tokens holds those and 64 KiB at
    most beside them."""
    p = torch.full((seqs, vocab), 1.0 / vocab, device="cuda")
    lens = dev(np.arange(seqs) + 1)
    got = drafts.verify(p, dev(np.zeros(seqs)), torch.full((seqs,), 0.5, device="cuda"), lens=lens)
    assert all(x.untyped_storage().nbytes() <= 65536 + 4 * 3 * seqs for x in got)
    torch.cuda.synchronize()
    del p
    before = torch.cuda.memory_allocated()
    del got
    torch.cuda.synchronize()
    assert before - torch.cuda.memory_allocated() <= 65536 + 4 * 3 * seqs + 512
