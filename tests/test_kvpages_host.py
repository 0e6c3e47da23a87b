"""What the calls on a paged cache's blocks and on drafted tokens refuse,
without a GPU: every check comes before a kernel is launched.  A call that is
not refused finds no GPU here."""
from __future__ import annotations

import ctypes

import pytest
import torch

from hbfsim_amd import _native as nat
from hbfsim_amd import drafts, kvcache

BAD, OK, NO, RUNS = (nat.HBFSIM_INVALID_ARGUMENT, nat.HBFSIM_OK, nat.HBFSIM_UNSUPPORTED,
                     nat.HBFSIM_CUDA_ERROR)
HERE = 0x7f0000000000  # a device address that no call here reaches
FAR = 1 << 36
I32 = torch.int32
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="its addresses are not a GPU's")


def arrays(at=HERE, **kw):
    c = nat.KvCacheArrays(ctypes.sizeof(nat.KvCacheArrays), 8, 2, 64, 16, 0,
                          *[at + i * FAR for i in range(6)])
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def copy(a=None, b=None, src=HERE, dst=HERE, n=3, ws=HERE, nbytes=32):
    a = arrays() if a is None else a
    b = a if b is None else b
    return nat.load().hbfsim_amd_kv_copy(ctypes.byref(a), ctypes.byref(b), src, dst, n, ws, nbytes,
                                         None)


@no_gpu
def test_copy_refuses():
    assert copy() == RUNS
    assert copy(b=arrays(HERE + 8 * FAR)) == RUNS
    assert copy(n=0, src=None, dst=None, ws=None, nbytes=0) == OK
    assert copy(ws=None, nbytes=0) == RUNS  # few pairs need none
    for kw in (dict(src=None), dict(dst=None), dict(n=5000, ws=None), dict(n=5000, ws=HERE + 4),
               dict(n=5000, nbytes=31), dict(a=arrays(struct_size=3)), dict(a=arrays(blocks=0)), dict(a=arrays(kv_heads=0)),
               dict(a=arrays(d_keys=None)), dict(a=arrays(d_bounds=HERE + 8)),
               dict(b=arrays(HERE + 8 * FAR, kv_heads=4)), dict(b=arrays(HERE + 8 * FAR, head_dim=65)),
               dict(b=arrays(HERE + 8 * FAR, block_tokens=32)),
               dict(b=arrays(HERE + 8 * FAR, d_values=HERE + FAR + 16)),  # overlaps a's values
               dict(b=arrays(HERE + 8 * FAR, d_weight=HERE + 5 * FAR - 8)),
               dict(b=arrays(blocks=9))):
        assert copy(**kw) == BAD, kw
    assert copy(n=1 << 40, nbytes=1 << 50) == NO
    need = ctypes.c_size_t()
    assert nat.load().hbfsim_amd_kv_copy_workspace(ctypes.byref(arrays()), 3, None) == BAD
    for n, want in ((0, 0), (3, 0), (5000, 32)):
        assert nat.load().hbfsim_amd_kv_copy_workspace(ctypes.byref(arrays()), n,
                                                       ctypes.byref(need)) == OK
        assert need.value == want


def hold(refs=HERE, blocks=8, table=HERE, seqs=3, width=4, stride=4):
    return nat.load().hbfsim_amd_kv_hold(refs, blocks, table, seqs, width, stride, None)


def release(refs=HERE, blocks=8, t=16, table=HERE, lens=HERE, seqs=3, width=4, stride=4):
    return nat.load().hbfsim_amd_kv_release(refs, blocks, t, table, lens, seqs, width, stride, None)


def fork(refs=HERE, blocks=8, table=HERE + FAR, lens=HERE + 2 * FAR, seqs=3, width=4, stride=4,
         parents=HERE + 3 * FAR, rows=5, out=HERE + 4 * FAR, out_lens=HERE + 5 * FAR):
    return nat.load().hbfsim_amd_kv_fork(refs, blocks, table, lens, seqs, width, stride, parents,
                                         rows, out, out_lens, None)


@no_gpu
def test_tables_refused():
    for call in (hold, release, fork):
        assert call() == RUNS and call(stride=9) == RUNS
        for kw in (dict(refs=None), dict(blocks=0), dict(blocks=1 << 31), dict(stride=3),
                   dict(table=None), dict(seqs=0x7fffff01)):
            assert call(**kw) == BAD, (call, kw)
        assert call(seqs=1 << 25, width=1 << 10, stride=1 << 10) in (NO, RUNS)
        assert call(seqs=1 << 25) == NO
    for call in (hold, release):
        assert call(seqs=0, table=None) == OK and call(width=0, table=None, stride=0) == OK
    assert release(lens=None) == RUNS
    for kw in (dict(t=0), dict(t=8), dict(t=17), dict(width=1 << 28, stride=1 << 28)):
        assert release(**kw) == BAD, kw


@no_gpu
def test_fork_refuses():
    assert fork(rows=0, parents=None, out=None, out_lens=None) == RUNS  # the old rows end
    assert fork(rows=0, seqs=0, table=None, lens=None, parents=None, out=None, out_lens=None) == OK
    assert fork(seqs=0, table=None, lens=None) == RUNS                  # rows of no sequence
    assert fork(width=0, stride=0, table=None, out=None) == RUNS        # lengths alone
    for kw in (dict(parents=None), dict(out=None), dict(out_lens=None), dict(lens=None),
               dict(out=HERE + FAR), dict(out=HERE + FAR + 44), dict(out=HERE + FAR - 76),
               dict(out=HERE + 28), dict(out=HERE + 2 * FAR), dict(out=HERE + 3 * FAR),
               dict(out_lens=HERE + 2 * FAR + 8), dict(out_lens=HERE + 3 * FAR),
               dict(out_lens=HERE + FAR), dict(out_lens=HERE + 4 * FAR + 76)):
        assert fork(**kw) == BAD, kw
    assert fork(out=HERE + FAR + 48) == RUNS and fork(out=HERE + FAR - 80) == RUNS


def grow(c=None, refs=HERE, table=HERE, lens=HERE, first=None, seqs=3, tokens=3, width=4, stride=4,
         out=HERE, missing=HERE, ws=HERE, nbytes=1 << 20):
    c = arrays() if c is None else c
    return nat.load().hbfsim_amd_kv_grow(ctypes.byref(c), refs, table, lens, first, seqs, tokens,
                                         width, stride, out, missing, ws, nbytes, None)


@no_gpu
def test_grow_refuses():
    assert grow() == RUNS and grow(first=HERE, tokens=40) == RUNS
    assert grow(seqs=0, tokens=0, table=None, lens=None, out=None, missing=None, ws=None) == OK
    for kw in (dict(c=arrays(d_keys=None)), dict(refs=None), dict(table=None), dict(lens=None),
               dict(out=None), dict(missing=None), dict(ws=None), dict(ws=HERE + 4), dict(nbytes=64),
               dict(tokens=4), dict(stride=3), dict(tokens=0x7fffff01, first=HERE),
               dict(width=1 << 28, stride=1 << 28)):
        assert grow(**kw) == BAD, kw
    assert grow(first=HERE, tokens=0x7fffff00, nbytes=1 << 60) == NO
    assert grow(seqs=1 << 24, tokens=1 << 24, nbytes=1 << 60) == NO
    need = ctypes.c_size_t()
    for seqs, tokens in ((3, 3), (3, 400), (70, 9)):
        assert nat.load().hbfsim_amd_kv_grow_workspace(ctypes.byref(arrays()), seqs, tokens,
                                                       ctypes.byref(need)) == OK
        assert grow(first=HERE, seqs=seqs, tokens=tokens, nbytes=need.value) == RUNS
        assert grow(first=HERE, seqs=seqs, tokens=tokens, nbytes=need.value - 256) == BAD
    assert nat.load().hbfsim_amd_kv_grow_workspace(ctypes.byref(arrays()), 3, 3, None) == BAD


def compact(c=None, refs=HERE, table=HERE, seqs=3, width=4, stride=4, where=HERE, ws=HERE,
            nbytes=1 << 20):
    c = arrays() if c is None else c
    return nat.load().hbfsim_amd_kv_compact(ctypes.byref(c), refs, table, seqs, width, stride, where,
                                            ws, nbytes, None)


@no_gpu
def test_compact_refuses():
    assert compact() == RUNS and compact(seqs=0, table=None) == RUNS
    for kw in (dict(c=arrays(head_dim=0)), dict(refs=None), dict(table=None), dict(where=None),
               dict(ws=None), dict(ws=HERE + 8), dict(nbytes=100), dict(stride=3)):
        assert compact(**kw) == BAD, kw
    assert compact(seqs=1 << 25) == NO


def verify(target=HERE, draft=HERE, kind=2, vocab=100, stride=100, draft_stride=100,
           tokens=HERE + FAR, uniform=HERE + 2 * FAR, first=HERE + 3 * FAR, seqs=2, rows=5,
           lens=HERE + 4 * FAR, out=HERE + 5 * FAR, gained=HERE + 6 * FAR,
           out_lens=HERE + 4 * FAR, ws=HERE, nbytes=1 << 20):
    return nat.load().hbfsim_amd_verify(target, draft, kind, vocab, stride, draft_stride, tokens,
                                        uniform, first, seqs, rows, lens, out, gained, out_lens,
                                        ws, nbytes, None)


@no_gpu
def test_verify_refuses():
    assert verify() == RUNS and verify(draft=None) == RUNS
    assert verify(lens=None, out_lens=None) == RUNS
    assert verify(first=None, rows=2, tokens=None) == RUNS  # nothing is drafted
    assert verify(seqs=0, rows=0, first=None, out=None, gained=None, ws=None) == OK
    assert verify(seqs=0, gained=None, ws=None, nbytes=0) == RUNS  # rows of no sequence
    for kw in (dict(target=None), dict(tokens=None), dict(uniform=None), dict(out=None),
               dict(gained=None), dict(vocab=70_000, ws=None), dict(vocab=70_000, ws=HERE + 4),
               dict(vocab=70_000, nbytes=63), dict(kind=3),
               dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(first=None), dict(lens=None),
               dict(out_lens=None), dict(rows=0x7fffff01), dict(seqs=0x7fffff01),
               dict(out=HERE + FAR + 16), dict(out=HERE + 2 * FAR - 4), dict(out=HERE + 3 * FAR + 8),
               dict(out=HERE + 4 * FAR)):
        assert verify(**kw) == BAD, kw
    assert verify(vocab=1 << 22, seqs=1 << 20, nbytes=1 << 60) == NO
    need = ctypes.c_size_t()
    for seqs, vocab, kind in ((2, 100, 2), (70, 50_000, 0), (3, 1 << 22, 1)):
        assert nat.load().hbfsim_amd_verify_workspace(seqs, vocab, kind, ctypes.byref(need)) == OK
        assert verify(seqs=seqs, vocab=vocab, kind=kind, nbytes=need.value) == RUNS
        if need.value:  # short rows need none
            assert verify(seqs=seqs, vocab=vocab, kind=kind, nbytes=need.value - 1) == BAD
        else:
            assert verify(seqs=seqs, vocab=vocab, kind=kind, ws=None, nbytes=0) == RUNS
    for bad in ((3, 0, 0), (3, 5, 3), (3, (1 << 22) + 1, 0)):
        assert nat.load().hbfsim_amd_verify_workspace(*bad, ctypes.byref(need)) == BAD


def test_python_refuses():
    cache = kvcache.KvCache(8, 2, 64, device="cpu")
    other = kvcache.KvCache(5, 2, 64, device="cpu")
    table, lens = torch.zeros((3, 2), dtype=I32), torch.zeros(3, dtype=I32)
    ids, first = torch.zeros(3, dtype=I32), torch.arange(4, dtype=I32)
    p = torch.zeros((3, 50))
    u = torch.zeros(3)
    assert cache.refs.dtype == I32 and tuple(cache.refs.shape) == (8,)
    long = table.long()
    shared = torch.zeros(4, dtype=I32).as_strided((3, 2), (1, 1))
    for bad in (
            lambda: cache.copy(ids, ids[:2]), lambda: cache.copy(ids.long(), ids),
            lambda: cache.copy(ids, table), lambda: cache.hold(long), lambda: cache.hold(ids),
            lambda: kvcache.hold(cache.refs.long(), table),
            lambda: kvcache.hold(torch.zeros((2, 4), dtype=I32), table),
            lambda: kvcache.hold(torch.zeros(8, dtype=I32)[::2], table),
            lambda: kvcache.hold(torch.zeros(0, dtype=I32), table),
            lambda: cache.fork(table, lens[:2], ids), lambda: cache.fork(table, lens, table),
            lambda: cache.fork(table, lens, ids.float()), lambda: cache.fork(table.t(), lens, ids),
            lambda: cache.release(shared, lens), lambda: cache.release(table, lens[:1]),
            lambda: cache.grow(shared, lens), lambda: cache.grow(table, lens.long()),
            lambda: cache.grow(table, lens, first), lambda: cache.grow(table, lens, first[:3], 3),
            lambda: cache.grow(table, lens, None, 4), lambda: cache.grow(table, lens, first, -1),
            lambda: cache.grow(table, lens, first, 2 ** 32), lambda: cache.compact(shared),
            lambda: cache.compact(long), lambda: cache.compact(ids),
            lambda: drafts.verify(p[0], ids, u), lambda: drafts.verify(p.double(), ids, u),
            lambda: drafts.verify(p.t().contiguous().t(), ids, u),
            lambda: drafts.verify(p, ids[:2], u), lambda: drafts.verify(p, ids.long(), u),
            lambda: drafts.verify(p, ids, u.double()), lambda: drafts.verify(p, ids, u[:2]),
            lambda: drafts.verify(p, ids, torch.zeros(6)[::2]),
            lambda: drafts.verify(p, ids, u, first[:0]), lambda: drafts.verify(p, ids, u, table),
            lambda: drafts.verify(p, ids, u, first, draft=p[:, :49]),
            lambda: drafts.verify(p, ids, u, first, draft=p.bfloat16()),
            lambda: drafts.verify(p, ids, u, first, lens=lens[:2])):
        with pytest.raises(ValueError) as e:
            bad()
        assert "not on a GPU" not in str(e.value)
    for fine in (lambda: cache.copy(ids, ids, other), lambda: cache.hold(table),
                 lambda: cache.fork(table, lens, ids), lambda: cache.release(table),
                 lambda: cache.release(table, lens), lambda: cache.grow(table, lens),
                 lambda: cache.grow(table, lens, first, 3), lambda: cache.compact(table),
                 lambda: drafts.verify(p, ids, u), lambda: drafts.verify(p, ids, u, first, p, lens)):
        with pytest.raises(ValueError, match="not on a GPU"):
            fine()


def test_references_that_do_not_fit():
    c = kvcache.KvCache(8, 2, 64, device="cpu")
    own = [getattr(c, n) for n in ("keys", "values", "key_scale", "value_scale", "bounds", "weight")]
    refs = torch.arange(8, dtype=I32)
    assert kvcache.KvCache.from_tensors(*own, head_dim=64, refs=refs).refs is refs
    assert not kvcache.KvCache.from_tensors(*own, head_dim=64).refs.any()
    for bad in (refs[:7], refs.long(), refs.view(2, 4), torch.zeros(16, dtype=I32)[::2]):
        with pytest.raises(ValueError, match="refs"):
            kvcache.KvCache.from_tensors(*own, head_dim=64, refs=bad)
    # a cache's references may be replaced, but not by ones elsewhere
    table, lens = (torch.zeros(n, dtype=I32, device="meta") for n in ((3, 2), (3,)))
    c.refs = torch.zeros(8, dtype=I32, device="meta")
    for bad in (lambda: c.grow(table, lens), lambda: c.compact(table)):
        with pytest.raises(ValueError, match="refs is on meta"):
            bad()
