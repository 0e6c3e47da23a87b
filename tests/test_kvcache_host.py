"""What the paged cache's calls refuse, without a GPU: every check comes
before a kernel is launched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kvcache_ref as kr
from hbfsim_amd import _native as nat
from hbfsim_amd import kvcache

BAD, OK, NO = nat.HBFSIM_INVALID_ARGUMENT, nat.HBFSIM_OK, nat.HBFSIM_UNSUPPORTED
HERE = 0x7f0000000000  # a device address that no call here reaches


def arrays(**kw):
    c = nat.KvCacheArrays(ctypes.sizeof(nat.KvCacheArrays), 8, 2, 64, 16, 0, HERE, HERE, HERE,
                          HERE, HERE, HERE)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    b = nat.KvBatch(ctypes.sizeof(nat.KvBatch), 3, 4, 4, 3, 0, HERE, HERE, None)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def attend(c=None, b=None, q=HERE, kind=0, heads=4, scale=0.1, chosen=None, count=0, acc=0,
           out=HERE, ws=HERE, nbytes=1 << 30):
    c, b = arrays() if c is None else c, batch() if b is None else b
    return nat.load().hbfsim_amd_kv_attend(ctypes.byref(c), ctypes.byref(b), q, kind, heads, 256,
                                           64, scale, chosen, count, acc, out, ws, nbytes, None)


def append(c=None, b=None, k=HERE, v=HERE, kind=0, strides=(128, 64, 128, 64)):
    c, b = arrays() if c is None else c, batch() if b is None else b
    s = None if strides is None else (ctypes.c_int64 * 4)(*strides)
    return nat.load().hbfsim_amd_kv_append(ctypes.byref(c), ctypes.byref(b), k, v, kind, s, None)


def select(c=None, b=None, q=HERE, kind=0, heads=4, count=4, first=1, last=1, out=HERE, ws=HERE,
           nbytes=1 << 30):
    c, b = arrays() if c is None else c, batch() if b is None else b
    return nat.load().hbfsim_amd_kv_select(ctypes.byref(c), ctypes.byref(b), q, kind, heads, 256,
                                           64, count, first, last, out, ws, nbytes, None)


def evict(weight=HERE, blocks=8, kv=2, t=16, table=HERE, lens=HERE, seqs=3, width=4, stride=4,
          keep=2, first=1, last=1, out=HERE, out_lens=HERE, freed=HERE, count=HERE, ws=HERE,
          nbytes=1 << 20):
    return nat.load().hbfsim_amd_kv_evict(weight, blocks, kv, t, table, lens, seqs, width, stride,
                                          keep, first, last, out, out_lens, freed, count, ws,
                                          nbytes, None)


@pytest.mark.parametrize("field,value", [
    ("struct_size", 8), ("blocks", 0), ("blocks", 1 << 31), ("kv_heads", 0), ("kv_heads", 1025),
    ("head_dim", 0), ("head_dim", 257), ("block_tokens", 0), ("block_tokens", 24),
    ("block_tokens", 256), ("d_keys", None), ("d_keys", HERE + 8), ("d_values", None),
    ("d_values", HERE + 4), ("d_key_scale", None), ("d_value_scale", None), ("d_bounds", None),
    ("d_bounds", HERE + 1), ("d_weight", None)])
def test_caches_refused(field, value):
    c = arrays(**{field: value})
    for call in (append, attend, select):
        assert call(c=c) == BAD, call
    need = ctypes.c_size_t()
    b = batch()
    lib = nat.load()
    assert lib.hbfsim_amd_kv_attend_workspace(ctypes.byref(c), ctypes.byref(b), 4, 0, 0,
                                              ctypes.byref(need)) == BAD
    assert lib.hbfsim_amd_kv_select_workspace(ctypes.byref(c), ctypes.byref(b),
                                              ctypes.byref(need)) == BAD
    assert lib.hbfsim_amd_kv_read(ctypes.byref(c), HERE, 1, 0, HERE, HERE, HERE, HERE, None) == BAD


@pytest.mark.parametrize("fields", [
    dict(struct_size=4), dict(table_stride=3), dict(tokens=2), dict(d_lens=None),
    dict(d_table=None), dict(table_width=1 << 28, table_stride=1 << 28),
    dict(tokens=0x7fffffff, d_first=HERE), dict(seqs=0x7fffffff, tokens=0x7fffffff)])
def test_batches_refused(fields):
    b = batch(**fields)
    for call in (append, attend, select):
        assert call(b=b) == BAD, call


def test_null_structures_refused():
    lib = nat.load()
    b, c = batch(), arrays()
    assert lib.hbfsim_amd_kv_attend(None, ctypes.byref(b), HERE, 0, 4, 256, 64, 0.1, None, 0, 0,
                                    HERE, HERE, 1 << 30, None) == BAD
    assert lib.hbfsim_amd_kv_attend(ctypes.byref(c), None, HERE, 0, 4, 256, 64, 0.1, None, 0, 0,
                                    HERE, HERE, 1 << 30, None) == BAD


def test_arguments_refused():
    for kw in (dict(kind=2), dict(heads=0), dict(heads=3), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(q=None), dict(out=None), dict(count=3),
               dict(chosen=HERE), dict(chosen=HERE, count=2, acc=1), dict(ws=None, acc=1),
               dict(nbytes=0, acc=1), dict(ws=HERE + 4, acc=1),
               dict(chosen=HERE, count=1 << 27)):
        assert attend(**kw) == BAD, kw
    for kw in (dict(k=None), dict(v=None), dict(kind=3), dict(strides=None)):
        assert append(**kw) == BAD, kw
    for kw in (dict(kind=2), dict(heads=5), dict(heads=2 * 65), dict(count=0), dict(q=None),
               dict(out=None), dict(ws=None), dict(nbytes=95), dict(first=3, last=2),
               dict(first=0xffffffff, last=0xffffffff)):
        assert select(**kw) == BAD, kw
    for kw in (dict(weight=None), dict(blocks=0), dict(kv=0), dict(t=17), dict(table=None),
               dict(lens=None), dict(stride=3), dict(keep=0), dict(last=0), dict(keep=1),
               dict(first=0xffffffff), dict(out=None), dict(out_lens=None), dict(freed=None),
               dict(count=None), dict(ws=None), dict(nbytes=95), dict(ws=HERE + 4)):
        assert evict(**kw) == BAD, kw


def test_empty_calls_launch_nothing():
    none = batch(seqs=0, tokens=0, d_table=None, d_lens=None)
    assert append(b=none, k=None, v=None) == OK
    assert attend(b=none, q=None, out=None, ws=None, nbytes=0) == OK
    assert select(b=none, q=None, out=None, ws=None, nbytes=0) == OK
    assert evict(seqs=0, table=None, lens=None) == OK
    assert append(b=batch(table_width=0)) == OK
    c = arrays()
    lib = nat.load()
    assert lib.hbfsim_amd_kv_read(ctypes.byref(c), None, 0, 0, None, None, None, None, None) == OK
    need = ctypes.c_size_t(5)
    assert lib.hbfsim_amd_kv_attend_workspace(ctypes.byref(c), ctypes.byref(none), 4, 0, 0,
                                              ctypes.byref(need)) == OK and need.value == 0


def test_batches_beyond_a_launch_refused():
    many = batch(seqs=1 << 24, tokens=1 << 24)
    assert append(b=many) == NO
    assert attend(b=many, nbytes=1 << 62) == NO
    assert select(b=many, nbytes=1 << 62) == NO
    assert evict(seqs=1 << 24, nbytes=1 << 62) == NO


def test_python_refusals():
    c = kvcache.KvCache(4, 2, 64, device="cpu")
    i32 = torch.int32
    table, lens = torch.zeros((3, 2), dtype=i32), torch.zeros(3, dtype=i32)
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16)
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    first = torch.zeros(4, dtype=i32)
    for bad in (lambda: kvcache.KvCache(4, 2, 64, 24), lambda: kvcache.KvCache(4, 2, 257),
                lambda: kvcache.KvCache(0, 2, 64),
                lambda: c.append(k, k.half(), table, lens, stream=0),
                lambda: c.append(k[:2], k, table, lens, stream=0),
                lambda: c.append(q, q, table, lens, stream=0),
                lambda: c.append(k, k, table.long(), lens, stream=0),
                lambda: c.append(k, k, table, lens[:2], stream=0),
                lambda: c.append(k[:2], k[:2], table, lens, stream=0),
                lambda: c.append(k, k, table, lens, first[:3], stream=0),
                lambda: c.append(k, k, table.t().contiguous().t(), lens, stream=0),
                lambda: c.append(k.double(), k.double(), table, lens, stream=0),
                lambda: c.attend(q.float(), table, lens, stream=0),
                lambda: c.attend(q[:, :3], table, lens, stream=0),
                lambda: c.attend(q[:, :, :32], table, lens, stream=0),
                lambda: c.attend(q, table, lens, out=q.half(), stream=0),
                lambda: c.attend(q, table, lens, selected=lens, stream=0),
                lambda: c.attend(q, table, lens, selected=torch.zeros((3, 2, 0), dtype=i32)),
                lambda: c.attend(q, table, lens, selected=torch.zeros((3, 4, 1), dtype=i32)),
                lambda: c.attend(q, table, lens, selected=torch.zeros((3, 2, 1), dtype=i32),
                                 accumulate=True),
                lambda: c.attend(q.transpose(0, 2).contiguous().transpose(0, 2), table, lens),
                lambda: c.select(q, table, lens, -1, stream=0),
                lambda: c.evict(table, lens, -2, stream=0),
                lambda: kvcache.evict(c.weight.int(), table, lens, 2, stream=0),
                lambda: c.read(lens.long()), lambda: c.read(lens, torch.int8),
                lambda: kvcache.KvCache.from_tensors(c.keys, c.values, c.key_scale,
                                                     c.value_scale, c.bounds, c.weight, 65),
                lambda: kvcache.KvCache.from_tensors(c.keys, c.keys, c.key_scale, c.value_scale,
                                                     c.bounds, c.weight, 64)):
        with pytest.raises(ValueError):
            bad()


def test_the_definition_itself():
    """The oracle's quantisation is within half a step, its bounds hold, and a
    planted mistake in it is seen."""
    rng = np.random.default_rng(1)
    ref = kr.RefCache(3, 2, 64, 16)
    k = rng.normal(0, 1, (40, 2, 64)).astype(np.float32)
    table = np.array([[2, 0, 1]], np.int32)
    ref.append(k, -k, table, [40], [0, 40])
    for n, ident in ((16, 2), (16, 0), (8, 1)):
        at = {2: 0, 0: 16, 1: 32}[ident]
        x = k[at:at + n].transpose(1, 0, 2)
        s = ref.scale[0][ident][:, None, None]
        back = ref.codes[0][ident][:, :n] * s
        assert (np.abs(back - x) <= s * (0.5 + 2.0 ** -16)).all()
        assert (ref.bounds[ident, :, 0] == ref.codes[0][ident][:, :n].min(1)).all()
        assert not ref.codes[0][ident][:, n:].any()
    q = rng.normal(0, 1, (1, 4, 64))
    out, bound, weight, _ = ref.attend(q, table, [40])
    k64, v64 = (np.concatenate([ref.codes[w][i, 0].astype(np.float64) * float(ref.scale[w][i, 0])
                                for i in (2, 0, 1)])[:40] for w in (0, 1))
    z, v = k64 @ q[0, 0] / 8, v64
    p = np.exp(z) / np.exp(z).sum()
    assert np.allclose(out[0, 0], p @ v, rtol=1e-9)
    assert abs(weight.sum() - 4) < 1e-9
    ref.codes[1][0, 0, 5, 7] += 40  # a planted mistake shows in what attends to it
    wrong, _, _, _ = ref.attend(q, table, [40])
    assert abs(wrong[0, 0, 7] - out[0, 0, 7]) > bound[0, 0, 7]
