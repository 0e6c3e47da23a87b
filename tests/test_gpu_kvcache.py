"""The paged 8-bit cache on the GPU against its definition (kvcache_ref)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvcache_ref as kr
from hbfsim_amd import kvcache

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half a unit in the last place, relative: the output's own rounding
ULP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x)).to("cuda" if dtype is None else "cuda",
                                                        dtype=dtype)


def ints(x):
    return None if x is None else dev(np.asarray(x, np.int32))


def rows(rng, shape, dtype, size=1.0):
    """Values of the type, as a GPU tensor and as float32 numpy."""
    x = torch.from_numpy(rng.normal(0, size, shape).astype(np.float32)).to(DT[dtype])
    return x.cuda(), x.float().numpy()


def pair(kv, dim, t, blocks):
    return (kvcache.KvCache(blocks, kv, dim, t), kr.RefCache(blocks, kv, dim, t))


def same_cache(cache, ref, blocks):
    dim = ref.shape[3]
    for got, want in zip(kr.codes_of(cache), ref.codes):
        np.testing.assert_array_equal(got[blocks][..., :dim], want[blocks])
        assert not got[blocks][..., dim:].any()
    for got, want in ((cache.key_scale, ref.scale[0]), (cache.value_scale, ref.scale[1])):
        np.testing.assert_array_equal(got.cpu().numpy()[blocks], want[blocks])
    np.testing.assert_array_equal(cache.bounds.cpu().numpy()[blocks][..., :dim],
                                  ref.bounds[blocks])
    np.testing.assert_array_equal(cache.weight.cpu().numpy()[blocks], ref.weight[blocks])


# ---- append and read ------------------------------------------------------


@pytest.mark.parametrize("kv,dim,t,dtype", [(8, 128, 16, "bf16"), (4, 64, 16, "f16"),
                                            (1, 80, 32, "bf16"), (3, 256, 64, "f32"),
                                            (2, 37, 128, "f16"), (5, 192, 16, "f32"),
                                            (2, 1, 16, "bf16")])
def test_append_matches_definition(kv, dim, t, dtype):
    """Prompts, single tokens and small chunks into blocks begun before, whose
    scales grow in some and stay in others; strided rows."""
    rng = np.random.default_rng(dim * t)
    lens = np.array([0, 3, 2 * t - 1, t, 5 * t + 7], np.int64)
    total = [int(n) + 40 for n in lens]
    blocks = sum(-(-n // t) for n in total) + 2
    table = kr.make_table(rng, total, t, blocks)
    cache, ref = pair(kv, dim, t, blocks)
    cache.weight.fill_(7)
    ref.weight[:] = 7
    steps = [("chunk", lens.copy()), ("one", None), ("chunk", np.array([0, 1, 17, t, 2])),
             ("one", None), ("one", None)]
    now = np.zeros(len(lens), np.int64)
    for i, (kind, new) in enumerate(steps):
        new = np.ones(len(lens), np.int64) if kind == "one" else new
        now = now + new
        first = np.concatenate([[0], np.cumsum(new)])
        tokens = int(first[-1])
        x = rng.normal(0, [1.0, 0.2, 1.5, 0.5, 3.0][i], (tokens, 2 * kv * dim + 3))
        x = torch.from_numpy(x.astype(np.float32)).to(DT[dtype])
        g = x.cuda()
        k, v = (g[:, a:a + kv * dim].view(tokens, kv, dim) for a in (0, kv * dim))
        kn, vn = (y.float().cpu().numpy() for y in (k, v))
        cache.append(k, v, ints(table), ints(now), None if kind == "one" else ints(first))
        ref.append(kn, vn, table, now, first)
    same_cache(cache, ref, np.unique(table[table >= 0]))


def test_append_zero_tiny_huge_and_not_finite():
    rng = np.random.default_rng(3)
    kv, dim, t, blocks = 2, 64, 16, 8
    cache, ref = pair(kv, dim, t, blocks)
    table = np.arange(8, dtype=np.int32).reshape(8, 1)
    k = rng.normal(0, 1, (8, kv, dim)).astype(np.float32)
    v = k[::-1].copy()
    k[0] = 0
    k[1] = 1e-20
    k[2, 0, 3] = np.inf
    k[3, 1, 5] = np.nan
    v[4, 0, 0] = 3e38          # scale beyond 2^40
    v[5] = -0.0
    k[6, 0] = 127 * 2.0 ** 40  # the largest scale that is kept
    one = np.ones(8, np.int64)
    cache.append(dev(k), dev(v), ints(table), ints(one))
    ref.append(k, v, table, one)
    same_cache(cache, ref, np.arange(8))
    assert torch.isnan(cache.key_scale[2, 0]) and torch.isnan(cache.key_scale[3, 1])
    assert torch.isnan(cache.value_scale[4, 0]) and not torch.isnan(cache.key_scale[6, 0])
    # a NaN block stays NaN while it fills, and is fine once begun anew
    k2 = rng.normal(0, 1, (8, kv, dim)).astype(np.float32)
    cache.append(dev(k2), dev(k2), ints(table), ints(one * 2))
    ref.append(k2, k2, table, one * 2)
    same_cache(cache, ref, np.arange(8))
    assert torch.isnan(cache.key_scale[2, 0])
    cache.append(dev(k2), dev(k2), ints(table), ints(one))
    ref.append(k2, k2, table, one)
    same_cache(cache, ref, np.arange(8))
    assert not torch.isnan(cache.key_scale).any()


def test_append_leaves_out_what_has_no_place():
    """Blocks that are not there, positions past the table, tokens of no
    sequence, lengths below the step's tokens: nothing else changes."""
    rng = np.random.default_rng(4)
    kv, dim, t, blocks = 2, 64, 16, 6
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table = np.array([[0, -1], [1, 6], [2, 3], [4, 5]], np.int32)
    lens = np.array([20, 32, 40, 2], np.int64)
    first = np.array([0, 20, 37, 45, 50], np.int64)  # the last two have no room or too few tokens
    x, xn = rows(rng, (50, kv, dim), "bf16")
    cache.append(x, x, ints(table), ints(lens), ints(first))
    ref.append(xn, xn, table, lens, first)
    same_cache(cache, ref, np.arange(blocks))


def test_append_rows_at_odd_addresses():
    rng = np.random.default_rng(5)
    kv, dim, t = 3, 64, 16
    cache, ref = pair(kv, dim, t, 4)
    big = torch.from_numpy(rng.normal(0, 1, 4 + 40 * 211).astype(np.float32)).to(torch.bfloat16).cuda()
    x = big[1:1 + 40 * 211].view(40, 211)[:, 5:5 + kv * dim].view(40, kv, dim)
    table, lens, first = np.array([[2, 0, 1]], np.int32), [40], [0, 40]
    cache.append(x, x, ints(table), ints(lens), ints(first))
    ref.append(x.float().cpu().numpy(), x.float().cpu().numpy(), table, lens, first)
    same_cache(cache, ref, np.array([0, 1, 2]))


@pytest.mark.parametrize("kv,dim,t", [(8, 128, 16), (2, 72, 32), (1, 256, 128), (3, 37, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_read_gives_code_times_scale(kv, dim, t, dtype):
    rng = np.random.default_rng(6)
    cache, ref = pair(kv, dim, t, 9)
    kr.fill(cache, ref, rng)
    ids = np.array([4, 0, 8, 4, -1, 9], np.int32)
    got = cache.read(ints(ids), DT[dtype])
    inside = (ids >= 0) & (ids < 9)
    at = np.where(inside, ids, 0)
    for g, codes, scale in ((got[0], ref.codes[0], ref.scale[0]), (got[1], ref.codes[1], ref.scale[1]),
                            (got[2], ref.bounds[:, :, 0], ref.scale[0]),
                            (got[3], ref.bounds[:, :, 1], ref.scale[0])):
        s = scale[at].reshape(len(ids), kv, *([1] * (codes.ndim - 2)))
        want = codes[at].astype(np.float32) * s
        want[~inside] = 0
        assert torch.equal(g.cpu(), torch.from_numpy(want).to(DT[dtype]))
    assert cache.read(ints(np.zeros(0, np.int32)))[0].shape[0] == 0


# ---- attend ---------------------------------------------------------------


def check_attend(cache, ref, q, qn, table, lens, first=None, selected=None, scale=None,
                 dtype="bf16", **kw):
    got = cache.attend(q, ints(table), ints(lens), ints(first), scale=scale,
                       selected=None if selected is None else dev(selected), **kw)
    want, bound, weight, wbound = ref.attend(qn, table, lens, first, selected, scale)
    bound = bound + ULP[dtype] * (np.abs(want) + bound) + 2.0 ** -24 * (dtype == "f16")
    bad = np.abs(got.double().cpu().numpy() - want) > bound
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4])
    return got, weight, wbound


@pytest.mark.parametrize("kv,g,dim,t,dtype", [(8, 4, 128, 16, "bf16"), (4, 8, 64, 16, "f16"),
                                              (1, 1, 80, 32, "bf16"), (2, 16, 256, 16, "f16"),
                                              (3, 5, 192, 64, "bf16"), (1, 20, 64, 128, "f16"),
                                              (2, 3, 37, 16, "bf16"), (1, 71, 128, 32, "bf16")])
def test_attend_one_token(kv, g, dim, t, dtype):
    """One token per sequence: empty ones, one token, ends of tiles, blocks
    and splits, one past them, and a table wider than any of them needs."""
    rng = np.random.default_rng(kv * 100 + g)
    lens = [0, 1, 2, 15, 16, 17, 31, 33, t, t + 1, 127, 128, 129, 300, 511, 513, 1030]
    blocks = sum(-(-n // t) for n in lens) + 3
    table = kr.make_table(rng, lens, t, blocks, width=-(-1030 // t) + 5)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    q, qn = rows(rng, (len(lens), kv * g, dim), dtype, 2.0)
    got, _, _ = check_attend(cache, ref, q, qn, table, lens, dtype=dtype)
    assert not got[0].any()
    again = cache.attend(q, ints(table), ints(lens))
    assert torch.equal(got, again)


@pytest.mark.parametrize("kv,g,dim,t,dtype", [(2, 4, 128, 16, "bf16"), (4, 1, 64, 32, "f16"),
                                              (1, 7, 96, 16, "bf16"), (1, 32, 64, 16, "f16"),
                                              (2, 2, 256, 64, "bf16")])
def test_attend_chunks(kv, g, dim, t, dtype):
    """Ragged chunks: no token, one, several, a whole prompt; some queries of
    the last sequence see nothing."""
    rng = np.random.default_rng(kv * 100 + g)
    lens, new = [90, 40, 333, 200, 0, 5], [0, 1, 9, 200, 0, 8]
    first = np.concatenate([[0], np.cumsum(new)])
    blocks = sum(-(-n // t) for n in lens) + 3
    table = kr.make_table(rng, lens, t, blocks)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    q, qn = rows(rng, (int(first[-1]), kv * g, dim), dtype, 2.0)
    got, _, _ = check_attend(cache, ref, q, qn, table, lens, first, dtype=dtype)
    assert not got[-8:-5].any() and got[-5].any()


def test_attend_many_rows_over_a_long_cache():
    """A chunk long enough for any form that takes many rows at once, whose
    last tokens cross a block, over a cache of several splits."""
    rng = np.random.default_rng(11)
    kv, g, dim, t = 2, 4, 128, 16
    lens, new = [2777, 700], [301, 130]
    first = np.concatenate([[0], np.cumsum(new)])
    blocks = sum(-(-n // t) for n in lens) + 1
    table = kr.make_table(rng, lens, t, blocks)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng, spread=1.0)
    for dtype in ("bf16", "f16"):
        q, qn = rows(rng, (int(first[-1]), kv * g, dim), dtype, 2.0)
        check_attend(cache, ref, q, qn, table, lens, first, dtype=dtype)


def test_attend_holes_garbage_and_not_finite_places():
    """Blocks that are not there count as masked; so do slots past a
    sequence's end, whatever they and their block's neighbours hold."""
    rng = np.random.default_rng(12)
    kv, g, dim, t = 2, 2, 64, 16
    lens = [100, 64, 70, 33]
    cache, ref = pair(kv, dim, t, 24)
    kr.fill(cache, ref, rng)
    table = kr.make_table(rng, lens, t, 20)
    table = np.concatenate([table, np.full((4, 2), 21, np.int32)], 1)  # past the ends: NaN blocks
    cache.key_scale[20:] = np.nan
    cache.value_scale[20:] = np.inf
    table[0, 2] = -1
    table[1, 0] = 24
    table[2, 4] = -2 ** 31
    table[3, :3] = -1          # a sequence none of whose blocks is there
    q, qn = rows(rng, (4, kv * g, dim), "bf16", 2.0)
    got, _, _ = check_attend(cache, ref, q, qn, table, lens)
    assert not got[3].any()
    # a query that is not finite makes its own row NaN and no other
    q[1, 2, 5] = np.nan
    q[2, 0, 0] = np.inf
    after = cache.attend(q, ints(table), ints(lens))
    nan = torch.isnan(after).all(-1)
    assert nan[1, 2] and nan[2, 0] and int(nan.sum()) == 2
    keep = ~nan
    assert torch.equal(after[keep], got[keep])
    # a block of NaN scale makes what reads it NaN
    cache.value_scale[int(table[0, 0]), 0] = np.nan
    after = cache.attend(q, ints(table), ints(lens))
    assert torch.isnan(after[0, :g]).all() and torch.equal(after[0, g:], got[0, g:])


@pytest.mark.parametrize("spread", [0.0, 6.0])
def test_attend_peaks_and_scales_far_apart(spread):
    """One token of nearly all the weight, placed anywhere; blocks whose value
    scales are powers apart; scale arguments of zero and below."""
    rng = np.random.default_rng(13)
    kv, g, dim, t = 2, 4, 128, 16
    lens = [700] * 6
    cache, ref = pair(kv, dim, t, 6 * 44 + 1)
    kr.fill(cache, ref, rng, spread=spread)
    table = kr.make_table(rng, lens, t, 6 * 44 + 1)
    q, qn = rows(rng, (6, kv * g, dim), "bf16", 1.0)
    for s, at in enumerate((0, 699, 17, 350, 511, 512)):
        block, slot = table[s, at // t], at % t
        for h in range(kv):
            key = ref.codes[0][block, h, slot].astype(np.float32) * ref.scale[0][block, h]
            norm = np.linalg.norm(key)
            x = torch.from_numpy(key * (60 / norm)).to(torch.bfloat16)
            q[s, h * g:(h + 1) * g] = x.cuda()
            qn[s, h * g:(h + 1) * g] = x.float().numpy()
    for scale in (None, 1.0, 0.0, -0.05, 30.0):
        check_attend(cache, ref, q, qn, table, lens, scale=scale)


@pytest.mark.parametrize("kv,g,dim,t,count", [(8, 4, 128, 16, 9), (2, 16, 64, 32, 3),
                                              (1, 1, 256, 16, 40), (3, 20, 80, 64, 1)])
def test_attend_selected(kv, g, dim, t, count):
    rng = np.random.default_rng(count)
    lens, new = [500, 77, 1, 0, 800], [1, 3, 1, 1, 2]
    first = np.concatenate([[0], np.cumsum(new)])
    blocks = sum(-(-n // t) for n in lens) + 1
    table = kr.make_table(rng, lens, t, blocks)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    tokens = int(first[-1])
    selected = np.full((tokens, kv, count), -1, np.int32)
    for s in range(len(lens)):
        for i in range(first[s], first[s + 1]):
            for h in range(kv):
                n = -(-lens[s] // t)
                pick = np.sort(rng.permutation(max(n, 1))[:rng.integers(0, count + 1)])
                selected[i, h, :len(pick)] = pick
    selected[0, 0] = -1                     # nothing selected
    selected[0, -1, 0] = table.shape[1]     # past the table: masked
    selected[0, -1, 1:] = -5
    q, qn = rows(rng, (tokens, kv * g, dim), "f16", 2.0)
    got, _, _ = check_attend(cache, ref, q, qn, table, lens, first, selected, dtype="f16")
    assert not got[0, :g].any() and not got[0, -g:].any()
    # every visible block selected is the same attention as none
    if lens[0] and -(-max(lens) // t) <= 64:
        whole = np.broadcast_to(np.arange(-(-max(lens) // t), dtype=np.int32),
                                (tokens, kv, -(-max(lens) // t)))
        check_attend(cache, ref, q, qn, table, lens, first, np.ascontiguousarray(whole), dtype="f16")


@pytest.mark.parametrize("kv,g,dim,t,chunk", [(8, 4, 128, 16, False), (2, 8, 64, 32, False),
                                              (1, 20, 80, 128, False), (2, 3, 128, 16, True),
                                              (1, 1, 256, 64, True), (4, 8, 128, 16, True)])
def test_accumulated_weights(kv, g, dim, t, chunk):
    """Weights gained by blocks, two sequences sharing a prefix's blocks; two
    runs give the same integers."""
    rng = np.random.default_rng(kv + g)
    lens, new = [1500, 300, 0, 65], [40, 33, 0, 70] if chunk else [1, 1, 1, 1]
    first = np.concatenate([[0], np.cumsum(new)]) if chunk else None
    blocks = sum(-(-n // t) for n in lens) + 1
    table = kr.make_table(rng, lens, t, blocks)
    shared = min(128 // t, 2)
    table[1, :shared] = table[0, :shared]
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    q, qn = rows(rng, (sum(new), kv * g, dim), "bf16", 2.0)
    got, weight, wbound = check_attend(cache, ref, q, qn, table, lens, first, accumulate=True)
    first_run = cache.weight.clone()
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= wbound + 2.0 ** -24 * weight).all()
    assert abs(float(cache.weights().double().sum()) - weight.sum()) <= 1e-3 * weight.sum()
    again = cache.attend(q, ints(table), ints(lens), ints(first), accumulate=True)
    assert torch.equal(got, again) and torch.equal(cache.weight, 2 * first_run)
    assert torch.equal(got, cache.attend(q, ints(table), ints(lens), ints(first)))


def test_strided_queries_and_given_output():
    rng = np.random.default_rng(21)
    kv, g, dim, t = 2, 3, 64, 16
    cache, ref = pair(kv, dim, t, 30)
    kr.fill(cache, ref, rng)
    lens = [200, 180]
    table = kr.make_table(rng, lens, t, 30)
    wide = torch.from_numpy(np.concatenate([table, table], 1)).cuda()
    big, _ = rows(rng, (2, 2, 7, kv * g, dim + 3), "bf16", 2.0)
    q = big[:, 1, 3, :, 1:1 + dim]
    out = torch.full((2, kv * g, dim), 9.0, dtype=torch.bfloat16, device="cuda")
    got = cache.attend(q, wide[:, :table.shape[1]], ints(lens), out=out)
    assert got is out
    assert torch.equal(out, cache.attend(q.contiguous(), ints(table), ints(lens)))
    check_attend(cache, ref, q, q.float().cpu().numpy(), table, lens)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes of keys: the last block and the first."""
    kv, dim, t = 8, 128, 16
    blocks = (1 << 32) // (kv * dim * t) + 3
    cache = kvcache.KvCache(blocks, kv, dim, t)
    small, ref = pair(kv, dim, t, 4)
    rng = np.random.default_rng(22)
    table = np.array([[blocks - 1, 0, blocks - 2]], np.int32)
    near = np.array([[2, 0, 1]], np.int32)
    x, xn = rows(rng, (45, kv, dim), "bf16")
    q, qn = rows(rng, (1, 4 * kv, dim), "bf16", 2.0)
    for c, tab in ((cache, table), (small, near)):
        c.append(x, x, ints(tab), ints([45]), ints([0, 45]))
    ref.append(xn, xn, near, [45], [0, 45])
    assert torch.equal(cache.keys[blocks - 1], small.keys[2])
    assert torch.equal(cache.values[blocks - 2], small.values[1])
    got, _, _ = check_attend(small, ref, q, qn, near, [45], accumulate=True)
    assert torch.equal(got, cache.attend(q, ints(table), ints([45]), accumulate=True))
    assert torch.equal(cache.weight[[blocks - 1, 0, blocks - 2]], small.weight[[2, 0, 1]])
    for a, b in zip(cache.read(ints(table[0])), small.read(ints(near[0]))):
        assert torch.equal(a, b)
    assert torch.equal(cache.select(q, ints(table), ints([45]), 2),
                       small.select(q, ints(near), ints([45]), 2))
    del cache
    torch.cuda.empty_cache()


def test_another_stream_and_a_graph():
    """The step on a side stream, and captured and replayed with other work
    between the replays."""
    rng = np.random.default_rng(23)
    kv, g, dim, t = 4, 4, 128, 16
    lens = [3000, 700, 64]
    blocks = sum(-(-n // t) for n in lens) + 1
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table = ints(kr.make_table(rng, lens, t, blocks))
    n = ints(lens)
    k, _ = rows(rng, (3, kv, dim), "bf16", 0.5)
    q, _ = rows(rng, (3, kv * g, dim), "bf16", 2.0)

    def step(stream=None):
        cache.append(k, k, table, n, stream=stream)
        chosen = cache.select(q, table, n, 20, stream=stream)
        out = cache.attend(q, table, n, selected=chosen, stream=stream)
        whole = cache.attend(q, table, n, accumulate=True, stream=stream)
        return chosen, out, whole, *cache.evict(table, n, 30, stream=stream)

    want = [x.clone() for x in step()]
    weight = cache.weight.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for handle in (side, side.cuda_stream):
        cache.weight.zero_()
        torch.cuda.synchronize()
        got = step(handle)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(cache.weight, weight)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.weight.zero_()
        got = step()
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(cache.weight, weight)
        step()


# ---- select ---------------------------------------------------------------


@pytest.mark.parametrize("kv,g,dim,t,count,dtype", [
    (8, 4, 128, 16, 12, "bf16"), (4, 8, 64, 16, 7, "f16"), (1, 1, 80, 32, 2, "bf16"),
    (2, 16, 256, 16, 100, "f16"), (3, 5, 192, 64, 3, "bf16"), (1, 64, 37, 16, 5, "bf16")])
def test_select_matches_definition(kv, g, dim, t, count, dtype):
    rng = np.random.default_rng(kv * 10 + count)
    lens, new = [0, 1, t, 900, 40, 1500], [1, 1, 2, 20, 0, 3]
    first = np.concatenate([[0], np.cumsum(new)])
    blocks = sum(-(-n // t) for n in lens) + 2
    table = kr.make_table(rng, lens, t, blocks)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table[3, 2] = -1
    table[5, 0] = blocks
    ref.scale[0][table[3, 4 % table.shape[1]], 0] = np.nan
    kr.upload(cache, ref)
    q, qn = rows(rng, (int(first[-1]), kv * g, dim), dtype, 2.0)
    for keep in ((1, 1), (0, 0), (0, 2), (2, 0)):
        got = cache.select(q, ints(table), ints(lens), count, ints(first), *keep)
        np.testing.assert_array_equal(got.cpu().numpy(),
                                      ref.select(qn, table, lens, count, first, *keep))
    got = cache.select(q[:6], ints(table), ints(lens), count)
    np.testing.assert_array_equal(got.cpu().numpy(), ref.select(qn[:6], table, lens, count))


def test_select_ties_go_to_the_lower_block():
    """Equal bounds and scales everywhere, and queries of zeros: the lowest
    blocks; a few distinct scores over many blocks."""
    rng = np.random.default_rng(31)
    kv, g, dim, t = 2, 2, 64, 16
    lens = [16 * 700, 16 * 333]
    cache, ref = pair(kv, dim, t, 1033)
    table = kr.make_table(rng, lens, t, 1033)
    ref.bounds[:, :, 0], ref.bounds[:, :, 1] = -3, 9
    kr.upload(cache, ref)
    q, qn = rows(rng, (2, kv * g, dim), "bf16")
    q[1], qn[1] = 0, 0
    for count in (3, 300, 333, 699, 700, 900):
        got = cache.select(q, ints(table), ints(lens), count).cpu().numpy()
        np.testing.assert_array_equal(got, ref.select(qn, table, lens, count))
    ref.scale[0][:] = (2.0 ** rng.integers(-2, 2, ref.scale[0].shape)).astype(np.float32)
    kr.upload(cache, ref)
    for count in (3, 300, 699):
        got = cache.select(q, ints(table), ints(lens), count).cpu().numpy()
        np.testing.assert_array_equal(got, ref.select(qn, table, lens, count))


def test_select_odd_queries():
    """Elements that are not numbers count as 0; an infinite one leaves no
    code but 0; the smallest values; far apart in size within a group."""
    rng = np.random.default_rng(32)
    kv, g, dim, t = 1, 4, 128, 16
    lens = [2000] * 5
    cache, ref = pair(kv, dim, t, 640)
    kr.fill(cache, ref, rng)
    table = kr.make_table(rng, lens, t, 640)
    q, qn = rows(rng, (5, g, dim), "bf16")
    q[0, 0, :7] = float("nan")
    q[1, 1, 1] = float("inf")
    q[2] *= 1e-38
    q[3, 0] *= 1e4
    q[4, 2, 3] = float("nan")
    q[4, 1, 3] = float("-inf")
    got = cache.select(q, ints(table), ints(lens), 25).cpu().numpy()
    np.testing.assert_array_equal(got, ref.select(q.float().cpu().numpy(), table, lens, 25))


# ---- evict ----------------------------------------------------------------


@pytest.mark.parametrize("t,kv,keep,first,last", [(16, 8, 20, 1, 1), (32, 1, 3, 0, 3),
                                                  (128, 5, 2, 1, 1), (16, 2, 300, 4, 9),
                                                  (64, 3, 1, 0, 1)])
@pytest.mark.parametrize("levels", [2, 1 << 40])
def test_evict_matches_definition(t, kv, keep, first, last, levels):
    rng = np.random.default_rng(keep)
    lens = [0, 1, t, keep * t, keep * t + 1, (keep + 1) * t, 700 * 16, 333 * 16 + 5]
    blocks = sum(-(-n // t) for n in lens) + 2
    table = kr.make_table(rng, lens, t, blocks)
    if table.shape[1] > 6:
        table[6, 3] = -1
        table[7, 5] = blocks
    weight = rng.integers(0, levels, (blocks, kv)).astype(np.int64)
    got = kvcache.evict(dev(weight), ints(table), ints(lens), keep, t, first, last)
    want = kr.evict(weight, table, lens, keep, t, first, last)
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.cpu().numpy(), b)


def test_evict_wide_table_and_large_weights():
    rng = np.random.default_rng(41)
    n = 20_000
    table = rng.permutation(n).astype(np.int32)[None]
    weight = (rng.integers(0, 1 << 20, (n, 4)) << 40).astype(np.int64)
    for keep in (2, 777, 19_999, 20_000):
        got = kvcache.evict(dev(weight), ints(table), ints([n * 16 - 3]), keep)
        want = kr.evict(weight, table, [n * 16 - 3], keep, 16)
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a.cpu().numpy(), b)


def test_decode_after_eviction():
    """A study's loop: prompt, steps with weights, eviction, more steps."""
    rng = np.random.default_rng(42)
    kv, g, dim, t, keep = 2, 4, 64, 16, 6
    cache, ref = pair(kv, dim, t, 40)
    table = kr.make_table(rng, [160, 130], t, 40, width=12)
    lens, first = np.array([150, 100]), np.array([0, 150, 250])
    x, xn = rows(rng, (250, kv, dim), "bf16")
    cache.append(x, x, ints(table), ints(lens), ints(first))
    ref.append(xn, xn, table, lens, first)
    tab, n = ints(table), ints(lens)
    for step in range(8):
        lens = lens + 1
        n = n + 1
        x, xn = rows(rng, (2, kv, dim), "bf16", 1.0 + 0.2 * step)
        q, qn = rows(rng, (2, kv * g, dim), "bf16", 2.0)
        cache.append(x, x, tab, n)
        ref.append(xn, xn, table, lens)
        check_attend(cache, ref, q, qn, table, lens, accumulate=True)
        if step == 4:
            weight = cache.weight.cpu().numpy()
            tab, n, _, _ = cache.evict(tab, n, keep)
            table, lens, _, _ = kr.evict(weight, table, lens, keep, t)
            np.testing.assert_array_equal(tab.cpu().numpy(), table)
            np.testing.assert_array_equal(n.cpu().numpy(), lens)
            spare = [b for b in range(40) if b not in set(table.ravel().tolist())]
            for s in range(2):  # room for the tokens to come
                table[s, -(-lens[s] // t):-(-lens[s] // t) + 2] = spare[2 * s:2 * s + 2]
            tab = ints(table)
