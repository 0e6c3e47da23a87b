"""Attention of many query rows where blocks' value scales are far apart: a
block of small or zero values still has its share of the denominator."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvcache_ref as kr
from hbfsim_amd import kvcache
from test_gpu_kvcache import check_attend, ints, pair, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("new", [1, 280])
def test_blocks_of_zero_values_take_their_share(dim, new):
    """Queries of zeros weigh every token alike, so a row is the mean of the
    values that it sees: ones in the even blocks, zeros in the odd ones, whose
    scale is the least there is.  The bound is the output's own rounding and
    that of the sums."""
    t, n = 16, 320
    v = (torch.arange(n) // t % 2 == 0).float()
    cache = kvcache.KvCache(n // t, 1, dim, t)
    table, lens = ints(np.arange(n // t)[None]), ints([n])
    k = torch.randn((n, 1, dim), generator=torch.Generator().manual_seed(dim))
    cache.append(k.cuda(), v[:, None, None].expand(n, 1, dim).cuda(), table, lens, ints([0, n]))
    assert cache.value_scale.min() == 2.0 ** -40
    q = torch.zeros((new, 1, dim), dtype=torch.float16, device="cuda")
    got = cache.attend(q, table, lens, ints([0, new]), accumulate=True).double().cpu()
    seen = torch.arange(n - new + 1, n + 1)
    want = (torch.cumsum(v.double(), 0) / torch.arange(1, n + 1))[seen - 1]
    assert ((got[:, 0] - want[:, None]).abs() <= 2.0 ** -10 * want[:, None]).all()
    # each block's weight: the tokens of it that a row sees, over all it sees
    inside = (seen[:, None] - torch.arange(n // t) * t).clamp(0, t)
    share = (inside / seen[:, None]).double().sum(0)
    assert torch.allclose(cache.weights()[:, 0].double().cpu(), share, rtol=1e-5)


@pytest.mark.parametrize("kv,g,dim,t,dtype", [(1, 4, 64, 16, "bf16"), (2, 3, 128, 16, "f16"),
                                              (1, 2, 192, 32, "bf16"), (1, 2, 256, 16, "bf16"),
                                              (2, 1, 200, 128, "f16"), (1, 5, 250, 64, "bf16")])
def test_value_scales_from_the_least_up(kv, g, dim, t, dtype):
    """Every power of two from 2^-40 to 2^3 among the blocks of a sequence, zero
    values in some, with and without the weights."""
    rng = np.random.default_rng(dim + t)
    lens, first = [44 * t - 5, 300], [0, 270, 340]
    blocks = sum(-(-n // t) for n in lens)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    power = rng.permutation(blocks)[:, None] % 44 - 40
    ref.scale[1][:] = 2.0 ** power.astype(np.float32)
    ref.codes[1][(power == -40)[:, 0]] = 0
    kr.upload(cache, ref)
    table = kr.make_table(rng, lens, t, blocks)
    q, qn = rows(rng, (340, kv * g, dim), dtype, 1.0)
    check_attend(cache, ref, q, qn, table, lens, first, dtype=dtype)
    _, weight, wbound = check_attend(cache, ref, q, qn, table, lens, first, dtype=dtype,
                                     accumulate=True)
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= wbound + 2.0 ** -24 * weight).all()


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("new", [1, 3, 120])
def test_blocks_of_scale_zero_hold_zeros(dim, new):
    """Arrays that a caller made of zeros: a block not begun yet stands for
    zeros, and what sees it weighs it as that (the oracle's block has codes of
    zero; 2^-33 is the largest code at the least scale)."""
    rng = np.random.default_rng(dim + new)
    kv, g, t, n = 2, 4, 16, 500
    blocks = -(-n // t)
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table = kr.make_table(rng, [n], t, blocks)
    zero = table[0, [0, 3, 4, 17, 31]]
    scales = [x.clone() for x in (cache.key_scale, cache.value_scale)]
    for x in scales:
        x[torch.from_numpy(zero).long().cuda()] = 0
    for codes in ref.codes:
        codes[zero] = 0
    q, qn = rows(rng, (new, kv * g, dim), "f16", 1.0)
    first = [0, new]
    want, bound, weight, wbound = ref.attend(qn, table, [n], first)
    bound = bound + 2.0 ** -33 + 2.0 ** -11 * (np.abs(want) + bound) + 2.0 ** -24
    cache.key_scale.copy_(scales[0])
    cache.value_scale.copy_(scales[1])
    got = cache.attend(q, ints(table), ints([n]), ints(first), accumulate=True)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    diff = np.abs(cache.weights().double().cpu().numpy() - weight)
    assert (diff <= wbound + 2.0 ** -24 * weight).all()
    cache.keys.zero_(), cache.values.zero_(), cache.key_scale.zero_(), cache.value_scale.zero_()
    assert not cache.attend(q, ints(table), ints([n]), ints(first)).any()
