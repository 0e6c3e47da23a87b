"""The paged cache's operators on another stream than the current one, beside
work that still uses memory the current stream has given back."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvcache_ref as kr
from hbfsim_amd import kvcache
from test_gpu_kvcache import ints, pair, rows

pytestmark = pytest.mark.gpu


def operators():
    """(name, call of a stream) over a filled cache, of several splits and of
    scratch in each that takes any."""
    rng = np.random.default_rng(61)
    kv, g, dim, t = 4, 4, 128, 16
    lens, first = [5000, 700, 64], [0, 3, 5, 6]
    blocks = sum(-(-n // t) for n in lens) + 1
    cache, ref = pair(kv, dim, t, blocks)
    kr.fill(cache, ref, rng)
    table, n, first = ints(kr.make_table(rng, lens, t, blocks)), ints(lens), ints(first)
    q, _ = rows(rng, (6, kv * g, dim), "bf16", 2.0)
    chosen = cache.select(q, table, n, 20, first)
    cache.weight.copy_(torch.from_numpy(rng.integers(0, 1 << 40, (blocks, kv))))
    ids = ints(np.arange(40))
    return cache, [
        ("attend", lambda s: [cache.attend(q[:3], table, n, stream=s)]),
        ("attend first", lambda s: [cache.attend(q, table, n, first, stream=s)]),
        ("attend selected", lambda s: [cache.attend(q, table, n, first, chosen, stream=s)]),
        ("attend weigh", lambda s: [cache.attend(q, table, n, first, accumulate=True, stream=s)]),
        ("select", lambda s: [cache.select(q, table, n, 20, first, stream=s)]),
        ("read", lambda s: list(cache.read(ids, stream=s))),
        ("evict", lambda s: list(cache.evict(table, n, 30, stream=s))),
        ("evict weights", lambda s: list(kvcache.evict(cache.weight, table, n, 30, stream=s)))]


def pending(load):
    """Buffers of every size whose copies wait behind a long product on the
    current stream, and that have been given back by the time this returns."""
    used = [torch.full((1 << k,), 7, dtype=torch.uint8, device="cuda")
            for k in range(9, 25) for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(12):
        torch.mm(load, load)
    return [x.clone() for x in used]


@pytest.mark.parametrize("raw", [False, True])
def test_memory_given_back_with_work_pending_is_left_alone(raw):
    cache, calls = operators()
    side = torch.cuda.Stream()
    load = torch.zeros((8192, 8192), dtype=torch.bfloat16, device="cuda")
    torch.mm(load, load)
    weight = cache.weight.clone()
    for name, call in calls:
        cache.weight.copy_(weight)
        want = [x.clone() for x in call(None)]
        gained = cache.weight.clone()
        cache.weight.copy_(weight)
        torch.cuda.synchronize()  # the side stream needs no more than the inputs
        copies = pending(load)
        got = call(side.cuda_stream if raw else side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
        torch.cuda.synchronize()
        assert all(bool((x == 7).all()) for x in copies), name
        assert torch.equal(cache.weight, gained), name


def test_outputs_given_back_while_the_caller_still_reads_them():
    """An output of the side stream, read by work queued on the current one and
    then given back, is not handed to the side stream's next call."""
    _, calls = operators()
    side = torch.cuda.Stream()
    load = torch.zeros((8192, 8192), dtype=torch.bfloat16, device="cuda")
    torch.mm(load, load)
    call = dict(calls)["read"]
    want = [x.clone() for x in call(None)]
    torch.cuda.synchronize()
    got = call(side)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(12):
        torch.mm(load, load)
    copies = [x.clone() for x in got]
    del got
    with torch.cuda.stream(side):
        over = [torch.full_like(x, 9) for x in want]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(copies, want))
    del over
