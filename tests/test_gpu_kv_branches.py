"""A branching, drafting decode as it is run: grow, append, fork, attend,
verify, release, compact on one cache, against a cache in which every sequence
has blocks of its own; and the study that does so with flash timing."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvpages_ref as pr
from hbfsim_amd import drafts, kvcache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,heads,dim,t", [(2, 8, 64, 16), (1, 3, 100, 32)])
def test_shared_blocks_attend_as_blocks_of_their_own(kv, heads, dim, t):
    """Both caches see the same appends, so that every block's codes are the
    same; attention over them is then equal to the last bit."""
    gen = torch.Generator(device="cuda").manual_seed(t)
    rng = np.random.default_rng(t)
    rows, width, steps = 9, 12, 14
    shared = kvcache.KvCache(rows * width, kv, dim, t)
    alone = kvcache.KvCache(2 * rows * width, kv, dim, t)
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")

    def private(n, half):
        at = half * rows * width + torch.arange(n * width, device="cuda")
        return at.view(n, width).to(torch.int32)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").bfloat16()

    own, half = private(3, 0), 0
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    counts = torch.tensor([37, 3 * t, t + 1], dtype=torch.int32, device="cuda")
    vocab, forks, compactions = 70, 0, 0
    for step in range(steps):
        n = table.shape[0]
        first = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        first[1:] = counts.cumsum(0)
        total = int(first[-1])
        now, missing = shared.grow(table, lens + counts, first, total)
        assert not missing.any() and torch.equal(now, lens + counts)
        k, v, q = normal(total, kv, dim), normal(total, kv, dim), normal(total, heads, dim)
        shared.append(k, v, table, now, first)
        alone.append(k, v, own, now, first)
        a = shared.attend(q, table, now, first)
        b = alone.attend(q, own, now, first)
        assert torch.equal(a, b) and torch.isfinite(a.float()).all()
        # drafts: some stay
        p = torch.softmax(torch.randn((total, vocab), generator=gen, device="cuda") * 3, 1)
        d = torch.softmax(torch.log(p) + torch.randn((total, vocab), generator=gen, device="cuda"), 1)
        said = d.argmax(1).roll(1).to(torch.int32)
        u = torch.rand((total,), generator=gen, device="cuda")
        out, gained, lens = drafts.verify(p, said, u, first, draft=d, lens=now)
        want = pr.verify(p.cpu().numpy(), said.cpu().numpy(), u.cpu().numpy(), first.tolist(),
                         d.cpu().numpy(), now.cpu().numpy())
        for got, x in zip((out, gained, lens), want):
            np.testing.assert_array_equal(got.cpu(), x)
        shared.release(table, lens)
        np.testing.assert_array_equal(shared.refs.cpu(), pr.count(table.cpu().numpy(), rows * width))
        blocks = (lens + t - 1) // t
        assert torch.equal((table >= 0).sum(1), blocks.long())
        if step % 3 == 2:  # branches, and some sequences end
            parents = torch.from_numpy(rng.integers(0, n, rows if step < 9 else 4).astype(np.int32))
            parents = parents.cuda()
            table, lens = shared.fork(table, lens, parents)
            half = 1 - half
            new = private(len(parents), half)
            alone.copy(own[parents.long()].reshape(-1), new.reshape(-1))
            own = new
            forks += 1
        if step % 4 == 3:
            shared.compact(table)
            used = int((shared.refs > 0).sum())
            assert (shared.refs[:used] > 0).all() and int(table.max()) < used
            compactions += 1
        counts = torch.from_numpy(rng.integers(0, 6, table.shape[0]).astype(np.int32)).cuda()
        # no sequence outgrows its row
        counts = torch.minimum(counts, (width * t - lens).clamp(min=0))
    assert forks == 4 and compactions == 3


def test_study_of_branches_and_drafts():
    from hbfsim_amd import kv_study

    got = kv_study.run_drafts(seqs=2, tokens=520, steps=10, branches=3, drafts=3, vocab=500, heads=4,
                              kv_heads=2, head_dim=64, seed=1)
    assert got["missing"] == 0
    for part in ("before", "after"):
        assert 1 < got[part]["gained"] <= 4 and got[part]["accesses"] > 0
    moved = got["compaction"]
    # a prompt's 32 full blocks are held once, whatever shares them: of rows 0,
    # 2 and 4, which stay, the first two are of the first prompt
    assert moved["named_by_rows"] - moved["blocks"] == 32
    assert moved["ms_before"] > 0 and moved["ms_after"] > 0
    plain = kv_study.run_drafts(seqs=2, tokens=520, steps=4, branches=1, drafts=0, vocab=500, heads=4,
                                kv_heads=2, head_dim=64, seed=1)
    assert plain["before"]["gained"] == 1.0
