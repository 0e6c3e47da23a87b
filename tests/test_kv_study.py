"""The paged cache's flash accesses (host) and the study that runs the cache's
operators and the timing engine together (GPU)."""
from __future__ import annotations

import numpy as np
import pytest

from hbfsim_amd import workloads as w


def test_cache_spans_cover_what_a_step_touches():
    kv, head = 3, 2048
    reads = np.array([[5, 0], [5, 2], [0, 1]])
    base, first, op = w.kv_cache_spans(1 << 30, 1 << 31, head, kv, reads, np.array([7, 2]))
    rec = w.span_records(base, first, op, 128, 64_000, 256)
    assert len(rec) == int(first[-1]) == (2 * 2 * kv * head + 2 * 3 * head) // 128
    want = []
    for pool in (1 << 30, 1 << 31):
        want += [(pool + b * kv * head + i, 1) for b in (7, 2) for i in range(0, kv * head, 128)]
        want += [(pool + (b * kv + h) * head + i, 0) for b, h in reads for i in range(0, head, 128)]
    assert sorted((int(r[0]), int(r[3])) for r in rec) == sorted((int(a), o) for a, o in want)
    none = w.kv_cache_spans(0, 1 << 30, head, kv, np.zeros((0, 2)), np.zeros(0))
    assert none[1].tolist() == [0]
    assert int(w.kv_cache_spans(0, 1 << 30, head, kv, reads, np.zeros(0))[1][-1]) == 6 * head // 128


@pytest.mark.parametrize("kw", [dict(head_bytes=100), dict(head_bytes=0), dict(key_base=64),
                                dict(value_base=1), dict(reads=np.array([[1, 3]])),
                                dict(reads=np.array([[-1, 0]])), dict(writes=np.array([-1]))])
def test_cache_spans_refused(kw):
    args = dict(key_base=0, value_base=1 << 20, head_bytes=2048, kv_heads=3,
                reads=np.array([[0, 0]]), writes=np.zeros(0))
    args.update(kw)
    with pytest.raises(ValueError):
        w.kv_cache_spans(**args)


@pytest.mark.gpu
def test_study_runs_the_step_and_its_flash_together():
    from hbfsim_amd import kv_study

    got = kv_study.run(seqs=3, tokens=1024, steps=20, count=12, keep=20, heads=8, kv_heads=2,
                       head_dim=64, seed=5)
    # the cut comes after 10 steps: 1034 tokens, 65 blocks a sequence, 20 kept
    assert got["evicted_blocks"] == 3 * (65 - 20)
    before, after = got["dense"]["before"], got["dense"]["after"]
    # 64 full blocks of 1 KiB a pool and head, 16 tokens a block
    assert before["accesses"] == 3 * 2 * 2 * 64 * 1024 // 128
    assert after["accesses"] < before["accesses"] / 3
    some = got["selected"]["before"]
    # of 12 blocks one is the last, which is not full
    assert some["accesses"] == 3 * 2 * 2 * 11 * 1024 // 128
    assert 0 < some["ms"] < before["ms"]
    # the blocks that the queries lean towards are found
    assert got["attention_held"]["before"] > 0.5
    assert got["output_error"] < 0.6
