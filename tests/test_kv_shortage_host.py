"""What `verify` refuses of the lengths before a step, without a GPU."""
from __future__ import annotations

import pytest
import torch

from hbfsim_amd import _native as nat
from hbfsim_amd import drafts
from test_kvpages_host import BAD, FAR, HERE, RUNS, no_gpu


def verify(lens=HERE + 4 * FAR, stored=HERE + 7 * FAR, out=HERE + 5 * FAR,
           out_lens=HERE + 8 * FAR, first=HERE + 3 * FAR, seqs=2, rows=5, vocab=100):
    return nat.load().hbfsim_amd_verify_step(
        HERE, HERE, 2, vocab, vocab, vocab, HERE + FAR, HERE + 2 * FAR, first, seqs, rows, lens, stored,
        out, HERE + 6 * FAR, out_lens, HERE, 1 << 20, None)


@no_gpu
def test_the_c_call():
    assert verify() == RUNS and verify(stored=None) == RUNS
    assert verify(lens=None, stored=None, out_lens=None) == RUNS
    assert verify(out_lens=HERE + 4 * FAR) == RUNS and verify(out_lens=HERE + 7 * FAR) == RUNS
    for kw in (dict(lens=None), dict(lens=None, out_lens=None), dict(out_lens=None),
               dict(stored=HERE + 5 * FAR + 16), dict(stored=HERE + 5 * FAR - 4)):
        assert verify(**kw) == BAD, kw


def test_the_python_call():
    p, u = torch.zeros((3, 50)), torch.zeros(3)
    ids = torch.zeros(3, dtype=torch.int32)
    for bad in (dict(stored=ids), dict(lens=ids, stored=ids[:2]), dict(lens=ids, stored=ids.long())):
        with pytest.raises(ValueError) as e:
            drafts.verify(p, ids, u, **bad)
        assert "not on a GPU" not in str(e.value)
    with pytest.raises(ValueError, match="not on a GPU"):
        drafts.verify(p, ids, u, lens=ids, stored=ids)
