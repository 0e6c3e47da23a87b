"""What `verify` refuses of lengths and outputs, without a GPU."""
from __future__ import annotations

import pytest
import torch

from hbfsim_amd import _native as nat
from hbfsim_amd import drafts
from test_kvpages_host import BAD, FAR, HERE, RUNS, no_gpu


def verify(lens=HERE + 4 * FAR, stored=HERE + 7 * FAR, out=HERE + 5 * FAR,
           out_lens=HERE + 8 * FAR, first=HERE + 3 * FAR, gained=HERE + 6 * FAR, seqs=2, rows=5,
           vocab=100):
    return nat.load().hbfsim_amd_verify_step(
        HERE, HERE, 2, vocab, vocab, vocab, HERE + FAR, HERE + 2 * FAR, first, seqs, rows, lens, stored,
        out, gained, out_lens, HERE, 1 << 20, None)


@no_gpu
def test_the_c_call():
    assert verify() == RUNS and verify(stored=None) == RUNS
    assert verify(lens=None, stored=None, out_lens=None) == RUNS
    assert verify(out_lens=HERE + 4 * FAR) == RUNS and verify(out_lens=HERE + 7 * FAR) == RUNS
    for kw in (dict(lens=None), dict(lens=None, out_lens=None), dict(out_lens=None),
               dict(stored=HERE + 5 * FAR + 16), dict(stored=HERE + 5 * FAR - 4)):
        assert verify(**kw) == BAD, kw


@no_gpu
def test_outputs_that_overlap():
    """A sequence's results are written while others are read.  Tokens and
    uniforms hold 20 bytes, offsets 12, lengths 8."""
    for name in ("gained", "out_lens"):
        for at in (HERE + FAR, HERE + FAR + 16, HERE + 2 * FAR - 4, HERE + 2 * FAR + 8, HERE + 3 * FAR,
                   HERE + 3 * FAR + 8, HERE + 5 * FAR - 4, HERE + 5 * FAR + 16, HERE + 4 * FAR + 4,
                   HERE + 4 * FAR - 4, HERE + 7 * FAR + 4):
            assert verify(**{name: at}) == BAD, (name, at - HERE)
        for at in (HERE + FAR + 20, HERE + 2 * FAR - 8, HERE + 3 * FAR + 12, HERE + 4 * FAR + 8,
                   HERE + 5 * FAR + 20):
            assert verify(**{name: at}) == RUNS, (name, at - HERE)
    assert verify(gained=HERE + 4 * FAR) == BAD and verify(gained=HERE + 7 * FAR) == BAD
    assert verify(gained=HERE + 8 * FAR + 4) == BAD and verify(gained=HERE + 8 * FAR + 8) == RUNS
    assert verify(first=None, seqs=5, out_lens=HERE + 3 * FAR) == RUNS


def test_the_python_call():
    p, u = torch.zeros((3, 50)), torch.zeros(3)
    ids = torch.zeros(3, dtype=torch.int32)
    for bad in (dict(stored=ids), dict(lens=ids, stored=ids[:2]), dict(lens=ids, stored=ids.long())):
        with pytest.raises(ValueError) as e:
            drafts.verify(p, ids, u, **bad)
        assert "not on a GPU" not in str(e.value)
    with pytest.raises(ValueError, match="not on a GPU"):
        drafts.verify(p, ids, u, lens=ids, stored=ids)
