"""How the paged cache's calls reach the library, without a GPU: a stub stands
in its place."""
from __future__ import annotations

import pytest
import torch

from hbfsim_amd import _native as nat
from hbfsim_amd import kvcache

I32 = torch.int32


class Library:
    """Notes every call; nothing is queued."""

    def __init__(self, seen=lambda name, args: None):
        self.calls, self.seen = [], seen

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            self.seen(name, args)
            return nat.HBFSIM_OK
        return call


def every_call(cache, device, **kw):
    """(name, call) of each operator with arguments that fit."""
    table, lens = (torch.zeros(s, dtype=I32, device=device) for s in ((3, 2), (3,)))
    first = torch.arange(4, dtype=I32, device=device)
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device=device)
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device=device)
    chosen = torch.zeros((3, 2, 1), dtype=I32, device=device)
    return [("append", lambda: cache.append(k, k, table, lens, **kw)),
            ("append", lambda: cache.append(k, k, table, lens, first, **kw)),
            ("read", lambda: cache.read(lens, **kw)),
            ("attend", lambda: cache.attend(q, table, lens, **kw)),
            ("attend", lambda: cache.attend(q, table, lens, out=torch.zeros_like(q), **kw)),
            ("attend", lambda: cache.attend(q, table, lens, first, accumulate=True, **kw)),
            ("attend", lambda: cache.attend(q, table, lens, selected=chosen, **kw)),
            ("select", lambda: cache.select(q, table, lens, 2, **kw)),
            ("evict", lambda: cache.evict(table, lens, 2, **kw)),
            ("evict", lambda: kvcache.evict(cache.weight, table, lens, 2, **kw))]


@pytest.mark.parametrize("stream", [None, 0, 12345])
def test_host_memory_reaches_no_kernel(monkeypatch, stream):
    """A cache may be built of host tensors, but no operator runs on it: the
    kernels would be handed host addresses."""
    library = Library()
    monkeypatch.setattr(nat, "load", lambda: library)
    cache = kvcache.KvCache(4, 2, 64, device="cpu")
    for name, call in every_call(cache, "cpu", stream=stream):
        with pytest.raises(ValueError, match="GPU"):
            call()
    assert library.calls == []
