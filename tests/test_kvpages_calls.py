"""How the calls on a paged cache's blocks and on drafted tokens reach the
library, without a GPU: a stub stands in its place."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from hbfsim_amd import _native as nat
from hbfsim_amd import drafts, kvcache
from test_kvcache_calls import Library, Machine

I32 = torch.int32
MAKES = {"fork", "grow", "compact", "verify", "verify without lengths"}  # outputs of their own
QUIET = {"hold", "release"}  # nor scratch memory


def every_call(cache, device, **kw):
    table, lens = (torch.zeros(s, dtype=I32, device=device) for s in ((3, 2), (3,)))
    first = torch.arange(4, dtype=I32, device=device)
    p, u = (torch.zeros(s, device=device) for s in ((3, 9), (3,)))
    return [("copy", lambda: cache.copy(lens, lens, **kw)),
            ("hold", lambda: cache.hold(table, **kw)),
            ("fork", lambda: cache.fork(table, lens, lens, **kw)),
            ("release", lambda: cache.release(table, **kw)),
            ("release", lambda: kvcache.release(cache.refs, table, lens, 32, **kw)),
            ("grow", lambda: cache.grow(table, lens, **kw)),
            ("grow", lambda: cache.grow(table, lens, first, 3, **kw)),
            ("compact", lambda: cache.compact(table, **kw)),
            ("verify", lambda: drafts.verify(p, lens, u, first, p, lens, **kw)),
            ("verify without lengths", lambda: drafts.verify(p, lens, u, **kw))]


@pytest.mark.parametrize("stream", [None, 0, 12345])
def test_host_memory_reaches_no_kernel(monkeypatch, stream):
    library = Library()
    monkeypatch.setattr(nat, "load", lambda: library)
    cache = kvcache.KvCache(4, 2, 64, device="cpu")
    for name, call in every_call(cache, "cpu", stream=stream):
        with pytest.raises(ValueError, match="GPU"):
            call()
    assert library.calls == []


def on_machine(monkeypatch, device, stream):
    rows = []
    with FakeTensorMode(), monkeypatch.context() as patch:
        machine = Machine(patch)

        def seen(name, args):
            if name.endswith("workspace"):
                args[-1]._obj.value = 4096
            else:
                rows.append((machine.device, args[-1], machine.made[:]))

        patch.setattr(nat, "load", lambda: Library(seen))
        patch.setattr(drafts, "_need", {})
        cache = kvcache.KvCache(4, 2, 64, device=device)
        got = []
        for name, call in every_call(cache, device, stream=stream(machine)):
            rows.clear(), machine.made.clear(), machine.recorded.clear()
            call()
            (current, handle, made), = rows
            got.append((name, current, handle, made, machine.recorded[:]))
            assert machine.device == 0 and machine.stream == {0: 0, 1: 0}
    return got


@pytest.mark.parametrize("raw", [False, True])
def test_memory_comes_from_the_pool_of_the_stream_that_writes_it(monkeypatch, raw):
    for name, _, handle, made, recorded in on_machine(
            monkeypatch, "cuda:0", lambda m: 77 if raw else m.Stream(77, "cuda:0")):
        assert handle == 77
        assert set(made) <= {(0, 77)} and bool(made) == (name not in QUIET), (name, made)
        assert set(recorded) <= {(0, 0)} and bool(recorded) == (name in MAKES), (name, recorded)
    for _, _, handle, made, recorded in on_machine(monkeypatch, "cuda:0", lambda m: None):
        assert handle == 0 and set(made) <= {(0, 0)} and not recorded


def test_the_cache_s_gpu_is_current_in_its_calls(monkeypatch):
    for stream, handle in ((lambda m: None, 0), (lambda m: 0, 0), (lambda m: 77, 77),
                           (lambda m: m.Stream(77, "cuda:1"), 77)):
        for name, current, got, made, _ in on_machine(monkeypatch, "cuda:1", stream):
            assert (current, got) == (1, handle), (name, current, got)
            assert set(made) <= {(1, handle)}, (name, made)


def test_a_stream_of_another_gpu_is_refused(monkeypatch):
    for device, other in (("cuda:0", "cuda:1"), ("cuda:1", "cuda:0")):
        with pytest.raises(ValueError, match="stream"):
            on_machine(monkeypatch, device, lambda m: m.Stream(77, other))


def test_arguments_past_32_bits(monkeypatch):
    with FakeTensorMode(), monkeypatch.context() as patch:
        Machine(patch)
        got = []
        patch.setattr(nat, "load", lambda: Library(lambda name, args: got.append(name)))
        cache = kvcache.KvCache(4, 2, 64, device="cuda:0")
        lens = torch.zeros((3,), dtype=I32, device="cuda:0")
        first = torch.zeros((4,), dtype=I32, device="cuda:0")
        far = torch.empty_strided((3, 2), (2 ** 32 + 2, 1), dtype=I32, device="cuda:0")
        table = torch.zeros((3, 2), dtype=I32, device="cuda:0")
        for bad in (lambda: cache.hold(far), lambda: cache.fork(far, lens, lens),
                    lambda: cache.release(far), lambda: cache.grow(far, lens),
                    lambda: cache.compact(far), lambda: cache.grow(table, lens, first, 2 ** 32 + 3),
                    lambda: kvcache.release(cache.refs, table, lens, 2 ** 32 + 16)):
            with pytest.raises(ValueError):
                bad()
        assert got == []
