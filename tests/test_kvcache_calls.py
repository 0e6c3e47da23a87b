"""How the paged cache's calls reach the library, without a GPU: a stub stands
in its place."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

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
            ("attend into", lambda: cache.attend(q, table, lens, out=torch.zeros_like(q), **kw)),
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


class Machine:
    """Two GPUs that are not there: which of them and which stream is current,
    and what is allocated where.  Streams are named (device, handle)."""

    def __init__(self, patch):
        self.device, self.stream = 0, {0: 0, 1: 0}
        self.made, self.recorded = [], []
        machine = self

        class Stream:
            def __init__(self, handle, device):
                self.cuda_stream, self.device = handle, torch.device(device)

        class Device:
            def __init__(self, device):
                self.index = torch.device(device).index

            def __enter__(self):
                self.before, machine.device = machine.device, self.index

            def __exit__(self, *_):
                machine.device = self.before

        class On(Device):
            def __init__(self, stream):
                super().__init__(stream.device)
                self.handle = stream.cuda_stream

            def __enter__(self):
                super().__enter__()
                self.was = machine.stream[self.index]
                machine.stream[self.index] = self.handle

            def __exit__(self, *_):
                machine.stream[self.index] = self.was
                super().__exit__()

        empty = torch.empty

        def make(*args, device, **kw):
            if torch.device(device).type == "cuda":
                index = torch.device(device).index
                self.made.append((index, self.stream[index]))
            return empty(*args, device=device, **kw)

        self.Stream = Stream
        patch.setattr(torch.cuda, "ExternalStream", Stream)
        patch.setattr(torch.cuda, "device", Device)
        patch.setattr(torch.cuda, "stream", On)
        patch.setattr(torch.cuda, "current_device", lambda: self.device)
        patch.setattr(torch.cuda, "current_stream",
                      lambda device=None: Stream(self.stream[self.index(device)],
                                                 f"cuda:{self.index(device)}"))
        patch.setattr(torch._C, "_cuda_getDevice", lambda: self.device, raising=False)
        patch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: self.stream[index],
                      raising=False)
        patch.setattr(torch.Tensor, "data_ptr", lambda t: 4096)
        patch.setattr(torch.Tensor, "record_stream", lambda t, s: self.recorded.append(
            (s.device.index, s.cuda_stream)))
        patch.setattr(torch, "empty", make)

    def index(self, device):
        return self.device if device is None else torch.device(device).index


def on_machine(monkeypatch, device, stream):
    """Every operator of a cache on `device`: (what was current when the
    library was called, the stream it was given, where it had tensors made,
    streams that the outputs were recorded on)."""
    launches = {"append", "read", "attend", "select", "evict"}
    rows = []
    with FakeTensorMode(), monkeypatch.context() as patch:
        machine = Machine(patch)

        def seen(name, args):
            if name.removeprefix("hbfsim_amd_kv_") in launches:
                rows.append((machine.device, args[-1], machine.made[:]))
            elif name.endswith("workspace"):
                args[-1]._obj.value = 4096

        library = Library(seen)
        patch.setattr(nat, "load", lambda: library)
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
    """Scratch and outputs of a call on another stream: a block just freed on
    the current one may have work queued on it that the other is not ordered
    behind.  The outputs are recorded on the caller's stream, which reads them."""
    for name, _, handle, made, recorded in on_machine(
            monkeypatch, "cuda:0", lambda m: 77 if raw else m.Stream(77, "cuda:0")):
        assert handle == 77
        assert set(made) <= {(0, 77)} and bool(made) == (name != "append"), (name, made)
        own = name not in ("append", "attend into")  # outputs that the call makes itself
        assert set(recorded) <= {(0, 0)} and bool(recorded) == own, (name, recorded)
    for _, _, handle, made, recorded in on_machine(monkeypatch, "cuda:0", lambda m: None):
        assert handle == 0 and set(made) <= {(0, 0)} and not recorded


def test_the_cache_s_gpu_is_current_in_its_calls(monkeypatch):
    """Handle 0 is the current device's default stream: with another GPU
    current, the launch would go there."""
    for stream, handle in ((lambda m: None, 0), (lambda m: 0, 0), (lambda m: 77, 77),
                           (lambda m: m.Stream(77, "cuda:1"), 77)):
        for name, current, got, made, _ in on_machine(monkeypatch, "cuda:1", stream):
            assert (current, got) == (1, handle), (name, current, got)
            assert set(made) <= {(1, handle)}, (name, made)


def test_a_stream_of_another_gpu_is_refused(monkeypatch):
    for device, other in (("cuda:0", "cuda:1"), ("cuda:1", "cuda:0")):
        with pytest.raises(ValueError, match="stream"):
            on_machine(monkeypatch, device, lambda m: m.Stream(77, other))


HERE = 0x7f0000000000  # a device address that no call here reaches


def attend_at(q, out, token_stride, head_stride, tokens=3, first=None, acc=0, heads=4, dim=64):
    """The C call with queries and output at these addresses; what it does not
    refuse has no GPU to run on."""
    c = nat.KvCacheArrays(ctypes.sizeof(nat.KvCacheArrays), 8, 2, dim, 16, 0, *[HERE] * 6)
    b = nat.KvBatch(ctypes.sizeof(nat.KvBatch), 3, 4, 4, tokens, 0, HERE, HERE, first)
    return nat.load().hbfsim_amd_kv_attend(
        ctypes.byref(c), ctypes.byref(b), q, nat.KV_BF16, heads, token_stride, head_stride, 0.1,
        None, 0, acc, out, HERE, 1 << 30, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="its addresses are not a GPU's")
def test_outputs_over_the_queries():
    """An output may be the queries themselves, row for row, unless they are
    read again for the weights; any other overlap would have rows read after
    they are overwritten."""
    at, row = HERE + (1 << 20), 4 * 64
    bad, runs = nat.HBFSIM_INVALID_ARGUMENT, nat.HBFSIM_CUDA_ERROR
    size = 3 * row * 2
    for out, strides, kw, want in (
            (at, (row, 64), {}, runs),                          # in place
            (at, (row, 64), dict(acc=1), runs),                 # one token each: not read again
            (at, (row, 64), dict(first=HERE), runs),
            (at, (row, 64), dict(first=HERE, acc=1), bad),
            (at + size, (row, 64), dict(first=HERE, acc=1), runs),
            (at - size, (row, 64), dict(first=HERE, acc=1), runs),
            (at + 128, (row, 64), {}, bad),                     # a head further
            (at - 512, (row, 64), {}, bad),                     # a token before
            (at + size - 2, (row, 64), {}, bad),
            (at, (2 * row, 64), {}, bad),                       # rows of a wider buffer
            (at, (row, 0), {}, bad),
            (at + 2 * row, (10 * row, 64), {}, runs),           # between its rows
            (at + 2 * row - 2, (10 * row, 64), {}, bad),
            (at + 2 * row, (4 * row - 2, 64), {}, bad),
            (at + 20 * row * 2, (10 * row, 64), {}, bad),
            (at + 2, (row, 64), dict(tokens=3), bad)):
        assert attend_at(at, out, *strides, **kw) == want, (out - at, strides, kw)


@pytest.mark.skipif(torch.cuda.is_available(), reason="its addresses are not a GPU's")
@pytest.mark.parametrize("seqs,tokens", [(0x7fffff00, 0x3000), (1 << 23, 5), (1 << 22, 1 << 21),
                                         (0x7fffff00, 0x7fffff00)])
def test_steps_of_more_sequences_than_a_launch_holds(seqs, tokens):
    """Most of them without a token: the slots are counted in 64 bits."""
    c = nat.KvCacheArrays(ctypes.sizeof(nat.KvCacheArrays), 8, 2, 64, 16, 0, *[HERE] * 6)
    b = nat.KvBatch(ctypes.sizeof(nat.KvBatch), seqs, 4, 4, tokens, 0, HERE, HERE, HERE)
    lib, refs = nat.load(), (ctypes.byref(c), ctypes.byref(b))
    strides = (ctypes.c_int64 * 4)(128, 64, 128, 64)
    assert lib.hbfsim_amd_kv_append(*refs, HERE, HERE, 0, strides, None) == nat.HBFSIM_UNSUPPORTED
    assert lib.hbfsim_amd_kv_select(*refs, HERE, 0, 4, 256, 64, 4, 1, 1, HERE, HERE, 1 << 62,
                                    None) == nat.HBFSIM_UNSUPPORTED
    for acc in (0, 1):
        assert lib.hbfsim_amd_kv_attend(*refs, HERE, 0, 4, 256, 64, 0.1, None, 0, acc, 2 * HERE,
                                        HERE, 1 << 62, None) == nat.HBFSIM_UNSUPPORTED


def test_arguments_past_32_bits(monkeypatch):
    """The library takes 32-bit counts: larger ones do not arrive as their low
    halves.  To keep more blocks than there can be is to keep all."""
    with FakeTensorMode(), monkeypatch.context() as patch:
        Machine(patch)
        got = []
        patch.setattr(nat, "load", lambda: Library(lambda name, args: got.append((name, args))))
        cache = kvcache.KvCache(4, 2, 64, device="cuda:0")
        table, lens = (torch.zeros(s, dtype=I32, device="cuda:0") for s in ((3, 2), (3,)))
        q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda:0")
        k = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda:0")
        for keep in (2 ** 32, 2 ** 32 + 5, 2 ** 63 - 1, 2 ** 80):
            cache.evict(table, lens, keep)
            kvcache.evict(cache.weight, table, lens, keep)
            assert [args[9] for _, args in got] == [2 ** 32 - 1] * 2
            got.clear()
        far = torch.empty_strided((3, 2), (2 ** 32 + 2, 1), dtype=I32, device="cuda:0")
        for bad in (lambda: cache.evict(table, lens, 2, 2 ** 32),
                    lambda: cache.evict(table, lens, 2, 0, 2 ** 32 + 1),
                    lambda: kvcache.evict(cache.weight, table, lens, 2, 2 ** 32 + 16),
                    lambda: cache.select(q, table, lens, 2, None, 2 ** 32, 1),
                    lambda: cache.select(q, table, lens, 2, None, 0, 2 ** 32 + 1),
                    lambda: cache.evict(far, lens, 2), lambda: cache.append(k, k, far, lens),
                    lambda: cache.select(q, far, lens, 2), lambda: cache.attend(q, far, lens)):
            with pytest.raises(ValueError):
                bad()
        assert got == []
