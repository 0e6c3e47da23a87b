"""A paged key/value cache in 8 bits and the operators of a step on it
(hbfsim_amd_kv_*, include/hbfsim_amd.h section 7).

`KvCache` owns the device arrays.  A step names its sequences by a block table
(int32 [seqs, width], -1 for a block that is not there), their lengths after
the step (int32 [seqs]) and, when a sequence has other than one token in the
step, the offsets of their rows in the batch (`first`, int32 [seqs + 1]).  Rows
that belong to no sequence store and select nothing and attend to nothing.  All
tensors are on the cache's GPU; calls queue their work on `stream` (the
current one by default) and return without waiting for it.

    cache = KvCache(blocks=4096, kv_heads=8, head_dim=128)
    cache.append(k, v, table, lens)               # one new token per sequence
    chosen = cache.select(q, table, lens, 128)    # blocks to read
    out = cache.attend(q, table, lens, selected=chosen)
    out = cache.attend(q, table, lens, accumulate=True)
    table, lens, freed, count = cache.evict(table, lens, keep=512)

No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math
from typing import Any

import torch

from . import _native as nat

BLOCK_TOKENS = (16, 32, 64, 128)
WEIGHT_UNIT = 2.0 ** -32
_TYPES = {torch.bfloat16: nat.KV_BF16, torch.float16: nat.KV_F16, torch.float32: nat.KV_F32}


def padded_dim(head_dim: int) -> int:
    """Dims stored per token: head_dim rounded up to a multiple of 64."""
    return -(-head_dim // 64) * 64


def _refuse(rc: int, what: str) -> None:
    if rc in (nat.HBFSIM_INVALID_ARGUMENT, nat.HBFSIM_UNSUPPORTED):
        raise ValueError(f"{what} refused: {nat.status_name(rc)} ({rc})")
    nat.check(rc, what)


def _gpu(x: Any) -> int | None:
    """The index of the tensor's GPU, None on another kind of device."""
    return x.device.index if x.is_cuda else None


def _elsewhere(gpu: int | None, stream: Any) -> bool:
    """Whether a call has to make another GPU or stream current first."""
    return gpu is not None and (stream is not None or torch._C._cuda_getDevice() != gpu)


def _there(device: Any, stream: Any, call: Any, own: bool = True) -> Any:
    """`call` with the cache's GPU current (handle 0 is the current one's
    default stream, and a kernel runs where it is launched, not where its
    tensors are) and `stream`, a torch stream or a handle, current on it, so
    that scratch and outputs come from its pool: a block of the current
    stream's may have work queued there that `stream` is not ordered behind.
    Its outputs, if it makes them itself, are recorded on the caller's stream,
    which reads them: none is handed out again before that is done."""
    if stream is None:
        with torch.cuda.device(device):
            return call()
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(stream, device=device)
    elif stream.device != device:
        raise ValueError(f"stream is of {stream.device}, the cache on {device}")
    caller = torch.cuda.current_stream(device)
    with torch.cuda.stream(stream):
        got = call()
    if own and got is not None:
        for t in got if isinstance(got, tuple) else (got,):
            t.record_stream(caller)
    return got


def _handle(gpu: int) -> int:
    """The current stream's handle.  (The raw accessor costs a tenth of
    building a Stream.)"""
    return torch._C._cuda_getCurrentRawStream(gpu)


def _on_gpu(gpu: int | None) -> None:
    """Kernels follow the tensors' addresses: only a GPU's may reach them."""
    if gpu is None:
        raise ValueError("the cache is not on a GPU")


def _workspace(nbytes: int, device: Any) -> Any:
    """Scratch of one call, handed back to torch's allocator after it: work
    queued later on the same stream is ordered behind the call."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _ints(x: Any, name: str, device: Any, dims: int) -> Any:
    if x.dtype != torch.int32 or x.dim() != dims or x.device != device:
        raise ValueError(f"{name} must be an int32 tensor of {dims} dimension(s) on {device}")
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return x


def _counts(bits: int) -> None:
    """The library's counts are of 32 bits; ctypes would pass their low half.
    `bits` are those of all counts of a call together."""
    if bits >> 32:
        raise ValueError("counts and strides must be in 0..2^32 - 1")


def _batch(table: Any, lens: Any, first: Any, tokens: int, device: Any) -> nat.KvBatch:
    _ints(table, "table", device, 2)
    _ints(lens, "lens", device, 1)
    seqs, width = table.shape
    if lens.shape[0] != seqs:
        raise ValueError(f"{lens.shape[0]} lengths for {seqs} sequences")
    if first is not None:
        _ints(first, "first", device, 1)
        if first.shape[0] != seqs + 1:
            raise ValueError("first must hold one offset more than there are sequences")
    elif tokens != seqs:
        raise ValueError(f"{tokens} tokens for {seqs} sequences of one token each")
    stride = table.stride(0) if seqs > 1 else width
    if stride < width:
        raise ValueError("table rows overlap")
    _counts(seqs | width | stride | tokens)
    return nat.KvBatch(ctypes.sizeof(nat.KvBatch), seqs, width, stride, tokens, 0,
                       table.data_ptr(), lens.data_ptr(),
                       first.data_ptr() if first is not None else None)


def evict(weight: Any, table: Any, lens: Any, keep: int, block_tokens: int = 16,
          keep_first: int = 1, keep_last: int = 1, stream: Any = None) -> tuple:
    """The blocks that leave a cache of per-block weights (int64 [blocks,
    kv_heads]): every sequence of more than `keep` blocks keeps its first
    `keep_first`, its last `keep_last` and the others of the largest weight
    summed over kv heads.  Returns (table, lens, freed, freed_count), new
    tensors: kept blocks in order, the tokens left, and the blocks that left,
    -1 beyond.  ValueError for what the library refuses."""
    device = weight.device
    gpu = _gpu(weight)
    if _elsewhere(gpu, stream):
        return _there(device, stream, lambda: evict(weight, table, lens, keep, block_tokens,
                                                    keep_first, keep_last))
    _ints(table, "table", device, 2)
    _ints(lens, "lens", device, 1)
    seqs, width = table.shape
    if weight.dtype != torch.int64 or weight.dim() != 2 or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous int64 tensor [blocks, kv_heads]")
    if lens.shape[0] != seqs:
        raise ValueError(f"{lens.shape[0]} lengths for {seqs} sequences")
    if min(keep, keep_first, keep_last) < 0:
        raise ValueError("keep, keep_first and keep_last must not be negative")
    stride = table.stride(0) if seqs > 1 else width
    keep = min(keep, 2 ** 32 - 1)  # no table has more blocks
    _counts(weight.shape[0] | weight.shape[1] | block_tokens | seqs | width | stride | keep_first
            | keep_last)
    _on_gpu(gpu)
    out_table, freed = torch.empty((2, seqs, width), dtype=torch.int32, device=device).unbind()
    out_lens, count = torch.empty((2, seqs), dtype=torch.int32, device=device).unbind()
    ws = _workspace(seqs * width * 8, device)
    _refuse(nat.load().hbfsim_amd_kv_evict(
        weight.data_ptr(), weight.shape[0], weight.shape[1], block_tokens, table.data_ptr(),
        lens.data_ptr(), seqs, width, stride, keep, keep_first, keep_last, out_table.data_ptr(),
        out_lens.data_ptr(), freed.data_ptr(), count.data_ptr(),
        ws.data_ptr() if ws is not None else None, seqs * width * 8, _handle(gpu)), "evict")
    return out_table, out_lens, freed, count


class KvCache:
    """A pool of blocks of `block_tokens` tokens of every kv head."""

    def __init__(self, blocks: int, kv_heads: int, head_dim: int, block_tokens: int = 16,
                 device: Any = "cuda"):
        if block_tokens not in BLOCK_TOKENS:
            raise ValueError(f"block_tokens must be one of {BLOCK_TOKENS}")
        if not (0 < blocks < 2 ** 31 and 0 < kv_heads <= 1024 and 0 < head_dim <= 256):
            raise ValueError("blocks, kv_heads (at most 1024) and head_dim (at most 256) must be "
                             "positive")
        dims, tiles = padded_dim(head_dim), block_tokens // 16
        shape = (blocks, kv_heads, tiles, dims // 64, 4, 16)
        new = dict(device=device)
        self._take(torch.zeros((*shape, 16), dtype=torch.int8, **new),
                   torch.zeros((*shape, 4, 4), dtype=torch.int8, **new),
                   torch.ones((blocks, kv_heads), dtype=torch.float32, **new),
                   torch.ones((blocks, kv_heads), dtype=torch.float32, **new),
                   torch.zeros((blocks, kv_heads, 2, dims), dtype=torch.int8, **new),
                   torch.zeros((blocks, kv_heads), dtype=torch.int64, **new), head_dim)

    @classmethod
    def from_tensors(cls, keys: Any, values: Any, key_scale: Any, value_scale: Any, bounds: Any,
                     weight: Any, head_dim: int) -> "KvCache":
        """A cache over arrays the caller keeps, in the library's layout (the
        tensors' shapes as the constructor makes them)."""
        self = cls.__new__(cls)
        self._take(keys, values, key_scale, value_scale, bounds, weight, head_dim)
        return self

    def _take(self, keys, values, key_scale, value_scale, bounds, weight, head_dim):
        if keys.dim() != 7 or not 0 < head_dim <= 256:
            raise ValueError("keys must have 7 dimensions and head_dim be in 1..256")
        blocks, kv_heads, tiles, chunks = keys.shape[:4]
        dims, shape = padded_dim(head_dim), (blocks, kv_heads, tiles, chunks, 4, 16)
        if chunks * 64 != dims or tiles * 16 not in BLOCK_TOKENS:
            raise ValueError("keys do not have the layout of blocks of this head_dim")
        for x, want, dtype, name in (
                (keys, (*shape, 16), torch.int8, "keys"),
                (values, (*shape, 4, 4), torch.int8, "values"),
                (key_scale, (blocks, kv_heads), torch.float32, "key_scale"),
                (value_scale, (blocks, kv_heads), torch.float32, "value_scale"),
                (bounds, (blocks, kv_heads, 2, dims), torch.int8, "bounds"),
                (weight, (blocks, kv_heads), torch.int64, "weight")):
            if tuple(x.shape) != want or x.dtype != dtype or not x.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {want}")
            if x.device != keys.device:
                raise ValueError(f"{name} is on {x.device}, keys on {keys.device}")
        self.keys, self.values = keys, values
        self.key_scale, self.value_scale = key_scale, value_scale
        self.bounds, self.weight = bounds, weight
        self.blocks, self.kv_heads = blocks, kv_heads
        self.head_dim, self.block_tokens = head_dim, tiles * 16
        self.device, self._gpu = keys.device, _gpu(keys)
        self._lib = nat.load()
        self._c = nat.KvCacheArrays(ctypes.sizeof(nat.KvCacheArrays), blocks, kv_heads, head_dim,
                                    tiles * 16, 0, keys.data_ptr(), values.data_ptr(),
                                    key_scale.data_ptr(), value_scale.data_ptr(),
                                    bounds.data_ptr(), weight.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._need: dict = {}  # workspace bytes by a call's sizes

    # -- checks -----------------------------------------------------------
    def _rows(self, x: Any, heads: int | None, name: str) -> tuple[int, int, int]:
        """(tokens, heads, type) of [tokens, heads, head_dim] rows."""
        if x.dim() != 3 or x.shape[2] != self.head_dim or x.device != self.device:
            raise ValueError(f"{name} must be [tokens, heads, {self.head_dim}] on {self.device}")
        if heads is not None and x.shape[1] != heads:
            raise ValueError(f"{name} has {x.shape[1]} heads, not {heads}")
        if x.dtype not in _TYPES:
            raise ValueError(f"{name} must be bfloat16, float16 or float32")
        if x.stride(2) != 1 and self.head_dim > 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
        return x.shape[0], x.shape[1], _TYPES[x.dtype]

    def _queries(self, q: Any) -> tuple[int, int, int]:
        tokens, heads, kind = self._rows(q, None, "q")
        if kind == nat.KV_F32:
            raise ValueError("q must be bfloat16 or float16")
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads do not divide among {self.kv_heads} kv heads")
        return tokens, heads, kind

    def _remember(self, sizes: tuple, nbytes: int) -> int:
        if len(self._need) >= 4096:
            self._need.clear()
        self._need[sizes] = nbytes
        return nbytes

    # -- operators --------------------------------------------------------
    def append(self, k: Any, v: Any, table: Any, lens: Any, first: Any = None,
               stream: Any = None) -> None:
        """Stores the step's keys and values [tokens, kv_heads, head_dim]
        (bfloat16, float16 or float32, any token and head strides) as the
        sequences' last tokens."""
        if _elsewhere(self._gpu, stream):
            return _there(self.device, stream, lambda: self.append(k, v, table, lens, first))
        tokens, _, kind = self._rows(k, self.kv_heads, "k")
        if self._rows(v, self.kv_heads, "v") != (tokens, self.kv_heads, kind):
            raise ValueError("k and v differ in tokens or type")
        b = _batch(table, lens, first, tokens, self.device)
        strides = (ctypes.c_int64 * 4)(k.stride(0), k.stride(1), v.stride(0), v.stride(1))
        _on_gpu(self._gpu)
        _refuse(self._lib.hbfsim_amd_kv_append(self._ref, ctypes.byref(b), k.data_ptr(),
                                               v.data_ptr(), kind, strides,
                                               _handle(self._gpu)), "append")

    def read(self, blocks: Any, dtype: Any = torch.bfloat16, stream: Any = None) -> tuple:
        """The values that the blocks (int32 ids) stand for: keys and values
        [n, kv_heads, block_tokens, head_dim] and the keys' lower and upper
        bounds [n, kv_heads, head_dim]."""
        if _elsewhere(self._gpu, stream):
            return _there(self.device, stream, lambda: self.read(blocks, dtype))
        _ints(blocks, "blocks", self.device, 1)
        if dtype not in _TYPES:
            raise ValueError("dtype must be bfloat16, float16 or float32")
        _on_gpu(self._gpu)
        n = blocks.shape[0]
        k, v = torch.empty((2, n, self.kv_heads, self.block_tokens, self.head_dim), dtype=dtype,
                           device=self.device).unbind()
        low, high = torch.empty((2, n, self.kv_heads, self.head_dim), dtype=dtype,
                                device=self.device).unbind()
        _refuse(self._lib.hbfsim_amd_kv_read(self._ref, blocks.data_ptr(), n, _TYPES[dtype],
                                             k.data_ptr(), v.data_ptr(), low.data_ptr(),
                                             high.data_ptr(), _handle(self._gpu)), "read")
        return k, v, low, high

    def attend(self, q: Any, table: Any, lens: Any, first: Any = None, selected: Any = None,
               scale: float | None = None, accumulate: bool = False, out: Any = None,
               stream: Any = None) -> Any:
        """Attention of the step's queries [tokens, heads, head_dim] (bfloat16
        or float16) over the cache, each over its sequence up to itself;
        `selected` (int32 [tokens, kv_heads, count], logical blocks, negative
        for none) limits it to those blocks; `scale` defaults to
        head_dim ** -0.5.  With `accumulate` the blocks' weights grow by the
        probabilities.  `out` may be q itself, but not where weights accumulate
        with `first`.  Returns [tokens, heads, head_dim] in q's type."""
        if _elsewhere(self._gpu, stream):
            return _there(self.device, stream, lambda: self.attend(
                q, table, lens, first, selected, scale, accumulate, out), out is None)
        tokens, heads, kind = self._queries(q)
        b = _batch(table, lens, first, tokens, self.device)
        count, chosen = 0, None
        if selected is not None:
            _ints(selected, "selected", self.device, 3)
            count = selected.shape[2]
            if tuple(selected.shape[:2]) != (tokens, self.kv_heads) or not count \
                    or not selected.is_contiguous():
                raise ValueError("selected must be a contiguous [tokens, kv_heads, count], count "
                                 "at least 1")
            if accumulate:
                raise ValueError("weights accumulate over every visible block, not a selection")
            chosen = selected.data_ptr()
        if out is not None and (tuple(out.shape) != tuple(q.shape) or out.dtype != q.dtype
                                or out.device != self.device or not out.is_contiguous()):
            raise ValueError("out must be a contiguous tensor of q's shape and type")
        _on_gpu(self._gpu)
        ref = ctypes.byref(b)
        sizes = (b.seqs, b.table_width, tokens, first is None, heads, count, accumulate)
        need = self._need.get(sizes)
        if need is None:
            got = ctypes.c_size_t()
            _refuse(self._lib.hbfsim_amd_kv_attend_workspace(self._ref, ref, heads, count,
                                                             int(accumulate), ctypes.byref(got)),
                    "attend")
            need = self._remember(sizes, got.value)
        if out is None:
            out = torch.empty((tokens, heads, self.head_dim), dtype=q.dtype, device=self.device)
        ws = _workspace(need, self.device)
        _refuse(self._lib.hbfsim_amd_kv_attend(
            self._ref, ref, q.data_ptr(), kind, heads, q.stride(0), q.stride(1),
            1.0 / math.sqrt(self.head_dim) if scale is None else scale, chosen, count,
            int(accumulate), out.data_ptr(), ws.data_ptr() if ws is not None else None,
            need, _handle(self._gpu)), "attend")
        return out

    def select(self, q: Any, table: Any, lens: Any, count: int, first: Any = None,
               keep_first: int = 1, keep_last: int = 1, stream: Any = None) -> Any:
        """The `count` blocks for each query token and kv head to attend to,
        int32 [tokens, kv_heads, count], ascending, -1 beyond: the first
        `keep_first` and the last `keep_last` that the token sees, and the
        best by the blocks' key bounds."""
        if _elsewhere(self._gpu, stream):
            return _there(self.device, stream, lambda: self.select(
                q, table, lens, count, first, keep_first, keep_last))
        tokens, heads, kind = self._queries(q)
        if min(count, keep_first, keep_last) < 0:
            raise ValueError("count, keep_first and keep_last must not be negative")
        _counts(count | keep_first | keep_last)
        b = _batch(table, lens, first, tokens, self.device)
        _on_gpu(self._gpu)
        ref = ctypes.byref(b)
        sizes = (b.seqs, b.table_width, tokens, first is None)
        need = self._need.get(sizes)
        if need is None:
            got = ctypes.c_size_t()
            _refuse(self._lib.hbfsim_amd_kv_select_workspace(self._ref, ref, ctypes.byref(got)),
                    "select")
            need = self._remember(sizes, got.value)
        out = torch.empty((tokens, self.kv_heads, count), dtype=torch.int32, device=self.device)
        ws = _workspace(need, self.device)
        _refuse(self._lib.hbfsim_amd_kv_select(
            self._ref, ref, q.data_ptr(), kind, heads, q.stride(0), q.stride(1), count, keep_first,
            keep_last, out.data_ptr(), ws.data_ptr() if ws is not None else None, need,
            _handle(self._gpu)), "select")
        return out

    def evict(self, table: Any, lens: Any, keep: int, keep_first: int = 1, keep_last: int = 1,
              stream: Any = None) -> tuple:
        """`evict` by this cache's weights."""
        return evict(self.weight, table, lens, keep, self.block_tokens, keep_first, keep_last,
                     stream)

    def weights(self) -> Any:
        """The accumulated weights as float32 probabilities."""
        return self.weight * WEIGHT_UNIT
