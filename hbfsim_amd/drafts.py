"""Drafted tokens: which of a step's stay (hbfsim_amd_verify_step,
include/hbfsim_amd.h section 9).

A step of drafts over a paged cache appends and attends to several tokens of
each sequence at once, the last known one and those that a draft proposes;
`verify` says from the target's probabilities which of them stay and which
token follows, and the cache's `release` gives back the blocks of the others.

    step, missing = cache.grow(table, lens + rows, first, tokens)  # rows of each sequence
    cache.append(k, v, table, step, first)
    out = cache.attend(q, table, step, first)
    new, gained, lens = verify(target, tokens, uniform, first, draft=draft, lens=step, stored=lens)
    cache.release(table, lens)

A sequence that lacks blocks has length 0 in `step`; by `stored` it keeps the
length that it had, and so its row, and can go on in a later step.

No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
from typing import Any

import torch

from . import _native as nat
from .kvcache import (_TYPES, _counts, _elsewhere, _flat, _gpu, _handle, _on_gpu, _refuse, _there,
                      _workspace)

_need: dict = {}  # workspace bytes by a call's sizes


def _probabilities(x: Any, name: str) -> Any:
    if x.dim() != 2 or x.dtype not in _TYPES or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"{name} must be [rows, vocab] of bfloat16, float16 or float32, "
                         "contiguous in its last dimension")
    return x


def verify(target: Any, tokens: Any, uniform: Any, first: Any = None, draft: Any = None,
           lens: Any = None, stream: Any = None, stored: Any = None) -> tuple:
    """Which of a step's drafted tokens stay, and the token behind them.

    Sequence s has rows first[s] .. first[s + 1] - 1 of the batch (`first`
    int32 [seqs + 1]; one row each without it): `tokens` (int32 [rows]) holds
    its last token, then the drafted ones; target[r] and draft[r] [rows, vocab]
    are the probabilities of the token after row r (no `draft`: the drafted
    tokens were sure).  Draft x after row r stays while
    uniform[r] * draft[r, x] < target[r, x]; at the first that does not, the
    next token is drawn from max(target - draft, 0), behind the last one from
    target, both by the `uniform` (float32 [rows], in [0, 1)) of the sequence's
    last row.  The drawing is in whole numbers, 2^40 to a probability of one.

    Returns (out, gained, lens): int32 [rows] with each sequence's tokens from
    its first row on, -1 beyond; how many they are; and, from `lens` (tokens
    stored with all of the step's), those that remain, None without it.  A
    sequence whose `lens` is below its rows was left out of the step: it gains
    nothing and remains as `lens` says, or as `stored` does (int32 [seqs], the
    lengths before the step), which a step that `grow` has given lengths needs
    before blocks are released by them."""
    gpu = _gpu(target)
    if _elsewhere(gpu, stream):
        return _there(target.device, stream, lambda: verify(target, tokens, uniform, first, draft,
                                                            lens, stored=stored))
    device = target.device
    rows, vocab = _probabilities(target, "target").shape
    if draft is not None and (_probabilities(draft, "draft").shape != target.shape
                              or draft.dtype is not target.dtype
                              or draft.get_device() != target.get_device()):
        raise ValueError("draft must be of target's shape, type and device")
    if _flat(tokens, "tokens", target) != rows:
        raise ValueError(f"{tokens.shape[0]} tokens for {rows} rows")
    if uniform.dtype is not torch.float32 or uniform.dim() != 1 or uniform.shape[0] != rows \
            or uniform.get_device() != target.get_device() or not uniform.is_contiguous():
        raise ValueError(f"uniform must be a contiguous float32 tensor [{rows}] on {device}")
    seqs = rows
    if first is not None:
        seqs = _flat(first, "first", target) - 1
        if seqs < 0:
            raise ValueError("first must hold one offset more than there are sequences")
    if lens is not None and _flat(lens, "lens", target) != seqs:
        raise ValueError(f"{lens.shape[0]} lengths for {seqs} sequences")
    if stored is not None:
        if lens is None:
            raise ValueError("stored lengths without the step's")
        if _flat(stored, "stored", target) != seqs:
            raise ValueError(f"{stored.shape[0]} stored lengths for {seqs} sequences")
    _counts(rows | seqs | vocab)
    _on_gpu(gpu)
    kind = _TYPES[target.dtype]
    need = _need.get((seqs, vocab, kind))
    if need is None:
        got = ctypes.c_size_t()
        _refuse(nat.load().hbfsim_amd_verify_workspace(seqs, vocab, kind, ctypes.byref(got)),
                "verify")
        if len(_need) >= 4096:
            _need.clear()
        need = _need[seqs, vocab, kind] = got.value
    # Outputs and scratch are parts of one allocation, scratch first (it is
    # aligned), if the scratch is small: whoever keeps an output keeps all of it.
    held = need // 4 if need <= 65536 else 0
    ws, out, gained, left = torch.empty((held + rows + 2 * seqs,), dtype=torch.int32,
                                        device=device).split_with_sizes((held, rows, seqs, seqs))
    if need > 4 * held:
        ws = _workspace(need, device)
    _refuse(nat.load().hbfsim_amd_verify_step(
        target.data_ptr(), draft.data_ptr() if draft is not None else None, kind, vocab,
        target.stride(0), draft.stride(0) if draft is not None else 0, tokens.data_ptr(),
        uniform.data_ptr(), first.data_ptr() if first is not None else None, seqs, rows,
        lens.data_ptr() if lens is not None else None,
        stored.data_ptr() if stored is not None else None, out.data_ptr(), gained.data_ptr(),
        left.data_ptr() if lens is not None else None, ws.data_ptr() if need else None, need,
        _handle(gpu)), "verify")
    return out, gained, left if lens is not None else None
