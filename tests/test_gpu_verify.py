"""Verification of drafted tokens on the GPU against its definition
(kvpages_ref): whole numbers, equal or wrong."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kvpages_ref as pr
from hbfsim_amd import drafts

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def dev(x, dtype=np.int32):
    return torch.from_numpy(np.array(x, dtype)).cuda()


def steps(rng, counts, vocab, dtype, sure=False, sharp=3.0):
    """(target, draft, tokens, uniform, first) of sequences with so many rows."""
    first = np.concatenate([[0], np.cumsum(counts)])
    rows = int(first[-1])
    x = rng.normal(0, sharp, (rows, vocab))
    y = x + rng.normal(0, 0.8, (rows, vocab))
    p, q = (np.exp(z - z.max(1, keepdims=True, initial=0)) for z in (x, y))
    p, q = (torch.from_numpy((z / z.sum(1, keepdims=True)).astype(np.float32)).to(DT[dtype])
            for z in (p, q))
    tokens = np.zeros(rows, np.int32)
    drawn = (q.double().numpy() / rng.exponential(size=(rows, vocab))).argmax(1)
    tokens[1:] = drawn[:-1]
    tokens[rng.random(rows) < 0.05] = rng.choice([-1, vocab, 2 ** 31 - 1, -2 ** 31])
    return p, None if sure else q, tokens, rng.random(rows).astype(np.float32), first


def check(p, q, tokens, u, first, lens=True, padded=0):
    seqs = (len(p) if first is None else len(first) - 1)
    stored = np.arange(seqs, dtype=np.int32) + 1000 if lens else None
    want = pr.verify(p.float().numpy(), tokens, u, first,
                     None if q is None else q.float().numpy(), stored)
    got = drafts.verify(p.cuda(), dev(tokens), dev(u, np.float32),
                        None if first is None else dev(first), draft=None if q is None else q.cuda(),
                        lens=None if stored is None else dev(stored))
    np.testing.assert_array_equal(got[0].cpu(), want[0])
    np.testing.assert_array_equal(got[1].cpu(), want[1])
    if lens:
        np.testing.assert_array_equal(got[2].cpu(), want[2])
    else:
        assert got[2] is None
    return want


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("vocab,seqs,rows", [(1, 3, 3), (2, 9, 2), (5, 40, 6), (257, 6, 9),
                                             (2048, 2, 3), (8192, 2, 2), (8193, 2, 3),
                                             (20011, 3, 4), (32000, 1, 5), (32768, 1, 2),
                                             (32769, 2, 2), (65536, 1, 2), (65541, 2, 2),
                                             (40_001, 80, 3)])
def test_verify(dtype, sure, vocab, seqs, rows):
    rng = np.random.default_rng(vocab + seqs)
    counts = rng.integers(0, rows + 1, seqs)
    counts[0] = rows
    check(*steps(rng, counts, vocab, dtype, sure))


@pytest.mark.parametrize("vocab", [3, 700, 9001])
def test_one_row_each_draws_from_the_target(vocab):
    rng = np.random.default_rng(vocab)
    p, q, tokens, u, _ = steps(rng, np.ones(11, int), vocab, "f32")
    u[:4] = [0.0, 1.0 - 2 ** -24, 1.0, 2 ** -31]
    check(p, None, tokens, u, None, lens=False)
    check(p, q, tokens, u, None)


def test_every_place_can_be_drawn():
    """A uniform target over sizes that end inside every tile: the drawn token
    is the one whose share of [0, 1) holds the number."""
    for vocab in (4, 1000, 1024, 4095, 12288, 33001, 100_003):
        at = np.unique(np.concatenate([np.arange(min(vocab, 40)), vocab - 1 - np.arange(min(vocab, 40)),
                                       np.linspace(0, vocab - 1, 60).astype(int)]))
        w = int(pr.whole(np.float32(1.0 / vocab)))
        u = ((at + 0.5) / vocab).astype(np.float32)
        want = [(int(float(x) * 2 ** 31) * w * vocab >> 31) // w for x in u]
        p = torch.full((len(at), vocab), 1.0 / vocab, device="cuda")
        got, gained, _ = drafts.verify(p, dev(at), dev(u, np.float32))
        np.testing.assert_array_equal(got.cpu(), want)
        assert (gained == 1).all()


def test_borders():
    """A draft stays only while u q < p, to the last bit; equal is refused."""
    vocab = 8
    p = np.full((6, vocab), 0.125, np.float32)
    q = np.full((6, vocab), 0.25, np.float32)
    u = np.array([0.5, 0.3, np.nextafter(np.float32(0.5), np.float32(0)), 0.3, 0.0, 0.3], np.float32)
    tokens = np.array([0, 3, 0, 3, 0, 3], np.int32)
    p[4, 3] = 0.0  # 0 < 0 is not
    first = [0, 2, 4, 6]
    want = check(torch.from_numpy(p), torch.from_numpy(q), tokens, u, first)
    assert want[1].tolist() == [1, 2, 1]


def test_nothing_left_and_no_probabilities_at_all():
    """Where target and draft agree nothing is left to draw from: the target
    itself is.  Rows of zeros and of what is not a number draw -1."""
    vocab = 600
    rng = np.random.default_rng(1)
    x = rng.random((12, vocab)).astype(np.float32)
    x /= x.sum(1, keepdims=True)
    p, q = x.copy(), x.copy()
    tokens = np.full(12, 7, np.int32)
    u = np.full(12, 0.9, np.float32)
    u[0::2] = 2.0                      # refuses
    p[2:4], p[4:6], q[6:8] = 0, np.nan, np.nan
    p[8, 3], p[9, 5], q[8, 9] = np.inf, -np.inf, -1.0
    p[10, :] = -0.0
    p[10, vocab - 1] = 1e-30           # below what is counted
    q[10, :] = 0
    u[11] = np.nan
    want = check(torch.from_numpy(p), torch.from_numpy(q), tokens, u, np.arange(0, 13, 2))
    assert want[0][2] == -1 and want[0][4] == -1 and want[0][0] >= 0


def test_many_drafts():
    """More than a wave tests at once; all stay, none does, the 64th or 65th is the first that does not."""
    vocab = 50
    rng = np.random.default_rng(2)
    counts = np.array([200, 130, 65, 66, 129, 1, 0, 64])
    p, q, tokens, u, first = steps(rng, counts, vocab, "f32")
    tokens = np.clip(tokens, 0, vocab - 1)
    u[:] = 0.0
    for s, at in ((1, 64), (2, 63), (3, 64), (4, 127)):
        u[first[s] + at] = 2.0 ** 20
    u[np.array(first[1:]) - 1] = rng.random(len(counts))
    want = check(p + 1e-4, q, tokens, u, first)
    assert want[1].tolist() == [200, 65, 64, 65, 128, 1, 0, 64]


def test_rows_of_no_sequence():
    """Padded batches, sequences that end past the rows, no sequence at all."""
    rng = np.random.default_rng(3)
    p, q, tokens, u, _ = steps(rng, [3, 4, 2, 5], 90, "f32")
    tokens = np.clip(tokens, 0, 89)
    for first in ([2, 5, 5, 9], [0, 3, 20], [0], [14, 14], [3, 3, 4]):
        check(p, q, tokens, u, np.array(first))
    got = drafts.verify(torch.zeros((0, 5), device="cuda"), dev([]), dev([], np.float32))
    assert got[0].shape == (0,) and got[1].shape == (0,)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("start,stride", [(0, 1003), (1, 1008), (3, 1001), (8, 1016)])
def test_strides_and_odd_addresses(dtype, start, stride):
    rng = np.random.default_rng(4)
    vocab = 1001
    p, q, tokens, u, first = steps(rng, [3, 2, 4], vocab, dtype)
    want = pr.verify(p.float().numpy(), tokens, u, first, q.float().numpy())
    views = []
    for x in (p, q):
        buffer = torch.full((start + 9 * stride,), 0.5, dtype=DT[dtype], device="cuda")
        view = buffer[start:].as_strided((9, vocab), (stride, 1), start)
        view.copy_(x)
        views.append(view)
    got = drafts.verify(views[0], dev(tokens), dev(u, np.float32), dev(first), draft=views[1])
    np.testing.assert_array_equal(got[0].cpu(), want[0])
    # one row for all: a stride of 0
    one = p[:1].cuda().expand(9, vocab)
    got = drafts.verify(one, dev(tokens), dev(u, np.float32), dev(first), draft=views[1])
    want = pr.verify(p[:1].float().numpy().repeat(9, 0), tokens, u, first, q.float().numpy())
    np.testing.assert_array_equal(got[0].cpu(), want[0])


def test_a_large_vocabulary():
    """The largest that is taken, and sums near their limit."""
    vocab = 1 << 22
    p = torch.ones((2, vocab), device="cuda")  # nothing says that they sum to one
    u = dev([0.25, 1.0], np.float32)
    got, _, _ = drafts.verify(p, dev([0, 0]), u)
    assert got.tolist() == [1 << 20, ((1 << 31) - 1) >> 9]
    with pytest.raises(ValueError):
        drafts.verify(torch.ones((2, vocab + 1), device="cuda"), dev([0, 0]), u)


def test_rows_past_2_31_elements():
    vocab, rows = 1 << 20, 2100
    target = torch.zeros((rows, vocab), dtype=torch.bfloat16, device="cuda")
    target[:, 5] = 1.0
    target[rows - 1, 5] = 0.0
    target[rows - 1, vocab - 1] = 1.0
    first = dev([0, 1, rows - 1, rows])
    tokens = dev(np.full(rows, 5))
    out, gained, _ = drafts.verify(target, tokens, torch.full((rows,), 0.5, device="cuda"), first)
    assert gained.tolist() == [1, rows - 2, 1]
    assert (out[:-1] == 5).all() and out[-1] == vocab - 1


def test_shares_of_many_draws():
    """What a step gains first is distributed as the target: 200,000 sequences
    of one draft each, every count within six standard deviations."""
    rng = np.random.default_rng(5)
    n, vocab = 200_000, 6
    p = np.array([0.30, 0.05, 0.25, 0.25, 0.05, 0.10])
    q = np.array([0.10, 0.40, 0.20, 0.05, 0.05, 0.20])
    tokens = np.zeros((n, 2), np.int32)
    tokens[:, 1] = rng.choice(vocab, n, p=q)
    u = rng.random((n, 2)).astype(np.float32)
    rows = [torch.tensor(x, dtype=torch.float32, device="cuda").expand(2 * n, vocab) for x in (p, q)]
    out, gained, _ = drafts.verify(rows[0], dev(tokens.reshape(-1)), dev(u.reshape(-1), np.float32),
                                   dev(2 * np.arange(n + 1)), draft=rows[1])
    got = np.bincount(out.view(n, 2)[:, 0].cpu().numpy(), minlength=vocab)
    assert (np.abs(got - n * p) < 6 * np.sqrt(n * p * (1 - p))).all(), got / n
    # and a draft stays with the chance sum(min(p, q))
    kept = float((gained == 2).sum()) / n
    a = np.minimum(p, q).sum()
    assert abs(kept - a) < 6 * np.sqrt(a * (1 - a) / n)


@pytest.mark.parametrize("vocab", [5000, 20_001])
def test_on_another_stream_and_in_a_graph(vocab):
    rng = np.random.default_rng(6)
    counts = [3, 1, 5, 2]
    runs = [steps(rng, counts, vocab, "f32") for _ in range(4)]
    first = dev(runs[0][4])
    p, q = (torch.zeros((11, vocab), device="cuda") for _ in range(2))
    tokens, u, lens = dev(np.zeros(11)), dev(np.zeros(11), np.float32), dev([9, 8, 7, 6])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        drafts.verify(p, tokens, u, first, draft=q, lens=lens)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = drafts.verify(p, tokens, u, first, draft=q, lens=lens)
    for x, y, z, v, f in runs + runs[::-1]:
        p.copy_(x), q.copy_(y), tokens.copy_(dev(z)), u.copy_(dev(v, np.float32))
        torch.cuda.synchronize()
        want = pr.verify(x.numpy(), z, v, f, y.numpy(), np.array([9, 8, 7, 6]))
        graph.replay()
        eager = drafts.verify(p, tokens, u, first, draft=q, lens=lens, stream=stream)
        torch.cuda.synchronize()
        for got in (captured, eager):
            for a, b in zip(got, want):
                np.testing.assert_array_equal(a.cpu(), b)


def test_two_streams_at_once_and_lengths_in_place():
    """Two calls side by side share nothing; the C call may write the lengths
    that remain over the lengths."""
    import ctypes

    from hbfsim_amd import _native as nat

    rng = np.random.default_rng(7)
    runs = [steps(rng, rng.integers(0, 6, 40), 9000 + i, "bf16") for i in range(2)]
    args = [(p.cuda(), q.cuda(), dev(t), dev(u, np.float32), dev(f)) for p, q, t, u, f in runs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[drafts.verify(p, t, u, f, draft=q, stream=s) for _ in range(5)]
           for s, (p, q, t, u, f) in zip(streams, args)]
    torch.cuda.synchronize()
    lens = np.arange(40, dtype=np.int32) + 50
    for (p, q, t, u, f), results, (gp, gq, gt, gu, gf) in zip(runs, got, args):
        want = pr.verify(p.float().numpy(), t, u, f, q.float().numpy(), lens)
        for out, gained, _ in results:
            np.testing.assert_array_equal(out.cpu(), want[0])
            np.testing.assert_array_equal(gained.cpu(), want[1])
        need, at = ctypes.c_size_t(), dev(lens)
        assert nat.load().hbfsim_amd_verify_workspace(40, p.shape[1], nat.KV_BF16,
                                                      ctypes.byref(need)) == 0
        ws = torch.empty(max(16, need.value), dtype=torch.uint8, device="cuda")
        out, gained = dev(np.zeros(len(t))), dev(np.zeros(40))
        assert nat.load().hbfsim_amd_verify(
            gp.data_ptr(), gq.data_ptr(), nat.KV_BF16, p.shape[1], p.shape[1], p.shape[1],
            gt.data_ptr(), gu.data_ptr(), gf.data_ptr(), 40, len(t), at.data_ptr(), out.data_ptr(),
            gained.data_ptr(), at.data_ptr(), ws.data_ptr(), need.value,
            torch.cuda.current_stream().cuda_stream) == 0
        np.testing.assert_array_equal(out.cpu(), want[0])
        np.testing.assert_array_equal(at.cpu(), want[2])
