"""Log probabilities of given tokens against the formulas in 64 bits.

Tolerances, u = 2^-24: with d = (x - m) / T and w = exp(d), a term's relative error is at most (3 |d| + 8) u (the
difference, the scaling and the exponential), and a sum over the row adds at most 128 u (the longest chain of
additions: 9 in a tile of a thread, up to 64 tiles, 5 and 3 levels in a block, up to 8 pieces in a thread of the join
and its 7 levels: 96). The largest's own 1 is exact. So
log(1 + R) is off by at most u sum_others p (3 |d| + 136) and a log probability by that and 3 u |x - m| / T of the
subtraction and the division; entropy's second sum weighs each term by |d| again. Ids, ranks and their order are exact.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from muyo_llm_b200 import nodes

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def score(logits, tokens, top_k, temperature=1.0, vocab=None, entropy=True, rank=True, stream=None):
    rows, stride = logits.shape[0], logits.stride(0)
    vocab = vocab or logits.shape[1]
    p = nodes.token_logprobs_params(rows, vocab, stride=stride, top_k=top_k, temperature=temperature)
    size = nodes.token_logprobs_workspace_size(p)
    ws = torch.full((size,), 0xCD, dtype=torch.uint8, device="cuda")
    f = lambda *s: torch.full(s, 7.0, device="cuda")  # noqa: E731
    lp, h, rk = f(rows + 1), f(rows + 1), torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    ids, tops = torch.full((rows + 1, max(top_k, 1)), -7, dtype=torch.int32, device="cuda"), f(rows + 1, max(top_k, 1))
    nodes.token_logprobs(p, logits, tokens, lp, ws, size, entropy=h if entropy else None, rank=rk if rank else None,
                         top_ids=ids if top_k else None, top_logprobs=tops if top_k else None, stream=stream)
    torch.cuda.synchronize()
    assert float(lp[rows]) == 7.0 and float(h[rows]) == 7.0 and int(rk[rows]) == -7 and int(ids[rows, 0]) == -7
    return lp[:rows], h[:rows], rk[:rows], ids[:rows], tops[:rows]


def check(logits, tokens, top_k, temperature=1.0, vocab=None, stream=None):
    lp, h, rk, ids, tops = score(logits, tokens, top_k, temperature, vocab, stream=stream)
    x = logits[:, :vocab] if vocab else logits
    T = float(np.float32(temperature))
    index = torch.arange(x.shape[1], device="cuda")
    for i in range(x.shape[0]):
        row, t = x[i].double(), int(tokens[i])
        best = int(x[i].argmax())
        d = (row - row.max()) / T
        w = torch.exp(d)
        w[best] = 0.0
        finite = d.clamp(min=-1e4).abs()
        R = w.sum()
        norm = torch.log1p(R)
        p = w / (1 + R)
        tol = U * float((p * (3 * finite + 136)).sum()) + 2 * U * float(norm)
        if 0 <= t < x.shape[1]:
            want = float(d[t] - norm)
            assert (float(lp[i]) == want) or abs(float(lp[i]) - want) <= tol + 3 * U * abs(float(d[t])) + U * abs(want), (i, float(lp[i]), want)
            before = int(((x[i] > x[i, t]) | ((x[i] == x[i, t]) & (index < t))).sum())
            assert int(rk[i]) == before, i
        else:
            assert float(lp[i]) == -math.inf and int(rk[i]) == x.shape[1]
        entropy = float(norm + (p * finite).sum())
        tol_h = U * float((p * (finite + 1) * (3 * finite + 300)).sum()) + 2 * U * entropy
        assert abs(float(h[i]) - entropy) <= tol_h, (i, float(h[i]), entropy, tol_h)
        if top_k:
            order = torch.sort(x[i], descending=True, stable=True).indices[:top_k]
            assert ids[i].tolist() == order.tolist(), i
            want = d[order] - norm
            ok = (tops[i].double() == want) | ((tops[i].double() - want).abs() <= tol + 3 * U * d[order].abs() + U * want.abs())
            assert bool(ok.all()), (i, tops[i], want)


@pytest.mark.parametrize("rows,vocab,top_k,temperature", [
    (1, 151936, 5, 1.0), (3, 151936, 20, 0.7), (1, 1, 1, 1.0), (2, 2, 2, 3.0), (5, 31, 31, 1.0), (4, 32, 32, 0.1), (9, 33, 32, 1.0),
    (40, 1000, 0, 1.0), (7, 32001, 7, 1.3), (3, 2047, 32, 1.0), (3, 2049, 32, 1.0), (2, 8191, 32, 1.0), (2, 8193, 32, 1.0),
    (300, 4099, 20, 1.0), (1, 300007, 32, 0.5), (160, 151936, 3, 1.0), (1, 3000001, 20, 1.0),
])
def test_token_logprobs(cuda, rows, vocab, top_k, temperature):
    g = gen(rows + vocab)
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * 3.0
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    tokens[::2] = logits[::2].argmax(1).to(torch.int32)
    check(logits, tokens, top_k, temperature)


@pytest.mark.parametrize("stride,vocab", [(1001, 1000), (1003, 997), (9000, 8999), (20010, 20001)])
def test_strides_and_alignments(cuda, stride, vocab):
    """Rows that start off 16 bytes, what lies between them NaN."""
    g = gen(stride)
    rows = 6
    store = torch.full((rows * stride + 3,), math.nan, device="cuda")
    for shift in (0, 1, 3):
        logits = torch.as_strided(store, (rows, vocab), (stride, 1), shift)
        store.fill_(math.nan)
        logits.copy_(torch.randn((rows, vocab), generator=g, device="cuda"))
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
        check(logits, tokens, 11)


@pytest.mark.parametrize("vocab", [40, 3001, 2046, 4094, 4095, 4096, 8190, 8192, 65534, 151936])
def test_masks_and_ties(cuda, vocab):
    """Rows with -inf or the type's lowest value for all but a few, rows of one value, zeros of both signs, ties around
    the last alternative."""
    g = gen(vocab)
    logits = torch.randn((9, vocab), generator=g, device="cuda") * 2.0
    keep = torch.randperm(vocab, generator=g, device="cuda")[:6]
    masked = torch.ones(vocab, dtype=torch.bool, device="cuda")
    masked[keep] = False
    logits[0, masked] = -math.inf
    logits[1, masked] = torch.finfo(torch.float32).min
    logits[2] = 3.25
    logits[3] = torch.finfo(torch.float32).min
    logits[4] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    logits[5] = torch.round(logits[5])  # a handful of values
    logits[6, masked] = -math.inf
    logits[6, keep] = 1.0
    logits[7] = -torch.arange(vocab, device="cuda").float()  # the best first
    logits[8] = torch.arange(vocab, device="cuda").float() * 0.001  # the best last
    tokens = torch.tensor([int(keep[0]), int(keep[1]), vocab // 2, 7, vocab - 1, 3, int(keep[2]), 0, vocab - 1], dtype=torch.int32,
                          device="cuda")
    check(logits, tokens, 20)
    masked_token = torch.tensor([int(masked.nonzero()[0])] * 9, dtype=torch.int32, device="cuda")
    check(logits, masked_token, 32)


@pytest.mark.parametrize("gap", [5.0, 12.0, 40.0, 90.0])
def test_almost_certain_tokens(cuda, gap):
    """log p near 0 keeps its relative accuracy."""
    logits = torch.zeros((3, 5000), device="cuda")
    logits[0, 17] = logits[1, 4999] = logits[2, 0] = gap
    check(logits, torch.tensor([17, 4999, 0], dtype=torch.int32, device="cuda"), 3)
    if gap == 40.0:
        lp = score(logits, torch.tensor([17, 4999, 0], dtype=torch.int32, device="cuda"), 0)[0]
        assert bool((lp < 0).all())  # -4999 exp(-40) = -2e-14: not rounded to 0


@pytest.mark.parametrize("rows", [1, 3, 30, 64, 200])
def test_masked_tokens_of_many_rows(cuda, rows):
    """Ranks of masked tokens and alternatives of masked rows, where rows are cut into pieces of every kind."""
    vocab = 32766
    g = gen(rows)
    logits = torch.randn((rows, vocab), generator=g, device="cuda")
    masked = torch.rand((rows, vocab), generator=g, device="cuda") < 0.999
    logits[masked] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    check(logits[:12], tokens[:12], 32) if rows < 12 else None
    lp, _, rk, ids, _ = score(logits, tokens, 32)
    row, index = torch.arange(rows, device="cuda"), torch.arange(vocab, device="cuda")
    given = logits[row, tokens.long()][:, None]
    before = ((logits > given) | ((logits == given) & (index[None, :] < tokens[:, None]))).sum(1)
    assert torch.equal(rk.long(), before)
    assert torch.equal(ids.long(), torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :32])
    want = torch.log_softmax(logits.double(), 1)[row, tokens.long()]
    same = (lp.double() == want) | ((lp.double() - want).abs() <= 400 * U)  # |d| below 12: (136 + 3 * 12) roundings
    assert bool(same.all())


def test_rising_rows(cuda):
    """Every later logit larger, and by whole tiles: the list of what reaches the threshold runs over."""
    vocab = 60000
    rows = [torch.arange(vocab, device="cuda") * 1e-3, (torch.arange(vocab, device="cuda") // 4096).float(),
            (torch.arange(vocab, device="cuda") % 1024).float() * 0.01]
    logits = torch.stack(rows)
    check(logits, torch.tensor([59999, 0, 1023], dtype=torch.int32, device="cuda"), 32)
    check(logits.repeat(300, 1)[:4], torch.tensor([5, 59000, 7, 8], dtype=torch.int32, device="cuda"), 20)


def test_nothing_left_nan_and_infinity(cuda):
    vocab = 9001
    logits = torch.randn((4, vocab), generator=gen(1), device="cuda")
    logits[0] = -math.inf
    logits[1, 5000] = math.nan
    logits[2, 77] = math.inf
    tokens = torch.tensor([5, 6, 7, 8], dtype=torch.int32, device="cuda")
    lp, h, rk, ids, tops = score(logits, tokens, 8)
    assert float(lp[0]) == -math.inf and float(h[0]) == 0.0 and int(rk[0]) == 5
    assert ids[0].tolist() == list(range(8)) and bool((tops[0] == -math.inf).all())
    for i in (1, 2):
        assert math.isnan(float(lp[i])) and math.isnan(float(h[i])) and bool(torch.isnan(tops[i]).all())
    best = torch.sort(logits[1].nan_to_num(nan=-math.inf), descending=True, stable=True).indices[:8]
    assert ids[1].tolist() == best.tolist() and int(ids[2, 0]) == 77
    logits[1] = math.nan
    logits[1, 4000] = logits[1, 100] = 1.0
    ids = score(logits, tokens, 4)[3]
    assert ids[1].tolist() == [100, 4000, -1, -1]
    check(logits[3:], tokens[3:], 8)


def test_ids_outside(cuda):
    logits = torch.randn((4, 700), generator=gen(2), device="cuda")
    check(logits, torch.tensor([-1, 700, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32, device="cuda"), 3)


def test_optional_outputs_and_one_row_apart(cuda):
    logits = torch.randn((3, 40000), generator=gen(3), device="cuda")
    tokens = torch.tensor([1, 2, 39999], dtype=torch.int32, device="cuda")
    full = score(logits, tokens, 20)
    bare = score(logits, tokens, 0, entropy=False, rank=False)
    assert torch.equal(full[0], bare[0])
    assert bool((bare[1] == 7.0).all()) and bool((bare[2] == -7).all())
    again = score(logits, tokens, 20)
    assert all(torch.equal(a, b) for a, b in zip(full, again))


def test_captured_after_the_pick(cuda):
    """As a server uses it: the greedy pick of a batch of logits, then its log probability, replayed on new logits."""
    rows, vocab = 5, 151936
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        logits = torch.zeros((rows, vocab), device="cuda")
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        lp, h = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        am = nodes.argmax_params(vocab, rows)
        am_bytes = nodes.argmax_workspace_size(am)
        am_ws = torch.empty(am_bytes, dtype=torch.uint8, device="cuda")
        p = nodes.token_logprobs_params(rows, vocab)
        size = nodes.token_logprobs_workspace_size(p)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")

        def step():
            nodes.argmax(am, logits, tokens, am_ws, am_bytes, stream=stream)
            nodes.token_logprobs(p, logits, tokens, lp, ws, size, entropy=h, stream=stream)

        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for seed in range(4):
            logits.copy_(torch.randn((rows, vocab), generator=gen(seed), device="cuda") * 4)
            graph.replay()
            stream.synchronize()
            want = torch.log_softmax(logits.double(), 1).amax(1)
            assert torch.equal(tokens.long(), logits.argmax(1))
            # at most 136 + 3 |d| roundings of log(1 + R), |d| below 60 here
            assert bool(((lp.double() - want).abs() <= 400 * U).all())
        del graph
    torch.cuda.synchronize()
