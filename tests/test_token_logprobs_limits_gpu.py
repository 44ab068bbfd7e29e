"""Log probabilities where single weights show, where sums are far below 1, and where rows are cut in every way.

U = 2^-24. A weight w = exp(d), d = (x - m) / T, is off by at most (3 |d| + 8) U of itself: the difference, the scaling's
two roundings, and the exponential (2^-22, or 4 U)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from muyo_llm_b200 import nodes
from test_token_logprobs_gpu import gen, score

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("vocab", [2, 40, 5000, 151936])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 30.0])
def test_single_weights(cuda, vocab, temperature):
    """Two tokens and masked ones: log p of the larger is -log(1 + w), of the smaller d - log(1 + w), with one weight w. log(1 + w) is off by the
    weight's error, w (3 |d| + 8) U, and by the 3 U of its logarithm and of the rounding of 1 + w's argument."""
    T = float(np.float32(temperature))
    gaps = torch.cat([torch.linspace(0.01, 6.0, 500), torch.linspace(6.0, 80.0, 50), torch.linspace(80.0, 86.0, 5)])
    gaps = ((gaps.double() * T).float()).cuda()
    if vocab > 5000:
        gaps = gaps[::9].contiguous()
    rows = len(gaps)
    logits = torch.full((rows, vocab), -math.inf, device="cuda")
    at = torch.randint(0, vocab, (rows,), generator=gen(vocab), device="cuda")
    to = (at + 1 + torch.randint(0, vocab - 1, (rows,), generator=gen(vocab + 1), device="cuda")) % vocab
    row = torch.arange(rows, device="cuda")
    logits[row, at] = 0.0
    logits[row, to] = -gaps
    d = -gaps.double() / T
    w = torch.exp(d)
    norm = torch.log1p(w)
    tol = w / (1 + w) * (3 * d.abs() + 8) * U + 3 * U * norm
    for tokens, want, more in ((at, -norm, 0.0), (to, d - norm, 4 * U * d.abs())):
        for top in (0, 2):
            lp, h, rank, ids, tops = score(logits, tokens.to(torch.int32), top, temperature)
            err = (lp.double() - want).abs()
            assert bool((err <= tol + more).all()), ((err / (tol + more)).max().item(), gaps[int((err / (tol + more)).argmax())].item())
            entropy = norm - d * w / (1 + w)
            tol_h = (w / (1 + w) * (d.abs() + 1) * (3 * d.abs() + 16)) * U + 4 * U * entropy
            assert bool(((h.double() - entropy).abs() <= tol_h).all())
            if top:
                assert bool(((tops[:, 0].double() + norm).abs() <= tol).all())


@pytest.mark.parametrize("rows", [1, 30, 700])
@pytest.mark.parametrize("fill", [-math.inf, torch.finfo(torch.float32).min])
def test_sums_far_below_one(cuda, rows, fill):
    """1 + R with R from 1e-35 to 1e-10, of many equal weights or of a few in the largest's own thread, piece and
    elsewhere: R keeps its relative accuracy. |d| is below 90, the sum adds 128 U."""
    vocab = 32003
    logits = torch.full((rows, vocab), fill, device="cuda")
    best = torch.randint(0, vocab, (rows,), generator=gen(rows), device="cuda")
    gap = torch.linspace(25.0, 80.0, rows, device="cuda")
    kind = torch.arange(rows, device="cuda") % 3
    for i in range(rows):
        b, lo = int(best[i]), -float(gap[i])
        if kind[i] == 0:
            logits[i] = lo
        elif kind[i] == 1:  # neighbours share a thread
            logits[i, max(b - 3, 0):b + 4] = lo
        else:
            logits[i, (b + 17000) % vocab] = lo
        logits[i, b] = 0.0
    d = logits.double()
    w = torch.exp(d)
    w[torch.arange(rows, device="cuda"), best] = 0.0
    R = w.sum(1)
    weighed = (w * d.clamp(min=-1e4)).sum(1)
    for top in (0, 5):
        lp, h, _, _, _ = score(logits, best.to(torch.int32), top)
        want = -torch.log1p(R)
        assert bool(((lp.double() - want).abs() <= 410 * U * want.abs()).all()), ((lp.double() - want) / want).abs().max().item()
        entropy = torch.log1p(R) - weighed / (1 + R)
        assert bool(((h.double() - entropy).abs() <= 800 * U * entropy).all())


def test_differences_beyond_f32(cuda):
    """Finite logits whose difference is not: log p is finite where (x - m) / T is, within 4 U of it."""
    big = torch.finfo(torch.float32).max
    logits = torch.full((2, 100), -math.inf, device="cuda")
    logits[:, 7], logits[:, 8], logits[:, 50] = big, -big, 0.0
    for temperature in (1e6, 3.0, 1.0):
        lp, h, rank, ids, tops = score(logits, torch.tensor([8, 7], dtype=torch.int32, device="cuda"), 4, temperature)
        T = float(np.float32(temperature))
        want = -2.0 * big / T
        if abs(want) < big:
            assert abs(float(lp[0]) - want) <= 4 * U * abs(want) and abs(float(tops[0, 2]) - want) <= 4 * U * abs(want)
        else:
            assert float(lp[0]) == -math.inf and float(tops[0, 2]) == -math.inf
        assert float(lp[1]) == 0.0 and float(h[0]) == 0.0
        assert rank.tolist() == [2, 0] and ids[0].tolist() == [7, 50, 8, 0] and float(tops[0, 3]) == -math.inf


def test_logits_of_the_kernel_before(cuda):
    """Logits written by a kernel of the library right in front, replayed with new ones."""
    rows, vocab = 64, 4001
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        a, b = (torch.zeros((rows, vocab), device="cuda") for _ in range(2))
        logits = torch.zeros((rows, vocab), device="cuda")
        tokens = torch.randint(0, vocab, (rows,), generator=gen(70), device="cuda").to(torch.int32)
        lp, rank = torch.zeros(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
        p = nodes.token_logprobs_params(rows, vocab)
        size = nodes.token_logprobs_workspace_size(p)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")

        def step():
            nodes.add(nodes.add_params(rows * vocab), a, b, logits, stream=stream)
            nodes.token_logprobs(p, logits, tokens, lp, ws, size, rank=rank, stream=stream)

        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(3):
                step()
        for seed in range(20):
            a.copy_(torch.randn(a.shape, generator=gen(seed), device="cuda") * 3)
            b.copy_(torch.randn(b.shape, generator=gen(seed + 100), device="cuda"))
            graph.replay()
            stream.synchronize()
            x = a + b
            given = x.gather(1, tokens.long()[:, None])
            assert torch.equal(rank.long(), (x > given).sum(1) + ((x == given) & (torch.arange(vocab, device="cuda")[None] < tokens[:, None])).sum(1))
            want = torch.log_softmax(x.double(), 1).gather(1, tokens.long()[:, None])[:, 0]
            # the largest weights' d is below 40: 136 + 3 * 40 roundings, and 3 of d
            assert bool(((lp.double() - want).abs() <= 400 * U).all())
        del graph
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [4, 40, 200, 900])
@pytest.mark.parametrize("vocab,top_k", [(60000, 32), (60001, 20), (8190, 32)])
def test_overfull_lists_in_rows_of_every_cut(cuda, rows, vocab, top_k):
    """Rising rows, steps of whole tiles, repeated ramps, constant rows, the lowest value, a few values: more logits reach the
    threshold than are listed, in rows of one piece, of a cluster and of many pieces."""
    index = torch.arange(vocab, device="cuda")
    lowest = torch.full((vocab,), torch.finfo(torch.float32).min, device="cuda")
    kinds = [index * 1e-3, (index // 4096).float(), (index % 1024).float() * 0.01, torch.full((vocab,), 2.5, device="cuda"), lowest,
             -(index // 600).float(), torch.round(torch.randn(vocab, generator=gen(vocab), device="cuda")),
             torch.where(index % 13 == 5, 1.0, lowest), torch.where(index % 2 == 0, index * 1e-4, -math.inf)]
    base = torch.stack(kinds)
    kind = torch.arange(rows, device="cuda") % len(kinds)
    logits = base[kind].contiguous()
    tokens = torch.randint(0, vocab, (rows,), generator=gen(rows), device="cuda")
    lp, h, rank, ids, tops = score(logits, tokens.to(torch.int32), top_k)
    d = (base.double() - base.double().amax(1, keepdim=True))
    w = torch.exp(d)
    best = base.argmax(1, keepdim=True)
    w = w.scatter(1, best, 0.0)
    R = w.sum(1, keepdim=True)
    norm, p = torch.log1p(R), w / (1 + R)
    finite = d.clamp(min=-1e4).abs()
    tol = U * (p * (3 * finite + 136)).sum(1, keepdim=True) + 2 * U * norm
    order = torch.sort(base, dim=1, descending=True, stable=True).indices[:, :top_k]
    place = torch.empty_like(base, dtype=torch.int64)
    place.scatter_(1, torch.sort(base, dim=1, descending=True, stable=True).indices, index.expand_as(place))
    assert torch.equal(ids.long(), order[kind])
    assert torch.equal(rank.long(), place[kind, tokens])

    def near(got, at_kind, at_id):
        dd = d[at_kind, at_id]
        want = dd - norm[at_kind, 0]
        return bool(((got.double() == want) | ((got.double() - want).abs() <= tol[at_kind, 0] + 3 * U * dd.abs() + U * want.abs())).all())

    assert near(lp, kind, tokens)
    for k in range(top_k):
        assert near(tops[:, k], kind, ids[:, k].long())
    entropy = (norm + (p * finite).sum(1, keepdim=True))[:, 0]
    tol_h = U * (p * (finite + 1) * (3 * finite + 300)).sum(1) + 2 * U * entropy
    assert bool(((h.double() - entropy[kind]).abs() <= tol_h[kind]).all())
