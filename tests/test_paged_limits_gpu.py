"""Paged-cache entry points at the ends of their ranges: stored values next to a rounding border, scores far beyond
the weights' range, batches around the default limit of shared memory, rows of the most slots, a step as a host drives it.

U = 2^-24, half a step of F32."""
from __future__ import annotations

import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT
from muyo_llm_b200 import _abi, nodes
from test_paged_gpu import DTYPES, as_bits, attention64, gen, ints, plan_case, plan_reference, randn, rotated64, run_plan

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ---- stored values ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n_dims,n_offs", [(0, 0), (6, 2)])  # units of two float4, and pairs
@pytest.mark.parametrize("dtype", [_abi.KV_F32, _abi.KV_F16, _abi.KV_F8])
@pytest.mark.parametrize("scale", [0.03, 0.02, 1.0 / 3.0, 0.7, 3.0, 1.0, 2.0 ** -99 * 1.5, 1e20])
def test_append_stores_the_quotient(cuda, dtype, scale, n_dims, n_offs):
    """Every value next to a border of e4m3's or F16's rounding, bit for bit: x / scale rounded to F32, then to the pool's
    type (to e4m3: at most +-448). Both roundings are of the quotient, so there is no tolerance."""
    kv, hd, page = 2, 64, 16
    s = np.float32(scale)
    steps = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    if dtype == _abi.KV_F16:
        steps = np.concatenate([steps, np.arange(0x3C00, 0x3C00 + 600, dtype=np.uint16).view(np.float16).astype(np.float32)])
    mid = ((steps[1:].astype(np.float64) + steps[:-1]) / 2 * float(s)).astype(np.float32)
    near, up, down = [mid], mid, mid
    for _ in range(3):
        up, down = np.nextafter(up, np.float32(np.inf)), np.nextafter(down, np.float32(-np.inf))
        near += [up, down]
    x = np.concatenate(near + [np.array([0.0, np.inf, np.finfo(np.float32).max, np.nan], np.float32)])
    x = np.concatenate([x, -x])
    tokens = -(-len(x) // (kv * hd))
    x = np.concatenate([x, np.zeros(tokens * kv * hd - len(x), np.float32)])
    with np.errstate(over="ignore", invalid="ignore"):
        q = torch.from_numpy(x / s).reshape(tokens, kv, hd)
    want = as_bits((q.clamp(-448, 448) if dtype == _abi.KV_F8 else q).to(DTYPES[dtype]))
    pages = -(-tokens // page)
    cache = nodes.paged_cache_params(kv, kv, hd, page_size=page, num_pages=pages, kv_dtype=dtype, order="nhd", k_scale=scale, v_scale=scale)
    pools = [torch.zeros((pages * page, kv, hd), device="cuda").to(DTYPES[dtype]) for _ in range(2)]
    xd, at = torch.from_numpy(x).cuda(), torch.arange(tokens, dtype=torch.int32, device="cuda")
    freqs = torch.zeros(n_dims // 2 + 1, dtype=torch.float64, device="cuda")
    freqs[-1] = 1.0  # turned by nothing: x cos 0 - y sin 0 is x for finite x and y
    nodes.paged_rope_append(nodes.paged_append_params(cache, tokens, n_dims=n_dims, n_offs=n_offs), None, xd, xd, torch.zeros_like(at), at,
                            freqs, None, *pools)
    torch.cuda.synchronize()
    for name, pool in zip("kv", pools):
        got = as_bits(pool.cpu())[:tokens]
        keep = torch.ones(hd, dtype=torch.bool)
        if name == "k":
            keep[n_offs:n_offs + n_dims] = False  # infinities meet zeros there
        if dtype == _abi.KV_F8:
            same = (got == want) | ((got & 0x7F == 0x7F) & (want & 0x7F == 0x7F))
        else:
            same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        assert bool(same[..., keep].all()), (name, int((~same[..., keep]).sum()))


# ---- plan -----------------------------------------------------------------------------------------------------

def test_plan_around_the_default_limit_of_shared_memory(cuda):
    """In a process of its own, smaller batches first: a larger one raises the limit for all that follow."""
    code = """
import torch
from muyo_llm_b200 import _abi, nodes
_abi.call("muyo_cuda_init", 0)
for n in (3023, 3024, 3040, 3071, 3073):
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    lens, starts, positions, slots, table = i32(n), i32(n + 1), i32(n), i32(n), i32(n, 1)
    state = torch.tensor([0, n, 0, 0], device="cuda")
    nodes.paged_plan(nodes.paged_plan_params(n, page_size=4, num_pages=n, table_stride=1, max_tokens=n), lens, i32(n) + 1, table,
                     torch.arange(n, dtype=torch.int32, device="cuda"), state, lens, starts, positions, slots, state)
    assert torch.equal(slots, 4 * torch.arange(n, dtype=torch.int32, device="cuda")) and bool((lens == 1).all()), n
    assert state.tolist() == [n, n, 0, n], n
print("done")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True,
                          timeout=600)
    assert done.returncode == 0 and "done" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("page,width,pages", [(1 << 29, 2, 3), (1 << 30, 1, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_of_rows_of_the_most_slots(cuda, page, width, pages, in_place):
    """A full row holds 2^30 tokens: idle, refused and ended ones, one with room for a last token, lengths past the row."""
    full = 1 << 30
    cached = [full, full, full - 1, full, (1 << 31) - 1, 0, full - 2]
    new = [0, 1, 1, -1, 0, -1, 3]
    table = [[(i + j) % pages for j in range(width)] for i in range(len(cached))]
    args = (cached, new, table, list(range(pages)), (5, 5))
    got = run_plan(*args, page, 6, in_place)
    want = plan_reference(*args, page, 6)
    assert want[2] == [full, full, full, 0, full, 0, full - 2] and want[6][2] == 2
    assert list(got) == list(want)


def room_reference(cached, new, page, width, free, max_tokens):
    """(lengths, refused, pages taken) where requests that need no page pass those that wait for some."""
    lens, refused, taken, asked, total = [], 0, 0, 0, 0
    for c, n in zip(cached, new):
        total += max(n, 0)
        fits = n > 0 and c + n <= width * page
        need = -(-(c + n) // page) - -(-c // page) if fits else 0
        asked += need
        ok = fits and total <= max_tokens and (need == 0 or asked <= free)
        taken += need if ok else 0
        refused += n > 0 and not ok
        lens.append(c + n if ok else 0 if n < 0 else c)
    return lens, refused, taken


@pytest.mark.parametrize("seqs,page,width,free,max_tokens,most", [
    (2, 8, 4, 0, 2, 1), (60, 8, 20, 0, 200, 5), (300, 8, 20, 50, 9000, 30), (300, 8, 20, 50, 700, 30), (40, 1, 30, 9, 99, 4), (700, 16, 9, 0, 800, 2),
])
def test_plan_passes_requests_that_need_no_page(cuda, seqs, page, width, free, max_tokens, most):
    """With MUYO_PLAN_ROOM a request that has room in its last page gets its tokens behind one that found no pages."""
    rng = np.random.default_rng(seqs + free)
    cached = [8, 3] if seqs == 2 else [int(rng.integers(0, page * width + 1)) for _ in range(seqs)]
    new = [1, 1] if seqs == 2 else [int(rng.integers(-1, most + 1)) for _ in range(seqs)]
    had = [-(-c // page) for c in cached]
    ids = rng.permutation(sum(had) + free + 1).tolist()
    table, at = [], 0
    for h in had:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    head, pages = 11, len(ids)
    ring = [-1] * pages
    for k in range(free):
        ring[(head + k) % pages] = ids[at + k]
    lens, refused, taken = room_reference(cached, new, page, width, free, max_tokens)
    p = nodes.paged_plan_params(seqs, page_size=page, num_pages=pages, table_stride=width, max_tokens=max_tokens, flags=_abi.PLAN_ROOM)
    table_d, ring_d, lens_d, starts = ints(table), ints(ring), ints(cached), ints([0] * (seqs + 1))
    positions, slots = ints([77] * max_tokens), ints([77] * max_tokens)
    state = torch.tensor([head, head + free, 0, 0], device="cuda")
    nodes.paged_plan(p, lens_d, ints(new), table_d, ring_d, state, lens_d, starts, positions, slots, state)
    torch.cuda.synchronize()
    back = sum(h for h, n in zip(had, new) if n < 0)
    total = sum(max(n, 0) for n in new)
    assert lens_d.tolist() == lens and state.tolist() == [head + taken, head + free + min(back, pages - free), refused, total]
    if seqs == 2:
        assert lens == [8, 4] and refused == 1
    fresh = iter(ids[at:at + free])
    slots, positions, table_d, t = slots.tolist(), positions.tolist(), table_d.tolist(), 0
    for i, (c, n) in enumerate(zip(cached, new)):
        row = table[i][:had[i]]
        if lens[i] > c:
            row += [next(fresh) for _ in range(-(-lens[i] // page) - had[i])]
        assert table_d[i][:len(row)] == row and table_d[i][len(row):] == [-1] * (width - len(row))
        for u in range(max(n, 0)):
            if t < max_tokens:
                pos = c + u if lens[i] > c else 0
                assert (positions[t], slots[t]) == (pos, row[pos // page] * page + pos % page if lens[i] > c else -1), (i, t)
            t += 1
    assert all(s == -1 and x == 0 for s, x in zip(slots[t:], positions[t:]))


# ---- attention ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [_abi.KV_F32, _abi.KV_F16, _abi.KV_F8])
@pytest.mark.parametrize("heads,kv,hd", [(8, 1, 64), (16, 1, 64), (6, 2, 128), (32, 2, 128), (12, 1, 16)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_of_scores_up_to_1e9(cuda, dtype, heads, kv, hd, sign):
    """Scores of 1e4 to 1e9 and far apart: one key takes all weight. The output is its value, with the weight's two F16
    halves (2^-22 of it, or 4 u), a product, a division and a sum on top: 16 u. The log-sum-exp is its score, of hd products of one sign: at
    most (2 hd + 16) u of it, and 4 u."""
    page, lens = 16, [1, 2, 15, 40, 700, 3000]
    g = gen(heads + hd)
    pages = sum(-(-n // page) for n in lens)
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), -(-max(lens) // page)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        had = -(-n // page)
        table[i, :had] = ids[at:at + had]
        at += had
    pattern = torch.where(torch.rand((kv, hd), generator=g, device="cuda") < 0.5, 1.0, -1.0)
    level = torch.randint(2, 15, (pages * page,), generator=g, device="cuda").float()  # exact in e4m3
    best = []
    for i, n in enumerate(lens):
        rows = table[i].long().clamp(min=0)[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page
        low, high = int(rows[n // 3]), int(rows[n - 1])
        level[low], level[high] = (1.0, 15.0) if low != high else (5.0, 5.0)
        best.append(high if sign > 0 else low)
    k = (level[:, None, None] * pattern).to(DTYPES[dtype])
    v = torch.randn((pages * page, kv, hd), generator=g, device="cuda").to(DTYPES[dtype])
    # of each head another size: scores of size * 15 at most, a step of the levels apart
    size = torch.logspace(4, 9, len(lens) * heads, device="cuda", dtype=torch.float64).float()[torch.randperm(len(lens) * heads, generator=g, device="cuda")]
    size = size.reshape(len(lens), heads) / 15
    q = (size / hd)[..., None] * pattern.repeat_interleave(heads // kv, 0)
    p = nodes.paged_attention_params(nodes.paged_cache_params(heads, kv, hd, page_size=page, num_pages=pages, kv_dtype=dtype, order="nhd"),
                                     len(lens), table_stride=table.shape[1], scale=sign)
    out, lse = torch.empty((len(lens), heads, hd), device="cuda"), torch.empty((len(lens), heads), device="cuda")
    n_bytes = nodes.paged_attention_workspace_size(p)
    nodes.paged_attention_decode(p, q.contiguous(), k.reshape(pages, page, kv, hd), v.reshape(pages, page, kv, hd), table, ints(lens), out,
                                 torch.empty(n_bytes, dtype=torch.uint8, device="cuda"), n_bytes, lse=lse)
    torch.cuda.synchronize()
    for i, row in enumerate(best):
        want = v[row].double().repeat_interleave(heads // kv, 0)
        assert bool(((out[i].double() - want).abs() <= 16 * U * want.abs()).all()), (i, lens[i])
        score = sign * (q[i].double() * k[row].double().repeat_interleave(heads // kv, 0)).sum(-1)
        assert bool(((lse[i].double() - score).abs() <= (2 * hd + 20) * U * score.abs()).all()), (i, lse[i], score)


# ---- a host's step ---------------------------------------------------------------------------------------------

class Host:
    """A decode step of several layers as a host makes it from the library's calls alone. The step's tokens are packed in
    the requests' order. Each layer's q lies one row behind the start of its buffer, so that the row of request i's last
    token is row query_start[i + 1] of the buffer (row 0 stands for no token); `owner`, which the host writes beside new_lens, brings the attention's
    rows back to the tokens'. The layers are x + attention(x, x, x's first channels and its last ones)."""

    def __init__(self, layers, seqs, heads, kv, hd, page, pages, width, stream):
        self.stream, self.row, self.kv_row = stream, heads * hd, kv * hd
        cache = nodes.paged_cache_params(heads, kv, hd, page_size=page, num_pages=pages, kv_dtype=_abi.KV_F32)
        self.plan_p = nodes.paged_plan_params(seqs, page_size=page, num_pages=pages, table_stride=width, max_tokens=seqs, flags=_abi.PLAN_ROOM)
        self.append_p = nodes.paged_append_params(cache, seqs, stride_k=self.row, stride_v=self.row)
        self.attn_p = nodes.paged_attention_params(cache, seqs, table_stride=width)
        self.gather_p, self.back_p = nodes.get_rows_params(self.row, seqs + 1, seqs), nodes.get_rows_params(self.row, seqs, seqs)
        self.lens, self.new, self.owner, self.positions, self.slots = (ints([0] * seqs) for _ in range(5))
        self.starts, self.ring = ints([0] * (seqs + 1)), ints(range(pages))
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
        self.state = torch.tensor([0, pages, 0, 0], device="cuda")
        self.x, self.q_of, self.out, self.back = (torch.zeros((seqs, self.row), device="cuda") for _ in range(4))
        self.y = torch.zeros((seqs, self.row), device="cuda")
        self.q_rows = torch.zeros((seqs + 1, self.row), device="cuda")
        self.pools = [[torch.full((pages, kv, page, hd), math.nan, device="cuda") for _ in range(2)] for _ in range(layers)]
        self.freqs = torch.zeros(hd // 2 + 1, dtype=torch.float64, device="cuda")
        nodes.rope_frequencies(nodes.rope_params(1, hd), self.freqs, stream=stream)
        size = nodes.paged_attention_workspace_size(self.attn_p)
        self.ws, self.ws_bytes = torch.empty(size, dtype=torch.uint8, device="cuda"), size

    def step(self):
        s = self.stream
        nodes.paged_plan(self.plan_p, self.lens, self.new, self.table, self.ring, self.state, self.lens, self.starts,
                         self.positions, self.slots, self.state, stream=s)
        self.y.copy_(self.x)
        for pools in self.pools:
            nodes.paged_rope_append(self.append_p, self.y, self.y, self.y[:, self.row - self.kv_row:], self.positions, self.slots,
                                    self.freqs, self.q_rows[1:], *pools, stream=s)
            nodes.get_rows_f32(self.gather_p, self.q_rows, self.starts[1:], self.q_of, stream=s)
            nodes.paged_attention_decode(self.attn_p, self.q_of, *pools, self.table, self.lens, self.out, self.ws, self.ws_bytes, stream=s)
            nodes.get_rows_f32(self.back_p, self.out, self.owner, self.back, stream=s)
            self.y.add_(self.back)


@pytest.mark.parametrize("captured", [False, True])
def test_step_of_a_host(cuda, captured):
    """Ended, idle and refused requests among the others, two layers: each token against its request's own cache in
    64 bits. The first layer's error D (its tolerance, and the roundings of x + y) changes the second's scores by at
    most scale hd D (max |q| + max |k|) and its values by D."""
    layers, seqs, heads, kv, hd, page, pages, width = 2, 7, 8, 2, 64, 4, 22, 9
    scale, row = 1.0 / math.sqrt(hd), heads * hd
    g, rng, stream = gen(50), np.random.default_rng(51), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        s = Host(layers, seqs, heads, kv, hd, page, pages, width, stream)
        if captured:
            s.step()  # nothing asked for: loads the modules
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                s.step()
        empty = torch.zeros((0, kv, hd), dtype=torch.float64, device="cuda")
        own = [[[empty, empty] for _ in range(layers)] for _ in range(seqs)]
        length, answered, refused = [0] * seqs, 0, 0
        for number in range(60):
            new = [-1 if n and rng.random() < 0.04 else int(rng.random() < 0.8) for n in length]
            owner = [i for i, n in enumerate(new) if n == 1]
            s.new.copy_(ints(new))
            s.owner.copy_(ints(owner + [-1] * (seqs - len(owner))))
            s.x.copy_(randn(s.x.shape, g))
            graph.replay() if captured else s.step()
            stream.synchronize()
            lens = s.lens.tolist()
            for t, i in enumerate(owner):
                if lens[i] == length[i]:
                    refused += 1
                    assert s.slots[t].item() == -1
                    continue
                x, D, pos = s.x[t].double().reshape(1, heads, hd), 0.0, s.positions[t:t + 1]
                assert pos.item() == length[i] == lens[i] - 1
                for k in range(layers):
                    q = rotated64(x, pos, s.freqs, _abi.ROPE_NEOX, hd, 0)
                    key, value = q[:, :kv], x[:, heads - kv:]
                    own[i][k] = [torch.cat([own[i][k][0], key]), torch.cat([own[i][k][1], value])]
                    out, _, tol, _ = attention64(q[0], *own[i][k], scale)
                    most = [float(v.abs().max()) for v in (q, *own[i][k])]
                    moved = scale * hd * (D + 2 * U * most[1]) * (most[0] + most[1])
                    x = x + out
                    D += float(tol.max()) + 4 * U * float(x.abs().max()) + 2 * moved * most[2] + D
                assert float((s.y[t].double().reshape(heads, hd) - x[0]).abs().max()) <= D, (number, i)
                length[i], answered = lens[i], answered + 1
            for i, n in enumerate(new):
                if n < 0:
                    own[i], length[i] = [[empty, empty] for _ in range(layers)], 0
                assert lens[i] == length[i], (number, i)
        assert answered > 100 and refused > 3
        if captured:
            del graph
    torch.cuda.synchronize()


def test_step_is_repeated_after_a_refusal(cuda):
    """In place: whoever got tokens asks for none in the repeated plan, one request ends, and a third plan serves the refused one from the pages
    given back; no position is given twice and no page is lost."""
    page, width, pages = 8, 6, 6
    plan = nodes.paged_plan_params(4, page_size=page, num_pages=pages, table_stride=width, max_tokens=64)
    lens, table, ring = ints([0] * 4), torch.full((4, width), -1, dtype=torch.int32, device="cuda"), ints(range(pages))
    state, starts = torch.tensor([0, pages, 0, 0], device="cuda"), ints([0] * 5)
    positions, slots = ints([0] * 64), ints([0] * 64)

    def step(new):
        nodes.paged_plan(plan, lens, ints(new), table, ring, state, lens, starts, positions, slots, state)
        torch.cuda.synchronize()
        first = starts.tolist()
        return [a for a, n in enumerate(new) if n > 0 and slots[first[a]].item() == -1]  # the refused

    assert step([10, 16, 30, 4]) == [2, 3] and lens.tolist() == [10, 16, 0, 0]
    assert step([0, -1, 30, 4]) == [2, 3]  # the pages of ended requests serve the plans that follow
    assert step([0, 0, 30, 4]) == [3] and lens.tolist() == [10, 0, 30, 0]
    assert positions[:30].tolist() == list(range(30))
    assert step([0, 0, 2, 0]) == [] and positions[:2].tolist() == [30, 31]
    held = [x for i, n in enumerate(lens.tolist()) for x in table[i, :-(-n // page)].tolist()]
    head, tail = state.tolist()[:2]
    assert sorted(held + [ring[k % pages].item() for k in range(head, tail)]) == list(range(pages))


def test_plan_apart_is_made_again_with_other_lengths(cuda):
    """Outputs apart from the inputs: a plan that was not taken over leaves what the next one needs."""
    args = plan_case(np.random.default_rng(8), 60, 8, 20, lambda r: r.integers(-1, 30), 40, 3)
    cached, first, table, ring, state = args
    second = [-1 if i % 7 == 3 else 0 if n > 20 else max(n, 0) for i, n in enumerate(first)]
    p = nodes.paged_plan_params(60, page_size=8, num_pages=len(ring), table_stride=20, max_tokens=2000)
    cached_d, table_d, ring_d = ints(cached), ints(table), ints(ring)
    state_d, state_out = torch.tensor([*state, 0, 0], device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    lens, starts, positions, slots = ints([0] * 60), ints([0] * 61), ints([0] * 2000), ints([0] * 2000)
    for new in (first, second):
        nodes.paged_plan(p, cached_d, ints(new), table_d, ring_d, state_d, lens, starts, positions, slots, state_out)
    torch.cuda.synchronize()
    want = plan_reference(cached, second, table, ring, state, 8, 2000)
    assert [lens.tolist(), starts.tolist(), positions.tolist(), slots.tolist(), state_out.tolist()] == list(want[2:])
    for got, row, n in zip(table_d.tolist(), want[0], want[2]):
        assert got[:-(-n // 8)] == row[:-(-n // 8)]
    got = ring_d.tolist()
    assert all(got[k % len(ring)] == want[1][k % len(ring)] for k in range(want[6][0], want[6][1]))


def test_append_reads_a_table_made_before_it(cuda):
    """Two tables by turns into one buffer, between appends of one captured graph."""
    tokens, hd = 40, 64
    g, stream = gen(60), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x = randn((tokens, hd), g)
        positions, slots = ints(range(100, 100 + tokens)), ints(range(tokens))
        cache = nodes.paged_cache_params(1, 1, hd, page_size=tokens, num_pages=1, kv_dtype=_abi.KV_F32)
        freqs = torch.zeros(hd // 2 + 1, dtype=torch.float64, device="cuda")
        pools = [torch.zeros((tokens, hd), device="cuda") for _ in range(5)]
        bases = [10000.0, 500000.0, 30.0, 1e6]

        def run():
            for base, pool in zip(bases, pools):
                nodes.rope_frequencies(nodes.rope_params(1, hd, freq_base=base), freqs, stream=stream)
                nodes.paged_rope_append(nodes.paged_append_params(cache, tokens), None, x, x, positions, slots, freqs, None, pool, pools[4],
                                        stream=stream)

        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run()
        for _ in range(20):
            x.copy_(randn(x.shape, g))
            graph.replay()
            stream.synchronize()
            for base, pool in zip(bases, pools):
                j = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
                table = torch.cat([base ** (-2.0 * j / hd), torch.ones(1, dtype=torch.float64, device="cuda")])
                want = rotated64(x.double().reshape(tokens, 1, hd), positions, table, _abi.ROPE_NEOX, hd, 0)[:, 0]
                # one rounding, and angles of at most 140 off by 2^-45
                assert bool(((pool.double() - want).abs() <= U * want.abs() + 1e-11).all()), base
        del graph
    torch.cuda.synchronize()
