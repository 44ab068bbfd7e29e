"""The paged-cache entry points against plain forms in 64 bits: block tables and slot maps, rotary append, one-token
attention, and a run of them together as a server makes it (eager and as a replayed CUDA graph).

Tolerances count roundings, u = 2^-24 per F32 operation:
* rotary append: the rotation is evaluated in float64 and rounded once to F32, then once to the pool's type: half a
  step of each (F32 u, F16 2^-11, e4m3 2^-4 relative; below the normal range half the smallest step), plus one
  division by the scale, plus 1e-9 of the pair's size for the angle (positions to 2^18 times 2^-52, and the sine's own
  rounding, are far below it).
* attention: a score's error is at most (2 HD + 16) u sum_d |scale q_d k_d| (products of exact values, an addition per
  channel that may drop a last bit, the two halves that F32 operands are split into, the scale); the exponential adds
  2^-21. A weight's relative error d moves the output by at most 2 d sum_j p_j |v_j|, and each of the n additions
  in the sums by 2 u of that at most.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from muyo_llm_b200 import _abi, nodes

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {_abi.KV_F32: torch.float32, _abi.KV_F16: torch.float16, _abi.KV_F8: torch.float8_e4m3fn}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(shape, g, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stored(x, dtype):
    return (x.clamp(-448, 448) if dtype == _abi.KV_F8 else x).to(DTYPES[dtype])


def as_bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


# ---- plan ---------------------------------------------------------------------------------------------------

def plan_reference(cached, new, table, ring, state, page, max_tokens):
    """One request after the other."""
    table, ring = [list(r) for r in table], list(ring)
    pages, width = len(ring), len(table[0])
    head, tail = state
    free = min(max(tail - head, 0), pages)
    taken = refused = total = need_so_far = 0
    lens, starts, positions, slots = [], [0], [0] * max_tokens, [-1] * max_tokens
    before = [list(r) for r in table]
    back = []
    for i, (c, n) in enumerate(zip(cached, new)):
        c = min(max(c, 0), width * page)
        had = -(-c // page)
        start, total = total, total + max(n, 0)
        starts.append(total)
        if n < 0:
            back += before[i][:had]
        fits = n > 0 and c + n <= width * page
        need = -(-(c + n) // page) - had if fits else 0
        need_so_far += need
        ok = fits and need_so_far <= free and total <= max_tokens
        refused += n > 0 and not ok
        lens.append(c + n if ok else 0 if n < 0 else c)
        if ok:
            for k in range(need):
                table[i][had + k] = ring[(head + taken) % pages]
                taken += 1
            for t in range(start, total):
                pos = c + t - start
                positions[t] = pos
                at = table[i][pos // page]
                slots[t] = at * page + pos % page if 0 <= at < pages else -1
    back = back[:pages - free]
    out = list(ring)
    for k, b in enumerate(back):
        out[(tail + k) % pages] = b
    return table, out, lens, starts, positions, slots, [head + taken, tail + len(back), refused, total]


def run_plan(cached, new, table, ring, state, page, max_tokens, in_place=False):
    n = len(cached)
    p = nodes.paged_plan_params(n, page_size=page, num_pages=len(ring), table_stride=len(table[0]), max_tokens=max_tokens)
    cached_d, table_d, ring_d = ints(cached), ints(table), ints(ring)
    state_d = torch.tensor([state[0], state[1], 0, 0], dtype=torch.int64, device="cuda")
    lens = cached_d if in_place else torch.empty(n, dtype=torch.int32, device="cuda")
    state_out = state_d if in_place else torch.empty(4, dtype=torch.int64, device="cuda")
    starts = torch.empty(n + 1, dtype=torch.int32, device="cuda")
    positions, slots = (torch.full((max_tokens + 3,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    nodes.paged_plan(p, cached_d, ints(new), table_d, ring_d, state_d, lens, starts, positions, slots, state_out)
    torch.cuda.synchronize()
    for t in (positions, slots):
        assert t[max_tokens:].tolist() == [77] * 3
    return (table_d.tolist(), ring_d.tolist(), lens.tolist(), starts.tolist(), positions[:max_tokens].tolist(),
            slots[:max_tokens].tolist(), state_out.tolist())


def plan_case(rng, seqs, page, width, new_of, free, head):
    cached = [int(rng.integers(0, page * width + 1)) for _ in range(seqs)]
    new = [int(new_of(rng)) for _ in range(seqs)]
    had = [-(-c // page) for c in cached]
    pages = sum(had) + free
    ids = rng.permutation(pages).tolist() if pages else []
    pages = max(pages, 1)
    table, at = [], 0
    for h in had:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    ring = [-1] * pages
    for k in range(free):
        ring[(head + k) % pages] = ids[at + k]
    return cached, new, table, ring, (head, head + free)


PLAN_CASES = [
    # seqs, page, width, new tokens of a request, free pages, head, tokens buffer
    (1, 16, 4, lambda r: 1, 3, 0, 1),
    (1, 1, 1, lambda r: 1, 1, 5, 2),
    (5, 16, 8, lambda r: r.integers(-1, 40), 40, 7, 200),
    (33, 3, 50, lambda r: r.integers(-1, 9), 60, 12345678901, 300),
    (250, 16, 130, lambda r: 1, 40, 99, 256),
    (1025, 32, 9, lambda r: r.integers(-1, 60), 900, 3, 20000),  # more than a request per thread, a row too narrow
    (300, 8, 20, lambda r: r.integers(0, 30), 50, 0, 9000),  # the free pages run out
    (300, 8, 20, lambda r: r.integers(0, 30), 2000, 0, 700),  # the tokens' buffer runs out
    (40, 8, 20, lambda r: -1, 10, 4, 5),  # everything ends
    (40, 8, 20, lambda r: 0, 10, 4, 5),  # nothing happens
    (12, 8, 20, lambda r: r.integers(0, 5), 0, 4, 100),  # no free page: only room in the last page
    (3, 64, 40, lambda r: 900, 60, 1, 2700),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(PLAN_CASES)))
def test_plan(cuda, case, in_place):
    seqs, page, width, new_of, free, head, max_tokens = PLAN_CASES[case]
    args = plan_case(np.random.default_rng(case), seqs, page, width, new_of, free, head)
    want = plan_reference(*args, page, max_tokens)
    got = run_plan(*args, page, max_tokens, in_place)
    for name, g, w in zip(("table", "ring", "lens", "starts", "positions", "slots", "state"), got, want):
        assert g == w, (name, case)


def test_plan_largest_batch(cuda):
    args = plan_case(np.random.default_rng(5), 8192, 16, 3, lambda r: r.integers(-1, 20), 12000, 1)
    assert list(run_plan(*args, 16, 90000)) == list(plan_reference(*args, 16, 90000))


def test_plan_without_tokens_buffer(cuda):
    args = plan_case(np.random.default_rng(6), 9, 4, 6, lambda r: -1 if r.random() < 0.5 else 0, 3, 1)
    assert list(run_plan(*args, 4, 0)) == list(plan_reference(*args, 4, 0))


def test_plan_with_the_largest_max_tokens(cuda):
    """Every place of buffers of 2^31 - 2 tokens is written, and none behind them."""
    tokens = (1 << 31) - 2
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    p = nodes.paged_plan_params(2, page_size=16, num_pages=8, table_stride=4, max_tokens=tokens)
    positions, slots = (torch.full((tokens + 2,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    lens, starts, state = ints([0, 0]), ints([0, 0, 0]), torch.tensor([0, 8, 0, 0], device="cuda")
    nodes.paged_plan(p, ints([0, 0]), ints([3, 20]), table, torch.arange(8, dtype=torch.int32, device="cuda"), state, lens, starts,
                     positions, slots, state)
    torch.cuda.synchronize()
    assert slots[:23].tolist() == [*range(3), *range(16, 36)] and positions[:23].tolist() == [*range(3), *range(20)]
    assert bool((slots[23:tokens] == -1).all()) and bool((positions[23:tokens] == 0).all())
    assert slots[tokens:].tolist() == positions[tokens:].tolist() == [77, 77]
    assert lens.tolist() == [3, 20] and state.tolist() == [3, 8, 0, 23]


@pytest.mark.parametrize("state", [(10, 5), (0, 1 << 40), (-7, 3)])
def test_plan_survives_bad_content(cuda, state):
    """Lengths past the row, page numbers and counters that make no sense: nothing is touched out of bounds, lengths and
    slots stay in their ranges."""
    rng = np.random.default_rng(3)
    n, page, width, pages = 70, 8, 5, 64
    cached = rng.integers(-(1 << 31), 1 << 31, n).tolist()
    new = rng.integers(-5, 60, n).tolist()
    new[3] = (1 << 31) - 1
    table = rng.integers(-(1 << 31), 1 << 31, (n, width)).tolist()
    ring = rng.integers(-(1 << 31), 1 << 31, pages).tolist()
    got = run_plan(cached, new, table, ring, state, page, 400)
    assert all(0 <= v <= page * width for v in got[2])
    assert all(-1 <= v < page * pages for v in got[5])


# ---- rotary append ------------------------------------------------------------------------------------------

def frequencies(n_dims, base, freq_scale=1.0, ext=0.0, attn=1.0, corr=(0.0, 0.0), ff=None):
    j = np.arange(n_dims // 2)
    f = float(np.float32(base)) ** (-2.0 * j / n_dims)
    if ff is not None:
        f = f / ff.astype(np.float64)
    mix = np.zeros(n_dims // 2)
    size = attn
    if ext:
        mix = (1 - np.clip((j - corr[0]) / max(0.001, corr[1] - corr[0]), 0, 1)) * ext
        size = attn * (1 + 0.1 * math.log(1 / freq_scale))
    return np.append(f * (freq_scale * (1 - mix) + mix), size)


@pytest.mark.parametrize("kw", [dict(), dict(freq_scale=0.25), dict(freq_scale=0.25, ext=1.0, corr=(6.0, 14.0)),
                                dict(freq_scale=0.125, ext=0.5, attn=1.5, corr=(3.0, 3.0)), dict(with_ff=True)])
@pytest.mark.parametrize("n_dims", [2, 64, 128])
def test_rope_frequencies(cuda, n_dims, kw):
    kw = dict(kw)
    ff = np.linspace(1, 9, n_dims // 2).astype(np.float32) if kw.pop("with_ff", False) else None
    p = nodes.rope_params(1, n_dims, freq_base=500000.0)
    p.freq_scale, p.ext_factor, p.attn_factor = kw.get("freq_scale", 1.0), kw.get("ext", 0.0), kw.get("attn", 1.0)
    p.corr_dims[0], p.corr_dims[1] = kw.get("corr", (0.0, 0.0))
    p.has_ff = ff is not None
    table = torch.zeros(n_dims // 2 + 2, dtype=torch.float64, device="cuda")
    nodes.rope_frequencies(p, table, None if ff is None else torch.from_numpy(ff).cuda())
    want = frequencies(n_dims, 500000.0, ff=ff, **kw)
    got = table.cpu().numpy()
    # a power, a division and a mix in float64: a few steps of 2^-53, and pow's exponent of at most log2(5e5) = 19
    assert np.all(np.abs(got[:-1] - want) <= 64 * 2.0 ** -53 * np.abs(want)) and got[-1] == 0


def rotated64(x, positions, freqs, mode, n_dims, n_offs):
    """x [tokens][heads][head_dim] float64."""
    half = n_dims // 2
    y = x.clone()
    a = positions.double()[:, None] * freqs[:half][None, :]
    c, s = (torch.cos(a) * freqs[half])[:, None], (torch.sin(a) * freqs[half])[:, None]
    one = torch.arange(half, device=x.device) * (1 if mode == _abi.ROPE_NEOX else 2) + n_offs
    two = one + (half if mode == _abi.ROPE_NEOX else 1)
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., one] * s + x[..., two] * c
    return y


STEP = {_abi.KV_F32: (U, 2.0 ** -150), _abi.KV_F16: (2.0 ** -11, 2.0 ** -25), _abi.KV_F8: (2.0 ** -4, 2.0 ** -10)}


def check_rounded(got, want, dtype, size):
    rel, least = STEP[dtype]
    want = want.clamp(-448, 448) if dtype == _abi.KV_F8 else want
    tol = rel * want.abs() + least + 2 * U * want.abs() + 1e-9 * size
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()


APPEND_CASES = [
    # tokens, heads, kv_heads, head_dim, n_dims, n_offs, mode, dtype, order, page, far, extra row stride, in place
    (1, 14, 2, 64, 64, 0, _abi.ROPE_NEOX, _abi.KV_F16, "hnd", 16, 100, 0, False),
    (65, 14, 2, 64, 64, 0, _abi.ROPE_NEOX, _abi.KV_F32, "nhd", 16, 2048, 8, True),
    (37, 32, 8, 128, 64, 0, _abi.ROPE_NORMAL, _abi.KV_F8, "nhd", 32, 131000, 0, False),
    (300, 8, 8, 128, 128, 0, _abi.ROPE_NORMAL, _abi.KV_F16, "hnd", 24, 262000, 4, False),
    (7, 16, 1, 32, 24, 6, _abi.ROPE_NEOX, _abi.KV_F16, "hnd", 1, 5000, 0, True),
    (7, 16, 1, 32, 24, 6, _abi.ROPE_NORMAL, _abi.KV_F8, "hnd", 3, 5000, 12, False),
    (19, 3, 3, 16, 16, 0, _abi.ROPE_NEOX, _abi.KV_F8, "nhd", 8, 70, 0, False),
    (19, 3, 3, 16, 2, 14, _abi.ROPE_NEOX, _abi.KV_F32, "nhd", 8, 70, 0, False),
    (9, 4, 2, 64, 0, 0, _abi.ROPE_NEOX, _abi.KV_F16, "hnd", 16, 70, 0, False),
    (9, 4, 2, 64, 56, 8, _abi.ROPE_NEOX, _abi.KV_F16, "hnd", 16, 70, 0, False),
    (33, 48, 4, 128, 120, 4, _abi.ROPE_NEOX, _abi.KV_F32, "hnd", 16, 70, 0, True),
]


@pytest.mark.parametrize("case", range(len(APPEND_CASES)))
def test_rope_append(cuda, case):
    tokens, heads, kv, hd, n_dims, n_offs, mode, dtype, order, page, far, extra, in_place = APPEND_CASES[case]
    g = gen(case)
    scales = (0.04, 0.5) if dtype == _abi.KV_F8 else (0.0, 0.0) if case % 2 else (2.0, 0.25)
    pages = -(-tokens // page) + 2
    cache = nodes.paged_cache_params(heads, kv, hd, page_size=page, num_pages=pages, kv_dtype=dtype, order=order,
                                     k_scale=scales[0], v_scale=scales[1])
    row = (heads + 2 * kv) * hd + extra  # q, k and v as one projection's rows
    qkv = randn((tokens, row), g, 3.0)
    q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:(heads + 2 * kv) * hd]
    x = [t.double().reshape(tokens, -1, hd).clone() for t in (q, k, v)]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
    left_out = torch.rand(tokens, generator=g, device="cuda") < 0.2
    if tokens > 1:
        slots[left_out] = -1
        if bool(left_out.any()):
            slots[int(left_out.nonzero()[0])] = pages * page  # past the pool: left out as well
    live = (slots >= 0) & (slots < pages * page)
    positions = torch.randint(0, far, (tokens,), generator=g, device="cuda").to(torch.int32)
    freqs = torch.from_numpy(frequencies(n_dims, 10000.0, 0.5, 1.0, 1.25, (2.0, 9.0))).cuda() if n_dims else None
    fill = 0.5
    shape = (pages, kv, page, hd) if order == "hnd" else (pages, page, kv, hd)
    k_pool, v_pool = (torch.full(shape, fill, device="cuda").to(DTYPES[dtype]) for _ in range(2))
    q_out = q if in_place else torch.full((tokens, heads * hd + extra), 7.0, device="cuda")
    p = nodes.paged_append_params(cache, tokens, n_dims=n_dims, n_offs=n_offs, rope_mode=mode, stride_q=row, stride_k=row,
                                  stride_v=row, stride_q_out=q_out.stride(0))
    nodes.paged_rope_append(p, q, k, v, positions, slots, freqs, q_out, k_pool, v_pool)
    torch.cuda.synchronize()
    size = [t.abs().amax() * 2 for t in x]
    if n_dims:
        x[0], x[1] = (rotated64(t, positions, freqs, mode, n_dims, n_offs) for t in x[:2])
    got_q = q_out[:, :heads * hd].reshape(tokens, heads, hd)
    check_rounded(got_q[live], x[0][live], _abi.KV_F32, size[0])
    if not in_place:
        assert bool((q_out[~live] == 7.0).all()) and bool((q_out[:, heads * hd:] == 7.0).all())
    at = slots.long()[live]
    for pool, want, scale, s in ((k_pool, x[1], scales[0], size[1]), (v_pool, x[2], scales[1], size[2])):
        rows = as_bits(pool).transpose(1, 2) if order == "hnd" else as_bits(pool)
        rows = rows.reshape(pages * page, kv, hd)
        got = rows[at]
        got = got.view(torch.float8_e4m3fn).float() if dtype == _abi.KV_F8 else got
        check_rounded(got, want[live] / (np.float32(scale) or 1.0), dtype, s / (scale or 1.0))
        rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        rest[at] = False
        assert bool((rows[rest] == as_bits(torch.full((1,), fill, device="cuda").to(DTYPES[dtype]))).all())


def test_rope_append_keys_only(cuda):
    """q may be absent; values beyond e4m3 are stored as its largest, NaN stays NaN."""
    cache = nodes.paged_cache_params(4, 2, 16, page_size=4, num_pages=3, kv_dtype=_abi.KV_F8)
    k = torch.tensor([1e9, -1e9, float("nan"), 448.0, 464.0, -3.0, 2.0 ** -9, 0.0] * 4, device="cuda").reshape(1, 32)
    pools = [torch.zeros((3, 2, 4, 16), device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    p = nodes.paged_append_params(cache, 1, n_dims=0)
    nodes.paged_rope_append(p, None, k, k, ints([0]), ints([6]), None, None, *pools)
    torch.cuda.synchronize()
    want = torch.tensor([448.0, -448.0, float("nan"), 448.0, 448.0, -3.0, 2.0 ** -9, 0.0] * 2, device="cuda")
    for pool in pools:
        assert torch.equal(torch.nan_to_num(pool.float()[1, :, 2], nan=-99.0), torch.nan_to_num(want, nan=-99.0).expand(2, 16))
        assert int((as_bits(pool) != 0).sum()) == 2 * 14


def test_rope_append_agrees_with_kv_append(cuda):
    """One token of one sequence, as muyo_cuda_kv_append stores it (the same float64 rotation, rounded once)."""
    kv, hd, S, pos = 2, 64, 32, 19
    g = gen(3)
    k, v = randn((kv, hd), g), randn((kv, hd), g)
    kc, vc = (torch.zeros((kv, S, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    nodes.kv_append(nodes.attention_params(4, kv, hd, S), 1e6, k, v, kc, vc, ints([pos]))
    cache = nodes.paged_cache_params(4, kv, hd, page_size=S, num_pages=1)
    kp, vp = (torch.zeros((1, kv, S, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    freqs = torch.zeros(hd // 2 + 1, dtype=torch.float64, device="cuda")
    nodes.rope_frequencies(nodes.rope_params(1, hd, freq_base=1e6), freqs)
    nodes.paged_rope_append(nodes.paged_append_params(cache, 1), None, k, v, ints([pos]), ints([pos]), freqs, None, kp, vp)
    torch.cuda.synchronize()
    assert torch.equal(vp[0], vc)
    # both round the same real number; their angles differ by float64 roundings
    assert bool(((kp[0].double() - kc.double()).abs() <= 2.0 ** -10 * kc.double().abs() + 2.0 ** -24).all())


# ---- attention ------------------------------------------------------------------------------------------------

def attention64(q, k, v, scale):
    """q [heads][hd], k, v [keys][kv][hd] (float64): (out, lse, tolerance of out, tolerance of lse)."""
    heads, hd = q.shape
    n, kv = k.shape[:2]
    if n == 0:
        z = torch.zeros_like(q)
        return z, torch.full((heads,), -math.inf, dtype=q.dtype, device=q.device), z, torch.zeros_like(z[:, 0])
    qg = q.reshape(kv, heads // kv, hd)
    s = torch.einsum("hgd,thd->hgt", qg, k) * scale
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    out = torch.einsum("hgt,thd->hgd", p, v)
    ds = (2 * hd + 16) * U * torch.einsum("hgd,thd->hgt", qg.abs(), k.abs()).amax(-1) * abs(scale) + 2.0 ** -21
    tol = (2 * ds + 2 * (n + 16) * U)[..., None] * torch.einsum("hgt,thd->hgd", p, v.abs())
    return out.reshape(heads, hd), lse.reshape(heads), tol.reshape(heads, hd), (ds + 2 * (n + 16) * U + 4 * U * lse.abs()).reshape(heads)


def make_paged(lens, kv, hd, dtype, order, page, g, width=None, spread=1.0, scales=(0.0, 0.0), strides=None):
    """Pools with random keys and values of the given lengths on shuffled pages; every other slot holds NaN."""
    lens_t = torch.tensor(lens, device="cuda")
    had = (lens_t + page - 1) // page
    width = width or max(1, int(had.max()))
    held = int(had.sum())
    pages = held + 3
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < had[:, None]] = ids[:held]
    key = torch.arange(width * page, device="cuda")
    slot = table.long().clamp(min=0)[:, key // page] * page + key % page
    used = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    used[slot[key[None, :] < lens_t[:, None]]] = True
    cache = dict(page_size=page, num_pages=pages, kv_dtype=dtype, order=order, k_scale=scales[0], v_scale=scales[1])
    values, pools = [], []
    for scale in scales:
        x = stored(randn((pages * page, kv, hd), g, spread), dtype)
        real = x.double() * float(np.float32(scale) or 1.0)
        bits = as_bits(x).clone()
        bits[~used] = 0x7F if dtype == _abi.KV_F8 else math.nan
        shaped = bits.reshape(pages, page, kv, hd)
        shaped = (shaped.transpose(1, 2) if order == "hnd" else shaped).contiguous()
        if strides:  # rows apart from one another, the space between them NaN
            ps, hs, ss = strides(page, kv, hd)
            flat = torch.full((pages * ps,), 0x7F if dtype == _abi.KV_F8 else math.nan, dtype=bits.dtype, device="cuda")
            torch.as_strided(flat, (pages, page, kv, hd), (ps, ss, hs, 1)).copy_(bits.reshape(pages, page, kv, hd))
            shaped = flat
            cache.update(page_stride=ps, head_stride=hs, slot_stride=ss)
        pools.append(shaped)
        values.append(real)
    rows = [slot[i, :n] for i, n in enumerate(lens)]
    return cache, pools, table, values, rows


def run_attention(cache, heads, kv, hd, q, pools, table, lens, *, window=0, scale=None, extra=0, stream=None, ws=None, lse=True):
    p = nodes.paged_attention_params(nodes.paged_cache_params(heads, kv, hd, **cache), len(lens), table_stride=table.shape[1],
                                     window=window, scale=scale, stride_q=q.stride(0), stride_out=heads * hd + extra)
    out = torch.full((len(lens) + 1, heads * hd + extra), 5.0, device="cuda")
    lse_t = torch.full((len(lens) + 1, heads), 5.0, device="cuda") if lse else None
    size = nodes.paged_attention_workspace_size(p)
    ws = torch.full((size,), 0xAB, dtype=torch.uint8, device="cuda") if ws is None else ws
    nodes.paged_attention_decode(p, q, *pools, table, ints(lens), out, ws, size, lse=lse_t, stream=stream)
    return out, lse_t


def check_attention(out, lse, q, values, rows, lens, heads, kv, hd, window, scale):
    torch.cuda.synchronize()
    n = len(lens)
    assert bool((out[n:] == 5.0).all()) and bool((out[:, heads * hd:] == 5.0).all())  # behind the last row, between rows
    for i in range(n):
        at = rows[i][max(0, len(rows[i]) - window):] if window else rows[i]
        want, want_lse, tol, tol_lse = attention64(q[i, :heads * hd].double().reshape(heads, hd), values[0][at], values[1][at], scale)
        err = (out[i, :heads * hd].double().reshape(heads, hd) - want).abs()
        assert bool((err <= tol).all()), (i, len(at), err.max().item(), tol.max().item())
        if lse is not None:
            same = (lse[i].double() == want_lse) | ((lse[i].double() - want_lse).abs() <= tol_lse)
            assert bool(same.all()), (i, lse[i], want_lse)
    if lse is not None:
        assert bool((lse[n:] == 5.0).all())


HEADS = [(14, 2, 64), (32, 8, 128), (16, 1, 128), (9, 9, 64), (22, 2, 32), (3, 1, 16), (32, 2, 64), (13, 1, 16)]


@pytest.mark.parametrize("dtype", [_abi.KV_F32, _abi.KV_F16, _abi.KV_F8])
@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("order,page,window", [("hnd", 16, 0), ("nhd", 24, 0), ("nhd", 1, 70), ("hnd", 64, 100)])
def test_attention(cuda, dtype, heads, kv, hd, order, page, window):
    g = gen(heads * 7 + hd + page)
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 129, 0, 300, 511, 1030, 5]
    scales = (0.03, 0.5) if dtype == _abi.KV_F8 else (0.0, 0.0)
    cache, pools, table, values, rows = make_paged(lens, kv, hd, dtype, order, page, g, scales=scales,
                                                   spread=20.0 if dtype == _abi.KV_F8 else 1.0)
    q = randn((len(lens), heads * hd), g, 2.0)
    scale = 1.0 / math.sqrt(hd)
    out, lse = run_attention(cache, heads, kv, hd, q, pools, table, lens, window=window)
    check_attention(out, lse, q, values, rows, lens, heads, kv, hd, window, scale)


@pytest.mark.parametrize("dtype", [_abi.KV_F32, _abi.KV_F16, _abi.KV_F8])
@pytest.mark.parametrize("lens", [[40000], [9000, 1, 20000, 0, 3], [2500] * 30, [1] * 700, [7, 0] * 500])
def test_attention_splits(cuda, dtype, lens):
    """Long caches with few rows (split and joined), and many short ones."""
    heads, kv, hd = (8, 2, 64) if len(lens) < 100 else (4, 2, 32)
    g = gen(len(lens))
    cache, pools, table, values, rows = make_paged(lens, kv, hd, dtype, "nhd", 16, g)
    q = randn((len(lens), heads * hd), g, 2.0)
    out, lse = run_attention(cache, heads, kv, hd, q, pools, table, lens)
    check_attention(out, lse, q, values, rows, lens, heads, kv, hd, 0, 1.0 / math.sqrt(hd))


@pytest.mark.parametrize("dtype", [_abi.KV_F32, _abi.KV_F16])
def test_attention_wide_pages_and_strides(cuda, dtype):
    """All layers of a page side by side (page strides far apart), padded rows of q and out, no lse."""
    heads, kv, hd, page = 14, 2, 64, 16
    lens = [5, 77, 300, 1000]
    g = gen(21)
    cache, pools, table, values, rows = make_paged(lens, kv, hd, dtype, "hnd", page, g, width=100,
                                                   strides=lambda page, kv, hd: (5 * page * kv * (hd + 8), hd + 8, kv * (hd + 8)))
    q = randn((len(lens), heads * hd + 24), g)
    out, _ = run_attention(cache, heads, kv, hd, q, pools, table, lens, extra=12, lse=False)
    check_attention(out, None, q, values, rows, lens, heads, kv, hd, 0, 0.125)


def test_attention_offsets_past_32_bits(cuda):
    """Pages 2^31 elements and more into the pool."""
    heads, kv, hd, page = 8, 1, 128, 16
    stride = 1 << 24  # elements from page to page
    pages = 300       # 5.0e9 elements: the pool is an F8 one, 5 GB
    pool = torch.full((pages * stride,), 0x7F, dtype=torch.uint8, device="cuda")
    g = gen(4)
    ids = [0, 299, 127, 128, 255, 256, 3]
    n = 7 * page - 3
    x = [stored(randn((7 * page, hd), g), _abi.KV_F8) for _ in range(2)]
    rows = pool.reshape(pages, stride)
    for j, i in enumerate(ids):
        rows[i, :page * hd] = as_bits(x[0])[j * page:(j + 1) * page].reshape(-1)
        rows[i, 1 << 20:(1 << 20) + page * hd] = as_bits(x[1])[j * page:(j + 1) * page].reshape(-1)
    cache = dict(page_size=page, num_pages=pages, kv_dtype=_abi.KV_F8, page_stride=stride, head_stride=page * hd, slot_stride=hd)
    q = randn((1, heads * hd), g)
    out, lse = run_attention(cache, heads, kv, hd, q, (pool, pool[1 << 20:]), ints([ids]), [n])
    values = [t.double().reshape(-1, 1, hd) for t in x]
    check_attention(out, lse, q, values, [torch.arange(n, device="cuda")], [n], heads, kv, hd, 0, 1.0 / math.sqrt(hd))
    del pool


@pytest.mark.parametrize("dtype", [_abi.KV_F32, _abi.KV_F16])
@pytest.mark.parametrize("size", [1e-20, 1e5, 3e4, 0.0])
def test_attention_query_range(cuda, dtype, size):
    """Queries far outside F16's range, against a scale that brings the scores back, and queries of zeros."""
    heads, kv, hd = 14, 2, 64
    lens = [1, 50, 333]
    g = gen(8)
    cache, pools, table, values, rows = make_paged(lens, kv, hd, dtype, "hnd", 16, g)
    q = randn((len(lens), heads * hd), g) * size
    scale = 0.3 / (size or 1.0)
    out, lse = run_attention(cache, heads, kv, hd, q, pools, table, lens, scale=scale)
    check_attention(out, lse, q, values, rows, lens, heads, kv, hd, 0, float(np.float32(scale)))


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attention_sharp_scores(cuda, sign):
    """Scores of hundreds, of both signs: one key takes all weight, early or late in the cache."""
    heads, kv, hd = 6, 1, 64
    lens = [700, 64, 2000]
    g = gen(9)
    cache, pools, table, values, rows = make_paged(lens, kv, hd, _abi.KV_F16, "hnd", 16, g)
    q = randn((len(lens), heads * hd), g, 30.0)
    out, lse = run_attention(cache, heads, kv, hd, q, pools, table, lens, scale=sign * 0.5)
    check_attention(out, lse, q, values, rows, lens, heads, kv, hd, 0, sign * 0.5)


def test_attention_bad_pages_and_lengths(cuda):
    """Keys on pages outside the pool are left out; lengths outside the row are clamped."""
    heads, kv, hd, page = 4, 2, 32, 16
    lens = [100, 100, 100, 40]
    g = gen(10)
    cache, pools, table, values, rows = make_paged(lens, kv, hd, _abi.KV_F16, "nhd", page, g)
    table[0, 2], table[0, 6], table[1, :] = -5, cache["num_pages"], 1 << 30
    rows[0] = torch.cat([rows[0][:32], rows[0][48:96]])
    rows[1] = rows[1][:0]
    q = randn((4, heads * hd), g)
    out, lse = run_attention(cache, heads, kv, hd, q, pools, table, lens)
    check_attention(out, lse, q, values, rows, lens, heads, kv, hd, 0, 1.0 / math.sqrt(hd))
    width = table.shape[1] * page  # 112 slots: the fourth request's row ends at 40, its table holds -1 behind
    out2, lse2 = run_attention(cache, heads, kv, hd, q, pools, table, [-7, 100, -(1 << 31), (1 << 31) - 1])
    torch.cuda.synchronize()
    assert width == 112 and bool((out2[[0, 2], :heads * hd] == 0).all()) and bool((lse2[[0, 2]] == -math.inf).all())
    assert torch.equal(out2[1], out[1])
    at = table[3, torch.arange(48, device="cuda") // page].long() * page + torch.arange(48, device="cuda") % page
    for kind in range(2):  # slots 40..47 of the fourth request's last page were never written: give them numbers
        assert bool(torch.isnan(pools[kind].reshape(-1, kv, hd)[at[40:]]).all())
        pools[kind].reshape(-1, kv, hd)[at[40:]] = values[kind][at[40:]].to(torch.float16)
    out2, lse2 = run_attention(cache, heads, kv, hd, q, pools, table, [-7, 100, -(1 << 31), (1 << 31) - 1])
    check_attention(out2, lse2, q, values, [at[:0], at[:0], at[:0], at], lens, heads, kv, hd, 0, 1.0 / math.sqrt(hd))


def test_attention_agrees_with_contiguous(cuda):
    """One request whose pages lie in order is muyo_cuda_attention_decode's contiguous cache."""
    heads, kv, hd, S, n = 14, 2, 64, 512, 389
    g = gen(12)
    K, V = (randn((kv, S, hd), g).half() for _ in range(2))
    q = randn((1, heads * hd), g)
    p = nodes.attention_params(heads, kv, hd, S, n_keys=n)
    size = nodes.attention_workspace_size(p)
    want = torch.empty(heads * hd, device="cuda")
    nodes.attention_decode(p, q, K, V, want, torch.empty(size, dtype=torch.uint8, device="cuda"), size)
    cache = dict(page_size=16, num_pages=S // 16, kv_dtype=_abi.KV_F16, page_stride=16 * hd, head_stride=S * hd, slot_stride=hd)
    table = torch.arange(S // 16, dtype=torch.int32, device="cuda").reshape(1, -1)
    out, _ = run_attention(cache, heads, kv, hd, q, (K, V), table, [n])
    torch.cuda.synchronize()
    _, _, tol, _ = attention64(q.double().reshape(heads, hd), K[:, :n].transpose(0, 1).double(), V[:, :n].transpose(0, 1).double(), 0.125)
    assert bool(((out[0] - want).abs().double() <= 2 * tol.reshape(-1)).all())


@pytest.mark.parametrize("window", [0, 50])
def test_attention_of_prompt_tokens(cuda, window):
    """Each token of a prompt as a row: its request's table row again, the keys up to its own."""
    heads, kv, hd, page = 14, 2, 64, 16
    prompts = [70, 1, 33]
    g = gen(14)
    cache, pools, table, values, rows = make_paged(prompts, kv, hd, _abi.KV_F16, "nhd", page, g)
    owner = [i for i, n in enumerate(prompts) for _ in range(n)]
    lens = [t + 1 for n in prompts for t in range(n)]
    q = randn((len(lens), heads * hd), g, 2.0)
    out, lse = run_attention(cache, heads, kv, hd, q, pools, table[owner].contiguous(), lens, window=window)
    check_attention(out, lse, q, values, [rows[i][:n] for i, n in zip(owner, lens)], lens, heads, kv, hd, window, 0.125)


def test_attention_repeats_bit_for_bit(cuda):
    heads, kv, hd = 14, 2, 64
    lens = [1500, 3, 700, 8000]
    g = gen(13)
    cache, pools, table, _, _ = make_paged(lens, kv, hd, _abi.KV_F16, "hnd", 16, g)
    q = randn((4, heads * hd), g)
    first, lse = run_attention(cache, heads, kv, hd, q, pools, table, lens)
    for _ in range(5):
        again, lse2 = run_attention(cache, heads, kv, hd, q, pools, table, lens)
        torch.cuda.synchronize()
        assert torch.equal(first, again) and torch.equal(lse, lse2)


# ---- the step, as a server makes it ------------------------------------------------------------------------------

class Server:
    """A one-layer step over device state: plan, append, attention; all buffers fixed, so that it can be captured."""

    def __init__(self, seqs, heads, kv, hd, page, pages, width, tokens, dtype=_abi.KV_F16, stream=None):
        self.stream = stream
        self.cache = nodes.paged_cache_params(heads, kv, hd, page_size=page, num_pages=pages, kv_dtype=dtype)
        self.plan_p = nodes.paged_plan_params(seqs, page_size=page, num_pages=pages, table_stride=width, max_tokens=tokens)
        self.append_p = nodes.paged_append_params(self.cache, tokens)
        self.attn_p = nodes.paged_attention_params(self.cache, seqs, table_stride=width)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.new = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
        self.ring = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.state = torch.tensor([0, pages, 0, 0], dtype=torch.int64, device="cuda")
        self.starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
        self.positions, self.slots = (torch.zeros(tokens, dtype=torch.int32, device="cuda") for _ in range(2))
        self.q, self.q_rot = (torch.zeros((tokens, heads * hd), device="cuda") for _ in range(2))
        self.k, self.v = (torch.zeros((tokens, kv * hd), device="cuda") for _ in range(2))
        self.q_last, self.out = (torch.zeros((seqs, heads * hd), device="cuda") for _ in range(2))
        self.pools = [torch.full((pages, kv, page, hd), math.nan, device="cuda").to(DTYPES[dtype]) for _ in range(2)]
        self.freqs = torch.zeros(hd // 2 + 1, dtype=torch.float64, device="cuda")
        nodes.rope_frequencies(nodes.rope_params(1, hd), self.freqs)
        size = nodes.paged_attention_workspace_size(self.attn_p)
        self.ws, self.ws_bytes = torch.empty(size, dtype=torch.uint8, device="cuda"), size

    def step(self):
        nodes.paged_plan(self.plan_p, self.lens, self.new, self.table, self.ring, self.state, self.lens, self.starts,
                         self.positions, self.slots, self.state, stream=self.stream)
        nodes.paged_rope_append(self.append_p, self.q, self.k, self.v, self.positions, self.slots, self.freqs, self.q_rot,
                                *self.pools, stream=self.stream)
        # the last new token of each request asks (a request without new tokens asks with some row: not looked at)
        last = (self.starts[1:].long() - 1).clamp(0, self.q.shape[0] - 1)
        self.q_last.copy_(self.q_rot[last])
        nodes.paged_attention_decode(self.attn_p, self.q_last, *self.pools, self.table, self.lens, self.out, self.ws,
                                     self.ws_bytes, stream=self.stream)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", [_abi.KV_F16, _abi.KV_F32])
def test_server_steps(cuda, captured, dtype):
    """Requests that come with prompts, decode, end and make room, over 24 steps with pages running short; each request's
    output against a cache of its own."""
    seqs, heads, kv, hd, page, pages, width, tokens = 6, 14, 2, 64, 8, 40, 12, 96
    stream = torch.cuda.Stream()
    g = gen(30)
    rng = np.random.default_rng(31)
    with torch.cuda.stream(stream):
        s = Server(seqs, heads, kv, hd, page, pages, width, tokens, dtype, stream)
        if captured:
            s.step()  # nothing asked for: loads the modules
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                s.step()
        own_k, own_v = ([torch.zeros((0, kv, hd), dtype=torch.float64, device="cuda") for _ in range(seqs)] for _ in range(2))
        length, refused_steps, checked = [0] * seqs, 0, 0
        for step in range(24):
            new = [int(rng.integers(1, 40)) if n == 0 and rng.random() < 0.7 else 1 if n else 0 for n in length]
            new = [-1 if n > 60 or (n and rng.random() < 0.06) else a for n, a in zip(length, new)]
            s.new.copy_(ints(new))
            for t in (s.q, s.k, s.v):
                t.copy_(randn(t.shape, g))
            graph.replay() if captured else s.step()
            stream.synchronize()
            lens, starts = s.lens.tolist(), s.starts.tolist()
            refused_steps += s.state[2].item() > 0
            at = 0
            for i, a in enumerate(new):
                assert starts[i] == at
                mine = slice(at, at + max(a, 0))
                at += max(a, 0)
                if a < 0:
                    own_k[i], own_v[i], length[i] = own_k[i][:0], own_v[i][:0], 0
                elif a and lens[i] != length[i]:
                    assert lens[i] == length[i] + a
                    assert s.positions[mine].tolist() == list(range(length[i], lens[i]))
                    k = rotated64(s.k[mine].double().reshape(a, kv, hd), s.positions[mine], s.freqs, _abi.ROPE_NEOX, hd, 0)
                    own_k[i] = torch.cat([own_k[i], k.float().to(DTYPES[dtype]).double()])
                    own_v[i] = torch.cat([own_v[i], s.v[mine].reshape(a, kv, hd).to(DTYPES[dtype]).double()])
                    length[i] = lens[i]
                    q = rotated64(s.q[mine].double().reshape(a, heads, hd), s.positions[mine], s.freqs, _abi.ROPE_NEOX, hd, 0)[-1]
                    want, _, tol, _ = attention64(q, own_k[i], own_v[i], 1.0 / math.sqrt(hd))
                    # q and the keys themselves are off by their roundings: u of q, and a key may round to its neighbour
                    assert bool(((s.out[i].double().reshape(heads, hd) - want).abs() <= 4 * tol + 1e-6).all()), (step, i)
                    checked += 1
                assert lens[i] == length[i]
            used = sum(-(-n // page) for n in length)
            head, tail = s.state.tolist()[:2]
            assert tail - head == pages - used
            free = [s.ring[j % pages].item() for j in range(head, tail)]
            held = [x for i, n in enumerate(length) for x in s.table[i, :-(-n // page)].tolist()]
            assert sorted(free + held) == list(range(pages))  # every page is free or held, once
        assert checked > 60 and refused_steps > 0
        if captured:
            del graph
    torch.cuda.synchronize()


def test_two_streams_with_workspaces_of_their_own(cuda):
    heads, kv, hd = 8, 2, 128
    cases = []
    for k, lens in enumerate(([9000, 40, 700], [3, 12000])):
        g = gen(40 + k)
        cases.append((lens, make_paged(lens, kv, hd, _abi.KV_F16, "hnd", 16, g), randn((len(lens), heads * hd), g)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(4):
        for st, (lens, (cache, pools, table, values, rows), q) in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append((run_attention(cache, heads, kv, hd, q, pools, table, lens, stream=st), lens, q, values, rows))
    for (out, lse), lens, q, values, rows in got:
        check_attention(out, lse, q, values, rows, lens, heads, kv, hd, 0, 1.0 / math.sqrt(hd))
