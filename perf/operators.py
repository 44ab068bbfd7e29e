"""The operators of a serving step over a paged key-value cache, as cases to be timed and compared.

* ``plan``: block tables, positions and slots of a ragged batch, built on the GPU from request lengths and a ring of free pages
* ``append``: rotary positions on the queries and keys of the batch, keys and values stored in their slots
* ``attend``: attention of one new token per request over the pages
* ``score``: log probabilities of given tokens, with entropy, rank and the top alternatives

``own = False`` computes each in elementary torch operations, ``own = True`` calls muyo_llm_b200.nodes."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "f8": torch.float8_e4m3fn}
F8_MAX = 448.0


# ---- cases -------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 250 requests: one token each, every 16th token opens a page
        dict(name="plan decode 250", op="plan", seqs=250, lo=20, hi=2000, new=1, release=0, page=16, spare=6, shortage=False),
        # prompts arrive, others decode, a seventh of the requests ends: the widest ragged step
        dict(name="plan mixed 1501", op="plan", seqs=1501, lo=1, hi=4000, new=600, release=7, page=32, spare=1000, shortage=False),
        # the decode step of the 0.5B model for 64 requests, F16 cache
        dict(name="append decode 64 f16", op="append", tokens=64, heads=14, kv_heads=2, dim=64, rot=64, mode="half", dtype="f16",
             base=1000000.0, scaled=False, order="hnd", page=16, far=2000, pad=0),
        # a prompt pass of a 7B-class layer into an 8-bit cache: interleaved, half of the head, scaled for a long context
        dict(name="append prompt 6001 f8", op="append", tokens=6001, heads=32, kv_heads=8, dim=128, rot=64, mode="pairs", dtype="f8",
             base=500000.0, scaled=True, order="nhd", page=32, far=131000, pad=40),
        # one request of the 0.5B model halfway through its context: latency
        dict(name="attend 1 x 1023 f16", op="attend", seqs=1, lo=1023, hi=1023, heads=14, kv_heads=2, dim=64, dtype="f16", order="hnd", page=16, window=0),
        # 200 requests of the 0.5B model up to its context
        dict(name="attend 200 x 2048 f16", op="attend", seqs=200, lo=60, hi=2048, heads=14, kv_heads=2, dim=64, dtype="f16", order="hnd", page=16, window=0),
        # one long document of a 7B-class layer: the split over the cache's length
        dict(name="attend 1 x 131071 f16", op="attend", seqs=1, lo=131071, hi=131071, heads=32, kv_heads=8, dim=128, dtype="f16", order="nhd", page=64, window=0),
        # a full batch of a 7B-class layer in an 8-bit cache
        dict(name="attend 64 x 16000 f8", op="attend", seqs=64, lo=2000, hi=16000, heads=32, kv_heads=8, dim=128, dtype="f8", order="nhd", page=32, window=0),
        # sixteen query heads on one key head, F32 cache, a sliding window, pages of an odd size
        dict(name="attend 33 x 9000 f32", op="attend", seqs=33, lo=500, hi=9000, heads=16, kv_heads=1, dim=128, dtype="f32", order="hnd", page=24, window=4096),
        # the token just sampled, with the usual five alternatives
        dict(name="score 1 x 151936", op="score", rows=1, vocab=151936, top=5, temperature=1.0, allowed=0),
        # a decode step's tokens, 20 alternatives, an eighth of the rows under a grammar's mask
        dict(name="score 97 x 151936", op="score", rows=97, vocab=151936, top=20, temperature=0.7, allowed=8),
        # a scored document: odd vocabulary (rows without alignment), no alternatives
        dict(name="score 2001 x 32001", op="score", rows=2001, vocab=32001, top=0, temperature=1.0, allowed=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "score"])
    if op == "plan":
        return dict(op=op, seqs=_log_int(rng, 1, 2000), lo=rng.choice([0, 1, 30]), hi=_log_int(rng, 40, 4000), new=rng.choice([1, 1, _log_int(rng, 2, 600)]),
                    release=rng.choice([0, 3, 11]), page=rng.choice([1, 8, 16, 24, 64, 128]), spare=rng.randint(0, 500), shortage=rng.random() < 0.2)
    if op == "append":
        dim = rng.choice([16, 32, 64, 128])
        kv = rng.choice([1, 2, 4, 8])
        return dict(op=op, tokens=_log_int(rng, 1, 6000), heads=kv * rng.randint(1, 16 if kv < 4 else 4), kv_heads=kv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, dim - 8]), mode=rng.choice(["half", "pairs"]), dtype=rng.choice(["f32", "f16", "f8"]),
                    base=rng.choice([10000.0, 500000.0, 1000000.0]), scaled=rng.random() < 0.5, order=rng.choice(["hnd", "nhd"]),
                    page=rng.choice([8, 16, 24, 64]), far=_log_int(rng, 50, 200000), pad=rng.randint(0, 30))
    if op == "attend":
        dim = rng.choice([16, 32, 64, 64, 128, 128])
        kv = rng.choice([1, 2, 4, 8])
        group = rng.randint(1, 16)
        size = {"f32": 4, "f16": 2, "f8": 1}
        dtype = rng.choice(["f32", "f16", "f16", "f8"])
        seqs = _log_int(rng, 1, 400)
        most = int(min(130000, 900e6 / (seqs * 2 * kv * dim * size[dtype])))
        hi = _log_int(rng, 16, max(17, most))
        return dict(op=op, seqs=seqs, lo=rng.choice([0, 1, hi // 3, hi]), hi=hi, heads=kv * group, kv_heads=kv, dim=dim, dtype=dtype,
                    order=rng.choice(["hnd", "nhd"]), page=rng.choice([1, 8, 16, 16, 24, 64, 128]), window=rng.choice([0, 0, 0, 100, 1024]))
    vocab = rng.choice([151936, 32001, 128256, _log_int(rng, 40, 250000)])
    return dict(op=op, rows=_log_int(rng, 1, max(2, min(4000, int(6.4e7 / vocab)))), vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]),
                temperature=rng.choice([1.0, 1.0, 0.6, 1.7]), allowed=rng.choice([0, 0, 5]))


def lengths(n, lo, hi):
    """n lengths spread over [lo, hi], more of them short: the same ones for every seed (their order is the seed's)."""
    if lo == hi:
        return np.full(n, hi, np.int64)
    u = (0.5 + np.arange(n) * 0.6180339887498949) % 1.0
    got = np.floor((lo + 1) * ((hi + 1) / (lo + 1)) ** u).astype(np.int64) - 1 + (lo > 0)
    got = np.clip(got, lo, hi)
    got[0] = hi
    return got


def new_tokens(case):
    """Tokens asked for by each request of a plan (-1: it ends), before the seed's order."""
    n = case["seqs"]
    got = np.ones(n, np.int64)
    if case["new"] > 1:  # a third of the requests bring a prompt
        got[::3] = lengths(len(got[::3]), 1, case["new"])
        got[5::13] = 0
    if case["release"]:
        got[case["release"] - 1::case["release"]] = -1
    return got


def plan_sizes(case):
    cached, new, page = lengths(case["seqs"], case["lo"], case["hi"]), new_tokens(case), case["page"]
    had, ask = -(-cached // page), np.maximum(new, 0)
    need = np.where(new > 0, -(-(cached + ask) // page) - had, 0)
    return cached, new, had, int(ask.sum()), int(need.sum())


def work(case):
    op = case["op"]
    if op == "plan":
        _, new, had, tokens, need = plan_sizes(case)
        ended = int(had[new < 0].sum())
        # lengths in and out, starts, pages from the ring into the tables and back, positions and slots
        return {"bytes": 16 * case["seqs"] + 8 * need + 8 * ended + 8 * (tokens + case["spare"]) + 64, "flops": 0}
    size = {"f32": 4, "f16": 2, "f8": 1}.get(case.get("dtype"))
    if op == "append":
        t, q, kv = case["tokens"], case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        return {"bytes": t * (8 * q + 8 * kv + 2 * kv * size + 8), "flops": 6 * t * (case["heads"] + case["kv_heads"]) * case["rot"] // 2}
    if op == "attend":
        lens = lengths(case["seqs"], case["lo"], case["hi"])
        if case["window"]:
            lens = np.minimum(lens, case["window"])
        keys = int(lens.sum())
        row = case["heads"] * case["dim"]
        return {"bytes": keys * 2 * case["kv_heads"] * case["dim"] * size + 8 * case["seqs"] * row + 4 * keys // case["page"],
                "flops": 4 * keys * row}
    n = case["rows"] * case["vocab"]
    return {"bytes": 4 * n + case["rows"] * (16 + 8 * case["top"]), "flops": 5 * n}


# ---- inputs ------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    state = {"plan": prepare_plan, "append": prepare_append, "attend": prepare_attend, "score": prepare_score}[case["op"]](case, g)
    state["case"] = dict(case)
    if own:  # the parameter block and the workspace that a program sets up once
        from muyo_llm_b200 import nodes

        state["nodes"] = nodes
        {"plan": setup_plan, "append": setup_append, "attend": setup_attend, "score": setup_score}[case["op"]](case, state, nodes)
    return state


def order_of(n, g):
    return torch.randperm(n, generator=g, device=DEVICE)


def int32(a):
    return torch.as_tensor(np.ascontiguousarray(a), device=DEVICE).to(torch.int32)


def prepare_plan(case, g):
    cached, new, had, tokens, need = plan_sizes(case)
    width = int((-(-(cached + np.maximum(new, 0)) // case["page"])).max()) + 1
    held = int(had.sum())
    free = need // 2 if case["shortage"] else need + 5
    pages = held + free
    shuffle = order_of(case["seqs"], g)
    cached, new = int32(cached)[shuffle].contiguous(), int32(new)[shuffle].contiguous()
    ids = order_of(pages, g).to(torch.int32)
    had = ((cached.long() + case["page"] - 1) // case["page"])
    col = torch.arange(width, device=DEVICE)
    mine = col[None, :] < had[:, None]
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEVICE)
    table[mine] = ids[:held]
    head = int(torch.randint(0, 1 << 20, (1,), generator=g, device=DEVICE))
    ring = torch.full((pages,), -1, dtype=torch.int32, device=DEVICE)
    ring[(head + torch.arange(free, device=DEVICE)) % pages] = ids[held:]
    return dict(cached=cached, new=new, table=table, ring=ring, state=torch.tensor([head, head + free, 0, 0], dtype=torch.int64, device=DEVICE),
                pages=pages, max_tokens=tokens + case["spare"])


def rope_settings(case):
    """(frequency scale, extrapolation factor, attention factor, first and last corrected pair)."""
    return (0.25, 1.0, 1.0, 6.0, 14.0) if case["scaled"] else (1.0, 0.0, 1.0, 0.0, 0.0)


def frequency_table(case):
    """Radians per position of each pair in float64, then the magnitude that scaling puts on the rotated values."""
    scale, ext, attn, low, high = rope_settings(case)
    j = np.arange(case["rot"] // 2, dtype=np.float64)
    freq = case["base"] ** (-2.0 * j / case["rot"])
    mix = (1.0 - np.clip((j - low) / max(0.001, high - low), 0.0, 1.0)) * ext if ext else np.zeros_like(j)
    freq = freq * (scale * (1.0 - mix) + mix)
    size = attn * (1.0 + 0.1 * math.log(1.0 / scale)) if ext else attn
    return np.concatenate([freq, [size]])


def pool_shape(case, pages):
    if case["order"] == "hnd":
        return (pages, case["kv_heads"], case["page"], case["dim"])
    return (pages, case["page"], case["kv_heads"], case["dim"])


def prepare_append(case, g):
    t, page = case["tokens"], case["page"]
    q_row, kv_row = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    qkv = torch.randn((t, q_row + 2 * kv_row), generator=g, device=DEVICE) * 2.0
    pages = -(-t // page) + 3
    slots = order_of(pages, g)[:, None] * page + torch.arange(page, device=DEVICE)[None, :]
    slots = slots.reshape(-1)[:t].to(torch.int32).contiguous()
    if case["pad"] and t > case["pad"]:
        slots[t - case["pad"]:] = -1  # the rest of a batch of a fixed size
    start = torch.randint(0, case["far"], (1,), generator=g, device=DEVICE)
    positions = ((start + torch.arange(t, device=DEVICE)) % case["far"]).to(torch.int32)
    pools = [torch.zeros(pool_shape(case, pages), device=DEVICE).to(TORCH[case["dtype"]]) for _ in range(2)]
    return dict(qkv=qkv, q=qkv[:, :q_row], k=qkv[:, q_row:q_row + kv_row], v=qkv[:, q_row + kv_row:], slots=slots, positions=positions,
                k_pool=pools[0], v_pool=pools[1], freqs=torch.as_tensor(frequency_table(case), device=DEVICE),
                q_out=torch.zeros((t, q_row), device=DEVICE), pages=pages)


def scales_of(case):
    """What a stored value stands for: value times scale (keys, values)."""
    return (0.03, 0.02) if case["dtype"] == "f8" else (1.0, 1.0)


def stored(x, dtype):
    return x.clamp(-F8_MAX, F8_MAX).to(TORCH[dtype]) if dtype == "f8" else x.to(TORCH[dtype])


def prepare_attend(case, g):
    page, n = case["page"], case["seqs"]
    lens = int32(lengths(n, case["lo"], case["hi"]))[order_of(n, g)].contiguous()
    width = -(-case["hi"] // page)
    had = (lens.long() + page - 1) // page
    held = int((-(-lengths(n, case["lo"], case["hi"]) // page)).sum())
    pages = held + 2
    ids = order_of(pages, g).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEVICE)
    table[torch.arange(width, device=DEVICE)[None, :] < had[:, None]] = ids[:held]
    # slots that no key was written to hold what the memory held before: here NaN
    key = torch.arange(width * page, device=DEVICE)
    used = torch.zeros(pages * page, dtype=torch.bool, device=DEVICE)
    where = table.long().clamp(min=0)[:, key // page] * page + key % page
    used[where[key[None, :] < lens[:, None]]] = True
    used = used.reshape((pages, 1, page, 1) if case["order"] == "hnd" else (pages, page, 1, 1))
    pools = []
    for scale in scales_of(case):
        x = torch.randn(pool_shape(case, pages), generator=g, device=DEVICE)
        pools.append(stored(x.div_(scale).masked_fill_(~used, math.nan), case["dtype"]))
        del x
    q = torch.randn((n, case["heads"] * case["dim"]), generator=g, device=DEVICE) * 1.5
    return dict(q=q, k_pool=pools[0], v_pool=pools[1], table=table, lens=lens, pages=pages, out=torch.empty_like(q),
                lse=torch.empty((n, case["heads"]), device=DEVICE))


def prepare_score(case, g):
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn((rows, vocab), generator=g, device=DEVICE) * 2.5
    best = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE)
    row = torch.arange(rows, device=DEVICE)
    logits[row, best] += 12.0
    tokens = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.6, best, torch.randint(0, vocab, (rows,), generator=g, device=DEVICE))
    if case["allowed"]:  # every so many rows leave a few tokens: the others are -inf
        few = torch.rand((len(row[::case["allowed"]]), vocab), generator=g, device=DEVICE) < 30.0 / vocab
        few[torch.arange(few.shape[0], device=DEVICE), best[::case["allowed"]]] = True
        logits[::case["allowed"]] = logits[::case["allowed"]].masked_fill(~few, -math.inf)
    top = (rows, case["top"])
    return dict(logits=logits, tokens=tokens.to(torch.int32), logprob=torch.empty(rows, device=DEVICE), entropy=torch.empty(rows, device=DEVICE),
                rank=torch.empty(rows, dtype=torch.int32, device=DEVICE), top_ids=torch.empty(top, dtype=torch.int32, device=DEVICE),
                top_logprobs=torch.empty(top, device=DEVICE))


# ---- the framework's calls ---------------------------------------------------------------------------------

def setup_cache(case, pages, nodes):
    from muyo_llm_b200 import _abi

    scales = scales_of(case)
    return nodes.paged_cache_params(case["heads"], case["kv_heads"], case["dim"], page_size=case["page"], num_pages=pages,
                                    kv_dtype={"f32": _abi.KV_F32, "f16": _abi.KV_F16, "f8": _abi.KV_F8}[case["dtype"]], order=case["order"],
                                    k_scale=scales[0], v_scale=scales[1])


def setup_plan(case, s, nodes):
    s["params"] = nodes.paged_plan_params(case["seqs"], page_size=case["page"], num_pages=s["pages"], table_stride=s["table"].shape[1],
                                          max_tokens=s["max_tokens"])
    s["seq_lens"] = torch.empty(case["seqs"], dtype=torch.int32, device=DEVICE)
    s["query_start"] = torch.empty(case["seqs"] + 1, dtype=torch.int32, device=DEVICE)
    s["positions"] = torch.empty(s["max_tokens"], dtype=torch.int32, device=DEVICE)
    s["slots"] = torch.empty(s["max_tokens"], dtype=torch.int32, device=DEVICE)
    s["state_out"] = torch.empty(4, dtype=torch.int64, device=DEVICE)


def setup_append(case, s, nodes):
    from muyo_llm_b200 import _abi

    row = s["qkv"].shape[1]
    s["params"] = nodes.paged_append_params(setup_cache(case, s["pages"], nodes), case["tokens"], n_dims=case["rot"],
                                            rope_mode=_abi.ROPE_NEOX if case["mode"] == "half" else _abi.ROPE_NORMAL, stride_q=row, stride_k=row, stride_v=row)


def setup_attend(case, s, nodes):
    s["params"] = nodes.paged_attention_params(setup_cache(case, s["pages"], nodes), case["seqs"], table_stride=s["table"].shape[1],
                                               window=case["window"])
    s["ws_bytes"] = nodes.paged_attention_workspace_size(s["params"])
    s["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device=DEVICE)


def setup_score(case, s, nodes):
    s["params"] = nodes.token_logprobs_params(case["rows"], case["vocab"], top_k=case["top"], temperature=case["temperature"])
    s["ws_bytes"] = nodes.token_logprobs_workspace_size(s["params"])
    s["ws"] = torch.empty(s["ws_bytes"], dtype=torch.uint8, device=DEVICE)


def own_plan(s):
    s["nodes"].paged_plan(s["params"], s["cached"], s["new"], s["table"], s["ring"], s["state"], s["seq_lens"], s["query_start"], s["positions"],
                          s["slots"], s["state_out"])
    return dict(table=s["table"], ring=s["ring"], lens=s["seq_lens"], starts=s["query_start"], positions=s["positions"], slots=s["slots"],
                state=s["state_out"])


def own_append(s):
    s["nodes"].paged_rope_append(s["params"], s["q"], s["k"], s["v"], s["positions"], s["slots"], s["freqs"], s["q_out"], s["k_pool"], s["v_pool"])
    return dict(q=s["q_out"], k=s["k_pool"], v=s["v_pool"])


def own_attend(s):
    s["nodes"].paged_attention_decode(s["params"], s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"], s["out"], s["ws"], s["ws_bytes"], lse=s["lse"])
    return dict(out=s["out"], lse=s["lse"])


def own_score(s):
    s["nodes"].token_logprobs(s["params"], s["logits"], s["tokens"], s["logprob"], s["ws"], s["ws_bytes"], entropy=s["entropy"], rank=s["rank"],
                              top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
    return dict(logprob=s["logprob"], entropy=s["entropy"], rank=s["rank"], top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": own_plan, "append": own_append, "attend": own_attend, "score": own_score}[op](state)
    return {"plan": plain_plan, "append": plain_append, "attend": plain_attend, "score": plain_score}[op](state)


# ---- the plain forms ---------------------------------------------------------------------------------------

def plain_plan(s):
    """A request asks for new[i] tokens behind the cached[i] that it has, or ends (new < 0) and gives its pages back. Requests get pages from the
    ring's head in their order, while it has enough, the row is wide enough and the batch's buffers are; the pages of ended ones go to its tail."""
    page, pages, max_tokens = s["case"]["page"], s["pages"], s["max_tokens"]
    table, width = s["table"].long(), s["table"].shape[1]
    cached, new = s["cached"].long().clamp(0, width * page), s["new"].long()
    ask = new.clamp(min=0)
    stop = ask.cumsum(0)
    start = stop - ask
    had = (cached + page - 1) // page
    fits = (new > 0) & (cached + ask <= width * page)
    need = torch.where(fits, (cached + ask + page - 1) // page - had, 0)
    upto = need.cumsum(0)
    first = upto - need
    head, tail = s["state"][0], s["state"][1]
    free = (tail - head).clamp(0, pages)
    ok = fits & (upto <= free) & (stop <= max_tokens)
    lens = torch.where(ok, cached + ask, torch.where(new < 0, 0, cached))
    taken = torch.where(ok, need, 0)
    back = torch.where(new < 0, had, 0)
    last = len(ask) - 1
    # tokens
    t = torch.arange(max_tokens, device=DEVICE)
    i = torch.searchsorted(stop, t, right=True).clamp(max=last)
    live = ok[i] & (t < stop[-1])
    pos = torch.where(live, cached[i] + t - start[i], 0)
    at = pos // page
    fresh = s["ring"].long()[(head + first[i] + (at - had[i]).clamp(min=0)) % pages]
    slot = torch.where(at < had[i], table[i, at], fresh) * page + pos % page
    slot = torch.where(live, slot, -1)
    # pages into the tables, and back into the ring; one more place takes what is not there
    p = torch.arange(pages, device=DEVICE)
    i = torch.searchsorted(upto, p, right=True).clamp(max=last)
    to = torch.where((p < taken.sum()), i * width + (had[i] + p - first[i]).clamp(max=width - 1), len(ask) * width)
    flat = torch.cat([s["table"].reshape(-1), s["table"].new_zeros(1)])
    flat = flat.index_put((to,), s["ring"][(head + p) % pages])
    ended = back.cumsum(0)
    i = torch.searchsorted(ended, p, right=True).clamp(max=last)
    gives = p < torch.minimum(ended[-1], pages - free)
    to = torch.where(gives, (tail + p) % pages, pages)
    ring = torch.cat([s["ring"], s["ring"].new_zeros(1)])
    ring = ring.index_put((to,), s["table"][i, (p - ended[i] + back[i]).clamp(0, width - 1)])
    refused = ((new > 0) & ~ok).sum()
    return dict(table=flat[:-1].reshape(s["table"].shape), ring=ring[:-1], lens=lens.to(torch.int32),
                starts=torch.cat([stop.new_zeros(1), stop]).to(torch.int32), positions=pos.to(torch.int32), slots=slot.to(torch.int32),
                state=torch.stack([head + taken.sum(), tail + torch.minimum(ended[-1], pages - free), refused, stop[-1]]))


def plain_append(s):
    case = s["case"]
    dim, rot, page, half = case["dim"], case["rot"], case["page"], case["rot"] // 2
    live = s["slots"] >= 0
    angle = s["positions"].double()[:, None] * s["freqs"][None, :half]
    size = s["freqs"][half]
    c, si = (angle.cos() * size).float()[:, None, :], (angle.sin() * size).float()[:, None, :]

    def rotated(x, heads):
        x = x.reshape(-1, heads, dim)
        a, b = (x[..., :half], x[..., half:rot]) if case["mode"] == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
        y = (a * c - b * si, a * si + b * c)
        y = torch.cat(y, -1) if case["mode"] == "half" else torch.stack(y, -1).flatten(-2)
        return torch.cat([y, x[..., rot:]], -1)

    q = torch.where(live[:, None], rotated(s["q"], case["heads"]).reshape(s["q_out"].shape), s["q_out"])
    values = (rotated(s["k"], case["kv_heads"]), s["v"].reshape(-1, case["kv_heads"], dim))
    slot = s["slots"].long()[live]
    pools = []
    for pool, x, scale in zip((s["k_pool"], s["v_pool"]), values, scales_of(case)):
        x = stored(x / scale, case["dtype"])
        bits, x = (pool.view(torch.uint8), x.view(torch.uint8)) if case["dtype"] == "f8" else (pool, x)
        rows = bits.transpose(1, 2) if case["order"] == "hnd" else bits
        rows[slot // page, slot % page] = x[live]
        pools.append(pool)
    return dict(q=q, k=pools[0], v=pools[1])


def plain_attend(s):
    case = s["case"]
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    n, width = s["table"].shape
    group = case["heads"] // kv
    pages = s["table"].long().clamp(min=0)
    key = torch.arange(width * page, device=DEVICE)
    seen = key[None, :] < s["lens"][:, None]
    if case["window"]:
        seen = seen & (key[None, :] >= s["lens"][:, None] - case["window"])

    def gathered(pool, scale):
        bits = pool.view(torch.uint8) if case["dtype"] == "f8" else pool
        x = bits[pages]  # [n, width, heads and slots, dim]
        x = x.transpose(2, 3) if case["order"] == "nhd" else x
        x = x.transpose(1, 2).reshape(n, kv, width * page, dim)
        x = x.view(TORCH["f8"]) if case["dtype"] == "f8" else x
        return x.float().masked_fill_(~seen[:, None, :, None], 0.0).mul_(scale)

    k_scale, v_scale = scales_of(case)
    q = s["q"].reshape(n, kv, group, dim)
    scores = torch.matmul(q, gathered(s["k_pool"], k_scale).transpose(2, 3)) / math.sqrt(dim)
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    most = scores.amax(-1, keepdim=True) if width else scores.new_full((n, kv, group, 1), -math.inf)
    most = torch.where(most == -math.inf, 0.0, most)
    p = torch.exp(scores - most)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, gathered(s["v_pool"], v_scale)) / torch.where(total == 0, 1.0, total)
    lse = (most + torch.log(total)).reshape(n, case["heads"])
    return dict(out=out.reshape(n, case["heads"] * dim), lse=lse)


def plain_score(s):
    case = s["case"]
    x, tokens = s["logits"], s["tokens"].long()
    given = x.gather(1, tokens[:, None])
    index = torch.arange(case["vocab"], device=DEVICE)
    rank = ((x > given) | ((x == given) & (index[None, :] < tokens[:, None]))).sum(1)
    y = x / case["temperature"]
    best = y.argmax(1, keepdim=True)
    y = y - y.gather(1, best)
    e = torch.exp(y)
    others = e.scatter(1, best, 0.0).sum(1, keepdim=True)  # without the largest, so that 1 + others does not round what is certain to 0
    logp = y - torch.log1p(others)
    entropy = torch.log1p(others) - torch.where(e > 0, e * y, 0.0).sum(1, keepdim=True) / (1 + others)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    return dict(logprob=logp.gather(1, tokens[:, None])[:, 0], entropy=entropy[:, 0], rank=rank.to(torch.int32), top_ids=ids.to(torch.int32),
                top_logprobs=logp.gather(1, ids))


# ---- 64 bits -----------------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    if case["op"] == "append":
        return exact_append(case, prepare_append(case, g))
    if case["op"] == "attend":
        return exact_attend(case, prepare_attend(case, g))
    return exact_score(case, prepare_score(case, g))


def exact_append(case, s):
    """The pairs as complex numbers, turned by exp(i * position * frequency)."""
    dim, rot, page = case["dim"], case["rot"], case["page"]
    scale, ext, attn, low, high = rope_settings(case)
    turn = torch.empty(rot // 2, dtype=torch.float64, device=DEVICE)
    for j in range(rot // 2):
        f = math.exp(-2.0 * j / rot * math.log(case["base"]))
        if ext:
            keep = ext * (1.0 - min(1.0, max(0.0, (j - low) / max(0.001, high - low))))
            f = f * scale + keep * (f - f * scale)
        turn[j] = f
    size = attn * (1.0 + 0.1 * math.log(1.0 / scale)) if ext else attn
    angle = torch.outer(s["positions"].double(), turn)
    z = torch.polar(torch.full_like(angle, size), angle)[:, None, :]

    def rotated(x, heads):
        x = x.double().reshape(-1, heads, dim)
        y = x.clone()
        one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if case["mode"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        w = torch.complex(x[..., one], x[..., two]) * z
        y[..., one], y[..., two] = w.real, w.imag
        return y

    live = (s["slots"] >= 0).nonzero()[:, 0]
    slot = s["slots"].long()[live]
    q = s["q_out"].double()
    q[live] = rotated(s["q"], case["heads"])[live].flatten(1)
    got = {"q": q}
    for name, x, unit in (("k", rotated(s["k"], case["kv_heads"]), scales_of(case)[0]),
                          ("v", s["v"].double().reshape(-1, case["kv_heads"], dim), scales_of(case)[1])):
        pool = torch.zeros(s["k_pool"].shape, dtype=torch.float64, device=DEVICE)
        if case["order"] == "hnd":
            pool[slot // page, :, slot % page] = x[live] / unit
        else:
            pool[slot // page, slot % page] = x[live] / unit
        got[name] = pool.clamp(-F8_MAX, F8_MAX) if case["dtype"] == "f8" else pool
    return got


def exact_attend(case, s):
    """Request by request: softmax over the keys that it sees."""
    page, kv, dim, heads = case["page"], case["kv_heads"], case["dim"], case["heads"]
    k_scale, v_scale = scales_of(case)
    out = torch.zeros((case["seqs"], heads, dim), dtype=torch.float64, device=DEVICE)
    lse = torch.full((case["seqs"], heads), -math.inf, dtype=torch.float64, device=DEVICE)
    lens = s["lens"].tolist()
    for i, n in enumerate(lens):
        begin = max(0, n - case["window"]) if case["window"] else 0
        if n == begin:
            continue
        t = torch.arange(begin, n, device=DEVICE)
        where = (s["table"][i, t // page].long(), t % page)

        def rows(pool):
            x = pool.view(torch.uint8) if case["dtype"] == "f8" else pool
            x = x[where[0], :, where[1]] if case["order"] == "hnd" else x[where[0], where[1]]
            return (x.view(TORCH["f8"]) if case["dtype"] == "f8" else x).double()

        k, v = rows(s["k_pool"]), rows(s["v_pool"])
        q = s["q"][i].double().reshape(kv, heads // kv, dim)
        sc = torch.einsum("hgd,thd->hgt", q, k) * (k_scale / math.sqrt(dim))
        norm = torch.logsumexp(sc, -1)
        out[i] = torch.einsum("hgt,thd->hgd", torch.exp(sc - norm[..., None]), v).reshape(heads, dim) * v_scale
        lse[i] = norm.reshape(heads)
    return {"out": out.reshape(case["seqs"], heads * dim), "lse": lse}


def exact_score(case, s):
    logprob, entropy, best = [], [], []
    for i in range(0, case["rows"], 256):
        x = s["logits"][i:i + 256].double() / case["temperature"]
        lp = torch.log_softmax(x, 1)
        logprob.append(lp.gather(1, s["tokens"][i:i + 256].long()[:, None])[:, 0])
        entropy.append(-(lp.exp() * lp.clamp(min=-1e4)).sum(1))
        best.append(lp.sort(1, descending=True).values[:, :case["top"]])
    return {"logprob": torch.cat(logprob), "entropy": torch.cat(entropy), "rank": None, "top_ids": None, "top_logprobs": torch.cat(best)}
