"""Refusals of the paged-cache and log-probability entry points: arguments are checked on the host before any
CUDA call, so these run without a device."""
from __future__ import annotations

import ctypes as C

import pytest

from muyo_llm_b200 import _abi, build, nodes

EINVAL, EUNSUPPORTED = -1, -5
A = 4096  # a non-null, aligned stand-in for a device address; a refused call never reads it


@pytest.fixture(scope="module")
def lib():
    build()
    return _abi.lib()


def refused(rc_expected, fn, p, *args, match):
    rc = getattr(_abi.lib(), fn)(None if p is None else C.byref(p), *args)
    assert rc == rc_expected, (fn, rc, _abi.last_error())
    assert match in _abi.last_error(), _abi.last_error()


def cache(**kw):
    kw = {**dict(page_size=16, num_pages=64), **kw}
    heads, kv, hd = kw.pop("heads", 14), kw.pop("kv_heads", 2), kw.pop("head_dim", 64)
    return nodes.paged_cache_params(heads, kv, hd, **kw)


BAD_CACHES = [
    (EINVAL, dict(heads=14, kv_heads=3), "multiple of kv_heads"),
    (EINVAL, dict(heads=0), "positive multiple"),
    (EINVAL, dict(heads=34, kv_heads=2), "16 query heads"),
    (EUNSUPPORTED, dict(head_dim=48), "head_dim 48"),
    (EUNSUPPORTED, dict(head_dim=256), "head_dim 256"),
    (EINVAL, dict(kv_dtype=3), "kv_dtype 3"),
    (EINVAL, dict(page_size=0, page_stride=64, head_stride=64, slot_stride=64), "page_size"),
    (EINVAL, dict(num_pages=0), "num_pages"),
    (EINVAL, dict(page_size=1 << 16, num_pages=1 << 15), "INT32_MAX"),
    (EINVAL, dict(k_scale=-1.0), "k_scale"),
    (EINVAL, dict(v_scale=float("inf")), "v_scale"),
    (EINVAL, dict(k_scale=2.0 ** -101), "k_scale"),
    (EINVAL, dict(v_scale=2.0 ** 101), "v_scale"),
    (EINVAL, dict(page_stride=64, head_stride=64, slot_stride=32), "below head_dim"),
    (EINVAL, dict(page_stride=4096), "below head_dim"),  # all three strides or none
    (EINVAL, dict(page_stride=4100, head_stride=64, slot_stride=64), "16 bytes"),
    (EINVAL, dict(page_stride=1 << 45, head_stride=64, slot_stride=64), "too large"),
]


@pytest.mark.parametrize("rc,kw,match", BAD_CACHES)
def test_bad_caches(lib, rc, kw, match):
    p = nodes.paged_attention_params(cache(**kw), 4, table_stride=8)
    refused(rc, "muyo_cuda_paged_attention_decode", p, A, A, A, A, A, A, None, A, 1 << 30, None, match=match)
    assert lib.muyo_cuda_paged_attention_workspace_size(C.byref(p)) == 0
    p = nodes.paged_append_params(cache(**kw), 4, n_dims=0)
    refused(rc, "muyo_cuda_paged_rope_append", p, A, A, A, A, A, A, A, A, A, None, match=match)


def attention(**kw):
    p = nodes.paged_attention_params(cache(), 4, table_stride=8)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,match", [
    (dict(seqs=0), "seqs"), (dict(seqs=1 << 31), "seqs"), (dict(seqs=(1 << 28) + 1), "seqs"), (dict(table_stride=0), "table_stride"),
    (dict(table_stride=1 << 28), "2^30"), (dict(window=1 << 31), "window"), (dict(scale=float("nan")), "scale"),
    (dict(stride_q=892), "row stride"), (dict(stride_out=892), "row stride"), (dict(stride_q=898), "multiples of 4"),
])
def test_attention_refuses(lib, kw, match):
    refused(EINVAL, "muyo_cuda_paged_attention_decode", attention(**kw), A, A, A, A, A, A, None, A, 1 << 30, None, match=match)


def test_attention_refuses_buffers(lib):
    fn = "muyo_cuda_paged_attention_decode"
    refused(EINVAL, fn, None, A, A, A, A, A, A, None, A, 1 << 30, None, match="null parameter")
    for i in range(6):
        args = [A] * 6
        args[i] = None
        refused(EINVAL, fn, attention(), *args, None, A, 1 << 30, None, match="null buffer")
    for i in (0, 1, 2, 5):
        args = [A] * 6
        args[i] = A + 8
        refused(EINVAL, fn, attention(), *args, None, A, 1 << 30, None, match="16-byte aligned")
    refused(EINVAL, fn, attention(), A, A, A, A, A, A, None, None, 1 << 30, None, match="workspace")
    need = lib.muyo_cuda_paged_attention_workspace_size(C.byref(attention()))
    assert need > 0
    refused(EINVAL, fn, attention(), A, A, A, A, A, A, None, A, need - 1, None, match="workspace of")
    refused(EINVAL, fn, attention(), A, A, A, A, A, A, None, A + 4, 1 << 30, None, match="workspace must be")


def append(**kw):
    p = nodes.paged_append_params(cache(), 4)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,match", [
    (dict(rope_mode=8), "rope mode"), (dict(n_dims=63), "even"), (dict(n_dims=66), "even"), (dict(n_offs=2), "even"),
    (dict(n_dims=32, n_offs=34), "even"), (dict(n_dims=32, n_offs=1), "even"), (dict(tokens=1 << 31), "tokens"),
    (dict(stride_q=890), "row stride"), (dict(stride_k=64), "row stride"), (dict(stride_v=130), "multiples of 4"),
    (dict(stride_q_out=64), "row stride"),
])
def test_append_refuses(lib, kw, match):
    refused(EINVAL, "muyo_cuda_paged_rope_append", append(**kw), A, A, A, A, A, A, 2 * A, A, A, None, match=match)


def test_append_refuses_buffers(lib):
    fn = "muyo_cuda_paged_rope_append"
    refused(EINVAL, fn, None, A, A, A, A, A, A, A, A, A, None, match="null parameter")
    for i in (1, 2, 3, 4, 7, 8):
        args = [A] * 9
        args[i] = None
        refused(EINVAL, fn, append(), *args, None, match="null buffer")
    refused(EINVAL, fn, append(), A, A, A, A, A, None, A, A, A, None, match="freqs are needed")
    refused(EINVAL, fn, append(), A, A, A, A, A, A, None, A, A, None, match="q without q_out")
    refused(EINVAL, fn, append(), A, A, A, A, A, A + 4, A, A, A, None, match="8-byte")
    refused(EINVAL, fn, append(), A, A + 4, A, A, A, A, A, A, A, None, match="16-byte")
    refused(EINVAL, fn, append(stride_q=1152), A, A, A, A, A, A, A, A, A, None, match="equal strides")
    assert lib.muyo_cuda_paged_rope_append(C.byref(append(tokens=0)), A, A, A, A, A, A, A, A, A, None) == 0  # nothing to do


@pytest.mark.parametrize("rc,kw,match", [
    (EINVAL, dict(seqs=0), "seqs"), (EUNSUPPORTED, dict(seqs=8193), "8192"), (EINVAL, dict(page_size=0), "page_size"),
    (EINVAL, dict(num_pages=0), "num_pages"), (EINVAL, dict(table_stride=0), "table_stride"),
    (EINVAL, dict(num_pages=1 << 28), "INT32_MAX"), (EINVAL, dict(table_stride=1 << 28), "2^30"),
    (EINVAL, dict(max_tokens=(1 << 31) - 1), "max_tokens"),
])
def test_plan_refuses(lib, rc, kw, match):
    p = nodes.paged_plan_params(4, page_size=16, num_pages=64, table_stride=8, max_tokens=32)
    for k, v in kw.items():
        setattr(p, k, v)
    refused(rc, "muyo_cuda_paged_plan", p, *[A] * 10, None, match=match)


def test_plan_refuses_buffers(lib):
    fn = "muyo_cuda_paged_plan"
    p = nodes.paged_plan_params(4, page_size=16, num_pages=64, table_stride=8, max_tokens=32)
    refused(EINVAL, fn, None, *[A] * 10, None, match="null parameter")
    for i in range(10):
        args = [A] * 10
        args[i] = None
        refused(EINVAL, fn, p, *args, None, match="positions and slots" if i in (7, 8) else "null buffer")
    for i in (4, 9):
        args = [A] * 10
        args[i] = A + 4
        refused(EINVAL, fn, p, *args, None, match="8-byte")


@pytest.mark.parametrize("kw,match", [
    (dict(n_dims=0), "n_dims"), (dict(n_dims=7), "n_dims"), (dict(freq_base=0.0), "freq_base"),
    (dict(ext_factor=1.0, freq_scale=0.0), "freq_scale"), (dict(has_ff=1), "freq_factors"),
])
def test_frequencies_refuse(lib, kw, match):
    p = nodes.rope_params(1, 64)
    for k, v in kw.items():
        setattr(p, k, v)
    refused(EINVAL, "muyo_cuda_rope_frequencies", p, None, A, None, match=match)


def test_frequencies_refuse_buffers(lib):
    refused(EINVAL, "muyo_cuda_rope_frequencies", None, None, A, None, match="null")
    refused(EINVAL, "muyo_cuda_rope_frequencies", nodes.rope_params(1, 64), None, None, None, match="null")
    refused(EINVAL, "muyo_cuda_rope_frequencies", nodes.rope_params(1, 64), None, A + 4, None, match="8-byte")


@pytest.mark.parametrize("kw,match", [
    (dict(rows=0), "rows"), (dict(rows=1 << 31), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 28) + 1), "vocab"),
    (dict(stride=99), "stride"), (dict(top_k=33), "top_k"), (dict(vocab=5, top_k=6), "top_k"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
])
def test_token_logprobs_refuse(lib, kw, match):
    p = nodes.token_logprobs_params(4, 100, top_k=2)
    for k, v in kw.items():
        setattr(p, k, v)
    refused(EINVAL, "muyo_cuda_token_logprobs", p, *[A] * 8, 1 << 30, None, match=match)
    assert lib.muyo_cuda_token_logprobs_workspace_size(C.byref(p)) == 0


def test_token_logprobs_refuse_buffers(lib):
    fn = "muyo_cuda_token_logprobs"
    p = nodes.token_logprobs_params(4, 100, top_k=2)
    refused(EINVAL, fn, None, *[A] * 8, 1 << 30, None, match="null parameter")
    for i in range(3):
        args = [A] * 8
        args[i] = None
        refused(EINVAL, fn, p, *args, 1 << 30, None, match="null buffer")
    for i in (5, 6):
        args = [A] * 8
        args[i] = None
        refused(EINVAL, fn, p, *args, 1 << 30, None, match="top_ids")
    need = lib.muyo_cuda_token_logprobs_workspace_size(C.byref(p))
    refused(EINVAL, fn, p, *[A] * 8, need - 1, None, match="workspace of")
    refused(EINVAL, fn, p, *[A] * 7, A + 4, 1 << 30, None, match="workspace must be")
    refused(EINVAL, fn, p, A + 2, *[A] * 7, 1 << 30, None, match="4-byte")


def test_orders_of_a_pool():
    hnd, nhd = cache(), cache(order="nhd")
    assert (hnd.page_stride, hnd.head_stride, hnd.slot_stride) == (2 * 16 * 64, 16 * 64, 64)
    assert (nhd.page_stride, nhd.head_stride, nhd.slot_stride) == (2 * 16 * 64, 64, 2 * 64)
    with pytest.raises(ValueError):
        cache(order="dnh")
