"""Refusals of the paged-cache entry points at the ends of their ranges, before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

from muyo_llm_b200 import _abi, nodes
from test_paged_cpu import EINVAL, EUNSUPPORTED, A, cache, lib, refused  # noqa: F401


def test_plan_refuses_unknown_flags(lib):  # noqa: F811
    p = nodes.paged_plan_params(4, page_size=16, num_pages=64, table_stride=8, max_tokens=32, flags=2)
    refused(EINVAL, "muyo_cuda_paged_plan", p, *[A] * 10, None, match="flags")


@pytest.mark.parametrize("scale,k_scale", [(1e30, 2.0 ** 100), (-3e38, 2.0), (3e38, 1.0)])
def test_attention_refuses_scales_whose_product_overflows(lib, scale, k_scale):  # noqa: F811
    """Each is in its range, but scores are scaled by both (and by log2 e): an infinite factor would give NaN."""
    p = nodes.paged_attention_params(cache(kv_dtype=_abi.KV_F8, k_scale=k_scale), 4, table_stride=8, scale=scale)
    refused(EINVAL, "muyo_cuda_paged_attention_decode", p, A, A, A, A, A, A, None, A, 1 << 30, None, match="scale")
    assert lib.muyo_cuda_paged_attention_workspace_size(C.byref(p)) == 0


@pytest.mark.parametrize("heads,page,width,seqs", [(1, 25, 38177487, 18), (1, 1 << 20, 1 << 10, 16)])
def test_attention_refuses_more_tiles_than_a_count_holds(lib, heads, page, width, seqs):  # noqa: F811
    """2^31 - 2 tiles fit the count, but not what is added to it to round up to whole CTAs."""
    p = nodes.paged_attention_params(cache(heads=heads, kv_heads=1, page_size=page, num_pages=4), seqs, table_stride=width)
    refused(EUNSUPPORTED, "muyo_cuda_paged_attention_decode", p, A, A, A, A, A, A, None, A, 1 << 30, None, match="tiles")
    assert lib.muyo_cuda_paged_attention_workspace_size(C.byref(p)) == 0
