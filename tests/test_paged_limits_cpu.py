"""Refusals of the paged-cache entry points at the ends of their ranges, before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

from muyo_llm_b200 import _abi, nodes
from test_paged_cpu import EINVAL, EUNSUPPORTED, A, cache, lib, refused  # noqa: F401


def test_plan_refuses_unknown_flags(lib):  # noqa: F811
    p = nodes.paged_plan_params(4, page_size=16, num_pages=64, table_stride=8, max_tokens=32, flags=2)
    refused(EINVAL, "muyo_cuda_paged_plan", p, *[A] * 10, None, match="flags")
