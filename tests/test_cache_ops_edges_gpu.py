"""Edges of the operators around a paged key/value cache on the GPU."""

import math

import pytest
import torch

from ninetoothed_amd import kernels

from test_cache_ops_gpu import BF16, DEV, E4M3, F16, caches, i32, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", (math.inf, math.nan))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("page", (16, 32, 24))
def test_a_missing_page_takes_no_scale(page, dim, odd):
    # Page 0 holds no sequence, so its scales may hold anything; pages that are missing have none.
    heads, kv_heads, pages = 4, 2, 14
    q = randn(3, heads, dim, dtype=BF16)
    kc, vc = caches((pages, page, kv_heads, dim), E4M3)
    tables = i32([[1, -1, 2, 3, 1 << 30], [4, 5, 6, pages, 7], [-1, -1, -1, -1, -1]])
    lengths = i32([5 * page - 3, 4 * page, 2 * page])
    outs = []
    for first in (1.0, odd):
        ks, vs = (torch.full((pages, kv_heads), 2.0**-6, device=DEV) for _ in range(2))
        ks[0], vs[0] = first, first
        outs.append(kernels.cache_attention(q, kc, vc, tables, lengths, torch.full_like(q, math.nan), ks, vs))
    assert outs[0].isfinite().all() and (outs[0][2] == 0).all() and torch.equal(outs[0], outs[1])
