"""Edges of the operators of a layer's step over a paged cache on the GPU.

Tolerances are those of test_layer_ops_gpu, where the norm's sum of squares may have 256 terms a lane (rows of up to
65,536 elements in the form for any strides): with 6 steps over lanes and 4 over waves 266 roundings of 2^-24, half of
which reaches the root, and two more of fp32 in each of root, quotient and products: (133 + 8) 2^-24 < 2^-16.
"""

import math

import pytest
import torch

from ninetoothed_amd import kernels

from test_cache_ops_gpu import BF16, DEV, E4M3, F16, caches, i32, paged, randn

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------------------------- chunk
@pytest.mark.parametrize("cache", (F16, E4M3))
@pytest.mark.parametrize("tokens", (1, 300, 2000))
def test_chunk_of_many_tokens_without_keys(tokens, cache):
    # a cache without pages, or tables without room, at any number of tokens: zeros
    q, (kc, vc) = randn(tokens + 2, 8, 64), caches((4, 32, 2, 64), cache)
    scales = [torch.ones(4, 2, device=DEV) for _ in range(2)] if cache == E4M3 else [None, None]
    tables, lengths, starts = i32([[0, 1], [2, 3]]), i32([9, 40]), i32([0, tokens // 3, tokens])
    for pages, t in ((0, tables), (4, tables[:, :0])):
        out = torch.full_like(q, 7.0)
        kernels.chunk_attention(q, kc[:pages], vc[:pages], t, lengths, starts, out,
                                *(s if s is None else s[:pages] for s in scales))
        assert (out[:tokens] == 0).all() and (out[tokens:] == 7).all()


@pytest.mark.parametrize("page", (16, 24))
def test_chunk_a_v_scale_of_zero_holds_nothing(page):
    # ... whatever its values are, and whether or not a masked NaN elsewhere has the rows taken key by key
    tables, pages = paged([110], page)
    kc, vc = caches((pages, page, 2, 64), E4M3)
    ks, vs = (torch.full((pages, 2), 2.0**-6, device=DEV) for _ in range(2))
    q, starts, at = randn(60, 4, 64, dtype=BF16), i32([0, 60]), lambda key: (int(tables[0, key // page]), key % page)
    vs[at(page)[0]] = 0.0
    vc[at(100) + (0, 5)] = math.nan
    outs = []
    for value in (1.0, math.nan):
        vc[at(page + 3) + (0, 9)] = value
        outs.append(kernels.chunk_attention(q, kc, vc, tables, i32([110]), starts, torch.empty_like(q), ks, vs))
    seen = 100 - (110 - 60)  # the first query that sees key 100
    assert outs[0][:seen].isfinite().all() and outs[0][seen:, :2, 5].isnan().all()
    assert torch.equal(outs[0].nan_to_num(), outs[1].nan_to_num())
