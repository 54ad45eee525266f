"""Edges of the operators around a paged key/value cache on the GPU."""

import math

import pytest
import torch

from ninetoothed_amd import kernels

from test_cache_ops_gpu import BF16, DEV, E4M3, F16, attended, attention_tol, caches, close, i32, randn, starts_of

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


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("dim", (64, 128, 30))
def test_keys_of_no_weight_come_first(dim, dtype, causal):
    # The first keys of a sequence score minus infinity, and what comes behind them far below zero.
    lengths, none = [300, 70, 40], 70
    starts = starts_of(lengths)
    total = sum(lengths)
    q = randn(total, 4, dim, dtype=dtype)
    k, v = randn(total, 2, dim, dtype=dtype, seed=1), randn(total, 2, dim, dtype=dtype, seed=2)
    q[..., 0], q[..., 1] = 1.0, 8.0
    k[..., 1] = -100.0 * (dim / 64) ** 0.5  # scores of about -100
    for a in starts[:-1].tolist():
        k[a:a + none, :, 0] = -math.inf
    out = kernels.prompt_attention(q, k, v, torch.full_like(q, math.nan), starts, starts, causal=causal)
    for a, n in zip(starts.tolist(), lengths):
        last = torch.arange(n, device=DEV) if causal else None
        for h in range(4):
            o, size = attended(q[a:a + n, h], k[a:a + n, h // 2], v[a:a + n, h // 2], dim**-0.5, last)
            # (dim sums of less than 2,048 in 32 bits, rounded by 2^-14 at most, times the scale: the scores are off by
            # less than 2^-10, and the weights and their sum by as much)
            close(out[a:a + n, h], o, attention_tol(o, size, dtype, n, 5.0) + 2.0**-9 * size, f"{n} keys, head {h}")
    assert (out[starts[2]:] == 0).all()  # (nothing but keys of no weight)
