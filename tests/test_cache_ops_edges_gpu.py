"""Edges of the operators around a paged key/value cache on the GPU."""

import math

import pytest
import torch

from ninetoothed_amd import kernels

from test_cache_ops_gpu import (BF16, DEV, E4M3, F16, attended, attention_tol, caches, check_append, close, i32, paged,
                                randn, rotary_tol, run_append, starts_of, turned)

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


def test_rotary_of_more_tokens_than_one_launch_takes():
    # 2^32 threads and more: a grid of 2^24 workgroups of 256 takes 2^26 tokens
    tokens = (1 << 26) + 1027
    x = torch.empty(tokens, 1, 2, dtype=BF16, device=DEV)
    x[..., 0], x[..., 1] = 1.0, 0.5
    positions = torch.arange(tokens, dtype=torch.int32, device=DEV)
    freqs = torch.full((1,), 0.001, dtype=torch.float64, device=DEV)
    out = kernels.rotary(x, positions, freqs, torch.zeros_like(x))
    for part in (slice(0, 5000), slice((1 << 26) - 5000, tokens)):
        want, size = turned(x[part], positions[part], freqs, False)
        close(out[part], want, rotary_tol(want, size, BF16))
    assert (out != 0).any(-1).all()


def test_append_of_more_sequences_than_one_launch_takes():
    # 2^23 sequences have 2^24 workgroups kept for them; one token each, of which eight have a page
    tokens, dim = (1 << 23) + 77, 16
    kc, vc = (torch.zeros(8, 4, 1, dim, dtype=F16, device=DEV) for _ in range(2))
    tables = torch.full((tokens, 1), -1, dtype=torch.int32, device=DEV)
    tables[:4, 0], tables[-4:, 0] = torch.arange(4, device=DEV), torch.arange(4, 8, device=DEV)
    starts = torch.arange(tokens + 1, dtype=torch.int32, device=DEV)
    k = torch.arange(tokens, device=DEV).remainder(1009).to(F16)[:, None, None].expand(tokens, 1, dim)
    kernels.cache_append(k, -k, kc, vc, tables, torch.zeros_like(tables[:, 0]), starts)
    used = torch.cat([k[:4], k[-4:]])
    assert torch.equal(kc[:, 0], used) and torch.equal(vc[:, 0], -used) and (kc[:, 1:] == 0).all()


def test_append_of_more_pages_than_one_launch_takes():
    # pages of one slot: a workgroup each
    tokens, dim = (1 << 24) + 1027, 16
    kc, vc = (torch.zeros(tokens, 1, 1, dim, dtype=E4M3, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(tokens, 1, device=DEV) for _ in range(2))
    tables = torch.arange(tokens, dtype=torch.int32, device=DEV)[None]
    k = torch.exp2(torch.arange(tokens, device=DEV).remainder(13).float()).to(F16)[:, None, None].expand(tokens, 1, dim)
    kernels.cache_append(k, -k, kc, vc, tables, i32([0]), i32([0, tokens]), k_scale=ks, v_scale=vs)
    for c, s, sign in ((kc, ks, 1), (vc, vs, -1)):
        for a in range(0, tokens, 1 << 22):
            at = slice(a, a + (1 << 22))
            assert torch.equal(c[at, 0].float() * s[at][:, :, None] * sign, k[at].float())


def test_prompts_of_more_sequences_than_one_launch_takes():
    # one token each, so that each query's output is its value; 16 heads of 2^20 sequences are 2^24 workgroups
    sequences, heads, dim = (1 << 20) + 77, 16, 8
    v = (torch.arange(sequences * heads, device=DEV).remainder(2003).to(F16)).view(sequences, heads, 1).expand(-1, -1, dim)
    v = v.contiguous()
    q = torch.ones(sequences, heads, dim, dtype=F16, device=DEV)
    starts = torch.arange(sequences + 1, dtype=torch.int32, device=DEV)
    out = kernels.prompt_attention(q, q, v, torch.full_like(q, math.nan), starts, starts)
    assert torch.equal(out, v)


def test_joins_of_more_states_than_one_launch_takes():
    # 32,768 sequences of 512 heads: 2^24 workgroups; sequence 16,416 is split between two workgroups a head
    sequences, heads, dim, page = (1 << 15) + 64, 512, 16, 16
    few = 16
    q = randn(few, heads, dim, dtype=F16)
    kc, vc = caches((9, page, heads, dim), E4M3)
    ks, vs = (torch.full((9, heads), 2.0**-7, device=DEV) for _ in range(2))
    tables = torch.arange(9, dtype=torch.int32, device=DEV)[None]
    want = kernels.cache_attention(q, kc, vc, tables.expand(few, 9), i32([144] * few), torch.empty_like(q), ks, vs)
    lengths = torch.full((sequences,), 144, dtype=torch.int32, device=DEV)
    lengths[0] = 100  # (one block of 128 keys, the others two)
    many = q.repeat(sequences // few, 1, 1)
    out = kernels.cache_attention(many, kc, vc, tables.expand(sequences, 9), lengths, torch.full_like(many, math.nan), ks, vs)
    # either is off by its rounding and that of its weights, 2^-11 each, and by 2^-12 for its scores, of at most 3.5
    tol = 2 * (want.abs().double() * 2.0**-11 + 3.5 * (2.0**-11 + 2.0**-12 + 144 * 2.0**-25))
    err = (out.view(-1, few, heads, dim) - want).double().abs().view(sequences, heads, dim)[1:]
    assert (err <= tol.repeat(sequences // few, 1, 1)[1:]).all() and out[0].isfinite().all()


@pytest.mark.parametrize("cache", (F16, E4M3))
@pytest.mark.parametrize("dim,part", ((4, 4), (4, 2), (20, 16), (36, 36), (124, 2)))
def test_append_of_heads_of_whole_fours(dim, part, cache):
    run_append([33, 1, 70], [5, 31, 40], 32, 3, dim, part, F16, cache, interleaved=dim == 36)


@pytest.mark.parametrize("cache", (F16, E4M3))
@pytest.mark.parametrize("lengths,cached,page,heads,dim,part", (
    ([200, 128], [70, 0], 128, 2, 80, 40),  # 8-byte vectors, more of a page's items than its lanes hold
    ([40, 5, 1], [9, 17, 40], 32, 2, 48, 22),  # element by element, into pages that were begun
    ([90, 300], [31, 100], 128, 2, 128, 128),  # 16-byte vectors, four items a lane
))
def test_append_of_every_width(lengths, cached, page, heads, dim, part, cache):
    for dtype in (F16, BF16) if cache == E4M3 else (cache,):
        run_append(lengths, cached, page, heads, dim, part, dtype, cache, interleaved=part == 22)


@pytest.mark.parametrize("cache", (BF16, E4M3))
@pytest.mark.parametrize("which", ("elements", "tokens", "caches"))
def test_append_of_strided_and_unaligned_tensors(which, cache):
    # k and v every other element of a wider tensor, or one element behind 16 bytes; caches one element behind them
    lengths, cached, page, heads, dim = [100, 1, 60], [33, 15, 0], 64, 3, 64
    tables, pages = paged([n + c for n, c in zip(lengths, cached)], page)
    total = sum(lengths)
    kc, vc = caches((pages, page, heads, dim), cache)
    if which == "elements":
        k, v = (randn(total, heads, 2 * dim, dtype=BF16, seed=i)[..., ::2] for i in (1, 2))
    elif which == "tokens":
        k, v = (randn(total * heads * dim + 1, dtype=BF16, seed=i)[1:].view(total, heads, dim) for i in (1, 2))
    else:
        k, v = (randn(total, heads, dim, dtype=BF16, seed=i) for i in (1, 2))
        for i, c in enumerate((kc, vc)):
            moved = torch.zeros(c.numel() + 1, dtype=cache, device=DEV)[1:].view(c.shape)
            moved.copy_(c)
            kc, vc = (moved, vc) if i == 0 else (kc, moved)
    ks, vs = (torch.full((pages, heads), 2.0**-12, device=DEV) for _ in range(2)) if cache == E4M3 else (None, None)
    freqs = kernels.rotary_frequencies(dim)
    before = [None if t is None else t.clone() for t in (kc, vc, ks, vs)]
    kernels.cache_append(k, v, kc, vc, tables, i32(cached), starts_of(lengths), k_scale=ks, v_scale=vs, freqs=freqs)
    check_append(k, v, kc, vc, ks, vs, before, tables, cached, lengths, page, freqs, False)
