"""Edges of the operators of a layer's step over a paged cache on the GPU.

Tolerances are those of test_layer_ops_gpu, where the norm's sum of squares may have 256 terms a lane (rows of up to
65,536 elements in the form for any strides): with 6 steps over lanes and 4 over waves 266 roundings of 2^-24, half of
which reaches the root, and two more of fp32 in each of root, quotient and products: (133 + 8) 2^-24 < 2^-16.
"""

import math

import pytest
import torch

from ninetoothed_amd import kernels

from test_cache_ops_gpu import (BF16, DEV, E4M3, F16, F32, attended, caches, check_append, close, half_step, i32, paged, randn,
                                starts_of)
from test_layer_ops_gpu import Layer, check_linear, check_norm, weights

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("out", ("same", "row", 64))
@pytest.mark.parametrize("residual", (False, True))
@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("rows,dim,step", ((5, 64, 1), (4, 1024, 1), (3, 4096, 1), (2, 16384, 1), (1, 65536, 1), (3, 4096, 2)))
def test_norm_of_elements_whose_squares_pass_fp32(rows, dim, step, dtype, residual, out):
    # Sums of squares from 2^112 to 2^256, and (with an eps of zero) down to 2^-194.
    for power, eps in ((56, 1e-5), (58, 1e-5), (63, 1e-5), (64, 1e-5), (100, 1e-5), (120, 1e-5), (58, 0.0), (-40, 0.0), (-50, 0.0),
                       (-60, 1e-35), (-75, 0.0), (-100, 0.0)):
        x, weight = randn(rows, dim * step, dtype=dtype)[:, ::step].mul_(2.0**power), randn(dim, dtype=dtype, seed=1)
        r = randn(rows, dim, dtype=dtype, seed=2).mul_(2.0**power) if residual else None
        total = torch.full_like(r, math.nan) if residual else None
        y = torch.full((rows, dim), 7.0, device=DEV).to(dtype if out == "same" else E4M3)
        group = out if isinstance(out, int) else 0
        scale = None if out == "same" else torch.full((rows, dim // group) if group else (rows,), math.nan, device=DEV)
        kernels.rms_norm(x, weight, y, residual=r, total=total, scale=scale, eps=eps)
        check_norm(x, weight, y, r, total, scale, group, eps)


@pytest.mark.parametrize("dim", (128, 1000, 4096))
def test_norm_beside_rows_whose_squares_pass_fp32(dim):
    # ordinary rows keep their bits, whatever their neighbours hold; infinities and NaN as ever
    x, weight = randn(300, dim, dtype=BF16), randn(dim, dtype=BF16, seed=1)
    want = kernels.rms_norm(x, weight, torch.empty_like(x))
    odd = x.clone()
    odd[::3] *= 2.0**70
    odd[1, 3], odd[4, 5], odd[7, 0] = math.inf, math.nan, -math.inf
    odd[1, 9] = odd[4, 9] = 2.0**100
    got = kernels.rms_norm(odd, weight, torch.empty_like(x))
    keep = [i for i in range(300) if i % 3 and i not in (1, 4, 7)]
    assert torch.equal(got[keep], want[keep])
    check_norm(odd[::3], weight, got[::3], None, None, None, 0, 1e-6)
    assert got[4].isnan().all()
    for row, at in ((1, 3), (7, 0)):
        assert got[row, at].isnan() and (got[row, :at] == 0).all() and (got[row, at + 1:] == 0).all()


# -------------------------------------------------------------------------------------------- linear
def unaligned(t):
    return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)


@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("rows,n", ((2, 40), (20, 40), (90, 40), (130, 6400)))
def test_linear_of_infinite_x(rows, n, dtype, zeros):
    """A row with an infinity is NaN, whichever form the call's strides and sizes take; the other rows keep their bits."""
    k = 256
    weight, scales, z = weights(n, k, 64, dtype, zeros)
    x = randn(rows, k, dtype=dtype)
    odd = x.clone()
    odd[1, 7], odd[rows - 1, k - 1] = math.inf, -math.inf
    rest = [i for i in range(rows) if i not in (1, rows - 1)]
    for form in (lambda t: t, unaligned, lambda t: t.t().contiguous().t(), lambda t: t.repeat_interleave(2, 1)[:, ::2]):
        for w in (weight, weight.t().contiguous().t()):
            for c in (None, randn(rows, n, dtype=dtype, seed=4)):
                want = kernels.linear_4bit(form(x), w, scales, torch.empty(rows, n, dtype=dtype, device=DEV), zeros=z, c=c)
                got = kernels.linear_4bit(form(odd), w, scales, torch.empty_like(want), zeros=z, c=c)
                assert got[1].isnan().all() and got[rows - 1].isnan().all()
                assert torch.equal(got[rest], want[rest])
                check_linear(x, weight, scales, want, z, c)


@pytest.mark.parametrize("rows,k,n,group", ((9700, 4096, 128, 128), (4800, 1024, 512, 64), (1300, 1024, 1152, 32), (9601, 256, 100, 128),
                                            (1210, 384, 1030, 128), (4736, 128, 257, 32)))
def test_linear_of_many_rows_and_few_columns(rows, k, n, group):
    """As test_linear_of_many_rows, of up to 9 tiles of columns."""
    x, (weight, scales, z) = randn(rows, k, dtype=BF16), weights(n, k, group, BF16, True)
    for c in (None, randn(n, rows, dtype=BF16, seed=5).t()):
        out = torch.full((rows, n), math.nan, dtype=BF16, device=DEV)
        kernels.linear_4bit(x, weight, scales, out, zeros=z, c=c)
        check_linear(x, weight, scales, out, z, c, roundings=2 * group + 2 + k / group)


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


# ------------------------------------------------------------------------------------------ together
def prompts(cache, dtype, pages, width, pieces):
    """A layer with the prompts' pieces of three sequences in its cache, and a function that goes on from there."""
    layer = Layer(cache, dtype, pages)
    n, total = layer.heads * layer.dim, [sum(p[b] for p in pieces) for b in range(3)]
    x, r = ([randn(total[b], n, dtype=dtype, seed=s + b, scale=scale) for b in range(3)] for s, scale in ((0, 1.0), (10, 2.0)))
    tables, lengths, at = torch.arange(3 * width, device=DEV).view(3, width).to(torch.int32), i32([0, 0, 0]), [0, 0, 0]
    for rows in pieces:
        take = lambda t: torch.cat([t[b][at[b]:at[b] + m] for b, m in enumerate(rows)])  # noqa: E731
        positions = torch.cat([torch.arange(at[b], at[b] + m) for b, m in enumerate(rows)]).to(DEV)
        layer.step(layer.buffers(sum(rows)), take(x), take(r), tables, lengths, starts_of(rows), positions)
        at = [a + m for a, m in zip(at, rows)]
    return layer, tables, lengths, at


@pytest.mark.parametrize("cache,dtype", ((BF16, BF16), (F16, F16), (E4M3, BF16)))
def test_a_fork_gives_what_a_cache_of_its_own_gives(cache, dtype):
    """Sequence 1 forks, and both go on.  The fork shares its full pages and has a copy of the begun one, or has all of its
    pages to itself, filled byte for byte: the same bits.  Without the copy, or without the copied scales, others."""
    pages, width, page = 60, 12, Layer.page
    layer, tables, lengths, at = prompts(cache, dtype, pages, width, ([20, 33, 1], [60, 0, 7], [1, 40, 30]))
    full, begun = at[1] // page, at[1] % page
    assert full > 1 and 1 < begun < page - 3
    n, own = layer.heads * layer.dim, pages - 1
    held = [t.clone() for t in (*layer.caches, *layer.scales) if t is not None]
    new = [[randn(4, n, dtype=dtype, seed=50 + 2 * i + j, scale=1.0 + j) for j in range(2)] for i in range(3)]

    def go_on(how):
        for t, was in zip((*layer.caches, *layer.scales), held):
            t.copy_(was)
        fork = tables[1].clone()
        if how == "pages of its own":
            fork[:full + 1] = torch.arange(pages - full - 2, own, device=DEV)
            for t in (*layer.caches, *layer.scales):
                if t is not None:
                    t = t.view(torch.uint8) if t.dtype == E4M3 else t
                    t[fork[:full + 1].long()] = t[tables[1, :full + 1].long()]
        else:
            fork[full] = own
            if how != "no copy":
                kernels.cache_copy(*layer.caches, tables[1, full:full + 1].contiguous(), i32([own]), *layer.scales,
                                   counts=i32([begun]))
            if how == "no scales":
                for s in layer.scales:
                    s[own] = 1.0
        all_tables, all_lengths, got = torch.cat([tables, fork[None]]), torch.cat([lengths, lengths[1:2]]), []
        for x, r in new:
            b = layer.buffers(4)
            residual, up = layer.step(b, x, r.clone(), all_tables, all_lengths, starts_of([1] * 4), all_lengths.long())
            got += [residual, up, b["out"]]
        return got

    want = go_on("pages of its own")
    for a, b in zip(go_on("copy"), want):
        assert torch.equal(a, b)
    for how in ("no copy", "no scales") if layer.eight else ("no copy",):
        for a, b in zip(go_on(how), want):
            assert torch.equal(a[:3], b[:3]) and not torch.equal(a[3], b[3]), how


@pytest.mark.parametrize("cache,dtype", ((BF16, BF16), (F16, F16), (E4M3, BF16)))
def test_each_stage_of_a_layer(cache, dtype):
    """Each operator of a layer's step against 64 bits of what it was given, for a mix of pieces and single tokens."""
    pages, width = 40, 12
    layer, tables, lengths, at = prompts(cache, dtype, pages, width, ([20, 33, 1], [60, 0, 7]))
    n, kv, rows = layer.heads * layer.dim, layer.kv_heads * layer.dim, [1, 40, 30]
    b, starts = layer.buffers(sum(rows)), starts_of(rows)
    positions = torch.cat([torch.arange(a, a + m) for a, m in zip(at, rows)]).to(DEV)
    x, residual = randn(sum(rows), n, dtype=dtype, seed=3), randn(sum(rows), n, dtype=dtype, seed=4, scale=2.0)
    was = residual.clone()
    kernels.rms_norm(x, layer.norms[0], b["h"], residual=residual)
    check_norm(x, layer.norms[0], b["h"], was, residual, None, 0, 1e-6)
    kernels.linear_4bit(b["h"], *layer.qkv[:2], b["qkv"], zeros=layer.qkv[2])
    check_linear(b["h"], *layer.qkv[:2], b["qkv"], layer.qkv[2], None)
    q = b["qkv"][:, :n].view(-1, layer.heads, layer.dim)
    k, v = (b["qkv"][:, n + i * kv:n + (i + 1) * kv].view(-1, layer.kv_heads, layer.dim) for i in range(2))
    before = [None if t is None else t.clone() for t in (*layer.caches, *layer.scales)]
    kernels.rotary(q, positions, layer.freqs, q)
    kernels.cache_append(k, v, *layer.caches, tables, lengths, starts, *layer.scales, freqs=layer.freqs)
    check_append(k, v, *layer.caches, *layer.scales, before, tables, at, rows, layer.page, layer.freqs, False)
    lengths.add_(starts[1:] - starts[:-1])
    o = b["out"].view(-1, layer.heads, layer.dim)
    kernels.chunk_attention(q, *layer.caches, tables, lengths, starts, o, *layer.scales)
    weight_type, first = F16 if layer.eight else dtype, 0
    for s, (a, m) in enumerate(zip(at, rows)):
        held = tables[s].long()
        kk, vv = ((c.double() * (1.0 if e is None else e.double()[:, None, :, None]))[held].flatten(0, 1)[:a + m]
                  for c, e in zip(layer.caches, layer.scales))
        for h in range(layer.heads):
            g = h // (layer.heads // layer.kv_heads)
            want, size = attended(q[first:first + m, h], kk[:, g], vv[:, g], layer.dim**-0.5, torch.arange(a, a + m, device=DEV))
            tol = half_step(dtype) * want.abs() + half_step(weight_type) * (want.abs() + size) + 2.0**-12 * size
            close(o[first:first + m, h], want, tol + (a + m) * 2.0**-25 * float(vv.abs().max()) + 1e-30, f"sequence {s}, head {h}")
        first += m
    was = residual.clone()
    kernels.linear_4bit(b["out"], *layer.o[:2], residual, zeros=layer.o[2], c=residual)
    check_linear(b["out"], *layer.o[:2], residual, layer.o[2], was)
    kernels.rms_norm(residual, layer.norms[1], b["y"], scale=b["scale"])
    check_norm(residual, layer.norms[1], b["y"], None, None, b["scale"], 0, 1e-6)
    kernels.gemm(b["y"], layer.up, b["up"])
    y, up = b["y"].double(), layer.up.double()
    # (sums of n products in fp32, twice the roundings for the matrix core's order, and one rounding to fp16)
    tol = (y @ up).abs() * 2.0**-11 + y.abs() @ up.abs() * n * 2.0**-23 + 2.0**-25
    close(b["up"], y @ up, tol, "up")


# --------------------------------------------------------------------------------------------- large
def test_norm_past_32_bits():
    rows, dim = 540_000, 4096  # x, residual and output of 4.4 GB each
    x = torch.empty(rows, dim, dtype=BF16, device=DEV).normal_()
    r, weight, out = x.flip(1), randn(dim, dtype=BF16, seed=1), torch.empty_like(x)
    tail = [t[-50:].clone() for t in (x, r)]
    kernels.rms_norm(x, weight, out, residual=r)
    check_norm(tail[0], weight, out[-50:], tail[1], r[-50:], None, 0, 1e-6)
    scale, y = torch.empty(rows, dim // 32, device=DEV), torch.empty(rows, dim, dtype=E4M3, device=DEV)
    kernels.rms_norm(x, weight, y, scale=scale)
    check_norm(x[-50:], weight, y[-50:], None, None, scale[-50:], 32, 1e-6)
    columns = x.view(dim, rows).t()  # (the form for any strides)
    kernels.rms_norm(columns, weight, r)
    check_norm(columns[-50:], weight, r[-50:], None, None, None, 0, 1e-6)


@pytest.mark.parametrize("rows,k,n", ((540_000, 4096, 64), (300_000, 64, 8192), (3, 8192, 1_100_000), (70, 8192, 1_100_000)))
def test_linear_past_32_bits(rows, k, n):
    # x, the output, or the weights, of more than 4 GB
    x, (weight, scales, z) = torch.empty(rows, k, dtype=BF16, device=DEV).normal_(), weights(32, k, 32, BF16, True)
    weight, scales, z = (t.repeat(-(-n // 32), 1)[:n] for t in (weight, scales, z))
    out = torch.full((rows, n), math.nan, dtype=BF16, device=DEV)
    kernels.linear_4bit(x, weight, scales, out, zeros=z)
    for at in (slice(0, 3), slice(rows - 3, rows)):
        for cols in (slice(0, 40), slice(n - 40, n)):
            check_linear(x[at], weight[cols], scales[cols], out[at, cols], z[cols], None, roundings=2 * 32 + 2 + k / 32)


def test_chunk_past_32_bits():
    tokens, heads, kv_heads, dim = 540_000, 32, 8, 128  # q and out of 4.4 GB
    q = torch.empty(tokens, heads, dim, dtype=BF16, device=DEV).normal_()
    kc, vc = caches((6, 32, kv_heads, dim), BF16)
    tables, keys, starts = i32([[0, 1, 2], [3, 4, 5]]), [70, 90], i32([0, tokens - 100, tokens])
    out = torch.full_like(q, math.nan)
    kernels.chunk_attention(q, kc, vc, tables, i32(keys), starts, out, causal=False)
    for b, rows in ((0, slice(tokens - 150, tokens - 100)), (1, slice(tokens - 100, tokens))):
        for head in (0, 13, 31):
            kk, vv = (c[tables[b].long(), :, head // 4].flatten(0, 1)[:keys[b]] for c in (kc, vc))
            want, size = attended(q[rows, head], kk, vv, dim**-0.5)
            tol = half_step(BF16) * (2 * want.abs() + size) + 2.0**-12 * size
            close(out[rows, head], want, tol + keys[b] * 2.0**-25 * float(vv.abs().max()) + 1e-30)


# --------------------------------------------------------------------------------------- other calls
@pytest.mark.parametrize("cache", (F16, E4M3))
@pytest.mark.parametrize("heads,kv_heads", ((300, 1), (3, 3), (64, 2)))
def test_chunk_of_wide_groups_and_shared_pages(heads, kv_heads, cache):
    """More heads of q to one of k than a block has rows; tables that share pages, among them one row for all sequences."""
    for dim, page in ((16, 16), (48, 24), (128, 128)):
        new, keys = [2, 0, 5, 1], [150, 9, 200, 40]
        kc, vc = caches((9, page, kv_heads, dim), cache)
        ks, vs = ((torch.full((9, kv_heads), 2.0**-7, device=DEV) for _ in range(2)) if cache == E4M3 else (None, None))
        q = randn(8, heads, dim, dtype=F16)
        row = (torch.arange(14, device=DEV) % 9).to(torch.int32)
        outs = [kernels.chunk_attention(q, kc, vc, t, i32(keys), starts_of(new), torch.empty_like(q), ks, vs)
                for t in (row.expand(4, 14), row.repeat(4, 1), torch.stack([row] * 8)[::2])]
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        first = 0
        for m, n in zip(new, keys):
            last = torch.arange(n - m, n, device=DEV)
            for head in range(0, heads, 7):
                h = head // (heads // kv_heads)
                kk, vv = ((c[row.long(), :, h].double() * (1.0 if s is None else s[0, 0].double())).flatten(0, 1)[:n]
                          for c, s in ((kc, ks), (vc, vs)))
                want, size = attended(q[first:first + m, head], kk, vv, dim**-0.5, last)
                tol = half_step(F16) * (2 * want.abs() + size) + 2.0**-12 * size
                close(outs[0][first:first + m, head], want, tol + n * 2.0**-25 * float(vv.abs().max()) + 1e-30)
            first += m


@pytest.mark.parametrize("cache", (BF16, E4M3))
def test_a_captured_chunk_replays_with_other_lengths(cache):
    """A padded batch: sequences, tables and lengths change between the replays, and the rows behind the last one stay."""
    q, (kc, vc) = randn(60, 8, 64, dtype=BF16), caches((200, 16, 2, 64), cache)
    scales = [torch.full((200, 2), 2.0**-6, device=DEV) for _ in range(2)] if cache == E4M3 else [None, None]
    order = torch.randperm(200, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    tables, lengths, starts, out = torch.zeros(4, 50, dtype=torch.int32, device=DEV), i32([0] * 4), i32([0] * 5), torch.zeros_like(q)
    steps = (([5, 1, 0, 40], [100, 800, 0, 77]), ([1, 1, 1, 1], [700, 3, 9, 50]), ([0, 0, 0, 0], [4, 4, 4, 4]),
             ([60, 0, 0, 0], [790, 0, 0, 0]), ([1, 30, 2, 1], [-1, 31, 600, 1]))
    call = lambda o: kernels.chunk_attention(q, kc, vc, tables, lengths, starts, o, *scales)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(torch.zeros_like(q))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for i, (new, keys) in enumerate(steps * 2):
        tables.copy_(order.roll(i).view(4, 50))
        lengths.copy_(i32(keys))
        starts.copy_(starts_of(new))
        want = call(torch.full_like(q, 7.0))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (out[sum(new):] == 7).all()
