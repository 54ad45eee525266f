"""The operators of a layer's step over a paged cache on the GPU (norm, products with 4-bit weights, attention of
chunks, page copies), against plain forms in 64 bits.

Tolerances, from the arithmetic (e: the type's half step, finfo.eps / 2):
- norm: the sum of squares is off by less than 150 roundings of fp32 (128 terms a lane at most, 16 steps over lanes
  and waves), half of which reaches its root; with the root, quotient and products less than 2^-16 of y, and one
  rounding of the output.  Of 8 bits half a step of e4m3, 2^-4 of the value or 2^-10, on y / scale; scales within 2^-15.
- products with 4-bit weights: fp32 sums of at most `group` products each (exact, twice the roundings allowed for the
  matrix core's order), and of groups / 8 of them and 16 more: 2^-23 (group + groups / 8 + 16) times
  sum s |x| (16 + q + 16 + z); one rounding of the output.
- attention of chunks: as prompt attention (test_cache_ops_gpu), with weights in fp16 for 8 bits.
- copies: equal.
"""

import math

import pytest
import torch

from ninetoothed_amd import kernels

from test_cache_ops_gpu import (BF16, DEV, E4M3, F16, F32, attended, caches, close, e4m3_tol, half_step, i32, paged, randn,
                                starts_of)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- norm
def check_norm(x, weight, out, residual, total, scale, group, eps):
    s = x.double() if residual is None else x.double() + residual.double()
    if residual is not None:
        close(total, s, s.abs() * (half_step(x.dtype) + 2.0**-23) + (2.0**-25 if x.dtype == F16 else 0), "total")
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double()
    if scale is None:
        close(out, y, y.abs() * (half_step(x.dtype) + 2.0**-16) + (2.0**-25 if x.dtype == F16 else 0) + 1e-38, "out")
        return
    parts = y.unflatten(-1, (-1, group)) if group else y[:, None]
    largest = torch.where(parts.isfinite(), parts.abs(), 0.0).amax(-1).view(scale.shape)
    want = (largest / 448).clamp_min(2.0**-64)
    close(scale, want, want * 2.0**-15, "scale")
    q = (parts / scale.double().view(parts.shape[:2])[..., None]).view_as(y)
    close(out.double(), q, e4m3_tol(q) + q.abs() * 2.0**-15, "out")


@pytest.mark.parametrize("residual", (False, True))
@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("rows,dim,out", [
    (rows, dim, out) for rows, dim in (
        (1, 1), (3, 7), (1, 8), (5, 64), (700, 128), (2, 200), (9, 520), (5000, 384), (33, 1024), (7, 2048), (3, 4096), (2, 5120),
        (4, 8192), (1, 8320), (2, 16384), (1, 32768), (2, 65536), (3, 65535), (0, 64))
    for out in ("same", "row", 32, 64, 128) if not isinstance(out, int) or dim % out == 0])
def test_norm(rows, dim, dtype, out, residual):
    group = out if isinstance(out, int) else 0
    x, weight = randn(rows, dim, dtype=dtype), randn(dim, dtype=dtype, seed=1)
    r = randn(rows, dim, dtype=dtype, seed=2, scale=4.0) if residual else None
    total = torch.full_like(x, math.nan) if residual else None
    eight = out != "same"
    y = torch.full((rows, dim), 7.0, device=DEV).to(E4M3 if eight else dtype)
    scale = torch.full((rows, dim // group) if group else (rows,), math.nan, device=DEV) if eight else None
    got = kernels.rms_norm(x, weight, y, residual=r, total=total, scale=scale, eps=1e-5)
    assert got is y
    check_norm(x, weight, y, r, total, scale, group, 1e-5)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("dim", (96, 1000, 4096, 9000, 1001))
def test_norm_in_place(dim, dtype):
    x, weight, r = randn(37, dim, dtype=dtype), randn(dim, dtype=dtype, seed=1), randn(37, dim, dtype=dtype, seed=2)
    want, total = torch.empty_like(x), torch.empty_like(x)
    kernels.rms_norm(x, weight, want, residual=r, total=total)
    for into_x in (False, True):  # the sum into the residual (the default) or into x, the norm into x
        a, b = x.clone(), r.clone()
        out = torch.empty_like(x) if into_x else a
        kernels.rms_norm(a, weight, out, residual=b, total=a if into_x else None)
        assert torch.equal(out, want) and torch.equal(a if into_x else b, total)
    a = x.clone()
    assert torch.equal(kernels.rms_norm(a, weight, a), kernels.rms_norm(x, weight, torch.empty_like(x)))


@pytest.mark.parametrize("eight", (0, "row", 64))
@pytest.mark.parametrize("dtype", (F32, F16, BF16))
def test_norm_strides(dtype, eight):
    dim = 192

    def made(i, how):
        if how == "rows":  # of a wider tensor
            return randn(21, 640, dtype=dtype, seed=i)[:, 64:64 + dim]
        if how == "unaligned":
            return randn(21 * dim + 1, dtype=dtype, seed=i)[1:].view(21, dim)
        if how == "every":
            return randn(21, 2 * dim, dtype=dtype, seed=i)[:, ::2]
        return randn(dim, 21, dtype=dtype, seed=i).t()

    for how in ("rows", "unaligned", "every", "columns"):
        x, r, total = made(0, how), made(1, how), made(2, how)
        weight = randn(2 * dim, dtype=dtype, seed=3)[::2] if how != "rows" else randn(dim, dtype=dtype, seed=3)
        scale, out = None, made(4, how)
        if eight:
            scale = torch.zeros((21,) if eight == "row" else (21, dim // 64), device=DEV)
            out = torch.zeros(21, 2 * dim, device=DEV).to(E4M3)[:, 1:dim + 1] if how != "columns" else torch.zeros(
                dim, 21, device=DEV).to(E4M3).t()
        kernels.rms_norm(x, weight, out, residual=r, total=total, scale=scale, eps=0.25)
        check_norm(x, weight, out, r, total, scale, eight if eight == 64 else 0, 0.25)


@pytest.mark.parametrize("eight", (0, "row", 32))
@pytest.mark.parametrize("dim", (128, 130 * 32, 224))
def test_norm_odd_values(dim, eight):
    x, weight = randn(6, dim, dtype=BF16), randn(dim, dtype=BF16, seed=1)
    x[1] = 0  # a row of nothing
    x[2, 5], x[3, 7], x[4] = math.inf, math.nan, 2.0**-60
    weight[40] = 3e38  # (y of more than fp32's largest in row 0)
    x[0, 40] = 60.0
    x[5, :32] = 0  # a group of nothing
    out = torch.empty(6, dim, dtype=E4M3 if eight else BF16, device=DEV)
    scale = torch.empty((6,) if eight == "row" else (6, dim // 32), device=DEV) if eight else None
    kernels.rms_norm(x, weight, out, scale=scale, eps=1e-6)
    got = out.float()
    assert (got[1] == 0).all() and got[2, 5].isnan() and got[3].isnan().all()
    assert (got[2, :5] == 0).all()  # over a norm of infinity
    if not eight:
        assert got[0, 40] == math.inf
        return
    assert got[0, 40].isnan() and scale.isfinite().all()  # (e4m3 has no infinity, and its scale is of the others)
    assert (scale.flatten()[scale.shape[-1] if eight == 32 else 1] == 2.0**-64).all()
    if eight == 32:
        assert (got[5, :32] == 0).all() and scale[5, 0] == 2.0**-64
        rest = slice(64, None)
        s = x[0].double()
        y = (s / torch.sqrt(s.square().mean() + 1e-6) * weight.double())[rest]
        q = (y.view(-1, 32) / scale[0, 2:].double()[:, None]).flatten()
        close(out[0, rest].double(), q, e4m3_tol(q) + q.abs() * 2.0**-15)


# -------------------------------------------------------------------------------------------- linear
def check_linear(x, weight, scales, out, zeros, c, roundings=None):
    n, k = weight.shape[0], x.shape[1]
    group = k // scales.shape[1]
    q = torch.stack((weight & 15, weight >> 4), -1).reshape(n, -1, group).double()
    z = 8.0 if zeros is None else zeros.double()[..., None]
    s = scales.double()[..., None]
    want = x.double() @ ((q - z) * s).reshape(n, k).t()
    size = x.double().abs() @ ((32 + q + abs(z)) * s.abs()).reshape(n, k).t()
    if c is not None:
        want, size = want + c.double(), size + c.double().abs()
    tol = 2.0**-23 * (roundings or group + scales.shape[1] / 8 + 16) * size + want.abs() * half_step(x.dtype)
    close(out, want, tol + (2.0**-25 if x.dtype == F16 else 0), f"{x.shape[0]} rows of {k}, {n} columns")


def weights(n, k, group, dtype, zeros, seed=0):
    g = torch.Generator().manual_seed(seed)
    weight = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).to(DEV)
    scales = (torch.rand(n, k // group, generator=g) / math.sqrt(20 * k) + 1e-4).to(dtype).to(DEV)
    if zeros:
        zeros = (torch.rand(n, k // group, generator=g) * 15).to(dtype).to(DEV)
    return weight, scales, zeros if zeros is not False else None


@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("rows,k,n,group", (
    (1, 32, 1, 32), (1, 64, 17, 64), (1, 4096, 64, 128), (2, 1024, 100, 32), (5, 160, 33, 32), (16, 768, 48, 96),
    (17, 1536, 31, 64), (32, 256, 16, 256), (33, 512, 80, 128), (64, 1152, 65, 64), (65, 384, 20, 384), (200, 2048, 130, 128),
    (3, 11008, 40, 64), (130, 96, 300, 32), (257, 1024, 515, 512), (1, 2080, 1000, 32), (100, 11008, 24, 128)))
def test_linear(rows, k, n, group, dtype, zeros):
    x, (weight, scales, z) = randn(rows, k, dtype=dtype), weights(n, k, group, dtype, zeros)
    for c in (None, randn(rows, n, dtype=dtype, seed=5), randn(n, dtype=dtype, seed=6).expand(rows, n)):
        out = torch.full((rows, n), math.nan, dtype=dtype, device=DEV)
        got = kernels.linear_4bit(x, weight, scales, out, zeros=z, c=c)
        assert got is out
        check_linear(x, weight, scales, out, z, c)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("rows", (1, 20, 150))
def test_linear_strides(rows, dtype):
    k, n, group = 320, 70, 64
    weight, scales, z = weights(n, k, group, dtype, True)
    x = randn(rows, k, dtype=dtype)
    forms = dict(
        x=[randn(rows, 3 * k, dtype=dtype)[:, k:2 * k], randn(rows * k + 1, dtype=dtype)[1:].view(rows, k),
           randn(k, rows, dtype=dtype).t(), randn(rows, k + 4, dtype=dtype)[:, :k]],
        weight=[torch.cat([weight, weight], 1)[:, :k // 2], torch.cat([weight, weight[:, :1]], 1)[:, :k // 2],
                weight.t().contiguous().t()],
        scales=[scales.t().contiguous().t(), torch.cat([scales, z], 1)[:, :k // group]],
        zeros=[z.t().contiguous().t()],
        c=[randn(n, rows, dtype=dtype).t(), randn(rows, 1, dtype=dtype).expand(rows, n)],
        out=[torch.zeros(n, rows, dtype=dtype, device=DEV).t(), torch.zeros(rows, 2 * n, dtype=dtype, device=DEV)[:, ::2],
             torch.zeros(rows, n + 3, dtype=dtype, device=DEV)[:, 1:n + 1]])
    for name, tensors in forms.items():
        for t in tensors:
            a = dict(x=x, weight=weight, scales=scales, out=torch.zeros(rows, n, dtype=dtype, device=DEV), zeros=z, c=None)
            a[name] = t
            kernels.linear_4bit(**a)
            check_linear(a["x"], a["weight"], a["scales"], a["out"], a["zeros"], a["c"])
    c = randn(rows, n, dtype=dtype, seed=9)  # onto itself
    want = kernels.linear_4bit(x, weight, scales, torch.empty_like(c), c=c)
    assert torch.equal(kernels.linear_4bit(x, weight, scales, c, c=c), want)


@pytest.mark.parametrize("rows", (2, 90))
def test_linear_odd_values(rows):
    k, n = 256, 40
    weight, scales, z = weights(n, k, 64, BF16, True)
    x = randn(rows, k, dtype=BF16)
    x[1, 7] = math.nan
    scales[3, 2] = math.inf
    want = torch.empty(rows, n, dtype=BF16, device=DEV)
    kernels.linear_4bit(x, weight, scales, want, zeros=z)
    assert want[1].isnan().all() and not want[0, 3].isfinite()
    keep = [i for i in range(n) if i != 3]
    check_linear(x[:1], weight[keep], scales[keep], want[:1, keep], z[keep], None)  # (the other rows and columns)
    out = torch.full((rows, n), 7.0, dtype=BF16, device=DEV)  # k of zero: c, or nothing
    kernels.linear_4bit(x[:, :0], weight[:, :0], scales[:, :0], out)
    assert (out == 0).all()
    kernels.linear_4bit(x[:, :0], weight[:, :0], scales[:, :0], out, c=want.nan_to_num())
    assert torch.equal(out, want.nan_to_num())


@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("rows,k,n,group", (
    (65, 32, 9601, 32), (130, 160, 6401, 32), (129, 4064, 6300, 32), (70, 96, 9545, 96), (200, 192, 4800, 64),
    (200, 1152, 4750, 64), (257, 2048, 3800, 128), (90, 640, 9600, 128), (300, 768, 3800, 256), (128, 128, 9600, 128)))
def test_linear_of_many_rows(rows, k, n, group, dtype, zeros):
    """Tiles of 64 rows.  Sums in fp32: of 128 products at most and of as many x (their order is the matrix core's: twice
    the roundings), two products with scale and zero point, and then a sum for every 32, 64 or 128 elements of k."""
    x, (weight, scales, z) = randn(rows, k, dtype=dtype), weights(n, k, group, dtype, zeros)
    piece = 128 if group % 128 == 0 else 64 if group % 64 == 0 else 32
    for c in (None, randn(n, rows, dtype=dtype, seed=5).t()):
        out = torch.full((rows, n), math.nan, dtype=dtype, device=DEV)
        kernels.linear_4bit(x, weight, scales, out, zeros=z, c=c)
        check_linear(x, weight, scales, out, z, c, roundings=2 * piece + 2 + k / piece)
    again = c.clone()  # onto c itself, the same bits
    assert torch.equal(kernels.linear_4bit(x, weight, scales, again, zeros=z, c=again), out)
    # columns of a wider output, groups along the other side, rows of a wider x
    wide = torch.full((rows, 2 * n), 3.0, dtype=dtype, device=DEV)
    xs = torch.cat([x, x], 1)[:, k:]
    kernels.linear_4bit(xs, weight, scales.t().contiguous().t(), wide[:, ::2], c=c,
                        zeros=None if z is None else z.t().contiguous().t())
    assert torch.equal(wide[:, ::2], out) and (wide[:, 1::2] == 3).all()


def test_linear_odd_values_of_many_rows():
    rows, k, n = 130, 256, 6400
    weight, scales, z = weights(n, k, 64, BF16, True)
    x = randn(rows, k, dtype=BF16)
    x[70, 7] = math.nan
    scales[3, 2] = math.inf
    out = torch.empty(rows, n, dtype=BF16, device=DEV)
    kernels.linear_4bit(x, weight, scales, out, zeros=z)
    assert out[70].isnan().all() and not out[:, 3].isfinite().any()
    rest, keep = [i for i in range(rows) if i != 70], [i for i in range(n) if i != 3]
    check_linear(x[rest], weight[keep], scales[keep], out[rest][:, keep], z[keep], None, roundings=2 * 64 + 2 + 4)
    none = torch.full((rows, n), 7.0, dtype=BF16, device=DEV)  # k of zero
    kernels.linear_4bit(x[:, :0], weight[:, :0], scales[:, :0], none)
    assert (none == 0).all()


def test_linear_of_quantized_weights():
    w = randn(96, 512, dtype=BF16, scale=0.05)
    x = randn(9, 512, dtype=BF16, seed=1)
    exact = x.double() @ w.double().t()
    for symmetric in (False, True):
        weight, scales, zeros = kernels.quantize_4bit(w, 64, symmetric)
        out = kernels.linear_4bit(x, weight, scales, torch.empty(9, 96, dtype=BF16, device=DEV), zeros=zeros)
        check_linear(x, weight, scales, out, zeros, None)
        # each weight is off by a step at most (see the steps' own test), of some 0.05 * 6 / 15
        step = scales.double().repeat_interleave(64, 1)
        close(out, exact, x.double().abs() @ (step * (1 + 15 * half_step(BF16))).t() + exact.abs() * 2.0**-7)


# ---------------------------------------------------------------------------------------------- copy
def run_copy(kc, vc, ks, vs, sources, destinations, counts):
    want = []
    for t in (kc, vc):
        t = t.clone()
        held = t.view(torch.uint8) if t.dtype == E4M3 else t
        for i, (a, b) in enumerate(zip(sources, destinations)):
            if 0 <= a < kc.shape[0] and 0 <= b < kc.shape[0]:
                n = kc.shape[1] if counts is None else min(max(counts[i], 0), kc.shape[1])
                held[b, :n] = held[a, :n]
        want.append(t)
    for s in (ks, vs):
        s = None if s is None else s.clone()
        for a, b in zip(sources, destinations):
            if s is not None and 0 <= a < kc.shape[0] and 0 <= b < kc.shape[0]:
                s[b] = s[a]
        want.append(s)
    kernels.cache_copy(kc, vc, i32(sources), i32(destinations), k_scale=ks, v_scale=vs,
                       counts=None if counts is None else i32(counts))
    for got, w, name in zip((kc, vc, ks, vs), want, ("k", "v", "k_scale", "v_scale")):
        if w is not None:
            as_bits = (lambda t: t.contiguous().view(torch.uint8)) if name in "kv" else (lambda t: t)
            assert torch.equal(as_bits(got), as_bits(w)), name


def made_cache(shape, cache, layout):
    kc, vc = caches(shape, cache, layout)
    scales = [None, None]
    if cache == E4M3:
        scales = [torch.rand(shape[0], shape[2], generator=torch.Generator().manual_seed(i)).to(DEV) for i in range(2)]
    return kc, vc, *scales


@pytest.mark.parametrize("layout", ("slots", "heads", "joint"))
@pytest.mark.parametrize("cache", (F16, BF16, E4M3))
@pytest.mark.parametrize("pages,page,heads,dim", ((4, 1, 1, 4), (6, 16, 2, 64), (9, 7, 3, 20), (40, 64, 8, 128), (8, 33, 1, 12),
                                                  (5, 100, 600, 8)))
def test_copy(pages, page, heads, dim, cache, layout):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
    n = pages // 2
    for counts in (None, [(7 * i) % (page + 2) - 1 for i in range(n)]):
        run_copy(*made_cache((pages, page, heads, dim), cache, layout), order[:n], order[n:2 * n], counts)


@pytest.mark.parametrize("cache", (F16, E4M3))
def test_copy_of_no_such_pages(cache):
    # out of range, onto itself, one source for several
    run_copy(*made_cache((12, 16, 2, 64), cache, "slots"), [0, -1, 3, 12, 5, 5, 5, 2**31 - 1, -2**31, 7],
             [1, 2, 12, 4, 5, 6, 8, 9, 10, -5], None)
    run_copy(*made_cache((12, 16, 2, 64), cache, "slots"), [], [], None)


@pytest.mark.parametrize("cache", (F16, E4M3))
def test_copy_of_strided_and_unaligned_caches(cache):
    g = torch.Generator().manual_seed(1)
    base = [(torch.randn(7 * 16 * 3 * 40 + 1, generator=g) * 8).to(cache).to(DEV) for _ in range(2)]
    for at in (0, 1):
        kc, vc = (b[at:at + 7 * 16 * 3 * 40].view(7, 16, 3, 40)[..., :36] for b in base)
        scales = [torch.rand(7, 3).to(DEV) for _ in range(2)] if cache == E4M3 else [None, None]
        run_copy(kc, vc, *scales, [0, 1, 2], [3, 4, 5], [16, 3, 9])


def test_copy_past_32_bits():
    # pages whose places pass 2^32 bytes
    page, heads, dim, pages = 64, 8, 128, 1 << 16
    kc, vc = (torch.empty(pages, page, heads, dim, dtype=F16, device=DEV) for _ in range(2))
    near = caches((2, page, heads, dim), F16)
    for c, n in zip((kc, vc), near):
        c[pages - 1], c[1] = n[0], n[1]
    kernels.cache_copy(kc, vc, i32([pages - 1, 1]), i32([2, pages - 3]))
    for c, n in zip((kc, vc), near):
        assert torch.equal(c[2], n[0]) and torch.equal(c[pages - 3], n[1])


# --------------------------------------------------------------------------------------------- chunk
def run_chunk(new, keys, heads, kv_heads, dim, page, dtype, cache, causal=True, layout="slots", edit=None, width=None,
              scale=None, spare=2, make=None, scales=None):
    """new: query tokens of each sequence; keys: what its length says."""
    tables, pages = paged([max(n, 0) for n in keys], page)
    if width:
        tables = tables[:, :width] if width < tables.shape[1] else torch.cat(
            [tables, tables.new_full((tables.shape[0], width - tables.shape[1]), -5)], 1)
    tokens = sum(new)
    make = make or (lambda n, seed: randn(n, heads, dim, dtype=dtype, seed=seed))
    q = make(tokens + spare, 0)
    kc, vc = caches((pages, page, kv_heads, dim), cache, layout)
    ks = vs = None
    if cache == E4M3:
        g = torch.Generator().manual_seed(3)
        ks, vs = scales or (torch.exp(torch.randn(pages, kv_heads, generator=g) - 4).to(DEV) for _ in range(2))
        if scales is None:
            ks[0, 0] = vs[1, 0] = 0.0
    for b, n in enumerate(keys):  # slots behind a sequence's end hold anything
        if n > 0 and n % page and n // page < tables.shape[1] and 0 <= tables[b, n // page] < pages:
            for c in (kc, vc):
                c[int(tables[b, n // page]), n % page:] = math.nan
    if edit:
        edit(q, kc, vc, tables)
    out = make(tokens + spare, 9)
    out.fill_(7.0)
    got = kernels.chunk_attention(q, kc, vc, tables, i32(keys), starts_of(new), out, k_scale=ks, v_scale=vs,
                                  causal=causal, scale=scale)
    assert got is out and (out[tokens:] == 7).all()
    group, scale, at_token = heads // kv_heads, dim**-0.5 if scale is None else scale, 0
    weight_type = F16 if cache == E4M3 else dtype
    for b, (m, n) in enumerate(zip(new, keys)):
        n = min(max(n, 0), tables.shape[1] * page)
        at = tables[b, :-(-n // page)].long()
        real = (at >= 0) & (at < pages)
        keep = real.repeat_interleave(page)[:n]
        place = torch.arange(n, device=DEV)[keep]
        last = torch.arange(m, device=DEV) + n - m if causal else torch.full((m,), n, device=DEV)
        # (the number of kept keys up to each row's last, less one)
        last = torch.searchsorted(place, last, right=True) - 1
        for h in range(kv_heads):
            kk, vv = (c[:, :, h][torch.where(real, at, 0)].double() if cache != E4M3 else
                      c[:, :, h].view(torch.uint8)[torch.where(real, at, 0)].view(E4M3).double() for c in (kc, vc))
            if cache == E4M3:
                kk = kk * ks[torch.where(real, at, 0), h].double()[:, None, None]
                vv = vv * vs[torch.where(real, at, 0), h].double()[:, None, None]
            kk, vv = kk.flatten(0, 1)[:n][keep], vv.flatten(0, 1)[:n][keep]
            vmax = float(vv[vv.isfinite()].abs().max()) if vv.isfinite().any() else 0.0
            for head in range(h * group, (h + 1) * group):
                o, size = attended(q[at_token:at_token + m, head], kk, vv, scale, last)
                o = torch.where((last >= 0)[:, None], o, 0.0)
                flat, size = torch.nan_to_num(o, 0, 0, 0), torch.nan_to_num(size, 0, 0, 0)
                tol = half_step(dtype) * flat.abs() + half_step(weight_type) * (flat.abs() + size) + 2.0**-12 * size
                close(out[at_token:at_token + m, head], o, tol + n * 2.0**-25 * vmax + 1e-30, f"sequence {b}: {m} over {n}, head {head}")
        at_token += m
    return out


MIXED = [1, 0, 5, 64, 65, 1, 300, 2, 33, 7]
CACHED = [0, 9, 63, 0, 64, 700, 130, 1, 400, 2000]


@pytest.mark.parametrize("cache", ("same", "e4m3"))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("heads,kv_heads,dim,page", ((1, 1, 64, 32), (8, 2, 128, 16), (4, 4, 128, 64), (7, 1, 64, 24),
                                                     (40, 2, 128, 32), (6, 1, 80, 128), (6, 3, 16, 1), (4, 2, 96, 48),
                                                     (3, 3, 112, 7)))
def test_chunk(heads, kv_heads, dim, page, dtype, cache):
    run_chunk(MIXED, [a + b for a, b in zip(MIXED, CACHED)], heads, kv_heads, dim, page, dtype,
              dtype if cache == "same" else E4M3)


@pytest.mark.parametrize("cache", (BF16, E4M3))
@pytest.mark.parametrize("page", (32, 24))
def test_chunk_without_a_mask(page, cache):
    run_chunk(MIXED, [a + b for a, b in zip(MIXED, CACHED)], 8, 2, 64, page, BF16, cache, causal=False)


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("cache", (F16, E4M3))
def test_chunk_of_more_queries_than_keys(cache, causal):
    # the first queries see no key; sequences without any; lengths below zero
    run_chunk([100, 3, 70, 5, 600], [40, 0, -3, 4, 100], 4, 2, 128, 16, F16, cache, causal=causal)


@pytest.mark.parametrize("cache", (F16, E4M3))
@pytest.mark.parametrize("new,cached", (([3], [20000]), ([600], [9000]), ([1, 300, 1, 1], [30000, 0, 5000, 17]),
                                        ([40] * 9, [1000 * i for i in range(9)])))
def test_chunk_split_keys(new, cached, cache):
    for heads, kv_heads, dim in ((4, 1, 128), (6, 6, 64)):
        run_chunk(new, [a + b for a, b in zip(new, cached)], heads, kv_heads, dim, 64, F16, cache, width=700)


@pytest.mark.parametrize("page", (16, 64))
@pytest.mark.parametrize("cache", (F16, E4M3))
def test_chunk_of_many_tiles_a_workgroup(cache, page):
    """64 heads share the CUs, so that a stretch is some hundred tiles long; pages are missing here and there, among them
    those around each 64th tile."""
    def edit(q, kc, vc, tables):
        kc[0], vc[0] = math.nan, math.nan
        tables[tables == 0] = -1
        tables[:, ::63 * 64 // page] = -3
        tables[:, 64 * 64 // page] = 1 << 30
        tables[0, 100:100 + 64 // page] = -1

    run_chunk([3, 0, 40], [20000, 50, 17001], 64, 64, 64, page, F16, cache, edit=edit)


@pytest.mark.parametrize("cache", (BF16, E4M3))
def test_chunk_many_sequences(cache):
    g = torch.Generator().manual_seed(7)
    new = torch.randint(0, 4, (1300,), generator=g).tolist()
    cached = torch.randint(0, 90, (1300,), generator=g).tolist()
    run_chunk(new, [a + b for a, b in zip(new, cached)], 2, 1, 64, 16, BF16, cache)


@pytest.mark.parametrize("cache", (BF16, E4M3))
@pytest.mark.parametrize("layout", ("heads", "joint"))
def test_chunk_layouts(layout, cache):
    run_chunk([30, 1, 90], [330, 78, 90], 8, 4, 128, 32, BF16, cache, layout=layout)


@pytest.mark.parametrize("cache", (F16, E4M3))
@pytest.mark.parametrize("scale", (0.0, -0.3, 3.0, 1e-4))
def test_chunk_scales(scale, cache):
    run_chunk([70, 4], [300, 90], 4, 2, 64, 32, F16, cache, scale=scale)


@pytest.mark.parametrize("page", (16, 8))
def test_chunk_far_apart_scales(page):
    # pages of 8 bits whose scales lie far apart: the weights stay within fp16 for any
    keys = [330, 200]
    _, pages = paged(keys, page)
    g = torch.Generator().manual_seed(5)
    ks = torch.exp2(torch.randint(-12, -6, (pages, 2), generator=g).float()).to(DEV)
    vs = torch.exp2(torch.randint(-40, 40, (pages, 2), generator=g).float()).to(DEV)
    run_chunk([70, 4], keys, 4, 2, 64, page, BF16, E4M3, scales=(ks, vs))


@pytest.mark.parametrize("page", (16, 24, 64))
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("cache", (F16, BF16, E4M3))
def test_chunk_odd_values_and_pages(cache, dim, page):
    def edit(q, kc, vc, tables):
        def at(b, key):
            return int(tables[b, key // page]), key % page

        vc[at(0, 150) + (0, 5)] = math.nan  # among the new tokens: hidden from some of them
        kc[at(0, 170) + (1, 7)] = math.nan
        vc[at(1, 20) + (1, 9)] = math.nan  # seen by all
        if cache != E4M3:
            vc[at(0, 180) + (1, 4)] = math.inf
            vc[at(2, 99) + (0, 4)] = -math.inf  # the last key
        kc[0], vc[0] = math.nan, math.nan  # what a missing page may not reach
        tables[tables == 0] = -1
        tables[3, 1], tables[3, 2] = -7, 1 << 30

    dtype = BF16 if cache == BF16 else F16
    run_chunk([100, 3, 40, 200, 2, 5], [200, 200, 100, 300, -3, 3000], 4, 2, dim, page, dtype, cache, edit=edit)


@pytest.mark.parametrize("dtype", (F16, BF16))
def test_chunk_keys_of_no_weight_come_first(dtype):
    # a sequence's first tiles score minus infinity, what comes behind them far below zero
    def edit(q, kc, vc, tables):
        q[..., 0], q[..., 1] = 1.0, 8.0
        kc[..., 1] = -100.0
        kc[tables[0, :5].long(), :, :, 0] = -math.inf

    tables, _ = paged([400], 32)
    out = run_chunk([50], [400], 2, 1, 64, 32, dtype, dtype, edit=edit, spare=0, scale=2.0**-3)
    assert out.isfinite().all()


def test_chunk_strides():
    for make in (lambda n, s: randn(n, 12, 64, dtype=BF16, seed=s)[:, 4:8],
                 lambda n, s: randn(4, n, 64, dtype=BF16, seed=s).transpose(0, 1),
                 lambda n, s: randn(n, 4, 128, dtype=BF16, seed=s)[..., ::2],
                 lambda n, s: randn(n, 64, 4, dtype=BF16, seed=s).transpose(1, 2),
                 lambda n, s: randn(n * 4 * 64 + 1, dtype=BF16, seed=s)[1:].view(n, 4, 64)):
        run_chunk([90, 1, 20], [200, 3000, 20], 4, 2, 64, 32, BF16, BF16, make=make)


def test_chunk_lengths_past_the_table():
    run_chunk([40, 3], [500, 64], 4, 2, 64, 32, F16, F16, width=5)
    q, (kc, vc) = randn(9, 2, 64), caches((4, 32, 2, 64), F16)
    out = torch.full_like(q, math.nan)
    for c, t in ((kc[:0], i32([[0, 1]])), (kc, i32([[0, 1]])[:, :0])):  # no pages, or no room: no keys
        kernels.chunk_attention(q, c, c, t, i32([9]), i32([0, 9]), out)
        assert (out == 0).all()
        out.fill_(math.nan)


def test_chunk_starts_past_the_tokens_and_falling():
    # starts are cut to the tokens; a sequence that would end before it begins has none
    q, (kc, vc) = randn(10, 2, 64), caches((8, 32, 2, 64), F16)
    tables, lengths = i32([[0, 1], [2, 3], [4, 5]]), i32([40, 33, 64])
    out, want = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    kernels.chunk_attention(q, kc, vc, tables, lengths, i32([-4, 6, 6, 50]), out)
    kernels.chunk_attention(q, kc, vc, tables, lengths, i32([0, 6, 6, 10]), want)
    assert torch.equal(out, want)
    out.fill_(7.0)
    kernels.chunk_attention(q, kc, vc, tables, lengths, i32([0, 6, 4, 4]), out)
    kernels.chunk_attention(q, kc, vc, tables, lengths, i32([0, 6, 6, 6]), want.fill_(7.0))
    assert torch.equal(out, want)


def test_chunk_pages_past_32_bits():
    page, heads, dim, pages = 64, 8, 128, 1 << 17
    kc, vc = (torch.empty(pages, page, heads, dim, dtype=E4M3, device=DEV) for _ in range(2))
    near = caches((4, page, heads, dim), E4M3)
    used = [pages - 1, 1, pages - 2, pages // 2]
    for c, n in zip((kc, vc), near):
        for i, p in enumerate(used):
            c[p].copy_(n[i])
    scales = [[torch.full((n, heads), 2.0**-6, device=DEV) for _ in range(2)] for n in (pages, 4)]
    q, starts, lengths = randn(50, 16, dim, dtype=BF16), i32([0, 30, 50]), i32([128, 100])
    got = kernels.chunk_attention(q, kc, vc, i32([used[:2], used[2:]]), lengths, starts, torch.empty_like(q), *scales[0])
    want = kernels.chunk_attention(q, *near, i32([[0, 1], [2, 3]]), lengths, starts, torch.empty_like(q), *scales[1])
    assert torch.equal(got, want) and want.isfinite().all()


# ------------------------------------------------------------------------------------------ together
class Layer:
    """One layer over a paged cache: norm, 4-bit projections, rotation, append, attention of the chunk, 4-bit projection
    onto the residual, norm in 8 bits and an 8-bit product."""

    heads, kv_heads, dim, page = 8, 2, 64, 16

    def __init__(self, cache, dtype, pages):
        n = self.heads * self.dim
        self.dtype, self.eight = dtype, cache == E4M3
        w = [randn(m, n, dtype=dtype, seed=20 + i, scale=n**-0.5) for i, m in enumerate((n + 2 * self.kv_heads * self.dim, n))]
        self.qkv, self.o = (kernels.quantize_4bit(x, 64) for x in w)
        self.norms = [(1 + 0.1 * randn(n, dtype=F32, seed=30 + i)).to(dtype) for i in range(2)]
        self.up = randn(128, n, dtype=F16, seed=40).to(E4M3).t()
        self.freqs = kernels.rotary_frequencies(self.dim)
        self.caches = [torch.zeros(pages, self.page, self.kv_heads, self.dim, dtype=cache, device=DEV) for _ in range(2)]
        self.scales = [torch.ones(pages, self.kv_heads, device=DEV) for _ in range(2)] if self.eight else [None, None]

    def buffers(self, tokens):
        n, kv = self.heads * self.dim, self.kv_heads * self.dim
        e = lambda *shape, dtype=self.dtype: torch.zeros(*shape, dtype=dtype, device=DEV)  # noqa: E731
        return dict(h=e(tokens, n), qkv=e(tokens, n + 2 * kv), out=e(tokens, n), y=e(tokens, n, dtype=E4M3),
                    scale=e(tokens, dtype=F32), up=e(tokens, 128, dtype=F16))

    def step(self, b, x, residual, tables, lengths, starts, positions):
        n, kv = self.heads * self.dim, self.kv_heads * self.dim
        kernels.rms_norm(x, self.norms[0], b["h"], residual=residual)
        kernels.linear_4bit(b["h"], *self.qkv[:2], b["qkv"], zeros=self.qkv[2])
        q = b["qkv"][:, :n].view(-1, self.heads, self.dim)
        k, v = (b["qkv"][:, n + i * kv:n + (i + 1) * kv].view(-1, self.kv_heads, self.dim) for i in range(2))
        kernels.rotary(q, positions, self.freqs, q)
        kernels.cache_append(k, v, *self.caches, tables, lengths, starts, *self.scales, freqs=self.freqs)
        lengths.add_(starts[1:] - starts[:-1])
        o = b["out"].view(-1, self.heads, self.dim)
        kernels.chunk_attention(q, *self.caches, tables, lengths, starts, o, *self.scales)
        kernels.linear_4bit(b["out"], *self.o[:2], residual, zeros=self.o[2], c=residual)
        kernels.rms_norm(residual, self.norms[1], b["y"], scale=b["scale"])
        kernels.gemm(b["y"], self.up, b["up"])
        return residual, (b["up"].float() * b["scale"][:, None])

    def plain(self, x, residual):
        """The same for one whole sequence, in 64 bits."""
        n, kv = self.heads * self.dim, self.kv_heads * self.dim

        def norm(x, w):
            return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()

        def linear(x, w):
            q = torch.stack((w[0] & 15, w[0] >> 4), -1).reshape(w[0].shape[0], -1, 64).double()
            return x @ ((q - w[2].double()[..., None]) * w[1].double()[..., None]).flatten(1).t()

        r = x.double() + residual.double()
        qkv = linear(norm(r, self.norms[0]), self.qkv)
        q, k, v = (t.reshape(x.shape[0], -1, self.dim) for t in qkv.split((n, kv, kv), 1))
        angle = torch.arange(x.shape[0], device=DEV)[:, None, None] * self.freqs
        turn = lambda t: torch.cat([t[..., :32] * angle.cos() - t[..., 32:] * angle.sin(),  # noqa: E731
                                    t[..., 32:] * angle.cos() + t[..., :32] * angle.sin()], -1)
        q, k, last = turn(q), turn(k), torch.arange(x.shape[0], device=DEV)
        o = torch.cat([attended(q[:, h], k[:, h // 4], v[:, h // 4], self.dim**-0.5, last)[0] for h in range(self.heads)], 1)
        r = r + linear(o, self.o)
        return r, norm(r, self.norms[1]) @ self.up.double()


@pytest.mark.parametrize("cache,dtype", ((BF16, BF16), (F16, F16), (E4M3, BF16)))
def test_a_layer_in_chunks_and_a_fork(cache, dtype):
    """Prompts in pieces, a fork, then tokens one by one, against each whole sequence in 64 bits."""
    pages, width = 40, 12
    layer = Layer(cache, dtype, pages)
    n = layer.heads * layer.dim
    pieces = ([20, 33, 1], [60, 0, 7], [1, 40, 30])  # of three sequences
    x = [randn(sum(p[b] for p in pieces) + 3, n, dtype=dtype, seed=b) for b in range(3)]
    r = [randn(*t.shape, dtype=dtype, seed=10 + b, scale=2.0) for b, t in enumerate(x)]
    tables = torch.arange(3 * width, device=DEV).view(3, width).to(torch.int32)
    lengths, at = i32([0, 0, 0]), [0, 0, 0]
    got = [[] for _ in range(4)]

    def run(rows, which, lengths, tables):
        """rows[i] tokens of sequence which[i]"""
        take = lambda t: torch.cat([t[b][at[b]:at[b] + m] for b, m in zip(which, rows)])  # noqa: E731
        positions = torch.cat([torch.arange(at[b], at[b] + m) for b, m in zip(which, rows)]).to(DEV)
        return layer.step(layer.buffers(sum(rows)), take(x), take(r), tables, lengths, starts_of(rows), positions)

    for rows in pieces:
        out = run(rows, (0, 1, 2), lengths, tables)
        for b, parts in enumerate(zip(*(t.split(rows) for t in out))):
            got[b].append([p.clone() for p in parts])
        at = [a + m for a, m in zip(at, rows)]
    # sequence 1 forks: it shares its full pages, and takes a copy of the begun one
    full, begun = at[1] // layer.page, at[1] % layer.page
    own = pages - 1
    kernels.cache_copy(*layer.caches, tables[1, full:full + 1].contiguous(), i32([own]), *layer.scales, counts=i32([begun]))
    fork = tables[1].clone()
    fork[full], fork[full + 1] = own, own - 1
    tables, lengths = torch.cat([tables, fork[None]]), torch.cat([lengths, lengths[1:2]])
    at.append(at[1])
    x.append(torch.cat([x[1][:at[1]], randn(3, n, dtype=dtype, seed=50)]))
    r.append(torch.cat([r[1][:at[1]], randn(3, n, dtype=dtype, seed=51, scale=2.0)]))
    got[3] = list(got[1])
    for _ in range(3):
        out = run([1] * 4, (0, 1, 2, 3), lengths, tables)
        for b in range(4):
            got[b].append([t[b:b + 1].clone() for t in out])
        at = [a + 1 for a in at]
    assert lengths.tolist() == at
    for b in range(4):
        want = layer.plain(x[b], r[b])
        residual, up = (torch.cat([p[i] for p in got[b]]).double() for i in range(2))
        # Each step rounds what is at most some 8 wide by e, five times on a path (the norm, q k v, the attention's weights
        # and output, the residual), and a projection sums n such errors at random, of weights of about n^-0.5: 5 e 8
        # at four times their deviation.  8 bits: keys and values are off by 2^-4 of their size, about as in a
        # step of the cache's own test, 0.5 in all.
        tol = 4 * 5 * half_step(dtype) * 8 + (0.5 if cache == E4M3 else 0)
        close(residual, want[0], torch.tensor(tol), f"sequence {b}")
        # the product of 8-bit values: n terms off by 2^-4 of about 1 times weights of about 1, at six times the deviation
        # (n^0.5 2^-4 / 3^0.5), and what the residual's error above makes of it
        close(up, want[1], torch.tensor(6 * (n / 3)**0.5 * 2.0**-4 + n**0.5 * tol), f"sequence {b}, up")


def test_a_captured_layer_replays():
    layers = [Layer(E4M3, BF16, 80) for _ in range(2)]
    n = 8 * 64
    rows = [5, 1, 1, 30]
    x, r0 = randn(37, n, dtype=BF16), randn(37, n, dtype=BF16, seed=1)
    tables, starts = torch.arange(80, device=DEV).view(4, 20).to(torch.int32), starts_of(rows)
    state = [dict(b=layer.buffers(37), r=r0.clone(), lengths=i32([0, 10, 47, 100]), copies=i32([[61, 2], [79, 78]]))
             for layer in layers]

    def step(layer, s):
        s["r"].copy_(r0)
        positions = torch.cat([s["lengths"][i:i + 1] + torch.arange(m, device=DEV) for i, m in enumerate(rows)])
        s["up"] = layer.step(s["b"], x, s["r"], tables, s["lengths"], starts, positions)[1]
        kernels.cache_copy(*layer.caches, s["copies"][0], s["copies"][1], *layer.scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = Layer(E4M3, BF16, 80)
        step(warm, dict(state[0], b=warm.buffers(37), r=r0.clone(), lengths=i32([0, 10, 47, 100])))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(layers[1], state[1])
    for _ in range(4):
        step(layers[0], state[0])
        graph.replay()
        torch.cuda.synchronize()
        for name in ("h", "qkv", "out", "scale", "up"):
            assert torch.equal(state[0]["b"][name], state[1]["b"][name]), name
        assert torch.equal(state[0]["b"]["y"].view(torch.uint8), state[1]["b"]["y"].view(torch.uint8))
        assert torch.equal(state[0]["r"], state[1]["r"]) and torch.equal(state[0]["lengths"], state[1]["lengths"])
        for a, b in zip(layers[0].caches, layers[1].caches):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_streams_at_once():
    """The same calls on two streams at once, each with its own outputs."""
    q, (kc, vc) = randn(80, 8, 128, dtype=BF16), caches((300, 32, 2, 128), BF16)
    tables, lengths, starts = torch.arange(300, device=DEV).view(3, 100).to(torch.int32), i32([3200, 1000, 77]), i32([0, 3, 4, 80])
    x, w, (weight, scales, z) = randn(9, 1024, dtype=BF16), randn(1024, dtype=BF16), weights(512, 1024, 128, BF16, True)

    def calls():
        return (kernels.chunk_attention(q, kc, vc, tables, lengths, starts, torch.empty_like(q)),
                kernels.rms_norm(x, w, torch.empty_like(x)),
                kernels.linear_4bit(x, weight, scales, torch.empty(9, 512, dtype=BF16, device=DEV), zeros=z))

    want = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for each in got for a, b in zip(each, want))
