"""The operators around a paged key/value cache on the GPU, against plain forms in 64 bits.

Tolerances, from the arithmetic (e: the type's half step, finfo.eps / 2):
- rotation: one rounding of the result, plus cos and sin within 2^-21 of the 64-bit values (the turn's
  fraction is rounded to 2^-25 of a turn, 2 pi 2^-25 < 2^-22, and sincospif and the fp32 products add less
  than that again), times |a| + |b|;
- prompt attention: the output's rounding, e |o|; each weight rounded for the product and in its sum,
  e (A + |o|) with A = sum p |v|; scores within (D + 4) 2^-24 sum |q k| scale, which for these
  inputs stays below 2^-13 and moves each weight by as much, and so does exp2: 2^-12 A;
  weights below fp16's normal range are off by 2^-25 at most each, out of a sum of at least 1;
- cache attention: the same with the sum in fp32, and weights in fp16 for 8-bit caches;
- 8-bit pages: half a step of e4m3, 2^-4 of the value or 2^-10, on x / scale; scales are equal.
"""

import math

import pytest
import torch

from ninetoothed_amd import _lib, kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def randn(*shape, dtype=F16, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def starts_of(lengths):
    return i32([0] + list(torch.tensor(lengths).cumsum(0))) if lengths else i32([0])


def close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol) & ~(got.double() == want) & ~(got.isnan() & want.isnan())
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {err[bad].max()} at {bad.nonzero()[0].tolist()}"


# -------------------------------------------------------------------------------------- rotation
def turned(x, positions, freqs, interleaved, inverse=False, magnitude=1.0):
    """(the rotation in 64 bits, |a| + |b| of each element's pair)"""
    x, part = x.double(), 2 * freqs.numel()
    angle = positions.double()[:, None, None] * freqs.double()
    c, s = magnitude * angle.cos(), magnitude * angle.sin() * (-1 if inverse else 1)
    one = slice(0, part, 2) if interleaved else slice(0, part // 2)
    two = slice(1, part, 2) if interleaved else slice(part // 2, part)
    y, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one] = size[..., two] = a.abs() + b.abs()
    return y, size


def rotary_tol(y, size, dtype, magnitude=1.0):
    return y.abs() * half_step(dtype) + size * magnitude * 2.0**-21 + (2.0**-25 if dtype == F16 else 0)


@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("tokens,heads,dim,part", ((1, 1, 2, 2), (1, 32, 128, 128), (37, 8, 128, 128), (513, 5, 80, 32),
                                                   (64, 3, 80, 40), (9, 2, 66, 22), (5, 7, 16, 16), (3, 2, 512, 512),
                                                   (4, 3, 24, 0), (3, 1200, 64, 64), (2, 3, 24, 12)))
def test_rotary(tokens, heads, dim, part, dtype, interleaved):
    x = randn(tokens, heads, dim, dtype=dtype)
    positions = torch.randint(0, 2_000_000, (tokens,), generator=torch.Generator().manual_seed(1)).to(DEV)
    freqs = kernels.rotary_frequencies(part) if part else torch.empty(0, dtype=torch.float64, device=DEV)
    out = torch.full_like(x, float("nan"))
    for inverse, magnitude in ((False, 1.0), (True, 1.25)):
        got = kernels.rotary(x, positions, freqs, out, interleaved=interleaved, inverse=inverse, magnitude=magnitude)
        assert got is out
        want, size = turned(x, positions, freqs, interleaved, inverse, magnitude)
        close(out, want, rotary_tol(want, size, dtype, magnitude), f"inverse={inverse}")
        if 2 * freqs.numel() < dim:
            assert torch.equal(out[..., part:], x[..., part:])


def test_rotary_in_place_strided_and_padded():
    fused = randn(50, 12, 64, dtype=BF16)  # q, k and v heads of one projection
    positions = i32(list(range(100, 150)))
    positions[[3, 49]] = -1  # padding
    freqs = kernels.rotary_frequencies(64)
    want, size = turned(fused[:, :8], positions, freqs, False)
    before = fused.clone()
    kernels.rotary(fused[:, :8], positions, freqs, fused[:, :8])
    live = positions >= 0
    close(fused[live, :8], want[live], rotary_tol(want, size, BF16)[live])
    assert torch.equal(fused[~live], before[~live]) and torch.equal(fused[:, 8:], before[:, 8:])
    # any strides: every other element, heads before tokens, positions of a wider table
    x = randn(6, 40, 48, dtype=F16, seed=3).transpose(0, 1)[..., ::2]
    out = torch.zeros(40, 24, 6, dtype=F16, device=DEV).transpose(1, 2)
    positions = torch.arange(80, device=DEV)[::2]
    freqs = kernels.rotary_frequencies(24)
    kernels.rotary(x, positions, freqs, out, interleaved=True)
    want, size = turned(x, positions, freqs, True)
    close(out, want, rotary_tol(want, size, F16))
    # one element off 16 bytes
    base = randn(40 * 2 * 64 + 1, dtype=F16)
    x = base[1:].view(40, 2, 64)
    out = torch.empty(40, 2, 64, dtype=F16, device=DEV)
    freqs = kernels.rotary_frequencies(64)
    kernels.rotary(x, positions, freqs, out)
    want, size = turned(x, positions, freqs, False)
    close(out, want, rotary_tol(want, size, F16))
    with pytest.raises(ValueError):
        kernels.rotary(x, positions, freqs, x.view(2, 40, 64).transpose(0, 1))


def test_rotary_gradient():
    x, positions, freqs = randn(7, 2, 32, dtype=F32), torch.arange(7, device=DEV), kernels.rotary_frequencies(24)
    g, direction = randn(7, 2, 32, dtype=F32, seed=1), randn(7, 2, 32, dtype=F32, seed=2)
    grad = kernels.rotary(g, positions, freqs, torch.empty_like(g), interleaved=True, inverse=True, magnitude=1.5)

    def loss(x):
        y = kernels.rotary(x, positions, freqs, torch.empty_like(x), interleaved=True, magnitude=1.5)
        return (y.double() * g).sum()

    # the map is linear: its difference quotient is exact but for fp32 roundings of 448 products
    slope = (loss(x + direction) - loss(x - direction)) / 2
    assert abs(slope - (grad.double() * direction).sum()) < 1e-3
    leaf = x.double().requires_grad_()
    y, _ = turned(leaf, positions, freqs, True, magnitude=1.5)
    y.backward(g.double())
    close(grad, leaf.grad, rotary_tol(leaf.grad, turned(g, positions, freqs, True)[1], F32, 1.5))


# ---------------------------------------------------------------------------------------- append
def paged(lengths, page, pages_extra=2, seed=0):
    """Tables over pages in no order for sequences of these total lengths, and the number of pages."""
    counts = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(counts) + pages_extra, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(counts + [1])
    tables, at = [], 0
    for n in counts:
        tables.append(order[at:at + n] + [10**6] * (width - n))  # (numbers no page has)
        at += n
    return i32(tables).view(len(lengths), width), sum(counts) + pages_extra


def caches(shape, dtype, layout="slots", seed=5):
    """A pair of caches [pages, page, heads, dim] full of numbers, stored as the layout says."""
    pages, page, heads, dim = shape
    stored = {"slots": shape, "heads": (pages, heads, page, dim), "joint": (pages, 2, page, heads, dim)}[layout]
    both = []
    for i in range(1 if layout == "joint" else 2):
        x = randn(*stored, seed=seed + i)
        both.append((x * 64).clamp(-448, 448).to(E4M3) if dtype == E4M3 else x.to(dtype))
    if layout == "joint":
        return both[0][:, 0], both[0][:, 1]
    return [c if layout == "slots" else c.transpose(1, 2) for c in both]


def read(cache, page, slot):
    return cache[page, slot].double()


def e4m3_tol(want):
    return torch.maximum(want.abs() * half_step(E4M3), torch.tensor(2.0**-10)) * (1 + 2.0**-18)


def check_append(k, v, kc, vc, ks, vs, before, tables, cached, lengths, page, freqs, interleaved, magnitude=1.0):
    """Every slot of every page against the definition, page by page."""
    kc0, vc0, ks0, vs0 = before
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    touched = set()
    tables = tables.tolist()
    for b, n in enumerate(lengths):
        at, last = cached[b], cached[b] + n
        while at < last:
            stop = min(last, at // page * page + page)
            index = at // page
            if index < len(tables[b]) and 0 <= tables[b][index] < kc.shape[0]:
                p, slot, t = tables[b][index], at % page, starts[b] + at - cached[b]
                count = stop - at
                touched.add(p)
                positions = torch.arange(at, stop, device=DEV)
                wk, size = turned(k[t:t + count], positions, freqs, interleaved, magnitude=magnitude)
                for x, tol, c, c0, s, s0 in ((wk, rotary_tol(wk, size, k.dtype, magnitude), kc, kc0, ks, ks0),
                                             (v[t:t + count].double(), 0, vc, vc0, vs, vs0)):
                    new = slice(slot, slot + count)
                    if s is None:
                        close(c[p, new], x, tol)
                        old = torch.ones(page, dtype=torch.bool)
                        old[new] = False
                        assert torch.equal(c[p][old], c0[p][old])
                        continue
                    finite = torch.where(x.isfinite(), x, 0.0).abs().amax((0, 2))
                    fit = torch.exp2(torch.ceil(torch.log2(finite / 448)).clamp_min(-64))
                    scale = torch.maximum(fit, s0[p].double()) if slot else fit
                    assert torch.equal(s[p].double(), scale), (s[p], scale)
                    want = torch.where(x.isfinite(), x / scale[None, :, None], float("nan"))
                    close(read(c, p, new), want, e4m3_tol(want) + want.abs() * 2.0**-18)
                    # the other slots keep their values where the page's scale grows, behind the new ones too
                    old = [s for s in range(page) if not slot <= s < slot + count]
                    kept = (s0[p].double() / scale if slot else torch.ones_like(scale))[None, :, None]
                    want = read(c0, p, old) * kept
                    close(read(c, p, old), want, torch.full_like(want, 2.0**-10) * (kept != 1))
            at = stop
    rest = [p for p in range(kc.shape[0]) if p not in touched]
    for c, c0 in ((kc, kc0), (vc, vc0)):
        assert torch.equal(c[rest].contiguous().view(torch.uint8), c0[rest].contiguous().view(torch.uint8))
    if ks is not None:
        assert torch.equal(ks[rest], ks0[rest]) and torch.equal(vs[rest], vs0[rest])


def run_append(lengths, cached, page, heads, dim, part, dtype, cache, layout="slots", interleaved=False, spare=3, seed=0,
               edit=None, fused=False):
    tables, pages = paged([n + c for n, c in zip(lengths, cached)], page)
    total = sum(lengths) + spare  # rows behind the last sequence are nobody's
    if fused:
        kv = randn(total, 3 * heads, dim, dtype=dtype, seed=seed)
        k, v = kv[:, heads:2 * heads], kv[:, 2 * heads:]
    else:
        k, v = randn(total, heads, dim, dtype=dtype, seed=seed), randn(total, heads, dim, dtype=dtype, seed=seed + 1)
    kc, vc = caches((pages, page, heads, dim), cache, layout)
    ks = vs = None
    if cache == E4M3:
        ks, vs = (torch.exp2(torch.randint(-12, -4, (pages, heads), generator=torch.Generator().manual_seed(i)).float()).to(DEV)
                  for i in (1, 2))
    if edit:
        tables = edit(k, v, tables) if edit else tables
    freqs = kernels.rotary_frequencies(part)
    before = [None if t is None else t.clone() for t in (kc, vc, ks, vs)]
    kernels.cache_append(k, v, kc, vc, tables, i32(cached), starts_of(lengths), k_scale=ks, v_scale=vs, freqs=freqs,
                         interleaved=interleaved)
    torch.cuda.synchronize()
    check_append(k, v, kc, vc, ks, vs, before, tables, cached, lengths, page, freqs, interleaved)


@pytest.mark.parametrize("cache", ("same", "e4m3"))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("lengths,cached,page,heads,dim,part", (
    ([1], [0], 16, 1, 16, 16),
    ([1] * 70, [7 * i for i in range(70)], 16, 2, 64, 64),
    ([1, 0, 300, 17, 0, 64, 1], [5, 9, 0, 130, 0, 64, 63], 64, 4, 128, 128),
    ([130, 257], [3, 0], 128, 3, 128, 64),
    ([300], [70], 128, 2, 128, 128),
    ([33, 5, 12], [0, 31, 17], 5, 2, 80, 40),
    ([3, 4, 9], [0, 2, 1], 1, 2, 48, 22),
    ([40, 700], [0, 100], 24, 8, 96, 96),
))
def test_append(lengths, cached, page, heads, dim, part, dtype, cache):
    run_append(lengths, cached, page, heads, dim, part, dtype, dtype if cache == "same" else E4M3,
               interleaved=len(lengths) % 2 == 0)


@pytest.mark.parametrize("cache", (BF16, E4M3))
@pytest.mark.parametrize("layout", ("heads", "joint"))
def test_append_layouts(layout, cache):
    run_append([50, 1, 90], [0, 40, 11], 32, 4, 64, 64, BF16, cache, layout=layout, fused=True)


@pytest.mark.parametrize("cache", (BF16, E4M3))
def test_append_many_sequences(cache):
    g = torch.Generator().manual_seed(7)
    lengths, cached = (torch.randint(0, 90, (150,), generator=g).tolist() for _ in range(2))
    run_append(lengths, cached, 32, 2, 64, 64, BF16, cache)


@pytest.mark.parametrize("cache", (BF16, E4M3))
def test_append_pages_past_32_bits(cache):
    # pages whose slots lie past 2^32 elements, in a cache of 2^33 and in one with pages far apart
    page, heads, dim, far = 64, 8, 128, 1 << 31
    for pages, stride in ((1 << 17, page * heads * dim), (5, far)):
        kc, vc = (torch.empty((pages - 1) * stride + page * heads * dim, dtype=cache, device=DEV).as_strided(
            (pages, page, heads, dim), (stride, heads * dim, dim, 1)) for _ in range(2))
        used = [pages - 1, 1, pages - 2, pages // 2]
        tables, lengths, cached = i32([used[:2], used[2:]]), [100, 20], [5, 60]
        few = i32([[3, 1], [2, 0]])
        near = caches((4, page, heads, dim), cache)
        for c, n in zip((kc, vc), near):
            for i, p in enumerate((used[3], 1, used[2], used[0])):
                c[p].copy_(n[i])
        k, v = randn(120, heads, dim, dtype=BF16), randn(120, heads, dim, dtype=BF16, seed=1)
        scales = [[None] * 2] * 2
        if cache == E4M3:
            scales = [[torch.full((n, heads), 2.0**-6, device=DEV) for _ in range(2)] for n in (pages, 4)]
        starts, freqs = starts_of(lengths), kernels.rotary_frequencies(dim)
        kernels.cache_append(k, v, kc, vc, tables, i32(cached), starts, *scales[0], freqs=freqs)
        kernels.cache_append(k, v, *near, few, i32(cached), starts, *scales[1], freqs=freqs)
        for c, n in zip((kc, vc), near):
            for i, p in enumerate((used[3], 1, used[2], used[0])):
                assert torch.equal(c[p].contiguous().view(torch.uint8), n[i].view(torch.uint8)), (pages, i)
        # and read again from there
        q, total = randn(2, 16, dim, dtype=BF16), i32([105, 80])
        got = kernels.cache_attention(q, kc, vc, tables, total, torch.empty_like(q), *scales[0])
        want = kernels.cache_attention(q, *near, few, total, torch.empty_like(q), *scales[1])
        assert torch.equal(got, want) and want.isfinite().all()


def test_rows_past_32_bits():
    # tokens far apart: the last ones' rows lie past 2^32 elements
    n, heads, dim, stride = 70, 2, 64, 1 << 26
    far = [torch.empty((n - 1) * stride + heads * dim, dtype=BF16, device=DEV).as_strided((n, heads, dim), (stride, dim, 1))
           for _ in range(2)]
    x, y = randn(n, heads, dim, dtype=BF16), randn(n, heads, dim, dtype=BF16, seed=1)
    far[0].copy_(x)
    positions, freqs, starts = torch.arange(n, device=DEV), kernels.rotary_frequencies(dim), i32([0, 3, n])
    want, size = turned(x, positions, freqs, False)
    kernels.rotary(far[0], positions, freqs, far[1])
    close(far[1].contiguous(), want, rotary_tol(want, size, BF16))
    far[1].copy_(y)
    out = kernels.prompt_attention(x, far[0], far[1], torch.empty_like(x), starts, starts)
    check_prompt(x, x, y, out, [3, n - 3], [3, n - 3], True)
    kernels.prompt_attention(far[0], x, y, far[1], starts, starts)
    check_prompt(x, x, y, far[1].contiguous(), [3, n - 3], [3, n - 3], True)


def test_append_large_pages_of_16_bits():
    run_append([600, 3], [100, 255], 256, 2, 128, 128, F16, F16)


@pytest.mark.parametrize("cache", (F16, E4M3))
def test_append_odd_values_and_pages(cache):
    def edit(k, v, tables):
        k[0, 0, 3], k[5, 1, 7], v[2, 0, 0], v[9, 1, 5] = float("inf"), float("nan"), float("-inf"), float("nan")
        v[20:52] = 0  # a page of zeros
        k[60] = 60000.0
        tables[0, 2], tables[1, 0] = -1, tables.max() + 7  # pages the cache does not have
        return tables

    run_append([100, 20, 40], [12, 0, 5], 32, 2, 64, 64, F16, cache, edit=edit)
    # a table too narrow for the tokens
    run_append([100, 20], [12, 0], 32, 2, 64, 64, F16, cache, edit=lambda k, v, tables: tables[:, :2])


def test_append_step_by_step_grows_a_page():
    # one token at a time, each twice as large as the last: the scale follows, the old values stay in place
    page, heads, dim = 16, 2, 32
    kc, vc = (torch.zeros(1, page, heads, dim, dtype=E4M3, device=DEV) for _ in range(2))
    ks, vs = (torch.full((1, heads), float("nan"), device=DEV) for _ in range(2))
    rows = randn(page, heads, dim, dtype=BF16) * torch.exp2(torch.arange(page, device=DEV))[:, None, None].to(BF16)
    tables, starts = i32([[0]]), i32([0, 1])
    for i in range(page):
        kernels.cache_append(rows[i:i + 1], rows[i:i + 1], kc, vc, tables, i32([i]), starts, k_scale=ks, v_scale=vs)
    scale = torch.exp2(torch.ceil(torch.log2(rows.double().abs().amax((0, 2)) / 448)))
    assert torch.equal(ks[0].double(), scale) and torch.equal(vs, ks)
    want = rows.double() / scale[None, :, None]
    # each halving rounds what lies below 2^-6 once more, by 2^-10 at most; the sum halves each time
    close(kc[0].double(), want, e4m3_tol(want) + 2.0**-9)


# ------------------------------------------------------------------------------ prompt attention
def attended(q, k, v, scale, last=None):
    """(o, sum p |v|) of q [n, dim] over k, v in 64 bits; row i sees keys up to last[i]."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    seen = torch.ones(q.shape[0], k.shape[0], dtype=torch.bool, device=q.device)
    if last is not None:
        seen = torch.arange(k.shape[0], device=q.device) <= last[:, None]
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if not s.isnan().any() else torch.softmax(s, -1)
    if v.isfinite().all():
        return p @ v, p @ v.abs()
    o = torch.where(seen[:, :, None], p[:, :, None] * v[None], 0.0).sum(1)  # (what is not seen does not count)
    return o, torch.where(seen[:, :, None], p[:, :, None] * v.abs()[None], 0.0).sum(1)


def attention_tol(o, size, dtype, keys, vmax):
    e = half_step(dtype)
    return e * (2 * o.abs() + size) + 2.0**-12 * size + (keys * 2.0**-25 * vmax if dtype == F16 else 0) + 1e-30


def check_prompt(q, k, v, out, q_lengths, k_lengths, causal, scale=None):
    dim, group = q.shape[2], q.shape[1] // k.shape[1]
    scale = dim**-0.5 if scale is None else scale
    a = b = 0
    for nq, nk in zip(q_lengths, k_lengths):
        last = torch.arange(nq, device=DEV) + nk - nq if causal else None
        for h in range(q.shape[1]):
            kk, vv = k[b:b + nk, h // group], v[b:b + nk, h // group]
            o, size = attended(q[a:a + nq, h], kk, vv, scale, last)
            finite = vv[vv.isfinite()]
            vmax = float(finite.abs().max()) if finite.numel() else 0.0
            tol = attention_tol(torch.nan_to_num(o, 0, 0, 0), torch.nan_to_num(size, 0, 0, 0), q.dtype, nk, vmax)
            close(out[a:a + nq, h], o, tol, f"sequence of {nq} over {nk}, head {h}")
        a, b = a + nq, b + nk
    return a


def run_prompt(q_lengths, k_lengths, heads, kv_heads, dim, dtype, causal, edit=None, scale=None, spare=2, make=None):
    nq, nk = sum(q_lengths) + spare, sum(k_lengths) + spare
    make = make or (lambda n, h, seed: randn(n, h, dim, dtype=dtype, seed=seed))
    q, k, v = make(nq, heads, 0), make(nk, kv_heads, 1), make(nk, kv_heads, 2)
    k[sum(k_lengths):] = float("nan")  # nobody's
    v[sum(k_lengths):] = float("nan")
    if edit:
        edit(q, k, v)
    out = torch.full((nq, heads, dim), 7.0, dtype=dtype, device=DEV)
    got = kernels.prompt_attention(q, k, v, out, starts_of(q_lengths), starts_of(k_lengths), causal=causal, scale=scale)
    assert got is out
    end = check_prompt(q, k, v, out, q_lengths, k_lengths, causal, scale)
    assert (out[end:] == 7).all()


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("heads,kv_heads,dim", ((1, 1, 64), (4, 4, 128), (8, 2, 128), (7, 1, 64), (6, 2, 80), (3, 1, 40),
                                                (2, 2, 17), (32, 1, 96), (4, 2, 8)))
def test_prompt_attention(heads, kv_heads, dim, dtype, causal):
    lengths = [1, 0, 63, 64, 65, 300, 2, 257]
    run_prompt(lengths, lengths, heads, kv_heads, dim, dtype, causal)


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dtype", (F16, BF16))
def test_prompt_attention_over_other_keys(dtype, causal):
    # cached prefixes, fewer keys than queries (rows that see nothing), none at all
    run_prompt([10, 5, 100, 70, 8, 1, 33], [200, 5, 40, 1, 0, 500, 34], 4, 2, 128, dtype, causal)


def test_prompt_attention_scales():
    # (of 0: every key counts alike; negative: the least score wins)
    for scale in (0.0, -0.2, 3.0):
        run_prompt([100, 70], [100, 130], 4, 2, 64, BF16, True, scale=scale)
        run_prompt([40], [40], 2, 2, 30, F16, True, scale=scale)


def test_prompt_attention_long():
    run_prompt([2049], [2049], 2, 1, 128, BF16, True)
    run_prompt([700, 1500], [2500, 1500], 2, 2, 64, F16, True, scale=0.3)


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("dtype,dim", ((F16, 64), (BF16, 128), (BF16, 72)))
def test_prompt_attention_split_keys(dtype, dim, causal):
    # few rows over many keys: workgroups that each take some of the keys, and join their states
    def edit(q, k, v):
        v[4190, 0, 5], v[4199, 1, 9], v[3000, 1, 1] = float("inf"), float("nan"), float("-inf")
        v[5000, 0, 0] = float("inf")
        k[4150, 1] = float("nan")

    queries, keys = [40, 3, 0, 70], [4200, 3600, 900, 30]
    assert _lib.load().nt_prompt_attention_workspace_size(115, 8732, 4, 4, 2, dim) > 0
    run_prompt(queries, keys, 4, 2, dim, dtype, causal)
    run_prompt(queries, keys, 4, 2, dim, dtype, causal, edit=edit, scale=-0.1)


def test_prompt_attention_split_keys_captured():
    # two graphs on two streams, each with its own workspace, beside the eager call
    queries, keys = [40, 3, 70], [4200, 2600, 300]
    q, k, v = randn(113, 4, 64, dtype=BF16), randn(7100, 2, 64, dtype=BF16, seed=1), randn(7100, 2, 64, dtype=BF16, seed=2)
    starts, k_starts = starts_of(queries), starts_of(keys)
    assert _lib.load().nt_prompt_attention_workspace_size(113, 7100, 3, 4, 2, 64) > 0
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(2):
        outs.append(torch.empty_like(q))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            kernels.prompt_attention(q, k, v, outs[-1], starts, k_starts)
    for i in range(4):
        q.copy_(randn(113, 4, 64, dtype=BF16, seed=10 + i))
        want = kernels.prompt_attention(q, k, v, torch.empty_like(q), starts, k_starts)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
    check_prompt(q, k, v, want, queries, keys, True)


def test_prompt_attention_many_sequences():
    g = torch.Generator().manual_seed(0)
    lengths = torch.randint(0, 6, (5000,), generator=g).tolist()
    q = randn(sum(lengths), 2, 32, dtype=BF16)
    out = torch.full_like(q, float("nan"))
    starts = starts_of(lengths)
    kernels.prompt_attention(q, q, q, out, starts, starts)
    picked = [i for i in range(5000) if i % 97 == 0 or i > 4990]
    for i in picked:
        a, b = int(starts[i]), int(starts[i + 1])
        for h in range(2):
            o, size = attended(q[a:b, h], q[a:b, h], q[a:b, h], 32**-0.5, torch.arange(b - a, device=DEV))
            close(out[a:b, h], o, attention_tol(o, size, BF16, 5, 5.0))
    assert out.isfinite().all()


@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("group", (1, 4))
def test_prompt_attention_many_turns(group, dim):
    # more workgroups than the card holds several times over, of sequences of very different lengths
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 1600, (40,), generator=g).tolist()
    heads = 32
    q = randn(sum(lengths) + 3, heads, dim, dtype=BF16)
    k, v = (randn(sum(lengths) + 3, heads // group, dim, dtype=BF16, seed=i) for i in (1, 2))
    out = torch.full_like(q, float("nan"))
    starts = starts_of(lengths)
    kernels.prompt_attention(q, k, v, out, starts, starts)
    assert out[:sum(lengths)].isfinite().all() and out[sum(lengths):].isnan().all()
    for i in range(0, 40, 3):
        a, n = int(starts[i]), lengths[i]
        for h in (i % heads, heads - 1):
            o, size = attended(q[a:a + n, h], k[a:a + n, h // group], v[a:a + n, h // group], dim**-0.5,
                               torch.arange(n, device=DEV))
            close(out[a:a + n, h], o, attention_tol(o, size, BF16, n, 5.0), f"sequence {i} of {n}, head {h}")


@pytest.mark.parametrize("dim", (64, 128, 72))
@pytest.mark.parametrize("dtype", (F16, BF16))
def test_prompt_attention_masked_infinities(dtype, dim):
    # an infinite or NaN key or value reaches the rows that see it, and no other
    def edit(q, k, v):
        for at, x in ((70, float("inf")), (200, float("-inf")), (201, float("nan")), (290, float("inf")), (299, float("nan"))):
            v[at, 0, at % dim] = x
        k[150, 1] = float("nan")
        k[298, 0] = float("nan")

    run_prompt([300, 40], [300, 40], 4, 2, dim, dtype, True, edit=edit)


def test_prompt_attention_strides():
    def fused(n, h, seed):
        return randn(n, h + 4, 64, dtype=BF16, seed=seed)[:, 2:2 + h]

    def heads_first(n, h, seed):
        return randn(h, n, 64, dtype=BF16, seed=seed).transpose(0, 1)

    def every_other(n, h, seed):
        return randn(n, h, 128, dtype=BF16, seed=seed)[..., ::2]

    def unaligned(n, h, seed):
        return randn(n * h * 64 + 1, dtype=BF16, seed=seed)[1:].view(n, h, 64)

    for make in (fused, heads_first, every_other, unaligned):
        run_prompt([100, 30], [100, 30], 4, 2, 64, BF16, True, make=make)


# ------------------------------------------------------------------------------- cache attention
def run_step(lengths, heads, kv_heads, dim, page, dtype, cache, layout="slots", edit=None, width=None, seed=0,
             scale=None):
    tables, pages = paged([max(n, 0) for n in lengths], page)
    if width:
        tables = torch.cat([tables, tables.new_full((tables.shape[0], width - tables.shape[1]), -5)], 1)
    q = randn(len(lengths), heads, dim, dtype=dtype, seed=seed)
    kc, vc = caches((pages, page, heads if kv_heads is None else kv_heads, dim), cache, layout)
    ks = vs = None
    if cache == E4M3:
        g = torch.Generator().manual_seed(3)
        ks, vs = (torch.exp(torch.randn(pages, kv_heads, generator=g) - 4).to(DEV) for _ in range(2))
        ks[0, 0] = vs[1, 0] = 0.0
    # slots behind a sequence's end hold anything
    for b, n in enumerate(lengths):
        if n > 0 and n % page:
            for c in (kc, vc):
                c[int(tables[b, n // page]), n % page:] = float("nan")
    if edit:
        edit(q, kc, vc, tables)
    out = torch.full_like(q, float("nan"))
    got = kernels.cache_attention(q, kc, vc, tables, i32(lengths), out, k_scale=ks, v_scale=vs, scale=scale)
    assert got is out
    group, scale = heads // kv_heads, dim**-0.5 if scale is None else scale
    weight_type = F16 if cache == E4M3 else dtype
    for b, n in enumerate(lengths):
        n = min(max(n, 0), tables.shape[1] * page)
        at = tables[b, :-(-n // page)].long()
        real = (at >= 0) & (at < kc.shape[0])
        for h in range(kv_heads):
            kk, vv = (c[:, :, h][torch.where(real, at, 0)].double() if cache != E4M3 else
                      c[:, :, h].view(torch.uint8)[torch.where(real, at, 0)].view(E4M3).double() for c in (kc, vc))
            if cache == E4M3:
                kk = kk * ks[torch.where(real, at, 0), h].double()[:, None, None]
                vv = vv * vs[torch.where(real, at, 0), h].double()[:, None, None]
            keep = real.repeat_interleave(page)[:n]
            kk, vv = kk.flatten(0, 1)[:n][keep], vv.flatten(0, 1)[:n][keep]
            rows = slice(h * group, (h + 1) * group)
            o, size = attended(q[b, rows], kk, vv, scale)
            vmax = float(torch.nan_to_num(vv).abs().max()) if kk.shape[0] else 0.0
            tol = half_step(dtype) * o.abs() + half_step(weight_type) * size + 2.0**-12 * size + n * 2.0**-25 * vmax + 1e-30
            close(out[b, rows], o, tol, f"sequence {b} of {n}, kv head {h}")


@pytest.mark.parametrize("cache", ("same", "e4m3"))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("heads,kv_heads,dim,page", ((1, 1, 64, 32), (8, 2, 128, 16), (8, 8, 128, 64), (7, 1, 64, 24),
                                                     (40, 2, 128, 32), (16, 1, 80, 128), (6, 3, 16, 1), (12, 2, 96, 48)))
def test_cache_attention(heads, kv_heads, dim, page, dtype, cache):
    run_step([1, 0, 31, 32, 33, 127, 128, 129, 640, 1000, 2], heads, kv_heads, dim, page, dtype,
             dtype if cache == "same" else E4M3)


@pytest.mark.parametrize("cache", (F16, E4M3))
@pytest.mark.parametrize("page", (16, 64))
def test_cache_attention_split_keys(page, cache):
    # one long sequence over all workgroups; long and short ones beside each other; a table with room
    run_step([40001], 4, 1, 128, page, F16, cache)
    run_step([9000, 5, 0, 3000, 1, 129], 8, 2, 64, page, F16, cache, width=700)


@pytest.mark.parametrize("cache", (BF16, E4M3))
def test_cache_attention_scales(cache):
    for scale in (0.0, -0.1, 1.5):
        run_step([100, 70, 300], 4, 2, 64, 16, BF16, cache, scale=scale)
        run_step([100, 70, 300], 4, 2, 64, 10, BF16, cache, scale=scale)


@pytest.mark.parametrize("cache", (F16, E4M3))
def test_cache_attention_missing_odd_pages(cache):
    # pages of no whole sixteens: a missing one reaches no output, though the first page is NaN
    def edit(q, kc, vc, tables):
        kc[0], vc[0] = float("nan"), float("nan")
        tables[tables == 0] = -1
        tables[0, 1], tables[1, 0] = -7, 1 << 30

    run_step([100, 20, 300], 4, 2, 64, 24, F16, cache, edit=edit)


def test_cache_attention_many_sequences():
    g = torch.Generator().manual_seed(0)
    run_step(torch.randint(0, 300, (300,), generator=g).tolist(), 4, 2, 64, 16, BF16, E4M3)


@pytest.mark.parametrize("layout", ("heads", "joint"))
@pytest.mark.parametrize("cache", (BF16, E4M3))
def test_cache_attention_layouts(layout, cache):
    run_step([300, 77, 0, 1500], 8, 4, 128, 32, BF16, cache, layout=layout)


@pytest.mark.parametrize("page", (16, 32))
@pytest.mark.parametrize("cache", (F16, E4M3))
def test_cache_attention_odd_values_and_pages(page, cache):
    def edit(q, kc, vc, tables):
        vc[int(tables[0, 0]), 3, 0, 5] = float("nan")
        kc[int(tables[1, 1]), 2, 1, 7] = float("nan")
        if cache == F16:
            vc[int(tables[2, 0]), 9, 1, 4] = float("inf")
            vc[int(tables[2, 99 // page]), 99 % page, 0, 4] = float("-inf")  # the last key
        kc[0], vc[0] = float("nan"), float("nan")  # what a missing page may not reach
        tables[tables == 0] = -1
        tables[3, 1], tables[3, 2] = -7, 1 << 30

    run_step([100, 200, 100, 300, -3, 3000], 4, 2, 64, page, F16, cache, edit=edit)


def test_cache_attention_lengths_past_the_table():
    q, (kc, vc) = randn(2, 2, 64), caches((4, 32, 2, 64), F16)
    tables = i32([[0, 1], [2, 3]])
    a, b = torch.empty_like(q), torch.empty_like(q)
    kernels.cache_attention(q, kc, vc, tables, i32([64, 64]), a)
    kernels.cache_attention(q, kc, vc, tables, i32([65, 2**31 - 1]), b)
    assert torch.equal(a, b)
    # no pages, or no room in the tables: no keys
    for c, t in ((kc[:0], tables), (kc, tables[:, :0])):
        b.fill_(float("nan"))
        kernels.cache_attention(q, c, c, t, i32([5, 5]), b)
        assert (b == 0).all()


def test_cache_attention_strided_queries():
    fused = randn(5, 12, 64, dtype=BF16)
    kc, vc = caches((10, 32, 2, 64), BF16)
    tables, lengths = i32([[0, 1], [2, 3], [4, 5], [6, 7], [8, 9]]), i32([64, 3, 40, 0, 33])
    want = kernels.cache_attention(fused[:, 4:].contiguous(), kc, vc, tables, lengths, torch.empty_like(fused[:, 4:]))
    out = torch.zeros(5, 64, 8, dtype=BF16, device=DEV).transpose(1, 2)
    kernels.cache_attention(fused[:, 4:], kc, vc, tables, lengths, out)
    assert torch.equal(out, want)


# --------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("cache,dtype", ((BF16, BF16), (E4M3, F16)))
def test_a_prompt_and_its_steps(cache, dtype):
    """Prompts, then tokens one by one through the cache, against whole prompts in one call."""
    heads, kv_heads, dim, page, steps = 8, 2, 64, 16, 5
    prompts = [37, 1, 130]
    total = [n + steps for n in prompts]
    freqs = kernels.rotary_frequencies(dim, factor=2.0)
    q, k, v = (randn(sum(total), h, dim, dtype=dtype, seed=i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    tables, pages = paged(total, page)
    kc, vc = (torch.zeros(pages, page, kv_heads, dim, dtype=cache, device=DEV) for _ in range(2))
    scales = [torch.ones(pages, kv_heads, device=DEV) for _ in range(2)] if cache == E4M3 else [None, None]
    first = starts_of(total)[:-1].tolist()
    where = torch.cat([torch.arange(n) for n in total]).to(DEV)
    rq, rk = (kernels.rotary(x, where, freqs, torch.empty_like(x)) for x in (q, k))
    whole = kernels.prompt_attention(rq, rk, v, torch.empty_like(q), starts_of(total), starts_of(total))

    head = torch.cat([torch.arange(a, a + n) for a, n in zip(first, prompts)]).to(DEV)
    lengths = i32([0, 0, 0])
    kernels.cache_append(k[head], v[head], kc, vc, tables, lengths, starts_of(prompts), *scales, freqs=freqs)
    got = kernels.prompt_attention(rq[head], rk[head], v[head], torch.empty_like(q[head]), starts_of(prompts),
                                   starts_of(prompts))
    # (a row's tiles fall otherwise in the longer sequence: alike but for the rounding of weights and output)
    tol = 4 * half_step(dtype) * 4.0
    close(got, whole[head].double(), tol)
    lengths += i32(prompts)
    for s in range(steps):
        rows = torch.tensor([a + n + s for a, n in zip(first, prompts)], device=DEV)
        now = kernels.rotary(q[rows], lengths, freqs, torch.empty_like(q[rows]))
        kernels.cache_append(k[rows], v[rows], kc, vc, tables, lengths, i32([0, 1, 2, 3]), *scales, freqs=freqs)
        lengths += 1
        out = kernels.cache_attention(now, kc, vc, tables, lengths, torch.empty_like(now), *scales)
        # 8 bits: keys and values are off by 2^-4 of their size each at most, about a step in all
        close(out, whole[rows].double(), tol if cache != E4M3 else 0.5)


def test_a_captured_step_replays():
    heads, kv_heads, dim, page, n = 8, 2, 128, 32, 6
    q, k, v = randn(n, heads, dim, dtype=BF16), randn(n, kv_heads, dim, dtype=BF16, seed=1), randn(n, kv_heads, dim, dtype=BF16, seed=2)
    tables = torch.arange(n * 40, device=DEV).view(n, 40).to(torch.int32)
    freqs, starts = kernels.rotary_frequencies(dim), starts_of([1] * n)
    lengths = i32([0, 5, 31, 32, 700, 1200])
    prompt_starts = i32([0, 2, 6])

    def fresh():
        kc, vc = caches((n * 40, page, kv_heads, dim), E4M3)
        ks, vs = (torch.full((n * 40, kv_heads), 2.0**-6, device=DEV) for _ in range(2))
        return dict(kc=kc, vc=vc, ks=ks, vs=vs, rq=torch.zeros_like(q), out=torch.zeros_like(q), whole=torch.zeros_like(q),
                    lengths=lengths.clone())

    def step(s):
        kernels.rotary(q, s["lengths"], freqs, s["rq"])
        kernels.cache_append(k, v, s["kc"], s["vc"], tables, s["lengths"], starts, s["ks"], s["vs"], freqs=freqs)
        s["lengths"].add_(1)
        kernels.cache_attention(s["rq"], s["kc"], s["vc"], tables, s["lengths"], s["out"], s["ks"], s["vs"])
        kernels.prompt_attention(s["rq"], k, v, s["whole"], prompt_starts, prompt_starts)

    eager, captured = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured)
    for s in (captured,):
        for name, t in fresh().items():  # (the capture ran nothing)
            s[name].copy_(t)
    for _ in range(4):
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        for name in ("rq", "out", "whole", "lengths", "ks", "vs"):
            assert torch.equal(eager[name], captured[name]), name
        for name in ("kc", "vc"):
            assert torch.equal(eager[name].view(torch.uint8), captured[name].view(torch.uint8)), name


def test_other_streams_do_not_share_state():
    """The same call on two streams at once, each with its own outputs."""
    q, (kc, vc) = randn(3, 8, 128, dtype=BF16), caches((300, 32, 2, 128), BF16)
    tables, lengths = torch.arange(300, device=DEV).view(3, 100).to(torch.int32), i32([3200, 1000, 17])
    want = kernels.cache_attention(q, kc, vc, tables, lengths, torch.empty_like(q))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(20)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                kernels.cache_attention(q, kc, vc, tables, lengths, o[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for both in outs for o in both)
