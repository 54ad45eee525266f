"""What a layer of a model that answers from a paged key/value cache runs beside its rotation and its
appends: the norm before a product with the residual's addition, products with 4-bit weights, attention of
pieces of prompts (or several drafted tokens) over the cache's pages, and pages copied where sequences
fork or move.

``own`` tells which form ``run`` takes: elementary torch operations in 32 bits, or this package's entry
points.  ``exact`` states each operator once more in 64 bits.  Sizes are those of linear layers and heads
that the repository's benchmark uses (4096, 11008, 32 heads of 128) and generic ones around them.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}
E4M3_MAX = 448.0
LEAST_SCALE = 2.0**-64  # of a row or group of a norm in 8 bits
EPS = 1e-6


def listed():
    return [
        # the residual stream of one decode step of 48 sequences
        dict(name="norm_step", kind="norm", rows=48, dim=4096, dtype="bf16", out="bf16", group=0, residual=True),
        # the same of a long packed prompt, for a product in 8 bits with a scale a token
        dict(name="norm_prompt_8bit", kind="norm", rows=8192, dim=4096, dtype="bf16", out="e4m3", group=0, residual=True),
        # a first layer's norm (nothing to add) of a ragged batch, with scales for groups of 128
        dict(name="norm_groups_8bit", kind="norm", rows=1237, dim=5120, dtype="f16", out="e4m3", group=128,
             residual=False),
        # 60 sequences fork (two answers each): the begun last page of each is copied, as far as it is filled
        dict(name="copy_fork", kind="copy", pages=60, spare=600, page=64, heads=8, dim=128, dtype="e4m3", partly=True),
        # a cache is compacted: pages from behind go to the free ones in front
        dict(name="copy_compact", kind="copy", pages=1500, spare=1300, page=16, heads=8, dim=128, dtype="f16",
             partly=False),
        # one token through one linear layer
        dict(name="linear_one", kind="linear", rows=1, k=4096, n=4096, group=128, dtype="f16", zeros=False, add=False),
        # a decode step of 24 sequences, down projection onto the residual
        dict(name="linear_step", kind="linear", rows=24, k=11008, n=4096, group=64, dtype="bf16", zeros=True, add=True),
        # a piece of a prompt
        dict(name="linear_chunk", kind="linear", rows=300, k=4096, n=11008, group=128, dtype="bf16", zeros=True,
             add=False),
        # five drafted tokens of each of 32 sequences are looked over at once, 8 bits
        dict(name="chunk_drafts_8bit", kind="chunk", sequences=32, singles=0, low=5, high=5, cached_low=500,
             cached_high=6000, spread=1, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", cache="e4m3"),
        # sequences of one new token each beside two that are at pieces of their prompts, pages of 16
        dict(name="chunk_mixed", kind="chunk", sequences=40, singles=38, low=400, high=700, cached_low=200,
             cached_high=4000, spread=2, heads=32, kv_heads=8, dim=128, page=16, dtype="f16", cache="f16"),
        # three prompts' next pieces of about 2,000 tokens
        dict(name="chunk_prompts", kind="chunk", sequences=3, singles=0, low=1500, high=2048, cached_low=3500,
             cached_high=7000, spread=3, heads=32, kv_heads=8, dim=128, page=32, dtype="bf16", cache="bf16"),
        # a question of 512 tokens behind one very long cached document, 8 bits
        dict(name="chunk_long_8bit", kind="chunk", sequences=1, singles=0, low=512, high=512, cached_low=60001,
             cached_high=60001, spread=4, heads=28, kv_heads=4, dim=128, page=64, dtype="f16", cache="e4m3"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("norm", "copy", "linear", "chunk"))
    dtype = rng.choice(("f16", "bf16"))
    if kind == "norm":
        out = rng.choice(("same", "same", "e4m3"))
        group = rng.choice((0, 0, 32, 64, 128)) if out == "e4m3" else 0
        dim = rng.choice((1024, 2048, 4096, 5120, 8192, _log(rng, 16, 16000)))
        dim = max(1, dim // (group or 1)) * (group or 1)
        dtype = rng.choice((dtype, dtype, "f32"))
        return dict(kind=kind, rows=_log(rng, 1, max(2, 8192 * 4096 // max(dim, 1024))), dim=dim, dtype=dtype,
                    out=dtype if out == "same" else out, group=group, residual=rng.random() < 0.6)
    if kind == "copy":
        dim, heads = rng.choice((64, 80, 96, 128, 128)), rng.choice((1, 2, 4, 8))
        page = rng.choice((16, 32, 64, 128, 7))
        pages = _log(rng, 1, max(2, 20_000_000 // (page * heads * dim)))
        return dict(kind=kind, pages=pages, spare=rng.randrange(pages + 1), page=page, heads=heads, dim=dim,
                    dtype=rng.choice((dtype, "e4m3")), partly=rng.random() < 0.5)
    if kind == "linear":
        group = rng.choice((32, 64, 128, 128))
        k = rng.choice((1024, 2048, 4096, 11008, _log(rng, 128, 12000))) // group * group
        return dict(kind=kind, rows=rng.choice((1, 2, _log(rng, 1, 64), _log(rng, 1, 300))), k=max(k, group),
                    n=rng.choice((1024, 4096, 11008, _log(rng, 16, 12000))), group=group, dtype=dtype,
                    zeros=rng.random() < 0.5, add=rng.random() < 0.4)
    group = rng.choice((1, 2, 4, 7, 8))
    kv_heads = rng.choice((1, 2, 4, 8)) if group < 8 else rng.choice((1, 2, 4))
    sequences = _log(rng, 1, 64)
    cached = _log(rng, 1, max(2, min(40000, 200000 // sequences)))
    high = _log(rng, 1, max(2, min(2000, 6000 // sequences, 12_000_000 // cached)))
    return dict(kind=kind, sequences=sequences, singles=rng.choice((0, 0, rng.randrange(sequences))),
                low=max(1, high // 3), high=high, cached_low=cached // 6, cached_high=cached,
                spread=rng.randrange(1, 1 << 20), heads=group * kv_heads, kv_heads=kv_heads,
                dim=rng.choice((64, 80, 96, 128, 128)), page=rng.choice((16, 32, 64, 128)), dtype=dtype,
                cache=rng.choice((dtype, "e4m3")))


def _lengths(case):
    """New tokens and cached keys of each sequence: part of the case, not of the seed."""
    rng = random.Random(case["spread"])
    new = [1 if i < case["singles"] else rng.randint(case["low"], case["high"]) for i in range(case["sequences"])]
    return new, [rng.randint(case["cached_low"], case["cached_high"]) for _ in new]


def _tables(page_counts, gen):
    """Page tables [sequences, most pages] over pages handed out in no order, and the number of pages."""
    total = sum(page_counts) + 3
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
    width, tables, at = max(page_counts), [], 0
    for n in page_counts:
        tables.append(torch.cat([order[at:at + n], order.new_zeros(width - n)]))
        at += n
    return torch.stack(tables), total


def _pages(shape, kind, gen):
    """Random cache contents and, for 8 bits, a scale for each page and head."""
    x = torch.empty(shape, dtype=torch.float16, device=DEVICE).normal_(generator=gen)
    if kind != "e4m3":
        return x.to(TYPES[kind]), None
    scale = torch.exp2(torch.randint(-8, -4, (shape[0], shape[2]), generator=gen, device=DEVICE).float())
    return (x * 64).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE).to(TYPES[case["dtype"]])

    state, kind = dict(case=case), case["kind"]
    if kind == "norm":
        rows, dim, group = case["rows"], case["dim"], case["group"]
        x = normal(rows, dim)
        residual = normal(rows, dim).mul_(4) if case["residual"] else None
        weight = (torch.rand(dim, generator=gen, device=DEVICE) + 0.5).to(TYPES[case["dtype"]])
        scale = torch.empty((rows, dim // group) if group else (rows,), device=DEVICE) if case["out"] == "e4m3" else None
        return dict(state, x=x, residual=residual, weight=weight, total=None if residual is None else torch.empty_like(x),
                    out=torch.empty(rows, dim, dtype=TYPES[case["out"]], device=DEVICE), scale=scale)
    if kind == "copy":
        n, total = case["pages"], 2 * case["pages"] + case["spare"]
        shape = (total, case["page"], case["heads"], case["dim"])
        kc, ks = _pages(shape, case["dtype"], gen)
        vc, vs = _pages(shape, case["dtype"], gen)
        order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
        counts = None
        if case["partly"]:
            counts = torch.randint(0, case["page"] + 1, (n,), generator=gen, device=DEVICE).to(torch.int32)
        return dict(state, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, sources=order[:n].contiguous(),
                    destinations=order[n:2 * n].contiguous(), counts=counts)
    if kind == "linear":
        n, k, groups = case["n"], case["k"], case["k"] // case["group"]
        weight = torch.randint(0, 256, (n, k // 2), generator=gen, device=DEVICE, dtype=torch.uint8)
        scales = ((torch.rand(n, groups, generator=gen, device=DEVICE) + 0.2) / math.sqrt(20 * k)).to(TYPES[case["dtype"]])
        zeros = None
        if case["zeros"]:
            zeros = torch.randint(4, 12, (n, groups), generator=gen, device=DEVICE).to(TYPES[case["dtype"]])
        return dict(state, x=normal(case["rows"], k), weight=weight, scales=scales, zeros=zeros,
                    c=normal(case["rows"], n) if case["add"] else None,
                    out=torch.empty(case["rows"], n, dtype=TYPES[case["dtype"]], device=DEVICE))
    new, cached = _lengths(case)
    keys = [n + c for n, c in zip(new, cached)]
    tables, pages = _tables([-(-n // case["page"]) for n in keys], gen)
    kc, ks = _pages((pages, case["page"], case["kv_heads"], case["dim"]), case["cache"], gen)
    vc, vs = _pages((pages, case["page"], case["kv_heads"], case["dim"]), case["cache"], gen)
    q = normal(sum(new), case["heads"], case["dim"])
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEVICE)
    return dict(state, q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, tables=tables, new=new, keys=keys,
                lengths=torch.tensor(keys, dtype=torch.int32, device=DEVICE), starts=starts, out=torch.empty_like(q))


def run(state):
    case = state["case"]
    return _RUN[case["kind"]](state, case)


# ------------------------------------------------------------------------------------------------ norm
def _run_norm(state, case):
    x, weight, out, scale = state["x"], state["weight"], state["out"], state["scale"]
    residual, total = state["residual"], state["total"]
    if own:
        from ninetoothed_amd import kernels

        kernels.rms_norm(x, weight, out, residual=residual, total=total, scale=scale, eps=EPS)
    else:
        s = x.float()
        if residual is not None:
            s = s + residual.float()
            total.copy_(s)
        y = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS) * weight.float()
        if scale is None:
            out.copy_(y)
        else:
            parts = y.view(*scale.shape, -1) if case["group"] else y
            scale.copy_((parts.abs().amax(-1) / E4M3_MAX).clamp_min(LEAST_SCALE))
            out.copy_((parts / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).view_as(y))
    return [t for t in (out, scale, total) if t is not None]


# ------------------------------------------------------------------------------------------------ copy
def _run_copy(state, case):
    kc, vc, ks, vs = state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"]
    sources, destinations, counts = state["sources"], state["destinations"], state["counts"]
    if own:
        from ninetoothed_amd import kernels

        kernels.cache_copy(kc, vc, sources, destinations, k_scale=ks, v_scale=vs, counts=counts)
    else:
        for cache, scale in ((kc, ks), (vc, vs)):
            held = cache.view(torch.uint8) if scale is not None else cache
            pages = held[sources]
            if counts is not None:
                filled = torch.arange(case["page"], device=DEVICE) < counts[:, None]
                pages = torch.where(filled[..., None, None], pages, held[destinations])
            held[destinations] = pages
            if scale is not None:
                scale[destinations] = scale[sources]
    return [t for t in (kc, vc, ks, vs) if t is not None]


# ---------------------------------------------------------------------------------------------- linear
def _run_linear(state, case):
    x, weight, scales, zeros, c, out = (state[name] for name in ("x", "weight", "scales", "zeros", "c", "out"))
    if own:
        from ninetoothed_amd import kernels

        return kernels.linear_4bit(x, weight, scales, out, zeros=zeros, c=c)
    values = torch.stack((weight & 15, weight >> 4), -1).view(case["n"], -1, case["group"]).float()
    w = (values - (8.0 if zeros is None else zeros.float()[..., None])) * scales.float()[..., None]
    y = torch.matmul(x.float(), w.view(case["n"], -1).t())
    return out.copy_(y if c is None else y + c.float())


# ----------------------------------------------------------------------------------------------- chunk
def _gathered(cache, scale, tables, kv_heads, dim):
    """The sequences' pages as [sequences, kv_heads, positions, dim] in 32 bits."""
    at = tables.long()
    x = cache.view(torch.uint8)[at].view(cache.dtype).float() if scale is not None else cache[at].float()
    if scale is not None:
        x = x.mul_(scale[at][:, :, None, :, None])
    return x.view(at.shape[0], -1, kv_heads, dim).transpose(1, 2)


def _attend(state, case, first, last):
    """The sequences [first, last), padded to their longest."""
    kv_heads, dim, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    starts, lengths, n = state["starts"][first:last + 1], state["lengths"][first:last], last - first
    most_q, most_k = max(state["new"][first:last]), max(state["keys"][first:last])
    tables = state["tables"][first:last, :-(-most_k // case["page"])]
    i, new = torch.arange(most_q, device=DEVICE), starts.diff()
    at = (starts[:-1, None] + i).clamp_max(state["q"].shape[0] - 1)
    q = state["q"][at].float().view(n, most_q, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(n, kv_heads, group * most_q, dim)
    k = _gathered(state["k_cache"], state["k_scale"], tables, kv_heads, dim)
    v = _gathered(state["v_cache"], state["v_scale"], tables, kv_heads, dim).contiguous()
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim))
    scores = scores.view(n, kv_heads, group, most_q, -1)
    seen = torch.arange(scores.shape[-1], device=DEVICE) <= (i + (lengths - new)[:, None])[..., None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    scores.div_(scores.sum(-1, keepdim=True))
    o = torch.matmul(scores.view(n, kv_heads, group * most_q, -1), v)
    o = o.view(n, kv_heads, group, most_q, dim).permute(0, 3, 1, 2, 4).reshape(n, most_q, -1, dim)
    return o[i < new[:, None]]


def _run_chunk(state, case):
    if own:
        from ninetoothed_amd import kernels

        return kernels.chunk_attention(state["q"], state["k_cache"], state["v_cache"], state["tables"], state["lengths"],
                                       state["starts"], state["out"], k_scale=state["k_scale"],
                                       v_scale=state["v_scale"])
    # (single tokens apart from the rest, which would pad them)
    bounds = sorted({0, case["singles"], case["sequences"]})
    return state["out"].copy_(torch.cat([_attend(state, case, a, b) for a, b in zip(bounds, bounds[1:])]))


_RUN = dict(norm=_run_norm, copy=_run_copy, linear=_run_linear, chunk=_run_chunk)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "norm":
        elements = case["rows"] * case["dim"]
        moved = BYTES[case["dtype"]] * (3 if case["residual"] else 1) + BYTES[case["out"]]
        scales = 4 * case["rows"] * (case["dim"] // case["group"] if case["group"] else 1) * (case["out"] == "e4m3")
        return dict(bytes=elements * moved + case["dim"] * BYTES[case["dtype"]] + scales, flops=4 * elements)
    if kind == "copy":
        # (partly: half of a page on average)
        slots = case["pages"] * (case["page"] / 2 if case["partly"] else case["page"])
        return dict(bytes=int(4 * slots * case["heads"] * case["dim"] * BYTES[case["dtype"]]), flops=0)
    if kind == "linear":
        n, k, rows = case["n"], case["k"], case["rows"]
        of_groups = n * (k // case["group"]) * (4 if case["zeros"] else 2)
        return dict(bytes=n * k // 2 + of_groups + 2 * rows * (k + n * (2 if case["add"] else 1)), flops=2 * rows * n * k)
    new, cached = _lengths(case)
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
    keys = sum(new) + sum(cached)
    return dict(bytes=2 * keys * case["kv_heads"] * case["dim"] * BYTES[case["cache"]]
                + 2 * sum(new) * case["heads"] * case["dim"] * BYTES[case["dtype"]],
                flops=4 * pairs * case["heads"] * case["dim"])


# ----------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed), case)


def _exact_norm(state, case):
    s = state["x"].double() if state["residual"] is None else state["x"].double() + state["residual"].double()
    y = torch.nn.functional.normalize(s, dim=-1, eps=0.0) * math.sqrt(case["dim"])
    # 1 / sqrt(mean + eps) out of 1 / sqrt(mean)
    mean = (s * s).sum(-1, keepdim=True) / case["dim"]
    y = y * torch.sqrt(mean / (mean + EPS)) * state["weight"].double()
    answer = []
    if state["scale"] is None:
        answer.append(y)
    else:
        parts = y.unflatten(-1, (-1, case["group"] or case["dim"]))
        scale = torch.maximum(parts.amax(-1), -parts.amin(-1)) / E4M3_MAX
        scale = torch.where(scale < LEAST_SCALE, LEAST_SCALE, scale)
        answer += [(parts / scale.unsqueeze(-1)).flatten(-2), scale.view(state["scale"].shape)]
    return answer + ([] if state["residual"] is None else [s])


def _exact_copy(state, case):
    counts = [case["page"]] * case["pages"] if state["counts"] is None else state["counts"].tolist()
    pairs = list(zip(state["sources"].tolist(), state["destinations"].tolist(), counts))
    answer = []
    for name in ("k_cache", "v_cache"):
        held = state[name].double()
        for source, destination, count in pairs:
            held[destination, :count] = held[source, :count]
        answer.append(held)
    for name in ("k_scale", "v_scale"):
        if state[name] is not None:
            held = state[name].double()
            for source, destination, _ in pairs:
                held[destination] = held[source]
            answer.append(held)
    return answer


def _exact_linear(state, case):
    w = torch.empty(case["n"], case["k"], dtype=torch.float64, device=DEVICE)
    w[:, ::2], w[:, 1::2] = state["weight"] % 16, state["weight"].div(16, rounding_mode="floor")
    w -= 8.0 if state["zeros"] is None else state["zeros"].double().repeat_interleave(case["group"], 1)
    w *= state["scales"].double().repeat_interleave(case["group"], 1)
    y = (w @ state["x"].double().t()).t()
    return y if state["c"] is None else state["c"].double() + y


def _exact_chunk(state, case):
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    group, starts, kind = case["heads"] // case["kv_heads"], state["starts"].tolist(), TYPES[case["cache"]]
    for b, (new, keys) in enumerate(zip(state["new"], state["keys"])):
        at = state["tables"][b, :-(-keys // case["page"])].long()
        rows = slice(starts[b], starts[b + 1])
        hidden = torch.ones(new, keys, dtype=torch.bool, device=DEVICE).triu(keys - new + 1)
        for h in range(case["kv_heads"]):
            kv = []
            for x in "kv":
                page = state[x + "_cache"][:, :, h]
                page = page.view(torch.uint8)[at].view(kind) if kind == torch.float8_e4m3fn else page[at]
                page = page.double()
                if state[x + "_scale"] is not None:
                    page = page * state[x + "_scale"][at, h].double()[:, None, None]
                kv.append(page.flatten(0, 1)[:keys])
            for head in range(h * group, (h + 1) * group):
                scores = state["q"][rows, head].double() @ kv[0].t() / math.sqrt(case["dim"])
                out[rows, head] = torch.softmax(scores.masked_fill_(hidden, -math.inf), -1) @ kv[1]
    return out


_EXACT = dict(norm=_exact_norm, copy=_exact_copy, linear=_exact_linear, chunk=_exact_chunk)
