"""The operators around a paged key/value cache, as a program that answers with a model calls them:
the rotation of queries by position, keys and values appended to the cache, attention over packed
prompts, and the attention of one new token a sequence over what the cache holds.

``own`` tells which form ``run`` takes: elementary torch operations in 32 bits (angles in 64), or
this package's entry points.  ``exact`` states each operator once more in 64 bits.  Sizes are
those of linear layers and heads that the repository's benchmark uses (32 heads of 128, 4,000
cached keys) and generic ones around them.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}
E4M3_MAX = 448.0
LEAST_EXPONENT = -64  # of a page's scale


def listed():
    return [
        # the queries of one decode step of 48 sequences
        dict(name="rotary_step", kind="rotary", tokens=48, heads=32, dim=128, part=128, dtype="bf16",
             interleaved=False, first=3900, factor=1.0, magnitude=1.0),
        # the queries of a long packed prompt
        dict(name="rotary_prompt", kind="rotary", tokens=8192, heads=32, dim=128, part=128, dtype="bf16",
             interleaved=False, first=0, factor=1.0, magnitude=1.0),
        # a model that rotates part of an 80-wide head, pairs side by side, far into a stretched context
        dict(name="rotary_part_far", kind="rotary", tokens=5001, heads=16, dim=80, part=32, dtype="f16",
             interleaved=True, first=1_000_000, factor=8.0, magnitude=1.2079),
        # one new token for each of 64 sequences, into 8-bit pages that were begun earlier
        dict(name="append_step_8bit", kind="append", sequences=64, low=1, high=1, spread=0, heads=8, dim=128,
             part=128, page=32, dtype="bf16", cache="e4m3", interleaved=False, cached=4000),
        # nine prompts of different lengths into 8-bit pages
        dict(name="append_prompt_8bit", kind="append", sequences=9, low=500, high=3200, spread=1, heads=8, dim=128,
             part=128, page=64, dtype="bf16", cache="e4m3", interleaved=False, cached=0),
        # pieces of prompts behind what is cached already, ungrouped 64-wide heads, 16-bit pages of 16
        dict(name="append_chunk_16bit", kind="append", sequences=7, low=100, high=1100, spread=2, heads=32, dim=64,
             part=64, page=16, dtype="f16", cache="f16", interleaved=True, cached=777),
        # many short questions packed into one call
        dict(name="prompt_short", kind="prompt", sequences=24, low=16, high=200, spread=3, heads=32, kv_heads=8,
             dim=128, dtype="bf16", causal=True, prefix=0),
        # a later piece of a prompt over all the keys before it, ungrouped 64-wide heads
        dict(name="prompt_chunk", kind="prompt", sequences=2, low=512, high=512, spread=0, heads=16, kv_heads=16,
             dim=64, dtype="f16", causal=True, prefix=3500),
        # three long documents
        dict(name="prompt_long", kind="prompt", sequences=3, low=3000, high=8000, spread=5, heads=32, kv_heads=8,
             dim=128, dtype="bf16", causal=True, prefix=0),
        # a decode step of a few sequences against about 4,000 cached keys in 8 bits
        dict(name="step_8bit_few", kind="step", sequences=8, low=3500, high=4500, spread=6, heads=32, kv_heads=8,
             dim=128, page=32, dtype="bf16", cache="e4m3"),
        # a full batch of sequences of very different lengths, 8 bits
        dict(name="step_8bit_many", kind="step", sequences=128, low=100, high=9000, spread=7, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bf16", cache="e4m3"),
        # two very long contexts in 16-bit pages of 16
        dict(name="step_16bit_long", kind="step", sequences=2, low=90000, high=100001, spread=8, heads=28, kv_heads=4,
             dim=128, page=16, dtype="f16", cache="f16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "prompt", "step"))
    dim = rng.choice((64, 80, 96, 128, 128))
    dtype = rng.choice(("f16", "bf16"))
    if kind == "rotary":
        heads = rng.choice((1, 8, 12, 16, 32))
        return dict(kind=kind, tokens=_log(rng, 1, 8192 * 32 // max(heads, 16)), heads=heads, dim=dim,
                    part=rng.choice((dim, dim, dim // 2, 32)), dtype=rng.choice(("f16", "bf16", "f32")),
                    interleaved=rng.random() < 0.5, first=_log(rng, 1, 2_000_000), factor=rng.choice((1.0, 4.0, 8.0)),
                    magnitude=rng.choice((1.0, 1.1386)))
    spread = rng.randrange(1, 1 << 20)
    if kind == "append":
        sequences, step = _log(rng, 1, 200), rng.random() < 0.4
        high = 1 if step else _log(rng, 2, max(2, 16000 // sequences))
        return dict(kind=kind, sequences=sequences, low=1 if step else max(1, high // 4), high=high, spread=spread,
                    heads=rng.choice((1, 2, 4, 8)), dim=dim, part=rng.choice((dim, dim, 32)),
                    page=rng.choice((16, 32, 64, 128)), dtype=dtype, cache=rng.choice((dtype, "e4m3", "e4m3")),
                    interleaved=rng.random() < 0.5, cached=rng.choice((0, _log(rng, 1, 3000))))
    group = rng.choice((1, 2, 4, 7, 8))
    kv_heads = rng.choice((1, 2, 4, 8)) if group < 8 else rng.choice((1, 2, 4))
    if kind == "prompt":
        sequences = _log(rng, 1, 40)
        high = _log(rng, 2, max(2, min(8000, 14000 // sequences)))
        return dict(kind=kind, sequences=sequences, low=max(1, high // 3), high=high, spread=spread,
                    heads=group * kv_heads, kv_heads=kv_heads, dim=dim, dtype=dtype, causal=rng.random() < 0.75,
                    prefix=rng.choice((0, 0, _log(rng, 1, 1500))))
    sequences = _log(rng, 1, 128)
    high = _log(rng, 2, max(2, min(100000, 500000 // sequences)))
    return dict(kind=kind, sequences=sequences, low=max(1, high // 8), high=high, spread=spread,
                heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64, 128)), dtype=dtype,
                cache=rng.choice((dtype, "e4m3", "e4m3")))


def _lengths(case):
    """The sequences' lengths: part of the case, not of the seed."""
    rng = random.Random(case["spread"])
    return [rng.randint(case["low"], case["high"]) for _ in range(case["sequences"])]


def _starts(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(DEVICE)


def _frequencies(part, factor=1.0, base=10000.0):
    return (base ** -(torch.arange(0, part, 2, dtype=torch.float64) / part) / factor).to(DEVICE)


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

    state, kind, dim = dict(case=case), case["kind"], case["dim"]
    if kind == "rotary":
        x = normal(case["tokens"], case["heads"], dim)
        positions = case["first"] + torch.randperm(case["tokens"], generator=gen, device=DEVICE)
        return dict(state, x=x, positions=positions, freqs=_frequencies(case["part"], case["factor"]),
                    out=torch.empty_like(x))
    lengths = _lengths(case)
    if kind == "append":
        page, heads = case["page"], case["heads"]
        cached = [max(0, case["cached"] - 5 * i) for i in range(len(lengths))]
        tables, pages = _tables([-(-(n + c) // page) for n, c in zip(lengths, cached)], gen)
        kc, ks = _pages((pages, page, heads, dim), case["cache"], gen)
        vc, vs = _pages((pages, page, heads, dim), case["cache"], gen)
        total = sum(lengths)
        return dict(state, k=normal(total, heads, dim), v=normal(total, heads, dim), k_cache=kc, v_cache=vc, k_scale=ks,
                    v_scale=vs, tables=tables, lengths=torch.tensor(cached, dtype=torch.int32, device=DEVICE),
                    starts=_starts(lengths), freqs=_frequencies(case["part"]))
    if kind == "prompt":
        keys = [n + case["prefix"] for n in lengths]
        q = normal(sum(lengths), case["heads"], dim)
        return dict(state, q=q, k=normal(sum(keys), case["kv_heads"], dim), v=normal(sum(keys), case["kv_heads"], dim),
                    q_starts=_starts(lengths), k_starts=_starts(keys), most_q=max(lengths), most_k=max(keys),
                    out=torch.empty_like(q))
    tables, pages = _tables([-(-n // case["page"]) for n in lengths], gen)
    kc, ks = _pages((pages, case["page"], case["kv_heads"], dim), case["cache"], gen)
    vc, vs = _pages((pages, case["page"], case["kv_heads"], dim), case["cache"], gen)
    q = normal(case["sequences"], case["heads"], dim)
    return dict(state, q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, tables=tables,
                lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE), out=torch.empty_like(q))


def run(state):
    case = state["case"]
    return _RUN[case["kind"]](state, case)


# ------------------------------------------------------------------------------------------- rotation
def _rotated(x, positions, freqs, interleaved, magnitude=1.0):
    """x [tokens, heads, dim] in 32 bits with its first 2 * len(freqs) elements rotated."""
    angle = positions.to(torch.float64)[:, None, None] * freqs
    c, s = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    part = 2 * freqs.numel()
    y = x.float().clone()
    first = slice(0, part, 2) if interleaved else slice(0, part // 2)
    second = slice(1, part, 2) if interleaved else slice(part // 2, part)
    a, b = x[..., first].float(), x[..., second].float()
    y[..., first] = a * c - b * s
    y[..., second] = b * c + a * s
    return y


def _run_rotary(state, case):
    if own:
        from ninetoothed_amd import kernels

        return kernels.rotary(state["x"], state["positions"], state["freqs"], state["out"],
                              interleaved=case["interleaved"], magnitude=case["magnitude"])
    y = _rotated(state["x"], state["positions"], state["freqs"], case["interleaved"], case["magnitude"])
    return state["out"].copy_(y)


# --------------------------------------------------------------------------------------------- append
def _slots(state, page):
    """Page and slot of each new token, and its position."""
    starts, tables = state["starts"], state["tables"]
    token = torch.arange(state["k"].shape[0], device=DEVICE)
    seq = torch.searchsorted(starts[1:].contiguous(), token.to(torch.int32), right=True)
    position = state["lengths"][seq] + token - starts[seq]
    return tables[seq, position // page].long(), position % page, position


def _store_16(cache, x, pages, slots):
    cache[pages, slots] = x.to(cache.dtype)


def _store_8(cache, scale, x, pages, slots):
    """Values into 8-bit pages; the scale of a page and head is the least power of two that holds its largest
    value, kept from before (what is stored then follows it) where the page was begun earlier."""
    largest = torch.zeros_like(scale).index_reduce_(0, pages, x.abs().amax(-1), "amax")
    first = torch.full((scale.shape[0],), cache.shape[1], device=DEVICE).index_reduce_(0, pages, slots, "amin")
    mantissa, exponent = torch.frexp(largest)
    exponent = (exponent - 9 + (mantissa > E4M3_MAX / 512).int()).clamp_min(LEAST_EXPONENT)
    fitting = torch.ldexp(torch.ones_like(scale), torch.where(largest > 0, exponent, LEAST_EXPONENT))
    touched = (first < cache.shape[1])[:, None]
    begun = touched & (first > 0)[:, None]
    new = torch.where(begun, torch.maximum(scale, fitting), torch.where(touched, fitting, scale))
    held = torch.unique(pages)
    ratio = torch.where(begun, scale / new, 1.0)[held][:, None, :, None]
    cache[held] = (cache[held].float() * ratio).to(cache.dtype)
    scale.copy_(new)
    cache.view(torch.uint8)[pages, slots] = (x / new[pages][..., None]).to(cache.dtype).view(torch.uint8)


def _run_append(state, case):
    kc, vc, ks, vs = state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"]
    if own:
        from ninetoothed_amd import kernels

        kernels.cache_append(state["k"], state["v"], kc, vc, state["tables"], state["lengths"], state["starts"],
                             k_scale=ks, v_scale=vs, freqs=state["freqs"], interleaved=case["interleaved"])
    else:
        pages, slots, position = _slots(state, case["page"])
        k = _rotated(state["k"], position, state["freqs"], case["interleaved"])
        v = state["v"].float()
        if ks is None:
            _store_16(kc, k, pages, slots)
            _store_16(vc, v, pages, slots)
        else:
            _store_8(kc, ks, k, pages, slots)
            _store_8(vc, vs, v, pages, slots)
    return [kc, vc] if ks is None else [kc, vc, ks, vs]


# -------------------------------------------------------------------------------------- prompt attention
def _weights(scores, visible):
    """Softmax over the last axis of the visible places, zeros where there are none; works in place."""
    scores.masked_fill_(~visible, -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp_min(-3.0e38)).exp_()
    return scores.div_(scores.sum(-1, keepdim=True).clamp_min(1e-30))


def _padded(x, starts, most):
    """Packed rows as [sequences, most, ...] in 32 bits (rows past a sequence's end are some other row)."""
    at = (starts[:-1, None] + torch.arange(most, device=DEVICE)).clamp_max(x.shape[0] - 1)
    return x[at].float()


def _run_prompt(state, case):
    q, k, v, out = state["q"], state["k"], state["v"], state["out"]
    if own:
        from ninetoothed_amd import kernels

        return kernels.prompt_attention(q, k, v, out, state["q_starts"], state["k_starts"], causal=case["causal"])
    qs, ks, group = state["q_starts"], state["k_starts"], case["heads"] // case["kv_heads"]
    lq, lk = qs.diff()[:, None], ks.diff()[:, None]
    most_q, most_k, dim = state["most_q"], state["most_k"], case["dim"]
    n = lq.shape[0]
    qp = _padded(q, qs, most_q).view(n, most_q, -1, group, dim).permute(0, 2, 3, 1, 4).reshape(n, -1, group * most_q, dim)
    kp = _padded(k, ks, most_k).permute(0, 2, 3, 1).contiguous()
    vp = _padded(v, ks, most_k).permute(0, 2, 1, 3).contiguous()
    i, j = torch.arange(most_q, device=DEVICE), torch.arange(most_k, device=DEVICE)
    visible = (j < lk)[:, None, :].expand(n, most_q, most_k)
    if case["causal"]:
        visible = visible & (j[None, None, :] <= (i[None, :] + lk - lq)[:, :, None])
    scores = torch.matmul(qp, kp).mul_(1.0 / math.sqrt(dim)).view(n, -1, group, most_q, most_k)
    p = _weights(scores, visible[:, None, None]).view(n, -1, group * most_q, most_k)
    o = torch.matmul(p, vp).view(n, -1, group, most_q, dim).permute(0, 3, 1, 2, 4).reshape(n, most_q, -1, dim)
    return out.copy_(o[i[None, :] < lq])


# --------------------------------------------------------------------------------------- cache attention
def _gathered(cache, scale, tables, kv_heads, dim):
    """The sequences' pages as [sequences, kv_heads, positions, dim] in 32 bits."""
    at = tables.long()
    x = cache.view(torch.uint8)[at].view(cache.dtype).float() if scale is not None else cache[at].float()
    if scale is not None:
        x = x.mul_(scale[at][:, :, None, :, None])
    return x.view(at.shape[0], -1, kv_heads, dim).transpose(1, 2)


def _run_step(state, case):
    q, kc, vc, out = state["q"], state["k_cache"], state["v_cache"], state["out"]
    if own:
        from ninetoothed_amd import kernels

        return kernels.cache_attention(q, kc, vc, state["tables"], state["lengths"], out, k_scale=state["k_scale"],
                                       v_scale=state["v_scale"])
    dim, kv_heads = case["dim"], case["kv_heads"]
    k = _gathered(kc, state["k_scale"], state["tables"], kv_heads, dim)
    v = _gathered(vc, state["v_scale"], state["tables"], kv_heads, dim)
    qg = q.float().view(q.shape[0], kv_heads, -1, dim)
    scores = torch.matmul(qg, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(dim))
    visible = torch.arange(k.shape[2], device=DEVICE) < state["lengths"][:, None, None, None]
    return out.copy_(torch.matmul(_weights(scores, visible), v.contiguous()).view(q.shape))


_RUN = dict(rotary=_run_rotary, append=_run_append, prompt=_run_prompt, step=_run_step)


# -------------------------------------------------------------------------------------------------- work
def work(case):
    kind, dim = case["kind"], case["dim"]
    if kind == "rotary":
        elements = case["tokens"] * case["heads"] * dim
        return dict(bytes=2 * elements * BYTES[case["dtype"]] + 8 * case["tokens"],
                    flops=3 * case["tokens"] * case["heads"] * case["part"])
    lengths = _lengths(case)
    if kind == "append":
        elements = 2 * sum(lengths) * case["heads"] * dim
        return dict(bytes=elements * (BYTES[case["dtype"]] + BYTES[case["cache"]]),
                    flops=3 * sum(lengths) * case["heads"] * case["part"])
    if kind == "prompt":
        pairs = sum(n * case["prefix"] + (n * (n + 1) // 2 if case["causal"] else n * n) for n in lengths)
        rows = 2 * sum(lengths) * case["heads"] + 2 * sum(n + case["prefix"] for n in lengths) * case["kv_heads"]
        return dict(bytes=rows * dim * BYTES[case["dtype"]], flops=4 * pairs * case["heads"] * dim)
    keys = sum(lengths)
    return dict(bytes=2 * keys * case["kv_heads"] * dim * BYTES[case["cache"]]
                + 2 * case["sequences"] * case["heads"] * dim * BYTES[case["dtype"]],
                flops=4 * keys * case["heads"] * dim)


# ------------------------------------------------------------------------------------------------- exact
def _turned(x, positions, freqs, interleaved, magnitude=1.0):
    """The rotation as a product of complex numbers, in 64 bits."""
    x, half = x.double(), freqs.numel()
    turned = x[..., :2 * half]
    pairs = turned.unflatten(-1, (half, 2)) if interleaved else turned.unflatten(-1, (2, half)).transpose(-1, -2)
    turn = torch.polar(torch.full_like(freqs, magnitude).expand(positions.numel(), half),
                       positions.double()[:, None] * freqs)
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
    turned = pairs.flatten(-2) if interleaved else pairs.transpose(-1, -2).flatten(-2)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _attended(q, k, v, first=None):
    """Attention of q [rows, dim] over k, v [keys, dim]; row i sees keys up to first[i]."""
    scores = q @ k.t() / math.sqrt(q.shape[1])
    if first is not None:
        scores.masked_fill_(torch.arange(k.shape[0], device=q.device) > first[:, None], -math.inf)
    return torch.softmax(scores, -1) @ v


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "rotary":
        return _turned(state["x"], state["positions"], state["freqs"], case["interleaved"], case["magnitude"])
    if kind == "append":
        return _exact_append(state, case)
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    group = case["heads"] // case["kv_heads"]
    if kind == "prompt":
        qs, ks = state["q_starts"].tolist(), state["k_starts"].tolist()
        for b in range(case["sequences"]):
            rows, keys = slice(qs[b], qs[b + 1]), slice(ks[b], ks[b + 1])
            first = torch.arange(rows.stop - rows.start, device=DEVICE) + case["prefix"] if case["causal"] else None
            for h in range(case["heads"]):
                k, v = (state[x][keys, h // group].double() for x in "kv")
                out[rows, h] = _attended(state["q"][rows, h].double(), k, v, first)
        return out
    for b, n in enumerate(state["lengths"].tolist()):
        at = state["tables"][b, :-(-n // case["page"])].long()
        for h in range(case["kv_heads"]):
            k, v = (state[x + "_cache"][:, :, h].view(torch.uint8 if state["k_scale"] is not None else TYPES[case["cache"]])[at]
                    .view(TYPES[case["cache"]]).double() for x in "kv")
            if state["k_scale"] is not None:
                k, v = k * state["k_scale"][at, h].double()[:, None, None], v * state["v_scale"][at, h].double()[:, None, None]
            heads = slice(h * group, (h + 1) * group)
            out[b, heads] = _attended(state["q"][b, heads].double(), k.flatten(0, 1)[:n], v.flatten(0, 1)[:n])
    return out


def _exact_append(state, case):
    """Page by page: what each holds over its scale, before the rounding to 8 (or 16) bits."""
    page, eight = case["page"], state["k_scale"] is not None
    starts, cached, tables = state["starts"].tolist(), state["lengths"].tolist(), state["tables"].tolist()
    token, position = [], []
    for b in range(case["sequences"]):
        token += range(starts[b], starts[b + 1])
        position += range(cached[b], cached[b] + starts[b + 1] - starts[b])
    where = torch.tensor(position, device=DEVICE)
    new = [_turned(state["k"], where, state["freqs"], case["interleaved"]), state["v"].double()]
    held = [state[x].double() for x in ("k_cache", "v_cache")]
    scales = [state["k_scale"].double(), state["v_scale"].double()] if eight else []
    for b in range(case["sequences"]):
        at, last = cached[b], cached[b] + starts[b + 1] - starts[b]
        while at < last:
            stop = min(last, at // page * page + page)
            p, slot, t = tables[b][at // page], at % page, starts[b] + at - cached[b]
            for i in range(2):
                x = new[i][t:t + stop - at]
                if eight:
                    # the least power of two that 448 times is at least the largest value
                    power = torch.ceil(torch.log2(x.abs().amax((0, 2)) / E4M3_MAX)).clamp_min(LEAST_EXPONENT)
                    scale = torch.exp2(power)
                    if slot:
                        scale = torch.maximum(scale, scales[i][p])
                        held[i][p, :slot] *= (scales[i][p] / scale)[None, :, None]
                    scales[i][p] = scale
                    x = x / scale[None, :, None]
                held[i][p, slot:slot + stop - at] = x
            at = stop
    return held + scales
