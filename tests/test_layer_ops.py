"""Refusals of the operators of a layer's step over a paged cache (norm, products with 4-bit weights, attention of chunks,
page copies), and what needs no GPU of them: on the CPU, before any launch."""

import ctypes
import math

import pytest
import torch

from ninetoothed_amd import _lib, kernels

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
INVALID = 1


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def norm_args(eight=False, **change):
    a = dict(x=z(3, 256), weight=z(256), out=z(3, 256, dtype=E4M3 if eight else F16))
    if eight:
        a |= dict(scale=torch.zeros(3))
    return {**a, **change}


def linear_args(**change):
    a = dict(x=z(3, 256), weight=z(10, 128, dtype=torch.uint8), scales=z(10, 4), out=z(3, 10))
    return {**a, **change}


def copy_args(eight=False, **change):
    cache = z(5, 16, 2, 64, dtype=E4M3 if eight else F16)
    a = dict(k_cache=cache, v_cache=cache.clone(), sources=_i32(0, 1), destinations=_i32(2, 3))
    if eight:
        a |= dict(k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2))
    return {**a, **change}


def chunk_args(eight=False, **change):
    cache = z(5, 16, 2, 64, dtype=E4M3 if eight else F16)
    a = dict(q=z(6, 4, 64), k_cache=cache, v_cache=cache.clone(), tables=torch.zeros(2, 2, dtype=torch.int32),
             lengths=_i32(3, 4), starts=_i32(0, 2, 6), out=z(6, 4, 64))
    if eight:
        a |= dict(k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2))
    return {**a, **change}


OPS = dict(rms_norm=norm_args, linear_4bit=linear_args, cache_copy=copy_args, chunk_attention=chunk_args)


@pytest.mark.parametrize("op", OPS)
def test_a_good_call_passes_the_checks_and_is_refused_on_the_cpu(op):
    args = OPS[op]()
    getattr(kernels, f"check_{op}")(**args)
    with pytest.raises(TypeError, match="GPU"):
        getattr(kernels, f"bind_{op}")(**args)
    with pytest.raises(TypeError, match="GPU"):
        getattr(kernels, op)(**args)


def test_what_the_checks_find():
    assert kernels.check_rms_norm(**norm_args()) == 0
    assert kernels.check_rms_norm(**norm_args(True)) == 0
    for groups in (8, 4, 2):
        assert kernels.check_rms_norm(**norm_args(True, scale=torch.zeros(3, groups))) == 256 // groups
    assert kernels.check_linear_4bit(**linear_args()) == 64
    assert kernels.check_linear_4bit(**linear_args(scales=z(10, 1), zeros=z(10, 1), c=z(10).expand(3, 10))) == 256
    for op in ("cache_copy", "chunk_attention"):
        assert getattr(kernels, f"check_{op}")(**OPS[op](True)) == _lib.DTYPE_E4M3
    # nothing there is nothing to refuse
    kernels.check_rms_norm(z(0, 256), z(256), z(0, 256))
    kernels.check_linear_4bit(z(3, 0), z(10, 0, dtype=torch.uint8), z(10, 0), z(3, 10))
    kernels.check_cache_copy(**copy_args(sources=_i32(), destinations=_i32()))


BAD = [
    ("rms_norm", dict(x=z(256), out=z(256)), ValueError),
    ("rms_norm", dict(out=z(3, 128)), ValueError),
    ("rms_norm", dict(out=z(3, 256, dtype=BF16)), TypeError),
    ("rms_norm", dict(x=z(3, 256, dtype=torch.float64), out=z(3, 256, dtype=torch.float64)), TypeError),
    ("rms_norm", dict(weight=z(256, dtype=F32)), TypeError),
    ("rms_norm", dict(weight=z(128)), ValueError),
    ("rms_norm", dict(residual=z(3, 256, dtype=F32)), TypeError),
    ("rms_norm", dict(residual=z(2, 256)), ValueError),
    ("rms_norm", dict(total=z(3, 256)), ValueError),
    ("rms_norm", dict(residual=z(1, 256).expand(3, 256)), ValueError),
    ("rms_norm", dict(residual=z(3, 256), total=z(3, 1).expand(3, 256)), ValueError),
    ("rms_norm", dict(residual=z(3, 256), total=z(3, 256, dtype=BF16)), TypeError),
    ("rms_norm", dict(out=z(1, 256).expand(3, 256)), ValueError),
    ("rms_norm", dict(scale=torch.zeros(3)), ValueError),
    ("rms_norm", dict(eight=True, scale=None), ValueError),
    ("rms_norm", dict(eight=True, scale=torch.zeros(3, dtype=F16)), TypeError),
    ("rms_norm", dict(eight=True, scale=torch.zeros(4)), ValueError),
    ("rms_norm", dict(eight=True, scale=torch.zeros(3, 3)), ValueError),
    ("rms_norm", dict(eight=True, scale=torch.zeros(3, 16)), ValueError),  # groups of 16
    ("rms_norm", dict(eight=True, scale=torch.zeros(3, 1)), ValueError),  # of 256
    ("rms_norm", dict(eight=True, scale=torch.zeros(6)[::2]), ValueError),
    ("rms_norm", dict(x=z(1, 65537), weight=z(65537), out=z(1, 65537)), ValueError),
    ("rms_norm", dict(eps="no"), ValueError),
    ("linear_4bit", dict(x=z(256)), ValueError),
    ("linear_4bit", dict(x=z(3, 256, dtype=F32), scales=z(10, 4, dtype=F32), out=z(3, 10, dtype=F32)), TypeError),
    ("linear_4bit", dict(weight=z(10, 128, dtype=torch.int8)), TypeError),
    ("linear_4bit", dict(weight=z(10, 256, dtype=torch.uint8)), ValueError),
    ("linear_4bit", dict(scales=z(10, 4, dtype=BF16)), TypeError),
    ("linear_4bit", dict(scales=z(9, 4)), ValueError),
    ("linear_4bit", dict(scales=z(10, 3)), ValueError),
    ("linear_4bit", dict(scales=z(10, 16)), ValueError),  # groups of 16
    ("linear_4bit", dict(scales=z(10, 0)), ValueError),
    ("linear_4bit", dict(zeros=z(10, 2)), ValueError),
    ("linear_4bit", dict(zeros=z(10, 4, dtype=torch.uint8)), TypeError),
    ("linear_4bit", dict(c=z(10)), ValueError),
    ("linear_4bit", dict(c=z(3, 10, dtype=BF16)), TypeError),
    ("linear_4bit", dict(out=z(3, 9)), ValueError),
    ("linear_4bit", dict(out=z(3, 10, dtype=BF16)), TypeError),
    ("linear_4bit", dict(out=z(10).expand(3, 10)), ValueError),
    ("cache_copy", dict(k_cache=z(16, 2, 64)), ValueError),
    ("cache_copy", dict(v_cache=z(4, 16, 2, 64)), ValueError),
    ("cache_copy", dict(k_cache=z(5, 16, 2, 64, dtype=F32), v_cache=z(5, 16, 2, 64, dtype=F32)), TypeError),
    ("cache_copy", dict(v_cache=z(5, 16, 2, 64, dtype=BF16)), TypeError),
    ("cache_copy", dict(k_cache=z(5, 16, 2, 66), v_cache=z(5, 16, 2, 66)), ValueError),
    ("cache_copy", dict(k_cache=z(5, 16, 64, 2).transpose(2, 3), v_cache=z(5, 16, 2, 64)), ValueError),
    ("cache_copy", dict(k_cache=z(1, 16, 2, 64).expand(5, 16, 2, 64)), ValueError),
    ("cache_copy", dict(k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2)), ValueError),
    ("cache_copy", dict(eight=True, k_scale=None), ValueError),
    ("cache_copy", dict(eight=True, v_scale=torch.ones(2, 5).t()), ValueError),
    ("cache_copy", dict(sources=torch.zeros(2, dtype=torch.int64)), TypeError),
    ("cache_copy", dict(destinations=_i32(1)), ValueError),
    ("cache_copy", dict(sources=_i32(1, 0, 2, 0)[::2]), ValueError),
    ("cache_copy", dict(counts=_i32(1)), ValueError),
    ("cache_copy", dict(counts=torch.zeros(2)), TypeError),
    ("chunk_attention", dict(out=z(6, 4, 32)), ValueError),
    ("chunk_attention", dict(out=z(6, 4, 64, dtype=BF16)), TypeError),
    ("chunk_attention", dict(q=z(6, 3, 64), out=z(6, 3, 64)), ValueError),
    ("chunk_attention", dict(q=z(6, 4, 72), out=z(6, 4, 72), k_cache=z(5, 16, 2, 72), v_cache=z(5, 16, 2, 72)), ValueError),
    ("chunk_attention", dict(q=z(6, 4, 144), out=z(6, 4, 144), k_cache=z(5, 16, 2, 144), v_cache=z(5, 16, 2, 144)), ValueError),
    ("chunk_attention", dict(q=z(6, 4, 64, dtype=BF16), out=z(6, 4, 64, dtype=BF16)), TypeError),
    ("chunk_attention", dict(k_cache=z(16, 2, 64)), ValueError),
    ("chunk_attention", dict(k_cache=z(5, 16, 2, 68)[..., :64], v_cache=z(5, 16, 2, 64)), ValueError),
    ("chunk_attention", dict(tables=torch.zeros(3, 2, dtype=torch.int32)), ValueError),
    ("chunk_attention", dict(tables=torch.zeros(2, 2, dtype=torch.int64)), TypeError),
    ("chunk_attention", dict(lengths=_i32(1, 2, 3)), ValueError),
    ("chunk_attention", dict(starts=_i32(0, 6)), ValueError),
    ("chunk_attention", dict(starts=torch.tensor([0, 2, 6])), TypeError),
    ("chunk_attention", dict(eight=True, v_scale=None), ValueError),
    ("chunk_attention", dict(eight=True, k_cache=z(5, 256, 2, 64, dtype=E4M3), v_cache=z(5, 256, 2, 64, dtype=E4M3)), ValueError),
    ("chunk_attention", dict(out=z(6, 1, 64).expand(6, 4, 64)), ValueError),
    ("chunk_attention", dict(scale="no"), ValueError),
]


@pytest.mark.parametrize("op,change,error", BAD, ids=[f"{op}-{i}" for i, (op, _, _) in enumerate(BAD)])
def test_bad_calls_are_refused(op, change, error):
    with pytest.raises(error):
        getattr(kernels, f"check_{op}")(**OPS[op](**change))


# ------------------------------------------------------------------ the C entry points, unlaunched
S2 = (ctypes.c_int64 * 2)(256, 1)
S3 = (ctypes.c_int64 * 3)(128, 64, 1)
P = 1 << 12  # an address that nothing reads: each call returns before a launch


def _norm(lib, x=P, residual=None, total=None, scale=None, group=0, dtype=1, out=1, rows=3, dim=256):
    return lib.nt_rms_norm(x, S2, P, 1, residual, S2, total, S2, P, S2, scale, group, dtype, out, rows, dim, 1e-6, None)


def _linear(lib, x=P, weight=P, out=P, dtype=1, rows=3, n=10, k=256, group=64):
    return lib.nt_linear_4bit(x, S2, weight, S2, P, S2, None, None, None, None, out, S2, dtype, rows, n, k, group, None)


def _copy(lib, k=P, sources=P, scale=None, dtype=1, pairs=2, pages=5, page=16, heads=2, dim=64):
    return lib.nt_cache_copy(k, S3, P, S3, dtype, scale, scale, sources, P, None, pairs, pages, page, heads, dim, None)


def _chunk(lib, dtype=1, cache=1, q=P, k=P, scale=P, starts=P, strides=S3, tokens=6, seqs=2, heads=4, kv=2, dim=64, pages=5,
           page=16, width=64, ws=None, nbytes=0):
    return lib.nt_chunk_attention(q, S3, k, strides, P, strides, cache, scale, scale, P, S3, dtype, P, width, P, starts, tokens,
                                  seqs, heads, kv, dim, pages, page, width, 1.0, 1, None, ws, nbytes)


def test_entry_points_reject_before_they_launch():
    lib = _lib.load()
    for bad in (dict(dtype=3), dict(out=2), dict(x=None), dict(rows=-1), dict(dim=65537), dict(residual=P), dict(out=4),
                dict(out=4, scale=P, group=48), dict(out=4, scale=P, group=128, dim=200)):
        assert _norm(lib, **bad) == INVALID, bad
    for bad in (dict(dtype=0), dict(x=None), dict(weight=None), dict(out=None), dict(rows=-1), dict(group=16), dict(group=48),
                dict(group=96), dict(group=0), dict(k=1 << 31), dict(n=1 << 31)):
        assert _linear(lib, **bad) == INVALID, bad
    for bad in (dict(dtype=0), dict(k=None), dict(sources=None), dict(dtype=4), dict(pairs=-1), dict(pages=-1),
                dict(page=1 << 30, heads=1 << 10, dim=1 << 10), dict(pairs=1 << 31)):
        assert _copy(lib, **bad) == INVALID, bad
    # (a table of 64 pages has room for splits, which want a workspace)
    for bad in (dict(dtype=0), dict(cache=2), dict(q=None), dict(starts=None), dict(dim=72), dict(dim=144), dict(kv=0),
                dict(heads=3), dict(page=0), dict(cache=4, scale=None), dict(), dict(ws=P, nbytes=64), dict(k=P + 8),
                dict(strides=(ctypes.c_int64 * 3)(128, 60, 1)), dict(page=1 << 20, width=1 << 12), dict(tokens=1 << 31),
                dict(tokens=1 << 30, heads=8)):
        assert _chunk(lib, **bad) == INVALID, bad
    # nothing to do: no launch, no error, whatever the pointers
    assert _norm(lib, rows=0, x=None) == 0 and _norm(lib, dim=0, x=None) == 0
    assert _linear(lib, rows=0, x=None) == 0 and _linear(lib, n=0, x=None) == 0
    assert _copy(lib, pairs=0, k=None) == 0 and _copy(lib, pages=0) == 0
    assert _chunk(lib, tokens=0, q=None) == 0 and _chunk(lib, seqs=0) == 0
    for op in OPS:
        assert getattr(lib, f"nt_{op}_packed")(None) == INVALID


def test_chunk_workspace_size():
    size = _lib.load().nt_chunk_attention_workspace_size
    for cache in (_lib.DTYPE_F16, _lib.DTYPE_E4M3):
        assert size(0, 4, 8, 8, 128, 16, 8, cache) == 0 and size(4, 4, 8, 3, 128, 16, 8, cache) == 0
        assert size(1, 1, 8, 8, 128, 16, 8, cache) == 0  # two tiles of keys at most: one workgroup
        assert size(1, 1, 8, 8, 128, 16, 100, cache) > 0
        assert size(10**6, 300, 512, 512, 128, 16, 1000, cache) == 0  # a head a workgroup
        assert size(10**6, 300, 32, 8, 128, 32, 1000, cache) < 100 << 20


# ------------------------------------------------------------------------------- 4-bit weights
@pytest.mark.parametrize("symmetric", (False, True))
@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("group", (32, 64, 256))
def test_quantize(group, dtype, symmetric):
    w = torch.randn(7, 256, generator=torch.Generator().manual_seed(1)).to(dtype)
    w[2, :32], w[3], w[4] = 0.0, w[3].abs() + 0.5, -w[4].abs()
    weight, scales, zeros = kernels.quantize_4bit(w, group, symmetric)
    assert weight.dtype == torch.uint8 and weight.shape == (7, 128) and scales.shape == (7, 256 // group)
    assert (zeros is None) == symmetric and scales.dtype == dtype
    q = torch.stack((weight & 15, weight >> 4), -1).view(7, 256 // group, group).double()
    s = scales.double()[..., None]
    back = (q - (8.0 if symmetric else zeros.double()[..., None])) * s
    x = w.double().view_as(back)
    # Half a step of the group (a whole one at the ends, for the zero point's rounding), and of the rounded scale what 15
    # steps gather: 15 steps times the type's half step, plus 2^-20 for the products in 32 bits.
    tol = s * (1.0 if not symmetric else 0.5) + 15 * s * (torch.finfo(dtype).eps / 2) + s * 2.0**-20
    assert ((back - x).abs() <= tol).all()
    assert (back[2, : 32 // group or 1][..., :32] == 0).all() or group > 32
    with pytest.raises(ValueError):
        kernels.quantize_4bit(w, 48)
    with pytest.raises(TypeError):
        kernels.quantize_4bit(w.float())
