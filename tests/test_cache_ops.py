"""Refusals of the operators around a paged key/value cache: on the CPU, before any launch.

Every ``check_<op>`` runs without a device or the library; a call on CPU tensors that passes it is
refused for its device.  The C entry points return their status before they launch anything.
"""

import ctypes

import pytest
import torch

from ninetoothed_amd import _lib, kernels

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
INVALID = 1


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def rotary_args(**change):
    a = dict(x=torch.zeros(3, 2, 64, dtype=F16), positions=torch.arange(3), freqs=torch.ones(32, dtype=torch.float64),
             out=torch.zeros(3, 2, 64, dtype=F16))
    return {**a, **change}


def append_args(eight=False, **change):
    cache = torch.zeros(5, 16, 2, 64, dtype=E4M3 if eight else F16)
    a = dict(k=torch.zeros(3, 2, 64, dtype=F16), v=torch.zeros(3, 2, 64, dtype=F16), k_cache=cache, v_cache=cache.clone(),
             tables=torch.zeros(2, 2, dtype=torch.int32), lengths=_i32(0, 4), starts=_i32(0, 1, 3))
    if eight:
        a |= dict(k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2))
    return {**a, **change}


def prompt_args(**change):
    a = dict(q=torch.zeros(5, 4, 64, dtype=F16), k=torch.zeros(7, 2, 64, dtype=F16), v=torch.zeros(7, 2, 64, dtype=F16),
             out=torch.zeros(5, 4, 64, dtype=F16), q_starts=_i32(0, 2, 5), k_starts=_i32(0, 3, 7))
    return {**a, **change}


def step_args(eight=False, **change):
    cache = torch.zeros(5, 16, 2, 64, dtype=E4M3 if eight else F16)
    a = dict(q=torch.zeros(2, 4, 64, dtype=F16), k_cache=cache, v_cache=cache.clone(),
             tables=torch.zeros(2, 2, dtype=torch.int32), lengths=_i32(3, 4), out=torch.zeros(2, 4, 64, dtype=F16))
    if eight:
        a |= dict(k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2))
    return {**a, **change}


OPS = {"rotary": rotary_args, "cache_append": append_args, "prompt_attention": prompt_args, "cache_attention": step_args}


@pytest.mark.parametrize("op", OPS)
def test_a_good_call_passes_its_check_and_is_refused_for_its_device(op):
    args = OPS[op]()
    getattr(kernels, f"check_{op}")(**args)
    with pytest.raises(TypeError, match="GPU"):
        getattr(kernels, op)(**args)


@pytest.mark.parametrize("op", ("cache_append", "cache_attention"))
def test_8_bit_caches_pass(op):
    assert getattr(kernels, f"check_{op}")(**OPS[op](eight=True)) == _lib.DTYPE_E4M3


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


BAD = [
    ("rotary", dict(x=z(3, 128), out=z(3, 128)), ValueError),
    ("rotary", dict(out=z(3, 2, 32)), ValueError),
    ("rotary", dict(out=z(3, 2, 64, dtype=BF16)), TypeError),
    ("rotary", dict(x=z(3, 2, 64, dtype=torch.float64), out=z(3, 2, 64, dtype=torch.float64)), TypeError),
    ("rotary", dict(positions=torch.arange(4)), ValueError),
    ("rotary", dict(positions=torch.zeros(3)), TypeError),
    ("rotary", dict(freqs=torch.ones(32)), TypeError),
    ("rotary", dict(freqs=torch.ones(33, dtype=torch.float64)), ValueError),
    ("rotary", dict(freqs=torch.ones(64, dtype=torch.float64)[::2]), ValueError),
    ("rotary", dict(out=z(3, 1, 64).expand(3, 2, 64)), ValueError),
    ("rotary", dict(x=z(3, 2, 514), out=z(3, 2, 514)), ValueError),
    ("cache_append", dict(v=z(3, 2, 32)), ValueError),
    ("cache_append", dict(v=z(3, 2, 64, dtype=BF16)), TypeError),
    ("cache_append", dict(k=z(3, 2, 64, dtype=torch.float32), v=z(3, 2, 64, dtype=torch.float32)), TypeError),
    ("cache_append", dict(k_cache=z(5, 16, 2, 64, dtype=BF16), v_cache=z(5, 16, 2, 64, dtype=BF16)), TypeError),
    ("cache_append", dict(k_cache=z(5, 16, 3, 64), v_cache=z(5, 16, 3, 64)), ValueError),
    ("cache_append", dict(v_cache=z(5, 8, 2, 64)), ValueError),
    ("cache_append", dict(k_cache=z(5, 16, 64, 2).transpose(2, 3), v_cache=z(5, 16, 2, 64)), ValueError),
    ("cache_append", dict(k_cache=z(1, 16, 2, 64).expand(5, 16, 2, 64)), ValueError),
    ("cache_append", dict(k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2)), ValueError),
    ("cache_append", dict(eight=True, k_scale=None), ValueError),
    ("cache_append", dict(eight=True, v_scale=torch.ones(2, 5)), ValueError),
    ("cache_append", dict(eight=True, v_scale=torch.ones(2, 5).t()), ValueError),
    ("cache_append", dict(eight=True, k_scale=torch.ones(5, 2, dtype=F16)), TypeError),
    ("cache_append", dict(eight=True, k_cache=z(5, 256, 2, 64, dtype=E4M3), v_cache=z(5, 256, 2, 64, dtype=E4M3)), ValueError),
    ("cache_append", dict(tables=torch.zeros(2, 2, dtype=torch.int64)), TypeError),
    ("cache_append", dict(tables=torch.zeros(2, 2, dtype=torch.int32).t()), ValueError),
    ("cache_append", dict(tables=torch.zeros(3, 2, dtype=torch.int32)), ValueError),
    ("cache_append", dict(lengths=torch.zeros(2, dtype=torch.int64)), TypeError),
    ("cache_append", dict(lengths=torch.zeros(4, dtype=torch.int32)[::2]), ValueError),
    ("cache_append", dict(starts=_i32(0, 3)), ValueError),
    ("cache_append", dict(starts=torch.tensor([0, 1, 3])), TypeError),
    ("cache_append", dict(freqs=torch.ones(33, dtype=torch.float64)), ValueError),
    ("prompt_attention", dict(out=z(5, 2, 64)), ValueError),
    ("prompt_attention", dict(v=z(6, 2, 64)), ValueError),
    ("prompt_attention", dict(out=z(5, 4, 64, dtype=BF16)), TypeError),
    ("prompt_attention", dict(k=z(7, 2, 32), v=z(7, 2, 32)), ValueError),
    ("prompt_attention", dict(k=z(7, 3, 64), v=z(7, 3, 64)), ValueError),
    ("prompt_attention", dict(k=z(7, 0, 64), v=z(7, 0, 64)), ValueError),
    ("prompt_attention", dict(q=z(5, 4, 136), k=z(7, 2, 136), v=z(7, 2, 136), out=z(5, 4, 136)), ValueError),
    ("prompt_attention", dict(q_starts=_i32(0, 5)), ValueError),
    ("prompt_attention", dict(k_starts=torch.tensor([0, 3, 7])), TypeError),
    ("prompt_attention", dict(q_starts=_i32()), ValueError),
    ("prompt_attention", dict(out=z(5, 1, 64).expand(5, 4, 64)), ValueError),
    ("cache_attention", dict(out=z(2, 4, 32)), ValueError),
    ("cache_attention", dict(out=z(2, 4, 64, dtype=BF16)), TypeError),
    ("cache_attention", dict(q=z(2, 3, 64), out=z(2, 3, 64)), ValueError),
    ("cache_attention", dict(q=z(2, 4, 72), out=z(2, 4, 72), k_cache=z(5, 16, 2, 72), v_cache=z(5, 16, 2, 72)), ValueError),
    ("cache_attention", dict(q=z(2, 4, 144), out=z(2, 4, 144), k_cache=z(5, 16, 2, 144), v_cache=z(5, 16, 2, 144)), ValueError),
    ("cache_attention", dict(k_cache=z(16, 2, 64)), ValueError),
    ("cache_attention", dict(tables=torch.zeros(3, 2, dtype=torch.int32), lengths=_i32(1, 2, 3)), ValueError),
    ("cache_attention", dict(lengths=_i32(1, 2, 3)), ValueError),
    ("cache_attention", dict(k_cache=z(5, 16, 2, 68)[..., :64], v_cache=z(5, 16, 2, 64)), ValueError),
    ("cache_attention", dict(eight=True, v_scale=None), ValueError),
    ("cache_attention", dict(out=z(2, 1, 64).expand(2, 4, 64)), ValueError),
]


@pytest.mark.parametrize("op,change,error", BAD, ids=[f"{op}-{i}" for i, (op, _, _) in enumerate(BAD)])
def test_bad_calls_are_refused(op, change, error):
    with pytest.raises(error):
        getattr(kernels, f"check_{op}")(**OPS[op](**change))


def test_frequencies():
    f = kernels.rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert torch.allclose(kernels.rotary_frequencies(8, base=100.0, factor=4.0, device="cpu"), f / 4)
    # over 200 positions: 31.8, 10.1, 3.2 and 1.007 turns; kept from 10 on, divided up to 2
    g = kernels.rotary_frequencies(8, base=100.0, factor=4.0, original_length=200, low=2.0, high=10.0, device="cpu")
    kept = (200 * 0.1 / (2 * torch.pi) - 2.0) / 8.0
    assert torch.allclose(g / f, torch.tensor([1.0, 1.0, kept + (1 - kept) / 4, 0.25], dtype=torch.float64))
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, factor=0.0), dict(dim=8, low=2.0, high=2.0)):
        with pytest.raises(ValueError):
            kernels.rotary_frequencies(device="cpu", **bad)


# ------------------------------------------------------------------ the C entry points, unlaunched
S3 = (ctypes.c_int64 * 3)(128, 64, 1)
P = 1 << 12  # an address that nothing reads: each call returns before a launch


def _rotary(lib, dtype=1, bits=32, tokens=4, heads=2, dim=64, pairs=32, x=P, freqs=P):
    return lib.nt_rotary(x, S3, P, S3, dtype, P, 1, bits, freqs, tokens, heads, dim, pairs, 0, 0, 1.0, None)


def _append(lib, dtype=1, cache=1, k=P, scale=P, tokens=4, seqs=2, heads=2, dim=64, pages=5, page=16, width=2, pairs=0):
    return lib.nt_cache_append(k, S3, P, S3, dtype, P, S3, P, S3, cache, scale, scale, P, 2, P, P, None, tokens, seqs, heads,
                               dim, pages, page, width, pairs, 0, 1.0, None)


def _prompt(lib, dtype=1, q=P, tokens=4, keys=4, seqs=2, heads=2, kv=2, dim=64):
    return lib.nt_prompt_attention(q, S3, P, S3, P, S3, P, S3, dtype, P, P, tokens, keys, seqs, heads, kv, dim, 1.0, 1, None,
                                   None, 0)


def _step(lib, dtype=1, cache=1, q=P, scale=P, seqs=2, heads=2, kv=2, dim=64, pages=5, page=16, width=2, ws=None, nbytes=0,
          strides=S3, k=P):
    return lib.nt_cache_attention(q, S3, k, strides, P, strides, cache, scale, scale, P, S3, dtype, P, 2, P, seqs, heads, kv, dim,
                                  pages, page, width, 1.0, None, ws, nbytes)


def test_entry_points_reject_before_they_launch():
    lib = _lib.load()
    for bad in (dict(dtype=3), dict(bits=16), dict(tokens=-1), dict(dim=514), dict(pairs=33), dict(x=None), dict(freqs=None)):
        assert _rotary(lib, **bad) == INVALID, bad
    for bad in (dict(dtype=0), dict(cache=2), dict(k=None), dict(tokens=-1), dict(dim=132), dict(dim=62), dict(page=0),
                dict(cache=4, scale=None), dict(cache=4, page=129), dict(pairs=33), dict(pairs=8)):
        assert _append(lib, **bad) == INVALID, bad
    for bad in (dict(dtype=0), dict(q=None), dict(dim=129), dict(kv=0), dict(heads=3), dict(keys=-1), dict(seqs=-1)):
        assert _prompt(lib, **bad) == INVALID, bad
    # 2 pages of 16 are one block of keys: no workspace; 128 of them want one
    for bad in (dict(dtype=0), dict(cache=2), dict(q=None), dict(dim=72), dict(dim=144), dict(kv=0), dict(heads=3), dict(page=0),
                dict(cache=4, scale=None), dict(width=128), dict(width=128, ws=P, nbytes=64), dict(k=P + 8),
                dict(strides=(ctypes.c_int64 * 3)(128, 60, 1)), dict(page=1 << 20, width=1 << 12)):
        assert _step(lib, **bad) == INVALID, bad
    # nothing to do: no launch, no error, whatever the pointers
    assert _rotary(lib, tokens=0, x=None) == 0
    assert _append(lib, tokens=0, k=None) == 0 and _append(lib, pages=0) == 0 and _append(lib, seqs=0) == 0
    assert _prompt(lib, tokens=0, q=None) == 0 and _prompt(lib, seqs=0) == 0
    assert _step(lib, seqs=0, q=None) == 0
    for name in ("rotary", "cache_append", "prompt_attention", "cache_attention"):
        assert getattr(lib, f"nt_{name}_packed")(None) == INVALID
    # sizes whose product passes 64 bits are no empty call (2^16 tokens of 2^8 sequences, ..., 2^64 in all)
    big = dict(tokens=1 << 16, seqs=1 << 8, heads=1 << 3, dim=1 << 7, pages=1 << 20, width=1 << 10, k=None)
    assert _append(lib, **big) == INVALID
    assert _prompt(lib, tokens=1 << 30, seqs=1 << 20, heads=1 << 8, kv=1 << 8, dim=1 << 6, q=None) == INVALID
    assert _rotary(lib, tokens=1 << 33, heads=1 << 20, dim=1 << 9, x=None) == INVALID


def test_workspace_size():
    size = _lib.load().nt_prompt_attention_workspace_size
    assert size(100000, 100000, 4, 32, 8, 128) == 0  # rows enough for every workgroup
    assert size(0, 100, 1, 8, 8, 64) == 0 and size(10, 100, 1, 8, 3, 64) == 0
    assert size(100, 50000, 1, 8, 8, 64) > 0
    size = _lib.load().nt_cache_attention_workspace_size
    for cache in (_lib.DTYPE_F16, _lib.DTYPE_E4M3):
        assert size(4, 8, 8, 128, 16, 8, cache) == 0  # at most one block of keys a sequence
        assert size(0, 8, 8, 128, 16, 100, cache) == 0
        assert size(1, 8, 8, 128, 16, 100, cache) > 0
        assert size(100, 32, 8, 128, 32, 1000, cache) < 32 << 20
