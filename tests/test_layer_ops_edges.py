"""What needs no GPU of the edges of a layer's operators."""

import ctypes

import pytest
import torch

from ninetoothed_amd import _lib, kernels

INVALID, P = 1, 1 << 12  # (an address that nothing reads: each call returns before a launch)


@pytest.mark.parametrize("pages,width", ((5, 0), (0, 0), (0, 64)))
@pytest.mark.parametrize("tokens", (1, 300, 2000, 10**6))
def test_chunk_workspace_of_calls_without_keys(tokens, pages, width):
    # Without keys a call splits its rows over workgroups all the same, and says what it needs for that.
    lib, strides = _lib.load(), (ctypes.c_int64 * 3)(128, 64, 1)
    nbytes = lib.nt_chunk_attention_workspace_size(tokens, 2, 8, 2, 64, 16, width, _lib.DTYPE_F16)
    without = lib.nt_chunk_attention_workspace_size(tokens, 2, 8, 2, 64, 16, 0, _lib.DTYPE_F16)
    assert nbytes >= without and (without > 0 or tokens == 1)
    if without:
        assert lib.nt_chunk_attention(P, strides, P, strides, P, strides, 1, None, None, P, strides, 1, P, width, P, P, tokens, 2,
                                      8, 2, 64, pages, 16, width, 1.0, 1, None, P, without - 1) == INVALID
    assert lib.nt_chunk_attention_workspace_size(tokens, 2, 8, 2, 64, 16, -1, _lib.DTYPE_F16) == 0


def test_quantized_weights_keep_no_graph():
    # (of a parameter: scales that ask for a gradient would keep its copy in fp32 alive)
    w = torch.nn.Parameter(torch.randn(8, 64).to(torch.float16))
    for symmetric in (False, True):
        assert not any(t.requires_grad for t in kernels.quantize_4bit(w, 32, symmetric) if t is not None)


def test_quantized_weights_lie_row_by_row():
    # linear_4bit reads rows of 16 bytes at a time; what the weights were made from may lie in any order
    w = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    for symmetric in (False, True):
        want = kernels.quantize_4bit(w, 32, symmetric)
        for other in (w.t().contiguous().t(), torch.cat([w, w], 1)[:, :128], w.repeat_interleave(2, 0)[::2]):
            got = kernels.quantize_4bit(other, 32, symmetric)
            for a, b in zip(got, want):
                assert a is b is None or (torch.equal(a, b) and a.is_contiguous())
