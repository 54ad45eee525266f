"""Calls whose workgroups pass the 2^32 threads of one launch, which a larger grid leaves out without an error: softmax
takes several launches, attention refuses the call."""

import ctypes

import pytest
import torch

from ninetoothed_amd import _lib, kernels

INVALID = 1
S4 = (ctypes.c_int64 * 4)(64, 64, 64, 1)
P = 1 << 12  # an address that nothing reads: the calls return before a launch


@pytest.mark.parametrize("entry,batch,queries,dim", (
    ("nt_attention_f16", 1 << 17, 1, 64),  # 256 threads a query block
    ("nt_attention_bf16", 1 << 16, 200, 64),  # 512
    ("nt_attention_f16", 1 << 17, 100, 63),  # 256
    ("nt_attention_f32", 1 << 19, 1, 64),  # 64
))
def test_attention_refuses_more_blocks_than_a_launch_takes(entry, batch, queries, dim):
    fn = getattr(_lib.load(), entry)
    args = (P, S4, P, S4, P, S4, P, S4, {"f16": 1, "bf16": 2, "f32": 0}[entry.rsplit("_", 1)[1]])
    assert fn(*args, batch, 128, queries, 8, dim, 1.0, 0, None) == INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("out", (torch.float16, torch.float32))
def test_softmax_of_more_segments_than_one_launch_takes(out):
    rows = (1 << 24) + 1027
    x = (torch.arange(3 * rows, device="cuda").remainder(1009) / 256).to(torch.float16).view(3, rows).t()
    y = torch.zeros(3, rows, dtype=out, device="cuda").t()
    kernels.softmax(x, y)
    # the largest is 1 at most: half a step of its rounding, and exp's and the quotient's in 32 bits
    tol = (2.0**-12 if out == torch.float16 else 0) + 2.0**-20
    for a in range(0, rows, 1 << 22):
        part = slice(a, a + (1 << 22))
        assert (y[part].double() - torch.softmax(x[part].double(), 1)).abs().max() < tol
    # and of one long row, in segments of two
    n = 2 * rows
    x = (torch.arange(2 * n, device="cuda").remainder(1009) / 256).to(torch.float16)[None, ::2]
    y = torch.zeros(1, n, dtype=out, device="cuda")
    kernels.softmax(x, y, block=2)
    assert (y.view(-1, 2).double() - torch.softmax(x.reshape(-1, 2).double(), 1)).abs().max() < tol
