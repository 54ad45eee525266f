"""Edges of the checks of the operators around a paged key/value cache, on the CPU."""

import pytest

from ninetoothed_amd import kernels

from test_cache_ops import append_args, step_args, z


def test_an_append_takes_heads_of_whole_fours_and_attention_of_sixteens():
    def heads(args, dim, names):
        return {**args, **{n: z(*args[n].shape[:-1], dim, dtype=args[n].dtype) for n in names}}

    for eight in (False, True):
        for dim in (4, 20, 36, 124, 128):
            kernels.check_cache_append(**heads(append_args(eight), dim, ("k", "v", "k_cache", "v_cache")))
        for dim in (2, 6, 18, 132):
            with pytest.raises(ValueError, match="multiple of 4 up to 128"):
                kernels.check_cache_append(**heads(append_args(eight), dim, ("k", "v", "k_cache", "v_cache")))
        for dim in (4, 20, 36, 144):
            with pytest.raises(ValueError, match="multiple of 16 up to 128"):
                kernels.check_cache_attention(**heads(step_args(eight), dim, ("q", "out", "k_cache", "v_cache")))
