"""Calls with nothing in them: no columns under leading dimensions, a cache of no sequences read through the C entry."""
import ctypes as ct

import pytest
import torch

from test_mx4_gpu import TYPES, ops  # noqa: F401

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("lead", [(2, 3), (4,), (2, 0), (3, 2, 5)])
def test_linear_without_columns(ops, lead):  # noqa: F811
    """a sum of no terms: the bias, for any leading dimensions"""
    w, bias = ops.mx4_quantize(torch.empty(7, 0, device="cuda")), torch.arange(7.0, device="cuda")
    got = ops.mx4_linear(torch.empty(*lead, 0, device="cuda"), w, bias)
    assert got.shape == (*lead, 7) and torch.equal(got, bias.expand(*lead, 7))
    assert bool((ops.mx4_linear(torch.empty(*lead, 0, device="cuda"), w) == 0).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_read_of_no_sequences(ops, dtype):  # noqa: F811
    """every token is outside cu: zeros, through the C entry as through the Python one, and nothing beside the rows"""
    from fufft_b200._lib import lib
    none = ops.seq_cache(0, 16, 64, torch.zeros(0, 0, dtype=torch.int32, device="cuda"))
    cu, starts = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    for tokens in (1, 5, 300):
        out = torch.full((tokens, 80), 7.0, dtype=dtype, device="cuda")
        rc = lib().fufft_cache_read(ct.addressof(none.desc), out[:, 8:].data_ptr(), TYPES.index(dtype), 80, cu.data_ptr(),
                                    starts.data_ptr() or None, tokens, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert bool((out[:, 8:72] == 0).all()) and bool((out[:, :8] == 7).all()) and bool((out[:, 72:] == 7).all())
        assert bool((ops.cache_read(none, cu, starts, tokens, dtype) == 0).all())
