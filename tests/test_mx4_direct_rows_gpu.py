"""Rows quantised inside the product, over summed axes that go round its ring of stages and are split over a cluster (the
last CTAs of which may have nothing to sum), at the limit of that path and one row above it: as rows quantised before the
product, to the last bit, and within the derived bound of the 64-bit product."""
import pytest
import torch

import mx_reference as ref
from test_mx4_gpu import TYPES, _values, ops  # noqa: F401
from fufft_b200._lib import MX4_DIRECT_ROWS

gpu = pytest.mark.gpu
ROWS = range(1, MX4_DIRECT_ROWS + 2)
LONG = [257, 1000, 1111, 1300, 4096, 4396, 8192]   # 4396: 18 chunks, over eight CTAs of three


def _weights(ops, n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(n, k, device="cuda", generator=g) * 0.3
    return w, ops.mx4_quantize(w), torch.randn(n, device="cuda", generator=g)


def _same(got, want):
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))


def _bounds(x, stored, bias, dtype):
    qx = ref.stored(x)
    want = qx @ stored.t() + bias
    return want, ref.sum_tolerance(want, qx.abs() @ stored.abs().t() + bias.abs(), x.shape[1], dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", LONG)
@pytest.mark.parametrize("n", [130, 2500])
def test_long_sums(ops, n, k, dtype):  # noqa: F811
    w, q, bias = _weights(ops, n, k, 8)
    stored = ref.stored(w.cpu())
    for m in ROWS:
        x = _values((m, k + 1), dtype, m)
        for off in (0, 1):                    # wide loads, and rows from any address
            d = x.cuda()[:, off:off + k]
            got = ops.mx4_linear(d, q, bias, dtype=torch.float32)
            _same(got, ops.mx4_matmul(ops.mx4_quantize(d), q, torch.float32, bias))
            want, tol = _bounds(x[:, off:off + k], stored, bias.cpu().double(), torch.float32)
            err = (got.cpu().double() - want).abs()
            assert bool((err <= tol).all()), float((err - tol).max())


@gpu
@pytest.mark.parametrize("k", LONG)
def test_nan_block_anywhere(ops, k):  # noqa: F811
    """a block that is NaN, in the first chunk, inside and in the ragged last one: its row alone"""
    _, q, bias = _weights(ops, 300, k, 9)
    for m in ROWS:
        for at in (0, k // 2, k - 1):
            x = torch.randn(m, k, device="cuda")
            x[m - 1, at] = float("inf")
            got = ops.mx4_linear(x, q, bias)
            assert bool(torch.isnan(got[m - 1]).all()) and not bool(torch.isnan(got[:m - 1]).any())
            _same(got, ops.mx4_matmul(ops.mx4_quantize(x), q, torch.float32, bias))


@gpu
@pytest.mark.parametrize("k", [1300, 4096])
def test_unsplit_sums(ops, k):  # noqa: F811
    """enough columns that every CTA sums the whole axis: six chunks and sixteen through five stages"""
    n = 19200
    w, q, bias = _weights(ops, n, k, 10)
    stored = ref.stored(w.cpu()[::37])
    for m in ROWS:
        x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(torch.bfloat16)
        for dtype in TYPES:
            got = ops.mx4_linear(x.cuda(), q, bias, dtype=dtype)
            _same(got, ops.mx4_matmul(ops.mx4_quantize(x.cuda()), q, dtype, bias))
            want, tol = _bounds(x, stored, bias.cpu()[::37].double(), dtype)
            assert bool(((got.cpu()[:, ::37].double() - want).abs() <= tol).all())
