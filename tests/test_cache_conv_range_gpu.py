"""The single-token convolution at the ends of the scales' range, in both kernels: blocks whose scale times a tap passes
32 bits or falls below their normal numbers, blocks of zeros, blocks that are NaN."""
import pytest
import torch

import mx_reference as ref
from test_seq_cache_gpu import KINDS, Model, _cu, _step, ops  # noqa: F401

gpu = pytest.mark.gpu
# channels, heads: the direct kernel with a tap per channel, per block, per 16 channels, for groups of 8; then the ring
# with a tap per channel and per block
FORMS = [(96, 96), (96, 3), (96, 6), (96, 12), (1024, 1024), (1024, 32)]
TAPS = [torch.float32, torch.bfloat16]


def _store(m, parts):
    """tokens of every sequence, fp32"""
    counts = [len(p) for p in parts]
    starts = torch.zeros(len(parts), dtype=torch.int32, device="cuda")
    m.ops.cache_append(m.cache, torch.cat(parts).cuda(), _cu(counts).cuda(), starts)
    m.rows = [ref.stored(p, m.kind) for p in parts]


def _subnormal(terms):
    """each of the products may round in the subnormals, by half of their spacing; the gate's product once more"""
    return (terms + 1) * 2.0 ** -150


@gpu
@pytest.mark.parametrize("batch", [1, 2, 5])
@pytest.mark.parametrize("taps_dtype", TAPS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", KINDS)
def test_large_scales(ops, kind, form, taps_dtype, batch):  # noqa: F811
    """1e38 in one channel of a block: its neighbours, zeros and small values, keep their finite products with a tap that
    is above 2^128 over the block's scale"""
    channels, heads = form
    m = Model(ops, batch, 100, channels, 16, kind)
    # scale 2^124 (mx4) or 2^118 (mx8); the tap times it is 2^128 or more, times the small value beside 1e38 it is not
    big, small = (16.0, 2.0 ** 123) if kind == "mx4" else (4096.0, 2.0 ** 110)
    parts = []
    for b in range(batch):
        x = torch.randn(100 - 7 * b, channels, generator=m.g)
        for t in (0, len(x) // 2, len(x) - 1):
            x[t] = 0.0
            x[t, 0::32] = 1e38
        x[-1, 1::32], x[-1, 2::32] = small, -small
        parts.append(x)
    _store(m, parts)
    taps = (big * torch.randint(0, 2, (90, heads), generator=m.g) * 2 - big).to(taps_dtype)
    want, tol = _step(m, taps, None, torch.float32)
    absolute = torch.stack([(r.flip(0)[:90].abs() * taps[:len(r)].double().abs().repeat_interleave(channels // heads, 1)).sum(0)
                            for r in m.rows])
    finite = absolute < 1.9 * 2.0 ** 127                 # no partial sum can pass 32 bits
    assert bool(finite.view(batch, -1, 32)[:, :, 1:].all())
    got = ops.cache_conv(m.cache, m.lengths.cuda(), taps.cuda(), dtype=torch.float32).cpu().double()
    err = (got - want).abs()
    assert bool((err <= tol)[finite].all()), float(err[finite].max())


@gpu
@pytest.mark.parametrize("batch", [1, 2, 5])
@pytest.mark.parametrize("taps_dtype", TAPS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", KINDS)
def test_small_scales(ops, kind, form, taps_dtype, batch):  # noqa: F811
    """blocks at the smallest scale, with taps that take it into the subnormals: the stored values times the taps are
    rounded once each, not the scale times the tap"""
    channels, heads = form
    m = Model(ops, batch, 100, channels, 16, kind)
    top = -118 if kind == "mx8" else -124                # the largest values that scale 2^-127 still holds
    parts = [torch.randn(100 - 7 * b, channels, generator=m.g).clamp(-1.5, 1.5) * 2.0 ** top for b in range(batch)]
    _store(m, parts)
    taps = (torch.randn(90, heads, generator=m.g) * 2.0 ** -16).to(taps_dtype)
    want, tol = _step(m, taps, None, torch.float32)
    got = ops.cache_conv(m.cache, m.lengths.cuda(), taps.cuda(), dtype=torch.float32).cpu().double()
    err = (got - want).abs()
    assert bool((err <= tol + _subnormal(90)).all()), float((err - tol).max())


@gpu
@pytest.mark.parametrize("batch", [1, 2, 5])
@pytest.mark.parametrize("taps_dtype", TAPS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", KINDS)
def test_scales_of_every_size(ops, kind, form, taps_dtype, batch):  # noqa: F811
    """scales from 2^-120 to 2^110 side by side, zero blocks, zero tokens, and a NaN block, which reaches the channels of
    its block in its sequence alone"""
    channels, heads = form
    m = Model(ops, batch, 100, channels, 16, kind)
    parts = []
    for b in range(batch):
        n = 100 - 7 * b
        scale = torch.exp2(torch.randint(-110, 100, (n, channels // 32), generator=m.g).float())
        scale[torch.rand(n, channels // 32, generator=m.g) < 0.2] = 0.0
        scale[n // 3] = 0.0
        parts.append(torch.randn(n, channels, generator=m.g) * scale.repeat_interleave(32, 1))
    parts[-1][-2, 40] = float("nan")
    _store(m, parts)
    taps = torch.randn(90, heads, generator=m.g).to(taps_dtype)
    want, tol = _step(m, taps, None, torch.float32)
    got = ops.cache_conv(m.cache, m.lengths.cuda(), taps.cuda(), dtype=torch.float32).cpu().double()
    nan = torch.zeros(batch, channels, dtype=torch.bool)
    nan[-1, 32:64] = True
    assert torch.equal(torch.isnan(want), nan)
    assert torch.equal(torch.isnan(got), nan)
    err = (got - want).abs()
    assert bool((err <= tol + _subnormal(90))[~nan].all()), float((err - tol)[~nan].max())
