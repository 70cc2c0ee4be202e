"""The convolution ring where scales are read byte by byte (channel counts that are no multiple of 128) and where the chunks
of channels have a ragged last one, against the stored values in 64 bits."""
import pytest
import torch

import mx_reference as ref
from test_seq_cache_gpu import KINDS, _cu, ops  # noqa: F401

gpu = pytest.mark.gpu
# channels, heads, batch, longest: histories above 64 MB, the ring's condition for such channel counts
FORMS = [(2112, 2112, 5, 8000), (2112, 66, 5, 16000), (2112, 22, 3, 24000), (1088, 1088, 9, 12000), (576, 576, 37, 8192), (1984, 62, 37, 5000)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
def test_ring_of_odd_channels(ops, form, kind):  # noqa: F811
    channels, heads, batch, longest = form
    g = torch.Generator(device="cuda").manual_seed(51)
    page = 48
    per = -(-longest // page)
    table = torch.randperm(batch * per, device="cuda", generator=g).view(batch, per).int()
    cache = ops.seq_cache(batch * per, page, channels, table, kind)
    cache.codes.random_(0, 256, generator=g)
    if kind == "mx8":
        cache.codes.bitwise_and_(0xBF)               # below the code of NaN
    cache.scales.random_(120, 131, generator=g)
    lengths = [max(0, longest - 331 * b) if b % 4 != 2 else 17 * b for b in range(batch)]
    lengths[batch // 2] = 0
    cache.scales[table[0, 5].long(), 7, 1::3] = 0    # blocks whose scale is no half-precision number, and NaN
    cache.scales[table[0, 9].long(), 3, 4] = 255
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cu, zero = _cu(lengths).cuda(), torch.zeros(batch, dtype=torch.int32, device="cuda")
    stored = ops.cache_read(cache, cu, zero, sum(lengths), torch.float32).split(lengths)
    for taps_dtype in (torch.float32, torch.bfloat16):
        taps = torch.randn(longest - 100, heads, device="cuda", generator=g).to(taps_dtype)
        got = ops.cache_conv(cache, lens, taps, dtype=torch.float32)
        assert torch.equal(torch.nan_to_num(ops.cache_conv(cache, lens, taps, dtype=torch.float32)), torch.nan_to_num(got))
        for b, v in enumerate(stored):
            t = v.flip(0)[:len(taps)].double() * taps[:len(v)].double().repeat_interleave(channels // heads, 1)
            want, tol = t.sum(0), ref.sum_tolerance(t.sum(0), t.abs().sum(0), len(t), torch.float32)
            assert torch.equal(torch.isnan(got[b]), torch.isnan(want))
            there = ~torch.isnan(want)
            assert bool(((got[b].double() - want).abs() <= tol)[there].all())
