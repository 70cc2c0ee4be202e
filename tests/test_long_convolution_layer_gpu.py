"""The example layer: stepping through the cache gives what the whole prompt
gives, training in 4 bits learns; and the torch.ops forms of the operators."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.gpu
@pytest.mark.parametrize("width,tokens", [(64, 100), (256, 300)])
def test_layer(width, tokens):
    """The two ways differ by fp32 rounding of the convolution, then by bfloat16 and 4-bit rounding of y that
    those differences tip over: a value of y on the edge between two codes moves by a quarter of itself at most
    (2^-2), and of bfloat16 values at most one in 2^8 * 2^-16 ~ 1% is that near an edge after an error of 2^-16, so
    the result is off by about sqrt(0.01) * 2^-2 < 5%."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import long_convolution_layer as example
    got = example.main(width=width, tokens=tokens, steps=5)
    assert got["stepped against whole prompt"] < 0.05
    assert got["last loss"] < 0.1 * got["first loss"]


def test_ops_registered_with_fake_shapes():
    import fufft_b200.torch_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    f = torch.ops.fufft
    with FakeTensorMode():
        x, w = torch.empty(7, 300, dtype=torch.bfloat16), torch.empty(130, 300, dtype=torch.bfloat16)
        codes, scales = f.mx4_quantize(w, False)
        assert codes.shape == (130, 256) and scales.shape == (2, 4, 32, 4, 4)
        assert f.mx4_quantize(w, True)[0].shape == (300, 128)
        assert f.mx4_linear(x, codes, scales, 130, None).shape == (7, 130)
        y, *kept = f.mx4_train(x, w)
        assert y.shape == (7, 130)
        gx, gw = f.mx4_train_grad(y, *kept)
        assert gx.shape == x.shape and gw.shape == w.shape
        c, s, t = torch.empty(9, 16, 64, dtype=torch.uint8), torch.empty(9, 16, 2, dtype=torch.uint8), torch.empty(2, 4, dtype=torch.int32)
        i = torch.empty(2, dtype=torch.int32)
        assert f.cache_read(c, s, t, "mx8", torch.empty(3, dtype=torch.int32), i, 5, torch.float16).shape == (5, 64)
        assert f.cache_read_channels(c, s, t, "mx8", i, i, 32).shape == (2, 64, 32)
        assert f.cache_conv(c, s, t, "mx8", i, torch.empty(8, 64), None, torch.float32).shape == (2, 64)


@pytest.mark.gpu
def test_ops_match_direct_calls():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import fufft_b200.torch_ops as torch_ops
    from fufft_b200 import ops
    f = torch.ops.fufft
    x, w = torch.randn(7, 300, device="cuda"), torch.randn(130, 300, device="cuda")
    q = ops.mx4_quantize(w)
    codes, scales = f.mx4_quantize(w, False)
    assert torch.equal(codes, q.codes)
    assert torch.equal(f.mx4_linear(x, codes, scales, 130, None), ops.mx4_linear(x, q))
    x.requires_grad_()
    w.requires_grad_()
    y = torch_ops.mx4_linear_train(x, w)
    gy = torch.randn_like(y)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    want = ops.mx4_linear_grad(gy, ops.mx4_quantize(x.detach(), transpose=True), ops.mx4_quantize(w.detach(), transpose=True))
    assert torch.equal(gx, want[0]) and torch.equal(gw, want[1])
    table = torch.tensor([[1, 0], [2, 3]], dtype=torch.int32, device="cuda")
    cache = ops.seq_cache(4, 4, 64, table, "mx4")
    v = torch.randn(10, 64, device="cuda")
    cu, zero, n = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 6, 10], [0, 0], [6, 4]))
    parts = cache.codes, cache.scales, table, "mx4"
    f.cache_append(v, *parts, cu, zero)
    read = f.cache_read(*parts, cu, zero, 10, torch.float32)
    assert torch.equal(read, ops.cache_read(cache, cu, zero, 10, torch.float32)) and bool((read != 0).any())
    assert torch.equal(f.cache_read_channels(*parts, zero, n, 16), ops.cache_read_channels(cache, zero, n, 16))
    taps = torch.randn(8, 64, device="cuda")
    assert torch.equal(f.cache_conv(*parts, n, taps, None, torch.float32), ops.cache_conv(cache, n, taps, dtype=torch.float32))
