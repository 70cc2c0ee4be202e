"""Gradients of the 4-bit product where activations and weights differ in type: each is the 64-bit product within the bound
of one rounding to its own type."""
import pytest
import torch

from test_mx4_gpu import TYPES, _product, ops  # noqa: F401

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("w_dtype", TYPES)
@pytest.mark.parametrize("x_dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 130, 70), (300, 65, 513)])
def test_each_gradient_in_its_type(ops, shape, x_dtype, w_dtype):  # noqa: F811
    import fufft_b200.torch_ops as torch_ops
    m, n, k = shape
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(m, k, generator=g).to(x_dtype), torch.randn(n, k, generator=g).to(w_dtype)
    gy = (torch.randn(m, n, generator=g) * 2.0 ** -8).to(x_dtype)
    dx, dw = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    gx, gw = torch.autograd.grad(torch_ops.mx4_linear_train(dx, dw), (dx, dw), gy.cuda())
    xt, wt = ops.mx4_quantize(x.cuda(), transpose=True), ops.mx4_quantize(w.cuda(), transpose=True)
    direct = ops.mx4_linear_grad(gy.cuda(), xt, wt, w_dtype=w_dtype)
    for got, same, dtype, (want, tol) in ((gx, direct[0], x_dtype, _product(gy, w.t(), None, x_dtype)),
                                          (gw, direct[1], w_dtype, _product(gy.t(), x.t(), None, w_dtype))):
        assert got.dtype == dtype and torch.equal(got, same)
        err = (got.cpu().double() - want).abs()
        assert bool((err <= tol).all()), float((err - tol).max())


def test_weight_gradient_type_of_the_fake():
    import fufft_b200.torch_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    f = torch.ops.fufft
    with FakeTensorMode():
        x, w = torch.empty(7, 300, dtype=torch.bfloat16), torch.empty(130, 300)
        y, *kept = f.mx4_train(x, w)
        gx, gw = f.mx4_train_grad(y, *kept, torch.float32)
        assert (gx.dtype, gw.dtype) == (torch.bfloat16, torch.float32) and gw.shape == w.shape
        gx, gw = f.mx4_train_grad(y, *kept)
        assert (gx.dtype, gw.dtype) == (torch.bfloat16, torch.bfloat16)
