"""4-bit microscaled matrices: quantisation bit for bit against a plain 64-bit
restatement, products and gradients within derived bounds, refusals."""
import pytest
import torch

import mx_reference as ref

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(1, 1), (1, 32), (2, 31), (5, 33), (16, 256), (31, 257), (129, 130), (200, 1000), (257, 96), (300, 515)]


@pytest.fixture()
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from fufft_b200 import ops
    return ops


def _values(shape, dtype, seed):
    """normal values over channels of unequal size, with zero blocks, ties and saturating values among them"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-8, 8, (1, shape[1]), generator=g).double())
    pick = torch.rand(shape, generator=g)
    x = torch.where(pick < 0.05, 0.0, x)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -5.0, -0.25], dtype=torch.float64)
    x = torch.where(pick > 0.8, ties[torch.randint(0, 10, shape, generator=g)], x)
    if shape[0] > 2:
        x[1] = 0.0
    return x.to(dtype)


def _check_bits(q, x):
    codes, tiles = ref.pack(x)
    assert torch.equal(q.codes.cpu(), codes)
    assert torch.equal(ref.untile(q.scales.cpu(), x.shape[0]), ref.untile(tiles, x.shape[0]))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_bits(ops, shape, dtype):
    x = _values(shape, dtype, 1)
    d = x.cuda()
    _check_bits(ops.mx4_quantize(d), x)
    _check_bits(ops.mx4_quantize(d, transpose=True), x.t().contiguous())
    q, qt = ops.mx4_quantize_both(d)
    _check_bits(q, x)
    _check_bits(qt, x.t().contiguous())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_special_values(ops, dtype):
    fin = torch.finfo(dtype)
    x = torch.zeros(12, 96, dtype=dtype)
    x[0, 3], x[0, 40] = float("nan"), 1.0          # one NaN block, its neighbours untouched
    x[1, 32], x[2, 95] = float("inf"), float("-inf")
    x[3, :] = fin.max
    x[4, :] = fin.min
    x[5, 5] = fin.tiny
    x[6, 6] = fin.smallest_normal / 2              # a subnormal
    x[7, :] = -0.0
    x[8, :32] = torch.linspace(-6, 6, 32).to(dtype)
    x[9, 0], x[9, 1] = 1.0, fin.smallest_normal    # far below its block's scale
    x[10, 64], x[10, 65] = 7.9, -7.9               # saturates
    d = x.cuda()
    q, qt = ops.mx4_quantize_both(d)
    for got, want in ((ops.mx4_quantize(d), x), (q, x), (qt, x.t().contiguous())):
        _check_bits(got, want)
        back = ops.mx4_dequantize(got, torch.float32).cpu().double()
        assert torch.equal(torch.nan_to_num(back, nan=12345.0), torch.nan_to_num(ref.stored(want), nan=12345.0))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_and_turned(ops, dtype):
    """rows apart by more than their length, from addresses that no vector load may take, and transposed views"""
    base = _values((70, 301), dtype, 2)
    d = base.cuda()
    for r, c0, c1 in ((1, 1, 300), (3, 7, 76), (0, 8, 264)):
        _check_bits(ops.mx4_quantize(d[r:, c0:c1]), base[r:, c0:c1])
        _check_bits(ops.mx4_quantize(d[r:, c0:c1], transpose=True), base[r:, c0:c1].t())
        _check_bits(ops.mx4_quantize(d[r:, c0:c1].t()), base[r:, c0:c1].t())
        a, b = ops.mx4_quantize_both(d[r:, c0:c1].t())
        _check_bits(a, base[r:, c0:c1].t())
        _check_bits(b, base[r:, c0:c1])
    _check_bits(ops.mx4_quantize(d[::2]), base[::2])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_dequantize(ops, shape, dtype):
    x = _values(shape, dtype, 3)
    q = ops.mx4_quantize(x.cuda())
    assert torch.equal(ops.mx4_dequantize(q, dtype).cpu().double(), ref.stored(x).to(dtype).double())
    wide = torch.full((shape[0], shape[1] + 3), 7.0, dtype=dtype, device="cuda")
    ops.mx4_dequantize(q, dtype, out=wide[:, 1:1 + shape[1]])
    assert torch.equal(wide[:, 1:1 + shape[1]].cpu().double(), ref.stored(x).to(dtype).double())
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 1 + shape[1]:] == 7).all())


# m, n, k: one token, few tokens, ragged tiles, k from one block to many, more tiles than one launch holds at once
PRODUCTS = [(1, 1, 1), (1, 64, 32), (1, 4096, 1024), (2, 130, 97), (7, 257, 300), (16, 512, 4096), (17, 1000, 513), (33, 384, 256),
            (64, 127, 640), (65, 129, 255), (100, 1025, 2049), (128, 256, 512), (130, 200, 31), (255, 257, 8192), (300, 4100, 768),
            (513, 511, 1111), (1024, 1280, 384), (2000, 2300, 130)]


def _product(a, b, bias, dtype):
    qa, qb = ref.stored(a), ref.stored(b)
    want = qa @ qb.t() + (0 if bias is None else bias.double())
    absolute = qa.abs() @ qb.abs().t() + (0 if bias is None else bias.double().abs())
    return want, ref.sum_tolerance(want, absolute, a.shape[1], dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", PRODUCTS)
def test_matmul(ops, shape, dtype):
    m, n, k = shape
    g = torch.Generator().manual_seed(m + n + k)
    a, b = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g) * 0.25
    bias = torch.randn(n, generator=g) if (m + n) % 2 else None
    want, tol = _product(a, b, bias, dtype)
    got = ops.mx4_matmul(ops.mx4_quantize(a.cuda()), ops.mx4_quantize(b.cuda()), dtype, None if bias is None else bias.cuda())
    assert got.dtype == dtype and got.shape == (m, n)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@gpu
@pytest.mark.parametrize("shape", [(1, 300, 64), (5, 129, 500), (70, 257, 300), (400, 515, 700)])
def test_matmul_out_strides(ops, shape):
    """rows of the result apart by more than their length and not aligned; nothing beside them is written"""
    m, n, k = shape
    g = torch.Generator().manual_seed(9)
    a, b = torch.randn(m, k, generator=g), torch.randn(n, k, generator=g)
    want, tol = _product(a, b, None, torch.bfloat16)
    for off, pitch in ((0, n), (1, n + 1), (3, n + 8), (8, n + 24)):
        buf = torch.full((m, pitch + off), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.mx4_matmul(ops.mx4_quantize(a.cuda()), ops.mx4_quantize(b.cuda()), torch.bfloat16, out=buf[:, off:off + n])
        assert bool(((buf[:, off:off + n].cpu().double() - want).abs() <= tol).all())
        assert bool((buf[:, :off] == 7).all()) and bool((buf[:, off + n:] == 7).all())


@gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_matmul_nan_block_stays_in_its_row_and_column(ops, m):
    a, b = torch.ones(m, 200), torch.ones(140, 200)
    a[m // 2, 70] = float("nan")
    b[131, 199] = float("inf")
    got = ops.mx4_matmul(ops.mx4_quantize(a.cuda()), ops.mx4_quantize(b.cuda()), torch.float32).cpu()
    nan = torch.zeros(m, 140, dtype=torch.bool)
    nan[m // 2], nan[:, 131] = True, True
    assert torch.equal(torch.isnan(got), nan)
    assert bool((got[~nan] == 200).all())


@gpu
@pytest.mark.parametrize("m", [1, 300])
def test_matmul_extreme_scales(ops, m):
    """scales from 2^-127 up: products below, inside and above the range of 32 bits"""
    a, b = torch.zeros(m, 64), torch.zeros(130, 64)
    a[:, 0], b[:, 0] = 2.0 ** 60, 2.0 ** 50
    a[:, 33], b[:, 33] = 2.0 ** -100, 2.0 ** 20
    got = ops.mx4_matmul(ops.mx4_quantize(a.cuda()), ops.mx4_quantize(b.cuda()), torch.float32).cpu()
    assert bool((got == 2.0 ** 110).all())
    a[:, 0] = 0.0
    got = ops.mx4_matmul(ops.mx4_quantize(a.cuda()), ops.mx4_quantize(b.cuda()), torch.float32).cpu()
    assert bool((got == 2.0 ** -80).all())


@gpu
def test_empty(ops):
    for r, c in ((0, 5), (5, 0), (0, 0)):
        x = torch.empty(r, c, device="cuda")
        q, qt = ops.mx4_quantize_both(x)
        assert q.shape == (r, c) and qt.shape == (c, r)
        assert ops.mx4_dequantize(q).shape == (r, c)
    w = ops.mx4_quantize(torch.ones(7, 64, device="cuda"))
    assert ops.mx4_linear(torch.ones(0, 64, device="cuda"), w).shape == (0, 7)
    a, b = ops.mx4_quantize(torch.ones(3, 0, device="cuda")), ops.mx4_quantize(torch.ones(200, 0, device="cuda"))
    bias = torch.arange(200.0, device="cuda")
    assert torch.equal(ops.mx4_matmul(a, b, torch.float32, bias), bias.expand(3, 200))
    assert bool((ops.mx4_matmul(a, b) == 0).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_linear(ops, dtype):
    g = torch.Generator().manual_seed(4)
    x, w, bias = torch.randn(2, 3, 300, generator=g).to(dtype), torch.randn(130, 300, generator=g), torch.randn(130, generator=g)
    want, tol = _product(x.reshape(6, 300), w, bias, dtype)
    got = ops.mx4_linear(x.cuda(), ops.mx4_quantize(w.cuda()), bias.cuda())
    assert got.shape == (2, 3, 130) and got.dtype == dtype
    assert bool(((got.cpu().double().view(6, 130) - want).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 130, 1), (1, 300, 31), (2, 64, 256), (5, 129, 257), (15, 200, 1000), (16, 4096, 4096), (16, 100, 40), (17, 100, 300)])
def test_linear_few_rows(ops, shape, dtype):
    """rows quantised inside the product: as those quantised before it, to the last bit, from any address, NaN and empty
    blocks among them"""
    m, n, k = shape
    x = _values((m, k + 5), dtype, 7)
    x[m // 2, (k - 1) // 2] = float("nan")
    w = ops.mx4_quantize((torch.randn(n, k, generator=torch.Generator().manual_seed(8)) * 0.3).cuda())
    bias = torch.randn(n, generator=torch.Generator().manual_seed(9)).cuda()
    for off in (0, 1, 4):
        d = x.cuda()[:, off:off + k]
        for out in TYPES:
            got = ops.mx4_linear(d, w, bias, dtype=out)
            want = ops.mx4_matmul(ops.mx4_quantize(d), w, out, bias)
            assert got.dtype == out
            assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))
            assert torch.equal(torch.isnan(got), torch.isnan(want))


GRADS = [(1, 1, 1), (5, 130, 70), (64, 96, 32), (130, 257, 300), (300, 65, 513)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", GRADS)
def test_linear_grad_formula(ops, shape, dtype):
    m, n, k = shape
    g = torch.Generator().manual_seed(5)
    x, w, gy = torch.randn(m, k, generator=g).to(dtype), torch.randn(n, k, generator=g).to(dtype), torch.randn(m, n, generator=g).to(dtype)
    gx, gw = ops.mx4_linear_grad(gy.cuda(), ops.mx4_quantize(x.cuda(), transpose=True), ops.mx4_quantize(w.cuda(), transpose=True))
    want, tol = _product(gy, w.t(), None, dtype)
    assert bool(((gx.cpu().double() - want).abs() <= tol).all())
    want, tol = _product(gy.t(), x.t(), None, dtype)
    assert bool(((gw.cpu().double() - want).abs() <= tol).all())


@gpu
def test_linear_grad_differences(ops):
    """On values that the blocks hold exactly (multiples of a half up to 2, no rounding anywhere: sums stay whole multiples
    of a quarter below 2^22) the product is linear, so the gradient is the difference quotient, to the last bit."""
    m, n, k = 6, 40, 33
    g = torch.Generator().manual_seed(6)
    pick = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, -0.5, -1.0, -1.5, -2.0])
    x, w, gy = (pick[torch.randint(0, 9, s, generator=g)].cuda() for s in ((m, k), (n, k), (m, n)))
    gx, gw = ops.mx4_linear_grad(gy, ops.mx4_quantize(x, transpose=True), ops.mx4_quantize(w, transpose=True), torch.float32)

    def loss(x, w):
        return float((ops.mx4_matmul(ops.mx4_quantize(x), ops.mx4_quantize(w), torch.float32).double() * gy.double()).sum())

    for i, j in ((0, 0), (5, 32), (3, 17)):
        up, down = x.clone(), x.clone()
        up[i, j], down[i, j] = 2.0, -2.0
        assert (loss(up, w) - loss(down, w)) / 4 == float(gx[i, j])
    for i, j in ((0, 0), (39, 32), (21, 5)):
        up, down = w.clone(), w.clone()
        up[i, j], down[i, j] = 2.0, -2.0
        assert (loss(x, up) - loss(x, down)) / 4 == float(gw[i, j])


@gpu
def test_other_stream_and_graph(ops):
    x, w = torch.randn(20, 500, device="cuda"), torch.randn(300, 500, device="cuda")
    wq = ops.mx4_quantize(w)
    want = ops.mx4_linear(x, wq)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 2.0
        got = ops.mx4_linear(y * 0.5, wq)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    static = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mx4_linear(static, wq)
    static.copy_(x)
    graph.replay()
    assert torch.equal(out, want)


@gpu
def test_repeats_are_bit_equal(ops):
    for m, n, k in ((1, 4096, 4096), (48, 1000, 3000), (700, 900, 1100)):
        a, b = ops.mx4_quantize(torch.randn(m, k, device="cuda")), ops.mx4_quantize(torch.randn(n, k, device="cuda"))
        first = ops.mx4_matmul(a, b, torch.float32)
        for _ in range(5):
            assert torch.equal(ops.mx4_matmul(a, b, torch.float32), first)


@gpu
def test_refusals(ops):
    x = torch.zeros(4, 64, device="cuda")
    q = ops.mx4_quantize(x)
    with pytest.raises(ValueError):
        ops.mx4_quantize(x.cpu())
    with pytest.raises(ValueError):
        ops.mx4_quantize(torch.zeros(4, 64, 2, device="cuda")[:, :, 0])
    with pytest.raises(ValueError):
        ops.mx4_quantize(torch.zeros(4, device="cuda"))
    with pytest.raises(TypeError):
        ops.mx4_quantize(x.double())
    with pytest.raises(ValueError):
        ops.mx4_matmul(q, ops.mx4_quantize(torch.zeros(4, 65, device="cuda")))
    with pytest.raises(TypeError):
        ops.mx4_matmul(q, q, torch.float64)
    with pytest.raises(ValueError):
        ops.mx4_matmul(q, q, bias=torch.zeros(5, device="cuda"))
    with pytest.raises(ValueError):
        ops.mx4_matmul(q, q, bias=torch.zeros(4, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.mx4_matmul(q, q, torch.float32, out=torch.zeros(4, 5, device="cuda"))
    with pytest.raises(ValueError):
        ops.Mx4(q.codes, q.scales, 4, 300)
    with pytest.raises(ValueError):
        ops.mx4_linear_grad(x, q, q)
    with pytest.raises(ops.FufftError):
        ops.mx4_matmul(ops.Mx4(torch.zeros(4 * 128 + 1, dtype=torch.uint8, device="cuda")[1:], q.scales, 4, 64), q)


def test_refusals_before_device():
    from fufft_b200._lib import lib
    L, P = lib(), 1 << 20
    SIZE, MISALIGNED, ARG = 1, 3, 7
    assert L.fufft_mx4_quantize(P, 3, 4, 64, 64, P, P, None, None, None) == ARG
    assert L.fufft_mx4_quantize(P, 0, -1, 64, 64, P, P, None, None, None) == SIZE
    assert L.fufft_mx4_quantize(P, 0, 1 << 29, 1 << 29, 1 << 29, P, P, None, None, None) == SIZE
    assert L.fufft_mx4_quantize(P, 0, 4, 64, 63, P, P, None, None, None) == ARG
    assert L.fufft_mx4_quantize(None, 0, 4, 64, 64, P, P, None, None, None) == ARG
    assert L.fufft_mx4_quantize(P, 0, 4, 64, 64, None, None, None, None, None) == ARG
    assert L.fufft_mx4_quantize(P, 0, 4, 64, 64, P, None, None, None, None) == ARG
    assert L.fufft_mx4_quantize(P, 0, 4, 64, 64, P + 8, P, None, None, None) == MISALIGNED
    assert L.fufft_mx4_quantize(P + 2, 0, 4, 64, 64, P, P, None, None, None) == MISALIGNED
    assert L.fufft_mx4_quantize(None, 0, 0, 64, 64, None, None, None, None, None) == 0
    assert L.fufft_mx4_dequantize(P, P, 4, 64, None, 0, 64, None) == ARG
    assert L.fufft_mx4_dequantize(P, P, 4, 64, P, 9, 64, None) == ARG
    assert L.fufft_mx4_matmul(P, P, P, P, None, P, 0, -1, 4, 64, 4, None) == SIZE
    assert L.fufft_mx4_matmul(P, P, P, P, None, P, 0, 4, 4, 64, 3, None) == ARG
    assert L.fufft_mx4_matmul(P, P, None, P, None, P, 0, 4, 4, 64, 4, None) == ARG
    assert L.fufft_mx4_matmul(P, P + 4, P, P, None, P, 0, 4, 4, 64, 4, None) == MISALIGNED
    assert L.fufft_mx4_matmul(None, None, None, None, None, None, 0, 0, 4, 64, 4, None) == 0
    linear = lambda m, x=P, c=P, stride=64, dtype=0: L.fufft_mx4_linear(x, dtype, m, 64, stride, c, c, P, P, 8, None, P, 0, 8, None)  # noqa: E731
    assert linear(4, x=None) == ARG and linear(4, stride=63) == ARG and linear(4, dtype=3) == ARG and linear(4, x=P + 2) == MISALIGNED
    assert linear(40, c=None) == ARG and linear(40, c=P + 8) == MISALIGNED and linear(0) == 0
    assert L.fufft_mx4_codes_bytes(3, 257) == 3 * 256 and L.fufft_mx4_scales_bytes(129, 1) == 2 * 2 * 512
    assert L.fufft_mx4_codes_bytes(-1, 4) == 0
