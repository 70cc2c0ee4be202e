"""All bytes of a quantised matrix are its values', those of rows beyond the last among them (zeros): the same input gives
the same buffers, whatever the memory held; and the torch.ops forms pass the dispatcher's own checks."""
import pytest
import torch

import mx_reference as ref
from test_mx4_gpu import TYPES, _values, ops  # noqa: F401

gpu = pytest.mark.gpu
SHAPES = [(1, 32), (5, 33), (16, 4096), (127, 515), (128, 256), (129, 130), (200, 1000), (257, 96), (300, 2049), (640, 4100)]


def _same(codes, scales, x):
    want_codes, want_scales = ref.pack(x)
    assert torch.equal(codes.cpu().view_as(want_codes), want_codes)
    assert torch.equal(scales.cpu().view_as(want_scales), want_scales)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_every_byte_is_written(ops, shape, dtype):  # noqa: F811
    """into buffers full of 255, which as a scale is NaN, for all forms of the call and rows from any address"""
    from fufft_b200._lib import lib
    rows, cols = shape
    x = _values((rows, cols + 1), dtype, 17)
    code = TYPES.index(dtype)
    for off in (0, 1):
        d, part = x.cuda()[:, off:off + cols], x[:, off:off + cols]
        for along_rows, along_cols in ((True, False), (False, True), (True, True)):
            q, t = ops.mx4_empty(rows, cols), ops.mx4_empty(cols, rows)
            for b in (q.codes, q.scales, t.codes, t.scales):
                b.fill_(255)
            at = (*(q.at if along_rows else (None, None)), *(t.at if along_cols else (None, None)))
            assert lib().fufft_mx4_quantize(d.data_ptr(), code, rows, cols, cols + 1, *at, torch.cuda.current_stream().cuda_stream) == 0
            if along_rows:
                _same(q.codes, q.scales, part)
            if along_cols:
                _same(t.codes, t.scales, part.t().contiguous())


@gpu
def test_nothing_beside_the_buffers_is_written(ops):  # noqa: F811
    from fufft_b200._lib import lib
    for rows, cols in ((5, 33), (129, 130), (200, 1000), (16, 4096)):
        x = torch.randn(rows, cols, device="cuda")
        bufs = []
        for r, c in ((rows, cols), (cols, rows)):
            for n in (lib().fufft_mx4_codes_bytes(r, c), lib().fufft_mx4_scales_bytes(r, c)):
                bufs.append((n, torch.full((n + 4096,), 77, dtype=torch.uint8, device="cuda")))
        for a, b in ((True, False), (False, True), (True, True)):
            at = [t[1].data_ptr() if (a if i < 2 else b) else None for i, t in enumerate(bufs)]
            assert lib().fufft_mx4_quantize(x.data_ptr(), 0, rows, cols, cols, *at, torch.cuda.current_stream().cuda_stream) == 0
        for n, t in bufs:
            assert bool((t[n:] == 77).all())


@gpu
def test_opcheck(ops):  # noqa: F811
    import fufft_b200.torch_ops  # noqa: F401
    f, i32 = torch.ops.fufft, torch.int32
    x, w = torch.randn(7, 300, device="cuda"), torch.randn(130, 300, device="cuda")
    codes, scales = f.mx4_quantize(w, False)
    _, *kept = f.mx4_train(x, w)
    cache = ops.seq_cache(4, 4, 64, torch.tensor([[1, 0], [2, 3]], dtype=i32, device="cuda"), "mx4")
    parts = cache.codes, cache.scales, cache.page_table, "mx4"
    cu, zero, n = (torch.tensor(t, dtype=i32, device="cuda") for t in ([0, 6, 10], [0, 0], [6, 4]))
    junk = [torch.full((1 << 20,), 201, dtype=torch.uint8, device="cuda") for _ in range(8)]   # what new buffers may be made of
    del junk
    for name, args in {"mx4_quantize": (w, False), "mx4_linear": (x, codes, scales, 130, None),
                       "mx4_train": (x.clone().requires_grad_(), w.clone().requires_grad_()),
                       "mx4_train_grad": (torch.randn(7, 130, device="cuda"), *kept, torch.float32),
                       "cache_append": (torch.randn(10, 64, device="cuda"), *parts, cu, zero),
                       "cache_read": (*parts, cu, zero, 10, torch.float32), "cache_read_channels": (*parts, zero, n, 16),
                       "cache_conv": (*parts, n, torch.randn(8, 64, device="cuda"), None, torch.float32)}.items():
        torch.library.opcheck(getattr(f, name).default, args)
    f.mx4_quantize(w, True)
