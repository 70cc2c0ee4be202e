"""torch.ops registration of the library's main entry points.

``import fufft_b200.torch_ops`` registers, under the ``fufft`` namespace:

  torch.ops.fufft.conv(a, b, n, layout, mid, filter_stride) -> Tensor
  torch.ops.fufft.conv2d(a, b, h, w, layout, mid, filter_stride) -> Tensor
  torch.ops.fufft.c2c(a, n, sign) -> Tensor
  torch.ops.fufft.filter_from_taps(taps, n, layout) -> Tensor

and, for the layers around a long convolution,

  torch.ops.fufft.mx4_quantize(x, transpose) -> (codes, scales)
  torch.ops.fufft.mx4_linear(x, w_codes, w_scales, n, bias) -> Tensor
  torch.ops.fufft.mx4_train(x, w) -> (y, xt codes, xt scales, wt codes, wt scales)
  torch.ops.fufft.mx4_train_grad(gy, xt codes, xt scales, wt codes, wt scales, w_dtype) -> (gx, gw)
  torch.ops.fufft.cache_append(x, codes, scales, page_table, kind, cu, starts) -> ()
  torch.ops.fufft.cache_read(codes, scales, page_table, kind, cu, starts, tokens, dtype) -> Tensor
  torch.ops.fufft.cache_read_channels(codes, scales, page_table, kind, starts, counts, n) -> Tensor
  torch.ops.fufft.cache_conv(codes, scales, page_table, kind, lengths, taps, gate, dtype) -> Tensor

The convolution's tensors are complex64 CUDA tensors (flat or any shape whose element count is
a whole number of transforms); every op returns a new tensor of a's shape and
launches exactly the kernels of the matching fufft_b200.ops call on the
current stream.  Each op has a fake (shape-only) implementation, so the ops
trace under torch.compile / torch.export and show up as single graph nodes.
mx4_train has an autograd formula (mx4_linear_train is its product alone); the
others have none.
"""
from __future__ import annotations

import torch

from . import ops

_NS = "fufft"


@torch.library.custom_op(f"{_NS}::conv", mutates_args=())
def conv(a: torch.Tensor, b: torch.Tensor | None, n: int, layout: int, mid: int, filter_stride: int) -> torch.Tensor:
    return ops.conv(a.contiguous().view(-1), None if b is None else b.contiguous().view(-1), n, layout, mid,
                    filter_stride=filter_stride).view(a.shape)


@conv.register_fake
def _(a, b, n, layout, mid, filter_stride):
    return torch.empty_like(a)


@torch.library.custom_op(f"{_NS}::conv2d", mutates_args=())
def conv2d(a: torch.Tensor, b: torch.Tensor | None, h: int, w: int, layout: int, mid: int,
           filter_stride: int) -> torch.Tensor:
    return ops.conv2d(a.contiguous().view(-1), None if b is None else b.contiguous().view(-1), h, w, layout, mid,
                      filter_stride=filter_stride).view(a.shape)


@conv2d.register_fake
def _(a, b, h, w, layout, mid, filter_stride):
    return torch.empty_like(a)


@torch.library.custom_op(f"{_NS}::c2c", mutates_args=())
def c2c(a: torch.Tensor, n: int, sign: int) -> torch.Tensor:
    return ops.c2c(a.contiguous().view(-1), n, sign).view(a.shape)


@c2c.register_fake
def _(a, n, sign):
    return torch.empty_like(a)


@torch.library.custom_op(f"{_NS}::filter_from_taps", mutates_args=())
def filter_from_taps(taps: torch.Tensor, n: int, layout: int) -> torch.Tensor:
    return ops.filter_from_taps(taps.contiguous().view(-1), n, layout).view(taps.shape)


@filter_from_taps.register_fake
def _(taps, n, layout):
    return torch.empty_like(taps)


# ---- microscaled 4-bit matrices --------------------------------------------------
def _mx4_sizes(rows, cols):
    tiles = -(-cols // 256) * 2
    return (rows, tiles * 64), (-(-rows // 128), tiles, 32, 4, 4)


def _mx4_fake(like: torch.Tensor, rows, cols):
    codes, scales = _mx4_sizes(rows, cols)
    return like.new_empty(codes, dtype=torch.uint8), like.new_empty(scales, dtype=torch.uint8)


def _own(q: ops.Mx4) -> tuple[torch.Tensor, torch.Tensor]:
    """codes and scales with a storage each: an op's results may not share one"""
    return q.codes, q.scales.clone()


@torch.library.custom_op(f"{_NS}::mx4_quantize", mutates_args=())
def mx4_quantize(x: torch.Tensor, transpose: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _own(ops.mx4_quantize(x, transpose))


@mx4_quantize.register_fake
def _(x, transpose):
    rows, cols = x.shape[::-1] if transpose else x.shape
    return _mx4_fake(x, rows, cols)


@torch.library.custom_op(f"{_NS}::mx4_linear", mutates_args=())
def mx4_linear(x: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor, n: int,
               bias: torch.Tensor | None) -> torch.Tensor:
    return ops.mx4_linear(x, ops.Mx4(w_codes, w_scales, n, x.shape[-1]), bias)


@mx4_linear.register_fake
def _(x, w_codes, w_scales, n, bias):
    return x.new_empty((*x.shape[:-1], n))


@torch.library.custom_op(f"{_NS}::mx4_train", mutates_args=())
def mx4_train(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    xq, xt = ops.mx4_quantize_both(x)
    wq, wt = ops.mx4_quantize_both(w)
    return ops.mx4_matmul(xq, wq, x.dtype), *_own(xt), *_own(wt)


@mx4_train.register_fake
def _(x, w):
    return x.new_empty((x.shape[0], w.shape[0])), *_mx4_fake(x, x.shape[1], x.shape[0]), *_mx4_fake(x, w.shape[1], w.shape[0])


@torch.library.custom_op(f"{_NS}::mx4_train_grad", mutates_args=())
def mx4_train_grad(gy: torch.Tensor, xt_codes: torch.Tensor, xt_scales: torch.Tensor, wt_codes: torch.Tensor,
                   wt_scales: torch.Tensor, w_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    k = wt_codes.shape[0]
    return ops.mx4_linear_grad(gy, ops.Mx4(xt_codes, xt_scales, k, gy.shape[0]), ops.Mx4(wt_codes, wt_scales, k, gy.shape[1]),
                               w_dtype=w_dtype)


@mx4_train_grad.register_fake
def _(gy, xt_codes, xt_scales, wt_codes, wt_scales, w_dtype=None):
    k = wt_codes.shape[0]
    return gy.new_empty((gy.shape[0], k)), gy.new_empty((gy.shape[1], k), dtype=w_dtype or gy.dtype)


def _train_context(ctx, inputs, output):
    ctx.save_for_backward(*output[1:])
    ctx.w_dtype = inputs[1].dtype


def _train_backward(ctx, gy, *_):
    return torch.ops.fufft.mx4_train_grad(gy.contiguous(), *ctx.saved_tensors, ctx.w_dtype)


mx4_train.register_autograd(_train_backward, setup_context=_train_context)


def mx4_linear_train(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """x [m, k] times w [n, k] with both in 4 bits, differentiable: the backward products are in 4 bits too, the
    quantisers passed straight through, and keep x and w in 4 bits in between"""
    return torch.ops.fufft.mx4_train(x, w)[0]


# ---- quantised sequence cache -----------------------------------------------------
@torch.library.custom_op(f"{_NS}::cache_append", mutates_args=("codes", "scales"))
def cache_append(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, kind: str,
                 cu: torch.Tensor, starts: torch.Tensor) -> None:
    ops.cache_append(ops.SeqCache(codes, scales, page_table, kind), x, cu, starts)


@cache_append.register_fake
def _(x, codes, scales, page_table, kind, cu, starts):
    return None


@torch.library.custom_op(f"{_NS}::cache_read", mutates_args=())
def cache_read(codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, kind: str, cu: torch.Tensor,
               starts: torch.Tensor, tokens: int, dtype: torch.dtype) -> torch.Tensor:
    return ops.cache_read(ops.SeqCache(codes, scales, page_table, kind), cu, starts, tokens, dtype)


@cache_read.register_fake
def _(codes, scales, page_table, kind, cu, starts, tokens, dtype):
    return codes.new_empty((tokens, scales.shape[2] * 32), dtype=dtype)


@torch.library.custom_op(f"{_NS}::cache_read_channels", mutates_args=())
def cache_read_channels(codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, kind: str,
                        starts: torch.Tensor, counts: torch.Tensor, n: int) -> torch.Tensor:
    return ops.cache_read_channels(ops.SeqCache(codes, scales, page_table, kind), starts, counts, n)


@cache_read_channels.register_fake
def _(codes, scales, page_table, kind, starts, counts, n):
    return codes.new_empty((page_table.shape[0], scales.shape[2] * 32, n), dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::cache_conv", mutates_args=())
def cache_conv(codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, kind: str, lengths: torch.Tensor,
               taps: torch.Tensor, gate: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    return ops.cache_conv(ops.SeqCache(codes, scales, page_table, kind), lengths, taps, gate, dtype)


@cache_conv.register_fake
def _(codes, scales, page_table, kind, lengths, taps, gate, dtype):
    return codes.new_empty((page_table.shape[0], scales.shape[2] * 32), dtype=dtype)
