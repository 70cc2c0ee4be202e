"""Python mirror of the reference's entry points over the C ABI.

The reference (weiwang217/FuFFT, fufft.cuh) exposes kernel templates that the
caller launches with a mid-op policy struct; here each becomes a function over
CUDA tensors that calls the corresponding C entry point on the current torch
stream.  Names follow the reference:

    pipeline_ip(a, b_dr)        fufft_pipeline_ip   (radix-8 chain, any mid-op)
    pipeline_fused(a, bperm)    fufft_pipeline_fused (radix-8 register boundary)
    pipeline_v16(a, b16)        fufft_pipeline_v16  (radix-16 chain)
    pipeline_v16f(a, bperm16)   fufft_pipeline_v16f (radix-16 register boundary)
    pipeline_r16(a, b16)        fufft_pipeline_r16  (same math as v16)
    pipeline_fwd / pipeline_apply   split forward / apply
    conv_r2                     fufft_conv_r2 (two-for-one real)
    pipeline_v16_bfp            fufft_pipeline_v16_bfp (int16 BFP)

Complex data: torch.complex64 (or float32 with a trailing dim of 2), one
transform per row of n points.  int16 BFP data: torch.int16 with a trailing
dim of 2 (re, im) plus one float32 scale per transform.

Operators without a counterpart there, for the layers around a long
convolution of a sequence model: 4-bit microscaled matrices (Mx4,
mx4_quantize, mx4_quantize_both, mx4_dequantize, mx4_matmul, mx4_linear,
mx4_linear_grad) and the quantised sequence cache (SeqCache, cache_append,
cache_read, cache_read_channels, cache_conv).  They take float32, float16 and
bfloat16.
"""
from __future__ import annotations

import ctypes as ct

import torch
from torch import _C

from ._lib import (CACHE_MX4, CACHE_MX8, DTYPE_BF16, DTYPE_F16, DTYPE_F32, LAYOUT_NATURAL, LAYOUT_R8,
                   LAYOUT_R8_BPERM, LAYOUT_R16, LAYOUT_R16_BPERM, MID_CONJ_MULTIPLY, MID_MULTIPLY, MID_NONE,
                   MX4_DIRECT_ROWS, CacheDesc, FufftError, check, lib)

__all__ = [
    "MID_NONE", "MID_MULTIPLY", "MID_CONJ_MULTIPLY",
    "LAYOUT_R8", "LAYOUT_R8_BPERM", "LAYOUT_R16", "LAYOUT_R16_BPERM", "LAYOUT_NATURAL",
    "FufftError", "chain", "chain_rev", "chain_rev_table", "filter_permute", "filter_permute_host", "filter_permute2d", "conv",
    "conv2d", "fwd", "apply",
    "conv_r2", "bfp_pack", "bfp_unpack", "conv_bfp", "pipeline_ip", "pipeline_fused", "pipeline_v16",
    "pipeline_v16f", "pipeline_r16", "pipeline_fwd", "pipeline_apply", "pipeline_v16_bfp", "init",
    "device_status", "launch_count", "max_n", "large_plan", "conv_large", "conv_large_bfp",
    "Mx4", "mx4_empty", "mx4_quantize", "mx4_quantize_both", "mx4_dequantize", "mx4_matmul", "mx4_linear",
    "mx4_linear_grad", "SeqCache", "seq_cache", "cache_append", "cache_read", "cache_read_channels", "cache_conv",
]


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _hptr(t: torch.Tensor | None):
    """address of a contiguous HOST tensor"""
    if t is None:
        return None
    if t.is_cuda or not t.is_contiguous():
        raise ValueError("expected a contiguous host tensor")
    return t.data_ptr()


def _ptr(t: torch.Tensor | None):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("fufft_b200 operates on CUDA tensors")
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return t.data_ptr()


def _complex(t: torch.Tensor) -> torch.Tensor:
    if t.dtype == torch.complex64:
        return t
    if t.dtype == torch.float32 and t.shape[-1] == 2:
        return torch.view_as_complex(t)
    raise TypeError("complex data must be complex64 (or float32 [..., 2])")


def _batch(t: torch.Tensor, n: int, per_point: int = 1) -> int:
    total = t.numel() // per_point
    if total % n:
        raise ValueError(f"{total} points is not a whole number of transforms of {n}")
    return total // n


# ---- library / index maps ---------------------------------------------------
def init() -> None:
    check(lib().fufft_init(), "fufft_init")


def max_n(layout: int) -> int:
    return lib().fufft_max_n(layout)


def launch_count() -> int:
    return int(lib().fufft_launch_count())


def device_status() -> int:
    v = ct.c_uint32()
    check(lib().fufft_device_status(ct.byref(v), _stream()), "fufft_device_status")
    return v.value


def chain(n: int, radix: int) -> list[int]:
    buf = (ct.c_int * 32)()
    p = lib().fufft_chain(n, radix, buf)
    if p < 0:
        raise ValueError(f"n={n} radix={radix}")
    return list(buf[:p])


def chain_rev(idx: int, radices) -> int:
    arr = (ct.c_int * len(radices))(*radices)
    return int(lib().fufft_chain_rev(idx, arr, len(radices)))


def chain_rev_table(radices, device=None) -> torch.Tensor:
    """natural (frequency) index of every chain position of the radix chain
    `radices` (pass 0 first), as an int64 tensor: the digits of p, pass 0 most
    significant, written back in reverse order -- fufft_chain_rev for all p at
    once (verify_kernel.cpp:460-477 chain_rev)"""
    n = 1
    for r in radices:
        n *= int(r)
    p = torch.arange(n, dtype=torch.int64, device=device)
    out = torch.zeros_like(p)
    rest, op = n, 1          # weight of the current digit in p; in the output
    for r in radices:
        rest //= int(r)
        out += ((p // rest) % int(r)) * op
        op *= int(r)
    return out


def filter_permute(spec_natural: torch.Tensor, n: int, layout: int) -> torch.Tensor:
    """natural-order spectrum (device) -> kernel layout, per transform"""
    s = _complex(spec_natural).contiguous()
    out = torch.empty_like(s)
    check(lib().fufft_filter_permute(_ptr(s), _ptr(out), n, _batch(s, n), layout, _stream()),
          "fufft_filter_permute")
    return out


def filter_permute_host(spec_natural, n: int, layout: int):
    """numpy complex64 natural-order spectrum -> kernel layout (host)"""
    import numpy as np
    s = np.ascontiguousarray(spec_natural, dtype=np.complex64)
    out = np.empty_like(s)
    check(lib().fufft_filter_permute_host(s.ctypes.data, out.ctypes.data, n, s.size // n, layout),
          "fufft_filter_permute_host")
    return out


# ---- fused convolutions -------------------------------------------------------
def conv(a: torch.Tensor, b: torch.Tensor | None, n: int, layout: int = LAYOUT_R16_BPERM,
         mid: int = MID_MULTIPLY, filter_stride: int | None = None,
         out: torch.Tensor | None = None) -> torch.Tensor:
    a = _complex(a)
    bt = None if b is None else _complex(b)
    out = torch.empty_like(a) if out is None else _complex(out)
    fs = n if filter_stride is None else filter_stride
    check(lib().fufft_conv_c2c_f32(_ptr(a), _ptr(bt), _ptr(out), n, _batch(a, n), layout, mid, fs, _stream()),
          "fufft_conv_c2c_f32")
    return out


def filter_permute2d(spec_natural: torch.Tensor, h: int, w: int, layout: int) -> torch.Tensor:
    """natural-order 2-D spectrum (device, row-major) -> 2-D kernel layout"""
    s = _complex(spec_natural).contiguous()
    out = torch.empty_like(s)
    check(lib().fufft_filter_permute2d(_ptr(s), _ptr(out), h, w, _batch(s, h * w), layout, 0, _stream()),
          "fufft_filter_permute2d")
    return out


def conv2d(a: torch.Tensor, b: torch.Tensor | None, h: int, w: int, layout: int = LAYOUT_R16_BPERM,
           mid: int = MID_MULTIPLY, filter_stride: int | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """fufft_conv2d<H, W, CPB>: fused 2-D cyclic convolution of row-major h x w images"""
    a = _complex(a)
    bt = None if b is None else _complex(b)
    out = torch.empty_like(a) if out is None else _complex(out)
    fs = h * w if filter_stride is None else filter_stride
    check(lib().fufft_conv2d_f32(_ptr(a), _ptr(bt), _ptr(out), h, w, _batch(a, h * w), layout, mid, fs, _stream()),
          "fufft_conv2d_f32")
    return out


def conv_host_workspace(n: int, batch: int, filter_stride: int, device=None) -> torch.Tensor:
    """device workspace for conv_host (allocate once, reuse across calls)"""
    need = int(lib().fufft_conv_host_workspace(n, batch, filter_stride))
    return torch.empty(max(need, 1), dtype=torch.uint8, device=device or "cuda")


def conv_host(a: torch.Tensor, b: torch.Tensor | None, out: torch.Tensor, n: int, layout: int = LAYOUT_R16_BPERM,
              mid: int = MID_MULTIPLY, filter_stride: int | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """fused convolution of HOST tensors (pinned for overlap): chunked upload /
    convolve / download pipeline on the current device, asynchronous on the
    current stream"""
    a, out = _complex(a), _complex(out)
    if a.is_cuda or out.is_cuda or (b is not None and b.is_cuda):
        raise ValueError("conv_host takes host tensors")
    bt = None if b is None else _complex(b)
    batch = _batch(a, n)
    if out.numel() < a.numel():
        raise ValueError("out is smaller than a")
    fs = (n if bt is None or bt.numel() > n else 0) if filter_stride is None else filter_stride
    if workspace is None:
        workspace = conv_host_workspace(n, batch, fs)
    check(lib().fufft_conv_c2c_f32_host(_hptr(a), _hptr(bt), _hptr(out), n, batch, layout, mid, fs, _ptr(workspace),
                                        workspace.numel(), _stream()), "fufft_conv_c2c_f32_host")
    return out


def filter_from_taps(taps: torch.Tensor, n: int, layout: int = LAYOUT_R16_BPERM) -> torch.Tensor:
    """complex filter taps (natural order) -> filter spectrum x 1/n in `layout`, on the device"""
    taps = _complex(taps)
    out = torch.empty_like(taps)
    check(lib().fufft_filter_from_taps_f32(_ptr(taps), _ptr(out), n, _batch(taps, n), layout, _stream()),
          "fufft_filter_from_taps_f32")
    return out


def c2c(a: torch.Tensor, n: int, sign: int = -1, out: torch.Tensor | None = None) -> torch.Tensor:
    """natural-order DFT of each n-point transform (sign -1), or the unnormalised inverse (+1)"""
    a = _complex(a)
    out = torch.empty_like(a) if out is None else _complex(out)
    check(lib().fufft_c2c_f32(_ptr(a), _ptr(out), n, _batch(a, n), sign, _stream()), "fufft_c2c_f32")
    return out


def fwd(a: torch.Tensor, n: int, layout: int = LAYOUT_R8) -> torch.Tensor:
    a = _complex(a)
    spec = torch.empty_like(a)
    check(lib().fufft_fwd_f32(_ptr(a), _ptr(spec), n, _batch(a, n), layout, _stream()), "fufft_fwd_f32")
    return spec


def apply(spec: torch.Tensor, b: torch.Tensor | None, n: int, layout: int = LAYOUT_R8,
          mid: int = MID_MULTIPLY, batch: int | None = None, spec_stride: int | None = None,
          filter_stride: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    spec = _complex(spec)
    bt = None if b is None else _complex(b)
    batch = _batch(spec, n) if batch is None else batch
    ss = n if spec_stride is None else spec_stride
    fs = n if filter_stride is None else filter_stride
    if out is None:
        out = torch.empty(batch * n, dtype=torch.complex64, device=spec.device)
    check(lib().fufft_apply_f32(_ptr(spec), _ptr(bt), _ptr(out), n, batch, layout, mid, ss, fs, _stream()),
          "fufft_apply_f32")
    return out


def fwd_r2(xr: torch.Tensor, yr: torch.Tensor, n: int, layout: int = LAYOUT_R16) -> torch.Tensor:
    """chain-order spectra of the packed pairs xr + i*yr (two real signals per transform)"""
    if xr.shape != yr.shape:
        raise ValueError("xr and yr must have the same shape")
    spec = torch.empty(xr.numel(), dtype=torch.complex64, device=xr.device)
    check(lib().fufft_fwd_r2_f32(_ptr(xr), _ptr(yr), _ptr(spec), n, _batch(xr, n), layout, _stream()),
          "fufft_fwd_r2_f32")
    return spec


def apply_grid(spec: torch.Tensor, b: torch.Tensor, n: int, layout: int = LAYOUT_R16, mid: int = MID_MULTIPLY,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """every spectrum against every filter in one launch: out[s][f] = IDFT(spec_s (x) b_f), complex"""
    spec, bt = _complex(spec), _complex(b)
    ns, nf = _batch(spec, n), _batch(bt, n)
    if out is None:
        out = torch.empty(ns * nf * n, dtype=torch.complex64, device=spec.device)
    else:
        out = _complex(out)
        if out.numel() < ns * nf * n:
            raise ValueError("out must hold n_spec * n_filt * n complex points")
    check(lib().fufft_apply_grid_f32(_ptr(spec), ns, _ptr(bt), nf, _ptr(out), n, layout, mid, _stream()),
          "fufft_apply_grid_f32")
    return out


def apply_grid_r2(spec: torch.Tensor, b: torch.Tensor, n: int, layout: int = LAYOUT_R16, mid: int = MID_MULTIPLY,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """packed real pairs x real filters: out[2s + j][f][0..n) real (j = 0: xr of pair s, 1: yr)"""
    spec, bt = _complex(spec), _complex(b)
    ns, nf = _batch(spec, n), _batch(bt, n)
    if out is None:
        out = torch.empty(2 * ns * nf * n, dtype=torch.float32, device=spec.device)
    elif out.dtype != torch.float32 or out.numel() < 2 * ns * nf * n:
        raise ValueError("out must be float32 with 2 * n_pairs * n_filt * n elements")
    check(lib().fufft_apply_grid_r2_f32(_ptr(spec), ns, _ptr(bt), nf, _ptr(out), n, layout, mid, _stream()),
          "fufft_apply_grid_r2_f32")
    return out


def conv_r2(xr: torch.Tensor, yr: torch.Tensor, b: torch.Tensor, n: int, layout: int = LAYOUT_R8,
            mid: int = MID_MULTIPLY, filter_stride: int | None = None):
    bt = _complex(b)
    ur, vr = torch.empty_like(xr), torch.empty_like(yr)
    fs = n if filter_stride is None else filter_stride
    check(lib().fufft_conv_r2_f32(_ptr(xr), _ptr(yr), _ptr(bt), _ptr(ur), _ptr(vr), n, _batch(xr, n),
                                  layout, mid, fs, _stream()), "fufft_conv_r2_f32")
    return ur, vr


# ---- four-step large N ------------------------------------------------------------
def large_plan(n: int, layout: int = LAYOUT_R16) -> tuple[int, int]:
    r, m = ct.c_int(), ct.c_int()
    check(lib().fufft_large_plan(n, layout, ct.byref(r), ct.byref(m)), "fufft_large_plan")
    return r.value, m.value


def conv_large(buf: torch.Tensor, b: torch.Tensor | None, n: int, layout: int = LAYOUT_R16,
               mid: int = MID_MULTIPLY, r_out: int | None = None, mid_size: int | None = None) -> torch.Tensor:
    """run_large: in-place four-step convolution of transforms of n points"""
    buf = _complex(buf)
    if r_out is None or mid_size is None:
        r_out, mid_size = large_plan(n, layout)
    bt = None if b is None else _complex(b)
    check(lib().fufft_conv_large_f32(_ptr(buf), _ptr(bt), n, _batch(buf, n), r_out, mid_size, layout, mid,
                                     _stream()), "fufft_conv_large_f32")
    return buf


def conv_large_bfp(aq, a_scale, bq, b_scale, n: int, layout: int = LAYOUT_R16, mid: int = MID_MULTIPLY,
                   r_out: int | None = None, mid_size: int | None = None, workspace: torch.Tensor | None = None):
    if r_out is None or mid_size is None:
        r_out, mid_size = large_plan(n, layout)
    batch = _batch(aq, n, 2)
    need = int(lib().fufft_conv_large_bfp_workspace(n, batch))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=aq.device)
    oq = torch.empty_like(aq)
    os_ = torch.empty(batch, dtype=torch.float32, device=aq.device)
    check(lib().fufft_conv_large_bfp(_ptr(aq), _ptr(a_scale), _ptr(bq), _ptr(b_scale), _ptr(oq), _ptr(os_), n, batch,
                                     r_out, mid_size, layout, mid, _ptr(workspace), workspace.numel(), _stream()),
          "fufft_conv_large_bfp")
    return oq, os_


# ---- int16 block floating point -------------------------------------------------
def bfp_pack(x: torch.Tensor, n: int):
    x = _complex(x)
    batch = _batch(x, n)
    q = torch.empty(x.numel(), 2, dtype=torch.int16, device=x.device)
    s = torch.empty(batch, dtype=torch.float32, device=x.device)
    check(lib().fufft_bfp_pack(_ptr(x), _ptr(q), _ptr(s), n, batch, _stream()), "fufft_bfp_pack")
    return q, s


def bfp_unpack(q: torch.Tensor, s: torch.Tensor, n: int) -> torch.Tensor:
    batch = _batch(q, n, 2)
    x = torch.empty(batch * n, dtype=torch.complex64, device=q.device)
    check(lib().fufft_bfp_unpack(_ptr(q), _ptr(s), _ptr(x), n, batch, _stream()), "fufft_bfp_unpack")
    return x


def conv_bfp(aq: torch.Tensor, a_scale: torch.Tensor, bq: torch.Tensor | None, b_scale: torch.Tensor | None,
             n: int, layout: int = LAYOUT_R16, mid: int = MID_MULTIPLY, filter_stride: int | None = None,
             out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """int16-BFP fused convolution; out = (oq, o_scale) to reuse output buffers"""
    batch = _batch(aq, n, 2)
    oq, os_ = out if out is not None else (torch.empty_like(aq),
                                           torch.empty(batch, dtype=torch.float32, device=aq.device))
    fs = n if filter_stride is None else filter_stride
    check(lib().fufft_conv_c2c_bfp(_ptr(aq), _ptr(a_scale), _ptr(bq), _ptr(b_scale), _ptr(oq), _ptr(os_), n,
                                   batch, layout, mid, fs, _stream()), "fufft_conv_c2c_bfp")
    return oq, os_


# ---- the reference's entry-point names ----------------------------------------------
def pipeline_ip(a, b_dr, n, mid=MID_MULTIPLY):
    """fufft_pipeline_ip<N, LEAD, NR8, CPB, Mid>: radix-8 chain, filter in mixedrev order"""
    return conv(a, b_dr, n, LAYOUT_R8, mid)


def pipeline_fused(a, bperm, n):
    """fufft_pipeline_fused: radix-8 chain, filter in the register-boundary layout"""
    return conv(a, bperm, n, LAYOUT_R8_BPERM, MID_MULTIPLY)


def pipeline_v16(a, b16, n, mid=MID_MULTIPLY):
    """fufft_pipeline_v16: radix-16 chain, filter in mixedrev16 order"""
    return conv(a, b16, n, LAYOUT_R16, mid)


def pipeline_v16f(a, bperm16, n):
    """fufft_pipeline_v16f: radix-16 chain, filter in the register-boundary layout"""
    return conv(a, bperm16, n, LAYOUT_R16_BPERM, MID_MULTIPLY)


def pipeline_r16(a, b16, n, mid=MID_MULTIPLY):
    """fufft_pipeline_r16: same transform and filter order as pipeline_v16"""
    return conv(a, b16, n, LAYOUT_R16, mid)


def pipeline_fwd(a, n):
    """fufft_pipeline_fwd: radix-8 chain-order spectrum"""
    return fwd(a, n, LAYOUT_R8)


def pipeline_apply(spec, b_dr, n, mid=MID_MULTIPLY):
    """fufft_pipeline_apply: spectrum x filter, inverse (radix-8 chain)"""
    return apply(spec, b_dr, n, LAYOUT_R8, mid)


def pipeline_v16_bfp(aq, a_scale, bq, b_scale, n):
    """fufft_pipeline_v16_bfp: int16 BFP in and out, radix-16 chain"""
    return conv_bfp(aq, a_scale, bq, b_scale, n, LAYOUT_R16, MID_MULTIPLY)


# ---- microscaled 4-bit matrices -------------------------------------------------------
# These operators run at a few microseconds, the time of their own Python: one
# allocation for the two buffers of a matrix, no check made twice.
_DTYPES = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}


def _queue(device: int, *others) -> int:
    """the current stream of the current device, as _stream, without making a stream object; `device`, an operand's, and
    the call's other operands (tensors, None) have to be there, since only their addresses go on"""
    current = _C._cuda_getDevice()   # looked up here: a torch without CUDA has no such name, and still imports this
    if device != current:
        raise ValueError(f"an operand is on {_name(device)}, the current device is {_name(current)}")
    for t in others:
        if t is not None and t.get_device() != current:
            raise ValueError(f"an operand is on {_name(t.get_device())}, the current device is {_name(current)}")
    return _C._cuda_getCurrentRawStream(current)


def _name(device: int) -> str:
    return "the host" if device < 0 else f"cuda:{device}"


def _at(t: torch.Tensor) -> int:
    """address of a contiguous tensor whose device is checked by itself (_queue)"""
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return t.data_ptr()


def _dtype(t: torch.dtype) -> int:
    d = _DTYPES.get(t)
    if d is None:
        raise TypeError(f"expected float32, float16 or bfloat16, got {t}")
    return d


def _rows(t: torch.Tensor, what: str) -> tuple[int, int, int]:
    """(rows, columns, row stride) of a 2-D CUDA tensor with unit stride along its rows"""
    if not t.is_cuda:
        raise ValueError("fufft_b200 operates on CUDA tensors")
    if t.dim() == 2:
        (rows, cols), (pitch, unit) = t.shape, t.stride()
        if rows <= 1:
            pitch = cols
        if (unit == 1 or cols <= 1) and pitch >= cols:
            return rows, cols, pitch
    raise ValueError(f"{what} must be a 2-D tensor with unit stride along its rows")


def _i32(t: torch.Tensor, n: int, what: str):
    if t.dtype != torch.int32 or t.shape != (n,):
        raise ValueError(f"{what} must be int32 with {n} entries")
    return _at(t)


def _result(out: torch.Tensor | None, like: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> tuple[torch.Tensor, int]:
    """a [rows, cols] result and its row stride: the caller's `out`, or a new one on like's device"""
    if out is None:
        return like.new_empty((rows, cols), dtype=dtype), cols
    if out.dtype != dtype or out.shape != (rows, cols):
        raise ValueError(f"out must be {dtype} {(rows, cols)}")
    if out.get_device() != like.get_device():
        raise ValueError(f"out is on {_name(out.get_device())}, the operands are on {_name(like.get_device())}")
    return out, _rows(out, "out")[2]


class Mx4:
    """A [rows, cols] matrix in 4-bit microscaled blocks along its columns:
    codes uint8 [rows, ceil(cols / 256) * 128] and the tiled E8M0 scales uint8
    [ceil(rows / 128), ceil(cols / 256) * 2, 32, 4, 4] (layout in
    include/fufft_b200.h, fufft_mx4_*)"""
    __slots__ = ("_codes", "_scales", "_buffer", "rows", "cols", "at", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        tiles = -(-cols // 256) * 2
        if codes.numel() != rows * tiles * 64 or scales.numel() != -(-rows // 128) * tiles * 512:
            raise ValueError(f"codes or scales do not fit a {rows} x {cols} matrix")
        self._codes, self._scales, self._buffer, self.rows, self.cols = codes, scales, codes, rows, cols
        self.at = _at(codes), _at(scales)
        self.device = device = codes.get_device()
        if device < 0 or scales.get_device() != device:
            raise ValueError(f"codes and scales must be on one CUDA device, not {_name(device)} and {_name(scales.get_device())}")

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            pitch = -(-self.cols // 256) * 128
            self._codes = self._buffer[: self.rows * pitch].view(self.rows, pitch)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            row_tiles, tiles = -(-self.rows // 128), -(-self.cols // 256) * 2
            at = self._buffer.numel() - row_tiles * tiles * 512
            self._scales = self._buffer[at:].view(row_tiles, tiles, 32, 4, 4)
        return self._scales

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols


def _mx4_new(like: torch.Tensor, rows: int, cols: int) -> Mx4:
    """uninitialised: codes, then scales, in one buffer on like's device"""
    q = Mx4.__new__(Mx4)
    tiles = -(-cols // 256) * 2
    codes = rows * tiles * 64          # a multiple of 128
    q._buffer = like.new_empty(codes + -(-rows // 128) * tiles * 512, dtype=torch.uint8)
    q._codes = q._scales = None
    q.rows, q.cols, q.device = rows, cols, q._buffer.get_device()
    at = q._buffer.data_ptr()
    q.at = at, at + codes
    return q


def mx4_empty(rows: int, cols: int, device=None) -> Mx4:
    """uninitialised buffers of a 4-bit matrix"""
    return _mx4_new(torch.empty(0, device=device or "cuda"), rows, cols)


def _turned(x: torch.Tensor) -> bool:
    """a transposed view: quantised along the other axis of what it is a view of"""
    return x.dim() == 2 and x.stride(0) == 1 and x.stride(1) != 1 and x.shape[0] > 1


def mx4_quantize(x: torch.Tensor, transpose: bool = False) -> Mx4:
    """x [rows, cols] quantised in blocks of 32 along its rows, or, with
    `transpose`, x^T quantised along the columns of x"""
    if _turned(x):
        x, transpose = x.t(), not transpose
    rows, cols, pitch = _rows(x, "x")
    dtype = _dtype(x.dtype)
    if transpose:
        q = _mx4_new(x, cols, rows)
        at = None, None, *q.at
    else:
        q = _mx4_new(x, rows, cols)
        at = *q.at, None, None
    rc = lib().fufft_mx4_quantize(x.data_ptr(), dtype, rows, cols, pitch, *at, _queue(x.get_device()))
    if rc:
        check(rc, "fufft_mx4_quantize")
    return q


def mx4_quantize_both(x: torch.Tensor) -> tuple[Mx4, Mx4]:
    """(mx4_quantize(x), mx4_quantize(x, transpose=True)) from one read of x"""
    if _turned(x):
        return mx4_quantize_both(x.t())[::-1]
    rows, cols, pitch = _rows(x, "x")
    dtype = _dtype(x.dtype)
    q, qt = _mx4_new(x, rows, cols), _mx4_new(x, cols, rows)
    rc = lib().fufft_mx4_quantize(x.data_ptr(), dtype, rows, cols, pitch, *q.at, *qt.at, _queue(x.get_device()))
    if rc:
        check(rc, "fufft_mx4_quantize")
    return q, qt


def mx4_dequantize(q: Mx4, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """the values that q stands for"""
    code = _dtype(dtype)
    out, pitch = _result(out, q._buffer, q.rows, q.cols, dtype)
    rc = lib().fufft_mx4_dequantize(*q.at, q.rows, q.cols, out.data_ptr(), code, pitch, _queue(q.device))
    if rc:
        check(rc, "fufft_mx4_dequantize")
    return out


def _bias(bias: torch.Tensor | None, n: int):
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,)):
        raise ValueError(f"bias must be float32 with {n} entries")
    return None if bias is None else _at(bias)


def mx4_matmul(a: Mx4, b: Mx4, dtype: torch.dtype = torch.bfloat16, bias: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """a b^T + bias: [a.rows, b.rows] in `dtype`, summed in float32; both are
    blocked along the summed axis, bias is float32 [b.rows]"""
    if a.cols != b.cols:
        raise ValueError(f"the summed axes differ: {a.shape} and {b.shape}")
    if a.device != b.device:
        raise ValueError(f"the operands are on {_name(a.device)} and {_name(b.device)}")
    code = _dtype(dtype)
    out, pitch = _result(out, a._buffer, a.rows, b.rows, dtype)
    rc = lib().fufft_mx4_matmul(*a.at, *b.at, _bias(bias, b.rows), out.data_ptr(), code, a.rows, b.rows, a.cols, pitch,
                                _queue(a.device, bias))
    if rc:
        check(rc, "fufft_mx4_matmul")
    return out


def mx4_linear(x: torch.Tensor, w: Mx4, bias: torch.Tensor | None = None,
               dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., k] quantised along k, times w [n, k]: [..., n] in x's dtype unless another is given"""
    flat = x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), x.shape[-1])
    if flat.shape[1] != w.cols:
        raise ValueError(f"the summed axes differ: {tuple(x.shape)} and {w.shape}")
    if _turned(flat):
        flat = flat.contiguous()
    m, k, pitch = _rows(flat, "x")
    dtype = dtype or x.dtype
    codes, out_code = _dtype(x.dtype), _dtype(dtype)
    out = flat.new_empty((m, w.rows), dtype=dtype)
    q = None if m <= MX4_DIRECT_ROWS else _mx4_new(flat, m, k)   # few rows are quantised inside the product
    rc = lib().fufft_mx4_linear(flat.data_ptr(), codes, m, k, pitch, *(q.at if q else (None, None)), *w.at, w.rows,
                                _bias(bias, w.rows), out.data_ptr(), out_code, w.rows, _queue(w.device, flat, bias))
    if rc:
        check(rc, "fufft_mx4_linear")
    return out if x.dim() == 2 else out.view(*x.shape[:-1], w.rows)


def mx4_linear_grad(gy: torch.Tensor, xt: Mx4, wt: Mx4, dtype: torch.dtype | None = None,
                    w_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """gradients of y = x w^T [m, n] with every operand in 4 bits, the
    quantiser passed straight through: gx [m, k] = Q(gy) Q(w^T)^T and
    gw [n, k] = Q(gy^T) Q(x^T)^T, from xt = mx4_quantize(x, transpose=True)
    [k, m] and wt = mx4_quantize(w, transpose=True) [k, n].  gx in `dtype`
    (gy's unless given), gw in `w_dtype` (as gx unless given), each rounded
    once from its float32 sums"""
    if gy.dim() != 2 or xt.cols != gy.shape[0] or wt.cols != gy.shape[1] or xt.rows != wt.rows:
        raise ValueError(f"gy {tuple(gy.shape)} does not fit xt {xt.shape} and wt {wt.shape}")
    gq, gt = mx4_quantize_both(gy)
    dtype = dtype or gy.dtype
    return mx4_matmul(gq, wt, dtype), mx4_matmul(gt, xt, w_dtype or dtype)


# ---- quantised sequence cache -----------------------------------------------------------
_KINDS = {"mx4": CACHE_MX4, "mx8": CACHE_MX8}


class SeqCache:
    """Past inputs of a batch of sequences in pages, each token's channels in
    microscaled blocks of 32 (`kind` "mx4" or "mx8"):
      codes       uint8 [pages, page_size, channels / 2 (mx4) or channels (mx8)]
      scales      uint8 [pages, page_size, channels / 32]
      page_table  int32 [batch, max_pages], -1 where there is no page"""
    __slots__ = ("codes", "scales", "page_table", "kind", "channels", "batch", "desc", "at", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, kind: str):
        code = _KINDS.get(kind)
        if code is None:
            raise ValueError(f"kind must be one of {sorted(_KINDS)}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or page_table.dtype != torch.int32:
            raise TypeError("codes and scales must be uint8, page_table int32")
        if codes.dim() != 3 or scales.dim() != 3 or page_table.dim() != 2:
            raise ValueError("codes and scales must be [pages, page_size, ...], page_table [batch, max_pages]")
        pages, page_size, width = codes.shape
        channels = scales.shape[2] * 32
        if scales.shape[:2] != (pages, page_size) or width * (2 if code == CACHE_MX4 else 1) != channels:
            raise ValueError("codes and scales differ in their pages or channels")
        self.batch, max_pages, stride = _rows(page_table, "page_table")
        self.codes, self.scales, self.page_table, self.kind, self.channels = codes, scales, page_table, kind, channels
        self.desc = CacheDesc(_at(codes), _at(scales), page_table.data_ptr(), stride, code, channels, page_size, pages,
                              max_pages, self.batch)
        self.at = ct.addressof(self.desc)
        self.device = device = codes.get_device()
        if device < 0 or scales.get_device() != device or page_table.get_device() != device:
            raise ValueError(f"codes, scales and page_table must be on one CUDA device, not {_name(device)}, "
                             f"{_name(scales.get_device())} and {_name(page_table.get_device())}")


def seq_cache(pages: int, page_size: int, channels: int, page_table: torch.Tensor, kind: str = "mx8") -> SeqCache:
    """an empty cache on page_table's device"""
    if channels % 32:
        raise ValueError("channels must be a multiple of 32")
    make = dict(dtype=torch.uint8, device=page_table.device)
    return SeqCache(torch.zeros(pages, page_size, channels // 2 if kind == "mx4" else channels, **make),
                    torch.zeros(pages, page_size, channels // 32, **make), page_table, kind)


def cache_append(cache: SeqCache, x: torch.Tensor, cu: torch.Tensor, starts: torch.Tensor) -> None:
    """quantise the tokens x [tokens, channels] into the cache: tokens
    cu[b] .. cu[b + 1] - 1 go to sequence b from position starts[b] on"""
    tokens, channels, pitch = _rows(x, "x")
    if channels != cache.channels:
        raise ValueError(f"x must have {cache.channels} channels")
    rc = lib().fufft_cache_append(cache.at, x.data_ptr(), _dtype(x.dtype), pitch, _i32(cu, cache.batch + 1, "cu"),
                                  _i32(starts, cache.batch, "starts"), tokens, _queue(cache.device, x, cu, starts))
    if rc:
        check(rc, "fufft_cache_append")


def cache_read(cache: SeqCache, cu: torch.Tensor, starts: torch.Tensor, tokens: int,
               dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """stored values [tokens, channels] of the ragged run (cu, starts), as in cache_append"""
    code = _dtype(dtype)
    out, pitch = _result(out, cache.codes, tokens, cache.channels, dtype)
    rc = lib().fufft_cache_read(cache.at, out.data_ptr(), code, pitch, _i32(cu, cache.batch + 1, "cu"),
                                _i32(starts, cache.batch, "starts"), tokens, _queue(cache.device, cu, starts))
    if rc:
        check(rc, "fufft_cache_read")
    return out


def cache_read_channels(cache: SeqCache, starts: torch.Tensor, counts: torch.Tensor, n: int,
                        dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[batch, channels, n]: positions starts[b] .. starts[b] + counts[b] - 1 of
    every sequence, channel by channel, zeros from counts[b] on -- two of
    these rows are what conv_r2 takes"""
    code = _dtype(dtype)
    out = cache.codes.new_empty((cache.batch, cache.channels, n), dtype=dtype)
    rc = lib().fufft_cache_read_channels(cache.at, out.data_ptr(), code, n, _i32(starts, cache.batch, "starts"),
                                         _i32(counts, cache.batch, "counts"), _queue(cache.device, starts, counts))
    if rc:
        check(rc, "fufft_cache_read_channels")
    return out


def cache_conv(cache: SeqCache, lengths: torch.Tensor, taps: torch.Tensor, gate: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """newest output of a causal convolution per sequence, [batch, channels]:
    gate[b, c] * sum_j taps[j, c // (channels // heads)] * x[b, lengths[b] - 1 - j, c]
    over j < min(lengths[b], len(taps)); taps [n_taps, heads] float32 or
    bfloat16, gate [batch, channels] of `dtype` or None.  The same call gives
    the same bits; in long histories another sequence's length can move the
    last of them (the work is dealt by the lengths of the whole batch)"""
    n, heads, taps_pitch = _rows(taps, "taps")
    if taps.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("taps must be float32 or bfloat16")
    code = _dtype(dtype)
    out, pitch = _result(out, cache.codes, cache.batch, cache.channels, dtype)
    gate_at, gate_pitch = None, 0
    if gate is not None:
        if gate.dtype != dtype or gate.shape != out.shape:
            raise ValueError(f"gate must be {dtype} {tuple(out.shape)}")
        gate_at, gate_pitch = gate.data_ptr(), _rows(gate, "gate")[2]
    if workspace is None:
        need = lib().fufft_cache_conv_workspace(cache.at, n)
        if need:
            workspace = out.new_empty(need, dtype=torch.uint8)
    rc = lib().fufft_cache_conv(cache.at, _i32(lengths, cache.batch, "lengths"), taps.data_ptr(), _DTYPES[taps.dtype], n,
                                heads, taps_pitch, gate_at, gate_pitch, out.data_ptr(), code, pitch, _ptr(workspace),
                                0 if workspace is None else workspace.numel(),
                                _queue(cache.device, lengths, taps, gate, workspace))
    if rc:
        check(rc, "fufft_cache_conv")
    return out
