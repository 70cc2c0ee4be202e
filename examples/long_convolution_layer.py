"""A gated long-convolution layer of a sequence model on this library: trained,
run over prompts, and stepped token by token.

    gate, v = x w_in^T          4-bit microscaled products (mx4_linear)
    y = gate * (taps (*) v)     causal convolution along the sequence, per channel
    out = y w_out^T

Prompts store v in the quantised cache, read it back channel by channel, and
convolve two sequences per transform (conv_r2).  Generation appends one v per
sequence and takes the newest output straight from the cache (cache_conv).

    python examples/long_convolution_layer.py
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fufft_b200 import ops, torch_ops  # noqa: E402


class LongConvolution:
    def __init__(self, width: int, longest: int, batch: int, page: int = 64, kind: str = "mx8", device="cuda", seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.width, self.batch = width, batch
        self.w_in = torch.randn(2 * width, width, device=device, generator=g) / math.sqrt(width)
        self.w_out = torch.randn(width, width, device=device, generator=g) / math.sqrt(width)
        lag = torch.arange(longest, device=device)[:, None]
        decay = torch.exp(torch.rand(width, device=device, generator=g) * math.log(longest))
        self.taps = torch.exp(-lag / decay) * torch.randn(longest, width, device=device, generator=g) / decay.sqrt()
        # what serving keeps: weights in 4 bits, the filters' spectra, the cache
        self.q_in, self.q_out = ops.mx4_quantize(self.w_in), ops.mx4_quantize(self.w_out)
        self.n = 1 << max(4, (2 * longest - 1).bit_length())
        rows = torch.zeros(width, self.n, dtype=torch.complex64, device=device)
        rows[:, :longest] = self.taps.t()
        self.spectrum = ops.filter_from_taps(rows.view(-1), self.n)
        per = -(-longest // page)
        table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
        self.cache = ops.seq_cache(batch * per, page, width, table, kind)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.one_each = torch.arange(batch + 1, dtype=torch.int32, device=device)

    def _project(self, x):
        u = ops.mx4_linear(x, self.q_in)
        return u[..., : self.width], u[..., self.width:]

    def prompt(self, x):
        """x [batch, tokens, width] -> [batch, tokens, width]; an even batch, two sequences a transform"""
        b, t, _ = x.shape
        gate, v = self._project(x.reshape(b * t, -1))
        ops.cache_append(self.cache, v, self.one_each * t, torch.zeros_like(self.lengths))
        self.lengths.fill_(t)
        rows = ops.cache_read_channels(self.cache, torch.zeros_like(self.lengths), self.lengths, self.n)
        y = torch.empty_like(rows)
        for i in range(0, b, 2):
            u, w = ops.conv_r2(rows[i].view(-1), rows[i + 1].view(-1), self.spectrum, self.n, ops.LAYOUT_R16_BPERM)
            y[i], y[i + 1] = u.view_as(y[i]), w.view_as(y[i])
        y = y[:, :, :t].transpose(1, 2).reshape(b * t, -1) * gate
        return ops.mx4_linear(y.to(x.dtype), self.q_out).view(b, t, -1)

    def step(self, x):
        """x [batch, width], the next token of every sequence -> [batch, width]"""
        gate, v = self._project(x)
        ops.cache_append(self.cache, v, self.one_each, self.lengths)
        self.lengths += 1
        y = ops.cache_conv(self.cache, self.lengths, self.taps, gate=gate, dtype=x.dtype)
        return ops.mx4_linear(y, self.q_out)


def train_projection(x, target, w, steps: int = 20, rate: float = 0.5):
    """a few steps of gradient descent on w with every product in 4 bits; the losses"""
    w = w.clone().requires_grad_()
    losses = []
    for _ in range(steps):
        loss = (torch_ops.mx4_linear_train(x, w) - target).square().mean()
        (grad,) = torch.autograd.grad(loss, w)
        with torch.no_grad():
            w -= rate * grad * x.shape[1]
        losses.append(float(loss.detach()))
    return losses


def main(width: int = 256, tokens: int = 300, steps: int = 8, batch: int = 4, dtype=torch.bfloat16) -> dict:
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(batch, tokens + steps, width, device="cuda", generator=g).to(dtype)
    layer = LongConvolution(width, tokens + steps, batch)
    whole = layer.prompt(x)
    layer.prompt(x[:, :tokens].contiguous())
    stepped = torch.stack([layer.step(x[:, tokens + i].contiguous()) for i in range(steps)], 1)
    want = whole[:, tokens:].float()
    apart = float((stepped.float() - want).norm() / want.norm())
    flat = torch.randn(512, width, device="cuda", generator=g)
    losses = train_projection(flat, flat @ layer.w_in.t(), torch.zeros_like(layer.w_in))
    return {"stepped against whole prompt": apart, "first loss": losses[0], "last loss": losses[-1]}


if __name__ == "__main__":
    for name, value in main().items():
        print(f"{name}: {value:.4g}")
