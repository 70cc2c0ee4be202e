"""Cases of the block-scaled operators: microscaled 4-bit quantisation and
product, the quantised sequence cache, and the single-token convolution that
reads it.

Layouts (the library's own, made here from plain torch so that both forms take
the same data):

  4-bit matrix [rows, cols]   codes: uint8 [rows, pitch], two E2M1 codes a byte
                              (the lower index in the low half), pitch =
                              ceil(cols / 256) * 128, zero beyond cols;
                              scales: E8M0 bytes, one per 32 columns, in tiles
                              of 128 rows x 4 blocks: [rows/128][pitch/64][32][4][4]
                              = [row tile][block tile][row % 32][row / 32 % 4][block % 4]
  sequence cache              codes: uint8 [pages, page_size, C / 2] (mx4) or
                              [pages, page_size, C] (mx8, E4M3); scales: uint8
                              [pages, page_size, C / 32]; page_table: int32
                              [sequences, max_pages]
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_CACHE_BYTES = {"mx4": 17 / 32, "mx8": 33 / 32}   # a stored value with its share of the scale


# ---- cases -----------------------------------------------------------------
def listed():
    return [
        # activations of one decoding step of a small batch, quantised for the product that follows
        {"name": "quantise-step", "op": "quantise", "rows": 16, "cols": 4096, "dtype": "bf16", "mode": "rows"},
        # master weights of one layer before a training step: along both axes, for the product and its gradient
        {"name": "quantise-weights", "op": "quantise", "rows": 8192, "cols": 8192, "dtype": "fp32", "mode": "both"},
        # one token through a projection, weights in 4 bits
        {"name": "linear-token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "bias": True},
        # a ragged batch of prompt tokens, sizes that fill no tile
        {"name": "linear-odd", "op": "linear", "m": 333, "n": 1537, "k": 1111, "dtype": "fp16", "bias": True},
        # prompt tokens of a large batch
        {"name": "linear-prompt", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "bias": False},
        # one training step of a projection: the product and both gradients
        {"name": "linear-train", "op": "train", "m": 8192, "n": 4096, "k": 2048, "dtype": "bf16"},
        # generation with a short filter: one token stored per sequence, the last 16 read back
        {"name": "cache-step", "op": "cache", "batch": 64, "channels": 2048, "new": 1, "ragged": False, "history": 1000,
         "read": 16, "page": 64, "kind": "mx8", "dtype": "bf16", "order": "tokens"},
        # prompts of unequal length stored and read back token by token
        {"name": "cache-prompt", "op": "cache", "batch": 8, "channels": 4096, "new": 8192, "ragged": True, "history": 0,
         "read": 0, "page": 64, "kind": "mx4", "dtype": "bf16", "order": "tokens"},
        # prompts stored and read back channel by channel, zero padded: the rows that the FFT convolution takes
        {"name": "cache-channels", "op": "cache", "batch": 8, "channels": 1056, "new": 2048, "ragged": True, "history": 37,
         "read": 0, "page": 48, "kind": "mx8", "dtype": "fp32", "order": "channels"},
        # one sequence, one token: where latency counts
        {"name": "conv-one", "op": "conv", "batch": 1, "channels": 1024, "length": 4096, "taps": 4096, "heads": 1024,
         "page": 64, "kind": "mx8", "dtype": "bf16", "taps_dtype": "fp32", "gate": True, "ragged": False},
        # a small ragged batch, filters shared by heads of 96 channels, pages that end inside a tile
        {"name": "conv-heads", "op": "conv", "batch": 5, "channels": 2112, "length": 5000, "taps": 3001, "heads": 22,
         "page": 100, "kind": "mx4", "dtype": "fp16", "taps_dtype": "fp32", "gate": False, "ragged": True},
        # a serving batch with long histories
        {"name": "conv-batch", "op": "conv", "batch": 16, "channels": 2048, "length": 32768, "taps": 32768, "heads": 2048,
         "page": 64, "kind": "mx4", "dtype": "bf16", "taps_dtype": "bf16", "gate": True, "ragged": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantise", "linear", "train", "cache", "conv", "conv", "linear", "cache"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "quantise":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 32, 8192), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "mode": rng.choice(["rows", "cols", "both"])}
    if op == "linear":
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 8192), "k": _log(rng, 64, 8192), "dtype": dtype,
                "bias": rng.random() < 0.5}
    if op == "train":
        return {"op": op, "m": _log(rng, 64, 8192), "n": _log(rng, 64, 4096), "k": _log(rng, 64, 2048), "dtype": dtype}
    kind = rng.choice(["mx4", "mx8"])
    page = rng.choice([16, 48, 64, 100, 128])
    if op == "cache":
        order = rng.choice(["tokens", "channels"])
        new = rng.choice([1, _log(rng, 2, 4096)])
        history = 0 if rng.random() < 0.3 else _log(rng, 1, 2000)
        return {"op": op, "batch": _log(rng, 1, 16), "channels": 32 * _log(rng, 1, 64), "new": new, "ragged": rng.random() < 0.5,
                "history": history, "read": rng.choice([0, _log(rng, 1, 64)]), "page": page, "kind": kind,
                "dtype": "fp32" if order == "channels" else rng.choice(["bf16", "fp16", "fp32"]), "order": order}
    channels = 32 * _log(rng, 1, 64)
    heads = rng.choice([channels, channels // 32, 1])
    return {"op": op, "batch": _log(rng, 1, 16), "channels": channels, "length": _log(rng, 1, 16384), "taps": _log(rng, 1, 16384),
            "heads": heads, "page": page, "kind": kind, "dtype": dtype, "taps_dtype": rng.choice(["fp32", "bf16"]),
            "gate": rng.random() < 0.5, "ragged": rng.random() < 0.5}


def _lengths(case, most):
    """sequence lengths of a ragged batch, the longest first, one of them empty where there are several"""
    b = case["batch"]
    if not case["ragged"]:
        return [most] * b
    out = [max(1, most * (2 * b - i) // (2 * b) - 3 * i) for i in range(b)]
    if b > 2:
        out[b // 2] = 0
    return out


def work(case):
    op = case["op"]
    if op == "quantise":
        n = case["rows"] * case["cols"]
        sides = 2 if case["mode"] == "both" else 1
        return {"bytes": n * (_BYTES[case["dtype"]] * (1 + sides) + sides * 17 / 32), "flops": 2.0 * n * sides}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m * k + m * n) * _BYTES[case["dtype"]] + n * k * 17 / 32 + (4 * n if case["bias"] else 0),
                "flops": 2.0 * m * n * k}
    if op == "train":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * (m * k + n * k + m * n) * _BYTES[case["dtype"]], "flops": 6.0 * m * n * k}
    if op == "cache":
        new = _lengths(case, case["new"])
        read = [case["read"] and min(case["read"], case["history"] + t) or case["history"] + t for t in new]
        c, size, stored = case["channels"], _BYTES[case["dtype"]], _CACHE_BYTES[case["kind"]]
        if case["order"] == "channels":
            written = case["batch"] * _padded(max(read)) * c * 4
        else:
            written = sum(read) * c * size
        return {"bytes": sum(new) * c * (size + stored) + sum(read) * c * stored + written,
                "flops": 2.0 * c * (sum(new) + sum(read))}
    lens = [min(t, case["taps"]) for t in _lengths(case, case["length"])]
    c = case["channels"]
    small = case["batch"] * c * _BYTES[case["dtype"]] * (2 if case["gate"] else 1)
    return {"bytes": sum(lens) * c * _CACHE_BYTES[case["kind"]] + max(lens) * case["heads"] * _BYTES[case["taps_dtype"]] + small,
            "flops": 2.0 * sum(lens) * c}


def _padded(t):
    """the transform that holds t samples and as many zeros"""
    n = 16
    while n < 2 * t:
        n *= 2
    return n


# ---- plain form of the formats (32 bits) ------------------------------------
def _two(e):
    """2 ** e in 32 bits from its bits, for whole -127 <= e <= 127: a power function may be off by a bit"""
    return torch.where(e < -126, 1 << 22, (e + 127).clamp(min=0) << 23).int().view(torch.float32)


def _round_e2m1(y):
    mag = y.abs()
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    return torch.copysign((torch.round(mag / step) * step).clamp(max=6.0), y)


def _round_e4m3(y):
    mag = y.abs()
    ex = (torch.frexp(mag)[1] - 1).clamp(min=-6)
    step = _two(ex - 3)
    return torch.copysign((torch.round(mag / step) * step).clamp(max=448.0), y)


def _blocks(x, emax):
    """x [..., C] in 32 bits, C a multiple of 32: (values over the block's scale [..., C / 32, 32], exponent [..., C / 32])"""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    e = (torch.frexp(b.abs().amax(-1))[1] - 1 - emax).clamp(min=-127)
    return b * _two(-e)[..., None], e


def _fill(x, multiple):
    more = -x.shape[-1] % multiple
    return torch.nn.functional.pad(x, (0, more)) if more else x


def _quantised(x):
    """x [rows, cols] -> the values its 4-bit blocks stand for, in 32 bits"""
    y, e = _blocks(_fill(x.float(), 32), 2)
    return (_round_e2m1(y) * _two(e)[..., None]).reshape(x.shape[0], -1)[:, : x.shape[1]]


def _e2m1_codes(q):
    mag = q.abs()
    code = torch.where(mag < 2, mag * 2, torch.where(mag < 4, mag + 2, mag / 2 + 4))
    return code.to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)


def _e2m1_values(codes):
    """uint8 [..., n] of two codes a byte -> [..., 2 n] in 32 bits"""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)
    return table[both.int()]


def _pack(x):
    """x [rows, cols] -> codes and tiled scales of the library's 4-bit matrix"""
    rows = x.shape[0]
    y, e = _blocks(_fill(x.float(), 256), 2)
    codes = _e2m1_codes(_round_e2m1(y).reshape(rows, -1))
    codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    s = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, 0, 0, -rows % 128))
    s = s.reshape(s.shape[0] // 128, 4, 32, s.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return codes.contiguous(), s


def _unpack(codes, scales, cols):
    s = scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[: codes.shape[0]]
    v = _e2m1_values(codes).reshape(codes.shape[0], -1, 32)
    return (v * _two(s.int() - 127)[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def _encode(x, kind):
    """tokens [T, C] -> cache codes and scales"""
    y, e = _blocks(x.float(), 2 if kind == "mx4" else 8)
    s = (e + 127).to(torch.uint8)
    if kind == "mx4":
        q = _e2m1_codes(_round_e2m1(y).reshape(x.shape))
        return q[:, 0::2] | (q[:, 1::2] << 4), s
    return _round_e4m3(y).reshape(x.shape).to(torch.float8_e4m3fn).view(torch.uint8), s


def _decode(codes, scales, kind):
    """cache codes [..., C / 2 or C] and scales [..., C / 32] -> values in 32 bits"""
    v = _e2m1_values(codes) if kind == "mx4" else codes.contiguous().view(torch.float8_e4m3fn).float()
    b = v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    return (b * _two(scales.int() - 127)[..., None]).reshape(v.shape)


# ---- inputs ------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(g, rows, cols, dtype):
    """normal values over channels of unequal spread, a few of them large"""
    spread = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=g))
    spread = torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 20.0 * spread, spread)
    return (torch.randn(rows, cols, device="cuda", generator=g) * spread).to(_TYPES[dtype])


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    st = {"case": case}
    if op == "quantise":
        st["x"] = _activations(g, case["rows"], case["cols"], case["dtype"])
    elif op == "linear":
        st["x"] = _activations(g, case["m"], case["k"], case["dtype"])
        w = torch.randn(case["n"], case["k"], device="cuda", generator=g) / math.sqrt(case["k"])
        st["codes"], st["scales"] = _pack(w)
        st["bias"] = 0.1 * torch.randn(case["n"], device="cuda", generator=g) if case["bias"] else None
    elif op == "train":
        t = _TYPES[case["dtype"]]
        st["x"] = _activations(g, case["m"], case["k"], case["dtype"])
        st["w"] = (torch.randn(case["n"], case["k"], device="cuda", generator=g) / math.sqrt(case["k"])).to(t)
        st["gy"] = (0.01 * torch.randn(case["m"], case["n"], device="cuda", generator=g)).to(t)
    elif op == "cache":
        new = torch.tensor(_lengths(case, case["new"]), device="cuda")
        total = case["history"] + new
        read = total.clamp(max=case["read"]) if case["read"] else total
        st |= _cache(g, case, case["history"] + case["new"], case["history"])
        st["x"] = _activations(g, int(new.sum()), case["channels"], case["dtype"])
        st["new_cu"], st["new_at"] = _cu(new), torch.full_like(new, case["history"]).int()
        st["read_cu"], st["read_at"], st["read_counts"] = _cu(read), (total - read).int(), read.int()
        st["read_tokens"], st["padded"] = int(read.sum()), _padded(int(read.max()))
    else:
        lens = _lengths(case, case["length"])
        st |= _cache(g, case, case["length"], case["length"])
        st["lengths"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
        lag = torch.arange(case["taps"], device="cuda")[:, None]
        decay = torch.exp(torch.rand(case["heads"], device="cuda", generator=g) * math.log(4096.0) + 1.0)
        taps = torch.exp(-lag / decay) * torch.randn(case["taps"], case["heads"], device="cuda", generator=g)
        st["taps"] = taps.to(_TYPES[case["taps_dtype"]])
        st["gate"] = torch.randn(case["batch"], case["channels"], device="cuda", generator=g).to(_TYPES[case["dtype"]]) if case["gate"] else None
    return st


def _cu(counts):
    return torch.nn.functional.pad(counts.cumsum(0), (1, 0)).int()


def _cache(g, case, longest, filled):
    """a paged cache with pages in shuffled order, `filled` tokens of history in every sequence's pages"""
    b, c, page, kind = case["batch"], case["channels"], case["page"], case["kind"]
    per = -(-longest // page)
    pages = b * per + 3
    table = torch.randperm(pages, device="cuda", generator=g)[: b * per].reshape(b, per).int()
    codes = torch.zeros(pages, page, c // 2 if kind == "mx4" else c, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(pages, page, c // 32, dtype=torch.uint8, device="cuda")
    if filled:
        step = max(1, (1 << 26) // (page * c))
        for at in range(0, pages, step):
            n = min(step, pages - at)
            q, s = _encode(torch.randn(n * page, c, device="cuda", generator=g), kind)
            codes[at:at + n], scales[at:at + n] = q.reshape(n, page, -1), s.reshape(n, page, -1)
    return {"codes": codes, "scales": scales, "table": table}


# ---- one pass ------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from fufft_b200 import ops
    case = st["case"]
    op, dtype = case["op"], _TYPES[case["dtype"]]
    if op == "quantise":
        out = {}
        if case["mode"] == "both":
            q, t = ops.mx4_quantize_both(st["x"])
        else:
            q = t = ops.mx4_quantize(st["x"], transpose=case["mode"] == "cols")
        if case["mode"] != "cols":
            out["rows"] = ops.mx4_dequantize(q, dtype)
        if case["mode"] != "rows":
            out["cols"] = ops.mx4_dequantize(t, dtype)
        return out
    if op == "linear":
        w = ops.Mx4(st["codes"], st["scales"], case["n"], case["k"])
        return ops.mx4_linear(st["x"], w, st["bias"])
    if op == "train":
        xq, xt = ops.mx4_quantize_both(st["x"])
        wq, wt = ops.mx4_quantize_both(st["w"])
        y = ops.mx4_matmul(xq, wq, dtype)
        gx, gw = ops.mx4_linear_grad(st["gy"], xt, wt)
        return {"y": y, "gx": gx, "gw": gw}
    cache = ops.SeqCache(st["codes"], st["scales"], st["table"], case["kind"])
    if op == "cache":
        ops.cache_append(cache, st["x"], st["new_cu"], st["new_at"])
        if case["order"] == "channels":
            return ops.cache_read_channels(cache, st["read_at"], st["read_counts"], st["padded"])
        return ops.cache_read(cache, st["read_cu"], st["read_at"], st["read_tokens"], dtype)
    return ops.cache_conv(cache, st["lengths"], st["taps"], gate=st["gate"], dtype=dtype)


def _slots(st, cu, at, tokens):
    """row of the flattened pages for each token of a ragged run of positions"""
    t = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    pos = at[b].long() + t - cu[b].long()
    page = st["codes"].shape[1]
    return st["table"][b, pos // page].long() * page + pos % page


def _run_plain(st):
    case = st["case"]
    op, dtype = case["op"], _TYPES[case["dtype"]]
    if op == "quantise":
        out = {}
        if case["mode"] != "cols":
            out["rows"] = _quantised(st["x"]).to(dtype)
        if case["mode"] != "rows":
            out["cols"] = _quantised(st["x"].t()).to(dtype)
        return out
    if op == "linear":
        y = _quantised(st["x"]) @ _unpack(st["codes"], st["scales"], case["k"]).t()
        return (y if st["bias"] is None else y + st["bias"]).to(dtype)
    if op == "train":
        x, w, gy = st["x"], st["w"], st["gy"]
        y = _quantised(x) @ _quantised(w).t()
        gx = _quantised(gy) @ _quantised(w.t()).t()
        gw = _quantised(gy.t()) @ _quantised(x.t()).t()
        return {"y": y.to(dtype), "gx": gx.to(dtype), "gw": gw.to(dtype)}
    kind, c = case["kind"], case["channels"]
    codes, scales = st["codes"].flatten(0, 1), st["scales"].flatten(0, 1)
    if op == "cache":
        at = _slots(st, st["new_cu"], st["new_at"], st["x"].shape[0])
        codes[at], scales[at] = _encode(st["x"], kind)
        if case["order"] == "tokens":
            at = _slots(st, st["read_cu"], st["read_at"], st["read_tokens"])
            return _decode(codes[at], scales[at], kind).to(dtype)
        i = torch.arange(st["padded"], device="cuda")
        live = i < st["read_counts"][:, None]
        pos = torch.where(live, st["read_at"][:, None] + i, 0)
        page = st["codes"].shape[1]
        at = st["table"].gather(1, pos // page).long() * page + pos % page
        return torch.where(live[..., None], _decode(codes[at], scales[at], kind), 0.0).transpose(1, 2).contiguous()
    lag = torch.arange(min(case["taps"], case["length"]), device="cuda")
    pos = st["lengths"][:, None].long() - 1 - lag
    live = pos >= 0
    pos = pos.clamp(min=0)
    page = st["codes"].shape[1]
    at = st["table"].gather(1, pos // page).long() * page + pos % page
    x = torch.where(live[..., None], _decode(codes[at], scales[at], kind), 0.0)
    taps = st["taps"][: lag.numel()].float().repeat_interleave(c // case["heads"], 1)
    y = (x * taps).sum(1)
    return (y if st["gate"] is None else y * st["gate"].float()).to(dtype)


# ---- the definition in 64 bits ----------------------------------------------------
def _power(e):
    """2 ** e in 64 bits, exactly"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _grid(kind):
    """the non-negative values of an element type, in order of their codes"""
    if kind == "mx4":
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return [m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127]


def _nearest(v, kind):
    """v >= 0 in 64 bits -> nearest value of the type, ties to the even code, saturating"""
    grid = torch.tensor(_grid(kind), dtype=torch.float64, device=v.device)
    mid = (grid[1:] + grid[:-1]) / 2
    i = torch.bucketize(v.contiguous(), mid)      # mid[i - 1] < v <= mid[i]
    tie = (i < mid.numel()) & (v == mid[i.clamp(max=mid.numel() - 1)]) & (i % 2 == 1)
    return grid[i + tie.long()]


def _stored(x, kind="mx4"):
    """x [rows, cols] of any type -> what its blocks of 32 columns stand for, in 64 bits"""
    rows, cols = x.shape
    v = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    v = v.reshape(rows, -1, 32)
    top = v.abs().max(-1, keepdim=True)[0]
    e = (torch.where(top > 0, top, 1.0).view(torch.int64) >> 52) - 1023 - (2 if kind == "mx4" else 8)
    scale = _power(e.clamp(min=-127))
    return (_nearest(v.abs() / scale, kind) * scale * torch.sign(v)).reshape(rows, -1)[:, :cols]


def _read(codes, scales, kind):
    """cache rows [T, bytes] -> values [T, C] in 64 bits"""
    grid = torch.tensor(_grid(kind), dtype=torch.float64, device=codes.device)
    if kind == "mx4":
        i = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.long, device=codes.device)
        i[:, 0::2], i[:, 1::2] = codes % 16, codes // 16
        v = grid[i % 8] * (1 - 2 * (i // 8))
    else:
        i = codes.long()
        v = grid[(i % 128).clamp(max=126)] * (1 - 2 * (i // 128))
    s = _power(scales.long() - 127)
    return v * s.repeat_interleave(32, 1)


def _weights(st, case):
    n, k = case["n"], case["k"]
    i = torch.empty(n, st["codes"].shape[1] * 2, dtype=torch.long, device="cuda")
    i[:, 0::2], i[:, 1::2] = st["codes"] % 16, st["codes"] // 16
    grid = torch.tensor(_grid("mx4"), dtype=torch.float64, device="cuda")
    r, b = torch.arange(n, device="cuda")[:, None], torch.arange(st["codes"].shape[1] // 16, device="cuda")
    s = st["scales"][r // 128, b // 4, r % 32, r // 32 % 4, b % 4].long()
    v = grid[i % 8] * (1 - 2 * (i // 8)) * _power(s - 127).repeat_interleave(32, 1)
    return v[:, :k]


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "quantise":
        out = {}
        if case["mode"] != "cols":
            out["rows"] = _stored(st["x"])
        if case["mode"] != "rows":
            out["cols"] = _stored(st["x"].t().contiguous())
        return out
    if op == "linear":
        y = torch.einsum("mk,nk->mn", _stored(st["x"]), _weights(st, case))
        return y if st["bias"] is None else y + st["bias"].double()
    if op == "train":
        x, w, gy = st["x"], st["w"], st["gy"]
        cols = lambda v: _stored(v.t().contiguous()).t()  # noqa: E731
        return {"y": torch.einsum("mk,nk->mn", _stored(x), _stored(w)),
                "gx": torch.einsum("mn,nk->mk", _stored(gy), cols(w)),
                "gw": torch.einsum("mn,mk->nk", cols(gy), cols(x))}
    page, kind, c = case["page"], case["kind"], case["channels"]
    codes, scales = st["codes"].flatten(0, 1), st["scales"].flatten(0, 1)
    if op == "cache":
        new, cu, parts = _stored(st["x"], kind), st["new_cu"].tolist(), []
        out = torch.zeros(case["batch"], c, st["padded"], dtype=torch.float64, device="cuda") if case["order"] == "channels" else None
        for b, (at, n) in enumerate(zip(st["read_at"].tolist(), st["read_counts"].tolist())):
            pos = torch.arange(at, at + n, device="cuda")
            row = st["table"][b][pos // page].long() * page + pos % page
            v = _read(codes[row], scales[row], kind)
            fresh = pos >= case["history"]
            v[fresh] = new[cu[b]:cu[b + 1]][pos[fresh] - case["history"]]
            if out is None:
                parts.append(v)
            else:
                out[b, :, :n] = v.t()
        return torch.cat(parts) if out is None else out
    y = torch.zeros(case["batch"], c, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lengths"].tolist()):
        n_lags = min(n, case["taps"])
        for lo in range(0, n_lags, 4096):
            lag = torch.arange(lo, min(lo + 4096, n_lags), device="cuda")
            pos = n - 1 - lag
            row = st["table"][b][pos // page].long() * page + pos % page
            v = _read(codes[row], scales[row], kind).reshape(lag.numel(), case["heads"], -1)
            y[b] += (v * st["taps"][lag].double()[:, :, None]).sum(0).reshape(-1)
    return y if st["gate"] is None else y * st["gate"].double()
