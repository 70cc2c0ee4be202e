"""The quantised sequence cache: stored bits, both ways of reading back, and
the single-token convolution against a plain 64-bit restatement."""
import pytest
import torch

import mx_reference as ref

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
KINDS = ["mx4", "mx8"]


@pytest.fixture()
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from fufft_b200 import ops
    return ops


def _cu(counts):
    return torch.nn.functional.pad(torch.tensor(counts).cumsum(0), (1, 0)).int()


class Model:
    """sequences as plain lists of stored 64-bit rows beside a cache of the library"""

    def __init__(self, ops, batch, longest, channels, page, kind, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        per = -(-longest // page)
        table = torch.randperm(batch * per + 2, generator=self.g)[: batch * per].reshape(batch, per).int()
        self.ops, self.channels, self.kind = ops, channels, kind
        self.cache = ops.seq_cache(batch * per + 2, page, channels, table.cuda(), kind)
        self.rows = [torch.zeros(0, channels, dtype=torch.float64) for _ in range(batch)]

    def append(self, counts, dtype):
        x = torch.randn(sum(counts), self.channels, generator=self.g) * torch.exp2(torch.randint(-6, 6, (1, self.channels), generator=self.g))
        x = x.to(dtype)
        starts = torch.tensor([len(r) for r in self.rows], dtype=torch.int32)
        self.ops.cache_append(self.cache, x.cuda(), _cu(counts).cuda(), starts.cuda())
        for b, part in enumerate(x.split(counts)):
            self.rows[b] = torch.cat((self.rows[b], ref.stored(part, self.kind)))

    @property
    def lengths(self):
        return torch.tensor([len(r) for r in self.rows], dtype=torch.int32)


LAYOUTS = [(1, 1, 32, 16), (3, 70, 96, 16), (2, 130, 1056, 48), (5, 33, 64, 100), (4, 9, 256, 1), (1, 300, 32, 7)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_append_and_read(ops, layout, dtype, kind):
    batch, longest, channels, page = layout
    m = Model(ops, batch, longest, channels, page, kind)
    first = [max(0, longest - 1 - 5 * b) if b % 3 != 1 else 0 for b in range(batch)]
    m.append(first, dtype)
    m.append([1] * batch, dtype)
    counts = m.lengths.tolist()
    got = ops.cache_read(m.cache, _cu(counts).cuda(), torch.zeros(batch, dtype=torch.int32, device="cuda"), sum(counts), dtype)
    assert torch.equal(got.cpu().double(), torch.cat(m.rows).to(dtype).double())
    tail = [min(3, c) for c in counts]
    at = m.lengths - torch.tensor(tail, dtype=torch.int32)
    got = ops.cache_read(m.cache, _cu(tail).cuda(), at.cuda(), sum(tail), torch.float32)
    assert torch.equal(got.cpu().double(), torch.cat([r[len(r) - t:] for r, t in zip(m.rows, tail)]))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_stored_bits(ops, kind):
    """codes, scales and their places: a slot holds what the format says, the other slots are untouched"""
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    cache = ops.seq_cache(3, 4, 64, table, kind)
    x = torch.randn(3, 64, generator=torch.Generator().manual_seed(1))
    x[1, 32:] = 0.0
    x[2, 5] = float("nan")
    ops.cache_append(cache, x.cuda(), torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"))
    codes, s = ref.quantise(x, kind)
    if kind == "mx4":
        codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    want_codes, want_scales = torch.zeros(12, codes.shape[1], dtype=torch.uint8), torch.zeros(12, 2, dtype=torch.uint8)
    at = [2 * 4 + 3, 0, 1]
    want_codes[at], want_scales[at] = codes.to(torch.uint8), s.to(torch.uint8)
    assert torch.equal(cache.codes.cpu().view(12, -1), want_codes) and torch.equal(cache.scales.cpu().view(12, -1), want_scales)
    got = ops.cache_read(cache, torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"), 3, torch.float32)
    assert torch.equal(torch.isnan(got[2]).cpu(), torch.arange(64) < 32)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_missing_pages(ops, kind):
    """tokens without a page are dropped, read as zeros and add nothing to a convolution"""
    table = torch.tensor([[0, -1], [7, 1]], dtype=torch.int32, device="cuda")
    cache = ops.seq_cache(2, 4, 32, table, kind)
    x = torch.ones(16, 32, device="cuda")
    cu = torch.tensor([0, 8, 16], dtype=torch.int32, device="cuda")
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    ops.cache_append(cache, x, cu, zero)
    held = torch.tensor([1.0] * 4 + [0.0] * 4 + [0.0] * 4 + [1.0] * 4, device="cuda")
    assert torch.equal(ops.cache_read(cache, cu, zero, 16, torch.float32)[:, 0], held)
    got = ops.cache_read_channels(cache, zero, torch.tensor([8, 8], dtype=torch.int32, device="cuda"), 8)
    assert torch.equal(got[:, 3], held.view(2, 8))
    y = ops.cache_conv(cache, torch.tensor([8, 8], dtype=torch.int32, device="cuda"), torch.ones(8, 32, device="cuda"), dtype=torch.float32)
    assert bool((y == 4).all())
    beyond = ops.cache_read(cache, cu, torch.tensor([8, -8], dtype=torch.int32, device="cuda"), 16, torch.float32)
    assert bool((beyond == 0).all())
    y = ops.cache_conv(cache, torch.tensor([20, 20], dtype=torch.int32, device="cuda"), torch.ones(30, 32, device="cuda"), dtype=torch.float32)
    assert bool((y == 4).all())


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 16, 100, 513])
def test_read_channels(ops, n, dtype, kind):
    m = Model(ops, 3, 200, 96, 48, kind, seed=3)
    m.append([200, 0, 131], dtype)
    starts, counts = torch.tensor([17, 0, 100], dtype=torch.int32), torch.tensor([183, 0, 31], dtype=torch.int32)
    got = ops.cache_read_channels(m.cache, starts.cuda(), counts.cuda(), n, dtype).cpu().double()
    want = torch.zeros(3, 96, n, dtype=torch.float64)
    for b in range(3):
        r = m.rows[b][starts[b]:starts[b] + counts[b]][:n]
        want[b, :, :len(r)] = r.t()
    assert torch.equal(got, want.to(dtype).double())


@gpu
def test_append_strided(ops):
    m = Model(ops, 2, 40, 64, 16, "mx8")
    base = torch.randn(50, 100, generator=m.g)
    for off in (3, 4):
        x = base.cuda()[:, off:off + 64]
        ops.cache_append(m.cache, x, _cu([30, 20]).cuda(), torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
        got = torch.full((50, 80), 7.0, device="cuda")
        ops.cache_read(m.cache, _cu([30, 20]).cuda(), torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 50, torch.float32, out=got[:, 5:69])
        assert torch.equal(got[:, 5:69].cpu().double(), ref.stored(base[:, off:off + 64], "mx8"))
        assert bool((got[:, :5] == 7).all()) and bool((got[:, 69:] == 7).all())


# batch, lengths, channels, page, taps, heads: one token to long histories, filters shorter and longer than them
STEPS = [(1, [1], 32, 16, 1, 32), (1, [700], 64, 16, 700, 64), (3, [0, 5, 33], 96, 48, 20, 3), (2, [64, 65], 1056, 64, 300, 1056),
         (5, [100, 0, 257, 31, 1], 288, 100, 256, 9), (9, [300, 299, 1, 2, 0, 128, 64, 200, 17], 128, 7, 129, 128),
         (1, [5000], 256, 64, 4999, 1), (2, [1500, 800], 2080, 64, 1024, 65), (17, [90 - 5 * i for i in range(17)], 32, 16, 64, 16),
         (2, [400, 401], 96, 16, 350, 32), (3, [70, 90, 200], 96, 16, 150, 8), (4, [0, 0, 0, 0], 64, 16, 10, 64),
         (6, [1000, 0, 333, 999, 64, 1], 1024, 64, 900, 1024), (3, [300, 299, 2], 2048, 16, 300, 2048), (1, [513], 1088, 100, 700, 1088),
         (2, [0, 0], 512, 64, 200, 512), (4, [129, 128, 127, 0], 3200, 64, 128, 100)]


def _step(m, taps, gate, dtype):
    n, heads = taps.shape
    want = torch.zeros(len(m.rows), m.channels, dtype=torch.float64)
    absolute, terms = want.clone(), 0
    for b, r in enumerate(m.rows):
        k = min(len(r), n)
        t = r.flip(0)[:k] * taps[:k].double().repeat_interleave(m.channels // heads, 1)
        want[b], absolute[b], terms = t.sum(0), t.abs().sum(0), max(terms, k)
    if gate is not None:
        want, absolute = want * gate.double(), absolute * gate.double().abs()
    return want, ref.sum_tolerance(want, absolute, terms, dtype)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("step", STEPS)
def test_conv(ops, step, dtype, kind):
    batch, lengths, channels, page, n, heads = step
    m = Model(ops, batch, max(max(lengths), 1), channels, page, kind, seed=channels)
    m.append(lengths, torch.float32)
    for taps_dtype, gated in ((torch.float32, True), (torch.bfloat16, False)):
        taps = torch.randn(n, heads, generator=m.g).to(taps_dtype)
        gate = torch.randn(batch, channels, generator=m.g).to(dtype) if gated else None
        want, tol = _step(m, taps, gate, dtype)
        got = ops.cache_conv(m.cache, m.lengths.cuda(), taps.cuda(), None if gate is None else gate.cuda(), dtype)
        assert got.dtype == dtype
        err = (got.cpu().double() - want).abs()
        assert bool((err <= tol).all()), float((err - tol).max())


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_conv_missing_pages_in_long_rows(ops, kind):
    """pages that are not there, and codes beside them that are NaN (mx8) or anything (mx4), add nothing"""
    m = Model(ops, 4, 400, 1024, 16, kind, seed=21)
    m.append([400, 399, 17, 200], torch.float32)
    taps = torch.randn(350, 1024, generator=m.g)
    for b, k in ((0, 24), (0, 3), (1, 0), (1, 10), (3, 12)):      # page k of sequence b
        m.cache.codes[m.cache.page_table[b, k].long()] = 0x7F
        m.cache.page_table[b, k] = -1 if k % 2 else m.cache.codes.shape[0]
        m.rows[b][16 * k:16 * k + 16] = 0.0
    want, tol = _step(m, taps, None, torch.float32)
    got = ops.cache_conv(m.cache, m.lengths.cuda(), taps.cuda(), dtype=torch.float32)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    heads = torch.randn(350, 32, generator=m.g)
    want, tol = _step(m, heads, None, torch.float32)
    got = ops.cache_conv(m.cache, m.lengths.cuda(), heads.cuda(), dtype=torch.float32)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("heads", [2048, 64, 2048 // 16])
@pytest.mark.parametrize("kind", KINDS)
def test_conv_long(ops, kind, heads):
    """histories that several launches' worth of CTAs share; the reference from the values read back, in 64 bits"""
    g = torch.Generator(device="cuda").manual_seed(31)
    batch, n, channels, page = 5, 9000, 2048, 64
    per = -(-n // page)
    table = torch.randperm(batch * per, device="cuda", generator=g).view(batch, per).int()
    cache = ops.seq_cache(batch * per, page, channels, table, kind)
    lengths = torch.tensor([9000, 8999, 0, 4097, 100], dtype=torch.int32)
    x = torch.randn(int(lengths.sum()), channels, device="cuda", generator=g)
    cu, zero = _cu(lengths.tolist()).cuda(), torch.zeros(batch, dtype=torch.int32, device="cuda")
    ops.cache_append(cache, x, cu, zero)
    stored = ops.cache_read(cache, cu, zero, x.shape[0], torch.float32).split(lengths.tolist())
    for taps_dtype in (torch.float32, torch.bfloat16):
        taps = torch.randn(8500, heads, device="cuda", generator=g).to(taps_dtype)
        got = ops.cache_conv(cache, lengths.cuda(), taps, dtype=torch.float32).double()
        for b, v in enumerate(stored):
            k = min(len(v), 8500)
            t = v.flip(0)[:k].double() * taps[:k].double().repeat_interleave(channels // heads, 1)
            tol = ref.sum_tolerance(t.sum(0), t.abs().sum(0), k, torch.float32)
            assert bool(((got[b] - t.sum(0)).abs() <= tol).all())
        assert torch.equal(ops.cache_conv(cache, lengths.cuda(), taps, dtype=torch.float32).double(), got)


@gpu
@pytest.mark.parametrize("spread", ["one", "none", "equal", "falling", "any"])
def test_conv_long_unequal(ops, spread):
    """ten groups of sequences whose lengths decide how many CTAs each of them gets"""
    g = torch.Generator(device="cuda").manual_seed(41)
    batch, n, channels, page = 37, 8192, 512, 64
    lengths = {"one": [0] * 30 + [8192] + [0] * 6, "none": [0] * 37, "equal": [8192] * 37,
               "falling": [8192 - 220 * b for b in range(37)],
               "any": torch.randint(0, 8193, (37,), generator=torch.Generator().manual_seed(3)).tolist()}[spread]
    per = n // page
    table = torch.randperm(batch * per, device="cuda", generator=g).view(batch, per).int()
    cache = ops.seq_cache(batch * per, page, channels, table, "mx4")
    cache.codes.random_(0, 256, generator=g)
    cache.scales.random_(120, 131, generator=g)
    lens = torch.tensor(lengths, dtype=torch.int32)
    cu, zero = _cu(lengths).cuda(), torch.zeros(batch, dtype=torch.int32, device="cuda")
    stored = ops.cache_read(cache, cu, zero, sum(lengths), torch.float32).split(lengths)
    for taps_dtype, heads in ((torch.float32, 512), (torch.bfloat16, 16)):
        taps = torch.randn(n, heads, device="cuda", generator=g).to(taps_dtype)
        got = ops.cache_conv(cache, lens.cuda(), taps, dtype=torch.float32).double()
        for b, v in enumerate(stored):
            t = v.flip(0).double() * taps[:len(v)].double().repeat_interleave(channels // heads, 1)
            tol = ref.sum_tolerance(t.sum(0), t.abs().sum(0), len(v), torch.float32)
            assert bool(((got[b] - t.sum(0)).abs() <= tol).all())
        assert torch.equal(ops.cache_conv(cache, lens.cuda(), taps, dtype=torch.float32).double(), got)


@gpu
def test_conv_strides_and_repeats(ops):
    """taps, gate and result as parts of wider rows, unaligned among them; the same bits on every call"""
    m = Model(ops, 3, 900, 96, 16, "mx4", seed=8)
    m.append([900, 77, 450], torch.float32)
    wide = torch.randn(800, 110, generator=m.g)
    gate = torch.randn(3, 110, generator=m.g)
    for off in (0, 1, 4):
        taps, g = wide[:, off:off + 96], gate[:, off:off + 96]
        want, tol = _step(m, taps, g, torch.float32)
        out = torch.full((3, 110), 7.0, device="cuda")
        ops.cache_conv(m.cache, m.lengths.cuda(), wide.cuda()[:, off:off + 96], gate.cuda()[:, off:off + 96], torch.float32, out=out[:, off:off + 96])
        assert bool(((out[:, off:off + 96].cpu().double() - want).abs() <= tol).all())
        assert bool((out[:, :off] == 7).all()) and bool((out[:, off + 96:] == 7).all())
        again = ops.cache_conv(m.cache, m.lengths.cuda(), wide.cuda()[:, off:off + 96], gate.cuda()[:, off:off + 96], torch.float32)
        assert torch.equal(again, out[:, off:off + 96])


@gpu
def test_conv_matches_the_transform(ops):
    """the cache read back channel by channel and convolved by FFT gives the same last outputs, within fp32"""
    n, channels, length = 512, 32, 200
    m = Model(ops, 2, length, channels, 16, "mx8", seed=11)
    m.append([length, length], torch.float32)
    taps = torch.randn(length, channels, generator=m.g)
    rows = ops.cache_read_channels(m.cache, torch.zeros(2, dtype=torch.int32, device="cuda"), m.lengths.cuda(), n)
    h = torch.zeros(channels, n, dtype=torch.complex64)
    h[:, :length] = taps.t()
    spec = ops.filter_from_taps(h.cuda().view(-1), n, ops.LAYOUT_R16_BPERM)
    u, v = ops.conv_r2(rows[0].reshape(-1), rows[1].reshape(-1), spec, n, ops.LAYOUT_R16_BPERM)
    want, tol = _step(m, taps, None, torch.float32)
    got = torch.stack((u.view(channels, n)[:, length - 1], v.view(channels, n)[:, length - 1])).cpu().double()
    assert float((got - want).norm() / want.norm()) <= 2e-6
    y = ops.cache_conv(m.cache, m.lengths.cuda(), taps.cuda(), dtype=torch.float32)
    assert bool(((y.cpu().double() - want).abs() <= tol).all())


@gpu
def test_large_offsets(ops):
    """slots whose byte offset passes 2^31 and 2^32"""
    page, channels = 64, 4096
    pages = (1 << 32) // (page * channels) + 40
    table = torch.tensor([[pages - 1, (1 << 31) // (page * channels) + 1, 0]], dtype=torch.int32, device="cuda")
    cache = ops.seq_cache(pages, page, channels, table, "mx8")
    x = torch.randn(page * 3, channels, generator=torch.Generator().manual_seed(2))
    cu, zero = torch.tensor([0, page * 3], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.cache_append(cache, x.cuda(), cu, zero)
    want = ref.stored(x, "mx8")
    assert torch.equal(ops.cache_read(cache, cu, zero, page * 3, torch.float32).cpu().double(), want)
    taps = torch.ones(page * 3, channels)
    y = ops.cache_conv(cache, torch.tensor([page * 3], dtype=torch.int32, device="cuda"), taps.cuda(), dtype=torch.float32)
    tol = ref.sum_tolerance(want.sum(0), want.abs().sum(0), page * 3, torch.float32)
    assert bool(((y[0].cpu().double() - want.sum(0)).abs() <= tol).all())


@gpu
def test_conv_stream_and_graph(ops):
    m = Model(ops, 2, 300, 64, 16, "mx4", seed=5)
    m.append([300, 200], torch.float32)
    taps, lengths = torch.randn(300, 64, device="cuda"), m.lengths.cuda()
    want = ops.cache_conv(m.cache, lengths, taps)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        t = taps * 2.0
        got = ops.cache_conv(m.cache, lengths, t * 0.5)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    static = torch.zeros_like(lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.cache_conv(m.cache, static, taps)
    static.copy_(lengths)
    graph.replay()
    assert torch.equal(out, want)


@gpu
def test_empty(ops):
    none = ops.seq_cache(0, 16, 64, torch.zeros(0, 0, dtype=torch.int32, device="cuda"))
    zero = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert ops.cache_conv(none, zero, torch.ones(4, 64, device="cuda")).shape == (0, 64)
    assert ops.cache_read_channels(none, zero, zero, 8).shape == (0, 64, 8)
    m = Model(ops, 2, 10, 64, 4, "mx4")
    m.append([0, 0], torch.float32)
    lengths = m.lengths.cuda()
    assert bool((ops.cache_conv(m.cache, lengths, torch.ones(4, 64, device="cuda")) == 0).all())
    assert bool((ops.cache_conv(m.cache, lengths + 3, torch.ones(0, 64, device="cuda")) == 0).all())
    assert ops.cache_read(m.cache, _cu([0, 0]).cuda(), lengths, 0).shape == (0, 64)
    assert bool((ops.cache_read_channels(m.cache, lengths, lengths, 5) == 0).all())


@gpu
@pytest.mark.parametrize("channels", [96, 2048])
def test_no_pages(ops, channels):
    """lengths and a page table, but no page at all: nothing is read, and the outputs are zeros"""
    table = torch.zeros(2, 100, dtype=torch.int32, device="cuda")
    none = ops.seq_cache(0, 16, channels, table)
    lengths = torch.tensor([1600, 3], dtype=torch.int32, device="cuda")
    for heads in (channels, channels // 32, 3 if channels == 96 else 256):
        out = ops.cache_conv(none, lengths, torch.full((700, heads), float("inf"), device="cuda"), dtype=torch.float32)
        assert bool((out == 0).all())
    assert bool((ops.cache_read_channels(none, lengths - lengths, lengths, 300) == 0).all())


@gpu
def test_conv_non_finite_taps(ops):
    """a tap that is infinite or NaN meets only rows that are there, in both kernels"""
    for channels, batch in ((96, 3), (1024, 4)):
        m = Model(ops, batch, 900, channels, 16, "mx4", seed=13)
        lengths = [900, 70, 450, 0][:batch]
        m.append(lengths, torch.float32)
        taps = torch.randn(900, channels, generator=m.g)
        taps[500:], taps[890:] = float("inf"), float("nan")
        got = ops.cache_conv(m.cache, m.lengths.cuda(), taps.cuda(), dtype=torch.float32).cpu()
        assert not bool(got[0].isfinite().any())
        finite = taps.clone()
        finite[500:] = 0.0
        want, tol = _step(m, finite, None, torch.float32)
        assert bool(((got[1:].double() - want[1:]).abs() <= tol[1:]).all())


@gpu
def test_refusals(ops):
    m = Model(ops, 2, 32, 64, 16, "mx4")
    c, cu, at = m.cache, _cu([1, 1]).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    x, taps = torch.zeros(2, 64, device="cuda"), torch.ones(8, 64, device="cuda")
    bad = [lambda: ops.cache_append(c, x[:, :32], cu, at), lambda: ops.cache_append(c, x, cu.long(), at),
           lambda: ops.cache_append(c, x, at, at), lambda: ops.cache_append(c, x.cpu(), cu, at),
           lambda: ops.cache_read(c, cu, at, 2, torch.float32, out=torch.zeros(3, 64, device="cuda")),
           lambda: ops.cache_conv(c, at, taps, gate=torch.zeros(2, 64, device="cuda")),
           lambda: ops.cache_conv(c, at, taps, dtype=torch.float32, out=torch.zeros(2, 64, device="cuda")[:, ::2]),
           lambda: ops.SeqCache(c.codes, c.scales, c.page_table, "mx8"), lambda: ops.SeqCache(c.codes, c.scales, c.page_table, "mx5"),
           lambda: ops.seq_cache(3, 16, 33, c.page_table)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        ops.cache_conv(c, at, taps.half())
    with pytest.raises(TypeError):
        ops.cache_append(c, x.double(), cu, at)
    with pytest.raises(ops.FufftError):
        ops.cache_conv(c, at, torch.ones(8, 7, device="cuda"))

def test_refusals_before_device():
    import ctypes as ct
    from fufft_b200._lib import CacheDesc, lib
    L, P = lib(), 1 << 20
    SIZE, BATCH, MISALIGNED, ARG = 1, 2, 3, 7

    def desc(**kw):
        d = dict(codes=P, scales=P, page_table=P, table_stride=4, kind=0, channels=64, page_size=16, pages=8, max_pages=4, batch=2)
        d.update(kw)
        return ct.addressof(keep.setdefault(str(kw), CacheDesc(**d)))

    keep = {}
    append = lambda d, **kw: L.fufft_cache_append(d, *[kw.get(k, v) for k, v in (  # noqa: E731
        ("x", P), ("dtype", 0), ("row_stride", 64), ("cu", P), ("starts", P), ("tokens", 3))], None)
    assert append(None) == ARG
    assert append(desc(kind=2)) == ARG
    assert append(desc(channels=48)) == SIZE and append(desc(channels=0)) == SIZE and append(desc(page_size=0)) == SIZE
    assert append(desc(batch=-1)) == BATCH
    assert append(desc(table_stride=3)) == ARG and append(desc(codes=None)) == ARG and append(desc(page_table=None)) == ARG
    assert append(desc(codes=P + 8)) == MISALIGNED
    assert append(desc(), dtype=3) == ARG and append(desc(), tokens=-1) == SIZE and append(desc(), row_stride=63) == ARG
    assert append(desc(), x=None) == ARG and append(desc(), x=P + 2) == MISALIGNED
    assert append(desc(), tokens=0) == 0 and append(desc(batch=0)) == 0
    assert L.fufft_cache_read(desc(), None, 0, 64, P, P, 3, None) == ARG
    assert L.fufft_cache_read_channels(desc(), P, 0, -1, P, P, None) == SIZE
    assert L.fufft_cache_read_channels(desc(), P, 0, 16, None, P, None) == ARG
    conv = lambda d, **kw: L.fufft_cache_conv(d, *[kw.get(k, v) for k, v in (  # noqa: E731
        ("lengths", P), ("taps", P), ("taps_dtype", 0), ("n", 8), ("heads", 64), ("taps_stride", 64), ("gate", None), ("gate_stride", 0),
        ("out", P), ("dtype", 0), ("out_stride", 64), ("workspace", None), ("bytes", 0))], None)
    assert conv(desc(), taps_dtype=1) == ARG and conv(desc(), dtype=5) == ARG
    assert conv(desc(), heads=0) == SIZE and conv(desc(), heads=7) == SIZE and conv(desc(), n=-1) == SIZE
    assert conv(desc(), taps=None) == ARG and conv(desc(), out=None) == ARG and conv(desc(), taps_stride=63) == ARG
    assert conv(desc(), out_stride=63) == ARG and conv(desc(), gate=P, gate_stride=63) == ARG
    assert conv(desc(), taps=P + 2) == MISALIGNED and conv(desc(), workspace=P + 4) == MISALIGNED
    assert conv(desc(batch=0)) == 0
