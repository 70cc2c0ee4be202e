"""Plain 64-bit restatement of the microscaled formats and of the operators
over them, on the CPU, for the tests."""
import torch

GRID = {"mx4": [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
        "mx8": [m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127]}
EMAX = {"mx4": 2, "mx8": 8}
SIGN = {"mx4": 8, "mx8": 128}


def quantise(x, kind="mx4"):
    """x [rows, cols], cols a multiple of 32 -> (codes int64 [rows, cols], scale bytes int64 [rows, cols / 32])"""
    b = x.double().reshape(x.shape[0], x.shape[1] // 32, 32)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    top = torch.where(bad | (top == 0), 1.0, top)
    e = (torch.frexp(top)[1].long() - 1 - EMAX[kind]).clamp(min=-127)
    e = torch.where(b.abs().amax(-1) == 0, -127, e)
    y = b / torch.exp2(e.double())[..., None]
    y = torch.where(bad[..., None], 0.0, y)
    grid = torch.tensor(GRID[kind], dtype=torch.float64)
    mid = (grid[1:] + grid[:-1]) / 2
    i = torch.bucketize(y.abs().contiguous(), mid)
    i = i + ((i < mid.numel()) & (y.abs() == mid[i.clamp(max=mid.numel() - 1)]) & (i % 2 == 1)).long()
    codes = i + SIGN[kind] * (torch.signbit(y) & ~bad[..., None]).long()
    s = torch.where(bad, 255, e + 127)
    return codes.reshape(x.shape), s


def values(codes, s, kind="mx4"):
    grid = torch.tensor(GRID[kind] + [float("nan")] * (SIGN[kind] - len(GRID[kind])), dtype=torch.float64)
    v = grid[codes % SIGN[kind]] * torch.where(codes >= SIGN[kind], -1.0, 1.0)
    scale = torch.where(s == 255, float("nan"), torch.exp2(s.double() - 127))
    return (v.reshape(*s.shape, 32) * scale[..., None]).reshape(codes.shape)


def padded(x, multiple):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % multiple))


def stored(x, kind="mx4"):
    """what the blocks along the rows of x [rows, cols] stand for, in 64 bits"""
    return values(*quantise(padded(x.double(), 32), kind), kind)[:, : x.shape[1]]


def pack(x):
    """codes uint8 [rows, pitch] and tiled scales uint8 of the library's 4-bit matrix; rows beyond x's are 0"""
    rows = x.shape[0]
    c, s = quantise(padded(x.double(), 256))
    s = torch.where(torch.isnan(s.double()), 0, s)
    codes = (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8)
    tiles = torch.zeros(-(-rows // 128), s.shape[1] // 4, 32, 4, 4, dtype=torch.uint8)
    r = torch.arange(rows)[:, None]
    b = torch.arange(s.shape[1])[None, :]
    tiles[r // 128, b // 4, r % 32, r // 32 % 4, b % 4] = s.to(torch.uint8)
    return codes, tiles


def untile(tiles, rows):
    """scale bytes [rows, blocks] of tiled scales"""
    r = torch.arange(rows)[:, None]
    b = torch.arange(tiles.shape[1] * 4)[None, :]
    return tiles[r // 128, b // 4, r % 32, r // 32 % 4, b % 4]


#: unit roundoff of the output types, and half the spacing of their subnormals
ROUND = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134)}


def sum_tolerance(want, absolute, terms, dtype):
    """bound on |got - want| of a sum of `terms` products accumulated in 32 bits in any order with every addition off by
    at most one unit in the last place (2^-23 of the partial sum, which `absolute`, the sum of the terms' magnitudes,
    bounds), two more operations after it (bias or gate), rounded once to dtype"""
    u, tiny = ROUND[dtype]
    return (terms + 2) * 2.0 ** -23 * absolute + u * want.abs() + tiny
