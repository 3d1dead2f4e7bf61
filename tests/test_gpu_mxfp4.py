"""gr_quant_mxfp4, gr_dequant_mxfp4 and gr_linear_mxfp4 against float64.

Rows to 4 bits and back are exact: the same codes, scales and values as rounding the
float64 quotients gives.  A product's bound: the matrix core joins four blocks of 32
exact products within 2^-24 of their sum of magnitudes and adds them to a float32 sum
(half a unit, 2^-24 of it), K / 128 times; eight partial sums may be added, and a last
rounding: (2 K / 128 + 16) 2^-24 of the sum of magnitudes in all.  An output of 16
bits adds half a step of it (2^-8 bf16, 2^-11 fp16)."""

import pytest
import torch

from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NUMBERS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BORDERS = (NUMBERS[1:] + NUMBERS[:-1]) / 2
POWERS = torch.pow(2.0, torch.arange(-127, 128, dtype=torch.float64))


def scale_bytes(amax):
    """float64 largest magnitudes -> scale bytes: the least power of two with amax < 7 * 2^e."""
    return torch.searchsorted(7.0 * POWERS, amax, right=True)


def quantise(x):
    """float64 [..., K] -> (codes [..., K], scale bytes [..., K / 32]), on the CPU."""
    b = x.unflatten(-1, (-1, 32))
    byte = scale_bytes(b.abs().amax(-1))
    a = (b / POWERS[byte][..., None]).abs()
    i = torch.bucketize(a, BORDERS)  # the lower of two at a border
    i += ((a == BORDERS[i.clamp_max(6)]) & (i < 7) & (i % 2 == 1)).long()
    return (i + 8 * torch.signbit(b).long()).flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def values(codes, byte):
    """float64 values of codes [..., K] and scale bytes."""
    v = NUMBERS[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    return v * POWERS[byte.long()].repeat_interleave(32, -1)


def operand(g, rows, K, spread=1.0):
    """Packed codes, scale bytes and float64 values of random rows."""
    x = torch.randn(rows, K, generator=g) * torch.exp(spread * torch.randn(1, K, generator=g))
    codes, byte = quantise(x.double())
    return pack(codes), byte, values(codes, byte)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,K", [(1, 32), (3, 96), (5, 160), (17, 2048), (300, 6144), (1025, 416), (4099, 4096)])
def test_quant_and_back(device, dtype, T, K):
    g = torch.Generator().manual_seed(T + K)
    x = (torch.randn(T, K + 32, generator=g) * torch.exp(2 * torch.randn(T, 1, generator=g))).to(dtype)
    x[0, :K // 2] = 0
    x[-1, 1:K:3] *= 0.01
    got, s = ops.quant_mxfp4(x.to(device)[:, :K])  # strided rows
    want, ws = quantise(x[:, :K].double())
    assert got.shape == (T, K // 2) and s.shape == (T, K // 32) and got.dtype == s.dtype == torch.uint8
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(got.cpu(), pack(want))
    v = values(want, ws)
    for to in (torch.bfloat16, torch.float16, torch.float32):
        back = ops.dequant_mxfp4(got, s, dtype=to)
        assert back.dtype == to and torch.equal(back.cpu(), v.to(to))


def test_quant_on_borders(device):
    """Values on and next to the borders between two numbers, and largest values on and
    next to the borders between two scales (1.75 times a power of two), over the whole
    range of scales."""
    rows = []
    for e in (-127, -126, -100, -1, 0, 1, 60, 124, 125):
        unit = 2.0 ** e
        near = torch.cat([BORDERS, NUMBERS, torch.tensor([6.5], dtype=torch.float64)]) * unit
        near = near.float()
        near = torch.cat([near, torch.nextafter(near, torch.tensor(0.0)), torch.nextafter(near, torch.tensor(3e38))])
        for top in (4.0, 6.999999, 7.0, 7.000001, 3.499999):
            block = torch.cat([near[:31 * (len(near) // 31)], -near[:31 * (len(near) // 31)]]).view(-1, 31)
            block = block.clamp(-top * unit, top * unit)
            rows.append(torch.cat([block, torch.full((len(block), 1), top * unit)], 1))
    x = torch.cat(rows).float()
    x = x[:len(x) // 3 * 3].view(-1, 96)
    got, s = ops.quant_mxfp4(x.to(device))
    want, ws = quantise(x.double())
    assert torch.equal(s.cpu(), ws) and torch.equal(got.cpu(), pack(want))


def test_every_16_bit_value(device):
    """Each finite bf16 and fp16 value as its block's largest, and beside a larger one."""
    for dtype in (torch.bfloat16, torch.float16):
        v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
        v = v[torch.isfinite(v)]
        v = v[:len(v) // 32 * 32]
        x = torch.zeros(len(v), 64, dtype=dtype)
        x[:, 5] = v
        x[:, 32:] = v.view(-1, 32).repeat_interleave(32, 0)
        got, s = ops.quant_mxfp4(x.to(device))
        want, ws = quantise(x.double())
        assert torch.equal(s.cpu(), ws) and torch.equal(got.cpu(), pack(want))


def test_quant_not_finite_and_strided_outputs(device):
    x = torch.randn(6, 96, generator=torch.Generator().manual_seed(2))
    x[1, 33] = float("inf")
    x[2, 5] = float("nan")
    x[3] = 0
    x[4, :32] = 1e-45
    x[5, :32] = 3.4e38
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype)
        out = torch.full((6, 64), 0xEE, dtype=torch.uint8, device=device)
        scale = torch.full((6, 5), 7, dtype=torch.uint8, device=device)
        got, s = ops.quant_mxfp4(xd.to(device), out=out[:, :48], scale=scale[:, 1:4])
        back = ops.dequant_mxfp4(got, s, dtype=torch.float32).cpu().view(6, 3, 32)
        bad = ~torch.isfinite(xd.view(6, 3, 32)).all(-1)
        assert torch.isnan(back).all(-1).equal(bad) and torch.isnan(back).any(-1).equal(bad)
        want, ws = quantise(torch.where(bad.repeat_interleave(32, 1), 0, xd.double()))
        assert torch.equal(s.cpu(), torch.where(bad, 255, ws))
        assert torch.equal(unpack(got.cpu())[~bad.repeat_interleave(32, 1)], want[~bad.repeat_interleave(32, 1)])
        assert (scale[:, [0, 4]] == 7).all() and (out[:, 48:] == 0xEE).all()


def test_every_code_and_scale_back(device):
    """Each code with each scale byte, in each type; byte 255 is NaN."""
    codes = torch.arange(32).to(torch.uint8) % 16
    x = pack(codes).repeat(256, 1)
    byte = torch.arange(256).to(torch.uint8)[:, None]
    want = values(codes.repeat(256, 1)[:255], byte[:255])
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        got = ops.dequant_mxfp4(x.to(device), byte.to(device), dtype=dtype).cpu()
        assert torch.isnan(got[255]).all()
        assert torch.equal(got[:255], want.to(dtype))
        out = torch.full((256, 48), 3.0, dtype=dtype, device=device)
        ops.dequant_mxfp4(x.to(device), byte.to(device).view(torch.float8_e8m0fnu), dtype=dtype, out=out[:, 8:40])
        assert torch.equal(out[:255, 8:40].cpu(), want.to(dtype)) and (out[:, :8] == 3).all() and (out[:, 40:] == 3).all()


def unit(K):
    return (2 * -(-K // 128) + 16) * 2.0 ** -24


def gated(gate, up, dg, du):
    """silu(gate) * up and how far it may be off for errors dg, du of its operands:
    |silu'| <= 1.1, |silu| <= |gate|; the exponential's and the reciprocal's own error
    2^-21 of the result."""
    y = gate * torch.sigmoid(gate) * up
    return y, 1.01 * (1.1 * dg * up.abs() + gate.abs() * du) + y.abs() * 2.0 ** -21 + 2.0 ** -60


def operands(M, N, K, swiglu, device, seed=0):
    g = torch.Generator().manual_seed(M + N + K + seed)
    x4, xs, x = operand(g, M, K)
    w4, ws, w = operand(g, 2 * N if swiglu else N, K, 0.2)
    w, ws = w * 2.0 ** -5, ws - 5  # (weights of ordinary size; random rows' scales are near 127)
    y, err = x @ w.t(), x.abs() @ w.abs().t() * unit(K)
    if swiglu:
        y, err = gated(y[:, :N], y[:, N:], err[:, :N], err[:, N:])
    return [t.to(device) for t in (x4, xs, w4, ws)], y, err


def check(got, y, err):
    half = HALF[got.dtype]
    assert ((got.cpu().double() - y).abs() <= err + (y.abs() + err) * half + 2.0 ** -25).all()


def check_4bit(packed, byte, y, err):
    """Codes and scales of results that are off by err at most: the scale is one that a
    largest value within its error has, the number a nearest one of a value within its."""
    top = y.abs().unflatten(-1, (-1, 32))
    off = err.unflatten(-1, (-1, 32))
    lo, hi = scale_bytes((top - off).clamp_min(0).amax(-1)), scale_bytes((top + off).amax(-1))
    byte = byte.cpu().long()
    assert ((byte >= lo) & (byte <= hi)).all()
    got = values(unpack(packed.cpu()), byte)
    grid = NUMBERS * torch.ones(()).double()
    a = (y / POWERS[byte].repeat_interleave(32, -1)).abs()
    nearest = torch.stack([(a - n).abs() for n in grid]).amin(0) * POWERS[byte].repeat_interleave(32, -1)
    assert ((got - y).abs() <= nearest + 2 * err).all()


# one row to many, columns that end inside a tile, a fragment or a group of four, depth
# that ends inside a stage, an instruction or four scales
SIZES = [(1, 16, 32), (1, 2048, 2048), (8, 4096, 512), (15, 100, 160), (16, 48, 6144), (17, 33, 288), (33, 257, 1024),
         (64, 256, 128), (65, 128, 640), (127, 400, 2080), (129, 1, 384), (250, 1000, 256), (257, 513, 544),
         (520, 768, 2048), (1000, 272, 416), (300, 4097, 96)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(device, M, N, K):
    ops_, y, err = operands(M, N, K, False, device)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        check(ops.linear_mxfp4(*ops_, out_dtype=dtype), y, err)


@pytest.mark.parametrize("M,N,K", [(1, 32, 32), (8, 6144, 2048), (15, 96, 160), (16, 48, 6144), (33, 256, 1024),
                                   (65, 128, 640), (127, 416, 2080), (250, 1024, 256), (520, 768, 2048), (1001, 2048, 352)])
def test_swiglu_and_quantized(device, M, N, K):
    ops_, y, err = operands(M, N, K, True, device)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        check(ops.linear_mxfp4(*ops_, swiglu=True, out_dtype=dtype), y, err)
    if N % 32 == 0:
        check_4bit(*ops.linear_mxfp4(*ops_, swiglu=True, quantized=True), y, err)
        ops_, y, err = operands(M, N, K, False, device)
        check_4bit(*ops.linear_mxfp4(*ops_, quantized=True), y, err)


def test_linear_operand_layout(device):
    """Whole numbers, whose sums are exact: each feature, row and scale in its place."""
    for M, N, K in ((3, 40, 288), (70, 200, 544), (300, 520, 1024), (600, 2100, 512)):
        g = torch.Generator().manual_seed(K)
        cx, cw = (torch.randint(0, 16, (n, K), generator=g, dtype=torch.uint8) for n in (M, N))
        bx, bw = (torch.randint(125, 130, (n, K // 32), generator=g, dtype=torch.uint8) for n in (M, N))
        y = values(cx, bx) @ values(cw, bw).t()
        got = ops.linear_mxfp4(*(t.to(device) for t in (pack(cx), bx, pack(cw), bw)), out_dtype=torch.float32)
        assert torch.equal(got.cpu().double(), y)  # (multiples of 2^-6, and sums far below 2^18)
