"""gr_quant_fp8 and gr_linear_fp8 against float64.

The quantiser is exact: the same e4m3 numbers and scales as rounding the float64
quotient gives.  A product's bound: float32 sums of K terms are off by at most
K 2^-24 of the sum of their magnitudes (here K / 8: errors of both signs, and 8
more units for the scales and the last additions); an output of 16 bits adds half
a unit in the last place (2^-8 bf16, 2^-11 fp16).  Results of 16 bits come from the
8-bit matrix instruction, which cuts products off below 2^-13 of the largest power
of two of their group of 8: at most 7 x 2^-13 of the group's largest product, so of
the sum of magnitudes; the cuts are of either sign, so in the norm of many results
sqrt(7 / 3) 2^-13 times the largest over the root of the sum of squares, below 2^-11."""

import pytest
import torch

from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def quantise(x):
    """float64 [T, K] -> (e4m3 numbers, scales) in float64, on the CPU."""
    T, K = x.shape
    G = -(-K // 128)
    xp = torch.zeros(T, G * 128, dtype=torch.float64)
    xp[:, :K] = x
    xp = xp.view(T, G, 128)
    s = (xp.abs().amax(-1) / 448).float().double().clamp_min(2.0 ** -80)
    table = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    mid = (table[1:] + table[:-1]) / 2
    a = (xp / s[..., None]).abs().clamp_max(448)
    i = torch.bucketize(a, mid)
    i += ((a == mid[i.clamp_max(125)]) & (i < 126) & (i % 2 == 1)).long()
    return (table[i] * torch.sign(xp)).view(T, -1)[:, :K], s


def expand(s, n, axis):
    return s.repeat_interleave(128, axis).narrow(axis, 0, n)


def weights(g, N, K, std=0.05):
    w = torch.randn(N, K, generator=g) * std
    nb, kb = -(-N // 128), -(-K // 128)
    p = torch.zeros(nb * 128, kb * 128)
    p[:N, :K] = w
    s = p.view(nb, 128, kb, 128).abs().amax((1, 3)) / 448
    w8 = (w / expand(expand(s, N, 0), K, 1)).to(E4M3)
    return w8, s, w8.double() * expand(expand(s.double(), N, 0), K, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,K", [(1, 16), (3, 128), (5, 144), (17, 2048), (300, 6144), (1025, 400)])
def test_quant(device, dtype, T, K):
    g = torch.Generator().manual_seed(T + K)
    x = (torch.randn(T, K + 16, generator=g) * torch.exp(2 * torch.randn(T, 1, generator=g))).to(dtype)
    x[0, :K // 2] = 0  # a group (or half of one) of zeros
    got, s = ops.quant_fp8(x.to(device)[:, :K])  # strided rows
    want, ws = quantise(x[:, :K].double())
    assert got.dtype == E4M3 and s.shape == (T, -(-K // 128))
    assert torch.equal(s.cpu().double(), ws)
    assert torch.equal(got.cpu().double(), want)


def test_quant_on_borders(device):
    """Values whose float32 quotient falls on the border between two e4m3 numbers
    while the exact one does not, and ones that are on it: a scale with a full
    mantissa, and x next to (number + half a step) * scale."""
    g = torch.Generator().manual_seed(1)
    rows = []
    table = torch.arange(127, dtype=torch.uint8).view(E4M3).double()
    mid = (table[1:] + table[:-1]) / 2
    for _ in range(64):
        amax = (torch.rand(1, generator=g, dtype=torch.float64) * 3 + 1).float()
        s = (amax.double() / 448).float().double()
        x = (mid * s).float()
        near = torch.cat([x, torch.nextafter(x, torch.tensor(0.0)), torch.nextafter(x, torch.tensor(1e9)), -x])[:504]
        near = near[near.abs() <= amax]
        for i in range(0, len(near) - 127, 127):
            rows.append(torch.cat([near[i:i + 127], amax]))
    x = torch.stack(rows)
    got, s = ops.quant_fp8(x.to(device))
    want, ws = quantise(x.double())
    assert torch.equal(s.cpu().double(), ws) and torch.equal(got.cpu().double(), want)


def test_quant_not_finite_tiny_and_strided_outputs(device):
    x = torch.randn(6, 384, generator=torch.Generator().manual_seed(2))
    x[1, 130] = float("inf")
    x[2, 5] = float("nan")
    x[3] = 0
    x[4, :128] = 1e-30
    x[5, :128] = 3e38
    out = torch.zeros(6, 400, dtype=torch.uint8, device=device).view(E4M3)
    scale = torch.full((6, 5), 7.0, device=device)
    got, s = ops.quant_fp8(x.to(device), out=out[:, :384], scale=scale[:, 1:4])
    v = got.cpu().double() * expand(s.cpu().double(), 384, 1)
    bad = torch.zeros(6, 3, dtype=torch.bool)
    bad[1, 1] = bad[2, 0] = True
    assert torch.isnan(v.view(6, 3, 128)).all(-1).equal(bad)  # the whole group, and no other
    assert s[1, 1] == float("inf") and torch.isnan(s[2, 0])
    ok = ~expand(bad, 384, 1)
    want, ws = quantise(torch.where(ok, x.double(), 0))
    assert torch.equal(torch.where(ok, got.cpu().double(), 0), torch.where(ok, want, 0))
    assert (s[3] == 2.0 ** -80).all() and (v[3] == 0).all()
    assert (scale[:, [0, 4]] == 7).all() and (out.view(torch.uint8)[:, 384:] == 0).all()


def operands(M, N, K, swiglu, device, seed=0):
    g = torch.Generator().manual_seed(M + N + K + seed)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(1, K, generator=g))
    x8, xs = quantise(x.double())
    parts = [weights(g, N, K) for _ in range(2 if swiglu else 1)]
    w8, ws = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    xd = x8 * expand(xs, K, 1)
    ys = [xd @ p[2].t() for p in parts]
    errs = [xd.abs() @ p[2].abs().t() * (K / 8 + 8) * 2.0 ** -24 for p in parts]
    if swiglu:
        (gate, up), (dg, du) = ys, errs
        y = gate * torch.sigmoid(gate) * up
        # |silu'| <= 1.1, |silu| <= |gate|; the exponential's and the quotient's own error 2^-21 of the result
        err = 1.01 * (1.1 * dg * up.abs() + gate.abs() * du) + y.abs() * 2.0 ** -21 + 2.0 ** -60
    else:
        y, err = ys[0], errs[0]
    to = lambda t: t.to(device)
    unit = (K / 8 + 8) * 2.0 ** -24
    mag = 1.1 * errs[0] * ys[-1].abs() + ys[0].abs() * errs[-1] if swiglu else errs[0]
    return (to(x8.to(E4M3)), to(xs.float()), to(w8), to(ws)), y, err, mag / unit


# one row to many, columns that end inside a tile, a fragment or a group of four, depth that ends inside a block
SIZES = [(1, 16, 16), (1, 2048, 2048), (8, 4096, 512), (15, 100, 144), (16, 48, 6144), (17, 33, 272), (33, 257, 1024),
         (64, 256, 128), (65, 128, 640), (127, 400, 2064), (129, 1, 384), (250, 1000, 256), (257, 513, 528),
         (520, 768, 2048), (1000, 272, 400)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(device, M, N, K):
    (x8, xs, w8, ws), y, err, mag = operands(M, N, K, False, device)
    y32 = ops.linear_fp8(x8, xs, w8, ws, out_dtype=torch.float32)
    assert ((y32.cpu().double() - y).abs() <= err).all()
    for dtype in (torch.bfloat16, torch.float16):
        check_16(ops.linear_fp8(x8, xs, w8, ws, out_dtype=dtype), y, mag, err)


CUT = 7 * 2.0 ** -13


def check_16(got, y, mag, err):
    """A 16-bit result of sums whose products' magnitudes add up to mag (with the gate: what they move it by)."""
    d, half = (got.cpu().double() - y).abs(), HALF[got.dtype]
    assert (d <= 1.01 * (err + mag * CUT) + y.abs() * half * 1.01 + 2.0 ** -25).all()
    assert d.norm() <= (half + 2.0 ** -11) * y.norm() + 2.0 ** -25 * y.numel() ** 0.5


def check_quantised(got, s, y, err):
    """A quantised result: scales within the float32 sums' error, values within that
    and half a step (2^-4 of the value, 2^-10 of the scale below the normal range)."""
    N = y.shape[1]
    dev = expand((torch.nn.functional.pad(err, (0, -N % 128)).view(err.shape[0], -1, 128).amax(-1)), N, 1)
    s = s.cpu().double()
    want = quantise(y)[1]
    lim = torch.nn.functional.pad(err, (0, -N % 128)).view(err.shape[0], -1, 128).amax(-1) / 448
    assert ((s - want).abs() <= lim + want * 2.0 ** -23).all()
    v = got.cpu().double() * expand(s, N, 1)
    step = torch.maximum(y.abs() * 2.0 ** -4, expand(s, N, 1) * 2.0 ** -10)
    assert ((v - y).abs() <= (step + err) * 1.07 + dev * 2.0 ** -4).all()
    # and as the float32 results' own quantisation gives it, but for values at a border
    assert (got.cpu().double() != quantise(y)[0]).double().mean() <= 2e-3 + 4.0 / y.numel()


@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (8, 768, 512), (15, 96, 144), (17, 6144, 2048), (64, 128, 128), (65, 144, 640),
                                   (130, 400, 1024), (300, 272, 2064), (513, 640, 256)])
def test_linear_swiglu_and_quantized(device, M, N, K):
    (x8, xs, w8, ws), y, err, mag = operands(M, N, K, True, device)
    y32 = ops.linear_fp8(x8, xs, w8, ws, swiglu=True, out_dtype=torch.float32)
    assert ((y32.cpu().double() - y).abs() <= err).all()
    for dtype in (torch.bfloat16, torch.float16):
        check_16(ops.linear_fp8(x8, xs, w8, ws, swiglu=True, out_dtype=dtype), y, mag, err)
    check_quantised(*ops.linear_fp8(x8, xs, w8, ws, swiglu=True, quantized=True), y, err)
    (x8, xs, w8, ws), y, err, mag = operands(M, N, K, False, device)
    check_quantised(*ops.linear_fp8(x8, xs, w8, ws, quantized=True), y, err)


def test_linear_strides_and_special_values(device):
    """Padded rows, scales in either order, results into part of a wider tensor; a
    row of NaN or of infinite scale stays its own row's."""
    M, N, K = 70, 130, 272
    (x8, xs, w8, ws), y, err, mag = operands(M, N, K, False, device)
    xw = torch.zeros(M, K + 32, dtype=torch.uint8, device=device).view(E4M3)
    ww = torch.zeros(N, K + 16, dtype=torch.uint8, device=device).view(E4M3)
    xw[:, :K].copy_(x8)
    ww[:, :K].copy_(w8)
    xw.view(torch.uint8)[:, K:] = 0x7F  # NaN behind the rows
    ww.view(torch.uint8)[:, K:] = 0x7F
    plain = ops.linear_fp8(x8, xs, w8, ws, out_dtype=torch.float32)
    for scale in (xs, xs.t().contiguous().t()):
        out = torch.full((M + 2, N + 6), 9.0, device=device)
        ops.linear_fp8(xw[:, :K], scale, ww[:, :K], ws, out_dtype=torch.float32, out=out[1:-1, :N])
        assert torch.equal(out[1:-1, :N], plain)
        out[1:-1, :N] = 9.0
        assert (out == 9.0).all()
    xs2 = xs.clone()
    xs2[3] = float("nan")
    xs2[69, 1] = float("inf")
    got = ops.linear_fp8(x8, xs2, w8, ws, out_dtype=torch.float32)
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[69]).any()
    keep = [i for i in range(M) if i not in (3, 69)]
    assert torch.equal(got[keep], plain[keep])


def test_linear_alone_equals_among_others(device):
    """A row's result does not depend on which rows of its tile share the call."""
    (x8, xs, w8, ws), _, _, _ = operands(256, 256, 1024, False, device)
    full = ops.linear_fp8(x8, xs, w8, ws, out_dtype=torch.float32)
    again = ops.linear_fp8(x8.flip(0), xs.flip(0).contiguous(), w8, ws, out_dtype=torch.float32).flip(0)
    assert torch.equal(full, again)


def test_captured_chain(device):
    """quant -> gate_up with the gate, quantised -> down, captured and replayed on new rows."""
    H, F, T = 512, 640, 37
    g = torch.Generator().manual_seed(5)
    gu = [weights(g, F, H) for _ in range(2)]
    dn = weights(g, H, F)
    w8, ws = torch.cat([p[0] for p in gu]).to(device), torch.cat([p[1] for p in gu]).to(device)
    d8, ds = dn[0].to(device), dn[1].to(device)

    def chain(x):
        a8, a_s = ops.linear_fp8(*ops.quant_fp8(x), w8, ws, swiglu=True, quantized=True)
        return ops.linear_fp8(a8, a_s, d8, ds, out_dtype=torch.bfloat16)

    xs = [torch.randn(T, H, generator=g).to(torch.bfloat16).to(device) for _ in range(3)]
    static = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(static)
    for x in xs + xs:
        eager = chain(x)
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        # in float64: x quantised, the gated product quantised
        x8, s8 = quantise(x.cpu().double())
        xd = x8 * expand(s8, H, 1)
        gate, up = (xd @ p[2].t() for p in gu)
        a8, sa = quantise(gate * torch.sigmoid(gate) * up)
        y = (a8 * expand(sa, F, 1)) @ dn[2].t()
        # values at a border of the inner rounding move by a step: few, see check_quantised
        assert ((eager.cpu().double() - y).norm(dim=1) <= 2.0 ** -5 * y.norm(dim=1)).all()
        assert (eager.cpu().double() - y).norm() <= 2.0 ** -8 * y.norm()
