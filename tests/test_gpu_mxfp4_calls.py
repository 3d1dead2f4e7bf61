"""The 4-bit operators as programs call them: every tile, strided and misaligned tensors,
far rows, NaN in its place only, streams, captured graphs, a run of all of them, refusals.

Bounds as in test_gpu_mxfp4 (sums) and test_gpu_mxfp4_experts (the 4-bit form of inexact
values); references in float64, on the device where they are large."""

import pytest
import torch

from tests.test_gpu_mxfp4 import HALF, NUMBERS, POWERS, check, check_4bit, gated, operand, operands, quantise, unit, values
from tests.test_gpu_mxfp4_experts import four_bits, make, reference
from tests.test_gpu_mxfp4_experts import check as check_experts
from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu


def random_rows(g, rows, K, device):
    """Random codes and scale bytes of 2^-3 to 2^0, and their float64 values."""
    x4 = torch.randint(0, 256, (rows, K // 2), generator=g, device=device, dtype=torch.uint8)
    s = torch.randint(124, 128, (rows, K // 32), generator=g, device=device, dtype=torch.uint8)
    codes = torch.stack([x4 & 15, x4 >> 4], -1).flatten(-2)
    v = NUMBERS.to(device)[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    return x4, s, v * POWERS.to(device)[s.long()].repeat_interleave(32, -1)


# from a few rows over tiles of 64 x 64 to 256 x 256, rows
# and columns left over
@pytest.mark.parametrize("M,N,K", [(8, 8192, 6144), (20, 4000, 160), (64, 4096, 2048), (200, 2000, 96), (511, 8184, 2048),
                                   (1001, 2048, 6144), (512, 12280, 2048), (2047, 12300, 288), (8190, 12280, 512),
                                   (4090, 8190, 1056), (500, 2040, 6144), (250, 2000, 1056), (700, 2300, 2080),
                                   (300, 4128, 2304)])
def test_large_tiles(device, M, N, K):
    g = torch.Generator(device=device).manual_seed(M + N + K)
    x4, xs, x = random_rows(g, M, K, device)
    w4, ws, w = random_rows(g, N, K, device)
    y, err = x @ w.t(), (x.abs() @ w.abs().t()) * unit(K)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((M + 3, N), -7.0, dtype=dtype, device=device)
        got = ops.linear_mxfp4(x4, xs, w4, ws, out_dtype=dtype, out=out[:M])
        assert ((got.double() - y).abs() <= err + (y.abs() + err) * HALF[dtype]).all()
        assert (out[M:] == -7).all()


@pytest.mark.parametrize("M,N,K", [(20, 2016, 160), (200, 1024, 96), (511, 4096, 544), (520, 6144, 2048), (4100, 6112, 96),
                                   (4100, 2080, 1056), (500, 1024, 2336), (300, 2048, 2304), (4100, 6144, 1056)])
def test_large_gated_tiles(device, M, N, K):
    g = torch.Generator(device=device).manual_seed(M + N + K)
    x4, xs, x = random_rows(g, M, K, device)
    w4, ws, w = random_rows(g, 2 * N, K, device)
    w, ws = w * 2.0 ** -6, ws - 6
    y, err = x @ w.t(), (x.abs() @ w.abs().t()) * unit(K)
    y, err = gated(y[:, :N], y[:, N:], err[:, :N], err[:, N:])
    got = ops.linear_mxfp4(x4, xs, w4, ws, swiglu=True, out_dtype=torch.float32)
    assert ((got.double() - y).abs() <= err + (y.abs() + err) * 2.0 ** -24).all()
    out = torch.full((M + 2, N // 2), 0xEE, dtype=torch.uint8, device=device)
    scale = torch.full((M + 2, N // 32), 0xEE, dtype=torch.uint8, device=device)
    ops.linear_mxfp4(x4, xs, w4, ws, swiglu=True, quantized=True, out=out[:M], out_scale=scale[:M])
    check_4bit(out[:M], scale[:M], y.cpu(), err.cpu())
    assert (out[M:] == 0xEE).all() and (scale[M:] == 0xEE).all()


@pytest.mark.parametrize("M,N,K", [(5, 200, 256), (70, 208, 512), (300, 4112, 1024), (9, 48, 288)])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_strides_alignments_and_types(device, M, N, K, shift):
    """Rows apart, scale rows at any byte, results at any 8 bytes; the same bits as from tensors of whole rows."""
    (x4, xs, w4, ws), y, err = operands(M, N, K, False, device)
    want = ops.linear_mxfp4(x4, xs, w4, ws)

    def apart(t, extra, at):
        wide = torch.full((t.shape[0], t.shape[1] + extra), 255, dtype=torch.uint8, device=device)
        wide[:, at:at + t.shape[1]] = t
        return wide[:, at:at + t.shape[1]]

    fp4, e8 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
    a = [apart(x4, 48, 16).view(fp4), apart(xs, 3 + shift, shift).view(e8), apart(w4, 16, 0).view(fp4), apart(ws, 4, shift).view(e8)]
    out = torch.full((M, N + 13), 5.0, dtype=torch.bfloat16, device=device)
    got = ops.linear_mxfp4(*a, out=out[:, 4:N + 4])
    check(got, y, err)
    assert torch.equal(got, want) and (out[:, :4] == 5).all() and (out[:, N + 4:] == 5).all()
    out = torch.full((M, N + 9), 5.0, dtype=torch.float32, device=device)
    check(ops.linear_mxfp4(*a, out=out[:, 4:N + 4], out_dtype=torch.float32), y, err)
    assert (out[:, :4] == 5).all() and (out[:, N + 4:] == 5).all()
    n = N // 32 * 32
    o4 = torch.full((M, n // 2 + 32), 0xEE, dtype=torch.uint8, device=device)
    os = torch.full((M, n // 32 + 3), 0xEE, dtype=torch.uint8, device=device)
    into = o4[:, 16:16 + n // 2], os[:, 1:1 + n // 32]
    ops.linear_mxfp4(a[0], a[1], a[2][:n], a[3][:n], quantized=True, out=into[0], out_scale=into[1])
    check_4bit(*into, y[:, :n], err[:, :n])
    for rest in (os[:, :1], os[:, 1 + n // 32:], o4[:, :16], o4[:, 16 + n // 2:]):
        assert (rest == 0xEE).all()


@pytest.mark.parametrize("M,N,K", [(7, 64, 288), (130, 512, 256), (600, 4128, 320)])
def test_not_a_number_stays_in_its_row_and_column(device, M, N, K):
    """A scale byte of 255 makes its row (its column) NaN, whatever the codes, and nothing else."""
    (x4, xs, w4, ws), y, err = operands(M, N, K, False, device)
    want = ops.linear_mxfp4(x4, xs, w4, ws, out_dtype=torch.float32)
    xs, ws, x4 = xs.clone(), ws.clone(), x4.clone()
    xs[M // 2, -1] = 255
    x4[M // 2] = 0
    ws[N - 3, 0] = 255
    got = ops.linear_mxfp4(x4, xs, w4, ws, out_dtype=torch.float32)
    assert got[M // 2].isnan().all() and got[:, N - 3].isnan().all()
    got[M // 2], got[:, N - 3] = want[M // 2], want[:, N - 3]
    assert torch.equal(got, want)
    o4, os = ops.linear_mxfp4(x4, xs, w4, ws, quantized=True)
    bad = torch.zeros(M, N // 32, dtype=torch.bool, device=device)
    bad[M // 2] = True
    bad[:, (N - 3) // 32] = True
    assert torch.equal(os == 255, bad)


def test_zeros_of_every_scale(device):
    """Zeros times the largest and the least scale are zeros; so are empty rows of x."""
    for M in (3, 200):
        x4, w4 = (torch.zeros(n, 128, dtype=torch.uint8, device=device) for n in (M, 256))
        for sx, sw in ((254, 254), (0, 0), (254, 0)):
            xs, ws = (torch.full((n, 8), s, dtype=torch.uint8, device=device) for n, s in ((M, sx), (256, sw)))
            assert (ops.linear_mxfp4(x4, xs, w4, ws, out_dtype=torch.float32) == 0).all()
            o4, os = ops.linear_mxfp4(x4, xs, w4, ws, quantized=True)
            assert (o4 & 0x77 == 0).all() and (os == 0).all()
    none = ops.linear_mxfp4(x4[:0], xs[:0], w4, ws)
    assert none.shape == (0, 256)
    a, *_ = make(4, 3, 2, 64, 32, torch.bfloat16, device)
    assert ops.expert_mlp_mxfp4(a[0][:0], *a[1:5], a[5][:0], a[6][:0]).shape == (0, 64)
    o4, s = ops.quant_mxfp4(torch.zeros(0, 64, device=device))
    assert o4.shape == (0, 32) and s.shape == (0, 2) and ops.dequant_mxfp4(o4, s).shape == (0, 64)


@pytest.mark.parametrize("T", [6, 60, 400])
def test_experts_not_a_number_stays_with_its_tokens(device, T):
    E, k, H, F = 5, 2, 288, 96
    a, gu, dn, x, w, ids = make(T, E, k, H, F, torch.bfloat16, device)
    want = ops.expert_mlp_mxfp4(*a)
    y, err = reference(x, gu, dn, w, ids)
    check_experts(want, y, err)
    b = [t.clone() for t in a]
    b[0][1, 3] = float("nan")
    b[0][2, 40] = float("inf")
    b[0][3] = 3e38  # gated products past float32
    got = ops.expert_mlp_mxfp4(*b)
    assert got[1:4].isnan().all()
    got[1:4] = want[1:4]
    assert torch.equal(got, want)
    b = [t.clone() for t in a]
    b[4][2, 7, 1] = 255  # a scale of expert 2's row 7 of the down product
    got = ops.expert_mlp_mxfp4(*b)
    hit = (ids == 2).any(1).to(device)
    assert got[hit][:, 7].isnan().all() and torch.equal(got[~hit], want[~hit])
    beside = [c for c in range(H) if c != 7]
    check_experts(got[:, beside], y[:, beside], err[:, beside])


def test_rows_far_apart(device):
    """Operands and results whose rows pass 32 bits of bytes and of elements."""
    M, N, K, far = 1100, 96, 256, 1 << 22
    (x4, xs, w4, ws), y, err = operands(M, N, K, False, device)
    want = ops.linear_mxfp4(x4, xs, w4, ws)
    room = torch.empty(M * far, dtype=torch.uint8, device=device)  # 4.6 GB
    xf, sf = room.as_strided((M, K // 2), (far, 1)), room.as_strided((M, K // 32), (far, 1), 1024)
    xf.copy_(x4)
    sf.copy_(xs)
    out = torch.empty(M * far, dtype=torch.bfloat16, device=device).as_strided((M, N), (far, 1))
    got = ops.linear_mxfp4(xf, sf, w4, ws, out=out)
    assert torch.equal(got, want)
    back = ops.dequant_mxfp4(xf, sf, dtype=torch.bfloat16, out=out.as_strided((M, K), (far, 1)))
    assert torch.equal(back, ops.dequant_mxfp4(x4, xs))
    again, scale = ops.quant_mxfp4(back, out=room.as_strided((M, K // 2), (far, 1), 4096), scale=room.as_strided((M, K // 32), (far, 1), 8192))
    assert torch.equal(ops.dequant_mxfp4(again, scale), ops.dequant_mxfp4(x4, xs))
    wf, wsf = room[:N * far].as_strided((N, K // 2), (far, 1)), room.as_strided((N, K // 32), (far, 1), 1024)
    wf.copy_(w4)
    wsf.copy_(ws)
    assert torch.equal(ops.linear_mxfp4(x4, xs, wf, wsf), want)


@pytest.mark.parametrize("T", [3, 100])
def test_experts_past_32_bits(device, T):
    """Weights of more than 2^32 bytes, of which the first and the last expert are used."""
    E, H, F, k = 130, 4096, 8192, 2
    g = torch.Generator().manual_seed(T)
    gu4 = torch.empty(E, 2 * F, H // 2, dtype=torch.uint8, device=device)
    gus = torch.empty(E, 2 * F, H // 32, dtype=torch.uint8, device=device)
    dn4 = torch.empty(E, H, F // 2, dtype=torch.uint8, device=device)
    dns = torch.empty(E, H, F // 32, dtype=torch.uint8, device=device)
    assert gu4.numel() > 2 ** 32
    gd = torch.Generator(device=device).manual_seed(T)
    gu, dn = {}, {}
    for e in (0, E - 1):
        gu4[e], gus[e], gu[e] = random_rows(gd, 2 * F, H, device)
        dn4[e], dns[e], dn[e] = random_rows(gd, H, F, device)
        gus[e] -= 6
        dns[e] -= 6
        gu[e], dn[e] = gu[e] * 2.0 ** -6, dn[e] * 2.0 ** -6
    x = torch.randn(T, H, generator=g).bfloat16()
    ids = torch.tensor([[E - 1, 0]] * T, dtype=torch.int32)
    w = torch.rand(T, k, generator=g)
    got = ops.expert_mlp_mxfp4(x.to(device), gu4, gus, dn4, dns, w.to(device), ids.to(device))
    # gated products are inexact before they go to 4 bits: a share of them may be the next
    # number over, which is carried through the down product
    v = values(*quantise(x.double())).to(device)
    y = torch.zeros(T, H, dtype=torch.float64, device=device)
    err = torch.zeros_like(y)
    for j, e in enumerate((E - 1, 0)):
        s, d = v @ gu[e].t(), v.abs() @ gu[e].abs().t() * unit(H)
        act, da = four_bits(*(t.cpu() for t in gated(s[:, :F], s[:, F:], d[:, :F], d[:, F:])))
        act, da = act.to(device), da.to(device)
        r = act @ dn[e].t()
        dr = da @ dn[e].abs().t() + (act.abs() + da) @ dn[e].abs().t() * unit(F)
        dr = dr + (r.abs() + dr) * 2.0 ** -11 + (r.abs() + dr).amax(1, keepdim=True) * 2.0 ** -39
        wt = w[:, j].double().to(device)[:, None]
        y += wt * r
        err += wt * (dr + r.abs() * (k + 2) * 2.0 ** -24)
    check_experts(got, y.cpu(), err.cpu())


def layer(x, w1, w2, router, e):
    """A decoder's feed-forward part: a dense layer and the experts', and what each step gives."""
    x4, xs = ops.quant_mxfp4(x)
    a4, as_ = ops.linear_mxfp4(x4, xs, *w1, swiglu=True, quantized=True)
    dense = ops.linear_mxfp4(a4, as_, *w2, out_dtype=x.dtype)
    weights, ids = ops.route_experts(ops.linear(x, router), 4)
    return dense, ops.expert_mlp_mxfp4(x, *e, weights, ids), ops.dequant_mxfp4(a4, as_)


def parts(device, H=512, F=160, E=16, seed=3):
    g = torch.Generator().manual_seed(seed)
    (w1, s1, v1), (w2, s2, v2) = operand(g, 2 * F, H, 0.2), operand(g, H, F, 0.2)
    gu4, gus, _ = operand(g, E * 2 * F, H, 0.2)
    dn4, dns, _ = operand(g, E * H, F, 0.2)
    to = lambda *t: [a.to(device) for a in t]
    return (to(w1, s1 - 4), to(w2, s2 - 4), (torch.randn(E, H, generator=g) * 0.1).bfloat16().to(device),
            to(gu4.view(E, 2 * F, -1), (gus - 4).view(E, 2 * F, -1), dn4.view(E, H, -1), (dns - 4).view(E, H, -1))), v1 * 2.0 ** -4, v2 * 2.0 ** -4


@pytest.mark.parametrize("T", [1, 37, 300])
def test_run_of_all(device, T):
    p, v1, v2 = parts(device)
    H, F = v1.shape[1], v2.shape[1]
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).bfloat16()
    dense, experts, act = layer(x.to(device), *p)
    v = values(*quantise(x.double()))
    s, d = v @ v1.t(), v.abs() @ v1.abs().t() * unit(H)
    want, off = four_bits(*gated(s[:, :F], s[:, F:], d[:, :F], d[:, F:]))
    assert ((act.cpu().double() - want).abs() <= off + (want.abs() + off) * 2.0 ** -8).all()
    y = want @ v2.t()
    check(dense, y, off @ v2.abs().t() + (want.abs() + off) @ v2.abs().t() * unit(F))
    weights, ids = ops.route_experts(ops.linear(x.to(device), p[2]), 4)
    gu, dn = (ops.dequant_mxfp4(c.flatten(0, 1), s_.flatten(0, 1), dtype=torch.float32).cpu().double().view(c.shape[0], c.shape[1], -1)
              for c, s_ in ((p[3][0], p[3][1]), (p[3][2], p[3][3])))
    check_experts(experts, *reference(x, gu, dn, weights.cpu(), ids.cpu()))


def test_streams_and_calls_at_once(device):
    """Calls on two streams at a time, tensors of a third, give what each gives alone, each time."""
    p, _, _ = parts(device)
    xs = [torch.randn(n, 512, generator=torch.Generator().manual_seed(n)).bfloat16().to(device) for n in (300, 290)]
    want = [layer(x, *p) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer(xs[i], *p))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_captured_graphs(device):
    """Two graphs with a workspace between them, replayed in turn with eager work between and new inputs."""
    p, _, _ = parts(device)
    E, F, H = p[3][0].shape[0], p[3][0].shape[1] // 2, 512
    sizes = (40, 9)
    ws = torch.empty(max(ops.expert_mlp_mxfp4_workspace_bytes(n, 3, E, H, F) for n in sizes), dtype=torch.uint8, device=device)
    xs = [torch.zeros(n, H, dtype=torch.bfloat16, device=device) for n in sizes]
    w = [torch.rand(n, 3, generator=torch.Generator().manual_seed(n)).to(device) for n in sizes]
    ids = [torch.randint(-1, E, (n, 3), generator=torch.Generator().manual_seed(n)).int().to(device) for n in sizes]

    def run(i, workspace=None):
        x4, s = ops.quant_mxfp4(xs[i])
        a4, as_ = ops.linear_mxfp4(x4, s, *p[0], swiglu=True, quantized=True)
        return (ops.linear_mxfp4(a4, as_, *p[1]), ops.dequant_mxfp4(a4, as_),
                ops.expert_mlp_mxfp4(xs[i], *p[3], w[i], ids[i], workspace=workspace))

    graphs, results = [], []
    for i in range(2):
        run(i, ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(run(i, ws))
        graphs.append(g)
    for step in range(4):
        for i in range(2):
            xs[i].copy_(torch.randn(xs[i].shape, generator=torch.Generator().manual_seed(step)))
            want = run(i)
            graphs[i].replay()
            for a, b in zip(results[i], want):
                assert torch.equal(a, b), (step, i)
            torch.cuda.synchronize()


def test_same_bits_each_time(device):
    a, *_ = make(700, 6, 2, 544, 288, torch.bfloat16, device)
    first = ops.expert_mlp_mxfp4(*a)
    ops_, _, _ = operands(700, 1000, 2048, False, device)
    one = ops.linear_mxfp4(*ops_)
    for _ in range(5):
        assert torch.equal(ops.expert_mlp_mxfp4(*a), first) and torch.equal(ops.linear_mxfp4(*ops_), one)


def test_refusals(device):
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=device)
    x4, s = ops.quant_mxfp4(x)
    w4, ws = ops.quant_mxfp4(torch.zeros(64, 256, device=device))
    E = torch.zeros(2, 64, 128, dtype=torch.uint8, device=device), torch.zeros(2, 64, 8, dtype=torch.uint8, device=device)
    D = torch.zeros(2, 256, 16, dtype=torch.uint8, device=device), torch.zeros(2, 256, 1, dtype=torch.uint8, device=device)
    w, ids = torch.zeros(4, 2, device=device), torch.zeros(4, 2, dtype=torch.int32, device=device)
    assert (ops.expert_mlp_mxfp4(x, *E, *D, w, ids) == 0).all()
    wide = torch.zeros(4, 512, dtype=torch.bfloat16, device=device)
    for f in (lambda: ops.quant_mxfp4(x[:, :250]), lambda: ops.quant_mxfp4(wide[:, ::2]), lambda: ops.quant_mxfp4(x.double()),
              lambda: ops.quant_mxfp4(x[0]), lambda: ops.quant_mxfp4(x, out=x4[:3]), lambda: ops.quant_mxfp4(x, scale=s[:, :7]),
              lambda: ops.quant_mxfp4(x, out=x4.int()), lambda: ops.quant_mxfp4(x, scale=s.cpu()),
              lambda: ops.dequant_mxfp4(x4, s[:, :7]), lambda: ops.dequant_mxfp4(x4[:, :120], s), lambda: ops.dequant_mxfp4(x4, s.int()),
              lambda: ops.dequant_mxfp4(x4, s, dtype=torch.float64), lambda: ops.dequant_mxfp4(x4, s, out=x[:, :128]),
              lambda: ops.dequant_mxfp4(x4, s, dtype=torch.float16, out=x), lambda: ops.dequant_mxfp4(x4.t(), s),
              lambda: ops.linear_mxfp4(x4, s, w4[:, :64], ws[:, :4]), lambda: ops.linear_mxfp4(x4, s, w4[:63], ws[:63], swiglu=True),
              lambda: ops.linear_mxfp4(x4, s, w4[:48], ws[:48], quantized=True), lambda: ops.linear_mxfp4(x4, s, w4, ws[:63]),
              lambda: ops.linear_mxfp4(x4, s, w4, ws, out_scale=s), lambda: ops.linear_mxfp4(x4, s, w4, ws, out=x),
              lambda: ops.linear_mxfp4(x4, s, w4, ws, out_dtype=torch.int8), lambda: ops.linear_mxfp4(x4, s, w4.cpu(), ws),
              lambda: ops.expert_mlp_mxfp4(x, E[0], E[1][:, :, :7], *D, w, ids),
              lambda: ops.expert_mlp_mxfp4(x, *E, D[0][:1], D[1][:1], w, ids),
              lambda: ops.expert_mlp_mxfp4(x.float(), *E, *D, w, ids), lambda: ops.expert_mlp_mxfp4(x, *E, *D, w, ids.long()),
              lambda: ops.expert_mlp_mxfp4(x, *E, *D, w[:, :1], ids), lambda: ops.expert_mlp_mxfp4(x, *E, *D, w.half(), ids),
              lambda: ops.expert_mlp_mxfp4(x[:, :224], *E, *D, w, ids),
              lambda: ops.expert_mlp_mxfp4(x, E[0].transpose(0, 1).contiguous().transpose(0, 1), E[1], *D, w, ids),
              lambda: ops.expert_mlp_mxfp4(x, *E, *D, w, ids, out=x[:3])):
        with pytest.raises((ValueError, NotImplementedError)):
            f()
    odd = torch.zeros(4, 300, dtype=torch.uint8, device=device)
    for f in (lambda: ops.quant_mxfp4(wide[:, 4:260]), lambda: ops.quant_mxfp4(x, out=odd[:, :128]),
              lambda: ops.dequant_mxfp4(odd[:, 1:129], s), lambda: ops.linear_mxfp4(odd[:, 8:136], s, w4, ws),
              lambda: ops.linear_mxfp4(x4, s, w4[:40], ws[:40], swiglu=True),
              lambda: ops.linear_mxfp4(x4, s, w4, ws, out=wide[:, 1:65]),
              lambda: ops.expert_mlp_mxfp4(wide[:, 4:260], *E, *D, w, ids),
              lambda: ops.expert_mlp_mxfp4(x, *E, *D, w, ids, workspace=w)):
        with pytest.raises(RuntimeError):
            f()
