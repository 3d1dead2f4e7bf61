"""The 8-bit products, the experts and the router at the sizes that reach each of their
tiles and variants, and on several streams.  Bounds as in the modules of their other
tests, from which the float64 references come."""

import pytest
import torch

from tests.test_gpu_experts import HALF, check, make, route_ref
from tests.test_gpu_fp8_linear import check_16, check_quantised, operands
from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu

# Tiles of rows x weight rows by (16-bit results, float32's), with rows, columns and depth that end inside one.
LINEAR = [(1000, 1100, 272, False),  # 64 x 64, 64 x 128
          (700, 2100, 1040, False),  # 64 x 128 both
          (513, 12300, 272, False),  # 128 x 128, 128 x 256
          (2049, 2050, 1040, False),  # 128 x 256 both
          (2500, 4500, 272, False),  # 256 x 256, 128 x 128
          (700, 2112, 1040, True),  # 128 x 128 both
          (1300, 2704, 1040, True),  # 128 x 256 both
          (1500, 4112, 528, True)]  # 256 x 256, 128 x 256


@pytest.mark.parametrize("M,N,K,swiglu", LINEAR)
def test_linear_tiles(device, M, N, K, swiglu):
    (x8, xs, w8, ws), y, err, mag = operands(M, N, K, swiglu, device)
    y32 = ops.linear_fp8(x8, xs, w8, ws, swiglu=swiglu, out_dtype=torch.float32)
    assert ((y32.cpu().double() - y).abs() <= err).all()
    for dtype in (torch.bfloat16, torch.float16):
        check_16(ops.linear_fp8(x8, xs, w8, ws, swiglu=swiglu, out_dtype=dtype), y, mag, err)


@pytest.mark.parametrize("M,N,K,swiglu", [(1100, 2064, 272, True), (900, 1040, 400, False)])
def test_linear_quantised_tiles(device, M, N, K, swiglu):
    """More groups than the smaller tile is taken for; and the plain product's."""
    (x8, xs, w8, ws), y, err, _ = operands(M, N, K, swiglu, device)
    check_quantised(*ops.linear_fp8(x8, xs, w8, ws, swiglu=swiglu, quantized=True), y, err)


# rows per expert of 8 and fewer, some dozens, hundreds and more (16-bit weights: tiles of 16 to 256 rows; 8-bit: 32, 128)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,F", [(8, 16, 4, 144, 272), (200, 3, 1, 400, 80), (601, 3, 2, 272, 208),
                                       (700, 1, 1, 272, 144), (1050, 3, 2, 144, 272)])
def test_expert_tiles(device, T, E, k, H, F, dtype, fp8):
    x, args, wts, ids, xr, ref = make(T, E, k, H, F, dtype, fp8, T + F, device)
    check(ops.expert_mlp(x, weights=wts, ids=ids, **args), xr, ref, wts, ids, dtype, fp8)


@pytest.mark.parametrize("E,k,groups,top", [(1024, 64, 1, 1), (640, 64, 5, 2), (512, 64, 64, 8), (100, 60, 2, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [3, 600])
def test_route_most_choices_near_ties(device, T, E, k, groups, top, score):
    """All the choices there may be, of scores that float32 cannot tell apart."""
    k = min(k, E // groups * top)
    g = torch.Generator().manual_seed(E + T)
    x = torch.randn(T, 1, generator=g).expand(T, E).clone()
    for _ in range(2):
        x = torch.where(torch.randint(0, 2, (T, E), generator=g).bool(), torch.nextafter(x, torch.tensor(9.0)), x)
    b = (0.5 + 1e-7 * torch.randn(E, generator=g)) if groups > 1 else None
    w, ids = ops.route_experts(x.to(device), k, score=score, bias=None if b is None else b.to(device),
                               num_groups=groups, top_groups=top)
    few = slice(0, 40)  # rows of 600 tokens share a wave: the first ones show it
    rw, rids = route_ref(x[few], k, score, b, groups, top, True, 1.0)
    assert torch.equal(ids[few].cpu(), rids)
    # the sum that they are divided by is of k rounded scores
    assert ((w[few].cpu().double() - rw).abs() <= rw * 2.0 ** -22).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_two_streams_at_once(device, fp8):
    """Layers of two streams overlap, each with inputs that its own stream makes just before."""
    T, E, k, H, F = 400, 8, 2, 512, 256
    x, args, _, _, _, _ = make(T, E, k, H, F, torch.bfloat16, fp8, 1, device)
    router = torch.randn(H, E, generator=torch.Generator().manual_seed(2)).to(device)

    def layer(x):
        w, ids = ops.route_experts(x.float() @ router, k)
        y = ops.expert_mlp(x, weights=w, ids=ids, **args)
        return ops.quant_fp8(y)

    inputs = [x, x.flip(0).contiguous()]
    want = [layer(v) for v in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                late = torch.zeros_like(inputs[i])
                late += inputs[i]
                got[i].append(layer(late))
    torch.cuda.synchronize()
    for i in range(2):
        for y8, ys in got[i]:
            assert torch.equal(y8.view(torch.uint8), want[i][0].view(torch.uint8)) and torch.equal(ys, want[i][1])


def test_two_graphs_of_one_layer(device):
    """Two captured batches of one layer, replayed in turn: neither's workspace is the other's."""
    E, k, H, F = 6, 2, 256, 128
    _, args, _, _, _, _ = make(4, E, k, H, F, torch.bfloat16, True, 3, device)
    g = torch.Generator().manual_seed(7)
    runs = []
    for T in (5, 300):
        x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(device)
        w = torch.rand(T, k, generator=g).to(device)
        ids = torch.randint(-1, E, (T, k), generator=g).to(torch.int32).to(device)  # an expert twice, or none
        want = ops.expert_mlp(x, weights=w, ids=ids, **args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.expert_mlp(x, weights=w, ids=ids, **args)
        runs.append((graph, out, want, (x, w, ids)))  # a graph reads its inputs where they were
    for _ in range(4):
        for graph, out, _, _ in runs:
            out.fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in runs:
            assert torch.equal(out, want)


@pytest.mark.parametrize("M", [1, 300, 2000])
def test_gate_far_below_zero(device, M):
    """A gate whose sigmoid is below the normal float32 numbers still counts beside a huge
    factor: the exponential of g is off by |g| log2(e) 2^-24 and half a unit of the
    product g log2(e), 2^-18 of a value near 128."""
    N, K = 256, 128
    gates = [-88.0, -80.0, -72.0, -1.0, 0.0, 80.0]
    x = torch.zeros(M, K)
    x[:, 0] = 1
    w = torch.zeros(2 * N, K)
    w[:N, 0] = torch.tensor(gates).repeat(N // len(gates) + 1)[:N]
    w[N:, 0] = 448
    ws = torch.ones(4, 1)
    ws[2:] = 2.0 ** 90
    to8 = lambda t: t.to(torch.float8_e4m3fn).to(device)
    got = ops.linear_fp8(to8(x), torch.ones(M, 1, device=device), to8(w), ws.to(device), swiglu=True,
                         out_dtype=torch.float32).cpu().double()
    g = w[:N, 0].double()
    want = g * torch.sigmoid(g) * 448 * 2.0 ** 90
    assert (want[g == -88].abs() > 1e-8).all()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -16).all()
