"""The kernels that many tokens take, of which the other tests reach the ones for
fewer: eight router logits a lane with up to eight tokens a wave, and two rows at a
time in the quantiser, by itself and ahead of the experts.  The last tokens leave a
wave, a workgroup and a pair of rows part empty.  References and bounds as in the
modules of their other tests."""

import pytest
import torch

from tests.test_gpu_experts import check, make, route_ref
from tests.test_gpu_fp8_linear import E4M3, quantise
from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu

# just above 2^18 logits; groups that are whole lanes (8 slots each), and ones that are not
MANY = [(4373, 60, 6, 4, 2), (4099, 64, 8, 8, 3), (2623, 100, 9, 5, 2), (2051, 128, 16, 4, 2), (1313, 200, 5, 10, 4),
        (1027, 256, 8, 8, 4)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias,grouped", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("T,E,k,groups,top", MANY)
def test_route_of_many_tokens(device, T, E, k, groups, top, bias, grouped, score):
    """Ordinary rows, rows of nearly equal scores, masked ones and ones with NaN side by
    side in a wave, so that some of its tokens are ordered again and others are not."""
    g = torch.Generator().manual_seed(T + E)
    x = 2 * torch.randn(T, E, generator=g)
    kind = torch.randint(0, 8, (T,), generator=g)
    near = torch.randn(T, 1, generator=g).expand(T, E).clone()
    for _ in range(3):
        near = torch.where(torch.randint(0, 2, (T, E), generator=g).bool(), torch.nextafter(near, torch.tensor(9.0)), near)
    x = torch.where((kind < 3)[:, None], near, x)
    hit = torch.rand(T, E, generator=g)
    inf = float("inf")
    x = torch.where((kind == 3)[:, None] & (hit < 0.9), -inf, x)
    x = torch.where((kind == 4)[:, None] & (hit < 0.1), float("nan"), x)
    x[kind == 5, E // 2] = torch.finfo(torch.float32).min
    x[-1] = -inf
    b = (0.5 + 1e-7 * torch.randn(E, generator=g)) if bias else None
    n, t = (groups, top) if grouped else (1, 1)
    w, ids = ops.route_experts(x.to(device), k, score=score, bias=None if b is None else b.to(device), num_groups=n,
                               top_groups=t)
    w, ids = w.cpu().double(), ids.cpu()
    assert ((ids >= 0) & (ids < E)).all() and (ids.sort(1)[0].diff(dim=1) > 0).all()
    rows = torch.cat([torch.arange(24), torch.randperm(T, generator=g)[:40], torch.arange(T - 36, T)])
    rw, rids = route_ref(x[rows], k, score, b, n, t, True, 1.0)
    assert torch.equal(ids[rows], rids)
    w = w[rows]
    assert torch.equal(torch.isnan(w), torch.isnan(rw))
    ok = ~torch.isnan(rw)
    assert ((w[ok] - rw[ok]).abs() <= rw[ok].abs() * 2.0 ** -23 + 1e-40).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_route_of_many_tokens_in_16_bits(device, dtype):
    """Strided rows of 16-bit logits, not renormalised."""
    T, E, k = 4373, 60, 6
    g = torch.Generator().manual_seed(2)
    wide = (2 * torch.randn(T, E + 5, generator=g)).to(dtype)
    b = 0.1 * torch.randn(E, generator=g)
    w, ids = ops.route_experts(wide.to(device)[:, :E], k, score="softmax", bias=b.to(device), renormalize=False, scale=2.5)
    rows = torch.cat([torch.arange(40), torch.arange(T - 40, T)])
    rw, rids = route_ref(wide[rows, :E], k, "softmax", b, 1, 1, False, 2.5)
    assert torch.equal(ids.cpu()[rows], rids)
    assert ((w.cpu().double()[rows] - rw).abs() <= rw.abs() * 2.0 ** -23 + 1e-40).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,K", [(2731, 6144), (65537, 144)])
def test_quant_of_many_groups(device, T, K, dtype):
    """An odd number of rows and 2^17 groups: two rows a lane.  Strided in and out; the row
    behind the last keeps what it holds."""
    g = torch.Generator(device=device).manual_seed(T)
    size = torch.exp(2 * torch.randn(T, 1, generator=g, device=device))
    x = (torch.randn(T, K + 16, generator=g, device=device) * size).to(dtype)
    x[5] = 0
    x[T - 1, :128] = 0
    out = torch.full((T + 1, K + 32), 0x33, dtype=torch.uint8, device=device)
    scale = torch.full((T + 1, -(-K // 128)), 7.0, device=device)
    got, s = ops.quant_fp8(x[:, :K], out=out[:T, :K].view(E4M3), scale=scale[:T])
    part = T // 5 + 1  # which takes a row a lane
    for r in range(0, T, part):
        p8, ps = ops.quant_fp8(x[r:r + part, :K])
        assert torch.equal(got[r:r + part].view(torch.uint8), p8.view(torch.uint8)) and torch.equal(s[r:r + part], ps)
    assert (out[T] == 0x33).all() and (out[:, K:] == 0x33).all() and (scale[T] == 7).all()
    rows = torch.cat([torch.arange(0, T, T // 200), torch.arange(T - 5, T)])
    want, ws = quantise(x[rows.to(device), :K].cpu().double())
    assert torch.equal(s.cpu()[rows].double(), ws) and torch.equal(got.cpu()[rows].double(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,F", [(8193, 4, 2, 2048, 48), (65537, 3, 1, 144, 32)])
def test_experts_of_many_quantised_rows(device, T, E, k, H, F, dtype):
    """8-bit experts whose tokens are quantised two rows at a time, beside the sort."""
    x, args, wts, ids, xr, ref = make(T, E, k, H, F, dtype, True, T, device)
    got = ops.expert_mlp(x, weights=wts, ids=ids, **args)
    rows = torch.cat([torch.randperm(T, generator=torch.Generator().manual_seed(1))[:160], torch.arange(T - 40, T)])
    at = rows.to(device)
    check(got[at], xr[rows], ref, wts[at], ids[at], dtype, True)
