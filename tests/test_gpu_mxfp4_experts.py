"""gr_expert_mlp_mxfp4 against float64.

The tokens' 4-bit form is exact.  A gated product is off by its float32 sums' bound
(as for gr_linear_mxfp4); its 4-bit form may then be any that values within that bound
have, which is carried through the down product.  Each expert's result is rounded to
fp16 multiples of a power of two (2^-11 of it, 2^-39 of the largest of its
neighbouring columns), summed in float32 and rounded to the output's type."""

import pytest
import torch

from tests.test_gpu_mxfp4 import BORDERS, HALF, NUMBERS, POWERS, gated, operand, quantise, scale_bytes, unit, values
from vllm_gr_amd import _C, ops

pytestmark = pytest.mark.gpu


def rounded(y, byte):
    """Nearest numbers (ties to even) times the given scales."""
    unit_ = POWERS[byte].repeat_interleave(32, -1)
    a = (y / unit_).abs()
    i = torch.bucketize(a, BORDERS)
    i += ((a == BORDERS[i.clamp_max(6)]) & (i < 7) & (i % 2 == 1)).long()
    return NUMBERS[i] * torch.sign(y) * unit_


def four_bits(y, err):
    """The 4-bit form's values, and how far that of values within err may be from them."""
    codes, byte = quantise(y)
    v = values(codes, byte)
    top, off = y.abs().unflatten(-1, (-1, 32)), err.unflatten(-1, (-1, 32))
    d = torch.zeros_like(v)
    for b in (scale_bytes((top - off).clamp_min(0).amax(-1)), scale_bytes((top + off).amax(-1))):
        for e in (-err, err):
            d = torch.maximum(d, (rounded(y + e, b) - v).abs())
    return v, d


def make(T, E, k, H, F, dtype, device, seed=0, away=0.0):
    g = torch.Generator().manual_seed(T + E + H + F + seed)
    x = (torch.randn(T, H, generator=g) * torch.exp(0.5 * torch.randn(1, H, generator=g))).to(dtype)
    gu4, gus, gu = operand(g, E * 2 * F, H, 0.2)
    dn4, dns, dn = operand(g, E * H, F, 0.2)
    gus, dns, gu, dn = gus - 4, dns - 4, gu * 2.0 ** -4, dn * 2.0 ** -4
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    ids[torch.rand(T, k, generator=g) < away] = -1
    w = torch.rand(T, k, generator=g)
    a = [x, gu4.view(E, 2 * F, -1), gus.view(E, 2 * F, -1), dn4.view(E, H, -1), dns.view(E, H, -1), w, ids]
    return [t.to(device) for t in a], gu.view(E, 2 * F, H), dn.view(E, H, F), x, w, ids


def reference(x, gu, dn, w, ids):
    v = values(*quantise(x.double()))
    E, F, H = gu.shape[0], gu.shape[1] // 2, gu.shape[2]
    out, err = torch.zeros_like(v), torch.zeros_like(v)
    for e in range(E):
        tok, j = torch.nonzero(ids == e, as_tuple=True)
        if not len(tok):
            continue
        s = v[tok] @ gu[e].t()
        d = v[tok].abs() @ gu[e].abs().t() * unit(H)
        act, da = four_bits(*gated(s[:, :F], s[:, F:], d[:, :F], d[:, F:]))
        y = act @ dn[e].t()
        dy = da @ dn[e].abs().t() + (act.abs() + da) @ dn[e].abs().t() * unit(F)
        dy = dy + (y.abs() + dy) * 2.0 ** -11 + (y.abs() + dy).amax(1, keepdim=True) * 2.0 ** -39 + 2.0 ** -112
        wt = w[tok, j].double()[:, None]
        out.index_add_(0, tok, wt * y)
        err.index_add_(0, tok, wt.abs() * (dy + y.abs() * (ids.shape[1] + 2) * 2.0 ** -24))
    return out, err


def check(got, y, err):
    half = HALF[got.dtype]
    assert ((got.cpu().double() - y).abs() <= err + (y.abs() + err) * half + 2.0 ** -25).all()


# tokens: one, a few rows an expert, tiles of every size, more choices than one workgroup sorts
CASES = [(1, 1, 1, 32, 32), (1, 8, 2, 256, 128), (3, 4, 4, 96, 160), (8, 64, 8, 2048, 768), (16, 20, 8, 544, 288),
         (5, 40, 25, 288, 96), (17, 100, 8, 256, 128), (40, 64, 2, 544, 288), (33, 5, 3, 416, 96),
         (100, 8, 2, 544, 288), (257, 6, 4, 512, 256), (640, 4, 2, 288, 352), (1500, 16, 8, 256, 64), (700, 2, 1, 1024, 512), (16, 60, 8, 2080, 800)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k,H,F", CASES)
def test_expert_mlp(device, dtype, T, E, k, H, F):
    a, gu, dn, x, w, ids = make(T, E, k, H, F, dtype, device)
    y, err = reference(x, gu, dn, w, ids)
    check(ops.expert_mlp_mxfp4(*a), y, err)


def test_absent_bad_and_repeated_experts(device):
    """Ids of another rank, ids past the end (flagged), a token without any expert, one expert twice, all tokens on one."""
    T, E, k, H, F = 70, 6, 3, 256, 128
    a, gu, dn, x, w, ids = make(T, E, k, H, F, torch.bfloat16, device, seed=5, away=0.4)
    ids[0] = -1
    ids[1] = torch.tensor([2, 2, 4], dtype=torch.int32)
    ids[2, 1] = E
    ids[3, 0] = 2 ** 31 - 1
    a[6] = ids.to(device)
    status = torch.zeros(1, dtype=torch.int32, device=device)
    y, err = reference(x, gu, dn, w, torch.where(ids >= E, -1, ids))
    got = ops.expert_mlp_mxfp4(*a, status=status)
    check(got, y, err)
    assert status.item() == _C.GR_DEV_BAD_EXPERT and (got[0] == 0).all()
    one = torch.full_like(ids, 3)
    a[6] = one.to(device)
    y, err = reference(x, gu, dn, w, one)
    check(ops.expert_mlp_mxfp4(*a), y, err)
    a[6] = torch.full_like(one, -1).to(device)
    assert (ops.expert_mlp_mxfp4(*a) == 0).all()


def test_few_tokens_absent_bad_and_repeated_experts(device):
    """The same for 16 tokens: more rows of one expert than a fragment holds among them."""
    T, E, k, H, F = 16, 5, 8, 288, 96
    a, gu, dn, x, w, ids = make(T, E + 3, k, H, F, torch.float16, device, seed=6, away=0.3)
    ids[0] = -1
    ids[1] = torch.tensor([2, 2, 4, 0, -1, E + 3, 2 ** 31 - 1, 1], dtype=torch.int32)
    for choices in (ids, torch.full_like(ids, 3), torch.full_like(ids, -7)):
        a[6] = choices.to(device)
        status = torch.zeros(1, dtype=torch.int32, device=device)
        y, err = reference(x, gu, dn, w, torch.where(choices >= E + 3, -1, choices))
        got = ops.expert_mlp_mxfp4(*a, status=status)
        check(got, y, err)
        assert status.item() == (_C.GR_DEV_BAD_EXPERT if choices is ids else 0)
    assert (got == 0).all()


@pytest.mark.parametrize("T", [9, 40])
def test_strided_tensors_and_workspace(device, T):
    E, k, H, F = 4, 2, 160, 96
    a, gu, dn, x, w, ids = make(T, E, k, H, F, torch.float16, device)
    y, err = reference(x, gu, dn, w, ids)
    wide = torch.zeros(T, H + 24, dtype=torch.float16, device=device)
    wide[:, 8:H + 8] = a[0]
    out = torch.full((T, H + 12), 9.0, dtype=torch.float16, device=device)
    need = ops.expert_mlp_mxfp4_workspace_bytes(T, k, E, H, F)
    for fill in (0, 255):  # no initial contents
        ws = torch.full((need,), fill, dtype=torch.uint8, device=device)
        got = ops.expert_mlp_mxfp4(wide[:, 8:H + 8], *a[1:], out=out[:, 4:H + 4], workspace=ws)
        check(got, y, err)
        assert (out[:, :4] == 9).all() and (out[:, H + 4:] == 9).all()
    with pytest.raises(RuntimeError):
        ops.expert_mlp_mxfp4(*a, workspace=ws[:need - 256])
    with pytest.raises(ValueError, match="contiguous"):
        ops.expert_mlp_mxfp4(*a, workspace=torch.zeros(2 * need, dtype=torch.uint8, device=device)[::2])
