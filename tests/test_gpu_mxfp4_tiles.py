"""gr_linear_mxfp4 and gr_expert_mlp_mxfp4 in every form that their sizes choose, against float64.

Each mode's forms (tiles, those that share a CU, the few rows' kernel) with rows and columns
left over, more stages than are on their way, and scales that come by 16 bytes, by words and
by single bytes (features in multiples of 512, of 128 and of 32).  Bounds as in test_gpu_mxfp4
and test_gpu_mxfp4_experts."""

import pytest
import torch

from tests.test_gpu_mxfp4 import BORDERS, HALF, NUMBERS, POWERS, gated, scale_bytes, unit
from tests.test_gpu_mxfp4_calls import random_rows
from tests.test_gpu_mxfp4_experts import check as check_experts
from tests.test_gpu_mxfp4_experts import make, reference
from vllm_gr_amd import _C, ops

pytestmark = pytest.mark.gpu

# mode: {gr_linear_mxfp4_tile: sizes (rows, columns, features) by the width of their scales}
TILES = {
    "plain": {
        16016: [(17, 15, 1536), (17, 15, 1152), (17, 15, 1056)],
        16032: [(17, 2135, 1536), (17, 2056, 1152), (17, 2179, 1056)],
        1064064: [(65, 1752, 1536), (67, 1696, 1152), (65, 1867, 1056)],
        1064128: [(65, 8432, 1536), (65, 8633, 1408), (65, 9118, 1376)],
        1128128: [(132, 10946, 1536), (130, 11126, 1152), (129, 11719, 1056)],
        1128256: [(321, 10919, 1536), (269, 13277, 1152), (258, 14348, 1056)],
        1256256: [(525, 14726, 1536), (578, 13674, 1152), (546, 14624, 1056)],
        2064064: [(402, 4632, 1536), (67, 8249, 1152), (65, 9005, 1056)],
        2064128: [(259, 11266, 1536), (261, 11186, 1152), (268, 11006, 1056)],
        2128128: [(729, 10801, 1536), (784, 9222, 1152), (782, 9258, 1056)],
    },
    "gated": {
        16032: [(17, 16, 1536), (17, 16, 1152), (17, 16, 1056)],
        16064: [(17, 2080, 1536), (17, 2176, 1152), (17, 2176, 1056)],
        1064064: [(65, 1648, 1536), (65, 1776, 1152), (66, 1648, 1056)],
        1064128: [(65, 4256, 1536), (65, 4320, 1408), (66, 4576, 1376)],
        1128128: [(132, 5536, 1536), (143, 5456, 1152), (129, 5584, 1056)],
        1128256: [(132, 11312, 1536), (129, 11424, 1152), (135, 11216, 1056)],
        1256256: [(263, 13344, 1536), (270, 13200, 1152), (257, 13920, 1056)],
        2064064: [(1257, 784, 1536), (66, 4176, 1152), (65, 4592, 1056)],
        2064128: [(132, 8208, 1536), (130, 8336, 1152), (130, 8976, 1056)],
        2128128: [(708, 5424, 1536), (805, 4656, 1152), (773, 4656, 1056)],
    },
    "plain_q": {
        16032: [(17, 32, 1536), (17, 32, 1152), (17, 32, 1056)],
        1064128: [(65, 1696, 1536), (65, 1824, 1408), (68, 1696, 1376)],
        1128128: [(129, 11040, 1536), (133, 11104, 1152), (135, 11712, 1056)],
        1128256: [(273, 13280, 1536), (261, 13888, 1152), (270, 13664, 1056)],
        1256256: [(542, 14528, 1536), (520, 14944, 1152), (608, 13248, 1056)],
        2064128: [(283, 11072, 1536), (66, 1696, 1152), (69, 1760, 1056)],
        2128128: [(1655, 4928, 1536), (734, 10816, 1152), (775, 9248, 1056)],
    },
    "gated_q": {
        16064: [(17, 32, 1536), (17, 32, 1152), (17, 32, 1056)],
        1064128: [(68, 1760, 1536), (66, 1696, 1408), (65, 1824, 1376)],
        1128128: [(132, 5536, 1536), (133, 5792, 1152), (135, 5472, 1056)],
        1128256: [(132, 11456, 1536), (131, 11168, 1152), (132, 11072, 1056)],
        1256256: [(273, 13216, 1536), (274, 13216, 1152), (259, 13248, 1056)],
        2064128: [(129, 8608, 1536), (65, 1888, 1152), (81, 1376, 1056)],
        2128128: [(1178, 3232, 1536), (774, 4640, 1408), (822, 4640, 1056)],
    },
}

# gr_expert_mlp_mxfp4_tile: sizes (tokens, experts, experts a token, hidden, features) by the width of both scales
EXPERT_TILES = {
    2032064: [(53, 48, 1, 1024, 1024), (7, 26, 4, 640, 1920), (15, 76, 7, 544, 544)],
    2032256: [(13, 56, 5, 2560, 1024), (12, 78, 7, 1920, 640), (95, 79, 2, 1376, 544)],
    3032064: [(40, 7, 3, 1024, 512), (33, 6, 2, 640, 384), (50, 9, 3, 544, 288)],
    3032256: [(11, 75, 7, 2048, 1024), (12, 71, 6, 2176, 640), (27, 66, 3, 2080, 544)],
    3064128: [(66, 9, 4, 1024, 1024), (47, 5, 3, 640, 1920), (485, 17, 1, 544, 544)],
    3128128: [(233, 15, 5, 1024, 1024), (137, 7, 4, 640, 2176), (514, 7, 1, 544, 2080)],
    2256256: [(1100, 8, 2, 512, 2048), (1100, 8, 2, 640, 1920), (1100, 8, 2, 544, 2080)],
}


def tile(mode, M, N, K):
    return _C.lib().gr_linear_mxfp4_tile(M, N, K, mode.startswith("gated"), _C.GR_DTYPE_MXFP4 if mode.endswith("q") else _C.GR_DTYPE_BF16)


def check_4bit(packed, byte, y, err):
    """As in test_gpu_mxfp4, on the device: a scale that a largest value within its error has, a nearest number."""
    top, off = y.abs().unflatten(-1, (-1, 32)), err.unflatten(-1, (-1, 32))
    lo, hi = (scale_bytes(t.amax(-1).cpu()).to(y.device) for t in ((top - off).clamp_min(0), top + off))
    assert ((byte >= lo) & (byte <= hi)).all()
    scale = POWERS.to(y.device)[byte.long()].repeat_interleave(32, -1)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    numbers = NUMBERS.to(y.device)
    got = numbers[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0) * scale
    a = (y / scale).abs()
    i = torch.bucketize(a, BORDERS.to(y.device))
    assert ((got - y).abs() <= (a - numbers[i]).abs() * scale + 2 * err).all()


def run(device, mode, M, N, K):
    g = torch.Generator(device=device).manual_seed(M + N + K)
    x4, xs, x = random_rows(g, M, K, device)
    swiglu = mode.startswith("gated")
    w4, ws, w = random_rows(g, 2 * N if swiglu else N, K, device)
    w, ws = w * 2.0 ** -6, ws - 6
    y, err = x @ w.t(), (x.abs() @ w.abs().t()) * unit(K)
    if swiglu:
        y, err = gated(y[:, :N], y[:, N:], err[:, :N], err[:, N:])
    if mode.endswith("q"):
        out = torch.full((M + 2, N // 2 + 16), 0xEE, dtype=torch.uint8, device=device)
        scale = torch.full((M + 2, N // 32 + 1), 0xEE, dtype=torch.uint8, device=device)
        ops.linear_mxfp4(x4, xs, w4, ws, swiglu=swiglu, quantized=True, out=out[:M, :N // 2], out_scale=scale[:M, :N // 32])
        check_4bit(out[:M, :N // 2], scale[:M, :N // 32], y, err)
        for rest in (out[M:], out[:, N // 2:], scale[M:], scale[:, N // 32:]):
            assert (rest == 0xEE).all()
        return
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        out = torch.full((M + 2, N + 8), -7.0, dtype=dtype, device=device)
        got = ops.linear_mxfp4(x4, xs, w4, ws, swiglu=swiglu, out_dtype=dtype, out=out[:M, :N])
        assert ((got.double() - y).abs() <= err + (y.abs() + err) * HALF[dtype] + 2.0 ** -25).all()
        assert (out[M:] == -7).all() and (out[:, N:] == -7).all()


@pytest.mark.parametrize("scales", [16, 4, 1])
@pytest.mark.parametrize("mode,form", [(m, t) for m, forms in TILES.items() for t in forms])
def test_linear_every_form(device, mode, form, scales):
    M, N, K = TILES[mode][form][(16, 4, 1).index(scales)]
    assert tile(mode, M, N, K) == form and (K % 512 == 0, K % 128 == 0) == (scales == 16, scales >= 4)
    run(device, mode, M, N, K)


def test_gated_product_of_whole_prompts(device):
    """The decoder's: 2048 features, 6144 of the layer, almost 8192 rows."""
    assert tile("gated_q", 8190, 6144, 2048) % 1000000 == 256256
    run(device, "gated_q", 8190, 6144, 2048)


@pytest.mark.parametrize("scales", [16, 4, 1])
@pytest.mark.parametrize("form", EXPERT_TILES)
def test_experts_every_form(device, form, scales):
    T, E, k, H, F = EXPERT_TILES[form][(16, 4, 1).index(scales)]
    assert _C.lib().gr_expert_mlp_mxfp4_tile(T, k, E, H, F) == form
    for size in (H, F):
        assert (size % 512 == 0, size % 128 == 0) == (scales == 16, scales >= 4)
    a, gu, dn, x, w, ids = make(T, E, k, H, F, torch.float16 if scales == 4 else torch.bfloat16, device)
    check_experts(ops.expert_mlp_mxfp4(*a), *reference(x, gu, dn, w, ids))
