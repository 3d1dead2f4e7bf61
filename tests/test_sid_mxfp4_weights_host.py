"""4-bit weights of a decoder, on the CPU: weights that are not finite, and what the making of them holds."""

import pytest
import torch

from tests.test_gpu_mxfp4 import pack, quantise
from vllm_gr_amd.v1.sid_decoder import quantize_mxfp4, quantize_weights


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_weights_that_are_not_finite_stay_visible(dtype):
    """A block with an infinity or a NaN has the scale byte 255, which reads back as NaN, and codes of 0, as
    gr_quant_mxfp4 leaves it; the others are what they are without it."""
    w = torch.randn(3, 40, 96, generator=torch.Generator().manual_seed(4)).to(dtype)
    codes, byte = quantise(w.double())
    bad = torch.zeros(byte.shape, dtype=torch.bool)
    for at, value in (((0, 0, 0), float("inf")), ((0, 7, 33), -float("inf")), ((1, 39, 95), float("nan")), ((2, 5, 64), float("nan"))):
        w[at] = value
        bad[at[0], at[1], at[2] // 32] = True
    w[2, 6, 32], w[2, 6, 40] = float("inf"), float("nan")
    bad[2, 6, 1] = True
    codes[bad.repeat_interleave(32, -1)], byte[bad] = 0, 255
    for w4, scale in (quantize_mxfp4(w), list(quantize_weights({"layers.0.expert_down": w}, "mxfp4").values())):
        assert torch.equal(scale, byte) and torch.equal(w4, pack(codes))
