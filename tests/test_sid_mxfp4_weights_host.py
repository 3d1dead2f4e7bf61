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


def test_weights_are_taken_piece_by_piece():
    """Temporaries stay at 2^22 weights at a time, whatever the tensor, and give the definition's codes and scales."""
    from torch.utils._python_dispatch import TorchDispatchMode

    largest = 0

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            nonlocal largest
            out = func(*args, **(kwargs or {}))
            for t in out if isinstance(out, (list, tuple)) else (out,):
                if isinstance(t, torch.Tensor) and not t._is_view():
                    largest = max(largest, t.numel() * t.element_size())
            return out

    w = torch.randn(5, 1000, 2080, generator=torch.Generator().manual_seed(6)).bfloat16()
    with Watch():
        w4, scale = quantize_mxfp4(w)
    assert largest <= 8 * 2 ** 22
    codes, byte = quantise(w.double())
    assert torch.equal(scale, byte) and torch.equal(w4, pack(codes))
    w = w.transpose(1, 2)[:, :, :992]
    w4, scale = quantize_mxfp4(w)
    codes, byte = quantise(w.double())
    assert torch.equal(scale, byte) and torch.equal(w4, pack(codes))
    assert [t.shape for t in quantize_mxfp4(w[:0])] == [(0, 2080, 496), (0, 2080, 31)]
