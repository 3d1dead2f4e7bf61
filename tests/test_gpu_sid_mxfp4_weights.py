"""4-bit weights of a decoder are made on the device by gr_quant_mxfp4, without temporaries of the weights' size."""

import pytest
import torch

from tests.test_gpu_mxfp4 import pack, quantise
from tests.test_gpu_sid_experts import BF16, EXPERTS
from tests.test_sid_mxfp4_types_host import typed
from vllm_gr_amd.v1.sid_decoder import SidDecoder, init_weights, quantize_mxfp4, quantize_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_memory(device, dtype):
    w = torch.randn(16, 1024, 1024, generator=torch.Generator(device=device).manual_seed(1), device=device).to(dtype)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    w4, scale = quantize_mxfp4(w)
    assert torch.cuda.max_memory_allocated() - before <= w4.numel() + scale.numel() + 2 ** 20
    for e in (0, 15):
        codes, byte = quantise(w[e].cpu().double())
        assert torch.equal(scale[e].cpu(), byte) and torch.equal(w4[e].cpu(), pack(codes))


def test_layouts(device):
    """Weights that the kernel's loads do not fit (not aligned, columns apart, float64), and none."""
    wide = torch.randn(2, 70, 417, generator=torch.Generator().manual_seed(2))
    for dtype in (torch.float32, torch.bfloat16, torch.float64):
        w = wide.to(dtype).to(device)
        flat = w.flatten()[3:3 + 2 * 70 * 416].view(2, 70, 416)
        for v in (w[:, :, 1:], flat, flat[0], w[:, :64].transpose(1, 2), w[0, :64].t(), flat[:, ::2], flat[0, :1].expand(5, 416)):
            codes, byte = quantise(v.cpu().double())
            w4, scale = quantize_mxfp4(v)
            assert torch.equal(scale.cpu(), byte) and torch.equal(w4.cpu(), pack(codes))
            assert w4.is_contiguous() and scale.is_contiguous()
    assert [t.shape for t in quantize_mxfp4(flat[:0])] == [(0, 70, 208), (0, 70, 13)]


@pytest.mark.parametrize("cfg", [BF16, EXPERTS], ids=["dense", "experts"])
def test_types_of_codes_and_scales(device, cfg):
    """A layer gives the same bits with torch's own types of 4-bit codes and scales as with uint8."""
    w = {k: v.to(device) for k, v in quantize_weights(init_weights(cfg, 2), "mxfp4").items()}
    models = [SidDecoder(cfg, t, max_position=8) for t in (w, typed(w))]
    x = torch.randn(40, cfg.hidden, generator=torch.Generator().manual_seed(3)).to(device).to(cfg.dtype)
    for f in (lambda m: m._project(x, "layers.1.qkv"), lambda m: m._mlp(x, "layers.1.")):
        a, b = map(f, models)
        assert torch.equal(a, b) and a.isfinite().all() and (a != 0).any()
