"""Decoder weights in 4 bits, on the CPU: what quantize_weights makes of them, and what
the decoder refuses when it is built."""

import dataclasses

import pytest
import torch

from tests.test_gpu_mxfp4 import pack, quantise
from vllm_gr_amd.v1.sid_decoder import DecoderConfig, SidDecoder, init_weights, quantize_mxfp4, quantize_weights

DENSE = DecoderConfig(num_layers=2, hidden=64, num_heads=4, num_kv_heads=2, head_dim=32, ffn=160, vocab=96)
EXPERTS = dataclasses.replace(DENSE, num_experts=8, experts_per_token=2, expert_ffn=96)


def build(cfg, weights):
    return SidDecoder(cfg, weights, max_position=8)


@pytest.mark.parametrize("shape", [(1, 32), (16, 96), (3, 130, 288), (2, 2, 48, 64)])
def test_quantize_mxfp4(shape):
    """The definition's codes and scales, with blocks of zeros, tiny and large values and borders among them."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(*shape, generator=g) * torch.exp(20 * torch.randn(*shape[:-1], 1, generator=g)).clamp(2e-38, 1e37)
    w[..., :1, :32] = 0
    w[..., -1:, :8] = torch.tensor([7.0, 0.25, 0.75, 1.25, 2.5, 3.5, 5.0, -0.25])
    w4, s = quantize_mxfp4(w)
    codes, byte = quantise(w.double())
    assert w4.dtype == s.dtype == torch.uint8 and w4.is_contiguous() and s.is_contiguous()
    assert w4.shape == (*shape[:-1], shape[-1] // 2) and s.shape == (*shape[:-1], shape[-1] // 32)
    assert torch.equal(s, byte) and torch.equal(w4, pack(codes))
    with pytest.raises(ValueError, match="multiple of 32"):
        quantize_mxfp4(torch.zeros(4, 48))


def test_quantize_weights():
    for cfg in (DENSE, EXPERTS):
        w = init_weights(cfg, 2)
        q = quantize_weights(w, "mxfp4")
        assert quantize_weights(q, "mxfp4").keys() == quantize_weights(q).keys() == q.keys()  # once is enough
        for name, v in w.items():
            kind = name.rsplit(".", 1)[-1]
            if kind in ("qkv", "o", "gate_up", "down", "expert_gate_up", "expert_down"):
                assert q[name].dtype == q[name + "_scale"].dtype == torch.uint8
                assert q[name].shape == (*v.shape[:-1], v.shape[-1] // 2)
                assert q[name + "_scale"].shape == (*v.shape[:-1], v.shape[-1] // 32)
                assert quantize_weights(q, "mxfp4")[name] is q[name]
            else:
                assert q[name] is v and name + "_scale" not in q
        build(cfg, q)
    with pytest.raises(ValueError, match="quantization"):
        quantize_weights(w, "int4")


def test_sizes_that_4_bits_do_not_take():
    w = init_weights(dataclasses.replace(DENSE, ffn=144), 1)
    with pytest.raises(ValueError, match="multiple of 32"):  # down's features
        quantize_weights(w, "mxfp4")
    q = quantize_weights(init_weights(DENSE, 1), "mxfp4")
    p = "layers.0."
    for name, rows in (("gate_up", 2 * 144), ("gate_up", 319)):  # gate and up's rows, which are the next product's features
        bad = dict(q)
        bad[p + name], bad[p + name + "_scale"] = q[p + name][:rows], q[p + name + "_scale"][:rows]
        with pytest.raises(ValueError, match="multiples of 32"):
            build(DENSE, bad)


def test_weights_and_scales_that_do_not_match():
    w = init_weights(DENSE, 1)
    q = quantize_weights(w, "mxfp4")
    q8 = quantize_weights(w)
    p = "layers.1."
    for change in (dict(qkv_scale=None), dict(gate_up_scale=None), dict(down_scale=None),
                   dict(qkv=torch.zeros(q[p + "qkv"].shape, dtype=torch.bfloat16)), dict(o_scale=q[p + "o_scale"].float()),
                   dict(gate_up_scale=q[p + "gate_up_scale"][:2]), dict(qkv_scale=q8[p + "qkv_scale"]),
                   dict(down_scale=q[p + "down_scale"].t().contiguous().t()),
                   dict(down=q8[p + "down"], down_scale=q8[p + "down_scale"]), dict(gate_up=w[p + "gate_up"], gate_up_scale=None)):
        bad = dict(q)
        for name, t in change.items():
            if t is None:
                del bad[p + name]
            else:
                bad[p + name] = t
        with pytest.raises(ValueError, match="layers.1"):
            build(DENSE, bad)
    mixed = dict(q)  # attention in 8 bits beside an MLP in 4 is fine
    for n in ("qkv", "qkv_scale", "o", "o_scale"):
        mixed[p + n] = q8[p + n]
    build(DENSE, mixed)
