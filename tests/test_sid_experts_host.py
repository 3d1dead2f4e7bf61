"""Decoder weights with experts and in 8 bits, on the CPU: what init_weights draws,
what quantize_weights makes of it, and the oracle's hooks for both."""

import dataclasses

import pytest
import torch

from oracle import sid_beam as so
from vllm_gr_amd.v1.sid_decoder import DecoderConfig, SidDecoder, init_weights, quantize_blocks, quantize_weights

DENSE = DecoderConfig(num_layers=2, hidden=64, num_heads=4, num_kv_heads=2, head_dim=32, ffn=144, vocab=96,
                      dtype=torch.float32)
EXPERTS = dataclasses.replace(DENSE, num_experts=6, experts_per_token=2, expert_ffn=48, router_bias=True)


@pytest.mark.parametrize("cfg", [DENSE, EXPERTS, dataclasses.replace(EXPERTS, router_bias=False, tie_embeddings=False)])
def test_num_params_and_shapes(cfg):
    w = init_weights(cfg, 1)
    n = sum(v.numel() for k, v in w.items() if not (k == "lm_head" and cfg.tie_embeddings))
    assert n == cfg.num_params()
    assert ("layers.0.gate_up" in w) == (cfg.num_experts == 0)
    if cfg.num_experts:
        assert w["layers.1.expert_gate_up"].shape == (6, 96, 64) and w["layers.1.expert_down"].shape == (6, 64, 48)
        assert w["layers.1.router"].shape == (6, 64)
        assert ("layers.1.router_bias" in w) == cfg.router_bias


def test_dense_weights_are_drawn_as_ever():
    """A dense model's draws (embedding, then qkv, o, gate_up, down of each layer) do not depend on the options for experts."""
    g = torch.Generator().manual_seed(3)
    w = init_weights(DENSE, 3)
    for name, shape in (("embed", (96, 64)), ("layers.0.qkv", (256, 64)), ("layers.0.o", (64, 128)),
                        ("layers.0.gate_up", (288, 64)), ("layers.0.down", (64, 144)), ("layers.1.qkv", (256, 64))):
        assert torch.equal(w[name], torch.randn(*shape, generator=g).mul_(DENSE.init_std)), name


@pytest.mark.parametrize("shape", [(16, 16), (128, 256), (3, 130, 272), (2, 2, 48, 400)])
def test_quantize_blocks(shape):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(1))
    w[..., :4, :] = 0
    w8, s = quantize_blocks(w)
    N, K = shape[-2:]
    assert w8.shape == w.shape and w8.dtype == torch.float8_e4m3fn
    assert s.shape == (*shape[:-2], -(-N // 128), -(-K // 128)) and s.is_contiguous()
    for b in range(s.shape[-2]):
        for c in range(s.shape[-1]):
            part = w[..., 128 * b:128 * b + 128, 128 * c:128 * c + 128]
            got = w8[..., 128 * b:128 * b + 128, 128 * c:128 * c + 128].float() * s[..., b:b + 1, c:c + 1]
            amax = part.abs().amax((-2, -1))
            assert torch.equal(s[..., b, c], (amax / 448).clamp_min(2.0 ** -80))
            # half a step: 2^-4 of the value, 2^-10 of the scale below the normal range
            assert ((got - part).abs() <= torch.maximum(part.abs() * 2.0 ** -4, s[..., b:b + 1, c:c + 1] * 2.0 ** -10)
                    * 1.0001).all()
    assert quantize_blocks(torch.zeros(32, 32))[1].item() == 2.0 ** -80


def test_quantize_weights():
    for cfg in (DENSE, EXPERTS):
        w = init_weights(cfg, 2)
        q = quantize_weights(w)
        assert quantize_weights(q).keys() == q.keys()  # once is enough
        for name, v in w.items():
            kind = name.rsplit(".", 1)[-1]
            if kind in ("qkv", "o", "gate_up", "down", "expert_gate_up", "expert_down"):
                assert q[name].dtype == torch.float8_e4m3fn and q[name].shape == v.shape
                assert quantize_weights(q)[name] is q[name]
            else:
                assert q[name] is v and name + "_scale" not in q
        p = "layers.0."
        if cfg is DENSE:  # gate's 144 rows and up's are blocks of their own
            assert q[p + "gate_up_scale"].shape == (4, 1)
            up = w[p + "gate_up"][144:]
            assert torch.equal(q[p + "gate_up"][144:].float(), quantize_blocks(up)[0].float())
        else:
            assert q[p + "expert_gate_up_scale"].shape == (6, 2, 1) and q[p + "expert_down_scale"].shape == (6, 1, 1)


def test_experts_need_sixteen_bits():
    with pytest.raises(ValueError, match="16-bit"):
        SidDecoder(EXPERTS, init_weights(EXPERTS, 1))


def test_oracle_hooks_are_the_plain_model():
    w = so.weights_f64(init_weights(DENSE, 4))

    def mlp(h, p):
        g, u = (h @ w[p + "gate_up"].T).chunk(2, -1)
        return (torch.nn.functional.silu(g) * u) @ w[p + "down"].T

    toks = [3, 9, 27, 81]
    plain = so.decoder_logits(w, DENSE, toks)
    assert torch.equal(so.decoder_logits(w, DENSE, toks, linear=lambda h, n: h @ w[n].T), plain)
    assert torch.allclose(so.decoder_logits(w, DENSE, toks, mlp=mlp), plain, rtol=1e-12, atol=1e-12)
