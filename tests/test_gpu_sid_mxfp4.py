"""The decoder with 4-bit weights on the GPU: its layers are the entry points' products in
their order, a float32 model's logits are float64's, and graph replays are eager runs."""

import dataclasses

import numpy as np
import pytest
import torch

from oracle import sid_beam as so
from tests.test_gpu_mxfp4 import quantise, unpack, values
from tests.test_gpu_sid_experts import BF16, EXPERTS, F32, prompts
from vllm_gr_amd import ops
from vllm_gr_amd.entrypoints.beam_search import BeamSearchParams
from vllm_gr_amd.entrypoints.llm import LLM
from vllm_gr_amd.v1.sid_decoder import SidDecoder, init_weights, quantize_mxfp4, quantize_weights
from vllm_gr_amd.v1.sid_runner import SidModelRunner, blocks_needed

pytestmark = pytest.mark.gpu


def test_quantize_mxfp4_on_the_device_is_the_kernels(device):
    w = torch.randn(300, 416, generator=torch.Generator().manual_seed(3)).to(device)
    for t in (w, w.bfloat16()):
        assert all(torch.equal(a, b) for a, b in zip(quantize_mxfp4(t), ops.quant_mxfp4(t)))


def test_prefill_logits_against_float64():
    cfg = dataclasses.replace(F32, num_layers=1)
    w = quantize_weights(init_weights(cfg, 7), "mxfp4")
    ps = prompts(7, [70, 129, 16], cfg.vocab)
    runner = SidModelRunner(SidDecoder(cfg, {k: v.cuda() for k, v in w.items()}, max_position=256), 64)
    got = runner.prefill(ps, ["a", "b", "c"])[0].cpu().double()
    wd = {k: values(unpack(v), w[k + "_scale"]) if k + "_scale" in w else v.double() for k, v in w.items()
          if not k.endswith("_scale")}
    linear = lambda h, name: values(*quantise(h)) @ wd[name].T
    far = []
    for i, p in enumerate(ps):
        ref = so.decoder_logits(wd, cfg, p, linear=linear)[-1]
        far.append(float((got[i] - ref).norm() / ref.norm()))
    # float32 sums leave about one value in 10^5 on the other side of a border: of a token's 64 inputs of a product at
    # most one, and that by half a unit where their root mean square is 2.2 (blocks' largest being 4 to 7): 2.8 %
    assert max(far) <= 2.0 ** -5, far


@pytest.mark.parametrize("T", [1, 40, 600])
@pytest.mark.parametrize("cfg", [F32, BF16, EXPERTS], ids=["float32", "bf16", "experts"])
def test_layers_are_the_entry_points(device, cfg, T):
    w = {k: v.to(device) for k, v in quantize_weights(init_weights(cfg, 2), "mxfp4").items()}
    model = SidDecoder(cfg, w, max_position=8)
    p = "layers.1."
    x = torch.randn(T, cfg.hidden, generator=torch.Generator().manual_seed(T)).to(device).to(cfg.dtype)
    x4 = ops.quant_mxfp4(x)
    want = ops.linear_mxfp4(*x4, w[p + "qkv"], w[p + "qkv_scale"], out_dtype=cfg.dtype)
    assert torch.equal(model._project(x, p + "qkv"), want)
    if cfg.num_experts:
        logits = ops.linear(x, w[p + "router"], out_f32=True) if cfg.hidden >= 512 else x.float() @ w[p + "router"].float().T
        weights, ids = ops.route_experts(logits, cfg.experts_per_token)
        want = ops.expert_mlp_mxfp4(x, *(w[p + n] for n in ("expert_gate_up", "expert_gate_up_scale", "expert_down",
                                                           "expert_down_scale")), weights, ids)
    else:
        act = ops.linear_mxfp4(*x4, w[p + "gate_up"], w[p + "gate_up_scale"], swiglu=True, quantized=True)
        want = ops.linear_mxfp4(*act, w[p + "down"], w[p + "down_scale"], out_dtype=cfg.dtype)
    assert torch.equal(model._mlp(x, p), want)


@pytest.mark.parametrize("cfg", [F32, BF16, EXPERTS, dataclasses.replace(EXPERTS, dtype=torch.float16)],
                         ids=["float32", "bf16", "experts", "experts fp16"])
def test_graph_replays_match_eager(cfg):
    """Captured decode steps, workspaces and all: replays, with eager batches between them, give the eager run's beams
    and scores."""
    lens, W, steps = [19, 44], 8, 4
    nb = blocks_needed(len(lens), max(lens), W, steps, 16) + 8
    kw = dict(weights={k: v.cuda() for k, v in init_weights(cfg, 7).items()}, num_blocks=nb, quantization="mxfp4")
    eager, graphed = LLM(cfg, use_graphs=False, **kw), LLM(cfg, use_graphs=True, **kw)
    params, ps = BeamSearchParams(W, steps), prompts(7, lens, cfg.vocab)
    ref = eager.beam_search(ps, params)
    for i in range(3):
        got = graphed.beam_search(ps, params)
        torch.cuda.synchronize()
        for o, r in zip(got, ref):
            assert [s.tokens for s in o.sequences] == [s.tokens for s in r.sequences], i
            assert np.allclose([s.cum_logprob for s in o.sequences], [s.cum_logprob for s in r.sequences], rtol=0,
                               atol=1e-5), i
        eager.beam_search(ps, params)
    assert len(graphed.runner._graphs) == 1
