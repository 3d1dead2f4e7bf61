"""The decoder with 8-bit weights and with experts, end to end on the GPU.

Models with experts, with and without 8-bit weights, and dense ones with them: a
layer's logits against float64, graph replays against eager runs, options of the
router.  (Whole beam searches are not compared with the oracle's: rounding to e4m3 is
a step, and a value that float32 sums leave on the other side of one -- one in about
10^5, of some 10^4 in a short prompt's layers -- moves what follows by per cents.)"""

import dataclasses

import numpy as np
import pytest
import torch

from oracle import sid_beam as so
from tests.test_gpu_fp8_linear import expand, quantise
from vllm_gr_amd.entrypoints.beam_search import BeamSearchParams
from vllm_gr_amd.entrypoints.llm import LLM
from vllm_gr_amd.v1.sid_decoder import DecoderConfig, SidDecoder, init_weights, quantize_weights
from vllm_gr_amd.v1.sid_runner import SidModelRunner, blocks_needed

pytestmark = pytest.mark.gpu

F32 = DecoderConfig(num_layers=2, hidden=64, num_heads=4, num_kv_heads=2, head_dim=32, ffn=96, vocab=96,
                    init_std=0.25, dtype=torch.float32)
BF16 = DecoderConfig(num_layers=2, hidden=256, num_heads=4, num_kv_heads=2, head_dim=128, ffn=512, vocab=512,
                     init_std=0.05, dtype=torch.bfloat16)
EXPERTS = dataclasses.replace(BF16, num_experts=16, experts_per_token=4, expert_ffn=128)


def prompts(seed, lens, vocab):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


def dequantised(w):
    """float64 weights: the e4m3 ones by their blocks."""
    out = {}
    for name, v in w.items():
        if name.endswith("_scale"):
            continue
        v = v.double()
        s = w.get(name + "_scale")
        if s is not None:
            s = s.double()
            N, K = v.shape[-2:]
            if name.endswith("gate_up"):
                half = s.shape[-2] // 2
                rows = torch.cat([expand(p, N // 2, -2) for p in s.split(half, -2)], -2)
            else:
                rows = expand(s, N, -2)
            v = v * expand(rows, K, -1)
        out[name] = v
    return out


def quantised(h):
    q, s = quantise(h)
    return q * expand(s, h.shape[1], 1)


def hooks(cfg, w, q):
    """The oracle's products and MLP for weights w (float64) with quantised inputs (q) and experts."""
    act = quantised if q else (lambda h: h)
    linear = lambda h, name: act(h) @ w[name].T
    if not cfg.num_experts:
        return dict(linear=linear)

    def mlp(h, p):
        logits = h @ w[p + "router"].T
        score = torch.softmax(logits, -1) if cfg.router_score == "softmax" else torch.sigmoid(logits)
        choice = score + w[p + "router_bias"] if p + "router_bias" in w else logits
        out = torch.zeros_like(h)
        for t in range(len(h)):
            c = choice[t].clone()
            if cfg.router_groups > 1:
                g = c.view(cfg.router_groups, -1)
                val = g.topk(2, 1)[0].sum(1) if p + "router_bias" in w else g.amax(1)
                drop = torch.ones(cfg.router_groups, dtype=torch.bool)
                drop[val.topk(cfg.router_top_groups)[1]] = False
                g[drop] = -float("inf")
            ids = c.topk(cfg.experts_per_token)[1]
            wt = score[t, ids]
            if cfg.router_renormalize:
                wt = wt / wt.sum()
            for e, v in zip(ids.tolist(), (wt * cfg.router_scale).tolist()):
                gate, up = (act(h[t:t + 1]) @ w[p + "expert_gate_up"][e].T).chunk(2, -1)
                a = torch.nn.functional.silu(gate) * up
                out[t] += v * (act(a) @ w[p + "expert_down"][e].T)[0]
        return out

    return dict(linear=linear, mlp=mlp)


CONFIGS = {
    "bf16 softmax": (EXPERTS, False), "bf16 8-bit": (EXPERTS, True),
    "sigmoid, bias, groups": (dataclasses.replace(EXPERTS, router_score="sigmoid", router_bias=True, router_groups=4,
                                                  router_top_groups=2, router_scale=2.5), False),
    "fp16, no renormalisation": (dataclasses.replace(EXPERTS, dtype=torch.float16, router_renormalize=False), True),
    "dense 8-bit": (BF16, True), "dense 8-bit, float32": (F32, True),
}


@pytest.mark.parametrize("name", CONFIGS)
def test_prefill_logits_against_float64(name):
    cfg, q = CONFIGS[name]
    cfg = dataclasses.replace(cfg, num_layers=1)
    w = init_weights(cfg, 7)
    if cfg.router_bias:
        w["layers.0.router_bias"] = 0.02 * torch.randn(cfg.num_experts, generator=torch.Generator().manual_seed(5))
    if q:
        w = quantize_weights(w)
    ps = prompts(7, [70, 129, 16], cfg.vocab)
    print(f"[sid] prefill {name}", flush=True)
    runner = SidModelRunner(SidDecoder(cfg, {k: v.cuda() for k, v in w.items()}, max_position=256), 64)
    got = runner.prefill(ps, ["a", "b", "c"])[0].cpu().double()
    wd = dequantised(w)
    far = []
    for i, p in enumerate(ps):
        ref = so.decoder_logits(wd, cfg, p, **hooks(cfg, wd, q))[-1]
        far.append(float((got[i] - ref).norm() / ref.norm()))
    # 16 bits: roundings of the residual stream and of every stage, about ten of 2^-9 each in one layer.  With e4m3
    # inputs, such a rounding ahead of a quantisation lands some of them a step s (2^-4 to 2^-3 of the value, about
    # 0.09) away, and the next quantisation sees that much more: at worst the two sides' rounding errors, s / sqrt(12)
    # each, have nothing in common, and a product's inputs differ by sqrt(2) s / sqrt(12) = 3.7 % of the norm.  qkv, o,
    # gate, up and down: five of them, 8.3 %.  float32: one or two single steps among 64 inputs, 2^-6 of the norm each.
    lim = 2.0 ** -5 if cfg.dtype == torch.float32 else 2.0 ** -3 if q else 2.0 ** -5.5
    assert max(far) <= lim, far


@pytest.mark.parametrize("name", CONFIGS)
def test_graph_replays_match_eager(name):
    """Captured decode steps with routing, workspaces and all: replays, with eager batches between them, give the
    eager run's beams and scores."""
    cfg, q = CONFIGS[name]
    seed, lens, W, steps = 7, [19, 44], 8, 4
    w = init_weights(cfg, seed)
    nb = blocks_needed(len(lens), max(lens), W, steps, 16) + 8
    wd = {k: v.cuda() for k, v in w.items()}
    kw = dict(weights=wd, num_blocks=nb, quantization="fp8" if q else None)
    eager, graphed = LLM(cfg, use_graphs=False, **kw), LLM(cfg, use_graphs=True, **kw)
    params = BeamSearchParams(W, steps)
    ps = prompts(seed, lens, cfg.vocab)
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


def test_llm_refuses_other_quantization():
    with pytest.raises(ValueError, match="quantization"):
        LLM(F32, num_blocks=8, quantization="int4")
