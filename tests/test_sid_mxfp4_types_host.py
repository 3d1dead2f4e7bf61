"""A decoder takes 4-bit weights in the types that its products take, on the CPU."""

import pytest
import torch

from tests.test_sid_mxfp4_host import DENSE, EXPERTS, build
from vllm_gr_amd.v1.sid_decoder import init_weights, quantize_weights

FP4, E8 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def typed(q, codes=FP4, scales=E8):
    return {k: v.view(scales) if k.endswith("_scale") else v.view(codes) if k + "_scale" in q else v for k, v in q.items()}


@pytest.mark.parametrize("cfg", [DENSE, EXPERTS], ids=["dense", "experts"])
def test_types_of_codes_and_scales(cfg):
    q = quantize_weights(init_weights(cfg, 2), "mxfp4")
    for codes in (torch.uint8, FP4):
        for scales in (torch.uint8, E8):
            build(cfg, typed(q, codes, scales))
    t = typed(q)
    assert all(quantize_weights(t, "mxfp4")[k] is v for k, v in t.items())
    p = "layers.0."
    down = p + ("expert_down" if cfg.num_experts else "down")
    build(cfg, {**t, down: q[down]})  # gate and up in one of the types, down in the other


def test_refusals():
    q = quantize_weights(init_weights(DENSE, 1), "mxfp4")
    t = typed(q)
    p = "layers.1."
    for change in (dict(qkv_scale=None), dict(o_scale=q[p + "o_scale"].float()), dict(gate_up_scale=t[p + "gate_up_scale"][:2]),
                   dict(qkv=torch.zeros(q[p + "qkv"].shape, dtype=torch.bfloat16)), dict(qkv=t[p + "qkv"].view(torch.int8))):
        bad = {**t, **{p + k: v for k, v in change.items()}}
        with pytest.raises(ValueError, match="layers.1"):
            build(DENSE, {k: v for k, v in bad.items() if v is not None})
