"""How far the rounding of an expert's result on its way to the sum over a token's
experts goes: half a step of fp16, 2^-11 of the value, reached."""

import pytest
import torch

from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 700])
def test_waiting_result_is_off_by_up_to_half_a_step(device, T):
    """One expert, e4m3 weights, fp16 results.  The expert's result is just below half a
    step of fp16 above a power of two and waits as that power; a weight just below half a
    step above 1 makes the last rounding lose as much again."""
    H = F = 128
    x = torch.zeros(T, H)
    x[:, 0] = 1
    gu = torch.zeros(1, 2 * F, H)
    gu[0, 0, 0] = 4.0
    gu[0, F, 0] = 2.0
    dn = torch.zeros(1, H, F)
    dn[0, :, 0] = 1.0
    act = float(torch.sigmoid(torch.tensor(4.0, dtype=torch.float64)) * 8)
    part = 0.99 * 2.0 ** -11  # (1 % of 2^-11 is 2^-18: more than the float32 roundings on the way)
    ds = torch.tensor((1 + part) / act)
    w = torch.tensor(1 + part)
    to8 = lambda t: t.to(torch.float8_e4m3fn).to(device)
    out = ops.expert_mlp(x.half().to(device), to8(gu), to8(dn), w.expand(T, 1).contiguous().to(device),
                         torch.zeros(T, 1, dtype=torch.int32, device=device),
                         gate_up_scale=torch.ones(1, 2, 1, device=device), down_scale=ds.view(1, 1, 1).to(device))
    y = act * float(ds) * float(w)
    off = (out.cpu().double() - y).abs() / y
    assert (off <= 2 * 2.0 ** -11 + 2.0 ** -20).all()  # the waiting result's half step and the output's
    assert (off > 2.0 ** -11 + 2.0 ** -12).all()       # and not half of the first
