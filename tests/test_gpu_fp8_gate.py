"""silu(gate) * up where the gate's sigmoid leaves the normal float32 numbers: as
long as gate * sigmoid(gate) is one (down to a gate of -91.8), the result counts."""

import pytest
import torch

from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 300, 2000])
def test_gate_to_the_end_of_the_normal_numbers(device, M):
    """The gates are exact in float32 (a row's scale times -88).  Their exponential's
    argument is off by half a unit of a number below 128 (2^-18) and by its constant's
    rounding (92 x 1.45 x 2^-25): ln 2 of it, 5.3e-6 with the last roundings, below 2^-17."""
    N, K = 256, 128
    gates = [-88.0, -80.0, -72.0, -1.0, 0.0, 80.0]
    rows = torch.tensor([1.0, 65 / 64, 33 / 32, 133 / 128]).repeat(M // 4 + 1)[:M] if M > 1 else torch.tensor([133 / 128])
    x = torch.zeros(M, K)
    x[:, 0] = 1
    w = torch.zeros(2 * N, K)
    w[:N, 0] = torch.tensor(gates).repeat(N // len(gates) + 1)[:N]
    w[N:, 0] = 448
    ws = torch.ones(4, 1)
    ws[2:] = 2.0 ** 90
    to8 = lambda t: t.to(torch.float8_e4m3fn).to(device)
    got = ops.linear_fp8(to8(x), rows[:, None].to(device), to8(w), ws.to(device), swiglu=True,
                         out_dtype=torch.float32).cpu().double()
    g = w[None, :N, 0].double() * rows[:, None].double()
    assert (g.min() == -88.0 * 133 / 128) and ((g * torch.sigmoid(g))[g != 0].abs() >= 2.0 ** -126).all()
    want = g * torch.sigmoid(g) * 448 * rows[:, None].double() * 2.0 ** 90
    assert ((got - want).abs() <= want.abs() * 2.0 ** -17).all()


def test_gate_beside_an_infinity(device):
    """An infinite up is not a NaN before the sigmoid is 0."""
    M, N, K = 4, 32, 128
    x = torch.zeros(M, K)
    x[:, 0] = 1
    w = torch.zeros(2 * N, K)
    w[:N, 0] = -88
    w[N:, 0] = 448
    ws = torch.tensor([[1.0], [float("inf")]])
    to8 = lambda t: t.to(torch.float8_e4m3fn).to(device)
    scale = torch.full((M, 1), 33 / 32, device=device)
    got = ops.linear_fp8(to8(x), scale, to8(w), ws.to(device), swiglu=True, out_dtype=torch.float32)
    assert (got == -float("inf")).all()
