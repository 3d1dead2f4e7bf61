"""The sum over a token's experts of gr_expert_mlp_mxfp4 holds float32 throughout.

Operands whose products are exact: a token's only feature is 4, each gate sum 64 (whose
sigmoid is 1 in float32), each up sum a quarter of an e2m1 number, with a 6 in each block
of 32, so that the gated product is sixteen times that number in 4 bits too.  A down sum is
then a multiple of 2^-1 and below 2^23, exact in any order.  What is left is the weighted sum, k steps of
2^-24 of the magnitudes so far, and the rounding of the result: half a step, 2^-8 bf16, 2^-11 fp16.  The experts come in
pairs of nearly opposite results, so that a result that waits in fewer bits shows."""

import pytest
import torch

from tests.test_gpu_mxfp4 import HALF, pack, values
from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
# (rows an expert on average for tiles of 32, 64, 128 and 256 rows; hidden sizes in tiles of 64 columns and not)
@pytest.mark.parametrize("T,E,k,H,F", [(5, 8, 4, 288, 96), (80, 8, 4, 1024, 128), (200, 4, 2, 544, 64), (600, 4, 2, 512, 256)])
def test_experts_results_wait_in_float32(device, dtype, T, E, k, H, F):
    g = torch.Generator().manual_seed(T)
    x = torch.zeros(T, H, dtype=dtype)
    x[:, 0] = 4.0
    gu = torch.zeros(E, 2 * F, H, dtype=torch.uint8)
    gu[:, :F, 0] = 6  # a 4, times 2^2: the gate's sum is 4 * 16
    up = torch.randint(0, 16, (E // 2, F), generator=g, dtype=torch.uint8)
    up[:, ::32] = 7
    up = torch.cat([up, up ^ 8])  # expert e + E / 2 has the opposite of expert e's products
    gu[:, F:, 0] = up
    gus = torch.full((E, 2 * F, H // 32), 127, dtype=torch.uint8)
    gus[:, :F] = 129
    gus[:, F:] = 123
    dn = torch.randint(0, 16, (E // 2, H, F), generator=g, dtype=torch.uint8)
    dns = torch.randint(124, 130, (E // 2, H, F // 32), generator=g, dtype=torch.uint8)
    near = dn.clone()
    near[:, :, 3] ^= 5  # one feature's number is another
    dn, dns = torch.cat([dn, near]), torch.cat([dns, dns])
    act = 16.0 * values(up, torch.full((E, F // 32), 127, dtype=torch.uint8))
    y = torch.einsum("ehf,ef->eh", values(dn, dns), act)
    first = torch.stack([torch.randperm(E // 2, generator=g)[:k // 2] for _ in range(T)])
    ids = torch.stack([first, first + E // 2], 2).flatten(1)
    w = (1.0 + torch.rand(T, k, generator=g) * 2.0 ** -8).float()
    each = w.double()[..., None] * y[ids]
    want, size = each.sum(1), each.abs().sum(1)
    got = ops.expert_mlp_mxfp4(*(t.to(device) for t in (x, pack(gu), gus, pack(dn), dns, w, ids.int()))).cpu().double()
    off = size * k * 2.0 ** -24
    assert ((got - want).abs() <= off + (want.abs() + off) * HALF[dtype] + 2.0 ** -25).all()
