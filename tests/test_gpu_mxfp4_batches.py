"""A token's result of gr_expert_mlp_mxfp4 has the same bits in every call that holds it."""

import pytest
import torch

from tests.test_gpu_mxfp4_experts import make
from tests.test_mxfp4_tiles_host import experts_tile
from vllm_gr_amd import _C, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,F", [(512, 1024), (2080, 1056)])
def test_a_tokens_bits_do_not_depend_on_the_others(device, dtype, H, F):
    E, k = 16, 4
    a, *_ = make(1300, E, k, H, F, dtype, device)
    want = ops.expert_mlp_mxfp4(*a)
    tiles = {experts_tile(_C.lib(), 1300, k, E, H, F)}
    order = torch.randperm(1300, generator=torch.Generator().manual_seed(H)).to(device)
    for n in (1, 3, 17, 60, 130, 200, 260, 400, 700, 1100):
        pick = order[:n]
        got = ops.expert_mlp_mxfp4(a[0][pick], *a[1:5], a[5][pick].contiguous(), a[6][pick].contiguous())
        assert torch.equal(got, want[pick]), n
        tiles.add(experts_tile(_C.lib(), n, k, E, H, F))
    assert {rows for rows, _, _ in tiles} == {32, 64, 128, 256}, tiles
