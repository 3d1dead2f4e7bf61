"""gr_linear_fp8's results where a caller puts them: quantised ones at every row
count into the layouts that gr_experts.h allows.  Bounds and references as in the
module of its other tests."""

import pytest
import torch

from tests.test_gpu_fp8_linear import E4M3, check_quantised, operands
from vllm_gr_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("offset,stride", [(0, 256), (4, 260), (8, 256), (12, 268)])
@pytest.mark.parametrize("M", [1, 8, 64, 65, 300])
def test_quantised_out_in_a_wider_tensor(device, M, offset, stride, swiglu):
    """Rows 4 bytes aligned at least, some bytes behind the last, scales in either order:
    the same layouts for few rows as for many, and nothing around them is written."""
    N, K = 240, 272
    (x8, xs, w8, ws), y, err, _ = operands(M, N, K, swiglu, device)
    whole = torch.full((M + 1, stride), 0x33, dtype=torch.uint8, device=device)
    rows = whole.view(-1)[offset:offset + M * stride].view(M, stride)
    out = rows[:, :N].view(E4M3)
    scale = torch.full((M, 4), 7.0, device=device)
    part = scale[:, 1:3] if offset else scale.view(4, M).t()[:, 1:3]
    got, s = ops.linear_fp8(x8, xs, w8, ws, swiglu=swiglu, quantized=True, out=out, out_scale=part)
    assert got.data_ptr() == out.data_ptr() and s.data_ptr() == part.data_ptr()
    check_quantised(got, s, y, err)
    rest = whole.view(-1).clone()
    rest[offset:offset + M * stride].view(M, stride)[:, :N] = 0x33
    assert (rest == 0x33).all()
    assert int((scale == 7.0).sum()) == 2 * M
