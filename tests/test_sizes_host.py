"""Sizes that a C int does not hold are refused: ctypes would cut them off, and a
call of 2^32 + 8 rows would quietly do eight."""

import pytest
import torch

from vllm_gr_amd import ops


@pytest.mark.parametrize("shape", [(2 ** 32 + 8, 16), (2 ** 31, 1), (4, 2 ** 32 + 16)])
def test_rows_beyond_a_c_int(shape):
    with pytest.raises(ValueError, match="2\\^31"):
        ops._rows("x", torch.empty(shape, device="meta"))


def test_rows_that_a_c_int_holds():
    ops._rows("x", torch.empty(2 ** 31 - 1, 16, device="meta"))
    ops._rows("x", torch.empty(0, 16, device="meta"))


@pytest.mark.gpu
def test_route_options_beyond_a_c_int(device):
    """(refused on the host: no kernel is launched)"""
    logits = torch.zeros(3, 8, device=device)
    for kw in (dict(top_k=2 ** 32 + 2), dict(top_k=2, num_groups=2 ** 32 + 2), dict(top_k=2, num_groups=2, top_groups=2 ** 32 + 1),
               dict(top_k=2, num_groups=2 - 2 ** 32), dict(top_k=9), dict(top_k=2, num_groups=2, top_groups=3)):
        with pytest.raises(ValueError):
            ops.route_experts(logits, **kw)
