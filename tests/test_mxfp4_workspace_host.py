"""The 4-bit experts' workspace, without a GPU: one for the most tokens holds every smaller call's."""

import pytest


@pytest.mark.parametrize("E,k,H,F", [(1024, 1, 32, 32), (256, 2, 64, 64), (64, 8, 2048, 768), (1, 1, 32, 4096), (2, 2, 32, 128),
                                     (8, 2, 2048, 512), (1024, 8, 64, 32)])
def test_more_tokens_need_no_less(built_lib, E, k, H, F):
    size = built_lib.gr_expert_mlp_mxfp4_workspace_size
    needs = [size(T, k, E, H, F) for T in range(1, 40000)]
    assert all(a <= b for a, b in zip(needs, needs[1:]))
