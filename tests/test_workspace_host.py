"""A caller's workspace counts by the memory behind it: an expanded tensor has many
elements and little memory, so the entry points take contiguous ones only."""

import pytest
import torch

from vllm_gr_amd import ops


def test_bytes_of_a_workspace():
    assert ops._workspace_bytes(torch.empty(100, dtype=torch.uint8)) == 100
    assert ops._workspace_bytes(torch.empty(4, 8)[1:3]) == 64
    for t in (torch.empty(1, dtype=torch.uint8).expand(1 << 20), torch.empty(64, 4).t(), torch.empty(64)[::2]):
        with pytest.raises(ValueError, match="contiguous"):
            ops._workspace_bytes(t)


@pytest.mark.gpu
def test_entry_points_refuse_an_expanded_workspace(device):
    """(refused on the host: no kernel is launched)"""
    T, E, k, H, F = 4, 2, 1, 64, 32
    half = dict(dtype=torch.bfloat16, device=device)
    need = ops.expert_mlp_workspace_bytes(T, k, E, H, F, False)
    ws = torch.empty(1, dtype=torch.uint8, device=device).expand(need)
    with pytest.raises(ValueError, match="contiguous"):
        ops.expert_mlp(torch.zeros(T, H, **half), torch.zeros(E, 2 * F, H, **half), torch.zeros(E, H, F, **half),
                       torch.ones(T, k, device=device), torch.zeros(T, k, dtype=torch.int32, device=device), workspace=ws)
    ws = torch.empty(1, dtype=torch.uint8, device=device).expand(ops.prune_workspace_bytes(2, 4, 64, 4))
    with pytest.raises(ValueError, match="contiguous"):
        ops.beam_prune_topk(torch.zeros(2, 4, 64, device=device), torch.zeros(2, 4, device=device), 4, workspace=ws)
