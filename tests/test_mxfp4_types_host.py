"""The types of 4-bit tensors, without a GPU: a torch without its own 4-bit and scale types runs all the same."""

import importlib.util

import pytest
import torch

from vllm_gr_amd import ops


@pytest.mark.parametrize("missing", [("float4_e2m1fn_x2",), ("float4_e2m1fn_x2", "float8_e8m0fnu")])
def test_import_without_torchs_own_types(monkeypatch, missing):
    for name in missing:
        monkeypatch.delattr(torch, name)
    spec = importlib.util.spec_from_file_location("vllm_gr_amd._ops_again", ops.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    x4, scale = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    assert again._mx_rows("x", x4, scale) == (4, 64, 32, 2)
    for bad in ((x4.int(), scale), (x4, scale.int())):
        with pytest.raises(ValueError):
            again._mx_rows("x", *bad)
