"""Static checks of the built 8-bit and expert kernels' gfx950 code, without a GPU."""

import re

import pytest

from tests.test_device_code import VMEM, _disassembly, _kernels, _scratch_sizes

NAMES = ("block_mm", "few_mm", "quant_fp8_k", "route_experts_k", "expert_count_k", "expert_plan_k", "expert_start_k",
         "expert_combine_k")


def test_kernels_keep_no_stack():
    """Tiles, fragments and row states live in registers and LDS: no kernel touches scratch."""
    sizes = _scratch_sizes()
    for n in NAMES:
        found = {k: v for k, v in sizes.items() if n in k}
        assert found, n
        assert all(v == 0 for v in found.values()), {k: v for k, v in found.items() if v}


def _into_lds(ins):
    return (ins.startswith("buffer_load_dwordx4 ") and ins.endswith(" lds")) or ins.startswith("global_load_lds_dword ")


def _among_transfers(code):
    """Vector-memory operations between the first transfer into LDS and the last that are none."""
    at = [i for i, ins in enumerate(code) if _into_lds(ins)]
    return [ins for ins in code[at[0]:at[-1]] if VMEM.match(ins) and not _into_lds(ins)]


def _stages(code):
    """The transfers in each straight line of code that has any: (rows' parts, scales')."""
    run, runs = [], []
    for ins in code:
        if _into_lds(ins):
            run.append(ins)
        elif ins.startswith(("s_cbranch", "s_branch", "s_barrier", "s_endpgm")) and run:
            runs.append(run)
            run = []
    return [(sum(i.startswith("buffer") for i in r), sum(i.startswith("global") for i in r)) for r in runs]


def test_transfers_are_what_the_waits_count():
    """block_mm waits for whole stages of transfers into LDS by their number: nothing else may be counted among them,
    and the code sends whole stages."""
    kernels = _kernels(_disassembly(), "block_mm")
    assert len(kernels) >= 20
    for name, code in kernels.items():
        assert not _among_transfers(code), (name, _among_transfers(code)[:3])
        xt, bm, bn, wm, wn = map(int, re.search(r"block_mmILi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)", name).groups())
        per = (bm + bn) // 8 // (wm * wn)
        rows = sum(r for r, _ in _stages(code))
        scales = sum(s for _, s in _stages(code))
        assert rows % per == 0 and rows >= 2 * per, (name, rows, per)
        # a stage is sent whole or with a short end: two bodies of rows' transfers, then one of scales
        assert (scales > 0) == (xt == 3) and (xt != 3 or rows == 2 * per * scales), (name, rows, scales, per)


def test_checks_flag_a_miscount():
    rows = ["buffer_load_dwordx4 v0, s[0:3], s4 offen lds"] * 4
    assert _among_transfers(rows) == []
    assert _among_transfers(rows[:2] + ["global_load_dword v1, v[2:3], off"] + rows[2:]) != []
    more = ["s_branch 3"] + rows[:3] + ["global_load_lds_dword v[0:1], off", "s_barrier"]
    assert _stages(rows + more) == [(4, 0), (3, 1)]
