"""Static checks of the built 4-bit kernels' gfx950 code, without a GPU."""

import re

from tests.test_device_code import _disassembly, _kernels, _scratch_sizes

NAMES = ("mx_quant_k", "mx_dequant_k", "mx_mm", "mx_few", "mx_expert_start_k")


def test_kernels_keep_no_stack():
    sizes = _scratch_sizes()
    for n in NAMES:
        found = {k: v for k, v in sizes.items() if n in k}
        assert found, n
        assert all(v == 0 for v in found.values()), {k: v for k, v in found.items() if v}


def _rows(ins):
    return ins.startswith("buffer_load_dwordx4 ") and ins.endswith(" lds")


def _scales(ins):
    return ins.startswith(("global_load_lds_dword ", "global_load_lds_dwordx4 "))


def _late(code):
    """Transfers of scales that follow rows' in a straight line of code."""
    rows, late = 0, 0
    for ins in code:
        if ins.startswith(("s_cbranch", "s_branch", "s_barrier", "s_endpgm")):
            rows = 0
        rows += _rows(ins)
        late += _scales(ins) and rows > 0
    return late


def test_transfers_are_what_the_waits_count():
    """mx_mm's loop waits until only its ST - 2 youngest stages' transfers are under way: it sends whole stages, a
    stage's scales ahead of its rows, and its first wait counts those stages' rows."""
    kernels = _kernels(_disassembly(), "mx_mm")
    assert len(kernels) >= 20
    for name, code in kernels.items():
        bm, bn, wm, wn, kg, st = map(int, re.search(r"mx_mmI" + r"Li(\d+)E" * 6, name).groups())
        per = (bm + bn) // 8 // (wm * wn)  # of a wave: kg groups of them send kg stages
        # the first stages, then the loop's body, sent once each
        assert sum(map(_rows, code)) == st * per and _late(code) == 0, name
        waits = [code[i - 1] for i, ins in enumerate(code) if ins.startswith("s_barrier")]
        assert waits[0] == f"s_waitcnt vmcnt({(st - 2) * per}) lgkmcnt(0)", (name, waits)
        assert waits[1] == "s_waitcnt vmcnt(0) lgkmcnt(0)", (name, waits)


def test_checks_flag_a_miscount():
    row, scale = "buffer_load_dwordx4 v0, s[0:3], s4 offen lds", "global_load_lds_dword v[0:1], off"
    assert _late([scale, row, row, "s_branch 5", scale, row, "s_barrier", scale, "s_endpgm"]) == 0
    assert _late([row, scale, row, "s_barrier"]) == 1
