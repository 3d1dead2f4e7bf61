"""The tiles of the 4-bit experts' products, without a GPU."""

import pytest


def experts_tile(lib, *sizes):
    """Tile rows, stages of the gated product and columns of the down product of (tokens, top_k, experts, hidden, ffn)."""
    t = lib.gr_expert_mlp_mxfp4_tile(*sizes)
    return t // 1000 % 1000, t // 1000000, t % 1000


# (sizes, the fastest tile measured): few or small experts, whose rows alone would take tiles of which the CUs get few
@pytest.mark.parametrize("sizes,rows", [((1200, 1, 4, 512, 256), 32), ((700, 1, 2, 1024, 512), 32), ((2000, 2, 8, 2048, 512), 128),
                                        ((512, 2, 8, 4096, 1024), 64), ((2048, 1, 8, 2048, 256), 64), ((2048, 4, 16, 1024, 256), 128),
                                        ((4000, 1, 2, 512, 128), 32), ((80, 1, 1, 2048, 2048), 32), ((1024, 4, 16, 1024, 256), 64)])
def test_experts_tiles_reach_the_cus(built_lib, sizes, rows):
    assert experts_tile(built_lib, *sizes)[0] == rows


# and sizes with work for all of them: the tile that their rows take
@pytest.mark.parametrize("tokens,rows", [(1, 32), (224, 32), (512, 64), (640, 128), (2048, 128), (2400, 256), (8192, 256)])
def test_experts_tiles_by_rows(built_lib, tokens, rows):
    assert experts_tile(built_lib, tokens, 8, 64, 2048, 768)[0] == rows
    assert experts_tile(built_lib, 2048, 2, 8, 2048, 6144)[0] == 256


def test_experts_tile_arguments(built_lib):
    good = (4, 2, 8, 256, 128)
    for i in range(5):
        assert built_lib.gr_expert_mlp_mxfp4_tile(*good[:i], 0, *good[i + 1:]) == 0
    for bad in ((4, 2, 8, 2 ** 21 + 32, 128), (4, 2, 8, 256, 2 ** 31 - 1)):
        assert built_lib.gr_expert_mlp_mxfp4_tile(*bad) == 0
    assert experts_tile(built_lib, *good) == (32, 3, 64)
    assert experts_tile(built_lib, 64, 8, 64, 2048, 768) == (32, 2, 256)


def test_linear_tile_arguments(built_lib):
    f = built_lib.gr_linear_mxfp4_tile
    assert f(8, 64, 256, 0, 2) == 16016 and f(8, 64, 256, 1, 2) == 16032 and f(8, 64, 256, 0, 4) == 16032 and f(8, 64, 256, 1, 4) == 16064
    for bad in ((0, 64, 256), (8, 0, 256), (8, 64, 0), (2 ** 28 + 1, 64, 256), (8, 2 ** 28 + 1, 256)):
        assert f(*bad, 0, 2) == 0


def test_every_form_is_tested(built_lib):
    """The device tests name a size for each form that any size of a wide grid takes, and the form that it takes."""
    from tests.test_gpu_mxfp4_tiles import EXPERT_TILES, TILES, tile
    rows = [1, 2, 5, 9, 15, 17, 24, 33, 48, 64, 65, 90, 128, 129, 180, 256, 300, 400, 512, 700, 1000, 1500, 2048, 3000, 5000, 8192]
    columns = [32, 96, 256, 512, 1024, 1536, 2048, 2592, 4096, 5120, 6144, 8192, 10240, 12288, 16384, 24576]
    features = [32, 256, 512, 1024, 1536, 2048, 2592, 4096, 6144, 8192]
    for mode, forms in TILES.items():
        taken = {tile(mode, M, N, K) for M in rows for N in columns for K in features}
        assert taken == set(forms), mode
        for form, sizes in forms.items():
            assert all(tile(mode, *s) == form for s in sizes), (mode, form)
    f = built_lib.gr_expert_mlp_mxfp4_tile
    taken = {f(T, k, E, H, F) for T in rows for E in (1, 4, 8, 16, 48, 64, 80, 128) for k in (1, 2, 8)
             for H in (512, 1024, 2048, 2560, 4096) for F in (96, 256, 512, 768, 1024, 1536, 2048)}
    assert taken == set(EXPERT_TILES)
    for form, sizes in EXPERT_TILES.items():
        assert all(f(T, k, E, H, F) == form for T, E, k, H, F in sizes), form
