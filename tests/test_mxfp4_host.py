"""Argument checks of the 4-bit entry points, without a GPU: the C ones refuse before
any launch, the Python ones before the library."""

import pytest
import torch

from tests.test_experts_host import A, BAD, UNSUPPORTED, call
from vllm_gr_amd import _C, ops


def test_quant_refusals(built_lib):
    base = dict(out=A, ostr=128, scale=A, sstr=8, x=A, xstr=256, T=4, K=256, dtype=2, stream=None)
    f = lambda **o: call(built_lib.gr_quant_mxfp4, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(K=0), dict(dtype=3), dict(dtype=4), dict(out=None), dict(scale=None), dict(x=None),
              dict(ostr=127), dict(xstr=255), dict(sstr=7)):
        assert f(**o) == BAD, o
    for o in (dict(K=240), dict(x=A + 8), dict(xstr=260), dict(dtype=0, xstr=258), dict(out=A + 8), dict(ostr=136),
              dict(T=2 ** 31 - 1), dict(T=2 ** 26)):
        assert f(**o) == UNSUPPORTED, o


def test_dequant_refusals(built_lib):
    base = dict(out=A, ostr=256, x=A, xstr=128, scale=A, sstr=8, T=4, K=256, dtype=2, stream=None)
    f = lambda **o: call(built_lib.gr_dequant_mxfp4, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(K=0), dict(dtype=3), dict(out=None), dict(scale=None), dict(x=None), dict(ostr=255),
              dict(xstr=127), dict(sstr=7)):
        assert f(**o) == BAD, o
    for o in (dict(K=240), dict(x=A + 2), dict(xstr=130), dict(out=A + 8), dict(ostr=260), dict(T=2 ** 26)):
        assert f(**o) == UNSUPPORTED, o


def test_linear_refusals(built_lib):
    base = dict(out=A, ostr=128, os=None, osr=0, x=A, xstr=128, xs=A, xss=8, w=A, wstr=128, ws=A, wss=8, T=4, N=128, K=256,
                swiglu=0, odt=2, stream=None)
    f = lambda **o: call(built_lib.gr_linear_mxfp4, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(N=0), dict(K=0), dict(swiglu=2), dict(odt=3), dict(odt=5), dict(odt=-1), dict(out=None),
              dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(ostr=127), dict(xstr=127), dict(wstr=127),
              dict(xss=7), dict(wss=7), dict(odt=4, ostr=64), dict(odt=4, os=A, osr=3), dict(odt=4, os=A, osr=4, ostr=63)):
        assert f(**o) == BAD, o
    q = dict(odt=4, os=A, osr=4, ostr=64)
    for o in (dict(K=240), dict(swiglu=1, N=120), dict(q, N=112), dict(x=A + 8), dict(w=A + 8), dict(xstr=136),
              dict(wstr=136), dict(out=A + 2), dict(odt=0, out=A + 8), dict(q, out=A + 8), dict(q, ostr=72),
              dict(N=2 ** 28 + 16, ostr=2 ** 28 + 16), dict(T=2 ** 28, N=2 ** 27, ostr=2 ** 27),
              dict(xstr=2 ** 22 + 16), dict(wstr=2 ** 22 + 16)):
        assert f(**o) == UNSUPPORTED, o


def test_expert_mlp_refusals(built_lib):
    size = built_lib.gr_expert_mlp_mxfp4_workspace_size
    need = size(4, 2, 8, 256, 128)
    assert need > 0 and size(0, 2, 8, 256, 128) == 0
    base = dict(out=A, ostr=256, x=A, xstr=256, gu=A, gus=A, dn=A, dns=A, w=A, ids=A, T=4, k=2, E=8, H=256, F=128,
                dtype=2, ws=A, bytes=need, status=None, stream=None)
    f = lambda **o: call(built_lib.gr_expert_mlp_mxfp4, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(k=0), dict(E=0), dict(H=0), dict(F=0), dict(dtype=3), dict(out=None), dict(x=None),
              dict(gu=None), dict(gus=None), dict(dn=None), dict(dns=None), dict(w=None), dict(ids=None), dict(ostr=255),
              dict(xstr=255)):
        assert f(**o) == BAD, o
    for o in (dict(dtype=0), dict(H=240), dict(F=112), dict(E=1025), dict(x=A + 8), dict(xstr=260), dict(gu=A + 8),
              dict(dn=A + 8), dict(out=A + 4), dict(ostr=258), dict(T=2 ** 26, k=2), dict(T=2 ** 22, H=2048, ostr=2048, xstr=2048),
              dict(H=2 ** 21 + 32, xstr=2 ** 22, ostr=2 ** 22), dict(F=2 ** 21 + 32)):
        assert f(**o) == UNSUPPORTED, o
    for o in (dict(ws=None), dict(ws=A + 128), dict(bytes=need - 1)):
        assert f(**o) == _C.GR_ERR_WORKSPACE, o


def test_workspace_holds_every_part(built_lib):
    """The tokens, the sorted rows' gated products and results, for sizes whose bytes pass 32 bits too."""
    for T, k, E, H, F in ((1, 1, 1, 32, 32), (8192, 8, 64, 2048, 768), (65536, 8, 256, 4096, 2048)):
        need = built_lib.gr_expert_mlp_mxfp4_workspace_size(T, k, E, H, F)
        assert need >= T * H * 17 // 32 + T * k * (F * 17 // 32 + 2 * H)


def test_python_refusals():
    x, x4, s = torch.zeros(4, 256), torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 8, dtype=torch.uint8)
    for f in (lambda: ops.quant_mxfp4(x), lambda: ops.dequant_mxfp4(x4, s), lambda: ops.linear_mxfp4(x4, s, x4, s),
              lambda: ops.expert_mlp_mxfp4(x, x4, s, x4, s, x, x)):
        with pytest.raises(ValueError, match="HIP device"):
            f()
