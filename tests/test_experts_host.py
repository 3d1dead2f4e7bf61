"""Argument checks of the 8-bit products and the experts' layers, without a GPU:
the C entry points refuse before any launch, the Python ones before the library."""

import pytest
import torch

from vllm_gr_amd import _C, ops

A = 0x1000  # a non-null, aligned pointer that is never dereferenced: the checks reject first
BAD, UNSUPPORTED = _C.GR_ERR_INVALID_ARG, _C.GR_ERR_UNSUPPORTED


def call(fn, defaults, **over):
    assert set(over) <= set(defaults)
    return fn(*{**defaults, **over}.values())


def test_quant_refusals(built_lib):
    base = dict(out=A, ostr=256, scale=A, srow=1, sgrp=4, x=A, xstr=256, T=4, K=256, dtype=2, stream=None)
    f = lambda **o: call(built_lib.gr_quant_fp8, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(K=0), dict(dtype=3), dict(out=None), dict(scale=None), dict(x=None), dict(ostr=255),
              dict(xstr=255), dict(srow=-1), dict(sgrp=-1)):
        assert f(**o) == BAD, o
    for o in (dict(K=248), dict(x=A + 2), dict(xstr=257), dict(out=A + 8), dict(ostr=264), dict(T=2 ** 31 - 1)):
        assert f(**o) == UNSUPPORTED, o


def test_linear_refusals(built_lib):
    base = dict(out=A, ostr=128, os=None, osr=0, osg=0, x=A, xstr=256, xs=A, xsr=1, xsg=4, w=A, wstr=256, ws=A, T=4,
                N=128, K=256, swiglu=0, odt=2, stream=None)
    f = lambda **o: call(built_lib.gr_linear_fp8, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(N=0), dict(K=0), dict(swiglu=2), dict(odt=4), dict(odt=-1), dict(out=None), dict(x=None),
              dict(xs=None), dict(w=None), dict(ws=None), dict(ostr=127), dict(xstr=255), dict(wstr=255), dict(xsr=-1),
              dict(xsg=-1), dict(odt=3), dict(odt=3, os=A, osr=-1)):
        assert f(**o) == BAD, o
    for o in (dict(K=248), dict(swiglu=1, N=120), dict(odt=3, os=A, N=100), dict(x=A + 8), dict(w=A + 8),
              dict(xstr=264), dict(wstr=264), dict(out=A + 2), dict(odt=0, out=A + 8), dict(odt=3, os=A, ostr=130),
              dict(xs=A + 2), dict(ws=A + 1), dict(N=2 ** 28 + 16, ostr=2 ** 28 + 16),
              dict(T=2 ** 28, N=2 ** 27, ostr=2 ** 27), dict(xstr=2 ** 22 + 16), dict(wstr=2 ** 22 + 16)):
        assert f(**o) == UNSUPPORTED, o


def test_route_refusals(built_lib):
    base = dict(w=A, ids=A, logits=A, stride=64, bias=None, T=4, E=64, k=8, score=0, groups=1, top=1, renorm=1,
                scale=1.0, dtype=0, stream=None)
    f = lambda **o: call(built_lib.gr_route_experts, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(E=0), dict(k=0), dict(k=65), dict(groups=0), dict(groups=5), dict(groups=4, top=5),
              dict(top=0), dict(groups=16, top=1, k=5), dict(score=2), dict(dtype=3), dict(w=None), dict(ids=None),
              dict(logits=None), dict(stride=63)):
        assert f(**o) == BAD, o
    for o in (dict(E=1025, stride=1025), dict(E=1024, stride=1024, k=65), dict(E=1000, stride=1000, groups=100, top=50)):
        assert f(**o) == UNSUPPORTED, o


def test_expert_mlp_refusals(built_lib):
    need = built_lib.gr_expert_mlp_workspace_size(4, 2, 8, 256, 128, 0)
    assert need > 0 and built_lib.gr_expert_mlp_workspace_size(0, 2, 8, 256, 128, 0) == 0
    base = dict(out=A, ostr=256, x=A, xstr=256, gu=A, gus=None, dn=A, dns=None, w=A, ids=A, T=4, k=2, E=8, H=256, F=128,
                dtype=2, ws=A, bytes=need, status=None, stream=None)
    f = lambda **o: call(built_lib.gr_expert_mlp, base, **o)
    assert f(T=0) == _C.GR_OK
    for o in (dict(T=-1), dict(k=0), dict(E=0), dict(H=0), dict(F=0), dict(dtype=3), dict(out=None), dict(x=None),
              dict(gu=None), dict(dn=None), dict(w=None), dict(ids=None), dict(ostr=255), dict(xstr=255), dict(gus=A),
              dict(dns=A)):
        assert f(**o) == BAD, o
    for o in (dict(dtype=0), dict(H=248), dict(F=120), dict(E=1025), dict(x=A + 8), dict(xstr=260), dict(gu=A + 8),
              dict(dn=A + 8), dict(out=A + 4), dict(ostr=258), dict(T=2 ** 26, k=2), dict(gus=A + 2, dns=A),
              dict(T=2 ** 19, xstr=2048), dict(H=2 ** 21 + 16, xstr=2 ** 22, ostr=2 ** 22), dict(F=2 ** 21 + 16)):
        assert f(**o) == UNSUPPORTED, o
    for o in (dict(ws=None), dict(ws=A + 128), dict(bytes=need - 1)):
        assert f(**o) == _C.GR_ERR_WORKSPACE, o


def test_workspace_holds_every_part(built_lib):
    """At least the sorted rows' two intermediate results, for sizes whose bytes pass 32 bits too."""
    size = built_lib.gr_expert_mlp_workspace_size
    for T, k, E, H, F in ((1, 1, 1, 16, 16), (8192, 8, 64, 2048, 768), (65536, 8, 256, 4096, 2048)):
        assert size(T, k, E, H, F, 0) >= T * k * (2 * F + 4 * H)
        assert size(T, k, E, H, F, 1) >= T * k * (F + 4 * H) + T * H


def test_python_refusals():
    x = torch.zeros(4, 256)
    for f in (lambda: ops.quant_fp8(x), lambda: ops.route_experts(x, 2),
              lambda: ops.linear_fp8(x, x, x, x), lambda: ops.expert_mlp(x, x, x, x, x)):
        with pytest.raises(ValueError, match="HIP device"):
            f()
