"""Sizes whose launches would count more threads than 32 bits hold are refused before
any launch, and a scale's stride that the product's kernel would cut off."""

from tests.test_experts_host import A, UNSUPPORTED, call


def test_quant_limits(built_lib):
    base = dict(out=A, ostr=2 ** 17, scale=A, srow=1, sgrp=4, x=A, xstr=2 ** 17, T=2 ** 18 + 1, K=2 ** 17, dtype=2,
                stream=None)
    assert call(built_lib.gr_quant_fp8, base) == UNSUPPORTED


def test_linear_limits(built_lib):
    base = dict(out=A, ostr=2 ** 20, os=None, osr=0, osg=0, x=A, xstr=256, xs=A, xsr=1, xsg=4, w=A, wstr=256, ws=A,
                T=2 ** 15, N=2 ** 20, K=256, swiglu=0, odt=2, stream=None)
    assert call(built_lib.gr_linear_fp8, base) == UNSUPPORTED
    assert call(built_lib.gr_linear_fp8, base, T=4, xsg=2 ** 31) == UNSUPPORTED


def test_route_limits(built_lib):
    base = dict(w=A, ids=A, logits=A, stride=1024, bias=None, T=2 ** 28 + 1, E=8, k=8, score=0, groups=1, top=1, renorm=1,
                scale=1.0, dtype=0, stream=None)
    assert call(built_lib.gr_route_experts, base) == UNSUPPORTED
    assert call(built_lib.gr_route_experts, base, T=2 ** 24 + 1, E=1024) == UNSUPPORTED
    assert call(built_lib.gr_route_experts, base, T=2 ** 26, E=257) == UNSUPPORTED


def test_expert_mlp_limits(built_lib):
    base = dict(out=A, ostr=16, x=A, xstr=16, gu=A, gus=None, dn=A, dns=None, w=A, ids=A, T=2 ** 23, k=1, E=8, H=16,
                F=16, dtype=2, ws=A, wsb=2 ** 62, status=None, stream=None)
    assert call(built_lib.gr_expert_mlp, base) == UNSUPPORTED
    big = dict(T=2 ** 12, k=64, ostr=2 ** 16, xstr=2 ** 16, H=2 ** 16, F=2 ** 21)
    assert call(built_lib.gr_expert_mlp, base, **big) == UNSUPPORTED
