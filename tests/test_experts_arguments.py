"""Arguments that the calls of a mixture of experts refuse before they touch a
device: these run anywhere."""
import pytest

from dragonwing_edge_rs_amd import HipError, ops


class NoBackend:
    handle = None


class Fake:
    handle = 1  # never read: the refusals below come before


BE = NoBackend()
BIG = 1 << 40


def refused(match, f, *args, **kw):
    with pytest.raises(HipError, match=match):
        f(BE, *args, **kw)


def route(dtype=ops.DTYPE_F32, stride=64, off=0, tokens=5, experts=64, top_k=4, **kw):
    return (ops.route_experts, dtype, None, stride, off, None, None, None, tokens, experts, top_k), kw


@pytest.mark.parametrize("match,change", [
    ("dtype", dict(dtype=ops.DTYPE_I8)), ("dtype", dict(dtype=ops.DTYPE_MXFP4)),
    ("zero size", dict(tokens=0)), ("zero size", dict(experts=0)), ("zero size", dict(top_k=0)),
    ("1024 experts", dict(experts=1025, stride=2000)), ("2\\^24", dict(tokens=(1 << 24) // 4 + 1)),
    ("2\\^24", dict(tokens=BIG)), ("2\\^24", dict(tokens=(1 << 64) - 1)),
    ("top_k above 32", dict(top_k=33)), ("take part", dict(top_k=5, experts=4)),
    ("take part", dict(groups=8, top_groups=1, top_k=9)),
    ("groups", dict(groups=0)), ("groups", dict(groups=3)), ("groups", dict(groups=4, top_groups=0)),
    ("groups", dict(groups=4, top_groups=5)), ("groups", dict(groups=128)), ("groups", dict(groups=BIG)),
    ("unknown score", dict(score=2)), ("group_best", dict(group_best=0)), ("group_best", dict(group_best=3)),
    ("renorm", dict(renorm=2)), ("scale", dict(scale=float("nan"))), ("scale", dict(scale=float("inf"))),
    ("do not fit", dict(stride=63)), ("do not fit", dict(off=1)), ("do not fit", dict(off=BIG)),
    ("do not fit", dict(stride=(1 << 24) + 1)),
    ("null backend", dict()), ("null backend", dict(groups=8, top_groups=4, group_best=2, top_k=32)),
])
def test_route(match, change):
    args, kw = route(**change)
    refused(match, *args, **kw)


def test_order():
    refused("zero size", ops.order_experts, None, None, None, 0, 8)
    refused("zero size", ops.order_experts, None, None, None, 8, 0)
    refused("2\\^24", ops.order_experts, None, None, None, (1 << 24) + 1, 8)
    refused("1024 experts", ops.order_experts, None, None, None, 8, 1025)
    refused("null backend", ops.order_experts, None, None, None, 1 << 24, 1024)


def product(a=ops.DTYPE_F16, a_scales=None, c=ops.DTYPE_F16, slots=8, experts=4, n=64, k=64, order=Fake(), **kw):
    return (ops.gemm_mxfp4_experts, a, None, a_scales, None, None, None, c, None, None, order, slots, experts, n, k), kw


@pytest.mark.parametrize("match,change", [
    ("A must be", dict(a=ops.DTYPE_F32)), ("dtype", dict(c=ops.DTYPE_I8)), ("activation", dict(act=4)),
    ("activation", dict(act=-1)),
    ("zero size", dict(slots=0)), ("zero size", dict(experts=0)), ("zero size", dict(n=0)), ("zero size", dict(k=0)),
    ("2\\^24", dict(slots=(1 << 24) + 1)), ("1024 experts", dict(experts=1025)), ("2\\^24", dict(n=(1 << 24) + 1)),
    ("2\\^22", dict(k=(1 << 22) + 1)), ("pairs", dict(act=3, n=65)), ("gather must", dict(gather=3)),
    ("gather must", dict(gather=BIG)), ("need the order", dict(gather=2, order=None)),
    ("need the order", dict(scatter=True, order=None)), ("scatter must", dict(scatter=2)),
    ("scales of A", dict(a=ops.DTYPE_MXFP4)), ("scales of A", dict(a_scales=Fake())),
    ("64 GiB", dict(slots=1 << 24, k=1 << 12)), ("64 GiB", dict(slots=1 << 24, k=1 << 14, a=ops.DTYPE_MXFP4, a_scales=Fake())),
    ("null backend", dict(order=None)), ("null backend", dict(act=3, gather=2, scatter=True)),
])
def test_product(match, change):
    args, kw = product(**change)
    refused(match, *args, **kw)


def test_gated_activation_is_the_experts_product_alone():
    refused("activation", ops.gemm_mxfp4, ops.DTYPE_F16, None, None, None, None, None, ops.DTYPE_F16, None, 4, 4, 64,
            act=ops.ACT_SWIGLU)


def test_combine():
    def go(match, dtype=ops.DTYPE_F16, tokens=4, top_k=2, experts=8, n=64):
        refused(match, ops.combine_experts, dtype, None, None, None, None, None, tokens, top_k, experts, n)

    go("dtype", dtype=ops.DTYPE_U8)
    for zero in ("tokens", "top_k", "experts", "n"):
        go("zero size", **{zero: 0})
    go("top_k above", top_k=33)
    go("2\\^24", tokens=(1 << 23) + 1)
    go("2\\^24", tokens=BIG)
    go("1024 experts", experts=1025)
    go("n above", n=(1 << 24) + 1)
    go("null backend")
