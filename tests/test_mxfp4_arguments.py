"""Arguments that the 4-bit ops refuse before they touch a device: sizes,
types and options are checked ahead of the handles, so these run anywhere."""
import ctypes as C

import pytest

from dragonwing_edge_rs_amd import HipError, ops


class NoBackend:
    handle = None


BE = NoBackend()
BIG = 1 << 33


def refused(match, f, *args, **kw):
    with pytest.raises(HipError, match=match):
        f(BE, *args, **kw)


def test_rows():
    for f in (ops.quantize_mxfp4, ops.dequantize_mxfp4):
        refused("zero size", f, ops.DTYPE_F16, None, None, None, 0, 32)
        refused("zero size", f, ops.DTYPE_F16, None, None, None, 4, 0)
        refused("dtype", f, ops.DTYPE_U8, None, None, None, 4, 32)
        refused("size", f, ops.DTYPE_F16, None, None, None, BIG, 32)
        refused("size", f, ops.DTYPE_F16, None, None, None, 4, BIG)
        refused("null backend", f, ops.DTYPE_F16, None, None, None, 4, 32)


def gemm(m=4, n=4, k=64, a=ops.DTYPE_F16, a_scales=None, c=ops.DTYPE_F16, act=0):
    return (ops.gemm_mxfp4, a, None, a_scales, None, None, None, c, None, m, n, k, act)


class Fake:
    handle = 1  # never read: the refusals below come before


def test_product():
    for sizes in ((0, 4, 64), (4, 0, 64), (4, 4, 0)):
        refused("zero size", *gemm(*sizes))
    for sizes in ((BIG, 4, 64), (4, (1 << 24) + 1, 64), (4, 4, BIG), (4, 4, (1 << 22) + 1)):
        refused("2\\^24", *gemm(*sizes))
    refused("A must be", *gemm(a=ops.DTYPE_F32))
    refused("A must be", *gemm(a=17))
    refused("dtype", *gemm(c=ops.DTYPE_I8))
    refused("activation", *gemm(act=3))
    refused("scales of A", *gemm(a=ops.DTYPE_MXFP4))
    refused("scales of A", *gemm(a_scales=Fake()))
    refused("null backend", *gemm())


def rope(dtype=ops.DTYPE_F16, xs=512, xo=0, ys=512, yo=0, tokens=3, heads=4, dim=128, rotary=128, sections=(24, 20, 20),
         x=None, y=None, **kw):
    return dict(f=ops.rope_axes, args=(dtype, x, xs, xo, y, ys, yo, None, tokens, heads, dim, rotary, sections), kw=kw)


@pytest.mark.parametrize("match,change", [
    ("dtype", dict(dtype=ops.DTYPE_I32)),
    ("zero size", dict(tokens=0)), ("zero size", dict(heads=0)), ("zero size", dict(dim=0)),
    ("zero size", dict(rotary=0)), ("zero size", dict(sections=())),
    ("even", dict(rotary=127)), ("even", dict(rotary=130)),
    ("size", dict(dim=300, rotary=258, xs=1200, ys=1200)), ("size", dict(tokens=1 << 24)),
    ("size", dict(heads=5000)), ("size", dict(sections=(8,) * 9)),
    ("option", dict(order=2)), ("option", dict(pairs=-1)), ("option", dict(freq=7)),
    ("base", dict(base=0.0)), ("base", dict(base=-1.0)), ("base", dict(base=float("nan"))),
    ("base", dict(base=float("inf"))),
    ("add up", dict(sections=(24, 20, 19))), ("add up", dict(sections=(24, 20, 21))),
    ("add up", dict(sections=((1 << 64) - 1, 65, 0))),
    ("do not fit", dict(xs=511)), ("do not fit", dict(xo=1)), ("do not fit", dict(yo=513)),
    ("do not fit", dict(ys=1 << 40)),
    ("null backend", dict()),
])
def test_rope(match, change):
    r = rope(**change)
    refused(match, r["f"], *r["args"], **r["kw"])


@pytest.mark.parametrize("xo,yo,bad", [(0, 0, False), (0, 1, True), (511, 0, True), (512, 0, False), (0, 512, False)])
def test_rope_columns_of_one_buffer(xo, yo, bad):
    b = Fake()
    r = rope(xs=1024, ys=1024, xo=xo, yo=yo, x=b, y=b)
    refused("overlap" if bad else "null backend", r["f"], *r["args"])
    r = rope(xs=1024, ys=1025, x=b, y=b)
    refused("overlap", r["f"], *r["args"])


KV = dict(tokens=3, batch=2, kv_heads=2, head_dim=128, page_size=16, num_pages=5, max_pages=3)


@pytest.mark.parametrize("match,change", [
    ("zero size", dict(tokens=0)), ("zero size", dict(batch=0)), ("zero size", dict(kv_heads=0)),
    ("zero size", dict(num_pages=0)), ("zero size", dict(max_pages=0)),
    ("head_dim", dict(head_dim=96)), ("head_dim", dict(head_dim=0)), ("head_dim", dict(head_dim=512)),
    ("page_size", dict(page_size=8)), ("page_size", dict(page_size=48)), ("page_size", dict(page_size=0)),
    ("page_size", dict(page_size=1 << 17)),
    ("size", dict(tokens=1 << 24)), ("size", dict(batch=65536)), ("size", dict(num_pages=BIG)),
    ("size", dict(max_pages=1 << 24, page_size=256)), ("size", dict(max_pages=BIG)),
    ("null backend", dict()),
])
def test_cache_sizes(match, change):
    s = dict(KV, **change)
    row = s["kv_heads"] * s["head_dim"] or 256
    refused(match, ops.kv_append_mxfp4, None, row, 0, None, row, 0, *[None] * 7, *s.values())
    s = dict(tokens=s.pop("tokens"), batch=s.pop("batch"), heads=4 * max(1, s["kv_heads"]), **s)
    refused(match, ops.attention_mxfp4, None, 4 * row, 0, *[None] * 8, *s.values(), 0.1)


def test_append_columns_and_caches():
    s = KV.values()
    refused("do not fit", ops.kv_append_mxfp4, None, 255, 0, None, 256, 0, *[None] * 7, *s)
    refused("do not fit", ops.kv_append_mxfp4, None, 256, 0, None, 256, 1, *[None] * 7, *s)
    b = Fake()
    refused("share", ops.kv_append_mxfp4, None, 256, 0, None, 256, 0, b, None, b, None, None, None, None, *s)


def attend(heads=4, stride=512, off=0, scale=0.1, causal=True, window=0):
    s = dict(KV)
    return (ops.attention_mxfp4, None, stride, off, *[None] * 8, s["tokens"], s["batch"], heads, s["kv_heads"],
            s["head_dim"], s["page_size"], s["num_pages"], s["max_pages"], scale, causal, window)


def test_attention_options():
    refused("multiple", *attend(heads=3))
    refused("multiple", *attend(heads=0))
    refused("4096", *attend(heads=4098))
    refused("finite", *attend(scale=float("nan")))
    refused("finite", *attend(scale=float("inf")))
    refused("finite", *attend(scale=3e38))
    refused("causal", *attend(causal=2))
    refused("window", *attend(causal=False, window=5))
    refused("do not fit", *attend(stride=511))
    refused("do not fit", *attend(off=1))
    big = dict(KV, tokens=1 << 20, batch=2)
    refused("2\\^24 rows", ops.attention_mxfp4, None, 4096, 0, *[None] * 8, big["tokens"], 2, 32, *list(big.values())[2:],
            0.1)
    refused("2\\^22", ops.attention_mxfp4, None, 1 << 20, 0, *[None] * 8, 4, 60000, 128, *list(big.values())[2:], 0.1)
    refused("null backend", *attend())
