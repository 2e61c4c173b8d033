"""Experts' products whose lists overlap or name no rows, and operands that are
one buffer."""
import numpy as np
import pytest

import experts_reference as moe
from dragonwing_edge_rs_amd import HipError, ops
from test_gpu_experts import Case

pytestmark = pytest.mark.gpu

F16, F32, MX = ops.DTYPE_F16, ops.DTYPE_F32, ops.DTYPE_MXFP4
LEFT = np.float32(7.5)  # what C holds before the call


def of_each(c, rows):
    """The product of each place's row with each expert's weights, and what it may be off: [experts, places, n]."""
    both = [moe.product(c.wide[rows], c.w[e], None, 0) for e in range(c.experts)]
    return np.stack([y for y, _ in both]), np.stack([off for _, off in both])


def within(got, want, off):
    e = np.finfo(np.float32)
    tol = off + np.abs(want) * float(e.eps) / 2 + float(e.smallest_subnormal) / 2
    return np.abs(got.astype(np.float64) - want) <= tol


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("counts", [[5, 6, 7, 3], [16, 9, 12, 16], [60, 50, 40, 30], [90, 150, 200, 130], [300, 40, 500, 250]])
def test_rows_of_lists_that_overlap(backend, counts, kind):
    # the last expert's places are all of the buffer's, beside the others' own, and the one ahead of it has none: an
    # element is that of one of its row's claimants, or as it was
    rng = np.random.default_rng(sum(counts))
    c = Case(rng, counts, 64, 128, kind, gather=1)
    offsets = c.offsets.copy()
    offsets[3], offsets[4] = -2 ** 31, 2 ** 31 - 1
    order = c.order.copy()
    no_place = np.array([-1, 2 ** 31 - 1, -2 ** 31, c.slots], np.int32)
    order[c.offsets[3]:] = np.resize(no_place, counts[3])
    named = (order >= 0) & (order < c.slots)
    want, off = of_each(c, np.where(named, order, 0))  # entries that name no slot take A's first row
    place = np.arange(c.slots)
    claims = np.stack([(offsets[e] <= place) & (place < offsets[e + 1]) for e in range(c.experts)])
    assert claims[3].all() and not claims[2].any()
    got = c.run(backend, None, 0, np.float32, offsets=offsets, order=order)
    fits = np.stack([within(got, want[e], off[e]) for e in range(c.experts)])
    assert ((fits & claims[..., None]).any(0) | (got == LEFT)).all()

    c.scatter = True
    got = c.run(backend, None, 0, np.float32, offsets=offsets, order=order)
    rest = np.setdiff1d(place, order[named])
    assert len(rest) == counts[3]
    assert (got[rest] == LEFT).all()  # no entry names them
    at = order[named]
    fits = np.stack([within(got[at], want[e][named], off[e][named]) for e in range(c.experts)])
    assert ((fits & claims[:, named, None]).any(0) | (got[at] == LEFT)).all()


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("slots", [12, 200, 900])
def test_lists_that_all_descend_have_no_rows(backend, kind, slots):
    rng = np.random.default_rng(slots)
    c = Case(rng, [slots // 2, slots - slots // 2], 64, 128, kind)
    for offsets in ([slots, slots // 2, 0], [2 ** 31 - 1, slots, -2 ** 31], [-5, -2, -1], [slots, slots + 1, 2 ** 31 - 1]):
        got = c.run(backend, None, 0, np.float32, offsets=np.array(offsets, np.int32))
        assert (got == LEFT).all()


def test_outputs_that_are_operands_are_refused(backend):
    # sizes at which the operands have C's number of bytes, so that only their being one buffer is wrong
    be = backend

    def refused(a_dtype, size, c_dtype=F16, slots=8, experts=1, n=64, k=64, **same):
        buffers = {name: None if bytes_ is None else be.alloc(bytes_) for name, bytes_ in size.items()}
        buffers["c"] = buffers[same["c"]]
        with pytest.raises(HipError, match="C is an operand"):
            ops.gemm_mxfp4_experts(be, a_dtype, buffers["a"], buffers["as"], buffers["w"], buffers["ws"], buffers["bias"],
                                   c_dtype, buffers["c"], buffers["offsets"], buffers["order"], slots, experts, n, k)

    def sizes(a_dtype, slots, experts, n, k, es):
        blocks, mx = -(-k // 32), a_dtype == MX
        return {"a": slots * blocks * 16 if mx else slots * k * 2, "as": slots * blocks if mx else None,
                "w": experts * n * blocks * 16, "ws": experts * n * blocks, "bias": experts * n * es,
                "offsets": (experts + 1) * 4, "order": slots * 4}

    for name, a_dtype, c_dtype, slots, experts, n, k in (
            ("a", F16, F16, 8, 1, 64, 64), ("a", MX, F16, 8, 1, 16, 64), ("as", MX, F16, 8, 1, 1, 64),
            ("w", F16, F16, 16, 1, 64, 64), ("ws", F16, F16, 1, 1, 64, 64), ("bias", F16, F32, 3, 3, 64, 64),
            ("offsets", F16, F32, 4, 3, 1, 64), ("order", F16, F32, 5, 2, 1, 64)):
        es = 2 if c_dtype == F16 else 4
        size = sizes(a_dtype, slots, experts, n, k, es)
        assert size[name] == slots * n * es, name
        refused(a_dtype, size, c_dtype, slots, experts, n, k, c=name)


def test_outputs_that_are_inputs_are_refused(backend):
    be = backend

    def route(match, tokens, experts, top, ids, weights, logits=None, bias=None):
        with pytest.raises(HipError, match=match):
            ops.route_experts(be, F32, logits or be.alloc(tokens * experts * 4), experts, 0, bias, ids, weights, tokens, experts,
                              top)

    one, other = be.alloc(4 * 4 * 4), be.alloc(4 * 4 * 4)
    route("overlap", 4, 4, 4, one, other, logits=one)
    route("overlap", 4, 4, 4, one, other, logits=other)
    row, rest = be.alloc(4 * 4), be.alloc(4 * 4)
    route("overlap", 1, 4, 4, row, rest, bias=row)
    route("overlap", 1, 4, 4, row, rest, bias=rest)
    ids, lists = be.alloc(4 * 4), be.alloc(4 * 4)
    for same in ((ids, ids, lists), (ids, lists, ids), (ids, lists, lists)):
        with pytest.raises(HipError, match="overlap"):
            ops.order_experts(be, *same, 4, 3)
    x, y = be.alloc(4 * 4), be.alloc(4 * 4)
    for k in ("x", "ids", "weights"):
        v = {"x": x, "ids": ids, "weights": lists, k: y}
        with pytest.raises(HipError, match="an input"):
            ops.combine_experts(be, F32, v["x"], v["ids"], v["weights"], None, y, 4, 1, 8, 1)
