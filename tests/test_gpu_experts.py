"""A mixture of experts (routing, order, products, combination) against its
definitions in 64 bits (tests/experts_reference.py; no reference code exists
for them)."""
import numpy as np
import pytest

import experts_reference as moe
import mxfp4_reference as ref
from dragonwing_edge_rs_amd import HipError, ops

pytestmark = pytest.mark.gpu

F16, F32, MX = ops.DTYPE_F16, ops.DTYPE_F32, ops.DTYPE_MXFP4


def kind_of(dtype):
    return F16 if dtype == np.float16 else F32


# --- routing ---------------------------------------------------------------------------


def run_route(be, x, top, bias=None, sigmoid=False, groups=1, kept=1, best=1, renorm=True, scale=1.0, stride=None, off=0):
    tokens, experts = x.shape
    stride = stride or experts
    wide = np.full((tokens, stride), np.nan, x.dtype)
    wide[:, off:off + experts] = x
    ids = be.from_numpy(np.full((tokens, top), 77, np.int32))
    weights = be.from_numpy(np.full((tokens, top), np.nan, np.float32))
    ops.route_experts(be, kind_of(x.dtype), be.from_numpy(wide), stride, off, None if bias is None else be.from_numpy(bias),
                      ids, weights, tokens, experts, top, score=int(sigmoid), groups=groups, top_groups=kept,
                      group_best=best, renorm=renorm, scale=scale)
    return be.to_numpy(ids, np.int32, (tokens, top)), be.to_numpy(weights, np.float32, (tokens, top))


def check_route(be, x, top, **kw):
    got_ids, got = run_route(be, x, top, **kw)
    kw.pop("stride", None), kw.pop("off", None)
    ids, want, off = moe.route(x, top, **kw)
    np.testing.assert_array_equal(got_ids, ids)
    bad = ~(np.abs(got.astype(np.float64) - want) <= off)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], off[bad][:4])


@pytest.mark.parametrize("experts,top", [(1, 1), (2, 1), (3, 3), (8, 2), (16, 16), (17, 4), (31, 31), (33, 17), (61, 6), (64, 8),
                                         (65, 32), (128, 8), (129, 1), (255, 10), (257, 8), (500, 32), (512, 3), (777, 9),
                                         (1024, 32)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_route(backend, experts, top, dtype):
    rng = np.random.default_rng(experts * 31 + top)
    for tokens in (1, 3, 50):
        x = (rng.normal(0, 2, (tokens, experts)) + rng.normal(0, 1, experts)).astype(dtype)
        bias = rng.normal(0, 0.1, experts).astype(np.float32)
        for sigmoid in (False, True):
            for renorm in (False, True):
                check_route(backend, x, top, sigmoid=sigmoid, renorm=renorm)
                check_route(backend, x, top, sigmoid=sigmoid, renorm=renorm, bias=bias, scale=2.5)


@pytest.mark.parametrize("experts,groups,kept", [(8, 2, 1), (12, 4, 3), (16, 16, 5), (30, 3, 2), (64, 8, 4), (96, 32, 7),
                                                 (256, 8, 4), (256, 64, 20), (510, 17, 3), (1024, 1024, 40),
                                                 (1024, 2, 1)])
def test_route_within_groups(backend, experts, groups, kept):
    rng = np.random.default_rng(experts + groups)
    x = rng.normal(0, 1.5, (37, experts)).astype(np.float32)
    bias = rng.normal(0, 0.05, experts).astype(np.float32)
    top = min(8, kept * (experts // groups))
    for best in (1, 2):
        for sigmoid in (False, True):
            check_route(backend, x, top, sigmoid=sigmoid, groups=groups, kept=kept, best=best)
            check_route(backend, x, top, sigmoid=sigmoid, groups=groups, kept=kept, best=best, bias=bias, renorm=False)
    check_route(backend, x, top, groups=groups, kept=groups, best=2)  # all groups: as without


def test_route_ties_go_to_the_lowest_index(backend):
    rng = np.random.default_rng(3)
    x = rng.integers(-2, 3, (200, 67)).astype(np.float16)
    x[0] = 0
    bias = rng.integers(-1, 2, 67).astype(np.float32) * 0.125
    for sigmoid in (False, True):
        check_route(backend, x, 9, sigmoid=sigmoid)
        check_route(backend, x, 9, sigmoid=sigmoid, bias=bias)
    y = rng.integers(-2, 3, (200, 64)).astype(np.float32)
    y[:, 32:] = y[:, :32]
    for best in (1, 2):
        check_route(backend, y, 9, groups=8, kept=3, best=best)


def test_route_masks_infinities_and_nan(backend):
    rng = np.random.default_rng(4)
    x = rng.normal(0, 2, (64, 40)).astype(np.float32)
    x[0] = -np.inf
    x[1, 1:] = -np.inf
    x[2] = np.nan
    x[3, ::2] = np.nan
    x[4, 5] = np.inf
    x[5, [3, 30]] = np.inf
    x[6] = np.inf
    x[7] = -3e38
    x[8, 0] = 3e38
    x[8, 1] = -3e38
    x[9, :] = np.finfo(np.float32).min
    x[10:20][rng.random((10, 40)) < 0.9] = -np.inf
    x[20:30] = rng.normal(0, 80, (10, 40))
    x[30:34] = rng.normal(-150, 3, (4, 40))  # sigmoids that f32 does not hold
    x[34:38] = rng.normal(60, 3, (4, 40))  # and whose distance from 1 it does not
    bias = rng.normal(0, 0.1, 40).astype(np.float32)
    off = bias.copy()
    off[[0, 7, 8, 20]] = -np.inf, np.nan, np.inf, -1e30
    for sigmoid in (False, True):
        for renorm in (False, True):
            for b in (None, bias, off):
                check_route(backend, x, 6, sigmoid=sigmoid, renorm=renorm, bias=b)
                for best in (1, 2):
                    check_route(backend, x, 6, sigmoid=sigmoid, renorm=renorm, bias=b, groups=8, kept=3, best=best)


def test_route_where_scores_and_biases_nearly_tie(backend):
    # sums that f32 rounds to one value, in an order of their own
    rng = np.random.default_rng(8)
    x = np.full((300, 64), 20.0, np.float32) + rng.integers(0, 40, (300, 64)).astype(np.float32) * 0.25
    bias = rng.integers(0, 3, 64).astype(np.float32)
    check_route(backend, x, 8, sigmoid=True, bias=bias)
    check_route(backend, x, 8, sigmoid=True, bias=bias, groups=8, kept=4, best=2)
    x = rng.normal(0, 1e-6, (300, 64)).astype(np.float32)
    check_route(backend, x, 8, sigmoid=True, bias=bias)
    check_route(backend, x, 8, bias=bias, groups=4, kept=2, best=2)


def test_route_columns_of_wider_rows(backend):
    rng = np.random.default_rng(5)
    for dtype in (np.float16, np.float32):
        x = rng.normal(0, 1, (19, 45)).astype(dtype)
        check_route(backend, x, 4, stride=111, off=33)
        check_route(backend, x, 4, stride=46, off=1)


def test_route_many_tokens(backend):
    rng = np.random.default_rng(6)
    x = rng.normal(0, 1, (5001, 24)).astype(np.float32)
    check_route(backend, x, 3)


# --- order -----------------------------------------------------------------------------


def run_order(be, ids, experts):
    slots = ids.size
    offsets, out = be.from_numpy(np.full(experts + 1, -9, np.int32)), be.from_numpy(np.full(slots, -9, np.int32))
    ops.order_experts(be, be.from_numpy(ids), offsets, out, slots, experts)
    return be.to_numpy(offsets, np.int32, (experts + 1,)), be.to_numpy(out, np.int32, (slots,))


@pytest.mark.parametrize("slots,experts", [(1, 1), (1, 1024), (7, 3), (64, 64), (65, 2), (1023, 1024), (4096, 128), (4097, 17),
                                           (12288, 5), (12289, 300), (16385, 1), (70001, 1024), (300000, 256)])
def test_order(backend, slots, experts):
    rng = np.random.default_rng(slots + experts)
    for case in range(4):
        if case == 0:
            ids = rng.integers(0, experts, slots)
        elif case == 1:  # few experts have nearly all, some slots have none
            ids = np.minimum(rng.geometric(0.4, slots) - 1, experts - 1)
            ids[rng.random(slots) < 0.1] = -1
        elif case == 2:
            ids = np.full(slots, experts - 1)
        else:
            ids = rng.integers(-3, experts + 3, slots)
            ids[rng.random(slots) < 0.05] = -2 ** 31
            ids[rng.random(slots) < 0.05] = 2 ** 31 - 1
        ids = ids.astype(np.int32)
        offsets, out = moe.order(ids, experts)
        got_offsets, got = run_order(backend, ids, experts)
        np.testing.assert_array_equal(got_offsets, offsets)
        np.testing.assert_array_equal(got, out)


def test_order_of_no_experts_at_all(backend):
    for slots in (5, 20000):
        offsets, out = run_order(backend, np.full(slots, -1, np.int32), 9)
        assert (offsets == 0).all() and (out == -1).all()


def test_order_of_most_slots(backend):
    # more than 256 pieces of 4,096
    ids = np.random.default_rng(1).integers(-1, 700, 3000001).astype(np.int32)
    offsets, out = run_order(backend, ids, 700)
    want = np.argsort(np.where(ids < 0, 700, ids), kind="stable").astype(np.int32)
    n = int((ids >= 0).sum())
    np.testing.assert_array_equal(offsets, np.searchsorted(np.sort(ids[ids >= 0]), np.arange(701)).astype(np.int32))
    np.testing.assert_array_equal(out[:n], want[:n])
    assert (out[n:] == -1).all()


# --- products --------------------------------------------------------------------------


class Case:
    """Experts of the given numbers of rows; `none` slots have no expert."""

    def __init__(self, rng, counts, n, k, kind, none=0, gather=0, scatter=False, spread=1.0):
        self.experts, self.n, self.k, self.gather, self.scatter = len(counts), n, k, gather, scatter
        ids = np.concatenate([np.repeat(np.arange(len(counts)), counts), np.full(none, -1)])
        if gather:
            ids = np.concatenate([ids, np.full(-len(ids) % gather, -1)])
        self.ids = rng.permutation(ids).astype(np.int32)
        self.slots = self.ids.size
        self.offsets, self.order = moe.order(self.ids, self.experts)
        nb = ref.blocks(k)
        self.q, self.s = ref.encode(rng.normal(0, 1 / np.sqrt(k), (self.experts * n, k)) *
                                    np.exp(rng.normal(0, spread, (self.experts * n, 1))))
        self.w = ref.decode(self.q, self.s, k).reshape(self.experts, n, k)
        rows = self.slots // gather if gather else self.slots
        self.a = (rng.normal(0, 1, (rows, k)) * np.exp(rng.normal(0, 1, k))).astype(np.float16)
        self.wide = self.a.astype(np.float64)
        if kind == "mxfp4":
            self.a = ref.encode(self.wide)
            self.wide = ref.decode(*self.a, k)
        assert self.q.shape == (self.experts * n, nb * 16)

    def run(self, be, bias, act, dtype, offsets=None, order=None):
        mx = isinstance(self.a, tuple)
        cols = self.n // 2 if act == 3 else self.n
        c = be.from_numpy(np.full((self.slots, cols), 7.5, dtype))
        ops.gemm_mxfp4_experts(be, MX if mx else F16, be.from_numpy(self.a[0] if mx else self.a),
                               be.from_numpy(self.a[1]) if mx else None, be.from_numpy(self.q), be.from_numpy(self.s),
                               None if bias is None else be.from_numpy(bias), kind_of(dtype), c,
                               be.from_numpy(self.offsets if offsets is None else offsets),
                               be.from_numpy(self.order if order is None else order), self.slots, self.experts, self.n,
                               self.k, act=act, gather=self.gather, scatter=self.scatter)
        return be.to_numpy(c, dtype, (self.slots, cols))

    def check(self, be, bias, act, dtype):
        got = self.run(be, bias, act, dtype)
        want, off = moe.products(self.wide, self.w, bias, act, self.offsets, self.order, self.gather, self.scatter, self.slots)
        none = np.isnan(want[:, 0])
        assert none.sum() == self.slots - self.offsets[-1]
        assert (got[none] == 7.5).all()  # left as they were
        e = np.finfo(dtype)
        tol = off + np.abs(want) * float(e.eps) / 2 + float(e.smallest_subnormal) / 2
        bad = ~(np.abs(got.astype(np.float64) - want) <= tol) & ~none[:, None]
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


SHAPES = [
    ([1], 16, 32), ([0, 1, 0], 17, 33), ([2, 0, 3, 1], 6, 31), ([4, 5, 16, 17, 0, 33], 70, 100), ([1] * 70, 18, 64),
    ([16], 130, 1000), ([15, 1, 2], 258, 4096), ([64, 65, 0, 1, 31], 66, 257), ([128, 129, 7], 128, 512),
    ([0] * 66 + [40, 3], 34, 224), ([300, 2, 0, 0, 90], 140, 160), ([513, 100], 260, 288), ([600, 700, 3], 300, 1056),
    ([33] * 12, 48, 2050), ([3, 200] * 5, 64, 96),
]


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_products(backend, shape, kind):
    counts, n, k = SHAPES[shape]
    for i, (none, gather, scatter, use, act, dtype) in enumerate([
            (0, 0, False, False, 0, np.float16), (3, 0, True, True, 1, np.float32), (5, 2, False, True, 2, np.float16),
            (0, 3, True, False, 3, np.float16), (1, 0, False, True, 3, np.float32)]):
        if act == 3 and n % 2:
            act = 2
        rng = np.random.default_rng(shape * 10 + i)
        c = Case(rng, counts, n, k, kind, none, gather, scatter)
        bias = rng.normal(0, 1, (c.experts, n)).astype(dtype) if use else None
        c.check(backend, bias, act, dtype)


LONG = [([513, 300], 260, 1024), ([700, 17, 200], 516, 512), ([400], 300, 2048), ([257, 256, 255], 256, 1536), ([0, 900], 34, 4000)]


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
@pytest.mark.parametrize("shape", range(len(LONG)))
def test_products_of_prompts(backend, shape, kind):
    counts, n, k = LONG[shape]
    for i, (none, gather, scatter, use, act, dtype) in enumerate([
            (0, 2, False, True, 3, np.float16), (5, 0, True, False, 2, np.float32), (0, 0, False, False, 0, np.float16)]):
        rng = np.random.default_rng(500 + shape * 10 + i)
        c = Case(rng, counts, n, k, kind, none, gather, scatter)
        c.check(backend, rng.normal(0, 1, (c.experts, n)).astype(dtype) if use else None, act, dtype)


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
def test_products_of_few_rows_beside_many_take_turns(backend, kind):
    # more pieces of few rows than workgroups that look for them
    rng = np.random.default_rng(18)
    Case(rng, [300, 2, 1, 16], 16390, 96, kind, none=2).check(backend, None, 3, np.float16)


def test_products_of_prompts_with_weights_beyond_f16(backend):
    rng = np.random.default_rng(17)
    for k in (512, 544):
        c = Case(rng, [300, 200], 280, k, "f16", gather=0)
        q, s = c.q.reshape(c.experts, c.n, -1), c.s.reshape(c.experts, c.n, -1)
        s[1, ::3, 1] = 1
        s[1, 270, 9] = 200
        c.w = ref.decode(q, s, c.k)
        c.q, c.s = q.reshape(-1, q.shape[-1]), s.reshape(-1, s.shape[-1])
        c.check(backend, None, 0, np.float32)


def test_products_one_after_the_other_on_two_backends(backend):
    # workspaces that grow while earlier calls are in flight, of two backends on one device
    other, calls = type(backend)(0), []
    try:
        rng = np.random.default_rng(19)
        cases = [Case(rng, counts, 70, k, kind) for counts, k, kind in
                 (([40, 30], 99, "f16"), ([300, 250], 545, "mxfp4"), ([30, 3], 1001, "f16"), ([400, 9], 1130, "f16"))]
        alone = [c.run(backend, None, 0, np.float32) for c in cases]
        for be in (backend, other, backend, other):
            for c, want in zip(cases, alone):
                rows, scales = c.a if isinstance(c.a, tuple) else (c.a, None)
                held = [be.from_numpy(x) for x in (rows, c.q, c.s, c.offsets, c.order)]
                held.append(None if scales is None else be.from_numpy(scales))
                calls.append((be, c, want, held, be.alloc(c.slots * c.n * 4)))
        for be, c, _, (a, w, ws, offsets, order, scales), y in calls:
            ops.gemm_mxfp4_experts(be, F16 if scales is None else MX, a, scales, w, ws, None, F32, y, offsets, order,
                                   c.slots, c.experts, c.n, c.k)
        for be, c, want, _, y in calls:
            np.testing.assert_array_equal(be.to_numpy(y, np.float32, (c.slots, c.n)), want)
    finally:
        for _, _, _, held, y in calls:
            for buffer in (*held, y):
                if buffer is not None:
                    buffer.free()
        other.close()


def test_products_of_more_workgroups_than_a_grid_has_are_refused(backend):
    experts, n, slots = 1024, 1 << 20, 1024
    a, s, c = backend.alloc(slots * 64), backend.alloc(experts * n), backend.alloc(slots * n * 2)
    w, offsets = backend.alloc(experts * n * 16), backend.alloc((experts + 1) * 4)
    with pytest.raises(HipError, match="2\\^32 threads"):
        ops.gemm_mxfp4_experts(backend, F16, a, None, w, s, None, F16, c, offsets, None, slots, experts, n, 32)


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
def test_products_of_many_slots_without_an_expert(backend, kind):
    rng = np.random.default_rng(12)
    for counts in ([0, 0, 0], [0, 5, 0], [0, 40, 0]):
        Case(rng, counts, 96, 128, kind, none=300, gather=4, scatter=False).check(backend, None, 0, np.float16)
        Case(rng, counts, 96, 128, kind, none=300, gather=0, scatter=True).check(backend, None, 3, np.float16)


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
def test_products_of_one_expert_are_the_products(backend, kind):
    # rows in order, one weight matrix: the call without experts, to the last bit where sums are exact
    rng = np.random.default_rng(13)
    for m, n, k in ((3, 40, 100), (16, 33, 64), (70, 130, 288), (200, 140, 999)):
        a, q, s, wide, w, want = ref.whole_product(rng, m, n, k, kind)
        mx = kind == "mxfp4"
        c = backend.alloc(m * n * 4)
        ops.gemm_mxfp4_experts(backend, MX if mx else F16, backend.from_numpy(a[0] if mx else a),
                               backend.from_numpy(a[1]) if mx else None, backend.from_numpy(q), backend.from_numpy(s), None, F32,
                               c, backend.from_numpy(np.array([0, m], np.int32)), None, m, 1, n, k)
        np.testing.assert_array_equal(backend.to_numpy(c, np.float32, (m, n)), want)


def test_products_of_weights_beyond_f16(backend):
    # factors that f16 does not hold take the exact form, in the expert that has them
    rng = np.random.default_rng(14)
    for counts in ([3, 9, 2], [30, 90, 20], [300, 200]):
        c = Case(rng, counts, 48, 160, "f16", gather=0)
        q = c.q.reshape(c.experts, c.n, -1)
        s = c.s.reshape(c.experts, c.n, -1)
        s[1, ::3, 1] = 1
        s[1, 5, 2] = 200
        c.w = ref.decode(q, s, c.k)
        c.q, c.s = q.reshape(-1, q.shape[-1]), s.reshape(-1, s.shape[-1])
        c.check(backend, None, 0, np.float32)


def test_products_read_no_rows_but_their_own(backend):
    # NaN in another expert's weights, in rows of no expert and behind them stays there
    rng = np.random.default_rng(15)
    for counts in ([5, 0, 7], [40, 0, 70], [200, 0, 300]):
        c = Case(rng, counts, 50, 96, "f16", none=9)
        c.s.reshape(c.experts, -1)[1] = 255
        c.a[c.offsets[-1]:] = np.nan
        c.check(backend, None, 0, np.float16)


def test_lists_that_say_otherwise_stay_inside(backend):
    # offsets that descend or pass the slots, orders of other numbers: experts whose lists are sound get their rows
    rng = np.random.default_rng(16)
    for counts in ([5, 6, 7, 3], [60, 50, 40, 30]):
        for kind in ("f16", "mxfp4"):
            c = Case(rng, counts, 64, 128, kind, gather=1)
            want, off = moe.products(c.wide, c.w, None, 0, c.offsets, c.order, 1, False, c.slots)
            bad = c.offsets.copy()
            bad[3], bad[4] = -2 ** 31, 2 ** 31 - 1
            order = c.order.copy()
            order[c.offsets[3]:] = np.resize(np.array([-1, 2 ** 31 - 1, -2 ** 31, c.slots], np.int32), counts[3])
            got = c.run(backend, None, 0, np.float32, offsets=bad, order=order)
            sound = slice(0, c.offsets[2])
            # expert 3 now claims every place from 0 on, so that sound rows may be either's: run only for its bounds
            assert got.shape == want.shape
            got = c.run(backend, None, 0, np.float32, order=order)
            e = np.finfo(np.float32)
            tol = off + np.abs(want) * float(e.eps) / 2 + float(e.smallest_subnormal) / 2
            assert (np.abs(got.astype(np.float64) - want) <= tol)[sound].all()
            c.scatter = True
            c.run(backend, None, 0, np.float32, offsets=bad, order=order)


# --- the weighted sum --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("tokens,top,n", [(1, 1, 1), (1, 8, 7), (3, 2, 33), (50, 4, 256), (7, 32, 1000), (300, 6, 2049),
                                          (2, 3, 40001), (5000, 2, 64)])
def test_combine(backend, tokens, top, n, dtype):
    rng = np.random.default_rng(tokens + top + n)
    ids = rng.integers(-1, 9, (tokens, top)).astype(np.int32)  # -1 and 8: of no expert
    ids[0] = -1
    x = rng.normal(0, 1, (tokens * top, n)).astype(dtype)
    x[(ids.reshape(-1) < 0) | (ids.reshape(-1) >= 8)] = np.nan  # rows that are not read
    weights = rng.normal(0, 1, (tokens, top)).astype(np.float32)
    base = rng.normal(0, 1, (tokens, n)).astype(dtype)
    for b in (None, base):
        y = backend.from_numpy(np.full((tokens, n), np.nan, dtype))
        ops.combine_experts(backend, kind_of(dtype), backend.from_numpy(x), backend.from_numpy(ids),
                            backend.from_numpy(weights), None if b is None else backend.from_numpy(b), y, tokens, top, 8, n)
        got = backend.to_numpy(y, dtype, (tokens, n))
        want, off = moe.combine(x, ids, weights, b, 8)
        e = np.finfo(dtype)
        assert (np.abs(got.astype(np.float64) - want) <= off + np.abs(want) * float(e.eps) / 2 +
                float(e.smallest_subnormal) / 2).all()
    # in place
    y = backend.from_numpy(base)
    ops.combine_experts(backend, kind_of(dtype), backend.from_numpy(x), backend.from_numpy(ids), backend.from_numpy(weights),
                        y, y, tokens, top, 8, n)
    np.testing.assert_array_equal(backend.to_numpy(y, dtype, (tokens, n)), got)


# --- the whole layer -----------------------------------------------------------------------


@pytest.mark.parametrize("tokens,kind", [(1, "f16"), (9, "f16"), (9, "mxfp4"), (200, "f16"), (200, "mxfp4")])
def test_a_layer_of_experts(backend, tokens, kind):
    """Routing, order, two products and the sum, one after the other on the device; padded tokens take no work.  Each
    stage is checked on what the stage before gave."""
    be, experts, top, d, inner = backend, 12, 3, 160, 72
    rng = np.random.default_rng(tokens)
    x = rng.normal(0, 1, (tokens, d)).astype(np.float16)
    logits = rng.normal(0, 1, (tokens, experts)).astype(np.float32)
    logits[tokens // 3::7] = -np.inf
    slots = tokens * top
    w1 = ref.encode(rng.normal(0, 0.1, (experts * 2 * inner, d)))
    w2 = ref.encode(rng.normal(0, 0.1, (experts * d, inner)))
    up = {n: be.from_numpy(v) for n, v in (("x", x), ("logits", logits), ("w1", w1[0]), ("s1", w1[1]), ("w2", w2[0]),
                                           ("s2", w2[1]))}
    ids, weights, offsets, order = be.alloc(slots * 4), be.alloc(slots * 4), be.alloc((experts + 1) * 4), be.alloc(slots * 4)
    h = be.from_numpy(np.zeros((slots, inner), np.float16))
    z = be.from_numpy(np.zeros((slots, d), np.float16))
    y = be.alloc(tokens * d * 2)
    ops.route_experts(be, F32, up["logits"], experts, 0, None, ids, weights, tokens, experts, top)
    ops.order_experts(be, ids, offsets, order, slots, experts)
    if kind == "mxfp4":
        qx, sx = be.alloc(tokens * 5 * 16), be.alloc(tokens * 5)
        ops.quantize_mxfp4(be, F16, up["x"], qx, sx, tokens, d)
        ops.gemm_mxfp4_experts(be, MX, qx, sx, up["w1"], up["s1"], None, F16, h, offsets, order, slots, experts, 2 * inner, d,
                               act=ops.ACT_SWIGLU, gather=top)
        qh, sh = be.alloc(slots * 3 * 16), be.alloc(slots * 3)
        ops.quantize_mxfp4(be, F16, h, qh, sh, slots, inner)
        ops.gemm_mxfp4_experts(be, MX, qh, sh, up["w2"], up["s2"], None, F16, z, offsets, order, slots, experts, d, inner,
                               scatter=True)
    else:
        ops.gemm_mxfp4_experts(be, F16, up["x"], None, up["w1"], up["s1"], None, F16, h, offsets, order, slots, experts,
                               2 * inner, d, act=ops.ACT_SWIGLU, gather=top)
        ops.gemm_mxfp4_experts(be, F16, h, None, up["w2"], up["s2"], None, F16, z, offsets, order, slots, experts, d, inner,
                               scatter=True)
    ops.combine_experts(be, F16, z, ids, weights, up["x"], y, tokens, top, experts, d)

    got = {n: be.to_numpy(b, t, s) for n, b, t, s in (
        ("ids", ids, np.int32, (tokens, top)), ("weights", weights, np.float32, (tokens, top)),
        ("offsets", offsets, np.int32, (experts + 1,)), ("order", order, np.int32, (slots,)),
        ("h", h, np.float16, (slots, inner)), ("z", z, np.float16, (slots, d)), ("y", y, np.float16, (tokens, d)))}

    def near(value, want, off, some=slice(None)):
        tol = off + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        assert (np.abs(value.astype(np.float64) - want) <= tol)[some].all()

    want_ids, want_w, off_w = moe.route(logits, top)
    np.testing.assert_array_equal(got["ids"], want_ids)
    assert (np.abs(got["weights"] - want_w) <= off_w).all()
    want_offsets, want_order = moe.order(want_ids, experts)
    np.testing.assert_array_equal(got["offsets"], want_offsets)
    np.testing.assert_array_equal(got["order"], want_order)
    values = (lambda v: ref.decode(*ref.encode(v), v.shape[1])) if kind == "mxfp4" else (lambda v: v.astype(np.float64))
    n = want_offsets[-1]
    want, off = moe.products(values(x), ref.decode(*w1, d).reshape(experts, 2 * inner, d), None, 3, want_offsets, want_order,
                             top, False, slots)
    near(got["h"], want, off, slice(0, n))
    want, off = moe.products(values(got["h"]), ref.decode(*w2, inner).reshape(experts, d, inner), None, 0, want_offsets,
                             want_order, 0, True, slots)
    near(got["z"], want, off, want_order[:n])
    near(got["y"], *moe.combine(got["z"], got["ids"], got["weights"], x, experts))


# --- refusals that need buffers --------------------------------------------------------------


def test_buffers_of_another_size_or_shared_are_refused(backend):
    be = backend
    logits, ids, weights = be.alloc(4 * 8 * 4), be.alloc(4 * 2 * 4), be.alloc(4 * 2 * 4)

    def route(logits=logits, bias=None, ids=ids, weights=weights, match="mismatch"):
        with pytest.raises(HipError, match=match):
            ops.route_experts(be, F32, logits, 8, 0, bias, ids, weights, 4, 8, 2)

    route(logits=be.alloc(4 * 8 * 4 + 4))
    route(bias=be.alloc(4))
    route(ids=be.alloc(4))
    route(weights=be.alloc(4))
    route(weights=ids, match="overlap")
    route(logits=None, match="null buffer")
    offsets, order = be.alloc(9 * 4), be.alloc(8 * 4)
    for bad in ((be.alloc(4), offsets, order), (ids, be.alloc(4), order), (ids, offsets, be.alloc(4))):
        with pytest.raises(HipError, match="mismatch"):
            ops.order_experts(be, *bad, 8, 8)
    with pytest.raises(HipError, match="overlap"):
        ops.order_experts(be, ids, offsets, ids, 8, 8)

    a, w, s, c = be.alloc(8 * 64 * 2), be.alloc(8 * 16 * 32), be.alloc(8 * 16 * 2), be.alloc(8 * 16 * 2)

    def product(match="mismatch", **kw):
        v = dict(a=a, w=w, s=s, bias=None, c=c, offsets=offsets, order=order, gather=0, act=0)
        v.update(kw)
        with pytest.raises(HipError, match=match):
            ops.gemm_mxfp4_experts(be, F16, v["a"], None, v["w"], v["s"], v["bias"], F16, v["c"], v["offsets"], v["order"], 8, 8,
                                   16, 64, gather=v["gather"], act=v["act"])

    short = be.alloc(4)
    for name in ("a", "w", "s", "bias", "c", "offsets", "order"):
        product(**{name: short})
    product(gather=2)  # A has slots / gather rows then
    product(act=3)  # C half as many columns
    product(c=a, match="mismatch")
    y, x = be.alloc(4 * 16 * 2), be.alloc(8 * 16 * 2)
    with pytest.raises(HipError, match="mismatch"):
        ops.combine_experts(be, F16, x, ids, weights, short, y, 4, 2, 8, 16)
    with pytest.raises(HipError, match="mismatch"):
        ops.combine_experts(be, F16, y, ids, weights, None, y, 4, 2, 8, 16)
    with pytest.raises(HipError, match="an input"):
        ops.combine_experts(be, F32, be.alloc(8), ids8 := be.alloc(8), be.alloc(8), None, ids8, 2, 1, 8, 1)
