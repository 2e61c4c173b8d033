"""MXFP4 rows, rotary positions and attention over an MXFP4 cache, evaluated
in 64 bits with numpy from their definitions (no code of the backend)."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
VALUES = np.concatenate([GRID, -GRID])


def blocks(k):
    return -(-k // 32)


def encode(x, least=-127):
    """Rows x [rows, k] as (q, scales): from the definition, in f64."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    b = np.zeros((rows, blocks(k) * 32))
    b[:, :k] = x
    b = b.reshape(rows, -1, 32)
    with np.errstate(all="ignore"):
        amax = np.abs(b).max(-1)
        bad = ~np.isfinite(b).all(-1)
        e = np.frexp(np.where(bad | (amax == 0), 1.0, amax))[1] - 3
        e = np.where(amax == 0, least, np.maximum(e, least))
        v = np.where(bad[..., None], 0.0, np.ldexp(np.where(bad[..., None], 0.0, b), -e[..., None]))
    d = np.abs(np.abs(v)[..., None] - GRID)
    # the nearest; of two as near the even code: odd codes lose ties
    code = np.argmin(d + np.where(np.arange(8) % 2 == 1, 1e-13, 0.0), -1).astype(np.uint8)
    code = np.where(np.signbit(v), code | 8, code).astype(np.uint8)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    q = (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(rows, -1)
    return q, np.where(bad, 255, e + 127).astype(np.uint8)


def decode(q, s, k):
    """The f64 values of packed rows [..., blocks * 16]."""
    c = np.stack([q & 15, q >> 4], -1).reshape(q.shape[:-1] + (q.shape[-1] // 16, 32))
    f = np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))
    return (VALUES[c] * f[..., None]).reshape(q.shape[:-1] + (q.shape[-1] * 2,))[..., :k]


def product(a, w, bias=None, act=0):
    """act(a w^T + bias) in f64, and what an f32 evaluation may be off: each of the k + 2 additions rounds by at most
    an ulp (2^-23) of the terms' magnitudes, SiLU's slope is at most 1.1 and its own steps round 8 times."""
    y, size = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    off = (a.shape[1] + 2) * 2.0 ** -23 * size
    if act == 1:
        y = np.maximum(y, 0)
    if act == 2:
        with np.errstate(over="ignore"):
            y = y / (1 + np.exp(-y))
        off = 1.1 * off + 8 * 2.0 ** -24 * np.abs(y)
    return y, off


def pair_axes(sections, order):
    """Axis of each pair and its place among those of its axis."""
    left, out, place = list(sections), [], []
    used = [0] * len(left)
    a = 0
    while any(left):
        while not left[a]:
            a = (a + 1) % len(left)
        out.append(a)
        place.append(used[a])
        used[a] += 1
        left[a] -= 1
        if order:
            a = (a + 1) % len(left)
    return out, place


def rope(x, pos, rotary, sections, order=0, pairs=0, freq=0, base=10000.0):
    """x [tokens, heads, dim] f64, pos [axes, tokens]; angles in 80 bits."""
    half = rotary // 2
    axis, place = pair_axes(sections, order)
    y = x.copy()
    for i in range(half):
        e = np.longdouble(i) / half if freq == 0 else np.longdouble(place[i]) / sections[axis[i]]
        t = pos[axis[i]].astype(np.longdouble) * np.longdouble(base) ** -e
        c, s = np.cos(t).astype(np.float64)[:, None], np.sin(t).astype(np.float64)[:, None]
        a, b = (i, i + half) if pairs == 0 else (2 * i, 2 * i + 1)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


class Cache:
    """Pages of an MXFP4 cache and the lists that go with them: nq new tokens of each sequence and kv keys with them;
    `extra` rows behind the last sequence.  Places that no sequence owns hold NaN scales."""

    def __init__(self, rng, nq, kv, kv_heads, d, page, extra=0, spare=2, values=None):
        self.nq, self.kv, self.h, self.d, self.page = list(nq), list(kv), kv_heads, d, page
        self.batch, self.tokens = len(nq), sum(nq) + extra
        need = [-(-max(n, 0) // page) for n in kv]
        self.max_pages = max(1, max(need))
        self.num_pages = sum(need) + spare
        order = rng.permutation(self.num_pages).astype(np.int32)
        # entries that no token reaches are no pages
        self.table = np.full((self.batch, self.max_pages), np.int32(2 ** 31 - 1))
        self.table[:, 1::2] = -5
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
        self.len = np.array(kv, np.int32)
        shape = (self.num_pages, kv_heads, page)
        self.q, self.s = {}, {}
        for name in "kv":
            x = rng.normal(0, 1, shape + (d,)) * np.exp(rng.normal(0, 0.5, d)) if values is None else values(name, shape)
            q, s = encode(x.reshape(-1, d), -23)
            self.q[name], self.s[name] = q.reshape(shape + (d // 2,)), s.reshape(shape + (d // 32,))
            live = np.zeros(shape[::2], bool)  # [page, slot]
            for b in range(self.batch):
                for j in range(max(0, self.kv[b])):
                    live[self.table[b, j // page], j % page] = True
            self.s[name][~live.repeat(kv_heads, 0).reshape(self.num_pages, kv_heads, page)] = 255

    def rows(self, name, b, h):
        """The f64 values of sequence b's keys or values of head h."""
        j = np.arange(max(0, self.kv[b]))
        p, s = self.table[b, j // self.page], j % self.page
        return decode(self.q[name][p, h, s], self.s[name][p, h, s], self.d)


def attention(q, cache, scale, causal=True, window=0, some=None):
    """y [tokens, heads, d] in f64 (NaN rows where no sequence owns them, and where `some` [tokens, heads] is not), and what the kernel may be off:
    scores are f32 sums of d exact products, p rounds to f16 (2^-11, and 2^-25 absolute), sums of n terms in f32, the
    result to f16."""
    heads, d = q.shape[1], cache.d
    y, off = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    group = heads // cache.h
    for b in range(cache.batch):
        n = max(0, cache.kv[b])
        rows = np.arange(cache.start[b], cache.start[b + 1])
        pos = cache.kv[b] - len(rows) + np.arange(len(rows))
        j = np.arange(n)
        see = np.ones((len(rows), n), bool)
        if causal:
            see = j[None] <= pos[:, None]
            if window:
                see &= j[None] > pos[:, None] - window
        for h in range(heads):
            k, v = cache.rows("k", b, h // group), cache.rows("v", b, h // group)
            x = q[rows, h]
            for i, r in enumerate(rows):
                if some is not None and not some[r, h]:
                    continue
                m = see[i]
                if not m.any():
                    y[r, h], off[r, h] = 0, 0
                    continue
                with np.errstate(invalid="ignore"):
                    s = k[m] @ x[i] * scale
                    e = np.exp(s - s.max())
                    ds = (d + 3) * 2.0 ** -23 * (np.abs(k[m]) @ np.abs(x[i])).max() * abs(scale) + 2.0 ** -22 * (
                        1 + np.abs(s).max())
                    y[r, h] = e @ v[m] / e.sum()
                    mean = e @ np.abs(v[m]) / e.sum()
                    off[r, h] = (mean * (2 * ds + 2.0 ** -11 + (len(s) + 4) * 2.0 ** -23)
                                 + len(s) * 2.0 ** -25 * np.abs(v[m]).max(0) / e.sum()
                                 + 2.0 ** -11 * np.abs(y[r, h]) + 2.0 ** -25)
    return y, off


def whole_product(rng, m, n, k, kind):
    """Rows ("f16" or "mxfp4") and weights without a zero whose products f32 sums exactly in any order (whole numbers of
    1/16 or 1/32, together below 2^24 of them up to k = 33,000): the operands, the weights, and the product."""
    nb = blocks(k)
    codes = rng.integers(1, 8, (n, nb * 32), dtype=np.uint8) | rng.integers(0, 2, (n, nb * 32), dtype=np.uint8) << 3
    codes[:, k:] = 0
    s = rng.integers(124, 128, (n, nb), dtype=np.uint8)
    q = codes[:, 0::2] | codes[:, 1::2] << 4
    w = decode(q, s, k)
    if kind == "f16":
        a = (rng.integers(1, 4, (m, k)) * rng.choice([-1, 1], (m, k))).astype(np.float16)
        wide = a.astype(np.float64)
    else:
        codes = rng.integers(1, 5, (m, nb * 32), dtype=np.uint8) | rng.integers(0, 2, (m, nb * 32), dtype=np.uint8) << 3
        codes[:, k:] = 0
        a = codes[:, 0::2] | codes[:, 1::2] << 4, np.full((m, nb), 127, np.uint8)
        wide = decode(*a, k)
    # f32 holds every sum of them, in any order
    assert np.abs(wide).max() * np.abs(w).max() * k * (16 if kind == "f16" else 32) < 2 ** 24
    return a, q, s, wide, w, wide.astype(np.float32) @ w.astype(np.float32).T
