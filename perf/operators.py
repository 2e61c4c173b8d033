"""Operators of language-model layers on this backend, as timed cases.

Each case is one pass through an operator of the layer around a model's
4-bit products, as a serving program calls it on device buffers:

* ``quantize``  rows to MXFP4 (blocks of 32 with a shared power of two) and
                their values back, as a program rounds activations or checks
                weights it has quantized;
* ``product``   rows times MXFP4 weights, the rows in f16 or MXFP4
                themselves, with an optional bias and activation;
* ``rope``      rotary positions over several axes on the heads of a row;
* ``append``    new keys and values into the pages of an MXFP4 cache, and the
                cache's values read back;
* ``attend``    attention of one or many new tokens a sequence over such a
                cache.

With ``own`` false ``run`` computes the operators from elementary torch
operations in f32; with ``own`` true it calls this backend's op functions.
"""
import math

import torch

own = False  # True: run() calls this backend's op functions

BLOCK = 32  # elements that share a scale
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # The activations of a decoding batch before a 4-bit product.
        {"name": "quantize_tokens", "kind": "quantize", "dtype": "f16", "rows": 32, "k": 8192},
        # A whole weight matrix, its row length no multiple of the block.
        {"name": "quantize_weights", "kind": "quantize", "dtype": "f32", "rows": 8191, "k": 4099},
        # One token through a wide layer: the weights' bytes are everything.
        {"name": "product_token", "kind": "product", "a": "f16", "m": 1, "n": 14336, "k": 4096, "bias": False,
         "act": 0},
        # A prompt through a layer with f16 activations.
        {"name": "product_prompt", "kind": "product", "a": "f16", "m": 2048, "n": 8192, "k": 4096, "bias": True,
         "act": 2},
        # A decoding batch with 4-bit activations, odd sizes throughout.
        {"name": "product_mx_batch", "kind": "product", "a": "mxfp4", "m": 51, "n": 8190, "k": 8176, "bias": True,
         "act": 0},
        # A long prompt with 4-bit activations: the matrix cores' case.
        {"name": "product_mx_prompt", "kind": "product", "a": "mxfp4", "m": 4096, "n": 8192, "k": 8192,
         "bias": False, "act": 0},
        # Queries and keys of a decoding batch, three axes in contiguous sections.
        {"name": "rope_batch", "kind": "rope", "dtype": "f16", "tokens": 24, "heads": 40, "dim": 128, "rotary": 128,
         "axes": 3, "order": 0, "pairs": 0, "freq": 0},
        # A video's tokens through an image encoder: f32, part of each head, frequencies of each axis its own.
        {"name": "rope_video", "kind": "rope", "dtype": "f32", "tokens": 12289, "heads": 24, "dim": 80, "rotary": 72,
         "axes": 3, "order": 0, "pairs": 1, "freq": 1},
        # One new token for each of many sequences.
        {"name": "append_batch", "kind": "append", "batch": 64, "most_q": 1, "most_kv": 256, "kv_heads": 8,
         "dim": 128, "page": 16},
        # Prompts of ragged lengths.
        {"name": "append_prompt", "kind": "append", "batch": 3, "most_q": 4096, "most_kv": 4096, "kv_heads": 8,
         "dim": 128, "page": 64},
        # Decoding: ragged sequences, the longest with tens of thousands of keys.
        {"name": "attend_tokens", "kind": "attend", "batch": 16, "most_q": 1, "most_kv": 65536, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "causal": True, "window": 0},
        # Prompts after cached prefixes: causal, many queries.
        {"name": "attend_prompt", "kind": "attend", "batch": 2, "most_q": 1536, "most_kv": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "window": 0},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(max(round(v / step) * step, -(-lo // step) * step), hi // step * step))


def draw(rng):
    kind = rng.choice(("quantize", "product", "product", "rope", "append", "attend", "attend"))
    if kind == "quantize":
        k = _log_int(rng, 16, 16384, rng.choice((1, 8, 32)))
        return {"kind": kind, "dtype": rng.choice(("f16", "f32")), "rows": _log_int(rng, 1, max(1, 30000000 // k)),
                "k": k}
    if kind == "product":
        a = rng.choice(("f16", "mxfp4"))
        n, k = _log_int(rng, 256, 14336, rng.choice((1, 16))), _log_int(rng, 128, 14336, rng.choice((1, 8, 32)))
        most = 68e9 if a == "f16" else 270e9
        m = _log_int(rng, 1, max(1, min(4096, int(most / (n * k)))))
        return {"kind": kind, "a": a, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5, "act": rng.choice((0, 0, 2))}
    if kind == "rope":
        dim = rng.choice((64, 80, 96, 128, 256))
        axes = rng.choice((1, 2, 3, 4))
        heads = _log_int(rng, 2, 48)
        return {"kind": kind, "dtype": rng.choice(("f16", "f32")),
                "tokens": _log_int(rng, 1, 23000000 // (heads * dim)), "heads": heads, "dim": dim,
                "rotary": rng.choice((dim, dim // 2)), "axes": axes, "order": rng.choice((0, 1)),
                "pairs": rng.choice((0, 1)), "freq": rng.choice((0, 1))}
    kv_heads, dim, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 256)), rng.choice((16, 32, 64, 256))
    if kind == "append":
        most = 12500000 // (kv_heads * dim)
        kv = _log_int(rng, 16, min(8192, most))
        return {"kind": kind, "batch": _log_int(rng, 1, max(1, min(64, most // kv))),
                "most_q": rng.choice((1, 1, _log_int(rng, 2, kv))), "most_kv": kv, "kv_heads": kv_heads, "dim": dim,
                "page": page}
    causal = rng.random() < 0.8
    c = {"kind": kind, "heads": kv_heads * rng.choice((1, 2, 4, 7, 8)), "kv_heads": kv_heads, "dim": dim,
         "page": page, "causal": causal, "window": rng.choice((0, 0, 1000)) if causal else 0}
    if rng.random() < 0.6:
        kv = _log_int(rng, 16, min(65536, 67000000 // (kv_heads * dim)))
        return dict(c, batch=_log_int(rng, 1, max(1, min(64, 67000000 // (kv_heads * dim * kv)))),
                    most_q=rng.choice((1, 1, 1, 4)), most_kv=kv)
    kv = _log_int(rng, 128, 4096)
    q = _log_int(rng, 16, min(kv, max(16, int(4e8 / (kv * c["heads"] * dim / 128)))))
    return dict(c, batch=_log_int(rng, 1, max(1, min(8, int(4e8 / (q * kv * c["heads"] * dim / 128))))), most_q=q,
                most_kv=kv)


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------

_TYPES = {"f32": torch.float32, "f16": torch.float16}
_STR = {torch.float32: "<f4", torch.float16: "<f2", torch.uint8: "|u1", torch.int32: "<i4"}
_at = {}


def _backend():
    """The package's backend on the device, made by the first call."""
    if not _at:
        import __graft_entry__

        __graft_entry__.import_pkg()
        import dragonwing_edge_rs_amd as dw
        from dragonwing_edge_rs_amd import ops

        _at.update(be=dw.Backend(0), ops=ops)
    return _at["be"], _at["ops"]


class _Span:
    """A backend buffer as the CUDA array interface shows it to torch."""

    def __init__(self, buf, shape, typestr):
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "version": 2,
                                         "data": (buf.device_ptr(), False), "strides": None}


def _hold(st):
    """The tensors of a state as a program of this backend holds them: each in a buffer of the backend, beside a
    torch view of it.  Without the backend they stay what they are."""
    if own:
        be, _ = _backend()
        st["buf"] = {}
        for name in [n for n, v in st.items() if isinstance(v, torch.Tensor)]:
            t = st[name]
            buf = be.alloc(t.numel() * t.element_size())
            view = torch.as_tensor(_Span(buf, t.shape, _STR[t.dtype]), device="cuda")
            view.copy_(t)
            st["buf"][name], st[name] = buf, view
        torch.cuda.synchronize()  # the backend's stream is its own
    return st


def _gen(seed):
    return torch.Generator("cuda").manual_seed(int(seed))


def _normal(g, shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _tokens(g, shape, dtype=torch.float16):
    """Activations: of order one, some channels far larger than the others."""
    ch = torch.exp(torch.randn(shape[-1], generator=g, device="cuda") * 0.7)
    return (torch.randn(shape, generator=g, device="cuda") * ch).to(dtype)


def _lengths(case):
    """Ragged lengths on the host, the same for every seed (outputs keep their shapes): new tokens of each sequence,
    and its keys with them.  The first sequence has the most of both; the others are spread over the logarithm of the
    range."""
    r = torch.Generator().manual_seed(77 + case["batch"])
    b, mq, mk = case["batch"], case["most_q"], case["most_kv"]
    u, v = torch.rand(b, generator=r).tolist(), torch.rand(b, generator=r).tolist()
    nq = [max(1, round(mq ** (0.5 + 0.5 * x))) for x in u]
    kv = [max(n, round(mk ** (0.4 + 0.6 * x))) for n, x in zip(nq, v)]
    nq[0], kv[0] = mq, max(mq, mk)
    return nq, kv


def _pages(case, g):
    """Lengths, block table (pages in random order) and the sizes of the cache."""
    nq, kv = _lengths(case)
    each = [-(-n // case["page"]) for n in kv]
    total, most = sum(each), max(each)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["batch"], most), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(each):
        table[b, :n] = order[at:at + n]
        at += n
    start = [0]
    for n in nq:
        start.append(start[-1] + n)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"nq": nq, "kv": kv, "total": total, "most": most, "tokens": start[-1], "table": table,
            "start": ints(start), "len": ints(kv)}


def _cache(g, total, case):
    """Pages that hold keys or values of order one, as packed bytes and scales."""
    shape = (total, case["kv_heads"], case["page"], case["dim"])
    q, s = _pack(_tokens(g, shape, torch.float32).reshape(-1, case["dim"]))
    return q.reshape(shape[:3] + (-1,)), s.reshape(shape[:3] + (-1,))


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    st = {"case": case}
    if kind == "quantize":
        dt, shape = _TYPES[case["dtype"]], (case["rows"], case["k"])
        st["x"] = _tokens(g, shape, dt)
        blocks = -(-case["k"] // BLOCK)
        st["q"] = torch.zeros((case["rows"], blocks * 16), dtype=torch.uint8, device="cuda")
        st["s"] = torch.zeros((case["rows"], blocks), dtype=torch.uint8, device="cuda")
        st["y"] = torch.zeros(shape, dtype=dt, device="cuda")
    elif kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = _tokens(g, (m, k))
        st["w"], st["ws"] = _pack(_normal(g, (n, k), 1.0 / math.sqrt(k)))
        if case["a"] == "f16":
            st["a"] = a
        else:
            st["a"], st["as"] = _pack(a.float())
        if case["bias"]:
            st["bias"] = _normal(g, (n,), 0.5, torch.float16)
        st["y"] = torch.zeros((m, n), dtype=torch.float16, device="cuda")
    elif kind == "rope":
        dt, shape = _TYPES[case["dtype"]], (case["tokens"], case["heads"], case["dim"])
        st["x"] = _tokens(g, shape, dt)
        # a time axis that reaches far, and places within a frame
        st["pos"] = torch.stack([torch.randint(0, 500000 if i == 0 else 200, (case["tokens"],), generator=g,
                                               device="cuda", dtype=torch.int32) for i in range(case["axes"])])
        st["y"] = torch.zeros(shape, dtype=dt, device="cuda")
    else:
        p = _pages(case, g)
        st.update(p)
        st["kc"], st["ks"] = _cache(g, p["total"], case)
        st["vc"], st["vs"] = _cache(g, p["total"], case)
        if kind == "append":
            st["qkv"] = _tokens(g, (p["tokens"], 2 * case["kv_heads"] * case["dim"]))
            shape = st["kc"].shape[:3] + (case["dim"],)
            st["yk"], st["yv"] = (torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2))
        else:
            # queries in the rows of a fused projection, keys and values of the step beside them
            st["qkv"] = _normal(g, (p["tokens"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]), 1.0,
                                torch.float16)
            st["y"] = torch.zeros((p["tokens"], case["heads"], case["dim"]), dtype=torch.float16, device="cuda")
    return _hold(st)


def _sections(case):
    """Pairs of each axis: an even split, the rest to the first axes."""
    half = case["rotary"] // 2
    return [half // case["axes"] + (i < half % case["axes"]) for i in range(case["axes"])]


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------


def _power(e):
    """2^e in f32 for whole e in [-126, 127]."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _blocks(x):
    """Rows as blocks of 32, zeros behind the end."""
    r, k = x.shape
    pad = -k % BLOCK
    x = torch.nn.functional.pad(x, (0, pad)) if pad else x
    return x.reshape(r, -1, BLOCK)


def _codes(x, least=-127):
    """Block exponents and elements (on the grid, in units of the block's power of two) of f32 rows."""
    b = _blocks(x)
    amax = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(amax).exponent - 3).clamp(least, 127)
    e = torch.where(amax == 0, torch.full_like(e, least), e)
    v = b * _power(-e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return e.squeeze(-1), torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)


def _pack(x, least=-127):
    """f32 rows as MXFP4: two elements a byte, the first in the low half, and a scale byte for each block."""
    e, v = _codes(x, least)
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(v).to(torch.uint8) << 3)
    q = code[..., 0::2] | (code[..., 1::2] << 4)
    return q.reshape(x.shape[0], -1).contiguous(), (e + 127).to(torch.uint8).contiguous()


def _values(q, s, k):
    """The f32 values of packed rows (any leading shape)."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float32, device=q.device)
    v = torch.stack([grid[(q & 15).int()], grid[(q >> 4).int()]], -1).reshape(q.shape[:-1] + (-1, BLOCK))
    v = v * _power(s.int() - 127).unsqueeze(-1)
    return v.reshape(q.shape[:-1] + (-1,))[..., :k]


def _plain_product(st):
    c = st["case"]
    a = st["a"].float() if c["a"] == "f16" else _values(st["a"], st["as"], c["k"])
    y = a @ _values(st["w"], st["ws"], c["k"]).t()
    if c["bias"]:
        y = y + st["bias"].float()
    if c["act"] == 2:
        y = y / (1 + torch.exp(-y))
    return y.half()


def _axis_of_pair(case):
    """For each pair of a head, its axis and its place within the axis."""
    sections = _sections(case)
    if case["order"] == 0:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    else:
        axis = sorted(((j, a) for a, n in enumerate(sections) for j in range(n)))
        axis = [a for _, a in axis]
    place = [axis[:i].count(a) for i, a in enumerate(axis)]
    return axis, place, [sections[a] for a in axis]


def _plain_rope(st, wide=torch.float32):
    c, half = st["case"], st["case"]["rotary"] // 2
    axis, place, size = (torch.tensor(v, device="cuda") for v in _axis_of_pair(c))
    i = torch.arange(half, device="cuda", dtype=torch.float64)
    power = i / half if c["freq"] == 0 else place.double() / size
    angle = st["pos"].double()[axis].t() * torch.exp(-power * math.log(10000.0))  # far positions: in 64 bits
    cos, sin = (f(angle).to(wide).unsqueeze(1) for f in (torch.cos, torch.sin))
    x = st["x"].to(wide)
    r = x[..., :c["rotary"]]
    if c["pairs"] == 0:
        a, b = r[..., :half], r[..., half:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([r, x[..., c["rotary"]:]], -1).to(st["x"].dtype)


def _places(st):
    """For each new token its sequence and its place there."""
    t = torch.arange(st["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["start"], t, right=True) - 1
    ends, lens = st["start"][seq + 1], st["len"][seq]
    return seq, lens - ends + t


def _plain_append(st):
    """The values of the cache with the new tokens' keys and values in it."""
    c = st["case"]
    h, d, ps = c["kv_heads"], c["dim"], c["page"]
    seq, pos = _places(st)
    page, slot = st["table"][seq, (pos // ps).long()].long(), (pos % ps).long()
    rows = st["qkv"].float().reshape(-1, 2, h, d)
    out = []
    for j, (q, s) in enumerate(((st["kc"], st["ks"]), (st["vc"], st["vs"]))):
        y = _values(q, s, d)
        e, v = _codes(rows[:, j].reshape(-1, d), -23)
        y[page, :, slot] = (v * _power(e).unsqueeze(-1)).reshape(-1, h, d)
        out.append(y.half())
    return {"k": out[0], "v": out[1]}


def _plain_attend(st):
    """All sequences at once, padded to the longest."""
    c = st["case"]
    b, h, d, ps, group = c["batch"], c["kv_heads"], c["dim"], c["page"], c["heads"] // c["kv_heads"]
    nq, nk = max(st["nq"]), st["most"] * ps
    table = st["table"].long()
    k, v = (_values(q[table].transpose(1, 2).reshape(b, h, nk, -1), s[table].transpose(1, 2).reshape(b, h, nk, -1), d)
            for q, s in ((st["kc"], st["ks"]), (st["vc"], st["vs"])))
    row = st["start"][:-1].unsqueeze(1) + torch.arange(nq, device="cuda", dtype=torch.int32)
    real = row < st["start"][1:].unsqueeze(1)
    at = row.clamp(max=st["tokens"] - 1).long()
    x = st["qkv"].float()[:, :c["heads"] * d][at].reshape(b, nq, h, group, d).permute(0, 2, 3, 1, 4)
    s = (x.reshape(b, h, group * nq, d) @ k.transpose(2, 3)).reshape(b, h, group, nq, nk) / math.sqrt(d)
    j = torch.arange(nk, device="cuda", dtype=torch.int32)
    keys = (j < st["len"].unsqueeze(1)).unsqueeze(1)
    if c["causal"]:
        pos = (st["len"] - st["start"][1:] + st["start"][:-1]).unsqueeze(1)
        pos = (pos + torch.arange(nq, device="cuda", dtype=torch.int32)).unsqueeze(2)
        keys = keys & (j <= pos)
        if c["window"]:
            keys = keys & (j > pos - c["window"])
    s = s.masked_fill_(~keys.reshape(b, 1, 1, -1, nk), -math.inf)
    s = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    y = (s.reshape(b, h, group * nq, nk) @ v).reshape(b, h, group, nq, d) / s.sum(-1, keepdim=True)
    y = y.permute(0, 3, 1, 2, 4).reshape(b, nq, c["heads"], d)
    out = torch.zeros((st["tokens"], c["heads"], d), dtype=torch.float32, device="cuda")
    out[at[real]] = y[real]
    return out.half()


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _own(st):
    """The op functions' calls."""
    c, (be, ops), f = st["case"], _backend(), st["buf"]
    kind = c["kind"]
    if kind == "quantize":
        dt = ops.DTYPE_F16 if c["dtype"] == "f16" else ops.DTYPE_F32
        ops.quantize_mxfp4(be, dt, f["x"], f["q"], f["s"], c["rows"], c["k"])
        ops.dequantize_mxfp4(be, dt, f["q"], f["s"], f["y"], c["rows"], c["k"])
        return st["y"]
    if kind == "product":
        ops.gemm_mxfp4(be, ops.DTYPE_F16 if c["a"] == "f16" else ops.DTYPE_MXFP4, f["a"], f.get("as"), f["w"],
                       f["ws"], f.get("bias"), ops.DTYPE_F16, f["y"], c["m"], c["n"], c["k"], act=c["act"])
        return st["y"]
    if kind == "rope":
        row = c["heads"] * c["dim"]
        ops.rope_axes(be, ops.DTYPE_F16 if c["dtype"] == "f16" else ops.DTYPE_F32, f["x"], row, 0, f["y"], row, 0,
                      f["pos"], c["tokens"], c["heads"], c["dim"], c["rotary"], _sections(c), order=c["order"],
                      pairs=c["pairs"], freq=c["freq"], base=10000.0)
        return st["y"]
    cache = (f["kc"], f["ks"], f["vc"], f["vs"], f["table"], f["start"], f["len"])
    sizes = (c["dim"], c["page"], st["total"], st["most"])
    row = st["qkv"].shape[1]
    if kind == "append":
        hd = c["kv_heads"] * c["dim"]
        ops.kv_append_mxfp4(be, f["qkv"], row, 0, f["qkv"], row, hd, *cache, st["tokens"], c["batch"], c["kv_heads"],
                            *sizes)
        n = st["total"] * c["kv_heads"] * c["page"]
        ops.dequantize_mxfp4(be, ops.DTYPE_F16, f["kc"], f["ks"], f["yk"], n, c["dim"])
        ops.dequantize_mxfp4(be, ops.DTYPE_F16, f["vc"], f["vs"], f["yv"], n, c["dim"])
        return {"k": st["yk"], "v": st["yv"]}
    ops.attention_mxfp4(be, f["qkv"], row, 0, *cache, f["y"], st["tokens"], c["batch"], c["heads"], c["kv_heads"],
                        *sizes, scale=1.0 / math.sqrt(c["dim"]), causal=c["causal"], window=c["window"])
    return st["y"]


def run(st):
    if own:
        return _own(st)
    c, kind = st["case"], st["case"]["kind"]
    if kind == "quantize":
        e, v = _codes(st["x"].float())
        return (v * _power(e.clamp(min=-126)).unsqueeze(-1)).reshape(c["rows"], -1)[:, :c["k"]].to(st["x"].dtype)
    if kind == "product":
        return _plain_product(st)
    if kind == "rope":
        return _plain_rope(st)
    return _plain_append(st) if kind == "append" else _plain_attend(st)


def _seen(case, nq, kv):
    """Pairs of a query and a key it sees, summed over the sequences."""
    pairs = 0
    for n, m in zip(nq, kv):
        first = m - n + 1 if case["causal"] else m
        w = case["window"] or m
        low, high = min(first, w), min(m, w)
        if not case["causal"]:
            pairs += n * m
        elif first >= w:
            pairs += n * w
        else:
            up = high - low + 1  # queries before the window is full, then the others
            pairs += (low + high) * up // 2 + (n - up) * high
    return pairs


def work(case):
    kind = case["kind"]
    packed = 0.5 + 1.0 / BLOCK  # bytes of an element in the 4-bit format
    if kind == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 * (2 if case["dtype"] == "f16" else 4) + packed), "flops": 4 * n}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = m * k * (2 if case["a"] == "f16" else packed)
        return {"bytes": a + n * k * packed + 2 * m * n + 2 * n * case["bias"], "flops": 2.0 * m * n * k}
    if kind == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * (2 if case["dtype"] == "f16" else 4) + 4 * case["axes"] * case["tokens"],
                "flops": 3.0 * n}
    nq, kv = _lengths(case)
    row = case["kv_heads"] * case["dim"]
    if kind == "append":
        cache = 2 * sum(-(-n // case["page"]) for n in kv) * case["page"] * row
        return {"bytes": sum(nq) * row * 2 * (2 + packed) + cache * (packed + 2), "flops": 8.0 * sum(nq) * row}
    read = sum(min(m, n + case["window"]) if case["window"] else m for n, m in zip(nq, kv))
    return {"bytes": 2 * read * row * packed + 4 * sum(nq) * case["heads"] * case["dim"],
            "flops": 4.0 * case["heads"] * case["dim"] * _seen(case, nq, kv)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def _wide(q, s, k):
    """Packed rows from their bits: sign, two exponent bits, one mantissa bit, times the block's power of two."""
    n = torch.stack([q & 15, q >> 4], -1).flatten(-2).long()
    ex, man = (n >> 1) & 3, (n & 1).double()
    v = torch.where(ex == 0, man / 2, (1 + man / 2) * torch.pow(2.0, (ex - 1).double()))
    v = torch.where(n >= 8, -v, v)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=q.device), s.double() - 127)
    return (v * scale.repeat_interleave(BLOCK, -1))[..., :k]


def _nearest(x, least):
    """The values MXFP4 gives f64 rows: the block's exponent from its largest magnitude, then the nearest of the
    format's fifteen values, of two as near the one whose last bit is zero."""
    r, k = x.shape
    out = torch.empty_like(x)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    for at in range(0, r, max(1, 8000000 // k)):
        rows = x[at:at + max(1, 8000000 // k)]
        wide = torch.zeros((rows.shape[0], -(-k // BLOCK) * BLOCK), dtype=torch.float64, device=x.device)
        wide[:, :k] = rows
        b = wide.view(rows.shape[0], -1, BLOCK)
        e = torch.floor(torch.log2(b.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -140))) - 2
        unit = torch.pow(2.0, e.clamp(min=least))
        a = b.abs() / unit
        low = torch.searchsorted(middle, a)  # the count of midpoints below a: one that a equals is not below
        tie = (low < 7) & (a == middle[low.clamp(max=6)]) & (low % 2 == 1)
        out[at:at + rows.shape[0]] = (torch.sign(b) * grid[low + tie] * unit).flatten(1)[:, :k]
    return out


def exact(case, seed):
    global own
    kind, was = case["kind"], own
    own = False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if kind == "quantize":
        return _nearest(st["x"].double(), -127)
    if kind == "product":
        k = case["k"]
        a = st["a"].double() if case["a"] == "f16" else _wide(st["a"], st["as"], k)
        y = a @ _wide(st["w"], st["ws"], k).t()
        if case["bias"]:
            y += st["bias"].double()
        return y * torch.sigmoid(y) if case["act"] == 2 else y
    if kind == "rope":
        x, n = st["x"].double(), case["rotary"]
        axis, place, size = _axis_of_pair(case)
        out = x.clone()
        for i in range(n // 2):
            f = 10000.0 ** -(i / (n // 2) if case["freq"] == 0 else place[i] / size[i])
            turn = torch.polar(torch.ones(case["tokens"], dtype=torch.float64, device="cuda"),
                               st["pos"][axis[i]].double() * f)
            a, b = (i, i + n // 2) if case["pairs"] == 0 else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., a], x[..., b]) * turn.unsqueeze(1)
            out[..., a], out[..., b] = z.real, z.imag
        return out
    h, d, ps = case["kv_heads"], case["dim"], case["page"]
    if kind == "append":
        out = {}
        for name, q, s, j in (("k", "kc", "ks", 0), ("v", "vc", "vs", 1)):
            y = _wide(st[q], st[s], d)
            rows = st["qkv"].double()[:, j * h * d:(j + 1) * h * d]
            rows = _nearest(rows.reshape(-1, d), -23).reshape(-1, h, d)
            at = 0
            for b, (n, m) in enumerate(zip(st["nq"], st["kv"])):
                p = torch.arange(m - n, m, device="cuda")
                y[st["table"][b].long()[p // ps], :, p % ps] = rows[at:at + n]
                at += n
            out[name] = y
        return out
    group = case["heads"] // h
    y = torch.zeros((st["tokens"], case["heads"], d), dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(st["nq"], st["kv"])):
        pages = st["table"][b, :-(-m // ps)].long()
        q = st["qkv"][at:at + n, :case["heads"] * d].double().reshape(n, case["heads"], d)
        i, j = torch.arange(m - n, m, device="cuda").unsqueeze(1), torch.arange(m, device="cuda")
        see = (j <= i) if case["causal"] else torch.ones((n, m), dtype=torch.bool, device="cuda")
        if case["window"]:
            see = see & (i - j < case["window"])
        for e in range(h):
            k, v = (_wide(st[a][pages, e].reshape(-1, d // 2), st[z][pages, e].reshape(-1, d // BLOCK), d)[:m]
                    for a, z in (("kc", "ks"), ("vc", "vs")))
            for f in range(e * group, (e + 1) * group):
                w = (q[:, f] @ k.t() * d ** -0.5).masked_fill(~see, -math.inf)
                y[at:at + n, f] = torch.softmax(w, -1) @ v
        at += n
    return y
