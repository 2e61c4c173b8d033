"""Operators of a mixture of experts in 4 bits, as timed cases.

Each case is one pass through an operator of such a layer, as a serving
program calls it on device buffers:

* ``route``    each token's experts and their weights from the router's
               logits: softmax or sigmoid, a bias for balance, groups;
* ``order``    the choices of all tokens sorted by expert;
* ``product``  rows times their own expert's MXFP4 weights, the rows in f16
               or MXFP4, taken from the tokens by the sorted choices or put
               back by them;
* ``combine``  the weighted sum of each token's experts' rows.

With ``own`` false ``run`` computes the operators from elementary torch
operations; with ``own`` true it calls this backend's op functions.
"""
import math

import torch

own = False  # True: run() calls this backend's op functions

BLOCK = 32  # elements that share a scale
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SWIGLU = 3  # the gated activation


def listed():
    return [
        # A decoding batch's router: latency is everything.
        {"name": "route_tokens", "kind": "route", "dtype": "f32", "tokens": 32, "experts": 128, "top": 8, "sigmoid": False,
         "bias": False, "groups": 1, "kept": 1, "best": 1, "renorm": True, "masked": 0.0},
        # Long prompts, many experts in groups, a bias that balances their load, some rows of padding.
        {"name": "route_prompt", "kind": "route", "dtype": "f32", "tokens": 32768, "experts": 256, "top": 8,
         "sigmoid": True, "bias": True, "groups": 8, "kept": 4, "best": 2, "renorm": True, "masked": 0.03},
        # An odd number of experts, f16 logits (which tie), weights as the softmax gives them.
        {"name": "route_odd", "kind": "route", "dtype": "f16", "tokens": 4099, "experts": 61, "top": 6, "sigmoid": False,
         "bias": False, "groups": 1, "kept": 1, "best": 1, "renorm": False, "masked": 0.0},
        # The choices of a decoding batch.
        {"name": "order_tokens", "kind": "order", "tokens": 48, "top": 8, "experts": 128, "pad": 3},
        # Those of many prompts at a time.
        {"name": "order_prompt", "kind": "order", "tokens": 65537, "top": 8, "experts": 256, "pad": 1000},
        # Gate and up in one product for a decoding batch: one to four rows for most experts, the weights' bytes.
        {"name": "product_tokens", "kind": "product", "a": "f16", "tokens": 16, "top": 8, "experts": 64, "n": 2816, "k": 2048,
         "bias": False, "act": SWIGLU, "back": False, "pad": 0},
        # The way back for a larger batch: some dozens of rows an expert.
        {"name": "product_back", "kind": "product", "a": "f16", "tokens": 256, "top": 8, "experts": 64, "n": 4096, "k": 2048,
         "bias": False, "act": 0, "back": True, "pad": 5},
        # Rows in 4 bits, odd sizes, biases.
        {"name": "product_mx_batch", "kind": "product", "a": "mxfp4", "tokens": 51, "top": 4, "experts": 32, "n": 5782,
         "k": 2900, "bias": True, "act": SWIGLU, "back": False, "pad": 1},
        # Prompts over few large experts: the matrix cores' case, f16 rows.
        {"name": "product_prompt", "kind": "product", "a": "f16", "tokens": 4096, "top": 2, "experts": 8, "n": 14336,
         "k": 4096, "bias": False, "act": 2, "back": False, "pad": 0},
        # Prompts over many experts, rows in 4 bits.
        {"name": "product_mx_prompt", "kind": "product", "a": "mxfp4", "tokens": 8192, "top": 8, "experts": 128, "n": 4096,
         "k": 4096, "bias": False, "act": SWIGLU, "back": False, "pad": 100},
        # A decoding batch's sum.
        {"name": "combine_tokens", "kind": "combine", "dtype": "f16", "tokens": 24, "top": 8, "experts": 128, "n": 4096,
         "base": False, "pad": 1},
        # A prompt's, with the row of an expert that all tokens share; an odd row length.
        {"name": "combine_prompt", "kind": "combine", "dtype": "f16", "tokens": 8192, "top": 8, "experts": 128, "n": 5119,
         "base": True, "pad": 200},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(max(round(v / step) * step, -(-lo // step) * step), hi // step * step))


def draw(rng):
    kind = rng.choice(("route", "route", "order", "product", "product", "product", "combine"))
    if kind == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * _log_int(rng, max(2, 8 // groups), 512 // groups)
        kept = rng.randint(max(1, groups // 2), groups)
        return {"kind": kind, "dtype": rng.choice(("f16", "f32")), "tokens": _log_int(rng, 1, 8000000 // experts),
                "experts": experts, "top": rng.randint(1, min(10, kept * (experts // groups))),
                "sigmoid": rng.random() < 0.5, "bias": rng.random() < 0.5, "groups": groups, "kept": kept,
                "best": rng.choice((1, 2)), "renorm": rng.random() < 0.7, "masked": rng.choice((0.0, 0.0, 0.1))}
    experts = _log_int(rng, 4, 256)
    top = rng.randint(1, min(8, experts))
    if kind == "order":
        tokens = _log_int(rng, 1, 500000 // top)
        return {"kind": kind, "tokens": tokens, "top": top, "experts": experts, "pad": rng.randint(0, tokens // 8)}
    if kind == "combine":
        n = _log_int(rng, 64, 16384, rng.choice((1, 8, 64)))
        dtype = rng.choice(("f16", "f32"))
        tokens = _log_int(rng, 1, max(1, min(65536, 300000000 // (n * (top + 2)) // (2 if dtype == "f32" else 1))))
        return {"kind": kind, "dtype": dtype, "tokens": tokens, "top": top, "experts": experts, "n": n,
                "base": rng.random() < 0.5, "pad": rng.randint(0, tokens // 8)}
    a = rng.choice(("f16", "mxfp4"))
    n, k = 2 * _log_int(rng, 64, 7168, rng.choice((1, 8, 16))), _log_int(rng, 128, 8192, rng.choice((1, 8, 32)))
    experts = max(top, min(experts, 1800000000 // (n * k)))
    most = 450e9 if a == "f16" else 1000e9
    tokens = _log_int(rng, 1, max(1, min(8192, int(most / (n * k * top)))))
    return {"kind": kind, "a": a, "tokens": tokens, "top": top, "experts": experts, "n": n, "k": k,
            "bias": rng.random() < 0.4, "act": rng.choice((0, 0, 1, 2, SWIGLU, SWIGLU)), "back": rng.random() < 0.5,
            "pad": rng.randint(0, tokens // 8)}


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


def _zeros(shape, dtype):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _choices(case):
    """Experts of each token, some chosen far more often than others, -1 for the last `pad` tokens; on the host, the
    same for every seed but for which expert is which."""
    r = torch.Generator().manual_seed(91 + case["experts"] * 31 + case["tokens"])
    t, e = case["tokens"], case["experts"]
    u = torch.rand((t, e), generator=r).clamp(min=1e-9)
    score = torch.randn(e, generator=r) * 0.7 - torch.log(-torch.log(u).clamp(min=1e-9))
    ids = torch.topk(score, case["top"], dim=1).indices.to(torch.int32)
    if case["pad"]:
        ids[t - case["pad"]:] = -1
    return ids


def _lists(case, g):
    """The choices on the device, sorted by expert: ids, where each expert's begin (on the host too), and the sorted
    choices, -1 behind them."""
    which = torch.randperm(case["experts"], generator=g, device="cuda").to(torch.int32)
    ids = _choices(case).to("cuda")
    ids = torch.where(ids >= 0, which[ids.clamp(min=0).long()], ids).contiguous()
    flat = ids.flatten().long()
    count = torch.bincount(flat[flat >= 0], minlength=case["experts"])
    offsets = torch.cat([count.new_zeros(1), torch.cumsum(count, 0)]).to(torch.int32)
    key = torch.where(flat >= 0, flat, flat.new_full((), case["experts"]))
    order = torch.sort(key, stable=True).indices.to(torch.int32)
    order[int(offsets[-1]):] = -1
    return ids, offsets, order, offsets.tolist()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    st = {"case": case}
    if kind == "route":
        t, e = case["tokens"], case["experts"]
        # the logits of a router in use: some experts are liked by most tokens
        x = torch.randn((t, e), generator=g, device="cuda") * 1.5 + torch.randn(e, generator=g, device="cuda") * 0.5
        if case["masked"]:
            x[torch.rand(t, generator=g, device="cuda") < case["masked"]] = -math.inf
        st["x"] = x.to(_TYPES[case["dtype"]])
        if case["bias"]:
            st["b"] = _normal(g, (e,), 0.05)
        st["ids"], st["w"] = _zeros((t, case["top"]), torch.int32), _zeros((t, case["top"]), torch.float32)
        return _hold(st)
    ids, offsets, order, st["at"] = _lists(case, g)
    slots = ids.numel()
    if kind == "order":
        st["ids"] = ids
        st["offsets"], st["order"] = _zeros(case["experts"] + 1, torch.int32), _zeros(slots, torch.int32)
    elif kind == "combine":
        dt, n = _TYPES[case["dtype"]], case["n"]
        st["ids"] = ids
        st["x"] = _tokens(g, (slots, n), dt)
        st["w"] = torch.softmax(torch.randn(ids.shape, generator=g, device="cuda"), -1)
        if case["base"]:
            st["base"] = _tokens(g, (case["tokens"], n), dt)
        st["y"] = _zeros((case["tokens"], n), dt)
    else:
        n, k = case["n"], case["k"]
        a = _tokens(g, (slots if case["back"] else case["tokens"], k))
        if case["a"] == "f16":
            st["a"] = a
        else:
            st["a"], st["as"] = _pack(a.float())
        blocks = -(-k // BLOCK)
        st["w"] = _zeros((case["experts"], n, blocks * 16), torch.uint8)
        st["ws"] = _zeros((case["experts"], n, blocks), torch.uint8)
        for e in range(case["experts"]):
            st["w"][e], st["ws"][e] = _pack(_normal(g, (n, k), 1.0 / math.sqrt(k)))
        if case["bias"]:
            st["bias"] = _normal(g, (case["experts"], n), 0.5, torch.float16)
        st["offsets"], st["order"] = offsets, order
        st["y"] = _zeros((slots, n // 2 if case["act"] == SWIGLU else n), torch.float16)
    return _hold(st)


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------


def _power(e):
    """2^e in f32 for whole e in [-126, 127]."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _pack(x):
    """f32 rows as MXFP4: two elements a byte, the first in the low half, and a scale byte for each block."""
    pad = -x.shape[1] % BLOCK
    b = (torch.nn.functional.pad(x, (0, pad)) if pad else x).reshape(x.shape[0], -1, BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.where(amax == 0, -126, (torch.frexp(amax).exponent - 3).clamp(-126, 127))
    v = b * _power(-e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(v).to(torch.uint8) << 3)
    q = code[..., 0::2] | (code[..., 1::2] << 4)
    return q.reshape(x.shape[0], -1).contiguous(), (e.squeeze(-1) + 127).to(torch.uint8).contiguous()


def _values(q, s, k):
    """The f32 values of packed rows."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float32, device=q.device)
    v = torch.stack([grid[(q & 15).int()], grid[(q >> 4).int()]], -1).reshape(q.shape[:-1] + (-1, BLOCK))
    v = v * _power(s.int() - 127).unsqueeze(-1)
    return v.reshape(q.shape[:-1] + (-1,))[..., :k]


def _plain_route(st):
    """In 64 bits: which of two experts comes first may hang on the last bits of their scores."""
    c = st["case"]
    x = st["x"].double()
    if c["sigmoid"]:
        p = 1 / (1 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300))
        p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    # without a bias the logits have the scores' order, and tie only where they are equal
    choice = p + st["b"].double() if c["bias"] else x
    choice = torch.where(x > -math.inf, choice, -math.inf)
    if c["groups"] > 1:
        value = torch.where(x > -math.inf, p, -math.inf) if c["best"] == 2 and not c["bias"] else choice
        value = value.reshape(len(x), c["groups"], -1)
        best = torch.sort(value, -1, descending=True).values
        total = best[..., 0]
        if c["best"] == 2 and best.shape[-1] > 1:
            total = total + torch.where(best[..., 1] > -math.inf, best[..., 1], 0.0)
        order = torch.sort(total, dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        keep = torch.zeros((len(x), c["groups"]), dtype=torch.bool, device=x.device).scatter_(1, order, True)
        choice = choice.masked_fill(~keep.repeat_interleave(c["experts"] // c["groups"], 1), -math.inf)
    top = torch.sort(choice, dim=-1, descending=True, stable=True)
    ids, real = top.indices[:, :c["top"]], top.values[:, :c["top"]] > -math.inf
    w = torch.where(real, p.gather(1, ids), 0.0)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    return {"ids": torch.where(real, ids, -1).to(torch.int32), "weights": w.float()}


def _plain_order(st):
    flat, e = st["ids"].flatten().long(), st["case"]["experts"]
    key = torch.where((flat >= 0) & (flat < e), flat, e)
    s = torch.sort(key, stable=True)
    offsets = torch.searchsorted(s.values, torch.arange(e + 1, device=key.device))
    return {"offsets": offsets.to(torch.int32), "order": torch.where(s.values < e, s.indices, -1).to(torch.int32)}


def _plain_product(st):
    c = st["case"]
    y = torch.zeros_like(st["y"])
    a = st["a"].float() if c["a"] == "f16" else _values(st["a"], st["as"], c["k"])
    for e in range(c["experts"]):
        lo, hi = st["at"][e], st["at"][e + 1]
        if lo == hi:
            continue
        slot = st["order"][lo:hi].long()
        rows = a[lo:hi] if c["back"] else a[slot // c["top"]]
        v = rows @ _values(st["w"][e], st["ws"][e], c["k"]).t()
        if c["bias"]:
            v = v + st["bias"][e].float()
        if c["act"] == 1:
            v = v.clamp(min=0)
        elif c["act"] == 2:
            v = v / (1 + torch.exp(-v))
        elif c["act"] == SWIGLU:
            v = v[:, 0::2] / (1 + torch.exp(-v[:, 0::2])) * v[:, 1::2]
        if c["back"]:
            y[slot] = v.half()
        else:
            y[lo:hi] = v.half()
    return y


def _plain_combine(st):
    c = st["case"]
    w = torch.where(st["ids"] >= 0, st["w"], 0.0)
    x = st["x"].reshape(c["tokens"], c["top"], c["n"])
    y = st["base"].float() if c["base"] else torch.zeros((c["tokens"], c["n"]), device=x.device)
    for j in range(c["top"]):
        y = y + w[:, j:j + 1] * x[:, j].float()
    return y.to(x.dtype)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _own(st):
    """The op functions' calls."""
    c, (be, ops), f = st["case"], _backend(), st["buf"]
    kind = c["kind"]
    if kind == "route":
        ops.route_experts(be, ops.DTYPE_F16 if c["dtype"] == "f16" else ops.DTYPE_F32, f["x"], c["experts"], 0, f.get("b"),
                          f["ids"], f["w"], c["tokens"], c["experts"], c["top"],
                          score=ops.SCORE_SIGMOID if c["sigmoid"] else ops.SCORE_SOFTMAX, groups=c["groups"],
                          top_groups=c["kept"], group_best=c["best"], renorm=c["renorm"], scale=1.0)
        return {"ids": st["ids"], "weights": st["w"]}
    if kind == "order":
        ops.order_experts(be, f["ids"], f["offsets"], f["order"], c["tokens"] * c["top"], c["experts"])
        return {"offsets": st["offsets"], "order": st["order"]}
    dt = ops.DTYPE_F16 if c.get("dtype", "f16") == "f16" else ops.DTYPE_F32
    if kind == "combine":
        ops.combine_experts(be, dt, f["x"], f["ids"], f["w"], f.get("base"), f["y"], c["tokens"], c["top"], c["experts"],
                            c["n"])
        return st["y"]
    ops.gemm_mxfp4_experts(be, ops.DTYPE_F16 if c["a"] == "f16" else ops.DTYPE_MXFP4, f["a"], f.get("as"), f["w"], f["ws"],
                           f.get("bias"), ops.DTYPE_F16, f["y"], f["offsets"], f["order"], c["tokens"] * c["top"],
                           c["experts"], c["n"], c["k"], act=c["act"], gather=0 if c["back"] else c["top"],
                           scatter=c["back"])
    return st["y"]


def run(st):
    if own:
        return _own(st)
    return {"route": _plain_route, "order": _plain_order, "product": _plain_product,
            "combine": _plain_combine}[st["case"]["kind"]](st)


def work(case):
    kind = case["kind"]
    t = case["tokens"]
    size = 2 if case.get("dtype", "f16") == "f16" else 4
    if kind == "route":
        e = case["experts"]
        return {"bytes": t * (e * size + case["top"] * 8) + 4 * e * case["bias"], "flops": 5.0 * t * e}
    if kind == "order":
        return {"bytes": 8 * t * case["top"] + 4 * case["experts"], "flops": 2.0 * t * case["top"]}
    real = (t - case["pad"]) * case["top"]
    if kind == "combine":
        n = case["n"]
        return {"bytes": size * n * (real + t * (1 + case["base"])) + 8 * t * case["top"], "flops": 2.0 * real * n}
    packed = 0.5 + 1.0 / BLOCK  # bytes of an element in the 4-bit format
    n, k = case["n"], case["k"]
    ids = _choices(case)
    hit = int(torch.unique(ids[ids >= 0]).numel())
    rows = real if case["back"] else t - case["pad"]
    return {"bytes": rows * k * (2 if case["a"] == "f16" else packed) + hit * n * (k * packed + 2 * case["bias"])
            + real * (n // 2 if case["act"] == SWIGLU else n) * 2, "flops": 2.0 * real * n * k}


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


def _exact_route(st):
    c = st["case"]
    x = st["x"].double()
    p = torch.sigmoid(x) if c["sigmoid"] else torch.softmax(x, -1)
    there = x > -math.inf
    value = torch.where(there, p + st["b"].double() if c["bias"] else x, -math.inf)
    each = c["experts"] // c["groups"]
    if c["groups"] > 1:
        of = value if c["bias"] or c["best"] == 1 else torch.where(there, p, -math.inf)
        totals = []
        for i in range(c["groups"]):
            part = of[:, i * each:(i + 1) * each].clone()
            total = part.amax(-1)
            if c["best"] == 2:
                part.scatter_(1, part.argmax(-1, keepdim=True), -math.inf)
                next_one = part.amax(-1)
                total = torch.where(next_one > -math.inf, total + next_one, total)
            totals.append(total)
        totals = torch.stack(totals, -1)
        rank = torch.zeros_like(totals, dtype=torch.long)  # how many groups come before each
        for i in range(c["groups"]):
            for j in range(c["groups"]):
                rank[:, i] += (totals[:, j] > totals[:, i]) | ((totals[:, j] == totals[:, i]) & (j < i))
        value = torch.where((rank < c["kept"]).repeat_interleave(each, 1), value, -math.inf)
    ids, weights = [], []
    index = torch.arange(c["experts"], device=x.device)
    for _ in range(c["top"]):
        best = value.amax(-1, keepdim=True)
        at = torch.where(value == best, index, c["experts"]).amin(-1, keepdim=True)  # the lowest of equal ones
        real = best > -math.inf
        ids.append(torch.where(real, at, -1))
        weights.append(torch.where(real, p.gather(1, at), 0.0))
        value = value.scatter(1, at, -math.inf)
    w = torch.cat(weights, 1)
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return {"ids": torch.cat(ids, 1).to(torch.int32), "weights": w}


def exact(case, seed):
    global own
    kind, was = case["kind"], own
    own = False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if kind == "route":
        return _exact_route(st)
    if kind == "order":
        flat = st["ids"].flatten()
        found = [torch.nonzero(flat == e).flatten() for e in range(case["experts"])]
        order = torch.cat(found)
        count = torch.tensor([0] + [f.numel() for f in found], device="cuda")
        rest = torch.full((flat.numel() - order.numel(),), -1, dtype=order.dtype, device="cuda")
        return {"offsets": torch.cumsum(count, 0).to(torch.int32), "order": torch.cat([order, rest]).to(torch.int32)}
    top = case["top"]
    if kind == "combine":
        w = st["w"].double() * (st["ids"] >= 0)
        y = torch.zeros((case["tokens"], case["n"]), dtype=torch.float64, device="cuda")
        for t in range(0, case["tokens"], 512):
            x = st["x"].reshape(-1, top, case["n"])[t:t + 512].double()
            y[t:t + 512] = (w[t:t + 512].unsqueeze(-1) * x).sum(1)
        return y + st["base"].double() if case["base"] else y
    k, n = case["k"], case["n"]
    y = torch.zeros(st["y"].shape, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        slot = st["order"][st["at"][e]:st["at"][e + 1]].long()
        if not slot.numel():
            continue
        row = torch.arange(st["at"][e], st["at"][e + 1], device="cuda")
        take = row if case["back"] else torch.div(slot, top, rounding_mode="floor")
        a = st["a"][take].double() if case["a"] == "f16" else _wide(st["a"][take], st["as"][take], k)
        v = a @ _wide(st["w"][e], st["ws"][e], k).t()
        if case["bias"]:
            v += st["bias"][e].double()
        if case["act"] == 1:
            v = torch.relu(v)
        elif case["act"] == 2:
            v = v * torch.sigmoid(v)
        elif case["act"] == SWIGLU:
            v = v.reshape(-1, n // 2, 2)
            v = v[..., 0] * torch.sigmoid(v[..., 0]) * v[..., 1]
        y[slot if case["back"] else row] = v
    return y
