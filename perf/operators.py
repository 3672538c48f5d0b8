"""What the expert half of a mixture-of-experts block is asked to do in use, case by case, through
`moearc_amd.Context`: the operators beside the attention half that `perf/cases.py` holds.

Four kinds of call, in the sizes a program that serves a model makes them:

* ``norm``   ``norm_residual``: h += scale * gate * z, x = RMSNorm(h) * w_pre, where z is a block's output
             y, or RMSNorm(y) * w_post; without y the plain RMSNorm.
* ``route``  ``moe_route``: the n_used largest of each token's router logits, largest first, ties to
             the lowest expert, and their softmax weights, over all experts or over the selected.
* ``ffn``    ``moe_ffn``: sum over a token's experts of weight * (W_down act(W_gate x, W_up x) + bias).
* ``linear`` ``matmul_experts``: one product per token and selected expert, W[expert] x (+ bias).

Inputs are made on the GPU from a seed: N(0,1) activations, weights of a trained matrix's size in each
GGUF format, router logits with favoured and neglected experts. Every buffer is a torch tensor that the
library sees through a ``DeviceView``, as a program that holds its model in torch would pass it.

Where ``own`` is false the plain forms compute the same in float32 torch operations.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

ALPHA, LIMIT = 1.702, 7.0  # of the clamped activation
BLOCK = {"F16": (1, 2), "Q8_0": (32, 34), "MXFP4": (32, 17), "Q4_K": (256, 144), "Q5_K": (256, 176),
         "Q6_K": (256, 210)}  # elements and bytes of a GGUF block


# ---- the cases -----------------------------------------------------------------------------------

def _norm(name, rows, cols, y="f32", post=True, gate="shared", x="f32"):
    """y None: the plain norm; gate: one row of factors for all rows, one for each, or none."""
    c = dict(kind="norm", rows=rows, cols=cols, y=y, post=post, gate=gate, x=x)
    return dict(name=name, **c) if name else c


def _route(name, tokens, experts, used, over, scale=1.0):
    c = dict(kind="route", tokens=tokens, experts=experts, used=used, over=over, scale=scale)
    return dict(name=name, **c) if name else c


def _ffn(name, tokens, experts, used, embd, ff, types, act="silu", bias=False, io="f32", add=False):
    c = dict(kind="ffn", tokens=tokens, experts=experts, used=used, embd=embd, ff=ff, type=types[0], down=types[1],
             act=act, bias=bias, io=io, add=add)
    return dict(name=name, **c) if name else c


def _linear(name, tokens, experts, used, rows, cols, type, bias=False, io="f32", per_slot=False):
    c = dict(kind="linear", tokens=tokens, experts=experts, used=used, rows=rows, cols=cols, type=type, bias=bias,
             io=io, per_slot=per_slot)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # One decode step's residual update and norm of a block with norms on both sides: latency.
        _norm("norm_step", 1, 2880),
        # The same over a prompt chunk, the normed rows in f16 for the products behind it.
        _norm("norm_2k", 2048, 2880, gate="none", x="f16"),
        # A prompt chunk's query heads, normed one by one: many short rows.
        _norm("norm_heads", 65536, 128, y=None, post=False, gate="none"),
        # The router of one decode step, and of a long prompt's whole chunk.
        _route("route_step", 1, 128, 4, "used"),
        _route("route_16k", 16384, 128, 8, "all"),
        # One decode step of 128 MXFP4 experts, four to a token, into the residual stream: the four
        # experts' weights once, and the launches' latency.
        _ffn("ffn_step", 1, 128, 4, 2880, 2880, ("MXFP4", "MXFP4"), "clamp", True, add=True),
        # A serving batch of 24 sequences on the same layer: most experts wake for a token or two.
        _ffn("ffn_b24", 24, 128, 4, 2880, 2880, ("MXFP4", "MXFP4"), "clamp", True, add=True),
        # A long prompt's ragged chunk through 32 such experts: the matrix cores' case.
        _ffn("ffn_prompt_2k", 2000, 32, 4, 2880, 2880, ("MXFP4", "MXFP4"), "clamp", True, add=True),
        # A ragged prompt through 128 small K-quant experts, eight to a token, f16 activations.
        _ffn("ffn_q4k_1k", 1000, 128, 8, 2048, 768, ("Q4_K", "Q6_K"), io="f16"),
        # A short prompt through 64 Q8_0 experts, eight to a token.
        _ffn("ffn_q8_200", 200, 64, 8, 2048, 1024, ("Q8_0", "Q8_0")),
        # The largest product alone: unquantised experts over a chunk, f16 in and out.
        _linear("linear_f16_4k", 4096, 16, 2, 4096, 2048, "F16", io="f16"),
        # Eight sequences' step through a single K-quant matrix per expert.
        _linear("linear_q5k_8", 8, 64, 4, 2048, 2048, "Q5_K", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["norm", "route", "ffn", "ffn", "ffn", "linear"])
    if kind == "norm":
        cols = rng.choice([64, 128, 2048, 2880, 4096, _log_int(rng, 64, 8192)])
        y = rng.choice([None, "f32", "f32", "f16"])
        return _norm(None, _log_int(rng, 1, 16 * 1024 * 1024 // cols // 2), cols, y, y is not None and rng.choice([True, False]),
                     rng.choice(["none", "shared", "row"]) if y else "none", rng.choice(["f32", "f16"]))
    if kind == "route":
        experts = rng.choice([8, 32, 64, 128, 128, 256, 512])
        return _route(None, _log_int(rng, 1, 16384), experts, min(experts, rng.choice([1, 2, 4, 6, 8, 8])),
                      rng.choice(["all", "used"]), rng.choice([1.0, 1.0, 2.5]))
    experts, used, embd, ff, types = rng.choice([
        (128, 4, 2880, 2880, [("MXFP4", "MXFP4")]), (32, 4, 2880, 2880, [("MXFP4", "MXFP4"), ("Q8_0", "Q8_0")]),
        (128, 8, 2048, 768, [("Q4_K", "Q6_K"), ("Q5_K", "Q5_K"), ("Q8_0", "Q8_0"), ("Q4_K", "Q4_K")]),
        (64, 8, 2048, 1024, [("Q4_K", "Q6_K"), ("Q8_0", "Q8_0"), ("F16", "F16")]),
        (8, 2, 1024, 1792, [("F16", "F16"), ("Q6_K", "Q6_K"), ("Q8_0", "Q8_0")])])
    if kind == "ffn":
        io = rng.choice(["f32", "f32", "f16"])
        return _ffn(None, rng.choice([1, _log_int(rng, 1, 64), _log_int(rng, 1, 1900)]), experts, used, embd, ff,
                    rng.choice(types), rng.choice(["silu", "clamp"]), rng.choice([True, False]), io,
                    io == "f32" and rng.choice([True, False]))
    return _linear(None, _log_int(rng, 1, 2048), experts, used, ff, embd, rng.choice(types)[rng.choice([0, 1])],
                   rng.choice([True, False]), rng.choice(["f32", "f16"]), rng.choice([True, False]))


# ---- inputs --------------------------------------------------------------------------------------

def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dtype(io):
    return torch.float16 if io == "f16" else torch.float32


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _bytes_of(x):
    return x.contiguous().view(torch.uint8)


def _weights(g, type, experts, rows, cols):
    """The experts' matrices in a GGUF format, uint8 [experts, rows, row bytes], values of about
    N(0, 0.02)'s size: every payload byte is drawn, then the blocks' scales are set."""
    if type == "F16":
        return _bytes_of(_normal(g, experts, rows, cols, dtype=torch.float16).mul_(0.02)).view(experts, rows, -1)
    be, bb = BLOCK[type]
    w = torch.randint(0, 256, (experts, rows, cols // be, bb), generator=g, device="cuda", dtype=torch.uint8)

    def scale(size):
        d = torch.rand(experts, rows, cols // be, 1, generator=g, device="cuda").mul_(0.6).add_(0.7).mul_(size).half()
        return d

    if type == "MXFP4":
        w[..., 0] = torch.randint(119, 122, w.shape[:-1], generator=g, device="cuda", dtype=torch.uint8)
    elif type == "Q8_0":
        w[..., :2] = _bytes_of(scale(0.02 / 74))
    elif type == "Q6_K":
        w[..., 208:] = _bytes_of(scale(0.02 / 74 / 18.5))
    else:
        top = 16 if type == "Q4_K" else 32  # dmin: so that the mins take away the values' mean
        d = scale(0.02 / 36 / (top * 0.43))
        w[..., :2], w[..., 2:4] = _bytes_of(d), _bytes_of((d.float() * (top - 1) / 2).half())
    return w.view(experts, rows, -1)


def _logits(g, tokens, experts):
    """Router logits: some experts are asked for often, some hardly ever."""
    return _normal(g, tokens, experts) + _normal(g, experts)


def _chosen(g, case):
    v, i = _logits(g, case["tokens"], case["experts"]).topk(case["used"], dim=-1)
    return i.to(torch.int32).contiguous(), torch.softmax(v, -1)


def _inputs(case, seed):
    g, kind = _rng(seed), case["kind"]
    s = SimpleNamespace(case=case, held=None)
    if kind == "norm":
        n, c = case["rows"], case["cols"]
        s.h, s.w_pre = _normal(g, n, c), 1 + 0.2 * _normal(g, c)
        s.y = _normal(g, n, c, dtype=_dtype(case["y"])) if case["y"] else None
        s.w_post = 1 + 0.2 * _normal(g, c) if case["post"] else None
        s.gate = None if case["gate"] == "none" else _normal(g, n if case["gate"] == "row" else 1, c)
        s.scale = 0.22 if case["y"] else 1.0
        s.x = torch.empty(n, c, device="cuda", dtype=_dtype(case["x"]))
    elif kind == "route":
        s.logits = _logits(g, case["tokens"], case["experts"])
        s.ids = torch.empty(case["tokens"], case["used"], device="cuda", dtype=torch.int32)
        s.weights = torch.empty(case["tokens"], case["used"], device="cuda")
    elif kind == "ffn":
        t, e, c, f = case["tokens"], case["experts"], case["embd"], case["ff"]
        s.ids, s.weights = _chosen(g, case)
        s.x = _normal(g, t, c, dtype=_dtype(case["io"]))
        s.y = _normal(g, t, c) if case["add"] else torch.empty(t, c, device="cuda", dtype=_dtype(case["io"]))
        s.w = [_weights(g, case["type"], e, f, c), _weights(g, case["type"], e, f, c), _weights(g, case["down"], e, c, f)]
        s.bias = [_normal(g, e, n) * 0.1 if case["bias"] else None for n in (f, f, c)]
    else:
        t, e, k = case["tokens"], case["experts"], case["used"]
        s.ids, _ = _chosen(g, case)
        s.x = _normal(g, t, k if case["per_slot"] else 1, case["cols"], dtype=_dtype(case["io"]))
        s.w = _weights(g, case["type"], e, case["rows"], case["cols"])
        s.bias = _normal(g, e, case["rows"]) * 0.1 if case["bias"] else None
        s.y = torch.empty(t, k, case["rows"], device="cuda", dtype=_dtype(case["io"]))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    torch.cuda.synchronize()  # the library's context has a stream of its own
    return s


# ---- the plain forms -----------------------------------------------------------------------------

def _dequant(type, w, cols):
    """Rows of GGUF blocks, uint8 [..., row bytes] -> float32 [..., cols]."""
    lead = w.shape[:-1]
    if type == "F16":
        return w.view(torch.float16).float()
    be, bb = BLOCK[type]
    b = w.view(*lead, cols // be, bb)

    def half(at):
        return b[..., at:at + 2].contiguous().view(torch.float16).float()

    if type == "Q8_0":
        return (half(0) * b[..., 2:].view(torch.int8).float()).view(*lead, cols)
    if type == "MXFP4":
        q = torch.cat([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
        code = (q & 7).float()  # 0 .5 1 1.5 2 3 4 6
        v = torch.where(code < 4, code * 0.5, torch.where(code < 6, code - 2, 2 * code - 8))
        v = torch.where(q >= 8, -v, v)
        return (v * torch.exp2(b[..., :1].float() - 127)).view(*lead, cols)
    if type == "Q6_K":
        n = lead + (cols // 256,)
        ql, qh = b[..., :128].reshape(*n, 2, 64), b[..., 128:192].reshape(*n, 2, 32)
        low = torch.stack([ql[..., :32] & 15, ql[..., 32:] & 15, ql[..., :32] >> 4, ql[..., 32:] >> 4], -2)
        high = torch.stack([qh & 3, (qh >> 2) & 3, (qh >> 4) & 3, qh >> 6], -2)
        q = (low | high << 4).float() - 32
        sc = b[..., 192:208].contiguous().view(torch.int8).float()
        return (half(208).unsqueeze(-1) * sc.unsqueeze(-1) * q.reshape(*n, 16, 16)).view(*lead, cols)
    s = b[..., 4:16]  # 6-bit scales and mins
    sc = torch.cat([s[..., :4] & 63, (s[..., 8:] & 15) | (s[..., :4] >> 6) << 4], -1).float()
    mn = torch.cat([s[..., 4:8] & 63, s[..., 8:] >> 4 | (s[..., 4:8] >> 6) << 4], -1).float()
    n = lead + (cols // 256,)
    qs = b[..., -128:].reshape(*n, 4, 32)
    q = torch.stack([qs & 15, qs >> 4], -2).reshape(*n, 8, 32)
    if type == "Q5_K":
        bit = torch.arange(8, device=w.device, dtype=torch.uint8).view(8, 1)
        q = q | ((b[..., 16:48].unsqueeze(-2) >> bit) & 1) << 4
    return ((half(0) * sc).unsqueeze(-1) * q.float() - (half(2) * mn).unsqueeze(-1)).view(*lead, cols)


def _plan(ids, experts):
    """Slots (a token's j-th expert) grouped by expert in tiles of `size`: (each tile's expert, each
    slot's place in the tiles). There are at most as many tiles as `count`."""
    n = ids.numel()
    size = 1 << max(0, min(8, (n // experts).bit_length()))
    count = min(n, n // size + experts)
    e, order = ids.reshape(-1).long().sort(stable=True)
    each = torch.zeros(experts, device=ids.device, dtype=torch.long).scatter_add_(0, e, torch.ones_like(e))
    tiles = (each + size - 1) // size
    end = tiles.cumsum(0)
    rank = torch.arange(n, device=ids.device) - (each.cumsum(0) - each)[e]
    place = torch.empty_like(e)
    place[order] = (end - tiles)[e] * size + rank
    expert = torch.searchsorted(end, torch.arange(count, device=ids.device), right=True).clamp(max=experts - 1)
    return SimpleNamespace(size=size, count=count, expert=expert, place=place, slot_expert=ids.reshape(-1).long())


def _grouped(p, type, w, x, bias):
    """W[expert of slot] x[slot] (+ bias) for x [slots, cols] float32."""
    cols = x.shape[1]
    t = torch.zeros(p.count * p.size, cols, device=x.device)
    t[p.place] = x
    t = t.view(p.count, p.size, cols).transpose(1, 2).contiguous()
    y = torch.bmm(_dequant(type, w[p.expert], cols), t)  # [tiles, rows, size]
    y = y.transpose(1, 2).reshape(p.count * p.size, -1)[p.place]
    return y if bias is None else y + bias[p.slot_expert]


def _act(case, g, u):
    if case["act"] == "silu":
        return g / (1 + torch.exp(-g)) * u
    g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
    return g / (1 + torch.exp(-ALPHA * g)) * (u + 1)


def _unit(v, eps=1e-5):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def _plain(s):
    case, kind = s.case, s.case["kind"]
    if kind == "norm":
        if s.y is not None:
            z = s.y.float()
            if s.w_post is not None:
                z = _unit(z) * s.w_post
            if s.gate is not None:
                z = z * s.gate
            s.h.add_(s.scale * z)
        s.x.copy_(_unit(s.h) * s.w_pre)
        return {"h": s.h, "x": s.x} if s.y is not None else {"x": s.x}
    if kind == "route":
        v, i = s.logits.sort(dim=-1, descending=True, stable=True)
        v, k = v[:, :case["used"]], case["used"]
        e = torch.exp(v - v[:, :1])
        total = e if case["over"] == "used" else torch.exp(s.logits - v[:, :1])
        s.ids.copy_(i[:, :k])
        s.weights.copy_(case["scale"] * e / total.sum(-1, keepdim=True))
        return {"ids": s.ids, "weights": s.weights}
    p = _plan(s.ids, case["experts"])
    if kind == "ffn":
        x = s.x.float().repeat_interleave(case["used"], 0)
        m = _act(case, _grouped(p, case["type"], s.w[0], x, s.bias[0]), _grouped(p, case["type"], s.w[1], x, s.bias[1]))
        o = _grouped(p, case["down"], s.w[2], m, s.bias[2]).view(*s.weights.shape, -1)
        o = (s.weights.unsqueeze(-1) * o).sum(1)
        if case["add"]:
            s.y.add_(o)
        else:
            s.y.copy_(o)
        return s.y
    x = s.x.float().expand(-1, case["used"], -1).reshape(-1, case["cols"])
    s.y.copy_(_grouped(p, case["type"], s.w, x, s.bias).view(s.y.shape))
    return s.y


# ---- the framework's calls -----------------------------------------------------------------------

_kept = {}


def _context():
    """The program's one context."""
    if "ctx" not in _kept:
        from moearc_amd import Context
        _kept["ctx"] = Context()
    return _kept["ctx"]


def _held(s):
    """The program's buffers of a state as the library sees them, and an expert layer's descriptor."""
    if s.held is None:
        from moearc_amd import DeviceView, MoeAct, MoeDesc, QuantType, RouteMode, OUT_F16, OUT_F32

        def view(t):
            if t is None:
                return None
            owner = SimpleNamespace(ctx=_context(), ptr=t.data_ptr(), len=t.numel() * t.element_size(), tensor=t)
            return DeviceView(owner, 0)

        c = s.case
        s.held = b = SimpleNamespace(ctx=_context())
        for name in ("h", "x", "y", "w_pre", "w_post", "gate", "logits", "ids", "weights"):
            setattr(b, name, view(getattr(s, name, None)))
        b.io = {"f16": OUT_F16, "f32": OUT_F32, None: OUT_F32}
        b.mode = RouteMode.SOFTMAX_SELECTED if c.get("over") == "used" else RouteMode.SOFTMAX_ALL
        if c["kind"] == "ffn":
            b.desc = MoeDesc.make([QuantType[c["type"]]] * 2 + [QuantType[c["down"]]], [view(w) for w in s.w],
                                  [view(x) for x in s.bias], c["experts"], c["embd"], c["ff"],
                                  MoeAct.SWIGLU if c["act"] == "silu" else MoeAct.SWIGLU_CLAMPED, ALPHA, LIMIT)
        if c["kind"] == "linear":
            b.type, b.w, b.bias = QuantType[c["type"]], view(s.w), view(s.bias)
    return s.held


def _own(s):
    b, c, kind = s.held or _held(s), s.case, s.case["kind"]
    if kind == "norm":
        b.ctx.norm_residual(b.x, b.h, b.y, b.w_post, b.gate, c["cols"] if c["gate"] == "row" else 0, s.scale, b.w_pre,
                            c["rows"], c["cols"], 1e-5, x_type=b.io[c["x"]], y_type=b.io[c["y"]])
        return {"h": s.h, "x": s.x} if s.y is not None else {"x": s.x}
    if kind == "route":
        b.ctx.moe_route(b.ids, b.weights, b.logits, c["tokens"], c["experts"], c["used"], b.mode, c["scale"])
        return {"ids": s.ids, "weights": s.weights}
    if kind == "ffn":
        b.ctx.moe_ffn(b.desc, b.y, b.x, b.ids, b.weights, c["tokens"], c["used"], io_type=b.io[c["io"]],
                      accumulate=c["add"])
        return s.y
    b.ctx.matmul_experts(b.type, b.y, b.w, b.x, b.bias, b.ids, c["tokens"], c["used"], c["experts"], c["rows"],
                         c["cols"], io_type=b.io[c["io"]], x_per_slot=c["per_slot"])
    return s.y


def run(s):
    if own:
        return _own(s)
    return _plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------

def _awake(case):
    """The number of experts that some token asks for, were all asked for alike."""
    return case["experts"] * (1 - (1 - case["used"] / case["experts"]) ** case["tokens"])


def _size(type, n):
    return n * BLOCK[type][1] / BLOCK[type][0]


def work(case):
    kind, io = case["kind"], 2 if case.get("io") == "f16" else 4
    if kind == "norm":
        n, c = case["rows"], case["cols"]
        y = {None: 0, "f16": 2, "f32": 4}[case["y"]]
        per = 4 + (y + 4 if y else 0) + (2 if case["x"] == "f16" else 4) + (4 if case["gate"] == "row" else 0)
        return {"bytes": n * c * per + 4 * c * (1 + case["post"] + (case["gate"] == "shared")),
                "flops": n * c * (4 + (3 if y else 0) + (4 if case["post"] else 0))}
    t, k = case["tokens"], case["used"]
    if kind == "route":
        return {"bytes": 4 * t * case["experts"] + 8 * t * k, "flops": t * case["experts"] * 4}
    if kind == "ffn":
        c, f = case["embd"], case["ff"]
        weights = 2 * _size(case["type"], f * c) + _size(case["down"], f * c) + (4 * (2 * f + c) if case["bias"] else 0)
        return {"bytes": _awake(case) * weights + t * c * (2 * io + (io if case["add"] else 0)) + 8 * t * k,
                "flops": 6 * t * k * c * f}
    r, c = case["rows"], case["cols"]
    return {"bytes": _awake(case) * (_size(case["type"], r * c) + 4 * r * case["bias"]) +
            t * c * io * (k if case["per_slot"] else 1) + t * k * (r * io + 4), "flops": 2 * t * k * r * c}


# ---- in 64 bits, from the definition ---------------------------------------------------------------

def _matrix(type, raw, rows, cols):
    """One expert's matrix in float64, block by block as the format defines it."""
    if type == "F16":
        return raw.view(torch.float16).double()
    be, bb = BLOCK[type]
    b = raw.view(rows * (cols // be), bb).to(torch.int64)
    out = torch.empty(b.shape[0], be, device=raw.device, dtype=torch.float64)

    def f16(lo):
        return raw.view(-1, bb)[:, lo:lo + 2].contiguous().view(torch.float16).double()

    if type == "Q8_0":
        out[:] = f16(0) * torch.where(b[:, 2:] > 127, b[:, 2:] - 256, b[:, 2:])
    elif type == "MXFP4":
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=raw.device,
                             dtype=torch.float64)
        size = torch.exp2((b[:, :1] - 127).double())
        out[:, :16], out[:, 16:] = table[b[:, 1:] % 16] * size, table[b[:, 1:] // 16] * size
    elif type == "Q6_K":
        d = f16(208)
        for j in range(16):  # 16 elements to a scale: half j / 8, quarter j / 2 % 4, side j % 2
            h, quarter, side = j // 8, j // 2 % 4, j % 2
            at = 64 * h + 32 * (quarter % 2) + 16 * side
            low = b[:, at:at + 16] // (16 if quarter > 1 else 1) % 16
            at = 128 + 32 * h + 16 * side
            q = low + 16 * (b[:, at:at + 16] // 4 ** quarter % 4) - 32
            s = b[:, 192 + j:193 + j]
            out[:, 16 * j:16 * j + 16] = d * torch.where(s > 127, s - 256, s) * q
    else:
        d, dmin = f16(0), f16(2)
        for j in range(8):  # 32 elements to a scale and a min
            if j < 4:
                s, m = b[:, 4 + j] % 64, b[:, 8 + j] % 64
            else:
                s, m = b[:, 8 + j] % 16 + 16 * (b[:, j] // 64), b[:, 8 + j] // 16 + 16 * (b[:, 4 + j] // 64)
            at = bb - 128 + 32 * (j // 2)
            q = b[:, at:at + 32] // (16 if j % 2 else 1) % 16
            if type == "Q5_K":
                q = q + 16 * (b[:, 16:48] // 2 ** j % 2)
            out[:, 32 * j:32 * j + 32] = d * s.unsqueeze(1) * q - dmin * m.unsqueeze(1)
    return out.view(rows, cols)


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind == "norm":
        h = s.h.double()

        def rms(v):
            return v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-5)

        if s.y is not None:
            z = s.y.double()
            z = rms(z) * s.w_post.double() if case["post"] else z
            z = z * s.gate.double() if s.gate is not None else z
            h = h + s.scale * z
        x = rms(h) * s.w_pre.double()
        return {"h": h, "x": x} if s.y is not None else {"x": x}
    k = case["used"]
    if kind == "route":
        at = torch.argsort(-s.logits.double(), dim=1, stable=True)[:, :k]
        if case["over"] == "used":
            w = torch.softmax(s.logits.double().gather(1, at), 1)
        else:
            w = torch.softmax(s.logits.double(), 1).gather(1, at)
        return {"ids": at.to(torch.int32), "weights": w * case["scale"]}
    ids = s.ids.long()
    if kind == "linear":
        y = torch.zeros(*s.y.shape, device="cuda", dtype=torch.float64)
        for e in range(case["experts"]):
            t, j = (ids == e).nonzero(as_tuple=True)
            if len(t):
                x = s.x[t, j if case["per_slot"] else torch.zeros_like(j)].double()
                y[t, j] = x @ _matrix(case["type"], s.w[e], case["rows"], case["cols"]).t().contiguous()
                if case["bias"]:
                    y[t, j] += s.bias[e].double()
        return y
    y = s.y.double() if case["add"] else torch.zeros(s.y.shape, device="cuda", dtype=torch.float64)
    for e in range(case["experts"]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        v = [s.x[t].double() @ _matrix(case["type"], s.w[i][e], case["ff"], case["embd"]).t().contiguous() for i in (0, 1)]
        if case["bias"]:
            v = [v[i] + s.bias[i][e].double() for i in (0, 1)]
        if case["act"] == "silu":
            m = v[0] * torch.sigmoid(v[0]) * v[1]
        else:
            g = torch.minimum(v[0], torch.tensor(LIMIT, device="cuda", dtype=torch.float64))
            m = g * torch.sigmoid(ALPHA * g) * (v[1].clamp(-LIMIT, LIMIT) + 1)
        o = m @ _matrix(case["down"], s.w[2][e], case["embd"], case["ff"]).t().contiguous()
        if case["bias"]:
            o = o + s.bias[2][e].double()
        y.index_add_(0, t, s.weights[t, j].double().unsqueeze(1) * o)
    return y
