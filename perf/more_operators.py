"""What the attention half of a block is asked to do for a ragged batch in use, case by case, through
`moearc_amd.Context`: sequences with any number of new tokens each (decode steps, drafts to verify, chunks
of prompts) behind a paged cache, beside the single-sequence calls that `perf/cases.py` holds.

Two kinds of call, in the sizes a program that serves a model makes them:

* ``append``  ``rope_qkv_append_batched``: q and k normed head by head where the model has such norms and
              rotated at their positions, q written for the attention, k and v into their pages.
* ``attend``  ``attn_prefill_batched``: every new token's attention over its sequence's keys up to its own,
              or over the last ``window`` of them, with the heads' sinks where the model has them.

A sequence of n new tokens behind ``cached`` ones holds n + cached keys; its tokens sit at the last n
positions. Inputs are made on the GPU from a seed: N(0,1) queries, keys and values, caches in pages
scattered by a random permutation. Every buffer is a torch tensor that the library sees through a
``DeviceView``, as a program that holds its model in torch would pass it.

Where ``own`` is false the plain forms compute the same in float32 torch operations, angles in float64.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6  # of the heads' norms
YARN = dict(n_ctx_orig=4096, factor=32.0)  # the long-context scaling of the rotation


# ---- the cases -----------------------------------------------------------------------------------

def _append(name, seqs, new, cached, heads, kv_heads, dim, rot=None, neox=True, base=150000.0, yarn=False, factors=False,
            norm=False, fused=False, io="f32", q="f16", kv="f16", page=256, lens=1, mix="all"):
    """new, cached: the least and the most of a sequence; fused: q, k and v are one product's rows; mix: "all"
    sequences have new tokens by that range, some are "idle", or most are "steps" of one token."""
    c = dict(kind="append", seqs=seqs, new_min=new[0], new_max=new[1], cached_min=cached[0], cached_max=cached[1],
             heads=heads, kv_heads=kv_heads, dim=dim, rot=dim if rot is None else rot, neox=neox, base=base, yarn=yarn,
             factors=factors, norm=norm, fused=fused, io=io, q=q, kv=kv, page=page, lens=lens, mix=mix)
    return dict(name=name, **c) if name else c


def _attend(name, seqs, new, cached, heads, kv_heads, dim, window=0, sinks=False, page=256, out="f16", lens=1, mix="all"):
    c = dict(kind="attend", seqs=seqs, new_min=new[0], new_max=new[1], cached_min=cached[0], cached_max=cached[1],
             heads=heads, kv_heads=kv_heads, dim=dim, window=window, sinks=sinks, page=page, out=out, lens=lens, mix=mix)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # One user's decode step: latency. f32 queries, as the decode attention takes them.
        _append("append_step", 1, (1, 1), (4095, 4095), 64, 8, 64, yarn=True, q="f32"),
        # A decode step of 48 sequences with normed heads of 128 channels.
        _append("append_b48_norm", 48, (1, 1), (100, 20000), 32, 4, 128, base=1e6, norm=True),
        # A long prompt's chunk, q, k and v the rows of one product.
        _append("append_chunk_2k", 1, (2048, 2048), (2048, 2048), 64, 8, 64, yarn=True, fused=True),
        # A dozen prompts of mixed lengths, interleaved pairs in half of each head, their frequencies scaled
        # one by one, f16 products, an f32 cache in odd pages.
        _append("append_ragged_part", 12, (40, 900), (1, 3000), 32, 8, 128, rot=64, neox=False, base=500000.0, factors=True,
                io="f16", kv="f32", page=48),
        # Four users' drafts of a few tokens to verify: latency. Precise outputs.
        _attend("attend_drafts", 4, (3, 7), (500, 3000), 64, 8, 64, sinks=True, out="f32"),
        # A continuous batch's step: most sequences decode a token, some bring a piece of a prompt.
        _attend("attend_mixed_b32", 32, (1, 400), (200, 8000), 32, 4, 128, lens=3, mix="steps"),
        # Prompts of many lengths from the start, a windowed layer.
        _attend("attend_prompts_window", 16, (30, 1500), (0, 0), 64, 8, 64, window=128, sinks=True),
        # Four long prompts, a full layer of heads of 64.
        _attend("attend_prompts_2k", 4, (2048, 2048), (0, 0), 64, 8, 64, sinks=True),
        # One prompt, heads of 128: the matrix cores' case.
        _attend("attend_prompt_4k_d128", 1, (4096, 4096), (0, 0), 32, 4, 128),
        # A follow-up question behind a long document: the largest.
        _attend("attend_512_at_32k", 1, (512, 512), (32700, 32700), 32, 4, 128),
        # Odd sizes everywhere: 80 channels, five heads to a KV head, pages of 48, precise outputs.
        _attend("attend_odd", 6, (50, 700), (10, 900), 20, 4, 80, page=48, out="f32"),
    ]


def _log_int(rng, lo, hi):
    """Spread over the logarithm of lo .. hi."""
    if lo >= hi:
        return lo
    at = math.log(lo + 1) + rng.random() * (math.log(hi + 2) - math.log(lo + 1))
    return max(lo, min(hi, int(math.exp(at)) - 1))


def draw(rng):
    while True:
        seqs = rng.choice([1, 1, 2, 3, 5, 8, 13, 24, 48, 64])
        top = _log_int(rng, 1, 4096 if seqs < 4 else 900)
        new = (rng.choice([1, max(1, top // 4), top]), top)
        far = rng.choice([0, _log_int(rng, 1, 3000), _log_int(rng, 16, 32000 if seqs < 4 else 8000)])
        cached = (far // rng.choice([1, 4, 16]), far)
        heads, kv_heads, dim = rng.choice([(64, 8, 64), (64, 8, 64), (32, 4, 128), (32, 4, 128), (32, 8, 128), (16, 16, 128),
                                           (20, 4, 80), (12, 2, 96), (14, 2, 64), (16, 2, 256), (8, 1, 128)])
        page, lens, mix = rng.choice([16, 256, 256, 48]), rng.randrange(1 << 20), rng.choice(["all", "all", "idle", "steps"])
        if rng.random() < 0.4:
            c = _append(None, seqs, new, cached, heads, kv_heads, dim, rng.choice([dim, dim, dim // 2]), rng.choice([True, True, False]),
                        rng.choice([10000.0, 150000.0, 500000.0, 1e6]), rng.choice([False, True]), rng.choice([False, False, True]),
                        rng.choice([False, True]), rng.choice([False, True]), rng.choice(["f32", "f32", "f16"]),
                        rng.choice(["f16", "f16", "f32"]), rng.choice(["f16", "f16", "f32"]), page, lens, mix)
        else:
            c = _attend(None, seqs, new, cached, heads, kv_heads, dim, rng.choice([0, 0, 128, 1024]), rng.choice([False, True]), page,
                        rng.choice(["f16", "f16", "f32"]), lens, mix)
        new, kv = _lengths(c)
        whole = 4 * sum(m * n for m, n in zip(new, kv)) * heads * dim if c["kind"] == "attend" else 0  # without any mask
        if 0 < sum(new) <= 9000 and sum(kv) <= 200000 and whole <= 2.7e11:
            return c


def _lengths(case):
    """Each sequence's new tokens and its keys, these among them."""
    r = random.Random(case["lens"])
    new, kv = [], []
    for b in range(case["seqs"]):
        n = _log_int(r, case["new_min"], case["new_max"])
        c = _log_int(r, case["cached_min"], case["cached_max"])
        if case["mix"] == "idle" and b % 6 == 4:
            n = 0
        if case["mix"] == "steps" and b % 8 != 3:
            n = 1
        new.append(n)
        kv.append(n + c)
    return new, kv


# ---- inputs --------------------------------------------------------------------------------------

def _dtype(io):
    return torch.float16 if io == "f16" else torch.float32


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = SimpleNamespace(case=case, held=None)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    s.new, s.kv = _lengths(case)
    s.rows = [0]
    for n in s.new:
        s.rows.append(s.rows[-1] + n)
    total = s.rows[-1]
    counts = [-(-n // page) for n in s.kv]
    s.pages, s.stride = sum(counts), max(counts)
    perm = torch.randperm(s.pages, generator=g, device="cuda").to(torch.int32)
    s.tables = torch.zeros(len(counts), s.stride, device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        s.tables[b, :n] = perm[at:at + n]
        at += n
    kv_type = _dtype(case.get("kv", "f16"))
    s.k_pages = normal(s.pages, page, kv_heads, dim, dtype=kv_type)
    s.v_pages = normal(s.pages, page, kv_heads, dim, dtype=kv_type)
    if case["kind"] == "append":
        io = _dtype(case["io"])
        if case["fused"]:
            s.qkv = normal(total, heads + 2 * kv_heads, dim, dtype=io)
            s.q, s.k, s.v = s.qkv.split([heads, kv_heads, kv_heads], 1)
        else:
            s.q, s.k, s.v = (normal(total, n, dim, dtype=io) for n in (heads, kv_heads, kv_heads))
        s.q_norm, s.k_norm = ((1 + 0.2 * normal(dim) for _ in range(2)) if case["norm"] else (None, None))
        # as such tables come: ones for the fast pairs, up to eight for the slow ones
        s.factors = (1 + 7 * torch.linspace(-1, 1, case["rot"] // 2, device="cuda").clamp(min=0) *
                     torch.rand(case["rot"] // 2, generator=g, device="cuda")) if case["factors"] else None
        s.q_out = torch.empty(total, heads, dim, device="cuda", dtype=_dtype(case["q"]))
    else:
        s.q = normal(total, heads, dim, dtype=torch.float16)
        s.sinks = normal(heads) if case["sinks"] else None
        s.out = torch.empty(total, heads, dim, device="cuda", dtype=_dtype(case["out"]))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    torch.cuda.synchronize()  # the library's context has a stream of its own
    return s


# ---- the plain forms -----------------------------------------------------------------------------

def _corrections(case):
    """The pairs between which the long-context scaling fades in."""
    rot, ctx, base = case["rot"], YARN["n_ctx_orig"], case["base"]

    def pair(turns):
        return rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))

    return max(math.floor(pair(32.0)), 0.0), min(math.ceil(pair(1.0)), rot - 1.0)


def _positions(s):
    return torch.cat([torch.arange(n - m, n, device="cuda") for m, n in zip(s.new, s.kv)])


def _places(s, pos):
    """Each row's place in the pools as one index over pages and slots."""
    seq = torch.cat([torch.full((m,), b, device="cuda", dtype=torch.long) for b, m in enumerate(s.new)])
    page = s.case["page"]
    return s.tables[seq, pos // page].long() * page + pos % page


def _cos_sin(case, pos, factors):
    j = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
    f = case["base"] ** (-2 * j / case["rot"])
    if factors is not None:
        f = f / factors
    size = 1.0
    if case["yarn"]:
        lo, hi = _corrections(case)
        far = 1 - ((j - lo) / max(0.001, hi - lo)).clamp(0, 1)  # 1: as it is, 0: interpolated
        f = f * ((1 - far) / YARN["factor"] + far)
        size = 1 + 0.1 * math.log(YARN["factor"])
    angle = pos.double().unsqueeze(1) * f
    return (torch.cos(angle) * size).float().unsqueeze(1), (torch.sin(angle) * size).float().unsqueeze(1)


def _rotated(case, x, w, cos, sin):
    x, rot = x.float(), case["rot"]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    if case["neox"]:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    a, b = a * cos - b * sin, a * sin + b * cos
    y = torch.cat([a, b], -1) if case["neox"] else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain(s):
    case = s.case
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        pos = _positions(s)
        cos, sin = _cos_sin(case, pos, s.factors)
        at = _places(s, pos)
        s.q_out.copy_(_rotated(case, s.q, s.q_norm, cos, sin))
        s.k_pages.view(-1, kv_heads, dim)[at] = _rotated(case, s.k, s.k_norm, cos, sin).to(s.k_pages.dtype)
        s.v_pages.view(-1, kv_heads, dim)[at] = s.v.to(s.v_pages.dtype)
        return {"q": s.q_out, "k_pages": s.k_pages, "v_pages": s.v_pages}
    group = heads // kv_heads
    for b, (m, n) in enumerate(zip(s.new, s.kv)):
        if m == 0:
            continue
        r, first = s.rows[b], max(0, n - m + 1 - case["window"]) if case["window"] else 0
        table = s.tables[b, :-(-n // page)].long()
        k = s.k_pages[table].view(-1, kv_heads, dim)[first:n].float().transpose(0, 1)
        v = s.v_pages[table].view(-1, kv_heads, dim)[first:n].float().transpose(0, 1)
        q = s.q[r:r + m].float().view(m, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * m, dim)
        row, key = torch.arange(n - m, n, device="cuda").view(m, 1), torch.arange(first, n, device="cuda")
        hidden = key > row
        if case["window"]:
            hidden |= key <= row - case["window"]
        for h in range(kv_heads):
            x = (q[h] @ k[h].t()).view(group, m, n - first).mul_(dim ** -0.5).masked_fill_(hidden, -math.inf)
            top = x.amax(-1, keepdim=True)
            if s.sinks is not None:
                sink = s.sinks[h * group:(h + 1) * group].view(group, 1, 1)
                top = torch.maximum(top, sink)
            x = x.sub_(top).exp_()
            total = x.sum(-1, keepdim=True)
            if s.sinks is not None:
                total = total + torch.exp(sink - top)
            o = (x.view(group * m, -1) @ v[h]).view(group, m, dim) / total
            s.out[r:r + m, h * group:(h + 1) * group] = o.transpose(0, 1).to(s.out.dtype)
    return s.out


# ---- the framework's calls -----------------------------------------------------------------------

_kept = {}


def _context():
    """The program's one context."""
    if "ctx" not in _kept:
        from moearc_amd import Context
        _kept["ctx"] = Context()
    return _kept["ctx"]


def _held(s):
    """The program's buffers of a state as the library sees them, and a layer's descriptor of its rows."""
    if s.held is None:
        import numpy as np
        from moearc_amd import DeviceView, KvType, OUT_F16, OUT_F32, QkvAppendDesc, RopeKind, RopeScaling

        def view(t):
            if t is None:
                return None
            size = t.element_size()
            owner = SimpleNamespace(ctx=_context(), ptr=t.data_ptr(), tensor=t,
                                    len=size * (sum((n - 1) * m for n, m in zip(t.shape, t.stride())) + 1))
            return DeviceView(owner, 0)

        c = s.case
        s.held = b = SimpleNamespace(ctx=_context(), rows=np.array(s.rows, np.uint32), kv=np.array(s.kv, np.uint32))
        for name in ("q", "out", "k_pages", "v_pages", "tables", "sinks"):
            setattr(b, name, view(getattr(s, name, None)))
        types = {"f16": OUT_F16, "f32": OUT_F32}
        if c["kind"] == "append":
            scaling = RopeScaling.yarn(c["rot"], YARN["n_ctx_orig"], c["base"], YARN["factor"]) if c["yarn"] else None
            b.desc = QkvAppendDesc.make(
                view(s.q), view(s.k), view(s.v), view(s.q_out), b.k_pages, b.v_pages, s.pages, c["heads"], c["kv_heads"],
                c["dim"], c["page"], c["rot"], c["base"], scaling, RopeKind.NEOX if c["neox"] else RopeKind.NORMAL,
                in_type=types[c["io"]], q_type=types[c["q"]], kv=KvType.F16 if c["kv"] == "f16" else KvType.F32,
                q_stride=s.q.stride(0), k_stride=s.k.stride(0), v_stride=s.v.stride(0), q_norm=view(s.q_norm),
                k_norm=view(s.k_norm), eps=EPS, freq_factors=view(s.factors))
        else:
            b.scale, b.out_type = c["dim"] ** -0.5, types[c["out"]]
    return s.held


def _own(s):
    b, c = s.held or _held(s), s.case
    if c["kind"] == "append":
        b.ctx.rope_qkv_append_batched(b.desc, b.tables, s.stride, b.rows, b.kv)
        return {"q": s.q_out, "k_pages": s.k_pages, "v_pages": s.v_pages}
    b.ctx.attn_prefill_batched(b.out, b.q, b.k_pages, b.v_pages, s.pages, b.tables, s.stride, b.rows, b.kv, b.sinks,
                               c["window"], c["heads"], c["kv_heads"], c["dim"], c["page"], b.scale, out_type=b.out_type)
    return s.out


def run(s):
    if own:
        return _own(s)
    return _plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    new, kv = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size = {"f16": 2, "f32": 4}
    if case["kind"] == "append":
        per = (heads + 2 * kv_heads) * dim * size[case["io"]] + heads * dim * size[case["q"]] + 2 * kv_heads * dim * size[case["kv"]]
        return {"bytes": sum(new) * per, "flops": sum(new) * (heads + kv_heads) * (3 * case["rot"] + 4 * dim * case["norm"])}
    w = case["window"]
    seen = pairs = 0
    for m, n in zip(new, kv):
        if m:
            seen += min(n, m + w - 1) if w else n
            whole = max(0, min(m, w - (n - m))) if w else m  # rows whose window reaches back to the first key
            pairs += whole * (n - m) + whole * (whole + 1) // 2 + (m - whole) * w
    return {"bytes": seen * kv_heads * dim * 4 + sum(new) * heads * dim * (2 + size[case["out"]]),
            "flops": 4 * pairs * heads * dim}


# ---- in 64 bits, from the definition ---------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "append":
        half = case["rot"] // 2
        angle_per = torch.empty(half, device="cuda", dtype=torch.float64)
        size = 1.0
        for j in range(half):
            f = math.exp(-2 * j / case["rot"] * math.log(case["base"]))
            if s.factors is not None:
                f /= float(s.factors[j])
            if case["yarn"]:
                size = 1 + 0.1 * math.log(YARN["factor"])
                lo, hi = _corrections(case)
                ramp = min(1.0, max(0.0, (j - lo) / max(0.001, hi - lo)))
                f = f / YARN["factor"] * ramp + f * (1 - ramp)
            angle_per[j] = f
        q_out = s.q.double().clone()
        k_new = s.k.double().clone()
        k_pages, v_pages = s.k_pages.double(), s.v_pages.double()
        for x, w in ((q_out, s.q_norm), (k_new, s.k_norm)):
            if w is not None:
                x *= torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / dim + EPS) * w.double()
        for b, (m, n) in enumerate(zip(s.new, s.kv)):
            if m == 0:
                continue
            at = slice(s.rows[b], s.rows[b] + m)
            turn = torch.outer(torch.arange(n - m, n, device="cuda", dtype=torch.float64), angle_per)
            turn = torch.polar(torch.full_like(turn, size), turn).unsqueeze(1)
            for x in (q_out, k_new):
                part = x[at, :, :2 * half]
                if case["neox"]:
                    z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
                    part.copy_(torch.cat([z.real, z.imag], -1))
                else:
                    z = torch.view_as_complex(part.reshape(m, -1, half, 2).contiguous()) * turn
                    part.copy_(torch.view_as_real(z).reshape(m, -1, 2 * half))
            for i in range(m):
                p = n - m + i
                if i == 0 or p % page == 0:
                    take = min(m - i, page - p % page)
                    where = int(s.tables[b, p // page])
                    k_pages[where, p % page:p % page + take] = k_new[s.rows[b] + i:s.rows[b] + i + take]
                    v_pages[where, p % page:p % page + take] = s.v[s.rows[b] + i:s.rows[b] + i + take].double()
        return {"q": q_out, "k_pages": k_pages, "v_pages": v_pages}
    out = torch.empty(s.rows[-1], heads, dim, device="cuda", dtype=torch.float64)
    for b, (m, n) in enumerate(zip(s.new, s.kv)):
        place = torch.arange(n, device="cuda")
        place = s.tables[b].long()[place // page] * page + place % page
        for lo in range(0, m, 512):  # rows at a time, each head by itself
            hi = min(m, lo + 512)
            pos = torch.arange(n - m + lo, n - m + hi, device="cuda").unsqueeze(1)
            first = max(0, n - m + lo + 1 - case["window"]) if case["window"] else 0
            key = torch.arange(first, n - m + hi, device="cuda")
            sees = key <= pos
            if case["window"]:
                sees &= pos - key < case["window"]
            for h in range(heads):
                at = place[first:n - m + hi]
                k = s.k_pages.view(-1, kv_heads, dim)[at, h * kv_heads // heads].double()
                v = s.v_pages.view(-1, kv_heads, dim)[at, h * kv_heads // heads].double()
                score = s.q[s.rows[b] + lo:s.rows[b] + hi, h].double() @ k.t() / math.sqrt(dim)
                score = torch.where(sees, score, torch.full_like(score, -math.inf))
                if s.sinks is not None:
                    score = torch.cat([score, s.sinks[h].double().expand(hi - lo, 1)], 1)
                    v = torch.cat([v, torch.zeros(1, dim, device="cuda", dtype=torch.float64)])
                out[s.rows[b] + lo:s.rows[b] + hi, h] = torch.softmax(score, 1) @ v
    return out
