"""The operators of a K/V cache held in 8 bits, as cases to time.

A pool of e4m3 tiles of 16 tokens and one KV head, each with one power of two as its scale, holds twice the tokens of
a bf16 pool and halves what a decode step reads. Its operators are the steps that write it (`append`, and
`rope_append`, which normalises and rotates q and k first), the one that reads it back (`gather`), and the attention
over it: one new token per sequence (`decode_step`, which appends it too) and chunks of new tokens (`extend`).

Shapes are those of the benchmark configurations (28 query heads over 4 KV heads of 128 in bf16; 14 over 2 of 64 in
f32; 8 over 1 of 256) and draws of like ones. Lengths and tables are a function of the case; contents of the seed. One
layer's call is one pass.

The pool's tensors are in the tile order of the library: K [D/16][16 tokens][16 dims], V [D/64][4 token quads][16 dim
quads][4 dims][4 tokens], one tile per (K or V, block, head).
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False  # set from outside: False the plain forms, True the library's kernels

DEV = "cuda:0"
PAGE = 16
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
E_MIN = -100  # the least exponent of a tile
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------


def listed():
    big = dict(hkv=4, g=7, d=128, type="bf16")
    small = dict(hkv=2, g=7, d=64, type="f32")
    return [
        # The decode step of the ordinary batch: one row per sequence into a block that is partly full.
        dict(name="append_step", op="append", **big, seqs=64, lo=1, hi=1, past_lo=1000, past_hi=8000, lens=1),
        # A prefill step of 16 prompts' chunks, some of which begin inside a block.
        dict(name="append_prompts", op="append", **big, seqs=16, lo=700, hi=1300, past_lo=0, past_hi=40, lens=2),
        # The small f32 model's decode step, far into its context, rotated in the half layout, no norm.
        dict(name="rope_step_f32", op="rope_append", **small, seqs=8, lo=1, hi=1, past_lo=100, past_hi=600, lens=3,
             rd=64, interleaved=False, norm=False, gated=False, factor=1.0, base=0),
        # Chunks of a long-context model: half the head rotated in pairs, positions up to a million, scaled cos and sin.
        dict(name="rope_prompts", op="rope_append", **big, seqs=32, lo=512, hi=512, past_lo=0, past_hi=2000, lens=4,
             rd=64, interleaved=True, norm=True, gated=True, factor=1.2079, base=1000000),
        # A few short sequences read back, as for a layer that wants its cache in one piece.
        dict(name="gather_small_f32", op="gather", **small, seqs=8, past_lo=100, past_hi=600, lens=5),
        # The ordinary batch read back.
        dict(name="gather_batch", op="gather", **big, seqs=64, past_lo=1000, past_hi=8000, lens=6),
        # One user's decode step after a long context: latency.
        dict(name="decode_one", op="decode", **big, seqs=1, past_lo=8191, past_hi=8191, lens=7),
        # The ordinary serving step.
        dict(name="decode_batch", op="decode", **big, seqs=64, past_lo=1000, past_hi=8000, lens=8),
        # The small f32 model's step.
        dict(name="decode_small_f32", op="decode", **small, seqs=8, past_lo=100, past_hi=600, lens=9),
        # Draft checking and short turns after long contexts.
        dict(name="extend_short", op="extend", **big, seqs=16, lo=5, hi=24, past_lo=4000, past_hi=8000, lens=10),
        # A prefill step of chunks after a common length.
        dict(name="extend_chunks", op="extend", **big, seqs=8, lo=512, hi=512, past_lo=4096, past_hi=4096, lens=11),
        # The small f32 model's prompts.
        dict(name="extend_prompts_f32", op="extend", **small, seqs=8, lo=32, hi=512, past_lo=0, past_hi=0, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "rope_append", "gather", "decode", "decode", "extend", "extend"])
    hkv, g = rng.choice([(1, 8), (1, 16), (2, 7), (2, 4), (3, 5), (4, 7), (4, 1), (8, 4), (8, 1), (5, 3)])
    d, t = rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "bf16", "f32"])
    c = dict(op=op, hkv=hkv, g=g, d=d, type=t, lens=rng.randrange(1 << 30))
    if op in ("append", "rope_append"):
        rows = max(64, min(16384, 16384 * 36 * 128 // ((hkv * (g + 2) if op == "rope_append" else 9 * hkv) * d)))
        hi = _log(rng, 1, rows)
        c.update(seqs=_log(rng, 1, min(256, rows // hi)), lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, past_lo=0,
                 past_hi=_log(rng, 1, 3000))
        if op == "rope_append":
            c.update(rd=rng.choice([d, d, d // 2, d // 4, 8 * rng.randrange(1, d // 8)]), norm=rng.random() < 0.5,
                     interleaved=rng.random() < 0.5, gated=rng.random() < 0.5, factor=rng.choice([1.0, 1.3466]),
                     base=rng.choice([0, 0, 30000, 900000]))
        return c
    tokens = max(256, min(1 << 19, 64 * 4500 * 4 * 128 // (hkv * d)))
    if op == "gather" or op == "decode":
        past = _log(rng, 1, min(tokens, 40000))
        return dict(c, seqs=_log(rng, 1, min(256, max(1, tokens // past))), past_lo=rng.choice([0, past // 3, past]),
                    past_hi=past)
    flops = (250 << 30) // (16 if t == "f32" else 1)
    past = _log(rng, 1, 16000)
    hi = _log(rng, 1, min(2048, max(1, flops // (4 * hkv * g * d * (past + 2048)))))
    most = max(1, min(64, flops // (4 * hkv * g * d * hi * (past + hi)), tokens // (past + hi)))
    return dict(c, seqs=_log(rng, 1, most), lo=rng.choice([0, 1, hi // 2, hi]), hi=hi,
                past_lo=rng.choice([0, past // 2, past]), past_hi=past)


def _lengths(c):
    """New tokens and the tokens after them, of every sequence; the first one has the most."""
    r = random.Random(c["lens"])
    past = [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["seqs"])]
    past[0] = c["past_hi"]
    if c["op"] == "gather":
        return [0] * c["seqs"], past
    new = [1 if c["op"] == "decode" else r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    new[0] = 1 if c["op"] == "decode" else c["hi"]
    return new, [a + b for a, b in zip(past, new)]


def _tables(c):
    """Number of blocks, indptr and the ids of every sequence's blocks, scattered over the pool."""
    _, ctx = _lengths(c)
    need = [-(-n // PAGE) for n in ctx]
    total = sum(need) + 3
    ids = np.array(random.Random(c["lens"] + 1).sample(range(total), sum(need)), np.int32)
    return total, np.concatenate([[0], np.cumsum(need)]).astype(np.int32), ids


def work(c):
    new, ctx = _lengths(c)
    es, row = 4 if c["type"] == "f32" else 2, c["hkv"] * c["d"]
    n, total, op, hq = sum(new), sum(ctx), c["op"], c["hkv"] * c["g"]
    blocks = sum(-(-x // PAGE) for x in ctx)
    q = n * hq * c["d"] * es
    if op == "append":
        return {"bytes": n * row * 2 * (es + 1), "flops": 4 * n * row}
    if op == "rope_append":
        return {"bytes": 2 * q + n * row * 2 * (es + 1), "flops": 10 * n * (hq + c["hkv"]) * c["d"]}
    if op == "gather":
        return {"bytes": total * row * 2 * (1 + es) + 2 * blocks * c["hkv"], "flops": 2 * total * row}
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(new, ctx))
    size = total * row * 2 + 2 * blocks * c["hkv"] + 2 * q + (n * row * 2 * es if op == "decode" else 0)
    return {"bytes": size, "flops": 4 * hq * c["d"] * pairs}


# ---- inputs -----------------------------------------------------------------


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _fill(c, g, blocks):
    """A pool's tiles and exponents: rows of uneven size from block to block, with large channels in K."""
    hkv, d = c["hkv"], c["d"]
    kv = torch.empty(2, blocks, hkv, PAGE * d, dtype=F8, device=DEV)
    ex = torch.empty(2, blocks, hkv, dtype=torch.int8, device=DEV)
    for p in range(2):
        x = _normal(g, blocks, hkv, PAGE * d) * torch.exp2(2 * torch.rand(blocks, hkv, 1, generator=g, device=DEV) - 1)
        if p == 0:
            x = (x.view(blocks, hkv, d // 16, 16, 16) * _channels(g, hkv, d).view(hkv, d // 16, 1, 16)).view(x.shape)
        e = _exponent(x.abs().amax(-1))
        kv[p] = (x * torch.exp2(-e.float())[..., None]).to(F8)
        ex[p] = e
    return kv, ex


def _channels(g, hkv, d):
    return torch.exp(0.7 * _normal(g, hkv, d))


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    t = TYPES[c["type"]]
    new, ctx = _lengths(c)
    blocks, indptr, ids = _tables(c)
    n, hkv, d = sum(new), c["hkv"], c["d"]
    hq = hkv * c["g"]
    s = dict(case=c, new=new, ctx=ctx, indptr=indptr, ids=ids, scale=d ** -0.5)
    s["kv"], s["exp"] = _fill(c, g, blocks)
    chan = _channels(g, hkv, d)
    if c["op"] != "gather":
        s["k"], s["v"] = (_normal(g, n, hkv, d) * chan).to(t), _normal(g, n, hkv, d).to(t)
        s["q"] = _normal(g, n, hq, d).to(t)
    if c["op"] == "rope_append":
        if c["gated"]:
            s["q"] = torch.stack([s["q"], _normal(g, n, hq, d).to(t)], 2)
        s["wq"], s["wk"] = 0.2 * _normal(g, d), 0.2 * _normal(g, d)
        # Frequencies of a base of a million; positions of a sequence start where its earlier part, held elsewhere, ends.
        s["freq"] = (1e6 ** (-torch.arange(0, c["rd"], 2, dtype=torch.float64) / c["rd"])).float().to(DEV)
        r = random.Random(c["lens"] + 2)
        pos = [r.randint(0, c["base"]) + x - a + i for a, x in zip(new, ctx) for i in range(a)]
        s["pos"] = torch.tensor(pos, dtype=torch.int32, device=DEV)
    if own:
        _own(s)
    return s


def _own(s):
    """The pool and the device arrays of the step that a serving program holds."""
    from mitten_amd import DeviceKv8Pool, PoolDesc

    c = s["case"]
    pool = DeviceKv8Pool(PoolDesc(1, c["hkv"], c["hkv"] * c["g"], c["d"], s["exp"].shape[1], c["type"]))
    pool.tensor()[0].copy_(s["kv"].view(torch.uint8))
    pool.exponents()[0].copy_(s["exp"])
    s["pool"], s["kv"], s["exp"] = pool, pool.tensor()[0].view(F8), pool.exponents()[0]

    def dev(x):
        return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(DEV)

    tables = (dev(s["indptr"]), dev(s["ids"]), dev(s["ctx"]))
    at = dev(np.concatenate([[0], np.cumsum(s["new"])]))
    longest, most = max(s["ctx"]), max(s["new"])
    if c["op"] == "append":
        s["call"] = lambda: pool.append(0, s["k"], s["v"], at, *tables, max_q_len=most)
    elif c["op"] == "rope_append":
        w = (s["wq"], s["wk"]) if c["norm"] else (None, None)
        s["call"] = lambda: pool.qk_norm_rope_append(
            0, s["q"], s["k"], s["v"], at, *tables, max_q_len=most, positions=s["pos"], q_norm_w=w[0], k_norm_w=w[1],
            inv_freq=s["freq"], eps=EPS, interleaved=c["interleaved"], rope_factor=c["factor"], gated=c["gated"])
    elif c["op"] == "gather":
        s["call"] = lambda: pool.gather(0, *tables, max_ctx_len=longest, total_tokens=sum(s["ctx"]))
    elif c["op"] == "decode":  # bound once for an engine step, run for every layer
        s["out"] = torch.empty_like(s["q"])
        step = pool.bind_decode_step(s["k"], s["v"], s["q"], *tables, s["out"], max_ctx_len=longest, scale=s["scale"])
        s["call"] = lambda: step(0)
    else:
        s["call"] = lambda: pool.extend_attention(0, s["q"], at, *tables, max_q_len=most, max_ctx_len=longest,
                                                  scale=s["scale"])


# ---- one pass ---------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        r = s["call"]()
        if op == "gather":
            return {"k": r[0], "v": r[1]}
        if op == "extend":
            return {"out": r}
        got = {"kv": s["kv"], "exp": s["exp"]}
        return dict(got, q=r) if op == "rope_append" else dict(got, out=s["out"]) if op == "decode" else got
    if op == "gather":
        return _gather(s)
    if op == "extend":
        return {"out": _attend(s)}
    if op == "decode":
        _append(s, s["k"].float(), s["v"].float())
        return {"kv": s["kv"], "exp": s["exp"], "out": _attend(s)}
    if op == "append":
        _append(s, s["k"].float(), s["v"].float())
        return {"kv": s["kv"], "exp": s["exp"]}
    c = s["case"]
    q = s["q"][:, :, 0] if c["gated"] else s["q"]
    a = s["pos"].double()[:, None] * s["freq"].double()  # angles of far positions in 64 bits
    cos, sin = (torch.cos(a) * c["factor"]).float()[:, None], (torch.sin(a) * c["factor"]).float()[:, None]
    q = _rope(c, _norm(c, q.float(), s["wq"]), cos, sin)
    _append(s, _rope(c, _norm(c, s["k"].float(), s["wk"]), cos, sin), s["v"].float())
    return {"kv": s["kv"], "exp": s["exp"], "q": q.to(TYPES[c["type"]])}


def _exponent(amax):
    """The least e with amax <= 448 * 2^e = 0.875 * 2^(e + 9)."""
    m, x = torch.frexp(amax)
    return torch.where(m > 0.875, x - 8, torch.where(amax > 0, x - 9, E_MIN)).clamp_min(E_MIN)


def _norm(c, x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w) if c["norm"] else x


def _rope(c, x, cos, sin):
    rd = c["rd"]
    y = x.clone()
    if c["interleaved"]:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        y[..., 0:rd:2], y[..., 1:rd:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., : rd // 2], x[..., rd // 2: rd]
        y[..., : rd // 2], y[..., rd // 2: rd] = a * cos - b * sin, b * cos + a * sin
    return y


def _rows(tiles, p, d):
    """Tiles [..., 16 * d] of K (p = 0) or V as rows [..., 16, d]."""
    lead = tiles.shape[:-1]
    if p == 0:
        return tiles.view(*lead, d // 16, 16, 16).transpose(-3, -2).reshape(*lead, 16, d)
    x = tiles.view(*lead, d // 64, 4, 16, 4, 4)  # dims 64 i + 4 q + n, tokens 4 t + j as [i][t][q][n][j]
    k = len(lead)
    return x.permute(*range(k), k + 1, k + 4, k, k + 2, k + 3).reshape(*lead, 16, d)


def _tiles(rows, p):
    lead, d = rows.shape[:-2], rows.shape[-1]
    if p == 0:
        return rows.reshape(*lead, 16, d // 16, 16).transpose(-3, -2).reshape(*lead, 16 * d)
    k = len(lead)
    x = rows.reshape(*lead, 4, 4, d // 64, 16, 4)  # [t][j][i][q][n]
    return x.permute(*range(k), k + 2, k, k + 3, k + 4, k + 1).reshape(*lead, 16 * d)


def _touched(s):
    """For every block that the new tokens go to: its id and whether it is fresh; for every token its place among them."""
    ids, fresh, place, row = [], [], [], []
    for b, (n, ctx) in enumerate(zip(s["new"], s["ctx"])):
        for pos in range(ctx - n, ctx):
            if pos == ctx - n or pos % PAGE == 0:
                ids.append(int(s["ids"][s["indptr"][b] + pos // PAGE]))
                fresh.append(pos % PAGE == 0)
            place.append(len(ids) - 1)
            row.append(pos % PAGE)
    return [torch.tensor(x, device=DEV, dtype=t) for x, t in ((ids, torch.int64), (fresh, torch.bool), (place, torch.int64),
                                                              (row, torch.int64))]


def _append(s, k, v):
    if not sum(s["new"]):
        return
    if "touched" not in s:  # the indexes of the step, kept for its layers
        s["touched"] = _touched(s)
    ids, fresh, place, row = s["touched"]
    d = s["case"]["d"]
    for p, x in enumerate((k, v)):
        new = torch.zeros(len(ids), x.shape[1], PAGE, d, device=DEV)
        new[place, :, row] = x
        written = torch.zeros(len(ids), 1, PAGE, 1, dtype=torch.bool, device=DEV)
        written[place, 0, row, 0] = True
        e = _exponent(torch.where(new.isfinite(), new.abs(), 0.0).amax((-2, -1)))
        was = s["exp"][p][ids].to(e.dtype)
        e = torch.where(fresh[:, None], e, torch.maximum(e, was))
        old = _rows(s["kv"][p].view(torch.uint8)[ids].view(F8), p, d).float() * torch.exp2((was - e).float())[..., None, None]
        old = torch.where(fresh[:, None, None, None], 0.0, old)
        x = torch.where(written, new * torch.exp2(-e.float())[..., None, None], old)
        s["kv"][p].view(torch.uint8)[ids] = _tiles(x, p).to(F8).view(torch.uint8)
        s["exp"][p][ids] = e.to(torch.int8)


def _held(s, b, p, dtype=torch.float32):
    """Sequence b's rows of K or V, [hkv][ctx][d]."""
    at = torch.from_numpy(s["ids"][s["indptr"][b]: s["indptr"][b + 1]].astype(np.int64)).to(DEV)
    x = _rows(s["kv"][p].view(torch.uint8)[at].view(F8).to(dtype), p, s["case"]["d"])
    x = x * torch.exp2(s["exp"][p][at].to(dtype))[..., None, None]
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, : s["ctx"][b]]


def _gather(s):
    t = TYPES[s["case"]["type"]]
    return {n: torch.cat([_held(s, b, p).to(t).reshape(-1) for b in range(len(s["ctx"]))]) for p, n in enumerate("kv")}


def _attend(s):
    c = s["case"]
    out, at = torch.empty_like(s["q"]), 0
    for b, (n, ctx) in enumerate(zip(s["new"], s["ctx"])):
        if not n:
            continue
        k, v = _held(s, b, 0), _held(s, b, 1)
        q = s["q"][at: at + n].float().view(n, c["hkv"], c["g"], c["d"]).permute(1, 0, 2, 3).reshape(c["hkv"], n * c["g"], -1)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
        if n > 1:
            pos = torch.arange(ctx - n, ctx, device=DEV).repeat_interleave(c["g"])
            x = torch.where(torch.arange(ctx, device=DEV) <= pos[:, None], x, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(x, v.contiguous()) / x.sum(-1, keepdim=True)
        out[at: at + n] = o.view(c["hkv"], n, c["g"], -1).permute(1, 0, 2, 3).reshape(n, -1, c["d"]).to(out.dtype)
        at += n
    return out


# ---- the definition in 64 bits ----------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c, op, d = s["case"], case["op"], case["d"]
    kv, ex = s["kv"].double(), s["exp"].long()
    if op == "rope_append":
        q = (s["q"][:, :, 0] if c["gated"] else s["q"]).double()
        k = s["k"].double()
        if c["norm"]:
            q, k = (x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * (w.double() + 1)
                    for x, w in ((q, s["wq"]), (k, s["wk"])))
        q, k = (_turn(c, x, s) for x in (q, k))
    elif op != "gather":
        q, k = s["q"].double(), s["k"].double()
    if op in ("append", "rope_append", "decode"):
        held = _exact_append(c, s, kv, ex, k, s["v"].double())
        if op == "append":
            return {"kv": kv, "exp": ex.to(torch.int8)}
        if op == "rope_append":
            return {"kv": kv, "exp": None, "q": q}
    else:
        held = kv
    kv = [held[p] * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=DEV), ex[p])[..., None] for p in range(2)]
    blocks = [torch.from_numpy(s["ids"][a:b].astype(np.int64)).to(DEV) for a, b in zip(s["indptr"][:-1], s["indptr"][1:])]

    def rows(p, b):  # [hkv][ctx][d]
        x = kv[p][blocks[b]]
        n = len(blocks[b])
        if p == 0:
            x = x.view(n, c["hkv"], d // 16, PAGE, 16).permute(1, 0, 3, 2, 4)
        else:
            x = x.view(n, c["hkv"], d // 64, 4, 16, 4, 4).permute(1, 0, 3, 6, 2, 4, 5)
        return x.reshape(c["hkv"], n * PAGE, d)[:, : s["ctx"][b]]

    if op == "gather":
        return {n: torch.cat([rows(p, b).flatten() for b in range(c["seqs"])]) for p, n in enumerate("kv")}
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), 0
    for b, (n, ctx) in enumerate(zip(s["new"], s["ctx"])):
        k, v = rows(0, b), rows(1, b)
        for h in range(c["hkv"] * c["g"] if n else 0):
            x = (q[at: at + n, h] @ k[h // c["g"]].T.contiguous()) * s["scale"]
            hidden = torch.arange(ctx, device=DEV)[None] > torch.arange(ctx - n, ctx, device=DEV)[:, None]
            out[at: at + n, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // c["g"]]
        at += n
    # (The rows as the tiles hold them; the new ones before their rounding in what is returned.)
    return {"out": out} if op == "extend" else {"kv": s["unrounded"], "exp": ex.to(torch.int8), "out": out}


def _turn(c, x, s):
    """Every pair as a complex number, turned by its angle."""
    rd = c["rd"]
    i = torch.arange(rd // 2, device=DEV)
    a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rd // 2)
    z = torch.complex(x[..., a], x[..., b])
    angle = s["pos"].double()[:, None, None] * s["freq"].double()
    z = z * torch.polar(torch.full_like(angle, c["factor"]), angle)
    y = x.clone()
    y[..., a], y[..., b] = z.real, z.imag
    return y


_GRID = torch.tensor([(m / 8 + (1 if x else 0)) * 2.0 ** ((x or 1) - 7) for x in range(16) for m in range(8)][:127],
                     dtype=torch.float64)  # what e4m3 holds, from 0 to 448


def _nearest(x):
    """x (at most 448) to the nearest value of the grid, ties to the even byte."""
    grid = _GRID.to(DEV)
    a = x.abs().contiguous()
    hi = torch.searchsorted(grid, a).clamp(1, 126)
    lo = hi - 1
    up = (grid[hi] - a < a - grid[lo]) | ((grid[hi] - a == a - grid[lo]) & (hi % 2 == 0))
    return torch.where(up, grid[hi], grid[lo]).copysign(x)


def _exact_append(c, s, kv, ex, k, v):
    """Writes the rows, unrounded, and the exponents block by block; returns the tiles as they are held."""
    d, at = c["d"], 0
    held = kv.clone()
    dim = torch.arange(d, device=DEV)
    for b, (n, ctx) in enumerate(zip(s["new"], s["ctx"])):
        pos = ctx - n
        while pos < ctx:
            end = min(ctx, pos - pos % PAGE + PAGE)
            blk, rows = int(s["ids"][s["indptr"][b] + pos // PAGE]), torch.arange(pos, end, device=DEV) % PAGE
            for p, x in enumerate((k, v)):
                new = x[at: at + end - pos].transpose(0, 1)  # [hkv][rows][d]
                amax = new.abs().flatten(1).max(1).values.clamp_min(1e-300)
                e = torch.floor(torch.log2(amax / F8_MAX)).long() - 1
                for _ in range(3):
                    e += amax > F8_MAX * torch.pow(2.0, e.double())
                e = e.clamp_min(E_MIN)
                if pos % PAGE == 0:
                    kv[p, blk] = 0.0
                else:
                    e = torch.maximum(e, ex[p, blk])
                    kv[p, blk] *= torch.pow(2.0, (ex[p, blk] - e).double())[:, None]
                ex[p, blk] = e
                held[p, blk] = _nearest(kv[p, blk])
                if p == 0:
                    place = (dim // 16 * PAGE + rows[:, None]) * 16 + dim % 16
                else:
                    place = ((dim // 64 * 4 + rows[:, None] // 4) * 16 + dim % 64 // 4) * 16 + dim % 4 * 4 + rows[:, None] % 4
                y = new / torch.pow(2.0, e.double())[:, None, None]
                kv[p, blk, :, place.flatten()] = y.flatten(1)
                held[p, blk, :, place.flatten()] = _nearest(y).flatten(1)
            at += end - pos
            pos = end
    s["unrounded"] = kv
    return held
