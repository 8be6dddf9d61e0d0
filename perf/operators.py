"""The operators of a hybrid model's linear-attention layers, and of the step between layers, as cases to time.

An engine that serves a hybrid model keeps, beside the paged K/V of its attention layers, one state matrix per value
head and sequence for its linear-attention layers. Prompts come in as ragged batches of chunks that read a state,
attend and leave the state after them (`linear_extend`); every engine step then moves each running sequence on by one
token (`linear_step`); states are copied between slots when a prefix's snapshot is shared or slots are compacted
(`state_copy`). Between layers the residual is added and the sum normalised for the next projections, in the model's
type or in 8 bits with scales (`add_rms_norm`).

Shapes are those of the benchmark configurations (28 query heads over 4 key heads of 128, width 3,584; 14 over 2 of
64 in f32, width 896) and one generic geometry of 32 value and 16 key heads of 128. Lengths and slots are a function
of the case; contents of the seed. One layer's call is one pass.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False  # set from outside: False the plain forms, True the library's kernels

DEV = "cuda:0"
NONE = 0xFFFFFFFF  # a source slot that says: start from a zero state
CHUNK = 64
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
FP8_MAX = 448.0
AMAX_MIN = 2.0 ** -100


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # One long prompt alone: 32 heads of work only, unless the length is split.
        dict(name="extend_one_prompt", op="linear_extend", hk=16, hv=32, dk=128, dv=128, type="bf16", seqs=1, lo=8192,
             hi=8192, carried=0.0, lens=1),
        # A scheduler's ordinary prefill batch: ragged prompts, half of them going on from an earlier chunk.
        dict(name="extend_batch", op="linear_extend", hk=4, hv=28, dk=128, dv=128, type="bf16", seqs=8, lo=300, hi=1500,
             carried=0.5, lens=2),
        # Draft checking and multi-turn chat: short chunks that all carry a state.
        dict(name="extend_short", op="linear_extend", hk=16, hv=32, dk=128, dv=128, type="bf16", seqs=16, lo=5, hi=24,
             carried=1.0, lens=3),
        # The small f32 model's prompts.
        dict(name="extend_f32", op="linear_extend", hk=2, hv=14, dk=64, dv=64, type="f32", seqs=8, lo=33, hi=512,
             carried=0.25, lens=4),
        # One user's decode step: the launch.
        dict(name="step_one", op="linear_step", hk=16, hv=32, dk=128, dv=128, type="bf16", seqs=1, carried=1.0, lens=5),
        # The ordinary serving step.
        dict(name="step_batch", op="linear_step", hk=4, hv=28, dk=128, dv=128, type="bf16", seqs=64, carried=1.0, lens=6),
        # A full pool's decode step: every byte of the states moves once each way.
        dict(name="step_full", op="linear_step", hk=16, hv=32, dk=128, dv=128, type="bf16", seqs=504, carried=0.95,
             lens=7),
        # Two requests fork a prefix's snapshot: a few states of every layer.
        dict(name="copy_fork", op="state_copy", hk=4, hv=28, dk=128, dv=128, layers=6, pairs=3, slots=24, lens=8),
        # Compaction of a pool after a wave of requests finished.
        dict(name="copy_compaction", op="state_copy", hk=16, hv=32, dk=128, dv=128, layers=4, pairs=85, slots=192,
             lens=9),
        # The small f32 model's decode step: a few narrow rows.
        dict(name="norm_small_f32", op="add_rms_norm", type="f32", rows=8, dim=896, group=-1, residual=True, lens=10),
        # The ordinary decode step's rows, quantised for 8-bit projections, one scale per row.
        dict(name="norm_step_fp8", op="add_rms_norm", type="bf16", rows=64, dim=3584, group=0, residual=True, lens=11),
        # A prefill batch's rows with scales per group of 128, as block-scaled products take them.
        dict(name="norm_prefill_fp8", op="add_rms_norm", type="bf16", rows=16384, dim=3584, group=128, residual=True,
             lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear_extend", "linear_extend", "linear_step", "add_rms_norm", "state_copy"])
    c = dict(op=op, lens=rng.randrange(1 << 30))
    if op == "add_rms_norm":
        dim = 8 * _log(rng, 8, 2048)
        rows = _log(rng, 1, min(16384, 16384 * 3584 // dim))
        group = rng.choice([-1, 0, 128, 64])
        if group > 0:
            dim = max(group, dim - dim % group)
        return dict(c, type=rng.choice(["bf16", "bf16", "f32"]), rows=rows, dim=dim, group=group,
                    residual=rng.random() < 0.8)
    hk = rng.choice([1, 2, 3, 4, 8, 16])
    hv = hk * rng.choice([1, 2, 4, 7])
    dk, dv = rng.choice([64, 128, 128, 256]), rng.choice([64, 128, 128, 256])
    c.update(hk=hk, hv=hv, dk=dk, dv=dv)
    per_state = hv * dk * dv
    if op == "state_copy":
        layers = rng.randrange(1, 7)
        slots = _log(rng, 6, max(7, min(300, (1 << 28) // (per_state * layers))))
        return dict(c, layers=layers, slots=slots, pairs=rng.randrange(1, slots // 2 + 1))
    c.update(type=rng.choice(["bf16", "bf16", "f32"]), carried=rng.choice([0.0, 0.5, 1.0]))
    if op == "linear_step":
        return dict(c, seqs=_log(rng, 1, max(2, min(504, (1 << 28) // per_state))))
    # Tokens in all, so that no draw costs more than the largest listed case; some sequences may be empty.
    total = max(16, min(8192, 8192 * 32 * 128 * 128 // per_state))
    if c["type"] == "f32":
        total = max(16, total // 8)
    hi = _log(rng, 1, total)
    seqs = max(1, min(64, _log(rng, 1, max(1, total // hi)), (1 << 27) // per_state))
    return dict(c, seqs=seqs, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi)


def _lengths(c):
    r = random.Random(c["lens"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]


def _slots(c):
    """(number of slots, source slots with NONE where a sequence is new, destination slots)."""
    r = random.Random(c["lens"] + 1)
    n = c["seqs"] + 3
    dst = r.sample(range(n), c["seqs"])
    return n, [s if r.random() < c["carried"] else NONE for s in dst], dst


def _pairs(c):
    r = random.Random(c["lens"] + 1)
    at = r.sample(range(c["slots"]), 2 * c["pairs"])
    src, dst = at[: c["pairs"]], at[c["pairs"]:]
    if c["pairs"] > 1 and c["pairs"] < 8:  # a fork: one snapshot to several slots
        src = [src[0]] * c["pairs"]
    return src, dst


def work(c):
    op = c["op"]
    if op == "add_rms_norm":
        n, es = c["rows"] * c["dim"], 4 if c["type"] == "f32" else 2
        size = n * es * (3 if c["residual"] else 1) + 4 * c["dim"]
        size += n * es if c["group"] < 0 else n + 4 * c["rows"] * (c["dim"] // c["group"] if c["group"] else 1)
        return {"bytes": size, "flops": 6 * n}
    state = 4 * c["hv"] * c["dk"] * c["dv"]
    if op == "state_copy":
        return {"bytes": 2 * c["layers"] * c["pairs"] * state, "flops": 0}
    es = 4 if c["type"] == "f32" else 2
    lens = [1] * c["seqs"] if op == "linear_step" else _lengths(c)
    _, src, _ = _slots(c)
    row = es * (2 * c["hk"] * c["dk"] + 2 * c["hv"] * c["dv"]) + 4 * c["hv"]
    read = sum(s != NONE for s in src)
    return {"bytes": sum(lens) * row + (read + c["seqs"]) * state,
            "flops": 4 * c["hv"] * c["dk"] * c["dv"] * sum(lens)}


# ---- inputs -----------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    c, g = case, _gen(seed)
    op = c["op"]
    if op == "add_rms_norm":
        t = TYPES[c["type"]]
        # A residual stream: channels of uneven size, a few of them large.
        size = torch.exp(_normal(g, c["dim"]))
        x = (_normal(g, c["rows"], c["dim"]) * size).to(t)
        res = (_normal(g, c["rows"], c["dim"]) * size * 2).to(t) if c["residual"] else None
        return dict(case=c, x=x, res=res, w=0.3 * _normal(g, c["dim"]))
    if op == "state_copy":
        src, dst = _pairs(c)
        s = dict(case=c, states=_normal(g, c["layers"], c["slots"], c["hv"], c["dk"], c["dv"]),
                 src=np.array(src, np.uint32), dst=np.array(dst, np.uint32))
        if own:
            s["pool"] = _pool(c, c["layers"], c["slots"], s["states"], "f32")
            s["states"] = s["pool"].tensor()
        return s
    t = TYPES[c["type"]]
    slots, src, dst = _slots(c)
    lens = [1] * c["seqs"] if op == "linear_step" else _lengths(c)
    n = sum(lens)
    # Heads forget at rates from a few tokens to a few thousand, modulated token by token.
    rate = torch.exp(torch.rand(c["hv"], generator=g, device=DEV) * math.log(1e3) - math.log(2e3))
    decay = -rate * (0.2 + 1.6 * torch.rand(n, c["hv"], generator=g, device=DEV))
    s = dict(case=c, q=_normal(g, n, c["hk"], c["dk"]).to(t),
             k=(_normal(g, n, c["hk"], c["dk"]) * c["dk"] ** -0.5).to(t), v=_normal(g, n, c["hv"], c["dv"]).to(t),
             decay=decay, states=0.5 * _normal(g, 1, slots, c["hv"], c["dk"], c["dv"]),
             lens=np.array(lens, np.int32), src=np.array(src, np.uint32), dst=np.array(dst, np.uint32),
             scale=c["dk"] ** -0.5)
    if own:
        s["pool"] = _pool(c, 1, slots, s["states"], c["type"])
        s["states"] = s["pool"].tensor()
        # The call of one engine step, bound once and run for every layer.
        s["out"] = torch.empty_like(s["v"])
        bind = s["pool"].bind_linear_step if op == "linear_step" else s["pool"].bind_linear_extend
        more = () if op == "linear_step" else (s["lens"],)
        s["call"] = bind(s["q"], s["k"], s["v"], s["decay"], *more, s["dst"], s["out"], src_slots=s["src"],
                         scale=s["scale"])
    return s


def _pool(c, layers, slots, states, dtype):
    from mitten_amd import DeviceStatePool, StateDesc

    pool = DeviceStatePool(StateDesc(layers, c["hk"], c["hv"], c["dk"], c["dv"], slots, dtype))
    pool.tensor().copy_(states)
    return pool


# ---- one pass ---------------------------------------------------------------


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        if op == "add_rms_norm":
            from mitten_amd import add_rms_norm

            r = add_rms_norm(s["x"], s["w"], EPS, residual=s["res"], fp8=c["group"] >= 0, group=max(c["group"], 0))
            return {k: v for k, v in zip(("sum", "out", "fp8", "scales"), r) if v is not None}
        if op == "state_copy":
            s["pool"].copy_states(s["src"], s["dst"])
            return {"states": s["states"]}
        s["call"](0)
        return {"out": s["out"], "states": s["states"]}
    if op == "add_rms_norm":
        return _norm(s)
    if op == "state_copy":
        src = torch.from_numpy(s["src"].astype(np.int64)).to(DEV)
        dst = torch.from_numpy(s["dst"].astype(np.int64)).to(DEV)
        s["states"][:, dst] = s["states"][:, src]
        return {"states": s["states"]}
    return _step(s) if op == "linear_step" else _extend(s)


def _norm(s):
    c = s["case"]
    t = s["x"].dtype
    r = s["x"].float() if s["res"] is None else s["x"].float() + s["res"].float()
    y = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS) * (1.0 + s["w"])
    got = {} if s["res"] is None else {"sum": r.to(t)}
    if c["group"] < 0:
        return dict(got, out=y.to(t))
    y = y.view(c["rows"], -1, c["group"] or c["dim"])
    a = y.abs().amax(-1, keepdim=True).clamp_min(AMAX_MIN)
    q = (y * (FP8_MAX / a)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return dict(got, fp8=q.view(c["rows"], c["dim"]), scales=(a / FP8_MAX).squeeze(-1))


def _start(s):
    """The states that a pass begins with, [B][Hv][Dk][Dv], and their slots on the device."""
    src = torch.from_numpy(s["src"].astype(np.int64)).to(DEV)
    dst = torch.from_numpy(s["dst"].astype(np.int64)).to(DEV)
    new = src == NONE
    s0 = s["states"][0][torch.where(new, 0, src)]
    return torch.where(new.view(-1, 1, 1, 1), 0.0, s0), dst


def _step(s):
    c = s["case"]
    rep = c["hv"] // c["hk"]
    q, k = (s[x].float().repeat_interleave(rep, 1) for x in "qk")
    s0, dst = _start(s)
    new = torch.exp(s["decay"])[:, :, None, None] * s0 + k[..., None] * s["v"].float()[:, :, None, :]
    s["states"][0][dst] = new
    o = torch.matmul(q[:, :, None, :], new)[:, :, 0] * s["scale"]
    return {"out": o.to(s["v"].dtype), "states": s["states"]}


def _extend(s):
    """Chunks of 64 tokens of all sequences at once (padded to the longest), their local states joined by one product
    with the matrix of decays between chunks."""
    c = s["case"]
    rep = c["hv"] // c["hk"]
    lens = torch.from_numpy(s["lens"].astype(np.int64)).to(DEV)
    s0, dst = _start(s)
    B, nc = c["seqs"], max(1, -(-int(s["lens"].max()) // CHUNK))
    first = torch.cumsum(lens, 0) - lens
    at = torch.arange(nc * CHUNK, device=DEV)
    live = at < lens[:, None]
    if not s["lens"].any():
        s["states"][0][dst] = s0
        return {"out": torch.empty_like(s["v"]), "states": s["states"]}
    rows = torch.where(live, first[:, None] + at, 0)

    def lay(x):  # [B][Hv][nc][CHUNK][D], zeros past a sequence's end
        x = torch.where(live[..., None, None], x[rows].float(), 0.0)
        if x.shape[2] != c["hv"]:
            x = x.repeat_interleave(rep, 2)
        return x.view(B, nc, CHUNK, c["hv"], -1).permute(0, 3, 1, 2, 4).contiguous()

    q, k, v = lay(s["q"]), lay(s["k"]), lay(s["v"])
    g = torch.where(live[..., None], s["decay"][rows].double(), 0.0)
    G = torch.cumsum(g.view(B, nc, CHUNK, c["hv"]).permute(0, 3, 1, 2), -1)  # [B][Hv][nc][CHUNK], 64 bits
    below = at[:CHUNK, None] >= at[None, :CHUNK]
    w = torch.where(below, torch.exp(G[..., :, None] - G[..., None, :]), 0.0).float()
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * w, v)
    kw = k * torch.exp(G[..., -1:] - G).float()[..., None]
    local = torch.matmul(kw.transpose(-1, -2).contiguous(), v)  # [B][Hv][nc][Dk][Dv]
    E = torch.cumsum(G[..., -1], -1)  # decay up to each chunk's end
    E0 = torch.cat([torch.zeros_like(E[..., :1]), E], -1)  # up to each boundary 0 .. nc
    i = torch.arange(nc + 1, device=DEV)
    M = torch.where(i[:, None] > i[None, :nc], torch.exp(E0[..., :, None] - E[..., None, :]), 0.0).float()
    S = torch.matmul(M, local.view(B, c["hv"], nc, -1)).view(B, c["hv"], nc + 1, c["dk"], c["dv"])
    S = S + torch.exp(E0).float()[..., None, None] * s0[:, :, None]
    o = (o + torch.matmul(q * torch.exp(G).float()[..., None], S[:, :, :nc])) * s["scale"]
    out = torch.empty_like(s["v"])
    o = o.permute(0, 2, 3, 1, 4).reshape(B, nc * CHUNK, c["hv"], c["dv"])
    out[rows[live]] = o[live].to(out.dtype)
    s["states"][0][dst] = S[:, :, nc]
    return {"out": out, "states": s["states"]}


# ---- the definition in 64 bits ----------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "add_rms_norm":
        r = s["x"].double()
        if s["res"] is not None:
            r = r + s["res"].double()
        y = r / torch.sqrt((r ** 2).sum(1, keepdim=True) / c["dim"] + EPS) * (s["w"].double() + 1)
        got = {} if s["res"] is None else {"sum": r}
        if c["group"] < 0:
            return dict(got, out=y)
        parts = y.reshape(c["rows"], -1, c["group"] or c["dim"])
        scale = torch.clamp(parts.abs().max(2).values, min=AMAX_MIN) / FP8_MAX
        return dict(got, fp8=(parts / scale[..., None]).reshape(c["rows"], c["dim"]), scales=scale)
    states = s["states"].double()
    if c["op"] == "state_copy":
        was = states.clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            states[:, b] = was[:, a]
        return {"states": states}
    # The recurrence, token by token, every sequence that still has one.
    lens = s["lens"].tolist()
    first = np.concatenate([[0], np.cumsum(lens)[:-1]])
    order = np.argsort(-np.array(lens), kind="stable")  # longest first: those with a token t are a prefix
    S = torch.stack([states[0, s["src"][b]] if s["src"][b] != NONE else torch.zeros_like(states[0, 0])
                     for b in order.tolist()])
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=DEV)
    head = torch.arange(c["hv"], device=DEV) // (c["hv"] // c["hk"])
    a = torch.exp(s["decay"].double())
    ordered = torch.from_numpy(first[order]).to(DEV)
    for t in range(max(lens)):
        m = int((np.array(lens) > t).sum())
        row = ordered[:m] + t
        S[:m] *= a[row][:, :, None, None]
        S[:m] += s["k"][row][:, head].double()[..., None] * s["v"][row].double()[:, :, None]
        out[row] = s["scale"] * (s["q"][row][:, head].double()[..., None] * S[:m]).sum(2)
    for i, b in enumerate(order.tolist()):
        states[0, s["dst"][b]] = S[i]
    return {"out": out, "states": states}
