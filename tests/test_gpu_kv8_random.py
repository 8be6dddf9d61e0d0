"""Random calls of the 8-bit pool's attention against 64 bits: heads, lengths, chunks, scales of
V, tiles of zeros, score gaps, bounds above the lengths and workspaces of any size."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv8

from kv8_helpers import Batch, assert_attention, dev, fill, host, make_pool, read, values

pytestmark = pytest.mark.gpu


def lengths(r, n):
    c = np.exp(r.uniform(0, np.log(2500), n)).astype(int) + r.integers(0, 2, n)
    return [int(x) for x in np.where(r.random(n) < 0.1, 0, c)]


@pytest.mark.parametrize("seed", range(48))
def test_attention(seed):
    import torch

    r = np.random.default_rng(1000 + seed)
    dtype = ("bf16", "f32")[seed % 2]
    d = int(r.choice([64, 128, 256]))
    hkv, g = int(r.integers(1, 5)), int(r.choice([1, 2, 3, 5, 7, 8, 16, 19]))
    ctx = lengths(r, int(r.integers(1, 9)))
    kind = ("decode", "extend")[seed // 2 % 2]
    new = [1] * len(ctx) if kind == "decode" else [int(r.integers(0, min(c, 70) + 1)) for c in ctx]
    b = Batch(new, ctx, seed=seed, spare=int(r.integers(0, 2)))
    with make_pool(b, hkv, g, d, dtype) as pool:
        lo = int(r.choice([-5, -30, -100]))
        fill(pool, seed, zero_tiles=float(r.choice([0.0, 0.2])))
        e = r.integers(lo, int(r.choice([-4, 0, 60, 100])) + 1, tuple(pool.exponents()[0, 1].shape))
        zero = (pool.tensor()[0, 1] & 0x7F).sum(-1).cpu().numpy() == 0
        pool.exponents()[0, 1] = torch.from_numpy(np.where(zero, -100, e)).to(torch.int8).cuda()
        want = read(pool)
        q = values(r.standard_normal((b.tokens, hkv * g, d)), dtype)
        scale = float(np.float32(r.choice([0.02, d ** -0.5, 0.6])))
        sink = bool(r.integers(0, 2))
        kw = dict(scale=scale, zero_sink=sink, max_ctx_len=max(max(ctx), 1) + int(r.choice([0, 1, 3000, 30000])))
        if r.integers(0, 2):
            size = int(r.choice([0, 300, 1 << 14, 1 << 18, 1 << 22]))
            kw["workspace"] = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        if kind == "decode":
            o = pool.decode_attention(0, dev(q, dtype), *b.device(), **kw)
        else:
            most = max(max(new), 1)
            o = pool.extend_attention(0, dev(q, dtype), b.q_indptr(), *b.device(),
                                      max_q_len=int(r.choice([most, min(most + 9, kw["max_ctx_len"])])), **kw)
        pool.check()
        ref = want.attend(q, new, ctx, b.tables, scale, sink)
        # (Results of scores far below a zero tile's reach 1e-53; both types end at 2^-126, and
        # what lies below may be 0.)
        ref[3][:] += 2.0 ** -126
        assert_attention(host(o), ref, dtype)
