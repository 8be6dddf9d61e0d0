"""Shared by the tests of the 8-bit K/V pool: a pool with its oracle, batches, tolerances."""
from __future__ import annotations

import numpy as np

from mitten_amd import DeviceKv8Pool, PoolDesc
from oracle import kv8
from oracle import oracle as orc

ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}  # half a step, relative
WEIGHT = {"f32": 2.0 ** -22, "bf16": 2.0 ** -11}  # a weight of the product with V


def values(x, dtype):
    """What the device rows hold of x, in 64 bits."""
    x = np.asarray(x, np.float32)
    return x.astype(np.float64) if dtype == "f32" else orc.bf16_to_f32(orc.f32_to_bf16(x)).astype(np.float64)


def dev(x, dtype=None):
    """A device tensor: rows of that type, or int32 without one."""
    import torch

    if dtype is None:
        return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(torch.float32 if dtype == "f32" else torch.bfloat16)


def host(t):
    return t.detach().cpu().double().numpy()


class Batch:
    """Sequences with scattered tables over a pool of their own blocks and some more."""

    def __init__(self, new, ctx, seed=0, extra=3, spare=0):
        self.new, self.ctx = list(new), list(ctx)
        need = [-(-c // 16) + spare for c in ctx]
        self.blocks = sum(need) + extra
        ids = np.random.default_rng(seed).permutation(self.blocks)[: sum(need)]
        self.indptr = np.concatenate([[0], np.cumsum(need)]).astype(np.uint32)
        self.ids = ids.astype(np.uint32)
        self.tables = [ids[a:b].tolist() for a, b in zip(self.indptr[:-1], self.indptr[1:])]
        self.tokens = sum(self.new)

    def host(self):
        return self.indptr, self.ids, np.array(self.ctx, np.int32)

    def device(self):
        return dev(self.indptr), dev(self.ids), dev(self.ctx)

    def q_indptr(self):
        return dev(np.concatenate([[0], np.cumsum(self.new)]))


def make_pool(batch, hkv, g, d, dtype, layers=1):
    return DeviceKv8Pool(PoolDesc(layers, hkv, hkv * g, d, batch.blocks, dtype))


def fill(pool, seed=0, exps=(-7, -4), zero_tiles=0.0):
    """Random bytes without NaN and exponents; returns the oracle of layer 0."""
    r = np.random.default_rng(seed)
    d = pool.desc
    shape = (d.num_layers, 2, d.num_blocks, d.num_kv_heads)
    b = kv8.to_e4m3(np.clip(r.standard_normal(shape + (16 * d.head_dim,)) * 120, -448, 448))
    if zero_tiles:
        b[r.random(shape) < zero_tiles] = 0.0
    import torch

    pool.tensor().copy_(torch.from_numpy(b).float().to(torch.float8_e4m3fn).view(torch.uint8))
    pool.exponents().copy_(torch.from_numpy(r.integers(exps[0], exps[1] + 1, shape)).to(torch.int8))
    return read(pool)


def read(pool, layer=0):
    return kv8.Kv8.read(pool.tensor()[layer].cpu().numpy(), pool.exponents()[layer].cpu().numpy())


def assert_same(pool, want, layer=0):
    """The pool's bytes stand for what the oracle holds, bit for bit."""
    got = read(pool, layer)
    assert np.array_equal(got.exp, want.exp), np.argwhere(got.exp != want.exp)[:4]
    assert np.array_equal(got.val, want.val, equal_nan=True), np.argwhere(~((got.val == want.val) | (np.isnan(got.val) & np.isnan(want.val))))[:4]


def assert_attention(got, want, dtype):
    """got against (o, a, s, f) of the oracle: the output is rounded once; a weight's error is its
    rounding and its score's, in the numerator and the denominator, and what f16 drops; f32
    sums of thousands of terms round by less than 2^-18 of a."""
    o, a, s, f = want
    fine = np.isfinite(o)
    assert np.array_equal(np.isnan(o), np.isnan(got))
    tol = ROUND[dtype] * np.abs(o) + a * (2 * WEIGHT[dtype] + 2 * s + 2.0 ** -18) + f
    err = np.abs(got - o)
    bad = fine & ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], err[bad][:4], tol[bad][:4])
    # Over all values: a rounding's mean square is a third of its largest; the errors of
    # scores, which move a whole row, as above.
    norm = np.linalg.norm(o[fine])
    if fine.sum() > 1000 and fine.all() and norm:
        rms = np.linalg.norm((got - o)[fine]) / norm
        assert rms <= ROUND[dtype] / np.sqrt(3) + 2 * WEIGHT[dtype] + 2 * s.max() + 2.0 ** -18, rms
