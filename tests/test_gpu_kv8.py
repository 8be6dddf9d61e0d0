"""The 8-bit K/V pool on the GPU: append, norm + RoPE + append, read-back, block copies,
refusals, streams and captured graphs. Bytes and exponents against a numpy oracle in
64 bits (oracle/kv8.py)."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import BackendError, DeviceIndexError, DeviceKv8Pool, PoolDesc, rope_inv_freq, rope_scaled_inv_freq
from mitten_amd import _lib
from oracle import kv8

from kv8_helpers import Batch, assert_attention, assert_same, dev, fill, host, make_pool, read, values

pytestmark = pytest.mark.gpu

TABLE, BLOCK, COPY, CTX = 4, 2, 8, 16  # device error bits


def rows(r, n, h, d, dtype, spread=True):
    """Rows whose magnitudes differ by powers of two from token to token."""
    x = r.standard_normal((n, h, d))
    if spread:
        x *= 2.0 ** r.integers(-9, 8, (n, 1, 1))
    return values(x, dtype)


# -- append -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hkv", [(64, 1), (64, 5), (128, 2), (256, 3)])
@pytest.mark.parametrize("form", ["host", "device"])
def test_append(d, hkv, dtype, form):
    r = np.random.default_rng(d + hkv)
    # Fresh tiles, parts of one, ends inside tiles, whole chunks; one with nothing new and padding.
    b = Batch([1, 16, 17, 5, 40, 33, 1, 0, 0, 2], [1, 16, 17, 21, 71, 33, 32, 9, 0, 17], spare=1)
    with make_pool(b, hkv, 1, d, dtype) as pool:
        want = fill(pool, 1)
        k, v = (rows(r, b.tokens, hkv, d, dtype) for _ in range(2))
        if form == "host":
            pool.append(0, dev(k, dtype), dev(v, dtype), b.new, *b.host())
        else:
            pool.append(0, dev(k, dtype), dev(v, dtype), b.q_indptr(), *b.device(), max_q_len=40)
        pool.check()
        want.append(k, v, b.new, b.ctx, b.tables)
        assert_same(pool, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 256])
def test_append_token_by_token_and_rolled_back(d, dtype):
    """A tile grown a row at a time, its scale rising, then cut back and written again."""
    r = np.random.default_rng(7)
    b = Batch([1], [60])
    with make_pool(b, 2, 1, d, dtype) as pool:
        want = fill(pool, 2)
        for ctx in list(range(1, 38)) + [20, 21, 22] + list(range(17, 40)):
            k, v = (rows(r, 1, 2, d, dtype) for _ in range(2))
            pool.append(0, dev(k, dtype), dev(v, dtype), [1], b.indptr, b.ids, [ctx])
            want.append(k, v, [1], [ctx], b.tables)
        pool.check()
        assert_same(pool, want)


def test_append_extreme_values():
    """Zeros, subnormals, the largest numbers, values on ties, infinities and NaN."""
    d, n = 64, 16 * 8
    big = float(np.finfo(np.float32).max)
    x = np.zeros((n, 1, d), np.float32)
    x[16:32] = 1e-40
    x[32:48] = big
    x[33] = -big
    x[48:64, 0] = np.resize(np.concatenate([kv8.GRID[1:] + kv8.GRID[:-1], [896.0]]) / 2, (16, d))
    x[64:80] = np.nan
    x[80:96, 0, ::2] = np.inf
    x[80:96, 0, 1::4] = -np.inf
    x[80:96, 0, 3::4] = 3.0
    x[96:112] = 448.0
    x[112:128] = np.nextafter(np.float32(448.0), np.float32(449.0))
    x[120] = -0.0
    b = Batch([n], [n])
    with make_pool(b, 1, 1, d, "f32") as pool:
        want = fill(pool, 3)
        pool.append(0, dev(x, "f32"), dev(x[::-1], "f32"), b.new, *b.host())
        want.append(x.astype(np.float64), x[::-1].astype(np.float64), b.new, b.ctx, b.tables)
        assert_same(pool, want)
        # A row of NaN into a tile of numbers: the numbers stay.
        y = np.full((1, 1, d), np.nan)
        b.ctx[0] = 40
        pool.append(0, dev(y, "f32"), dev(y, "f32"), [1], *b.host())
        want.append(y, y, [1], b.ctx, b.tables)
        assert_same(pool, want)


def test_append_longer_chunk_than_the_launch():
    r = np.random.default_rng(3)
    b = Batch([3, 100, 1], [20, 130, 5])
    with make_pool(b, 2, 1, 128, "bf16") as pool:
        want = fill(pool, 4)
        k, v = (rows(r, b.tokens, 2, 128, "bf16") for _ in range(2))
        pool.append(0, dev(k, "bf16"), dev(v, "bf16"), b.q_indptr(), *b.device(), max_q_len=1)
        pool.check()
        want.append(k, v, b.new, b.ctx, b.tables)
        assert_same(pool, want)


def test_bad_sequences_are_skipped_and_reported():
    """Each bad sequence by itself, between good ones; the good ones are written."""
    import torch

    r = np.random.default_rng(5)
    b = Batch([4, 4, 4], [20, 36, 50])
    q = 4
    for what, bit in (("ctx", CTX), ("q_len", CTX), ("table", TABLE), ("id", BLOCK), ("negative id", BLOCK)):
        with make_pool(b, 2, 2, 64, "bf16") as pool:
            want = fill(pool, 6)
            k, v = (rows(r, b.tokens, 2, 64, "bf16") for _ in range(2))
            indptr, ids, ctx = b.indptr.astype(np.int64), b.ids.astype(np.int64), list(b.ctx)
            at = np.array([0, 4, 8, 12])
            good = [0, 2]
            if what == "ctx":
                ctx[1] = -3
            elif what == "q_len":
                ctx[1] = 2  # fewer tokens than new ones
            elif what == "table":
                indptr[2] -= 1  # the second has a block too few, the third one more
            elif what == "id":
                ids[indptr[1] + 2] = b.blocks
            else:
                ids[indptr[1] + 2] = -1
            tables = [list(ids[indptr[i]: indptr[i + 1]]) for i in range(3)]
            out = torch.full((12, 4, 64), 7.0, device="cuda", dtype=torch.bfloat16)
            pool.append(0, dev(k, "bf16"), dev(v, "bf16"), dev(at), dev(indptr), dev(ids), dev(ctx), max_q_len=q)
            with pytest.raises(DeviceIndexError) as ei:
                pool.check()
            assert ei.value.bits == bit, what
            pool.check()  # (cleared)
            for i in good:
                want.append(k[4 * i: 4 * i + 4], v[4 * i: 4 * i + 4], [4], [ctx[i]], [tables[i]])
            assert_same(pool, want)  # (a bad id: positions 32 .. 35 lie in that block alone)
            # The fused call reports it too, and leaves the bad sequence's q (but for a bad id) alone.
            qr = dev(rows(r, 12, 4, 64, "bf16", False), "bf16")
            pool.qk_norm_rope_append(0, qr, dev(k, "bf16"), dev(v, "bf16"), dev(at), dev(indptr), dev(ids), dev(ctx),
                                     max_q_len=q, gated=False, out=out)
            with pytest.raises(DeviceIndexError) as ei:
                pool.check()
            assert ei.value.bits == bit, what
            for i in good:
                want.append(k[4 * i: 4 * i + 4], v[4 * i: 4 * i + 4], [4], [ctx[i]], [tables[i]])
                assert torch.equal(out[4 * i: 4 * i + 4], qr[4 * i: 4 * i + 4])
            if "id" not in what:
                assert bool((out[4:8] == 7.0).all())
            assert_same(pool, want)


# -- norm + RoPE + append ---------------------------------------------------------------


def assert_prepared(pool, want, k, pairs, b):
    """K tiles hold each value of `k` to half a step of its byte (the kernel's f32 value may lie
    on the other side of a tie or of an exponent's limit, off by `pairs`)."""
    got = read(pool)
    assert np.array_equal(got.val[1], want.val[1], equal_nan=True) and np.array_equal(got.exp[1], want.exp[1])
    at = 0
    for n, c, table in zip(b.new, b.ctx, b.tables):
        x, off = k[at: at + n].transpose(1, 0, 2), pairs[at: at + n].transpose(1, 0, 2)
        y = got.rows(0, table, c)[:, c - n:]
        e = got.exp[0][table[: -(-c // 16)]].repeat(16, 0)[c - n: c].T[..., None]
        # (Half a step of bf16 or f32 does not enter: a byte is rounded from f32.)
        tol = np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** (e - 10.0)) + off
        bad = ~(np.abs(y - x) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:3], y[bad][:3], x[bad][:3])
        first = c - n - (c - n) % 16
        for p in range(first, c, 16):
            if p >= c - n:  # a fresh tile: its exponent is that of its values
                amax = np.abs(x[:, p - c + n: p - c + n + 16]).max((1, 2))
                ee = got.exp[0][table[p // 16]]
                slack = off[:, p - c + n: p - c + n + 16].max((1, 2))
                assert np.all(448.0 * 2.0 ** ee >= amax - slack)
                assert np.all((ee == kv8.MIN_EXP) | (224.0 * 2.0 ** ee < amax + slack))
        at += n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hkv,g,rd,interleaved,norm,gated,given", [
    (64, 2, 3, 64, False, True, True, False),
    (64, 1, 1, 32, True, False, False, True),
    (64, 3, 2, 8, False, True, False, True),
    (64, 2, 2, 24, True, True, True, False),
    (128, 4, 7, 128, False, True, False, False),
    (128, 2, 5, 128, True, False, True, True),
    (128, 1, 3, 40, False, True, True, False),
    (128, 2, 2, 0, False, True, False, False),
    (256, 2, 4, 64, False, True, True, True),
    (256, 1, 2, 256, True, True, False, False),
    (256, 2, 1, 256, False, False, False, False),
    (256, 2, 1, 136, False, True, True, False),
])
def test_norm_rope_append(d, hkv, g, rd, interleaved, norm, gated, given, dtype):
    import torch

    r = np.random.default_rng(d + rd)
    b = Batch([1, 16, 17, 5, 0, 35, 0], [1, 16, 17, 21, 9, 50, 0])
    n = b.tokens
    with make_pool(b, hkv, g, d, dtype) as pool:
        want = fill(pool, 1, exps=(-6, -6))
        hq = hkv * g
        q = rows(r, n, hq * (2 if gated else 1), d, dtype, False).reshape((n, hq, 2, d) if gated else (n, hq, d))
        k, v = rows(r, n, hkv, d, dtype, False), rows(r, n, hkv, d, dtype)
        wq, wk = (r.standard_normal(d).astype(np.float32) * 0.2 for _ in range(2)) if norm else (None, None)
        pos = np.concatenate([np.arange(c - m, c) for m, c in zip(b.new, b.ctx)]) if not given else \
            r.integers(0, 2 ** 31 - 1, n)
        freq, factor = rope_scaled_inv_freq(rd, 1e4, 4.0, 4096) if rd else (np.zeros(0, np.float32), 1.0)
        args = dict(q_norm_w=None if wq is None else torch.from_numpy(wq).cuda(),
                    k_norm_w=None if wk is None else torch.from_numpy(wk).cuda(),
                    inv_freq=torch.from_numpy(freq).cuda() if rd else None, eps=1e-6, rope_factor=factor,
                    interleaved=interleaved, gated=gated)
        kw = norm_rope_pairs(k, wk, freq, pos, factor, interleaved, d, given)
        qw = norm_rope_pairs(q[:, :, 0] if gated else q, wq, freq, pos, factor, interleaved, d, given)
        for form in ("host", "device"):
            fill(pool, 1, exps=(-6, -6))
            if form == "host":
                out = pool.qk_norm_rope_append(0, dev(q, dtype), dev(k, dtype), dev(v, dtype), b.new, *b.host(),
                                               positions=pos.astype(np.int32) if given else None, **args)
                first = out
            else:
                qd = dev(q, dtype)
                out = pool.qk_norm_rope_append(0, qd, dev(k, dtype), dev(v, dtype), b.q_indptr(), *b.device(),
                                               max_q_len=35, positions=dev(pos) if given else None,
                                               out=None if gated else qd, **args)  # (in place)
                assert torch.equal(out, first)
            pool.check()
            if form == "host":
                want.append(np.zeros_like(v), v, b.new, b.ctx, b.tables)  # (its K is not looked at)
            assert_prepared(pool, want, kw[0], kw[1], b)
            y, tol = qw
            err = np.abs(host(out) - y)
            tol = tol + np.abs(y) * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24)
            assert np.all(err <= tol), (err - tol).max()


def norm_rope_pairs(x, w, freq, pos, factor, interleaved, d, given):
    """Values in 64 bits and a bound on the f32 kernel's error before its rounding: the norm's
    sum of d squares, a few products, and the angle (position * frequency in f64: 2^31 turns
    leave 2^-22 of one)."""
    y = kv8.norm_rope(x, w, 1e-6, freq, pos, factor, interleaved)
    flat = kv8.norm_rope(x, w, 1e-6, freq[:0], pos, 1.0, False)
    half = len(freq)
    mag = np.abs(flat)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    both = (mag[..., a] + mag[..., b]) * factor
    mag[..., a], mag[..., b] = both, both
    return y, mag * ((d / 2 if w is not None else 0) + 16) * 2.0 ** -24 + mag * (2.0 ** -20 if given else 0.0)


# -- read-back and copies ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hkv", [(64, 3), (128, 2), (256, 1)])
def test_gather(d, hkv, dtype):
    import torch

    b = Batch([0] * 7, [1, 16, 0, 17, 100, 31, 48], spare=1)
    with make_pool(b, hkv, 1, d, dtype, layers=2) as pool:
        fill(pool, 5, exps=(-30, 20))
        pool.tensor()[1, :, int(b.ids[0]), 0, 5] = 0x7F  # a NaN is read back
        want = read(pool, 1)
        total = sum(b.ctx)
        outs = [pool.gather(1, *b.host()),
                pool.gather(1, *b.device(), max_ctx_len=100, total_tokens=total + 3,
                            out_k=torch.full(((total + 3) * hkv * d,), 9.0, device="cuda", dtype=pool.torch_dtype),
                            out_v=torch.full(((total + 3) * hkv * d,), 9.0, device="cuda", dtype=pool.torch_dtype))]
        pool.check()
        for out in outs:
            for kv in range(2):
                y = host(out[kv])
                ref = np.concatenate([want.rows(kv, t, c).ravel() for t, c in zip(b.tables, b.ctx)])
                assert np.array_equal(y[: ref.size], ref, equal_nan=True)  # (4 bits: exact in either type)
                assert np.all(y[ref.size:] == 9.0)


def test_gather_what_does_not_fit():
    import torch

    b = Batch([0] * 3, [20, 30, 40])
    with make_pool(b, 1, 1, 64, "bf16") as pool:
        want = fill(pool, 5)
        ip, ix, cl = b.device()
        for what, bit in (("capacity", CTX), ("max", CTX), ("id", BLOCK)):
            out = [torch.full((90 * 64,), 9.0, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
            ids = ix.clone()
            if what == "id":
                ids[b.indptr[2]] = b.blocks + 5
            size = 70 * 64 if what == "capacity" else 90 * 64
            pool.gather(0, ip, ids, cl, max_ctx_len=35 if what == "max" else 40, total_tokens=size // 64,
                        out_k=out[0][:size], out_v=out[1][:size])
            with pytest.raises(DeviceIndexError) as ei:
                pool.check()
            assert ei.value.bits == bit
            y = host(out[0])
            ref = np.concatenate([want.rows(0, t, c).ravel() for t, c in zip(b.tables[:2], b.ctx[:2])])
            assert np.array_equal(y[: ref.size], ref)
            left = y[ref.size:].reshape(40, 64)
            assert np.all(left[: 16 if what == "id" else 40] == 9.0)


@pytest.mark.parametrize("d,hkv", [(64, 1), (128, 3), (256, 2)])
def test_copy_blocks(d, hkv):
    import torch

    with DeviceKv8Pool(PoolDesc(3, hkv, hkv, d, 9, "bf16")) as pool:
        fill(pool, 1, exps=(-100, 100))
        tiles, exps = pool.tensor().clone(), pool.exponents().clone()
        src, dst = [0, 0, 8, 3], [1, 7, 2, 5]
        for form in (list, lambda x: dev(np.array(x))):
            pool.tensor().copy_(tiles)
            pool.exponents().copy_(exps)
            torch.cuda.synchronize()
            pool.copy_blocks(form(src), form(dst))
            pool.check()
            t, e = tiles.clone(), exps.clone()
            t[:, :, dst], e[:, :, dst] = tiles[:, :, src], exps[:, :, src]
            assert torch.equal(pool.tensor(), t) and torch.equal(pool.exponents(), e)
        pool.copy_blocks([], [])
        for pair in (([0], [9]), ([9], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 1])):
            with pytest.raises(BackendError):
                pool.copy_blocks(*pair)
        pool.copy_blocks(dev([0, 9, -1]), dev([4, 1, 1]))
        with pytest.raises(DeviceIndexError) as ei:
            pool.check()
        assert ei.value.bits == COPY
        t[:, :, 4], e[:, :, 4] = t[:, :, 0].clone(), e[:, :, 0].clone()
        assert torch.equal(pool.tensor(), t) and torch.equal(pool.exponents(), e)


def test_offsets_past_32_bits():
    """Blocks whose tiles lie more than 4 GiB into a plane."""
    r = np.random.default_rng(0)
    hkv, d, blocks = 8, 128, 270_000  # 16 KiB of a block and plane
    with DeviceKv8Pool(PoolDesc(1, hkv, hkv, d, blocks, "bf16")) as pool:
        table = [blocks - 1, 3, blocks - 7]
        k, v = (rows(r, 40, hkv, d, "bf16") for _ in range(2))
        pool.append(0, dev(k, "bf16"), dev(v, "bf16"), [40], [0, 3], table, [40])
        out = pool.gather(0, [0, 3], table, [40])
        pool.check()
        want = kv8.Kv8(3, hkv, d)
        want.append(k, v, [40], [40], [[0, 1, 2]])
        for kv in range(2):
            assert np.array_equal(host(out[kv]).reshape(hkv, 40, d), want.rows(kv, [0, 1, 2], 40))
        pool.copy_blocks([blocks - 1], [blocks - 2])
        again = pool.gather(0, [0, 1], [blocks - 2], [16])
        assert np.array_equal(host(again[0]).reshape(hkv, 16, d), want.rows(0, [0], 16))
        q = rows(r, 1, hkv, d, "bf16", False)
        o = host(pool.decode_attention(0, dev(q, "bf16"), [0, 3], table, [40]))
        o2 = host(pool.extend_attention(0, dev(q, "bf16"), [1], [0, 3], table, [40]))
        ref = want.attend(q, [1], [40], [[0, 1, 2]], d ** -0.5)
        assert_attention(o, ref, "bf16")
        assert_attention(o2, ref, "bf16")


# -- refusals ---------------------------------------------------------------------------


def test_refusals():
    import torch

    b = Batch([2, 3], [20, 30])
    with make_pool(b, 2, 2, 64, "bf16") as pool:
        k = dev(np.zeros((5, 2, 64)), "bf16")
        ip, ix, cl = b.host()
        pool.append(0, k, k, b.new, ip, ix, cl)
        shared = ix.copy()
        shared[ip[1] + 1] = ix[1]  # the block that the first sequence writes
        prefix = ix.copy()
        prefix[ip[1]] = ix[0]      # one that nothing writes
        pool.append(0, k, k, b.new, ip, prefix, cl)
        bad_id = ix.copy()
        bad_id[0] = b.blocks
        q = dev(np.zeros((5, 4, 64)), "bf16")
        freq = torch.from_numpy(rope_inv_freq(64, 1e4)).cuda()
        for call in (
            lambda: pool.append(0, k, k, b.new, ip, shared, cl),
            lambda: pool.append(0, k, k, b.new, ip, bad_id, cl),
            lambda: pool.append(1, k, k, b.new, ip, ix, cl),
            lambda: pool.append(-1, k, k, b.new, ip, ix, cl),
            lambda: pool.append(0, k, k, [2, 2], ip, ix, cl),
            lambda: pool.append(0, k, k, [4, 1], ip, ix, [3, 30]),
            lambda: pool.append(0, k, k, [6, -1], ip, ix, cl),
            lambda: pool.append(0, k, k, b.new, ip, ix, [20, 64]),
            lambda: pool.append(0, k, k, b.new, [0, 3, 2], ix, cl),
            lambda: pool.append(0, k, k, b.new, [1, 2, 4], ix, cl),
            lambda: pool.append(0, k, k, b.new, [0, 2, 99], ix, cl),
            lambda: pool.append(0, k.float(), k, b.new, ip, ix, cl),
            lambda: pool.append(0, k.cpu(), k, b.new, ip, ix, cl),
            lambda: pool.append(0, k, k.transpose(0, 1).contiguous().transpose(0, 1), b.new, ip, ix, cl),
            lambda: pool.append(0, k, k, b.new, dev(ip), dev(ix), dev(cl)),
            lambda: pool.append(0, k, k, b.q_indptr(), *b.device()),
            lambda: pool.append(0, k, k, b.q_indptr().long(), *b.device(), max_q_len=3),
            lambda: pool.append(0, k, k, b.q_indptr(), *b.device(), max_q_len=-3),
            lambda: pool.qk_norm_rope_append(0, q, k, k, b.new, ip, ix, cl, gated=True),
            lambda: pool.qk_norm_rope_append(0, q, k, k, b.new, ip, ix, cl, gated=False, q_norm_w=freq),
            lambda: pool.qk_norm_rope_append(0, q, k, k, b.new, ip, ix, cl, gated=False, inv_freq=freq[:5]),
            lambda: pool.qk_norm_rope_append(0, q, k, k, b.new, ip, ix, cl, gated=False, inv_freq=torch.cat([freq, freq])),
            lambda: pool.qk_norm_rope_append(0, q, k, k, b.new, ip, ix, cl, gated=False, inv_freq=freq,
                                             rope_factor=float("inf")),
            lambda: pool.qk_norm_rope_append(0, q, k, k, b.new, ip, ix, cl, gated=False, positions=[1, 2, 3]),
            lambda: pool.qk_norm_rope_append(0, q, k, k, b.new, ip, ix, cl, gated=False, positions=[1, 2, 3, 4, -1]),
            lambda: pool.qk_norm_rope_append(0, q, q[:, :2].contiguous(), k, b.new, ip, ix, cl, gated=False,
                                             out=k.view(-1)[:0]),
            lambda: pool.gather(0, ip, ix, [20, -1]),
            lambda: pool.gather(0, ip, bad_id, cl),
            lambda: pool.gather(0, ip, ix, cl, out_k=torch.empty(9, device="cuda", dtype=torch.bfloat16)),
            lambda: pool.gather(0, *b.device(), max_ctx_len=30),
            lambda: pool.copy_blocks([1], dev([2])),
            lambda: pool.copy_blocks([1, 2], [3]),
        ):
            with pytest.raises(BackendError):
                call()
        x = torch.zeros(5 * 4 * 64 + 64, device="cuda", dtype=torch.bfloat16)
        with pytest.raises(BackendError):  # an output that overlaps its input by a part
            pool.qk_norm_rope_append(0, x[:1280].view(5, 4, 64), k, k, b.new, ip, ix, cl, gated=False,
                                     out=x[64:].view(5, 4, 64))
        with pytest.raises(BackendError):  # 8-byte aligned
            y = torch.zeros(5 * 2 * 64 + 8, device="cuda", dtype=torch.bfloat16)[4:644].view(5, 2, 64)
            pool.append(0, y, y, b.new, ip, ix, cl)
        pool.check()
    with pytest.raises(BackendError):  # closed
        pool.append(0, k, k, b.new, ip, ix, cl)


def test_null_arguments():
    """The C entry points refuse NULL where a pointer is needed, with a pool and without."""
    import ctypes

    lib = _lib.device_lib()
    names = [n for n in _lib.DEVICE_SIGNATURES if n.startswith("mkv_kv8_") and n != "mkv_kv8_pool_destroy"]
    assert len(names) > 15
    with DeviceKv8Pool(PoolDesc(1, 1, 1, 64, 4, "f32")) as pool:
        for name in names:
            fn = getattr(lib, name)
            zeros = [t(0) if t in (ctypes.c_float, ctypes.c_int32, ctypes.c_int, ctypes.c_int64, ctypes.c_uint32,
                                   ctypes.c_uint64) else None for t in fn.argtypes]
            assert fn(*zeros) == 1, name  # MKV_ERR_INVALID_ARGUMENT
            if not ("append" in name or "gather" in name or "attention" in name or "copy" in name):
                continue
            ones = [z if z is None else type(z)(1) for z in zeros]
            ones[0] = pool._h
            ones[1] = type(ones[1])(0) if ones[1] is not None else None  # the layer
            assert fn(*ones) == 1, name
        pool.check()


def test_host_metadata_is_not_captured():
    import torch

    b = Batch([2], [20])
    with make_pool(b, 1, 1, 64, "bf16") as pool:
        want = fill(pool, 1)
        x = rows(np.random.default_rng(1), 2, 1, 64, "bf16")
        k, qi, t = dev(x, "bf16"), b.q_indptr(), b.device()
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(BackendError):
                pool.append(0, k, k, b.new, *b.host())
            with pytest.raises(BackendError):
                pool.copy_blocks([0], [1])
            pool.append(0, k, k, qi, *t, max_q_len=2)
        graph.replay()
        torch.cuda.synchronize()
        want.append(x, x, b.new, b.ctx, b.tables)
        assert_same(pool, want)


# -- streams, graphs --------------------------------------------------------------------


def test_captured_steps_follow_lengths_and_tables():
    """append and norm + RoPE + append in a graph, replayed with other lengths and rows, eager
    work and synchronizations in between."""
    import torch

    r = np.random.default_rng(11)
    b = Batch([3, 1], [3, 1], spare=4)
    with make_pool(b, 2, 2, 64, "bf16", layers=2) as pool:
        fill(pool, 1)
        wants = [read(pool, layer) for layer in range(2)]
        k, v, q = dev(np.zeros((4, 2, 64)), "bf16"), dev(np.zeros((4, 2, 64)), "bf16"), dev(np.zeros((4, 4, 64)), "bf16")
        qi, (ip, ix, cl) = b.q_indptr(), b.device()
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pool.append(0, k, v, qi, ip, ix, cl, max_q_len=3)
            pool.qk_norm_rope_append(1, q, k, v, qi, ip, ix, cl, max_q_len=3, gated=False, out=out)
        ctx = [3, 1]
        for step in range(6):
            x, y = (rows(r, 4, 2, 64, "bf16") for _ in range(2))
            z = rows(r, 4, 4, 64, "bf16")
            k.copy_(dev(x, "bf16"))
            v.copy_(dev(y, "bf16"))
            q.copy_(dev(z, "bf16"))
            cl.copy_(dev(ctx))
            graph.replay()
            torch.cuda.synchronize()
            for layer, w in enumerate(wants):
                w.append(x, y, b.new, ctx, b.tables)
                assert_same(pool, w, layer)
            assert np.array_equal(host(out), z)
            ctx = [c + n + step for c, n in zip(ctx, b.new)]
            torch.zeros(1000, device="cuda").sum()
        pool.check()


def test_another_stream():
    """A call given a stream runs there, after what that stream has before it."""
    import torch

    r = np.random.default_rng(12)
    b = Batch([64] * 4, [64, 80, 100, 64])
    with make_pool(b, 4, 1, 128, "bf16") as pool:
        want = fill(pool, 1)
        k, v = (rows(r, b.tokens, 4, 128, "bf16") for _ in range(2))
        kd, vd = dev(k, "bf16"), dev(v, "bf16")
        late = [torch.zeros_like(kd), torch.zeros_like(vd)]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        big = torch.randn(4096, 4096, device="cuda")
        with torch.cuda.stream(side):
            for _ in range(8):
                big = big @ big * 1e-3
            late[0].copy_(kd)
            late[1].copy_(vd)
        pool.append(0, *late, b.new, *b.host(), stream=side)
        out = pool.gather(0, *b.host(), stream=side)
        pool.check(stream=side)
        want.append(k, v, b.new, b.ctx, b.tables)
        assert_same(pool, want)
        assert np.array_equal(host(out[1]), np.concatenate([want.rows(1, t, c).ravel() for t, c in zip(b.tables, b.ctx)]))
