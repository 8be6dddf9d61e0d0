"""Attention over the 8-bit K/V pool on the GPU against 64 bits (oracle/kv8.py): decode steps
with their append, chunks of new tokens, both decompositions of each, what a mask hides, and
a run of the operators together. The tolerances stand in kv8_helpers.assert_attention."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import BackendError, DeviceIndexError, rope_inv_freq
from oracle import kv8

from kv8_helpers import Batch, assert_attention, assert_same, dev, fill, host, make_pool, read, values

pytestmark = pytest.mark.gpu

TABLE, BLOCK, CTX = 4, 2, 16
SHAPES = [(64, 2, 1), (64, 1, 7), (128, 4, 7), (128, 2, 16), (256, 2, 4), (64, 2, 20), (256, 1, 33), (128, 8, 1)]


def randn(seed, shape, dtype, scale=1.0):
    return values(np.random.default_rng(seed).standard_normal(shape) * scale, dtype)


# -- decode -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hkv,g", SHAPES)
@pytest.mark.parametrize("ctx", [[1, 0, 16, 17, 32, 33, 100, 0, 200, 5], [1, 3000, 0, 31, 700, 64, 33, 0]])
def test_decode_step(d, hkv, g, dtype, ctx):
    """Short contexts (one launch) and longer ones (pieces and a merge); the rows appended."""
    b = Batch([1] * len(ctx), ctx, spare=1)
    n = len(ctx)
    with make_pool(b, hkv, g, d, dtype) as pool:
        want = fill(pool, 1, zero_tiles=0.05)
        k, v = randn(2, (n, hkv, d), dtype, 3.0), randn(3, (n, hkv, d), dtype, 3.0)
        q = randn(4, (n, hkv * g, d), dtype)
        # What lies behind a context is not looked at.
        live = [c for c in ctx]
        want.append(k[[i for i in range(n) if ctx[i]]], v[[i for i in range(n) if ctx[i]]],
                    [1 if c else 0 for c in ctx], ctx, b.tables)
        poison(pool, b, live)
        for form in ("host", "device"):
            args = b.host() if form == "host" else b.device()
            kw = {} if form == "host" else dict(max_ctx_len=max(ctx) + 7)
            for sink in (False, True):
                o = pool.decode_step(0, dev(k, dtype), dev(v, dtype), dev(q, dtype), *args, zero_sink=sink, **kw)
                pool.check()
                assert_attention(host(o), want.attend(q, [1] * n, ctx, b.tables, d ** -0.5, sink), dtype)
            o2 = pool.decode_attention(0, dev(q, dtype), *args, zero_sink=True, **kw)
            assert np.array_equal(host(o), host(o2))
        got = read(pool)
        assert np.array_equal(got.exp, want.exp)
        for c, t in zip(ctx, b.tables):
            for kv in range(2):
                assert np.array_equal(got.rows(kv, t, c), want.rows(kv, t, c))


def poison(pool, b, ctx):
    """NaN bytes in every row behind a context that a new row does not clear."""
    tiles = pool.tensor().cpu().numpy()
    for c, table in zip(ctx, b.tables):
        first = c % 16
        if first < 2:  # (row 0 new: the tile is made anew)
            continue
        for kv in range(2):
            at = kv8.tile_index(kv, pool.desc.head_dim)[first:].ravel()
            for h in range(pool.desc.num_kv_heads):
                tiles[0, kv, table[c // 16], h, at] = 0x7F
    import torch

    pool.tensor().copy_(torch.from_numpy(tiles))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 256])
def test_workspace_sizes(d, dtype):
    """A workspace that holds every piece, a few, and none."""
    import torch

    ctx = [2000, 17, 1024, 900]
    b = Batch([1] * 4, ctx)
    with make_pool(b, 2, 3, d, dtype) as pool:
        want = fill(pool, 1)
        q = randn(4, (4, 6, d), dtype)
        ref = want.attend(q, [1] * 4, ctx, b.tables, d ** -0.5)
        ext = Batch([9, 0, 30, 1], ctx)
        ext.indptr, ext.ids, ext.tables = b.indptr, b.ids, b.tables
        qe = randn(5, (40, 6, d), dtype)
        refe = want.attend(qe, ext.new, ctx, b.tables, d ** -0.5)
        assert pool.workspace_size() >= 1 << 20
        one = 2 * 6 * (8 + 4 * d) + 256  # one piece of the decode kernel
        for size in (0, 16, one, 5 * one, 64 * one, pool.workspace_size()):
            ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # (NaN)
            o = pool.decode_attention(0, dev(q, dtype), *b.device(), max_ctx_len=2000, workspace=ws)
            assert_attention(host(o), ref, dtype)
            o = pool.extend_attention(0, dev(qe, dtype), ext.q_indptr(), *b.device(), max_q_len=30, max_ctx_len=2000,
                                      workspace=ws)
            assert_attention(host(o), refe, dtype)
        pool.check()


def test_more_sequences_than_one_scan():
    """5,000 sequences, one of them long."""
    n = 5000
    ctx = np.random.default_rng(0).integers(0, 40, n)
    ctx[4999], ctx[17] = 900, 500
    b = Batch([1] * n, ctx.tolist())
    with make_pool(b, 1, 2, 64, "bf16") as pool:
        want = fill(pool, 1)
        k, v, q = randn(1, (n, 1, 64), "bf16"), randn(2, (n, 1, 64), "bf16"), randn(3, (n, 2, 64), "bf16")
        o = pool.decode_step(0, *(dev(x, "bf16") for x in (k, v, q)), *b.device(), max_ctx_len=900)
        pool.check()
        live = ctx > 0
        want.append(k[live], v[live], live.astype(int), b.ctx, b.tables)
        assert_same(pool, want)
        assert_attention(host(o), want.attend(q, [1] * n, b.ctx, b.tables, 0.125), "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["decode", "extend"])
@pytest.mark.parametrize("spread", [(-60, 20), (-20, 0), (-100, 100)])
def test_exponents_far_apart(kind, dtype, spread):
    """V tiles whose scales differ by up to 2^200, in both orders; K's as usual."""
    import torch

    ctx = [40, 700, 2000]
    b = Batch([1, 40, 70] if kind == "extend" else [1] * 3, ctx)
    with make_pool(b, 2, 4, 128, dtype) as pool:
        fill(pool, 1)
        e = torch.from_numpy(np.random.default_rng(2).integers(spread[0], spread[1] + 1, pool.exponents()[:, 1].shape))
        pool.exponents()[:, 1] = e.to(torch.int8).cuda()
        want = read(pool)
        q = randn(4, (b.tokens, 8, 128), dtype)
        if kind == "extend":
            o = pool.extend_attention(0, dev(q, dtype), b.new, *b.host())
        else:
            o = pool.decode_attention(0, dev(q, dtype), *b.host())
        assert_attention(host(o), want.attend(q, b.new, ctx, b.tables, 128 ** -0.5), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["decode", "extend"])
@pytest.mark.parametrize("low", [0, 4, 8, 12, 16, 30])
def test_many_small_weights(kind, dtype, low):
    """One key far above thousands of others, whose values lie 2^-low below its own: each
    weight is small, their sum is not (e^-12 * 8191 = 0.05, and 0.4 for the second head)."""
    import torch

    d, ctx = 128, 8192
    b = Batch([1 if kind == "decode" else 20], [ctx])
    with make_pool(b, 1, 2, d, dtype) as pool:
        fill(pool, 1)
        t = b.tables[0]
        at = kv8.tile_index(0, d)[0]
        pool.tensor()[0, 0] = 0
        pool.tensor()[0, 0, t[0], 0, torch.from_numpy(at.copy()).cuda()] = 0x54  # 12 = 1.5 * 2^3
        pool.exponents()[0, 0] = 0
        pool.exponents()[0, 1] = -low
        pool.exponents()[0, 1, t[0]] = 0
        want = read(pool)
        q = np.full((b.tokens, 2, d), 1 / 128)
        q[:, 1] = 0.828125 / 128
        o = host(pool.decode_attention(0, dev(q, dtype), *b.host(), scale=1.0) if kind == "decode" else
                 pool.extend_attention(0, dev(q, dtype), b.new, *b.host(), scale=1.0))
        assert_attention(o, want.attend(q, b.new, [ctx], b.tables, 1.0), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_and_small_scores(dtype):
    """Scores of thousands (one key takes all), and of almost nothing (all alike)."""
    ctx = [50, 1500]
    b = Batch([20, 33], ctx)
    with make_pool(b, 2, 3, 64, dtype) as pool:
        want = fill(pool, 1)
        for scale in (40.0, 1e-6):
            q = randn(4, (b.tokens, 6, 64), dtype)
            o = pool.extend_attention(0, dev(q, dtype), b.new, *b.host(), scale=scale)
            assert_attention(host(o), want.attend(q, b.new, ctx, b.tables, float(np.float32(scale))), dtype)
            o = pool.decode_attention(0, dev(q[:2], dtype), *b.host(), scale=scale)
            assert_attention(host(o), want.attend(q[:2], [1, 1], ctx, b.tables, float(np.float32(scale))), dtype)


def test_nan_reaches_those_that_see_it():
    """NaN in a query row, in K and in V: rows that see it are NaN, others as without it."""
    ctx = [300, 90]
    for dtype in ("f32", "bf16"):
        b = Batch([150, 90], ctx)
        with make_pool(b, 2, 3, 64, dtype) as pool:
            fill(pool, 1)
            for s, pos, kv, h, dim in ((0, 200, 1, 0, 5), (0, 299, 1, 1, 63), (0, 20, 1, 1, 8), (1, 40, 0, 0, 7),
                                       (1, 71, 1, 1, 0), (1, 89, 0, 1, 1)):
                at = int(kv8.tile_index(kv, 64)[pos % 16, dim])
                pool.tensor()[0, kv, b.tables[s][pos // 16], h, at] = 0xFF if dim % 2 else 0x7F
            want = read(pool)
            q = randn(4, (b.tokens, 6, 64), dtype)
            q[17, 2, 9] = np.nan
            ref = want.attend(q, b.new, ctx, b.tables, 0.125)
            assert np.isnan(ref[0]).any() and np.isfinite(ref[0]).any()
            assert_attention(host(pool.extend_attention(0, dev(q, dtype), b.new, *b.host())), ref, dtype)
            one = want.attend(q[16:18], [1, 1], ctx, b.tables, 0.125)
            assert_attention(host(pool.decode_attention(0, dev(q[16:18], dtype), *b.host())), one, dtype)


@pytest.mark.parametrize("long", [False, True])
def test_bad_sequences_are_skipped_and_reported(long):
    import torch

    ctx = [20, 36, 900 if long else 50, 40]
    b = Batch([4] * 4, ctx)
    d = 64
    for what, bit in (("ctx", CTX), ("max", CTX), ("table", TABLE), ("id", BLOCK)):
        with make_pool(b, 2, 2, d, "bf16") as pool:
            want = fill(pool, 6)
            indptr, ids, lens = b.indptr.astype(np.int64), b.ids.astype(np.int64), list(ctx)
            tables = [list(t) for t in b.tables]
            if what == "ctx":
                lens[1] = -1
            elif what == "max":
                lens[1] = 2_000_000_000
            elif what == "table":
                indptr[2] -= 1
                tables[2] = list(ids[indptr[2]: indptr[3]])
            else:
                ids[indptr[1] + 1] = b.blocks  # (the middle block of three)
            t = dev(indptr), dev(ids), dev(lens)
            top = max(ctx)
            q = randn(4, (16, 4, d), "bf16")
            good = [0, 2, 3]
            for kind in ("decode", "step", "extend"):
                n = 4 if kind == "extend" else 1
                x = q[: 4 * n]
                out = torch.full((4 * n + 2, 4, d), 7.0, device="cuda", dtype=torch.bfloat16)
                if kind == "extend":
                    pool.extend_attention(0, dev(x, "bf16"), b.q_indptr(), *t, max_q_len=4, max_ctx_len=top, out=out[:-2])
                elif kind == "decode":
                    pool.decode_attention(0, dev(x, "bf16"), *t, max_ctx_len=top, out=out[:-2])
                else:
                    k = randn(5, (4, 2, d), "bf16")
                    pool.decode_step(0, dev(k, "bf16"), dev(k, "bf16"), dev(x, "bf16"), *t, max_ctx_len=top, out=out[:-2])
                    for i in good + ([1] if what == "id" else []):  # (the last block's id is good)
                        want.append(k[i: i + 1], k[i: i + 1], [1], [lens[i]], [tables[i]])
                    assert_same(pool, want)
                with pytest.raises(DeviceIndexError) as ei:
                    pool.check()
                assert ei.value.bits == bit, (what, kind)
                y = host(out)
                assert np.all(y[-2:] == 7.0)
                for i in good:
                    ref = want.attend(x[n * i: n * i + n], [n], [lens[i]], [tables[i]], d ** -0.5)
                    assert_attention(y[n * i: n * i + n], ref, "bf16")
                if what == "id":  # attended without that block
                    assert np.isfinite(y[n: 2 * n]).all()
                else:
                    assert np.all(y[n: 2 * n] == 7.0)


# -- extend -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,hkv,g", SHAPES)
def test_extend(d, hkv, g, dtype):
    """Whole prompts and chunks after a cache, one token and many, ends inside blocks, nothing
    new; the last rows of the buffers belong to nobody."""
    import torch

    for new, ctx in (([1, 16, 17, 0, 33, 5], [1, 16, 17, 9, 33, 700]), ([130, 1, 0, 77], [1100, 64, 0, 77]),
                     ([1, 2, 3], [1500, 33, 1000])):
        b = Batch(new, ctx, spare=1)
        n = b.tokens
        with make_pool(b, hkv, g, d, dtype) as pool:
            fill(pool, 1, zero_tiles=0.05)
            poison(pool, b, ctx)
            want = read(pool)
            q = randn(4, (n, hkv * g, d), dtype)
            for sink in (False, True):
                ref = want.attend(q, new, ctx, b.tables, d ** -0.5, sink)
                o = pool.extend_attention(0, dev(q, dtype), new, *b.host(), zero_sink=sink)
                assert_attention(host(o), ref, dtype)
            out = torch.full((n + 3, hkv * g, d), 7.0, device="cuda", dtype=pool.torch_dtype)
            qd = torch.full((n + 3, hkv * g, d), float("nan"), device="cuda", dtype=pool.torch_dtype)
            qd[:n] = dev(q, dtype)
            pool.extend_attention(0, qd, b.q_indptr(), *b.device(), max_q_len=max(new), max_ctx_len=max(ctx),
                                  zero_sink=True, out=out)
            pool.check()
            assert_attention(host(out[:n]), ref, dtype)
            assert bool((out[n:] == 7.0).all())
            # Launched for shorter chunks and longer contexts than it finds.
            o = pool.extend_attention(0, dev(q, dtype), b.q_indptr(), *b.device(), max_q_len=1, max_ctx_len=5000,
                                      zero_sink=True)
            assert_attention(host(o), ref, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_extend_many_sequences(d, dtype):
    """Enough work that key ranges are not split, with both forms of the kernel."""
    for hkv, g, new, ctx in ((8, 2, 300, 500), (4, 1, 9, 700)):
        news = [new - i % 7 for i in range(40)]
        ctxs = [max(n, ctx - 31 * i % 400) for i, n in enumerate(news)]
        b = Batch(news, ctxs)
        with make_pool(b, hkv, g, d, dtype) as pool:
            want = fill(pool, 3)
            q = randn(4, (b.tokens, hkv * g, d), dtype)
            o = host(pool.extend_attention(0, dev(q, dtype), b.new, *b.host()))
            at = np.concatenate([[0], np.cumsum(news)])
            for i in (0, 1, 19, 38, 39):
                ref = want.attend(q[at[i]: at[i + 1]], [news[i]], [ctxs[i]], [b.tables[i]], d ** -0.5)
                assert_attention(o[at[i]: at[i + 1]], ref, dtype)


def test_extend_runs_of_ids():
    """A context of more blocks than are staged at a time (1,024), the chunk over the boundary."""
    ctx = [16400, 17000, 40000]
    new = [40, 3, 2]
    b = Batch(new, ctx)
    with make_pool(b, 1, 2, 64, "bf16") as pool:
        want = fill(pool, 3)
        q = randn(4, (b.tokens, 2, 64), "bf16", 2.0)
        ref = want.attend(q, new, ctx, b.tables, 0.125)
        import torch

        ws = torch.empty(0, dtype=torch.uint8, device="cuda")  # unsplit
        o = pool.extend_attention(0, dev(q, "bf16"), b.q_indptr(), *b.device(), max_q_len=40, max_ctx_len=40000,
                                  workspace=ws)
        assert_attention(host(o), ref, "bf16")
        assert_attention(host(pool.extend_attention(0, dev(q, "bf16"), new, *b.host())), ref, "bf16")


@pytest.mark.parametrize("count", [65, 130, 512, 513])
def test_extend_short_chunks_of_many_sequences(count):
    """Keys cut into pieces over more sequences than a wave scans at once, up to the most (and
    one more, uncut); some without new tokens, some bad."""
    import torch

    r = np.random.default_rng(count)
    ctx = r.integers(1, 2500, count)
    new = np.minimum(r.integers(0, 4, count), ctx)
    b = Batch(new.tolist(), ctx.tolist())
    with make_pool(b, 1, 2, 64, "bf16") as pool:
        want = fill(pool, 3)
        q = randn(4, (b.tokens, 2, 64), "bf16")
        lens = ctx.copy()
        bad = [i for i in (3, 64, count - 1) if new[i]]
        lens[bad] = 3000  # (more than the tables hold)
        at = np.concatenate([[0], np.cumsum(new)])
        ref = want.attend(q, b.new, b.ctx, b.tables, 0.125)
        for own in (None, torch.empty(0, dtype=torch.uint8, device="cuda")):
            out = torch.full((b.tokens, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16)
            pool.extend_attention(0, dev(q, "bf16"), b.q_indptr(), dev(b.indptr), dev(b.ids), dev(lens), max_q_len=3,
                                  max_ctx_len=3000, out=out, workspace=own)
            if bad:  # (none of the three has new tokens where there are 65)
                with pytest.raises(DeviceIndexError) as ei:
                    pool.check()
                assert ei.value.bits == TABLE
            pool.check()
            y = host(out)
            for i in bad:
                assert np.all(y[at[i]: at[i + 1]] == 7.0)
                y[at[i]: at[i + 1]] = ref[0][at[i]: at[i + 1]]
            assert_attention(y, ref, "bf16")


def test_bounds_far_above_the_lengths():
    """The largest max_ctx_len and max_q_len: sizes of launches, not of what they do."""
    top = 2 ** 31 - 1
    ctx = [40, 700, 3]
    b = Batch([9, 20, 3], ctx)
    with make_pool(b, 2, 4, 64, "f32") as pool:
        want = fill(pool, 1)
        k, v = randn(1, (32, 2, 64), "f32"), randn(2, (32, 2, 64), "f32")
        q = randn(3, (32, 8, 64), "f32")
        pool.append(0, dev(k, "f32"), dev(v, "f32"), b.q_indptr(), *b.device(), max_q_len=top)
        want.append(k, v, b.new, ctx, b.tables)
        assert_same(pool, want)
        for most in (100_000, top):
            o = pool.extend_attention(0, dev(q, "f32"), b.q_indptr(), *b.device(), max_q_len=most, max_ctx_len=most)
            assert_attention(host(o), want.attend(q, b.new, ctx, b.tables, 0.125), "f32")
            o = pool.decode_attention(0, dev(q[:3], "f32"), *b.device(), max_ctx_len=most)
            assert_attention(host(o), want.attend(q[:3], [1] * 3, ctx, b.tables, 0.125), "f32")
        out = pool.gather(0, *b.device(), max_ctx_len=top, total_tokens=sum(ctx))
        assert np.array_equal(host(out[0]), np.concatenate([want.rows(0, t, c).ravel() for t, c in zip(b.tables, ctx)]))
        pool.check()


def test_nothing_to_do():
    """No sequences, no tokens, padding alone."""
    import torch

    b = Batch([0, 0], [0, 0], spare=1)
    with make_pool(b, 2, 4, 64, "bf16") as pool:
        want = fill(pool, 1)
        none = dev(np.zeros((0, 2, 64)), "bf16")
        qn = dev(np.zeros((0, 8, 64)), "bf16")
        i0, i1 = dev([]), dev([0])
        pool.append(0, none, none, [], [0], [], [])
        pool.append(0, none, none, i1, i1, i0, i0, max_q_len=0)
        pool.append(0, none, none, [0, 0], *b.host())
        pool.append(0, none, none, b.q_indptr(), *b.device(), max_q_len=5)
        pool.qk_norm_rope_append(0, qn, none, none, [0, 0], *b.host(), gated=False)
        assert pool.decode_step(0, none, none, qn, [0], [], []).shape == (0, 8, 64)
        assert pool.extend_attention(0, qn, [], [0], [], []).shape == (0, 8, 64)
        assert pool.extend_attention(0, qn, b.q_indptr(), *b.device(), max_q_len=3, max_ctx_len=900).shape == (0, 8, 64)
        assert pool.gather(0, [0], [], [])[0].numel() == 0
        assert pool.gather(0, *b.device(), max_ctx_len=50, total_tokens=0)[1].numel() == 0
        q, k = dev(randn(1, (2, 8, 64), "bf16"), "bf16"), dev(randn(1, (2, 2, 64), "bf16"), "bf16")
        for most in (0, 40, 5000):
            out = torch.full((2, 8, 64), 7.0, device="cuda", dtype=torch.bfloat16)
            pool.decode_step(0, k, k, q, *b.device(), max_ctx_len=most, out=out)
            assert bool((out == 0).all())
        assert bool((pool.decode_step(0, k, k, q, *b.host()) == 0).all())
        pool.check()
        assert_same(pool, want)


# -- refusals ---------------------------------------------------------------------------


def test_refusals():
    import torch

    b = Batch([1, 1], [20, 30])
    with make_pool(b, 2, 2, 64, "bf16") as pool:
        fill(pool, 1)
        q, k = dev(np.zeros((2, 4, 64)), "bf16"), dev(np.zeros((2, 2, 64)), "bf16")
        ip, ix, cl = b.host()
        dv = b.device()
        shared = ix.copy()
        shared[ip[1] + 1] = ix[1]
        pool.decode_attention(0, q, ip, shared, cl)  # (nothing is written)
        odd = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")[8:]
        for call in (
            lambda: pool.decode_step(0, k, k, q, ip, shared, cl),
            lambda: pool.decode_step(0, k, None, q, ip, ix, cl),
            lambda: pool.decode_step(0, k[:1], k[:1], q, ip, ix, cl),
            lambda: pool.decode_step(0, k, k, q, ip, ix, cl, out=q),
            lambda: pool.decode_attention(0, q, ip, ix, [20, -1]),
            lambda: pool.decode_attention(0, q, ip, ix, [20, 33]),
            lambda: pool.decode_attention(0, q[:1], ip, ix, cl),
            lambda: pool.decode_attention(0, q, ip, ix, cl, scale=0.0),
            lambda: pool.decode_attention(0, q, ip, ix, cl, scale=float("nan")),
            lambda: pool.decode_attention(0, q, ip, ix, cl, workspace=odd),
            lambda: pool.decode_attention(0, q, *dv, max_ctx_len=4000, workspace=odd),
            lambda: pool.decode_attention(0, q, *dv, max_ctx_len=30, workspace=odd.cpu()),
            lambda: pool.decode_attention(0, q, *dv),
            lambda: pool.decode_attention(0, q, *dv, max_ctx_len=-1),
            lambda: pool.decode_attention(0, q, ip, dv[1], cl),
            lambda: pool.decode_attention(2, q, ip, ix, cl),
            lambda: pool.extend_attention(0, q, [1, 2], ip, ix, cl),
            lambda: pool.extend_attention(0, q, [1], ip, ix, cl),
            lambda: pool.extend_attention(0, q, b.q_indptr(), *dv, max_q_len=2),
            lambda: pool.extend_attention(0, q, b.q_indptr(), *dv, max_q_len=2, max_ctx_len=1),
            lambda: pool.extend_attention(0, q, b.q_indptr(), *dv, max_q_len=1, max_ctx_len=30, out=q),
            lambda: pool.extend_attention(0, q, b.q_indptr(), *dv, max_q_len=1, max_ctx_len=30, scale=-1.0),
            lambda: pool.bind_decode_step(k, k, q, ip, ix, cl, torch.empty_like(q), 30),
            lambda: pool.bind_decode_step(k, k, q, *dv, torch.empty_like(q)[:1], 30),
            lambda: pool.bind_decode_step(k, k, q, *dv, torch.empty_like(q), 30)(1),
        ):
            with pytest.raises(BackendError):
                call()
        pool.check()


# -- streams, graphs, the bound step ----------------------------------------------------


def test_bind_decode_step():
    import torch

    ctx = [40, 700, 0]
    b = Batch([1] * 3, ctx)
    L, hkv, g, d = 3, 2, 4, 64
    for lead in (True, False):
        pool = make_pool(b, hkv, g, d, "bf16", layers=L)
        fill(pool, 1)
        shape = (L,) if lead else ()
        k, v = (dev(randn(s, shape + (3, hkv, d), "bf16"), "bf16") for s in (1, 2))
        q = dev(randn(3, shape + (3, hkv * g, d), "bf16"), "bf16")
        out = torch.zeros_like(q)
        run = pool.bind_decode_step(k, v, q, *b.device(), out, max_ctx_len=700)
        for layer in (2, 0, 1):
            want = read(pool, layer)
            one = lambda t: t[layer] if lead else t  # noqa: E731
            run(layer)
            pool.check()
            live = [0, 1]
            want.append(host(one(k))[live], host(one(v))[live], [1, 1, 0], ctx, b.tables)
            assert_same(pool, want, layer)
            assert_attention(host(one(out)), want.attend(host(one(q)), [1] * 3, ctx, b.tables, d ** -0.5), "bf16")
        pool.close()
        with pytest.raises(BackendError):
            run(0)


@pytest.mark.parametrize("own", [False, True])
def test_captured_step(own):
    """A decode step and a chunk in a graph, replayed over growing contexts, with eager calls
    between the replays: every replay gives the eager call's bits."""
    import torch

    b = Batch([1, 1], [500, 30], spare=30)
    e = Batch([3, 2], [500, 30])
    hkv, g, d = 2, 4, 128
    with make_pool(b, hkv, g, d, "bf16") as pool:
        fill(pool, 1)
        ip, ix, cl = b.device()
        qi = e.q_indptr()
        k, v, q, qe = (dev(np.zeros(s), "bf16") for s in ((2, hkv, d), (2, hkv, d), (2, hkv * g, d), (5, hkv * g, d)))
        out, oute = torch.zeros_like(q), torch.zeros_like(qe)
        ws = torch.empty(pool.workspace_size(), dtype=torch.uint8, device="cuda") if own else None

        def step(ws):
            pool.decode_step(0, k, v, q, ip, ix, cl, max_ctx_len=960, out=out, workspace=ws)
            pool.extend_attention(0, qe, qi, ip, ix, cl, max_q_len=3, max_ctx_len=960, out=oute, workspace=ws)

        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(ws)
        ctx = [500, 30]
        for i in range(5):
            for s, t in enumerate((k, v, q, qe)):
                t.copy_(dev(randn(10 * i + s, t.shape, "bf16"), "bf16"))
            cl.copy_(dev(ctx))
            tiles, exps = pool.tensor().clone(), pool.exponents().clone()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone(), oute.clone(), pool.tensor().clone(), pool.exponents().clone()
            pool.tensor().copy_(tiles)
            pool.exponents().copy_(exps)
            want = read(pool)
            torch.cuda.synchronize()
            step(None)
            torch.cuda.synchronize()
            for x, y in zip(got, (out, oute, pool.tensor(), pool.exponents())):
                assert torch.equal(x, y)
            want.append(host(k), host(v), [1, 1], ctx, b.tables)
            assert_same(pool, want)
            assert_attention(host(oute), want.attend(host(qe), e.new, ctx, b.tables, d ** -0.5), "bf16")
            ctx = [ctx[0] + 1 + 40 * i, ctx[1] + 1]
        pool.check()


def test_two_streams_share_the_pool():
    """Calls that use the pool's workspace from two streams follow one another there."""
    import torch

    ctx = [3000, 2500]
    b = Batch([1, 1], ctx)
    hkv, g, d = 4, 7, 128
    with make_pool(b, hkv, g, d, "bf16") as pool:
        fill(pool, 1)
        t = b.device()
        qs = [dev(randn(i, (2, hkv * g, d), "bf16"), "bf16") for i in range(2)]
        want = [pool.decode_attention(0, q, *t, max_ctx_len=3000) for q in qs]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        outs = [[], []]
        for _ in range(20):
            for i, s in enumerate(streams):
                outs[i].append(pool.decode_attention(0, qs[i], *t, max_ctx_len=3000, stream=s))
        torch.cuda.synchronize()
        for i in range(2):
            for o in outs[i]:
                assert torch.equal(o, want[i])


def test_two_graphs_with_a_workspace_each():
    """Replayed at the same time on two streams."""
    import torch

    ctx = [3000, 2500]
    b, e = Batch([1, 1], ctx), Batch([4, 3], ctx)
    hkv, g, d = 4, 7, 128
    with make_pool(b, hkv, g, d, "bf16") as pool:
        fill(pool, 1)
        t, qi = b.device(), e.q_indptr()
        qs = [dev(randn(i, (2, hkv * g, d), "bf16"), "bf16") for i in range(2)]
        qe = [dev(randn(i, (7, hkv * g, d), "bf16"), "bf16") for i in range(2)]
        want = [(pool.decode_attention(0, qs[i], *t, max_ctx_len=3000),
                 pool.extend_attention(0, qe[i], qi, *t, max_q_len=4, max_ctx_len=3000)) for i in range(2)]
        outs = [(torch.zeros_like(qs[i]), torch.zeros_like(qe[i])) for i in range(2)]
        graphs = []
        torch.cuda.synchronize()
        for i in range(2):
            ws = torch.empty(pool.workspace_size(), dtype=torch.uint8, device="cuda")
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                pool.decode_attention(0, qs[i], *t, max_ctx_len=3000, out=outs[i][0], workspace=ws)
                pool.extend_attention(0, qe[i], qi, *t, max_q_len=4, max_ctx_len=3000, out=outs[i][1], workspace=ws)
            graphs.append((graph, torch.cuda.Stream(), ws))
        for _ in range(4):
            for x in outs:
                for y in x:
                    y.fill_(9.0)
            torch.cuda.synchronize()
            for _ in range(5):
                for graph, stream, _ws in graphs:
                    with torch.cuda.stream(stream):
                        graph.replay()
            torch.cuda.synchronize()
            for got, ref in zip(outs, want):
                assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_results_given_to_a_stream():
    from test_gpu_streams_given import check

    import torch

    b = Batch([8] * 4, [40, 80, 64, 900])
    with make_pool(b, 2, 4, 128, "bf16") as pool:
        fill(pool, 1)
        x = dev(randn(1, (32, 8, 128), "bf16"), "bf16")
        k = dev(randn(1, (32, 2, 128), "bf16"), "bf16")
        n = 32 * 8 * 256
        torch.cuda.synchronize()
        check(lambda s: [pool.extend_attention(0, x, b.new, *b.host(), stream=s)], [n])
        check(lambda s: [pool.qk_norm_rope_append(0, x, k, k, b.new, *b.host(), gated=False, stream=s)], [n])
        check(lambda s: [pool.decode_attention(0, x[:4], *b.host(), stream=s)], [n // 8])
        total = sum(b.ctx) * 2 * 256
        check(lambda s: list(pool.gather(0, *b.host(), stream=s)), [total] * 2)


# -- together ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,d,hkv,g", [("bf16", 128, 4, 7), ("f32", 64, 2, 7), ("bf16", 256, 2, 4)])
def test_serving_run(dtype, d, hkv, g):
    """Two layers of a serving run: prompts in two chunks, a fork that copies its last block,
    decode steps of a padded batch, a rollback, and the rows read back."""
    import torch

    r = np.random.default_rng(9)
    L, hq, freq = 2, hkv * g, rope_inv_freq(d, 1e6)
    b = Batch([0] * 4, [100, 45, 130, 0], spare=2)
    freq_d = torch.from_numpy(freq).cuda()
    w = [torch.from_numpy(r.standard_normal(d).astype(np.float32) * 0.1).cuda() for _ in range(2)]

    def put(pool, layer, new, ctx, tables, ip, ix):
        n = sum(new)
        q, k, v = (values(r.standard_normal((n, h, d)), dtype) for h in (hq, hkv, hkv))
        pos = np.concatenate([np.arange(c - m, c) for m, c in zip(new, ctx)])
        out = pool.qk_norm_rope_append(layer, dev(q, dtype), dev(k, dtype), dev(v, dtype), new, ip, ix, ctx,
                                       q_norm_w=w[0], k_norm_w=w[1], inv_freq=freq_d, gated=False)
        y = kv8.norm_rope(q, w[0].cpu().numpy(), 1e-6, freq, pos, 1.0, False)
        # sum of d squares, a few products, one rounding of pairs of up to sqrt(2) times the value
        both = np.sqrt(y ** 2 + np.roll(y, d // 2, -1) ** 2) * np.sqrt(2)
        assert np.all(np.abs(host(out) - y) <= np.abs(y) * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24) +
                      both * (d / 2 + 16) * 2.0 ** -24)
        return out

    with make_pool(b, hkv, g, d, dtype, layers=L) as pool:
        pool.tensor().fill_(0x7F)
        pool.exponents().fill_(127)
        torch.cuda.synchronize()
        ip, ix, _ = b.host()
        for new, ctx in (([64, 45, 1, 0], [64, 45, 1, 0]), ([36, 0, 129, 0], [100, 45, 130, 0])):
            for layer in range(L):
                qd = put(pool, layer, new, ctx, b.tables, ip, ix)
                o = pool.extend_attention(layer, qd, new, ip, ix, ctx)
                assert_attention(host(o), read(pool, layer).attend(host(qd), new, ctx, b.tables, d ** -0.5), dtype)
        # The fourth forks from the first at 100 tokens: six blocks shared, the seventh copied.
        spare = sorted(set(range(b.blocks)) - set(b.ids.tolist()))
        tables = [list(t) for t in b.tables]
        tables[3] = tables[0][:6] + spare[:2]
        pool.copy_blocks([tables[0][6]], [spare[0]])
        ip = np.concatenate([[0], np.cumsum([len(t) for t in tables])]).astype(np.uint32)
        ix = np.concatenate(tables).astype(np.uint32)
        ctx = [100, 45, 130, 100]
        for step in range(6):
            ctx = [c + 1 for c in ctx]
            if step == 4:
                ctx = [98, 40, 129, 99]  # back by some tokens
            for layer in range(L):
                k, v = (values(r.standard_normal((4, hkv, d)) * 2.0 ** step, dtype) for _ in range(2))
                q = values(r.standard_normal((4, hq, d)), dtype)
                want = read(pool, layer)
                o = pool.decode_step(layer, dev(k, dtype), dev(v, dtype), dev(q, dtype), ip, ix, ctx)
                want.append(k, v, [1] * 4, ctx, tables)
                got = read(pool, layer)
                for kv in range(2):
                    for c, t in zip(ctx, tables):
                        assert np.array_equal(got.rows(kv, t, c), want.rows(kv, t, c))
                assert_attention(host(o), want.attend(q, [1] * 4, ctx, tables, d ** -0.5), dtype)
        outs = pool.gather(1, ip, ix, ctx)
        want = read(pool, 1)
        for kv in range(2):
            assert np.array_equal(host(outs[kv]), np.concatenate([want.rows(kv, t, c).ravel() for t, c in zip(tables, ctx)]))
        pool.check()
