"""V tiles whose scales lie far apart: a low tile between or behind the others that takes the
scores, tiles that only some rows of a chunk see, and rejected blocks."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import DeviceIndexError

from kv8_forms import attend, chunks
from kv8_helpers import Batch, assert_attention, dev, fill, host, make_pool, read, values
from test_gpu_kv8_score_gaps import FORMS, check_gap, off

pytestmark = pytest.mark.gpu


def v_exponents(pool, b, exps):
    """Block j of every sequence under exps[j % len(exps)]."""
    fill(pool, 1)
    for t in b.tables:
        for j, blk in enumerate(t):
            pool.exponents()[0, 1, blk] = exps[j % len(exps)]
    return read(pool)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("low", [[0], [1], [7], [17, 18], [4, 5, 6, 10]])
@pytest.mark.parametrize("zeros", [True, False])
def test_a_low_tile_takes_the_scores(form, dtype, low, zeros):
    gaps = [10, 40, 60, 72, 80] if zeros else [10, 40, 52]
    check_gap(form, dtype, [300, 2000, 45], low, 16 * low[0] + 5, zeros, gaps)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", ["whole", "cut"])
@pytest.mark.parametrize("g", [1, 4, 7])
@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.parametrize("exps", [(-60, 20), (20, -60), (-100, 120), (-100, -50, 0, 50, 100)])
def test_rows_before_a_tile_of_another_scale(form, dtype, g, exps):
    """Prompts and chunks: a row's result does not depend on the scales of tiles behind it."""
    new, ctx = [32, 100, 1, 45], [32, 100, 17, 500]
    b = Batch(new, ctx)
    d = 64
    with make_pool(b, 2, g, d, dtype) as pool:
        want = v_exponents(pool, b, exps)
        q = values(np.random.default_rng(4).standard_normal((b.tokens, 2 * g, d)), dtype)
        for sink in (False, True):
            ref = want.attend(q, new, ctx, b.tables, d ** -0.5, sink)
            got = attend(form, pool, b, q, dtype, zero_sink=sink)
            # (Bytes up to 448 under 2^120 are 1.75 * 2^128, past f32 and so past what an append
            # writes: a mean of them is infinite where it passes the type's largest, 2^128 less
            # half a step, and either way within the tolerance of that.)
            ref[0][np.abs(ref[0]) > 0.98 * 2.0 ** 128] = np.inf
            assert_attention(got, ref, dtype)
            fine = np.isfinite(ref[0]).all(-1)
            got, ref = got[fine], [x[fine] for x in ref]
            assert fine.mean() > 0.5 and off(got, ref, 0.01) <= 1.0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
def test_any_scales_and_wide_scores(form, dtype, d):
    """Scales of every size from tile to tile, scores of tens."""
    import torch

    ctx = [33, 900, 260, 2100]
    b = Batch(chunks(form, ctx, 50), ctx)
    with make_pool(b, 2, 2, d, dtype) as pool:
        fill(pool, 1)
        e = torch.from_numpy(np.random.default_rng(2).integers(-100, 113, tuple(pool.exponents()[0, 1].shape)))
        pool.exponents()[0, 1] = e.to(torch.int8).cuda()
        want = read(pool)
        q = values(np.random.default_rng(4).standard_normal((b.tokens, 4, d)), dtype)
        for scale in (0.05, 0.5, 2.0):
            ref = want.attend(q, b.new, ctx, b.tables, scale)
            assert_attention(attend(form, pool, b, q, dtype, scale=scale), ref, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
def test_rejected_blocks_have_no_scale(form, dtype):
    """An id outside the pool is left out, whatever block 0 holds."""
    ctx = [64, 700]
    b = Batch(chunks(form, ctx, 16), ctx)  # (rows of the last blocks)
    d = 64
    with make_pool(b, 1, 2, d, dtype) as pool:
        free = min(set(range(b.blocks)) - {x for t in b.tables for x in t})
        for t in b.tables:  # (block 0 to nobody)
            t[:] = [free if x == 0 else x for x in t]
        b.ids = np.concatenate(b.tables).astype(np.int64)
        want = v_exponents(pool, b, (-40,))
        pool.exponents()[0, 1, 0] = 100
        want = read(pool)
        q = values(np.random.default_rng(4).standard_normal((b.tokens, 2, d)), dtype)
        # Without the blocks 1 and 2 of each: as if those keys were not there.
        bad = b.ids.copy()
        for at in b.indptr[:-1].astype(int):
            bad[at + 1: at + 3] = [-1, b.blocks]
        tables = [t[:1] + t[3:] for t in b.tables]
        ref = want.attend(q, b.new, [c - 32 for c in ctx], tables, d ** -0.5)
        b.ids = bad
        with pytest.raises(DeviceIndexError):
            attend(form, pool, b, q, dtype)
        import torch

        kw = dict(max_ctx_len=20000 if form in ("split", "cut") else 700)
        if form in ("seq", "whole"):
            kw["workspace"] = torch.empty(0, dtype=torch.uint8, device="cuda")
        if form in ("seq", "split"):
            o = pool.decode_attention(0, dev(q, dtype), *b.device(), **kw)
        else:
            o = pool.extend_attention(0, dev(q, dtype), b.q_indptr(), *b.device(), max_q_len=16, **kw)
        with pytest.raises(DeviceIndexError):
            pool.check()
        assert_attention(host(o), ref, dtype)
