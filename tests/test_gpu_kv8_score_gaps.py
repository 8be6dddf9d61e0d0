"""Keys whose values lie far below all others' (a sink of zeros, a tile of tiny numbers) and whose
scores lie far above: the products that count are the others', however small their weights."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv8

from kv8_forms import attend, chunks
from kv8_helpers import Batch, assert_attention, fill, make_pool, read, values

pytestmark = pytest.mark.gpu

FORMS = ["seq", "split", "whole", "cut"]


def set_gap(pool, b, low, at, zeros):
    """Blocks `low` of every sequence hold V under 2^-100; token `at` of every sequence alone has
    a first K dim (16), so that q's first dim is a sixteenth of its score."""
    import torch

    d = pool.desc.head_dim
    fill(pool, 1)
    first = torch.from_numpy(kv8.tile_index(0, d)[:, 0].copy()).cuda()
    pool.tensor()[0, 0, :, :, first] = 0
    for c, t in zip(b.ctx, b.tables):
        if at < c:
            pool.tensor()[0, 0, t[at // 16], :, first[at % 16]] = 0x78  # 256
            pool.exponents()[0, 0, t[at // 16]] = -4
        for j in low:
            if j < len(t):
                pool.exponents()[0, 1, t[j]] = -100
                if zeros:
                    pool.tensor()[0, 1, t[j]] = 0
    return read(pool)


def off(got, ref, part):
    """The greatest error of a row over `part` of its norm and what f16 weights drop of it."""
    size = part * np.linalg.norm(ref[0], axis=-1) + np.sqrt(got.shape[-1]) * ref[3][..., 0]
    err = np.linalg.norm(got - ref[0], axis=-1)
    return float(np.max(np.where(err > 0, err / np.maximum(size, 1e-300), 0.0)))


def check_gap(form, dtype, ctx, low, at, zeros, gaps, d=64, most=40):
    b = Batch(chunks(form, ctx, most), ctx)
    with make_pool(b, 2, 3, d, dtype) as pool:
        want = set_gap(pool, b, low, at, zeros)
        q = np.random.default_rng(3).standard_normal((b.tokens, 6, d)) * 0.07
        for gap in gaps:
            q[..., 0] = gap / 16
            x = values(q, dtype)
            for sink in (False, True):
                ref = want.attend(x, b.new, ctx, b.tables, 1.0, sink)
                got = attend(form, pool, b, x, dtype, scale=1.0, zero_sink=sink)
                assert_attention(got, ref, dtype)
                # (Not a bound that zeros would pass: a row is off by 0.05 of it, and by what f16
                # weights drop in each of its d values, ref[3], which at a gap of 80 is 45 * 448 * 2^-132
                # for 45 keys, beside results of 2^-117: weights e^-80 times V of 2^-5 * 100 or so.)
                if not sink:
                    assert off(got, ref, 0.05) <= 1.0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("zeros", [True, False])
def test_low_tiles_first(form, dtype, zeros):
    """The first 32 keys are the low ones: the scale rises by 90 binades behind them."""
    check_gap(form, dtype, [300, 2000, 45], [0, 1], 3, zeros, [10, 40, 52, 60, 72, 80] if zeros else [10, 40, 52])


@pytest.mark.parametrize("form", FORMS)
def test_low_tiles_first_wide_heads(form):
    check_gap(form, "bf16", [200, 700], [0, 1], 3, True, [60, 80], d=256)
