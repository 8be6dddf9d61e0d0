"""Attention over V rows near the largest numbers that f32 and bf16 hold, in every form of the
8-bit pool's kernels: partials of a split context must not leave f32 where the result does not."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import kv8

from kv8_forms import attend, chunks
from kv8_helpers import Batch, assert_attention, dev, fill, host, make_pool, read, values

pytestmark = pytest.mark.gpu


def large(pool, lo, hi):
    """V bytes up to 240 (240 * 2^120 is finite) under exponents lo..hi."""
    import torch

    fill(pool, 1)
    r = np.random.default_rng(2)
    v = kv8.to_e4m3(np.clip(r.standard_normal(tuple(pool.tensor()[0, 1].shape)) * 120, -240, 240))
    pool.tensor()[0, 1] = torch.from_numpy(v).float().to(torch.float8_e4m3fn).view(torch.uint8).cuda()
    pool.exponents()[0, 1] = torch.from_numpy(r.integers(lo, hi + 1, tuple(pool.exponents()[0, 1].shape))).to(torch.int8).cuda()
    return read(pool)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", ["seq", "split", "whole", "cut"])
@pytest.mark.parametrize("lo,hi", [(105, 120), (120, 120)])
@pytest.mark.parametrize("ctx", [[1, 40, 300], [9000, 1, 1030]])
def test_values_near_the_largest(form, dtype, lo, hi, ctx):
    b = Batch(chunks(form, ctx, 20), ctx)
    d = 64
    with make_pool(b, 2, 3, d, dtype) as pool:
        want = large(pool, lo, hi)
        q = values(np.random.default_rng(3).standard_normal((b.tokens, 6, d)), dtype)
        for sink in (False, True):
            ref = want.attend(q, b.new, ctx, b.tables, d ** -0.5, sink)
            assert np.isfinite(ref[0]).all() and np.abs(ref[0]).max() > 2.0 ** 110
            assert_attention(attend(form, pool, b, q, dtype, zero_sink=sink), ref, dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("form", ["seq", "split", "cut"])
def test_equal_keys_give_the_value(form, d):
    """Keys all alike and one value: the mean of thousands of them is the value itself."""
    ctx = [6000, 16, 333]
    b = Batch(chunks(form, ctx, 5), ctx)
    with make_pool(b, 1, 2, d, "f32") as pool:
        fill(pool, 1)
        pool.tensor()[0, 0] = 0
        pool.tensor()[0, 1] = 0x77  # 240
        pool.exponents()[0, 1] = 120
        o = attend(form, pool, b, values(np.random.default_rng(3).standard_normal((b.tokens, 2, d)), "f32"), "f32")
        assert np.all(np.abs(o / (240 * 2.0 ** 120) - 1) <= 2.0 ** -18)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_step_with_a_large_row(dtype):
    """A decode step of one token whose value is finite: the token's own value comes out."""
    b = Batch([1], [1])
    with make_pool(b, 1, 1, 64, dtype) as pool:
        k, v = np.ones((1, 1, 64)), np.full((1, 1, 64), 2.0 ** 121)
        o = pool.decode_step(0, dev(k, dtype), dev(v, dtype), dev(k, dtype), *b.host())
        assert np.array_equal(host(o), v)
