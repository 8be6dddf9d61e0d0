"""The 8-bit pool without a GPU: its oracle against torch's own e4m3, sizes and refusals of
descriptors, and the frequencies of stretched rotary positions."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import BackendError, DeviceKv8Pool, PoolDesc, kv8_required_bytes, rope_inv_freq, rope_scaled_inv_freq
from oracle import kv8


def test_oracle_rounds_as_torch_does():
    import torch

    x = np.concatenate([np.linspace(-448, 448, 20001), kv8.GRID, (kv8.GRID[1:] + kv8.GRID[:-1]) / 2,
                        np.random.default_rng(0).standard_normal(5000) * 2.0 ** np.random.default_rng(1).integers(-12, 8, 5000)])
    x = np.clip(x, -448, 448).astype(np.float32)
    t = torch.from_numpy(x).to(torch.float8_e4m3fn)
    assert np.array_equal(kv8.to_e4m3(x), t.float().numpy())
    assert np.array_equal(kv8.from_bytes(t.view(torch.uint8).numpy()), t.float().numpy())
    every = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(every).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(kv8.from_bytes(every), want, equal_nan=True)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_tile_orders_are_permutations(d):
    for kv in range(2):
        assert np.array_equal(np.sort(kv8.tile_index(kv, d).ravel()), np.arange(16 * d))


def test_exponents():
    for amax, e in ((0.0, -100), (448.0, 0), (448.5, 1), (224.0, -1), (1e-40, -100), (3.4028235e38, 120), (1.0, -8)):
        assert kv8.exponent(amax) == e


def test_required_bytes():
    assert kv8_required_bytes(PoolDesc(28, 4, 28, 128, 512, "bf16")) == (28 * 2 * 512 * 4 * 16 * 128, 28 * 2 * 512 * 4)
    assert kv8_required_bytes(PoolDesc(2, 2, 14, 64, 7, "f32")) == (2 * 2 * 7 * 2 * 16 * 64, 2 * 2 * 7 * 2)


@pytest.mark.parametrize("bad", [dict(head_dim=32), dict(head_dim=96), dict(head_dim=512), dict(num_kv_heads=3),
                                 dict(page_size=32), dict(num_blocks=0), dict(num_layers=0)])
def test_descriptors_refused(bad):
    kw = dict(num_layers=2, num_kv_heads=4, num_q_heads=28, head_dim=128, num_blocks=10, dtype="bf16")
    kw.update(bad)
    with pytest.raises(BackendError):
        kv8_required_bytes(PoolDesc(**kw))
    with pytest.raises(BackendError):
        DeviceKv8Pool(PoolDesc(**kw))


def test_pool_without_a_device():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a HIP device is present")
    with pytest.raises(BackendError) as ei:
        DeviceKv8Pool(PoolDesc(1, 1, 1, 64, 4, "f32"))
    assert ei.value.status == 5


def test_stretched_frequencies():
    base = rope_inv_freq(128, 1e6)
    f, m = rope_scaled_inv_freq(128, 1e6, 4.0, 32768, "linear")
    assert m == 1.0 and np.allclose(f, base / 4, rtol=1e-6)
    f, m = rope_scaled_inv_freq(128, 1e6, 4.0, 32768, "ntk")
    assert m == 1.0 and np.isclose(f[0], 1.0) and np.isclose(f[-1], base[-1] / 4, rtol=1e-5)
    f, m = rope_scaled_inv_freq(128, 1e6, 4.0, 32768)
    assert np.isclose(m, 0.1 * np.log(4.0) + 1.0)
    turns = 32768 * base.astype(np.float64) / (2 * np.pi)
    assert np.allclose(f[turns > 40], base[turns > 40], rtol=1e-5)
    assert np.allclose(f[turns < 0.8], base[turns < 0.8] / 4, rtol=1e-5)
    assert np.all(np.diff(f) < 0) and np.all(f <= base * (1 + 1e-6)) and np.all(f >= base / 4 * (1 - 1e-6))
    assert np.allclose(rope_scaled_inv_freq(64, 1e4, 1.0, 4096)[0], rope_inv_freq(64, 1e4), rtol=1e-6)
    for bad in (dict(rotary_dim=7), dict(factor=0.5), dict(method="other"), dict(original_len=0)):
        kw = dict(rotary_dim=64, theta=1e4, factor=2.0, original_len=4096)
        kw.update(bad)
        with pytest.raises(ValueError):
            rope_scaled_inv_freq(**kw)


def small_pool():
    r = np.random.default_rng(5)
    o = kv8.Kv8(9, 2, 64)
    tables = [[3, 0, 7], [8, 1], [5]]
    ctx, n = [40, 17, 3], [40, 17, 3]
    k, v = (r.standard_normal((60, 2, 64)) * 2.0 ** r.integers(-3, 4, (60, 1, 1)) for _ in range(2))
    o.append(k, v, n, ctx, tables)
    return o, tables, ctx, k, v


def test_oracle_appends_to_half_a_step():
    o, tables, ctx, k, v = small_pool()
    at = 0
    for t, c in zip(tables, ctx):
        for kv, x in enumerate((k, v)):
            y = x[at: at + c].transpose(1, 0, 2)
            e = o.exp[kv][t].repeat(16, 0)[:c].T[..., None]
            assert np.all(np.abs(o.rows(kv, t, c) - y) <= np.maximum(np.abs(y) * 2.0 ** -4, 2.0 ** (e - 10.0)))
        at += c
    # A larger row raises its tile's exponent; the others move by less than half a step of it.
    before, e0 = o.rows(0, tables[1], 17), int(o.exp[0, 1, 0])
    big = np.full((1, 2, 64), 3000.0)
    o.append(big, big, [1], [18], [tables[1]])
    e = int(o.exp[0, 1, 0])
    assert e > e0 and 224 * 2.0 ** e < 3000 <= 448 * 2.0 ** e
    after = o.rows(0, tables[1], 18)
    assert np.all(np.abs(after[0, 16] - before[0, 16]) <= np.maximum(np.abs(before[0, 16]) * 2.0 ** -4, 2.0 ** (e - 10)))
    assert np.array_equal(after[:, :16], before[:, :16]) and np.all(after[:, 17] == kv8.to_e4m3(3000 * 2.0 ** -e) * 2.0 ** e)


@pytest.mark.parametrize("sink", [False, True])
def test_oracle_attention(sink):
    import torch

    o, tables, ctx, _, _ = small_pool()
    new = [5, 17, 0]
    q = np.random.default_rng(6).standard_normal((22, 6, 64))
    got = o.attend(q, new, ctx, tables, 0.125, sink)[0]
    at = 0
    for n, c, t in zip(new, ctx, tables):
        if n == 0:
            continue
        k, v = (torch.from_numpy(o.rows(kv, t, c)).repeat_interleave(3, 0) for kv in range(2))
        mask = torch.ones(n, c, dtype=torch.bool).tril(c - n)
        if sink:  # a key of zeros with values of zeros that every row sees
            k, v = (torch.nn.functional.pad(x, (0, 0, 1, 0)) for x in (k, v))
            mask = torch.nn.functional.pad(mask, (1, 0), value=True)
        want = torch.nn.functional.scaled_dot_product_attention(
            torch.from_numpy(q[at: at + n]).transpose(0, 1), k, v, attn_mask=mask, scale=0.125)
        assert np.allclose(got[at: at + n], want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-13)
        at += n


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation(interleaved):
    r = np.random.default_rng(7)
    x, w, pos = r.standard_normal((4, 3, 64)), r.standard_normal(64), np.array([0, 1, 77, 2_000_000])
    f = rope_inv_freq(32, 1e4)
    y = kv8.norm_rope(x, w, 1e-6, f, pos, 1.5, interleaved)
    z = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * (1 + w)
    c = z[..., :32].reshape(4, 3, 16, 2) if interleaved else np.stack([z[..., :16], z[..., 16:32]], -1)
    turned = (c[..., 0] + 1j * c[..., 1]) * 1.5 * np.exp(1j * pos[:, None, None] * f.astype(np.float64))
    assert np.allclose(y[..., 32:], z[..., 32:], rtol=1e-14)
    a, b = (y[..., 0:32:2], y[..., 1:32:2]) if interleaved else (y[..., :16], y[..., 16:32])
    assert np.allclose(a, turned.real, atol=1e-9) and np.allclose(b, turned.imag, atol=1e-9)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tolerances_see_mistakes(dtype):
    """The rounded exact result passes; a lost token, another head's keys, an exponent off by
    one, or a dropped scale do not."""
    from kv8_helpers import assert_attention, values

    o, tables, ctx, _, _ = small_pool()
    new, q = [1, 1, 1], np.random.default_rng(8).standard_normal((3, 6, 64))
    want = o.attend(q, new, ctx, tables, 0.125)
    assert_attention(values(want[0], dtype), want, dtype)
    heads = kv8.Kv8(9, 2, 64)
    heads.val, heads.exp = o.val[:, :, ::-1], o.exp[:, :, ::-1]
    off = kv8.Kv8(9, 2, 64)
    off.val, off.exp = o.val, o.exp.copy()
    off.exp[1, 0] += 1
    for bad in (o.attend(q, new, [39, 17, 3], tables, 0.125)[0], heads.attend(q, new, ctx, tables, 0.125)[0],
                off.attend(q, new, ctx, tables, 0.125)[0], o.attend(q, new, ctx, tables, 0.13)[0]):
        with pytest.raises(AssertionError):
            assert_attention(values(bad, dtype), want, dtype)
