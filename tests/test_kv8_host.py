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
