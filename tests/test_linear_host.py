"""What the linear-attention and norm entry points refuse before they touch a
device, and the state pool's size (CPU)."""
from __future__ import annotations

import ctypes

import pytest

from mitten_amd import BackendError, DeviceStatePool, StateDesc, _lib, state_required_bytes

GOOD = dict(num_layers=2, num_k_heads=16, num_v_heads=32, k_dim=128, v_dim=128, num_slots=10, dtype="bf16")


def test_required_bytes():
    assert state_required_bytes(StateDesc(**GOOD)) == 2 * 10 * 32 * 128 * 128 * 4
    assert state_required_bytes(StateDesc(**{**GOOD, "dtype": "f32", "k_dim": 64, "v_dim": 256})) == \
        2 * 10 * 32 * 64 * 256 * 4


@pytest.mark.parametrize("bad", [
    dict(num_layers=0), dict(num_layers=65536), dict(num_k_heads=0), dict(num_k_heads=5), dict(num_v_heads=2048),
    dict(k_dim=32), dict(k_dim=96), dict(v_dim=512), dict(num_slots=0), dict(num_slots=2 ** 31), dict(dtype="fp8"),
    dict(num_layers=65535, num_slots=2 ** 31 - 1, num_v_heads=1024, k_dim=256, v_dim=256),
])
def test_descriptor_validation(bad):
    with pytest.raises((BackendError, KeyError)):
        state_required_bytes(StateDesc(**{**GOOD, **bad}))


def test_pool_without_device_fails_cleanly():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a HIP device is present")
    with pytest.raises(BackendError) as ei:
        DeviceStatePool(StateDesc(**GOOD))
    assert ei.value.status == 5  # MKV_ERR_NO_DEVICE


def test_null_pools_are_refused():
    lib = _lib.device_lib()
    for name, (_, args) in _lib.DEVICE_SIGNATURES.items():
        if name.startswith(("mkv_state_", "mkv_linear_")) and name not in ("mkv_state_required_bytes",
                                                                            "mkv_state_pool_destroy"):
            zeros = [None if a is _lib.P or hasattr(a, "contents") else a(0) for a in args]
            assert getattr(lib, name)(*zeros) == 1, name
    assert lib.mkv_state_pool_destroy(None) == 0


@pytest.mark.parametrize("change,msg", [
    (dict(dtype=2), "dtype"), (dict(dim=12), "dim"), (dict(dim=16392), "dim"), (dict(dim=0), "dim"),
    (dict(rows=-1), "num_rows"), (dict(rows=1 << 24), "num_rows"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(scales=None), "both"), (dict(fp8=None, out=None, scales=None), "output"),
    (dict(group=48), "group"), (dict(group=-8), "group"), (dict(group=4), "group"), (dict(group=128), "group"),
    (dict(fp8=None, scales=None, group=8), "group"),
])
def test_norm_refusals(change, msg):
    """Refused on its numbers alone: no pointer here is one."""
    a = dict(dtype=1, dim=64, rows=4, eps=1e-6, out=16, fp8=32, scales=48, group=0)
    a.update(change)
    lib = _lib.device_lib()
    p = ctypes.c_void_p
    st = lib.mkv_add_rms_norm(0, p(64), None, p(80), a["eps"], a["rows"], a["dim"], a["dtype"], None, p(a["out"]),
                              p(a["fp8"]), p(a["scales"]), a["group"], None)
    assert st == 1 and msg in lib.mkv_last_error().decode()


def test_norm_refuses_one_buffer_for_two_outputs():
    lib = _lib.device_lib()
    p = ctypes.c_void_p
    st = lib.mkv_add_rms_norm(0, p(64), p(96), p(80), 1e-6, 4, 64, 1, p(16), p(16), None, None, 0, None)
    assert st == 1 and "same" in lib.mkv_last_error().decode()


@pytest.mark.parametrize("place", [
    dict(fp8="x"), dict(fp8="residual"), dict(fp8="out"), dict(fp8="sum"), dict(fp8="weight"), dict(scales="x"),
    dict(scales="fp8"), dict(scales="weight"), dict(out="weight"), dict(sum="weight"), dict(out=("x", 16)),
    dict(out=("x", -16)), dict(sum=("residual", 512 - 16)), dict(sum=("out", 16)), dict(fp8=("scales", -240)),
])
def test_norm_refuses_outputs_over_other_buffers(place):
    """4 rows of 64 bf16: 512 bytes each, 256 of e4m3, 16 of scales (256 bytes after the e4m3 rows' end)."""
    at = dict(x=1 << 20, residual=2 << 20, weight=3 << 20, sum=4 << 20, out=5 << 20, fp8=6 << 20, scales=7 << 20)
    for k, v in place.items():
        at[k] = at[v] if isinstance(v, str) else at[v[0]] + v[1]
    lib, p = _lib.device_lib(), ctypes.c_void_p
    st = lib.mkv_add_rms_norm(0, p(at["x"]), p(at["residual"]), p(at["weight"]), 1e-6, 4, 64, 1, p(at["sum"]),
                              p(at["out"]), p(at["fp8"]), p(at["scales"]), 0, None)
    assert st == 1 and "overlaps" in lib.mkv_last_error().decode()
