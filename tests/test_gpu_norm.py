"""add_rms_norm against the formula in 64 bits:
    r = x + residual, y = r (mean r^2 + eps)^-1/2 (1 + w),
    e4m3: a = max(max |y|, 2^-100) per row or group, scale = a / 448, value e4m3(y 448 / a).

Tolerances, relative to the value: y is within (dim + 16) 2^-24 before its
rounding (a sum of dim squares, halved by the root, and a few operations; 2^-24 of the
sum x + residual's larger addend comes on top); a bf16 output adds 2^-8, an
e4m3 value 2^-4 (and half the least subnormal, 2^-10) of y 448 / a.
"""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import add_rms_norm
from mitten_amd import device_pool as dp
from oracle import oracle as orc
from tests.helpers import to_device, to_host, widen

pytestmark = pytest.mark.gpu

EPS = 1e-6


def reference(x, res, w, group):
    r = x.astype(np.float64) + (0 if res is None else res.astype(np.float64))
    with np.errstate(all="ignore"):
        y = r / np.sqrt((r * r).mean(-1, keepdims=True) + EPS) * (1 + w.astype(np.float64))
    p = y.reshape(len(y), -1, group or y.shape[1])
    scale = np.maximum(np.abs(p).max(-1), 2.0 ** -100) / 448
    return r, y, scale, (p / scale[..., None]).reshape(y.shape)


def make(rng, rows, dim, dtype, residual=True):
    size = np.exp(rng.standard_normal(dim))
    x = (rng.standard_normal((rows, dim)) * size).astype(np.float32)
    res = (2 * rng.standard_normal((rows, dim)) * size).astype(np.float32) if residual else None
    if dtype == "bf16":
        x, res = orc.f32_to_bf16(x), None if res is None else orc.f32_to_bf16(res)
    return x, res, (0.3 * rng.standard_normal(dim)).astype(np.float32)


def verify(x, res, w, dtype, got, group, fp8):
    r, y, scale, q = reference(widen(x), None if res is None else widen(res), w, group)
    big = np.abs(widen(x).astype(np.float64)) + (0 if res is None else np.abs(widen(res).astype(np.float64)))
    with np.errstate(all="ignore"):
        f = np.abs(y) / np.where(r == 0, 1, np.abs(r))
    err = (x.shape[1] + 16) * 2.0 ** -24 * np.abs(y) + 2.0 ** -24 * big * f
    step = 0 if dtype == "f32" else 2.0 ** -8
    s, o, b, c = got
    if s is not None:
        assert np.all(np.abs(widen(to_host(s)) - r) <= 2.0 ** -24 * big + step * np.abs(r))
    if o is not None:
        assert np.all(np.abs(widen(to_host(o)) - y) <= err + step * np.abs(y) * 1.01 + 1e-37)
    if fp8:
        b, c = b.float().cpu().numpy().astype(np.float64), c.cpu().numpy().astype(np.float64)
        most = err.reshape(*scale.shape, -1).max(-1) / 448 + 2.0 ** -23 * scale
        assert c.shape == scale.shape and np.all(np.abs(c - scale) <= most)
        wide = np.repeat(scale, y.shape[1] // scale.shape[1], 1)
        rel = err / wide + 2 * np.abs(q) * np.repeat(most / scale, y.shape[1] // scale.shape[1], 1)
        assert np.all(np.abs(b) <= 448) and np.all(np.abs(b - q) <= 2.0 ** -4 * np.abs(q) * 1.01 + 2.0 ** -10 + rel)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,dim", [(1, 8), (3, 64), (5, 512), (2, 520), (7, 896), (64, 2048), (3, 3584), (2, 4104),
                                      (2, 8192), (3, 11008), (2, 16384)])
def test_norm_matches_the_formula(rows, dim, dtype):
    rng = np.random.default_rng(dim + rows)
    x, res, w = make(rng, rows, dim, dtype)
    dx, dr, dw = (to_device(a) for a in (x, res, w))
    verify(x, res, w, dtype, add_rms_norm(dx, dw, EPS, residual=dr), 0, False)
    got = add_rms_norm(dx, dw, EPS)
    assert got[0] is None and got[2] is None and got[3] is None
    verify(x, None, w, dtype, got, 0, False)
    for group in {0, 8, dim if dim % 128 else 128, dim // 2 if dim % 16 == 0 else dim}:
        got = add_rms_norm(dx, dw, EPS, residual=dr, fp8=True, group=group, both=group == 8)
        assert (got[1] is not None) == (group == 8)
        verify(x, res, w, dtype, got, group, True)


def test_many_rows():
    rng = np.random.default_rng(1)
    x, res, w = make(rng, 5003, 896, "bf16")
    dx, dr, dw = (to_device(a) for a in (x, res, w))
    verify(x, res, w, "bf16", add_rms_norm(dx, dw, EPS, residual=dr, fp8=True, group=128, both=True), 128, True)


def test_in_place():
    """The sum into the residual and the output into x: what separate buffers get."""
    rng = np.random.default_rng(2)
    x, res, w = make(rng, 9, 3584, "bf16")
    dx, dr, dw = (to_device(a) for a in (x, res, w))
    want = add_rms_norm(dx, dw, EPS, residual=dr)
    got = add_rms_norm(dx, dw, EPS, residual=dr, residual_out=dr, out=dx)
    assert got[0] is dr and got[1] is dx
    assert all((a == b).all() for a, b in zip(want[:2], got[:2]))


def test_zero_rows_tiny_rows_and_no_rows():
    import torch

    w = torch.zeros(64, device="cuda")
    x = torch.zeros(3, 64, device="cuda")
    x[1] = 1e-30
    x[2, 5] = 3e18
    _, y, q, s = add_rms_norm(x, w, EPS, fp8=True, both=True)
    assert (y[0] == 0).all() and (q.float()[0] == 0).all() and s[0, 0].item() == np.float32(2.0 ** -100) / np.float32(448)
    assert torch.isfinite(y).all() and torch.isfinite(s).all() and torch.isfinite(q.float()).all()
    assert q.float()[1].unique().tolist() == [448.0] and q.float()[2].sum().item() == 448.0
    assert add_rms_norm(x[:0], w, EPS)[1].shape == (0, 64)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("group", [0, 64])
def test_a_nan_or_inf_stays_in_its_row(bad, group):
    """A NaN makes its row NaN, scales and bytes too; an infinity leaves
    itself NaN and the rest of its row zero, as the formula has it."""
    import torch

    rng = np.random.default_rng(3)
    x, res, w = make(rng, 4, 256, "f32")
    x[2, 70] = bad
    dx, dr, dw = (to_device(a) for a in (x, res, w))
    _, y, q, s = (t.float().cpu().numpy() for t in add_rms_norm(dx, dw, EPS, residual=dr, fp8=True, group=group, both=True))
    others = [0, 1, 3]
    assert np.isfinite(y[others]).all() and np.isfinite(q[others]).all() and np.isfinite(s[others]).all()
    hit = np.isnan(y[2])
    assert hit[70] and (hit.all() if np.isnan(bad) else hit.sum() == 1 and np.all(np.delete(y[2], 70) == 0))
    for j in range(s.shape[1]):
        part = slice(j * (group or 256), (j + 1) * (group or 256))
        assert np.isnan(s[2, j]) == hit[part].any() and np.isnan(q[2, part]).all() == hit[part].any()


def test_other_streams_and_captures():
    import torch

    rng = np.random.default_rng(4)
    x, res, w = make(rng, 33, 2048, "bf16")
    dx, dr, dw = (to_device(a) for a in (x, res, w))
    want = add_rms_norm(dx, dw, EPS, residual=dr, fp8=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = add_rms_norm(dx, dw, EPS, residual=dr, fp8=True, stream=side)
    side.synchronize()
    assert (got[0] == want[0]).all() and (got[2].float() == want[2].float()).all() and (got[3] == want[3]).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = add_rms_norm(dx, dw, EPS, residual=dr, fp8=True)
    for _ in range(3):
        for t in (got[0], got[3]):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (got[0] == want[0]).all() and (got[2].float() == want[2].float()).all() and (got[3] == want[3]).all()


def test_refusals():
    import torch

    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(64, device="cuda")
    for call, msg in (
        (lambda: add_rms_norm(x.cpu(), w, EPS), "device tensor"),
        (lambda: add_rms_norm(x[0], w, EPS), "device tensor"),
        (lambda: add_rms_norm(x.half(), w, EPS), "dtype"),
        (lambda: add_rms_norm(x.t(), torch.zeros(4, device="cuda"), EPS), "contiguous"),
        (lambda: add_rms_norm(x, w[:32], EPS), "weight has shape"),
        (lambda: add_rms_norm(x, w.double(), EPS), "weight has dtype"),
        (lambda: add_rms_norm(x, w, -1.0), "eps"),
        (lambda: add_rms_norm(x, w, float("nan")), "eps"),
        (lambda: add_rms_norm(x, w, EPS, residual=x.float()), "residual has dtype"),
        (lambda: add_rms_norm(x, w, EPS, residual=x[:2]), "residual has shape"),
        (lambda: add_rms_norm(x, w, EPS, fp8=True, group=48), "group"),
        (lambda: add_rms_norm(x, w, EPS, fp8=True, group=4), "group"),
        (lambda: add_rms_norm(x, w, EPS, group=8), "e4m3"),
        (lambda: add_rms_norm(torch.zeros(4, 12, device="cuda"), torch.zeros(12, device="cuda"), EPS), "dim (12)"),
        (lambda: add_rms_norm(torch.zeros(1, 16392, device="cuda"), torch.zeros(16392, device="cuda"), EPS), "dim (16392)"),
        (lambda: add_rms_norm(torch.zeros(4 * 64 + 1, device="cuda")[1:].view(4, 64), w, EPS), "aligned"),
    ):
        with pytest.raises(dp.BackendError) as ei:
            call()
        assert msg in str(ei.value), (msg, str(ei.value))
