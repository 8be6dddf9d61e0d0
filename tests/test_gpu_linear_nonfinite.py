"""Infinities and NaN in linear attention: the classes (finite, Inf with its
sign, NaN) of outputs and states are those of the recurrence in f32, whatever
form computes them (a step, a chunk, whole sequences, segments)."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import DeviceStatePool, StateDesc
from oracle import oracle as orc
from tests.helpers import to_device, to_host, widen
from tests.test_gpu_linear import f32_bound, inputs, out_bound, reference

pytestmark = pytest.mark.gpu


def run(form, q, k, v, g, s0, dtype):
    """(outputs, state) of one sequence: "step" token by token, "whole" (a
    workspace with no room), "segments" (as planned), "many" (with 140 others like
    it, which take workgroups of 128 columns where v has them)."""
    import torch

    hk, dk, (n, hv, dv) = q.shape[1], q.shape[2], v.shape
    dev = [to_device(orc.f32_to_bf16(x) if dtype == "bf16" else x) for x in (q, k, v)] + [to_device(g)]
    many = 141 if form == "many" else 1
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, many, dtype)) as pool:
        pool.tensor().copy_(torch.from_numpy(s0[None, None]))
        if form == "many":
            o = pool.linear_extend(0, *(torch.cat([x] * many) for x in dev), [n] * many, np.arange(many))
            o, states = o.view(many, n, hv, dv), pool.tensor()[0]
            bits = [x.view(torch.int16 if x.dtype == torch.bfloat16 else torch.int32) for x in (o, states)]
            assert all(bool((x == x[:1]).all()) for x in bits), "equal sequences differ"
            o = o[0]
        elif form == "step":
            o = torch.cat([pool.linear_step(0, *(x[t:t + 1] for x in dev), [0]) for t in range(n)])
        else:
            assert form == "whole" or pool.linear_extend_workspace_size(1, n, n) > 0
            ip, slots = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [0]))
            ws = torch.empty(16, dtype=torch.uint8, device="cuda") if form == "whole" else None
            o = pool.linear_extend_device(0, *dev, ip, slots, n, workspace=ws)
        pool.check()
        return widen(to_host(o)).astype(np.float64), pool.tensor().cpu().numpy()[0, 0].astype(np.float64)


def verify(form, q, k, v, g, s0, dtype):
    """Against the recurrence in 64 bits, its decays those of f32 (0 below e^-104)."""
    n, dk = q.shape[0], q.shape[2]
    o, s = run(form, q, k, v, g, s0, dtype)
    with np.errstate(all="ignore"):
        ro, rs, ao, as_ = reference(q, k, v, np.where(g < -104, -np.inf, g), s0, dk ** -0.5)
    for got, ref, bound in ((o, ro, out_bound(n, dk, dtype, ro, ao)), (s, rs, f32_bound(n, dk, as_))):
        fine = np.isfinite(ref)
        assert np.array_equal(np.isnan(ref), np.isnan(got))
        assert np.array_equal(ref[np.isinf(ref)], got[np.isinf(ref)])
        assert np.all(np.abs(got[fine] - ref[fine]) <= bound[fine])
    return ro, rs


def make(n, dk, dv, dtype, seed):
    rng = np.random.default_rng(seed)
    q, k, v, g = inputs(rng, n, 1, 2, dk, dv, "f32")
    if dtype == "bf16":
        q, k, v = (widen(orc.f32_to_bf16(x)) for x in (q, k, v))
    return q, k, v, g, rng.standard_normal((2, dk, dv)).astype(np.float32)


FORMS = [("step", 20), ("whole", 20), ("whole", 200), ("segments", 1400), ("many", 150)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 128), (256, 64), (256, 128)])
@pytest.mark.parametrize("form,n", FORMS)
@pytest.mark.parametrize("decay", [-np.inf, -200.0, -95.0, -3.0])
def test_an_infinite_state_behind_a_decay(form, n, dk, dv, decay, dtype):
    """A decay of 0 (minus infinity, or e^-200, which is 0 in f32) makes it a
    NaN; one that is not 0, however small, and a long row of others whose product
    is 0 only by underflow leave it infinite."""
    q, k, v, g, s0 = make(n, dk, dv, dtype, 3)
    q += np.where(q >= 0, 0.25, -0.25).astype(np.float32)  # (0 x Inf in an output is not the point here)
    if dtype == "bf16":
        q = widen(orc.f32_to_bf16(q))
    s0[0, 5, 7], s0[1, 9, 11] = np.inf, -np.inf
    if decay == -3.0:
        g[:] = decay
    else:
        g[n // 2, 0] = decay
        g[n // 3, 1] = decay
    _, s = verify(form, q, k, v, g, s0, dtype)
    assert np.isnan(s[0, 5, 7]) == (decay <= -104) and np.isinf(s[0, 5, 7]) == (decay > -104)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_nan_decay_beside_a_zero_one_stays(dtype):
    q, k, v, g, s0 = make(1400, 64, 64, dtype, 4)
    g[70, 0], g[71, 0] = np.nan, -np.inf
    g[1381, 1], g[1380, 1] = np.nan, -np.inf
    _, s = verify("segments", q, k, v, g, s0, dtype)
    assert np.isnan(s).all()


def recurrence32(q, k, v, g, s0, scale):
    """The recurrence with its state held in f32 (past 3.4e38 it is infinite),
    in f64 otherwise: (outputs, state, their sums of absolute values)."""
    top = 3.4028235e38
    rep = v.shape[1] // k.shape[1]
    q, k = (np.repeat(x.astype(np.float64), rep, 1) for x in (q, k))
    v = v.astype(np.float64)
    S, A = s0.astype(np.float64), np.abs(s0.astype(np.float64))
    o, Ao = np.zeros(v.shape), np.zeros(v.shape)
    for t in range(v.shape[0]):
        d = np.exp(g[t].astype(np.float64))[:, None, None]
        kv = k[t][:, :, None] * v[t][:, None, :]
        kv = np.where(np.abs(kv) > top, np.copysign(np.inf, kv), kv)
        S, A = d * S + kv, d * A + np.abs(kv)
        S = np.where(np.abs(S) > top, np.copysign(np.inf, S), S)
        o[t], Ao[t] = scale * np.einsum("hd,hdv->hv", q[t], S), scale * np.einsum("hd,hdv->hv", np.abs(q[t]), A)
    return np.where(np.abs(o) > top, np.copysign(np.inf, o), o), S, Ao, A


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 128), (256, 64), (256, 128)])
@pytest.mark.parametrize("form,n", FORMS + [("whole", 64)])
@pytest.mark.parametrize("what", ["state", "state and decays", "score", "score of two states", "q inf", "q nan"])
def test_overflow_and_odd_queries(form, n, dk, dv, what, dtype):
    """Finite rows whose product overflows a state inside a segment ("state"),
    before decays whose product is 0 ("state and decays"); a q . k past f32's
    range where the state and the output are within it ("score", with a
    value of 1e-25; "score of two states": the product of q with a state of 1e30
    likewise); a query that is not finite."""
    q, k, v, g, s0 = make(n, dk, dv, dtype, 5)
    q += np.where(q >= 0, 0.25, -0.25).astype(np.float32)
    at = n // 3
    if what.startswith("state"):
        k[at, 0, 3], v[at, 0, 2], v[at, 1, 5] = 1e30, 1e30, -1e30
        g[at + 1:] = -2.5 if what == "state and decays" else -1e-3
    elif what == "score":
        k[at, 0, 3], q[at:at + 9, 0, 3], v[at] = 1e25, 1e20, 1e-25
    elif what == "score of two states":
        s0[0, 3, 2], g[0, 0], q[at:at + 9, 0, 3] = 1e30, -100, 1e10
    else:
        q[at, 0, 3] = np.inf if what == "q inf" else np.nan
    if dtype == "bf16":
        q, k, v = (widen(orc.f32_to_bf16(x)) for x in (q, k, v))
    o, s = run(form, q, k, v, g, s0, dtype)
    with np.errstate(all="ignore"):
        ro, rs, ao, as_ = recurrence32(q, k, v, g, s0, dk ** -0.5)
    for got, ref, bound in ((o, ro, out_bound(n, dk, dtype, ro, ao)), (s, rs, f32_bound(n, dk, as_))):
        fine = np.isfinite(ref)
        assert np.array_equal(np.isnan(ref), np.isnan(got))
        assert np.array_equal(ref[np.isinf(ref)], got[np.isinf(ref)])
        assert np.all(np.abs(got[fine] - ref[fine]) <= bound[fine])
