"""How many bits linear_extend keeps, against the recurrence in 64 bits.

With bf16 rows an output has one rounding to bf16; its operands (scores, and
the state it reads) are held in two bf16 parts, and w V in two or three.
"""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import DeviceStatePool, StateDesc
from oracle import oracle as orc
from tests.helpers import to_device, to_host, widen
from tests.test_gpu_linear import inputs, reference

pytestmark = pytest.mark.gpu


def extend(q, k, v, g, s0, dtype, whole=False):
    """One sequence from state s0: (outputs, state after it, scale), in f32."""
    import torch

    hk, dk, (n, hv, dv) = q.shape[1], q.shape[2], v.shape
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 1, dtype)) as pool:
        pool.tensor().copy_(torch.from_numpy(s0[None, None]))
        ip, slots = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [0]))
        ws = torch.empty(16, dtype=torch.uint8, device="cuda") if whole else None  # no room for segments
        o = pool.linear_extend_device(0, *(to_device(x) for x in (q, k, v, g)), ip, slots, n, workspace=ws)
        pool.check()
        return widen(to_host(o)).astype(np.float64), pool.tensor().cpu().numpy()[0, 0].astype(np.float64)


def norm(x):
    return float(np.linalg.norm(x.astype(np.float64)))


LONG = [(64, 64), (64, 128), (128, 64), (128, 128), (256, 64), (256, 256)]


@pytest.mark.parametrize("dk,dv", LONG)
@pytest.mark.parametrize("n,whole", [(40, True), (200, True), (1500, False)])
@pytest.mark.parametrize("rate", [0.01, 1.0])
def test_bf16_outputs_have_one_rounding(dk, dv, n, whole, rate):
    """The error's norm is that of rounding the exact outputs to bf16. Each
    term of an output is otherwise held to 2^-14 (w V: two truncations to 8
    bits, 2^-7 each) + 2 x 2^-15 (a state, a score: truncated, its rest
    rounded) = 2^-13, and f32 sums. Those errors are not larger against the
    terms' sum than against the outputs' norm by more than the sum's own
    cancellation, and add to an independent rounding of 2^-8 / sqrt(3) x 0.7
    = 1.6e-3 in squares: 1.2e-4 of it is 0.3%. A fifth of its size (a bf16
    operand has all of it) would be 2%."""
    rng = np.random.default_rng(dk + dv + n)
    q, k, v, g = inputs(rng, n, 1, 2, dk, dv, "bf16", rate)
    s0 = (0.3 * rng.standard_normal((2, dk, dv))).astype(np.float32)
    o, _ = extend(q, k, v, g, s0, "bf16", whole)
    ref, _, _, _ = reference(*(widen(x) for x in (q, k, v)), g, s0, dk ** -0.5)
    rounding = norm(widen(orc.f32_to_bf16(ref.astype(np.float32))) - ref)
    assert norm(o - ref) <= 1.02 * rounding


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (256, 128)])
@pytest.mark.parametrize("strong,first", [(60, 61), (40, 44), (40, 61), (62, 62)])
def test_small_decays_after_strong_ones(dtype, dk, dv, strong, first):
    """`strong` tokens of a chunk decay by e^-95 to e^-104 each, those after
    them by 1e-3: the sum is past -5,000 where differences of it decide the
    scores. Two opposite values, at `first` and the token after, cancel but
    for the decay between them; q . k is 1 throughout. Per term, bf16: 2^-15
    (a score's second part is rounded) + 2^-16 (decay differences in steps
    of 2^-17, the exponential); f32: 2^-18 (f32 operations and their sums)."""
    n, hv = 64, 32
    rng = np.random.default_rng(strong + first)
    q, k, v = (np.zeros((n, h, d), np.float32) for h, d in ((1, dk), (1, dk), (hv, dv)))
    q[:, :, 3] = k[:, :, 3] = 1
    v[first] = 2.0 ** rng.integers(-3, 3, (hv, dv))
    v[first + 1] = -v[first]
    g = -rng.uniform(95, 104, (n, hv)).astype(np.float32)
    g[strong:] = -1e-3 * rng.uniform(0.1, 2, (n - strong, hv))
    if dtype == "bf16":
        q, k, v = (orc.f32_to_bf16(x) for x in (q, k, v))
    s0 = np.zeros((hv, dk, dv), np.float32)
    o, s = extend(q, k, v, g, s0, dtype)
    scale = float(np.float32(dk ** -0.5))
    ref, rs, ao, as_ = reference(*(widen(x) for x in (q, k, v)), g, s0, scale)
    bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -15 + 2.0 ** -16) * ao if dtype == "bf16" else 2.0 ** -18 * ao
    assert np.all(np.abs(o - ref) <= bound)
    assert np.all(np.abs(s - rs) <= 2.0 ** -18 * as_)


STATE_REL = 1.5e-6  # norm of a state's error, relative (test_linear_state_parts.py)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", LONG)
@pytest.mark.parametrize("n,whole", [(2, True), (64, True), (200, True), (1500, True), (1500, False)])
def test_states_keep_f32s_accuracy(dk, dv, n, whole, dtype):
    """w V against K in three bf16 parts (24 bits): the norm of a state's error
    is that of f32 sums, some 2^-24 for each of the operations that an element
    takes, in a random order of signs: 2^-24 sqrt(2 x 64) = 7e-7 over the tokens
    that a state remembers here (rates of 1e-1 to 1, so few). Two parts leave
    1e-5."""
    rng = np.random.default_rng(dk * dv + n)
    q, k, v, g = inputs(rng, n, 1, 2, dk, dv, dtype, 0.3)
    s0 = (0.3 * rng.standard_normal((2, dk, dv))).astype(np.float32)
    _, s = extend(q, k, v, g, s0, dtype, whole)
    _, ref, _, _ = reference(*(widen(x) for x in (q, k, v)), g, s0, dk ** -0.5)
    assert norm(s - ref) <= STATE_REL * norm(ref)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(64, 128), (128, 128), (128, 256), (256, 128)])
def test_many_sequences_are_as_accurate(dk, dv, dtype):
    """Enough of them for workgroups of 128 columns: one rounding per bf16
    output, states as f32 sums leave them."""
    import torch

    rng = np.random.default_rng(dk + dv)
    B, n, hk, hv = 70, 130, 2, 8
    q, k, v, g = inputs(rng, B * n, hk, hv, dk, dv, dtype, 0.3)
    s0 = (0.3 * rng.standard_normal((1, B, hv, dk, dv))).astype(np.float32)
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, B, dtype)) as pool:
        pool.tensor().copy_(torch.from_numpy(s0))
        o = pool.linear_extend(0, *(to_device(x) for x in (q, k, v, g)), [n] * B, np.arange(B))
        pool.check()
        o, s = widen(to_host(o)).astype(np.float64), pool.tensor().cpu().numpy()[0]
    for b in (0, 33, B - 1):
        r = slice(b * n, (b + 1) * n)
        ref, rs, _, _ = reference(*(widen(x[r]) for x in (q, k, v)), g[r], s0[0, b], dk ** -0.5)
        if dtype == "bf16":
            assert norm(o[r] - ref) <= 1.02 * norm(widen(orc.f32_to_bf16(ref.astype(np.float32))) - ref)
        else:
            assert norm(o[r] - ref) <= STATE_REL * norm(ref)
        assert norm(s[b] - rs) <= STATE_REL * norm(rs)
