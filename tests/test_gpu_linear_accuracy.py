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
