"""What the bound on a state's error (test_gpu_linear_accuracy.STATE_REL) can
see: the update K^T (w V) of a chunk with w V cut into truncated bf16 parts, in
64 bits otherwise. Three parts are within it, two are not: 2.3e-6 to 1e-5 (CPU)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import oracle as orc
from tests.test_gpu_linear import inputs, reference
from tests.test_gpu_linear_accuracy import STATE_REL


def parts_of(x, parts):
    """x (f32) as the sum of `parts` truncated bf16 values."""
    rest, total = x.astype(np.float32), np.zeros(x.shape)
    for _ in range(parts):
        top = (rest.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        total += top
        rest = rest - top
    return total


@pytest.mark.parametrize("parts,fits", [(1, False), (2, False), (3, True)])
@pytest.mark.parametrize("n", [2, 64, 200])
@pytest.mark.parametrize("dk", [64, 256])
def test_a_states_error_by_parts(parts, fits, n, dk):
    rng = np.random.default_rng(n + dk)
    q, k, v, g = inputs(rng, n, 1, 2, dk, 64, "bf16", 0.3)
    q, k, v = (orc.bf16_to_f32(x) for x in (q, k, v))
    s0 = (0.3 * rng.standard_normal((2, dk, 64))).astype(np.float32)
    _, ref, _, _ = reference(q, k, v, g, s0, 1.0)
    S = s0.astype(np.float64)
    for t0 in range(0, n, 64):
        G = np.cumsum(g[t0:t0 + 64].astype(np.float64), 0)
        w = np.exp(G[-1] - G).astype(np.float32)
        wv = parts_of((w[:, :, None] * v[t0:t0 + 64]).astype(np.float32), parts)
        S = np.exp(G[-1])[:, None, None] * S + np.einsum("td,thv->hdv", k[t0:t0 + 64, 0].astype(np.float64), wv)
    err = np.linalg.norm(S - ref) / np.linalg.norm(ref)
    assert (err <= STATE_REL) == fits
