"""A batch of padding alone: no block in any table, rows of zeros."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import DeviceIndexError, DeviceKv8Pool, PoolDesc

from kv8_helpers import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most", [0, 100, 100000])
def test_padding_alone(most):
    import torch

    none = dev(np.zeros(0)), dev(np.zeros(4)), dev(np.zeros(3))
    with DeviceKv8Pool(PoolDesc(1, 1, 2, 64, 4, "bf16")) as pool:
        q, k = dev(np.ones((3, 2, 64)), "bf16"), dev(np.ones((3, 1, 64)), "bf16")
        ids, indptr, ctx = none
        out = torch.full((3, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16)
        before = pool.tensor().clone()
        for run in (lambda: pool.decode_attention(0, q, indptr, ids, ctx, max_ctx_len=most, out=out),
                    lambda: pool.decode_step(0, k, k, q, indptr, ids, ctx, max_ctx_len=most, out=out),
                    lambda: pool.bind_decode_step(k, k, q, indptr, ids, ctx, out, max_ctx_len=most)(0)):
            out.fill_(7.0)
            run()
            pool.check()
            assert bool((out == 0.0).all())
        # Nothing of the three tokens' room is written.
        rows = [torch.full((3 * 64,), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        pool.gather(0, indptr, ids, ctx, max_ctx_len=most, total_tokens=3, out_k=rows[0], out_v=rows[1])
        empty = torch.empty((0, 2, 64), device="cuda", dtype=torch.bfloat16)
        pool.extend_attention(0, empty, indptr, indptr, ids, ctx, max_q_len=min(most, 5), max_ctx_len=most)
        pool.append(0, empty[:, :1].contiguous(), empty[:, :1].contiguous(), indptr, indptr, ids, ctx, max_q_len=5)
        pool.check()
        assert all(bool((x == 7.0).all()) for x in rows) and torch.equal(pool.tensor(), before)
        # By host metadata.
        o = pool.decode_step(0, k, k, q, [0, 0, 0, 0], [], [0, 0, 0])
        assert bool((o == 0.0).all())


def test_tokens_without_a_table():
    """An empty array of ids has no room for any token: reported, nothing read or written."""
    import torch

    ids, indptr, ctx = dev(np.zeros(0)), dev(np.array([0, 0, 0])), dev(np.array([5, 0]))
    with DeviceKv8Pool(PoolDesc(1, 1, 2, 64, 4, "bf16")) as pool:
        q, k = dev(np.ones((2, 2, 64)), "bf16"), dev(np.ones((2, 1, 64)), "bf16")
        out = torch.full((2, 2, 64), 7.0, device="cuda", dtype=torch.bfloat16)
        qi = dev(np.array([0, 2, 2]))
        before = pool.tensor().clone()
        for table in (indptr, dev(np.array([0, 1, 1]))):  # (and one that names an id which is not there)
            for run, last in ((lambda m: pool.decode_step(0, k, k, q, table, ids, ctx, max_ctx_len=m, out=out), 0.0),
                              (lambda m: pool.extend_attention(0, q, qi, table, ids, ctx, max_q_len=2, max_ctx_len=m, out=out), 7.0),
                              (lambda m: pool.append(0, k, k, qi, table, ids, ctx, max_q_len=2), 7.0),
                              (lambda m: pool.qk_norm_rope_append(0, q, k, k, qi, table, ids, ctx, max_q_len=2, gated=False, out=out), 7.0),
                              (lambda m: pool.gather(0, table, ids, ctx, max_ctx_len=m, total_tokens=5), 7.0)):
                for m in (5, 30000):
                    out.fill_(7.0)
                    run(m)
                    with pytest.raises(DeviceIndexError) as ei:
                        pool.check()
                    assert ei.value.bits == 4  # (the table)
                    assert bool((out[0] == 7.0).all()) and bool((out[1] == last).all())
        assert torch.equal(pool.tensor(), before)
