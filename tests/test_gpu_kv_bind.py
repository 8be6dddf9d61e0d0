"""Bound decode steps after their plan or pool has changed."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import DeviceKvPool, PoolDesc
from mitten_amd import device_pool as dp

pytestmark = pytest.mark.gpu

B, CTX, HQ, HKV, D, L = 3, 64, 4, 2, 128, 2


def setup(shared):
    import torch

    pool = DeviceKvPool(PoolDesc(L, HKV, HQ, D, 64, "bf16"))
    pool.tensor().zero_()
    ip, ids = np.arange(B + 1) * (CTX // 16), np.arange(B * CTX // 16)
    k, v = (torch.randn(L, B, HKV, D, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(L, B, HQ, D, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    if shared:
        plan = pool.plan_shared_prefix(np.array([60]), [CTX] * B, ip, ids)
        run = pool.bind_decode_step_shared_prefix(plan, k, v, q, None, None, None, out)
    else:
        plan = pool.plan([CTX] * B, block_indptr=ip, block_ids=ids)
        run = pool.bind_decode_step(plan, k, v, q, None, None, out)
    return pool, plan, run, out, ip, ids


@pytest.mark.parametrize("shared", [False, True])
def test_a_plan_built_again_for_other_sequences(shared):
    import torch

    pool, plan, run, out, ip, ids = setup(shared)
    pre = {"prefix_ids": np.array([60])} if shared else {}
    run(0)
    run(1)
    torch.cuda.synchronize()
    want = out.clone()
    plan.build([CTX] * B, block_indptr=ip, block_ids=ids, **pre)
    run(0)
    assert torch.equal(out, want)
    plan.build([CTX] * (B - 1), block_indptr=ip[:B], block_ids=ids[: ip[B - 1]], **pre)
    with pytest.raises(dp.BackendError) as ei:
        run(0)
    assert "bound for 3 sequences, the plan has 2" in str(ei.value)
    pool.check()
    plan.close()
    pool.close()


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("what", ["plan", "pool"])
def test_a_closed_plan_or_pool_is_refused(shared, what):
    import torch

    pool, plan, run, *_ = setup(shared)
    run(0)
    torch.cuda.synchronize()
    plan.close()
    if what == "pool":
        pool.close()
    with pytest.raises(dp.BackendError) as ei:
        run(0)
    assert "NULL" in str(ei.value)
    pool.close()


@pytest.mark.parametrize("shared", [False, True])
def test_a_bound_call_keeps_its_plan_and_pool(shared):
    import gc
    import weakref

    import torch

    pool, plan, run, out, *_ = setup(shared)
    refs = weakref.ref(pool), weakref.ref(plan)
    del pool, plan, _
    gc.collect()
    assert all(r() is not None for r in refs)
    run(0)
    torch.cuda.synchronize()
    assert bool(out[0].any())
