"""An 8-bit pool that is closed: no view of its memory, and no call."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import BackendError, DeviceKv8Pool, PoolDesc

from kv8_helpers import dev

pytestmark = pytest.mark.gpu


def test_closed_pool():
    pool = DeviceKv8Pool(PoolDesc(1, 1, 2, 64, 4, "bf16"))
    assert pool.tensor().shape == (1, 2, 4, 1, 1024) and pool.exponents().shape == (1, 2, 4, 1)
    pool.close()
    kv, q = dev(np.ones((1, 1, 64)), "bf16"), dev(np.ones((1, 2, 64)), "bf16")
    tables = np.array([0, 1], np.uint32), np.array([2], np.uint32), np.array([3], np.int32)
    for call in (pool.tensor, pool.exponents, pool.workspace_size, pool.check,
                 lambda: pool.append(0, kv, kv, [1], *tables),
                 lambda: pool.qk_norm_rope_append(0, q, kv, kv, [1], *tables, gated=False),
                 lambda: pool.gather(0, *tables), lambda: pool.copy_blocks([0], [1]),
                 lambda: pool.decode_step(0, kv, kv, q, *tables), lambda: pool.decode_attention(0, q, *tables),
                 lambda: pool.extend_attention(0, q, [1], *tables)):
        with pytest.raises(BackendError):
            call()
    pool.close()  # (again: nothing)


def test_a_view_keeps_the_pool():
    """A view of a pool that nobody holds any more reads its memory still."""
    import gc

    def view():
        pool = DeviceKv8Pool(PoolDesc(1, 1, 2, 64, 4, "bf16"))
        pool.tensor().fill_(7)
        return pool.tensor()

    t = view()
    gc.collect()
    assert bool((t == 7).all())
