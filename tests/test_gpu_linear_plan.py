"""How linear_extend is planned: bounds on the lengths, segments in captured
calls, workspaces."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import DeviceStatePool, StateDesc
from tests.helpers import to_device, to_host, widen
from tests.test_gpu_linear import check_close, f32_bound, inputs, out_bound, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hk,hv,dk,dv", [(16, 32, 128, 128), (1, 64, 256, 256), (1, 2, 64, 64)])
def test_no_sequence_is_longer_than_all_tokens(hk, hv, dk, dv, dtype):
    """A bound on the lengths past the number of tokens plans as that number:
    small batches stay whole, and ask for no workspace."""
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 1, dtype)) as pool:
        for seqs, tokens in ((1, 0), (1, 1), (1, 64), (8, 32), (1, 700), (3, 5000)):
            want = pool.linear_extend_workspace_size(seqs, tokens, tokens)
            for loose in (tokens + 1, 8192, 2 ** 31 - 1):
                assert pool.linear_extend_workspace_size(seqs, tokens, max(loose, tokens)) == want
        assert pool.linear_extend_workspace_size(8, 32, 8192) == pool.linear_extend_workspace_size(1, 64, 8192) == 0
