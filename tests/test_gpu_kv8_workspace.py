"""What the 8-bit pool says of workspaces: its size holds no decode call back, and extend calls
take what the given one has room for."""
from __future__ import annotations

import pytest

from mitten_amd import DeviceKv8Pool, PoolDesc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hkv,hq", [(1, 1), (4, 28), (2, 32), (8, 128), (1, 17), (64, 1024), (1, 4096)])
def test_size_holds_every_decode_piece(d, hkv, hq):
    """Two partials (a pair and a row of f32) for every piece and query head: 8 waves a CU, a
    wave per piece, KV head and 16 query heads."""
    import torch

    cus = torch.cuda.get_device_properties(0).multi_processor_count
    heads = hkv * -(-hq // hkv // 16)
    pieces = max(1, 8 * cus // heads)
    with DeviceKv8Pool(PoolDesc(1, hkv, hq, d, 4, "bf16")) as pool:
        assert pool.workspace_size() >= max(64 << 20, 256 + pieces * 2 * hq * (8 + 4 * d))
