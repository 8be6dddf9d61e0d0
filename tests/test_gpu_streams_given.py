"""Results that a call allocates for a stream that it is given: they are that
stream's memory, not what the current stream has just let go of, and dropping
one does not hand it to the current stream while the call may be running."""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import DeviceKvPool, DeviceStatePool, PoolDesc, StateDesc, add_rms_norm

pytestmark = pytest.mark.gpu


def check(call, sizes):
    """call(stream) -> the tensors that it allocated. `sizes`: bytes of them."""
    import torch

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(None)  # both streams have blocks to give
    call(side)
    torch.cuda.synchronize()
    for _ in range(3):
        freed = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
        was = {t.data_ptr() for t in freed}
        del freed
        got = call(side)
        at = {t.data_ptr() for t in got}
        assert len(at) == len(sizes) and not at & was
        del got
        again = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
        assert not at & {t.data_ptr() for t in again}
        del again
    torch.cuda.synchronize()


def test_add_rms_norm():
    import torch

    rows, dim = 64, 2048
    x, res = (torch.randn(rows, dim, device="cuda").bfloat16() for _ in range(2))
    w = torch.zeros(dim, device="cuda")
    n = rows * dim
    check(lambda s: add_rms_norm(x, w, 1e-6, residual=res, fp8=True, group=64, both=True, stream=s),
          [2 * n, 2 * n, n, n // 16])


@pytest.mark.parametrize("kind", ["step", "extend", "extend_device"])
def test_linear(kind):
    import torch

    with DeviceStatePool(StateDesc(1, 1, 2, 64, 64, 700, "bf16")) as pool:
        n = 640
        q, k = (torch.randn(n, 1, 64, device="cuda").bfloat16() for _ in range(2))
        v, g = torch.randn(n, 2, 64, device="cuda").bfloat16(), -torch.rand(n, 2, device="cuda")
        ip, slots = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [3]))
        pool.tensor().zero_()
        torch.cuda.synchronize()
        call = {"step": lambda s: [pool.linear_step(0, q, k, v, g, np.arange(n), stream=s)],
                "extend": lambda s: [pool.linear_extend(0, q, k, v, g, [n], [3], stream=s)],
                "extend_device": lambda s: [pool.linear_extend_device(0, q, k, v, g, ip, slots, n, stream=s)]}[kind]
        check(call, [2 * n * 2 * 64])
        pool.check()


def test_results_are_right_on_a_given_stream():
    import torch

    x = torch.randn(4096, 2048, device="cuda").bfloat16()
    w = torch.zeros(2048, device="cuda")
    want = add_rms_norm(x, w, 1e-6)[1]
    side = torch.cuda.Stream()
    for _ in range(20):
        junk = torch.empty_like(x).fill_(3.0)
        del junk
        side.wait_stream(torch.cuda.current_stream())
        got = add_rms_norm(x, w, 1e-6, stream=side)[1]
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["decode", "planned", "static", "extend", "extend_host", "prep", "gather",
                                  "gather_host", "wire"])
def test_kv_pool(kind):
    import torch

    B, ctx, hq, hkv, d = 64, 256, 8, 2, 128  # results of 512 KiB
    desc = PoolDesc(num_layers=1, num_kv_heads=hkv, num_q_heads=hq, head_dim=d, num_blocks=B * ctx // 16, dtype="bf16")
    with DeviceKvPool(desc) as pool:
        pool.tensor().zero_()
        q = torch.randn(B * 4, hq, d, device="cuda").bfloat16()
        kv = torch.randn(B * 4, hkv, d, device="cuda").bfloat16()
        host_ip, host_ids = np.arange(B + 1) * (ctx // 16), np.arange(B * ctx // 16)
        ip, ids, cl, qip = (torch.tensor(x, dtype=torch.int32, device="cuda")
                            for x in (host_ip, host_ids, [ctx] * B, 4 * np.arange(B + 1)))
        cip = torch.tensor(ctx * np.arange(B + 1), dtype=torch.int32, device="cuda")
        plan = pool.plan(np.full(B, ctx, np.int32))
        slots = np.arange(B * 4)
        torch.cuda.synchronize()
        out, one = 2 * B * 4 * hq * d, 2 * B * hq * d
        kvb = 2 * B * ctx * hkv * d
        call, sizes = {
            "decode": (lambda s: [pool.decode_attention(0, q[:B], ip, ids, cl, ctx, stream=s)], [one]),
            "planned": (lambda s: [pool.decode_attention_planned(0, plan, q[:B], ip, ids, stream=s)], [one]),
            "static": (lambda s: [pool.decode_attention_static(0, q[:B], ip, ids, cl, ctx, stream=s)], [one]),
            "extend": (lambda s: [pool.extend_attention(0, q, qip, ip, ids, cl, 4, ctx, stream=s)], [out]),
            "extend_host": (lambda s: [pool.extend_attention_host(0, q, [4] * B, [ctx] * B, host_ip, host_ids,
                                                                  stream=s)], [out]),
            "prep": (lambda s: [pool.qk_norm_rope_append(0, q, kv, kv, slots, slots, gated=False, stream=s)], [out]),
            "gather": (lambda s: pool.gather(0, ip, ids, cip, ctx, total_tokens=B * ctx, stream=s), [kvb, kvb]),
            "gather_host": (lambda s: pool.gather_host(0, host_ip, host_ids, [ctx] * B, stream=s), [kvb, kvb]),
            "wire": (lambda s: pool.wire_export(host_ids, stream=s), [2 * kvb, 8 * host_ids.size]),
        }[kind]
        check(call, sizes)
        pool.check()
