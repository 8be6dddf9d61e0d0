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


def long_prompt(rng, hk, hv, dk, dv, n, dtype):
    import torch

    host = inputs(rng, n, hk, hv, dk, dv, dtype)
    return host, [to_device(x) for x in host], torch.tensor([0, n], dtype=torch.int32, device="cuda")


def verify(pool, host, o, s0, slot, dtype):
    q, k, v, g = host
    n, dk = q.shape[0], q.shape[2]
    ro, rs, ao, as_ = reference(*(widen(x) for x in (q, k, v)), g, s0, dk ** -0.5)
    check_close(widen(to_host(o)), ro, out_bound(n, dk, dtype, ro, ao), "outputs")
    check_close(pool.tensor()[0, slot].cpu().numpy(), rs, f32_bound(n, dk, as_), "state")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bound", [320, 640, 1000, 1999])
def test_a_bound_too_small_still_in_segments(bound, dtype):
    """The last of the planned segments takes all that is left."""
    import torch

    rng = np.random.default_rng(bound)
    hk, hv, dk, dv, n = 1, 2, 128, 128, 2000
    host, dev, ip = long_prompt(rng, hk, hv, dk, dv, n, dtype)
    s0 = rng.standard_normal((1, 2, hv, dk, dv)).astype(np.float32)
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 2, dtype)) as pool:
        # (A planned length of 5 chunks is whole: 5 x 3.6 us against 12 and 7.4 of segments.)
        assert pool.linear_extend_workspace_size(1, n, bound) > 0 or bound == 320
        pool.tensor().copy_(torch.from_numpy(s0))
        slots = torch.tensor([1], dtype=torch.int32, device="cuda")
        o = pool.linear_extend_device(0, *dev, ip, slots, bound)
        pool.check()
        verify(pool, host, o, s0[0, 1], 1, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("given", [False, True])
def test_segments_in_a_captured_call(given, dtype):
    """Three launches over a workspace, the pool's or a given one, replayed
    with other extends of the pool between: each replay as the eager call."""
    import torch

    rng = np.random.default_rng(7)
    hk, hv, dk, dv, n = 1, 2, 128, 128, 2000
    host, dev, ip = long_prompt(rng, hk, hv, dk, dv, n, dtype)
    _, other, _ = long_prompt(rng, hk, hv, dk, dv, n, dtype)
    s0 = rng.standard_normal((1, 3, hv, dk, dv)).astype(np.float32)
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 3, dtype)) as pool:
        start = torch.from_numpy(s0).cuda()
        slots, src = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (1, 0))
        size = pool.linear_extend_workspace_size(1, n, n)
        assert size > 0
        ws = torch.empty(size, dtype=torch.uint8, device="cuda") if given else None
        o = torch.empty_like(dev[2])

        def call():
            pool.linear_extend_device(0, *dev, ip, slots, n, src_slots=src, out=o, workspace=ws)

        pool.tensor().copy_(start)
        call()
        pool.check()
        verify(pool, host, o, s0[0, 0], 1, dtype)
        want = o.clone(), pool.tensor()[0, 1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for _ in range(4):
            pool.tensor().copy_(start)
            o.zero_()
            pool.linear_extend(0, *other, [n], [2])
            torch.cuda.synchronize()
            graph.replay()
            pool.linear_extend(0, *other, [n], [2])
            torch.cuda.synchronize()
            assert torch.equal(o, want[0]) and torch.equal(pool.tensor()[0, 1], want[1])
        pool.check()


def test_graphs_with_workspaces_of_their_own_beside_each_other():
    """Two captured calls, each with a workspace, replayed at once on two streams."""
    import torch

    rng = np.random.default_rng(8)
    hk, hv, dk, dv, n = 1, 2, 128, 128, 3000
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 2, "bf16")) as pool:
        size = pool.linear_extend_workspace_size(1, n, n)
        new = torch.tensor([-1], dtype=torch.int32, device="cuda")
        graphs, outs, want, keep = [], [], [], []
        for b in range(2):
            _, dev, ip = long_prompt(rng, hk, hv, dk, dv, n, "bf16")
            slots = torch.tensor([b], dtype=torch.int32, device="cuda")
            ws = torch.empty(size, dtype=torch.uint8, device="cuda")
            o = torch.empty_like(dev[2])
            pool.linear_extend_device(0, *dev, ip, slots, n, src_slots=new, out=o, workspace=ws)
            torch.cuda.synchronize()
            want.append((o.clone(), pool.tensor()[0, b].clone()))
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                pool.linear_extend_device(0, *dev, ip, slots, n, src_slots=new, out=o, workspace=ws)
            outs.append(o)
            keep.append((dev, ip, slots, ws))
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(4):
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for b in range(2):
                assert torch.equal(outs[b], want[b][0]) and torch.equal(pool.tensor()[0, b], want[b][1])
        pool.check()


def test_an_empty_workspace_is_none_of_the_pools():
    """A workspace of no bytes has no room for segments: the call stays whole, as
    with one of 16, where the pool's own would have cut it."""
    import torch

    from mitten_amd import device_pool as dp

    rng = np.random.default_rng(9)
    hk, hv, dk, dv, n = 1, 2, 128, 128, 2000
    _, dev, ip = long_prompt(rng, hk, hv, dk, dv, n, "f32")
    slots, new = (torch.tensor([x], dtype=torch.int32, device="cuda") for x in (0, -1))
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 1, "f32")) as pool:
        got = []
        for ws in (None, torch.empty(16, device="cuda"), torch.empty(0, device="cuda")):
            o = pool.linear_extend_device(0, *dev, ip, slots, n, src_slots=new, workspace=ws)
            got.append((o, pool.tensor().clone()))
        pool.check()
        assert not torch.equal(got[0][1], got[1][1])  # (summed in another order)
        assert torch.equal(got[1][0], got[2][0]) and torch.equal(got[1][1], got[2][1])
        for bad, msg in ((np.zeros(1 << 20), "tensor"), (torch.empty(64), "cuda:0")):
            with pytest.raises(dp.BackendError) as ei:
                pool.linear_extend_device(0, *dev, ip, slots, n, workspace=bad)
            assert msg in str(ei.value)


def test_segments_that_overfill_an_xcd_are_counted():
    """28 value heads over 4: whole key heads go to one XCD, 5 segments each of 2
    prompts would leave 35 workgroups on its 32 CUs, two rounds of three
    launches (57 us; whole 47). 16 key heads of 2 fill every XCD evenly."""
    with DeviceStatePool(StateDesc(1, 4, 28, 128, 128, 1, "bf16")) as pool:
        assert pool.linear_extend_workspace_size(2, 1600, 800) == 0
        assert pool.linear_extend_workspace_size(1, 4000, 4000) > 0
    with DeviceStatePool(StateDesc(1, 16, 32, 128, 128, 1, "bf16")) as pool:
        assert pool.linear_extend_workspace_size(1, 1000, 1000) > 0
