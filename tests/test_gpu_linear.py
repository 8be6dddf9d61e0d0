"""Linear-attention extend and step over the state pool, against the
recurrence in 64 bits:
    S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t.

Tolerances, per element, from the same sums over absolute values (A_o for an
output, A_S for a state): every path forms them with at most 4 (n + k_dim +
64) f32 operations of relative error 2^-24 each (n tokens of the recurrence,
k_dim products of an output, the rest exponentials and joins). With bf16
rows an output also has its own rounding (2^-8 of itself) and the chunked
form's roundings of a state or of a score to bf16 (2^-8 of the term, so 2^-8
A_o in all); states stay within the f32 bound.
"""
from __future__ import annotations

import numpy as np
import pytest

from mitten_amd import STATE_NONE, DeviceStatePool, StateDesc
from mitten_amd import device_pool as dp
from oracle import oracle as orc
from tests.helpers import to_device, to_host, widen

pytestmark = pytest.mark.gpu


def reference(q, k, v, g, s0, scale):
    """One sequence in f64: q, k [n, Hk, Dk], v [n, Hv, Dv], g [n, Hv], s0
    [Hv, Dk, Dv] -> (o, S, A_o, A_S)."""
    rep = v.shape[1] // k.shape[1]
    q, k = (np.repeat(x.astype(np.float64), rep, 1) for x in (q, k))
    v = v.astype(np.float64)
    S, A = s0.astype(np.float64).copy(), np.abs(s0.astype(np.float64))
    o, Ao = np.zeros(v.shape), np.zeros(v.shape)
    for t in range(v.shape[0]):
        d = np.exp(g[t].astype(np.float64))[:, None, None]
        kv = k[t][:, :, None] * v[t][:, None, :]
        S = d * S + kv
        A = d * A + np.abs(kv)
        o[t] = scale * np.einsum("hd,hdv->hv", q[t], S)
        Ao[t] = abs(scale) * np.einsum("hd,hdv->hv", np.abs(q[t]), A)
    return o, S, Ao, A


def check_close(got, ref, bound, what):
    err = np.abs(got.astype(np.float64) - ref)
    assert np.all(np.isfinite(got)), what
    over = err - bound
    assert np.all(over <= 0), f"{what}: error {err.flat[over.argmax()]:.3e} over {bound.flat[over.argmax()]:.3e}"


def inputs(rng, n, hk, hv, dk, dv, dtype, rate=1.0):
    q = rng.standard_normal((n, hk, dk)).astype(np.float32)
    k = (rng.standard_normal((n, hk, dk)) * dk ** -0.5).astype(np.float32)
    v = rng.standard_normal((n, hv, dv)).astype(np.float32)
    if dtype == "bf16":
        q, k, v = (orc.f32_to_bf16(x) for x in (q, k, v))
    g = -(rate * np.exp(rng.uniform(np.log(1e-3), 0, hv))[None] * rng.uniform(0.2, 1.8, (n, hv))).astype(np.float32)
    return q, k, v, g


def f32_bound(n, dk, A):
    return 4 * (n + dk + 64) * 2.0 ** -24 * A + 1e-37


def out_bound(n, dk, dtype, o, Ao):
    b = f32_bound(n, dk, Ao)
    return b if dtype == "f32" else b + 2.0 ** -8 * (np.abs(o) + Ao)


def run_batch(lens, hk, hv, dk, dv, dtype, src, dst, nslots, seed, step=False, device_meta=False, layer=0, layers=1,
              rate=1.0, head_decay=False, scale=None, max_q_len=None, edit=None):
    """Runs one call and checks every output, every written state and every
    state that it must leave alone."""
    import torch

    rng = np.random.default_rng(seed)
    n = int(sum(lens))
    q, k, v, g = inputs(rng, n, hk, hv, dk, dv, dtype, rate)
    if head_decay:
        g = np.repeat(g[:1] if n else -np.ones((1, hv), np.float32), n, 0)
    if edit:
        edit(q, k, v, g)
    desc = StateDesc(layers, hk, hv, dk, dv, nslots, dtype)
    host = rng.standard_normal(desc.shape).astype(np.float32)
    scale = dk ** -0.5 if scale is None else scale
    dq, dk_, dv_, dg = (to_device(x) for x in (q, k, v, g[0] if head_decay and n else g))
    with DeviceStatePool(desc) as pool:
        pool.tensor().copy_(torch.from_numpy(host))
        if step:
            s, d = (np.array(x, np.uint32) for x in (src, dst))
            if device_meta:
                s, d = (torch.from_numpy(x.view(np.int32)).cuda() for x in (s, d))
            o = pool.linear_step(layer, dq, dk_, dv_, dg, d, src_slots=s, scale=scale)
        elif device_meta:
            ip = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
            s, d = (torch.from_numpy(np.array(x, np.uint32).view(np.int32)).cuda() for x in (src, dst))
            o = pool.linear_extend_device(layer, dq, dk_, dv_, dg, ip, d,
                                          max(lens, default=0) if max_q_len is None else max_q_len, src_slots=s,
                                          scale=scale)
        else:
            o = pool.linear_extend(layer, dq, dk_, dv_, dg, np.array(lens, np.int32), np.array(dst, np.uint32),
                                   src_slots=np.array(src, np.uint32), scale=scale)
        pool.check()
        got_o, got_s = widen(to_host(o)), pool.tensor().cpu().numpy()
    r0 = 0
    for b, m in enumerate(lens):
        s0 = np.zeros((hv, dk, dv)) if src[b] == STATE_NONE else host[layer, src[b]]
        ro, rs, ao, as_ = reference(*(widen(x[r0:r0 + m]) for x in (q, k, v)), g[r0:r0 + m], s0, scale)
        check_close(got_o[r0:r0 + m], ro, out_bound(m, dk, dtype, ro, ao), f"sequence {b} outputs")
        check_close(got_s[layer, dst[b]], rs, f32_bound(m, dk, as_), f"sequence {b} state")
        r0 += m
    left = np.ones((layers, nslots), bool)
    left[layer, dst] = False
    assert np.array_equal(got_s[left], host[left]), "a state that the call does not write has changed"


GEOMETRIES = [(1, 1, 64, 64), (2, 4, 128, 128), (1, 7, 128, 64), (2, 2, 256, 128), (1, 2, 64, 256), (1, 3, 256, 256)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("geom", GEOMETRIES)
@pytest.mark.parametrize("device_meta", [False, True])
def test_step_matches_the_recurrence(geom, dtype, device_meta):
    run_batch([1] * 5, *geom, dtype, [4, STATE_NONE, 2, 9, 2], [4, 1, 0, 3, 7], 10, 11, step=True,
              device_meta=device_meta, layer=1, layers=2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("geom", GEOMETRIES)
@pytest.mark.parametrize("lens", [[1], [63], [64], [65], [0, 5, 0, 130, 1, 16, 17, 0]])
def test_extend_matches_the_recurrence(geom, dtype, lens):
    B = len(lens)
    src = [STATE_NONE if b % 3 == 1 else b for b in range(B)]
    run_batch(lens, *geom, dtype, src, list(range(B)), B + 1, 21, layer=1, layers=2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,fork", [([700], False), ([1500], True), ([5, 1111, 64, 640], False)])
def test_extend_of_long_chunks(lens, fork, dtype):
    B = len(lens)
    run_batch(lens, 1, 2, 128, 128, dtype, [B] * B if fork else list(range(B)), list(range(B)), B + 1, 31)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 256), (256, 64), (256, 128)])
def test_extend_in_segments(dk, dv, dtype):
    """Prompts long enough for segments, beside short and empty ones, at every
    head dim; the source of a sequence among them is its own or another slot."""
    lens = [900, 0, 70, 1025]
    with DeviceStatePool(StateDesc(1, 1, 2, dk, dv, 1, dtype)) as pool:
        assert pool.linear_extend_workspace_size(len(lens), sum(lens), max(lens)) > 0
    run_batch(lens, 1, 2, dk, dv, dtype, [0, 4, STATE_NONE, 4], [0, 1, 2, 3], 6, 35)


@pytest.mark.parametrize("dk,dv", [(64, 128), (128, 128), (128, 256), (256, 128)])
def test_extend_of_many_sequences(dk, dv):
    """More sequences and heads than workgroups of 64 columns would fit at once."""
    rng = np.random.default_rng(37)
    lens = [int(x) for x in rng.integers(0, 90, 40)]
    dst = [int(x) for x in rng.permutation(42)[:40]]
    run_batch(lens, 2, 8, dk, dv, "bf16", [d if d % 3 else STATE_NONE for d in dst], dst, 42, 38)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("max_q_len", [0, 1, 70, 5000])
def test_device_metadata_with_any_bound(dtype, max_q_len):
    """max_q_len sizes the launch only."""
    run_batch([33, 0, 900], 1, 2, 128, 128, dtype, [0, STATE_NONE, 2], [0, 1, 2], 4, 41, device_meta=True,
              max_q_len=max_q_len)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rate", [0.0, 30.0, 3000.0])
def test_decays_from_none_to_all(dtype, rate):
    """No decay at all; decays that leave nothing after a few tokens; decays
    whose sum over a chunk leaves f32's exponent range by far."""
    run_batch([300, 40], 1, 4, 128, 128, dtype, [0, 1], [0, 1], 2, 51, rate=rate)


@pytest.mark.parametrize("step", [False, True])
def test_one_decay_per_head(step):
    run_batch([1, 1, 1] if step else [70, 200], 1, 4, 64, 128, "bf16", [0, 1, 2] if step else [0, 1],
              [0, 1, 2] if step else [0, 1], 3, 61, step=step, head_decay=True)


def test_a_decay_of_minus_infinity_forgets():
    def edit(q, k, v, g):
        g[40:42, 0] = -np.inf
        g[100, :] = -np.inf
        g[0, 1] = -np.inf

    for dtype in ("bf16", "f32"):
        run_batch([150, 7], 1, 2, 128, 128, dtype, [0, 1], [0, 1], 2, 71, edit=edit)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 60, 700])
def test_a_large_state_is_forgotten_wholly(dtype, n):
    """A finite state of 1e36 behind a decay of minus infinity leaves nothing,
    in one step, one chunk and in segments."""
    import torch

    rng = np.random.default_rng(72)
    q, k, v, g = inputs(rng, n, 1, 2, 64, 64, dtype)
    g[0] = -np.inf
    v[:] = 0
    with DeviceStatePool(StateDesc(1, 1, 2, 64, 64, 1, dtype)) as pool:
        pool.tensor().fill_(1e36)
        if n == 1:
            o = pool.linear_step(0, *(to_device(x) for x in (q, k, v, g)), [0])
        else:
            o = pool.linear_extend(0, *(to_device(x) for x in (q, k, v, g)), np.array([n], np.int32), [0])
        assert not torch.any(o.cpu() != 0) and not torch.any(pool.tensor().cpu() != 0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("where", ["v", "k", "state", "g"])
@pytest.mark.parametrize("n", [150, 700])
def test_an_inf_or_nan_reaches_only_what_follows_it(dtype, bad, where, n):
    """Token 70 of n (whole, or in segments) holds it: the tokens before, and
    the other sequences and heads, do not see it; the classes of what follows
    are the recurrence's."""
    import torch

    hk, hv, dk, dv, at = 1, 2, 128, 64, 70
    if where == "g" and bad == np.inf:
        pytest.skip("an infinite growth has no defined state")
    rng = np.random.default_rng(81)
    lens = [n, 20]
    q, k, v, g = inputs(rng, n + 20, hk, hv, dk, dv, "f32")
    if dtype == "bf16":
        q, k, v = (widen(orc.f32_to_bf16(x)) for x in (q, k, v))
    host = rng.standard_normal((1, 2, hv, dk, dv)).astype(np.float32)
    {"v": v[at, 0], "k": k[at, 0], "state": host[0, 0, 0, 5], "g": g[at, :1]}[where][0 if where == "g" else 3] = bad
    dev = [to_device(orc.f32_to_bf16(x) if dtype == "bf16" else x) for x in (q, k, v)]
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 2, dtype)) as pool:
        pool.tensor().copy_(torch.from_numpy(host))
        o = pool.linear_extend(0, *dev, to_device(g), np.array(lens, np.int32), [0, 1])
        got, st = widen(to_host(o)).astype(np.float64), pool.tensor().cpu().numpy()
    r0 = 0
    for b, m in enumerate(lens):
        with np.errstate(all="ignore"):
            ro, rs, ao, as_ = reference(q[r0:r0 + m], k[r0:r0 + m], v[r0:r0 + m], g[r0:r0 + m], host[0, b], dk ** -0.5)
        for x, ref, bound in ((got[r0:r0 + m], ro, out_bound(m, dk, dtype, ro, ao)), (st[0, b], rs, f32_bound(m, dk, as_))):
            fine = np.isfinite(ref)
            assert np.array_equal(fine, np.isfinite(x))
            assert np.array_equal(np.isnan(ref), np.isnan(x))
            assert np.array_equal(ref[np.isinf(ref)], x[np.isinf(ref)].astype(np.float64))
            check_close(x[fine], ref[fine], bound[fine], where)
        r0 += m


def test_rows_outside_the_sequences_and_bad_metadata_are_left_alone():
    """Device metadata that names a slot outside the pool, or rows outside the
    arrays, is reported and its sequence skipped; the others are computed."""
    import torch

    hk, hv, dk, dv, n = 1, 2, 64, 64, 90
    rng = np.random.default_rng(91)
    q, k, v, g = inputs(rng, n, hk, hv, dk, dv, "bf16")
    host = rng.standard_normal((1, 6, hv, dk, dv)).astype(np.float32)
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 6, "bf16")) as pool:
        dev = [to_device(x) for x in (q, k, v, g)]
        for ip, src, dst, good, bits in (
            ([0, 20, 40, 80], [0, 6, 2], [0, 1, 2], (0, 2), dp.DEVERR_SLOT),
            ([0, 20, 40, 80], [0, -2, 2], [0, 1, 2], (0, 2), dp.DEVERR_SLOT),
            ([0, 20, 40, 80], [0, 1, 2], [0, 6, 2], (0, 2), dp.DEVERR_SLOT),
            ([0, 20, 40, 80], [0, 1, 2], [0, -1, 2], (0, 2), dp.DEVERR_SLOT),
            ([0, 20, 10, 91], [0, 1, 2], [0, 1, 2], (0,), dp.DEVERR_CTX),
            ([-5, 20, 40, 2 ** 31 - 1], [0, 1, 2], [0, 1, 2], (1,), dp.DEVERR_CTX),
        ):
            pool.tensor().copy_(torch.from_numpy(host))
            out = torch.full((n, hv, dv), 7.0, dtype=torch.bfloat16, device="cuda")
            i32 = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ip, dst, src)]
            pool.linear_extend_device(0, *dev, i32[0], i32[1], 40, src_slots=i32[2], out=out)
            with pytest.raises(dp.DeviceIndexError) as ei:
                pool.check()
            assert ei.value.bits == bits
            pool.check()
            got, st = widen(to_host(out)), pool.tensor().cpu().numpy()
            rows = np.zeros(n, bool)
            slots = np.zeros(6, bool)
            for b in good:
                r = slice(ip[b], ip[b + 1])
                ro, rs, ao, as_ = reference(*(widen(x[r]) for x in (q, k, v)), g[r], host[0, src[b]], dk ** -0.5)
                check_close(got[r], ro, out_bound(len(ro), dk, "bf16", ro, ao), "outputs")
                check_close(st[0, dst[b]], rs, f32_bound(len(ro), dk, as_), "state")
                rows[r] = True
                slots[dst[b]] = True
            assert np.all(got[~rows] == 7.0) and np.array_equal(st[0][~slots], host[0][~slots])


def test_a_view_of_the_states_keeps_the_pool():
    import gc
    import weakref

    pool = DeviceStatePool(StateDesc(1, 1, 1, 64, 64, 2, "f32"))
    view = pool.tensor()[0]
    alive = weakref.ref(pool)
    del pool
    gc.collect()
    assert alive() is not None
    view.fill_(3.0)
    assert view.sum().item() == 3.0 * view.numel()
    del view
    gc.collect()
    assert alive() is None


def test_copies_and_forks():
    import torch

    desc = StateDesc(3, 1, 3, 64, 128, 9, "bf16")
    host = np.random.default_rng(5).standard_normal(desc.shape).astype(np.float32)
    with DeviceStatePool(desc) as pool:
        for src, dst, device in (([0, 0, 4], [8, 2, 3], False), ([0, 0, 4], [8, 2, 3], True), ([], [], False)):
            pool.tensor().copy_(torch.from_numpy(host))
            s, d = np.array(src, np.uint32), np.array(dst, np.uint32)
            if device:
                s, d = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (s, d))
            pool.copy_states(s, d)
            pool.check()
            want = host.copy()
            want[:, dst] = host[:, src]
            assert np.array_equal(pool.tensor().cpu().numpy(), want)
        many = DeviceStatePool(StateDesc(2, 1, 1, 64, 64, 150, "f32"))  # more pairs than travel as arguments
        for n in (64, 65, 70):
            was = torch.randn(many.desc.shape, device="cuda")
            many.tensor().copy_(was)
            many.copy_states(np.arange(n), np.arange(149, 149 - n, -1))
            many.check()
            was[:, 150 - n:] = was[:, :n].flip(1)
            assert torch.equal(many.tensor(), was)
        pool.copy_states(*(torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 9, -1, 1], [5, 4, 3, -1])))
        with pytest.raises(dp.DeviceIndexError) as ei:
            pool.check()
        assert ei.value.bits == dp.DEVERR_COPY
        got = pool.tensor().cpu().numpy()
        want = np.concatenate([host[:, :5], host[:, :1], host[:, 6:]], 1)
        assert np.array_equal(got, want)


def test_refusals():
    import torch

    desc = StateDesc(2, 1, 2, 64, 64, 8, "bf16")
    with DeviceStatePool(desc) as pool:
        def row(n, h=2, d=64, dt=torch.bfloat16, dev="cuda"):
            return torch.zeros(n, h, d, dtype=dt, device=dev)

        g = torch.zeros(3, 2, device="cuda")
        good = (row(3, 1), row(3, 1), row(3), g)
        pool.linear_step(1, *good, [0, 1, 2])
        bad = [
            (lambda: pool.linear_step(2, *good, [0, 1, 2]), "layer 2"),
            (lambda: pool.linear_step(-1, *good, [0, 1, 2]), "layer -1"),
            (lambda: pool.linear_step(0, *good, [0, 1]), "3 rows for 2 slots"),
            (lambda: pool.linear_step(0, *good, [0, 1, 8]), "outside"),
            (lambda: pool.linear_step(0, *good, [0, 1, 1]), "written twice"),
            (lambda: pool.linear_step(0, *good, [0, 1, STATE_NONE]), "outside"),
            (lambda: pool.linear_step(0, *good, [0, 1, 2], src_slots=[0, 1, 9]), "outside"),
            (lambda: pool.linear_step(0, *good, [0, 1, 2], src_slots=[1, 3, 3]), "is written by sequence 1"),
            (lambda: pool.linear_step(0, *good, [0, 1, 2], src_slots=[1, 3]), "differ in length"),
            (lambda: pool.linear_step(0, *good, [0, 1, 2], scale=float("nan")), "scale"),
            (lambda: pool.linear_step(0, row(3, 2), *good[1:], [0, 1, 2]), "q has shape"),
            (lambda: pool.linear_step(0, *good[:2], row(3, dt=torch.float32), g, [0, 1, 2]), "dtype"),
            (lambda: pool.linear_step(0, *good[:2], row(3, dev="cpu"), g, [0, 1, 2]), "cuda:0"),
            (lambda: pool.linear_step(0, *good[:2], row(6)[::2], g, [0, 1, 2]), "contiguous"),
            (lambda: pool.linear_step(0, *good[:3], g.double(), [0, 1, 2]), "dtype"),
            (lambda: pool.linear_extend(0, *good, [1, 1], [0, 1]), "add up to 2"),
            (lambda: pool.linear_extend(0, *good, [4, -1], [0, 1]), "negative"),
            (lambda: pool.linear_extend(0, *good, [3, 0], [0, 0]), "written twice"),
            (lambda: pool.linear_step(0, *good, torch.arange(3, dtype=torch.int32, device="cuda"), src_slots=[0, 1, 2]),
             "both be host"),
            (lambda: pool.linear_extend(0, *good, [1, 2], torch.arange(2, dtype=torch.int32, device="cuda")), "host array"),
            (lambda: pool.linear_extend_device(0, *good, g, [0, 1], 3), "device tensor"),
            (lambda: pool.linear_step(0, *good, torch.arange(3, device="cuda")), "dtype"),
            (lambda: pool.copy_states(torch.arange(2, dtype=torch.int32, device="cuda"), [4, 5]), "both be host"),
            (lambda: pool.copy_states([0, 1], [2]), "differ in length"),
            (lambda: pool.copy_states([0, 1], [2, 2]), "written twice"),
            (lambda: pool.copy_states([0, 1], [1, 2]), "both a source and a destination"),
            (lambda: pool.copy_states([0, 8], [1, 2]), "outside"),
        ]
        for call, msg in bad:
            with pytest.raises(dp.BackendError) as ei:
                call()
            assert msg in str(ei.value), (msg, str(ei.value))
        odd = torch.zeros(3 * 2 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 2, 64)
        with pytest.raises(dp.BackendError) as ei:
            pool.linear_step(0, *good[:2], odd, g, [0, 1, 2])
        assert "aligned" in str(ei.value)
        pool.check()
        assert pool.linear_step(0, *(x[:0] for x in good), []).shape == (0, 2, 64)


def test_captured_steps_replay_and_host_slots_are_refused_in_capture():
    """A captured chain of an extend and two steps on another stream, replayed
    with other work between, equals the eager one every time."""
    import torch

    hk, hv, dk, dv = 1, 2, 128, 128
    rng = np.random.default_rng(7)
    lens = [70, 300, 0]
    n = sum(lens)
    ext = [to_device(x) for x in inputs(rng, n, hk, hv, dk, dv, "bf16")]
    one = [to_device(x) for x in inputs(rng, 3, hk, hv, dk, dv, "bf16")]
    host = torch.from_numpy(rng.standard_normal((1, 4, hv, dk, dv)).astype(np.float32)).cuda()
    ip = torch.tensor([0, 70, 370, 370], dtype=torch.int32, device="cuda")
    slots = torch.tensor([2, 0, 3], dtype=torch.int32, device="cuda")
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 4, "bf16")) as pool:
        oe = torch.empty(n, hv, dv, dtype=torch.bfloat16, device="cuda")
        o1, o2 = (torch.empty(3, hv, dv, dtype=torch.bfloat16, device="cuda") for _ in range(2))

        def chain():
            pool.linear_extend_device(0, *ext, ip, slots, 300, out=oe)
            pool.linear_step(0, *one, slots, out=o1)
            pool.linear_step(0, *one, slots, out=o2)

        pool.tensor().copy_(host)
        chain()
        torch.cuda.synchronize()
        want = [x.clone() for x in (oe, o1, o2, pool.tensor())]
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(dp.BackendError) as ei:
                pool.linear_step(0, *one, [0, 1, 2], out=o1)
            assert "captured" in str(ei.value)
            chain()
        for _ in range(4):
            pool.tensor().copy_(host)
            for o in (oe, o1, o2):
                o.zero_()
            (host @ host.transpose(-1, -2).contiguous()).sum()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for got, ref in zip((oe, o1, o2, pool.tensor()), want):
                assert torch.equal(got, ref)
        pool.check()


def test_a_prompt_then_steps_as_an_engine_runs_them():
    """Two prompts in two chunks each, a fork of the first after its first
    chunk, then steps of all three: equal to the recurrence over the whole
    sequences, with slots staged again when they change and reused when not."""
    import torch

    hk, hv, dk, dv, L = 2, 4, 128, 128, 2
    rng = np.random.default_rng(17)
    n = [90, 161, 100]  # tokens of sequences 0, 1 and 2 (2 shares sequence 0's first 50)
    q, k, v, g = (list(x) for x in zip(*(inputs(rng, m, hk, hv, dk, dv, "bf16") for m in n)))
    for x in (q, k, v, g):
        x[2][:50] = x[0][:50]
    at = [0, 0, 0]
    outs = [np.zeros((L, m, hv, dv), np.float32) for m in n]
    with DeviceStatePool(StateDesc(L, hk, hv, dk, dv, 5, "bf16")) as pool:
        def go(seqs, lens, src, dst, step=False):
            cat = [to_device(np.concatenate([x[b][at[b]:at[b] + m] for b, m in zip(seqs, lens)])) for x in (q, k, v, g)]
            for layer in range(L):
                if step:
                    o = pool.linear_step(layer, *cat, dst, src_slots=src)
                else:
                    o = pool.linear_extend(layer, *cat, lens, dst, src_slots=src)
                r = 0
                for b, m in zip(seqs, lens):
                    outs[b][layer, at[b]:at[b] + m] = widen(to_host(o))[r:r + m]
                    r += m
            for b, m in zip(seqs, lens):
                at[b] += m

        go([0, 1], [50, 100], [STATE_NONE, STATE_NONE], [3, 1])
        pool.copy_states([3], [4])  # the prefix's snapshot
        outs[2][:, :50] = outs[0][:, :50]
        at[2] = 50
        go([0, 1, 2], [39, 58, 47], [3, 1, 4], [3, 1, 0])
        for _ in range(1):
            go([0, 1, 2], [1, 1, 1], [3, 1, 0], [3, 1, 0], step=True)
        for _ in range(2):
            go([1, 2], [1, 1], [1, 0], [1, 0], step=True)
        pool.check()
        st = pool.tensor().cpu().numpy()
    assert at == n
    for b, slot in ((0, 3), (1, 1), (2, 0)):
        ro, rs, ao, as_ = reference(*(widen(x[b]) for x in (q, k, v)), g[b], np.zeros((hv, dk, dv)), dk ** -0.5)
        for layer in range(L):
            check_close(outs[b][layer], ro, out_bound(n[b], dk, "bf16", ro, ao), f"sequence {b}")
            check_close(st[layer, slot], rs, f32_bound(n[b], dk, as_), f"state {b}")


def test_thousands_of_sequences_of_large_states():
    """4,100 sequences of 64 heads of 256 x 256 (the scan over segments could
    not be launched for them, and need not be). One has a slot; the others'
    are outside the pool, and are reported."""
    import torch

    rng = np.random.default_rng(93)
    q, k, v, g = inputs(rng, 1, 1, 64, 256, 256, "bf16")
    B = 4100
    with DeviceStatePool(StateDesc(1, 1, 64, 256, 256, 1, "bf16")) as pool:
        pool.tensor().zero_()
        ip = torch.ones(B + 1, dtype=torch.int32, device="cuda")
        ip[0] = 0
        slots = torch.ones(B, dtype=torch.int32, device="cuda")
        slots[0] = 0
        assert pool.linear_extend_workspace_size(B, 1, 1) == 0
        o = pool.linear_extend_device(0, *(to_device(x) for x in (q, k, v, g)), ip, slots, 1)
        with pytest.raises(dp.DeviceIndexError) as ei:
            pool.check()
        assert ei.value.bits == dp.DEVERR_SLOT
        ro, rs, ao, as_ = reference(*(widen(x) for x in (q, k, v)), g, np.zeros((64, 256, 256)), 1 / 16)
        check_close(widen(to_host(o)), ro, out_bound(1, 256, "bf16", ro, ao), "outputs")
        check_close(pool.tensor().cpu().numpy()[0, 0], rs, f32_bound(1, 256, as_), "state")


def test_a_loose_bound_on_the_lengths_costs_no_time():
    """max_q_len is only a bound: the largest one is planned as fast as any."""
    import time

    import torch

    rng = np.random.default_rng(94)
    q, k, v, g = (to_device(x) for x in inputs(rng, 5, 1, 64, 256, 256, "bf16"))
    with DeviceStatePool(StateDesc(1, 1, 64, 256, 256, 1, "bf16")) as pool:
        ip, slots = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 5], [0]))
        outs, times = [], []
        for bound in (5, 2 ** 31 - 1):
            pool.tensor().zero_()
            pool.linear_extend_device(0, q, k, v, g, ip, slots, bound)
            pool.tensor().zero_()
            torch.cuda.synchronize()
            t = time.perf_counter()
            outs.append(pool.linear_extend_device(0, q, k, v, g, ip, slots, bound).float())
            times.append(time.perf_counter() - t)
            torch.cuda.synchronize()
        ro, _, ao, _ = reference(*(widen(to_host(x)) for x in (q, k, v)), to_host(g), np.zeros((64, 256, 256)), 1 / 16)
        for o in outs:
            check_close(o.cpu().numpy(), ro, out_bound(5, 256, "bf16", ro, ao), "outputs")
        assert times[1] < 0.02 + times[0]


@pytest.mark.parametrize("i", range(16))
def test_random_batches(i):
    rng = np.random.default_rng(900 + i)
    hk = int(rng.choice([1, 2, 3]))
    hv = hk * int(rng.choice([1, 2, 5]))
    dk, dv = int(rng.choice([64, 128, 256])), int(rng.choice([64, 128, 256]))
    B = int(rng.integers(1, 7))
    lens = [int(x) for x in rng.choice([0, 1, 3, 15, 16, 31, 64, 100, 129, 257], B)]
    n = B + 2
    dst = [int(x) for x in rng.permutation(n)[:B]]
    free = [s for s in range(n) if s not in dst]
    src = [STATE_NONE if r < 0.3 else free[0] if r < 0.5 else d for r, d in zip(rng.random(B), dst)]
    dtype = "f32" if rng.random() < 0.4 else "bf16"
    print(f"case {i}: heads {hk}/{hv} dims {dk}/{dv} {dtype} lens {lens} src {src} dst {dst}", flush=True)
    run_batch(lens, hk, hv, dk, dv, dtype, src, dst, n, 1000 + i, device_meta=bool(rng.integers(2)),
              rate=float(rng.choice([0.1, 1.0, 10.0])), scale=float(rng.uniform(0.1, 2.0)))


def _long_call(pool, rng, hk, hv, dk, dv, n):
    import torch

    rows = [to_device(x) for x in inputs(rng, n, hk, hv, dk, dv, "bf16")]
    ip = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    return rows, ip


def test_workspaces_given_and_too_small_and_of_the_pool():
    """A long prompt in segments from the pool's workspace and from a given one
    is the same to the bit; with too little room it stays whole."""
    import torch

    hk, hv, dk, dv, n = 1, 2, 128, 128, 2000
    rng = np.random.default_rng(23)
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 2, "bf16")) as pool:
        rows, ip = _long_call(pool, rng, hk, hv, dk, dv, n)
        slots = torch.tensor([1], dtype=torch.int32, device="cuda")
        new = torch.tensor([-1], dtype=torch.int32, device="cuda")
        size = pool.linear_extend_workspace_size(1, n, n)
        assert size > 0 and pool.linear_extend_workspace_size(0, 0, 0) == 0
        got = []
        for ws in (None, torch.empty(size, dtype=torch.uint8, device="cuda"),
                   torch.empty(16, dtype=torch.uint8, device="cuda")):
            o = pool.linear_extend_device(0, *rows, ip, slots, n, src_slots=new, workspace=ws)
            pool.check()
            got.append((o.float(), pool.tensor()[0, 1].clone()))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
        assert (got[0][0] - got[2][0]).norm() <= 2.0 ** -7 * got[2][0].norm()
        assert (got[0][1] - got[2][1]).norm() <= 2.0 ** -20 * got[2][1].norm()
        with pytest.raises(dp.BackendError) as ei:
            pool.linear_extend_device(0, *rows, ip, slots, n, workspace=torch.empty(size + 8, dtype=torch.uint8,
                                                                                   device="cuda")[8:])
        assert "aligned" in str(ei.value)


def test_two_streams_share_the_pools_workspace():
    """Long prompts of two pairs of slots on two streams at once: each as alone."""
    import torch

    hk, hv, dk, dv, n = 1, 2, 128, 128, 3000
    rng = np.random.default_rng(29)
    with DeviceStatePool(StateDesc(1, hk, hv, dk, dv, 4, "bf16")) as pool:
        calls = [inputs(rng, n, hk, hv, dk, dv, "bf16") for _ in range(2)]
        calls = [[to_device(x) for x in c] for c in calls]
        want = []
        for b, c in enumerate(calls):
            o = pool.linear_extend(0, *c, [n], [b], src_slots=[STATE_NONE])
            want.append((o.clone(), pool.tensor()[0, b].clone()))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in calls]
        for _ in range(3):
            outs = []
            for b, (c, st) in enumerate(zip(calls, streams)):
                outs.append(pool.linear_extend(0, *c, [n], [b + 2], src_slots=[STATE_NONE], out=torch.empty_like(want[b][0]),
                                               stream=st))
            torch.cuda.synchronize()
            for b in range(2):
                assert torch.equal(outs[b], want[b][0]) and torch.equal(pool.tensor()[0, b + 2], want[b][1])
        pool.check()
