"""Linear-attention states and the step between layers, in Python.

`DeviceStatePool` owns one libmitten_kv state pool (HBM, f32, layout
[num_layers][num_slots][num_v_heads][k_dim][v_dim]) and runs linear attention
with a scalar decay per head over it (S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t =
scale S_t^T q_t; not the delta rule, which also erases):

    linear_extend(layer, q, k, v, log_decay, q_lens, slots)    ragged prompts
    linear_step(layer, q, k, v, log_decay, slots)              one token per sequence
    copy_states(src, dst)                                      fork, compaction

`add_rms_norm` is the residual add and RMSNorm(1 + w) around a layer's blocks
(inference-model-qwen/src/model.rs:84-109,348-365), with an output in the
model's type or in e4m3 with scales.

torch is used only for device memory and streams, as in `device_pool`.

With `stream=`, what a call allocates is that stream's memory. Operands of
another stream's have to be ready there, and to be kept (or noted with
`record_stream`) until it has passed the call, as with any work on a second stream.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from functools import partial

import numpy as np

from . import _lib
from .device_pool import (
    DTYPES,
    MKV_ERR_DEVICE_INDEX,
    MKV_ERR_INVALID_ARGUMENT,
    BackendError,
    DeviceIndexError,
    _dptr,
    _empty_on,
    _host_i32,
    _host_u32,
    _i32p,
    _is_host,
    _raise,
    _torch,
    _tptr,
    _u32p,
)

STATE_NONE = 0xFFFFFFFF  # source slot: the sequence starts from zeros (device slots: -1)
LINEAR_HEAD_DECAY = 1


@dataclass(frozen=True)
class StateDesc:
    """Geometry of a state pool: heads and dims of a model's linear-attention
    layers, and how many sequences' states it holds."""

    num_layers: int
    num_k_heads: int
    num_v_heads: int
    k_dim: int
    v_dim: int
    num_slots: int
    dtype: str = "bf16"  # of q, k, v and the output; states are f32

    def c(self) -> _lib.StateDescC:
        return _lib.StateDescC(self.num_layers, self.num_k_heads, self.num_v_heads, self.k_dim, self.v_dim,
                               DTYPES[self.dtype], self.num_slots)

    @property
    def shape(self):
        return (self.num_layers, self.num_slots, self.num_v_heads, self.k_dim, self.v_dim)


def state_required_bytes(desc: StateDesc) -> int:
    out = ctypes.c_uint64()
    _raise(_lib.device_lib().mkv_state_required_bytes(ctypes.byref(desc.c()), ctypes.byref(out)))
    return out.value


def _bad(msg: str):
    return BackendError(MKV_ERR_INVALID_ARGUMENT, msg)


def _check(t, device: int, shape, dtype, name: str) -> None:
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.device.index != device:
        raise _bad(f"{name} must be a tensor on cuda:{device}")
    if t.dtype != dtype:
        raise _bad(f"{name} has dtype {t.dtype}, expected {dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise _bad(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise _bad(f"{name} must be contiguous")


def _stream(stream, device: int) -> ctypes.c_void_p:
    """The given stream, or the current one of the operands' device."""
    if stream is None:
        stream = _torch().cuda.current_stream(device)
    return ctypes.c_void_p(stream.cuda_stream)


def _raw_stream(stream, device: int) -> int:
    """_stream as a number, without a Stream object for the current one where torch offers that."""
    if stream is not None:
        return stream.cuda_stream
    raw = getattr(_torch()._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else _torch().cuda.current_stream(device).cuda_stream


def _host_copy(x):
    """Host metadata as an array of its own; anything else as it is."""
    return np.array(x.numpy() if hasattr(x, "numpy") else x) if x is not None and _is_host(x) else x


def _torch_type(name: str):
    torch = _torch()
    return torch.float32 if name == "f32" else torch.bfloat16


class DeviceStatePool:
    """The states of a hybrid model's linear-attention layers. Pool, forks and
    copies fit any layer with one matrix per head (the DeltaNet variant of
    KVCacheState, inference-model-common/src/lib.rs:5-13, too); linear_extend and
    linear_step compute the scalar-decay recurrence only."""

    def __init__(self, desc: StateDesc, device: int = 0):
        self.desc = desc
        self.device = device
        self._lib = _lib.device_lib()
        h = ctypes.c_void_p()
        _raise(self._lib.mkv_state_pool_create(ctypes.byref(desc.c()), device, ctypes.byref(h)))
        self._h = h
        ptr, nbytes = ctypes.c_void_p(), ctypes.c_uint64()
        _raise(self._lib.mkv_state_pool_buffer(self._h, ctypes.byref(ptr), ctypes.byref(nbytes)))
        self.data_ptr = ptr.value
        self.nbytes = nbytes.value

    # -- lifecycle -------------------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.mkv_state_pool_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def torch_dtype(self):
        return _torch_type(self.desc.dtype)

    def check(self, stream=None) -> None:
        """Synchronise and raise DeviceIndexError if a kernel met a bad id."""
        bits = ctypes.c_uint32()
        st = self._lib.mkv_state_pool_check(self._h, _stream(stream, self.device), ctypes.byref(bits))
        if st == MKV_ERR_DEVICE_INDEX:
            raise DeviceIndexError(st, self._lib.mkv_last_error().decode(), bits.value)
        _raise(st)

    def tensor(self):
        """Zero-copy torch view of the states, shape `desc.shape` (f32). It
        keeps the pool alive; after close() it must not be read."""

        class _View:
            pass

        view = _View()
        view.pool = self  # the tensor holds the view: states are not freed under it
        view.__cuda_array_interface__ = {"shape": tuple(int(x) for x in self.desc.shape), "typestr": "<f4",
                                         "data": (self.data_ptr, False), "version": 3, "strides": None}
        return _torch().as_tensor(view, device=f"cuda:{self.device}")

    # -- operations -----------------------------------------------------------------------
    def copy_states(self, src, dst, stream=None) -> None:
        """states[:, dst[i]] = states[:, src[i]]. src, dst: device int32
        tensors, or host u32 slots (mkv_state_copy_host, which also checks
        that no copy reads or writes what another writes)."""
        sh = _stream(stream, self.device)
        if _is_host(src) != _is_host(dst):
            raise _bad("src and dst must both be host arrays or both device tensors")
        if _is_host(src):
            s, d = _host_u32(src, "src"), _host_u32(dst, "dst")
            if s.size != d.size:
                raise _bad("src and dst differ in length")
            _raise(self._lib.mkv_state_copy_host(self._h, _u32p(s), _u32p(d), s.size, sh))
            return
        torch = _torch()
        n = src.shape[0]
        _check(src, self.device, (n,), torch.int32, "src")
        _check(dst, self.device, (n,), torch.int32, "dst")
        _raise(self._lib.mkv_state_copy(self._h, _dptr(src), _dptr(dst), n, sh))

    def _rows(self, q, k, v, log_decay, out, scale, lead=(), stream=None):
        """Checks a call's rows ([*lead, tokens, heads, dim]) and returns
        (tokens, out, scale, flags). log_decay: f32 [*lead, tokens, Hv], or
        [*lead, Hv] for one decay per head."""
        torch = _torch()
        d = self.desc
        lead = tuple(lead)
        if not isinstance(q, torch.Tensor) or q.dim() != len(lead) + 3:
            raise _bad(f"q must be a tensor of {len(lead) + 3} dimensions")
        n = q.shape[len(lead)]
        dt = self.torch_dtype
        _check(q, self.device, lead + (n, d.num_k_heads, d.k_dim), dt, "q")
        _check(k, self.device, lead + (n, d.num_k_heads, d.k_dim), dt, "k")
        _check(v, self.device, lead + (n, d.num_v_heads, d.v_dim), dt, "v")
        per_head = isinstance(log_decay, torch.Tensor) and log_decay.dim() == len(lead) + 1
        _check(log_decay, self.device, lead + ((d.num_v_heads,) if per_head else (n, d.num_v_heads)), torch.float32,
               "log_decay")
        if out is None:
            out = _empty_on(stream, v.shape, dt, v.device)
        _check(out, self.device, lead + (n, d.num_v_heads, d.v_dim), dt, "out")
        return n, out, d.k_dim ** -0.5 if scale is None else scale, LINEAR_HEAD_DECAY if per_head else 0

    def _slots(self, slots, src_slots):
        """(num_seqs, destination pointer, source pointer, whether they are host slots, the arrays)."""
        torch = _torch()
        if src_slots is not None and _is_host(slots) != _is_host(src_slots):
            raise _bad("slots and src_slots must both be host arrays or both device tensors")
        if _is_host(slots):
            d = _host_u32(slots, "slots")
            s = None if src_slots is None else _host_u32(src_slots, "src_slots")
            if s is not None and s.size != d.size:
                raise _bad("slots and src_slots differ in length")
            return d.size, _u32p(d), None if s is None else _u32p(s), True, (d, s)
        n = slots.shape[0]
        _check(slots, self.device, (n,), torch.int32, "slots")
        if src_slots is not None:
            _check(src_slots, self.device, (n,), torch.int32, "src_slots")
        return n, _dptr(slots), _tptr(src_slots), False, (slots, src_slots)

    def linear_step(self, layer: int, q, k, v, log_decay, slots, src_slots=None, out=None, scale: float | None = None,
                    stream=None):
        """One token per sequence: row b moves the state of src_slots[b]
        (default: slots[b]; STATE_NONE, or -1 in a device tensor: zeros) on
        and leaves it in slots[b]. Slots: host u32 (validated, copied) or
        device int32. Returns o [B, Hv, v_dim]."""
        n, out, scale, flags = self._rows(q, k, v, log_decay, out, scale, stream=stream)
        B, dst, src, host, _ = self._slots(slots, src_slots)
        if B != n:
            raise _bad(f"{n} rows for {B} slots")
        fn = self._lib.mkv_linear_step_host if host else self._lib.mkv_linear_step
        _raise(fn(self._h, layer, _dptr(q), _dptr(k), _dptr(v), _dptr(log_decay), _dptr(out), src, dst, B, scale,
                  flags, _stream(stream, self.device)))
        return out

    def linear_extend(self, layer: int, q, k, v, log_decay, q_lens, slots, src_slots=None, out=None,
                      scale: float | None = None, stream=None):
        """A chunk of q_lens[b] tokens per sequence, its rows one after
        another; slots as in linear_step. Host q_lens and slots (validated,
        copied). Returns o [tokens, Hv, v_dim]."""
        n, out, scale, flags = self._rows(q, k, v, log_decay, out, scale, stream=stream)
        lens, slots, src_slots = self._extend_meta(n, q_lens, slots, src_slots)
        _raise(self._lib.mkv_linear_extend_host(
            self._h, layer, _dptr(q), _dptr(k), _dptr(v), _dptr(log_decay), _dptr(out), _i32p(lens),
            None if src_slots is None else _u32p(src_slots), _u32p(slots), slots.size, scale, flags,
            _stream(stream, self.device)))
        return out

    def _extend_meta(self, n, q_lens, slots, src_slots):
        for x, name in ((q_lens, "q_lens"), (slots, "slots"), (src_slots, "src_slots")):
            if x is not None and not _is_host(x):
                raise _bad(f"{name} must be a host array (linear_extend_device takes device tensors)")
        lens, d = _host_i32(q_lens, "q_lens"), _host_u32(slots, "slots")
        s = None if src_slots is None else _host_u32(src_slots, "src_slots")
        if lens.size != d.size or (s is not None and s.size != d.size):
            raise _bad("q_lens, slots and src_slots differ in length")
        if lens.size and int(lens.min()) < 0:
            raise _bad("q_lens holds a negative length")
        if int(lens.astype(np.int64).sum()) != n:
            raise _bad(f"q_lens add up to {int(lens.astype(np.int64).sum())} tokens, q has {n}")
        return lens, d, s

    def linear_extend_workspace_size(self, num_seqs: int, num_tokens: int, max_q_len: int) -> int:
        """Bytes of a workspace for linear_extend_device calls of that size (0: none is used)."""
        out = ctypes.c_uint64()
        _raise(self._lib.mkv_linear_extend_workspace_size(self._h, num_seqs, num_tokens, max_q_len, ctypes.byref(out)))
        return out.value

    def linear_extend_device(self, layer: int, q, k, v, log_decay, q_indptr, slots, max_q_len: int, src_slots=None,
                             out=None, scale: float | None = None, workspace=None, stream=None):
        """linear_extend with device metadata (int32 q_indptr [B + 1], slots,
        src_slots), read when the kernels run: it can be captured into a
        graph. workspace: a device tensor of linear_extend_workspace_size
        bytes (with less, of none too, sequences stay whole), or None for the
        pool's own."""
        torch = _torch()
        n, out, scale, flags = self._rows(q, k, v, log_decay, out, scale, stream=stream)
        if _is_host(slots):
            raise _bad("slots must be a device tensor")
        B, dst, src, _, _ = self._slots(slots, src_slots)
        _check(q_indptr, self.device, (B + 1,), torch.int32, "q_indptr")
        ws, nws = None, 0
        if workspace is not None:
            _check(workspace, self.device, None, getattr(workspace, "dtype", None), "workspace")
            nws = workspace.numel() * workspace.element_size()
            # (An empty tensor has no address, and no address is the pool's own.)
            ws = workspace.data_ptr() or self.data_ptr
        _raise(self._lib.mkv_linear_extend(
            self._h, layer, _dptr(q), _dptr(k), _dptr(v), _dptr(log_decay), _dptr(out), _dptr(q_indptr), src, dst, B,
            n, max_q_len, scale, flags, ws, nws, _stream(stream, self.device)))
        return out

    def bind_linear_step(self, q, k, v, log_decay, slots, out, src_slots=None, scale: float | None = None,
                         stream=None):
        """Checks, once, the buffers of one engine step (with a leading layer
        dimension, [L, B, ...], or without one, then shared by every layer)
        and returns `run(layer)`, which enqueues linear_step for that layer
        with no per-call Python checks. Host slots are copied here: a later
        change of the caller's arrays does not reach the bound call. Device
        slots are read by every call's kernel. A run goes to the given stream,
        or to the one that is current then; after close() it raises."""
        return self._bind(q, k, v, log_decay, None, slots, out, src_slots, scale, stream)

    def bind_linear_extend(self, q, k, v, log_decay, q_lens, slots, out, src_slots=None, scale: float | None = None,
                           stream=None):
        """bind_linear_step for linear_extend."""
        return self._bind(q, k, v, log_decay, q_lens, slots, out, src_slots, scale, stream)

    def _bind(self, q, k, v, log_decay, q_lens, slots, out, src_slots, scale, stream):
        L = self.desc.num_layers
        if out is None:
            raise _bad("a bound call needs out")
        lead = (L,) if getattr(q, "ndim", 0) == 4 else ()
        n, out, scale, flags = self._rows(q, k, v, log_decay, out, scale, lead, stream)
        # (The lengths are checked against q's rows here, and here only.)
        q_lens, slots, src_slots = (_host_copy(x) for x in (q_lens, slots, src_slots))
        if q_lens is None:
            B, dst, src, host, keep = self._slots(slots, src_slots)
            if B != n:
                raise _bad(f"{n} rows for {B} slots")
            fn = self._lib.mkv_linear_step_host if host else self._lib.mkv_linear_step
            meta = (src, dst, B)
        else:
            lens, d, s = keep = self._extend_meta(n, q_lens, slots, src_slots)
            fn = self._lib.mkv_linear_extend_host
            meta = (_i32p(lens), None if s is None else _u32p(s), _u32p(d), d.size)

        def at(t, layer):
            return ctypes.c_void_p(t.data_ptr() + (layer * (t.numel() // L) * t.element_size() if lead else 0))

        args = [(layer,) + tuple(at(t, layer) for t in (q, k, v, log_decay, out)) + meta + (scale, flags)
                for layer in range(L)]
        device = self.device

        def run(layer: int) -> None:
            if not 0 <= layer < L:
                raise _bad(f"layer {layer} out of range [0, {L})")
            # (self._h is None after close(), which the library refuses.)
            st = fn(self._h, *args[layer], _raw_stream(stream, device))
            if st:
                _raise(st)

        run.keep_alive = (self, q, k, v, log_decay, out, keep)
        return run


def add_rms_norm(x, weight, eps: float, residual=None, residual_out=None, out=None, fp8: bool = False,
                 group: int = 0, both: bool = False, stream=None):
    """r = x + residual, y = r * (mean(r^2) + eps)^-1/2 * (1 + weight) per row
    (mkv_add_rms_norm). x, residual: [rows, dim] f32 or bf16; weight: f32
    [dim]. Returns (r, y, fp8, scales), None for what was not asked for: r
    with a residual (in `residual_out`, which may be `residual`); y in x's type
    unless `fp8`; with `fp8`, e4m3 [rows, dim] and f32 scales [rows, dim /
    group] (group 0: one per row, [rows, 1]), and y beside them with `both`."""
    torch = _torch()
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() != 2:
        raise _bad("x must be a device tensor [rows, dim]")
    dt, shape, device = x.dtype, x.shape, x.device
    if dt != torch.float32 and dt != torch.bfloat16:
        raise _bad(f"x has dtype {dt}, expected float32 or bfloat16")
    dev = device.index
    rows, dim = shape
    if not x.is_contiguous():
        raise _bad("x must be contiguous")

    def like_x(t, name):  # (_check names what is wrong)
        if not isinstance(t, torch.Tensor) or t.dtype != dt or t.shape != shape or t.device != device or \
                not t.is_contiguous():
            _check(t, dev, shape, dt, name)
        return t.data_ptr()

    if not isinstance(weight, torch.Tensor) or weight.dtype != torch.float32 or weight.device != device or \
            weight.dim() != 1 or weight.shape[0] != dim or not weight.is_contiguous():
        _check(weight, dev, (dim,), torch.float32, "weight")
    if residual is not None and residual_out is None:
        residual_out = torch.empty_like(x) if stream is None else _empty_on(stream, shape, dt, device)
    if out is None and (both or not fp8):
        out = torch.empty_like(x) if stream is None else _empty_on(stream, shape, dt, device)
    q8 = scales = None
    if fp8:
        if group < 0 or (group and dim % group):
            raise _bad(f"group ({group}) does not divide dim ({dim})")
        new = torch.empty if stream is None else partial(_empty_on, stream)
        q8 = new((rows, dim), dtype=torch.float8_e4m3fn, device=device)
        scales = new((rows, dim // group if group else 1), dtype=torch.float32, device=device)
    elif group:
        raise _bad("group is for an e4m3 output")
    st = _lib.device_lib().mkv_add_rms_norm(
        dev, x.data_ptr(), None if residual is None else like_x(residual, "residual"), weight.data_ptr(), eps, rows, dim,
        0 if dt == torch.float32 else 1, None if residual_out is None else like_x(residual_out, "residual_out"),
        None if out is None else like_x(out, "out"), None if q8 is None else q8.data_ptr(),
        None if scales is None else scales.data_ptr(), group, _raw_stream(stream, dev))
    if st:
        _raise(st)
    return residual_out, out, q8, scales
