"""The K/V cache in 8 bits, in Python.

`DeviceKv8Pool` owns one libmitten_kv 8-bit pool: e4m3 tiles of 16 tokens and one
KV head with a power of two each as their scale (mkv_kv8_*; the tile order is
described there). It holds twice the tokens of a bf16 `DeviceKvPool`, and its
attention reads half the bytes. Rows that go in and out are bf16 or f32
(`PoolDesc.dtype`).

    append(layer, k, v, q_lens, block_indptr, block_ids, ctx_lens)
    qk_norm_rope_append(layer, q, k, v, q_lens, block_indptr, block_ids, ctx_lens, ...)
    gather(layer, block_indptr, block_ids, ctx_lens)
    copy_blocks(src, dst)
    decode_step(layer, k_new, v_new, q, block_indptr, block_ids, ctx_lens)
    decode_attention(layer, q, block_indptr, block_ids, ctx_lens)
    extend_attention(layer, q, q_lens, block_indptr, block_ids, ctx_lens)

A call's sequences come in one of two forms, as elsewhere in this package:

* host arrays (numpy, lists, CPU tensors): checked and copied by the call; q_lens
  holds the new tokens of each sequence;
* device int32 tensors, read when the kernels run, so that a call can be captured
  into a graph: q_lens is then their indptr [B + 1], and max_q_len / max_ctx_len,
  the largest chunk and length that the call (or any replay) will find, are given.

The new rows of a sequence are its last ones, positions ctx - n .. ctx - 1 (its
ctx_lens counts them). A block that a call writes belongs to one sequence.

With `stream=`, what a call allocates is that stream's memory.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from .device_pool import (
    ATTN_ZERO_SINK,
    MKV_ERR_DEVICE_INDEX,
    PREP_NO_NORM,
    PREP_PLAIN_Q,
    DeviceIndexError,
    PoolDesc,
    _empty_on,
    _host_i32,
    _host_u32,
    _i32p,
    _is_host,
    _raise,
    _torch,
    _u32p,
    rope_inv_freq,
)
from .state_pool import _bad, _check, _raw_stream, _stream, _torch_type

PREP_INTERLEAVED = 4
KV8_MIN_EXP = -100  # the least exponent of a tile


def kv8_required_bytes(desc: PoolDesc):
    """(bytes of the tiles, bytes of the exponents)."""
    a, b = ctypes.c_uint64(), ctypes.c_uint64()
    _raise(_lib.device_lib().mkv_kv8_required_bytes(ctypes.byref(desc.c()), ctypes.byref(a), ctypes.byref(b)))
    return a.value, b.value


def rope_scaled_inv_freq(rotary_dim: int, theta: float, factor: float, original_len: int, method: str = "yarn",
                         beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(inv_freq f32 [rotary_dim / 2], rope_factor) for contexts `factor` times
    the original length.

    "linear": every frequency divided by `factor` (positions interpolated);
    "ntk": theta grown so that the lowest frequency is divided by `factor`;
    "yarn": YaRN (Peng et al., 2023): frequencies with more than beta_fast turns in
    original_len stay, those with fewer than beta_slow are divided by `factor`, a
    linear ramp between, and cos and sin are scaled by 0.1 ln(factor) + 1."""
    if rotary_dim < 2 or rotary_dim % 2 or factor < 1.0 or original_len < 1:
        raise ValueError("rotary_dim must be even, factor >= 1 and original_len >= 1")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    if method == "linear":
        return (rope_inv_freq(rotary_dim, theta) / np.float32(factor)).astype(np.float32), 1.0
    if method == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk needs a rotary_dim of 4 or more")
        theta = float(theta) * float(factor) ** (rotary_dim / (rotary_dim - 2))
        return (theta ** (-2.0 * i / rotary_dim)).astype(np.float32), 1.0
    if method != "yarn":
        raise ValueError(f"unknown method {method!r}")
    freq = float(theta) ** (-2.0 * i / rotary_dim)

    def pair(turns):  # the pair that makes that many turns in original_len
        return rotary_dim * np.log(original_len / (turns * 2 * np.pi)) / (2 * np.log(theta))

    lo, hi = max(np.floor(pair(beta_fast)), 0.0), min(np.ceil(pair(beta_slow)), rotary_dim - 1.0)
    ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)  # 0: kept, 1: interpolated
    return ((1 - ramp) * freq + ramp * freq / factor).astype(np.float32), float(0.1 * np.log(factor) + 1.0)


class DeviceKv8Pool:
    """The K/V pool in 8 bits (see the module)."""

    def __init__(self, desc: PoolDesc, device: int = 0):
        self.desc = desc
        self.device = device
        self._lib = _lib.device_lib()
        h = ctypes.c_void_p()
        _raise(self._lib.mkv_kv8_pool_create(ctypes.byref(desc.c()), device, ctypes.byref(h)))
        self._h = h
        t, e, tn, en = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_uint64(), ctypes.c_uint64()
        _raise(self._lib.mkv_kv8_pool_buffers(self._h, ctypes.byref(t), ctypes.byref(tn), ctypes.byref(e),
                                              ctypes.byref(en)))
        self.tiles_ptr, self.tile_bytes, self.exponents_ptr, self.exponent_bytes = t.value, tn.value, e.value, en.value
        self._dtype = _torch_type(desc.dtype)
        self._tensor, self._int32 = _torch().Tensor, _torch().int32
        self._device = _torch().device("cuda", device)
        self._scale = float(np.float32(desc.head_dim ** -0.5))

    # -- lifecycle -------------------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "_h", None):
            self._lib.mkv_kv8_pool_destroy(self._h)
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
        return self._dtype

    def check(self, stream=None) -> None:
        """Synchronise and raise DeviceIndexError if a kernel met a bad id or length."""
        bits = ctypes.c_uint32()
        st = self._lib.mkv_kv8_pool_check(self._h, _stream(stream, self.device), ctypes.byref(bits))
        if st == MKV_ERR_DEVICE_INDEX:
            raise DeviceIndexError(st, self._lib.mkv_last_error().decode(), bits.value)
        _raise(st)

    def workspace_size(self) -> int:
        """Bytes of the pool's own workspace, with which no decode call is held back. An
        extend call of n tokens takes min(32, (bytes - 256) // (n * Hq * (8 + 4 * D)))
        partials a row, and is not cut with fewer than 2: a larger one allows more."""
        out = ctypes.c_uint64()
        _raise(self._lib.mkv_kv8_workspace_size(self._h, ctypes.byref(out)))
        return out.value

    def _view(self, ptr, shape, typestr):
        if not self._h:
            raise _bad("the pool is closed")

        class _View:
            pass

        view = _View()
        view.pool = self  # the tensor holds the view: the pool lives as long, but for a close()
        view.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 3,
                                         "strides": None}
        return _torch().as_tensor(view, device=f"cuda:{self.device}")

    def tensor(self):
        """Zero-copy uint8 view of the tiles, [L, 2, num_blocks, Hkv, 16 * D] (bytes in
        tile order; `.view(torch.float8_e4m3fn)` for their values). It keeps the pool
        alive; after close() it must not be read."""
        d = self.desc
        return self._view(self.tiles_ptr, (d.num_layers, 2, int(d.num_blocks), d.num_kv_heads, 16 * d.head_dim), "|u1")

    def exponents(self):
        """Zero-copy int8 view of the exponents, [L, 2, num_blocks, Hkv], as tensor()."""
        d = self.desc
        return self._view(self.exponents_ptr, (d.num_layers, 2, int(d.num_blocks), d.num_kv_heads), "|i1")

    # -- checks ------------------------------------------------------------------------
    def _rows(self, t, shape, name, dtype=None):
        """Address of a contiguous tensor of that shape on the pool's device."""
        dtype = dtype or self._dtype
        if not isinstance(t, self._tensor) or t.dtype != dtype or t.shape != shape or t.device != self._device or \
                not t.is_contiguous():
            _check(t, self.device, shape, dtype, name)  # (names what is wrong)
        return t.data_ptr()

    def _num_rows(self, t, name, dims):
        if not isinstance(t, self._tensor) or t.dim() != dims:
            raise _bad(f"{name} must be a tensor of {dims} dimensions")
        return t.shape[0]

    def _i32(self, t, name, n=None):
        if not isinstance(t, self._tensor) or t.dtype != self._int32 or t.device != self._device or t.dim() != 1 or \
                not t.is_contiguous() or (n is not None and t.shape[0] != n):
            _check(t, self.device, None if n is None else (n,), self._int32, name)
            raise _bad(f"{name} must have one dimension")
        return t.data_ptr()

    def _form(self, block_indptr, block_ids, ctx_lens, q_lens=None):
        """Whether the metadata is the host's; all of it has to be, or none."""
        tensor = self._tensor
        if isinstance(ctx_lens, tensor) and ctx_lens.is_cuda:
            return False  # (the others are checked one by one)
        host = None
        for x in (ctx_lens, block_indptr, block_ids, q_lens):
            if x is None and x is q_lens:
                continue
            h = not x.is_cuda if isinstance(x, tensor) else _is_host(x)
            if host is not None and h != host:
                raise _bad("lengths and tables must all be host arrays or all device tensors")
            host = h
        return host

    def _tables(self, block_indptr, block_ids, ctx_lens):
        """Host arrays of the tables, and the number of sequences."""
        ip, ix = _host_u32(block_indptr, "block_indptr"), _host_u32(block_ids, "block_ids")
        cl = _host_i32(ctx_lens, "ctx_lens")
        if ip.size != cl.size + 1:
            raise _bad("block_indptr must have num_seqs + 1 entries")
        if ip.size and int(ip[-1]) > ix.size:
            raise _bad(f"block_indptr ends at {int(ip[-1])}, block_ids has {ix.size}")
        return ip, ix, cl

    def _lens(self, q_lens, cl, n):
        ql = _host_i32(q_lens, "q_lens")
        if ql.size != cl.size:
            raise _bad("q_lens and ctx_lens differ in length")
        if ql.size and int(ql.min()) < 0:
            raise _bad("q_lens holds a negative length")
        if int(ql.astype(np.int64).sum()) != n:
            raise _bad(f"q_lens add up to {int(ql.astype(np.int64).sum())} tokens, there are rows of {n}")
        return ql

    @staticmethod
    def _need(x, name):
        if x is None:
            raise _bad(f"device metadata needs {name}")
        return x

    def _device_tables(self, block_indptr, block_ids, ctx_lens, q_indptr=None):
        B = ctx_lens.shape[0] if getattr(ctx_lens, "ndim", 0) == 1 else -1
        at = (self._i32(block_indptr, "block_indptr", B + 1), self._i32(block_ids, "block_ids"),
              self._i32(ctx_lens, "ctx_lens", B))
        return B, at, None if q_indptr is None else self._i32(q_indptr, "q_indptr", B + 1)

    def _out(self, out, shape, stream, name="out"):
        if out is None:
            out = _empty_on(stream, shape, self._dtype, self._device)
        else:
            self._rows(out, shape, name)
        return out

    def _workspace(self, workspace):
        """(address, bytes); (None, 0) for the pool's own."""
        if workspace is None:
            return None, 0
        torch = _torch()
        if not isinstance(workspace, torch.Tensor):
            raise _bad("workspace must be a tensor")
        _check(workspace, self.device, None, workspace.dtype, "workspace")
        # (An empty tensor has no address, and no address is the pool's own.)
        return workspace.data_ptr() or self.tiles_ptr, workspace.numel() * workspace.element_size()

    # -- writing -----------------------------------------------------------------------
    def append(self, layer: int, k, v, q_lens, block_indptr, block_ids, ctx_lens, max_q_len: int | None = None,
               stream=None) -> None:
        """Quantise and write the new rows k, v [tokens, Hkv, D] of every sequence."""
        d = self.desc
        n = self._num_rows(k, "k", 3)
        shape = (n, d.num_kv_heads, d.head_dim)
        kp, vp = self._rows(k, shape, "k"), self._rows(v, shape, "v")
        sh = _raw_stream(stream, self.device)
        if self._form(block_indptr, block_ids, ctx_lens, q_lens):
            ip, ix, cl = self._tables(block_indptr, block_ids, ctx_lens)
            ql = self._lens(q_lens, cl, n)
            st = self._lib.mkv_kv8_append_host(self._h, layer, kp, vp, _i32p(ql), _i32p(cl), _u32p(ip), _u32p(ix),
                                               cl.size, sh)
        else:
            B, t, qi = self._device_tables(block_indptr, block_ids, ctx_lens, q_lens)
            st = self._lib.mkv_kv8_append(self._h, layer, kp, vp, qi, *t, B, n, self._need(max_q_len, "max_q_len"), sh)
        if st:
            _raise(st)

    def qk_norm_rope_append(self, layer: int, q, k, v, q_lens, block_indptr, block_ids, ctx_lens,
                            max_q_len: int | None = None, positions=None, q_norm_w=None, k_norm_w=None, inv_freq=None,
                            eps: float = 1e-6, rope_factor: float = 1.0, interleaved: bool = False, gated: bool = True,
                            out=None, stream=None):
        """The step before attention: RMSNorm(1 + w) of the q and k heads (weights
        None: none), rotary positions on the first 2 * len(inv_freq) dims (None: none;
        pairs (i, i + half), or (2i, 2i + 1) if `interleaved`; cos and sin times
        `rope_factor`), k and v appended. q: [tokens, Hq, 2, D] (q then gate) when
        `gated`, else [tokens, Hq, D]. positions: int32 per token (host or device, as
        the tables), default the positions in the sequence. Returns the prepared q
        [tokens, Hq, D]."""
        torch = _torch()
        d = self.desc
        n = self._num_rows(k, "k", 3)
        shape = (n, d.num_kv_heads, d.head_dim)
        kp, vp = self._rows(k, shape, "k"), self._rows(v, shape, "v")
        qshape = (n, d.num_q_heads, d.head_dim)
        qp = self._rows(q, (n, d.num_q_heads, 2, d.head_dim) if gated else qshape, "q")
        flags = (0 if gated else PREP_PLAIN_Q) | (PREP_INTERLEAVED if interleaved else 0)
        if (q_norm_w is None) != (k_norm_w is None):
            raise _bad("give both norm weights or neither")
        wq = wk = fp = None
        if q_norm_w is None:
            flags |= PREP_NO_NORM
        else:
            wq = self._rows(q_norm_w, (d.head_dim,), "q_norm_w", torch.float32)
            wk = self._rows(k_norm_w, (d.head_dim,), "k_norm_w", torch.float32)
        rd = 0
        if inv_freq is not None:
            rd = 2 * self._num_rows(inv_freq, "inv_freq", 1)
            fp = self._rows(inv_freq, (rd // 2,), "inv_freq", torch.float32)
        out = self._out(out, qshape, stream)
        sh = _raw_stream(stream, self.device)
        if self._form(block_indptr, block_ids, ctx_lens, q_lens):
            ip, ix, cl = self._tables(block_indptr, block_ids, ctx_lens)
            ql = self._lens(q_lens, cl, n)
            pos = None
            if positions is not None:
                if not _is_host(positions):
                    raise _bad("positions must be a host array, as the tables")
                pos = _host_i32(positions, "positions")
                if pos.size != n:
                    raise _bad(f"{pos.size} positions for {n} tokens")
            st = self._lib.mkv_kv8_qk_norm_rope_append_host(
                self._h, layer, qp, kp, vp, wq, wk, fp, rd, eps, rope_factor, None if pos is None else _i32p(pos),
                _i32p(ql), _i32p(cl), _u32p(ip), _u32p(ix), cl.size, out.data_ptr(), flags, sh)
        else:
            B, t, qi = self._device_tables(block_indptr, block_ids, ctx_lens, q_lens)
            pos = None if positions is None else self._i32(positions, "positions", n)
            st = self._lib.mkv_kv8_qk_norm_rope_append(
                self._h, layer, qp, kp, vp, wq, wk, fp, rd, eps, rope_factor, pos, qi, *t, B, n,
                self._need(max_q_len, "max_q_len"), out.data_ptr(), flags, sh)
        if st:
            _raise(st)
        return out

    # -- reading back, copies ------------------------------------------------------------
    def gather(self, layer: int, block_indptr, block_ids, ctx_lens, max_ctx_len: int | None = None,
               total_tokens: int | None = None, out_k=None, out_v=None, stream=None):
        """The rows of every sequence in the pool's dtype: (k, v), each flat
        [sum(ctx) * Hkv * D] with sequence b's [Hkv][ctx_b][D] after those before it.
        Device metadata needs total_tokens (>= the sum of the lengths) and max_ctx_len."""
        d = self.desc
        row = d.num_kv_heads * d.head_dim
        host = self._form(block_indptr, block_ids, ctx_lens)
        if host:
            ip, ix, cl = self._tables(block_indptr, block_ids, ctx_lens)
            if cl.size and int(cl.min()) < 0:
                raise _bad("ctx_lens holds a negative length")
            total_tokens = int(cl.astype(np.int64).sum())
        n = self._need(total_tokens, "total_tokens") * row
        outs = []
        for t, name in ((out_k, "out_k"), (out_v, "out_v")):
            if t is None:
                t = _empty_on(stream, n, self._dtype, self._device)
            else:
                _check(t, self.device, None, self._dtype, name)
                if t.numel() < n:
                    raise _bad(f"{name} is too small")
            outs.append(t)
        if n == 0:
            return tuple(outs)
        cap = min(t.numel() for t in outs) // row
        sh = _raw_stream(stream, self.device)
        if host:
            st = self._lib.mkv_kv8_gather_host(self._h, layer, _u32p(ip), _u32p(ix), _i32p(cl), cl.size,
                                               outs[0].data_ptr(), outs[1].data_ptr(), cap, sh)
        else:
            B, t, _ = self._device_tables(block_indptr, block_ids, ctx_lens)
            st = self._lib.mkv_kv8_gather(self._h, layer, *t, B, self._need(max_ctx_len, "max_ctx_len"),
                                          outs[0].data_ptr(), outs[1].data_ptr(), cap, sh)
        if st:
            _raise(st)
        return tuple(outs)

    def copy_blocks(self, src, dst, stream=None) -> None:
        """Whole blocks with their exponents, all layers: block dst[i] becomes block
        src[i]. Host u32 ids (checked: distinct destinations, none a source), or
        device int32."""
        sh = _raw_stream(stream, self.device)
        if _is_host(src) != _is_host(dst):
            raise _bad("src and dst must both be host arrays or both device tensors")
        if _is_host(src):
            s, t = _host_u32(src, "src"), _host_u32(dst, "dst")
            if s.size != t.size:
                raise _bad("src and dst differ in length")
            _raise(self._lib.mkv_kv8_copy_blocks_host(self._h, _u32p(s), _u32p(t), s.size, sh))
            return
        sp = self._i32(src, "src")
        _raise(self._lib.mkv_kv8_copy_blocks(self._h, sp, self._i32(dst, "dst", src.shape[0]), src.shape[0], sh))

    # -- attention ---------------------------------------------------------------------
    def _decode(self, layer, k_new, v_new, q, block_indptr, block_ids, ctx_lens, max_ctx_len, out, scale, zero_sink,
                workspace, stream):
        d = self.desc
        B = self._num_rows(q, "q", 3)
        qshape, kshape = (B, d.num_q_heads, d.head_dim), (B, d.num_kv_heads, d.head_dim)
        qp = self._rows(q, qshape, "q")
        kp = vp = None
        if k_new is not None:
            kp, vp = self._rows(k_new, kshape, "k_new"), self._rows(v_new, kshape, "v_new")
        out = self._out(out, qshape, stream)
        flags = ATTN_ZERO_SINK if zero_sink else 0
        scale = self._scale if scale is None else scale
        sh = _raw_stream(stream, self.device)
        if self._form(block_indptr, block_ids, ctx_lens):
            ip, ix, cl = self._tables(block_indptr, block_ids, ctx_lens)
            if cl.size != B:
                raise _bad(f"{B} rows for {cl.size} sequences")
            if workspace is not None:
                raise _bad("a workspace is for device metadata")
            st = self._lib.mkv_kv8_decode_attention_host(self._h, layer, kp, vp, qp, out.data_ptr(), _i32p(cl),
                                                         _u32p(ip), _u32p(ix), B, scale, flags, sh)
        else:
            n, t, _ = self._device_tables(block_indptr, block_ids, ctx_lens)
            if n != B:
                raise _bad(f"{B} rows for {n} sequences")
            ws, nws = self._workspace(workspace)
            st = self._lib.mkv_kv8_decode_attention(self._h, layer, kp, vp, qp, out.data_ptr(), *t, B,
                                                    self._need(max_ctx_len, "max_ctx_len"), scale, flags, ws, nws, sh)
        if st:
            _raise(st)
        return out

    def decode_attention(self, layer: int, q, block_indptr, block_ids, ctx_lens, max_ctx_len: int | None = None,
                         out=None, scale: float | None = None, zero_sink: bool = False, workspace=None, stream=None):
        """One query row per sequence, q [B, Hq, D], over its first ctx tokens. Returns
        o [B, Hq, D]; zeros where ctx is 0. workspace: a device tensor of
        workspace_size() bytes (with less, long contexts are cut into fewer pieces),
        or None for the pool's own."""
        return self._decode(layer, None, None, q, block_indptr, block_ids, ctx_lens, max_ctx_len, out, scale, zero_sink,
                            workspace, stream)

    def decode_step(self, layer: int, k_new, v_new, q, block_indptr, block_ids, ctx_lens,
                    max_ctx_len: int | None = None, out=None, scale: float | None = None, zero_sink: bool = False,
                    workspace=None, stream=None):
        """decode_attention that first appends the step's rows k_new, v_new
        [B, Hkv, D] at position ctx - 1."""
        if k_new is None or v_new is None:
            raise _bad("decode_step needs k_new and v_new")
        return self._decode(layer, k_new, v_new, q, block_indptr, block_ids, ctx_lens, max_ctx_len, out, scale,
                            zero_sink, workspace, stream)

    def bind_decode_step(self, k_new, v_new, q, block_indptr, block_ids, ctx_lens, out, max_ctx_len: int,
                         scale: float | None = None, zero_sink: bool = False, workspace=None, stream=None):
        """Checks, once, the buffers of one engine step (with a leading layer
        dimension, [L, B, ...], or without one, then shared by every layer) and
        returns `run(layer)`, which enqueues decode_step for that layer with no
        per-call Python checks. Tables and lengths are device tensors, read by every
        call's kernels. A run goes to the given stream, or to the one that is current
        then; after close() it raises."""
        d = self.desc
        L = d.num_layers
        lead = (L,) if getattr(q, "ndim", 0) == 4 else ()
        B = q.shape[len(lead)] if getattr(q, "ndim", 0) >= 3 else -1
        qshape, kshape = lead + (B, d.num_q_heads, d.head_dim), lead + (B, d.num_kv_heads, d.head_dim)
        rows = [self._rows(t, s, n) for t, s, n in ((k_new, kshape, "k_new"), (v_new, kshape, "v_new"),
                                                    (q, qshape, "q"), (out, qshape, "out"))]
        if self._form(block_indptr, block_ids, ctx_lens):
            raise _bad("a bound step takes device tables and lengths")
        n, t, _ = self._device_tables(block_indptr, block_ids, ctx_lens)
        if n != B:
            raise _bad(f"{B} rows for {n} sequences")
        ws, nws = self._workspace(workspace)
        strides = [x.numel() // L * x.element_size() if lead else 0 for x in (k_new, v_new, q, out)]
        args = [(layer,) + tuple(p + layer * s for p, s in zip(rows, strides)) + t +
                (B, max_ctx_len, self._scale if scale is None else scale, ATTN_ZERO_SINK if zero_sink else 0, ws, nws)
                for layer in range(L)]
        fn, device = self._lib.mkv_kv8_decode_attention, self.device

        def run(layer: int) -> None:
            if not 0 <= layer < L:
                raise _bad(f"layer {layer} out of range [0, {L})")
            # (self._h is None after close(), which the library refuses.)
            st = fn(self._h, *args[layer], _raw_stream(stream, device))
            if st:
                _raise(st)

        run.keep_alive = (self, k_new, v_new, q, out, block_indptr, block_ids, ctx_lens, workspace)
        return run

    def extend_attention(self, layer: int, q, q_lens, block_indptr, block_ids, ctx_lens, max_q_len: int | None = None,
                         max_ctx_len: int | None = None, out=None, scale: float | None = None, zero_sink: bool = False,
                         workspace=None, stream=None):
        """Causal attention of each sequence's newest tokens, q [tokens, Hq, D], over
        its cache, whose rows are there already. Returns o [tokens, Hq, D]."""
        d = self.desc
        n = self._num_rows(q, "q", 3)
        shape = (n, d.num_q_heads, d.head_dim)
        qp = self._rows(q, shape, "q")
        out = self._out(out, shape, stream)
        flags = ATTN_ZERO_SINK if zero_sink else 0
        scale = self._scale if scale is None else scale
        sh = _raw_stream(stream, self.device)
        if self._form(block_indptr, block_ids, ctx_lens, q_lens):
            ip, ix, cl = self._tables(block_indptr, block_ids, ctx_lens)
            ql = self._lens(q_lens, cl, n)
            if workspace is not None:
                raise _bad("a workspace is for device metadata")
            st = self._lib.mkv_kv8_extend_attention_host(self._h, layer, qp, out.data_ptr(), _i32p(ql), _i32p(cl),
                                                         _u32p(ip), _u32p(ix), cl.size, scale, flags, sh)
        else:
            B, t, qi = self._device_tables(block_indptr, block_ids, ctx_lens, q_lens)
            ws, nws = self._workspace(workspace)
            st = self._lib.mkv_kv8_extend_attention(
                self._h, layer, qp, out.data_ptr(), qi, *t, B, n, self._need(max_q_len, "max_q_len"),
                self._need(max_ctx_len, "max_ctx_len"), scale, flags, ws, nws, sh)
        if st:
            _raise(st)
        return out
