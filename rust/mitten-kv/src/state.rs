//! The states of a hybrid model's linear-attention layers as a pool of slots
//! beside the K/V pool, linear attention with a scalar decay per head over them,
//! and the residual + norm between layers.
//!
//! Slots, forks and copies fit the `DeltaNet` variant of `KVCacheState`
//! (`inference-model-common/src/lib.rs:5-13`) as well; `linear_extend` and
//! `linear_step` do not compute its recurrence (the delta rule has a write
//! strength and an erase term, which they lack).
//!
//! A request holds one slot instead of a page table; slots come from the same
//! host allocator as pages (`KvCachePool`, one "page" per slot). A request
//! that starts from a prefix's snapshot reads the snapshot's slot and writes
//! its own: `src[b] != dst[b]` forks without a copy.

use crate::error::check;
use crate::pool::{KvDtype, Stream};
use inference_backend::EngineError;
use mitten_kv_sys as sys;
use std::ffi::c_void;
use std::ptr;

/// A source slot that holds no state: the request starts from zeros.
pub const STATE_NONE: u32 = sys::MKV_STATE_NONE;

/// The pool's shape: the linear-attention layers' heads and the slot count.
#[derive(Clone, Copy, Debug)]
pub struct StateGeometry {
    pub num_layers: usize,
    pub num_k_heads: usize,
    pub num_v_heads: usize,
    pub k_dim: usize,
    pub v_dim: usize,
    pub num_slots: usize,
    /// Of q, k, v and the output; states are f32.
    pub dtype: KvDtype,
}

impl StateGeometry {
    fn desc(&self) -> sys::mkv_state_desc {
        sys::mkv_state_desc {
            num_layers: self.num_layers as i32,
            num_k_heads: self.num_k_heads as i32,
            num_v_heads: self.num_v_heads as i32,
            k_dim: self.k_dim as i32,
            v_dim: self.v_dim as i32,
            dtype: self.dtype.raw(),
            num_slots: self.num_slots as i64,
        }
    }

    /// Bytes of the states.
    pub fn required_bytes(&self) -> Result<u64, EngineError> {
        let mut out = 0u64;
        check(unsafe { sys::mkv_state_required_bytes(&self.desc(), &mut out) })?;
        Ok(out)
    }
}

/// Device rows of one linear-attention call: q and k `[n][Hk][Dk]`, v and o
/// `[n][Hv][Dv]` in the pool's dtype, 16-byte aligned; log decays f32 `[n][Hv]`
/// (`[Hv]` with `MKV_LINEAR_HEAD_DECAY`).
#[derive(Clone, Copy, Debug)]
pub struct LinearIo {
    pub q: *const c_void,
    pub k: *const c_void,
    pub v: *const c_void,
    pub log_decay: *const f32,
    pub o: *mut c_void,
}

/// The state pool.
pub struct DeviceStatePool {
    raw: *mut sys::mkv_state_pool,
    geom: StateGeometry,
}

// Driven from one thread at a time, as DeviceKvPool.
unsafe impl Send for DeviceStatePool {}

impl DeviceStatePool {
    pub fn new(geom: StateGeometry, device: i32) -> Result<Self, EngineError> {
        let mut raw = ptr::null_mut();
        check(unsafe { sys::mkv_state_pool_create(&geom.desc(), device, &mut raw) })?;
        Ok(Self { raw, geom })
    }

    pub fn geometry(&self) -> &StateGeometry {
        &self.geom
    }

    /// The library handle, for the device-metadata forms. The pool keeps
    /// ownership.
    pub fn as_raw(&self) -> *mut sys::mkv_state_pool {
        self.raw
    }

    fn same_len(a: usize, b: usize) -> Result<(), EngineError> {
        if a == b {
            return Ok(());
        }
        Err(EngineError::Backend("linear attention: lengths and slots differ in count".into()))
    }

    /// The prefill requests of a step: request `b`'s `q_lens[b]` rows follow
    /// those of request `b - 1`; its state is read from `src[b]` (or
    /// `STATE_NONE`) and left in `dst[b]`.
    ///
    /// # Safety
    /// `io` holds device buffers of `sum(q_lens)` rows, valid until `stream`
    /// has run the call; `o` overlaps none of the others.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn linear_extend(&mut self, layer: usize, io: &LinearIo, q_lens: &[i32], src: &[u32], dst: &[u32],
                                scale: f32, flags: u32, stream: Stream) -> Result<(), EngineError> {
        Self::same_len(q_lens.len(), dst.len())?;
        Self::same_len(src.len(), dst.len())?;
        check(sys::mkv_linear_extend_host(self.raw, layer as i32, io.q, io.k, io.v, io.log_decay, io.o,
                                          q_lens.as_ptr(), src.as_ptr(), dst.as_ptr(), dst.len() as i32, scale, flags,
                                          stream))
    }

    /// The decode requests of a step: one row each.
    ///
    /// # Safety
    /// As for `linear_extend`, with `dst.len()` rows.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn linear_step(&mut self, layer: usize, io: &LinearIo, src: &[u32], dst: &[u32], scale: f32,
                              flags: u32, stream: Stream) -> Result<(), EngineError> {
        Self::same_len(src.len(), dst.len())?;
        check(sys::mkv_linear_step_host(self.raw, layer as i32, io.q, io.k, io.v, io.log_decay, io.o, src.as_ptr(),
                                        dst.as_ptr(), dst.len() as i32, scale, flags, stream))
    }

    /// Copies of whole slots, every layer: a prefix's snapshot, or compaction
    /// moves. Checked and copied before the call returns.
    pub fn copy_states(&mut self, src: &[u32], dst: &[u32], stream: Stream) -> Result<(), EngineError> {
        Self::same_len(src.len(), dst.len())?;
        check(unsafe { sys::mkv_state_copy_host(self.raw, src.as_ptr(), dst.as_ptr(), src.len() as i32, stream) })
    }

    /// Waits for `stream` and reports an out-of-range slot a kernel met.
    pub fn check(&mut self, stream: Stream) -> Result<(), EngineError> {
        let mut bits = 0u32;
        check(unsafe { sys::mkv_state_pool_check(self.raw, stream, &mut bits) })
    }
}

impl Drop for DeviceStatePool {
    fn drop(&mut self) {
        unsafe { sys::mkv_state_pool_destroy(self.raw) };
    }
}

/// `r = x + residual; y = r * (mean(r^2) + eps)^-1/2 * (1 + w)` per row
/// (`inference-model-qwen/src/model.rs:84-109,348-365`), `y` in `out` and / or
/// as e4m3 with scales per row (`group` 0) or group of columns.
///
/// # Safety
/// Device buffers of `rows * dim` elements (`weight`: f32 `[dim]`, `scales`:
/// f32 `[rows][dim / group]`), 16-byte aligned; `residual`, `sum`, `out`, `fp8`
/// and `scales` may be null as `mkv_add_rms_norm` has it.
#[allow(clippy::too_many_arguments)]
pub unsafe fn add_rms_norm(device: i32, x: *const c_void, residual: *const c_void, weight: *const f32, eps: f32,
                           rows: usize, dim: usize, dtype: KvDtype, sum: *mut c_void, out: *mut c_void,
                           fp8: *mut c_void, scales: *mut f32, group: usize, stream: Stream) -> Result<(), EngineError> {
    check(sys::mkv_add_rms_norm(device, x, residual, weight, eps, rows as i32, dim as i32, dtype.raw(), sum, out, fp8,
                                scales, group as i32, stream))
}
