//! The K/V pool in 8 bits: e4m3 tiles of 16 tokens and one KV head with a power of
//! two each, twice the tokens of a bf16 pool (`KvCachePool::required_bytes`,
//! `inference-engine/src/kv_pool.rs:58-68`, for half the bytes per element and
//! `KVCacheState::Attention`'s rows, `inference-model-common/src/lib.rs:5-13`).
//!
//! Its calls name the requests by their page tables and lengths, as the batch
//! carries them (`inference-backend/src/batch.rs:24-26`): the new rows of a
//! request are its last ones. A block that a call writes belongs to one request.

use crate::error::check;
use crate::pool::{PoolGeometry, Stream, Tables};
use inference_backend::EngineError;
use mitten_kv_sys as sys;
use std::ffi::c_void;
use std::ptr;

/// A step's requests: table `b`, the tokens it holds with the new ones, and how many
/// of them are new (`q_lens`; a decode step has one each).
#[derive(Clone, Copy, Debug)]
pub struct Requests<'a> {
    pub tables: &'a Tables,
    pub ctx_lens: &'a [i32],
    pub q_lens: &'a [i32],
}

/// What the fused step before attention applies to q and k heads: RMSNorm weights
/// (null: no norm) and rotary frequencies (`rotary_dim` 0: none), f32 on the device.
#[derive(Clone, Copy, Debug)]
pub struct Preparation {
    pub q_norm: *const f32,
    pub k_norm: *const f32,
    pub eps: f32,
    pub inv_freq: *const f32,
    pub rotary_dim: usize,
    /// Of cos and sin; 1 for plain RoPE.
    pub rope_factor: f32,
    /// `MKV_PREP_PLAIN_Q`, `MKV_PREP_INTERLEAVED`.
    pub flags: u32,
}

/// The pool.
pub struct DeviceKv8Pool {
    raw: *mut sys::mkv_kv8_pool,
    geom: PoolGeometry,
}

// Driven from one thread at a time, as DeviceKvPool.
unsafe impl Send for DeviceKv8Pool {}

impl DeviceKv8Pool {
    /// `geom.dtype` is the type of the rows that go in and out.
    pub fn new(geom: PoolGeometry, device: i32) -> Result<Self, EngineError> {
        let mut raw = ptr::null_mut();
        check(unsafe { sys::mkv_kv8_pool_create(&geom.desc(), device, &mut raw) })?;
        Ok(Self { raw, geom })
    }

    /// Bytes of the tiles and of their exponents.
    pub fn required_bytes(geom: &PoolGeometry) -> Result<(u64, u64), EngineError> {
        let (mut tiles, mut exponents) = (0u64, 0u64);
        check(unsafe { sys::mkv_kv8_required_bytes(&geom.desc(), &mut tiles, &mut exponents) })?;
        Ok((tiles, exponents))
    }

    pub fn geometry(&self) -> &PoolGeometry {
        &self.geom
    }

    /// The library handle, for the device-metadata forms. The pool keeps
    /// ownership.
    pub fn as_raw(&self) -> *mut sys::mkv_kv8_pool {
        self.raw
    }

    fn fits(r: &Requests, rows: bool) -> Result<i32, EngineError> {
        let n = r.tables.len();
        if r.ctx_lens.len() != n || (rows && r.q_lens.len() != n) {
            return Err(EngineError::Backend("8-bit pool: tables and lengths differ in count".into()));
        }
        Ok(n as i32)
    }

    /// Quantise and write the new rows k, v `[sum(q_lens)][Hkv][D]`.
    ///
    /// # Safety
    /// Device buffers of that many rows, 16-byte aligned, valid until `stream` has
    /// run the call.
    pub unsafe fn append(&mut self, layer: usize, k: *const c_void, v: *const c_void, r: &Requests,
                         stream: Stream) -> Result<(), EngineError> {
        let n = Self::fits(r, true)?;
        check(sys::mkv_kv8_append_host(self.raw, layer as i32, k, v, r.q_lens.as_ptr(), r.ctx_lens.as_ptr(),
                                       r.tables.indptr.as_ptr(), r.tables.ids.as_ptr(), n, stream))
    }

    /// `append` with norm and rotary positions of the q and k heads; q goes to
    /// `q_out` `[sum(q_lens)][Hq][D]`.
    ///
    /// # Safety
    /// As for `append`; `q` holds `[Hq][2][D]` per row, or `[Hq][D]` with
    /// `MKV_PREP_PLAIN_Q`.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn qk_norm_rope_append(&mut self, layer: usize, q: *const c_void, k: *const c_void, v: *const c_void,
                                      p: &Preparation, r: &Requests, q_out: *mut c_void,
                                      stream: Stream) -> Result<(), EngineError> {
        let n = Self::fits(r, true)?;
        let flags = p.flags | if p.q_norm.is_null() { sys::MKV_PREP_NO_NORM } else { 0 };
        check(sys::mkv_kv8_qk_norm_rope_append_host(self.raw, layer as i32, q, k, v, p.q_norm, p.k_norm, p.inv_freq,
                                                    p.rotary_dim as i32, p.eps, p.rope_factor, ptr::null(),
                                                    r.q_lens.as_ptr(), r.ctx_lens.as_ptr(), r.tables.indptr.as_ptr(),
                                                    r.tables.ids.as_ptr(), n, q_out, flags, stream))
    }

    /// The decode requests of a step, one row each: k_new and v_new are appended
    /// (both null: nothing is) and q attends to the first `ctx_lens[b]` tokens.
    ///
    /// # Safety
    /// As for `append`, with one row per request; `o` overlaps none of the others.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn decode_step(&mut self, layer: usize, k_new: *const c_void, v_new: *const c_void, q: *const c_void,
                              o: *mut c_void, r: &Requests, scale: f32, flags: u32,
                              stream: Stream) -> Result<(), EngineError> {
        let n = Self::fits(r, false)?;
        check(sys::mkv_kv8_decode_attention_host(self.raw, layer as i32, k_new, v_new, q, o, r.ctx_lens.as_ptr(),
                                                 r.tables.indptr.as_ptr(), r.tables.ids.as_ptr(), n, scale, flags,
                                                 stream))
    }

    /// Causal attention of the new tokens, whose rows are in the pool already.
    ///
    /// # Safety
    /// As for `append`: q and o `[sum(q_lens)][Hq][D]`, apart.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn extend_attention(&mut self, layer: usize, q: *const c_void, o: *mut c_void, r: &Requests, scale: f32,
                                   flags: u32, stream: Stream) -> Result<(), EngineError> {
        let n = Self::fits(r, true)?;
        check(sys::mkv_kv8_extend_attention_host(self.raw, layer as i32, q, o, r.q_lens.as_ptr(), r.ctx_lens.as_ptr(),
                                                 r.tables.indptr.as_ptr(), r.tables.ids.as_ptr(), n, scale, flags,
                                                 stream))
    }

    /// The rows of every request, `[Hkv][ctx][D]` each, into buffers of
    /// `capacity_tokens` rows.
    ///
    /// # Safety
    /// Device buffers of `capacity_tokens * Hkv * D` elements, 16-byte aligned.
    #[allow(clippy::too_many_arguments)]
    pub unsafe fn gather(&mut self, layer: usize, r: &Requests, out_k: *mut c_void, out_v: *mut c_void,
                         capacity_tokens: usize, stream: Stream) -> Result<(), EngineError> {
        let n = Self::fits(r, false)?;
        check(sys::mkv_kv8_gather_host(self.raw, layer as i32, r.tables.indptr.as_ptr(), r.tables.ids.as_ptr(),
                                       r.ctx_lens.as_ptr(), n, out_k, out_v, capacity_tokens as i64, stream))
    }

    /// Whole blocks with their exponents, every layer: copy-on-write pairs,
    /// compaction moves. Checked and copied before the call returns.
    pub fn copy_blocks(&mut self, src: &[u32], dst: &[u32], stream: Stream) -> Result<(), EngineError> {
        if src.len() != dst.len() {
            return Err(EngineError::Backend("8-bit pool: block copies differ in count".into()));
        }
        check(unsafe { sys::mkv_kv8_copy_blocks_host(self.raw, src.as_ptr(), dst.as_ptr(), src.len() as i32, stream) })
    }

    /// Waits for `stream` and reports a bad id or length that a kernel met.
    pub fn check(&mut self, stream: Stream) -> Result<(), EngineError> {
        let mut bits = 0u32;
        check(unsafe { sys::mkv_kv8_pool_check(self.raw, stream, &mut bits) })
    }
}

impl Drop for DeviceKv8Pool {
    fn drop(&mut self) {
        unsafe { sys::mkv_kv8_pool_destroy(self.raw) };
    }
}
