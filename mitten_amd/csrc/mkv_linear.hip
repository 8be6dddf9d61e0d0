// Linear-attention states: the pool that holds them, copies between slots, and
// the step that moves each sequence's on by one token.
//
// A linear-attention layer keeps, instead of K/V rows, one matrix per value
// head and sequence. The recurrence here is that of a scalar decay per head
// (the delta rule, which also erases along k_t, is another):
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <new>

#include "mkv_linear.h"

namespace mkv {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- kernels ------------------------------------------------------------------

template <bool BF16>
__device__ __forceinline__ float lin_elem(const void *p, int64_t i) {
  if constexpr (BF16) return __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
  else return static_cast<const float *>(p)[i];
}

// One step of the recurrence. A workgroup of 256 threads moves CW columns of one
// (sequence, value head) state: thread (rg, cg) the rows rg + R*i and the four
// columns 4*cg, so that each of its loads and stores covers R whole row pieces
// of CW floats, all of them in flight before k, q and v arrive in LDS. The R
// partial outputs of a column (a thread's own rows' share of S^T q) are added
// through LDS in order. Bound by HBM: the state moves once each way, without a
// stay in the caches (a step passes through every layer's states before it
// returns to one). 64 sequences of 28 heads 45 us, 504 of 32 heads 383 us: 5.2
// and 5.4 TB/s, what a copy of the same size reaches.
template <int DK, int CW, bool BF16>
__global__ void __launch_bounds__(256) linear_step_kernel(LinArgs a) {
  constexpr int CG = CW / 4, R = 256 / CG, NI = DK / R;
  static_assert(R <= DK && NI >= 1, "every thread holds at least one row");
  __shared__ float ks[DK], qs[DK];
  __shared__ __attribute__((aligned(16))) float vs[CW];
  __shared__ __attribute__((aligned(16))) float red[R][CW];
  const int tid = threadIdx.x, cg = tid % CG, rg = tid / CG;
  const int slices = a.DV / CW;
  const int sl = blockIdx.x % slices, h = (blockIdx.x / slices) % a.Hv, b = blockIdx.x / (slices * a.Hv);
  LinSeq s;
  if (!lin_seq(a, b, tid == 0 && h == 0 && sl == 0, s)) return;  // uniform over the workgroup
  const int kh = h / (a.Hv / a.Hk);
  const int64_t plane = (int64_t)a.Hv * DK * a.DV;
  const int64_t off = (int64_t)h * DK * a.DV + sl * CW + 4 * cg;
  // (A buffer of no bytes where there is no state: its loads are zeros.)
  const int src = __builtin_amdgcn_readfirstlane((int)s.src);
  const auto from = __builtin_amdgcn_make_buffer_rsrc(a.states + max(src, 0) * plane + (int64_t)h * DK * a.DV, 0,
                                                      src >= 0 ? DK * a.DV * 4 : 0, 0x00027000);
  constexpr int kNt = 2;  // non-temporal
  f32x4 S[NI];
#pragma unroll
  for (int i = 0; i < NI; i++)
    S[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                         from, ((rg + R * i) * a.DV + sl * CW + 4 * cg) * 4, 0, kNt));
  const int64_t krow = ((int64_t)s.row0 * a.Hk + kh) * DK, vrow = ((int64_t)s.row0 * a.Hv + h) * a.DV + sl * CW;
  if (tid < DK) {
    ks[tid] = lin_elem<BF16>(a.k, krow + tid);
    qs[tid] = lin_elem<BF16>(a.q, krow + tid);
  }
  if (tid < CW) vs[tid] = lin_elem<BF16>(a.v, vrow + tid);
  const float d = expf(a.g[(int64_t)s.row0 * a.g_stride + h]);
  __syncthreads();
  const f32x4 v = *reinterpret_cast<const f32x4 *>(&vs[4 * cg]);
  f32x4 o = {};
#pragma unroll
  for (int i = 0; i < NI; i++) {
    S[i] = d * S[i] + ks[rg + R * i] * v;
    o += qs[rg + R * i] * S[i];
    __builtin_nontemporal_store(
        S[i], reinterpret_cast<f32x4 *>(a.states + s.dst * plane + off + (int64_t)(rg + R * i) * a.DV));
  }
  *reinterpret_cast<f32x4 *>(&red[rg][4 * cg]) = o;
  __syncthreads();
  if (tid < CW) {
    float x = 0.0f;
#pragma unroll
    for (int r = 0; r < R; r++) x += red[r][tid];
    x *= a.scale;
    if constexpr (BF16) static_cast<uint16_t *>(a.o)[vrow + tid] = (uint16_t)f32_to_bf16_bits(x);
    else static_cast<float *>(a.o)[vrow + tid] = x;
  }
}

// grid.x = (pair, part), grid.y = layer: a workgroup copies one 32 KiB part
// of a slot's state of one layer, all its 16-byte loads first. (A state is
// 0.5 to 8 MiB: a workgroup per state left most of the device idle in a fork
// of a few, 78 us for 3 pairs of 6 layers against 12.)
// Bound by HBM: 85 pairs of 4 layers at 5.4 TB/s, as a plain copy.
constexpr int kStatePer = 8;

// A few pairs travel as kernel arguments (3 pairs of 6 layers 17 us with an
// upload ahead of the launch, 12 without).
constexpr int kArgPairs = 64;
struct ArgPairs {
  int32_t src[kArgPairs], dst[kArgPairs];
};
struct MemPairs {
  const int32_t *src, *dst;
};

template <class Pairs>
__global__ void __launch_bounds__(256) state_copy_kernel(float *__restrict__ states, Pairs pairs, int64_t nslots,
                                                         int64_t elems, int parts, uint32_t *__restrict__ d_err) {
  const int pair = blockIdx.x / parts, part = blockIdx.x % parts;
  const int32_t s = pairs.src[pair], d = pairs.dst[pair];
  if (s < 0 || s >= nslots || d < 0 || d >= nslots) {
    if (part == 0 && blockIdx.y == 0 && threadIdx.x == 0) record_error(d_err, MKV_DEVERR_COPY);
    return;
  }
  const int64_t plane = (int64_t)blockIdx.y * nslots * elems;
  const f32x4 *sp = reinterpret_cast<const f32x4 *>(states + plane + s * elems);
  f32x4 *dp = reinterpret_cast<f32x4 *>(states + plane + d * elems);
  const int64_t total = elems / 4, base = (int64_t)part * 256 * kStatePer + threadIdx.x;
  f32x4 r[kStatePer];
#pragma unroll
  for (int u = 0; u < kStatePer; u++) r[u] = __builtin_nontemporal_load(sp + min(base + u * 256, total - 1));
#pragma unroll
  for (int u = 0; u < kStatePer; u++)
    if (base + u * 256 < total) __builtin_nontemporal_store(r[u], dp + base + u * 256);
}

// ---- host side ------------------------------------------------------------------

static int validate_state_desc(const mkv_state_desc *d) {
  if (!d) return set_error(MKV_ERR_INVALID_ARGUMENT, "desc is NULL");
  if (d->num_layers < 1 || d->num_layers > 65535 || d->num_k_heads < 1 || d->num_v_heads < 1 || d->num_slots < 1)
    return set_error(MKV_ERR_INVALID_ARGUMENT,
                     "num_layers (at most 65535), num_k_heads, num_v_heads and num_slots must be >= 1");
  if (d->num_v_heads % d->num_k_heads || d->num_v_heads > 1024)
    return set_error(MKV_ERR_INVALID_ARGUMENT,
                     "num_v_heads (%d) must be a multiple of num_k_heads (%d) and at most 1024", d->num_v_heads,
                     d->num_k_heads);
  for (int32_t x : {d->k_dim, d->v_dim})
    if (x != 64 && x != 128 && x != 256)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "k_dim and v_dim must be 64, 128 or 256 (got %d)", x);
  if (d->dtype != MKV_DTYPE_F32 && d->dtype != MKV_DTYPE_BF16)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "unknown dtype %d", d->dtype);
  if (d->num_slots > INT32_MAX) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_slots too large for int32 slot ids");
  const unsigned __int128 bytes = (unsigned __int128)d->num_layers * d->num_slots * d->num_v_heads * d->k_dim * d->v_dim * 4;
  if (bytes > (unsigned __int128)INT64_MAX) return set_error(MKV_ERR_INVALID_ARGUMENT, "the pool's size overflows");
  return MKV_OK;
}

static int64_t state_elems(const mkv_state_desc *d) { return (int64_t)d->num_v_heads * d->k_dim * d->v_dim; }

int lin_args(StatePool *p, int32_t layer, const void *d_q, const void *d_k, const void *d_v, const float *d_g,
             void *d_o, const int32_t *d_src, const int32_t *d_dst, int32_t num_seqs, int32_t num_tokens, float scale,
             uint32_t flags, LinArgs &a) {
  const mkv_state_desc &d = p->desc;
  if (layer < 0 || layer >= d.num_layers)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "layer %d out of range [0, %d)", layer, d.num_layers);
  if (flags & ~(uint32_t)MKV_LINEAR_HEAD_DECAY) return set_error(MKV_ERR_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
  if (num_seqs < 0 || num_seqs > 65535)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs (%d) must be in [0, 65535]", num_seqs);
  if (!std::isfinite(scale)) return set_error(MKV_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (num_tokens < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_tokens < 0");
  // A batch of empty chunks has no rows: only its slots are looked at.
  if (num_seqs && (!d_dst || (num_tokens && (!d_q || !d_k || !d_v || !d_g || !d_o))))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v) || !aligned16(d_o))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "q, k, v and o must be 16-byte aligned");
  // (Heads that share q and k, and columns that share a row, are computed apart.)
  const uint64_t es = d.dtype == MKV_DTYPE_F32 ? 4 : 2, n = (uint64_t)num_tokens;
  const uint64_t kb = n * d.num_k_heads * d.k_dim * es, vb = n * d.num_v_heads * d.v_dim * es;
  const uint64_t gb = (flags & MKV_LINEAR_HEAD_DECAY ? 1 : n) * d.num_v_heads * 4;
  if (n && (overlap(d_o, vb, d_q, kb) || overlap(d_o, vb, d_k, kb) || overlap(d_o, vb, d_v, vb) ||
            overlap(d_o, vb, d_g, gb)))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "o overlaps q, k, v or the decays");
  a = LinArgs{};
  a.q = d_q;
  a.k = d_k;
  a.v = d_v;
  a.g = d_g;
  a.o = d_o;
  a.states = p->data + (int64_t)layer * d.num_slots * p->state_elems;
  a.src = d_src;
  a.dst = d_dst;
  a.d_err = p->d_err;
  a.nslots = d.num_slots;
  a.B = num_seqs;
  a.Hk = d.num_k_heads;
  a.Hv = d.num_v_heads;
  a.DV = d.v_dim;
  a.g_stride = (flags & MKV_LINEAR_HEAD_DECAY) ? 0 : d.num_v_heads;
  a.num_tokens = num_tokens;
  a.scale = scale;
  return MKV_OK;
}

int check_state_slots(StatePool *p, const uint32_t *src, const uint32_t *dst, int32_t n) {
  if (n < 0 || n > 65535) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs (%d) must be in [0, 65535]", n);
  if (n && !dst) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL destination slots");
  const uint64_t nslots = (uint64_t)p->desc.num_slots;
  try {
    if (p->mark.empty()) {
      p->owner.assign((size_t)nslots, 0);
      p->mark.assign((size_t)nslots, 0);
    }
  } catch (const std::bad_alloc &) {
    p->mark.clear();
    return set_error(MKV_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
  if (++p->epoch == 0) {  // wrapped: every mark is of an earlier call again
    std::fill(p->mark.begin(), p->mark.end(), 0u);
    p->epoch = 1;
  }
  for (int32_t i = 0; i < n; i++) {
    if (dst[i] >= nslots)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "dst slot[%d] = %u outside [0, %llu)", i, dst[i],
                       (unsigned long long)nslots);
    if (p->mark[dst[i]] == p->epoch)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "dst slot[%d] = %u is written twice", i, dst[i]);
    p->mark[dst[i]] = p->epoch;
    p->owner[dst[i]] = (uint32_t)i;
  }
  for (int32_t i = 0; src && i < n; i++) {
    if (src[i] == MKV_STATE_NONE) continue;
    if (src[i] >= nslots)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "src slot[%d] = %u outside [0, %llu)", i, src[i],
                       (unsigned long long)nslots);
    if (p->mark[src[i]] == p->epoch && p->owner[src[i]] != (uint32_t)i)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "src slot[%d] = %u is written by sequence %u", i, src[i],
                       p->owner[src[i]]);
  }
  return MKV_OK;
}

int refuse_capture(hipStream_t hs) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  MKV_CHECK_HIP(hipStreamIsCapturing(hs, &st));
  if (st != hipStreamCaptureStatusNone)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "host metadata cannot be captured: use the entry point with device arrays");
  return MKV_OK;
}

template <int DK, bool BF16>
static const void *step_fn(int cw) {
  if (cw == 64) return reinterpret_cast<const void *>(&linear_step_kernel<DK, 64, BF16>);
  if constexpr (DK < 256) return reinterpret_cast<const void *>(&linear_step_kernel<DK, 128, BF16>);
  return nullptr;
}

static int launch_step(StatePool *p, const LinArgs &a, hipStream_t hs) {
  const mkv_state_desc &d = p->desc;
  if (a.B == 0) return MKV_OK;
  // Columns per workgroup: as many as leave 16 or fewer 16-byte loads per
  // thread. (Narrower pieces to fill the device do not help one sequence: 32
  // workgroups of 128 columns and 128 of 32 both take 4.0 us, and 64 sequences
  // 44.8 us against 47.6.)
  const int cw = std::min(d.v_dim, d.k_dim == 256 ? 64 : 128);
  const int64_t wgs = (int64_t)a.B * a.Hv * (d.v_dim / cw);
  if (wgs > kMaxGrid) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs * num_v_heads too large for one launch");
  const bool bf = d.dtype == MKV_DTYPE_BF16;
  const void *fn = d.k_dim == 64    ? (bf ? step_fn<64, true>(cw) : step_fn<64, false>(cw))
                   : d.k_dim == 128 ? (bf ? step_fn<128, true>(cw) : step_fn<128, false>(cw))
                                    : (bf ? step_fn<256, true>(cw) : step_fn<256, false>(cw));
  LinArgs args = a;
  void *params[] = {&args};
  MKV_CHECK_HIP(hipLaunchKernel(fn, dim3((unsigned)wgs), dim3(256), params, 0, hs));
  return MKV_OK;
}

}  // namespace mkv

using namespace mkv;

// ---- C ABI: state pool lifecycle -----------------------------------------------------

extern "C" int mkv_state_required_bytes(const mkv_state_desc *desc, uint64_t *out_bytes) {
  int rc = validate_state_desc(desc);
  if (rc) return rc;
  if (!out_bytes) return set_error(MKV_ERR_INVALID_ARGUMENT, "out_bytes is NULL");
  *out_bytes = (uint64_t)desc->num_layers * (uint64_t)desc->num_slots * (uint64_t)state_elems(desc) * 4;
  return MKV_OK;
}

extern "C" int mkv_state_pool_create(const mkv_state_desc *desc, int device, mkv_state_pool **out_pool) {
  if (!out_pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "out_pool is NULL");
  *out_pool = nullptr;
  uint64_t bytes = 0;
  int rc = mkv_state_required_bytes(desc, &bytes);
  if (rc) return rc;
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0) {
    (void)hipGetLastError();
    return set_error(MKV_ERR_NO_DEVICE, "no HIP device available");
  }
  if (device < 0 || device >= ndev)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "device %d out of range (%d devices)", device, ndev);
  DeviceGuard guard(device);
  if (!guard.ok) return set_error(MKV_ERR_HIP, "hipSetDevice(%d) failed", device);
  StatePool *p = new (std::nothrow) StatePool();
  if (!p) return set_error(MKV_ERR_OUT_OF_MEMORY, "host allocation failed");
  p->desc = *desc;
  p->device = device;
  p->bytes = bytes;
  p->state_elems = state_elems(desc);
  hipError_t e = hipDeviceGetAttribute(&p->cus, hipDeviceAttributeMultiprocessorCount, device);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&p->data), bytes);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&p->d_err), 256);
  if (e == hipSuccess) e = hipMemset(p->d_err, 0, 256);
  p->ws_bytes = kLinWorkspace;
  if (e == hipSuccess) e = hipMalloc(&p->ws, p->ws_bytes);
  if (e == hipSuccess) e = hipEventCreateWithFlags(&p->ws_done, hipEventDisableTiming | hipEventDisableSystemFence);
  if (e != hipSuccess) {
    if (p->ws) (void)hipFree(p->ws);
    if (p->data) (void)hipFree(p->data);
    if (p->d_err) (void)hipFree(p->d_err);
    delete p;
    return hip_fail(e, "state pool allocation");
  }
  *out_pool = reinterpret_cast<mkv_state_pool *>(p);
  return MKV_OK;
}

extern "C" int mkv_state_pool_destroy(mkv_state_pool *pool) {
  if (!pool) return MKV_OK;
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  DeviceGuard guard(p->device);
  (void)hipDeviceSynchronize();
  meta_free(p);
  (void)hipEventDestroy(p->ws_done);
  (void)hipFree(p->ws);
  (void)hipFree(p->d_err);
  (void)hipFree(p->data);
  delete p;
  return MKV_OK;
}

extern "C" int mkv_state_pool_get_desc(const mkv_state_pool *pool, mkv_state_desc *out_desc) {
  if (!pool || !out_desc) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL argument");
  *out_desc = reinterpret_cast<const StatePool *>(pool)->desc;
  return MKV_OK;
}

extern "C" int mkv_state_pool_buffer(const mkv_state_pool *pool, void **out_dev_ptr, uint64_t *out_bytes) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  const StatePool *p = reinterpret_cast<const StatePool *>(pool);
  if (out_dev_ptr) *out_dev_ptr = p->data;
  if (out_bytes) *out_bytes = p->bytes;
  return MKV_OK;
}

extern "C" int mkv_state_pool_check(mkv_state_pool *pool, void *stream, uint32_t *out_bits) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  DeviceGuard guard(p->device);
  uint32_t bits = 0;
  MKV_CHECK_HIP(hipStreamSynchronize(reinterpret_cast<hipStream_t>(stream)));
  MKV_CHECK_HIP(hipMemcpy(&bits, p->d_err, sizeof(bits), hipMemcpyDeviceToHost));
  if (bits) MKV_CHECK_HIP(hipMemset(p->d_err, 0, sizeof(bits)));
  if (out_bits) *out_bits = bits;
  if (bits) return set_error(MKV_ERR_DEVICE_INDEX, "kernel met out-of-range ids (error bits 0x%x)", bits);
  return MKV_OK;
}

// ---- C ABI: copies -------------------------------------------------------------------

template <class Pairs>
static int launch_copy(StatePool *p, const Pairs &pairs, int32_t n, void *stream) {
  const int64_t parts = (p->state_elems / 4 + 256 * kStatePer - 1) / (256 * kStatePer);
  if (n * parts > kMaxGrid) return set_error(MKV_ERR_INVALID_ARGUMENT, "too many pairs for one launch");
  hipLaunchKernelGGL(state_copy_kernel<Pairs>, dim3((unsigned)(n * parts), (unsigned)p->desc.num_layers), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), p->data, pairs, p->desc.num_slots, p->state_elems, (int)parts,
                     p->d_err);
  MKV_CHECK_LAUNCH("state_copy_kernel");
  return MKV_OK;
}

extern "C" int mkv_state_copy(mkv_state_pool *pool, const int32_t *d_src_slots, const int32_t *d_dst_slots,
                              int32_t num_pairs, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  if (num_pairs < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_pairs < 0");
  if (num_pairs == 0) return MKV_OK;
  if (!d_src_slots || !d_dst_slots) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  DeviceGuard guard(p->device);
  return launch_copy(p, MemPairs{d_src_slots, d_dst_slots}, num_pairs, stream);
}

extern "C" int mkv_state_copy_host(mkv_state_pool *pool, const uint32_t *h_src_slots, const uint32_t *h_dst_slots,
                                   int32_t num_pairs, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  if (num_pairs < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_pairs < 0");
  if (num_pairs == 0) return MKV_OK;
  if (!h_src_slots || !h_dst_slots) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL host pointer");
  // The slots as check_state_slots has them, and no source that any pair
  // writes (the order of the copies is not defined).
  int rc = MKV_OK;
  for (int32_t i = 0; i < num_pairs; i++)
    if (h_src_slots[i] >= (uint64_t)p->desc.num_slots)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "src slot[%d] = %u outside [0, %lld)", i, h_src_slots[i],
                       (long long)p->desc.num_slots);
  if (num_pairs > 65535) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_pairs > 65535");
  if ((rc = check_state_slots(p, nullptr, h_dst_slots, num_pairs))) return rc;
  for (int32_t i = 0; i < num_pairs; i++)
    if (p->mark[h_src_slots[i]] == p->epoch)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "slot %u is both a source and a destination", h_src_slots[i]);
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  if ((rc = refuse_capture(hs))) return rc;
  if (num_pairs <= kArgPairs) {
    ArgPairs pairs = {};
    std::memcpy(pairs.src, h_src_slots, (size_t)num_pairs * 4);
    std::memcpy(pairs.dst, h_dst_slots, (size_t)num_pairs * 4);
    return launch_copy(p, pairs, num_pairs, stream);
  }
  MetaSlot *sl = nullptr;
  if ((rc = meta_acquire(p, 2 * (size_t)num_pairs, hs, &sl))) return rc;
  std::memcpy(sl->h, h_src_slots, (size_t)num_pairs * 4);
  std::memcpy(sl->h + num_pairs, h_dst_slots, (size_t)num_pairs * 4);
  if ((rc = meta_upload(sl, 2 * (size_t)num_pairs, hs))) return rc;
  rc = mkv_state_copy(pool, sl->d, sl->d + num_pairs, num_pairs, stream);
  const int rr = meta_release(sl, hs);
  return rc ? rc : rr;
}

// ---- C ABI: recurrent step -----------------------------------------------------------

extern "C" int mkv_linear_step(mkv_state_pool *pool, int32_t layer, const void *d_q, const void *d_k, const void *d_v,
                               const float *d_log_decay, void *d_o, const int32_t *d_src_slots,
                               const int32_t *d_dst_slots, int32_t num_seqs, float scale, uint32_t flags,
                               void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  LinArgs a;
  int rc = lin_args(p, layer, d_q, d_k, d_v, d_log_decay, d_o, d_src_slots, d_dst_slots, num_seqs, num_seqs, scale,
                    flags, a);
  if (rc) return rc;
  DeviceGuard guard(p->device);
  return launch_step(p, a, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int mkv_linear_step_host(mkv_state_pool *pool, int32_t layer, const void *d_q, const void *d_k,
                                    const void *d_v, const float *d_log_decay, void *d_o, const uint32_t *h_src_slots,
                                    const uint32_t *h_dst_slots, int32_t num_seqs, float scale, uint32_t flags,
                                    void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  int rc = check_state_slots(p, h_src_slots, h_dst_slots, num_seqs);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  if ((rc = refuse_capture(hs))) return rc;
  MetaSlot *sl = nullptr;
  try {
    std::vector<int32_t> &st = p->stage_tmp;
    st.resize(2 * (size_t)num_seqs);
    std::memcpy(st.data(), h_src_slots ? h_src_slots : h_dst_slots, (size_t)num_seqs * 4);
    std::memcpy(st.data() + num_seqs, h_dst_slots, (size_t)num_seqs * 4);
    if ((rc = stage_cached(p, p->step_cache, st.data(), st.size(), hs, &sl))) return rc;
  } catch (const std::bad_alloc &) {
    return set_error(MKV_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
  rc = mkv_linear_step(pool, layer, d_q, d_k, d_v, d_log_decay, d_o, sl->d, sl->d + num_seqs, num_seqs, scale, flags,
                       stream);
  const int rr = meta_release(sl, hs);
  return rc ? rc : rr;
}
