// The K/V pool in 8 bits: its lifecycle, the steps that write it (append, and
// norm + RoPE + append), read-back and block copies.
//
// All of it streams: what bounds these kernels is memory. Quantising needs the
// largest value of 16 tokens of a head before the first byte, so the unit of work
// is a tile: one wave holds its rows in registers (16 * D / 64 values a lane),
// reduces the maximum over the wave and writes the bytes, 16 a lane in tile
// order. No LDS but for the rotation table, no second pass.
#include "mkv_kv8.h"

namespace mkv {

// ---- append --------------------------------------------------------------------

// Block j of the chunk of sequence s: its id and the rows [o0, o1) that are new,
// the first of them row `row0` of the call. False for an id outside the pool.
__device__ __forceinline__ bool kv8_chunk_block(const Kv8Args &a, const Kv8Seq &s, int j, int32_t &blk, int &o0,
                                                int &o1, int64_t &row0) {
  const int p0 = s.ctx - s.n, first = p0 / kPageSize;
  const int base = (first + j) * kPageSize;
  o0 = max(p0 - base, 0);
  o1 = min(s.ctx - base, kPageSize);
  row0 = (int64_t)s.q0 + (base + o0 - p0);
  blk = ((const kv8_const_i32 *)a.ids)[(int64_t)s.tab0 + first + j];
  return blk >= 0 && blk < a.nblocks;
}

// grid (waves of (block of the chunk, K | V, head) / 4, sequence). The heads of
// one block stand in a workgroup's waves: they read whole rows together. Bound by
// memory: 16 prompts of 700 to 1,300 tokens, 53 MB in 12.3 us (4.3 TB/s); a decode
// step's rows by the chain of loads, 4.8 us.
template <int D, bool F32>
__global__ void __launch_bounds__(256) kv8_append_kernel(Kv8Args a, const uint8_t *__restrict__ k,
                                                         const uint8_t *__restrict__ v, int32_t max_ctx) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Kv8Seq s;
  const uint32_t err = kv8_seq(a, blockIdx.y, max_ctx, s);
  if (err && blockIdx.x == 0 && threadIdx.x == 0) record_error(a.d_err, err);
  if (err || s.n == 0) return;
  const int64_t units = (int64_t)((s.ctx - 1) / kPageSize - (s.ctx - s.n) / kPageSize + 1) * 2 * a.Hkv;
  const int64_t stride = (int64_t)a.Hkv * D * Kv8Row<F32>::ES;
  for (int64_t u = (int64_t)blockIdx.x * 4 + wave; u < units; u += (int64_t)gridDim.x * 4) {
    const int h = (int)(u % a.Hkv), kv = (int)(u / a.Hkv) & 1, j = (int)(u / (2 * a.Hkv));
    int32_t blk;
    int o0, o1;
    int64_t row0;
    if (!kv8_chunk_block(a, s, j, blk, o0, o1, row0)) {
      if (h == 0 && kv == 0 && lane == 0) record_error(a.d_err, MKV_DEVERR_BLOCK);
      continue;
    }
    const int64_t at = (int64_t)blk * a.Hkv + h;
    const int64_t src = row0 * stride + (int64_t)h * D * Kv8Row<F32>::ES;
    if (kv) kv8_write_v<D, F32>(v + src, stride, a.v_tiles + at * 16 * D, a.v_exps + at, lane, o0, o1);
    else kv8_write_k<D, F32>(k + src, stride, a.k_tiles + at * 16 * D, a.k_exps + at, lane, o0, o1);
  }
}

// ---- norm + RoPE + append ---------------------------------------------------------

struct Kv8PrepArgs {
  const uint8_t *q, *k, *v;
  const float *wq, *wk, *inv_freq;
  const int32_t *pos;  // per row, or null
  uint8_t *q_out;
  int32_t rd, q_stride;  // rotary dims; elements from one q head to the next
  int32_t norm, interleaved;
  float eps, factor;
};

// Workgroup = (block of the chunk, sequence, share z of the heads): up to 16
// tokens, whose table of cos and sin (rd/2 pairs each) it forms once in LDS, then
// one wave per head. A lane holds, per pass over the rows, two runs of VEC dims of one
// token that rotate against each other (half layout: dims i.. and i + rd/2..;
// interleaved, and dims that do not rotate: 2 VEC neighbours), so that the
// partner is always in the lane. A K head goes from there into its tile. Bound by
// memory: 32 chunks of 512 tokens, 285 MB in 72 us (4.0 TB/s; 86 us with no head
// loaded ahead). Without the angles it took 71.
// VEC: 8, or 4 where rd/2 (interleaved: rd/2) is not a multiple of 8.
template <int D, int VEC>
struct PrepLane {
  static constexpr int LPT = D / (2 * VEC);  // lanes of a token
  static constexpr int TPP = 64 / LPT;       // tokens of a pass
  static constexpr int NP = 16 / TPP;        // passes
  int tok0, a0, a1, pair;                    // token of pass 0, first dims of both runs, first pair (-1: none)
  __device__ __forceinline__ PrepLane(const Kv8PrepArgs &p, int lane) {
    const int u = lane % LPT, half = p.rd >> 1;
    tok0 = lane / LPT;
    if (p.interleaved) {
      a0 = 2 * u * VEC;
      a1 = a0 + VEC;
      pair = a0 < p.rd ? a0 / 2 : -1;
    } else if (u * VEC < half) {
      a0 = u * VEC;
      a1 = a0 + half;
      pair = a0;
    } else {
      a0 = p.rd + 2 * (u - half / VEC) * VEC;
      a1 = a0 + VEC;
      pair = -1;
    }
  }
};

// Waves of a SIMD that leave the kernel the registers for a head's rows twice.
#define KV8_EU(D, F32) ((D) * ((F32) ? 2 : 1) <= 64 ? 4 : (D) * ((F32) ? 2 : 1) <= 128 ? 3 : (D) * ((F32) ? 2 : 1) <= 256 ? 2 : 1)
// VEC values as they are loaded.
template <bool F32, int VEC>
struct PrepRaw {
  typedef uint32_t type __attribute__((ext_vector_type(F32 ? VEC : VEC / 2)));
  static __device__ __forceinline__ void widen(const type &w, float (&x)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; e++) {
      if constexpr (F32) x[e] = __uint_as_float(w[e]);
      else x[e] = e & 1 ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]);
    }
  }
};

template <int D, bool F32, int VEC>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(KV8_EU(D, F32)))) kv8_prep_kernel(Kv8Args a, Kv8PrepArgs p) {
  typedef Kv8Row<F32> Row;
  typedef PrepLane<D, VEC> Lane;
  constexpr int ES = Row::ES, NP = Lane::NP;
  constexpr int CW = D / 2 + 4;  // (padded: the tokens' rows start in other banks)
  __shared__ __attribute__((aligned(16))) float cs[16][2][CW];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Kv8Seq s;
  const uint32_t err = kv8_seq(a, blockIdx.y, INT32_MAX, s);
  if (err && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) record_error(a.d_err, err);
  if (err || s.n == 0) return;
  const int blocks = (s.ctx - 1) / kPageSize - (s.ctx - s.n) / kPageSize + 1;
  const int64_t kv_stride = (int64_t)a.Hkv * D * ES;
  const Lane ln(p, lane);
  const int half = p.rd >> 1;
  for (int64_t j = blockIdx.x; j < blocks; j += gridDim.x) {
    int32_t blk;
    int o0, o1;
    int64_t row0;
    const bool ok = kv8_chunk_block(a, s, (int)j, blk, o0, o1, row0);
    if (!ok && blockIdx.z == 0 && threadIdx.x == 0) record_error(a.d_err, MKV_DEVERR_BLOCK);
    // The angle in turns, in f64: p * inv_freq reaches millions of turns, of which
    // f32 keeps no fraction (2^-24 of 10^6 radians is 0.06).
    for (int i = threadIdx.x; i < (o1 - o0) * half; i += 256) {
      const int t = i / half, c = i - t * half;
      const int pos = p.pos ? p.pos[row0 + t] : s.ctx - s.n + (int)(row0 - s.q0) + t;
      const double turns = (double)pos * (double)p.inv_freq[c] * 0.15915494309189533577;
      float sn, cn;
      sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cn);
      cs[t][0][c] = cn * p.factor;
      cs[t][1][c] = sn * p.factor;
    }
    __syncthreads();
    // Heads of q and k in turn, the next one's rows loaded before this one is used.
    // Token t of a pass is row o0 + t of the tile; its rows lie at lane offsets of the
    // first one's (32 bits: 16 rows of a call).
    const int n = o1 - o0, by = gridDim.z * 4, heads = a.Hq + a.Hkv;
    typedef typename PrepRaw<F32, VEC>::type raw_t;
    raw_t cur[NP][2], nxt[NP][2];
    const uint8_t *q0 = p.q + row0 * a.Hq * p.q_stride * ES, *k0 = p.k + row0 * kv_stride;
    auto load = [&](int u, raw_t (&r)[NP][2]) {
      const bool is_k = u >= a.Hq;
      const uint8_t *src = is_k ? k0 + (u - a.Hq) * D * ES : q0 + u * p.q_stride * ES;
      const uint32_t stride = (is_k ? a.Hkv * D : a.Hq * p.q_stride) * ES;
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const uint32_t off = (uint32_t)min(ln.tok0 + i * Lane::TPP, n - 1) * stride;
        r[i][0] = *reinterpret_cast<const raw_t *>(src + (off + ln.a0 * ES));
        r[i][1] = *reinterpret_cast<const raw_t *>(src + (off + ln.a1 * ES));
      }
    };
    int u = blockIdx.z * 4 + wave;
    if (u < heads) load(u, cur);
    for (; u < heads; u += by) {
      const bool is_k = u >= a.Hq;
      const int h = is_k ? u - a.Hq : u;
      const float *w = is_k ? p.wk : p.wq;
      if (u + by < heads) load(u + by, nxt);
      float x[NP][2][VEC];
#pragma unroll
      for (int i = 0; i < NP; i++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          PrepRaw<F32, VEC>::widen(cur[i][r], x[i][r]);
          cur[i][r] = nxt[i][r];
        }
      float w0[VEC], w1[VEC];
      if (p.norm) {
        Kv8Row<true>::load(reinterpret_cast<const uint8_t *>(w + ln.a0), w0);
        Kv8Row<true>::load(reinterpret_cast<const uint8_t *>(w + ln.a1), w1);
      }
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int t = min(ln.tok0 + i * Lane::TPP, n - 1);
        if (p.norm) {  // x * (mean(x^2) + eps)^-1/2 * (1 + w)
          float ss = 0.0f;
#pragma unroll
          for (int e = 0; e < VEC; e++) ss += x[i][0][e] * x[i][0][e] + x[i][1][e] * x[i][1][e];
          const float inv = 1.0f / sqrtf(row_sum<Lane::LPT>(ss) / (float)D + p.eps);
#pragma unroll
          for (int e = 0; e < VEC; e++) {
            x[i][0][e] = x[i][0][e] * inv * (1.0f + w0[e]);
            x[i][1][e] = x[i][1][e] * inv * (1.0f + w1[e]);
          }
        }
        if (ln.pair >= 0) {
          float c[VEC], sn[VEC];
#pragma unroll
          for (int e = 0; e < VEC; e += 4) {
            const f32x4 c4 = *reinterpret_cast<const f32x4 *>(&cs[t][0][ln.pair + e]);
            const f32x4 s4 = *reinterpret_cast<const f32x4 *>(&cs[t][1][ln.pair + e]);
#pragma unroll
            for (int z = 0; z < 4; z++) c[e + z] = c4[z], sn[e + z] = s4[z];
          }
          if (p.interleaved) {
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
              for (int e = 0; e < VEC; e += 2) {
                const int z = (r * VEC + e) / 2;
                const float xa = x[i][r][e], xb = x[i][r][e + 1];
                x[i][r][e] = xa * c[z] - xb * sn[z];
                x[i][r][e + 1] = xb * c[z] + xa * sn[z];
              }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
              const float xa = x[i][0][e], xb = x[i][1][e];
              x[i][0][e] = xa * c[e] - xb * sn[e];
              x[i][1][e] = xb * c[e] + xa * sn[e];
            }
          }
        }
        if (is_k) {
#pragma unroll
          for (int e = 0; e < VEC; e++)
            amax = fmaxf(amax, fmaxf(kv8_finite_abs(x[i][0][e]), kv8_finite_abs(x[i][1][e])));
        } else if (ln.tok0 + i * Lane::TPP < n) {
          uint8_t *dst = p.q_out + (row0 * a.Hq + h) * D * ES;
          const uint32_t off = (uint32_t)t * (a.Hq * D * ES);
          Row::store(dst + (off + ln.a0 * ES), x[i][0]);
          Row::store(dst + (off + ln.a1 * ES), x[i][1]);
        }
      }
      if (!is_k || !ok) continue;
      const int64_t at = (int64_t)blk * a.Hkv + h;
      uint8_t *tile = a.k_tiles + at * 16 * D;
      const int e_old = a.k_exps[at];
      amax = wave_max(amax);
      bool grown;
      float f;
      const int e = kv8_new_exp(amax, o0, e_old, grown, f);
      kv8_k_others<D>(tile, lane, o0, o1, grown, f);
      const float inv = kv8_inv(e);
#pragma unroll
      for (int i = 0; i < NP; i++) {
        const int t = ln.tok0 + i * Lane::TPP;
        if (t >= n) continue;
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int d0 = r ? ln.a1 : ln.a0;
          uint32_t w[VEC / 4];
#pragma unroll
          for (int z = 0; z < VEC; z += 4)
            w[z / 4] = kv8_pack4(kv8_down(x[i][r][z], inv), kv8_down(x[i][r][z + 1], inv),
                                 kv8_down(x[i][r][z + 2], inv), kv8_down(x[i][r][z + 3], inv));
          uint8_t *dst = tile + (d0 >> 4) * 256 + (o0 + t) * 16 + (d0 & 15);
          if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
          else *reinterpret_cast<uint32_t *>(dst) = w[0];
        }
      }
      if (lane == 0 && e != e_old) a.k_exps[at] = (int8_t)e;
    }
    if (ok)
      for (; u < heads + a.Hkv; u += by) {
        const int h = u - heads;
        const int64_t at = (int64_t)blk * a.Hkv + h;
        kv8_write_v<D, F32>(p.v + row0 * kv_stride + (int64_t)h * D * ES, kv_stride, a.v_tiles + at * 16 * D,
                            a.v_exps + at, lane, o0, o1);
      }
    __syncthreads();  // the table is written again for the next block
  }
}

// ---- read-back -------------------------------------------------------------------

// grid (waves of (block, K | V, head) / 4, sequence); lane as in the tile order. Bound by
// memory: 64 sequences of 1 to 8k tokens, 973 MB in 196 us, 4.95 TB/s (a copy reaches
// 5.13). Loads past the caches, plain stores: 235 us with stores past them too.
template <int D, bool F32>
__global__ void __launch_bounds__(256) kv8_gather_kernel(Kv8Args a, int32_t max_ctx, uint8_t *__restrict__ out_k,
                                                         uint8_t *__restrict__ out_v, int64_t capacity) {
  typedef Kv8Row<F32> Row;
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ctx = ((const kv8_const_i32 *)a.ctx)[b];
  const kv8_const_i32 *ip = (const kv8_const_i32 *)a.indptr;
  const int tab0 = ip[b];
  const int64_t tabn = a.ids ? (int64_t)ip[b + 1] - tab0 : 0;
  // The token that the sequence starts at: the sum of the lengths before it (as
  // they are: a length that does not fit spoils its own sequence only).
  int64_t c0 = 0;
  for (int i = lane; i < b; i += 64) c0 += max(a.ctx[i], 0);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) c0 += __shfl_xor(c0, o);
  uint32_t err = 0;
  if (ctx < 0 || ctx > max_ctx || c0 + ctx > capacity) err = MKV_DEVERR_CTX;
  else if (ctx && (tab0 < 0 || tabn < ((int64_t)ctx + kPageSize - 1) / kPageSize)) err = MKV_DEVERR_TABLE;
  if (err) {
    if (blockIdx.x == 0 && threadIdx.x == 0) record_error(a.d_err, err);
    return;
  }
  const int64_t units = ((int64_t)ctx + kPageSize - 1) / kPageSize * 2 * a.Hkv;
  for (int64_t u = (int64_t)blockIdx.x * 4 + wave; u < units; u += (int64_t)gridDim.x * 4) {
    const int h = (int)(u % a.Hkv), kv = (int)(u / a.Hkv) & 1, j = (int)(u / (2 * a.Hkv));
    const int32_t blk = ((const kv8_const_i32 *)a.ids)[(int64_t)tab0 + j];
    if (blk < 0 || blk >= a.nblocks) {
      if (lane == 0) record_error(a.d_err, MKV_DEVERR_BLOCK);
      continue;
    }
    const int64_t at = (int64_t)blk * a.Hkv + h;
    const uint8_t *tile = (kv ? a.v_tiles : a.k_tiles) + at * 16 * D;
    u32x4 w[D / 64];
#pragma unroll
    for (int r = 0; r < D / 64; r++)
      w[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(tile + 1024 * r) + lane);
    const float scale = kv8_scale((kv ? a.v_exps : a.k_exps)[at]);
    const int nv = min(kPageSize, ctx - j * kPageSize), lo = lane & 15, hi = lane >> 4;
    const int64_t base = (c0 * a.Hkv + (int64_t)h * ctx + (int64_t)j * kPageSize) * D;
    if (!kv) {
      if (lo >= nv) continue;
#pragma unroll
      for (int r = 0; r < D / 64; r++) {
        float y[16];
#pragma unroll
        for (int z = 0; z < 4; z++) {
          float x[4];
          kv8_unpack4(w[r][z], x);
#pragma unroll
          for (int c = 0; c < 4; c++) y[4 * z + c] = x[c] * scale;
        }
        Row::store(out_k + (base + (int64_t)lo * D + 64 * r + 16 * hi) * Row::ES, y);
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
      float x[4][4];  // [dim][token]
#pragma unroll
      for (int n = 0; n < 4; n++) {
        kv8_unpack4(w[i][n], x[n]);
#pragma unroll
        for (int t = 0; t < 4; t++) x[n][t] *= scale;
      }
      if constexpr (F32) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const float y[4] = {x[0][t], x[1][t], x[2][t], x[3][t]};
          if (4 * hi + t < nv) Row::store(out_v + (base + (int64_t)(4 * hi + t) * D + 64 * i + 4 * lo) * 4, y);
        }
      } else {
        // Two neighbours trade two tokens each for 16-byte stores: the even lane takes
        // tokens 0 and 1 of eight dims, the odd one tokens 2 and 3.
        const bool odd = lane & 1;
        uint32_t p[4][2];
#pragma unroll
        for (int t = 0; t < 4; t++) p[t][0] = pack_bf16x2(x[0][t], x[1][t]), p[t][1] = pack_bf16x2(x[2][t], x[3][t]);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          uint32_t got[2];
#pragma unroll
          for (int z = 0; z < 2; z++)
            got[z] = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? p[t][z] : p[t + 2][z]), 0xb1, 0xf, 0xf, false);
          const int tok = 4 * hi + t + (odd ? 2 : 0);
          const u32x4 y = odd ? u32x4{got[0], got[1], p[t + 2][0], p[t + 2][1]} : u32x4{p[t][0], p[t][1], got[0], got[1]};
          if (tok < nv)
            *reinterpret_cast<u32x4 *>(out_v + (base + (int64_t)tok * D + 64 * i + 4 * (lo & ~1)) * 2) = y;
        }
      }
    }
  }
}

// ---- block copies ------------------------------------------------------------------

// grid (pair, plane = layer * 2 + (K | V)); the exponents by the first lanes.
__global__ void __launch_bounds__(256) kv8_copy_kernel(uint8_t *__restrict__ tiles, int8_t *__restrict__ exps,
                                                       const int32_t *__restrict__ src,
                                                       const int32_t *__restrict__ dst, int64_t nblocks,
                                                       int64_t block_bytes, int32_t Hkv, uint32_t *__restrict__ d_err) {
  constexpr int PER = 4;
  const int32_t s = src[blockIdx.x], d = dst[blockIdx.x];
  if (s < 0 || s >= nblocks || d < 0 || d >= nblocks) {
    if (blockIdx.y == 0 && threadIdx.x == 0) record_error(d_err, MKV_DEVERR_COPY);
    return;
  }
  const int64_t plane = (int64_t)blockIdx.y * nblocks;
  const u32x4 *sp = reinterpret_cast<const u32x4 *>(tiles + (plane + s) * block_bytes);
  u32x4 *dp = reinterpret_cast<u32x4 *>(tiles + (plane + d) * block_bytes);
  const int64_t chunks = block_bytes >> 4;
  for (int64_t base = threadIdx.x; base < chunks; base += 256 * PER) {
    u32x4 r[PER];
#pragma unroll
    for (int u = 0; u < PER; u++) r[u] = __builtin_nontemporal_load(sp + min(base + u * 256, chunks - 1));
#pragma unroll
    for (int u = 0; u < PER; u++)
      if (base + u * 256 < chunks) __builtin_nontemporal_store(r[u], dp + base + u * 256);
  }
  for (int i = threadIdx.x; i < Hkv; i += 256) exps[(plane + d) * Hkv + i] = exps[(plane + s) * Hkv + i];
}

// ---- host side ----------------------------------------------------------------------

int kv8_check_layer(const Kv8Pool *p, int32_t layer) {
  if (layer < 0 || layer >= p->g.L)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "layer %d out of range [0, %d)", layer, p->g.L);
  return MKV_OK;
}

static int kv8_geom(const mkv_pool_desc *d, Geom *g) {
  uint64_t bytes = 0;
  int rc = mkv_pool_required_bytes(d, &bytes);  // the checks of every pool
  if (rc) return rc;
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "an 8-bit pool needs head_dim 64, 128 or 256 (got %d)", d->head_dim);
  g->L = d->num_layers;
  g->Hkv = d->num_kv_heads;
  g->Hq = d->num_q_heads;
  g->D = d->head_dim;
  g->ps = d->page_size;
  g->dtype = d->dtype;
  g->nblocks = d->num_blocks;
  g->es = d->dtype == MKV_DTYPE_F32 ? 4 : 2;
  g->row_bytes = (int64_t)g->Hkv * g->D * g->es;
  g->block_bytes = (int64_t)g->Hkv * 16 * g->D;
  g->plane_bytes = g->nblocks * g->block_bytes;
  return MKV_OK;
}

int kv8_ws_begin(Kv8Pool *p, void *d_ws, uint64_t bytes, hipStream_t hs, Kv8Ws *out) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (d_ws) {
    out->ptr = d_ws;
    out->bytes = bytes;
    out->own = false;
    return MKV_OK;
  }
  out->ptr = p->ws;
  out->bytes = p->ws_bytes;
  MKV_CHECK_HIP(hipStreamIsCapturing(hs, &st));
  out->own = st == hipStreamCaptureStatusNone;
  if (out->own && p->ws_used) MKV_CHECK_HIP(hipStreamWaitEvent(hs, p->ws_done, 0));
  return MKV_OK;
}

int kv8_ws_end(Kv8Pool *p, const Kv8Ws &w, hipStream_t hs) {
  if (!w.own) return MKV_OK;
  MKV_CHECK_HIP(hipEventRecord(p->ws_done, hs));
  p->ws_used = true;
  return MKV_OK;
}

static int stage_checked(Kv8Pool *p, StagedCache &c, const int32_t *h_q_lens, const int32_t *h_ctx,
                         const uint32_t *h_indptr, const uint32_t *h_ids, const int32_t *h_pos, int32_t B, bool write,
                         hipStream_t hs, Kv8Meta *out) {
  const Geom &g = p->g;
  if (B < 0 || B > 65535) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs %d outside [0, 65535]", B);
  if (!h_indptr || !h_ctx) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL indptr or lengths");
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  MKV_CHECK_HIP(hipStreamIsCapturing(hs, &st));
  if (st != hipStreamCaptureStatusNone)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "host metadata cannot be captured into a graph: use the device form");
  if (h_indptr[0] != 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "block_indptr[0] = %u, expected 0", h_indptr[0]);
  for (int32_t b = 0; b < B; b++)
    if (h_indptr[b + 1] < h_indptr[b])
      return set_error(MKV_ERR_INVALID_ARGUMENT, "block_indptr not monotone at %d", b);
  if (h_indptr[B] > (uint32_t)INT32_MAX) return set_error(MKV_ERR_INVALID_ARGUMENT, "more than 2^31 - 1 block ids");
  const size_t nids = h_indptr[B];
  if (nids && !h_ids) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL block ids");
  int64_t tokens = 0, total = 0;
  int32_t max_q = 0, max_ctx = 0;
  for (int32_t b = 0; b < B; b++) {
    const int32_t n = h_q_lens ? h_q_lens[b] : 1, ctx = h_ctx[b];
    if (ctx < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "length[%d] = %d < 0", b, ctx);
    if (h_q_lens && (n < 0 || n > ctx))
      return set_error(MKV_ERR_INVALID_ARGUMENT, "sequence %d: %d new tokens outside [0, ctx %d]", b, n, ctx);
    tokens += n;
    total += ctx;
    max_q = std::max(max_q, n);
    max_ctx = std::max(max_ctx, ctx);
  }
  if (tokens > INT32_MAX || total > INT32_MAX) return set_error(MKV_ERR_INVALID_ARGUMENT, "more than 2^31 - 1 tokens");
  const size_t nx = h_pos ? (size_t)tokens : 0;
  // (The last three say how the rest is read: equal arrays are equal calls.)
  const size_t n = 3 * (size_t)B + 2 + nx + nids + 3;
  std::vector<int32_t> &t = p->stage_tmp;
  t.resize(n);
  int32_t *qi = t.data(), *ip = qi + B + 1, *cl = ip + B + 1, *ex = cl + B, *ix = ex + nx;
  qi[0] = 0;
  for (int32_t b = 0; b < B; b++) qi[b + 1] = qi[b] + (h_q_lens ? h_q_lens[b] : 1);
  for (int32_t b = 0; b <= B; b++) ip[b] = (int32_t)h_indptr[b];
  if (B) std::memcpy(cl, h_ctx, (size_t)B * 4);
  if (nx) std::memcpy(ex, h_pos, nx * 4);
  if (nids) std::memcpy(ix, h_ids, nids * 4);
  t[n - 3] = B;
  t[n - 2] = (int32_t)nx;
  t[n - 1] = write;
  const bool seen = c.vals.size() == n && std::memcmp(c.vals.data(), t.data(), n * 4) == 0;
  if (!seen) {
    for (size_t i = 0; i < nx; i++)
      if (h_pos[i] < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "position[%zu] = %d < 0", i, h_pos[i]);
    for (int32_t b = 0; b < B; b++) {
      const uint32_t need = (uint32_t)(((int64_t)h_ctx[b] + kPageSize - 1) / kPageSize);
      if (h_indptr[b + 1] - h_indptr[b] < need)
        return set_error(MKV_ERR_INVALID_ARGUMENT, "sequence %d: %u blocks cannot hold %d tokens", b,
                         h_indptr[b + 1] - h_indptr[b], h_ctx[b]);
      for (uint32_t i = h_indptr[b]; i < h_indptr[b] + need; i++)
        if (h_ids[i] >= (uint64_t)g.nblocks)
          return set_error(MKV_ERR_INVALID_ARGUMENT, "sequence %d: block id %u (table entry %u) outside the pool of %lld",
                           b, h_ids[i], i - h_indptr[b], (long long)g.nblocks);
    }
    if (write) {
      // owner[block]: this call's number, then the sequence that writes the block. Entries of
      // other calls count as none, so that a call costs what it names and not the pool.
      if (p->owner.empty() || ++p->calls == 0) {
        p->owner.assign((size_t)g.nblocks, 0);
        p->calls = 1;
      }
      const uint64_t tag = (uint64_t)p->calls << 32;
      auto writer = [&](uint32_t id) {  // the sequence, or -1
        const uint64_t o = p->owner[id];
        return o >> 32 == p->calls ? (int32_t)(uint32_t)o : -1;
      };
      for (int32_t b = 0; b < B; b++) {
        const int32_t nq = qi[b + 1] - qi[b];
        if (nq == 0 || h_ctx[b] == 0) continue;
        for (int32_t j = (h_ctx[b] - nq) / kPageSize; j <= (h_ctx[b] - 1) / kPageSize; j++) {
          const uint32_t id = h_ids[h_indptr[b] + j];
          if (writer(id) >= 0)
            return set_error(MKV_ERR_INVALID_ARGUMENT, "block %u would be written twice (sequences %d and %d)", id,
                             writer(id), b);
          p->owner[id] = tag | (uint32_t)b;
        }
      }
      for (int32_t b = 0; b < B; b++) {
        const uint32_t need = (uint32_t)(((int64_t)h_ctx[b] + kPageSize - 1) / kPageSize);
        const int32_t nq = qi[b + 1] - qi[b];
        for (uint32_t j = 0; j < need; j++) {
          const int32_t o = writer(h_ids[h_indptr[b] + j]);
          const bool own = nq && o == b && (int32_t)j >= (h_ctx[b] - nq) / kPageSize;
          if (o >= 0 && !own)
            return set_error(MKV_ERR_INVALID_ARGUMENT, "block %u is written by sequence %d and in another part (of sequence %d)",
                             h_ids[h_indptr[b] + j], o, b);
        }
      }
    }
  }
  int rc = stage_cached(p, c, t.data(), n, hs, &out->slot);
  if (rc) return rc;
  const int32_t *d = out->slot->d;
  out->q_indptr = d;
  out->indptr = d + B + 1;
  out->ctx = d + 2 * (B + 1);
  out->pos = out->ctx + B;
  out->ids = out->pos + nx;
  out->max_q = max_q;
  out->max_ctx = max_ctx;
  out->tokens = (int32_t)tokens;
  return MKV_OK;
}

int kv8_stage(Kv8Pool *p, StagedCache &c, const int32_t *h_q_lens, const int32_t *h_ctx, const uint32_t *h_indptr,
              const uint32_t *h_ids, const int32_t *h_pos, int32_t B, bool write, hipStream_t hs, Kv8Meta *out) {
  try {
    return stage_checked(p, c, h_q_lens, h_ctx, h_indptr, h_ids, h_pos, B, write, hs, out);
  } catch (const std::bad_alloc &) {
    c.slot = -1;
    c.vals.clear();
    return set_error(MKV_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
}

Kv8Args kv8_args(const Kv8Pool *p, int32_t layer, const int32_t *q_indptr, const int32_t *indptr,
                        const int32_t *ids, const int32_t *ctx, int32_t B, int32_t tokens) {
  const Geom &g = p->g;
  Kv8Args a;
  a.k_tiles = p->tiles + (int64_t)layer * 2 * g.plane_bytes;
  a.v_tiles = a.k_tiles + g.plane_bytes;
  a.k_exps = p->exps + (int64_t)layer * 2 * kv8_exp_plane(g);
  a.v_exps = a.k_exps + kv8_exp_plane(g);
  a.q_indptr = q_indptr;
  a.indptr = indptr;
  a.ids = ids;
  a.ctx = ctx;
  a.d_err = p->d_err;
  a.nblocks = g.nblocks;
  a.B = B;
  a.Hq = g.Hq;
  a.Hkv = g.Hkv;
  a.G = g.Hq / g.Hkv;
  a.tokens = tokens;
  return a;
}

// Blocks that a chunk of n tokens can touch.
static int64_t kv8_chunk_blocks(int32_t n) { return ((int64_t)n + 14) / kPageSize + 1; }

#define KV8_DISPATCH(KERNEL, GRID, STREAM, ...)                                                               \
  do {                                                                                                        \
    const bool f32 = g.dtype == MKV_DTYPE_F32;                                                                \
    switch (g.D) {                                                                                            \
      case 64: if (f32) hipLaunchKernelGGL((KERNEL<64, true>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);       \
               else hipLaunchKernelGGL((KERNEL<64, false>), GRID, dim3(256), 0, STREAM, __VA_ARGS__); break;   \
      case 128: if (f32) hipLaunchKernelGGL((KERNEL<128, true>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);     \
                else hipLaunchKernelGGL((KERNEL<128, false>), GRID, dim3(256), 0, STREAM, __VA_ARGS__); break; \
      default: if (f32) hipLaunchKernelGGL((KERNEL<256, true>), GRID, dim3(256), 0, STREAM, __VA_ARGS__);      \
               else hipLaunchKernelGGL((KERNEL<256, false>), GRID, dim3(256), 0, STREAM, __VA_ARGS__); break;  \
    }                                                                                                         \
  } while (0)

int kv8_append_rows(const Kv8Pool *p, const Kv8Args &a, const void *d_k, const void *d_v, int32_t max_ctx,
                    hipStream_t hs) {
  const Geom &g = p->g;
  KV8_DISPATCH(kv8_append_kernel, dim3((2 * g.Hkv + 3) / 4, a.B), hs, a, static_cast<const uint8_t *>(d_k),
               static_cast<const uint8_t *>(d_v), max_ctx);
  MKV_CHECK_LAUNCH("kv8_append_kernel");
  return MKV_OK;
}

static int kv8_check_batch(int32_t B, int32_t tokens, int32_t max_q) {
  if (B < 0 || B > 65535) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs %d outside [0, 65535]", B);
  if (tokens < 0 || max_q < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "negative sizes");
  return MKV_OK;
}

}  // namespace mkv

using namespace mkv;

// ---- C ABI: pool -----------------------------------------------------------------------

extern "C" int mkv_kv8_required_bytes(const mkv_pool_desc *desc, uint64_t *out_tile_bytes,
                                      uint64_t *out_exponent_bytes) {
  Geom g;
  int rc = kv8_geom(desc, &g);
  if (rc) return rc;
  if (!out_tile_bytes || !out_exponent_bytes) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL argument");
  *out_tile_bytes = (uint64_t)2 * g.L * (uint64_t)g.plane_bytes;
  *out_exponent_bytes = (uint64_t)2 * g.L * (uint64_t)kv8_exp_plane(g);
  return MKV_OK;
}

extern "C" int mkv_kv8_pool_create(const mkv_pool_desc *desc, int device, mkv_kv8_pool **out_pool) {
  Geom g;
  int rc = kv8_geom(desc, &g);
  if (rc) return rc;
  if (!out_pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "out_pool is NULL");
  *out_pool = nullptr;
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0) {
    (void)hipGetLastError();
    return set_error(MKV_ERR_NO_DEVICE, "no HIP device available");
  }
  if (device < 0 || device >= ndev)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "device %d out of range (%d devices)", device, ndev);
  DeviceGuard guard(device);
  if (!guard.ok) return set_error(MKV_ERR_HIP, "hipSetDevice(%d) failed", device);
  Kv8Pool *p = new (std::nothrow) Kv8Pool();
  if (!p) return set_error(MKV_ERR_OUT_OF_MEMORY, "host allocation failed");
  p->desc = *desc;
  p->g = g;
  p->device = device;
  p->tile_bytes = (uint64_t)2 * g.L * (uint64_t)g.plane_bytes;
  p->exp_bytes = (uint64_t)2 * g.L * (uint64_t)kv8_exp_plane(g);
  hipError_t e = hipMalloc(reinterpret_cast<void **>(&p->tiles), p->tile_bytes);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&p->exps), p->exp_bytes);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&p->cus, hipDeviceAttributeMultiprocessorCount, device);
  p->ws_bytes = std::max(kKv8Workspace, kv8_piece_bytes(g, kv8_most_pieces(g, p->cus)));
  if (e == hipSuccess) e = hipMalloc(&p->ws, p->ws_bytes);
  if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void **>(&p->d_err), 256);
  if (e == hipSuccess) e = hipMemset(p->d_err, 0, 256);
  if (e == hipSuccess) e = hipEventCreateWithFlags(&p->ws_done, hipEventDisableTiming);
  if (e != hipSuccess) {
    mkv_kv8_pool_destroy(reinterpret_cast<mkv_kv8_pool *>(p));
    return hip_fail(e, "8-bit pool allocation");
  }
  *out_pool = reinterpret_cast<mkv_kv8_pool *>(p);
  return MKV_OK;
}

extern "C" int mkv_kv8_pool_destroy(mkv_kv8_pool *pool) {
  if (!pool) return MKV_OK;
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  DeviceGuard guard(p->device);
  (void)hipDeviceSynchronize();
  meta_free(p);
  if (p->ws_done) (void)hipEventDestroy(p->ws_done);
  if (p->d_err) (void)hipFree(p->d_err);
  if (p->ws) (void)hipFree(p->ws);
  if (p->exps) (void)hipFree(p->exps);
  if (p->tiles) (void)hipFree(p->tiles);
  delete p;
  return MKV_OK;
}

extern "C" int mkv_kv8_pool_get_desc(const mkv_kv8_pool *pool, mkv_pool_desc *out_desc) {
  if (!pool || !out_desc) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL argument");
  *out_desc = reinterpret_cast<const Kv8Pool *>(pool)->desc;
  return MKV_OK;
}

extern "C" int mkv_kv8_pool_buffers(const mkv_kv8_pool *pool, void **out_tiles, uint64_t *out_tile_bytes,
                                    void **out_exponents, uint64_t *out_exponent_bytes) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  const Kv8Pool *p = reinterpret_cast<const Kv8Pool *>(pool);
  if (out_tiles) *out_tiles = p->tiles;
  if (out_tile_bytes) *out_tile_bytes = p->tile_bytes;
  if (out_exponents) *out_exponents = p->exps;
  if (out_exponent_bytes) *out_exponent_bytes = p->exp_bytes;
  return MKV_OK;
}

extern "C" int mkv_kv8_pool_check(mkv_kv8_pool *pool, void *stream, uint32_t *out_bits) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  DeviceGuard guard(p->device);
  uint32_t bits = 0;
  MKV_CHECK_HIP(hipStreamSynchronize(reinterpret_cast<hipStream_t>(stream)));
  MKV_CHECK_HIP(hipMemcpy(&bits, p->d_err, sizeof(bits), hipMemcpyDeviceToHost));
  if (bits) MKV_CHECK_HIP(hipMemset(p->d_err, 0, sizeof(bits)));
  if (out_bits) *out_bits = bits;
  if (bits) return set_error(MKV_ERR_DEVICE_INDEX, "kernel met out-of-range ids (error bits 0x%x)", bits);
  return MKV_OK;
}

extern "C" int mkv_kv8_workspace_size(const mkv_kv8_pool *pool, uint64_t *out_bytes) {
  if (!pool || !out_bytes) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL argument");
  *out_bytes = reinterpret_cast<const Kv8Pool *>(pool)->ws_bytes;
  return MKV_OK;
}

// ---- C ABI: append -----------------------------------------------------------------------

extern "C" int mkv_kv8_append(mkv_kv8_pool *pool, int32_t layer, const void *d_k, const void *d_v,
                              const int32_t *d_q_indptr, const int32_t *d_block_indptr, const int32_t *d_block_ids,
                              const int32_t *d_ctx_lens, int32_t num_seqs, int32_t num_tokens, int32_t max_q_len,
                              void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  const Geom &g = p->g;
  int rc = kv8_check_layer(p, layer);
  if (rc || (rc = kv8_check_batch(num_seqs, num_tokens, max_q_len))) return rc;
  if (num_seqs == 0 || num_tokens == 0 || max_q_len == 0) return MKV_OK;
  if (!d_k || !d_v || !d_q_indptr || !d_block_indptr || !d_ctx_lens)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(d_k) || !aligned16(d_v))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "K/V rows must be 16-byte aligned");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  const Kv8Args a = kv8_args(p, layer, d_q_indptr, d_block_indptr, d_block_ids, d_ctx_lens, num_seqs, num_tokens);
  const int64_t wgs = (kv8_chunk_blocks(std::min(max_q_len, num_tokens)) * 2 * g.Hkv + 3) / 4;
  const dim3 grid((unsigned)std::min<int64_t>(wgs, 1 << 20), (unsigned)num_seqs);
  KV8_DISPATCH(kv8_append_kernel, grid, hs, a, static_cast<const uint8_t *>(d_k), static_cast<const uint8_t *>(d_v),
               INT32_MAX);
  MKV_CHECK_LAUNCH("kv8_append_kernel");
  return MKV_OK;
}

extern "C" int mkv_kv8_append_host(mkv_kv8_pool *pool, int32_t layer, const void *d_k, const void *d_v,
                                   const int32_t *h_q_lens, const int32_t *h_ctx_lens, const uint32_t *h_block_indptr,
                                   const uint32_t *h_block_ids, int32_t num_seqs, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  int rc = kv8_check_layer(p, layer);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  if (!h_q_lens) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL q_lens");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  Kv8Meta m;
  if ((rc = kv8_stage(p, p->app_cache, h_q_lens, h_ctx_lens, h_block_indptr, h_block_ids, nullptr, num_seqs, true, hs,
                      &m)))
    return rc;
  rc = mkv_kv8_append(pool, layer, d_k, d_v, m.q_indptr, m.indptr, m.ids, m.ctx, num_seqs, m.tokens, m.max_q, stream);
  const int rr = meta_release(m.slot, hs);
  return rc ? rc : rr;
}

extern "C" int mkv_kv8_qk_norm_rope_append(mkv_kv8_pool *pool, int32_t layer, const void *d_q, const void *d_k,
                                           const void *d_v, const float *d_q_norm_w, const float *d_k_norm_w,
                                           const float *d_inv_freq, int32_t rotary_dim, float eps, float rope_factor,
                                           const int32_t *d_positions, const int32_t *d_q_indptr,
                                           const int32_t *d_block_indptr, const int32_t *d_block_ids,
                                           const int32_t *d_ctx_lens, int32_t num_seqs, int32_t num_tokens,
                                           int32_t max_q_len, void *d_q_out, uint32_t flags, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  const Geom &g = p->g;
  int rc = kv8_check_layer(p, layer);
  if (rc || (rc = kv8_check_batch(num_seqs, num_tokens, max_q_len))) return rc;
  if (flags & ~(uint32_t)(MKV_PREP_PLAIN_Q | MKV_PREP_NO_NORM | MKV_PREP_INTERLEAVED))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
  const bool norm = !(flags & MKV_PREP_NO_NORM), plain = flags & MKV_PREP_PLAIN_Q;
  if (rotary_dim < 0 || rotary_dim > g.D || rotary_dim % 8)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "rotary_dim %d must be a multiple of 8 in [0, %d]", rotary_dim, g.D);
  if (norm && !(eps >= 0.0f && eps < INFINITY))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  if (!std::isfinite(rope_factor)) return set_error(MKV_ERR_INVALID_ARGUMENT, "rope_factor must be finite");
  if (num_seqs == 0 || num_tokens == 0 || max_q_len == 0) return MKV_OK;
  if (!d_q || !d_k || !d_v || !d_q_out || !d_q_indptr || !d_block_indptr || !d_ctx_lens ||
      (norm && (!d_q_norm_w || !d_k_norm_w)) || (rotary_dim > 0 && !d_inv_freq))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(d_q) || !aligned16(d_k) || !aligned16(d_v) || !aligned16(d_q_out) ||
      (norm && (!aligned16(d_q_norm_w) || !aligned16(d_k_norm_w))))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "q, k, v, q_out and the norm weights must be 16-byte aligned");
  const uint64_t qn = (uint64_t)num_tokens * g.Hq * g.D * g.es, kn = (uint64_t)num_tokens * g.row_bytes;
  if ((overlap(d_q_out, qn, d_q, plain ? qn : 2 * qn) && !(plain && d_q_out == d_q)) || overlap(d_q_out, qn, d_k, kn) ||
      overlap(d_q_out, qn, d_v, kn))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "q_out overlaps q, k or v");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  const Kv8Args a = kv8_args(p, layer, d_q_indptr, d_block_indptr, d_block_ids, d_ctx_lens, num_seqs, num_tokens);
  Kv8PrepArgs r;
  r.q = static_cast<const uint8_t *>(d_q);
  r.k = static_cast<const uint8_t *>(d_k);
  r.v = static_cast<const uint8_t *>(d_v);
  r.wq = d_q_norm_w;
  r.wk = d_k_norm_w;
  r.inv_freq = d_inv_freq;
  r.pos = d_positions;
  r.q_out = static_cast<uint8_t *>(d_q_out);
  r.rd = rotary_dim;
  r.q_stride = plain ? g.D : 2 * g.D;
  r.norm = norm;
  r.interleaved = (flags & MKV_PREP_INTERLEAVED) ? 1 : 0;
  r.eps = eps;
  r.factor = rope_factor;
  const int64_t blocks = std::min<int64_t>(kv8_chunk_blocks(std::min(max_q_len, num_tokens)), 1 << 20);
  // The heads of a block are dealt to several workgroups, for 8 of them a CU: a decode
  // step's waves each take one head or two (32 chunks of 512 tokens: 73 us, with 4 a CU
  // 82, although each forms the angles again).
  const int64_t units = g.Hq + 2 * g.Hkv, wgs = blocks * num_seqs;
  const int64_t z = std::max<int64_t>(1, std::min<int64_t>((units + 3) / 4, (8 * p->cus + wgs - 1) / wgs));
  const dim3 grid((unsigned)blocks, (unsigned)num_seqs, (unsigned)z);
#define KV8_PREP(DD, FF)                                                                                     \
  do {                                                                                                       \
    if (rotary_dim % 16 == 0) hipLaunchKernelGGL((kv8_prep_kernel<DD, FF, 8>), grid, dim3(256), 0, hs, a, r); \
    else hipLaunchKernelGGL((kv8_prep_kernel<DD, FF, 4>), grid, dim3(256), 0, hs, a, r);                      \
  } while (0)
  const bool f32 = g.dtype == MKV_DTYPE_F32;
  switch (g.D) {
    case 64: if (f32) KV8_PREP(64, true); else KV8_PREP(64, false); break;
    case 128: if (f32) KV8_PREP(128, true); else KV8_PREP(128, false); break;
    default: if (f32) KV8_PREP(256, true); else KV8_PREP(256, false); break;
  }
#undef KV8_PREP
  MKV_CHECK_LAUNCH("kv8_prep_kernel");
  return MKV_OK;
}

extern "C" int mkv_kv8_qk_norm_rope_append_host(mkv_kv8_pool *pool, int32_t layer, const void *d_q, const void *d_k,
                                                const void *d_v, const float *d_q_norm_w, const float *d_k_norm_w,
                                                const float *d_inv_freq, int32_t rotary_dim, float eps,
                                                float rope_factor, const int32_t *h_positions, const int32_t *h_q_lens,
                                                const int32_t *h_ctx_lens, const uint32_t *h_block_indptr,
                                                const uint32_t *h_block_ids, int32_t num_seqs, void *d_q_out,
                                                uint32_t flags, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  int rc = kv8_check_layer(p, layer);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  if (!h_q_lens) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL q_lens");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  Kv8Meta m;
  if ((rc = kv8_stage(p, p->app_cache, h_q_lens, h_ctx_lens, h_block_indptr, h_block_ids, h_positions, num_seqs, true, hs,
                      &m)))
    return rc;
  rc = mkv_kv8_qk_norm_rope_append(pool, layer, d_q, d_k, d_v, d_q_norm_w, d_k_norm_w, d_inv_freq, rotary_dim, eps,
                                   rope_factor, h_positions ? m.pos : nullptr, m.q_indptr, m.indptr, m.ids, m.ctx,
                                   num_seqs, m.tokens, m.max_q, d_q_out, flags, stream);
  const int rr = meta_release(m.slot, hs);
  return rc ? rc : rr;
}

// ---- C ABI: read-back and copies ------------------------------------------------------------

extern "C" int mkv_kv8_gather(mkv_kv8_pool *pool, int32_t layer, const int32_t *d_block_indptr,
                              const int32_t *d_block_ids, const int32_t *d_ctx_lens, int32_t num_seqs,
                              int32_t max_ctx_len, void *d_out_k, void *d_out_v, int64_t out_capacity_tokens,
                              void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  const Geom &g = p->g;
  int rc = kv8_check_layer(p, layer);
  if (rc) return rc;
  if (num_seqs < 0 || num_seqs > 65535 || max_ctx_len < 0 || out_capacity_tokens < 0)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs outside [0, 65535], or negative sizes");
  if (num_seqs == 0 || max_ctx_len == 0) return MKV_OK;
  if (!d_block_indptr || !d_ctx_lens || !d_out_k || !d_out_v)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(d_out_k) || !aligned16(d_out_v))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "gather outputs must be 16-byte aligned");
  const uint64_t out_bytes = (uint64_t)out_capacity_tokens * g.row_bytes;
  if (overlap(d_out_k, out_bytes, d_out_v, out_bytes))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "gather outputs overlap");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  const Kv8Args a = kv8_args(p, layer, nullptr, d_block_indptr, d_block_ids, d_ctx_lens, num_seqs, 0);
  const int64_t units = ((int64_t)max_ctx_len + kPageSize - 1) / kPageSize * 2 * g.Hkv;
  const dim3 grid((unsigned)std::min<int64_t>((units + 3) / 4, 1 << 20), (unsigned)num_seqs);
  KV8_DISPATCH(kv8_gather_kernel, grid, hs, a, max_ctx_len, static_cast<uint8_t *>(d_out_k),
               static_cast<uint8_t *>(d_out_v), out_capacity_tokens);
  MKV_CHECK_LAUNCH("kv8_gather_kernel");
  return MKV_OK;
}

extern "C" int mkv_kv8_gather_host(mkv_kv8_pool *pool, int32_t layer, const uint32_t *h_block_indptr,
                                   const uint32_t *h_block_ids, const int32_t *h_ctx_lens, int32_t num_seqs,
                                   void *d_out_k, void *d_out_v, int64_t out_capacity_tokens, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  int rc = kv8_check_layer(p, layer);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  if (num_seqs > 0 && h_ctx_lens) {
    int64_t tokens = 0;
    for (int32_t b = 0; b < num_seqs; b++) tokens += std::max(h_ctx_lens[b], 0);
    if (tokens > out_capacity_tokens)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "outputs hold %lld tokens, the tables give %lld",
                       (long long)out_capacity_tokens, (long long)tokens);
  }
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  Kv8Meta m;
  if ((rc = kv8_stage(p, p->gather_cache, nullptr, h_ctx_lens, h_block_indptr, h_block_ids, nullptr, num_seqs, false, hs,
                      &m)))
    return rc;
  rc = mkv_kv8_gather(pool, layer, m.indptr, m.ids, m.ctx, num_seqs, m.max_ctx, d_out_k, d_out_v, out_capacity_tokens,
                      stream);
  const int rr = meta_release(m.slot, hs);
  return rc ? rc : rr;
}

extern "C" int mkv_kv8_copy_blocks(mkv_kv8_pool *pool, const int32_t *d_src_blocks, const int32_t *d_dst_blocks,
                                   int32_t num_pairs, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  if (num_pairs < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_pairs < 0");
  if (num_pairs == 0) return MKV_OK;
  if (!d_src_blocks || !d_dst_blocks) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (2 * (int64_t)p->g.L > 65535) return set_error(MKV_ERR_INVALID_ARGUMENT, "too many layers");
  DeviceGuard guard(p->device);
  hipLaunchKernelGGL(kv8_copy_kernel, dim3(num_pairs, 2 * p->g.L), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                     p->tiles, p->exps, d_src_blocks, d_dst_blocks, p->g.nblocks, p->g.block_bytes, p->g.Hkv, p->d_err);
  MKV_CHECK_LAUNCH("kv8_copy_kernel");
  return MKV_OK;
}

extern "C" int mkv_kv8_copy_blocks_host(mkv_kv8_pool *pool, const uint32_t *h_src_blocks, const uint32_t *h_dst_blocks,
                                        int32_t num_pairs, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  if (num_pairs < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "num_pairs < 0");
  if (num_pairs == 0) return MKV_OK;
  if (!h_src_blocks || !h_dst_blocks) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL block arrays");
  for (int32_t i = 0; i < num_pairs; i++)
    if (h_src_blocks[i] >= (uint64_t)p->g.nblocks || h_dst_blocks[i] >= (uint64_t)p->g.nblocks)
      return set_error(MKV_ERR_INVALID_ARGUMENT, "pair %d (%u -> %u) outside the pool of %lld blocks", i,
                       h_src_blocks[i], h_dst_blocks[i], (long long)p->g.nblocks);
  int rc = mkv_validate_copy_pairs(&p->desc, reinterpret_cast<const int32_t *>(h_src_blocks),
                                   reinterpret_cast<const int32_t *>(h_dst_blocks), num_pairs);
  if (rc) return rc;
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  MKV_CHECK_HIP(hipStreamIsCapturing(hs, &st));
  if (st != hipStreamCaptureStatusNone)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "host metadata cannot be captured into a graph: use the device form");
  MetaSlot *sl = nullptr;
  if ((rc = meta_acquire(p, 2 * (size_t)num_pairs, hs, &sl))) return rc;
  std::memcpy(sl->h, h_src_blocks, (size_t)num_pairs * 4);
  std::memcpy(sl->h + num_pairs, h_dst_blocks, (size_t)num_pairs * 4);
  if ((rc = meta_upload(sl, 2 * (size_t)num_pairs, hs))) return rc;
  rc = mkv_kv8_copy_blocks(pool, sl->d, sl->d + num_pairs, num_pairs, stream);
  const int rr = meta_release(sl, hs);
  return rc ? rc : rr;
}
