// The K/V pool in 8 bits: declarations and device helpers shared by its
// translation units.
//
// A tile holds 16 tokens of one KV head, K or V, as 16 * D e4m3 bytes; one int8
// exponent e per tile, a byte stands for its value times 2^e. The tile order is
// that of the matrix operands (lane = 16 * g4 + m16 of a wave):
//   K [D/16][16 tok][16 dim]: load r (1 KiB of the tile, 16 bytes a lane) gives the lane
//     token m16, dims 64r + 16 g4 .. +16: two A operands of S^T = K.Q^T (16x16x32),
//     whose k-slots are those dims;
//   V [D/64][4 tok quads][16 dim quads][4 dim][4 tok]: load i gives the lane tokens
//     4 g4 .. +4 of dims 64i + 4 m16 .. +4, where S^T leaves the weights of
//     those tokens: four A operands of O^T = V^T.P^T, one dword each and block.
// So a lane takes both straight from memory, each load instruction one
// contiguous KiB, with no transpose and no LDS.
#pragma once

#include "mkv_attn.h"

namespace mkv {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));

constexpr int kKv8MinExp = -100;
constexpr uint64_t kKv8Workspace = 64ull << 20;  // bytes of a pool's own workspace, at least
// Waves of a split decode launch.
constexpr int kSplitWavesPerCu = 8;

struct Kv8Pool : MetaRing {
  mkv_pool_desc desc;
  Geom g;  // es, row_bytes: of the rows; block_bytes, plane_bytes: of the tiles
  int device = 0;
  int cus = 256;
  uint8_t *tiles = nullptr;
  int8_t *exps = nullptr;
  uint64_t tile_bytes = 0, exp_bytes = 0;
  uint32_t *d_err = nullptr;
  void *ws = nullptr;  // ws_bytes, allocated with the pool
  uint64_t ws_bytes = 0;
  hipEvent_t ws_done = nullptr;
  bool ws_used = false;
  // The last host arrays of each kind of call.
  StagedCache app_cache, gather_cache, decode_cache, extend_cache;
  std::vector<int32_t> stage_tmp;
  // Per block, the last call of those that checked one that writes it, and the sequence.
  std::vector<uint64_t> owner;
  uint32_t calls = 0;
};

inline int64_t kv8_exp_plane(const Geom &g) { return g.nblocks * g.Hkv; }

// Pieces of a split decode launch, at most, and the workspace of n pieces: two partials each.
inline int64_t kv8_most_pieces(const Geom &g, int cus) {
  return std::max<int64_t>(1, (int64_t)cus * kSplitWavesPerCu / ((int64_t)g.Hkv * ((g.Hq / g.Hkv + 15) / 16)));
}
inline uint64_t kv8_piece_bytes(const Geom &g, int64_t n) { return 256 + (uint64_t)n * 2 * g.Hq * (8 + 4 * g.D); }

int kv8_check_layer(const Kv8Pool *p, int32_t layer);

// A call's hold on a workspace: the caller's, or the pool's own, whose calls
// follow one another across streams (outside captures).
struct Kv8Ws {
  void *ptr = nullptr;
  uint64_t bytes = 0;
  bool own = false;
};
int kv8_ws_begin(Kv8Pool *p, void *d_ws, uint64_t bytes, hipStream_t hs, Kv8Ws *out);
int kv8_ws_end(Kv8Pool *p, const Kv8Ws &w, hipStream_t hs);

// Host metadata of a call (null q_lens: one new row per sequence; null positions:
// none), checked and staged as q_indptr[B+1] | indptr[B+1] | ctx[B] | positions |
// ids. Arrays equal to the previous call's of the same kind are not checked
// again, nor uploaded again on the same stream. write: a block that new rows go
// to must be in no other place of the call's tables.
struct Kv8Meta {
  MetaSlot *slot = nullptr;
  const int32_t *q_indptr, *indptr, *ctx, *pos, *ids;
  int32_t max_q, max_ctx, tokens;
};
int kv8_stage(Kv8Pool *p, StagedCache &c, const int32_t *h_q_lens, const int32_t *h_ctx, const uint32_t *h_indptr,
              const uint32_t *h_ids, const int32_t *h_pos, int32_t B, bool write, hipStream_t hs, Kv8Meta *out);

// ---- device side --------------------------------------------------------------

// The planes of one layer and the tables of a call.
struct Kv8Args {
  uint8_t *k_tiles, *v_tiles;
  int8_t *k_exps, *v_exps;  // [blocks][Hkv]
  const int32_t *q_indptr, *indptr, *ids, *ctx;  // ids null: no table holds a block
  uint32_t *d_err;
  int64_t nblocks;
  int32_t B, Hq, Hkv, G, tokens;
};

Kv8Args kv8_args(const Kv8Pool *p, int32_t layer, const int32_t *q_indptr, const int32_t *indptr, const int32_t *ids,
                 const int32_t *ctx, int32_t B, int32_t tokens);

// One new row per sequence at position ctx - 1 (a without q_indptr).
int kv8_append_rows(const Kv8Pool *p, const Kv8Args &a, const void *d_k, const void *d_v, int32_t max_ctx,
                    hipStream_t hs);

// A sequence's numbers, checked: n new rows at row q0, ctx tokens, table at
// tab0. False (and reported by the caller's choice of thread) if they do not fit.
struct Kv8Seq {
  int q0, n, ctx, tab0;
};
typedef const __attribute__((address_space(4))) int32_t kv8_const_i32;

__device__ __forceinline__ uint32_t kv8_seq(const Kv8Args &a, int b, int32_t max_ctx, Kv8Seq &s) {
  const kv8_const_i32 *qi = (const kv8_const_i32 *)a.q_indptr, *ip = (const kv8_const_i32 *)a.indptr;
  s.ctx = ((const kv8_const_i32 *)a.ctx)[b];
  s.q0 = qi ? qi[b] : b;
  const int q1 = qi ? qi[b + 1] : b + (s.ctx > 0);  // (no indptr: one row each, none for padding)
  s.tab0 = ip[b];
  const int64_t tabn = a.ids ? (int64_t)ip[b + 1] - s.tab0 : 0;
  const int64_t n = (int64_t)q1 - s.q0;
  s.n = 0;
  if (n < 0 || s.q0 < 0 || q1 > a.tokens || s.ctx < 0 || n > s.ctx || s.ctx > max_ctx) return MKV_DEVERR_CTX;
  if (n == 0) return 0;
  if (s.tab0 < 0 || tabn < ((int64_t)s.ctx + kPageSize - 1) / kPageSize) return MKV_DEVERR_TABLE;
  s.n = (int)n;
  return 0;
}

__device__ __forceinline__ float kv8_scale(int e) { return __builtin_ldexpf(1.0f, e); }

// Least e >= kKv8MinExp with amax <= 448 * 2^e = 1.75 * 2^(e + 8); amax finite, >= 0.
__device__ __forceinline__ int kv8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kKv8MinExp);  // (zeros and subnormals too: their exponent field is 0)
}

// |x| where it is finite, else 0.
__device__ __forceinline__ float kv8_finite_abs(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? __uint_as_float(u) : 0.0f;
}
// x / 2^e for a byte: the format has no infinity, one becomes NaN.
__device__ __forceinline__ float kv8_down(float x, float inv) {
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : x * inv;
}
// (One power of two may pass f32's range: e from -128 of foreign bytes to 120.)
__device__ __forceinline__ float kv8_inv(int e) { return __builtin_ldexpf(1.0f, -e); }

__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ void kv8_unpack4(uint32_t w, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
}
// Four bytes under another exponent: f = 2^(e_old - e_new) <= 1.
__device__ __forceinline__ uint32_t kv8_rescale4(uint32_t w, float f) {
  float x[4];
  kv8_unpack4(w, x);
  return kv8_pack4(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
}
// Bytes of a V dword whose tokens 4 * tq + j are in [lo, hi): 0xff each.
__device__ __forceinline__ uint32_t kv8_tok_mask(int tq, int lo, int hi) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (4 * tq + j >= lo && 4 * tq + j < hi) m |= 0xffu << (8 * j);
  return m;
}

// Maximum over the 64 lanes of a wave, in every lane.
__device__ __forceinline__ float wave_max(float v) {
  v = row16_max(v);
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

template <bool F32>
struct Kv8Row;  // n values at p as f32
template <>
struct Kv8Row<true> {
  static constexpr int ES = 4;
  template <int N>
  static __device__ __forceinline__ void load(const uint8_t *p, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const f32x4 v = *reinterpret_cast<const f32x4 *>(p + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; j++) x[4 * i + j] = v[j];
    }
  }
  template <int N>
  static __device__ __forceinline__ void store(uint8_t *p, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; i++)
      *reinterpret_cast<f32x4 *>(p + 16 * i) = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
  }
};
template <>
struct Kv8Row<false> {
  static constexpr int ES = 2;
  template <int N>
  static __device__ __forceinline__ void load(const uint8_t *p, float (&x)[N]) {
    if constexpr (N == 4) {
      const uint2 w = *reinterpret_cast<const uint2 *>(p);
      x[0] = bf16_lo(w.x), x[1] = bf16_hi(w.x), x[2] = bf16_lo(w.y), x[3] = bf16_hi(w.y);
    } else {
#pragma unroll
      for (int i = 0; i < N / 8; i++) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(p + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; j++) x[8 * i + 2 * j] = bf16_lo(w[j]), x[8 * i + 2 * j + 1] = bf16_hi(w[j]);
      }
    }
  }
  template <int N>
  static __device__ __forceinline__ void store(uint8_t *p, const float (&x)[N]) {
    if constexpr (N == 4) {
      *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    } else {
#pragma unroll
      for (int i = 0; i < N / 8; i++)
        *reinterpret_cast<u32x4 *>(p + 16 * i) =
            u32x4{pack_bf16x2(x[8 * i], x[8 * i + 1]), pack_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                  pack_bf16x2(x[8 * i + 4], x[8 * i + 5]), pack_bf16x2(x[8 * i + 6], x[8 * i + 7])};
    }
  }
};

// ---- writing tiles -------------------------------------------------------------

// The rows of a K tile that this call does not write, [0, o0) and [o1, 16): zeros
// where the tile is fresh (o0 = 0), and expressed under the new exponent where
// that grew. Lane = (token m16, chunk g4) of each KiB.
template <int D>
__device__ __forceinline__ void kv8_k_others(uint8_t *tile, int lane, int o0, int o1, bool grown, float f) {
  const int tok = lane & 15;
  if (tok >= o0 && tok < o1) return;
  if (o0 != 0 && !grown) return;
#pragma unroll
  for (int r = 0; r < D / 64; r++) {
    u32x4 *p = reinterpret_cast<u32x4 *>(tile + 1024 * r) + lane;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (o0 != 0) {
      w = *p;
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = kv8_rescale4(w[j], f);
    }
    *p = w;
  }
}

// Exponent of a tile that takes values up to amax: e, and whether rows held
// before have to be expressed anew (f = 2^(e_old - e)).
__device__ __forceinline__ int kv8_new_exp(float amax, int o0, int e_old, bool &grown, float &f) {
  int e = kv8_exponent(amax);
  grown = false;
  f = 1.0f;
  if (o0 != 0) {
    grown = e > e_old;
    e = max(e, e_old);
    f = __builtin_ldexpf(1.0f, e_old - e);
  }
  return e;
}

// Rows [o0, o1) of a K tile from rows of `stride` bytes at src (row o0 first).
template <int D, bool F32>
__device__ __forceinline__ void kv8_write_k(const uint8_t *src, int64_t stride, uint8_t *tile, int8_t *exp, int lane,
                                            int o0, int o1) {
  typedef Kv8Row<F32> Row;
  const int tok = lane & 15, g4 = lane >> 4;
  const bool mine = tok >= o0 && tok < o1;
  const int e_old = *exp;
  float x[D / 64][16];
  float amax = 0.0f;
  const uint8_t *row = src + (int64_t)(mine ? tok - o0 : 0) * stride + 16 * g4 * Row::ES;
#pragma unroll
  for (int r = 0; r < D / 64; r++) Row::load(row + 64 * r * Row::ES, x[r]);
#pragma unroll
  for (int r = 0; r < D / 64; r++)
#pragma unroll
    for (int j = 0; j < 16; j++) amax = fmaxf(amax, kv8_finite_abs(x[r][j]));
  amax = wave_max(amax);  // (lanes of other rows hold row o0 once more)
  bool grown;
  float f;
  const int e = kv8_new_exp(amax, o0, e_old, grown, f);
  kv8_k_others<D>(tile, lane, o0, o1, grown, f);
  if (mine) {
    const float inv = kv8_inv(e);
#pragma unroll
    for (int r = 0; r < D / 64; r++) {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; j++)
        w[j] = kv8_pack4(kv8_down(x[r][4 * j], inv), kv8_down(x[r][4 * j + 1], inv), kv8_down(x[r][4 * j + 2], inv),
                         kv8_down(x[r][4 * j + 3], inv));
      *(reinterpret_cast<u32x4 *>(tile + 1024 * r) + lane) = w;
    }
  }
  if (lane == 0 && e != e_old) *exp = (int8_t)e;
}

// The same of a V tile. Lane = (token quad g4, dim quad m16) of each KiB.
template <int D, bool F32>
__device__ __forceinline__ void kv8_write_v(const uint8_t *src, int64_t stride, uint8_t *tile, int8_t *exp, int lane,
                                            int o0, int o1) {
  typedef Kv8Row<F32> Row;
  const int dq = lane & 15, tq = lane >> 4;
  const int e_old = *exp;
  float x[D / 64][4][4];  // [.][token j][dim n]
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int tok = 4 * tq + j;
    const uint8_t *row = src + (int64_t)(tok >= o0 && tok < o1 ? tok - o0 : 0) * stride + 4 * dq * Row::ES;
#pragma unroll
    for (int i = 0; i < D / 64; i++) Row::load(row + 64 * i * Row::ES, x[i][j]);
  }
#pragma unroll
  for (int i = 0; i < D / 64; i++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int n = 0; n < 4; n++) amax = fmaxf(amax, kv8_finite_abs(x[i][j][n]));
  amax = wave_max(amax);
  bool grown;
  float f;
  const int e = kv8_new_exp(amax, o0, e_old, grown, f);
  const uint32_t mask = kv8_tok_mask(tq, o0, o1);
  if (o0 == 0 || grown || mask) {
    const float inv = kv8_inv(e);
#pragma unroll
    for (int i = 0; i < D / 64; i++) {
      u32x4 *p = reinterpret_cast<u32x4 *>(tile + 1024 * i) + lane;
      u32x4 w = {0u, 0u, 0u, 0u};
      if (o0 != 0) {
        w = *p;
        if (grown)
#pragma unroll
          for (int n = 0; n < 4; n++) w[n] = kv8_rescale4(w[n], f);
      }
#pragma unroll
      for (int n = 0; n < 4; n++) {
        const uint32_t y = kv8_pack4(kv8_down(x[i][0][n], inv), kv8_down(x[i][1][n], inv), kv8_down(x[i][2][n], inv),
                                     kv8_down(x[i][3][n], inv));
        w[n] = (w[n] & ~mask) | (y & mask);
      }
      *p = w;
    }
  }
  if (lane == 0 && e != e_old) *exp = (int8_t)e;
}

}  // namespace mkv
