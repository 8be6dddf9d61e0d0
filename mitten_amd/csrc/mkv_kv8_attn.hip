// Attention over the K/V pool in 8 bits: one query row per sequence (decode, with
// the row's append fused in) and chunks of new tokens (extend).
//
// For a query row q and the keys it sees, with byte values k', v' and the
// exponents ek, ev of their tiles:
//   s_j = scale * log2(e) * q . (k'_j 2^ek),  o = sum_j 2^(s_j - m) v'_j 2^ev / sum_j 2^(s_j - m).
// S^T = K.Q^T runs on v_mfma_f32_16x16x32_bf16: a byte times its power of two is
// exact in bf16 (the conversion multiplies). A bf16 q is one operand, an f32 q three
// (8 + 8 + 8 bits), so the products are exact and the sums f32.
// O^T = V^T.P^T runs on v_mfma_f32_16x16x32_f16: a byte is exact in f16, and the
// weight carries the tile's exponent: with E the greatest ev so far and d = ev - E,
//   p_j = 2^(s_j + d - R),  O = sum_j p_j v'_j,  l = sum_j 2^(s_j - R - c),  o = 2^(E - c) O / l,
// R a running maximum of s_j + d (moved when one passes it by more than kRescaleSlack).
// c is 0 and l = sum_j 2^-d p_j, but where scales lie so far apart (a tile of zeros, by
// whose score no other is seen in l) that l relative to R would leave f32.
// p is f16 with 11 bits where it matters: it is held times 2^kBias, so at most
// 2^15, and a weight 2^-21 below the greatest is still a normal number. (In bf16 its
// 8 bits would add as much error as the rounding of a bf16 result, 1.41 of it
// together.) f32 rows take two f16 parts (22 bits).
//
// 32 keys (two blocks) per softmax step: the k-slots of lane group g4 in the PV
// product are keys 4 g4 .. +3 of the first block, then of the second, where S^T
// left the scores.
#include <cfloat>

#include "mkv_kv8.h"

namespace mkv {

constexpr float kBias = 15.0f - kRescaleSlack;
constexpr int kMaxRaise = 40;
// A tile with d below that of -kFarExp is summed into l from its scores: 2^-d p_j could leave f32.
constexpr int kFarExp = 40;
// The matrix unit sums the rounded weights of tiles with d >= -kSumExp: what f16 drops
// of one is below 2^-32 of the greatest s + d, 2^-28 of l. Behind that a long row of
// small weights could be missed, and l is summed from the f32 weights.
constexpr int kSumExp = 4;
constexpr int kNoExp = -1000;

template <int D, bool F32>
struct Kv8Q {
  static constexpr int QP = F32 ? 3 : 1;
  bf16x8 op[QP][D / 64][2];
  // Lane holds q[row of lane % 16][64 r + 16 g4 + 8 half .. +8].
  __device__ __forceinline__ void load(const void *q, int64_t row, int g4) {
#pragma unroll
    for (int r = 0; r < D / 64; r++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const int64_t at = row * D + 64 * r + 16 * g4 + 8 * half;
        if constexpr (F32) {
          const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(q) + at);
          const f32x4 a = p[0], b = p[1];
#pragma unroll
          for (int j = 0; j < 8; j++) {
            float x = j < 4 ? a[j & 3] : b[j & 3];
#pragma unroll
            for (int part = 0; part < 3; part++) {
              const __bf16 y = (__bf16)x;
              op[part][r][half][j] = y;
              x -= (float)y;
            }
          }
        } else {
          op[0][r][half] =
              __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(q) + at));
        }
      }
  }
};

// Eight bytes of K as an operand, times 2^ek.
__device__ __forceinline__ bf16x8 kv8_k_operand(uint32_t w0, uint32_t w1, float scale) {
  union {
    bf16x2v p[4];
    bf16x8 v;
  } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return u.v;
}
// Four bytes of V as f16.
__device__ __forceinline__ uint2 kv8_v_half(uint32_t w) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
  return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}

// Softmax state of 16 query rows: row of lane % 16. O[i][n][c] is dim 64 i + 16 g4 + 4 c + n.
// l: this lane's keys only, or with SUMS all keys, summed by the matrix unit (each of
// the four is the same sum).
template <int D, bool SUMS = false>
struct Kv8State {
  typedef typename std::conditional<SUMS, f32x4, float>::type sum_t;
  f32x4 O[D / 64][4];
  float R, c;  // (the four lanes of a row hold the same)
  sum_t l;
  __device__ __forceinline__ float sum() const {
    if constexpr (SUMS) return l[0];
    else return l;
  }
  __device__ __forceinline__ void join() {  // l of all keys
    if constexpr (!SUMS) {
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
    }
  }
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < D / 64; i++)
#pragma unroll
      for (int n = 0; n < 4; n++) O[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    R = -FLT_MAX;  // (finite: no difference of two of them is NaN)
    c = 0.0f;
    l = sum_t{};
  }
  __device__ __forceinline__ void scale_o(float f) {
#pragma unroll
    for (int i = 0; i < D / 64; i++)
#pragma unroll
      for (int n = 0; n < 4; n++) O[i][n] *= f;
  }
  // E grows by de: s + d and R fall by it, O stays. l goes with R as far as f32 allows
  // (2^40 at a time, and not from 2^60 on); the rest stands in c. Whether it does.
  __device__ __forceinline__ bool raise(int de) {
    const int dl = __ballot(sum() > 0x1p60f) ? 0 : min(de, kMaxRaise);
    R -= (float)de;
    c += (float)(de - dl);
    l *= __builtin_ldexpf(1.0f, dl);
    return dl != de;
  }
};

// The scale of a wave's state: E, and whether some row's l is apart from its R (c is not 0).
struct Kv8Scale {
  int E;
  bool apart;
  __device__ __forceinline__ void reset() {
    E = kNoExp;
    apart = false;
  }
};

// d of a step's two tiles. (Only a reference, E, stands between a row and tiles that it
// does not see: R follows s + d of the keys that it does.)
__device__ __forceinline__ void kv8_offsets(int E, int ev0, int ev1, int (&d)[2]) {
  d[0] = ev0 - E;
  d[1] = ev1 - E;
}

// E for a step with tile exponents ev: raised where needed.
template <int D, bool SUMS, int RT>
__device__ __forceinline__ void kv8_raise(Kv8Scale &sc, int ev0, int ev1, Kv8State<D, SUMS> (&st)[RT]) {
  const int top = max(ev0, ev1);
  if (top <= sc.E) return;
  if (sc.E != kNoExp)
#pragma unroll
    for (int i = 0; i < RT; i++) sc.apart |= st[i].raise(top - sc.E);
  sc.E = top;
}

// The greatest s + d of this lane's scores S (hidden keys -inf).
__device__ __forceinline__ float kv8_top(const float (&S)[2][4], float sl2, const int (&d)[2]) {
  const float a = fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3]));
  const float b = fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3]));
  return fmaxf(fmaf(a, sl2, (float)d[0]), fmaf(b, sl2, (float)d[1]));
}

// R for a step whose greatest s + d in this lane is top. R + c moves only where R passes it.
template <int D, bool SUMS>
__device__ __forceinline__ void kv8_rescale(float top, Kv8State<D, SUMS> &st) {
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  const float R = top > st.R + kRescaleSlack ? top : st.R;
  const float up = R - st.R;
  st.l *= fast_exp2(fminf(st.c - up, 0.0f));
  st.c = fmaxf(st.c - up, 0.0f);
  st.scale_o(fast_exp2(-up));
  st.R = R;
}
template <int D, bool SUMS, int RT>
__device__ __forceinline__ void kv8_rescale_all(const float (&top)[RT], Kv8Scale &sc, Kv8State<D, SUMS> (&st)[RT]) {
  bool apart = false;
#pragma unroll
  for (int i = 0; i < RT; i++) {
    kv8_rescale(top[i], st[i]);
    apart |= st[i].c != 0.0f;
  }
  sc.apart = __ballot(apart) != 0;
}

// Whether l takes a tile's weights by kv8_sum_low.
template <bool SUMS>
__device__ __forceinline__ bool kv8_low(int d, bool apart) {
  return d < -(SUMS ? kSumExp : kFarExp) || apart;
}

// The weights of two blocks: operands of the PV product in p (and the second part of
// f32 rows in p2), their sums in l but with SUMS and of low tiles.
template <int D, bool F32, bool SUMS>
__device__ __forceinline__ void kv8_weights(const float (&S)[2][4], float sl2, const int (&d)[2], bool apart,
                                            Kv8State<D, SUMS> &st, f16x8 &p, f16x8 &p2) {
#pragma unroll
  for (int kb = 0; kb < 2; kb++) {
    const float base = st.R - kBias - (float)d[kb];
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = fast_exp2(fmaf(S[kb][i], sl2, -base));
      const _Float16 h = (_Float16)w[i];
      p[4 * kb + i] = h;
      if constexpr (F32) p2[4 * kb + i] = (_Float16)(w[i] - (float)h);
    }
    if constexpr (!SUMS)
      st.l = fmaf((w[0] + w[1]) + (w[2] + w[3]), kv8_low<SUMS>(d[kb], apart) ? 0.0f : kv8_scale(-d[kb]), st.l);
  }
}

// 2^-d of each key, with which the matrix unit sums the weights (SUMS); 0 of a tile
// that kv8_sum_low takes.
__device__ __forceinline__ f16x8 kv8_ones(const int (&d)[2], bool apart) {
  _Float16 y[2];
#pragma unroll
  for (int kb = 0; kb < 2; kb++)
    y[kb] = (_Float16)(kv8_low<true>(d[kb], apart) ? 0.0f : __builtin_ldexpf(1.0f, -d[kb]));
  return f16x8{y[0], y[0], y[0], y[0], y[1], y[1], y[1], y[1]};
}
// The low tiles' weights into l, from their scores: 2^(s_j - R - c). First a score far above
// R + c, whose tile lies so low that R does not follow it, moves c; from then on every tile
// is low, until R has caught up.
template <int D, bool SUMS, int RT>
__device__ __forceinline__ void kv8_sum_low(const float (&S)[RT][2][4], float sl2, const int (&d)[2], Kv8Scale &sc,
                                            Kv8State<D, SUMS> (&st)[RT]) {
  bool apart = false;
#pragma unroll
  for (int x = 0; x < RT; x++) {
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
      if (kv8_low<SUMS>(d[kb], sc.apart))
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, S[x][kb][i] * sl2);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float M = st[x].R + st[x].c;
    if (top > M + (kRescaleSlack + kFarExp)) {  // (below, 2^31 such keys add up to less than 2^87)
      st[x].l *= fast_exp2(M - top);
      st[x].c = top - st[x].R;
      apart = true;
    }
  }
  sc.apart |= __ballot(apart) != 0;
#pragma unroll
  for (int x = 0; x < RT; x++) {
    const float base = st[x].R + st[x].c - kBias;
    float l = 0.0f;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
      if (kv8_low<SUMS>(d[kb], sc.apart))
#pragma unroll
        for (int i = 0; i < 4; i++) l += fast_exp2(fmaf(S[x][kb][i], sl2, -base));
    if constexpr (SUMS) {
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
    }
    st[x].l += l;
  }
}

// Partials. A row's weights are l 2^a, l in [0.5, 1), and the sum of its products o 2^b, a and
// b whole numbers: two powers, for the keys that make the one need not make the other (a
// tile of zeros), and 2^E stays out of o, so neither leaves f32 where the result does not. Held
// as (a, l 2^(b - a)) and o, a frexp apart; no merge takes an exponential.
__device__ __forceinline__ float kv8_pow2(float n) {  // of a whole number n <= 0
  return __builtin_ldexpf(1.0f, (int)fmaxf(n, -2000.0f));
}
__device__ __forceinline__ void kv8_part(float2 ml, float &a, float &b, float &l) {
  a = ml.x;
  l = __builtin_amdgcn_frexp_mantf(ml.y);
  b = a + (float)__builtin_amdgcn_frexp_expf(ml.y);
}
// The result of a row is f * 2^x times o. zero_sink: one more key, of weight 1 and value 0.
__device__ __forceinline__ void kv8_finish(float a, float b, float l, int32_t zero_sink, float &f, int &x) {
  const float top = zero_sink ? fmaxf(a, 0.0f) : a;
  f = 1.0f / (zero_sink ? l * kv8_pow2(a - top) + kv8_pow2(-top) : l);
  x = (int)fminf(fmaxf(b - top, -2000.0f), 2000.0f);
}

// A finished row: the result, or its partial for a merge.
template <int D, bool F32, bool SUMS>
__device__ __forceinline__ void kv8_store(const Kv8State<D, SUMS> &st, int E, int g4, bool final, void *o, int64_t row,
                                          float *ws_ml, float *ws_o, int64_t prow, int32_t zero_sink) {
  // (As the weights and their sums were formed: the same where c is 0.)
  const float m = st.R + st.c - kBias, r = st.R - kBias;
  const float ls = st.sum() * fast_exp2(m - floorf(m));
  const float a = floorf(m) + (float)__builtin_amdgcn_frexp_expf(ls), b = floorf(r) + (float)E;
  const float l = __builtin_amdgcn_frexp_mantf(ls);
  float f = fast_exp2(r - floorf(r));
  int x;
  float k = 0.0f;
  if (final) {
    float g;
    kv8_finish(a, b, l, zero_sink, g, x);
    f *= g;
  } else {  // (b - a past what an exponent holds: the rest to o, whose sum is nothing beside l then, or small)
    k = fminf(fmaxf(b - a, -120.0f), 120.0f);
    x = (int)fminf(fmaxf(b - a - k, -2000.0f), 2000.0f);
  }
#pragma unroll
  for (int i = 0; i < D / 64; i++) {
    float y[16];
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
      for (int n = 0; n < 4; n++) y[4 * c + n] = __builtin_ldexpf(st.O[i][n][c] * f, x);
    const int64_t at = (final ? row : prow) * D + 64 * i + 16 * g4;
    if (final && !F32) {
#pragma unroll
      for (int z = 0; z < 2; z++)
        reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(o) + at)[z] =
            u32x4{pack_bf16x2(y[8 * z], y[8 * z + 1]), pack_bf16x2(y[8 * z + 2], y[8 * z + 3]),
                  pack_bf16x2(y[8 * z + 4], y[8 * z + 5]), pack_bf16x2(y[8 * z + 6], y[8 * z + 7])};
    } else {
      f32x4 *p = reinterpret_cast<f32x4 *>((final ? static_cast<float *>(o) : ws_o) + at);
#pragma unroll
      for (int z = 0; z < 4; z++) p[z] = f32x4{y[4 * z], y[4 * z + 1], y[4 * z + 2], y[4 * z + 3]};
    }
  }
  if (!final && g4 == 0) *reinterpret_cast<float2 *>(ws_ml + 2 * prow) = make_float2(a, __builtin_ldexpf(l, (int)k));
}

// ===========================================================================
// Decode.
//
// A wave takes a run of steps (32 tokens) of one KV head and up to 16 query
// heads, tiles straight from memory into the operand layout, kRing steps deep.
// Two decompositions:
//   split: the steps of all sequences stand in one row, cut into equal pieces;
//     every workgroup finds its place itself by a scan over the lengths, so nothing
//     is planned on the host and a captured call follows the lengths it finds.
//     A sequence that lies in one piece is stored at once, others leave at most
//     two partials per piece, which a second launch merges;
//   seq: one workgroup of 8 waves (4 at head_dim 256) per (sequence, KV head, 16 query
//     heads), their states merged in LDS; one launch.
// What bounds it: memory for many long contexts (64 of 1 to 8k tokens, 286 MB: 55 us
// for the split kernel, 5.2 TB/s, and 5 for the merge), the chain of dependent loads for
// few or short ones (lengths, ids, tiles, partials: 9 us at the least, one of 8k tokens split
// 11 and a merge of 4).
// ===========================================================================

constexpr int kSplitSeqs = 4096;   // sequences of one split launch (their scan stands in LDS)
// Waves of the seq kernel (their states take 512 registers at head_dim 256).
constexpr int kv8_seq_waves(int D) { return D == 256 ? 4 : 8; }
constexpr int kKv8Step = 32;       // tokens of a step

struct Kv8Dec {
  const void *q;
  void *o;
  const uint8_t *new_k, *new_v;  // or null
  float *ws_ml, *ws_o;
  int32_t max_ctx, nqc;
  int32_t pieces, min_steps;  // pieces of a split launch, at least min_steps steps each
  float sl2;
  int32_t zero_sink;
};

// What a wave needs of one step, a step per lane.
struct Kv8Items {
  int32_t seq, id0, id1, exps, meta;  // exps: ek0 | ek1 | ev0 | ev1, one byte each
};
constexpr int kItemValid = 63;      // tokens inside the context, 1..32
constexpr int kItemBad0 = 1 << 6;   // block 0 (1) has an id outside the pool
constexpr int kItemBad1 = 1 << 7;
constexpr int kItemLast = 1 << 8;   // the sequence's last step

// Step j of sequence b, which has ctx tokens and its table at tab0.
__device__ __forceinline__ Kv8Items kv8_item(const Kv8Args &a, int b, int ctx, int tab0, int j) {
  Kv8Items it;
  const int left = ctx - kKv8Step * j;
  const bool two = left > kPageSize;
  const int32_t *t = a.ids + (int64_t)tab0 + 2 * j;
  it.seq = b;
  it.id0 = t[0];
  it.id1 = two ? t[1] : it.id0;
  it.meta = min(left, kKv8Step) | (left <= kKv8Step ? kItemLast : 0);
  if (it.id0 < 0 || it.id0 >= a.nblocks) {
    it.meta |= kItemBad0;
    it.id0 = 0;
    record_error(a.d_err, MKV_DEVERR_BLOCK);
  }
  if (it.id1 < 0 || it.id1 >= a.nblocks) {
    it.meta |= kItemBad1;
    it.id1 = 0;
    record_error(a.d_err, MKV_DEVERR_BLOCK);
  }
  it.exps = 0;
  return it;
}

template <int D>
struct Kv8Raw {
  u32x4 k[2][D / 64], v[2][D / 64];
};

// The new rows of the n steps whose ids `it` holds, written into their tiles before
// these are read: a step that is its sequence's last has one. (Put into the loaded
// registers inside the loop instead, they spilled: 36 registers at head_dim 128. This
// costs 2.4 of 63.4 us for 64 sequences of 1 to 8k tokens.)
template <int D, bool F32>
__device__ __forceinline__ void kv8_insert(const Kv8Args &a, const Kv8Dec &dc, int lane, int h, int n,
                                           const Kv8Items &it) {
  const int left = it.meta & kItemValid;  // tokens of the last step
  const bool bad = it.meta & (left > kPageSize ? kItemBad1 : kItemBad0);
  uint64_t last = __ballot(lane < n && (it.meta & kItemLast) && !bad);
  if (!last) return;
  const int64_t stride = (int64_t)a.Hkv * D * Kv8Row<F32>::ES;
  while (last) {
    const int k = __builtin_ctzll(last);
    last &= last - 1;
    const int nv = __builtin_amdgcn_readlane(it.meta, k) & kItemValid, kb = nv > kPageSize;
    const int row = nv - 1 - kPageSize * kb;
    const int id = kb ? __builtin_amdgcn_readlane(it.id1, k) : __builtin_amdgcn_readlane(it.id0, k);
    const int64_t at = (int64_t)id * a.Hkv + h;
    const int64_t src = __builtin_amdgcn_readlane(it.seq, k) * stride + (int64_t)h * D * Kv8Row<F32>::ES;
    kv8_write_k<D, F32>(dc.new_k + src, stride, a.k_tiles + at * 16 * D, a.k_exps + at, lane, row, row + 1);
    kv8_write_v<D, F32>(dc.new_v + src, stride, a.v_tiles + at * 16 * D, a.v_exps + at, lane, row, row + 1);
  }
  // Read again by this wave alone, through the cache that it wrote through.
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// The exponents of a step's tiles (after its new row is written).
__device__ __forceinline__ void kv8_item_exps(const Kv8Args &a, int h, Kv8Items &it) {
  const int64_t e0 = (int64_t)it.id0 * a.Hkv + h, e1 = (int64_t)it.id1 * a.Hkv + h;
  it.exps = (uint8_t)a.k_exps[e0] | (uint8_t)a.k_exps[e1] << 8 | (uint8_t)a.v_exps[e0] << 16 |
            (uint32_t)(uint8_t)a.v_exps[e1] << 24;
}

// One step: scores of both blocks, weights, O += P.V.
template <int D, bool F32>
__device__ __forceinline__ void kv8_step(float sl2, Kv8Raw<D> &raw, int lane, int exps, int meta,
                                         const Kv8Q<D, F32> &q, Kv8Scale &sc, Kv8State<D> (&st)[1]) {
  const int g4 = lane >> 4;
  int ek[2] = {(int8_t)exps, (int8_t)(exps >> 8)}, ev[2] = {(int8_t)(exps >> 16), exps >> 24};
  const int nv = meta & kItemValid;
  if (nv <= kPageSize) ev[1] = ev[0];
  const bool partial = (meta & (kItemBad0 | kItemBad1)) || nv < kKv8Step;
  if (partial) {
    // V of tokens past the context (or of a rejected block) counts as zero: bytes
    // there may be NaN, and 0 * NaN would poison the sum.
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
      const bool bad = meta & (kb ? kItemBad1 : kItemBad0);
      const uint32_t m = bad ? 0u : kv8_tok_mask(g4, 0, nv - kPageSize * kb);
#pragma unroll
      for (int i = 0; i < D / 64; i++)
#pragma unroll
        for (int n = 0; n < 4; n++) raw.v[kb][i][n] &= m;
    }
  }
  kv8_raise(sc, ev[0], ev[1], st);
  int d[2];
  kv8_offsets(sc.E, ev[0], ev[1], d);
  float t[1][2][4];
#pragma unroll
  for (int kb = 0; kb < 2; kb++) {
    const float ks = kv8_scale(ek[kb]);
    f32x4 S = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < D / 64; r++)
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const bf16x8 k = kv8_k_operand(raw.k[kb][r][2 * half], raw.k[kb][r][2 * half + 1], ks);
#pragma unroll
        for (int part = Kv8Q<D, F32>::QP - 1; part >= 0; part--)
          S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q.op[part][r][half], S, 0, 0, 0);
      }
    // Lane holds S[token 16 kb + 4 g4 + i][query lane % 16].
#pragma unroll
    for (int i = 0; i < 4; i++) t[0][kb][i] = S[i];
    if (partial) {
      const bool bad = meta & (kb ? kItemBad1 : kItemBad0);
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (bad || kPageSize * kb + 4 * g4 + i >= nv) t[0][kb][i] = -INFINITY;
    }
  }
  const float top[1] = {kv8_top(t[0], sl2, d)};
  if (__ballot(top[0] > st[0].R + kRescaleSlack)) kv8_rescale_all(top, sc, st);
  if (kv8_low<false>(min(d[0], d[1]), sc.apart)) kv8_sum_low(t, sl2, d, sc, st);  // (uniform, rare)
  f16x8 p, p2;
  kv8_weights<D, F32>(t[0], sl2, d, sc.apart, st[0], p, p2);
#pragma unroll
  for (int i = 0; i < D / 64; i++)
#pragma unroll
    for (int n = 0; n < 4; n++) {
      const uint2 v0 = kv8_v_half(raw.v[0][i][n]), v1 = kv8_v_half(raw.v[1][i][n]);
      const f16x8 v = __builtin_bit_cast(f16x8, u32x4{v0.x, v0.y, v1.x, v1.y});
      if constexpr (F32) st[0].O[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p2, st[0].O[i][n], 0, 0, 0);
      st[0].O[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p, st[0].O[i][n], 0, 0, 0);
    }
}

// The n steps that `it` holds (lane k: step k), carried on from sequence cur_b
// (-1: none). finish(b) stores a sequence that is done, start(b) loads the next
// one's q.
template <int D, bool F32, class Start, class Finish>
__device__ __forceinline__ void kv8_run(const Kv8Args &a, const Kv8Dec &dc, int lane, int h, int n, Kv8Items it,
                                        int &cur_b, const Kv8Q<D, F32> &q, Kv8Scale &sc,
                                        Kv8State<D> (&st)[1], Start start, Finish finish) {
  constexpr int RING = D == 256 ? 2 : 3;
  if (dc.new_k) kv8_insert<D, F32>(a, dc, lane, h, n, it);
  if (lane < n) kv8_item_exps(a, h, it);
  Kv8Raw<D> raw[RING];
  // (Past the caches: 63.4 us for 64 sequences of 1 to 8k tokens, plain loads 70.6.)
  auto issue = [&](Kv8Raw<D> &w, int k) {
    const bool live = k < n;
    const int kk = live ? k : n - 1;
    // Steps past the end read one line of the last tile again: every stage issues
    // the same loads, so that the compiler's wait counts cover the one in use.
    const int off = live ? lane : lane & 7;
    const int64_t t0 = ((int64_t)__builtin_amdgcn_readlane(it.id0, kk) * a.Hkv + h) * 16 * D;
    const int64_t t1 = ((int64_t)__builtin_amdgcn_readlane(it.id1, kk) * a.Hkv + h) * 16 * D;
    const u32x4 *k0 = reinterpret_cast<const u32x4 *>(a.k_tiles + t0) + off;
    const u32x4 *k1 = reinterpret_cast<const u32x4 *>(a.k_tiles + t1) + off;
    const u32x4 *v0 = reinterpret_cast<const u32x4 *>(a.v_tiles + t0) + off;
    const u32x4 *v1 = reinterpret_cast<const u32x4 *>(a.v_tiles + t1) + off;
#pragma unroll
    for (int r = 0; r < D / 64; r++) {
      w.k[0][r] = __builtin_nontemporal_load(k0 + 64 * r);
      w.k[1][r] = __builtin_nontemporal_load(k1 + 64 * r);
    }
#pragma unroll
    for (int r = 0; r < D / 64; r++) {
      w.v[0][r] = __builtin_nontemporal_load(v0 + 64 * r);
      w.v[1][r] = __builtin_nontemporal_load(v1 + 64 * r);
    }
  };
  auto stage = [&](int s, int k) {
    issue(raw[(s + RING - 1) % RING], k + RING - 1);
    const int b = __builtin_amdgcn_readlane(it.seq, k);
    if (b != cur_b) {
      if (cur_b >= 0) finish(cur_b);
      st[0].reset();
      sc.reset();
      cur_b = b;
      start(b);
    }
    kv8_step<D, F32>(dc.sl2, raw[s], lane, __builtin_amdgcn_readlane(it.exps, k),
                     __builtin_amdgcn_readlane(it.meta, k), q, sc, st);
  };
#pragma unroll
  for (int s = 0; s < RING - 1; s++) issue(raw[s], s);
  int k0 = 0;
  for (int i = 0; i < n / RING; i++, k0 += RING) {
#pragma unroll
    for (int s = 0; s < RING; s++) stage(s, k0 + s);
  }
#pragma unroll
  for (int s = 0; s < RING - 1; s++)
    if (k0 + s < n) stage(s, k0 + s);
}

// Steps of sequence b, 0 for one that does not fit or is padding.
__device__ __forceinline__ int kv8_steps(const Kv8Args &a, int b, int max_ctx, uint32_t &err) {
  const int ctx = a.ctx[b], tab0 = a.indptr[b];
  const int64_t tabn = a.ids ? (int64_t)a.indptr[b + 1] - tab0 : 0;
  err = 0;
  if (ctx == 0) return 0;
  if (ctx < 0 || ctx > max_ctx) err = MKV_DEVERR_CTX;
  else if (tab0 < 0 || tabn < ((int64_t)ctx + kPageSize - 1) / kPageSize) err = MKV_DEVERR_TABLE;
  return err ? 0 : (int)(((int64_t)ctx + kKv8Step - 1) / kKv8Step);
}

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// Query heads of chunk qc of a group.
__device__ __forceinline__ int kv8_chunk_heads(int G, int qc) { return min(16, G - 16 * qc); }

template <int D, bool F32>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
kv8_decode_split_kernel(Kv8Args a, Kv8Dec dc) {
  extern __shared__ int32_t pre[];  // [B + 1] steps before each sequence, then their lengths and tables
  int32_t *ctx_s = pre + a.B + 1, *tab_s = ctx_s + a.B;
  __shared__ int32_t wsum[4];
  const int lane = threadIdx.x & 63, m16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  {
    const int per = (a.B + 255) / 256, b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
    int sum = 0;
    for (int b = b0; b < b1; b++) {
      uint32_t err;
      const int n = kv8_steps(a, b, dc.max_ctx, err);
      if (err && blockIdx.x == 0) record_error(a.d_err, err);
      pre[b + 1] = n;  // (own entries only, turned into the scan below)
      ctx_s[b] = a.ctx[b];
      tab_s[b] = a.indptr[b];
      sum += n;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    int at = inc - sum;
    for (int w = 0; w < wave; w++) at += wsum[w];
    for (int b = b0; b < b1; b++) {
      at += pre[b + 1];
      pre[b + 1] = at;
    }
    if (threadIdx.x == 0) pre[0] = 0;
    __syncthreads();
  }
  const int total = pre[a.B], heads = a.Hkv * dc.nqc;
  const int per = max(dc.min_steps, (total + dc.pieces - 1) / dc.pieces);
  const int wid = (int)blockIdx.x * 4 + wave, p = wid / heads, hc = wid % heads;
  const int h = hc / dc.nqc, qc = hc % dc.nqc;
  if (p >= dc.pieces || (int64_t)p * per >= total) return;
  const int f0 = p * per, f1 = min(total, f0 + per);
  const int nq = kv8_chunk_heads(a.G, qc), q0 = h * a.G + 16 * qc;
  Kv8Q<D, F32> q;
  Kv8State<D> st[1];
  Kv8Scale sc;
  sc.reset();
  int cur = -1;
  auto start = [&](int b) { q.load(dc.q, (int64_t)b * a.Hq + q0 + min(m16, nq - 1), g4); };
  auto finish = [&](int b) {
    st[0].join();
    const int s0 = __builtin_amdgcn_readfirstlane(pre[b]), s1 = __builtin_amdgcn_readfirstlane(pre[b + 1]);
    if (m16 >= nq) return;
    // A sequence that starts in this piece and goes on behind it is its second partial.
    const int64_t slot = 2 * (int64_t)p + (s0 >= f0);
    kv8_store<D, F32, false>(st[0], sc.E, g4, s0 >= f0 && s1 <= f1, dc.o, (int64_t)b * a.Hq + q0 + m16, dc.ws_ml, dc.ws_o,
                      slot * a.Hq + q0 + m16, dc.zero_sink);
  };
  for (int c = f0; c < f1; c += 64) {
    const int n = min(64, f1 - c);
    Kv8Items it = {0, 0, 0, 0, 0};
    if (lane < n) {
      const int f = c + lane;
      int lo = 0, hi = a.B;  // the last sequence that starts at or before f
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= f) lo = mid;
        else hi = mid;
      }
      it = kv8_item(a, lo, ctx_s[lo], tab_s[lo], f - pre[lo]);
    }
    kv8_run<D, F32>(a, dc, lane, h, n, it, cur, q, sc, st, start, finish);
  }
  finish(cur);
}

// Merge of n partials by a wave: (a, l 2^(b - a)) of partial s at ml_at(s), o at o_at(s). Lane s
// holds the numbers of partial s of a round of 16, lane d dims d * DPL .. +DPL of every one.
template <int D, class MlAt, class OAt>
__device__ __forceinline__ void kv8_merge(int lane, int n, MlAt ml_at, OAt o_at, float &A, float &B, float &L,
                                          typename MergeVec<D>::type &acc) {
  constexpr int DPL = MergeVec<D>::DPL, SB = 16;
  typedef typename MergeVec<D>::type fvec;
  acc = fvec{};
  A = B = -FLT_MAX;
  L = 0.0f;
  auto first = [](float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
  };
  for (int s0 = 0; s0 < n; s0 += SB) {
    const int cnt = min(SB, n - s0);
    float2 ml = make_float2(-FLT_MAX, 0.0f);
    if (lane < cnt) ml = *reinterpret_cast<const float2 *>(ml_at(s0 + lane));
    fvec ov[SB];
#pragma unroll
    for (int i = 0; i < SB; i++) {
      ov[i] = fvec{};
      if (i < cnt) ov[i] = *reinterpret_cast<const fvec *>(o_at(s0 + i) + lane * DPL);
    }
    float a, b, l;
    kv8_part(ml, a, b, l);
    const float An = fmaxf(A, first(row16_max(a))), Bn = fmaxf(B, first(row16_max(b)));
    L = L * kv8_pow2(A - An) + first(row_sum<16>(l * kv8_pow2(a - An)));
    acc *= kv8_pow2(B - Bn);
    const float w = kv8_pow2(b - Bn);
#pragma unroll
    for (int i = 0; i < SB; i++)
      acc += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i)) * ov[i];
    A = An;
    B = Bn;
  }
}

// The merge of a split launch, a workgroup per (query head, sequence); also the
// zeros of padding sequences.
template <int D, bool F32>
__global__ void __launch_bounds__(256) kv8_decode_merge_kernel(Kv8Args a, Kv8Dec dc) {
  constexpr int NW = 4, DPL = MergeVec<D>::DPL;
  typedef typename MergeVec<D>::type fvec;
  __shared__ int32_t sums[2][NW];
  __shared__ float part[NW][3 + 64 * DPL];
  const int lane = threadIdx.x & 63, hq = blockIdx.x, b = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int before = 0, all = 0;
  uint32_t err;
  for (int i = threadIdx.x; i < a.B; i += 256) {
    const int n = kv8_steps(a, i, dc.max_ctx, err);
    all += n;
    before += i < b ? n : 0;
  }
  const int mine = kv8_steps(a, b, dc.max_ctx, err);
  before = wave_sum_int(before);
  all = wave_sum_int(all);
  if (lane == 0) sums[0][wave] = before, sums[1][wave] = all;
  __syncthreads();
  before = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
  all = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  if (err) return;
  const int64_t row = (int64_t)b * a.Hq + hq;
  if (mine == 0) {
    for (int i = threadIdx.x; i < D; i += 256) {
      if constexpr (F32) static_cast<float *>(dc.o)[row * D + i] = 0.0f;
      else static_cast<uint16_t *>(dc.o)[row * D + i] = 0;
    }
    return;
  }
  const int per = max(dc.min_steps, (all + dc.pieces - 1) / dc.pieces);
  const int p0 = before / per, p1 = (before + mine - 1) / per;
  if (p0 == p1) return;  // stored already
  const int n = p1 - p0 + 1, waves = n <= 16 ? 1 : NW;
  if (wave >= waves) return;  // (no barrier follows where waves is 1)
  const int s0 = (int)((int64_t)n * wave / waves), s1 = (int)((int64_t)n * (wave + 1) / waves);
  // Partial s: piece p0 + s; in the first one the sequence starts.
  auto at = [&](int s) {
    const int pc = p0 + s0 + s;
    return (2 * (int64_t)pc + (before >= pc * per)) * a.Hq + hq;
  };
  float A, B, L;
  fvec acc;
  kv8_merge<D>(
      lane, s1 - s0, [&](int s) { return dc.ws_ml + 2 * at(s); }, [&](int s) { return dc.ws_o + at(s) * D; }, A, B, L,
      acc);
  if (waves > 1) {
    if (lane == 0) part[wave][0] = A, part[wave][1] = B, part[wave][2] = L;
#pragma unroll
    for (int k = 0; k < DPL; k++) part[wave][3 + lane * DPL + k] = acc[k];
    __syncthreads();
    if (wave != 0) return;
    L = 0.0f;
    acc = fvec{};
#pragma unroll
    for (int w = 1; w < NW; w++) A = fmaxf(A, part[w][0]), B = fmaxf(B, part[w][1]);
#pragma unroll
    for (int w = 0; w < NW; w++) {
      L = fmaf(part[w][2], kv8_pow2(part[w][0] - A), L);
      const float f = kv8_pow2(part[w][1] - B);
#pragma unroll
      for (int k = 0; k < DPL; k++) acc[k] = fmaf(part[w][3 + lane * DPL + k], f, acc[k]);
    }
  }
  float f;
  int x;
  kv8_finish(A, B, L, dc.zero_sink, f, x);
  const int64_t to = row * D + lane * DPL;
#pragma unroll
  for (int k = 0; k < DPL; k++) acc[k] = __builtin_ldexpf(acc[k] * f, x);
  if constexpr (F32) *reinterpret_cast<fvec *>(static_cast<float *>(dc.o) + to) = acc;
  else {
    uint16_t *op = static_cast<uint16_t *>(dc.o) + to;
    if constexpr (DPL == 1) *op = (uint16_t)f32_to_bf16_bits(acc[0]);
    else if constexpr (DPL == 2) *reinterpret_cast<uint32_t *>(op) = pack_bf16x2(acc[0], acc[1]);
    else *reinterpret_cast<uint2 *>(op) = make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
  }
}

template <int D, bool F32>
__global__ void __launch_bounds__(64 * kv8_seq_waves(D)) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
kv8_decode_seq_kernel(Kv8Args a, Kv8Dec dc) {
  constexpr int NW = kv8_seq_waves(D);
  __shared__ __attribute__((aligned(16))) float part[NW][16][D];
  __shared__ float2 ml[NW][16];
  const int lane = threadIdx.x & 63, m16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y, h = blockIdx.x / dc.nqc, qc = blockIdx.x % dc.nqc;
  const int nq = kv8_chunk_heads(a.G, qc), q0 = h * a.G + 16 * qc;
  uint32_t err;
  const int steps = __builtin_amdgcn_readfirstlane(kv8_steps(a, b, dc.max_ctx, err));
  if (err) {
    if (blockIdx.x == 0 && threadIdx.x == 0) record_error(a.d_err, err);
    return;
  }
  const int f0 = (int)((int64_t)steps * wave / NW), f1 = (int)((int64_t)steps * (wave + 1) / NW);
  if (f0 < f1) {
    const int ctx = a.ctx[b], tab0 = a.indptr[b];
    Kv8Q<D, F32> q;
    Kv8State<D> st[1];
    Kv8Scale sc;
    int cur = b;
    sc.reset();
    st[0].reset();
    q.load(dc.q, (int64_t)b * a.Hq + q0 + min(m16, nq - 1), g4);
    for (int c = f0; c < f1; c += 64) {
      const int n = min(64, f1 - c);
      Kv8Items it = {b, 0, 0, 0, 0};
      if (lane < n) it = kv8_item(a, b, ctx, tab0, c + lane);
      kv8_run<D, F32>(a, dc, lane, h, n, it, cur, q, sc, st, [](int) {}, [](int) {});
    }
    st[0].join();
    kv8_store<D, true, false>(st[0], sc.E, g4, false, nullptr, 0, &ml[wave][0].x, &part[wave][0][0], m16, 0);
  }
  __syncthreads();
  const int used = min(NW, steps);
  for (int i = threadIdx.x; i < nq * (D / 4); i += 64 * NW) {
    const int r = i / (D / 4), dim = 4 * (i % (D / 4));
    float A = -FLT_MAX, B = -FLT_MAX, L = 0.0f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto live = [&](int w) { return (int64_t)steps * w / NW < (int64_t)steps * (w + 1) / NW; };
    for (int w = 0; w < NW; w++) {
      if (!live(w)) continue;
      float pa, pb, pl;
      kv8_part(ml[w][r], pa, pb, pl);
      A = fmaxf(A, pa), B = fmaxf(B, pb);
    }
    for (int w = 0; w < NW; w++) {
      if (!live(w)) continue;
      float pa, pb, pl;
      kv8_part(ml[w][r], pa, pb, pl);
      L = fmaf(pl, kv8_pow2(pa - A), L);
      acc += *reinterpret_cast<const f32x4 *>(&part[w][r][dim]) * kv8_pow2(pb - B);
    }
    float f = 0.0f;  // (No keys at all: a padding sequence, a row of zeros.)
    int x = 0;
    if (used) kv8_finish(A, B, L, dc.zero_sink, f, x);
#pragma unroll
    for (int k = 0; k < 4; k++) acc[k] = __builtin_ldexpf(acc[k] * f, x);
    const int64_t at = ((int64_t)b * a.Hq + q0 + r) * D + dim;
    if constexpr (F32) *reinterpret_cast<f32x4 *>(static_cast<float *>(dc.o) + at) = acc;
    else
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(dc.o) + at) =
          make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
  }
}

// ===========================================================================
// Extend: causal attention of the newest q_len tokens over the whole cache.
//
// The rows of one (sequence, KV head) are its (position, query head of the group)
// pairs in memory order. A workgroup of W waves takes 16 * RT * W of them, RT groups
// of 16 rows a wave, and streams the keys they see, 32 a step. A tile's bytes are
// converted once, on the way into LDS (K bf16 with its exponent, V f16), and lie
// there in operand order: 16 bytes a lane, contiguous, for all reads and for K's stores. V's
// stores are 8 bytes a lane at a stride of 16, one block's half of an operand: half the banks
// at a time (the SQ_LDS_BANK_CONFLICT of these kernels, 4% of the busy cycles in long chunks).
// An operand is read once for RT products: LDS gives 128 bytes a cycle and CU, so at
// RT = 1 the reads of a step take as long as twice its products, at RT = 2 as long.
// Loads run kKv8ExtRing - 1 steps ahead in registers (16 bytes a lane and 1 KiB of tile);
// one barrier a step.
// What bounds it: the matrix unit and the instructions around it. 8 chunks of 512 tokens
// after 4k, 28 query heads on 4 KV heads of 128 dims, bf16: 256 GFLOP in 323 us (790
// TFLOP/s). Tiles of 128 rows on 512 places, 4k tokens before them, of equal lengths: 896 take
// 302 us (847 TFLOP/s), 1,024 308 (957), 1,536 464 (983), 544 233 (613).
// With the next step's scores beside the weights; one after the other 420 us.
// ===========================================================================

constexpr int kKv8ExtRing = 4;    // steps in registers, the one in use included
constexpr int kKv8ExtIds = 1024;  // block ids staged in LDS at a time
constexpr int kCutSeqs = 512;     // sequences of a cut launch

// Two decompositions. Whole: a workgroup per (tile, KV head, sequence). Cut: the steps of
// all tiles stand in one row (a tile's as many as its sequence has), cut into equal
// pieces, as a decode launch's are; a tile that lies in one piece is stored at once, a
// row of others has a partial per piece, numbered from the tile's first, and a second
// launch merges them. Measured at 28 query heads on 4 KV heads of 128 dims, bf16, whole /
// cut in us: 16 chunks of 8 tokens after 2k 48 / 35, after 8k 170 / 55; of 40 after 8k
// 222 / 145; one of 200 after 30k 622 / 134. (16 chunks of 5 to 24 tokens after 4 to 8k
// take 73, in equal shares of every tile 87: their workgroups fill the CUs 1.3 times.)
struct Kv8Ext {
  const void *q;
  void *o;
  float *ws_ml, *ws_o;
  int32_t max_ctx, rows, tiles;  // rows of a tile; tiles of the longest chunk
  int32_t pieces, parts;         // of a cut launch; partials of a row, at most (1: whole)
  float sl2;
  int32_t zero_sink;
};
constexpr int kCutMinSteps = 4;  // steps of a piece, at least

// Tiles of a chunk of n tokens, and steps of each.
__device__ __forceinline__ int kv8_cut_tiles(const Kv8Args &a, const Kv8Ext &e, int n) {
  return (int)(((int64_t)n * a.G + e.rows - 1) / e.rows);
}
__device__ __forceinline__ int kv8_cut_steps(int ctx) { return (int)(((int64_t)ctx + kKv8Step - 1) / kKv8Step); }
// Steps of a piece, of `total`; no tile (of `longest` steps, at most) has more pieces than parts.
__device__ __forceinline__ int kv8_cut_per(const Kv8Ext &e, int total, int longest) {
  return max(kCutMinSteps, max((total + e.pieces - 1) / e.pieces, (longest + e.parts - 2) / (e.parts - 1)));
}

// Rows t0 .. of one sequence and KV head over the steps [s0, s1) of its keys: the whole
// result, or partial `part`.
template <int D, bool F32, int RT, int W>
__device__ __forceinline__ void kv8_extend_tile(const Kv8Args &a, const Kv8Ext &e, const Kv8Seq &s, int h, int t0,
                                                int s0, int s1, bool whole, int part) {
  constexpr int NR = D / 64, UNITS = 4 * NR;  // 1 KiB pieces of a step: (K | V, block, r)
  constexpr int LPL = UNITS / W;              // of them a wave loads
  static_assert(UNITS % W == 0, "every wave loads the same number of pieces");
  constexpr int HALF = 64 * D;                // bytes of K, or V, of a step in LDS
  constexpr int R = kKv8ExtRing;
  __shared__ __attribute__((aligned(16))) uint8_t kbuf[2][HALF], vbuf[2][HALF];
  __shared__ int32_t ids_s[kKv8ExtIds], exps_s[kKv8ExtIds];  // exps: ek, then ev, a byte each
  __shared__ int32_t odd_s;
  const int tid = threadIdx.x, lane = tid & 63, m16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t rows = (int64_t)s.n * a.G;
  const int p0 = s.ctx - s.n;
  const int last = (int)min(rows, (int64_t)t0 + 16 * RT * W) - 1;  // the tile's last row
  const int qlo_wg = p0 + t0 / a.G, qhi_wg = p0 + last / a.G;
  const int steps_all = qhi_wg / kKv8Step + 1;
  const int st0 = min(s0, steps_all), st1 = min(s1, steps_all);
  const int nblk = qhi_wg / kPageSize + 1;

  int qp[RT], qlo[RT], row0[RT];
  int64_t qrow[RT];
  Kv8Q<D, F32> q[RT];
  Kv8State<D, !F32> st[RT];
  Kv8Scale sc;
  sc.reset();
  int qhi = -1;  // last position of the wave's rows; -1: it has none
#pragma unroll
  for (int i = 0; i < RT; i++) {
    row0[i] = t0 + (wave * RT + i) * 16;
    const int r = min(row0[i] + m16, (int)rows - 1), pos = r / a.G;
    qp[i] = p0 + pos;
    qlo[i] = p0 + min(row0[i], (int)rows - 1) / a.G;
    qrow[i] = (int64_t)(s.q0 + pos) * a.Hq + h * a.G + (r - pos * a.G);
    if (row0[i] < rows) qhi = p0 + min(row0[i] + 15, (int)rows - 1) / a.G;
    q[i].load(e.q, qrow[i], g4);
    st[i].reset();
  }

  u32x4 raw[R][LPL];
  // Piece u = wave + W * i of a step: K or V (known at compile time but at head_dim 64),
  // block kb, KiB r; all of it wave-uniform.
  auto is_v = [&](int i) { return (2 * NR) % W == 0 ? (W * i) / (2 * NR) : (wave + W * i) / (2 * NR); };
  auto load = [&](int i, int32_t id, bool live) {
    const int r = (wave + W * i) % NR;
    const uint8_t *t = (is_v(i) ? a.v_tiles : a.k_tiles) + ((int64_t)max(id, 0) * a.Hkv + h) * 16 * D + 1024 * r;
    // (A step past the end reads one line of the last block again.)
    return *(reinterpret_cast<const u32x4 *>(t) + (live ? lane : lane & 7));
  };
  // A piece, converted, into buffer y: K times 2^ek, V as it is.
  auto put_k = [&](u32x4 w, int i, int y, int ek) {
    const int u = wave + W * i, kb = (u / NR) & 1, r = u % NR;
    const float f = kv8_scale(ek);
    uint8_t *p = kbuf[y] + ((kb * NR + r) * 2) * 1024 + lane * 16;
    *reinterpret_cast<bf16x8 *>(p) = kv8_k_operand(w[0], w[1], f);
    *reinterpret_cast<bf16x8 *>(p + 1024) = kv8_k_operand(w[2], w[3], f);
  };
  auto put_v = [&](u32x4 w, int i, int y) {
    const int u = wave + W * i, kb = (u / NR) & 1, r = u % NR;
#pragma unroll
    for (int n = 0; n < 4; n++)
      *reinterpret_cast<uint2 *>(vbuf[y] + (r * 4 + n) * 1024 + lane * 16 + 8 * kb) = kv8_v_half(w[n]);
  };
  auto read_k = [&](bf16x8 (&k)[2][2], int y, int r) {
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
        k[half][kb] = *reinterpret_cast<const bf16x8 *>(kbuf[y] + ((kb * NR + r) * 2 + half) * 1024 + lane * 16);
  };
  auto dot_k = [&](f32x4 (&S)[RT][2], const bf16x8 (&k)[2][2], int r) {
#pragma unroll
    for (int half = 0; half < 2; half++)
#pragma unroll
      for (int part = Kv8Q<D, F32>::QP - 1; part >= 0; part--)
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
          for (int x = 0; x < RT; x++)
            S[x][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[half][kb], q[x].op[part][r][half],
                                                               r == 0 && half == 0 && part == Kv8Q<D, F32>::QP - 1
                                                                   ? f32x4{0.f, 0.f, 0.f, 0.f} : S[x][kb], 0, 0, 0);
  };
  auto read_v = [&](f16x8 (&v)[4], int y, int r) {
#pragma unroll
    for (int n = 0; n < 4; n++) v[n] = *reinterpret_cast<const f16x8 *>(vbuf[y] + (r * 4 + n) * 1024 + lane * 16);
  };
  auto add_v = [&](const f16x8 (&v)[4], const f16x8 (&p)[RT], const f16x8 (&p2)[RT], int r) {
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
      for (int x = 0; x < RT; x++) {
        f32x4 &o = st[x].O[r][n];
        if constexpr (F32) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[n], p2[x], o, 0, 0, 0);
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[n], p[x], o, 0, 0, 0);
      }
  };
  auto sum_p = [&](const f16x8 (&p)[RT], const int (&d)[2]) {
    if constexpr (!F32) {
      const f16x8 ones = kv8_ones(d, sc.apart);
#pragma unroll
      for (int x = 0; x < RT; x++) st[x].l = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[x], st[x].l, 0, 0, 0);
    }
  };
  // E, R and what kv8_sum_low adds for the scores S of a step with V exponents ev0, ev1.
  auto settle = [&](const f32x4 (&S)[RT][2], int ev0, int ev1, float (&t)[RT][2][4], int (&d)[2], auto mask) {
    kv8_raise(sc, ev0, ev1, st);
    kv8_offsets(sc.E, ev0, ev1, d);
    float top[RT];
    bool move = false;
#pragma unroll
    for (int x = 0; x < RT; x++) {
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int c = 0; c < 4; c++) t[x][kb][c] = S[x][kb][c];
      mask(t[x], x);
      top[x] = kv8_top(t[x], e.sl2, d);
      move |= top[x] > st[x].R + kRescaleSlack;
    }
    if (__ballot(move)) kv8_rescale_all(top, sc, st);
    if (kv8_low<!F32>(min(d[0], d[1]), sc.apart)) kv8_sum_low(t, e.sl2, d, sc, st);  // (uniform, rare)
  };

  f32x4 S[2][RT][2];
  if (tid == 0) odd_s = 0;
  for (int c0 = st0; c0 < st1; c0 += kKv8ExtIds / 2) {
    const int c1 = min(st1, c0 + kKv8ExtIds / 2);
    const int nid = min(2 * c1, nblk) - 2 * c0;  // ids of this run; behind them the last one counts
    __syncthreads();
    int bad = 0;
    for (int i = tid; i < nid; i += 64 * W) {
      int32_t id = a.ids[(int64_t)s.tab0 + 2 * c0 + i];
      if (id < 0 || id >= a.nblocks) {
        id = -1;
        bad = 1;
        record_error(a.d_err, MKV_DEVERR_BLOCK);
      }
      ids_s[i] = id;
      const int64_t at = (int64_t)max(id, 0) * a.Hkv + h;
      exps_s[i] = (uint8_t)a.k_exps[at] | a.v_exps[at] * 256;
    }
    bad = __builtin_amdgcn_readfirstlane(__syncthreads_or(bad));
    auto block = [&](int step, int kb) { return min(2 * (step - c0) + kb, nid - 1); };
    auto kb_of = [&](int i) { return ((wave + W * i) / NR) & 1; };
    auto issue = [&](u32x4 (&w)[LPL], int step) {
#pragma unroll
      for (int i = 0; i < LPL; i++)
        w[i] = load(i, __builtin_amdgcn_readfirstlane(ids_s[block(step, kb_of(i))]), step < c1);
    };
    // Pieces of K of step ks and of V of step vs, with what has to be left out.
    auto put = [&](const u32x4 (&kw)[LPL], int ks, const u32x4 (&vw)[LPL], int vs) {
#pragma unroll
      for (int i = 0; i < LPL; i++) {
        if (!is_v(i)) {
          if (ks < c1) put_k(kw[i], i, ks - c0 & 1, (int8_t)exps_s[block(ks, kb_of(i))]);
          continue;
        }
        if (vs >= c1) continue;
        u32x4 w = vw[i];
        const int k = 2 * vs + kb_of(i);
        if (bad && ids_s[block(vs, kb_of(i))] < 0) w = u32x4{0u, 0u, 0u, 0u};
        if (kKv8Step * (vs + 1) - 1 > qlo_wg) {  // some row of the tile does not see all of it
          // Keys past the context count as zero (their bytes may be NaN, and 0 * NaN is
          // NaN), and so does a NaN that some row must not see: it is given to the rows
          // that do when the tile is done.
          const uint32_t in = kv8_tok_mask(g4, 0, s.ctx - kPageSize * k);
          const uint32_t later = kv8_tok_mask(g4, qlo_wg + 1 - kPageSize * k, kPageSize);
          uint32_t odd = 0;
#pragma unroll
          for (int n = 0; n < 4; n++) {
            w[n] &= in;
            const uint32_t one = (((w[n] & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u & later;
            w[n] &= ~((one << 8) - one);
            odd |= one;
          }
          if (odd) odd_s = 1;
        }
        put_v(w, i, vs - c0 & 1);
      }
    };
#pragma unroll
    for (int i = 0; i < R - 1; i++) issue(raw[i], c0 + i);
    put(raw[0], c0, raw[0], c0);
    put(raw[1], c0 + 1, raw[1], c1);
    __syncthreads();
    auto scores = [&](f32x4 (&N)[RT][2], int y) {
#pragma unroll
      for (int r = 0; r < NR; r++) {
        bf16x8 k[2][2];
        read_k(k, y, r);
        dot_k(N, k, r);
      }
    };
    if (kKv8Step * c0 <= qhi) scores(S[0], 0);
    __syncthreads();

    // Steps whose keys, and those of the two after, every row of the workgroup sees,
    // R at a time. A step's turn: its scores are in S, its V in buffer y. The scores of
    // the next step go into N beside its weights, so that the matrix and the vector units
    // both have work, and its products with V beside the conversion of later tiles: K
    // of the step after the next and V of the next, into the buffers that every wave
    // left at the last barrier. Ids and exponents of a round stand in lanes.
    const int full = bad ? c0 : min(c1, (qlo_wg + 1) / kKv8Step) - 2;
    int step = c0;
    int idw = ids_s[min(lane, nid - 1)], exw = exps_s[min(lane, nid - 1)];
    for (int it = 0, n = max(full - c0, 0) / R; it < n; it++, step += R) {
      const int at = min(2 * (step + R - c0) + lane, nid - 1);
      const int idn = ids_s[at], exn = exps_s[at];
#pragma unroll
      for (int i = 0; i < R; i++) {
        constexpr auto lane_of = [](int x, int kb) { return 2 * x + kb; };
        const int y = i & 1;
        f32x4(&cur)[RT][2] = S[y];
        f32x4(&nxt)[RT][2] = S[y ^ 1];
        u32x4(&in)[LPL] = raw[(i + R - 1) % R];
#pragma unroll
        for (int l = 0; l < LPL; l++) {
          // (Blocks past the last step are the last block again: step < c1 - 2 here.)
          const int32_t id = __builtin_amdgcn_readlane(idw, lane_of(i + R - 1, 0) + kb_of(l));
          in[l] = load(l, id, step + i + R - 1 < c1);
        }
        if (qhi >= 0) {
          bf16x8 k[2][2][2];
          read_k(k[0], y ^ 1, 0);
          float t[RT][2][4];
          int d[2];
          settle(cur, __builtin_amdgcn_readlane(exw, lane_of(i, 0)) >> 8, __builtin_amdgcn_readlane(exw, lane_of(i, 1)) >> 8,
                 t, d, [](float (&)[2][4], int) {});
          f16x8 p[RT], p2[RT], v[2][4];
#pragma unroll
          for (int r = 0; r < NR; r++) {
            if (r + 1 < NR) read_k(k[(r + 1) & 1], y ^ 1, r + 1);
            dot_k(nxt, k[r & 1], r);
          }
          read_v(v[0], y, 0);
#pragma unroll
          for (int x = 0; x < RT; x++) kv8_weights<D, F32, !F32>(t[x], e.sl2, d, sc.apart, st[x], p[x], p2[x]);
          // One product, then some of the weights' instructions, in turn.
#pragma unroll
          for (int g = 0; g < 4 * NR * RT * Kv8Q<D, F32>::QP; g++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, F32 ? 2 : 4, 0);
          }
          __builtin_amdgcn_sched_barrier(0);  // (362 us where the products with V may mix in, 323 here: 8 x 512 after 4k)
          sum_p(p, d);
#pragma unroll
          for (int r = 0; r < NR; r++) {
            if (r + 1 < NR) read_v(v[(r + 1) & 1], y, r + 1);
            add_v(v[r & 1], p, p2, r);
          }
        }
#pragma unroll
        for (int l = 0; l < LPL; l++) {
          if (!is_v(l)) {
            const int ek = (int8_t)__builtin_amdgcn_readlane(exw, lane_of(i + 2, 0) + kb_of(l));
            put_k(raw[(i + 2) % R][l], l, y, ek);
          } else {
            put_v(raw[(i + 1) % R][l], l, y ^ 1);
          }
        }
        __syncthreads();
      }
      idw = idn;
      exw = exn;
    }
    // The rest a step at a time, masked, the ring moved down, the next scores in the
    // place of these.
#pragma unroll 1
    for (; step < c1; step++) {
      const int y = step - c0 & 1;
      if (kKv8Step * step <= qhi) {
        float t[RT][2][4];
        int d[2];
        settle(S[0], __builtin_amdgcn_readfirstlane(exps_s[block(step, 0)]) >> 8,
               __builtin_amdgcn_readfirstlane(exps_s[block(step, 1)]) >> 8, t, d, [&](float (&u)[2][4], int x) {
                 if (!bad && kKv8Step * (step + 1) - 1 <= qlo[x]) return;
                 const int key = kKv8Step * step + 4 * g4;
#pragma unroll
                 for (int kb = 0; kb < 2; kb++) {
                   const bool none = bad && ids_s[block(step, kb)] < 0;
#pragma unroll
                   for (int c = 0; c < 4; c++)
                     if (none || key + kPageSize * kb + c > qp[x]) u[kb][c] = -INFINITY;
                 }
               });
        f16x8 p[RT], p2[RT];
#pragma unroll
        for (int x = 0; x < RT; x++) kv8_weights<D, F32, !F32>(t[x], e.sl2, d, sc.apart, st[x], p[x], p2[x]);
        scores(S[0], y ^ 1);
        sum_p(p, d);
#pragma unroll
        for (int r = 0; r < NR; r++) {
          f16x8 v[4];
          read_v(v, y, r);
          add_v(v, p, p2, r);
        }
      }
      put(raw[2], step + 2, raw[1], step + 1);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < LPL; i++) raw[1][i] = raw[2][i];
      issue(raw[2], step + 3);
    }
  }
  __syncthreads();
  const bool odd = odd_s;
#pragma unroll
  for (int i = 0; i < RT; i++) {
    st[i].join();
    if (row0[i] + m16 < rows)
      kv8_store<D, F32, !F32>(st[i], sc.E, g4, whole, e.o, qrow[i], e.ws_ml, e.ws_o, qrow[i] * e.parts + part,
                              e.zero_sink);
  }
  if (!odd) return;
  // NaN values of V behind the tile's first position, for the rows that see them.
  __syncthreads();
  const int key0 = max(qlo_wg + 1, kKv8Step * st0), key1 = min(s.ctx, kKv8Step * st1);
  for (int i = tid; i < (last - t0 + 1) * (D / 4); i += 64 * W) {
    const int r = t0 + i / (D / 4), dim = 4 * (i % (D / 4)), pos = r / a.G;
    uint32_t nan = 0;
    for (int key = key0; key < min(key1, p0 + pos + 1); key++) {
      const int32_t id = a.ids[(int64_t)s.tab0 + key / kPageSize];
      if (id < 0 || id >= a.nblocks) continue;
      const int tok = key % kPageSize;
      const uint8_t *t = a.v_tiles + ((int64_t)id * a.Hkv + h) * 16 * D + dim / 64 * 1024 + tok / 4 * 256 + dim % 64 * 4 + tok % 4;
#pragma unroll
      for (int n = 0; n < 4; n++)
        if ((t[4 * n] & 0x7f) == 0x7f) nan |= 1u << n;
    }
    const int64_t qr = (int64_t)(s.q0 + pos) * a.Hq + h * a.G + (r - pos * a.G);
#pragma unroll
    for (int n = 0; n < 4; n++) {
      if (!(nan >> n & 1)) continue;
      if (!whole) e.ws_o[(qr * e.parts + part) * D + dim + n] = __uint_as_float(0x7fc00000u);
      else if constexpr (F32) static_cast<float *>(e.o)[qr * D + dim + n] = __uint_as_float(0x7fc00000u);
      else static_cast<uint16_t *>(e.o)[qr * D + dim + n] = 0x7fc0;
    }
  }
}

template <int D, bool F32, int RT, int W>
__global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(D == 256 && F32 ? 1 : 2, D == 256 && F32 ? 1 : 2)))
kv8_extend_kernel(Kv8Args a, Kv8Ext e) {
  __shared__ int32_t pre[kCutSeqs + 1], longest_s;
  const int pairs = a.Hkv * a.B;
  const bool cut = e.parts > 1;
  int b = 0, h = 0, u = 0, u1 = 0, per = 1, first = 0;
  int64_t t = -1;
  Kv8Seq s;
  if (cut) {
    for (int i = threadIdx.x; i < a.B; i += 64 * W) {
      Kv8Seq x;
      const uint32_t err = kv8_seq(a, i, e.max_ctx, x);
      if (err && blockIdx.x == 0) record_error(a.d_err, err);
      const bool none = err || x.n == 0;
      pre[i + 1] = none ? 0 : a.Hkv * kv8_cut_tiles(a, e, x.n) * kv8_cut_steps(x.ctx);
    }
    if (threadIdx.x == 0) pre[0] = 0;
    __syncthreads();
    if (threadIdx.x < 64) {
      int at = 0, top = 0;
      for (int i0 = 0; i0 < a.B; i0 += 64) {
        const int i = i0 + (int)threadIdx.x;
        int v = i < a.B ? pre[i + 1] : 0;
        if (v > 0) top = max(top, kv8_cut_steps(a.ctx[i]));
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int up = __shfl_up(v, o);
          if ((int)threadIdx.x >= o) v += up;
        }
        if (i < a.B) pre[i + 1] = at + v;
        at += __shfl(v, 63);
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) top = max(top, __shfl_xor(top, o));
      if (threadIdx.x == 0) longest_s = top;
    }
    __syncthreads();
    const int total = __builtin_amdgcn_readfirstlane(pre[a.B]);
    per = kv8_cut_per(e, total, __builtin_amdgcn_readfirstlane(longest_s));
    // Neighbours, which read the same keys for other rows, on one XCD.
    const int x = blockIdx.x;
    first = e.pieces % 8 ? x : x % 8 * (e.pieces / 8) + x / 8;
    if ((int64_t)first * per >= total) return;
    u = first * per;
    u1 = min(total, u + per);
  } else {
    // Tiles with the most keys first, every (KV head, sequence) in turn. Where
    // their number is a multiple of the 8 XCDs, all tiles of a pair run on one and
    // share its L2.
    const int64_t L = blockIdx.x;
    const int pair = (int)(L % pairs);
    h = pair % a.Hkv;
    b = pair / a.Hkv;
    const uint32_t err = kv8_seq(a, b, e.max_ctx, s);
    if (err && L < pairs && h == 0 && threadIdx.x == 0) record_error(a.d_err, err);
    if (err || s.n == 0) return;
    // (A chunk longer than max_q_len takes further rounds.)
    t = kv8_cut_tiles(a, e, s.n) - 1 - L / pairs;
  }
  while (cut ? u < u1 : t >= 0) {
    int s0 = 0, s1 = INT32_MAX, part = 0;
    bool whole = true;
    if (cut) {
      int lo = 0, hi = a.B;  // the last sequence that starts at or before u
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__builtin_amdgcn_readfirstlane(pre[mid]) <= u) lo = mid;
        else hi = mid;
      }
      (void)kv8_seq(a, lo, e.max_ctx, s);
      const int steps = kv8_cut_steps(s.ctx), tiles = kv8_cut_tiles(a, e, s.n);
      const int r = u - __builtin_amdgcn_readfirstlane(pre[lo]), ht = r / steps;
      h = ht / tiles;
      t = ht % tiles;
      s0 = r - ht * steps;
      s1 = min(steps, s0 + u1 - u);
      whole = s0 == 0 && s1 == steps;
      part = first - (u - s0) / per;
      u += s1 - s0;
    }
    kv8_extend_tile<D, F32, RT, W>(a, e, s, h, (int)t * e.rows, s0, s1, whole, part);
    __syncthreads();
    if (!cut) t -= e.tiles;
  }
}

// The merge of a cut launch: a thread per 4 dims of a (token, query head) row of
// sequence blockIdx.y.
template <int D, bool F32>
__global__ void __launch_bounds__(256) kv8_extend_merge_kernel(Kv8Args a, Kv8Ext e) {
  constexpr int TPR = D / 4;  // threads of a row
  __shared__ int32_t part[4][3];
  Kv8Seq s;
  int before = 0, total = 0, longest = 0;
  for (int i = threadIdx.x; i < a.B; i += 256) {
    if (kv8_seq(a, i, e.max_ctx, s) || s.n == 0) continue;
    const int steps = kv8_cut_steps(s.ctx), n = a.Hkv * kv8_cut_tiles(a, e, s.n) * steps;
    total += n;
    before += i < (int)blockIdx.y ? n : 0;
    longest = max(longest, steps);
  }
  before = wave_sum_int(before);
  total = wave_sum_int(total);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) longest = max(longest, __shfl_xor(longest, o));
  if (threadIdx.x % 64 == 0) {
    int32_t *p = part[threadIdx.x / 64];
    p[0] = before, p[1] = total, p[2] = longest;
  }
  __syncthreads();
  before = part[0][0] + part[1][0] + part[2][0] + part[3][0];
  total = part[0][1] + part[1][1] + part[2][1] + part[3][1];
  longest = max(max(part[0][2], part[1][2]), max(part[2][2], part[3][2]));
  if (kv8_seq(a, blockIdx.y, e.max_ctx, s) || s.n == 0) return;
  const int per = kv8_cut_per(e, total, longest), steps = kv8_cut_steps(s.ctx), tiles = kv8_cut_tiles(a, e, s.n);
  const int64_t rows = (int64_t)s.n * a.Hq;
  const int dim = 4 * (threadIdx.x % TPR);
  for (int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR; r < rows; r += (int64_t)gridDim.x * (256 / TPR)) {
    const int pos = (int)(r / a.Hq), hq = (int)(r - (int64_t)pos * a.Hq), h = hq / a.G;
    const int tile = (int)(((int64_t)pos * a.G + (hq - h * a.G)) / e.rows);
    const int from = before + (h * tiles + tile) * steps;
    const int parts = (from + steps - 1) / per - from / per + 1;
    if (parts == 1) continue;  // stored already
    const int64_t at = ((int64_t)s.q0 * a.Hq + r) * e.parts;
    float A = -FLT_MAX, B = -FLT_MAX, L = 0.0f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    constexpr int N = 8;  // partials loaded at a time
    for (int i0 = 0; i0 < parts; i0 += N) {
      float2 y[N];
      f32x4 o[N];
#pragma unroll
      for (int i = 0; i < N; i++) {  // (past the last partial: the last one, with no weight)
        const int64_t c = at + min(i0 + i, parts - 1);
        y[i] = *reinterpret_cast<const float2 *>(e.ws_ml + 2 * c);
        o[i] = *reinterpret_cast<const f32x4 *>(e.ws_o + c * D + dim);
      }
      float pa[N], pb[N], pl[N], An = A, Bn = B;
#pragma unroll
      for (int i = 0; i < N; i++) {
        kv8_part(y[i], pa[i], pb[i], pl[i]);
        An = fmaxf(An, pa[i]);
        Bn = fmaxf(Bn, pb[i]);
      }
      L *= kv8_pow2(A - An);
      acc *= kv8_pow2(B - Bn);
#pragma unroll
      for (int i = 0; i < N; i++) {
        if (i0 + i >= parts) break;
        L = fmaf(pl[i], kv8_pow2(pa[i] - An), L);
        acc += o[i] * kv8_pow2(pb[i] - Bn);
      }
      A = An;
      B = Bn;
    }
    float f;
    int x;
    kv8_finish(A, B, L, e.zero_sink, f, x);
#pragma unroll
    for (int k = 0; k < 4; k++) acc[k] = __builtin_ldexpf(acc[k] * f, x);
    const int64_t out = ((int64_t)s.q0 * a.Hq + r) * D + dim;
    if constexpr (F32) *reinterpret_cast<f32x4 *>(static_cast<float *>(e.o) + out) = acc;
    else
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(e.o) + out) =
          make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
  }
}

// ---- host side ----------------------------------------------------------------------

static uint64_t kv8_ml_bytes(uint64_t rows) { return (rows * 8 + 255) / 256 * 256; }

#define KV8_LAUNCH(KERNEL, GRID, BLOCK, LDS, ...)                                                       \
  do {                                                                                                  \
    const bool f32 = g.dtype == MKV_DTYPE_F32;                                                          \
    switch (g.D) {                                                                                      \
      case 64: if (f32) hipLaunchKernelGGL((KERNEL<64, true>), GRID, BLOCK, LDS, hs, __VA_ARGS__);       \
               else hipLaunchKernelGGL((KERNEL<64, false>), GRID, BLOCK, LDS, hs, __VA_ARGS__); break;   \
      case 128: if (f32) hipLaunchKernelGGL((KERNEL<128, true>), GRID, BLOCK, LDS, hs, __VA_ARGS__);     \
                else hipLaunchKernelGGL((KERNEL<128, false>), GRID, BLOCK, LDS, hs, __VA_ARGS__); break; \
      default: if (f32) hipLaunchKernelGGL((KERNEL<256, true>), GRID, BLOCK, LDS, hs, __VA_ARGS__);      \
               else hipLaunchKernelGGL((KERNEL<256, false>), GRID, BLOCK, LDS, hs, __VA_ARGS__); break;  \
    }                                                                                                   \
  } while (0)

static int kv8_check_attn(const Kv8Pool *p, int32_t layer, float scale, uint32_t flags, const void *ws) {
  int rc = kv8_check_layer(p, layer);
  if (rc) return rc;
  if (!(scale > 0.0f) || !std::isfinite(scale))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "scale must be finite and > 0");
  if (flags & ~(uint32_t)MKV_ATTN_ZERO_SINK)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
  if (!aligned16(ws)) return set_error(MKV_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  return MKV_OK;
}

// ---- decode

// kSplitWavesPerCu, and the steps of a piece, at least. Measured, 64 sequences of 1 to
// 8k tokens (286 MB): 8 waves a CU 63.5 us, 7 the same, 12 (with a ring of 2, which
// their registers allow) 65.9, 16 73.0; one sequence of 8k: 4 steps 16.3 us, 2 the
// same, 8 18.6.
constexpr int kSplitMinSteps = 4;

// Steps of the longest context that a wave of the seq kernel may have to take; behind that
// the split kernel. The seq kernel saves the scan and the merge, but its longest sequence
// is on eight waves alone, and its workgroups are large. Measured at head_dim 128, 4 KV
// heads, seq / split in us: 8 sequences of 1,024 tokens 12.4 / 15.4, 1,536 15.5 / 15.7,
// 2,048 17.6 / 16.2; 64 of 1,024 16.8 / 26.8, 64 of 1 to 2,048 21.8 / 28.8, of 1 to
// 3,200 29.1 / 35.3, all but one of 100 17.3 / 16.7 and 23.0 / 16.6; 256 of 512
// 41.8 / 45.7, all but one of 100 34.8 / 26.8. Those are bf16, three batches in turn; other
// types and head dims follow the same steps. Of one batch, which stays in the caches: f32, 128
// dims, 8 of 1,024 12.6 / 18.4, of 2,048 17.2 / 19.0; f32, 256 dims, 8 of 1,024 21.7 / 24.9, of
// 1,536 28.4 / 25.1, 64 of 1,024 31.9 / 56.4; bf16, 64 dims, 8 of 1,536 9.7 / 15.3, of 2,048
// 10.6 / 15.5, 256 of 512 26.3 / 33.7. (So 64 dims are split early.) The bound on the lengths
// counts, not what a captured call finds.
static int kv8_seq_steps(int64_t wgs, int cus) { return 2 * wgs < cus ? 6 : wgs <= 2 * cus ? 10 : 0; }

// Up to kSplitSeqs sequences (any number for pieces = 0, the seq kernel).
static int launch_kv8_decode(const Kv8Pool *p, const Kv8Args &a, Kv8Dec &d, int64_t pieces, hipStream_t hs) {
  const Geom &g = p->g;
  const int64_t heads = (int64_t)g.Hkv * d.nqc;
  if (pieces < 1) {
    KV8_LAUNCH(kv8_decode_seq_kernel, dim3((unsigned)heads, (unsigned)a.B), dim3(64 * kv8_seq_waves(g.D)), 0, a, d);
    MKV_CHECK_LAUNCH("kv8_decode_seq_kernel");
    return MKV_OK;
  }
  d.pieces = (int32_t)pieces;
  KV8_LAUNCH(kv8_decode_split_kernel, dim3((unsigned)((pieces * heads + 3) / 4)), dim3(256), (3 * a.B + 1) * 4, a, d);
  MKV_CHECK_LAUNCH("kv8_decode_split_kernel");
  KV8_LAUNCH(kv8_decode_merge_kernel, dim3((unsigned)g.Hq, (unsigned)a.B), dim3(256), 0, a, d);
  MKV_CHECK_LAUNCH("kv8_decode_merge_kernel");
  return MKV_OK;
}

// ---- extend

// The forms of the extend kernel: rows and waves of a workgroup, and what a step of 32
// keys takes it in us, alone on a CU and beside a second one (0: none fits). Wide: an
// LDS operand feeds two groups of rows where the registers allow it. Measured: 16
// chunks of 5-24 tokens after 4-8k unsplit, and 8 of 512 after 4k. (Every tile is priced by
// the longest context; a cheaper form or cut by a few percent of this is not to be relied on.)
struct Kv8ExtForm {
  const void *fn;
  int rows, waves;
  double alone, beside;
};
static Kv8ExtForm kv8_ext_form(const Geom &g, bool wide) {
#define KV8_EXT(DD, FF, RR, WW, ALONE, BESIDE) \
  Kv8ExtForm { reinterpret_cast<const void *>(&kv8_extend_kernel<DD, FF, RR, WW>), 16 * RR * WW, WW, ALONE, BESIDE }
  const bool f32 = g.dtype == MKV_DTYPE_F32;
  switch (g.D) {
    case 64:
      if (f32) return wide ? KV8_EXT(64, true, 2, 4, .77, 1.37) : KV8_EXT(64, true, 1, 4, .56, .75);
      return wide ? KV8_EXT(64, false, 2, 4, .58, .92) : KV8_EXT(64, false, 1, 4, .48, .58);
    case 128:
      if (f32) return wide ? KV8_EXT(128, true, 1, 8, 1.26, 0) : KV8_EXT(128, true, 1, 4, .85, 1.15);
      return wide ? KV8_EXT(128, false, 2, 4, .76, 1.24) : KV8_EXT(128, false, 1, 4, .60, .78);
    default:
      if (f32) return KV8_EXT(256, true, 1, 4, 2.0, 0);
      return wide ? KV8_EXT(256, false, 1, 8, 1.0, 0) : KV8_EXT(256, false, 1, 4, .88, 1.28);
  }
#undef KV8_EXT
}

// What a call takes, by that: `tiles` tiles of `steps` each. Whole: in rounds of what the
// CUs hold. Cut: in equal pieces, started twice each, and the merge: a launch, and the
// partials' bytes both ways.
static double kv8_ext_whole(const Kv8ExtForm &f, double cus, double tiles, double steps) {
  const double wgs = tiles / cus;
  double step = f.alone;
  if (wgs > 1) step = f.beside > 0 ? std::max(f.beside, f.beside * std::ceil(wgs) / 2) : f.alone * std::ceil(wgs);
  return steps * step + 3.0;
}
static int kv8_ext_slots(const Kv8ExtForm &f, int cus) { return f.beside > 0 ? 2 * cus : cus; }
static double kv8_ext_cut(const Kv8ExtForm &f, int cus, double tiles, double steps, int parts, double values) {
  const double per = std::max({(double)kCutMinSteps, tiles * steps / kv8_ext_slots(f, cus), steps / (parts - 1)});
  const double step = f.beside > 0 && tiles * steps / per > cus ? f.beside : f.alone;
  return per * step + 6.0 + 6.0 + values * (steps / per + 1) * 8 / 5.0e6;
}

}  // namespace mkv

using namespace mkv;

extern "C" int mkv_kv8_decode_attention(mkv_kv8_pool *pool, int32_t layer, const void *d_k_new, const void *d_v_new,
                                        const void *d_q, void *d_o, const int32_t *d_block_indptr,
                                        const int32_t *d_block_ids, const int32_t *d_ctx_lens, int32_t num_seqs,
                                        int32_t max_ctx_len, float scale, uint32_t flags, void *d_workspace,
                                        uint64_t workspace_bytes, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  const Geom &g = p->g;
  int rc = kv8_check_attn(p, layer, scale, flags, d_workspace);
  if (rc) return rc;
  if (num_seqs < 0 || num_seqs > 65535 || max_ctx_len < 0)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs outside [0, 65535], or max_ctx_len < 0");
  if (!d_k_new != !d_v_new) return set_error(MKV_ERR_INVALID_ARGUMENT, "give both new rows, or neither");
  if (num_seqs == 0) return MKV_OK;
  if (!d_q || !d_o || !d_block_indptr || !d_ctx_lens)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(d_q) || !aligned16(d_o) || !aligned16(d_k_new) || !aligned16(d_v_new))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "q, o and the new rows must be 16-byte aligned");
  const uint64_t on = (uint64_t)num_seqs * g.Hq * g.D * g.es, kn = (uint64_t)num_seqs * g.row_bytes;
  if (overlap(d_o, on, d_q, on) || overlap(d_o, on, d_k_new, kn) || overlap(d_o, on, d_v_new, kn))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "o overlaps q or the new rows");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  const int G = g.Hq / g.Hkv, nqc = (G + 15) / 16;
  Kv8Args a = kv8_args(p, layer, nullptr, d_block_indptr, d_block_ids, d_ctx_lens, num_seqs, num_seqs);
  if (nqc > 1 && d_k_new) {
    // Several waves read a head's tiles: the rows are written before any of them.
    if ((rc = kv8_append_rows(p, a, d_k_new, d_v_new, max_ctx_len, hs))) return rc;
    d_k_new = d_v_new = nullptr;
  }
  Kv8Dec d{};
  d.max_ctx = max_ctx_len;
  d.nqc = nqc;
  d.min_steps = kSplitMinSteps;
  d.sl2 = scale * kLog2e;
  d.zero_sink = (flags & MKV_ATTN_ZERO_SINK) ? 1 : 0;
  const int64_t most = ((int64_t)max_ctx_len + kKv8Step - 1) / kKv8Step, heads = (int64_t)g.Hkv * nqc;
  int64_t pieces = 0;
  Kv8Ws ws;
  if (most > kv8_seq_waves(g.D) * kv8_seq_steps(heads * num_seqs, p->cus)) {
    if ((rc = kv8_ws_begin(p, d_workspace, workspace_bytes, hs, &ws))) return rc;
    // Two partials a piece; fewer pieces where there are no more steps, or the
    // workspace holds no more.
    pieces = kv8_most_pieces(g, p->cus);
    pieces = std::min(pieces, (most * num_seqs + kSplitMinSteps - 1) / kSplitMinSteps);
    if (kv8_piece_bytes(g, pieces) > ws.bytes)
      pieces = ws.bytes > 256 ? (int64_t)((ws.bytes - 256) / ((uint64_t)2 * g.Hq * (8 + 4 * g.D))) : 0;
    d.ws_ml = static_cast<float *>(ws.ptr);
    d.ws_o = reinterpret_cast<float *>(static_cast<uint8_t *>(ws.ptr) + kv8_ml_bytes((uint64_t)2 * pieces * g.Hq));
  }
  const int32_t chunk = pieces < 1 ? num_seqs : kSplitSeqs;
  for (int32_t b0 = 0; b0 < num_seqs; b0 += chunk) {
    Kv8Args c = a;
    c.B = c.tokens = std::min(chunk, num_seqs - b0);
    c.indptr += b0;
    c.ctx += b0;
    const int64_t rows = (int64_t)b0 * g.Hq * g.D * g.es, kv = (int64_t)b0 * g.row_bytes;
    d.q = static_cast<const uint8_t *>(d_q) + rows;
    d.o = static_cast<uint8_t *>(d_o) + rows;
    d.new_k = d_k_new ? static_cast<const uint8_t *>(d_k_new) + kv : nullptr;
    d.new_v = d_k_new ? static_cast<const uint8_t *>(d_v_new) + kv : nullptr;
    if ((rc = launch_kv8_decode(p, c, d, pieces, hs))) return rc;
  }
  return kv8_ws_end(p, ws, hs);
}

extern "C" int mkv_kv8_decode_attention_host(mkv_kv8_pool *pool, int32_t layer, const void *d_k_new,
                                             const void *d_v_new, const void *d_q, void *d_o,
                                             const int32_t *h_ctx_lens, const uint32_t *h_block_indptr,
                                             const uint32_t *h_block_ids, int32_t num_seqs, float scale,
                                             uint32_t flags, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  int rc = kv8_check_layer(p, layer);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  Kv8Meta m;
  if ((rc = kv8_stage(p, p->decode_cache, nullptr, h_ctx_lens, h_block_indptr, h_block_ids, nullptr, num_seqs,
                      d_k_new != nullptr, hs, &m)))
    return rc;
  rc = mkv_kv8_decode_attention(pool, layer, d_k_new, d_v_new, d_q, d_o, m.indptr, m.ids, m.ctx, num_seqs, m.max_ctx,
                                scale, flags, nullptr, 0, stream);
  const int rr = meta_release(m.slot, hs);
  return rc ? rc : rr;
}

extern "C" int mkv_kv8_extend_attention(mkv_kv8_pool *pool, int32_t layer, const void *d_q, void *d_o,
                                        const int32_t *d_q_indptr, const int32_t *d_block_indptr,
                                        const int32_t *d_block_ids, const int32_t *d_ctx_lens, int32_t num_seqs,
                                        int32_t num_tokens, int32_t max_q_len, int32_t max_ctx_len, float scale,
                                        uint32_t flags, void *d_workspace, uint64_t workspace_bytes, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  const Geom &g = p->g;
  int rc = kv8_check_attn(p, layer, scale, flags, d_workspace);
  if (rc) return rc;
  if (num_seqs < 0 || num_seqs > 65535 || num_tokens < 0 || max_q_len < 0 || max_ctx_len < 0)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs outside [0, 65535], or negative sizes");
  if (num_seqs == 0 || num_tokens == 0 || max_q_len == 0) return MKV_OK;
  if (max_q_len > max_ctx_len)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "max_q_len %d > max_ctx_len %d", max_q_len, max_ctx_len);
  if (!d_q || !d_o || !d_q_indptr || !d_block_indptr || !d_ctx_lens)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  if (!aligned16(d_q) || !aligned16(d_o)) return set_error(MKV_ERR_INVALID_ARGUMENT, "q and o must be 16-byte aligned");
  const uint64_t on = (uint64_t)num_tokens * g.Hq * g.D * g.es;
  if (overlap(d_o, on, d_q, on)) return set_error(MKV_ERR_INVALID_ARGUMENT, "o overlaps q");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  Kv8Args a = kv8_args(p, layer, d_q_indptr, d_block_indptr, d_block_ids, d_ctx_lens, num_seqs, num_tokens);
  Kv8Ext e{};
  e.q = d_q;
  e.o = d_o;
  e.max_ctx = max_ctx_len;
  e.sl2 = scale * kLog2e;
  e.zero_sink = (flags & MKV_ATTN_ZERO_SINK) ? 1 : 0;
  const int64_t pairs = (int64_t)g.Hkv * num_seqs, rows = (int64_t)std::min(max_q_len, num_tokens) * a.G;
  if ((int64_t)num_tokens * a.G > INT32_MAX / 2) return set_error(MKV_ERR_INVALID_ARGUMENT, "too many tokens");
  // The form and the decomposition that cost least, for chunks of the mean length (of
  // many lengths: half a tile more) and the longest context. A row has at most 32
  // partials, and no more than the workspace holds of all rows.
  const double mean = std::max(1.0, std::min<double>((double)rows, (double)num_tokens * a.G / num_seqs));
  auto tiles_of = [&](int n) {
    const double most = std::ceil((double)rows / n);
    return mean >= (double)rows ? most : std::max(1.0, std::min(most, mean / n + 0.5));
  };
  const int64_t steps = ((int64_t)max_ctx_len + kKv8Step - 1) / kKv8Step;
  const uint64_t row = (uint64_t)num_tokens * g.Hq * (8 + 4 * g.D);
  const uint64_t bytes = d_workspace ? workspace_bytes : p->ws_bytes, room = bytes > 256 ? bytes - 256 : 0;
  const int parts = (int)std::min<uint64_t>(room / row, 32);
  Kv8ExtForm form{};
  double best = INFINITY;
  e.parts = 1;
  for (int narrow = 0; narrow < 2; narrow++) {
    const Kv8ExtForm f = kv8_ext_form(g, !narrow);
    const double tiles = (double)pairs * tiles_of(f.rows);
    // (Units are 32-bit, also where the chunks' rows overlap.)
    const double most = (double)pairs * std::ceil((double)num_tokens * a.G / f.rows) * (double)steps;
    double c = kv8_ext_whole(f, p->cus, tiles, (double)steps);
    if (c < best) best = c, form = f, e.parts = 1;
    if (parts < 2 || num_seqs > kCutSeqs || most > INT32_MAX / 2) continue;
    c = kv8_ext_cut(f, p->cus, tiles, (double)steps, parts, (double)num_tokens * g.Hq * g.D);
    if (c < best) best = c, form = f, e.parts = parts;
  }
  e.rows = form.rows;
  const int64_t tiles = (rows + form.rows - 1) / form.rows;
  int64_t grid = tiles * pairs;
  Kv8Ws ws;
  if (e.parts > 1) {
    if ((rc = kv8_ws_begin(p, d_workspace, workspace_bytes, hs, &ws))) return rc;
    e.ws_ml = static_cast<float *>(ws.ptr);
    e.ws_o = reinterpret_cast<float *>(static_cast<uint8_t *>(ws.ptr) + kv8_ml_bytes((uint64_t)num_tokens * g.Hq * e.parts));
    e.pieces = kv8_ext_slots(form, p->cus);
    grid = e.pieces;
  }
  if (grid > INT32_MAX) return set_error(MKV_ERR_INVALID_ARGUMENT, "grid too large");
  e.tiles = (int32_t)tiles;
  void *args[] = {&a, &e};
  MKV_CHECK_HIP(hipLaunchKernel(form.fn, dim3((unsigned)grid), dim3(64 * form.waves), args, 0, hs));
  MKV_CHECK_LAUNCH("kv8_extend_kernel");
  if (e.parts > 1) {
    const int64_t per = 1024 / g.D, wgs = ((int64_t)std::min(max_q_len, num_tokens) * g.Hq + per - 1) / per;
    const dim3 mgrid((unsigned)std::min<int64_t>(wgs, 1 << 20), (unsigned)num_seqs);
    KV8_LAUNCH(kv8_extend_merge_kernel, mgrid, dim3(256), 0, a, e);
    MKV_CHECK_LAUNCH("kv8_extend_merge_kernel");
  }
  return kv8_ws_end(p, ws, hs);
}

extern "C" int mkv_kv8_extend_attention_host(mkv_kv8_pool *pool, int32_t layer, const void *d_q, void *d_o,
                                             const int32_t *h_q_lens, const int32_t *h_ctx_lens,
                                             const uint32_t *h_block_indptr, const uint32_t *h_block_ids,
                                             int32_t num_seqs, float scale, uint32_t flags, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  Kv8Pool *p = reinterpret_cast<Kv8Pool *>(pool);
  int rc = kv8_check_layer(p, layer);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  if (!h_q_lens) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL q_lens");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  Kv8Meta m;
  if ((rc = kv8_stage(p, p->extend_cache, h_q_lens, h_ctx_lens, h_block_indptr, h_block_ids, nullptr, num_seqs, false,
                      hs, &m)))
    return rc;
  rc = mkv_kv8_extend_attention(pool, layer, d_q, d_o, m.q_indptr, m.indptr, m.ids, m.ctx, num_seqs, m.tokens, m.max_q,
                                m.max_ctx, scale, flags, nullptr, 0, stream);
  const int rr = meta_release(m.slot, hs);
  return rc ? rc : rr;
}
