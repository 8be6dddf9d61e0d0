// Linear attention over ragged batches of chunks of tokens (prompts): the
// chunked form of the recurrence
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t.
// Over a chunk of tokens with G_t = g_1 + ... + g_t (t counted in the chunk),
//   o_t   = scale * ( e^{G_t} S_in^T q_t + sum_{s <= t} e^{G_t - G_s} (q_t . k_s) v_s )
//   S_out = e^{G_end} S_in + sum_s k_s (e^{G_end - G_s} v_s)^T,
// four matrix products per chunk instead of a rank-one update per token.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <new>
#include <type_traits>

#include "mkv_linear.h"

namespace mkv {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4s lds_i16x4;

constexpr int kChunk = 64;  // tokens per chunk

// A sequence's tokens are cut into segments of `len` tokens (the last takes
// what is left), computed side by side: each segment's own contribution to the
// state first (local form, from zero), then a scan over the segments, then
// the outputs of every segment from the state before it. One segment per
// sequence (nseg 1) is a single launch.
struct LinSegs {
  int32_t nseg, len;
  float *state;  // [B][nseg][Hv][DK * DV]: local states, then the state before each segment
  float *decay;  // [B][nseg][Hv]: exp of a segment's summed log decays, -0 with a decay of 0 among them
};

__device__ __forceinline__ int lin_nseg(const LinSegs &g, int n) {
  return n > 0 ? min(g.nseg, (n - 1) / g.len + 1) : 1;
}

// Row swizzles of the LDS tiles (16-byte chunk c of row r stands at c ^ swz(r)):
// lin_row_swz for 16-byte reads of one chunk of 16 rows, lin_tr_swz for the
// transposing reads of four rows by two chunks (linear over GF(2) in the row's
// low bits; its values over 8 rows are distinct modulo 8, so 16-byte reads
// stay free of conflicts too).
__device__ __forceinline__ int lin_row_swz(int r, int cpr) { return r & 15 & (cpr - 1); }
__device__ __forceinline__ int lin_tr_swz(int r, int cpr) {
  const int s = ((r & 1) << 1) ^ ((r & 2) << 1) ^ (((r >> 2) & 1) * 11) ^ ((r >> 3) & 1);
  return s & (cpr - 1);
}

// Byte offset of half `half` of 16-byte chunk c of row r. Rows 8-15 of every 16
// have their halves swapped: 16 lanes that read the same half of 16 rows (one
// 8-byte read each) then cover every bank.
__device__ __forceinline__ int lin_at(int r, int c, int half, int cpr, int swz) {
  return r * cpr * 16 + (c ^ swz) * 16 + (half ^ ((r >> 3) & 1)) * 8;
}

// v of another lane of the DPP pattern, 0 where the pattern has no source.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Inclusive sum over lanes 0..lane of the wave.
__device__ __forceinline__ double wave_scan(double v) {
  v += dpp_d<0x111, 0xf>(v);  // row_shr:1
  v += dpp_d<0x112, 0xf>(v);  // row_shr:2
  v += dpp_d<0x114, 0xf>(v);  // row_shr:4
  v += dpp_d<0x118, 0xf>(v);  // row_shr:8
  v += dpp_d<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp_d<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ double lane_d(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }  // below 2^-126: 0

// Whether a decay of that log2 is 0 in f32, as -inf is: it makes an infinity a NaN.
__device__ __forceinline__ bool decay_is_zero(double l) { return l < -150.0; }

// A token's log decay in base 2. Below e^-104 a decay is 0 in f32 whatever
// stands beside it: cutting there keeps sums of decays finite at -inf (a NaN
// stays one).
__device__ __forceinline__ double log2_decay(float g) {
  return (double)(g < -104.0f ? -104.0f : g) * 1.4426950408889634074;
}

// Difference of two summed log2 decays of a chunk, each in steps of 2^-17 (64
// tokens reach -9,603, within 31 bits): off by 2^-17 at most wherever the
// tokens stand, where f32 sums behind strong decays are off by 2^-10. A NaN is lost
// here; it reaches the outputs by e^G.
__device__ __forceinline__ float decay_diff(int a, int b) {
  return (float)(int)((uint32_t)a - (uint32_t)b) * 7.62939453125e-6f;
}

// A segment's decay for the scan, from its summed log2 (-inf: one of them was 0).
__device__ __forceinline__ float segment_decay(double total) {
  return total == -INFINITY ? -0.0f : exp2_f((float)total);
}

// c + the squares of a word's two bf16: not finite where one is an Inf, a NaN, or
// so large (2^64) that a product of two may pass f32's range.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float add_squares(uint32_t w, float c) {
  const bf16x2 x = __builtin_bit_cast(bf16x2, w);
  return __builtin_amdgcn_fdot2_f32_bf16(x, x, c, false);
}
__device__ __forceinline__ bool not_finite(float x) { return x - x != 0.0f; }

// Buffer resource over `bytes` bytes at p (wave-uniform): loads past the end
// return zeros and stores past it are dropped, without a branch.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00027000);
}
__device__ __forceinline__ u32x4 buffer_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ __forceinline__ float buffer_load4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}

// Eight bf16 as two halves of an operand.
__device__ __forceinline__ bf16x8 join_b64(uint64_t a, uint64_t b) {
  return __builtin_bit_cast(bf16x8, u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)});
}

// The upper halves of two f32: bf16 by truncation (a finite value stays finite).
__device__ __forceinline__ uint32_t upper_bf16x2(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
}
// What they leave of the two, exact in f32, rounded to bf16.
__device__ __forceinline__ uint32_t rest_bf16x2(float a, float b, uint32_t upper) {
  // -1 in the lower and in the upper half. (Opaque: as a constant the first is
  // encoded as the f32 -1.0, which is the second.)
  uint32_t lower = 0x0000bf80u, higher = 0xbf800000u;
  asm("" : "+s"(lower), "+s"(higher));
  const bf16x2 u = __builtin_bit_cast(bf16x2, upper);
  return pack_bf16x2(__builtin_amdgcn_fdot2_f32_bf16(u, __builtin_bit_cast(bf16x2, lower), a, false),
                     __builtin_amdgcn_fdot2_f32_bf16(u, __builtin_bit_cast(bf16x2, higher), b, false));
}

// Two tiles' accumulators as an operand of 32 rows in two parts, together 16
// bits or more of each. An Inf leaves a NaN in the second.
struct RowParts {
  bf16x8 hi, lo;
};
__device__ __forceinline__ RowParts split_rows(f32x4 x, f32x4 y) {
  const u32x4 hi = {upper_bf16x2(x[0], x[1]), upper_bf16x2(x[2], x[3]), upper_bf16x2(y[0], y[1]),
                    upper_bf16x2(y[2], y[3])};
  const u32x4 lo = {rest_bf16x2(x[0], x[1], hi[0]), rest_bf16x2(x[2], x[3], hi[1]), rest_bf16x2(y[0], y[1], hi[2]),
                    rest_bf16x2(y[2], y[3], hi[3])};
  return {__builtin_bit_cast(bf16x8, hi), __builtin_bit_cast(bf16x8, lo)};
}

// ===========================================================================
// bf16 rows. One workgroup of NW waves per (sequence, segment, value head,
// slice of 16 NW columns); wave w holds columns 16 w .. of the state, all DK
// rows, in the accumulators of 16x16 tiles (lane m16 + 16 g: column m16, rows
// 4 g .. 4 g + 3), which are the operand layout of the product with q:
//   O^T = S^T Q^T      S tiles 2p and 2p + 1 as one operand of 32 rows, in two
//                      parts of bf16 (8 + 8 bits: 2^-15 of a term)
//   P   = K Q^T        tiles of 16 keys by 16 tokens dealt over the waves, decayed
//                      and masked, through LDS in two parts as well
//   O^T += V^T P^T     V^T by the transposing LDS read
//                      (With one part of S and of P each an output's error was 1.41
//                      times that of its own rounding, now it is that rounding's:
//                      one prompt of 8,192 tokens 115 -> 122 us, 8 of 300-1,500
//                      67.5 -> 77.5.)
//   S   = e^G S + K^T (w V)   w V in f32 split into three bf16 (8 + 8 + 8 bits
//                      by truncation), so that the state keeps f32's accuracy
// The order of the 32 tokens (or rows) of an operand is (4 g + e, 16 + 4 g + e)
// throughout, which is how accumulator tiles and transposing reads deliver them.
// From a chunk with an Inf or NaN in k or v (or a number of 2^64 or more), in its
// scores or in its products with the state, the segment goes on token by token:
// masked products would carry them to tokens that do not see them, and what
// overflows in a product of a chunk is not what does in the recurrence.
// ===========================================================================
// kWhole: one segment per sequence, states read and written in their slots.
// kLocal and kOutputs: the first and the last of the three launches over
// segments; the scan between them has the states of both ends. Where states
// are only for the outputs, w V takes two parts (16 bits).
enum { kWhole, kLocal, kOutputs };
template <int DK, int NW, int MODE>
__global__ void __launch_bounds__(64 * NW, NW == 8 && DK < 256 ? 4 : DK < 256 ? 2 : 1) linear_chunk_kernel(LinArgs a, LinSegs sg) {
  constexpr bool OUT = MODE != kLocal;
  constexpr int TERMS = MODE == kOutputs ? 2 : 3;  // bf16 parts of w V
  constexpr int T = 64 * NW, W = 16 * NW;  // threads, columns of the workgroup
  constexpr int KRB = DK * 2, VRB = W * 2; // LDS row bytes
  constexpr int KC = DK / 8, VC = W / 8;   // 16-byte chunks per row
  constexpr int KL = kChunk * KC / T, VL = kChunk * VC / T;  // chunks per thread
  constexpr int NP = DK / 32;              // operands of 32 state rows
  constexpr int kPlane = kChunk * 128;     // bytes of one part of the scores
  // In this order every read's offset from its lane's part fits an instruction
  // (16 bits) at k_dim 128 (apart, the vectors came last and cost 5 registers).
  struct Tiles {
    // Per token: summed log2 decay G (in 2^-17, decay_diff), scale e^G, the weight
    // e^{G_end - G}, and e^{G' - G}, G' that of the last of its 16 tokens; then the
    // chunk's whole decay. Two of each: the next chunk's are made beside this
    // chunk's products.
    int gs2[2][kChunk];
    float es2[2][kChunk], ws2[2][kChunk], rs2[2][kChunk], gend2[2];
    int odd;   // the last chunk (counted from 1) with an Inf, a NaN or 2^64 in k or v
    int late;  // the chunk with one in its scores, or in its products with the state
    uint8_t vt[kChunk * VRB];
    uint8_t pt[OUT ? 2 * kPlane : 16];  // the scores' two parts
    uint8_t kt[kChunk * KRB], qt[OUT ? kChunk * KRB : 16];
  };
  static_assert(offsetof(Tiles, vt) % 16 == 0, "tiles are read 16 bytes at a time");
  __shared__ __attribute__((aligned(16))) Tiles lds;
  auto &gs2 = lds.gs2;
  auto &es2 = lds.es2, &ws2 = lds.ws2, &rs2 = lds.rs2;
  auto &gend2 = lds.gend2;
  uint8_t *const kt = lds.kt, *const qt = lds.qt, *const pt = lds.pt, *const vt = lds.vt;
  int &odd_s = lds.odd;

  const int slices = a.DV / W, rep = a.Hv / a.Hk;
  // Workgroups that share a key head's q and k (its value heads and their
  // slices) are dealt to one XCD, whose L2 then reads them once.
  const int members = rep * slices, grp = (int)((blockIdx.x >> 3) / members) * 8 + (int)(blockIdx.x & 7);
  const int mem = (int)((blockIdx.x >> 3) % members);
  const int inst = grp / a.Hk, kh = grp % a.Hk;
  const int seg = inst % sg.nseg, b = inst / sg.nseg;
  if (b >= a.B) return;
  const int h = kh * rep + mem / slices, sl = mem % slices;
  int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m16 = lane & 15, g4 = lane >> 4;
  // LDS offsets of a lane: a tile's rows are a power of two wide and swizzles
  // go by a row's low four bits, so another chunk is an XOR and another 16
  // rows an addition of a constant.
  const int tr = 4 * g4 + (m16 >> 2);  // transposing reads: its row
  int k_tr = lin_at(tr, (m16 >> 1) & 1, m16 & 1, KC, lin_tr_swz(tr, KC));
  int v_tr = lin_at(tr, (m16 >> 1) & 1, m16 & 1, VC, lin_tr_swz(tr, VC));
  int k_row = lin_at(m16, g4 >> 1, g4 & 1, KC, lin_tr_swz(m16, KC));  // 8 bytes of row m16 of K, Q and P
  int q_row = lin_at(m16, g4 >> 1, g4 & 1, KC, lin_row_swz(m16, KC));
  int p_row = lin_at(m16, g4 >> 1, g4 & 1, 8, lin_row_swz(m16, 8));
  LinSeq s;
  if (!lin_seq(a, b, MODE != kLocal && tid == 0 && seg == 0 && h == 0 && sl == 0, s)) return;
  s.row0 = __builtin_amdgcn_readfirstlane(s.row0);
  s.n = __builtin_amdgcn_readfirstlane(s.n);
  s.src = __builtin_amdgcn_readfirstlane((int)s.src);
  s.dst = __builtin_amdgcn_readfirstlane((int)s.dst);
  const int ns = lin_nseg(sg, s.n);
  if (seg >= ns) return;
  const int t_begin = seg * sg.len, t_end = seg == ns - 1 ? s.n : t_begin + sg.len;

  const int64_t plane = (int64_t)a.Hv * DK * a.DV;
  // The head's state: in its slot, where a lane's first element is row 4 g4 of
  // column m16 of the wave's; or between the launches, tile by tile in the
  // lanes' order.
  const int64_t hoff = (int64_t)h * DK * a.DV;
  const uint32_t lane_off = (uint32_t)(4 * g4 * a.DV + sl * W + 16 * wave + m16) * 4, srow = a.DV * 4;
  float *const frag = sg.state + ((int64_t)b * sg.nseg + seg) * plane + hoff + (sl * NW + wave) * (DK * 16) + lane * 4;
  f32x4 S[DK / 16];
  float z = 0.0f;  // a NaN where the state holds an Inf or a NaN
  const auto from = buffer(a.states + (s.src >= 0 ? s.src : 0) * plane + hoff, s.src >= 0 ? DK * srow : 0);  // none: zeros
#pragma unroll
  for (int j = 0; j < DK / 16; j++) {
    S[j] = f32x4{};
    if constexpr (MODE == kOutputs) S[j] = *reinterpret_cast<const f32x4 *>(frag + j * 256);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (MODE == kWhole) S[j][i] = buffer_load4(from, lane_off + (16 * j + i) * srow);
      z = fmaf(S[j][i], 0.0f, z);
    }
  }
  double total = 0.0, g_end = 0.0;  // summed log2 decays of the segment so far, and of this chunk (wave NW - 1)
  if (tid == 0) odd_s = lds.late = 0;

  const uint8_t *kp = static_cast<const uint8_t *>(a.k) + ((int64_t)s.row0 * a.Hk + kh) * KRB;
  const uint8_t *qp = static_cast<const uint8_t *>(a.q) + ((int64_t)s.row0 * a.Hk + kh) * KRB;
  const uint8_t *vp = static_cast<const uint8_t *>(a.v) + ((int64_t)s.row0 * a.Hv + h) * a.DV * 2 + sl * VRB;
  const int64_t krs = (int64_t)a.Hk * KRB, vrs = (int64_t)a.Hv * a.DV * 2;  // row strides
  u32x4 kr[KL], qr[OUT ? KL : 1], vr[VL];
  uint32_t k_off = tid / KC * (uint32_t)krs + tid % KC * 16, v_off = tid / VC * (uint32_t)vrs + tid % VC * 16;
  uint32_t o_off = m16 * (uint32_t)vrs + (wave * 16 + 4 * g4) * 2;
  // The loop has no branch around a load or a store of global memory (the
  // buffers' bounds drop them), so that a wait for the next chunk's rows does not
  // wait for the outputs stored after they were asked for.
  auto rows = [&](const uint8_t *base, int t0, int64_t stride, uint32_t bytes) {  // rows past the segment's end are zeros
    const bool any = t0 < t_end;
    return buffer(base + (any ? t0 : 0) * stride, any ? (min(kChunk, t_end - t0) - 1) * (uint32_t)stride + bytes : 0);
  };
  auto load_k = [&](int t0) {
    const auto r = rows(kp, t0, krs, KRB);
#pragma unroll
    for (int i = 0; i < KL; i++) kr[i] = buffer_load16(r, k_off + i * (T / KC) * (uint32_t)krs);
  };
  auto load_q = [&](int t0) {
    const auto r = rows(qp, t0, krs, KRB);
#pragma unroll
    for (int i = 0; i < (OUT ? KL : 0); i++) qr[i] = buffer_load16(r, k_off + i * (T / KC) * (uint32_t)krs);
  };
  auto load_v = [&](int t0) {
    const auto r = rows(vp, t0, vrs, VRB);
#pragma unroll
    for (int i = 0; i < VL; i++) vr[i] = buffer_load16(r, v_off + i * (T / VC) * (uint32_t)vrs);
  };
  // Token t0 + lane's decay, and (wave NW - 1, which has one tile of scores) a chunk's
  // vectors from it.
  auto load_g = [&](int t0) {
    const bool any = t0 < t_end;
    const uint32_t last = min(kChunk, t_end - t0) - 1, gs = a.g_stride * 4;
    return buffer_load4(buffer(a.g + (any ? (int64_t)(s.row0 + t0) * a.g_stride : 0), any ? last * gs + 4 * h + 4 : 0),
                        lane * gs + 4 * h);
  };
  float gr = load_g(t_begin);
  auto vectors = [&](int t0, int buf) {
    const double l = t0 + lane < t_end ? log2_decay(gr) : 0.0, G = wave_scan(l), end = lane_d(G, 63);
    gs2[buf][lane] = (int)rint(fmin(fmax(G, -16000.0), 16000.0) * 131072.0);
    es2[buf][lane] = exp2_f((float)G) * a.scale;
    ws2[buf][lane] = exp2_f((float)(end - G));
    rs2[buf][lane] = exp2_f((float)(__shfl(G, lane | 15) - G));
    if (lane == 0) gend2[buf] = exp2_f((float)end);
    return MODE == kLocal && __any(decay_is_zero(l)) ? end - INFINITY : end;  // (a NaN stays one)
  };
  auto stage = [&](int chunk) {  // the loaded rows into the LDS tiles
    float odd[4] = {};
    auto put = [&](const u32x4 &x, uint8_t *tile, int at, bool look) {
      if (look) {
#pragma unroll
        for (int e = 0; e < 4; e++) odd[e] = add_squares(x[e], odd[e]);
      }
      *reinterpret_cast<uint2 *>(tile + at) = make_uint2(x[0], x[1]);
      *reinterpret_cast<uint2 *>(tile + (at ^ 8)) = make_uint2(x[2], x[3]);
    };
#pragma unroll
    for (int i = 0; i < KL; i++) {
      const int r = tid / KC + i * (T / KC), c = tid % KC;
      put(kr[i], kt, lin_at(r, c, 0, KC, lin_tr_swz(r, KC)), true);
      if constexpr (OUT) put(qr[i], qt, lin_at(r, c, 0, KC, lin_row_swz(r, KC)), false);
    }
#pragma unroll
    for (int i = 0; i < VL; i++) {
      const int r = tid / VC + i * (T / VC), c = tid % VC;
      put(vr[i], vt, lin_at(r, c, 0, VC, lin_tr_swz(r, VC)), true);
    }
    if (not_finite((odd[0] + odd[1]) + (odd[2] + odd[3]))) odd_s = chunk;
  };

  load_k(t_begin);
  load_q(t_begin);
  load_v(t_begin);
  if constexpr (OUT) {
#pragma unroll
    for (int i = 0; i < 2 * kPlane / (16 * T); i++) *reinterpret_cast<u32x4 *>(pt + (tid + T * i) * 16) = u32x4{};
  }
  if (wave == NW - 1) g_end = vectors(t_begin, 0);
  gr = load_g(t_begin + kChunk);
  __syncthreads();  // (odd_s is set)
  stage(1);
  if (OUT && z != z) odd_s = 1;
  __syncthreads();
  int t0 = t_begin;
  for (int chunk = 1; t0 < t_end; chunk++) {
    const int nt = min(kChunk, t_end - t0);
    const int *gs = gs2[(chunk - 1) & 1];
    const float *es = es2[(chunk - 1) & 1], *ws = ws2[(chunk - 1) & 1], *rs = rs2[(chunk - 1) & 1];
    // (Opaque: the addresses made from these are formed where they are used,
    // not kept in registers over the loop.)
    asm volatile("" : "+v"(k_tr), "+v"(v_tr), "+v"(k_row), "+v"(q_row), "+v"(p_row));
    asm volatile("" : "+v"(k_off), "+v"(v_off), "+v"(o_off));
    // (And one of each per 16 tokens: two reads off the same register would be
    // paired across tokens, into registers that no operand has in that order.)
    int q_at[4] = {q_row, q_row, q_row, q_row}, p_at[4] = {p_row, p_row, p_row, p_row};
    int k_at[4] = {k_row, k_row, k_row, k_row};
    asm volatile("" : "+v"(q_at[1]), "+v"(q_at[2]), "+v"(q_at[3]), "+v"(p_at[1]), "+v"(p_at[2]), "+v"(p_at[3]),
                 "+v"(k_at[1]), "+v"(k_at[2]), "+v"(k_at[3]));
    if (odd_s == chunk) break;  // uniform over the workgroup
    // The next chunk's rows are asked for in three parts between the products.
    load_k(t0 + kChunk);
    double next_end = 0.0;
    if (wave == NW - 1) next_end = vectors(t0 + kChunk, chunk & 1);
    gr = load_g(t0 + 2 * kChunk);

    f32x4 acc[4];
    float bad[2] = {};  // a NaN where a product is an Inf or a NaN
    if constexpr (OUT) {
      // Scores: the ten tiles of 16 tokens (columns) by 16 keys on and below the
      // diagonal, up to three per wave; the two above it that a product of 32
      // keys reaches over are zeros from the start. A wave's tiles are straight
      // code: with a branch round each they wait for one another.
      auto read16 = [&](const uint8_t *tile, int at, int p) {  // 16 rows by 32 columns from column 32 p on
        return join_b64(*reinterpret_cast<const uint64_t *>(tile + (at ^ (p * 64))),
                        *reinterpret_cast<const uint64_t *>(tile + (at ^ (p * 64 + 32))));
      };
      // N tiles from n0 on. Four waves form O^T from the state with them, off one
      // read of q (their n0 is a constant, and so is the tile of q each takes).
      auto scores = [&](auto count, int n0, int step) {
        constexpr int N = decltype(count)::value;
        int tq[N], st[N];
        f32x4 c[N], r[N];
        i32x4 gk[N];
        int gt[N], e[N];
#pragma unroll
        for (int u = 0; u < N; u++) {  // tiles by rows from the last one: (3, 0) .. (3, 3), (2, 0) .. (0, 0)
          const int n = n0 + step * u;
          tq[u] = n < 4 ? 3 : n < 7 ? 2 : n < 9 ? 1 : 0;
          st[u] = n - (n < 4 ? 0 : n < 7 ? 4 : n < 9 ? 7 : 9);
          gt[u] = gs[16 * tq[u] + m16];
          e[u] = gs[16 * st[u] + 15];
          gk[u] = *reinterpret_cast<const i32x4 *>(&gs[16 * st[u] + 4 * g4]);
          r[u] = *reinterpret_cast<const f32x4 *>(&rs[16 * st[u] + 4 * g4]);
        }
#pragma unroll
        for (int p = 0; p < NP; p++) {
          bf16x8 q[4];
          if constexpr (NW == 4) {
            const RowParts sf = split_rows(S[2 * p], S[2 * p + 1]);
#pragma unroll
            for (int tt = 0; tt < 4; tt++) {
              q[tt] = read16(qt + tt * 16 * KRB, q_at[tt], p);
              acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sf.hi, q[tt], p ? acc[tt] : f32x4{}, 0, 0, 0);
            }
#pragma unroll
            for (int tt = 0; tt < 4; tt++)
              acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sf.lo, q[tt], acc[tt], 0, 0, 0);
          }
#pragma unroll
          for (int u = 0; u < N; u++) {
            const bf16x8 qf = NW == 4 ? q[tq[u]] : read16(qt + tq[u] * 16 * KRB, q_at[u], p);
            const bf16x8 kf = read16(kt + st[u] * 16 * KRB, k_at[u], p);
            c[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf, p ? c[u] : f32x4{}, 0, 0, 0);
          }
        }
#pragma unroll
        for (int u = 0; u < N; u++) {
          if (st[u] < tq[u]) {  // e^{G_t - G_end of tile} e^{G_end of tile - G_k}: one exponential per lane
            const float f = exp2_f(decay_diff(gt[u], e[u])) * a.scale;
#pragma unroll
            for (int i = 0; i < 4; i++) c[u][i] *= f * r[u][i];
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {  // (selected, not multiplied: past t it may be anything)
              const float f = exp2_f(decay_diff(gt[u], gk[u][i])) * a.scale;
              c[u][i] = 4 * g4 + i <= m16 ? c[u][i] * f : 0.0f;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; i++) bad[i & 1] = fmaf(c[u][i], 0.0f, bad[i & 1]);
          uint8_t *at = pt + (p_row ^ (st[u] * 32)) + tq[u] * 16 * 128;
          const uint32_t h0 = upper_bf16x2(c[u][0], c[u][1]), h1 = upper_bf16x2(c[u][2], c[u][3]);
          *reinterpret_cast<uint64_t *>(at) = (uint64_t)h1 << 32 | h0;
          *reinterpret_cast<uint64_t *>(at + kPlane) =
              (uint64_t)rest_bf16x2(c[u][2], c[u][3], h1) << 32 | rest_bf16x2(c[u][0], c[u][1], h0);
        }
      };
      constexpr int kFull = NW == 8 ? 2 : 3;  // that many waves have that many tiles, the others one
      const std::integral_constant<int, kFull> full;
      const std::integral_constant<int, 1> one;
      if constexpr (NW == 8) {
        if (wave < kFull) scores(full, wave, 8);
        else scores(one, wave, 0);
      } else {
        if (wave == 0) scores(full, 0, 1);
        else if (wave == 1) scores(full, 3, 1);
        else if (wave == 2) scores(full, 6, 1);
        else scores(one, 9, 0);
      }
      load_q(t0 + kChunk);
      // O^T from the state: eight waves, which have no registers for more at once.
#pragma unroll
      for (int p = 0; p < (NW == 8 ? NP : 0); p++) {
        const RowParts sf = split_rows(S[2 * p], S[2 * p + 1]);
#pragma unroll
        for (int tt = 0; tt < 4; tt++) {
          const bf16x8 q = read16(qt + tt * 16 * KRB, q_at[tt], p);
          acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sf.hi, q, p ? acc[tt] : f32x4{}, 0, 0, 0);
          acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sf.lo, q, acc[tt], 0, 0, 0);
        }
      }
#pragma unroll
      for (int tt = 0; tt < 4; tt++) {
#pragma unroll
        for (int i = 0; i < 4; i++) bad[i & 1] = fmaf(acc[tt][i], 0.0f, bad[i & 1]);
        acc[tt] *= es[16 * tt + m16];
      }
      if (bad[0] + bad[1] != 0.0f) lds.late = chunk;
      __syncthreads();  // the scores are written
    }
    const float dend = gend2[(chunk - 1) & 1];
    if constexpr (!OUT) {
      // (An Inf in a state without outputs only meets the chunk's decay.)
      if (__builtin_amdgcn_readfirstlane(__float_as_int(dend)) == 0) {
#pragma unroll
        for (int j = 0; j < DK / 16; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) bad[i & 1] = fmaf(S[j][i], 0.0f, bad[i & 1]);
        if (bad[0] + bad[1] != 0.0f) lds.late = chunk;
        __syncthreads();
      }
    }
    const int late = lds.late;

    load_v(t0 + kChunk);
    bf16x8 vf[2];  // [32 tokens][16 columns]
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const uint8_t *at = vt + (v_tr ^ (wave * 32)) + 32 * x * VRB;
      const i16x4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)at);
      const i16x4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(at + 16 * VRB));
      vf[x] = join_b64(__builtin_bit_cast(uint64_t, lo), __builtin_bit_cast(uint64_t, hi));
    }
    if (late == chunk) break;  // uniform over the workgroup
    if constexpr (OUT) {
      const auto ob = buffer(static_cast<uint8_t *>(a.o) + ((int64_t)(s.row0 + t0) * a.Hv + h) * a.DV * 2 + sl * VRB,
                             (uint32_t)(nt - 1) * (uint32_t)vrs + VRB);
#pragma unroll
      for (int tt = 0; tt < 4; tt++) {
#pragma unroll
        for (int x = 0; x <= tt / 2; x++) {
#pragma unroll
          for (int u = 0; u < 2; u++) {
            const uint8_t *at = pt + u * kPlane + tt * 16 * 128;
            const bf16x8 pf = join_b64(*reinterpret_cast<const uint64_t *>(at + (p_at[tt] ^ (x * 64))),
                                       *reinterpret_cast<const uint64_t *>(at + (p_at[tt] ^ (x * 64 + 32))));
            acc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[x], pf, acc[tt], 0, 0, 0);
          }
        }
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{pack_bf16x2(acc[tt][0], acc[tt][1]), pack_bf16x2(acc[tt][2], acc[tt][3])},
                                              ob, o_off + 16 * tt * (uint32_t)vrs, 0, 0);
      }
    }
    total += g_end;  // (past the last exit of the loop body)
    g_end = next_end;
#pragma unroll
    for (int j = 0; j < DK / 16; j++) S[j] *= dend;
#pragma unroll
    for (int x = 0; x < 2; x++) {  // 32 tokens
      uint32_t wv[TERMS][4];       // w V: high, middle and low bits
      const f32x4 w0 = *reinterpret_cast<const f32x4 *>(&ws[32 * x + 4 * g4]);
      const f32x4 w1 = *reinterpret_cast<const f32x4 *>(&ws[32 * x + 16 + 4 * g4]);
      const u32x4 raw = __builtin_bit_cast(u32x4, vf[x]);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float f[2] = {bf16_lo(raw[e]), bf16_hi(raw[e])};
        f[0] *= e < 2 ? w0[2 * e] : w1[2 * e - 4];
        f[1] *= e < 2 ? w0[2 * e + 1] : w1[2 * e - 3];
#pragma unroll
        for (int u = 0; u < TERMS; u++) {
          const uint32_t b0 = __float_as_uint(f[0]), b1 = __float_as_uint(f[1]);
          wv[u][e] = __builtin_amdgcn_perm(b1, b0, 0x07060302);  // the upper halves
          f[0] -= __uint_as_float(b0 & 0xffff0000u);
          f[1] -= __uint_as_float(b1 & 0xffff0000u);
        }
      }
#pragma unroll
      for (int j = 0; j < DK / 16; j++) {
        const uint8_t *at = kt + (k_tr ^ (j * 32)) + 32 * x * KRB;
        const i16x4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)at);
        const i16x4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(at + 16 * KRB));
        const bf16x8 kf = join_b64(__builtin_bit_cast(uint64_t, lo), __builtin_bit_cast(uint64_t, hi));
#pragma unroll
        for (int u = 0; u < TERMS; u++)
          S[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              kf, __builtin_bit_cast(bf16x8, u32x4{wv[u][0], wv[u][1], wv[u][2], wv[u][3]}), S[j], 0, 0, 0);
      }
    }
    t0 += kChunk;
    if (t0 >= t_end) break;
    __syncthreads();  // this chunk's tiles are read
    stage(chunk + 1);
    __syncthreads();
  }

  // From the first chunk that cannot be computed as one on: token by token, as the
  // recurrence has it. Lane: column m16 of each tile, its rows' share of an
  // output, summed over the four lane groups.
#pragma unroll 1
  for (; t0 < t_end; t0++) {
    const int64_t krow = ((int64_t)(s.row0 + t0) * a.Hk + kh) * DK + 4 * g4;
    const int64_t vrow = ((int64_t)(s.row0 + t0) * a.Hv + h) * a.DV + sl * W + 16 * wave + m16;
    const double l = log2_decay(a.g[(int64_t)(s.row0 + t0) * a.g_stride + h]);
    const float d = exp2f((float)l);
    total += decay_is_zero(l) ? -INFINITY : l;
    const float v = __uint_as_float((uint32_t)static_cast<const uint16_t *>(a.v)[vrow] << 16);
    float o = 0.0f;
#pragma unroll
    for (int j = 0; j < DK / 16; j++) {
      const uint2 kw = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.k) + krow + 16 * j);
      const float k[4] = {bf16_lo(kw.x), bf16_hi(kw.x), bf16_lo(kw.y), bf16_hi(kw.y)};
      float q[4] = {};
      if constexpr (OUT) {
        const uint2 qw = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(a.q) + krow + 16 * j);
        q[0] = bf16_lo(qw.x), q[1] = bf16_hi(qw.x), q[2] = bf16_lo(qw.y), q[3] = bf16_hi(qw.y);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        S[j][i] = d * S[j][i] + k[i] * v;
        if constexpr (OUT) o += q[i] * S[j][i];
      }
    }
    if constexpr (OUT) {
      o += __shfl_xor(o, 16);
      o += __shfl_xor(o, 32);
      if (g4 == 0) static_cast<uint16_t *>(a.o)[vrow] = (uint16_t)f32_to_bf16_bits(o * a.scale);
    }
  }

  if constexpr (MODE == kLocal) {
    if (tid == 64 * (NW - 1) && sl == 0)
      sg.decay[((int64_t)b * sg.nseg + seg) * a.Hv + h] = segment_decay(total);
#pragma unroll
    for (int j = 0; j < DK / 16; j++) *reinterpret_cast<f32x4 *>(frag + j * 256) = S[j];
  } else if constexpr (MODE == kWhole) {
    // (Formed again: not kept in a register over the loop.)
    int m = m16, g = g4;
    asm volatile("" : "+v"(m), "+v"(g));
    const uint32_t s_off = (uint32_t)(4 * g * a.DV + sl * W + 16 * wave + m) * 4;
    const auto to = buffer(a.states + s.dst * plane + hoff, DK * srow);
#pragma unroll
    for (int j = 0; j < DK / 16; j++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[j][i]), to, s_off + (16 * j + i) * srow, 0, 0);
  }
}

// ===========================================================================
// f32 rows: the same products on v_mfma_f32_16x16x4 (a fifth of the bf16 rate
// counted with its three parts, and exact), chunks of 32 tokens so that the
// tiles of k_dim 256 leave room for two workgroups per CU. Four waves on 64
// columns. The four products of an operand step take rows (or tokens) 4 g + i
// for i = 0 .. 3, again what accumulators and 16-byte reads deliver. Tiles are
// swizzled by chunk c ^ (r & 15): free of conflicts for 16-byte reads of one
// chunk of 16 rows and for 4-byte reads of 16 columns of rows 4 g + i.
// Decays are differences of sums kept in two floats, exact to f32's last bits.
// ===========================================================================
constexpr int kChunkF32 = 32;

template <int DK, int MODE>
__global__ void __launch_bounds__(256, DK == 256 ? 1 : 2) linear_chunk_f32_kernel(LinArgs a, LinSegs sg) {
  constexpr bool OUT = MODE != kLocal;
  constexpr int C = kChunkF32, W = 64, KC = DK / 4, VC = W / 4;  // 16-byte chunks per row
  constexpr int KL = C * KC / 256, VL = C * VC / 256;
  __shared__ __attribute__((aligned(16))) float kt[C * DK], qt[OUT ? C * DK : 4], vt[C * W], pt[OUT ? C * C : 4];
  // Summed log2 decay (two floats), scale e^G, and e^{G_end - G} per token.
  __shared__ __attribute__((aligned(16))) float gh[C], gl[C], es[C], ws[C];
  __shared__ float gend_s;
  __shared__ int odd_s;   // the last chunk (counted from 1) with an Inf, a NaN or 2^64 in k or v
  __shared__ int late_s;  // the chunk with one in its scores, or in its products with the state

  const int slices = a.DV / W, rep = a.Hv / a.Hk;
  const int members = rep * slices, grp = (int)((blockIdx.x >> 3) / members) * 8 + (int)(blockIdx.x & 7);
  const int mem = (int)((blockIdx.x >> 3) % members);
  const int inst = grp / a.Hk, kh = grp % a.Hk;
  const int seg = inst % sg.nseg, b = inst / sg.nseg;
  if (b >= a.B) return;
  const int h = kh * rep + mem / slices, sl = mem % slices;
  int tid = threadIdx.x;
  const int lane = tid & 63;
  int m16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  LinSeq s;
  if (!lin_seq(a, b, MODE != kLocal && tid == 0 && seg == 0 && h == 0 && sl == 0, s)) return;
  s.row0 = __builtin_amdgcn_readfirstlane(s.row0);
  s.n = __builtin_amdgcn_readfirstlane(s.n);
  s.src = __builtin_amdgcn_readfirstlane((int)s.src);
  s.dst = __builtin_amdgcn_readfirstlane((int)s.dst);
  const int ns = lin_nseg(sg, s.n);
  if (seg >= ns) return;
  const int t_begin = seg * sg.len, t_end = seg == ns - 1 ? s.n : t_begin + sg.len;

  const int64_t plane = (int64_t)a.Hv * DK * a.DV, hoff = (int64_t)h * DK * a.DV;
  uint32_t lane_off = (uint32_t)(4 * g4 * a.DV + sl * W + 16 * wave + m16) * 4, srow = a.DV * 4;
  float *const frag = sg.state + ((int64_t)b * sg.nseg + seg) * plane + hoff + (sl * 4 + wave) * (DK * 16) + lane * 4;
  f32x4 S[DK / 16];
  float z = 0.0f;  // a NaN where the state holds an Inf or a NaN
  const auto from = buffer(a.states + (s.src >= 0 ? s.src : 0) * plane + hoff, s.src >= 0 ? DK * srow : 0);  // none: zeros
#pragma unroll
  for (int j = 0; j < DK / 16; j++) {
    S[j] = f32x4{};
    if constexpr (MODE == kOutputs) S[j] = *reinterpret_cast<const f32x4 *>(frag + j * 256);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (MODE == kWhole) S[j][i] = buffer_load4(from, lane_off + (16 * j + i) * srow);
      z = fmaf(S[j][i], 0.0f, z);
    }
  }
  double total = 0.0;  // summed log2 decays of the segment so far (wave 0)
  if (tid == 0) odd_s = late_s = 0;

  const uint8_t *kp = static_cast<const uint8_t *>(a.k) + ((int64_t)s.row0 * a.Hk + kh) * (DK * 4);
  const uint8_t *qp = static_cast<const uint8_t *>(a.q) + ((int64_t)s.row0 * a.Hk + kh) * (DK * 4);
  const uint8_t *vp = static_cast<const uint8_t *>(a.v) + ((int64_t)s.row0 * a.Hv + h) * a.DV * 4 + sl * (W * 4);
  const int64_t krs = (int64_t)a.Hk * DK * 4, vrs = (int64_t)a.Hv * a.DV * 4;  // row strides
  f32x4 kr[KL], qr[OUT ? KL : 1], vr[VL];
  float gr = 0.0f;
  auto load = [&](int t0) {  // rows past the segment's end are zeros
    const bool any = t0 < t_end;
    const uint32_t last = min(C, t_end - t0) - 1;
    const int64_t at = any ? t0 : 0;
    const uint32_t kb = any ? last * (uint32_t)krs + DK * 4 : 0;
    const auto rk = buffer(kp + at * krs, kb), rq = buffer(qp + at * krs, kb);
    const auto rv = buffer(vp + at * vrs, any ? last * (uint32_t)vrs + W * 4 : 0);
#pragma unroll
    for (int i = 0; i < KL; i++) {
      const uint32_t off = (tid / KC + i * (256 / KC)) * (uint32_t)krs + tid % KC * 16;
      kr[i] = __builtin_bit_cast(f32x4, buffer_load16(rk, off));
      if constexpr (OUT) qr[i] = __builtin_bit_cast(f32x4, buffer_load16(rq, off));
    }
#pragma unroll
    for (int i = 0; i < VL; i++)
      vr[i] = __builtin_bit_cast(
          f32x4, buffer_load16(rv, (tid / VC + i * (256 / VC)) * (uint32_t)vrs + tid % VC * 16));
    const uint32_t gs = a.g_stride * 4;
    gr = buffer_load4(buffer(a.g + (any ? (int64_t)(s.row0 + t0) * a.g_stride : 0), any ? last * gs + 4 * h + 4 : 0),
                      (lane & (C - 1)) * gs + 4 * h);
  };
  // Element (r, c) of a tile of cpr chunks per row.
  auto at = [](int r, int c, int cpr) { return r * cpr * 4 + ((c >> 2) ^ (r & 15)) * 4 + (c & 3); };
  auto read4 = [&](const float *tile, int r, int c, int cpr) {
    return *reinterpret_cast<const f32x4 *>(tile + at(r, c, cpr));
  };

  load(t_begin);
  int chunk = 0, t0 = t_begin;
  for (; t0 < t_end; t0 += C) {
    const int nt = min(C, t_end - t0);
    chunk++;
    // (Opaque: addresses are formed where they are used, not kept over the loop.)
    asm volatile("" : "+v"(tid), "+v"(m16), "+v"(g4), "+v"(lane_off));
    __syncthreads();  // the previous chunk's tiles are read
    float odd = chunk == 1 && OUT ? z : 0.0f;
#pragma unroll
    for (int i = 0; i < KL; i++) {
      const int r = tid / KC + i * (256 / KC), c = tid % KC * 4;
      *reinterpret_cast<f32x4 *>(kt + at(r, c, KC)) = kr[i];
      if constexpr (OUT) *reinterpret_cast<f32x4 *>(qt + at(r, c, KC)) = qr[i];
#pragma unroll
      for (int e = 0; e < 4; e++) odd = fmaf(kr[i][e], kr[i][e], odd);
    }
#pragma unroll
    for (int i = 0; i < VL; i++) {
      const int r = tid / VC + i * (256 / VC), c = tid % VC * 4;
      *reinterpret_cast<f32x4 *>(vt + at(r, c, VC)) = vr[i];
#pragma unroll
      for (int e = 0; e < 4; e++) odd = fmaf(vr[i][e], vr[i][e], odd);
    }
    if (not_finite(odd)) odd_s = chunk;
    double end = 0.0;
    if (wave == 0) {
      const double l = lane < nt ? log2_decay(gr) : 0.0, G = wave_scan(l);
      end = lane_d(G, 63);
      if (lane < C) {
        gh[lane] = (float)G;
        gl[lane] = (float)(G - (double)(float)G);
        es[lane] = exp2_f((float)G) * a.scale;
        ws[lane] = exp2_f((float)(end - G));
      }
      if (lane == 0) gend_s = exp2_f((float)end);
      if (MODE == kLocal && __any(decay_is_zero(l))) end -= INFINITY;  // (a NaN stays one)
    }
    __syncthreads();
    if (odd_s == chunk) break;  // uniform over the workgroup
    load(t0 + C);

    f32x4 acc[2];
    float bad = 0.0f;  // a NaN where a product is an Inf or a NaN
    if constexpr (OUT) {
      // Scores: one tile of 16 tokens (columns) by 16 keys per wave; the one
      // that no column sees comes out as zeros.
      const int tq = wave & 1, st = wave >> 1, t = 16 * tq + m16;
      f32x4 c[4] = {};  // four chains
#pragma unroll
      for (int j = 0; j < DK / 16; j++) {
        const f32x4 kf = read4(kt, 16 * st + m16, 16 * j + 4 * g4, KC), qf = read4(qt, t, 16 * j + 4 * g4, KC);
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[i], qf[i], c[i], 0, 0, 0);
      }
      const f32x4 r = (c[0] + c[1]) + (c[2] + c[3]);
      f32x4 p;
#pragma unroll
      for (int i = 0; i < 4; i++) {  // (selected, not multiplied: past t it may be anything)
        const int k = 16 * st + 4 * g4 + i;
        const float e = exp2_f((gh[t] - gh[k]) + (gl[t] - gl[k])) * a.scale;
        p[i] = k <= t ? r[i] * e : 0.0f;
        bad = fmaf(p[i], 0.0f, bad);
      }
      *reinterpret_cast<f32x4 *>(pt + t * C + ((4 * st + g4) ^ (t & 7)) * 4) = p;
      // O^T from the state.
#pragma unroll
      for (int tt = 0; tt < 2; tt++) {
        f32x4 o[2] = {};
#pragma unroll
        for (int j = 0; j < DK / 16; j++) {
          const f32x4 qf = read4(qt, 16 * tt + m16, 16 * j + 4 * g4, KC);
#pragma unroll
          for (int i = 0; i < 4; i++)
            o[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[j][i], qf[i], o[i & 1], 0, 0, 0);
        }
        acc[tt] = o[0] + o[1];
#pragma unroll
        for (int i = 0; i < 4; i++) bad = fmaf(acc[tt][i], 0.0f, bad);
        acc[tt] *= es[16 * tt + m16];
      }
      if (bad != 0.0f) late_s = chunk;
      __syncthreads();  // the scores are written
    }
    const float dend = gend_s;
    if constexpr (!OUT) {
      // (An Inf in a state without outputs only meets the chunk's decay.)
      if (__builtin_amdgcn_readfirstlane(__float_as_int(dend)) == 0) {
#pragma unroll
        for (int j = 0; j < DK / 16; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) bad = fmaf(S[j][i], 0.0f, bad);
        if (bad != 0.0f) late_s = chunk;
        __syncthreads();
      }
    }
    const int late = late_s;
    float vf[2][4];  // [16 tokens][4 g + i] of the wave's columns
#pragma unroll
    for (int st = 0; st < 2; st++)
#pragma unroll
      for (int i = 0; i < 4; i++) vf[st][i] = vt[at(16 * st + 4 * g4 + i, 16 * wave + m16, VC)];
    if (late == chunk) break;  // uniform over the workgroup
    total += end;
    if constexpr (OUT) {
      const auto ob = buffer(static_cast<uint8_t *>(a.o) + ((int64_t)(s.row0 + t0) * a.Hv + h) * a.DV * 4 + sl * (W * 4),
                             (uint32_t)(nt - 1) * (uint32_t)vrs + W * 4);
#pragma unroll
      for (int tt = 0; tt < 2; tt++) {
        const int t = 16 * tt + m16;
#pragma unroll
        for (int st = 0; st <= tt; st++) {
          const f32x4 p = *reinterpret_cast<const f32x4 *>(pt + t * C + ((4 * st + g4) ^ (t & 7)) * 4);
#pragma unroll
          for (int i = 0; i < 4; i++) acc[tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[st][i], p[i], acc[tt], 0, 0, 0);
        }
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[tt]), ob,
                                               t * (uint32_t)vrs + (16 * wave + 4 * g4) * 4, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < DK / 16; j++) S[j] *= dend;
#pragma unroll
    for (int st = 0; st < 2; st++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = 16 * st + 4 * g4 + i;
        const float wv = vf[st][i] * ws[r];
#pragma unroll
        for (int j = 0; j < DK / 16; j++)
          S[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(kt[at(r, 16 * j + m16, KC)], wv, S[j], 0, 0, 0);
      }
  }

  // Token by token from there on, as the bf16 form.
#pragma unroll 1
  for (; t0 < t_end; t0++) {
    asm volatile("" : "+v"(m16), "+v"(g4));
    const int64_t krow = ((int64_t)(s.row0 + t0) * a.Hk + kh) * DK + 4 * g4;
    const int64_t vrow = ((int64_t)(s.row0 + t0) * a.Hv + h) * a.DV + sl * W + 16 * wave + m16;
    const double l = log2_decay(a.g[(int64_t)(s.row0 + t0) * a.g_stride + h]);
    const float d = exp2f((float)l), v = static_cast<const float *>(a.v)[vrow];
    total += decay_is_zero(l) ? -INFINITY : l;
    float o = 0.0f;
#pragma unroll
    for (int j = 0; j < DK / 16; j++) {
      const f32x4 k = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.k) + krow + 16 * j);
      const f32x4 q = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.q) + krow + 16 * j);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        S[j][i] = d * S[j][i] + k[i] * v;
        o += q[i] * S[j][i];
      }
    }
    if constexpr (OUT) {
      o += __shfl_xor(o, 16);
      o += __shfl_xor(o, 32);
      if (g4 == 0) static_cast<float *>(a.o)[vrow] = o * a.scale;
    }
  }

  if constexpr (MODE == kLocal) {
    if (tid == 0 && sl == 0) sg.decay[((int64_t)b * sg.nseg + seg) * a.Hv + h] = segment_decay(total);
#pragma unroll
    for (int j = 0; j < DK / 16; j++) *reinterpret_cast<f32x4 *>(frag + j * 256) = S[j];
  } else if constexpr (MODE == kWhole) {
    const auto to = buffer(a.states + s.dst * plane + hoff, DK * srow);
#pragma unroll
    for (int j = 0; j < DK / 16; j++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[j][i]), to, lane_off + (16 * j + i) * srow, 0, 0);
  }
}

// The scan over segments: from the state a sequence begins with and each
// segment's local state, the state before every segment (in place of its
// local one) and the sequence's last, into its slot. Elementwise; a thread
// takes four elements, which are four rows of one column in the order that
// states have between the launches.
__global__ void __launch_bounds__(256) linear_scan_kernel(LinArgs a, LinSegs sg, int DK) {
  const int elems = DK * a.DV, per = elems / 1024;
  const int part = blockIdx.x % per, h = (blockIdx.x / per) % a.Hv, b = blockIdx.x / (per * a.Hv);
  LinSeq s;
  if (!lin_seq(a, b, false, s)) return;
  const int ns = lin_nseg(sg, s.n);
  const int64_t plane = (int64_t)a.Hv * elems, hoff = (int64_t)h * elems;
  const int f = part * 256 + threadIdx.x, lane = f & 63, tile = f >> 6;  // tiles: 16 columns, then their rows
  const int row = tile % (DK / 16) * 16 + (lane >> 4) * 4, col = tile / (DK / 16) * 16 + (lane & 15);
  const int64_t slot_off = hoff + (int64_t)row * a.DV + col;
  f32x4 S = {};
  if (s.src >= 0)
#pragma unroll
    for (int i = 0; i < 4; i++) S[i] = (a.states + s.src * plane + slot_off)[i * a.DV];
  float *at = sg.state + (int64_t)b * sg.nseg * plane + hoff + f * 4;
  const float *dec = sg.decay + (int64_t)b * sg.nseg * a.Hv + h;
  constexpr int U = 8;  // segments loaded ahead
  for (int j0 = 0; j0 < ns; j0 += U) {
    f32x4 l[U];
    float d[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int j = min(j0 + u, ns - 1);
      l[u] = *reinterpret_cast<const f32x4 *>(at + j * plane);
      d[u] = dec[(int64_t)j * a.Hv];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (j0 + u >= ns) break;
      *reinterpret_cast<f32x4 *>(at + (j0 + u) * plane) = S;
      // (An infinity stays one under a product of decays that is 0 only by
      // underflow; a decay of 0 makes it a NaN.)
      const bool gone = d[u] < 1.17549435e-38f && !signbit(d[u]);
#pragma unroll
      for (int i = 0; i < 4; i++) S[i] = (gone && isinf(S[i]) ? S[i] : d[u] * S[i]) + l[u][i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) (a.states + s.dst * plane + slot_off)[i * a.DV] = S[i];
}

// ---- host side ------------------------------------------------------------------

static uint64_t segs_bytes(const StatePool *p, int64_t num_seqs, int64_t nseg) {
  const uint64_t n = (uint64_t)num_seqs * nseg;
  return n * p->state_elems * 4 + ((n * p->desc.num_v_heads * 4 + 15) & ~15ull);
}

// NW 0: f32 rows.
template <int DK, int NW, int MODE>
static void launch_chunks(const LinArgs &a, const LinSegs &sg, hipStream_t hs) {
  const int64_t groups = ((int64_t)a.B * sg.nseg * a.Hk + 7) / 8 * 8;
  const dim3 grid((unsigned)(groups * (a.Hv / a.Hk) * (a.DV / (NW ? 16 * NW : 64))));
  if constexpr (NW) hipLaunchKernelGGL((linear_chunk_kernel<DK, NW, MODE>), grid, dim3(64 * NW), 0, hs, a, sg);
  else hipLaunchKernelGGL((linear_chunk_f32_kernel<DK, MODE>), grid, dim3(256), 0, hs, a, sg);
}

// How a batch is computed.
struct LinPlan {
  int waves;      // per workgroup: 4 (64 columns) or 8 (128)
  int nseg, len;  // segments per sequence, tokens of one
};

// The costs are measured ones in microseconds at a k_dim of 128 (f32: 64) on 256
// CUs: whole sequences, 4.5 (f32: 2.5) and `lone` per chunk of 64 tokens of the
// longest, or `full` per chunk and CU (of 128 columns; f32: 64); segments, `seg`
// per chunk of one round of workgroups or `segs` of each of several, 14 for three
// launches, and the states between them, written, scanned and read at 5 TB/s. A
// chunk's products grow with k_dim, its latency less. Measured against the other
// way: 1,000 tokens of 32 heads of 128 in segments 38 us (whole 54), 4,000 80
// (199), 2 prompts of 800 of 28 heads whole 47 (57), 4 of 600 of 8 heads of 256 in
// segments 48 (61), 8 of 300 of 2 heads of 64 whole 17 (20); f32 1,000 tokens of 14
// heads of 64 in segments 28 (113), 8 of 300 whole 40 (44), 2 of 800 of 32 heads of
// 128 in segments 124 (136).
static LinPlan plan_extend(const StatePool *p, int64_t num_seqs, int64_t num_tokens, int64_t max_q_len,
                           uint64_t ws_bytes) {
  const mkv_state_desc &d = p->desc;
  const bool f32 = d.dtype == MKV_DTYPE_F32;
  // Chunks of the longest sequence (max_q_len may be a loose bound).
  const int64_t longest = std::max<int64_t>(1, (std::min(max_q_len, num_tokens) + kChunk - 1) / kChunk);
  const int64_t chunks = std::min(num_seqs * longest, num_tokens / kChunk + num_seqs);
  const int cols = f32 || d.v_dim == 64 ? 64 : 128;  // of a workgroup over segments
  const double load = (double)chunks * d.num_v_heads * d.v_dim / (f32 ? 64 : 128) / p->cus;
  const double dim = d.k_dim / (f32 ? 64.0 : 128.0);
  const double grown = f32 ? dim : std::max(0.56 + 0.44 * dim, 0.23 + 0.77 * dim);
  const double lone = f32 ? 6.8 * std::min(dim, (1.0 + dim) / 2) : 3.1 * grown, full = (f32 ? 5.6 : 3.3) * dim;
  const double seg = (f32 ? 8.4 : 7.4) * grown, segs = (f32 ? 6.0 : 6.2) * grown;
  LinPlan r = {cols / 16, 1, INT_MAX & ~(kChunk - 1)};
  double best = std::max((f32 ? 2.5 : 4.5) + lone * longest, full * load);
  for (int64_t want = 1; want < longest && want * segs < best; want += 1 + want / 64) {
    // Chunks of a segment, to 2%; the steps are the same whatever the workspace holds.
    const int64_t nseg = (longest + want - 1) / want;
    const uint64_t bytes = segs_bytes(p, num_seqs, nseg);
    if (bytes > ws_bytes) continue;
    // Workgroups of the fullest XCD, which has whole key heads' (5 segments each of 2
    // prompts, 28 heads over 4: 35 on 32 CUs, 57 us against 47 whole).
    const double heads = std::ceil(std::ceil((double)chunks / want) * d.num_k_heads / 8);
    const double wgs = heads * (d.num_v_heads / d.num_k_heads) * (d.v_dim / cols);
    const double rounds = std::max(1.0, std::ceil(wgs * 8 / p->cus - 0.05));
    const double t = 14.0 + 3.0 * (double)bytes / 5e6 + want * (rounds > 1.0 ? segs * rounds : seg);
    if (t < best) {
      best = t;
      r.nseg = (int)nseg;
      r.len = (int)want * kChunk;
    }
  }
  // Whole sequences of bf16 take 64 columns a workgroup while two to a CU hold
  // them all (8 prompts of 300-1,500 tokens, 28 heads: 78 us against 88 with
  // 128), else 128, which form the scores once for twice the columns.
  if (r.nseg == 1 && num_seqs * d.num_v_heads * (d.v_dim / 64) <= 2 * p->cus) r.waves = 4;
  return r;
}

template <int DK, int NW>
static void launch_plan(const StatePool *p, const LinArgs &a, const LinSegs &sg, hipStream_t hs) {
  if (sg.nseg == 1) {
    launch_chunks<DK, NW, kWhole>(a, sg, hs);
    return;
  }
  launch_chunks<DK, NW, kLocal>(a, sg, hs);
  hipLaunchKernelGGL(linear_scan_kernel, dim3((unsigned)((int64_t)a.B * a.Hv * (DK * a.DV / 1024))), dim3(256), 0, hs, a,
                     sg, DK);
  launch_chunks<DK, NW, kOutputs>(a, sg, hs);
}

static int launch_extend(StatePool *p, const LinArgs &a, int32_t max_q_len, void *ws, uint64_t ws_bytes,
                         hipStream_t hs) {
  const mkv_state_desc &d = p->desc;
  if (a.B == 0) return MKV_OK;
  const LinPlan pl = plan_extend(p, a.B, a.num_tokens, max_q_len, ws_bytes);
  const int64_t wgs = ((int64_t)a.B * pl.nseg * a.Hk + 7) / 8 * 8 * (a.Hv / a.Hk) * (d.v_dim / (16 * pl.waves));
  if (wgs * (pl.waves / 4) > kMaxGrid ||
      (pl.nseg > 1 && (int64_t)a.B * a.Hv * (d.k_dim * d.v_dim / 1024) > kMaxGrid))
    return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs * num_v_heads too large for one launch");
  LinSegs sg = {pl.nseg, pl.len, nullptr, nullptr};
  // Calls on different streams that share the pool's workspace follow one
  // another (a captured call cannot be ordered with what runs beside its graph).
  bool own_ws = false;
  if (pl.nseg > 1) {
    sg.state = static_cast<float *>(ws);
    sg.decay = sg.state + (int64_t)a.B * pl.nseg * p->state_elems;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    MKV_CHECK_HIP(hipStreamIsCapturing(hs, &st));
    own_ws = ws == p->ws && st == hipStreamCaptureStatusNone;
    if (own_ws && p->ws_used) MKV_CHECK_HIP(hipStreamWaitEvent(hs, p->ws_done, 0));
  }
  switch (d.k_dim * 10 + (d.dtype == MKV_DTYPE_BF16 ? pl.waves : 0)) {
    case 640: launch_plan<64, 0>(p, a, sg, hs); break;
    case 1280: launch_plan<128, 0>(p, a, sg, hs); break;
    case 2560: launch_plan<256, 0>(p, a, sg, hs); break;
    case 644: launch_plan<64, 4>(p, a, sg, hs); break;
    case 648: launch_plan<64, 8>(p, a, sg, hs); break;
    case 1284: launch_plan<128, 4>(p, a, sg, hs); break;
    case 1288: launch_plan<128, 8>(p, a, sg, hs); break;
    case 2564: launch_plan<256, 4>(p, a, sg, hs); break;
    default: launch_plan<256, 8>(p, a, sg, hs); break;
  }
  MKV_CHECK_LAUNCH("linear_chunk_kernel");
  if (own_ws) {
    MKV_CHECK_HIP(hipEventRecord(p->ws_done, hs));
    p->ws_used = true;
  }
  return MKV_OK;
}

}  // namespace mkv

using namespace mkv;

extern "C" int mkv_linear_extend_workspace_size(const mkv_state_pool *pool, int32_t num_seqs, int32_t num_tokens,
                                                int32_t max_q_len, uint64_t *out_bytes) {
  if (!pool || !out_bytes) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL argument");
  if (num_seqs < 0 || num_seqs > 65535 || num_tokens < 0 || max_q_len < 0)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "num_seqs must be in [0, 65535], num_tokens and max_q_len >= 0");
  const StatePool *p = reinterpret_cast<const StatePool *>(pool);
  *out_bytes = 0;
  if (num_seqs == 0) return MKV_OK;
  const LinPlan pl = plan_extend(p, num_seqs, num_tokens, max_q_len, UINT64_MAX);
  if (pl.nseg > 1) *out_bytes = segs_bytes(p, num_seqs, pl.nseg);
  return MKV_OK;
}

extern "C" int mkv_linear_extend(mkv_state_pool *pool, int32_t layer, const void *d_q, const void *d_k,
                                 const void *d_v, const float *d_log_decay, void *d_o, const int32_t *d_q_indptr,
                                 const int32_t *d_src_slots, const int32_t *d_dst_slots, int32_t num_seqs,
                                 int32_t num_tokens, int32_t max_q_len, float scale, uint32_t flags,
                                 void *d_workspace, uint64_t workspace_bytes, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  if (max_q_len < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "max_q_len < 0");
  LinArgs a;
  int rc = lin_args(p, layer, d_q, d_k, d_v, d_log_decay, d_o, d_src_slots, d_dst_slots, num_seqs, num_tokens, scale,
                    flags, a);
  if (rc) return rc;
  if (num_seqs && !d_q_indptr) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  a.q_indptr = d_q_indptr;
  DeviceGuard guard(p->device);
  if (!d_workspace) d_workspace = p->ws, workspace_bytes = p->ws_bytes;
  else if (!aligned16(d_workspace)) return set_error(MKV_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
  return launch_extend(p, a, max_q_len, d_workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int mkv_linear_extend_host(mkv_state_pool *pool, int32_t layer, const void *d_q, const void *d_k,
                                      const void *d_v, const float *d_log_decay, void *d_o, const int32_t *h_q_lens,
                                      const uint32_t *h_src_slots, const uint32_t *h_dst_slots, int32_t num_seqs,
                                      float scale, uint32_t flags, void *stream) {
  if (!pool) return set_error(MKV_ERR_INVALID_ARGUMENT, "pool is NULL");
  StatePool *p = reinterpret_cast<StatePool *>(pool);
  int rc = check_state_slots(p, h_src_slots, h_dst_slots, num_seqs);
  if (rc) return rc;
  if (num_seqs == 0) return MKV_OK;
  if (!h_q_lens) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL lengths");
  int64_t tokens = 0;
  int32_t longest = 0;
  for (int32_t b = 0; b < num_seqs; b++) {
    if (h_q_lens[b] < 0) return set_error(MKV_ERR_INVALID_ARGUMENT, "q_len[%d] = %d < 0", b, h_q_lens[b]);
    tokens += h_q_lens[b];
    longest = std::max(longest, h_q_lens[b]);
  }
  if (tokens > INT32_MAX) return set_error(MKV_ERR_INVALID_ARGUMENT, "more than 2^31 - 1 tokens");
  DeviceGuard guard(p->device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  if ((rc = refuse_capture(hs))) return rc;
  MetaSlot *sl = nullptr;
  const size_t B = (size_t)num_seqs;
  try {  // src | dst | q_indptr
    std::vector<int32_t> &st = p->stage_tmp;
    st.resize(3 * B + 1);
    std::memcpy(st.data(), h_src_slots ? h_src_slots : h_dst_slots, B * 4);
    std::memcpy(st.data() + B, h_dst_slots, B * 4);
    int32_t *ip = st.data() + 2 * B;
    ip[0] = 0;
    for (size_t b = 0; b < B; b++) ip[b + 1] = ip[b] + h_q_lens[b];
    if ((rc = stage_cached(p, p->extend_cache, st.data(), st.size(), hs, &sl))) return rc;
  } catch (const std::bad_alloc &) {
    return set_error(MKV_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
  rc = mkv_linear_extend(pool, layer, d_q, d_k, d_v, d_log_decay, d_o, sl->d + 2 * B, sl->d, sl->d + B, num_seqs,
                         (int32_t)tokens, longest, scale, flags, nullptr, 0, stream);
  const int rr = meta_release(sl, hs);
  return rc ? rc : rr;
}
