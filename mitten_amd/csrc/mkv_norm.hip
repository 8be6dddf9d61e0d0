// The step between two layers: the residual's addition, RMSNorm with weight
// (1 + w) (inference-model-qwen/src/model.rs:84-109), and the row's output in
// the model's type or in e4m3 with scales, for the projections that follow.
//
//   r = x + residual;  y = r * (mean(r^2) + eps)^-1/2 * (1 + w)
//   e4m3: a = max(max |y|, 2^-100) over a row or a group of columns,
//         scale = a / 448, stored value e4m3(y * (448 / a)).
#include <climits>
#include <cmath>

#include "mkv_internal.h"

namespace mkv {

struct NormArgs {
  const uint8_t *x, *res;  // [rows][dim]; res may be null
  const float *w;          // [dim]
  uint8_t *sum, *out;      // [rows][dim]; each may be null
  uint8_t *q8;             // [rows][dim] e4m3, or null
  float *scales;           // [rows][dim / group]
  int32_t dim, group;
  float eps;
};

constexpr float kFp8Max = 448.0f;
constexpr float kAmaxMin = 7.888609052210118e-31f;  // 2^-100: the least divisor, so that a zero row has scale > 0

// Eight consecutive elements as f32.
template <bool BF16>
__device__ __forceinline__ void load8(const uint8_t *p, int64_t i, float (&f)[8]) {
  if constexpr (BF16) {
    const uint4 r = *reinterpret_cast<const uint4 *>(p + i * 2);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; j++) f[2 * j] = bf16_lo(w[j]), f[2 * j + 1] = bf16_hi(w[j]);
  } else {
    const float4 r0 = *reinterpret_cast<const float4 *>(p + i * 4), r1 = *reinterpret_cast<const float4 *>(p + i * 4 + 16);
    f[0] = r0.x, f[1] = r0.y, f[2] = r0.z, f[3] = r0.w, f[4] = r1.x, f[5] = r1.y, f[6] = r1.z, f[7] = r1.w;
  }
}
template <bool BF16>
__device__ __forceinline__ void store8(uint8_t *p, int64_t i, const float (&f)[8]) {
  if constexpr (BF16) {
    *reinterpret_cast<uint4 *>(p + i * 2) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                       pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
    *reinterpret_cast<float4 *>(p + i * 4) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4 *>(p + i * 4 + 16) = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// Eight f32 -> e4m3 (round to nearest even, clamped to +-448; a NaN stays one).
__device__ __forceinline__ uint2 pack_fp8x8(const float (&f)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; j++) {
    float c[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float v = f[4 * j + e];
      c[e] = v > kFp8Max ? kFp8Max : v < -kFp8Max ? -kFp8Max : v;
    }
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], r, true);
    w[j] = (uint32_t)r;
  }
  return make_uint2(w[0], w[1]);
}

// Bits of |f|: as unsigned integers they order as the magnitudes do, with NaN
// above infinity, so that a maximum over them keeps a NaN.
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// One workgroup of W waves per row; thread t holds the 8-element chunks t, t +
// 64 W, ... of the row in registers, NC of them at most: one pass over memory,
// which bounds it (16,384 rows of 3,584 bf16 with a residual, sum and e4m3 out:
// 81 us, 5.1 TB/s, what a copy of that size reaches; 64 rows: 4.5 us, the
// launch and two trips to memory).
// A group's maximum is taken by each of its threads from the maxima of its
// chunks: nothing for groups of 64 or 128 columns, but reads that grow with the
// square of a large group (4,096 rows of 16,384 with groups of 512 columns 110 us,
// 2,048 152, 8,192 480; one scale per row, which goes by shuffles, 94).
template <int W, int NC, bool BF16>
__global__ void __launch_bounds__(64 * W) add_rms_norm_kernel(NormArgs a) {
  __shared__ float red_f[W];
  __shared__ uint32_t red_u[W];
  __shared__ uint32_t gmax[W * NC * 64];  // per-chunk maxima (groups)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = a.dim >> 3;
  const int64_t row = (int64_t)blockIdx.x * a.dim;
  float y[NC][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = tid + 64 * W * i;
#pragma unroll
    for (int e = 0; e < 8; e++) y[i][e] = 0.0f;
    if (c < chunks) {
      load8<BF16>(a.x, row + 8 * c, y[i]);
      if (a.res) {
        float r[8];
        load8<BF16>(a.res, row + 8 * c, r);
#pragma unroll
        for (int e = 0; e < 8; e++) y[i][e] += r[e];
      }
      if (a.sum) store8<BF16>(a.sum, row + 8 * c, y[i]);
#pragma unroll
      for (int e = 0; e < 8; e++) ss += y[i][e] * y[i][e];
    }
  }
  ss = row_sum<64>(ss);
  if (W > 1) {
    if (lane == 0) red_f[wave] = ss;
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) ss += red_f[w];
  }
  const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = tid + 64 * W * i;
    if (c < chunks) {
      float w[8];
      load8<false>(reinterpret_cast<const uint8_t *>(a.w), 8 * c, w);
      uint32_t mc = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        y[i][e] = (y[i][e] * inv) * (1.0f + w[e]);
        mc = max(mc, abs_bits(y[i][e]));
      }
      if (a.out) store8<BF16>(a.out, row + 8 * c, y[i]);
      if (a.q8 && a.group < a.dim) gmax[c] = mc;
      m = max(m, mc);
    }
  }
  if (!a.q8) return;
  if (a.group == a.dim) {
    for (int s = 1; s < 64; s <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, s));
    if (W > 1) {
      if (lane == 0) red_u[wave] = m;
      __syncthreads();
      m = 0;
#pragma unroll
      for (int w = 0; w < W; w++) m = max(m, red_u[w]);
    }
  } else {
    __syncthreads();
  }
  const int cpg = a.group >> 3;  // chunks per group
#pragma unroll
  for (int i = 0; i < NC; i++) {
    const int c = tid + 64 * W * i;
    if (c < chunks) {
      uint32_t mg = m;
      if (a.group < a.dim) {
        mg = 0;
        const int c0 = c / cpg * cpg;
        for (int j = 0; j < cpg; j++) mg = max(mg, gmax[c0 + j]);
      }
      const float amax = __uint_as_float(max(mg, __float_as_uint(kAmaxMin)));
      const float f = kFp8Max / amax;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = y[i][e] * f;
      *reinterpret_cast<uint2 *>(a.q8 + row + 8 * c) = pack_fp8x8(v);
      if (c % cpg == 0) a.scales[(int64_t)blockIdx.x * (a.dim / a.group) + c / cpg] = amax / kFp8Max;
    }
  }
}

}  // namespace mkv

using namespace mkv;

extern "C" int mkv_add_rms_norm(int device, const void *d_x, const void *d_residual, const float *d_weight,
                                float eps, int32_t num_rows, int32_t dim, int32_t dtype, void *d_sum, void *d_out,
                                void *d_fp8, float *d_scales, int32_t group, void *stream) {
  if (dtype != MKV_DTYPE_F32 && dtype != MKV_DTYPE_BF16)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (dim < 8 || dim > 16384 || dim % 8)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "dim (%d) must be a multiple of 8 in [8, 16384]", dim);
  if (num_rows < 0 || num_rows >= 1 << 24)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "num_rows (%d) must be in [0, 2^24)", num_rows);
  if (!(eps >= 0.0f && eps < INFINITY)) return set_error(MKV_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  if (num_rows == 0) return MKV_OK;
  if (!d_fp8 != !d_scales) return set_error(MKV_ERR_INVALID_ARGUMENT, "give both the e4m3 output and its scales, or neither");
  if (!d_out && !d_fp8) return set_error(MKV_ERR_INVALID_ARGUMENT, "no output asked for");
  if (d_sum && d_sum == d_out) return set_error(MKV_ERR_INVALID_ARGUMENT, "d_sum and d_out are the same");
  if (group && (!d_fp8 || group < 8 || group % 8 || group > dim || dim % group))
    return set_error(MKV_ERR_INVALID_ARGUMENT,
                     "group (%d) must be 0 (one scale per row) or a multiple of 8 that divides dim (%d), with an e4m3 output",
                     group, dim);
  // Outputs share no byte with anything else, but for the sum and the output in
  // place of x or of the residual (an element is read and written by one thread).
  const uint64_t n = (uint64_t)num_rows * dim, nb = n * (dtype == MKV_DTYPE_F32 ? 4 : 2);
  const struct {
    const void *p;
    uint64_t bytes;
  } bufs[] = {{d_sum, nb},   {d_out, nb}, {d_fp8, n},        {d_scales, (group ? n / group : num_rows) * 4ull},
              {d_weight, (uint64_t)dim * 4}, {d_x, nb}, {d_residual, nb}};
  for (int i = 0; i < 4; i++)
    for (int j = i + 1; j < 7; j++)
      if (overlap(bufs[i].p, bufs[i].bytes, bufs[j].p, bufs[j].bytes) && !(i < 2 && j >= 5 && bufs[i].p == bufs[j].p))
        return set_error(MKV_ERR_INVALID_ARGUMENT, "an output overlaps another buffer");
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0) {
    (void)hipGetLastError();
    return set_error(MKV_ERR_NO_DEVICE, "no HIP device available");
  }
  if (device < 0 || device >= ndev)
    return set_error(MKV_ERR_INVALID_ARGUMENT, "device %d out of range (%d devices)", device, ndev);
  if (!d_x || !d_weight) return set_error(MKV_ERR_INVALID_ARGUMENT, "NULL device pointer");
  const void *vec[] = {d_x, d_residual, d_weight, d_sum, d_out, d_fp8};
  for (const void *q : vec)
    if (!aligned16(q)) return set_error(MKV_ERR_INVALID_ARGUMENT, "device pointers must be 16-byte aligned");
  NormArgs a;
  a.x = static_cast<const uint8_t *>(d_x);
  a.res = static_cast<const uint8_t *>(d_residual);
  a.w = d_weight;
  a.sum = static_cast<uint8_t *>(d_sum);
  a.out = static_cast<uint8_t *>(d_out);
  a.q8 = static_cast<uint8_t *>(d_fp8);
  a.scales = d_scales;
  a.dim = dim;
  a.group = group ? group : dim;
  a.eps = eps;
  DeviceGuard guard(device);
  if (!guard.ok) return set_error(MKV_ERR_HIP, "hipSetDevice(%d) failed", device);
  hipStream_t hs = reinterpret_cast<hipStream_t>(stream);
  const bool bf = dtype == MKV_DTYPE_BF16;
  const int chunks = dim / 8;
#define MKV_NORM(WW, NN)                                                                                            \
  do {                                                                                                              \
    if (bf) hipLaunchKernelGGL((add_rms_norm_kernel<WW, NN, true>), dim3((unsigned)num_rows), dim3(64 * WW), 0, hs, a); \
    else hipLaunchKernelGGL((add_rms_norm_kernel<WW, NN, false>), dim3((unsigned)num_rows), dim3(64 * WW), 0, hs, a);   \
  } while (0)
  // Rows of up to 1,024 columns take one wave (no barrier: 16,384 rows of 512
  // 12.0 us against 20.1 with four waves, of 896 19.7 against 24.7), longer ones
  // four (of 2,048 43.6 us against 46.9 with one), with as many chunks per
  // thread as the row needs.
  if (chunks <= 64) MKV_NORM(1, 1);
  else if (chunks <= 128) MKV_NORM(1, 2);
  else if (chunks <= 256) MKV_NORM(4, 1);
  else if (chunks <= 512) MKV_NORM(4, 2);
  else if (chunks <= 1024) MKV_NORM(4, 4);
  else MKV_NORM(4, 8);
#undef MKV_NORM
  MKV_CHECK_LAUNCH("add_rms_norm_kernel");
  return MKV_OK;
}
