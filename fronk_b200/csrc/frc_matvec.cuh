// frc_matvec.cuh - products of one dense 4-bit matrix with 1-16 token vectors.
//
// y[t][r] = sum_j W[r][j] x[t][j], W in the row formats of the expert slices:
// Q4_K (w = d sc_g q - dmin mi_g, a 6-bit scale and minimum per 32 weights
// under fp16 super scales per 256) or MXFP4 (w = 2^(e-127) E2M1 per 32).
#pragma once
#include <cuda_bf16.h>

#include "../../include/fronk_b200.h"
#include "frc_device.cuh"

namespace frc {

struct MatvecParams {
  const uint8_t* w;  // rows x row_bytes
  const void* x;
  void* y;
  size_t x_stride, y_stride;  // elements between tokens
  unsigned rows, n, tokens, row_bytes;
  unsigned* status;
};

// Weight j of one row in the reference byte layout, exact in fp32.
template <unsigned TYPE>
__device__ __forceinline__ float matvec_weight(const uint8_t* row, unsigned j) {
  if (TYPE == kQ4K) {
    const uint8_t* b = row + j / 256 * 144;
    const unsigned g = j % 256 / 32, l = j % 32;
    const unsigned sc = g < 4 ? b[4 + g] & 63u : (b[8 + g] & 15u) | (b[g] >> 6) << 4;
    const unsigned mi = g < 4 ? b[8 + g] & 63u : static_cast<unsigned>(b[8 + g] >> 4) | (b[4 + g] >> 6) << 4;
    const unsigned q = b[16 + g / 2 * 32 + l] >> (4 * (g & 1)) & 15u;
    const float d = h2f(b[0] | b[1] << 8), m = h2f(b[2] | b[3] << 8);
    return __fmaf_rn(__fmul_rn(d, static_cast<float>(sc)), static_cast<float>(q), -__fmul_rn(m, static_cast<float>(mi)));
  }
  const uint8_t* b = row + j / 32 * 17;
  const unsigned l = j % 32, c = b[1 + l % 16] >> (l < 16 ? 0 : 4) & 15u;
  const float mag = byte_f((c & 4u) ? kE2M1Hi : kE2M1Lo, c & 3u);
  return (c & 8u ? -mag : mag) * pow2_m128(b[0]);
}

// Scales that are not finite (Q4_K super scales, MXFP4 exponent 255) raise
// the numeric bit; one thread a block of weights.
__global__ void matrix_check_kernel(const uint8_t* w, unsigned type, size_t blocks, unsigned* status) {
  const size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x;
  if (i >= blocks) return;
  bool bad;
  if (type == kQ4K) {
    const uint8_t* b = w + i * 144;
    bad = (b[1] & 0x7cu) == 0x7cu || (b[3] & 0x7cu) == 0x7cu;
  } else {
    bad = w[i * 17] == 255u;
  }
  if (bad) atomicOr(status, kStNumeric);
}

template <typename X>
__device__ __forceinline__ float matvec_load(const X* p);
template <>
__device__ __forceinline__ float matvec_load<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float matvec_load<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void matvec_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void matvec_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One warp a row, a lane every 32nd weight, fp32 sums.
template <unsigned TYPE, typename X, typename Y>
__global__ void __launch_bounds__(256) matvec_kernel(const MatvecParams a) {
  const unsigned row = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  const uint8_t* w = a.w + static_cast<size_t>(row) * a.row_bytes;
  const X* x = static_cast<const X*>(a.x);
  float acc[kMaxTokens] = {};
  for (unsigned j = lane; j < a.n; j += 32) {
    const float v = matvec_weight<TYPE>(w, j);
#pragma unroll
    for (unsigned t = 0; t < kMaxTokens; ++t)
      if (t < a.tokens) acc[t] = fmaf(v, matvec_load(x + t * a.x_stride + j), acc[t]);
  }
#pragma unroll
  for (unsigned t = 0; t < kMaxTokens; ++t) {
    if (t >= a.tokens) break;
    float s = acc[t];
#pragma unroll
    for (unsigned o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) {
      Y* y = static_cast<Y*>(a.y) + t * a.y_stride + row;
      matvec_store(y, s);
      if (!isfinite(matvec_load(y))) atomicOr(a.status, kStNumeric);
    }
  }
}

template <unsigned TYPE>
inline void launch_matvec(const MatvecParams& a, unsigned xt, unsigned yt, cudaStream_t s) {
  const unsigned grid = (a.rows + 7) / 8;
  if (xt == FRC_F32 && yt == FRC_F32) matvec_kernel<TYPE, float, float><<<grid, 256, 0, s>>>(a);
  else if (xt == FRC_F32) matvec_kernel<TYPE, float, __nv_bfloat16><<<grid, 256, 0, s>>>(a);
  else if (yt == FRC_F32) matvec_kernel<TYPE, __nv_bfloat16, float><<<grid, 256, 0, s>>>(a);
  else matvec_kernel<TYPE, __nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, s>>>(a);
}

}  // namespace frc
