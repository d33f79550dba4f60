// LayerNorm for training: the forward pass that keeps its statistics (and can leave its result as 8-bit blocks, the operand
// of sdamd_linear8 and its checkpoint), and the backward pass.  diffusion.py:109,117,126; clip.py:54,63,95.
//
//   mean = sum x / C,  rstd = (sum (x - mean)^2 / C + eps)^-1/2,  xh = (x - mean) rstd,  y = xh gamma + beta
//   a = dy gamma,  dx = rstd (a - sum a / C - xh sum(a xh) / C) (+ residual)
//   dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// G lanes share a row and keep it in registers, NV vectors of 8 values per lane.  Rows are read once per pass; both passes
// are bound by HBM where there are enough rows.  The variance is taken from the centred values, so a large mean costs no
// digits.
#pragma once
#include "blocks8.h"

constexpr int LNT_MAX_C = 256 * 6 * 8;

template <int N> __device__ __forceinline__ float rotate16(float v) {
  return __builtin_bit_cast(float, b8_rotate16<N>(__builtin_bit_cast(unsigned, v)));
}
// sum over the G lanes of a row (G = 256, 512: four or eight waves, through LDS; red: a float per wave of the workgroup)
template <int G> __device__ __forceinline__ float group_sum(float v, float* red) {
  constexpr int W = G < 64 ? G : 64;
  if constexpr (W > 32) v += __shfl_xor(v, 32, 64);
  if constexpr (W > 16) v += __shfl_xor(v, 16, 64);
  if constexpr (W >= 16) {                       // within 16 lanes by rotations in the vector unit, not through LDS
    v += rotate16<8>(v);
    v += rotate16<4>(v);
    v += rotate16<2>(v);
    v += rotate16<1>(v);
  } else {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  }
  if constexpr (G > 64) {
    const int first = G == 256 ? (threadIdx.x >> 8) * 4 : 0;
    __syncthreads();                             // (red may still be read from the previous call)
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[first] + red[first + 1]) + (red[first + 2] + red[first + 3]);
    if constexpr (G == 512) v += (red[4] + red[5]) + (red[6] + red[7]);
  }
  return v;
}
