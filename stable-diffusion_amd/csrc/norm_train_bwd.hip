// LayerNorm backward (norm_train.h): dx, and the weight gradients in two steps without atomics.  A workgroup walks rows
// blockIdx, blockIdx + grid, ... and keeps the sums of dy xh and dy of the columns its lanes hold in registers; at its end
// the lanes that hold the same columns are joined by shuffles within a wave and wave after wave in LDS, and the workgroup
// leaves one row of partial sums.  A second launch adds the partial rows.  Every order is fixed: the same bits every run.
#include "norm_train.h"

template <typename TX> struct RowX {             // x as values
  static __device__ __forceinline__ Raw8<TX> load(const TX* x, const unsigned char*, size_t row, int c, int C) { return raw8_load(x + row * C, c, C); }
  static __device__ __forceinline__ void get(const Raw8<TX>& r, int c, int C, int, float (&v)[8]) { raw8_get(r, c, C, v); }
};
struct RawQ { u32x2_t q; int e; };
template <> struct RowX<unsigned char> {         // x as 8-bit blocks
  static __device__ __forceinline__ RawQ load(const unsigned char* x, const unsigned char* scale, size_t row, int c, int C) {
    const int KB = (C + B8_BLOCK - 1) / B8_BLOCK, cc = min(c, KB * B8_BLOCK - 8);
    return {*reinterpret_cast<const u32x2_t*>(x + row * KB * B8_BLOCK + cc), (int)scale[row * ((KB + 3) / 4 * 4) + cc / B8_BLOCK]};
  }
  static __device__ __forceinline__ void get(const RawQ& r, int c, int C, int fmt, float (&v)[8]) {
    b8_unpack8(r.q, r.e, fmt, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) if (c + j >= C) v[j] = 0.f;
  }
};

template <typename TX, typename TD, int G, int NV>
__global__ __launch_bounds__(256) void ln_backward_kernel(const TD* __restrict__ dy, const TX* __restrict__ x, const unsigned char* __restrict__ xscale,
                                                          const float* __restrict__ gamma, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, const void* __restrict__ residual,
                                                          void* __restrict__ dx, float* __restrict__ part, int rows, int C, int dx_dtype, int fmt) {
  extern __shared__ __attribute__((aligned(16))) float smem[];   // [2][C] sums of the waves (G <= 64) | gamma, a row of whole vectors
  __shared__ float red[4];
  const int t = threadIdx.x, sub = t % G;
  const int VC = (C + 7) / 8 * 8;
  float* s_gamma = smem + (G <= 64 ? 2 * VC : 0);
  for (int c = t; c < VC; c += 256) s_gamma[c] = c < C ? gamma[c] : 0.f;
  __syncthreads();
  float sg[NV][8], sb[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) { sg[i][j] = 0.f; sb[i][j] = 0.f; }
  const float inv_c = 1.0f / (float)C;
  constexpr int RP = 256 / G;
  for (int base = blockIdx.x * RP; base < rows; base += gridDim.x * RP) {
    const int row0 = base + t / G;
    const bool live = row0 < rows;
    const size_t row = min(row0, rows - 1);
    decltype(RowX<TX>::load(x, xscale, row, 0, C)) rx[NV];
    Raw8<TD> rd[NV];
    const float mu = mean[row], rs = rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) rx[i] = RowX<TX>::load(x, xscale, row, (sub + i * G) * 8, C);
#pragma unroll
    for (int i = 0; i < NV; ++i) rd[i] = raw8_load(dy + row * C, (sub + i * G) * 8, C);
    float xh[NV][8], a[NV][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (sub + i * G) * 8;
      float xv[8], dv[8];
      RowX<TX>::get(rx[i], c, C, fmt, xv);
      raw8_get(rd[i], c, C, dv);
      const f32x4_t* gp = reinterpret_cast<const f32x4_t*>(s_gamma + min(c, VC - 8));
      const f32x4_t g0 = gp[0], g1 = gp[1];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[i][j] = (xv[j] - mu) * rs;            // (past C: dv = 0 keeps it out of every sum)
        a[i][j] = dv[j] * (j < 4 ? g0[j] : g1[j - 4]);
        s1 += a[i][j];
        s2 += a[i][j] * xh[i][j];
        if (live) { sg[i][j] += dv[j] * xh[i][j]; sb[i][j] += dv[j]; }
      }
    }
    s1 = group_sum<G>(s1, red) * inv_c;
    s2 = group_sum<G>(s2, red) * inv_c;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) a[i][j] = rs * (a[i][j] - s1 - xh[i][j] * s2);
    if (dx_dtype == SDAMD_F32) {
      if (residual) {
        Raw8<float> rr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) rr[i] = raw8_load((const float*)residual + row * C, (sub + i * G) * 8, C);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float r[8];
          raw8_get(rr[i], (sub + i * G) * 8, C, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) a[i][j] += r[j];
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (sub + i * G) * 8;
        if (live) row_store8((float*)dx + row * C + c, C - c, a[i]);
      }
    } else {
      if (residual) {
        Raw8<bf16_t> rr[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) rr[i] = raw8_load((const bf16_t*)residual + row * C, (sub + i * G) * 8, C);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float r[8];
          raw8_get(rr[i], (sub + i * G) * 8, C, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) a[i][j] += r[j];
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (sub + i * G) * 8;
        if (live) row_store8((bf16_t*)dx + row * C + c, C - c, a[i]);
      }
    }
  }
  float* pr = part + (size_t)blockIdx.x * 2 * C;
  if constexpr (G > 64) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (sub + i * G) * 8;
      row_store8(pr + c, C - c, sg[i]);
      row_store8(pr + C + c, C - c, sb[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int o = 32; o >= G; o >>= 1) { sg[i][j] += __shfl_xor(sg[i][j], o, 64); sb[i][j] += __shfl_xor(sb[i][j], o, 64); }
    for (int w = 0; w < 4; ++w) {
      if (t / 64 == w && (t & 63) < G) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (sub + i * G) * 8;
          if (c < C) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {        // (a partial vector's tail lands in the padding up to VC)
              smem[c + j] = (w ? smem[c + j] : 0.f) + sg[i][j];
              smem[VC + c + j] = (w ? smem[VC + c + j] : 0.f) + sb[i][j];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int c = t; c < C; c += 256) { pr[c] = smem[c]; pr[C + c] = smem[VC + c]; }
  }
}

// partial rows [nb][2C] -> dgamma [C], dbeta [C]: 16 columns x 16 row lanes per workgroup
__global__ __launch_bounds__(256) void ln_backward_reduce(const float* __restrict__ part, float* __restrict__ dgamma, float* __restrict__ dbeta, int nb, int C) {
  __shared__ float s[16][17];
  const int tc = threadIdx.x & 15, tr = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + tc;
  float acc = 0.f;
  if (c < 2 * C) {
    int r = tr;
    for (; r + 48 < nb; r += 64) {
      const float a0 = part[(size_t)r * 2 * C + c], a1 = part[(size_t)(r + 16) * 2 * C + c];
      const float a2 = part[(size_t)(r + 32) * 2 * C + c], a3 = part[(size_t)(r + 48) * 2 * C + c];
      acc += (a0 + a1) + (a2 + a3);
    }
    for (; r < nb; r += 16) acc += part[(size_t)r * 2 * C + c];
  }
  s[tr][tc] = acc;
  __syncthreads();
  if (tr == 0 && c < 2 * C) {
    float tot = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) tot += s[i][tc];
    if (c < C) dgamma[c] = tot; else dbeta[c - C] = tot;
  }
}

constexpr int LNB_MAX_GRID = 512;
static int lnb_grid(int rows, int C) {
  const int nvec = (C + 7) / 8;
  int rp = 1;
#define LNB_ROWS(G, NV) rp = 256 / G
  LNT_PICK(nvec, LNB_ROWS);
#undef LNB_ROWS
  return min((rows + rp - 1) / rp, LNB_MAX_GRID);
}

extern "C" size_t sdamd_layernorm_backward_ws_bytes(int rows, int C) {
  if (rows <= 0 || C <= 0 || C > LNT_MAX_C) return 0;
  return (size_t)lnb_grid(rows, C) * 2 * C * sizeof(float);
}

template <typename TX, typename TD>
static void lnb_launch(const void* dy, const void* x, const unsigned char* xs, const float* gamma, const float* mean, const float* rstd,
                       const void* residual, void* dx, float* part, int rows, int C, int dx_dtype, int fmt, hipStream_t st) {
  const int grid = lnb_grid(rows, C), VC = (C + 7) / 8 * 8;
#define LNB_CASE(G, NV)                                                                                             \
  ln_backward_kernel<TX, TD, G, NV><<<grid, 256, (size_t)(G <= 64 ? 3 : 1) * VC * sizeof(float), st>>>(              \
      (const TD*)dy, (const TX*)x, xs, gamma, mean, rstd, residual, dx, part, rows, C, dx_dtype, fmt)
  LNT_PICK((C + 7) / 8, LNB_CASE);
#undef LNB_CASE
}

extern "C" int sdamd_layernorm_backward(const void* dy, const void* x, const unsigned char* x_scale, const float* gamma, const float* mean,
                                        const float* rstd, const void* residual, void* dx, float* dgamma, float* dbeta, void* ws,
                                        size_t ws_bytes, int rows, int C, int dy_dtype, int x_dtype, int dx_dtype, void* stream) {
  SD_CHECK((dy_dtype == SDAMD_F32 || dy_dtype == SDAMD_BF16) && (dx_dtype == SDAMD_F32 || dx_dtype == SDAMD_BF16) &&
           x_dtype >= SDAMD_F32 && x_dtype <= SDAMD_E5M2, "layernorm_backward: unsupported dtypes dy=%d x=%d dx=%d", dy_dtype, x_dtype, dx_dtype);
  SD_CHECK(x_dtype < SDAMD_E4M3 || x_scale, "layernorm_backward: 8-bit x without its scales");
  SD_CHECK(rows > 0 && C > 0 && C <= LNT_MAX_C, "layernorm_backward: unsupported shape rows=%d C=%d (C <= %d)", rows, C, LNT_MAX_C);
  const size_t need = sdamd_layernorm_backward_ws_bytes(rows, C);
  SD_CHECK(ws && ws_bytes >= need, "layernorm_backward: workspace of %zu bytes, %zu needed", ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  float* part = (float*)ws;
#define LNB_TX(TD)                                                                                                                       \
  do {                                                                                                                                  \
    if (x_dtype == SDAMD_F32) lnb_launch<float, TD>(dy, x, x_scale, gamma, mean, rstd, residual, dx, part, rows, C, dx_dtype, x_dtype, st);   \
    else if (x_dtype == SDAMD_BF16) lnb_launch<bf16_t, TD>(dy, x, x_scale, gamma, mean, rstd, residual, dx, part, rows, C, dx_dtype, x_dtype, st); \
    else lnb_launch<unsigned char, TD>(dy, x, x_scale, gamma, mean, rstd, residual, dx, part, rows, C, dx_dtype, x_dtype, st);           \
  } while (0)
  if (dy_dtype == SDAMD_F32) LNB_TX(float); else LNB_TX(bf16_t);
#undef LNB_TX
  SD_LAUNCH_CHECK("layernorm_backward");
  ln_backward_reduce<<<(2 * C + 15) / 16, 256, 0, st>>>(part, dgamma, dbeta, lnb_grid(rows, C), C);
  SD_LAUNCH_CHECK("layernorm_backward");
  return 0;
}
