// LayerNorm forward for training (norm_train.h).  65536 x 320 f32 -> bf16: 21.3 us (5.9 TB/s), -> e4m3 blocks 21.7; 77 x 768: 3.8.
#include "norm_train.h"

// lanes per row and vectors per lane: at most 4 vectors where the row allows it.  (With 5 or 6 and fewer lanes no lane is
// idle at 320, 640 and 1280 columns, but each waits longer: 65536 x 320 -> e4m3 31.7 us against 21.6, 77 x 768 5.2 against 3.5.)
#define LNT_PICK(nvec, CASE)                                                                                          \
  do {                                                                                                                \
    const int nv_ = (nvec);                                                                                           \
    if (nv_ <= 16) { CASE(8, 2); } else if (nv_ <= 24) { CASE(8, 3); } else if (nv_ <= 48) { CASE(16, 3); }            \
    else if (nv_ <= 64) { CASE(32, 2); } else if (nv_ <= 96) { CASE(32, 3); } else if (nv_ <= 128) { CASE(64, 2); }    \
    else if (nv_ <= 192) { CASE(64, 3); } else if (nv_ <= 256) { CASE(64, 4); } else if (nv_ <= 512) { CASE(256, 2); } \
    else if (nv_ <= 768) { CASE(256, 3); } else if (nv_ <= 1024) { CASE(256, 4); } else { CASE(256, 6); }             \
  } while (0)

template <typename TX, int G, int NV>
__global__ __launch_bounds__(256) void ln_train_kernel(const TX* __restrict__ x, void* __restrict__ y, unsigned char* __restrict__ yscale,
                                                       const float* __restrict__ gamma, const float* __restrict__ beta,
                                                       float* __restrict__ mean_out, float* __restrict__ rstd_out, int rows, int C,
                                                       float eps, int out_dtype) {
  __shared__ float red[4];
  const int sub = threadIdx.x % G;
  const int row = blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = row < rows;
  const TX* xr = x + (size_t)min(row, rows - 1) * C;
  Raw8<TX> raw[NV];
  Raw8<float> gm[NV], bt[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) raw[i] = raw8_load(xr, (sub + i * G) * 8, C);
#pragma unroll
  for (int i = 0; i < NV; ++i) {                 // (they arrive while the statistics are reduced)
    gm[i] = raw8_load(gamma, (sub + i * G) * 8, C);
    bt[i] = raw8_load(beta, (sub + i * G) * 8, C);
  }
  float v[NV][8];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    raw8_get(raw[i], (sub + i * G) * 8, C, v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[i][j];
  }
  const float mean = group_sum<G>(sum, red) / (float)C;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = v[i][j] - mean;
      sq += (sub + i * G) * 8 + j < C ? d * d : 0.f;
    }
  const float rstd = 1.0f / sqrtf(group_sum<G>(sq, red) / (float)C + eps);
  if (live && sub == 0) { mean_out[row] = mean; rstd_out[row] = rstd; }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (sub + i * G) * 8;
    float g[8], b[8];
    raw8_get(gm[i], c, C, g);
    raw8_get(bt[i], c, C, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] - mean) * rstd * g[j] + b[j];
  }
  if (out_dtype == SDAMD_F32) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (sub + i * G) * 8;
      if (live) row_store8((float*)y + (size_t)row * C + c, C - c, v[i]);
    }
  } else if (out_dtype == SDAMD_BF16) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (sub + i * G) * 8;
      if (live) row_store8((bf16_t*)y + (size_t)row * C + c, C - c, v[i]);
    }
  } else {
    // 8-bit blocks: vector number sub + i G of the row belongs to block (sub + i G) / 16, so 16 lanes hold a block of one
    // step i (G >= 16) or 8 lanes hold it in two (G = 8)
    const int KB = (C + B8_BLOCK - 1) / B8_BLOCK, SP = (KB + 3) / 4 * 4;
    unsigned char* yr = (unsigned char*)y + (size_t)row * KB * B8_BLOCK;
    unsigned char* sr = yscale + (size_t)row * SP;
    constexpr int STEPS = G == 8 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < NV; i += STEPS) {
      unsigned m = 0;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (i + s >= NV) continue;
        const int c = (sub + (i + s) * G) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) if (c + j >= C) v[i + s][j] = 0.f;
        m = max(m, b8_mag8(v[i + s]));
      }
      if constexpr (G == 8) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
      } else {
        m = b8_max16(m);
      }
      const int e = b8_exponent_of(m, out_dtype);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (i + s >= NV) continue;
        const int vec = sub + (i + s) * G;
        if (live && vec < KB * 16) {
          *reinterpret_cast<u32x2_t*>(yr + vec * 8) = b8_pack8(v[i + s], e, out_dtype);
          if (vec % 16 == 0) sr[vec / 16] = (unsigned char)e;
        }
      }
    }
    if (live && KB + sub < SP) sr[KB + sub] = 127;
  }
}

template <typename TX>
static void ln_train_launch(const void* x, void* y, unsigned char* ys, const float* g, const float* b, float* mean, float* rstd, int rows, int C,
                            float eps, int out_dtype, hipStream_t st) {
  // 8-bit rows are written in whole blocks, so the lanes have to reach the end of the last one
  const int nvec = out_dtype >= SDAMD_E4M3 ? b8_kblocks(C) * 16 : (C + 7) / 8;
#define LNT_CASE(G, NV) \
  ln_train_kernel<TX, G, NV><<<(rows + 256 / G - 1) / (256 / G), 256, 0, st>>>((const TX*)x, y, ys, g, b, mean, rstd, rows, C, eps, out_dtype)
  LNT_PICK(nvec, LNT_CASE);
#undef LNT_CASE
}

extern "C" int sdamd_layernorm_train(const void* x, void* y, unsigned char* y_scale, const float* gamma, const float* beta, float* mean,
                                     float* rstd, int rows, int C, float eps, int dtype, int out_dtype, void* stream) {
  SD_CHECK((dtype == SDAMD_BF16 || dtype == SDAMD_F32) && out_dtype >= SDAMD_F32 && out_dtype <= SDAMD_E5M2,
           "layernorm_train: unsupported dtypes in=%d out=%d", dtype, out_dtype);
  SD_CHECK(out_dtype < SDAMD_E4M3 || y_scale, "layernorm_train: 8-bit output without room for its scales");
  SD_CHECK(rows > 0 && C > 0 && C <= LNT_MAX_C, "layernorm_train: unsupported shape rows=%d C=%d (C <= %d)", rows, C, LNT_MAX_C);
  SD_CHECK(rows < (1 << 24) || (rows <= (1 << 27) - 32 && C <= 512), "layernorm_train: too many rows, %d of %d", rows, C);   // (a launch's 2^32 threads)
  if (dtype == SDAMD_BF16) ln_train_launch<bf16_t>(x, y, y_scale, gamma, beta, mean, rstd, rows, C, eps, out_dtype, (hipStream_t)stream);
  else ln_train_launch<float>(x, y, y_scale, gamma, beta, mean, rstd, rows, C, eps, out_dtype, (hipStream_t)stream);
  SD_LAUNCH_CHECK("layernorm_train");
  return 0;
}
