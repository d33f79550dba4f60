// LayerNorm backward (norm_train.h): dx, and the weight gradients in two steps without atomics.  A workgroup walks rows
// blockIdx, blockIdx + grid, ... and keeps the sums of dy xh and dy of the columns its lanes hold in registers; at its end
// the lanes that hold the same columns are joined by shuffles within a wave and wave after wave in LDS, and the workgroup
// leaves one row of partial sums.  A second launch adds the partial rows.  Every order is fixed: the same bits every run.
// Few rows (LNB_ONE_LAUNCH): the weight gradients need nothing that the dx workgroups compute, so workgroups of their own
// read x and dy again by columns, in the same launch.
#include "norm_train.h"
#include <type_traits>

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

template <typename TX> __device__ __forceinline__ float row_x(const TX* x, const unsigned char*, size_t row, int c, int C, int) { return Cvt<TX>::ld(x + row * C + c); }
__device__ __forceinline__ float row_x(const unsigned char* x, const unsigned char* scale, size_t row, int c, int C, int fmt) {
  const int KB = (C + B8_BLOCK - 1) / B8_BLOCK;
  float v[8];
  b8_unpack8((u32x2_t){(unsigned)x[row * KB * B8_BLOCK + c], 0u}, scale[row * ((KB + 3) / 4 * 4) + c / B8_BLOCK], fmt, v);
  return v[0];
}

// dgamma, dbeta of 16 columns over all rows: NT / 16 row lanes, four rows requested at a time
template <typename TX, typename TD, int NT>
__device__ __forceinline__ void ln_columns(const TD* __restrict__ dy, const TX* __restrict__ x, const unsigned char* __restrict__ xscale,
                                           const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ dgamma,
                                           float* __restrict__ dbeta, int blk, int rows, int C, int fmt) {
  constexpr int RL = NT / 16;
  __shared__ float s[2][RL][17];
  const int tc = threadIdx.x & 15, tr = threadIdx.x >> 4;
  const int c = min(blk * 16 + tc, C - 1);
  float ag = 0.f, ab = 0.f;
  for (int r0 = tr; r0 < rows; r0 += 4 * RL) {
    float d[4], v[4], mu[4], rs[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const size_t r = min(r0 + RL * k, rows - 1);
      d[k] = Cvt<TD>::ld(dy + r * C + c);
      v[k] = row_x(x, xscale, r, c, C, fmt);
      mu[k] = mean[r];
      rs[k] = rstd[r];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r0 + RL * k < rows) { ag += d[k] * ((v[k] - mu[k]) * rs[k]); ab += d[k]; }
  }
  s[0][tr][tc] = ag;
  s[1][tr][tc] = ab;
  __syncthreads();
  if (tr < 2 && blk * 16 + tc < C) {
    float tot = 0.f;
#pragma unroll
    for (int i = 0; i < RL; ++i) tot += s[tr][i][tc];
    (tr ? dbeta : dgamma)[c] = tot;
  }
}

// the compiler would keep the unpacked values of the first use for the second: make it unpack again (registers)
__device__ __forceinline__ void again(Raw8<float>& r) { asm volatile("" : "+v"(r.a), "+v"(r.b)); }
__device__ __forceinline__ void again(Raw8<bf16_t>& r) { asm volatile("" : "+v"(r.a)); }
__device__ __forceinline__ void again(RawQ& r) { asm volatile("" : "+v"(r.q)); }

constexpr int LNB_THREADS = 512;   // two waves per SIMD: one waits for memory while the other computes

// lanes per row and vectors per lane: at most 4, so that the sums of both weight gradients (16 registers a vector), a row and
// the next fit 256 registers, two waves per SIMD.  (5 vectors a lane, four waves of 400 registers: 65536 x 320 bf16 in 41.5 us, this way 35.5.)
#define LNB_PICK(nvec, CASE)                                                                                       \
  do {                                                                                                             \
    const int nv_ = (nvec);                                                                                        \
    if (nv_ <= 16) { CASE(8, 2); } else if (nv_ <= 24) { CASE(8, 3); } else if (nv_ <= 48) { CASE(16, 3); }         \
    else if (nv_ <= 64) { CASE(32, 2); } else if (nv_ <= 96) { CASE(32, 3); } else if (nv_ <= 128) { CASE(64, 2); } \
    else if (nv_ <= 192) { CASE(64, 3); } else if (nv_ <= 256) { CASE(64, 4); } else if (nv_ <= 512) { CASE(256, 2); } \
    else if (nv_ <= 1024) { CASE(512, 2); } else { CASE(512, 3); }                                                 \
  } while (0)

template <typename TX, typename TD, int G, int NV>
__global__ __launch_bounds__(LNB_THREADS) void ln_backward_kernel(
    const TD* __restrict__ dy, const TX* __restrict__ x, const unsigned char* __restrict__ xscale, const float* __restrict__ gamma,
    const float* __restrict__ mean, const float* __restrict__ rstd, const void* __restrict__ residual, void* __restrict__ dx,
    float* __restrict__ part, float* __restrict__ dgamma, float* __restrict__ dbeta, int row_blocks, int rows, int C, int dx_dtype, int fmt) {
  constexpr int NT = LNB_THREADS, RP = NT / G;
  if ((int)blockIdx.x >= row_blocks) {
    ln_columns<TX, TD, NT>(dy, x, xscale, mean, rstd, dgamma, dbeta, blockIdx.x - row_blocks, rows, C, fmt);
    return;
  }
  extern __shared__ __attribute__((aligned(16))) float smem[];   // gamma [VC], at the end the sums of the waves [4][VC] (G <= 64) or of half the lanes [VC]
  __shared__ float red[8];
  const int t = threadIdx.x, sub = t % G;
  const int VC = (C + 7) / 8 * 8;
  typedef decltype(RowX<TX>::load(x, xscale, 0, 0, C)) raw_x;
  // The next rows are requested before this turn's are used, where two rows of raw values fit the registers beside the sums.
  constexpr bool AHEAD = NV <= 3;
  raw_x rx[NV], nx[AHEAD ? NV : 1];
  Raw8<TD> rd[NV], nd[AHEAD ? NV : 1];
  float mu, rs, nmu = 0.f, nrs = 0.f;
  auto request = [&](int base, raw_x* ax, Raw8<TD>* ad, float& am, float& ar) {
    const size_t row = min(base + t / G, rows - 1);
    am = mean[row];
    ar = rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) ax[i] = RowX<TX>::load(x, xscale, row, (sub + i * G) * 8, C);
#pragma unroll
    for (int i = 0; i < NV; ++i) ad[i] = raw8_load(dy + row * C, (sub + i * G) * 8, C);
  };
  if constexpr (AHEAD) request(blockIdx.x * RP, nx, nd, nmu, nrs);
  for (int c = t; c < VC; c += NT) smem[c] = c < C ? gamma[c] : 0.f;
  __syncthreads();
  float sg[NV][8], sb[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) { sg[i][j] = 0.f; sb[i][j] = 0.f; }
  const float inv_c = 1.0f / (float)C;
  for (int base = blockIdx.x * RP; base < rows; base += row_blocks * RP) {
    const bool live = base + t / G < rows;
    const size_t row = min(base + t / G, rows - 1);
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < NV; ++i) { rx[i] = nx[i]; rd[i] = nd[i]; }
      mu = nmu;
      rs = nrs;
      request(base + row_blocks * RP, nx, nd, nmu, nrs);
    } else {
      request(base, rx, rd, mu, rs);
    }
    float s1 = 0.f, s2 = 0.f;
    auto terms = [&](int i, float (&xh)[8], float (&dv)[8], float (&a)[8]) {
      const int c = (sub + i * G) * 8;
      RowX<TX>::get(rx[i], c, C, fmt, xh);
      raw8_get(rd[i], c, C, dv);
      const f32x4_t* gp = reinterpret_cast<const f32x4_t*>(smem + min(c, VC - 8));
      const f32x4_t g0 = gp[0], g1 = gp[1];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[j] = (xh[j] - mu) * rs;               // (past C: dv = 0 keeps it out of every sum)
        a[j] = dv[j] * (j < 4 ? g0[j] : g1[j - 4]);
      }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float xh[8], dv[8], a[8];
      terms(i, xh, dv, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s1 += a[j];
        s2 += a[j] * xh[j];
        if (live) { sg[i][j] += dv[j] * xh[j]; sb[i][j] += dv[j]; }
      }
      again(rx[i]);
      again(rd[i]);
    }
    auto finish = [&](auto* out, auto* res) {
      typedef typename std::remove_const<typename std::remove_pointer<decltype(res)>::type>::type TO;
      Raw8<TO> rr[NV];
      if (res) {
#pragma unroll
        for (int i = 0; i < NV; ++i) rr[i] = raw8_load(res + row * C, (sub + i * G) * 8, C);
      }
      s1 = group_sum<G>(s1, red) * inv_c;
      s2 = group_sum<G>(s2, red) * inv_c;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (sub + i * G) * 8;
        float xh[8], dv[8], a[8], r[8];
        terms(i, xh, dv, a);
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = rs * (a[j] - s1 - xh[j] * s2);
        if (res) {
          raw8_get(rr[i], c, C, r);
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] += r[j];
        }
        if (live) row_store8(out + row * C + c, C - c, a);
      }
    };
    if (dx_dtype == SDAMD_F32) finish((float*)dx, (const float*)residual);
    else finish((bf16_t*)dx, (const bf16_t*)residual);
  }
  if (!part) return;                             // (the column workgroups have the weight gradients)
  float* pr = part + (size_t)blockIdx.x * 2 * C;
  if constexpr (G > 64) {                        // two rows per turn: the second half's lanes hand theirs to the first's
    auto join = [&](float (&v)[NV][8], float* out) {
      if constexpr (G == LNB_THREADS) {          // (the whole workgroup has one row)
#pragma unroll
        for (int i = 0; i < NV; ++i) row_store8(out + (sub + i * G) * 8, C - (sub + i * G) * 8, v[i]);
        return;
      }
      __syncthreads();
      if (t >= 256) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (sub + i * G) * 8;
          f32x4_t* d = reinterpret_cast<f32x4_t*>(smem + c);
          if (c < C) { d[0] = (f32x4_t){v[i][0], v[i][1], v[i][2], v[i][3]}; d[1] = (f32x4_t){v[i][4], v[i][5], v[i][6], v[i][7]}; }
        }
      }
      __syncthreads();
      if (t < 256) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (sub + i * G) * 8;
          if (c < C) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] += smem[c + j];
            row_store8(out + c, C - c, v[i]);
          }
        }
      }
    };
    join(sg, pr);
    join(sb, pr + C);
  } else {
    float* s_sum = smem;                         // (gamma is not needed any more)
    auto join = [&](float (&v)[NV][8], float* out) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int o = 32; o >= G; o >>= 1) v[i][j] += __shfl_xor(v[i][j], o, 64);
#pragma unroll
      for (int half = 0; half < 2; ++half) {     // waves 0-3 write, waves 4-7 add to them
        __syncthreads();                         // (s_sum may still be read)
        if ((t >> 8) == half && (t & 63) < G) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (sub + i * G) * 8;
            f32x4_t* d = reinterpret_cast<f32x4_t*>(s_sum + ((t >> 6) & 3) * VC + c);
            if (c < C) {
              f32x4_t lo = {v[i][0], v[i][1], v[i][2], v[i][3]}, hi = {v[i][4], v[i][5], v[i][6], v[i][7]};
              if (half) { lo += d[0]; hi += d[1]; }
              d[0] = lo;
              d[1] = hi;
            }
          }
        }
      }
      __syncthreads();
      for (int c = t; c < C; c += NT) out[c] = (s_sum[c] + s_sum[VC + c]) + (s_sum[2 * VC + c] + s_sum[3 * VC + c]);
    };
    join(sg, pr);
    join(sb, pr + C);
  }
}

// partial rows [nb][2C] -> dgamma [C], dbeta [C]: 16 columns x 16 row lanes per workgroup, 16 rows requested at a time
__global__ __launch_bounds__(256) void ln_backward_reduce(const float* __restrict__ part, float* __restrict__ dgamma, float* __restrict__ dbeta, int nb, int C) {
  __shared__ float s[16][17];
  const int tc = threadIdx.x & 15, tr = threadIdx.x >> 4;
  const int c = min((int)blockIdx.x * 16 + tc, 2 * C - 1);
  float acc = 0.f;
  for (int r0 = tr; r0 < nb; r0 += 256) {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = part[(size_t)min(r0 + 16 * k, nb - 1) * 2 * C + c];
#pragma unroll
    for (int k = 0; k < 16; ++k) acc += r0 + 16 * k < nb ? v[k] : 0.f;
  }
  s[tr][tc] = acc;
  __syncthreads();
  if (tr == 0 && (int)blockIdx.x * 16 + tc < 2 * C) {
    float tot = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) tot += s[i][tc];
    if (c < C) dgamma[c] = tot; else dbeta[c - C] = tot;
  }
}

// One launch for both where the column workgroups' walk over all rows is short: they take as long as the rest up to about
// 1024 rows of 1024 (1024 x 768: 6.8 us, two launches 13.1; 2048 x 768: 18.9 and 12.7; 1024 x 2048: 16.8 and 13.7).
static bool lnb_one_launch(int rows, int C) { return rows <= 1024 && (long long)rows * C <= (1 << 20); }
// One workgroup per CU (256, never 257: 4099 x 1001 in 171 workgroups of three turns 16.0 us, in 257 of two 19.6): each
// leaves a row of partial sums and pays for joining its waves' (65536 x 320 bf16: 35.5 us, in 384 workgroups 49.2, in 512 42.2).
static int lnb_grid(int rows, int C) {
  const int nvec = (C + 7) / 8;
  int rp = 1;
#define LNB_ROWS(G, NV) rp = LNB_THREADS / G
  LNB_PICK(nvec, LNB_ROWS);
#undef LNB_ROWS
  const int blocks = (rows + rp - 1) / rp;
  if (lnb_one_launch(rows, C)) return blocks;
  const int turns = (blocks + 255) / 256;
  return (blocks + turns - 1) / turns;
}

extern "C" size_t sdamd_layernorm_backward_ws_bytes(int rows, int C) {
  if (rows <= 0 || C <= 0 || C > LNT_MAX_C || lnb_one_launch(rows, C)) return 0;
  return (size_t)lnb_grid(rows, C) * 2 * C * sizeof(float);
}

template <typename TX, typename TD>
static void lnb_launch(const void* dy, const void* x, const unsigned char* xs, const float* gamma, const float* mean, const float* rstd,
                       const void* residual, void* dx, float* part, float* dgamma, float* dbeta, int rows, int C, int dx_dtype, int fmt,
                       hipStream_t st) {
  const int row_blocks = lnb_grid(rows, C), VC = (C + 7) / 8 * 8, grid = row_blocks + (part ? 0 : (C + 15) / 16);
#define LNB_CASE(G, NV)                                                                                             \
  ln_backward_kernel<TX, TD, G, NV><<<grid, LNB_THREADS, (size_t)(G <= 64 && part ? 4 : 1) * VC * sizeof(float), st>>>(              \
      (const TD*)dy, (const TX*)x, xs, gamma, mean, rstd, residual, dx, part, dgamma, dbeta, row_blocks, rows, C, dx_dtype, fmt)
  LNB_PICK((C + 7) / 8, LNB_CASE);
#undef LNB_CASE
}

extern "C" int sdamd_layernorm_backward(const void* dy, const void* x, const unsigned char* x_scale, const float* gamma, const float* mean,
                                        const float* rstd, const void* residual, void* dx, float* dgamma, float* dbeta, void* ws,
                                        size_t ws_bytes, int rows, int C, int dy_dtype, int x_dtype, int dx_dtype, void* stream) {
  SD_CHECK((dy_dtype == SDAMD_F32 || dy_dtype == SDAMD_BF16) && (dx_dtype == SDAMD_F32 || dx_dtype == SDAMD_BF16) &&
           x_dtype >= SDAMD_F32 && x_dtype <= SDAMD_E5M2, "layernorm_backward: unsupported dtypes dy=%d x=%d dx=%d", dy_dtype, x_dtype, dx_dtype);
  SD_CHECK(x_dtype < SDAMD_E4M3 || x_scale, "layernorm_backward: 8-bit x without its scales");
  SD_CHECK(rows > 0 && C > 0 && C <= LNT_MAX_C, "layernorm_backward: unsupported shape rows=%d C=%d (C <= %d)", rows, C, LNT_MAX_C);
  SD_CHECK(rows <= (1 << 28), "layernorm_backward: too many rows, %d", rows);
  const size_t need = sdamd_layernorm_backward_ws_bytes(rows, C);
  SD_CHECK(need == 0 || (ws && ws_bytes >= need), "layernorm_backward: workspace of %zu bytes, %zu needed", ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  float* part = need ? (float*)ws : nullptr;
#define LNB_TX(TD)                                                                                                                       \
  do {                                                                                                                                  \
    if (x_dtype == SDAMD_F32) lnb_launch<float, TD>(dy, x, x_scale, gamma, mean, rstd, residual, dx, part, dgamma, dbeta, rows, C, dx_dtype, x_dtype, st);   \
    else if (x_dtype == SDAMD_BF16) lnb_launch<bf16_t, TD>(dy, x, x_scale, gamma, mean, rstd, residual, dx, part, dgamma, dbeta, rows, C, dx_dtype, x_dtype, st); \
    else lnb_launch<unsigned char, TD>(dy, x, x_scale, gamma, mean, rstd, residual, dx, part, dgamma, dbeta, rows, C, dx_dtype, x_dtype, st);           \
  } while (0)
  if (dy_dtype == SDAMD_F32) LNB_TX(float); else LNB_TX(bf16_t);
#undef LNB_TX
  SD_LAUNCH_CHECK("layernorm_backward");
  if (!need) return 0;
  ln_backward_reduce<<<(2 * C + 15) / 16, 256, 0, st>>>(part, dgamma, dbeta, lnb_grid(rows, C), C);
  SD_LAUNCH_CHECK("layernorm_backward");
  return 0;
}
