// 8-bit blocks (blocks8.h): quantise, dequantise, and GeGLU (diffusion.py:128-130) with its pre-activation kept in them.
// All of it is bound by HBM: one pass, 16-byte loads, nothing read twice.  (Sizes are limited by a launch's 2^32 threads.)
#include "blocks8.h"

// ---- rows -> blocks.  q [rows][KB*128], scale [rows][SP]; 16 lanes hold a block, a workgroup takes 16 * UN blocks, all of
// them requested before the first is used.  36864 x 1280 bf16: 23 - 24.4 us = 5.9 TB/s with UN = 2 (1: 31.1, 4: 26.3).
template <typename T, int UN>
__global__ __launch_bounds__(256) void quant8_kernel(const T* __restrict__ x, unsigned char* __restrict__ q,
                                                     unsigned char* __restrict__ scale, unsigned nblk, int KB, int K,
                                                     long long ldx, int SP, int fmt) {
  const int sub = threadIdx.x & 15;
  const unsigned b0 = blockIdx.x * (16u * UN) + (threadIdx.x >> 4);
  Raw8<T> raw[UN];
  unsigned row[UN], kb[UN];
#pragma unroll
  for (int u = 0; u < UN; ++u) {     // every block's values are requested before the first is used
    const unsigned b = min(b0 + 16u * u, nblk - 1);
    row[u] = b / (unsigned)KB;
    kb[u] = b - row[u] * (unsigned)KB;
    const int c = (int)kb[u] * B8_BLOCK + sub * 8;
    raw[u] = raw8_load(x + (long long)row[u] * ldx, c, K);
  }
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    float v[8];
    raw8_get(raw[u], (int)kb[u] * B8_BLOCK + sub * 8, K, v);
    const int e = b8_exponent_of(b8_max16(b8_mag8(v)), fmt);
    if (b0 + 16u * u < nblk) {
      *reinterpret_cast<u32x2_t*>(q + ((size_t)row[u] * KB + kb[u]) * B8_BLOCK + sub * 8) = b8_pack8(v, e, fmt);
      if (sub == 0) scale[(size_t)row[u] * SP + kb[u]] = (unsigned char)e;
      if (kb[u] == (unsigned)KB - 1 && KB + sub < SP) scale[(size_t)row[u] * SP + KB + sub] = 127;
    }
  }
}

// ---- weights -> 128 x 128 blocks.  One workgroup per block; the weight has any strides (w and w.t() alike).  ALONG = 1: its
// rows are contiguous, 16 lanes take 128 columns of a row and leave their bytes where they belong; 2: its columns are
// contiguous, the bytes turn in LDS; 0: neither, value by value.  10240 x 1280 bf16: 11.1 us
// (3.5 TB/s; value by value 53), its transpose 13.1; f32 12.8 and 14.8 (5.1 and 4.4 TB/s).  All 800 workgroups are on the
// chip at once, so loads, reduction and stores follow one another with no other block's beside them.
template <typename T, int ALONG>
__global__ __launch_bounds__(256) void quant8_weight_kernel(const T* __restrict__ w, unsigned char* __restrict__ q,
                                                            unsigned char* __restrict__ scale, int N, int K, long long sn,
                                                            long long sk, int KB, int SP) {
  __shared__ __attribute__((aligned(16))) unsigned char tile[ALONG == 1 ? 16 : 128 * 132];
  __shared__ unsigned red[4];
  const int n0 = blockIdx.y * B8_BLOCK, k0 = blockIdx.x * B8_BLOCK, t = threadIdx.x;
  const int c = (t & 15) * 8, r = t >> 4;                  // a thread's eight columns, and its rows r + 16 i (ALONG 2: of the transpose)
  float v[8][8];
  unsigned m = 0;
  if constexpr (ALONG != 0) {
    const int R = ALONG == 1 ? N : K, C = ALONG == 1 ? K : N, r0 = ALONG == 1 ? n0 : k0, c0 = ALONG == 1 ? k0 : n0;
    const long long ld = ALONG == 1 ? sn : sk;
    Raw8<T> raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = raw8_load(w + min(r0 + r + 16 * i, R - 1) * ld, c0 + c, C);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      raw8_get(raw[i], c0 + c, C, v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = r0 + r + 16 * i < R ? v[i][j] : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = n0 + r + 16 * i, k = k0 + c + j;
        const float x = Cvt<T>::ld(w + min(n, N - 1) * sn + min(k, K - 1) * sk);
        v[i][j] = n < N && k < K ? x : 0.f;
      }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, b8_mag8(v[i]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
  if ((t & 63) == 0) red[t >> 6] = m;
  __syncthreads();
  const int e = b8_exponent<8>(max(max(red[0], red[1]), max(red[2], red[3])));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const u32x2_t b = b8_pack8(v[i], e, SDAMD_E4M3);
    if constexpr (ALONG == 2) {
#pragma unroll
      for (int j = 0; j < 8; ++j) tile[(c + j) * 132 + r + 16 * i] = (unsigned char)(b[j >> 2] >> (j & 3) * 8);
    } else {
      if (n0 + r + 16 * i < N) *reinterpret_cast<u32x2_t*>(q + ((size_t)(n0 + r + 16 * i) * KB + blockIdx.x) * B8_BLOCK + c) = b;
    }
  }
  if constexpr (ALONG == 2) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = i * 256 + t, n = d >> 5, k = (d & 31) * 4;
      if (n0 + n < N)
        *reinterpret_cast<unsigned*>(q + ((size_t)(n0 + n) * KB + blockIdx.x) * B8_BLOCK + k) = *reinterpret_cast<const unsigned*>(tile + n * 132 + k);
    }
  }
  if (t == 0) scale[(size_t)blockIdx.y * SP + blockIdx.x] = (unsigned char)e;
  if ((int)blockIdx.x == KB - 1 && KB + t < SP) scale[(size_t)blockIdx.y * SP + KB + t] = 127;
}

// ---- blocks -> the values they stand for.  36864 x 1280 to bf16: 22.2 us = 6.4 TB/s, to f32 41.7.
template <typename TO>
__global__ __launch_bounds__(256) void dequant8_kernel(const unsigned char* __restrict__ q, const unsigned char* __restrict__ scale,
                                                       TO* __restrict__ out, unsigned nblk, int KB, int K, int SP, int row_shift, int fmt) {
  const int sub = threadIdx.x & 15;
  const unsigned b = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (b >= nblk) return;
  const unsigned row = b / (unsigned)KB, kb = b - row * (unsigned)KB;
  const int c = (int)kb * B8_BLOCK + sub * 8;
  if (c >= K) return;
  float v[8];
  b8_unpack8(*reinterpret_cast<const u32x2_t*>(q + (size_t)b * B8_BLOCK + sub * 8), scale[(size_t)(row >> row_shift) * SP + kb], fmt, v);
  row_store8(out + (size_t)row * K + c, K - c, v);
}

// ---- GeGLU that keeps its input in 8 bits: h [rows][2F] -> out [rows][F] = value * gelu(gate), of h's type or as blocks of
// another Linear's operand, and h's blocks.
// 65536 x 1280 bf16: 102 - 119 us = 5.7 - 6.6 TB/s, by what the caches hold; into blocks 114, where a quantiser behind it makes 154.
// F % 128 == 0: the 16 lanes that hold a value block hold the gate block of the same columns too, so h is read once.
enum GegluOut { GEGLU_DENSE, GEGLU_PAST, GEGLU_BLOCKS };    // PAST: past the cache (b8_past_cache)
template <typename T, GegluOut OUT>
__global__ __launch_bounds__(256) void geglu_train_kernel(const T* __restrict__ h, void* __restrict__ out, unsigned char* __restrict__ out_scale,
                                                          unsigned char* __restrict__ q, unsigned char* __restrict__ scale, unsigned nblk, int FB,
                                                          int SP, int fmt, int out_fmt) {
  const int sub = threadIdx.x & 15;
  const unsigned b = blockIdx.x * 16u + (threadIdx.x >> 4);
  const unsigned bb = min(b, nblk - 1), row = bb / (unsigned)FB, fb = bb - row * (unsigned)FB;
  const size_t vb = (size_t)row * 2 * FB + fb, gb = vb + FB;          // block numbers in h
  float v[8], g[8], o[8];
  const Raw8<T> rv = raw8_load(h + vb * B8_BLOCK, sub * 8, B8_BLOCK), rg = raw8_load(h + gb * B8_BLOCK, sub * 8, B8_BLOCK);
  raw8_get(rv, sub * 8, B8_BLOCK, v);
  raw8_get(rg, sub * 8, B8_BLOCK, g);
  const int ev = b8_exponent_of(b8_max16(b8_mag8(v)), fmt), eg = b8_exponent_of(b8_max16(b8_mag8(g)), fmt);
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = v[j] * gelu_erf_f(g[j]);
  const int eo = OUT == GEGLU_BLOCKS ? b8_exponent_of(b8_max16(b8_mag8(o)), out_fmt) : 0;
  if (b >= nblk) return;
  if constexpr (OUT == GEGLU_BLOCKS) {
    const int SO = (FB + 3) / 4 * 4;
    *reinterpret_cast<u32x2_t*>((unsigned char*)out + (size_t)bb * B8_BLOCK + sub * 8) = b8_pack8(o, eo, out_fmt);
    if (sub == 0) out_scale[(size_t)row * SO + fb] = (unsigned char)eo;
    if (fb == (unsigned)FB - 1 && FB + sub < SO) out_scale[(size_t)row * SO + FB + sub] = 127;
  } else {
    row_store8<OUT == GEGLU_PAST>((T*)out + (size_t)bb * B8_BLOCK + sub * 8, 8, o);
  }
  *reinterpret_cast<u32x2_t*>(q + vb * B8_BLOCK + sub * 8) = b8_pack8(v, ev, fmt);
  *reinterpret_cast<u32x2_t*>(q + gb * B8_BLOCK + sub * 8) = b8_pack8(g, eg, fmt);
  if (sub == 0) { scale[(size_t)row * SP + fb] = (unsigned char)ev; scale[(size_t)row * SP + FB + fb] = (unsigned char)eg; }
  if (fb == (unsigned)FB - 1 && 2 * FB + sub < SP) scale[(size_t)row * SP + 2 * FB + sub] = 127;
}
// any F: a value's block and its gate's do not line up.  A workgroup quantises R whole rows, then gates them; it finds them in
// the caches the second time.  (10000 x 1000 bf16: 19 - 22.5 us, as two launches 28.4; 65536 x
// 960 103 - 107 and 138.  R with 32 blocks together; with 64 and 128 10000 x 1000 f32 takes 40.6 and 41.7 instead of 34.4.)
template <typename T, bool BLOCKS>
__global__ __launch_bounds__(256) void geglu_rows_kernel(const T* __restrict__ h, void* __restrict__ out, unsigned char* __restrict__ out_scale,
                                                         unsigned char* __restrict__ q, unsigned char* __restrict__ scale, long long rows, int R,
                                                         int F, int KB, int SP, int fmt, int out_fmt) {
  const int t = threadIdx.x, sub = t & 15, VR = (F + 7) / 8;
  const long long r0 = (long long)blockIdx.x * R;
  const int n = (int)min((long long)R, rows - r0), blocks = n * KB, vecs = n * VR;
  h += r0 * 2 * F;
  q += r0 * KB * B8_BLOCK;
  scale += r0 * SP;
  for (int b0 = t >> 4; b0 < blocks; b0 += 32) {           // two blocks requested at a time
    Raw8<T> raw[2];
    int row[2], kb[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int b = min(b0 + 16 * u, blocks - 1);
      row[u] = b / KB;
      kb[u] = b - row[u] * KB;
      raw[u] = raw8_load(h + (size_t)row[u] * 2 * F, kb[u] * B8_BLOCK + sub * 8, 2 * F);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float v[8];
      raw8_get(raw[u], kb[u] * B8_BLOCK + sub * 8, 2 * F, v);
      const int e = b8_exponent_of(b8_max16(b8_mag8(v)), fmt);
      if (b0 + 16 * u < blocks) {
        *reinterpret_cast<u32x2_t*>(q + ((size_t)row[u] * KB + kb[u]) * B8_BLOCK + sub * 8) = b8_pack8(v, e, fmt);
        if (sub == 0) scale[(size_t)row[u] * SP + kb[u]] = (unsigned char)e;
        if (kb[u] == KB - 1 && KB + sub < SP) scale[(size_t)row[u] * SP + KB + sub] = 127;
      }
    }
  }
  auto gate = [&](int row, int c, float (&o)[8]) {
    const T* hr = h + (size_t)row * 2 * F;
    const Raw8<T> rv = raw8_load(hr, c, F), rg = raw8_load(hr + F, c, F);
    float v[8], g[8];
    raw8_get(rv, c, F, v);
    raw8_get(rg, c, F, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = v[j] * gelu_erf_f(g[j]);          // (zeros past F)
  };
  if constexpr (BLOCKS) {
    const int KO = (F + B8_BLOCK - 1) / B8_BLOCK, SO = (KO + 3) / 4 * 4;
    for (int b = t >> 4; b < n * KO; b += 16) {
      const int row = b / KO, kb = b - row * KO;
      float o[8];
      gate(row, kb * B8_BLOCK + sub * 8, o);
      const int e = b8_exponent_of(b8_max16(b8_mag8(o)), out_fmt);
      *reinterpret_cast<u32x2_t*>((unsigned char*)out + ((size_t)(r0 + row) * KO + kb) * B8_BLOCK + sub * 8) = b8_pack8(o, e, out_fmt);
      if (sub == 0) out_scale[(size_t)(r0 + row) * SO + kb] = (unsigned char)e;
      if (kb == KO - 1 && KO + sub < SO) out_scale[(size_t)(r0 + row) * SO + KO + sub] = 127;
    }
  } else {
    for (int i = t; i < vecs; i += 256) {
      const int row = i / VR, c = (i - row * VR) * 8;
      float o[8];
      gate(row, c, o);
      row_store8((T*)out + (size_t)(r0 + row) * F + c, F - c, o);
    }
  }
}

// gelu(x) = x Phi(x) and its slope Phi(x) + x phi(x), erf as in gelu_erf_f (its exponential is phi's)
__device__ __forceinline__ void gelu_slope(float x, float& gelu, float& slope) {
  const float z = __builtin_fabsf(x) * 0.70710678118654752440f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, z, 1.0f));
  float poly = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  poly = __builtin_fmaf(poly, t, 1.421413741f);
  poly = __builtin_fmaf(poly, t, -0.284496736f);
  poly = __builtin_fmaf(poly, t, 0.254829592f);
  const float e = __builtin_amdgcn_exp2f(-(z * z) * 1.4426950408889634f);
  const float tail = 0.5f * poly * t * e;                              // Phi(-|x|)
  const float cdf = x < 0.f ? tail : 1.0f - tail;
  gelu = x * cdf;
  slope = __builtin_fmaf(x * 0.39894228040143267794f, e, cdf);
}

// ---- GeGLU backward: dvalue = dout gelu(gate), dgate = dout value gelu'(gate); h as values (TH) or as 8-bit blocks
// (TH = unsigned char).  BLOCKS (F % 128 == 0, dh bf16): dh's blocks too, of the values as dh holds them, the operand of the Linear that
// takes it on.  65536 x 1280 bf16 from e4m3: 120 us = 5.6 TB/s, 133 right behind its forward pass; with blocks 155, where a quantiser behind it
// makes 212; from bf16 h 150 (5.6 TB/s), all f32 306.
template <typename TD, typename TH, typename TO, bool PAST, bool BLOCKS>
__global__ __launch_bounds__(256) void geglu_backward_kernel(const TD* __restrict__ dout, const TH* __restrict__ h,
                                                             const unsigned char* __restrict__ scale, TO* __restrict__ dh,
                                                             unsigned nvec, int VR, int F, int ldh, int SP, int fmt,
                                                             unsigned char* __restrict__ q, unsigned char* __restrict__ q_scale, int q_fmt) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= nvec) return;                         // (BLOCKS: in whole groups of 16)
  const unsigned row = i / (unsigned)VR;
  const int c = (int)(i - row * (unsigned)VR) * 8;
  const TH* hr = h + (size_t)row * ldh;
  float d[8], v[8], g[8], dv[8], dg[8];
  row_load8(dout + (size_t)row * F, c, F, d);
  if constexpr (sizeof(TH) == 1) {
    const unsigned char* sr = scale + (size_t)row * SP;
    if (F % 8 == 0) {
      const u32x2_t qv = *reinterpret_cast<const u32x2_t*>(hr + c), qg = *reinterpret_cast<const u32x2_t*>(hr + F + c);
      b8_unpack8(qv, sr[c / B8_BLOCK], fmt, v);
      b8_unpack8(qg, sr[(F + c) / B8_BLOCK], fmt, g);
    } else if (F > 8) {              // the gates start at any byte and may change block inside the vector
      const int cc = min(c, F - 8), s = c - cc;                          // (read inside the row; its last, partial vector shifted down)
      typedef unsigned long long __attribute__((aligned(1))) bytes8_t;
      auto eight = [&](int at, float (&o)[8]) {
        const unsigned long long b = *reinterpret_cast<const bytes8_t*>(hr + at + cc) >> s * 8;
        b8_unpack8((u32x2_t){(unsigned)b, (unsigned)(b >> 32)}, 127, fmt, o);
        const int from = at + c, to = B8_BLOCK - from % B8_BLOCK;        // (values to .. 7 are the next block's)
        const float s0 = b8_scale(sr[from / B8_BLOCK]), s1 = b8_scale(sr[min(from + 7, 2 * F - 1) / B8_BLOCK]);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] *= j < to ? s0 : s1;
      };
      eight(0, v);
      eight(F, g);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int cc = min(c + j, F - 1);
        float o[8];
        b8_unpack8((u32x2_t){(unsigned)hr[cc], 0u}, sr[cc / B8_BLOCK], fmt, o); v[j] = o[0];
        b8_unpack8((u32x2_t){(unsigned)hr[F + cc], 0u}, sr[(F + cc) / B8_BLOCK], fmt, o); g[j] = o[0];
      }
    }
  } else {
    row_load8(hr, c, F, v);
    row_load8(hr + F, c, F, g);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float ge, sl;
    gelu_slope(g[j], ge, sl);
    dv[j] = d[j] * ge;
    dg[j] = d[j] * v[j] * sl;
  }
  row_store8<PAST>(dh + (size_t)row * 2 * F + c, F - c, dv);
  row_store8<PAST>(dh + (size_t)row * 2 * F + F + c, F - c, dg);
  if constexpr (BLOCKS) {
    const int sub = threadIdx.x & 15, FB = F / B8_BLOCK, fb = c / B8_BLOCK;
    auto block = [&](float (&x)[8], int col) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = bf2f(f2bf(x[j]));
      const int e = b8_exponent_of(b8_max16(b8_mag8(x)), q_fmt);
      *reinterpret_cast<u32x2_t*>(q + (size_t)row * 2 * F + col) = b8_pack8(x, e, q_fmt);
      if (sub == 0) q_scale[(size_t)row * SP + col / B8_BLOCK] = (unsigned char)e;
    };
    block(dv, c);
    block(dg, F + c);
    if (fb == FB - 1 && 2 * FB + sub < SP) q_scale[(size_t)row * SP + 2 * FB + sub] = 127;
  }
}

// ---------------------------------------------------------------------------------------------
// host entry points
// ---------------------------------------------------------------------------------------------
static bool is_fmt(int f) { return f == SDAMD_E4M3 || f == SDAMD_E5M2; }
static bool is_val(int d) { return d == SDAMD_F32 || d == SDAMD_BF16; }

extern "C" int sdamd_quant8(const void* x, void* q, unsigned char* scale, long long rows, int K, long long ldx, int dtype, int fmt, void* stream) {
  SD_CHECK(is_val(dtype) && is_fmt(fmt), "quant8: unsupported dtypes in=%d out=%d", dtype, fmt);
  SD_CHECK(rows > 0 && K > 0 && K <= (1 << 30) && ldx >= 0, "quant8: bad shape rows=%lld K=%d", rows, K);
  const int KB = b8_kblocks(K);
  SD_CHECK(rows <= (1ll << 40) && rows * (long long)KB <= (1ll << 29) - 32, "quant8: too large, rows=%lld K=%d", rows, K);
  const unsigned nblk = (unsigned)(rows * KB);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SDAMD_BF16)
    quant8_kernel<bf16_t, 2><<<(nblk + 31) / 32, 256, 0, st>>>((const bf16_t*)x, (unsigned char*)q, scale, nblk, KB, K, ldx, b8_scale_stride(K), fmt);
  else
    quant8_kernel<float, 2><<<(nblk + 31) / 32, 256, 0, st>>>((const float*)x, (unsigned char*)q, scale, nblk, KB, K, ldx, b8_scale_stride(K), fmt);
  SD_LAUNCH_CHECK("quant8");
  return 0;
}

extern "C" int sdamd_quant8_weight(const void* w, void* q, unsigned char* scale, int N, int K, long long sn, long long sk, int dtype, void* stream) {
  SD_CHECK(is_val(dtype), "quant8_weight: unsupported dtype %d", dtype);
  SD_CHECK(N > 0 && K > 0 && K <= (1 << 30) && sn >= 0 && sk >= 0, "quant8_weight: bad shape N=%d K=%d", N, K);
  const int KB = b8_kblocks(K), NB = b8_kblocks(N);
  SD_CHECK(NB <= 65535, "quant8_weight: N=%d is too large", N);
  hipStream_t st = (hipStream_t)stream;
#define QW_LAUNCH(T, ALONG) \
  quant8_weight_kernel<T, ALONG><<<dim3(KB, NB), 256, 0, st>>>((const T*)w, (unsigned char*)q, scale, N, K, sn, sk, KB, b8_scale_stride(K))
#define QW(T) { if (sk == 1) QW_LAUNCH(T, 1); else if (sn == 1) QW_LAUNCH(T, 2); else QW_LAUNCH(T, 0); }
  if (dtype == SDAMD_BF16) QW(bf16_t) else QW(float)
#undef QW
#undef QW_LAUNCH
  SD_LAUNCH_CHECK("quant8_weight");
  return 0;
}

extern "C" int sdamd_dequant8(const void* q, const unsigned char* scale, void* out, long long rows, int K, int block_rows, int fmt, int out_dtype, void* stream) {
  SD_CHECK(is_val(out_dtype) && is_fmt(fmt), "dequant8: unsupported dtypes in=%d out=%d", fmt, out_dtype);
  SD_CHECK(rows > 0 && K > 0 && K <= (1 << 30) && (block_rows == 1 || block_rows == B8_BLOCK), "dequant8: bad shape rows=%lld K=%d block_rows=%d", rows, K, block_rows);
  const int KB = b8_kblocks(K);
  SD_CHECK(rows <= (1ll << 40) && rows * (long long)KB <= (1ll << 28) - 16, "dequant8: too large, rows=%lld K=%d", rows, K);
  const unsigned nblk = (unsigned)(rows * KB);
  const int shift = block_rows == 1 ? 0 : 7, SP = b8_scale_stride(K);
  hipStream_t st = (hipStream_t)stream;
  if (out_dtype == SDAMD_BF16)
    dequant8_kernel<bf16_t><<<(nblk + 15) / 16, 256, 0, st>>>((const unsigned char*)q, scale, (bf16_t*)out, nblk, KB, K, SP, shift, fmt);
  else
    dequant8_kernel<float><<<(nblk + 15) / 16, 256, 0, st>>>((const unsigned char*)q, scale, (float*)out, nblk, KB, K, SP, shift, fmt);
  SD_LAUNCH_CHECK("dequant8");
  return 0;
}

static int geglu_rows_of_a_workgroup(int KB) { return max(1, 32 / KB); }
template <typename T>
static void geglu_train_launch(const T* h, void* out, unsigned char* out_scale, unsigned char* q, unsigned char* scale, long long rows, int F,
                               int fmt, int out_dtype, hipStream_t st) {
  const int SP = b8_scale_stride(2 * F);
  if (F % B8_BLOCK == 0) {
    const unsigned nblk = (unsigned)(rows * (F / B8_BLOCK));
    auto k = is_fmt(out_dtype) ? geglu_train_kernel<T, GEGLU_BLOCKS>
             : b8_past_cache((double)rows * F * sizeof(T)) ? geglu_train_kernel<T, GEGLU_PAST> : geglu_train_kernel<T, GEGLU_DENSE>;
    k<<<(nblk + 15) / 16, 256, 0, st>>>(h, out, out_scale, q, scale, nblk, F / B8_BLOCK, SP, fmt, out_dtype);
  } else {
    const int KB = b8_kblocks(2 * F), R = geglu_rows_of_a_workgroup(KB);
    auto k = is_fmt(out_dtype) ? geglu_rows_kernel<T, true> : geglu_rows_kernel<T, false>;
    k<<<(unsigned)((rows + R - 1) / R), 256, 0, st>>>(h, out, out_scale, q, scale, rows, R, F, KB, SP, fmt, out_dtype);
  }
}

extern "C" int sdamd_geglu_train(const void* h, void* out, unsigned char* out_scale, void* q, unsigned char* scale, long long rows, int F, int dtype,
                                 int out_dtype, int fmt, void* stream) {
  SD_CHECK(is_val(dtype) && (out_dtype == dtype || is_fmt(out_dtype)) && is_fmt(fmt), "geglu_train: unsupported dtypes h=%d out=%d kept=%d", dtype, out_dtype, fmt);
  SD_CHECK(!is_fmt(out_dtype) || out_scale, "geglu_train: 8-bit output without room for its scales");
  SD_CHECK(rows > 0 && F > 0 && F <= (1 << 29), "geglu_train: bad shape rows=%lld F=%d", rows, F);
  SD_CHECK(rows <= (1ll << 40) && rows * (long long)((F + 7) / 8) < (1ll << 31) && (F % B8_BLOCK == 0 || rows / geglu_rows_of_a_workgroup(b8_kblocks(2 * F)) < (1ll << 24) - 1),
           "geglu_train: too large, rows=%lld F=%d", rows, F);
  if (dtype == SDAMD_BF16) geglu_train_launch<bf16_t>((const bf16_t*)h, out, out_scale, (unsigned char*)q, scale, rows, F, fmt, out_dtype, (hipStream_t)stream);
  else geglu_train_launch<float>((const float*)h, out, out_scale, (unsigned char*)q, scale, rows, F, fmt, out_dtype, (hipStream_t)stream);
  SD_LAUNCH_CHECK("geglu_train");
  return 0;
}

template <typename TD, typename TH, typename TO, typename... A>
static void geglu_backward_launch(dim3 grid, hipStream_t st, bool past, bool blocks, A... a) {
  auto k = past ? geglu_backward_kernel<TD, TH, TO, true, false> : geglu_backward_kernel<TD, TH, TO, false, false>;
  if constexpr (sizeof(TO) == 2) {
    if (blocks) k = past ? geglu_backward_kernel<TD, TH, TO, true, true> : geglu_backward_kernel<TD, TH, TO, false, true>;
  }
  k<<<grid, 256, 0, st>>>(a...);
}

extern "C" int sdamd_geglu_backward(const void* dout, const void* h, const unsigned char* h_scale, void* dh, void* q, unsigned char* q_scale,
                                    long long rows, int F, int dout_dtype, int h_dtype, int dh_dtype, int q_fmt, void* stream) {
  SD_CHECK(is_val(dout_dtype) && is_val(dh_dtype) && (is_val(h_dtype) || is_fmt(h_dtype)), "geglu_backward: unsupported dtypes dout=%d h=%d dh=%d",
           dout_dtype, h_dtype, dh_dtype);
  SD_CHECK(!is_fmt(h_dtype) || h_scale, "geglu_backward: 8-bit h without its scales");
  SD_CHECK(!q || (is_fmt(q_fmt) && q_scale && dh_dtype == SDAMD_BF16 && F % B8_BLOCK == 0), "geglu_backward: blocks of dh need room for scales, bf16 dh and F %% 128 == 0 (F=%d)", F);
  SD_CHECK(rows > 0 && F > 0 && F <= (1 << 29), "geglu_backward: bad shape rows=%lld F=%d", rows, F);
  const int VR = (F + 7) / 8;
  SD_CHECK(rows <= (1ll << 40) && rows * (long long)VR < (1ll << 31), "geglu_backward: too large, rows=%lld F=%d", rows, F);
  const unsigned nvec = (unsigned)(rows * VR);
  hipStream_t st = (hipStream_t)stream;
  const int SP = b8_scale_stride(2 * F), ldq = b8_kblocks(2 * F) * B8_BLOCK;
  const bool past = b8_past_cache((double)rows * 2 * F * (dh_dtype == SDAMD_F32 ? 4 : 2));
#define GB_LAUNCH(TD, TH, TO, LD) \
  geglu_backward_launch<TD, TH, TO>(dim3((nvec + 255) / 256), st, past, q != nullptr, (const TD*)dout, (const TH*)h, h_scale, (TO*)dh, nvec, VR, F, \
                                    LD, SP, h_dtype, (unsigned char*)q, q_scale, q_fmt)
#define GB_H(TD, TO) \
  { if (h_dtype == SDAMD_F32) GB_LAUNCH(TD, float, TO, 2 * F); else if (h_dtype == SDAMD_BF16) GB_LAUNCH(TD, bf16_t, TO, 2 * F); else GB_LAUNCH(TD, unsigned char, TO, ldq); }
  if (dout_dtype == SDAMD_F32) { if (dh_dtype == SDAMD_F32) GB_H(float, float) else GB_H(float, bf16_t) }
  else { if (dh_dtype == SDAMD_F32) GB_H(bf16_t, float) else GB_H(bf16_t, bf16_t) }
#undef GB_H
#undef GB_LAUNCH
  SD_LAUNCH_CHECK("geglu_backward");
  return 0;
}
