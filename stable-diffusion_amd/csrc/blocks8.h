// Device helpers of the 8-bit block format (SDAMD_E4M3 / SDAMD_E5M2, include/sdamd.h): 128 consecutive values of a row
// share one power-of-two scale 2^(e-127), kept as the byte e.
//
//   e = the smallest power of two with  max |x| <= top * 2^(e-127),  top = 448 (e4m3) or 57344 (e5m2)
//   q = x / 2^(e-127) rounded to nearest even in the 8-bit type
//
// A power of two, not max |x| / top: the division by the scale and the way back are exact, so the 8-bit rounding is the
// only one (half a step, 2^-4 of an e4m3 value); bf16 holds q * scale exactly, so a bf16 MFMA of a dequantised block has
// exact products; and the matrix core takes such a scale as an operand of its own.  In a floating 8-bit type the finer
// scale would buy nothing: the relative step is the same wherever in the range the block's maximum lands.
#pragma once
#include "common.h"

#define SDAMD_E4M3 2
#define SDAMD_E5M2 3

constexpr int B8_BLOCK = 128;      // values that share a scale (weights: 128 rows x 128 columns)

static inline int b8_kblocks(int K) { return (K + B8_BLOCK - 1) / B8_BLOCK; }
static inline int b8_scale_stride(int K) { return (b8_kblocks(K) + 3) / 4 * 4; }   // bytes of scale per row: whole 32-bit words

// bit pattern of |x| where x is finite, else 0: unsigned order = order of magnitudes
__device__ __forceinline__ unsigned b8_mag(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// scale byte of a block whose largest finite magnitude has the bits `mag`; TOP_EXP = exponent of the type's maximum
// 1.75 * 2^TOP_EXP.  A block of zeros (or without finite values) gets scale 1.
template <int TOP_EXP> __device__ __forceinline__ int b8_exponent(unsigned mag) {
  const int e = (int)(mag >> 23) - TOP_EXP + ((mag & 0x7fffffu) > 0x600000u ? 1 : 0);
  return mag == 0u ? 127 : max(e, 1);
}
// runtime choice of the type (uniform over the launch)
__device__ __forceinline__ int b8_exponent_of(unsigned mag, int fmt) {
  return fmt == SDAMD_E4M3 ? b8_exponent<8>(mag) : b8_exponent<15>(mag);
}
__device__ __forceinline__ float b8_scale(int e) {          // 2^(e-127); e = 0 is the subnormal 2^-127, 255 is NaN
  return __builtin_bit_cast(float, e == 0 ? 0x400000u : e == 255 ? 0x7fc00000u : (unsigned)e << 23);
}
__device__ __forceinline__ float b8_inverse(int e) {        // 2^(127-e) for 1 <= e <= 253
  return __builtin_bit_cast(float, (unsigned)(254 - e) << 23);
}
// four values (already divided by the scale) -> four bytes.  Infinities become NaN in e4m3, which has none.
__device__ __forceinline__ unsigned b8_pack4(float a, float b, float c, float d, int fmt) {
  int r = 0;
  if (fmt == SDAMD_E4M3) {
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  } else {
    r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
  }
  return (unsigned)r;
}
__device__ __forceinline__ u32x2_t b8_pack8(const float (&v)[8], int e, int fmt) {
  const float inv = b8_inverse(e);
  return (u32x2_t){b8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, fmt),
                   b8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv, fmt)};
}
// eight bytes -> the values they stand for
__device__ __forceinline__ void b8_unpack8(u32x2_t q, int e, int fmt, float (&v)[8]) {
  typedef __attribute__((ext_vector_type(2))) float v2;
  const float s = b8_scale(e);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v2 lo, hi;
    if (fmt == SDAMD_E4M3) {
      lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false);
      hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
    } else {
      lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)q[h], false);
      hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)q[h], true);
    }
    v[4 * h] = lo[0] * s; v[4 * h + 1] = lo[1] * s; v[4 * h + 2] = hi[0] * s; v[4 * h + 3] = hi[1] * s;
  }
}
// largest magnitude over the 16 lanes that hold a block: rotations within the 16, in the vector unit (data-parallel
// primitives; __shfl would go through LDS four times)
template <int N> __device__ __forceinline__ unsigned b8_rotate16(unsigned m) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x120 + N, 0xf, 0xf, true);
}
__device__ __forceinline__ unsigned b8_max16(unsigned m) {
  m = max(m, b8_rotate16<8>(m));
  m = max(m, b8_rotate16<4>(m));
  m = max(m, b8_rotate16<2>(m));
  return max(m, b8_rotate16<1>(m));
}
__device__ __forceinline__ unsigned b8_mag8(const float (&v)[8]) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, b8_mag(v[j]));
  return m;
}

// ---- rows of any width and alignment -------------------------------------------------------------------------------
// A row's eight values from column c on.  Global memory takes 16-byte accesses at any element alignment on this hardware,
// so odd widths keep the wide loads.  Loading is split from unpacking so that a kernel can request all its vectors before
// it uses the first: raw8_load reads at min(c, C - 8), inside the row whatever c is, without a branch around the load;
// raw8_get moves a row's last, partial vector into place and zeroes what lies past C.  C < 8 goes value by value.
typedef u32x4_t __attribute__((aligned(2))) b8_u32x4_a2;
typedef f32x4_t __attribute__((aligned(4))) b8_f32x4_a4;
template <typename T> struct Raw8;
template <> struct Raw8<float> { f32x4_t a, b; };
template <> struct Raw8<bf16_t> { u32x4_t a; };

template <typename T> __device__ __forceinline__ Raw8<T> raw8_load(const T* row, int c, int C) {
  Raw8<T> r;
  if (C < 8) {                                   // (uniform over the launch)
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) { r.a[j] = j < C ? row[j] : 0.f; r.b[j] = 4 + j < C ? row[4 + j] : 0.f; }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r.a[j] = (2 * j < C ? (unsigned)row[2 * j] : 0u) | (2 * j + 1 < C ? (unsigned)row[2 * j + 1] << 16 : 0u);
    }
    return r;
  }
  const T* p = row + min(c, C - 8);
  if constexpr (sizeof(T) == 4) {
    r.a = *reinterpret_cast<const b8_f32x4_a4*>(p);
    r.b = *reinterpret_cast<const b8_f32x4_a4*>(p + 4);
  } else {
    r.a = *reinterpret_cast<const b8_u32x4_a2*>(p);
  }
  return r;
}
template <typename T> __device__ __forceinline__ void raw8_get(const Raw8<T>& r, int c, int C, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = r.a[j]; v[4 + j] = r.b[j]; }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __builtin_bit_cast(float, r.a[i] << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, r.a[i] & 0xffff0000u);
    }
  }
  if (C % 8 != 0) {                              // (uniform) shift a partial vector down by c - (C - 8)
    const int s = C < 8 ? c : max(c - (C - 8), 0);
    if (s > 0) {                                 // (one vector of a row: most waves branch over it)
#pragma unroll
      for (int b = 4; b > 0; b >>= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = s & b ? (j + b < 8 ? v[j + b] : 0.f) : v[j];
    }
  }
  if (c >= C) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
  }
}
template <typename T> __device__ __forceinline__ void row_load8(const T* row, int c, int C, float (&v)[8]) {
  const Raw8<T> r = raw8_load(row, c, C);
  raw8_get(r, c, C, v);
}
// Results of half the last-level cache (256 MB) or more are written past it: whoever reads them next finds the larger part
// gone anyway, and the lines they would push out are the operands'.  (Alone, operands and results from rotating buffers: 36864 x
// 1280 -> 10240, 755 MB: 497 us kept, 473 past; 16384 x 640 -> 5120, 168 MB: 73.9 and 62.6, with the GeGLU that reads it
// 132.7 and 135.8; 65536 x 320 -> 2560, 336 MB, with its GeGLU 241 and 234; 4096 x 1280 -> 10240, 84 MB, with its GeGLU 93.1
// and 104.3: so not the smaller ones.)
static inline bool b8_past_cache(double bytes) { return bytes >= 134217728.0; }
// store the n (<= 8, may be <= 0) values that belong to the row; PAST: past the cache (a template argument: the compiler joins the two stores of a branch into a plain one)
template <bool PAST = false> __device__ __forceinline__ void row_store8(float* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    const f32x4_t lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
    b8_f32x4_a4* d = reinterpret_cast<b8_f32x4_a4*>(p);
    if constexpr (PAST) { __builtin_nontemporal_store(lo, d); __builtin_nontemporal_store(hi, reinterpret_cast<b8_f32x4_a4*>(p + 4)); }
    else { *d = lo; *reinterpret_cast<b8_f32x4_a4*>(p + 4) = hi; }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) p[j] = v[j];
  }
}
template <bool PAST = false> __device__ __forceinline__ void row_store8(bf16_t* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    u32x4_t t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = pack_bf2(v[2 * i], v[2 * i + 1]);
    if constexpr (PAST) __builtin_nontemporal_store(t, reinterpret_cast<b8_u32x4_a2*>(p));
    else *reinterpret_cast<b8_u32x4_a2*>(p) = t;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j < n) p[j] = f2bf(v[j]);
  }
}
