// Linear on 8-bit blocks (blocks8.h):  out[m][n] = act( sum_k A[m][k] W[n][k] + bias[n] + residual[m][n] )
//   A [M][KB*128] e4m3 or e5m2, one scale byte per row and 128 columns; W [N][KB*128] e4m3, one per 128 x 128 block.
//
// The matrix core multiplies two 8-bit blocks of 128 and their power-of-two scales in one instruction
// (v_mfma_scale_f32_16x16x128_f8f6f4): no vector instruction touches the products, the sums stay in f32 registers.
// Inside such an instruction the 128 products are aligned to the largest of them and cut about 2^-20 below it before they
// are added (measured against 64 bits: 1.4e-5 relative per block of normally distributed operands, no bias to speak of).
// That is 1/100 of a bf16 rounding, so a bf16 result takes this form (3.8 PFLOP/s measured from registers), but it is not
// an f32 sum: for an f32 result (EXACT) the bytes and their scales go to bf16, which holds them exactly, and through
// v_mfma_f32_16x16x32_bf16, whose products and sums are exact to f32 rounding (1.9 PFLOP/s from registers).
//
// "A" of the instruction = weight rows, "B" = activation rows: a lane ends up with 4 consecutive columns of one row.
// Which 32 of a block's 128 values a lane supplies does not matter as long as both operands agree, the scales covering
// the whole block.
#include "blocks8.h"
#include "gemm_common.h"

typedef __attribute__((address_space(3))) void lds_void8_t;
typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2v_t;

struct G8Args {
  const void* A;                   // blocks, or the rows themselves (XRAW)
  const unsigned char* As;
  const unsigned char* W;
  const unsigned char* Ws;
  void* out;
  const float* bias;
  const void* residual;
  int M, N, K, KB, SP, act;
  int tiles_m, tiles_n;
};

// one 128-wide step of a 16 x 16 tile
template <int FMT> __device__ __forceinline__ f32x4_t mfma8(i32x8_t w, i32x8_t a, f32x4_t c, int sw, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, FMT == SDAMD_E5M2 ? 1 : 0, 0, sw, 0, sa);
}
// the EXACT operand: 32 bytes and their scale -> four bf16 fragments
struct Bf4 { bf16x8_t q[4]; };
template <int FMT> __device__ __forceinline__ Bf4 to_bf16(i32x8_t v, float s) {
  Bf4 o;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    bf16x2v_t p[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (FMT == SDAMD_E4M3) {
        p[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * q + h], s, false);
        p[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * q + h], s, true);
      } else {
        p[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v[2 * q + h], s, false);
        p[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v[2 * q + h], s, true);
      }
    }
    o.q[q] = (bf16x8_t){p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
  }
  return o;
}

typedef u32x2_t __attribute__((aligned(2))) g8_u32x2_a2;
typedef f32x4_t __attribute__((aligned(4))) g8_f32x4_a4;
__device__ __forceinline__ float g8_act(float v, int act) {
  return act == ACT_SILU ? silu_f(v) : act == ACT_QUICK_GELU ? quick_gelu_f(v) : v;
}
// four consecutive columns of row m: + bias + residual, activation, one rounding to the output type
template <typename TO> __device__ __forceinline__ void g8_store(const G8Args& p, int m, int n, f32x4_t v) {
  if (m >= p.M || n >= p.N) return;
  const size_t at = (size_t)m * p.N + n;
  TO* o = (TO*)p.out + at;
  const TO* r = p.residual ? (const TO*)p.residual + at : nullptr;
  if (n + 4 <= p.N) {
    if (p.bias) v += *reinterpret_cast<const g8_f32x4_a4*>(p.bias + n);
    if (r) {
      if constexpr (sizeof(TO) == 4) v += *reinterpret_cast<const g8_f32x4_a4*>(r);
      else {
        const u32x2_t t = *reinterpret_cast<const g8_u32x2_a2*>(r);
        v += (f32x4_t){__builtin_bit_cast(float, t[0] << 16), __builtin_bit_cast(float, t[0] & 0xffff0000u),
                       __builtin_bit_cast(float, t[1] << 16), __builtin_bit_cast(float, t[1] & 0xffff0000u)};
      }
    }
    if (p.act) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = g8_act(v[j], p.act);
    }
    if constexpr (sizeof(TO) == 4) *reinterpret_cast<g8_f32x4_a4*>(o) = v;
    else *reinterpret_cast<g8_u32x2_a2*>(o) = (u32x2_t){pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) {
        float w = v[j];
        if (p.bias) w += p.bias[n + j];
        if (r) w += Cvt<TO>::ld(r + j);
        Cvt<TO>::st(o + j, g8_act(w, p.act));
      }
  }
}

// ---- large problems ------------------------------------------------------------------------------------------------
// Workgroup tile BM x BN, WGM x WGN waves, K step 128 = 128 bytes per row.  Both operands go global -> LDS by
// global_load_lds_dwordx4 (8 rows of 128 bytes per wave instruction) into two buffers: step t is multiplied while t + 1
// is on its way.  The 16-byte chunks of a row are permuted by (row >> 1) & 7 on the way in and on the way out, which
// spreads the rows a fragment read touches over all banks.
__device__ __forceinline__ void dma16(const void* g, void* lds) {
  // (inline assembly: the builtin makes the compiler wait for all of LDS at every later fragment read; its completion is
  // this kernel's business, s_waitcnt vmcnt(0) and a barrier before the data is read)
  const unsigned l = (unsigned)(unsigned long)(lds_void8_t*)lds;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(g) : "memory", "m0");
}

template <int BM, int BN, int WGM, int WGN, int FMT, bool EXACT, typename TO>
__global__ __launch_bounds__(64 * WGM * WGN) void gemm8_kernel(G8Args p) {
  constexpr int NW = WGM * WGN, TM = BM / WGM / 16, TN = BN / WGN / 16;
  constexpr int STAGE = (BM + BN) * 128, NI = (BM + BN) / 8 / NW;
  static_assert((BM + BN) % (8 * NW) == 0 && 128 % (BN / WGN) == 0, "tile shape");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;

  // Workgroups go round robin over the 8 XCDs, each with an L2 of its own: give every XCD a run of neighbouring tiles, in
  // groups of 8 row tiles that share their weight tiles.
  int id = blockIdx.x;
  {
    const int total = p.tiles_m * p.tiles_n, per = total / 8, rem = total % 8, x = id % 8, r = id / 8;
    id = x * per + min(x, rem) + r;
  }
  const int group = id / (8 * p.tiles_n), first = group * 8, gm = min(8, p.tiles_m - first), in = id - group * 8 * p.tiles_n;
  const int m0 = (first + in % gm) * BM, n0 = (in / gm) * BN;

  const unsigned char* src[NI];
  int dst[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = (wave * NI + i) * 8 + (lane >> 3), ch = (lane & 7) ^ ((row >> 1) & 7);
    const unsigned char* base = row < BM ? (const unsigned char*)p.A + (size_t)min(m0 + row, p.M - 1) * p.KB * B8_BLOCK
                                         : p.W + (size_t)min(n0 + row - BM, p.N - 1) * p.KB * B8_BLOCK;
    src[i] = base + ch * 16;
    dst[i] = (wave * NI + i) * 1024;
  }
  auto stage = [&](int kb, int buf) {
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16(src[i] + (size_t)kb * B8_BLOCK, smem + buf * STAGE + dst[i]);
  };
  // scales: four steps per 32-bit word; a lane holds those of the rows it supplies
  const unsigned char* sa[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) sa[i] = p.As + (size_t)min(m0 + (wm * TM + i) * 16 + (lane & 15), p.M - 1) * p.SP;
  const unsigned char* sw = p.Ws + (size_t)(min(n0 + wn * TN * 16, p.N - 1) / B8_BLOCK) * p.SP;
  unsigned sca[TM], scw, nxa[TM], nxw;
#pragma unroll
  for (int i = 0; i < TM; ++i) nxa[i] = *reinterpret_cast<const unsigned*>(sa[i]);
  nxw = *reinterpret_cast<const unsigned*>(sw);

  f32x4_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  const int r16 = lane & 15, g = lane >> 4;
  auto frag = [&](const char* base, int row) {
    const int o = row * 128 + ((g ^ ((row >> 1) & 7)) << 4);
    const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(base + o), hi = *reinterpret_cast<const u32x4_t*>(base + (o ^ 64));
    return (i32x8_t){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };

  stage(0, 0);
  for (int kb = 0; kb < p.KB; ++kb) {
    // step kb has landed (it was issued a whole step ago), and this wave's reads of step kb - 1 are done
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if ((kb & 3) == 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i) { asm volatile("" : "+v"(nxa[i])); sca[i] = nxa[i]; }   // (used here, where nothing is in flight)
      asm volatile("" : "+v"(nxw));
      scw = nxw;
    }
    __builtin_amdgcn_s_barrier();
    if (kb + 1 < p.KB) stage(kb + 1, (kb + 1) & 1);
    if ((kb & 3) == 3 && kb + 1 < p.KB) {
#pragma unroll
      for (int i = 0; i < TM; ++i) nxa[i] = *reinterpret_cast<const unsigned*>(sa[i] + kb + 1);
      nxw = *reinterpret_cast<const unsigned*>(sw + kb + 1);
    }
    const char* sA = smem + (kb & 1) * STAGE;
    const char* sW = sA + BM * 128;
    const int sh = (kb & 3) * 8;
    const int bw = (int)(scw >> sh);
    if constexpr (!EXACT) {
      i32x8_t w[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) w[j] = frag(sW, (wn * TN + j) * 16 + r16);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const i32x8_t a = frag(sA, (wm * TM + i) * 16 + r16);
        const int ba = (int)(sca[i] >> sh);
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma8<FMT>(w[j], a, acc[i][j], bw, ba);
      }
    } else {
      Bf4 w[TN];
      const float fw = b8_scale(bw & 255);
#pragma unroll
      for (int j = 0; j < TN; ++j) w[j] = to_bf16<SDAMD_E4M3>(frag(sW, (wn * TN + j) * 16 + r16), fw);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const Bf4 a = to_bf16<FMT>(frag(sA, (wm * TM + i) * 16 + r16), b8_scale((int)(sca[i] >> sh) & 255));
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j].q[q], a.q[q], acc[i][j], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
      g8_store<TO>(p, m0 + (wm * TM + i) * 16 + r16, n0 + (wn * TN + j) * 16 + g * 4, acc[i][j]);
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// 16 columns and up to 16 * MT rows per workgroup; its 8 waves share out the blocks of K and read them straight into
// registers (every weight byte is used once: LDS would only delay it), then join their sums in a fixed order in LDS.
// XRAW: A is the f32 / bf16 rows themselves, quantised on the way in (a block of a row lies in the four lanes 16 apart).
template <int MT, int FMT, bool EXACT, typename TO, typename TX>
__global__ __launch_bounds__(512) void gemm8_rows_kernel(G8Args p) {
  constexpr bool XRAW = sizeof(TX) != 1;
  constexpr int LD = 20;                                   // floats per row of the exchange: 16 columns, 16-byte aligned
  __shared__ __attribute__((aligned(16))) float ex[8][MT * 16][LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const unsigned char* wr = p.W + (size_t)min(n0 + r16, p.N - 1) * p.KB * B8_BLOCK + g * 32;
  const unsigned char* sw = p.Ws + (size_t)(n0 / B8_BLOCK) * p.SP;
  f32x4_t acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < p.KB; kb += 8) {
    const u32x4_t* wp = reinterpret_cast<const u32x4_t*>(wr + (size_t)kb * B8_BLOCK);
    const u32x4_t w0 = wp[0], w1 = wp[1];
    const int bw = sw[kb];
    i32x8_t a[MT];
    int ba[MT];
    if constexpr (!XRAW) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const size_t m = min(m0 + i * 16 + r16, p.M - 1);
        const u32x4_t* ap = reinterpret_cast<const u32x4_t*>((const unsigned char*)p.A + (m * p.KB + kb) * B8_BLOCK + g * 32);
        const u32x4_t a0 = ap[0], a1 = ap[1];
        ba[i] = p.As[m * p.SP + kb];
        a[i] = (i32x8_t){(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const size_t m = min(m0 + i * 16 + r16, p.M - 1);
        const TX* xr = (const TX*)p.A + m * p.K;
        Raw8<TX> raw[4];
        float v[4][8];
        unsigned mag = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[q] = raw8_load(xr, kb * B8_BLOCK + g * 32 + q * 8, p.K);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          raw8_get(raw[q], kb * B8_BLOCK + g * 32 + q * 8, p.K, v[q]);
          mag = max(mag, b8_mag8(v[q]));
        }
        mag = max(mag, (unsigned)__shfl_xor((int)mag, 16, 64));
        mag = max(mag, (unsigned)__shfl_xor((int)mag, 32, 64));
        ba[i] = b8_exponent_of(mag, FMT);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x2_t t = b8_pack8(v[q], ba[i], FMT);
          a[i][2 * q] = (int)t[0];
          a[i][2 * q + 1] = (int)t[1];
        }
      }
    }
    const i32x8_t w = {(int)w0[0], (int)w0[1], (int)w0[2], (int)w0[3], (int)w1[0], (int)w1[1], (int)w1[2], (int)w1[3]};
    if constexpr (!EXACT) {
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = mfma8<FMT>(w, a[i], acc[i], bw, ba[i]);
    } else {
      const Bf4 wb = to_bf16<SDAMD_E4M3>(w, b8_scale(bw));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const Bf4 ab = to_bf16<FMT>(a[i], b8_scale(ba[i]));
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb.q[q], ab.q[q], acc[i], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4_t*>(&ex[wave][i * 16 + r16][g * 4]) = acc[i];
  __syncthreads();
  for (int t = threadIdx.x; t < MT * 64; t += 512) {
    const int row = t >> 2, c = (t & 3) * 4;
    f32x4_t s = *reinterpret_cast<const f32x4_t*>(&ex[0][row][c]);
#pragma unroll
    for (int w = 1; w < 8; ++w) s += *reinterpret_cast<const f32x4_t*>(&ex[w][row][c]);
    g8_store<TO>(p, m0 + row, n0 + c, s);
  }
}

// ---------------------------------------------------------------------------------------------
// host entry points
// ---------------------------------------------------------------------------------------------
// Few tiles: the kernel without LDS staging, which also splits K over the waves of a workgroup.
static bool g8_few_rows(int M, int N) {
  const long long t128 = (long long)((M + 127) / 128) * ((N + 127) / 128);
  return M <= 64 || (t128 < 96 && (M + 63) / 64 <= 65535);
}
// That kernel can quantise rows on its way.  Every workgroup then repeats the work for its rows, so it does where that is
// cheaper than a launch of its own: up to G8_RAW_WORK values over all workgroups.
constexpr long long G8_RAW_WORK = 1ll << 24;
extern "C" int sdamd_linear8_quantises(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return g8_few_rows(M, N) && (long long)((N + 15) / 16) * M <= G8_RAW_WORK / K;
}

template <int BM, int BN, int WGM, int WGN, int FMT, bool EXACT, typename TO>
static int g8_tile_launch(G8Args p, hipStream_t st) {
  static std::atomic<unsigned long long> done{0};
  constexpr int lds = 2 * (BM + BN) * 128;
  auto k = gemm8_kernel<BM, BN, WGM, WGN, FMT, EXACT, TO>;
  const hipError_t e = sd_lds_opt_in(done, (const void*)k, lds);
  if (e != hipSuccess) return sdamd_set_error(2, "linear8: %s", hipGetErrorString(e));
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  k<<<p.tiles_m * p.tiles_n, 64 * WGM * WGN, lds, st>>>(p);
  return 0;
}

template <int FMT, bool EXACT, typename TO>
static int g8_launch(const G8Args& p, int x_dtype, hipStream_t st) {
  if (g8_few_rows(p.M, p.N)) {
    const dim3 grid((p.N + 15) / 16, p.M <= 32 ? 1 : (p.M + 63) / 64);
#define G8_ROWS(TX)                                                                              \
  do {                                                                                           \
    if (p.M <= 16) gemm8_rows_kernel<1, FMT, EXACT, TO, TX><<<grid, 512, 0, st>>>(p);            \
    else if (p.M <= 32) gemm8_rows_kernel<2, FMT, EXACT, TO, TX><<<grid, 512, 0, st>>>(p);       \
    else gemm8_rows_kernel<4, FMT, EXACT, TO, TX><<<grid, 512, 0, st>>>(p);                      \
  } while (0)
    if (x_dtype == SDAMD_F32) G8_ROWS(float); else if (x_dtype == SDAMD_BF16) G8_ROWS(bf16_t); else G8_ROWS(unsigned char);
#undef G8_ROWS
    return 0;
  }
  const long long t256 = (long long)((p.M + 255) / 256) * ((p.N + 255) / 256), t128 = (long long)((p.M + 127) / 128) * ((p.N + 127) / 128);
  SD_CHECK(t128 < (1ll << 31), "linear8: too large, M=%d N=%d", p.M, p.N);
  if constexpr (!EXACT) {
    if (t256 >= 192) return g8_tile_launch<256, 256, 2, 4, FMT, EXACT, TO>(p, st);
  }
  return g8_tile_launch<128, 128, 2, 2, FMT, EXACT, TO>(p, st);
}

extern "C" int sdamd_linear8(const void* x, const unsigned char* x_scale, const void* w, const unsigned char* w_scale, void* out, const float* bias,
                             const void* residual, int M, int N, int K, int act, int x_dtype, int fmt, int out_dtype, void* stream) {
  SD_CHECK((out_dtype == SDAMD_F32 || out_dtype == SDAMD_BF16) && (fmt == SDAMD_E4M3 || fmt == SDAMD_E5M2) &&
           (x_dtype == SDAMD_F32 || x_dtype == SDAMD_BF16 || x_dtype == fmt), "linear8: unsupported dtypes x=%d fmt=%d out=%d", x_dtype, fmt, out_dtype);
  SD_CHECK(M > 0 && N > 0 && K > 0 && N <= (1 << 30) && K <= (1 << 30), "linear8: bad shape M=%d N=%d K=%d", M, N, K);
  SD_CHECK(act == ACT_NONE || act == ACT_QUICK_GELU || act == ACT_SILU, "linear8: unsupported activation %d", act);
  SD_CHECK(x_dtype >= SDAMD_E4M3 || sdamd_linear8_quantises(M, N, K), "linear8: M=%d N=%d K=%d: the rows have to be quantised first", M, N, K);
  SD_CHECK(x_dtype < SDAMD_E4M3 || x_scale, "linear8: 8-bit rows without their scales");
  G8Args p{x, x_scale, (const unsigned char*)w, w_scale, out, bias, residual, M, N, K, b8_kblocks(K), b8_scale_stride(K), act, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (out_dtype == SDAMD_F32) rc = fmt == SDAMD_E4M3 ? g8_launch<SDAMD_E4M3, true, float>(p, x_dtype, st) : g8_launch<SDAMD_E5M2, true, float>(p, x_dtype, st);
  else rc = fmt == SDAMD_E4M3 ? g8_launch<SDAMD_E4M3, false, bf16_t>(p, x_dtype, st) : g8_launch<SDAMD_E5M2, false, bf16_t>(p, x_dtype, st);
  if (rc) return rc;
  SD_LAUNCH_CHECK("linear8");
  return 0;
}
