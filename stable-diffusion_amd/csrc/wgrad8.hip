// Weight and bias gradient of a Linear from the 8-bit checkpoint of its input (blocks8.h):
//   dW[n][k] = sum_t dy[t][n] x8[t][k],   db[n] = sum_t dy[t][n];   dy [T][N] bf16, x8 [T][KB*128] with a scale per row and 128
// The reduction runs over tokens, along which the scales change, so the 8-bit instruction (one scale per operand row)
// cannot take x8.  Its bytes go to bf16 on the way into LDS, scaled: bf16 holds every such value exactly, so all products
// are exact and the sums are f32, whatever the checkpoint's type.  Bound by the bf16 matrix rate for wide layers
// (16384 x 5120 x 640: 0.72 PFLOP/s, 8192^3 1.1); the narrow ones by their splits: 65536 x 320 x 320 in 54 of them 40 us (floor 13),
// 16384 x 640 x 640 in 10 35 (11), 8192 x 1280 x 1280 in 5 48 (22).  dy is bf16 as the instruction's other operand: an f32 gradient
// is rounded by whoever has it, or would take three such products.
//
// Workgroup tile BT_N x BT_K of dW, token steps of 64, two LDS buffers.  Both operands arrive as rows of one token and are
// needed as columns of 8 tokens: ds_read_b64_tr_b16 turns 4 x 16 blocks on the way out of LDS.  A row's 32-byte units (16
// columns) are permuted by f(t) = (t & 3) | ((t >> 3) & 1) << 2: the 16 rows such a read touches fall on all 64 banks.
// "A" of the instruction = columns k, "B" = columns n: a lane ends up with 4 consecutive k of one n.
// db costs one more instruction per n tile and step, against a row of ones, in the waves of the first k tile.
// Few tiles and many tokens: the tokens are split over workgroups, which leave f32 partial sums; a second launch adds them
// in a fixed order (no atomics: the same bits every run).
#include "blocks8.h"
#include "gemm_common.h"
#include <type_traits>

typedef __attribute__((address_space(3))) void lds_voidw_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2w_t;
typedef f32x4_t __attribute__((aligned(4))) w8_f32x4_a4;

static __device__ __attribute__((aligned(256))) const unsigned int g_wgrad_zero[4] = {0};

struct W8Args {
  const bf16_t* dy;
  const unsigned char* q;
  const unsigned char* qs;
  float* dw;        // [splits][N][K] partial sums, or the result
  float* db;        // [splits][N], or the result; null: not wanted
  int T, N, K, KB, SP;
  int tiles_n, tiles_k, steps;   // steps: token steps of 64 per split
};

template <int FMT> __device__ __forceinline__ void w8_to_bf16(u32x4_t v, float s, u32x4_t& lo, u32x4_t& hi) {
  unsigned o[8];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    bf16x2w_t a, b;
    if constexpr (FMT == SDAMD_E4M3) {
      a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)v[h], s, false);
      b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)v[h], s, true);
    } else {
      a = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)v[h], s, false);
      b = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)v[h], s, true);
    }
    o[2 * h] = __builtin_bit_cast(unsigned, a);
    o[2 * h + 1] = __builtin_bit_cast(unsigned, b);
  }
  lo = (u32x4_t){o[0], o[1], o[2], o[3]};
  hi = (u32x4_t){o[4], o[5], o[6], o[7]};
}
__device__ __forceinline__ int w8_swz(int t) { return (t & 3) | (((t >> 3) & 1) << 2); }

// How dy gets to LDS.  DMA: its rows are 16-byte aligned (N % 8 == 0 and an aligned base).  ROWS: any other rows of 8 columns or
// more, through registers (8192 x 1280 x 1280: 48 us, 1284 columns: 56).  NARROW: fewer columns, value by value.
enum W8Rows { W8_DMA, W8_ROWS, W8_NARROW };
template <int BT_N, int BT_K, int WGN, int WGK, int FMT, W8Rows HOW>
__global__ __launch_bounds__(64 * WGN * WGK) void wgrad8_kernel(W8Args p) {
  constexpr bool DMA = HOW == W8_DMA;
  constexpr int NT = 64 * WGN * WGK, TN = BT_N / WGN / 16, TK = BT_K / WGK / 16;
  constexpr int ROWN = BT_N * 2, ROWK = BT_K * 2, STAGE = 64 * (ROWN + ROWK);
  constexpr int QI = 64 * BT_K / 16 / NT;                  // 16-byte pieces of x8 per thread and step
  constexpr int DI = 64 * ROWN / 16 / NT;                  // 16-byte pieces of dy per thread and step
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WGN, wk = wave / WGN, r16 = lane & 15, g = lane >> 4;

  int id = blockIdx.x;                                     // neighbouring tiles on one XCD (see gemm8.hip)
  {
    const int total = p.tiles_n * p.tiles_k, per = total / 8, rem = total % 8, x = id % 8, r = id / 8;
    id = x * per + min(x, rem) + r;
  }
  const int n0 = (id / p.tiles_k) * BT_N, k0 = (id % p.tiles_k) * BT_K;
  const int t_begin = blockIdx.y * p.steps * 64, t_end = min(p.T, t_begin + p.steps * 64);
  const int steps = (t_end - t_begin + 63) / 64;           // (the launcher leaves no split empty)

  // Pieces of 16 bytes: a thread's places in the tiles are the same every step, so are its offsets from the step's first
  // token.  Columns past N or the row's last block are taken from inside the row (they only reach results that are not
  // stored); tokens past the end are zeros in both operands.
  const char* dy0 = reinterpret_cast<const char*>(p.dy) + (size_t)t_begin * p.N * 2;
  const unsigned char* q0 = p.q + (size_t)t_begin * p.KB * B8_BLOCK;
  const unsigned char* s0 = p.qs + (size_t)t_begin * p.SP;
  // A thread's pieces lie DROWS and QROWS tokens apart, in the same columns.
  constexpr int DROWS = NT / (ROWN / 16), QROWS = NT / (BT_K / 16);
  static_assert(NT % (ROWN / 16) == 0 && NT % (BT_K / 16) == 0 && DROWS % 16 == 0, "a piece's place and permutation");
  const int d_t = tid / (ROWN / 16), d_c = tid % (ROWN / 16), q_t = tid / (BT_K / 16);
  const int d_col = n0 + (DMA ? ((d_c >> 1) ^ w8_swz(d_t)) * 2 + (d_c & 1) : d_c) * 8;       // (DMA: the column whose 16 bytes belong at this place)
  const unsigned d_step = (unsigned)DROWS * (unsigned)p.N * 2u;
  const unsigned off_d = (unsigned)d_t * (unsigned)p.N * 2u + (unsigned)(HOW == W8_NARROW ? 0 : min(d_col, p.N - 8)) * 2u;
  const int kc = min(k0 + tid % (BT_K / 16) * 16, p.KB * B8_BLOCK - 16);
  const unsigned q_step = (unsigned)QROWS * (unsigned)(p.KB * B8_BLOCK), s_step = (unsigned)QROWS * (unsigned)p.SP;
  const unsigned off_q = (unsigned)q_t * (unsigned)(p.KB * B8_BLOCK) + (unsigned)kc;
  const unsigned off_s = (unsigned)q_t * (unsigned)p.SP + (unsigned)(kc / B8_BLOCK & ~3);    // (the word with the scale; a byte load's
  const int shift_s = (kc / B8_BLOCK & 3) * 8;                                               //  extension the compiler would wait for at once)
  u32x4_t rd[DMA ? 1 : DI];
  u32x4_t rq[QI];
  unsigned rs[QI];
  auto request = [&](int s, int buf) {
    const int left = t_end - (t_begin + s * 64);           // tokens from the step's first one to the end
    const unsigned char* q = q0 + (size_t)s * 64 * p.KB * B8_BLOCK;
    const unsigned char* sc = s0 + (size_t)s * 64 * p.SP;
    const char* d = dy0 + (size_t)s * 64 * p.N * 2;
    unsigned od = off_d, oq = off_q, os = off_s;
    asm volatile("" : "+v"(od), "+v"(oq), "+v"(os));       // (or every piece's offset takes a register of its own)
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      const bool in = q_t + i * QROWS < left;
      rq[i] = *reinterpret_cast<const u32x4_t*>(q + (in ? oq + i * q_step : 0u));
      rs[i] = *reinterpret_cast<const unsigned*>(sc + (in ? os + i * s_step : 0u));
    }
    auto place = [&](int i) {
      return __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)(lds_voidw_t*)(smem + buf * STAGE + (i * NT + (tid & ~63)) * 16));
    };
    if constexpr (DMA) {
      if (left >= 64) {
#pragma unroll
        for (int i = 0; i < DI; ++i)
          asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(place(i)), "v"(od + i * d_step), "s"(d) : "memory", "m0");
      } else {
#pragma unroll
        for (int i = 0; i < DI; ++i) {
          const void* src = d_t + i * DROWS < left ? (const void*)(d + od + i * d_step) : (const void*)g_wgrad_zero;
          asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(place(i)), "v"(src) : "memory", "m0");
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < DI; ++i) {
        const char* at = d + (d_t + i * DROWS < left ? od + i * d_step : 0u);
        if constexpr (HOW == W8_ROWS) rd[i] = *reinterpret_cast<const b8_u32x4_a2*>(at);
        else rd[DMA ? 0 : i] = raw8_load(reinterpret_cast<const bf16_t*>(at), 0, p.N).a;     // (no column past N is looked at)
      }
    }
  };
  // what came through registers goes to LDS
  auto write = [&](int s, int buf) {
    const int left = t_end - (t_begin + s * 64);
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      const int piece = i * NT + tid, t = piece / (BT_K / 16), u = piece % (BT_K / 16);
      u32x4_t lo, hi;
      w8_to_bf16<FMT>(rq[i], b8_scale((int)(rs[i] >> shift_s) & 255), lo, hi);
      if (t >= left) { lo = (u32x4_t){0u, 0u, 0u, 0u}; hi = lo; }
      char* d = smem + buf * STAGE + 64 * ROWN + t * ROWK + ((u ^ w8_swz(t)) << 5);
      *reinterpret_cast<u32x4_t*>(d) = lo;
      *reinterpret_cast<u32x4_t*>(d + 16) = hi;
    }
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < DI; ++i) {
        const int piece = i * NT + tid, t = piece / (ROWN / 16), c = piece % (ROWN / 16);
        u32x4_t o = rd[DMA ? 0 : i];
        const int s = max(n0 + c * 8 - (p.N - 8), 0);      // a row's last, partial piece was read s columns early
        if (HOW == W8_ROWS && s > 0) {
          if (s & 4) o = (u32x4_t){o[2], o[3], 0u, 0u};
          if (s & 2) o = (u32x4_t){o[1], o[2], o[3], 0u};
          if (s & 1) o = (u32x4_t){o[0] >> 16 | o[1] << 16, o[1] >> 16 | o[2] << 16, o[2] >> 16 | o[3] << 16, o[3] >> 16};
        }
        if (t >= left) o = (u32x4_t){0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4_t*>(smem + buf * STAGE + t * ROWN + (((c >> 1) ^ w8_swz(t)) * 2 + (c & 1)) * 16) = o;
      }
    }
  };
  // 8 tokens (8 g .. of a 32-token half) of the 16 columns of unit u.  A lane's address: its token and place in the unit,
  // and the unit's place u ^ f, of which the low three bits are permuted and f (the same for t and t + 4) is the lane's own.
  const int f_t = w8_swz(g * 8 + (r16 >> 2));
  auto frag = [&](unsigned at, int row_bytes, int half, int u) {
    typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
    const char* a = smem + at + half * 32 * row_bytes + ((u ^ f_t) << 5);
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)a);
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(a + 4 * row_bytes));
    typedef __attribute__((ext_vector_type(8))) short s16x8_t;
    return __builtin_bit_cast(bf16x8_t, (s16x8_t){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  };
  const unsigned lane_n = (g * 8 + (r16 >> 2)) * ROWN + (r16 & 3) * 8, lane_k = 64 * ROWN + (g * 8 + (r16 >> 2)) * ROWK + (r16 & 3) * 8;

  f32x4_t acc[TK][TN], accb[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    accb[j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TK; ++i) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  const bool want_db = p.db && k0 == 0 && wk == 0;
  const __bf16 one = (__bf16)1.0f;
  const bf16x8_t ones = {one, one, one, one, one, one, one, one};

  // (two loops: a test of want_db inside would make the compiler move all sums around it)
  auto run = [&](auto with_db) {
    request(0, 0);
    write(0, 0);
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");        // step s has landed and is written, step s - 1 is read
      __builtin_amdgcn_s_barrier();
      const bool more = s + 1 < steps;
      if (more) request(s + 1, (s + 1) & 1);
      const unsigned an = lane_n + (s & 1) * STAGE, ak = lane_k + (s & 1) * STAGE;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        bf16x8_t fn[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) fn[j] = frag(an, ROWN, half, wn * TN + j);
        if constexpr (decltype(with_db)::value) {
#pragma unroll
          for (int j = 0; j < TN; ++j) accb[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, fn[j], accb[j], 0, 0, 0);
        }
        constexpr int AHEAD = 2;                 // k fragments are read this many tiles ahead of their use
        bf16x8_t fk[AHEAD + 1];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fk[i] = frag(ak, ROWK, half, wk * TK + i);
#pragma unroll
        for (int i = 0; i < TK; ++i) {
          if (i + AHEAD < TK) fk[(i + AHEAD) % (AHEAD + 1)] = frag(ak, ROWK, half, wk * TK + i + AHEAD);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fk[i % (AHEAD + 1)], fn[j], acc[i][j], 0, 0, 0);
        }
      }
      if (more) write(s + 1, (s + 1) & 1);
    }
  };
  if (want_db) run(std::true_type{}); else run(std::false_type{});
  float* dw = p.dw + (size_t)blockIdx.y * p.N * p.K;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + (wn * TN + j) * 16 + r16;
    if (n < p.N) {
#pragma unroll
      for (int i = 0; i < TK; ++i) {
        const int k = k0 + (wk * TK + i) * 16 + g * 4;
        float* o = dw + (size_t)n * p.K + k;
        if (k + 4 <= p.K) *reinterpret_cast<w8_f32x4_a4*>(o) = acc[i][j];
        else {
#pragma unroll
          for (int e = 0; e < 4; ++e) if (k + e < p.K) o[e] = acc[i][j][e];
        }
      }
      if (want_db && g == 0) p.db[(size_t)blockIdx.y * p.N + n] = accb[j][0];
    }
  }
}

// partial sums -> dw [nk], db [N], in the order of the splits; part: [splits][nk] and behind them [splits][N]
__global__ __launch_bounds__(256) void wgrad8_reduce(const float* __restrict__ part, float* __restrict__ dw, float* __restrict__ db,
                                                     size_t nk, int N, int splits, unsigned dw_blocks) {
  const bool is_b = blockIdx.x >= dw_blocks;
  const float* src = is_b ? part + splits * nk : part;
  float* out = is_b ? db : dw;
  const size_t total = is_b ? (size_t)N : nk;
  const size_t i = ((size_t)(blockIdx.x - (is_b ? dw_blocks : 0u)) * 256 + threadIdx.x) * 4;
  if (i >= total) return;
  if (i + 4 <= total) {
    f32x4_t s = *reinterpret_cast<const w8_f32x4_a4*>(src + i);
    int k = 1;
    for (; k + 4 <= splits; k += 4) {            // four requested at a time
      f32x4_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const w8_f32x4_a4*>(src + (size_t)(k + u) * total + i);
#pragma unroll
      for (int u = 0; u < 4; ++u) s += v[u];
    }
    for (; k < splits; ++k) s += *reinterpret_cast<const w8_f32x4_a4*>(src + (size_t)k * total + i);
    *reinterpret_cast<w8_f32x4_a4*>(out + i) = s;
  } else {
    for (size_t e = i; e < total; ++e) {
      float s = src[e];
      for (int k = 1; k < splits; ++k) s += src[(size_t)k * total + e];
      out[e] = s;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// host entry points
// ---------------------------------------------------------------------------------------------
constexpr int W8_MAX_WIDTH = 1 << 24;            // (offsets within 64 rows are held in 32 bits)
struct W8Plan { bool big; int tiles_n, tiles_k, splits, steps; };
// Tile size and number of splits by the least estimated time, in us, from what the kernels measured: a step of 64 tokens
// takes 1.67 with one 256 x 256 workgroup on a CU, 0.8 with one of 128 x 128 and 1.17 with two; a split result costs its
// partial sums' way through memory (both ways at 4 TB/s) and a launch.  16384 x 5120 x 640: 60 large tiles in 4 splits
// 140 us (3: 174, 6: 182; 200 small tiles in 4: 166); 65536 x 320 x 320: small in 48, 42 us (large in 64: 51);
// 1024 x 1280 x 1280: small, not split, 19.8 us (in 2: 22.1; large in 6: 29.1).
static W8Plan w8_plan(int T, int N, int K) {
  static const int tries[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64, 80, 96, 112, 128};
  const int kp = b8_kblocks(K) * B8_BLOCK, all = (T + 63) / 64;
  W8Plan best{};
  double best_us = 0;
  for (int big = 0; big < (N < 8 ? 1 : 2); ++big) {
    const int b = big ? 256 : 128, tn = (N + b - 1) / b, tk = (kp + b - 1) / b;
    const long long tiles = (long long)tn * tk;
    for (int want : tries) {
      if (want > 1 && (want > all || tiles * (want - 1) > 1024)) break;
      const int steps = (all + want - 1) / want, splits = (all + steps - 1) / steps;
      const long long per_cu = (tiles * splits + 255) / 256;
      const double step = big ? 1.67 * per_cu : per_cu == 1 ? 0.8 : 1.17 * ((per_cu + 1) / 2);
      const double us = 4 + steps * step + (splits > 1 ? 4 + 8e-6 / 4 * splits * N * K : 0);
      if (best.steps == 0 || us < best_us) {
        best_us = us;
        best = W8Plan{big != 0, tn, tk, splits, steps};
      }
    }
  }
  return best;
}

extern "C" size_t sdamd_linear8_weight_grad_ws_bytes(int T, int N, int K) {
  if (T <= 0 || N <= 0 || K <= 0 || N > W8_MAX_WIDTH || K > W8_MAX_WIDTH) return 0;
  const W8Plan w = w8_plan(T, N, K);
  return w.splits > 1 ? (size_t)w.splits * ((size_t)N * K + N) * sizeof(float) : 0;
}

template <int B, int WGN, int WGK, int FMT, W8Rows HOW>
static int w8_launch(const W8Args& p, int splits, hipStream_t st) {
  static std::atomic<unsigned long long> done{0};
  constexpr int lds = 2 * 64 * 2 * B * 2;
  auto k = wgrad8_kernel<B, B, WGN, WGK, FMT, HOW>;
  const hipError_t e = sd_lds_opt_in(done, (const void*)k, lds);
  if (e != hipSuccess) return sdamd_set_error(2, "linear8_weight_grad: %s", hipGetErrorString(e));
  k<<<dim3(p.tiles_n * p.tiles_k, splits), 64 * WGN * WGK, lds, st>>>(p);
  return 0;
}

extern "C" int sdamd_linear8_weight_grad(const void* dy, const void* x8, const unsigned char* x8_scale, float* dw, float* db, void* ws, size_t ws_bytes,
                                         int T, int N, int K, int fmt, void* stream) {
  SD_CHECK(fmt == SDAMD_E4M3 || fmt == SDAMD_E5M2, "linear8_weight_grad: unsupported dtype %d", fmt);
  SD_CHECK(T > 0 && N > 0 && K > 0 && N <= W8_MAX_WIDTH && K <= W8_MAX_WIDTH && T <= (1 << 30),
           "linear8_weight_grad: bad shape T=%d N=%d K=%d (N, K <= %d)", T, N, K, W8_MAX_WIDTH);
  SD_CHECK(((uintptr_t)x8 & 15) == 0 && ((uintptr_t)x8_scale & 3) == 0, "linear8_weight_grad: blocks have to be 16-byte aligned, their scales 4-byte aligned");
  const W8Plan w = w8_plan(T, N, K);
  SD_CHECK((long long)w.tiles_n * w.tiles_k < (1ll << 23), "linear8_weight_grad: too large, N=%d K=%d", N, K);
  const size_t need = sdamd_linear8_weight_grad_ws_bytes(T, N, K), nk = (size_t)N * K;
  SD_CHECK(need == 0 || (ws && ws_bytes >= need), "linear8_weight_grad: workspace of %zu bytes, %zu needed", ws_bytes, need);
  float* part = (float*)ws;
  W8Args p{(const bf16_t*)dy, (const unsigned char*)x8, x8_scale, need ? part : dw, db ? (need ? part + w.splits * nk : db) : nullptr,
           T, N, K, b8_kblocks(K), b8_scale_stride(K), w.tiles_n, w.tiles_k, w.steps};
  hipStream_t st = (hipStream_t)stream;
  const bool dma = N % 8 == 0 && ((uintptr_t)dy & 15) == 0;
  int rc;
#define W8_FMT(F)                                                                                          \
  rc = w.big ? (dma ? w8_launch<256, 4, 2, F, W8_DMA>(p, w.splits, st) : w8_launch<256, 4, 2, F, W8_ROWS>(p, w.splits, st))              \
     : dma   ? w8_launch<128, 2, 2, F, W8_DMA>(p, w.splits, st)                                                                          \
     : N < 8 ? w8_launch<128, 2, 2, F, W8_NARROW>(p, w.splits, st) : w8_launch<128, 2, 2, F, W8_ROWS>(p, w.splits, st)
  if (fmt == SDAMD_E4M3) W8_FMT(SDAMD_E4M3); else W8_FMT(SDAMD_E5M2);
#undef W8_FMT
  if (rc) return rc;
  SD_LAUNCH_CHECK("linear8_weight_grad");
  if (need) {
    const unsigned dw_blocks = (unsigned)((nk + 1023) / 1024), db_blocks = db ? (N + 1023) / 1024 : 0;
    wgrad8_reduce<<<dw_blocks + db_blocks, 256, 0, st>>>(part, dw, db, nk, N, w.splits, dw_blocks);
    SD_LAUNCH_CHECK("linear8_weight_grad");
  }
  return 0;
}
