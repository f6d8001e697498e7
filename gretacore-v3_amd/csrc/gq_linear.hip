// gq_linear.hip -- the product with bias, activation and residual in its epilogue over T16 weights,
// any number of rows (few rows here, tiles in gq_linear_rb.hip), and its backward pass.
#include <algorithm>
#include <type_traits>

#include "gq_internal.h"
#include "gq_linear.h"
#include "gq_rows_frag.h"

namespace {

// ---- forward: up to 16 rows, units of 128 k ------------------------------------------
// The weights' bytes bound these: a workgroup takes R row tiles, its KS waves share K unit by unit with PD units in
// flight each, and their sums are added through LDS.
// Outputs of R tiles and up to ROWS rows, several a thread: their biases and residuals (which may be y, and are read before any
// output is written) are loaded first of all, so that nothing waits for them at the end.
template <int KS, int R, int ROWS>
struct LinOut {
  static constexpr int EACH = (16 * R * ROWS + 64 * KS - 1) / (64 * KS);
  LinTail t[EACH];
  __device__ __forceinline__ void ahead(const LinEpi &e, int M, int N, int block) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int o = threadIdx.x + 64 * KS * i, m = o / (16 * R), n = 16 * R * block + o % (16 * R);
      t[i] = m < M && n < N ? lin_tail(e, m, n, N) : LinTail{0.f, 0.f};
    }
  }
  template <typename At>
  __device__ __forceinline__ void put(At at, const float *rs, const LinEpi &e, int M, int N, int block) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int o = threadIdx.x + 64 * KS * i, nl = o % (16 * R), m = o / (16 * R), n = 16 * R * block + nl;
      if (m >= M || n >= N) continue;
      float y = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) y += at(k, nl >> 4, nl & 15, m);
      lin_put(e, m, n, N, rs ? y * rs[m] : y, t[i]);
    }
  }
};

// Up to 4 rows of 16-bit x: codes and x as they are, scales in fp32 (gq_rows_frag.h), x through LDS
template <int FMT, int XT, int MR, int R, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_lin_few(const uint8_t *__restrict__ w, size_t sc_off, const void *__restrict__ x, const float *__restrict__ rs, LinEpi e,
          int M, int N, int K, int C, int units) {
  constexpr int NG = kFewGroups<FMT>;
  __shared__ float red[KS][R][MR][64];
  extern __shared__ __attribute__((aligned(16))) uint8_t xs_s[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, ntiles = (int)gq_tiles(N);
  FTile<FMT> tl[R];
#pragma unroll
  for (int t = 0; t < R; ++t) {
    const int tile = (int)blockIdx.x * R + t;
    tl[t] = ftile<FMT>(w, sc_off, (size_t)(tile < ntiles ? tile : ntiles - 1), C);  // (clamped: not stored)
  }
  const int np = 128 * units, stride = (int)few_lds_stride(np);
  const bool mine = few_mine<FMT>(lane) && (lane & 3) < M;
  const uint32_t x0 = mine ? (uint32_t)((lane & 3) * stride + 32 * g) : (uint32_t)(M * stride), xd = mine ? 256u : 0u;
  constexpr int G = kGroup<FMT>;
  FUnit<FMT> us[PD][R][G];
  auto request = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < R; ++t) load_group<FMT>(tl[t], group, lane, us[st][t]);
  };
  float acc[R][MR] = {};
  uint32_t mg;  // (kept in a register)
  if constexpr (XT == GQ_DT_F16) asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(mg));
  else asm volatile("v_mov_b32 %0, 0x43004300" : "=v"(mg));
  auto compute = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < G; ++p)
      few_add<FMT, XT>(us[st], p, G * group + p, g, xs_s, x0 + xd * (uint32_t)(G * group + p), mg, acc);
  };
  LinOut<KS, R, MR> out;
  out.ahead(e, M, N, (int)blockIdx.x);
  // (x's loads go out before the weights': behind them they would wait for theirs)
  few_stage<64 * KS>(x, M, K, np, stride, kNibOrder<FMT>, xs_s, tid,
                     [&]() __attribute__((always_inline)) { walk_requests<PD, KS>(units / G, wave, request); });
  step_barrier<63>();  // (of LDS alone)
  walk_computes<PD, KS>(units / G, wave, request, compute);
#pragma unroll
  for (int t = 0; t < R; ++t)
#pragma unroll
    for (int v = 0; v < MR; ++v) red[wave][t][v][lane] = acc[t][v];
  __syncthreads();
  out.put(
      [&](int k, int t, int n, int m) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) y += red[k][t][MR == 1 ? 0 : m][16 * i + n];
        return y;
      },
      rs, e, M, N, (int)blockIdx.x);
}

// More rows: fp16 rows of x with a power-of-two scale each, the scale groups folded into the weights (gq_rows_frag.h)
template <int FMT, int MT, int R, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_lin_rows(const uint8_t *__restrict__ w, size_t sc_off, const _Float16 *__restrict__ a16, int lda,
           const float *__restrict__ rs, LinEpi e, int M, int N, int C, int units) {
  __shared__ gq_f4 red[KS][R][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15, ntiles = (int)gq_tiles(N);
  FTile<FMT> tl[R];
#pragma unroll
  for (int t = 0; t < R; ++t) {
    const int tile = (int)blockIdx.x * R + t;
    tl[t] = ftile<FMT>(w, sc_off, (size_t)(tile < ntiles ? tile : ntiles - 1), C);  // (clamped: not stored)
  }
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<_Float16 *>(a16), (short)0, (int)(2u * (uint32_t)M * (uint32_t)lda), 0x00020000);
  uint32_t xo[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int row = 16 * t + r;
    xo[t] = 2u * ((uint32_t)(row < M ? row : M - 1) * (uint32_t)lda + 16u * (uint32_t)g);  // (rows past M: not stored)
  }
  constexpr int G = kGroup<FMT>;
  FUnit<FMT> us[PD][R][G];
  gq_half8 xs[PD][G][MT][4];
  auto request = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < R; ++t) load_group<FMT>(tl[t], group, lane, us[st][t]);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint32_t o = G * group < units ? xo[t] + 256u * G * (uint32_t)group : 0xFFFFFC00u;
#pragma unroll
      for (int i = 0; i < 4 * G; ++i) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(xr, o + 128u * (i >> 1) + 16u * (i & 1), 0, 0);
        xs[st][i >> 2][t][i & 3] = __builtin_bit_cast(gq_half8, gq_u4{v[0], v[1], v[2], v[3]});
      }
    }
  };
  gq_f4 acc[R][MT];
#pragma unroll
  for (int t = 0; t < R; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[t][i] = gq_f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t mg = gq_nib_magic();
  auto compute = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < G; ++p)
#pragma unroll
      for (int t = 0; t < R; ++t) rows_add<FMT, MT>(us[st][t][p], G * group + p, g, mg, xs[st][p], acc[t]);
  };
  LinOut<KS, R, 16 * MT> out;
  out.ahead(e, M, N, (int)blockIdx.x);
  walk_units<PD, KS>(units / G, wave, request, compute);
#pragma unroll
  for (int t = 0; t < R; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wave][t][i][lane] = acc[t][i];
  __syncthreads();
  auto at = [&](int k, int t, int n, int m) {
    return reinterpret_cast<const float *>(&red[k][t][m >> 4][16 * ((m >> 2) & 3) + n])[m & 3];
  };
  out.put(at, rs, e, M, N, (int)blockIdx.x);
}

// the parts' sums, in their order, and the epilogue; a thread takes outputs of one row
__global__ void __launch_bounds__(256) k_lin_sum(const float *__restrict__ part, LinEpi e, int M, int N, int parts) {
  const int n = (int)blockIdx.x * 256 + (int)threadIdx.x, m = (int)blockIdx.y;
  if (n >= N) return;
  const LinTail t = lin_tail(e, m, n, N);
  float v = 0.f;
  for (int p = 0; p < parts; ++p) v += part[((size_t)p * M + m) * (size_t)N + n];
  lin_put(e, m, n, N, v, t);
}
template <int FMT, int XT>
int launch_few_t(const void *w, const void *x, const float *rs, const LinEpi &e, int M, int N, int K, hipStream_t s) {
  const int units = (int)(gq_kpad(FMT, K) / 128);
  const size_t tiles = gq_tiles(N), lds = few_lds_bytes(M, 128 * (size_t)units);
#define GQ_FEW(MR, R, KS, PD)                                                                                               \
  hipLaunchKernelGGL((k_lin_few<FMT, XT, MR, R, KS, group_stages<FMT>(PD)>), dim3((unsigned)((tiles + (R)-1) / (R))), dim3(64 * (KS)), lds, s,   \
                     (const uint8_t *)w, gq_sc_plane_offset(FMT, N, K), x, rs, e, M, N, K, (int)gq_chunks(FMT, K), units)
#define GQ_FEW_M(R, KS, PD)           \
  do {                                \
    if (M == 1) GQ_FEW(1, R, KS, PD); \
    else GQ_FEW(4, R, KS, PD);        \
  } while (0)
  // One tile and 16 waves up to a workgroup a CU, 8 waves up to two, then two tiles, which share what is done for x (one row, us by one tile and 16
  // waves / one and 8 / two and 8: 4096 x 14336 Q4_K 9.3 / 11.7 / 13.7; 5120 x 5120 Q6_K 10.2 / 8.0 / 8.7; 8192 x 8192 Q4_0 11.9 / 9.6 / 10.3;
  // 14336 x 4096 Q4_K 11.7 / 9.9 / 9.4, Q8_0 13.3 / 12.7 / 13.2)
  if (tiles <= 256) GQ_FEW_M(1, 16, 2);
  else if (tiles <= 512) GQ_FEW_M(1, 8, 2);
  else GQ_FEW_M(2, 8, 2);
#undef GQ_FEW_M
#undef GQ_FEW
  return gq_last_launch();
}
template <int FMT>
int launch_rows_t(const void *w, const _Float16 *a16, int lda, const float *rs, const LinEpi &e, int M, int N, int K, hipStream_t s) {
  const int units = (int)(gq_kpad(FMT, K) / 128);
  const size_t tiles = gq_tiles(N);
#define GQ_ROWS(R, KS, PD)                                                                                               \
  hipLaunchKernelGGL((k_lin_rows<FMT, 1, R, KS, group_stages<FMT>(PD)>), dim3((unsigned)((tiles + (R)-1) / (R))), dim3(64 * (KS)), 0, s,      \
                     (const uint8_t *)w, gq_sc_plane_offset(FMT, N, K), a16, lda, rs, e, M, N, (int)gq_chunks(FMT, K), units)
  // Two tiles share the rows of x (which every workgroup reads whole) where that leaves a workgroup for every other CU; long rows of one tile by few
  // waves.  16 rows, us by two tiles and 4 waves / two and 8 / one and 8 / one and 4, deeper:
  //   14336 x 4096 Q4_K 15.2 / 14.5 / 18.6 / 18.8, Q4_0 14.6 / 15.4 / 20.6 / 19.7    6144 x 14336 Q4_K 25.7 / 23.1 / - / 30.6, Q8_0 24.9 / 24.6 / - / 34.3
  //   4096 x 14336 Q4_K 24.9 / 22.4 / 19.4 / 19.5, Q8_0 23.7 / 23.4 / 20.3 / 19.5    8 rows, 4096 x 4096 Q8_0 8.5 / 8.3 / 6.5 / 6.9
  if (tiles > 512) GQ_ROWS(2, 4, 2);
  else if (tiles > 256) GQ_ROWS(2, 8, 2);
  else if (units > 64) GQ_ROWS(1, 4, 4);
  else GQ_ROWS(1, 8, 2);
#undef GQ_ROWS
  return gq_last_launch();
}

// ---- backward ----------------------------------------------------------------------
// dz = dy act'(z): one pass over dy and z, a workgroup a row at a time (row blockIdx.x, + gridDim.x, ...).  dz goes out in its own
// type where it is wanted, and, as it is before that rounding, to fp16 with one power-of-two scale per row (the row's
// largest to [2^14, 2^15); 2^-114 to 2^126), padded with zeros to np columns: the A operand of dx, of the matrix cores' types the one
// with the most bits (2.1e-4 of a row; products of fp32 would leave them).  The workgroup's rows are summed
// by column into its row of `part` (dbias), which a last kernel adds over the workgroups in their order.  The first RUNS * 4096
// columns of a row and their sums stay in registers, the rest (RUNS = 4 alone) is computed twice and summed in `part`.  The row's last,
// ragged run is one thread's, on a path of its own: a launch starts with its code to be fetched, and every unrolled run's
// copy of it counts (203 x 5003 fp16, tanh-GELU: 13.3 us with all activations and runs in one kernel, 8.0 so;
// 2048 x 14336 bf16, ReLU, 44 us, 250 MB).
constexpr int kDzThreads = 512;
template <int DT, int ACT, int RUNS>
__global__ void __launch_bounds__(kDzThreads) k_lin_dz(const void *dy, const void *z, void *dzo, _Float16 *a16, float *rs,
                                                       float *part, int add, int M, int N, int np) {
  __shared__ float top_s[2][kDzThreads / 64];
  constexpr int SPAN = 8 * kDzThreads * RUNS;
  constexpr bool GATED = ACT != GQ_ACT_NONE, LONG = RUNS == 4;
  const int tid = threadIdx.x;
  auto run = [&](int i) { return 8 * (tid + kDzThreads * i); };
  const int kt = N & ~7, it = kt / (8 * kDzThreads);  // the ragged run, and which of its thread's it is
  const bool last = kt < N && kt < SPAN && kt / 8 % kDzThreads == tid;
  float sum[RUNS][8];
  float *pr = part ? part + (size_t)blockIdx.x * (size_t)N : nullptr;
#pragma unroll
  for (int i = 0; i < RUNS; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[i][e] = pr && add && run(i) + e < N ? pr[run(i) + e] : 0.f;
  // whole runs of the next row are requested before a row's are used
  FRaw<DT> ra[RUNS], rb[RUNS];
  auto request = [&](int m) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      if (m >= M || run(i) + 8 > N) continue;
      px_load<DT>(dy, (size_t)m * (size_t)N + run(i), ra[i]);
      if (GATED) px_load<DT>(z, (size_t)m * (size_t)N + run(i), rb[i]);
    }
  };
  request((int)blockIdx.x);
  int buf = 0;
  for (int m = (int)blockIdx.x; m < M; m += (int)gridDim.x, buf ^= 1) {
    const size_t row = (size_t)m * (size_t)N;
    auto grads = [&](int k, float (&o)[8]) __attribute__((always_inline)) {
      float b[8];
      dgu_load<DT>(dy, row, k, N, o);
      if (!GATED) return;
      dgu_load<DT>(z, row, k, N, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = k + e < N ? o[e] * lin_act_d<ACT>(b[e]) : 0.f;
    };
    float d[RUNS][8], tail[8] = {}, top = 0.f;
    if (last) grads(kt, tail);
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      if (run(i) + 8 <= N) {
        float b[8];
        px_floats<DT>(ra[i], true, d[i]);
        if (GATED) {
          px_floats<DT>(rb[i], true, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) d[i][e] *= lin_act_d<ACT>(b[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[i][e] = last && i == it ? tail[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = fmaxf(top, fabsf(d[i][e]));
        sum[i][e] += d[i][e];
      }
    }
    request(m + (int)gridDim.x);
    if (LONG && a16)
      for (int k = SPAN + 8 * tid; k < N; k += 8 * kDzThreads) {
        float a[8];
        grads(k, a);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(a[e]));
      }
    float f2 = 0.f;
    if (a16) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
      if ((tid & 63) == 0) top_s[buf][tid >> 6] = top;
      __syncthreads();  // (two buffers: a row's maxima are read before the next row's barrier, the one after writes them)
#pragma unroll
      for (int w = 0; w < kDzThreads / 64; ++w) top = fmaxf(top, top_s[buf][w]);
      const int sh = gq_fp16_shift(top);
      f2 = gq_pow2(sh);
      if (tid == 0) rs[m] = gq_pow2(-sh);
    }
    auto put16 = [&](int k, const float (&a)[8]) __attribute__((always_inline)) {
      if (!a16 || k >= np) return;
      gq_half8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (_Float16)(a[e] * f2);
      *reinterpret_cast<gq_half8 *>(a16 + (size_t)m * (size_t)np + k) = x;
    };
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      if (dzo && run(i) + 8 <= N) dgu_store<DT>(dzo, row, run(i), run(i) + 8, d[i]);
      put16(run(i), d[i]);
    }
    if (dzo && last) dgu_store<DT>(dzo, row, kt, N, tail);
    if (LONG)
      for (int k = SPAN + 8 * tid; k < (a16 ? np : N); k += 8 * kDzThreads) {
        float a[8] = {};
        if (k < N) grads(k, a);
        if (dzo && k < N) dgu_store<DT>(dzo, row, k, N, a);
        put16(k, a);
        if (pr)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k + e < N) pr[k + e] = (add || m != (int)blockIdx.x ? pr[k + e] : 0.f) + a[e];
      }
  }
  if (!pr) return;
#pragma unroll
  for (int i = 0; i < RUNS; ++i) {
    if (run(i) + 8 <= N) {
      FRun32 r;
      r.v[0] = gq_f4{sum[i][0], sum[i][1], sum[i][2], sum[i][3]};
      r.v[1] = gq_f4{sum[i][4], sum[i][5], sum[i][6], sum[i][7]};
      *reinterpret_cast<FRun32 *>(pr + run(i)) = r;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (run(i) + e < N) pr[run(i) + e] = sum[i][e];
    }
  }
}
// dbias = the workgroups' sums, in an order of their own (none: zeros): 64 columns a workgroup, wave w adds parts w, w + 16, ...
constexpr int kDbWaves = 16;
__global__ void __launch_bounds__(64 * kDbWaves) k_lin_dbias(GqColSums s) {
  __shared__ double red[kDbWaves][64];
  gq_col_sums<64, kDbWaves>(s, 64 * (int)blockIdx.x, threadIdx.x & 63, threadIdx.x >> 6, red);
}
int launch_dbias(const GqColSums &c, hipStream_t s) {
  hipLaunchKernelGGL(k_lin_dbias, dim3((unsigned)((c.n + 63) / 64)), dim3(64 * kDbWaves), 0, s, c);
  return gq_last_launch();
}
template <int DT>
int launch_dz(const void *dy, const void *z, void *dz, _Float16 *a16, float *rs, float *part, int add, int wgs, int M, int N,
              int np, int act, hipStream_t s) {
#define GQ_DZ_RUNS(ACT, RUNS) \
  hipLaunchKernelGGL((k_lin_dz<DT, ACT, RUNS>), dim3((unsigned)wgs), dim3(kDzThreads), 0, s, dy, z, dz, a16, rs, part, add, M, N, np)
  // (np: whole runs of the fp16 row)
#define GQ_DZ_ACT(ACT)                                 \
  do {                                                 \
    if (np <= 8 * kDzThreads) GQ_DZ_RUNS(ACT, 1);      \
    else if (np <= 16 * kDzThreads) GQ_DZ_RUNS(ACT, 2); \
    else GQ_DZ_RUNS(ACT, 4);                           \
  } while (0)
  if (act == GQ_ACT_NONE) GQ_DZ_ACT(GQ_ACT_NONE);
  else if (act == GQ_ACT_RELU) GQ_DZ_ACT(GQ_ACT_RELU);
  else if (act == GQ_ACT_SILU) GQ_DZ_ACT(GQ_ACT_SILU);
  else GQ_DZ_ACT(GQ_ACT_GELU_TANH);
#undef GQ_DZ_ACT
#undef GQ_DZ_RUNS
  return gq_last_launch();
}

bool lin_act_valid(int act) { return act >= GQ_ACT_SILU && act <= GQ_ACT_RELU; }

int check_linear(int fmt, const void *w, size_t M, size_t N, size_t K, int act) {
  GQ_TRY(gq_check_shape(fmt, N, K));
  GQ_CHECK(M <= GQ_MAX_DIM, GQ_ERR_INVALID_ARGS);
  GQ_CHECK(lin_act_valid(act), GQ_ERR_UNSUPPORTED);
  GQ_CHECK(w || M == 0 || N == 0, GQ_ERR_INVALID_ARGS);
  GQ_CHECK(((uintptr_t)w & 15) == 0, GQ_ERR_INVALID_ARGS);  // (16-byte loads)
  // the kernels address a packed tensor with 32-bit offsets (the last 4 KiB: those that lie outside)
  GQ_CHECK(N == 0 || K == 0 || gq_packed_bytes(fmt, N, K) <= 0xFFFFF000u, GQ_ERR_INVALID_ARGS);
  return GQ_OK;
}

constexpr size_t kFew = 4, kRows = 16;
constexpr size_t kFewLds = 65536;  // values of x that LDS takes beside the waves' sums
// Rows a call takes at a time: their fp16 copies stay below 64 MiB, but for the rows that the kernels of few rows take at
// once (16 of at most 2^24 columns: 512 MiB)
size_t linear_rows(int fmt, size_t M, size_t K) {
  const size_t fit = ((size_t)64 << 20) / (2 * gq_kpad(fmt, K));
  const size_t mb = fit >= 256 ? fit & ~(size_t)255 : fit > kRows ? fit : kRows;
  return M < mb ? M : mb;
}

}  // namespace

int gq_launch_linear_sum(const float *part, const void *epi, int M, int N, int parts, hipStream_t s) {
  hipLaunchKernelGGL(k_lin_sum, dim3((unsigned)((N + 255) / 256), (unsigned)M), dim3(256), 0, s, part,
                     *reinterpret_cast<const LinEpi *>(epi), M, N, parts);
  return gq_last_launch();
}

extern "C" size_t gq_linear_workspace_bytes(int fmt, size_t M, size_t N, size_t K) {
  if (!gq_fmt_valid(fmt) || M > GQ_MAX_DIM || N > GQ_MAX_DIM || K > GQ_MAX_DIM || K == 0) return 0;
  const size_t mb = linear_rows(fmt, M, K);
  return gq_align256(mb * (gq_kpad(fmt, K) + 8) * 2) + gq_align256((mb + 256) * 4) + std::min(kLinParts * mb * N * 4, kLinPartBytes);
}

extern "C" int gq_linear(int fmt, const void *w, const void *x, int x_dtype, const void *bias, int bias_dtype, int act,
                         const void *resid, void *y, int y_dtype, void *z, size_t M, size_t N, size_t K, void *ws,
                         size_t ws_bytes, void *stream) {
  GQ_TRY(check_linear(fmt, w, M, N, K, act));
  GQ_CHECK(gq_dtype_valid(x_dtype) && gq_dtype_valid(y_dtype) && (!bias || gq_dtype_valid(bias_dtype)), GQ_ERR_UNSUPPORTED);
  if (M == 0 || N == 0) return GQ_OK;
  GQ_CHECK(x && y && K > 0, GQ_ERR_INVALID_ARGS);
  GQ_CHECK(N * 256 * gq_dtype_size(y_dtype) < ((size_t)1 << 31), GQ_ERR_INVALID_ARGS);  // (a tile's rows of outputs)
  hipStream_t s = (hipStream_t)stream;
  LinEpi e = {bias, resid, y, z, bias_dtype, y_dtype, act};
  auto few = [&](const void *xp, int xt, const float *rs) -> int {
#define GQ_FMT_X(F)                                                                             \
  (xt == GQ_DT_F16 ? launch_few_t<F, GQ_DT_F16>(w, xp, rs, e, (int)M, (int)N, (int)K, s)         \
                   : launch_few_t<F, GQ_DT_BF16>(w, xp, rs, e, (int)M, (int)N, (int)K, s))
    if (fmt == GQ_FMT_Q4_0) return GQ_FMT_X(GQ_FMT_Q4_0);
    if (fmt == GQ_FMT_Q8_0) return GQ_FMT_X(GQ_FMT_Q8_0);
    if (gq_fmt_is_q6k(fmt)) return GQ_FMT_X(GQ_FMT_Q6_K);
    return GQ_FMT_X(GQ_FMT_Q4_K);
#undef GQ_FMT_X
  };
  const bool is_few = M <= kFew && M * gq_kpad(fmt, K) <= kFewLds;
  if (is_few && x_dtype != GQ_DT_F32) return few(x, x_dtype, nullptr);
  const size_t need = gq_linear_workspace_bytes(fmt, M, N, K), mb = linear_rows(fmt, M, K), Kp = gq_kpad(fmt, K);
  GqScratch sc(ws ? 0 : need, s);
  if (ws) GQ_CHECK(ws_bytes >= need, GQ_ERR_WORKSPACE);
  else ws = sc.ptr;
  GQ_CHECK(ws, GQ_ERR_WORKSPACE);
  GQ_CHECK(((uintptr_t)ws & 15) == 0, GQ_ERR_INVALID_ARGS);
  _Float16 *a16 = (_Float16 *)ws;
  float *rs = (float *)((uint8_t *)ws + gq_align256(mb * (Kp + 8) * 2));
  const int q4 = fmt == GQ_FMT_Q4_0 || gq_fmt_is_q4k(fmt);
  // fp16 rows of whole chunks are what the matrix cores take already, but for the 4-bit formats' order
  const bool plain = x_dtype == GQ_DT_F16 && !q4 && K == Kp && ((uintptr_t)x & 15) == 0;
  if (is_few) {
    GQ_TRY(gq_launch_a_to_f16(x, x_dtype, a16, rs, (int)M, (int)K, (int)K, 0, s));
    return few(a16, GQ_DT_F16, rs);
  }
  float *part = (float *)((uint8_t *)rs + gq_align256((mb + 256) * 4));
  if (M <= kRows) {  // rows 16 bytes longer than a multiple of 4 KiB, where 16 of them would collide
    const int ld = (int)(plain ? K : Kp + 8);
    if (!plain) GQ_TRY(gq_launch_a_to_f16(x, x_dtype, a16, rs, (int)M, (int)K, ld, q4, s));
    const _Float16 *a = plain ? (const _Float16 *)x : a16;
    const float *f = plain ? nullptr : rs;
#define GQ_ROWS_F(F) launch_rows_t<F>(w, a, ld, f, e, (int)M, (int)N, (int)K, s)
    if (fmt == GQ_FMT_Q4_0) return GQ_ROWS_F(GQ_FMT_Q4_0);
    if (fmt == GQ_FMT_Q8_0) return GQ_ROWS_F(GQ_FMT_Q8_0);
    if (gq_fmt_is_q6k(fmt)) return GQ_ROWS_F(GQ_FMT_Q6_K);
    return GQ_ROWS_F(GQ_FMT_Q4_K);
#undef GQ_ROWS_F
  }
  const size_t xs = gq_dtype_size(x_dtype) * K, ys = gq_dtype_size(y_dtype) * N;
  for (size_t m0 = 0; m0 < M; m0 += mb) {
    const int m = (int)(M - m0 < mb ? M - m0 : mb);
    const _Float16 *a = plain ? (const _Float16 *)x + m0 * K : a16;
    if (!plain) GQ_TRY(gq_launch_a_to_f16((const uint8_t *)x + m0 * xs, x_dtype, a16, rs, m, (int)K, (int)Kp, q4, s));
    LinEpi b = e;
    b.resid = resid ? (const uint8_t *)resid + m0 * ys : nullptr;
    b.y = (uint8_t *)y + m0 * ys;
    b.z = z ? (uint8_t *)z + m0 * ys : nullptr;
    GQ_TRY(gq_launch_linear_rb(fmt, w, a, plain ? nullptr : rs, &b, part, m, (int)N, (int)K, s));
  }
  return GQ_OK;
}

// Workgroups that share the rows of dz (and so the sums in `part`): one a CU, of 64 MiB of sums together at most (N <= 2^24)
static size_t dz_groups(size_t M, size_t N) { return std::min({M, (size_t)256, ((size_t)1 << 24) / N}); }
static size_t dbias_bytes(size_t M, size_t N) { return gq_align256(dz_groups(M, N) * N * 4); }

extern "C" size_t gq_linear_bwd_workspace_bytes(int fmt, size_t M, size_t N, size_t K) {
  if (!gq_fmt_valid(fmt) || M > GQ_MAX_DIM || N > GQ_MAX_DIM || K > GQ_MAX_DIM || M == 0 || N == 0 || K == 0) return 0;
  return dbias_bytes(M, N) + gq_dx_most_bytes(M, N, K, 1);
}

extern "C" int gq_linear_bwd(int fmt, const void *w, const void *dy, const void *z, int dtype, int act, void *dz, void *dx,
                             int dx_dtype, float *dbias, size_t M, size_t N, size_t K, void *ws, size_t ws_bytes,
                             void *stream) {
  GQ_TRY(check_linear(fmt, w, M, N, K, act));
  GQ_CHECK(gq_dtype_valid(dtype) && gq_dtype_valid(dx_dtype), GQ_ERR_UNSUPPORTED);
  hipStream_t s = (hipStream_t)stream;
  if (M == 0) return dbias && N ? launch_dbias(GqColSums{nullptr, dbias, (int)N, 0}, s) : GQ_OK;  // (sums of nothing)
  if (!dz && !dx && !dbias) return GQ_OK;
  GQ_CHECK(K > 0, GQ_ERR_INVALID_ARGS);
  if (N == 0) return dx ? gq_launch_zeros(dx, dx_dtype, M, K, s) : GQ_OK;
  GQ_CHECK(dy && (z || act == GQ_ACT_NONE), GQ_ERR_INVALID_ARGS);
  const GqDxPlan plan = gq_dx_plan(M, N, K, 1);
  const size_t db = dbias ? dbias_bytes(M, N) : 0;
  GqScratch sc0(ws ? 0 : db, s), sc1(ws || !dx ? 0 : gq_dx_bytes(plan, K), s);  // (two blocks: each fits one)
  if (ws) GQ_CHECK(ws_bytes >= gq_linear_bwd_workspace_bytes(fmt, M, N, K), GQ_ERR_WORKSPACE);
  GQ_CHECK(((uintptr_t)ws & 15) == 0, GQ_ERR_INVALID_ARGS);
  float *sums = dbias ? (float *)(ws ? ws : sc0.ptr) : nullptr;
  uint8_t *at16 = dx ? (ws ? (uint8_t *)ws + db : (uint8_t *)sc1.ptr) : nullptr;
  GQ_CHECK((sums || !dbias) && (at16 || !dx), GQ_ERR_WORKSPACE);
  _Float16 *a16 = dx ? (_Float16 *)at16 : nullptr;
  float *rs = dx ? (float *)(at16 + gq_dx_a_bytes(plan)) : nullptr;
  float *part = dx ? (float *)((uint8_t *)rs + gq_dx_rs_bytes(plan)) : nullptr;
  const size_t es = gq_dtype_size(dtype) * N, xs = gq_dtype_size(dx_dtype) * K;
  const size_t step = dx ? plan.mb : (size_t)1 << 20, wgs = dz_groups(M < step ? M : step, N);
  const GqColSums cols = {sums, dbias, (int)N, (int)wgs};
  const bool with = dbias && dx && plan.parts > 1;
  for (size_t m0 = 0; m0 < M; m0 += step) {
    const int m = (int)(M - m0 < step ? M - m0 : step);
    auto at = [&](const void *p) { return p ? (void *)((uint8_t *)p + m0 * es) : nullptr; };
#define GQ_DZ(DT) launch_dz<DT>(at(dy), at(z), at(dz), a16, rs, sums, m0 > 0, (int)wgs, m, (int)N, (int)plan.np, act, s)
    if (dtype == GQ_DT_F32) GQ_TRY(GQ_DZ(GQ_DT_F32));
    else if (dtype == GQ_DT_F16) GQ_TRY(GQ_DZ(GQ_DT_F16));
    else GQ_TRY(GQ_DZ(GQ_DT_BF16));
#undef GQ_DZ
    // (the last block's sum of parts does dbias too: 203 x 5003 x 4096 Q6_K 39.0 us, 41.0 with a launch of its own)
    if (dx) GQ_TRY(gq_launch_dx(fmt, plan, w, w, a16, rs, part, (uint8_t *)dx + m0 * xs, dx_dtype, m, N, K, with && m0 + step >= M ? cols : GqColSums{}, s));
  }
  return dbias && !with ? launch_dbias(cols, s) : GQ_OK;
}
