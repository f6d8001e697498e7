// gq_ffn.hip -- the gated feed-forward front h = act(x W_gate^T) * (x W_up^T) over T16
// weights for any number of rows, and its backward pass.
#include <algorithm>
#include <type_traits>

#include "gq_act.h"
#include "gq_gemm_frag.h"
#include "gq_gemv_frag.h"
#include "gq_internal.h"
#include "gq_rows_frag.h"

namespace {

// ---- forward: up to 32 rows, units of 128 k ------------------------------------------
// The weights' bytes bound these.  A workgroup takes R row tiles of both matrices, its KS waves
// share K unit by unit (wave, wave + KS, ...) with PD units in flight each, and their sums are
// added through LDS.
// Sums of the waves, h and where they are kept g and u, of the R tiles `block`.  at(k, w, t, n, m): wave k's part of output
// (m, 16 t + n) of matrix w; rs: row scales of x
template <int KS, int R, typename At>
GQ_DEV void front_out(At at, const float *rs, void *h, void *go, void *uo, int dt, int M, int N, int act, int block) {
  for (int o = threadIdx.x; o < 16 * R * M; o += 64 * KS) {
    const int nl = o % (16 * R), m = o / (16 * R), n = 16 * R * block + nl;
    float y[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int k = 0; k < KS; ++k) y[w] += at(k, w, nl >> 4, nl & 15, m);
    if (n < N) {
      const float f = rs ? rs[m] : 1.f, g = y[0] * f, u = y[1] * f;
      const size_t i = (size_t)m * N + n;
      gq_st_dt(h, dt, i, gq_act_f(act, g) * u);
      if (go) gq_st_dt(go, dt, i, g);
      if (uo) gq_st_dt(uo, dt, i, u);
    }
  }
}
template <int FMT, int XT, int MR, int R, int KS>
__global__ void __launch_bounds__(64 * KS)
k_front_few(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off, const void *__restrict__ x,
            const float *__restrict__ rs, void *__restrict__ h, void *__restrict__ go, void *__restrict__ uo, int dt, int M,
            int N, int K, int C, int units, int act) {
  constexpr int NG = kFewGroups<FMT>, T = 2 * R, PD = R == 1 ? 3 : 2;
  constexpr float OFF = kFewOff<FMT, XT>;
  __shared__ float red[KS][T][MR][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, ntiles = (int)gq_tiles(N);
  FTile<FMT> tl[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int tile = (int)blockIdx.x * R + t % R;
    tl[t] = ftile<FMT>(t < R ? wg : wu, sc_off, (size_t)(tile < ntiles ? tile : ntiles - 1), C);  // (clamped: not stored)
  }
  const __amdgpu_buffer_rsrc_t xr =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(x), (short)0, (int)(2u * (uint32_t)M * (uint32_t)K), 0x00020000);
  const int xrow = lane & 3, xk = 64 * ((lane >> 3) & 1) + 16 * g + 8 * ((lane >> 2) & 1);
  FUnit<FMT> us[PD][T];
  gq_u4 xs[PD];
  auto request = [&](int unit, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < T; ++t) load_unit<FMT>(tl[t], unit, lane, us[st][t]);
    const uint32_t k = 128u * (uint32_t)unit + (uint32_t)xk;  // (K is whole 32-blocks: a run is wholly in or out)
    const bool in = xrow < M && k < (uint32_t)K;
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(xr, in ? 2u * ((uint32_t)xrow * (uint32_t)K + k) : 0xFFFFFFF0u, 0, 0);
    xs[st] = gq_u4{v[0], v[1], v[2], v[3]};
  };
  float acc[T][MR] = {};
  uint32_t mg;  // (kept in a register)
  if constexpr (XT == GQ_DT_F16) asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(mg));
  else asm volatile("v_mov_b32 %0, 0x43004300" : "=v"(mg));
  constexpr uint32_t one = XT == GQ_DT_F16 ? 0x3C003C00u : 0x3F803F80u;
  const gq_u4 ones = {one, one, one, one};
  const gq_f4 zero = {0.f, 0.f, 0.f, 0.f};
  auto compute = [&](int unit, int st) __attribute__((always_inline)) {
    const gq_u4 xv = kNibOrder<FMT> ? nib_order(xs[st]) : xs[st];
    float s[T][2], mn[T][2];
#pragma unroll
    for (int t = 0; t < T; ++t) few_scales<FMT>(us[st][t], unit, g & (NG - 1), s[t], mn[t]);
    auto step = [&](auto mc) __attribute__((always_inline)) {
      constexpr int m = decltype(mc)::value;
      const gq_u4 a0 = few_operand<NG, 2 * m>(xv), a1 = few_operand<NG, 2 * m + 1>(xv);
      gq_f4 sx = zero;
      if constexpr (OFF != 0.f || FMT == GQ_FMT_Q4_K) sx = few_mfma<XT>(a1, ones, few_mfma<XT>(a0, ones, zero));
#pragma unroll
      for (int t = 0; t < T; ++t) {
        gq_u4 b[2];
        few_codes<FMT, XT>(us[st][t], m, mg, b);
        const gq_f4 d = few_mfma<XT>(a1, b[1], few_mfma<XT>(a0, b[0], zero));
        const float o = FMT == GQ_FMT_Q4_K ? fmaf(s[t][m], OFF, mn[t][m]) : 0.f;
#pragma unroll
        for (int v = 0; v < MR; ++v) {
          if constexpr (FMT == GQ_FMT_Q4_K) acc[t][v] = fmaf(s[t][m], d[v], fmaf(-o, sx[v], acc[t][v]));
          else acc[t][v] = fmaf(s[t][m], OFF != 0.f ? fmaf(-OFF, sx[v], d[v]) : d[v], acc[t][v]);
        }
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
  };
  walk_units<PD, KS>(units, wave, request, compute);
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int v = 0; v < MR; ++v) red[wave][t][v][lane] = acc[t][v];
  __syncthreads();
  front_out<KS, R>(
      [&](int k, int w, int t, int n, int m) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) y += red[k][w * R + t][MR == 1 ? 0 : m][16 * i + n];
        return y;
      },
      rs, h, go, uo, dt, M, N, act, (int)blockIdx.x);
}

template <int FMT, int MT, int R, int KS>
__global__ void __launch_bounds__(64 * KS)
k_front_rows(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off,
             const _Float16 *__restrict__ a16, int lda, const float *__restrict__ rs, void *__restrict__ h,
             void *__restrict__ go, void *__restrict__ uo, int dt, int M, int N, int C, int units, int act) {
  constexpr int T = 2 * R, PD = R == 1 ? 3 : 2;
  __shared__ gq_f4 red[KS][T][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15, ntiles = (int)gq_tiles(N);
  FTile<FMT> tl[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int tile = (int)blockIdx.x * R + t % R;
    tl[t] = ftile<FMT>(t < R ? wg : wu, sc_off, (size_t)(tile < ntiles ? tile : ntiles - 1), C);  // (clamped: not stored)
  }
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<_Float16 *>(a16), (short)0, (int)(2u * (uint32_t)M * (uint32_t)lda), 0x00020000);
  uint32_t xo[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int row = 16 * t + r;
    xo[t] = 2u * ((uint32_t)(row < M ? row : M - 1) * (uint32_t)lda + 16u * (uint32_t)g);  // (rows past M: not stored)
  }
  FUnit<FMT> us[PD][T];
  gq_half8 xs[PD][MT][4];
  auto request = [&](int unit, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < T; ++t) load_unit<FMT>(tl[t], unit, lane, us[st][t]);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint32_t o = unit < units ? xo[t] + 256u * (uint32_t)unit : 0xFFFFFF00u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(xr, o, 128u * (i >> 1) + 16u * (i & 1), 0);
        xs[st][t][i] = __builtin_bit_cast(gq_half8, gq_u4{v[0], v[1], v[2], v[3]});
      }
    }
  };
  gq_f4 acc[T][MT];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[t][i] = gq_f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t mg = gq_nib_magic();
  auto compute = [&](int unit, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < T; ++t) rows_add<FMT, MT>(us[st][t], unit, g, mg, xs[st], acc[t]);
  };
  walk_units<PD, KS>(units, wave, request, compute);
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wave][t][i][lane] = acc[t][i];
  __syncthreads();
  front_out<KS, R>(
      [&](int k, int w, int t, int n, int m) {
        return reinterpret_cast<const float *>(&red[k][w * R + t][m >> 4][16 * ((m >> 2) & 3) + n])[m & 3];
      },
      rs, h, go, uo, dt, M, N, act, (int)blockIdx.x);
}

// K up to 4096: x stays in registers.  A wave's share of K is the same for every row tile, so a
// workgroup of 8 waves reads (and converts) x once and walks the tiles blockIdx.x, + gridDim.x, ...; while a
// unit of one tile is computed the same unit of the next tile is requested, NU units in
// flight a wave.  14336 x 4096, 16 rows, Q4_K / Q6_K: x read for every tile 27.5 / 31.3 us, so 21.8 / 26.2.
constexpr int kPxWaves = 8;
// Up to 4 rows of 16-bit x (the sums of k_front_few).  The operands made of x and its sums stay in
// registers too: 14336 x 4096 Q4_K one row 17.3 us with them made for every tile, 15.4 so.
template <int FMT, int XT, int MR, int NU>
__global__ void __launch_bounds__(64 * kPxWaves) __attribute__((amdgpu_waves_per_eu(2)))
k_front_few_px(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off, const void *__restrict__ x,
               void *__restrict__ h, void *__restrict__ go, void *__restrict__ uo, int dt, int M, int N, int K, int C,
               int units, int act) {
  constexpr int NG = kFewGroups<FMT>;
  constexpr float OFF = kFewOff<FMT, XT>;
  __shared__ float red[2][kPxWaves][2][MR][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, ntiles = (int)gq_tiles(N);
  constexpr bool SUMS = OFF != 0.f || FMT == GQ_FMT_Q4_K;
  gq_u4 ops[NU][4];
  float sums[NU][2][MR];
  constexpr uint32_t one = XT == GQ_DT_F16 ? 0x3C003C00u : 0x3F803F80u;
  const gq_u4 ones = {one, one, one, one};
  const gq_f4 zero = {0.f, 0.f, 0.f, 0.f};
  auto operands = [&](const gq_u4 &v, gq_u4 (&o)[4], float (&sx)[2][MR]) __attribute__((always_inline)) {
    o[0] = few_operand<NG, 0>(v);
    o[1] = few_operand<NG, 1>(v);
    o[2] = few_operand<NG, 2>(v);
    o[3] = few_operand<NG, 3>(v);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const gq_f4 t = SUMS ? few_mfma<XT>(o[2 * m + 1], ones, few_mfma<XT>(o[2 * m], ones, zero)) : zero;
#pragma unroll
      for (int e = 0; e < MR; ++e) sx[m][e] = t[e];
    }
  };
  const int row = lane & 3, xk = 128 * wave + 64 * ((lane >> 3) & 1) + 16 * g + 8 * ((lane >> 2) & 1);
  auto xin = [&](int i) { return row < M && xk + 128 * kPxWaves * i < K; };  // (whole 32-blocks: a run is wholly in or out)
  FRaw<XT> raw[NU];
  auto load_x = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NU; ++i) px_load<XT>(x, xin(i) ? (size_t)row * K + xk + 128 * kPxWaves * i : 0, raw[i]);
  };
  auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      gq_u4 v = raw[i].v[0];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = xin(i) ? v[e] : 0u;
      operands(kNibOrder<FMT> ? nib_order(v) : v, ops[i], sums[i]);
    }
  };
  FUnit<FMT> us[NU][2];
  auto request = [&](int tile, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
      load_unit<FMT>(ftile<FMT>(w ? wu : wg, sc_off, (size_t)tile, tile < ntiles ? C : 0), wave + kPxWaves * i, lane, us[i][w]);
  };
  float acc[2][MR] = {};
  uint32_t mg;  // (kept in a register)
  if constexpr (XT == GQ_DT_F16) asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(mg));
  else asm volatile("v_mov_b32 %0, 0x43004300" : "=v"(mg));
  auto compute = [&](int i) __attribute__((always_inline)) {
    float s[2][2], mn[2][2];
#pragma unroll
    for (int w = 0; w < 2; ++w) few_scales<FMT>(us[i][w], wave, g & (NG - 1), s[w], mn[w]);  // (8 i units on: the same half)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        gq_u4 b[2];
        few_codes<FMT, XT>(us[i][w], m, mg, b);
        const gq_f4 d = few_mfma<XT>(ops[i][2 * m + 1], b[1], few_mfma<XT>(ops[i][2 * m], b[0], zero));
        const float o = FMT == GQ_FMT_Q4_K ? fmaf(s[w][m], OFF, mn[w][m]) : 0.f;
#pragma unroll
        for (int v = 0; v < MR; ++v) {
          if constexpr (FMT == GQ_FMT_Q4_K) acc[w][v] = fmaf(s[w][m], d[v], fmaf(-o, sums[i][m][v], acc[w][v]));
          else acc[w][v] = fmaf(s[w][m], SUMS ? fmaf(-OFF, sums[i][m][v], d[v]) : d[v], acc[w][v]);
        }
      }
  };
  auto finish = [&](int tile, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int v = 0; v < MR; ++v) {
        red[buf][wave][w][v][lane] = acc[w][v];
        acc[w][v] = 0.f;
      }
    __syncthreads();
    front_out<kPxWaves, 1>(
        [&](int k, int w, int t, int n, int m) {
          float y = 0.f;
#pragma unroll
          for (int i = 0; i < NG; ++i) y += red[buf][k][w][MR == 1 ? 0 : m][16 * i + n];
          return y;
        },
        nullptr, h, go, uo, dt, M, N, act, tile);
  };
  walk_tiles<NU>(ntiles, load_x, request, begin, compute, finish);
}

// Up to 32 rows of any x (the weights of k_front_rows).  x to fp16 with a power-of-two scale per
// row and wave: the largest of the wave's share of a row is brought into [2^14, 2^15), one rounding
// to fp16, and the wave's sums are scaled back in fp32 before they are added to the other waves'.
template <int FMT, int XT, int MT, int NU>
__global__ void __launch_bounds__(64 * kPxWaves) __attribute__((amdgpu_waves_per_eu(2)))
k_front_rows_px(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off, const void *__restrict__ x,
                void *__restrict__ h, void *__restrict__ go, void *__restrict__ uo, int dt, int M, int N, int K, int C,
                int units, int act) {
  __shared__ gq_f4 red[2][kPxWaves][2][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15, ntiles = (int)gq_tiles(N);
  FUnit<FMT> us[NU][2];
  auto request = [&](int tile, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
      load_unit<FMT>(ftile<FMT>(w ? wu : wg, sc_off, (size_t)tile, tile < ntiles ? C : 0), wave + kPxWaves * i, lane, us[i][w]);
  };
  gq_half8 xs[NU][MT][4];
  float back[MT][4];  // what undoes the scales of this lane's rows of the result, 16 t + 4 g + v
  auto xin = [&](int t, int i, int f) {
    return 16 * t + r < M && 128 * (wave + kPxWaves * i) + 64 * (f >> 1) + 16 * g + 8 * (f & 1) < K;
  };
  FRaw<XT> raw[MT][NU][4];  // x as loaded
  auto load_x = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const int k = 128 * (wave + kPxWaves * i) + 64 * (f >> 1) + 16 * g + 8 * (f & 1);
          px_load<XT>(x, xin(t, i, f) ? (size_t)(16 * t + r) * K + k : 0, raw[t][i][f]);
        }
  };
  auto begin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          float v[8];
          px_floats<XT>(raw[t][i][f], xin(t, i, f), v);
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
        }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const int sh = gq_fp16_shift(top);
      const float f2 = gq_pow2(sh), inv = gq_pow2(-sh);
#pragma unroll
      for (int v = 0; v < 4; ++v) back[t][v] = __shfl(inv, 4 * g + v, 64);
#pragma unroll
      for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          float v[8];
          px_floats<XT>(raw[t][i][f], xin(t, i, f), v);
          constexpr int perm[8] = {0, 2, 4, 6, 1, 3, 5, 7};  // the nibbles' order, their 16 x divided out
#pragma unroll
          for (int e = 0; e < 8; ++e)
            xs[i][t][f][e] = (_Float16)(kNibOrder<FMT> ? ((e & 2) ? v[perm[e]] * 0.0625f : v[perm[e]]) * f2 : v[e] * f2);
        }
    }
  };
  gq_f4 acc[2][MT];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[w][t] = gq_f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t mg = gq_nib_magic();
  auto compute = [&](int i) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
      rows_add<FMT, MT>(us[i][w], wave, g, mg, xs[i], acc[w]);  // (8 i units on: the same half of a super-block)
  };
  auto finish = [&](int tile, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[w][t][v] *= back[t][v];
        red[buf][wave][w][t][lane] = acc[w][t];
        acc[w][t] = gq_f4{0.f, 0.f, 0.f, 0.f};
      }
    __syncthreads();
    front_out<kPxWaves, 1>(
        [&](int k, int w, int t, int n, int m) {
          return reinterpret_cast<const float *>(&red[buf][k][w][m >> 4][16 * ((m >> 2) & 3) + n])[m & 3];
        },
        nullptr, h, go, uo, dt, M, N, act, tile);
  };
  walk_tiles<NU>(ntiles, load_x, request, begin, compute, finish);
}

// ---- forward: register-B tiles ---------------------------------------------------
// gq_gemm's register-B kernel on two matrices at once: a wave owns NJ 32-column blocks of
// W_gate and the same of W_up, so one activation fragment read from LDS feeds the products of
// both, and the epilogue has g and u of an output in the same lane: h (and g, u where they
// are kept) goes out once, nothing comes back.  Operand order, swizzle and pipeline are those
// of gq_gemm_frag.h: fp16 activations by LDS DMA PD - 1 steps of 64 k ahead, weights PD steps
// ahead in registers.  So are the weights' roundings to fp16: Q4_0 and Q8_0 once (1.7e-4 and 2.1e-4 of a product's row), Q6_K
// d sc first (2.9e-4), Q4_K dmin m first (5.4e-4 where minima are 7.5 scales, as in weights about zero; as d sc (q - 8) + c, c
// rounded, 2.3e-4 there, but 2.8e-4 against 2.1e-4 where they are not).
// KG: groups of waves that share the tile and take every KG-th step,
// their sums added through LDS at the end.
template <int FMT, int BM, int WN, int NJ, int PD, int KG>
__global__ void __launch_bounds__(64 * WN * KG) __attribute__((amdgpu_waves_per_eu(front_wpe(WN *KG), front_wpe(WN *KG))))
k_front_rb(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, uint32_t sc_off,
           const _Float16 *__restrict__ a16, int lda, const float *__restrict__ rs, void *__restrict__ h,
           void *__restrict__ go, void *__restrict__ uo, int dt, int M, int N, int C, int nsteps, int tiles_m, int act) {
  constexpr int KS = BK / 16, NW = WN, TM = BM / 32, BN = 32 * NJ * WN;
  __shared__ __attribute__((aligned(16))) _Float16 As_0[KG * BM * BK];
  __shared__ __attribute__((aligned(16))) _Float16 As_1[KG * BM * BK];
  __shared__ __attribute__((aligned(16))) _Float16 As_2[PD >= 3 ? KG * BM * BK : 8];
  __shared__ __attribute__((aligned(16))) _Float16 As_3[PD >= 4 ? KG * BM * BK : 8];
  __shared__ __attribute__((aligned(16))) float rs_s[BM];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane((tid >> 6) / NW);
  const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) % NW);
  const int wn = wave;
  auto As_of = [&](auto b) -> _Float16 * {
    constexpr int v = decltype(b)::value;
    return (v == 0 ? As_0 : v == 1 ? As_1 : v == 2 ? As_2 : As_3) + kg * (BM * BK);
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  using B2 = std::integral_constant<int, 2>;
  using B3 = std::integral_constant<int, 3>;
  // loads a step may leave in flight: activations of steps s + 2 .. s + PD - 1, weights of s + 2 .. s + PD
  constexpr int NA = BM / (8 * NW), pend = (PD - 2) * NA + (PD - 1) * 2 * kRLoads<FMT> * NJ;
  int mt, nt;
  tile_of_g(blockIdx.x, gridDim.x, tiles_m, (N + BN - 1) / BN, 4, mt, nt);
  const int m0 = mt * BM, n0 = nt * BN, nl = nsteps / KG;
  const int ntiles = (int)gq_tiles(N), kh = lane >> 5, r = lane & 15;
  uint32_t qo[NJ], so[NJ];  // byte offsets of this lane's codes (slot kh) and scales, chunk 0
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    int t = (n0 + 32 * (NJ * wn + j) + (lane & 31)) >> 4;
    if (t >= ntiles) t = ntiles - 1;  // clamped; those columns are never stored
    const uint32_t tc = (uint32_t)t * (uint32_t)C;
    qo[j] = tc * (uint32_t)gq_chunk_qs_bytes(FMT) + 16u * (16u * (uint32_t)kh + (uint32_t)r);
    so[j] = sc_off + tc * (uint32_t)gq_chunk_sc_bytes(FMT) + (FMT == GQ_FMT_Q4_0 || FMT == GQ_FMT_Q8_0 ? 8u : 16u) * r;
  }
  gq_f16v acc[2][TM][NJ];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[w][i][j][v] = 0.f;
  RStep<FMT, NJ> st[2][PD];
  const uint32_t mg = gq_nib_magic();
  uint32_t ao[NA];
  a_offsets<BM, NW>(lda, M, m0, wave, lane, ao);
  const int arow = lane & 31, sw = a_swz(lane & 31);
  auto gstep = [&](int l) { return (l < nl ? l : nl - 1) * KG + kg; };
  auto run_step = [&](int l, auto buf_c) __attribute__((always_inline)) {
    constexpr int BUF = decltype(buf_c)::value;
    using NB = std::integral_constant<int, (BUF + PD - 1) % PD>;
    const int step = l * KG + kg, s1 = gstep(l + PD - 1), s2 = gstep(l + PD);
    load_a_lds_b<BM, NW>(a16, ao, s1, wave, As_of(NB{}));
    __builtin_amdgcn_sched_barrier(0);
    const _Float16 *As = As_of(buf_c) + arow * BK;
    gq_half8 af[2][TM];
    auto read_a = [&](int ks, int fb) __attribute__((always_inline)) {
      const int ch = (4 * (ks >> 1) + 2 * kh + (ks & 1)) ^ sw;
#pragma unroll
      for (int i = 0; i < TM; ++i) af[fb][i] = *reinterpret_cast<const gq_half8 *>(As + 32 * i * BK + 8 * ch);
    };
    read_a(0, 0);
    QKf qk[2][NJ][2];
    gq_half2 q6[2][NJ][2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if constexpr (FMT == GQ_FMT_Q4_K) q4k_factors<NJ>(st[w][BUF], step, qk[w]);
      if constexpr (FMT == GQ_FMT_Q6_K) q6k_factors<NJ>(st[w][BUF], kh, q6[w]);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS) read_a(ks + 1, (ks + 1) & 1);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const gq_half8 bf = rfrag<FMT, NJ>(st[w][BUF], j, ks, step, qk[w][j], q6[w][j], mg);
#pragma unroll
          for (int i = 0; i < TM; ++i) acc[w][i][j] = gq_mfma32(af[ks & 1][i], bf, acc[w][i][j]);
        }
    }
    load_rstep<FMT, NJ>(wg, qo, so, s2, st[0][BUF]);
    load_rstep<FMT, NJ>(wu, qo, so, s2, st[1][BUF]);
    step_barrier<pend>();
  };
  auto prime = [&](auto b) __attribute__((always_inline)) {
    constexpr int i = decltype(b)::value;
    const int s = gstep(i);
    if constexpr (i < PD - 1) load_a_lds_b<BM, NW>(a16, ao, s, wave, As_of(b));
    __builtin_amdgcn_sched_barrier(0);  // (pend counts this order)
    load_rstep<FMT, NJ>(wg, qo, so, s, st[0][i]);
    load_rstep<FMT, NJ>(wu, qo, so, s, st[1][i]);
    __builtin_amdgcn_sched_barrier(0);
  };
  const gq_f4 rs4 = *reinterpret_cast<const gq_f4 *>(rs + m0 + 4 * (tid % (BM / 4)));  // (padded past M)
  prime(B0{});
  prime(B1{});
  if constexpr (PD >= 3) prime(B2{});
  if constexpr (PD >= 4) prime(B3{});
  if (tid < BM / 4) *reinterpret_cast<gq_f4 *>(rs_s + 4 * tid) = rs4;
  step_barrier<pend>();
  for (int l = 0; l < nl; l += PD) {
    run_step(l, B0{});
    if (l + 1 < nl) run_step(l + 1, B1{});
    if constexpr (PD >= 3)
      if (l + 2 < nl) run_step(l + 2, B2{});
    if constexpr (PD >= 4)
      if (l + 3 < nl) run_step(l + 3, B3{});
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // (loads of no step still on their way to LDS)
  if constexpr (KG > 1) {
    __shared__ __attribute__((aligned(16))) gq_f4 xs[(KG - 1) * NW * 4 * 64];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          gq_f16v &a = acc[w][i][j];
          if (kg > 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              xs[(((kg - 1) * NW + wave) * 4 + q) * 64 + lane] = gq_f4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
          }
          __syncthreads();
          if (kg == 0) {
#pragma unroll
            for (int g = 0; g < KG - 1; ++g)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const gq_f4 t = xs[((g * NW + wave) * 4 + q) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) a[4 * q + e] += t[e];
              }
          }
          __syncthreads();
        }
    if (kg > 0) return;
  }
  // D layout (32x32): lane l holds column l % 32, rows 8 (v / 4) + 4 (l / 32) + v % 4.  Rows >= M lie
  // past the resource's end, whose check need not count a scalar offset: all of it is in the lane's
  // (host: a tile's rows span less than 2 GiB).
  auto store = [&](auto dtc) __attribute__((always_inline)) {
    constexpr int DT = decltype(dtc)::value;
    constexpr uint32_t ES = DT == GQ_DT_F32 ? 4u : 2u;
    const size_t left = (size_t)(M - m0) * (size_t)N * ES;
    const int range = (int)(uint32_t)(left < 0xFFFFFFFFu ? left : 0xFFFFFFFFu);
    auto rsrc = [&](void *p) {
      return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<uint8_t *>(p) + (p ? (size_t)m0 * N * ES : 0), (short)0,
                                               p ? range : 0, 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t hr = rsrc(h), gr = rsrc(go), ur = rsrc(uo);  // (an output not wanted: no range)
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int mb = 32 * i + 4 * (lane >> 5);
      float rsv[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const gq_f4 t = *reinterpret_cast<const gq_f4 *>(rs_s + mb + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) rsv[4 * q + e] = t[e];
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int n = n0 + 32 * (NJ * wn + j) + (lane & 31);
        if (n >= N) continue;
        const uint32_t vo = ((uint32_t)mb * (uint32_t)N + (uint32_t)n) * ES;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const uint32_t o = vo + (uint32_t)(8 * (v >> 2) + (v & 3)) * (uint32_t)N * ES;
          const float g = acc[0][i][j][v] * rsv[v], u = acc[1][i][j][v] * rsv[v];
          front_put<DT>(hr, o, dt, gq_act_f(act, g) * u);
          if (go) front_put<DT>(gr, o, dt, g);
          if (uo) front_put<DT>(ur, o, dt, u);
        }
      }
    }
  };
  if (dt == GQ_DT_F32) store(std::integral_constant<int, GQ_DT_F32>{});
  else store(std::integral_constant<int, GQ_DT_BF16>{});
}

// ---- backward --------------------------------------------------------------------
// dg = dh u act'(g), du = dh act(g): one pass over dh, g, u, a workgroup a row.  The products
// go out in their own type where they are wanted, and, as they are before that rounding, to fp16
// [dg | du] with one power-of-two scale per row (the row's largest to [2^14, 2^15); 2^-114 to 2^126), the A operand of
// dx, each half padded with zeros to np columns (whole steps of 64).  The first 4096 x 4 columns of a
// row stay in registers between the maximum and the conversion, the rest is computed twice.
GQ_DEV void front_grads(int act, float dh, float g, float u, float &dg, float &du) {
  float f, d;
  gq_act_fd(act, g, f, d);
  dg = dh * u * d;
  du = dh * f;
}
constexpr int kDguThreads = 512, kDguRuns = 4;
// (no __restrict__: dg may be g, du may be u or dh; every element is read by the thread that writes it, before)
template <int DT>
__global__ void __launch_bounds__(kDguThreads) k_front_dgu(const void *dh, const void *g, const void *u, void *dgo, void *duo,
                                                           _Float16 *a16, float *rs, int N, int np, int act) {
  __shared__ float top_s[kDguThreads / 64];
  const int tid = threadIdx.x;
  const size_t row = (size_t)blockIdx.x * (size_t)N;
  _Float16 *ar = a16 + (size_t)blockIdx.x * 2 * (size_t)np;
  float dg[kDguRuns][8], du[kDguRuns][8], top = 0.f;
  auto grads = [&](int k, float (&a)[8], float (&b)[8]) __attribute__((always_inline)) {
    float x[8], y[8], z[8];
    dgu_load<DT>(dh, row, k, N, x);
    dgu_load<DT>(g, row, k, N, y);
    dgu_load<DT>(u, row, k, N, z);
#pragma unroll
    for (int e = 0; e < 8; ++e) front_grads(act, x[e], y[e], z[e], a[e], b[e]);
  };
  auto put = [&](int k, const float (&a)[8], const float (&b)[8]) __attribute__((always_inline)) {
    if (k >= N) return;
    if (dgo) dgu_store<DT>(dgo, row, k, N, a);
    if (duo) dgu_store<DT>(duo, row, k, N, b);
  };
#pragma unroll
  for (int i = 0; i < kDguRuns; ++i) {
    const int k = 8 * (tid + kDguThreads * i);
#pragma unroll
    for (int e = 0; e < 8; ++e) dg[i][e] = du[i][e] = 0.f;
    if (k < N) grads(k, dg[i], du[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fmaxf(fabsf(dg[i][e]), fabsf(du[i][e])));
  }
  constexpr int SPAN = 8 * kDguThreads * kDguRuns;
  if (a16)
    for (int k = SPAN + 8 * tid; k < N; k += 8 * kDguThreads) {
      float a[8], b[8];
      grads(k, a, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fmaxf(fabsf(a[e]), fabsf(b[e])));
    }
  float f2 = 0.f;
  if (a16) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if ((tid & 63) == 0) top_s[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kDguThreads / 64; ++w) top = fmaxf(top, top_s[w]);
    const int sh = gq_fp16_shift(top);
    f2 = gq_pow2(sh);
    if (tid == 0) rs[blockIdx.x] = gq_pow2(-sh);
  }
  auto put16 = [&](int k, const float (&a)[8], const float (&b)[8]) __attribute__((always_inline)) {
    if (!a16 || k >= np) return;
    gq_half8 x, y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = (_Float16)(a[e] * f2);
      y[e] = (_Float16)(b[e] * f2);
    }
    *reinterpret_cast<gq_half8 *>(ar + k) = x;
    *reinterpret_cast<gq_half8 *>(ar + np + k) = y;
  };
#pragma unroll
  for (int i = 0; i < kDguRuns; ++i) {
    const int k = 8 * (tid + kDguThreads * i);
    put(k, dg[i], du[i]);
    put16(k, dg[i], du[i]);
  }
  for (int k = SPAN + 8 * tid; k < (a16 ? np : N); k += 8 * kDguThreads) {
    float a[8], b[8];
    grads(k, a, b);
    put(k, a, b);
    put16(k, a, b);
  }
}

// dx[m][k] = sum over n of dg[m][n] W_gate[n][k] + du[m][n] W_up[n][k]: the sum runs over the weights'
// rows, while a T16 record holds 16 rows of 128 k, each row's codes side by side.  Steps of 64 n (four row
// tiles), the first matrix's before the second's (`half` steps each; or one matrix alone, half = nsteps).  The records go to LDS as they are (by DMA, the slots of a 64-lane
// record XOR-swizzled), and a lane collects for its four columns the codes of 8 rows, 16 bits (Q8_0
// 32) a row: joined in pairs of rows they are masked into fp16 pairs that run along n, B
// fragments of v_mfma_f32_32x32x16_f16 without a transposition.  Lane c of 32 owns columns
//   4-bit and Q6_K: 32 (c / 8) + 16 (c / 4 % 2) + 8 (c / 2 % 2) + 2 (c % 2) + {0, 4, 1, 5}  Q8_0: 4 c + {0, 1, 2, 3}
// of 128, one per fragment; the second and fourth of the former come out 16 x (nibbles masked in place) and
// the sums are divided by 16 at the end.  Scales vary along n: a wave brings the step's 64 rows'
// scales to LDS as fp16 [group of columns][16 rows], a lane's 8 rows one 16-byte read.  (Q4_K: sc, -dmin m
// rounded to fp16, and d apart, so that sc q is exact and d sc q - dmin m rounded once.)
template <int FMT>
constexpr int kDxGroups = FMT == GQ_FMT_Q6_K ? 8 : 4;  // scale groups of 128 columns
template <int FMT>
constexpr int kDxRecs = FMT == GQ_FMT_Q8_0 || FMT == GQ_FMT_Q6_K ? 2 : 1;  // 1 KiB records of 128 columns and a row tile
template <int FMT>
constexpr int kDxRows = FMT == GQ_FMT_Q4_K ? 9 : kDxGroups<FMT>;  // [16 rows] of a tile's table: 4 sc, 4 minima, d; else the scales

// scales of row r (of a tile) for 128 columns, as loaded
template <int FMT>
GQ_DEV gq_u4 dx_load_scales(const __amdgpu_buffer_rsrc_t &w, uint32_t sc_off, uint32_t tc, uint32_t p, uint32_t r, bool in) {
  const uint32_t o = in ? sc_off + tc * HFmt<FMT>::SB : 0xFFFFF000u;  // (outside: zeros)
  gq_u4 v = {0, 0, 0, 0};
  if constexpr (FMT == GQ_FMT_Q4_K) {
    const auto t = __builtin_amdgcn_raw_buffer_load_b128(w, o + 16u * r, 0, 0);
    v = gq_u4{t[0], t[1], t[2], t[3]};
  } else if constexpr (FMT == GQ_FMT_Q6_K) {
    const auto t = __builtin_amdgcn_raw_buffer_load_b64(w, o + 16u * r + 8u * p, 0, 0);
    v[0] = t[0];
    v[1] = t[1];
    v[2] = __builtin_amdgcn_raw_buffer_load_b16(w, o + 256u + 2u * r, 0, 0);
  } else {
    const auto t = __builtin_amdgcn_raw_buffer_load_b64(w, o + 8u * r, 0, 0);
    v[0] = t[0];
    v[1] = t[1];
  }
  return v;
}
// -> the tables [table][group][16 rows] of the row's tile
template <int FMT>
GQ_DEV void dx_store_scales(const gq_u4 &v, uint32_t p, int r, _Float16 *t) {
  if constexpr (FMT == GQ_FMT_Q4_K) {
    const float dm = (float)bits_h(v[0] >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // sub-block 4 p + j
      const uint32_t sh = 16u * p + 8u * (j >> 1), b = ((j & 1) ? v[2] : v[1]) >> sh, m = v[3] >> (sh + 4u * (j & 1));
      t[16 * j + r] = (_Float16)(float)(b & 63u);
      t[16 * (4 + j) + r] = (_Float16)(-(dm * (float)(((b >> 6) & 3u) | ((m & 15u) << 2))));
    }
    t[16 * 8 + r] = bits_h(v[0]);
  } else if constexpr (FMT == GQ_FMT_Q6_K) {
    const float d = (float)bits_h(v[2]);
#pragma unroll
    for (int j = 0; j < 8; ++j) t[16 * j + r] = (_Float16)(d * (float)(int8_t)(v[j >> 2] >> (8 * (j & 3))));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) t[16 * j + r] = bits_h(v[j & 1] >> (16 * (j >> 1)));  // (d0 d2 | d1 d3)
  }
}

template <int FMT, int WN, int KG, int TM, int PD>
__global__ void __launch_bounds__(64 * WN * KG) k_front_dx(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, uint32_t w_bytes, uint32_t sc_off,
           const _Float16 *__restrict__ a16, const float *__restrict__ rs, void *__restrict__ y, int dt, int M, int K,
           int C, int ntiles, int nsteps, int half, int sps, int tiles_m) {
  constexpr int NW = WN, BM = 32 * TM, BN = 128 * WN, ROWS_T = 16 * kDxRows<FMT>, RECS = kDxRecs<FMT>;
  constexpr int NREC = 4 * WN * RECS, RPW = (NREC + NW - 1) / NW;  // records a step, per wave
  static_assert(NREC % NW == 0, "records");
  constexpr int A_B = BM * BK * 2, W_B = NREC * 1024, S_B = WN * 4 * ROWS_T * 2, STAGE = A_B + W_B + S_B;
  static_assert(PD == 2 || PD == 3, "pipeline depth");
  static_assert(KG * PD * STAGE <= 160 * 1024, "LDS");
  // an array a stage (activations, records, scales): no wait for a DMA into another one
  __shared__ __attribute__((aligned(1024))) uint8_t lds_0[KG * STAGE], lds_1[KG * STAGE], lds_2[PD == 3 ? KG * STAGE : 16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane((tid >> 6) / NW);
  const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) % NW);
  const int wn = wave;
  int mt, nt;
  tile_of_g(blockIdx.x, gridDim.x, tiles_m, (K + BN - 1) / BN, 4, mt, nt);
  const int m0 = mt * BM, kc0 = nt * WN;
  // this workgroup's steps of 64 n (part blockIdx.y), this group's every KG-th
  const int s0 = (int)blockIdx.y * sps, s1 = s0 + sps < nsteps ? s0 + sps : nsteps;
  const int nl = (s1 - s0 + KG - 1) / KG;
  __builtin_assume(nl > 0);  // (no part is empty; under a branch around the loop the loads in front of it may sink)
  const int lda = 64 * nsteps;
  auto stage = [&](int i) { return (i == 0 ? lds_0 : i == 1 ? lds_1 : lds_2) + kg * STAGE; };
  auto table = [&](int i) { return reinterpret_cast<_Float16 *>(stage(i) + A_B + W_B); };
  uint32_t ao[BM / (8 * NW)];
  a_offsets<BM, NW>(lda, M, m0, wave, lane, ao);
  auto mat = [&](bool up) __attribute__((always_inline)) {  // (the pointer is chosen, not one of two resources in memory)
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(up ? wu : wg), (short)0, (int)w_bytes, 0x00020000);
  };
  // the record's slot a lane fetches: 16 g + (rho ^ 2 g), Q8_0's second half-record (64 k on) ^ 1 more
  const uint32_t slot = 16u * (16u * (uint32_t)(lane >> 4) + (uint32_t)((lane & 15) ^ (2 * (lane >> 4))));
  auto step_of = [&](int l) { return s0 + l * KG + kg; };  // (past the part's end: skipped by the sums, A zero or not used)
  auto request = [&](int l, int st) __attribute__((always_inline)) {
    int s = step_of(l);
    s = s < s1 ? s : s1 - 1;
    load_a_lds_b<BM, NW>(a16, ao, s, wave, reinterpret_cast<_Float16 *>(stage(st)));
    const bool up = s >= half;
    const __amdgpu_buffer_rsrc_t wr = mat(up);
    const uint32_t t0 = 4u * (uint32_t)(up ? s - half : s);
    uint8_t *wl = stage(st) + A_B;
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int rec = wave * RPW + i;  // [column block][tile][record]
      const int b = rec / (4 * RECS), t = rec / RECS % 4, h = rec % RECS;
      const uint32_t kc = (uint32_t)(kc0 + b), c = kSuper<FMT> ? kc >> 1 : kc, p = kSuper<FMT> ? kc & 1u : 0u;
      // (outside: the last record, its scales are zero; clamped without a branch, which would copy the DMAs)
      const uint32_t tt = min(t0 + (uint32_t)t, (uint32_t)ntiles - 1u), cc = min(c, (uint32_t)C - 1u);
      uint32_t v = slot, o = (tt * (uint32_t)C + cc) * HFmt<FMT>::QB;
      if constexpr (FMT == GQ_FMT_Q8_0) {
        o += 1024u * (uint32_t)h;
        v ^= h ? 16u : 0u;
      } else if constexpr (FMT == GQ_FMT_Q6_K) {
        o += h ? 2048u : 1024u * p;
      } else {
        o += 1024u * p;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void *)(wl + 1024 * rec), 16, v, o, 0, 0);
    }
  };
  // scales: a wave those of its own column block, a row a lane
  const int srow = lane & 15, stile = lane >> 4;
  auto load_scales = [&](int l) __attribute__((always_inline)) {
    int s = step_of(l);
    s = s < s1 ? s : s1 - 1;
    const bool up = s >= half;
    const uint32_t t = 4u * (uint32_t)(up ? s - half : s) + (uint32_t)stile, kc = (uint32_t)(kc0 + wave);
    const uint32_t c = kSuper<FMT> ? kc >> 1 : kc;
    return dx_load_scales<FMT>(mat(up), sc_off, t * (uint32_t)C + c, kSuper<FMT> ? kc & 1u : 0u, (uint32_t)srow,
                               t < (uint32_t)ntiles && c < (uint32_t)C);
  };
  auto store_scales = [&](const gq_u4 &v, int st) __attribute__((always_inline)) {
    _Float16 *t = table(st) + (wave * 4 + stile) * ROWS_T;
    dx_store_scales<FMT>(v, kSuper<FMT> ? (uint32_t)(kc0 + wave) & 1u : 0u, srow, t);
  };

  gq_f16v acc[TM][4];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][f][v] = 0.f;
  const int c = lane & 31, kh = lane >> 5, sw = a_swz(lane & 31);
  // where this lane's codes lie in a record: slot group, byte in the slot; its scale group
  const bool q8 = FMT == GQ_FMT_Q8_0;
  const int cg = q8 ? (c >> 2) & 3 : 2 * ((c >> 3) & 1) + ((c >> 2) & 1), cm = c >> 4;
  const int cb = q8 ? 4 * (c & 3) : 8 * cm + 4 * ((c >> 1) & 1) + 2 * (c & 1);
  const int grp = FMT == GQ_FMT_Q6_K ? 4 * cm + cg : 2 * cm + (cg >> 1);
  const uint32_t mg = gq_nib_magic();
  const int par = FMT == GQ_FMT_Q6_K ? (kc0 + wn) & 1 : 0;
  // byte offset of row 8 kh + e: slot 16 cg + ((8 kh + e) ^ 2 cg ^ (Q8_0: cm))
  auto row_at = [&](int e) { return 16 * (16 * cg + ((8 * kh + e) ^ (2 * cg) ^ (q8 ? cm : 0))) + (q8 ? 1024 * cm : 0); };

  auto compute = [&](int st) __attribute__((always_inline)) {
    const _Float16 *As = reinterpret_cast<const _Float16 *>(stage(st)) + (lane & 31) * BK;
    const uint8_t *Ws = stage(st) + A_B + wn * (4 * RECS * 1024);
    const _Float16 *Ss = table(st) + wn * (4 * ROWS_T) + 8 * kh;
    // a row tile's operands as they lie in LDS, one tile ahead of the products
    gq_half8 af[2][TM], s8[2], m8[2], d8[2];
    uint32_t cw[2][8], hw[2][8];
    auto read = [&](int t, int x) __attribute__((always_inline)) {
      const uint8_t *W = Ws + t * (RECS * 1024) + cb;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (FMT == GQ_FMT_Q8_0) cw[x][e] = *reinterpret_cast<const uint32_t *>(W + row_at(e));
        else cw[x][e] = *reinterpret_cast<const uint16_t *>(W + row_at(e));
        // (Q6_K's high fields: bytes 2 hw, 2 hw + 1 of the step's word)
        if constexpr (FMT == GQ_FMT_Q6_K)
          hw[x][e] = *reinterpret_cast<const uint16_t *>(Ws + t * (RECS * 1024) + 1024 + 4 * (2 * par + cm) + 2 * (c & 1) + row_at(e));
      }
      const _Float16 *S = Ss + t * ROWS_T;
      s8[x] = *reinterpret_cast<const gq_half8 *>(S + 16 * grp);
      if constexpr (FMT == GQ_FMT_Q4_K) {
        m8[x] = *reinterpret_cast<const gq_half8 *>(S + 16 * (4 + grp));
        d8[x] = *reinterpret_cast<const gq_half8 *>(S + 16 * 8);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) af[x][i] = *reinterpret_cast<const gq_half8 *>(As + 32 * i * BK + 8 * ((2 * t + kh) ^ sw));
    };
    read(0, 0);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int x = t & 1;
      if (t < 3) read(t + 1, x ^ 1);
      gq_half8 bf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // rows 2 j, 2 j + 1
        uint32_t q[4];               // fp16 pairs 1024 + code (4-bit, Q6_K: of the second and fourth 16 x the code)
        if constexpr (FMT == GQ_FMT_Q8_0) {
#pragma unroll
          for (int f = 0; f < 4; ++f)
            q[f] = __builtin_amdgcn_perm(cw[x][2 * j + 1], cw[x][2 * j], 0x0C040C00u + 0x00010001u * (uint32_t)f) ^ 0x64806480u;
        } else {
          const uint32_t v = cw[x][2 * j] | cw[x][2 * j + 1] << 16, v8 = v >> 8;
          q[0] = (v & 0x000F000Fu) | mg;
          q[1] = (v & 0x00F000F0u) | mg;
          q[2] = (v8 & 0x000F000Fu) | mg;
          q[3] = (v8 & 0x00F000F0u) | mg;
          if constexpr (FMT == GQ_FMT_Q6_K) {  // (the word's half w in bits 4 w .. + 3 of a byte)
            const uint32_t h = (hw[x][2 * j] | hw[x][2 * j + 1] << 16) >> (4 * ((c >> 1) & 1)), h8 = h >> 8;
            q[0] |= (h << 4) & 0x00300030u;
            q[1] |= (h << 6) & 0x03000300u;
            q[2] |= (h8 << 4) & 0x00300030u;
            q[3] |= (h8 << 6) & 0x03000300u;
          }
        }
        const gq_half2 s2 = {s8[x][2 * j], s8[x][2 * j + 1]};
        gq_half2 m2 = s2, m16 = s2, d2 = s2, n2 = s2;
        if constexpr (FMT == GQ_FMT_Q4_K) {
          m2 = gq_half2{m8[x][2 * j], m8[x][2 * j + 1]};
          m16 = m2 * gq_half2{(_Float16)16.0f, (_Float16)16.0f};
          d2 = gq_half2{d8[x][2 * j], d8[x][2 * j + 1]};
          n2 = s2 * gq_half2{(_Float16)-1024.0f, (_Float16)-1024.0f};
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          const bool x16 = !q8 && (f & 1);
          const float off = q8                     ? -1152.f
                            : FMT == GQ_FMT_Q4_0 ? (x16 ? -1152.f : -1032.f)
                                                 : (x16 ? -1536.f : -1056.f);
          gq_half2 r;
          if constexpr (FMT == GQ_FMT_Q4_K)  // (sc q or 16 sc q, exact; then one rounding)
            r = __builtin_elementwise_fma(__builtin_elementwise_fma(gq_bits_h2(q[f]), s2, n2), d2, x16 ? m16 : m2);
          else
            r = (gq_bits_h2(q[f]) + gq_half2{(_Float16)off, (_Float16)off}) * s2;  // (the sum is exact)
          bf[f][2 * j] = r[0];
          bf[f][2 * j + 1] = r[1];
        }
      }
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][f] = gq_mfma32(af[x][i], bf[f], acc[i][f]);
    }
  };

  // Step l computes from stage l % PD; the loads of step l + PD - 1 go into the stage step l - 1 has
  // left, the scales of l + 2 into registers, those of l + 1 from there to LDS.  At its end the DMA of l + 1
  // must have landed.  Every step issues its DMAs first and its scales behind them (kept so by the
  // sched_barriers: the count is of that order), so behind the DMA of l + 1 come, PD = 2, the scales of l + 2; PD =
  // 3, those of l + 1, the DMA of l + 2 and the scales of l + 2.
  constexpr int ND = BM / (8 * NW) + RPW, SL = FMT == GQ_FMT_Q6_K ? 2 : 1, pend = (PD - 2) * ND + (PD - 1) * SL;
  gq_u4 sv[PD];
  const gq_u4 first = load_scales(0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < PD - 1; ++i) request(i, i);
  __builtin_amdgcn_sched_barrier(0);
  sv[1] = load_scales(1);
  __builtin_amdgcn_sched_barrier(0);  // (no wait for the scales before all of it is requested)
  store_scales(first, 0);
  step_barrier<(PD - 2) * ND>();
  for (int l = 0; l < nl; l += PD) {
#pragma unroll
    for (int i = 0; i < PD; ++i) {
      if (l + i >= nl) break;
      request(l + i + PD - 1, (i + PD - 1) % PD);
      __builtin_amdgcn_sched_barrier(0);
      sv[(i + 2) % PD] = load_scales(l + i + 2);
      __builtin_amdgcn_sched_barrier(0);
      // (the last group's step may lie past the part: nothing to add, the barriers are everyone's)
      if (KG == 1 || step_of(l + i) < s1) compute(i);
      store_scales(sv[(i + 1) % PD], (i + 1) % PD);
      step_barrier<pend>();
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // (loads of no step still on their way into the stages)
  // Out through LDS, 16 rows of the tile at a time: every wave puts its sums there by row, then the
  // groups' waves of a column block add them in group order, a share of the rows each, and store whole
  // runs.  (From the lanes that hold them, 8 bytes every 16 of a row, the stores took 12 of 46 us, 200 x
  // 5003 x 4096 Q4_K in 8 parts.)  Parts: fp32 sums [part][M][K], scaled by k_dx_sum; else dx itself.
  constexpr int LD = 132, SHARE = 16 / KG;
  static_assert(KG * NW * 16 * LD * 4 <= KG * STAGE, "LDS");
  float *xs = reinterpret_cast<float *>(lds_0);
  const bool parts = gridDim.y > 1;
  if (parts) y = reinterpret_cast<float *>(y) + (size_t)blockIdx.y * (size_t)M * (size_t)K;
  const int kl = q8 ? 4 * c : 32 * (c >> 3) + 16 * ((c >> 2) & 1) + 8 * ((c >> 1) & 1) + 2 * (c & 1);
  const int k0 = 128 * (kc0 + wn) + 4 * (lane & 31);  // the run of 4 this lane stores
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const int v = 8 * half + w;
        float *row = xs + ((kg * NW + wn) * 16 + 8 * (w >> 2) + 4 * kh + (w & 3)) * LD + kl;
        if constexpr (FMT == GQ_FMT_Q8_0) {
          *reinterpret_cast<gq_f4 *>(row) = gq_f4{acc[i][0][v], acc[i][1][v], acc[i][2][v], acc[i][3][v]};
        } else {  // (columns + 0, + 1 and + 4, + 5)
          *reinterpret_cast<float2 *>(row) = make_float2(acc[i][0][v], acc[i][2][v]);
          *reinterpret_cast<float2 *>(row + 4) = make_float2(acc[i][1][v] * 0.0625f, acc[i][3][v] * 0.0625f);
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < SHARE; j += 2) {
        const int r = kg * SHARE + j + (lane >> 5), m = m0 + 32 * i + 16 * half + r;
        gq_f4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const gq_f4 u = *reinterpret_cast<const gq_f4 *>(xs + ((g * NW + wn) * 16 + r) * LD + 4 * (lane & 31));
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] += u[e];
        }
        if (m >= M || k0 >= K) continue;  // (K is whole 32-blocks)
        const size_t at = (size_t)m * K + k0;
        const float f = parts ? 1.f : rs[m];
        if (parts || dt == GQ_DT_F32) {
          FRun32h o;
          o.v = gq_f4{t[0] * f, t[1] * f, t[2] * f, t[3] * f};
          *reinterpret_cast<FRun32h *>(reinterpret_cast<float *>(y) + at) = o;
        } else {
          uint32_t b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            b[e] = dt == GQ_DT_BF16 ? gq_f32_to_bf16(t[e] * f) : __builtin_bit_cast(uint16_t, (_Float16)(t[e] * f));
          FRun16h o;
          o.v = gq_u2{b[0] | b[1] << 16, b[2] | b[3] << 16};
          *reinterpret_cast<FRun16h *>(reinterpret_cast<uint16_t *>(y) + at) = o;
        }
      }
    }
}
// dx = rs[m] * the parts' sums, in part order (no parts: zeros).  Workgroups behind its own: a bias gradient, 16 columns each (db: gq_internal.h)
__global__ void __launch_bounds__(256) k_dx_sum(const float *__restrict__ part, const float *__restrict__ rs, void *__restrict__ y,
                                                int dt, size_t mk, int K, int parts, GqColSums db) {
  const unsigned own = (unsigned)((mk / 4 + 255) / 256);
  if (blockIdx.x >= own) {
    __shared__ double red[16][16];
    gq_col_sums<16, 16>(db, 16 * (int)(blockIdx.x - own), threadIdx.x & 15, threadIdx.x >> 4, red);
    return;
  }
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;  // (K % 32 == 0: four of one row)
  if (i >= mk) return;
  gq_f4 v = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < parts; ++p) {
    const gq_f4 t = *reinterpret_cast<const gq_f4 *>(part + (size_t)p * mk + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += t[e];
  }
  const float s = parts ? rs[i / (size_t)K] : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) gq_st_dt(y, dt, i + e, v[e] * s);
}

template <int FMT, int BM, int WN, int NJ, int PD, int KG>
int launch_front_rb(const void *wg, const void *wu, const _Float16 *a16, int lda, const float *rs, void *h, void *go,
                    void *uo, int dt, int M, int N, int K, int act, hipStream_t s) {
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (N + 32 * NJ * WN - 1) / (32 * NJ * WN);
  GQ_CHECK((size_t)tiles_m * (size_t)tiles_n <= 0x7FFFFFFFu, GQ_ERR_INVALID_ARGS);  // (one grid dimension)
  hipLaunchKernelGGL((k_front_rb<FMT, BM, WN, NJ, PD, KG>), dim3((unsigned)(tiles_m * tiles_n)), dim3(64 * WN * KG),
                     0, s, (const uint8_t *)wg, (const uint8_t *)wu, (uint32_t)gq_sc_plane_offset(FMT, N, K), a16, lda, rs,
                     h, go, uo, dt, M, N, (int)gq_chunks(FMT, K), (int)(gq_kpad(FMT, K) / BK), tiles_m, act);
  return gq_last_launch();
}
template <int FMT, int XT>
int launch_front_few_t(const void *wg, const void *wu, const void *x, const float *rs, void *h, void *go, void *uo, int dt,
                       int M, int N, int K, int act, hipStream_t s) {
  const int units = (int)(gq_kpad(FMT, K) / 128);
#define GQ_FEW(MR, R, KS)                                                                                             \
  hipLaunchKernelGGL((k_front_few<FMT, XT, MR, R, KS>), dim3((unsigned)((gq_tiles(N) + (R)-1) / (R))), dim3(64 * (KS)), 0, s, \
                     (const uint8_t *)wg, (const uint8_t *)wu, gq_sc_plane_offset(FMT, N, K), x, rs, h, go, uo, dt, M, N, K,  \
                     (int)gq_chunks(FMT, K), units, act)
  const size_t tiles = gq_tiles(N);
#define GQ_FEW_M(R, KS)          \
  do {                           \
    if (M == 1) GQ_FEW(1, R, KS); \
    else GQ_FEW(4, R, KS);       \
  } while (0)
  // (14336 x 4096 Q4_K one row: 17.6 us by one tile, 16.9 by two; 4096 x 4096 7.3 and 10.1)
  if (tiles <= 256) GQ_FEW_M(1, 8);
  else if (tiles <= 448) GQ_FEW_M(1, 4);
  else GQ_FEW_M(2, 4);
#undef GQ_FEW_M
#undef GQ_FEW
  return gq_last_launch();
}
// x in registers (front_px): any dtype and alignment of x, no workspace
template <int FMT, int XT, int NU>
int launch_front_px_n(const void *wg, const void *wu, const void *x, void *h, void *go, void *uo, int dt, int M, int N,
                      int K, int act, hipStream_t s) {
  const int tiles = (int)gq_tiles(N), cus = gq_device_cus();
  const int C = (int)gq_chunks(FMT, K), units = (int)(gq_kpad(FMT, K) / 128);
  const size_t so = gq_sc_plane_offset(FMT, N, K);
  const uint8_t *g8 = (const uint8_t *)wg, *u8 = (const uint8_t *)wu;
  const dim3 grid((unsigned)(cus > 0 && tiles > cus ? cus : tiles)), block(64 * kPxWaves);
#define GQ_PX(KERN) hipLaunchKernelGGL(KERN, grid, block, 0, s, g8, u8, so, x, h, go, uo, dt, M, N, K, C, units, act)
  if constexpr (XT != GQ_DT_F32) {
    if (M == 1) {
      GQ_PX((k_front_few_px<FMT, XT, 1, NU>));
      return gq_last_launch();
    }
    if (M <= 4) {
      GQ_PX((k_front_few_px<FMT, XT, 4, NU>));
      return gq_last_launch();
    }
  }
  if (M <= 16) {
    GQ_PX((k_front_rows_px<FMT, XT, 1, NU>));
  } else {
    if constexpr (NU <= 2) GQ_PX((k_front_rows_px<FMT, XT, 2, NU>));
  }
#undef GQ_PX
  return gq_last_launch();
}
template <int FMT, int XT>
int launch_front_px_t(const void *wg, const void *wu, const void *x, void *h, void *go, void *uo, int dt, int M, int N,
                      int K, int act, hipStream_t s) {
  const size_t units = gq_kpad(FMT, K) / 128;
  if (units <= kPxWaves) return launch_front_px_n<FMT, XT, 1>(wg, wu, x, h, go, uo, dt, M, N, K, act, s);
  if (units <= 2 * kPxWaves) return launch_front_px_n<FMT, XT, 2>(wg, wu, x, h, go, uo, dt, M, N, K, act, s);
  return launch_front_px_n<FMT, XT, 4>(wg, wu, x, h, go, uo, dt, M, N, K, act, s);
}
template <int FMT>
int launch_front_px_x(const void *wg, const void *wu, const void *x, int xt, void *h, void *go, void *uo, int dt, int M,
                      int N, int K, int act, hipStream_t s) {
  if (xt == GQ_DT_F32) return launch_front_px_t<FMT, GQ_DT_F32>(wg, wu, x, h, go, uo, dt, M, N, K, act, s);
  if (xt == GQ_DT_F16) return launch_front_px_t<FMT, GQ_DT_F16>(wg, wu, x, h, go, uo, dt, M, N, K, act, s);
  return launch_front_px_t<FMT, GQ_DT_BF16>(wg, wu, x, h, go, uo, dt, M, N, K, act, s);
}
// Up to 16 rows of K <= 4096, and 32 of K <= 2048 (with more units the registers spill: 16 rows of
// 8192 x 8192 Q4_K 40.6 us, x read for every tile 28.3; one row 20.0 and 18.6)
bool front_px(int fmt, size_t M, size_t K) {
  const size_t units = gq_kpad(fmt, K) / 128;
  return M <= 16 ? units <= 4 * kPxWaves : M <= 32 && units <= 2 * kPxWaves;
}
int launch_front_px(int fmt, const void *wg, const void *wu, const void *x, int xt, void *h, void *go, void *uo, int dt,
                    int M, int N, int K, int act, hipStream_t s) {
  if (fmt == GQ_FMT_Q4_0) return launch_front_px_x<GQ_FMT_Q4_0>(wg, wu, x, xt, h, go, uo, dt, M, N, K, act, s);
  if (fmt == GQ_FMT_Q8_0) return launch_front_px_x<GQ_FMT_Q8_0>(wg, wu, x, xt, h, go, uo, dt, M, N, K, act, s);
  if (gq_fmt_is_q6k(fmt)) return launch_front_px_x<GQ_FMT_Q6_K>(wg, wu, x, xt, h, go, uo, dt, M, N, K, act, s);
  return launch_front_px_x<GQ_FMT_Q4_K>(wg, wu, x, xt, h, go, uo, dt, M, N, K, act, s);
}

// x of xt (f16 or bf16), 4-byte aligned
int launch_front_few(int fmt, const void *wg, const void *wu, const void *x, int xt, const float *rs, void *h, void *go,
                     void *uo, int dt, int M, int N, int K, int act, hipStream_t s) {
#define GQ_FMT_X(F)                                                                                          \
  (xt == GQ_DT_F16 ? launch_front_few_t<F, GQ_DT_F16>(wg, wu, x, rs, h, go, uo, dt, M, N, K, act, s)         \
                   : launch_front_few_t<F, GQ_DT_BF16>(wg, wu, x, rs, h, go, uo, dt, M, N, K, act, s))
  if (fmt == GQ_FMT_Q4_0) return GQ_FMT_X(GQ_FMT_Q4_0);
  if (fmt == GQ_FMT_Q8_0) return GQ_FMT_X(GQ_FMT_Q8_0);
  if (gq_fmt_is_q6k(fmt)) return GQ_FMT_X(GQ_FMT_Q6_K);
  return GQ_FMT_X(GQ_FMT_Q4_K);
#undef GQ_FMT_X
}
template <int FMT>
int launch_front_rows_t(const void *wg, const void *wu, const _Float16 *a16, int lda, const float *rs, void *h, void *go,
                        void *uo, int dt, int M, int N, int K, int act, hipStream_t s) {
  const int units = (int)(gq_kpad(FMT, K) / 128);
#define GQ_ROWS(MT, R, KS)                                                                                           \
  hipLaunchKernelGGL((k_front_rows<FMT, MT, R, KS>), dim3((unsigned)((gq_tiles(N) + (R)-1) / (R))), dim3(64 * (KS)), 0, s, \
                     (const uint8_t *)wg, (const uint8_t *)wu, gq_sc_plane_offset(FMT, N, K), a16, lda, rs, h, go, uo, dt, \
                     M, N, (int)gq_chunks(FMT, K), units, act)
  // (as k_front_few; 17..32 rows by one tile, the host sends large N to the tiled kernel)
  if (M > 16) GQ_ROWS(2, 1, 4);
  else if (gq_tiles(N) <= 448) GQ_ROWS(1, 1, 4);
  else GQ_ROWS(1, 2, 4);
#undef GQ_ROWS
  return gq_last_launch();
}
int launch_front_rows(int fmt, const void *wg, const void *wu, const _Float16 *a16, int lda, const float *rs, void *h,
                      void *go, void *uo, int dt, int M, int N, int K, int act, hipStream_t s) {
  if (fmt == GQ_FMT_Q4_0) return launch_front_rows_t<GQ_FMT_Q4_0>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
  if (fmt == GQ_FMT_Q8_0) return launch_front_rows_t<GQ_FMT_Q8_0>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
  if (gq_fmt_is_q6k(fmt)) return launch_front_rows_t<GQ_FMT_Q6_K>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
  return launch_front_rows_t<GQ_FMT_Q4_K>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
}
template <int FMT>
int launch_front_fmt(const void *wg, const void *wu, const _Float16 *a16, int lda, const float *rs, void *h, void *go,
                     void *uo, int dt, int M, int N, int K, int act, hipStream_t s) {
#define GQ_FRONT(...) launch_front_rb<FMT, __VA_ARGS__>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s)
  auto wgs = [&](int bm, int bn) { return (size_t)((M + bm - 1) / bm) * (size_t)((N + bn - 1) / bn); };
  const int nsteps = (int)(gq_kpad(FMT, K) / BK);
  // About one workgroup per CU first, with K groups where the tiles alone give fewer waves
  // (Q4_K, K = 4096, us by 32 x 64 / 64 x 64 / 64 x 128 / 128 x 128 tiles: 32 x 14336 24.5 / 30.8 / 39.7 / -,
  // 64 x 14336 43.0 / 31.2 / 40.6 / 57.2, 128 x 14336 79.5 / 56.3 / 46.3 / 57.8, 256 x 4096 - / 31.5 / 40.6 / 56.2); 128
  // x 128 without groups, two workgroups a CU, for the rest: 2048 x 14336 450 us (with K groups 492,
  // 256 x 128 on 8 waves 470, on 4 waves of 256 rows 503)
  if (M <= 32 && nsteps % 4 == 0) return GQ_FRONT(32, 2, 1, 4, 4);
  if (wgs(64, 64) <= 288 && nsteps % 4 == 0) return GQ_FRONT(64, 2, 1, 3, 4);
  if (wgs(64, 128) <= 288) return GQ_FRONT(64, 4, 1, 3, 2);
  if (wgs(128, 128) <= 288) return GQ_FRONT(128, 4, 1, 3, 2);
  return GQ_FRONT(128, 4, 1, 2, 1);
#undef GQ_FRONT
}
int launch_front(int fmt, const void *wg, const void *wu, const _Float16 *a16, int lda, const float *rs, void *h, void *go,
                 void *uo, int dt, int M, int N, int K, int act, hipStream_t s) {
  if (fmt == GQ_FMT_Q4_0) return launch_front_fmt<GQ_FMT_Q4_0>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
  if (fmt == GQ_FMT_Q8_0) return launch_front_fmt<GQ_FMT_Q8_0>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
  if (gq_fmt_is_q6k(fmt)) return launch_front_fmt<GQ_FMT_Q6_K>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
  return launch_front_fmt<GQ_FMT_Q4_K>(wg, wu, a16, lda, rs, h, go, uo, dt, M, N, K, act, s);
}

int check_front(int fmt, const void *gate, const void *up, size_t M, size_t N, size_t K, int act) {
  GQ_TRY(gq_check_shape(fmt, N, K));
  GQ_CHECK(M <= GQ_MAX_DIM, GQ_ERR_INVALID_ARGS);
  GQ_CHECK(gq_act_valid(act), GQ_ERR_UNSUPPORTED);
  GQ_CHECK((gate && up) || M == 0 || N == 0, GQ_ERR_INVALID_ARGS);
  GQ_CHECK((((uintptr_t)gate | (uintptr_t)up) & 15) == 0, GQ_ERR_INVALID_ARGS);  // (16-byte loads)
  // the kernels address a packed tensor with 32-bit offsets (the last 4 KiB: those that lie outside)
  GQ_CHECK(N == 0 || K == 0 || gq_packed_bytes(fmt, N, K) <= 0xFFFFF000u, GQ_ERR_INVALID_ARGS);
  return GQ_OK;
}

}  // namespace

constexpr size_t kFewRows = 4;
// Rows that go into the few-row kernel without a conversion
static bool front_as_it_is(const void *x, int x_dtype, size_t M) {
  return M <= kFewRows && x_dtype != GQ_DT_F32 && (uintptr_t)x % 4 == 0;
}
// Rows a call takes at a time: their fp16 copies stay below 64 MiB, but for the rows that the kernels
// of few rows take at once (32 of at most 2^24 columns: 1 GiB, 32-bit offsets still)
constexpr size_t kOneBlock = 32;
static size_t front_rows(int fmt, size_t M, size_t K) {
  const size_t fit = ((size_t)64 << 20) / (2 * gq_kpad(fmt, K));
  const size_t mb = fit >= 256 ? fit & ~(size_t)255 : fit > kOneBlock ? fit : kOneBlock;
  return M < mb ? M : mb;
}

extern "C" size_t gq_ffn_gate_up_workspace_bytes(int fmt, size_t M, size_t N, size_t K) {
  if (!gq_fmt_valid(fmt) || M > GQ_MAX_DIM || N > GQ_MAX_DIM || K > GQ_MAX_DIM || K == 0) return 0;
  const size_t mb = front_rows(fmt, M, K);
  return gq_align256(mb * (gq_kpad(fmt, K) + 8) * 2) + gq_align256((mb + 256) * 4);
}

extern "C" int gq_ffn_gate_up(int fmt, const void *gate, const void *up, const void *x, int x_dtype, void *h,
                              int h_dtype, void *g, void *u, size_t M, size_t N, size_t K, int act, void *ws,
                              size_t ws_bytes, void *stream) {
  GQ_TRY(check_front(fmt, gate, up, M, N, K, act));
  GQ_CHECK(gq_dtype_valid(x_dtype) && gq_dtype_valid(h_dtype), GQ_ERR_UNSUPPORTED);
  if (M == 0 || N == 0) return GQ_OK;
  GQ_CHECK(x && h && K > 0, GQ_ERR_INVALID_ARGS);
  GQ_CHECK(N * 128 * gq_dtype_size(h_dtype) < ((size_t)1 << 31), GQ_ERR_INVALID_ARGS);  // (a tile's rows of outputs)
  hipStream_t s = (hipStream_t)stream;
  if (front_px(fmt, M, K))
    return launch_front_px(fmt, gate, up, x, x_dtype, h, g, u, h_dtype, (int)M, (int)N, (int)K, act, s);
  if (front_as_it_is(x, x_dtype, M))
    return launch_front_few(fmt, gate, up, x, x_dtype, nullptr, h, g, u, h_dtype, (int)M, (int)N, (int)K, act, s);
  const size_t need = gq_ffn_gate_up_workspace_bytes(fmt, M, N, K), mb = front_rows(fmt, M, K), Kp = gq_kpad(fmt, K);
  GqScratch sc(ws ? 0 : need, s);
  if (ws) GQ_CHECK(ws_bytes >= need, GQ_ERR_WORKSPACE);
  else ws = sc.ptr;
  GQ_CHECK(ws, GQ_ERR_WORKSPACE);
  GQ_CHECK(((uintptr_t)ws & 15) == 0, GQ_ERR_INVALID_ARGS);
  _Float16 *a16 = (_Float16 *)ws;
  float *rs = (float *)((uint8_t *)ws + gq_align256(mb * (Kp + 8) * 2));
  const int q4 = fmt == GQ_FMT_Q4_0 || gq_fmt_is_q4k(fmt);
  if (M <= kFewRows) {  // (x in fp32, or at an odd address)
    GQ_TRY(gq_launch_a_to_f16(x, x_dtype, a16, rs, (int)M, (int)K, (int)K, 0, s));
    return launch_front_few(fmt, gate, up, a16, GQ_DT_F16, rs, h, g, u, h_dtype, (int)M, (int)N, (int)K, act, s);
  }
  if (M <= 16 || (M <= kOneBlock && gq_tiles(N) <= 400)) {  // rows 16 bytes longer than a multiple of 4 KiB, where 16 of them would collide
    const int ld = (int)Kp + 8;
    GQ_TRY(gq_launch_a_to_f16(x, x_dtype, a16, rs, (int)M, (int)K, ld, q4, s));
    return launch_front_rows(fmt, gate, up, a16, ld, rs, h, g, u, h_dtype, (int)M, (int)N, (int)K, act, s);
  }
  const size_t xs = gq_dtype_size(x_dtype) * K, hs = gq_dtype_size(h_dtype) * N;
  for (size_t m0 = 0; m0 < M; m0 += mb) {
    const int m = (int)(M - m0 < mb ? M - m0 : mb);
    GQ_TRY(gq_launch_a_to_f16((const uint8_t *)x + m0 * xs, x_dtype, a16, rs, m, (int)K, (int)Kp, q4, s));
    auto at = [&](void *p) { return p ? (void *)((uint8_t *)p + m0 * hs) : nullptr; };
    GQ_TRY(launch_front(fmt, gate, up, a16, (int)Kp, rs, at(h), at(g), at(u), h_dtype, m, (int)N, (int)K, act, s));
  }
  return GQ_OK;
}

// The plan of sums over the weights' rows: rows at a time, the kernel's shape and the parts of the sum over n (gq_internal.h)
namespace {
struct DxShape {
  int bm, bn, kg;
  size_t rows;  // the largest block it is taken for
};
// (Q4_K, K = 4096: 128 x 14336 by the second shape 73.4 us, the third 94.5; 128 x 5003 41.4 and 54.8)
constexpr DxShape kDxShapes[3] = {{32, 128, 4, 32}, {64, 128, 4, 128}, {128, 256, 2, ~(size_t)0}};

size_t dx_tiles(const DxShape &t, size_t rows, size_t K) {
  return ((rows + t.bm - 1) / t.bm) * ((K + t.bn - 1) / t.bn);
}
GqDxPlan dx_plan(size_t M, size_t N, size_t K, int mats) {
  GqDxPlan p;
  p.mats = mats;
  p.np = (gq_tiles(N) * 16 + 63) & ~(size_t)63;
  // A below 120 MiB (what a scratch block holds with the rest), whole tiles of rows where they fit
  const size_t fit = ((size_t)120 << 20) / (2 * mats * p.np);  // (np <= 2^24: at least 1)
  p.mb = fit < 256 ? fit : fit & ~(size_t)255;
  if (M < p.mb) p.mb = M;
  const size_t nsteps = mats * p.np / 64;
  p.shape = 0;
  while (p.mb > kDxShapes[p.shape].rows) ++p.shape;
  // One matrix has half the steps to go round: the second shape also where it gives no more than a workgroup a CU (us by the second / the
  // third: 512 rows, 4096 x 4096 Q8_0 40.6 / 49.7; 203, 5003 x 4096 Q6_K 43.4 / 44.8; 256, 4096 x 14336 Q4_K 69.6 / 63.6)
  if (mats == 1 && p.shape == 2 && dx_tiles(kDxShapes[1], p.mb, K) <= 256) p.shape = 1;
  const DxShape &t = kDxShapes[p.shape];
  const size_t wgs = dx_tiles(t, p.mb, K);
  size_t want = wgs >= 192 ? 1 : 256 / wgs;
  const size_t most = nsteps / (4 * t.kg);  // at least four steps a group
  if (want > most) want = most < 1 ? 1 : most;
  p.sps = (int)((nsteps + want - 1) / want);
  p.parts = (int)((nsteps + p.sps - 1) / p.sps);
  // all of it below what one scratch block holds
  const size_t held = gq_align256(p.mb * 2 * mats * p.np) + gq_align256((p.mb + 256) * 4);
  while (p.parts > 1 && held + (size_t)p.parts * p.mb * K * 4 + 256 > kGqScratchMax) {
    p.sps = (int)((nsteps + p.parts - 2) / (p.parts - 1));
    p.parts = (int)((nsteps + p.sps - 1) / p.sps);
  }
  return p;
}
size_t dx_a_bytes(const GqDxPlan &p) { return gq_align256(p.mb * p.mats * p.np * 2); }
size_t dx_rs_bytes(const GqDxPlan &p) { return gq_align256((p.mb + 256) * 4); }
size_t dx_bytes(const GqDxPlan &p, size_t K) {
  return dx_a_bytes(p) + dx_rs_bytes(p) + (p.parts > 1 ? gq_align256((size_t)p.parts * p.mb * K * 4) : 0);
}

// No less than dx_bytes of any call of at most M rows, and never less for more rows (a call of fewer rows
// may have more parts, so its own bytes may be more than M's).  A plan with parts has at most 256 / workgroups of
// them, so parts * (rows, up to whole tiles) * (columns, up to whole tiles) <= 256 tiles; it has them only
// while its workgroups are at most 128.
size_t dx_most_bytes(size_t M, size_t N, size_t K, int mats) {
  const GqDxPlan p = dx_plan(M, N, K, mats);
  size_t most = dx_a_bytes(p) + dx_rs_bytes(p);  // (of the block of most rows)
  const size_t nsteps = mats * p.np / 64;
  for (int i = 0; i <= p.shape; ++i) {
    const DxShape &t = kDxShapes[i];
    const size_t tk = (K + t.bn - 1) / t.bn, tiles = 128 / tk, parts = std::min(nsteps / (4 * t.kg), 256 / tk);
    GqDxPlan q = p;  // the most rows of this shape that have parts
    q.mb = std::min({p.mb, mats == 1 && i == 1 ? p.mb : t.rows, tiles * t.bm});
    if (q.mb <= (i ? kDxShapes[i - 1].rows : 0) || parts < 2) continue;
    const size_t sums = std::min((size_t)256 * t.bm * t.bn, parts * q.mb * K);
    // (dx_plan keeps plans with parts below kGqScratchMax)
    most = std::max(most, std::min(dx_a_bytes(q) + dx_rs_bytes(q) + gq_align256(4 * sums), kGqScratchMax));
  }
  return most;
}

template <int FMT, int WN, int KG, int TM, int PD>
int launch_dx_t(const GqDxPlan &p, const void *wg, const void *wu, const _Float16 *a16, const float *rs, void *y, int dt, int M,
                size_t N, size_t K, hipStream_t s) {
  const int tiles_m = (M + 32 * TM - 1) / (32 * TM), tiles_k = (int)((K + 128 * WN - 1) / (128 * WN));
  GQ_CHECK((size_t)tiles_m * (size_t)tiles_k <= 0x7FFFFFFFu, GQ_ERR_INVALID_ARGS);  // (one grid dimension)
  hipLaunchKernelGGL((k_front_dx<FMT, WN, KG, TM, PD>), dim3((unsigned)(tiles_m * tiles_k), (unsigned)p.parts),
                     dim3(64 * WN * KG), 0, s, (const uint8_t *)wg, (const uint8_t *)wu,
                     (uint32_t)gq_packed_bytes(FMT, N, K), (uint32_t)gq_sc_plane_offset(FMT, N, K), a16, rs, y, dt, M, (int)K,
                     (int)gq_chunks(FMT, K), (int)gq_tiles(N), (int)(p.mats * p.np / 64),
                     (int)(p.np / 64), p.sps, tiles_m);
  return gq_last_launch();
}
template <int FMT>
int launch_dx(const GqDxPlan &p, const void *wg, const void *wu, const _Float16 *a16, const float *rs, void *y, int dt, int M,
              size_t N, size_t K, hipStream_t s) {
#define GQ_DX(...) launch_dx_t<FMT, __VA_ARGS__>(p, wg, wu, a16, rs, y, dt, M, N, K, s)
  switch (p.shape) {
  case 0: return GQ_DX(1, 4, 1, 3);
  case 1: return GQ_DX(1, 4, 2, FMT == GQ_FMT_Q8_0 || FMT == GQ_FMT_Q6_K ? 2 : 3);
  default: return GQ_DX(2, 2, 4, FMT == GQ_FMT_Q8_0 || FMT == GQ_FMT_Q6_K ? 2 : 3);
  }
#undef GQ_DX
}
int launch_dx_sum(const float *part, const float *rs, void *y, int dt, size_t M, size_t K, int parts, const GqColSums &db, hipStream_t s) {
  const size_t mk = M * K, wgs = (mk / 4 + 255) / 256 + (size_t)(db.n + 15) / 16;
  GQ_CHECK(wgs <= 0x7FFFFFFFu, GQ_ERR_INVALID_ARGS);  // (one grid dimension)
  hipLaunchKernelGGL(k_dx_sum, dim3((unsigned)wgs), dim3(256), 0, s, part, rs, y, dt, mk, (int)K, parts, db);
  return gq_last_launch();
}
template <int DT>
int launch_dgu(const void *dh, const void *g, const void *u, void *dg, void *du, _Float16 *a16, float *rs, int M, int N, int np,
               int act, hipStream_t s) {
  hipLaunchKernelGGL(k_front_dgu<DT>, dim3((unsigned)M), dim3(kDguThreads), 0, s, dh, g, u, dg, du, a16, rs, N, np, act);
  return gq_last_launch();
}
}  // namespace

GqDxPlan gq_dx_plan(size_t M, size_t N, size_t K, int mats) { return dx_plan(M, N, K, mats); }
size_t gq_dx_a_bytes(const GqDxPlan &p) { return dx_a_bytes(p); }
size_t gq_dx_rs_bytes(const GqDxPlan &p) { return dx_rs_bytes(p); }
size_t gq_dx_bytes(const GqDxPlan &p, size_t K) { return dx_bytes(p, K); }
size_t gq_dx_most_bytes(size_t M, size_t N, size_t K, int mats) { return dx_most_bytes(M, N, K, mats); }
int gq_launch_dx(int fmt, const GqDxPlan &p, const void *w0, const void *w1, const _Float16 *a16, const float *rs, float *part,
                 void *y, int dt, int M, size_t N, size_t K, const GqColSums &db, hipStream_t s) {
  void *to = p.parts > 1 ? (void *)part : y;
  if (fmt == GQ_FMT_Q4_0) GQ_TRY(launch_dx<GQ_FMT_Q4_0>(p, w0, w1, a16, rs, to, dt, M, N, K, s));
  else if (fmt == GQ_FMT_Q8_0) GQ_TRY(launch_dx<GQ_FMT_Q8_0>(p, w0, w1, a16, rs, to, dt, M, N, K, s));
  else if (gq_fmt_is_q6k(fmt)) GQ_TRY(launch_dx<GQ_FMT_Q6_K>(p, w0, w1, a16, rs, to, dt, M, N, K, s));
  else GQ_TRY(launch_dx<GQ_FMT_Q4_K>(p, w0, w1, a16, rs, to, dt, M, N, K, s));
  return p.parts > 1 ? launch_dx_sum(part, rs, y, dt, (size_t)M, K, p.parts, db, s) : GQ_OK;
}
int gq_launch_zeros(void *y, int dt, size_t M, size_t K, hipStream_t s) {
  return launch_dx_sum(nullptr, nullptr, y, dt, M, K, 0, GqColSums{}, s);
}

extern "C" size_t gq_ffn_gate_up_bwd_workspace_bytes(int fmt, size_t M, size_t N, size_t K) {
  if (!gq_fmt_valid(fmt) || M > GQ_MAX_DIM || N > GQ_MAX_DIM || K > GQ_MAX_DIM || M == 0 || N == 0 || K == 0) return 0;
  return dx_most_bytes(M, N, K, 2);
}

extern "C" int gq_ffn_gate_up_bwd(int fmt, const void *gate, const void *up, const void *dh, const void *g,
                                  const void *u, int dtype, void *dg, void *du, void *dx, int dx_dtype, size_t M,
                                  size_t N, size_t K, int act, void *ws, size_t ws_bytes, void *stream) {
  GQ_TRY(check_front(fmt, gate, up, M, N, K, act));
  GQ_CHECK(gq_dtype_valid(dtype) && gq_dtype_valid(dx_dtype), GQ_ERR_UNSUPPORTED);
  if (M == 0 || (!dg && !du && !dx)) return GQ_OK;
  GQ_CHECK(K > 0, GQ_ERR_INVALID_ARGS);
  hipStream_t s = (hipStream_t)stream;
  if (N == 0) return dx ? launch_dx_sum(nullptr, nullptr, dx, dx_dtype, M, K, 0, GqColSums{}, s) : GQ_OK;  // (sums of nothing)
  GQ_CHECK(dh && g && u, GQ_ERR_INVALID_ARGS);
  const GqDxPlan plan = dx_plan(M, N, K, 2);
  const size_t need = dx ? gq_ffn_gate_up_bwd_workspace_bytes(fmt, M, N, K) : 0;
  GqScratch sc(ws || !dx ? 0 : dx_bytes(plan, K), s);
  if (ws) GQ_CHECK(ws_bytes >= need, GQ_ERR_WORKSPACE);
  else ws = sc.ptr;
  GQ_CHECK(ws || !dx, GQ_ERR_WORKSPACE);
  GQ_CHECK(((uintptr_t)ws & 15) == 0, GQ_ERR_INVALID_ARGS);
  _Float16 *a16 = dx ? (_Float16 *)ws : nullptr;
  float *rs = dx ? (float *)((uint8_t *)ws + dx_a_bytes(plan)) : nullptr;
  float *part = dx ? (float *)((uint8_t *)rs + dx_rs_bytes(plan)) : nullptr;
  const size_t es = gq_dtype_size(dtype) * N, xs = gq_dtype_size(dx_dtype) * K;
  const size_t step = dx ? plan.mb : (size_t)1 << 20;
  for (size_t m0 = 0; m0 < M; m0 += step) {
    const int m = (int)(M - m0 < step ? M - m0 : step);
    auto at = [&](const void *p) { return p ? (void *)((uint8_t *)p + m0 * es) : nullptr; };
    if (dtype == GQ_DT_F32) GQ_TRY(launch_dgu<GQ_DT_F32>(at(dh), at(g), at(u), at(dg), at(du), a16, rs, m, (int)N, (int)plan.np, act, s));
    else if (dtype == GQ_DT_F16) GQ_TRY(launch_dgu<GQ_DT_F16>(at(dh), at(g), at(u), at(dg), at(du), a16, rs, m, (int)N, (int)plan.np, act, s));
    else GQ_TRY(launch_dgu<GQ_DT_BF16>(at(dh), at(g), at(u), at(dg), at(du), a16, rs, m, (int)N, (int)plan.np, act, s));
    if (!dx) continue;
    GQ_TRY(gq_launch_dx(fmt, plan, gate, up, a16, rs, part, (uint8_t *)dx + m0 * xs, dx_dtype, m, N, K, GqColSums{}, s));
  }
  return GQ_OK;
}
