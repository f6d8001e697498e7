// gq_moe.hip -- the mixture-of-experts layer of a few tokens over T16 expert tensors: router, choice of experts, their gated
// feed-forward products and the weighted sum.
//
//   l[m][e] = sum_k x[m][k] Wr[e][k]                    k_moe_logits, in 64 bits: which of two experts is larger decides the layer
//   S_m, w_me                                           k_moe_plan: the choice, and the list of each expert's tokens
//   h_me = act(Wg_e x_m) * (Wu_e x_m)                   k_moe_gu_*: one row of h a (token, expert) pair
//   y_m = r_m + sum over S_m of w_me Wd_e h_me          k_moe_down_*: a workgroup adds its 16 columns over all experts
//
// The weights of the experts taken bound all of it; each is read once for up to 16 of its tokens.
#include <algorithm>
#include <type_traits>

#include "gq_internal.h"
#include "gq_rows_frag.h"

namespace {

constexpr int kMoeFew = 4;  // tokens that the kernels of few rows take

// A block of an expert's work: up to 16 of its pairs (token * top + slot); few tokens (M <= 4): pair[m] is token m's, -1 none,
// and w[m] its weight.  expert -1: no block.
struct MoeBlk {
  int expert, count;
  int pair[16];
  float w[kMoeFew];
};
struct MoePlan {
  int *nblk;
  MoeBlk *blk;  // [maxblk], the blocks that there are first
  float *wsum;  // [pair] the weight (of the first pair of an expert that a token names twice: their sum); not for few tokens
  int maxblk;
};

// ---- router --------------------------------------------------------------------------
// Workgroup (e, b): logits of expert e for tokens TOK b .. TOK b + TOK - 1.  Products of two fp32 values are exact in 64 bits.
constexpr int kLogThreads = 256;
template <int XT, int RT, int TOK>
__global__ void __launch_bounds__(kLogThreads) k_moe_logits(const void *__restrict__ x, const void *__restrict__ wr,
                                                            double *__restrict__ logits, int M, int E, int K) {
  __shared__ double red[kLogThreads / 64][TOK];
  const int tid = threadIdx.x, e = blockIdx.x, m0 = TOK * (int)blockIdx.y;
  double acc[TOK] = {};
#pragma unroll 2
  for (int k = 8 * tid; k < K; k += 8 * kLogThreads) {  // (K is whole 8s)
    FRaw<RT> wv;
    FRaw<XT> xv[TOK];
    px_load<RT>(wr, (size_t)e * K + k, wv);
#pragma unroll
    for (int t = 0; t < TOK; ++t) px_load<XT>(x, (size_t)(m0 + t < M ? m0 + t : M - 1) * K + k, xv[t]);
    float wf[8], xf[8];
    px_floats<RT>(wv, true, wf);
#pragma unroll
    for (int t = 0; t < TOK; ++t) {
      px_floats<XT>(xv[t], true, xf);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[t] = fma((double)wf[i], (double)xf[i], acc[t]);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
#pragma unroll
    for (int t = 0; t < TOK; ++t) acc[t] += __shfl_xor(acc[t], o, 64);
  if ((tid & 63) == 0)
#pragma unroll
    for (int t = 0; t < TOK; ++t) red[tid >> 6][t] = acc[t];
  __syncthreads();
  if (tid < TOK && m0 + tid < M) {
    double v = 0.0;
#pragma unroll
    for (int w = 0; w < kLogThreads / 64; ++w) v += red[w][tid];
    logits[(size_t)(m0 + tid) * E + e] = v;
  }
}

struct RouteArgs {
  const double *logits;
  const float *bias;
  int *ids;
  float *weights;
  int score, renorm;
  float scale;
};
// The largest of a wave's values, in all lanes
GQ_DEV uint32_t wave_max(uint32_t v) {
#define GQ_DPP_MAX(CTRL, ROWS) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false))
  GQ_DPP_MAX(0x111, 0xF);  // row_shr 1, 2, 4, 8: lane 15 of each row has its largest
  GQ_DPP_MAX(0x112, 0xF);
  GQ_DPP_MAX(0x114, 0xF);
  GQ_DPP_MAX(0x118, 0xF);
  GQ_DPP_MAX(0x142, 0xA);  // row_bcast 15, 31: lane 63 the wave's
  GQ_DPP_MAX(0x143, 0xC);
#undef GQ_DPP_MAX
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
GQ_DEV double lane_d(double v, int lane) {  // (lane: the same in all lanes)
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// One wave chooses the experts of token m; lane j writes slot j.  A key is a 64-bit number in the values' order, 0 what is
// never taken (-Inf, none there, taken before): the largest's high word, then its low word, then the lowest
// expert that has both.
template <int NE>
GQ_DEV void moe_choose(const RouteArgs &a, int m, int E, int top, int lane, int *ids_s, float *w_s) {
  const double ninf = -__builtin_inf();
  const bool sm = a.score == GQ_MOE_SOFTMAX;
  double l[NE], lmax = ninf, sum = 0.0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = 64 * i + lane;
    l[i] = e < E ? a.logits[(size_t)m * E + e] : ninf;
    lmax = fmax(lmax, l[i]);  // (of those that are numbers)
  }
  if (sm) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lmax = fmax(lmax, __shfl_xor(lmax, o, 64));
    if (!a.renorm || a.bias) {  // (renormalised weights do without the sum over all experts)
#pragma unroll
      for (int i = 0; i < NE; ++i) sum += l[i] == ninf ? 0.0 : exp(l[i] - lmax);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    } else {
      sum = 1.0;
    }
  }
  auto score = [&](double v) { return sm ? (v == ninf ? 0.0 : exp(v - lmax) / sum) : 1.0 / (1.0 + exp(-v)); };
  uint32_t kh[NE], kl[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = 64 * i + lane;
    double key = l[i];
    if (a.bias && e < E) key = score(l[i]) + (double)a.bias[e];
    if (key != key) key = __builtin_inf();
    const uint64_t b = __builtin_bit_cast(uint64_t, key);
    const uint64_t o = e >= E || key == ninf ? 0 : b >> 63 ? ~b : b | (uint64_t)1 << 63;
    kh[i] = (uint32_t)(o >> 32);
    kl[i] = (uint32_t)o;
  }
  double mine = ninf;  // lane j: the logit of slot j
  int id = -1;
  for (int j = 0; j < top; ++j) {
    uint32_t h = 0, w = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) h = max(h, kh[i]);
    const uint32_t mh = wave_max(h);
    if (mh == 0) break;
#pragma unroll
    for (int i = 0; i < NE; ++i) w = max(w, kh[i] == mh ? kl[i] : 0u);
    const uint32_t mw = wave_max(w);
    bool found = false;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const uint64_t at = found ? 0 : __ballot(kh[i] == mh && kl[i] == mw);
      if (at == 0) continue;
      found = true;
      const int ln = __builtin_ctzll(at);
      const double v = lane_d(l[i], ln);
      if (lane == ln) kh[i] = kl[i] = 0;
      if (lane == j) {
        id = 64 * i + ln;
        mine = v;
      }
    }
  }
  double w = id < 0 ? 0.0 : score(mine), total = 0.0;
  if (a.renorm) {
    for (int j = 0; j < top; ++j) total += lane_d(w, j);
    w = total == 0.0 ? 0.0 : w / total;
  }
  if (lane < top) {
    const float f = id < 0 ? 0.f : (float)(w * (double)a.scale);
    ids_s[m * top + lane] = id;
    w_s[m * top + lane] = f;
    if (a.ids) a.ids[m * top + lane] = id;
    if (a.weights) a.weights[m * top + lane] = f;
  }
}

// ---- plan: one workgroup ------------------------------------------------------------
// The choice (NE: experts a lane; 0: ids and weights are given), each expert's pairs in order of their tokens, in blocks of `per`.
// Ids outside 0 .. E - 1 name no expert; an expert that a token names twice gets one pair with both weights.
constexpr int kPlanThreads = 1024;
template <int NE>
__global__ void __launch_bounds__(kPlanThreads) k_moe_plan(RouteArgs a, const int *__restrict__ ids, const float *__restrict__ weights,
                                                           MoePlan p, int M, int E, int top, int per) {
  constexpr int MP = GQ_MOE_MAX_TOKENS * GQ_MOE_MAX_TOP, FB = kMoeFew * GQ_MOE_MAX_TOP;
  static_assert(MP <= kPlanThreads && GQ_MOE_MAX_EXPERTS <= kPlanThreads, "a thread a pair, a thread an expert");
  __shared__ int id_s[MP], base_s[kPlanThreads], tot_s[kPlanThreads / 64], pair_s[FB][kMoeFew];
  __shared__ uint32_t tok_s[2][kPlanThreads];  // the tokens of an expert, a bit each
  __shared__ float w_s[MP], wsum_s[FB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = M * top;
  const bool few = M <= kMoeFew;
  tok_s[0][tid] = tok_s[1][tid] = 0;
  if (tid < FB * kMoeFew) pair_s[tid / kMoeFew][tid % kMoeFew] = -1;
  if constexpr (NE > 0) {
    for (int m = wave; m < M; m += kPlanThreads / 64) moe_choose<NE>(a, m, E, top, lane, id_s, w_s);
  } else if (tid < P) {
    id_s[tid] = ids[tid];
    w_s[tid] = weights[tid];
  }
  if (!p.blk) return;  // (the choice alone)
  __syncthreads();
  const int tok = tid / top;
  int id = -1;
  if (tid < P) {
    id = id_s[tid];
    if (id < 0 || id >= E) id = -1;
    float w = w_s[tid];
    if constexpr (NE == 0) {
      w = 0.f;
      for (int j = tok * top; j < tok * top + top; ++j) {
        if (id_s[j] != id) continue;
        if (j < tid) id = -1;  // (the first pair's)
        else w += w_s[j];
      }
    }
    if (few) wsum_s[tid] = w;
    else p.wsum[tid] = w;
    if (id >= 0) atomicOr(&tok_s[tok >> 5][id], 1u << (tok & 31));
  }
  __syncthreads();
  const int c = __popc(tok_s[0][tid]) + __popc(tok_s[1][tid]), nb = (c + per - 1) / per;
  int inc = nb;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(inc, o, 64);
    if (lane >= o) inc += v;
  }
  if (lane == 63) tot_s[wave] = inc;
  __syncthreads();
  int base = inc - nb, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    const int v = tot_s[w];
    if (w < wave) base += v;
    all += v;
  }
  base_s[tid] = base;
  for (int b = 0; b < nb; ++b) {
    p.blk[base + b].expert = tid;
    p.blk[base + b].count = c - per * b < per ? c - per * b : per;
  }
  for (int b = all + tid; b < p.maxblk; b += kPlanThreads) p.blk[b].expert = -1;
  if (tid == 0) *p.nblk = all;
  __syncthreads();
  if (id >= 0) {
    const uint32_t below = (1u << (tok & 31)) - 1u, w0 = tok_s[0][id], w1 = tok_s[1][id];
    const int rank = tok < 32 ? __popc(w0 & below) : __popc(w0) + __popc(w1 & below);
    if (few) pair_s[base_s[id]][tok] = tid;
    else p.blk[base_s[id] + rank / per].pair[rank % per] = tid;
  }
  if (!few) return;
  __syncthreads();
  if (tid < all * kMoeFew) {
    const int b = tid / kMoeFew, m = tid % kMoeFew, q = pair_s[b][m];
    p.blk[b].pair[m] = q;
    p.blk[b].w[m] = q < 0 ? 0.f : wsum_s[q];
  }
}

// ---- gate and up -----------------------------------------------------------------------
template <int KS, int R, int MR, typename At>
GQ_DEV void moe_gu_out(At at, float *__restrict__ h, int N, int act, int group, int rows, const int *pair, const float *rs, int top) {
  for (int o = threadIdx.x; o < 16 * R * rows; o += 64 * KS) {
    const int nl = o % (16 * R), m = o / (16 * R), n = 16 * R * group + nl, p = pair[m];
    if (n >= N || p < 0) continue;
    float y[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int k = 0; k < KS; ++k) y[w] += at(k, w, nl >> 4, nl & 15, m);
    const float f = rs ? rs[p / top] : 1.f, g = y[0] * f, u = y[1] * f;
    h[(size_t)p * N + n] = gq_act_f(act, g) * u;
  }
}

// Up to 4 tokens of 16-bit x: codes and x as they are, scales in fp32 (gq_rows_frag.h); row j is token j.
template <int FMT, int XT, int MR, int R, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_moe_gu_few(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off, const void *__restrict__ x,
             const float *__restrict__ rs, MoePlan p, float *__restrict__ h, int M, int N, int K, int C, int units, int act, int top) {
  constexpr int NG = kFewGroups<FMT>, T = 2 * R;
  constexpr float OFF = kFewOff<FMT, XT>;
  __shared__ float red[KS][T][MR][64];
  const MoeBlk &blk = p.blk[blockIdx.y];
  const int expert = __builtin_amdgcn_readfirstlane(blk.expert);
  if (expert < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, ntiles = N / 16;
  const size_t tile0 = (size_t)expert * (size_t)ntiles;
  FTile<FMT> tl[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int tile = (int)blockIdx.x * R + t % R;
    tl[t] = ftile<FMT>(t < R ? wg : wu, sc_off, tile0 + (size_t)(tile < ntiles ? tile : ntiles - 1), C);  // (clamped: not stored)
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
  moe_gu_out<KS, R, MR>(
      [&](int k, int w, int t, int n, int m) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) y += red[k][w * R + t][MR == 1 ? 0 : m][16 * i + n];
        return y;
      },
      h, N, act, (int)blockIdx.x, M, blk.pair, rs, top);
}

// More tokens: a block's rows are its pairs, fp16 rows of x gathered, the scale groups folded into the weights.
template <int FMT, int R, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_moe_gu_rows(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off, const _Float16 *__restrict__ a16,
              int lda, const float *__restrict__ rs, MoePlan p, float *__restrict__ h, int M, int N, int C, int units, int act,
              int top) {
  constexpr int T = 2 * R;
  __shared__ gq_f4 red[KS][T][64];
  const MoeBlk &blk = p.blk[blockIdx.y];
  const int expert = __builtin_amdgcn_readfirstlane(blk.expert);
  if (expert < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15, ntiles = N / 16;
  const size_t tile0 = (size_t)expert * (size_t)ntiles;
  FTile<FMT> tl[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int tile = (int)blockIdx.x * R + t % R;
    tl[t] = ftile<FMT>(t < R ? wg : wu, sc_off, tile0 + (size_t)(tile < ntiles ? tile : ntiles - 1), C);  // (clamped: not stored)
  }
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<_Float16 *>(a16), (short)0, (int)(2u * (uint32_t)M * (uint32_t)lda), 0x00020000);
  const bool row = r < blk.count;
  const uint32_t xo = row ? 2u * ((uint32_t)(blk.pair[r] / top) * (uint32_t)lda + 16u * (uint32_t)g) : 0u;
  FUnit<FMT> us[PD][T];
  gq_half8 xs[PD][1][4];
  auto request = [&](int unit, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < T; ++t) load_unit<FMT>(tl[t], unit, lane, us[st][t]);
    const uint32_t o = row && unit < units ? xo + 256u * (uint32_t)unit : 0xFFFFFF00u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(xr, o + 128u * (i >> 1) + 16u * (i & 1), 0, 0);
      xs[st][0][i] = __builtin_bit_cast(gq_half8, gq_u4{v[0], v[1], v[2], v[3]});
    }
  };
  gq_f4 acc[T][1];
#pragma unroll
  for (int t = 0; t < T; ++t) acc[t][0] = gq_f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t mg = gq_nib_magic();
  auto compute = [&](int unit, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < T; ++t) rows_add<FMT, 1>(us[st][t], unit, g, mg, xs[st], acc[t]);
  };
  walk_units<PD, KS>(units, wave, request, compute);
#pragma unroll
  for (int t = 0; t < T; ++t) red[wave][t][lane] = acc[t][0];
  __syncthreads();
  moe_gu_out<KS, R, 4>(
      [&](int k, int w, int t, int n, int m) {
        return reinterpret_cast<const float *>(&red[k][w * R + t][16 * (m >> 2) + n])[m & 3];
      },
      h, N, act, (int)blockIdx.x, blk.count, blk.pair, rs, top);
}

// ---- down ------------------------------------------------------------------------------
// A workgroup owns a row tile of every expert's W_down (16 columns of y); its KS waves take the units of all blocks in turn
// (block by block, unit by unit), so that the sum over a token's experts stays in the workgroup, in one order.
struct ItemAt {
  int b, u;
  __device__ __forceinline__ void next(int by, int units) {
    u += by;
    while (u >= units) {
      u -= units;
      ++b;
    }
  }
};
template <int PD, int KS, typename Request, typename Compute>
GQ_DEV void walk_items(int nblk, int units, int wave, Request request, Compute compute) {
  ItemAt rq = {0, 0}, at = {0, 0};
  rq.next(wave, units);
  at = rq;
#pragma unroll
  for (int i = 0; i < PD; ++i) {
    request(rq, i);
    rq.next(KS, units);
  }
  while (at.b < nblk) {
#pragma unroll
    for (int i = 0; i < PD; ++i) {
      if (at.b >= nblk) break;
      compute(at, i);
      at.next(KS, units);
      request(rq, i);
      rq.next(KS, units);
    }
  }
}

// Up to 4 tokens: rows are the tokens, h comes in fp32 and is rounded to fp16 after a power-of-two scale per row and unit; the
// scale's inverse and the expert's weight go onto the unit's fp32 sums.
template <int FMT, int MR, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_moe_down_few(const uint8_t *__restrict__ wd, size_t sc_off, const float *__restrict__ h, MoePlan p, const void *resid, void *y,
               int dt, int M, int N, int K, int C, int units, int top) {
  constexpr int NG = kFewGroups<FMT>, XT = GQ_DT_F16, MB = kMoeFew * GQ_MOE_MAX_TOP;
  constexpr float OFF = kFewOff<FMT, XT>;
  __shared__ float red[KS][MR][64];
  __shared__ int e_s[MB], p_s[MB][kMoeFew];
  __shared__ float w_s[MB][kMoeFew];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, ntiles = K / 16;
  const int nblk = __builtin_amdgcn_readfirstlane(*p.nblk);
  if (tid < p.maxblk) {  // (not nblk, which would have to arrive first)
    e_s[tid] = p.blk[tid].expert;
#pragma unroll
    for (int m = 0; m < kMoeFew; ++m) {
      p_s[tid][m] = p.blk[tid].pair[m];
      w_s[tid][m] = p.blk[tid].w[m];
    }
  }
  __syncthreads();
  const __amdgpu_buffer_rsrc_t hr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<float *>(h), (short)0, (int)(4u * (uint32_t)(M * top) * (uint32_t)N), 0x00020000);
  const int xrow = lane & 3, xk = 64 * ((lane >> 3) & 1) + 16 * g + 8 * ((lane >> 2) & 1);
  FUnit<FMT> us[PD];
  gq_f4 xs[PD][2];
  auto request = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
    const bool on = at.b < nblk;
    const int b = on ? at.b : 0;
    const size_t tile = (size_t)__builtin_amdgcn_readfirstlane(e_s[b]) * (size_t)ntiles + blockIdx.x;
    load_unit<FMT>(ftile<FMT>(wd, sc_off, tile, on ? C : 0), at.u, lane, us[st]);
    const int q = p_s[b][xrow], k = 128 * at.u + xk;  // (N is whole 32-blocks: a run is wholly in or out)
    const uint32_t o = on && q >= 0 && k < N ? 4u * ((uint32_t)q * (uint32_t)N + (uint32_t)k) : 0xFFFFFFE0u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(hr, o + 16u * i, 0, 0);
      xs[st][i] = __builtin_bit_cast(gq_f4, v);
    }
  };
  float acc[MR] = {};
  uint32_t mg;  // (kept in a register)
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(mg));
  const gq_u4 ones = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
  const gq_f4 zero = {0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
    float v[8], t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = xs[st][i >> 2][i & 3];
      t = fmaxf(t, fabsf(v[i]));
    }
#pragma unroll
    for (int o = 4; o < 64; o <<= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
    // 2^s, s = 14 - floor(log2(t)) at most 126 (at least -114: both have a normal inverse)
    const int sh = 14 + 127 - (int)((__float_as_uint(t) >> 23) & 0xFFu), cut = sh > 126 ? 126 : sh;
    const float f2 = __uint_as_float((uint32_t)(127 + cut) << 23), inv = __uint_as_float((uint32_t)(127 - cut) << 23);
    gq_u4 xv;
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = gq_h2_bits(gq_half2{(_Float16)(v[2 * i] * f2), (_Float16)(v[2 * i + 1] * f2)});
    if (kNibOrder<FMT>) xv = nib_order(xv);
    float s[2], mn[2], sum[MR] = {};
    few_scales<FMT>(us[st], at.u, g & (NG - 1), s, mn);
    auto step = [&](auto mc) __attribute__((always_inline)) {
      constexpr int m = decltype(mc)::value;
      const gq_u4 a0 = few_operand<NG, 2 * m>(xv), a1 = few_operand<NG, 2 * m + 1>(xv);
      const gq_f4 sx = few_mfma<XT>(a1, ones, few_mfma<XT>(a0, ones, zero));
      gq_u4 b[2];
      few_codes<FMT, XT>(us[st], m, mg, b);
      const gq_f4 d = few_mfma<XT>(a1, b[1], few_mfma<XT>(a0, b[0], zero));
      const float o = FMT == GQ_FMT_Q4_K ? fmaf(s[m], OFF, mn[m]) : 0.f;
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        if constexpr (FMT == GQ_FMT_Q4_K) sum[r] = fmaf(s[m], d[r], fmaf(-o, sx[r], sum[r]));
        else sum[r] = fmaf(s[m], fmaf(-OFF, sx[r], d[r]), sum[r]);
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    // (each quad of lanes holds the four rows' scales)
    const float inv0 = __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(inv), 0x00, 15, 15, true));
    acc[0] = fmaf(w_s[at.b][0] * inv0, sum[0], acc[0]);
    if constexpr (MR == 4) {
      const float inv1 = __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(inv), 0x55, 15, 15, true));
      const float inv2 = __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(inv), 0xAA, 15, 15, true));
      const float inv3 = __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(inv), 0xFF, 15, 15, true));
      acc[1] = fmaf(w_s[at.b][1] * inv1, sum[1], acc[1]);
      acc[2] = fmaf(w_s[at.b][2] * inv2, sum[2], acc[2]);
      acc[3] = fmaf(w_s[at.b][3] * inv3, sum[3], acc[3]);
    }
  };
  if (nblk > 0) walk_items<PD, KS>(nblk, units, wave, request, compute);
#pragma unroll
  for (int r = 0; r < MR; ++r) red[wave][r][lane] = acc[r];
  __syncthreads();
  if (tid < 16 * M) {
    const int n = tid & 15, m = tid >> 4;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < KS; ++w)
#pragma unroll
      for (int i = 0; i < NG; ++i) v += red[w][MR == 1 ? 0 : m][16 * i + n];
    const size_t o = (size_t)m * K + 16 * blockIdx.x + n;
    if (resid) v += gq_ld_dt(resid, dt, o);
    gq_st_dt(y, dt, o, v);
  }
}

// More tokens: a block's rows are its pairs (fp16 rows of h with a power-of-two scale each); a block's sums go, with the
// scale's inverse and the expert's weight, to the wave's own sums of the tokens in LDS.
template <int FMT, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_moe_down_rows(const uint8_t *__restrict__ wd, size_t sc_off, const _Float16 *__restrict__ h16, int ldh, const float *__restrict__ hs,
                MoePlan p, const void *resid, void *y, int dt, int M, int K, int C, int units, int top, int maxblk) {
  extern __shared__ float lds[];
  const int P = M * top;
  float *sum_s = lds;                                                    // [KS][M][16]
  float *f_s = sum_s + KS * M * 16;                                      // [P]: weight and scale of a pair
  uint16_t *p_s = reinterpret_cast<uint16_t *>(f_s + P);                 // [maxblk][16]: pairs, 0xFFFF none
  uint16_t *e_s = p_s + 16 * maxblk;                                     // [maxblk]
  uint8_t *t_s = reinterpret_cast<uint8_t *>(e_s + maxblk);              // [P]: token of a pair
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15, ntiles = K / 16;
  const int nblk = __builtin_amdgcn_readfirstlane(*p.nblk);
  for (int i = tid; i < KS * M * 16; i += 64 * KS) sum_s[i] = 0.f;
  for (int i = tid; i < P; i += 64 * KS) {
    f_s[i] = p.wsum[i] * hs[i];
    t_s[i] = (uint8_t)(i / top);
  }
  for (int i = tid; i < 16 * maxblk; i += 64 * KS) {
    const MoeBlk &b = p.blk[i >> 4];
    p_s[i] = (i & 15) < b.count ? (uint16_t)b.pair[i & 15] : (uint16_t)0xFFFF;
    if ((i & 15) == 0) e_s[i >> 4] = (uint16_t)b.expert;
  }
  __syncthreads();
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<_Float16 *>(h16), (short)0, (int)(2u * (uint32_t)P * (uint32_t)ldh), 0x00020000);
  FUnit<FMT> us[PD];
  gq_half8 xs[PD][1][4];
  auto request = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
    const bool on = at.b < nblk;
    const int b = on ? at.b : 0;
    const size_t tile = (size_t)__builtin_amdgcn_readfirstlane((int)e_s[b]) * (size_t)ntiles + blockIdx.x;
    load_unit<FMT>(ftile<FMT>(wd, sc_off, tile, on ? C : 0), at.u, lane, us[st]);
    const uint32_t q = p_s[16 * b + r];
    const uint32_t o = on && q != 0xFFFFu ? 2u * (q * (uint32_t)ldh + 16u * (uint32_t)g) + 256u * (uint32_t)at.u : 0xFFFFFF00u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(xr, o + 128u * (i >> 1) + 16u * (i & 1), 0, 0);
      xs[st][0][i] = __builtin_bit_cast(gq_half8, gq_u4{v[0], v[1], v[2], v[3]});
    }
  };
  gq_f4 acc[1] = {{0.f, 0.f, 0.f, 0.f}};
  const uint32_t mg = gq_nib_magic();
  int cur = -1;
  auto flush = [&]() __attribute__((always_inline)) {
    if (cur < 0) return;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const uint32_t q = p_s[16 * cur + 4 * g + v];
      if (q != 0xFFFFu) sum_s[(wave * M + t_s[q]) * 16 + r] += f_s[q] * acc[0][v];  // (a block's tokens differ)
      acc[0][v] = 0.f;
    }
  };
  auto compute = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
    if (at.b != cur) {
      flush();
      cur = at.b;
    }
    rows_add<FMT, 1>(us[st], at.u, g, mg, xs[st], acc);
  };
  if (nblk > 0) walk_items<PD, KS>(nblk, units, wave, request, compute);
  flush();
  __syncthreads();
  for (int i = tid; i < 16 * M; i += 64 * KS) {
    const int n = i & 15, m = i >> 4;
    float v = 0.f;
    for (int w = 0; w < KS; ++w) v += sum_s[(w * M + m) * 16 + n];
    const size_t o = (size_t)m * K + 16 * blockIdx.x + n;
    if (resid) v += gq_ld_dt(resid, dt, o);
    gq_st_dt(y, dt, o, v);
  }
}

// ---- host ----------------------------------------------------------------------------
int check_moe(const gq_moe *l, size_t M, bool route, bool ffn) {
  GQ_CHECK(l, GQ_ERR_INVALID_ARGS);
  GQ_CHECK(M <= GQ_MOE_MAX_TOKENS && l->n_experts <= GQ_MOE_MAX_EXPERTS, GQ_ERR_UNSUPPORTED);
  GQ_CHECK(l->top_k >= 1 && l->top_k <= GQ_MOE_MAX_TOP, GQ_ERR_UNSUPPORTED);
  GQ_CHECK(l->n_experts > 0 && l->K > 0 && l->K <= GQ_MAX_DIM, GQ_ERR_INVALID_ARGS);
  if (route) {
    GQ_CHECK(gq_dtype_valid(l->router_dtype), GQ_ERR_UNSUPPORTED);
    GQ_CHECK(l->score == GQ_MOE_SOFTMAX || l->score == GQ_MOE_SIGMOID, GQ_ERR_UNSUPPORTED);
    GQ_CHECK((size_t)l->top_k <= l->n_experts && l->K % 8 == 0, GQ_ERR_INVALID_ARGS);
    GQ_CHECK(l->router || M == 0, GQ_ERR_INVALID_ARGS);
  }
  if (ffn) {
    GQ_CHECK(gq_fmt_valid(l->fmt) && gq_fmt_valid(l->fmt_down), GQ_ERR_UNSUPPORTED);
    GQ_CHECK(l->act == GQ_ACT_SILU || l->act == GQ_ACT_GELU_TANH, GQ_ERR_UNSUPPORTED);
    GQ_CHECK(l->N > 0 && l->N <= GQ_MAX_DIM, GQ_ERR_INVALID_ARGS);
    GQ_TRY(gq_check_shape(l->fmt, l->n_experts * l->N, l->K));
    GQ_TRY(gq_check_shape(l->fmt_down, l->n_experts * l->K, l->N));
    GQ_CHECK((l->gate && l->up && l->down) || M == 0, GQ_ERR_INVALID_ARGS);
    GQ_CHECK((((uintptr_t)l->gate | (uintptr_t)l->up | (uintptr_t)l->down) & 15) == 0, GQ_ERR_INVALID_ARGS);
    // a tile's records, and the rows of h, lie within 32-bit offsets
    GQ_CHECK(gq_chunks(l->fmt, l->K) * gq_chunk_qs_bytes(l->fmt) < ((size_t)1 << 31), GQ_ERR_INVALID_ARGS);
    GQ_CHECK(gq_chunks(l->fmt_down, l->N) * gq_chunk_qs_bytes(l->fmt_down) < ((size_t)1 << 31), GQ_ERR_INVALID_ARGS);
    GQ_CHECK((size_t)GQ_MOE_MAX_TOKENS * l->top_k * (gq_kpad(l->fmt_down, l->N) + 8) * 4 < ((size_t)1 << 32) - 4096,
             GQ_ERR_INVALID_ARGS);
  }
  return GQ_OK;
}

// Where a call's intermediate values lie in its workspace
struct MoeWs {
  size_t logits, ids, weights, nblk, blk, wsum, a16, rs, h, h16, hs, bytes;
  int maxblk;
};
MoeWs moe_ws(const gq_moe &l, size_t M) {
  MoeWs w;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at += gq_align256(n);
    return o;
  };
  const size_t P = M * (size_t)l.top_k;
  const bool few = M <= (size_t)kMoeFew;
  // (an expert's last block may be short: at most a block an expert beyond whole ones)
  w.maxblk = (int)(few ? std::min(P, l.n_experts) : std::min(P, l.n_experts + P / 16));
  w.logits = take(M * l.n_experts * 8);
  w.ids = take(P * 4);
  w.weights = take(P * 4);
  w.nblk = take(4);
  w.blk = take((size_t)w.maxblk * sizeof(MoeBlk));
  w.wsum = take(P * 4);
  w.a16 = take(M * (gq_kpad(l.fmt, l.K) + 8) * 2);
  w.rs = take((M + 256) * 4);
  w.h = take(P * l.N * 4);
  w.h16 = take(P * (gq_kpad(l.fmt_down, l.N) + 8) * 2);
  w.hs = take((P + 256) * 4);
  w.bytes = at;
  return w;
}

template <int XT, int RT>
int launch_logits_t(const gq_moe &l, const void *x, double *logits, int M, hipStream_t s) {
#define GQ_LOG(TOK)                                                                                                            \
  hipLaunchKernelGGL((k_moe_logits<XT, RT, TOK>), dim3((unsigned)l.n_experts, (unsigned)((M + (TOK)-1) / (TOK))), dim3(kLogThreads), \
                     0, s, x, l.router, logits, M, (int)l.n_experts, (int)l.K)
  if (M == 1) GQ_LOG(1);
  else GQ_LOG(4);
#undef GQ_LOG
  return gq_last_launch();
}
template <int XT>
int launch_logits_x(const gq_moe &l, const void *x, double *logits, int M, hipStream_t s) {
  if (l.router_dtype == GQ_DT_F32) return launch_logits_t<XT, GQ_DT_F32>(l, x, logits, M, s);
  if (l.router_dtype == GQ_DT_F16) return launch_logits_t<XT, GQ_DT_F16>(l, x, logits, M, s);
  return launch_logits_t<XT, GQ_DT_BF16>(l, x, logits, M, s);
}
int launch_plan(const gq_moe &l, const RouteArgs &a, const int *ids, const float *weights, const MoePlan &plan, int M,
                hipStream_t s) {
  const int E = (int)l.n_experts;
#define GQ_PLAN(NE)                                                                                                       \
  hipLaunchKernelGGL(k_moe_plan<NE>, dim3(1), dim3(kPlanThreads), 0, s, a, ids, weights, plan, M, E, l.top_k, M <= kMoeFew ? kMoeFew : 16)
  if (!a.logits) GQ_PLAN(0);
  else if (E <= 64) GQ_PLAN(1);
  else if (E <= 128) GQ_PLAN(2);
  else if (E <= 256) GQ_PLAN(4);
  else GQ_PLAN(16);
#undef GQ_PLAN
  return gq_last_launch();
}
int launch_route(const gq_moe &l, const void *x, int xt, int M, double *logits, int *ids, float *weights, const MoePlan &plan,
                 hipStream_t s) {
  if (xt == GQ_DT_F32) GQ_TRY(launch_logits_x<GQ_DT_F32>(l, x, logits, M, s));
  else if (xt == GQ_DT_F16) GQ_TRY(launch_logits_x<GQ_DT_F16>(l, x, logits, M, s));
  else GQ_TRY(launch_logits_x<GQ_DT_BF16>(l, x, logits, M, s));
  const RouteArgs a = {logits, l.router_bias, ids, weights, l.score, l.renorm, l.scale};
  return launch_plan(l, a, nullptr, nullptr, plan, M, s);
}

template <int FMT, int XT>
int launch_gu_few_t(const gq_moe &l, const void *x, const float *rs, const MoePlan &p, float *h, int M, int maxblk, hipStream_t s) {
  const int N = (int)l.N, K = (int)l.K, units = (int)(gq_kpad(FMT, K) / 128), tiles = N / 16;
#define GQ_GU(MR, R, KS, PD)                                                                                              \
  hipLaunchKernelGGL((k_moe_gu_few<FMT, XT, MR, R, KS, PD>), dim3((unsigned)((tiles + (R)-1) / (R)), (unsigned)maxblk),    \
                     dim3(64 * (KS)), 0, s, (const uint8_t *)l.gate, (const uint8_t *)l.up,                               \
                     gq_sc_plane_offset(FMT, l.n_experts * l.N, K), x, rs, p, h, M, N, K, (int)gq_chunks(FMT, K), units,  \
                     l.act, l.top_k)
  if (M == 1) GQ_GU(1, 1, 4, 3);
  else GQ_GU(4, 1, 4, 3);
#undef GQ_GU
  return gq_last_launch();
}
template <int FMT>
int launch_gu_t(const gq_moe &l, const void *x, int xt, const _Float16 *a16, int lda, const float *rs, const MoePlan &p, float *h,
                int M, int maxblk, hipStream_t s) {
  if (M <= kMoeFew)
    return xt == GQ_DT_F16 ? launch_gu_few_t<FMT, GQ_DT_F16>(l, x, rs, p, h, M, maxblk, s)
                           : launch_gu_few_t<FMT, GQ_DT_BF16>(l, x, rs, p, h, M, maxblk, s);
  const int N = (int)l.N, K = (int)l.K, units = (int)(gq_kpad(FMT, K) / 128), tiles = N / 16;
  hipLaunchKernelGGL((k_moe_gu_rows<FMT, 1, 4, 3>), dim3((unsigned)tiles, (unsigned)maxblk), dim3(256), 0, s,
                     (const uint8_t *)l.gate, (const uint8_t *)l.up, gq_sc_plane_offset(FMT, l.n_experts * l.N, K), a16, lda, rs, p,
                     h, M, N, (int)gq_chunks(FMT, K), units, l.act, l.top_k);
  return gq_last_launch();
}
template <int FMT>
int launch_down_t(const gq_moe &l, const float *h, const _Float16 *h16, int ldh, const float *hs, const MoePlan &p,
                  const void *resid, void *y, int dt, int M, int maxblk, hipStream_t s) {
  const int N = (int)l.N, K = (int)l.K, units = (int)(gq_kpad(FMT, N) / 128), C = (int)gq_chunks(FMT, N);
  const size_t so = gq_sc_plane_offset(FMT, l.n_experts * l.K, N);
  const dim3 grid((unsigned)(K / 16));
  constexpr int KS = 8;
  if (M <= kMoeFew) {
#define GQ_DOWN(MR)                                                                                                    \
  hipLaunchKernelGGL((k_moe_down_few<FMT, MR, KS, 4>), grid, dim3(64 * KS), 0, s, (const uint8_t *)l.down, so, h, p, resid, y, \
                     dt, M, N, K, C, units, l.top_k)
    if (M == 1) GQ_DOWN(1);
    else GQ_DOWN(4);
#undef GQ_DOWN
    return gq_last_launch();
  }
  const size_t P = (size_t)M * l.top_k, lds = (size_t)KS * M * 64 + P * 4 + (size_t)maxblk * 34 + P + 16;
  hipLaunchKernelGGL((k_moe_down_rows<FMT, KS, 3>), grid, dim3(64 * KS), lds, s, (const uint8_t *)l.down, so, h16, ldh, hs, p, resid,
                     y, dt, M, K, C, units, l.top_k, maxblk);
  return gq_last_launch();
}

int moe_ffn(const gq_moe &l, const void *x, int xt, const MoePlan &plan, const MoeWs &w, uint8_t *ws, const void *resid, void *y,
            int dt, int M, hipStream_t s) {
  _Float16 *a16 = (_Float16 *)(ws + w.a16), *h16 = (_Float16 *)(ws + w.h16);
  float *rs = (float *)(ws + w.rs), *h = (float *)(ws + w.h), *hs = (float *)(ws + w.hs);
  const bool few = M <= kMoeFew;
  const int q4 = l.fmt == GQ_FMT_Q4_0 || gq_fmt_is_q4k(l.fmt), q4d = l.fmt_down == GQ_FMT_Q4_0 || gq_fmt_is_q4k(l.fmt_down);
  const int lda = few ? (int)l.K : (int)gq_kpad(l.fmt, l.K) + 8, ldh = (int)gq_kpad(l.fmt_down, l.N) + 8;
  const float *xs = nullptr;
  if (!few || xt == GQ_DT_F32 || (uintptr_t)x % 4) {  // (few rows of 16-bit x go in as they are)
    GQ_TRY(gq_launch_a_to_f16(x, xt, a16, rs, M, (int)l.K, lda, few ? 0 : q4, s));
    x = a16;
    xt = GQ_DT_F16;
    xs = rs;
  }
#define GQ_GU_F(F) launch_gu_t<F>(l, x, xt, a16, lda, xs, plan, h, M, w.maxblk, s)
  if (l.fmt == GQ_FMT_Q4_0) GQ_TRY(GQ_GU_F(GQ_FMT_Q4_0));
  else if (l.fmt == GQ_FMT_Q8_0) GQ_TRY(GQ_GU_F(GQ_FMT_Q8_0));
  else if (gq_fmt_is_q6k(l.fmt)) GQ_TRY(GQ_GU_F(GQ_FMT_Q6_K));
  else GQ_TRY(GQ_GU_F(GQ_FMT_Q4_K));
#undef GQ_GU_F
  if (!few) GQ_TRY(gq_launch_a_to_f16(h, GQ_DT_F32, h16, hs, M * l.top_k, (int)l.N, ldh, q4d, s));
#define GQ_DOWN_F(F) launch_down_t<F>(l, h, h16, ldh, hs, plan, resid, y, dt, M, w.maxblk, s)
  if (l.fmt_down == GQ_FMT_Q4_0) return GQ_DOWN_F(GQ_FMT_Q4_0);
  if (l.fmt_down == GQ_FMT_Q8_0) return GQ_DOWN_F(GQ_FMT_Q8_0);
  if (gq_fmt_is_q6k(l.fmt_down)) return GQ_DOWN_F(GQ_FMT_Q6_K);
  return GQ_DOWN_F(GQ_FMT_Q4_K);
#undef GQ_DOWN_F
}

// The workspace of a call: the caller's, or scratch memory of its own
struct MoeRoom {
  GqScratch sc;
  uint8_t *ptr = nullptr;
  int status = GQ_OK;
  MoeRoom(void *ws, size_t ws_bytes, size_t need, hipStream_t s) : sc(ws ? 0 : need, s) {
    if (ws && ws_bytes < need) status = GQ_ERR_WORKSPACE;
    else if (((uintptr_t)ws & 15) != 0) status = GQ_ERR_INVALID_ARGS;
    ptr = ws ? (uint8_t *)ws : (uint8_t *)sc.ptr;
    if (!ptr) status = GQ_ERR_WORKSPACE;
  }
};
MoePlan plan_of(const MoeWs &w, uint8_t *ws) {
  return MoePlan{(int *)(ws + w.nblk), (MoeBlk *)(ws + w.blk), (float *)(ws + w.wsum), w.maxblk};
}

}  // namespace

extern "C" size_t gq_moe_workspace_bytes(const gq_moe *l, size_t M) {
  if (check_moe(l, 0, false, true) != GQ_OK || M > GQ_MOE_MAX_TOKENS || M == 0) return 0;
  return moe_ws(*l, M).bytes;
}

extern "C" size_t gq_moe_route_workspace_bytes(const gq_moe *l, size_t M) {
  if (check_moe(l, 0, true, false) != GQ_OK || M > GQ_MOE_MAX_TOKENS) return 0;
  return M * l->n_experts * 8;
}

extern "C" int gq_moe_route(const gq_moe *l, const void *x, int x_dtype, int32_t *ids, float *weights, size_t M, void *ws,
                            size_t ws_bytes, void *stream) {
  GQ_TRY(check_moe(l, M, true, false));
  GQ_CHECK(gq_dtype_valid(x_dtype), GQ_ERR_UNSUPPORTED);
  if (M == 0) return GQ_OK;
  GQ_CHECK(x && ids && weights, GQ_ERR_INVALID_ARGS);
  hipStream_t s = (hipStream_t)stream;
  MoeRoom room(ws, ws_bytes, M * l->n_experts * 8, s);
  GQ_TRY(room.status);
  return launch_route(*l, x, x_dtype, (int)M, (double *)room.ptr, ids, weights, MoePlan{}, s);
}

extern "C" int gq_moe_ffn(const gq_moe *l, const void *x, int x_dtype, const int32_t *ids, const float *weights,
                          const void *resid, void *y, int y_dtype, size_t M, void *ws, size_t ws_bytes, void *stream) {
  GQ_TRY(check_moe(l, M, false, true));
  GQ_CHECK(gq_dtype_valid(x_dtype) && gq_dtype_valid(y_dtype), GQ_ERR_UNSUPPORTED);
  if (M == 0) return GQ_OK;
  GQ_CHECK(x && y && ids && weights, GQ_ERR_INVALID_ARGS);
  hipStream_t s = (hipStream_t)stream;
  const MoeWs w = moe_ws(*l, M);
  MoeRoom room(ws, ws_bytes, w.bytes, s);
  GQ_TRY(room.status);
  const MoePlan plan = plan_of(w, room.ptr);
  GQ_TRY(launch_plan(*l, RouteArgs{}, (const int *)ids, weights, plan, (int)M, s));
  return moe_ffn(*l, x, x_dtype, plan, w, room.ptr, resid, y, y_dtype, (int)M, s);
}

extern "C" int gq_moe_layer(const gq_moe *l, const void *x, int x_dtype, const void *resid, void *y, int y_dtype, int32_t *ids,
                            float *weights, size_t M, void *ws, size_t ws_bytes, void *stream) {
  GQ_TRY(check_moe(l, M, true, true));
  GQ_CHECK(gq_dtype_valid(x_dtype) && gq_dtype_valid(y_dtype), GQ_ERR_UNSUPPORTED);
  if (M == 0) return GQ_OK;
  GQ_CHECK(x && y, GQ_ERR_INVALID_ARGS);
  hipStream_t s = (hipStream_t)stream;
  const MoeWs w = moe_ws(*l, M);
  MoeRoom room(ws, ws_bytes, w.bytes, s);
  GQ_TRY(room.status);
  const MoePlan plan = plan_of(w, room.ptr);
  GQ_TRY(launch_route(*l, x, x_dtype, (int)M, (double *)(room.ptr + w.logits), ids, weights, plan, s));
  return moe_ffn(*l, x, x_dtype, plan, w, room.ptr, resid, y, y_dtype, (int)M, s);
}
