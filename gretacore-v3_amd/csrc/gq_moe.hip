// gq_moe.hip -- the mixture-of-experts layer of a few tokens over T16 expert tensors: router, choice of experts, their gated
// feed-forward products and the weighted sum.
//
//   l[m][e] = sum_k x[m][k] Wr[e][k]                    k_moe_logits, in 64 bits: which of two experts is larger decides the layer
//   S_m, w_me                                           k_moe_plan: the choice, and the list of each expert's tokens
//   h_me = act(Wg_e x_m) * (Wu_e x_m)                   k_moe_gu_*: one row of h a (token, expert) pair
//   y_m = r_m + sum over S_m of w_me Wd_e h_me          k_moe_down_*: a workgroup adds its row tiles' columns (16, more tokens: 32) over all
//                                                       experts, or over a part of them
//
// The weights of the experts taken bound all of it; each is read once for up to 16 of its tokens, 32 where experts have many (moe_tiles).
#include <algorithm>
#include <type_traits>

#include "gq_internal.h"
#include "gq_rows_frag.h"

#define GQ_DEV_M __device__ __forceinline__

namespace {

constexpr int kMoeFew = 4;  // tokens that the kernels of few rows take

// A block of an expert's work: up to 16 (with more tokens an expert 32: 2^MoePlan::sh) of its pairs (token * top + slot).  expert -1: no block.
constexpr int kMoeTiles = 2;  // row tiles of 16 of a block at most
struct MoeBlk {
  int expert, count;
  int pair[16 * kMoeTiles];
};
struct MoePlan {
  int *nblk;
  MoeBlk *blk;  // [maxblk], the blocks that there are first
  float *wsum;  // [pair] the weight (of the first pair of an expert that a token names twice: their sum)
  int maxblk, sh;  // 2^sh: rows of a block
  int *count;  // tokens chosen for (zeroed by k_moe_logits)
};

// ---- router --------------------------------------------------------------------------
// Where the rows of x go as fp16 with a power-of-two scale each (gq_launch_a_to_f16's), a16 NULL: nowhere
struct MoeConv {
  _Float16 *a16;
  float *rs;
  int lda, q4;
};
// One wave, one row
template <int XT>
GQ_DEV void moe_convert(const void *x, const MoeConv &c, int m, int K, int lane) {
  float top = 0.f;
  for (int k = 8 * lane; k < K; k += 512) {
    FRaw<XT> r;
    float v[8];
    px_load<XT>(x, (size_t)m * K + k, r);
    px_floats<XT>(r, true, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const int sh = gq_fp16_shift(top);
  const float f = gq_pow2(sh);
  if (lane == 0) c.rs[m] = gq_pow2(-sh);
  for (int k = 8 * lane; k < c.lda; k += 512) {
    FRaw<XT> r;
    float v[8];
    px_load<XT>(x, (size_t)m * K + (k < K ? k : 0), r);
    px_floats<XT>(r, k < K, v);
    gq_half8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)((c.q4 ? (kQ4Div16[i] ? v[kQ4Perm[i]] * 0.0625f : v[kQ4Perm[i]]) : v[i]) * f);
    *reinterpret_cast<gq_half8 *>(c.a16 + (size_t)m * c.lda + k) = h;
  }
}
// The sum of a wave's values, in all lanes: rows of 16 by rotations, then the rows
template <int CTRL>
GQ_DEV double dpp_d(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
GQ_DEV double wave_sum(double v) {
  v += dpp_d<0x128>(v);  // row_ror 8, 4, 2, 1
  v += dpp_d<0x124>(v);
  v += dpp_d<0x122>(v);
  v += dpp_d<0x121>(v);
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
// Workgroup (e, b): logits of expert e for tokens TOK b .. TOK b + TOK - 1.  Products of two fp32 values are exact in 64 bits.
// Workgroup (E, b): the conversion of those tokens' rows, a wave a row.
constexpr int kLogThreads = 256;
template <int XT, int RT, int TOK>
__global__ void __launch_bounds__(kLogThreads) k_moe_logits(const void *__restrict__ x, const void *__restrict__ wr,
                                                            double *__restrict__ logits, MoeConv conv, int *count, int M, int E, int K) {
  static_assert(TOK <= kLogThreads / 64, "a wave a row");
  __shared__ double red[kLogThreads / 64][TOK];
  const int tid = threadIdx.x, e = blockIdx.x, m0 = TOK * (int)blockIdx.y;
  if (count && tid == 0 && e == 0 && m0 == 0) *count = 0;
  if (e == E) {
    const int w = tid >> 6;
    if (w < TOK && m0 + w < M) moe_convert<XT>(x, conv, m0 + w, K, tid & 63);
    return;
  }
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
  for (int t = 0; t < TOK; ++t) acc[t] = wave_sum(acc[t]);
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
// Values that another workgroup of the launch reads: past the caches that it does not share
template <typename V>
GQ_DEV void st_agent(V *p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V>
GQ_DEV V ld_agent(const V *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
GQ_DEV double lane_d(double v, int lane) {  // (lane: the same in all lanes)
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int kFewNE = 2;  // experts a lane of the choice within k_moe_gu_few
// One wave chooses the experts of token m; lane j writes slot j (ids_s: in LDS, at the token's place).  A key is a 64-bit number in the values' order, 0 what is
// never taken (-Inf, none there, taken before): the largest's high word, then its low word, then the lowest
// expert that has both.
template <int NE>
GQ_DEV void moe_choose(const RouteArgs &a, int m, int E, int top, int lane, int *ids_s, float *w_s) {
  const double ninf = -__builtin_inf();
  const bool sm = a.score == GQ_MOE_SOFTMAX, weighed = w_s || a.weights;  // (else the ids alone)
  double l[NE], lmax = ninf, sum = 0.0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = 64 * i + lane;
    l[i] = e < E ? a.logits[(size_t)m * E + e] : ninf;
    lmax = fmax(lmax, l[i]);  // (of those that are numbers)
  }
  if (sm && (weighed || a.bias)) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lmax = fmax(lmax, __shfl_xor(lmax, o, 64));
    if (!a.renorm || a.bias) {  // (renormalised weights do without the sum over all experts)
#pragma unroll
      for (int i = 0; i < NE; ++i) sum += l[i] == ninf ? 0.0 : exp(l[i] - lmax);
      sum = wave_sum(sum);
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
    int same = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) same += __builtin_popcountll(__ballot(kh[i] == mh));
    uint32_t mw = 0;
    if (same > 1) {  // (low words count)
#pragma unroll
      for (int i = 0; i < NE; ++i) w = max(w, kh[i] == mh ? kl[i] : 0u);
      mw = wave_max(w);
    }
    bool found = false;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const uint64_t at = found ? 0 : __ballot(kh[i] == mh && kl[i] >= mw);
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
  if (lane < top) {
    if (ids_s) ids_s[m * top + lane] = id;
    if (a.ids) st_agent(a.ids + m * top + lane, id);
  }
  if (!weighed) return;
  double w = id < 0 ? 0.0 : score(mine), total = 0.0;
  if (a.renorm) {
    for (int j = 0; j < top; ++j) total += lane_d(w, j);
    w = total == 0.0 ? 0.0 : w / total;
  }
  if (lane < top) {
    const float f = id < 0 ? 0.f : (float)(w * (double)a.scale);
    if (w_s) w_s[m * top + lane] = f;
    if (a.weights) st_agent(a.weights + m * top + lane, f);
  }
}

template <int NE>
__global__ void __launch_bounds__(64) k_moe_choose(RouteArgs a, int E, int top) {
  moe_choose<NE>(a, (int)blockIdx.x, E, top, (int)threadIdx.x, nullptr, nullptr);
}

// ---- plan ---------------------------------------------------------------------------
// The choice (NE: experts a lane; 0: ids and weights are given), each expert's pairs in order of their tokens, in blocks of 16 or 32 (2^MoePlan::sh).
// Ids outside 0 .. E - 1 name no expert; an expert that a token names twice gets one pair with both weights.
constexpr int kPlanThreads = 1024;
// Is this workgroup the last of n to arrive at a counter (zero before the launch)?  What the others stored before they came, by st_agent, can
// be read then, by ld_agent (fences in their place, which write back and drop whole caches: 2 us more).
GQ_DEV bool arrives_last(int *counter, int n) {
  __shared__ int last_s;
  __builtin_amdgcn_s_waitcnt(0x0F70);  // (every wave's own stores have arrived)
  __syncthreads();
  if (threadIdx.x == 0)
    last_s = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
  __syncthreads();
  return last_s != 0;
}
// NE > 0: more tokens than a workgroup has waves are chosen for by a workgroup each, and the last to be done makes the plan.
template <int NE>
__global__ void __launch_bounds__(kPlanThreads) k_moe_plan(RouteArgs a, const int *__restrict__ ids, const float *__restrict__ weights,
                                                           MoePlan p, int M, int E, int top) {
  constexpr int MP = GQ_MOE_MAX_TOKENS * GQ_MOE_MAX_TOP;
  static_assert(MP <= kPlanThreads && GQ_MOE_MAX_EXPERTS <= kPlanThreads, "a thread a pair, a thread an expert");
  __shared__ int id_s[MP], base_s[kPlanThreads], tot_s[kPlanThreads / 64];
  __shared__ uint32_t tok_s[2][kPlanThreads];  // the tokens of an expert, a bit each
  __shared__ float w_s[MP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, P = M * top;
  if constexpr (NE > 0) {
    if (gridDim.x > 1) {
      if (wave == 0) moe_choose<NE>(a, (int)blockIdx.x, E, top, lane, nullptr, nullptr);
      if (!arrives_last(p.count, (int)gridDim.x)) return;
      if (tid < P) {
        id_s[tid] = ld_agent(a.ids + tid);
        w_s[tid] = ld_agent(a.weights + tid);
      }
    } else if (wave < M) {
      moe_choose<NE>(a, wave, E, top, lane, id_s, w_s);
    }
  } else if (tid < P) {
    id_s[tid] = ids[tid];
    w_s[tid] = weights[tid];
  }
  tok_s[0][tid] = tok_s[1][tid] = 0;
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
    p.wsum[tid] = w;
    if (id >= 0) atomicOr(&tok_s[tok >> 5][id], 1u << (tok & 31));
  }
  __syncthreads();
  const int c = __popc(tok_s[0][tid]) + __popc(tok_s[1][tid]), nb = (c + (1 << p.sh) - 1) >> p.sh;
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
    p.blk[base + b].count = min(c - (b << p.sh), 1 << p.sh);
  }
  for (int b = all + tid; b < p.maxblk; b += kPlanThreads) p.blk[b].expert = -1;
  if (tid == 0) *p.nblk = all;
  __syncthreads();
  if (id >= 0) {
    const uint32_t below = (1u << (tok & 31)) - 1u, w0 = tok_s[0][id], w1 = tok_s[1][id];
    const int rank = tok < 32 ? __popc(w0 & below) : __popc(w0) + __popc(w1 & below);
    p.blk[base_s[id] + (rank >> p.sh)].pair[rank & ((1 << p.sh) - 1)] = tid;
  }
}

// ---- few tokens: no plan --------------------------------------------------------------
// At most 64 pairs, a lane each.  An expert's block is that of the first pair that names it; row m is token m's first pair with it (-1:
// none), with the weights of all of that token's.
struct FewPairs {
  int id;       // this lane's pair
  uint64_t of;  // the pairs of the expert asked for
  GQ_DEV_M int expert(int q) const { return __builtin_amdgcn_readlane(id, q); }
  GQ_DEV_M bool leads(int q) {  // is q the first of its expert's
    const int e = expert(q);
    of = e < 0 ? 0 : __ballot(id == e);
    return e >= 0 && __builtin_ctzll(of) == q;
  }
  GQ_DEV_M uint64_t mine(int m, int top) const { return of & (((1ull << top) - 1ull) << (m * top)); }
  GQ_DEV_M int pair(int m, int top) const { return mine(m, top) ? __builtin_ctzll(mine(m, top)) : -1; }
};

// ---- gate and up -----------------------------------------------------------------------
// Output (m, 16 t + n) of the R tiles `group` in both matrices from the waves' parts at(k, w, t, n, m)
template <int KS, int R, typename At>
GQ_DEV float moe_gu_h(At at, int nl, int m, float f, int act) {
  float y[2] = {0.f, 0.f};
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int k = 0; k < KS; ++k) y[w] += at(k, w, nl >> 4, nl & 15, m);
  return gq_act_f(act, y[0] * f) * (y[1] * f);
}

// Up to 4 tokens of 16-bit x: codes and x as they are, scales in fp32 (gq_rows_frag.h); row j is token j.  h goes out in fp16 (nib:
// in the nibbles' order; as the matrix cores take it, 2.1e-4 of h) with a power-of-two scale for each 32 of a row, the scale groups of W_down's products; the inverse of block
// 2 m + i of 128 values to hs[pair][128s][i][m].
// Workgroup (j, q): 32 columns of the expert that pair q names first.  ROUTE: the choice is made here, by every workgroup for itself (8 of
// 64 experts of 1024 x 2048: 20.5 us the layer, 23.1 with the choice in a launch of its own); the first one keeps it.
template <int FMT, int XT, int MR, int KS, int PD, bool ROUTE>
__global__ void __launch_bounds__(64 * KS)
k_moe_gu_few(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off, const void *__restrict__ x,
             const float *__restrict__ rs, RouteArgs a, const int *__restrict__ ids, _Float16 *__restrict__ h, float *__restrict__ hs,
             int nib, int M, int N, int K, int C, int units, int act, int E, int top) {
  static_assert(KS >= kMoeFew, "a wave a token");
  constexpr int NG = kFewGroups<FMT>, R = 2, T = 2 * R;
  __shared__ float red[KS][T][MR][64];
  extern __shared__ __attribute__((aligned(16))) uint8_t xs_s[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, ntiles = N / 16;
  const int np = 128 * units, stride = (int)few_lds_stride(np);
  __shared__ int id_s[64];
  few_stage<64 * KS>(x, M, K, np, stride, kNibOrder<FMT>, xs_s, (int)threadIdx.x, [&]() __attribute__((always_inline)) {
    if constexpr (ROUTE) {  // (the weights are the first workgroup's alone)
      if (blockIdx.x > 0 || blockIdx.y > 0) a.ids = nullptr, a.weights = nullptr;
      if (wave < M) moe_choose<kFewNE>(a, wave, E, top, lane, id_s, nullptr);
    }
  });
  __syncthreads();
  FewPairs pairs;
  pairs.id = lane < M * top ? (ROUTE ? id_s[lane] : ids[lane]) : -1;
  if (pairs.id >= E) pairs.id = -1;
  const int expert = pairs.expert((int)blockIdx.y);
  if (!pairs.leads((int)blockIdx.y)) return;
  const size_t tile0 = (size_t)expert * (size_t)ntiles;
  FTile<FMT> tl[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int tile = (int)blockIdx.x * R + t % R;
    tl[t] = ftile<FMT>(t < R ? wg : wu, sc_off, tile0 + (size_t)(tile < ntiles ? tile : ntiles - 1), C);  // (clamped: not stored)
  }
  const bool mine = few_mine<FMT>(lane) && (lane & 3) < M;
  const uint32_t x0 = mine ? (uint32_t)((lane & 3) * stride + 32 * g) : (uint32_t)(M * stride), xd = mine ? 256u : 0u;
  constexpr int G = kGroup<FMT>;
  FUnit<FMT> us[PD][T][G];
  auto request = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < T; ++t) load_group<FMT>(tl[t], group, lane, us[st][t]);
  };
  float acc[T][MR] = {};
  uint32_t mg;  // (kept in a register)
  if constexpr (XT == GQ_DT_F16) asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(mg));
  else asm volatile("v_mov_b32 %0, 0x43004300" : "=v"(mg));
  auto compute = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < G; ++p)
      few_add<FMT, XT>(us[st], p, G * group + p, g, xs_s, x0 + xd * (uint32_t)(G * group + p), mg, acc);
  };
  walk_units<PD, KS>(units / G, wave, request, compute);
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int v = 0; v < MR; ++v) red[wave][t][v][lane] = acc[t][v];
  __syncthreads();
  const int m = threadIdx.x >> 5, nl = threadIdx.x & 31, n0 = 32 * (int)blockIdx.x;  // (N is whole 32-blocks)
  const int q = m < M ? pairs.pair(m, top) : -1;
  if (q < 0) return;  // (whole half-waves)
  const float v = moe_gu_h<KS, R>(
      [&](int k, int w, int t, int n, int mm) {
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) y += red[k][w * R + t][MR == 1 ? 0 : mm][16 * i + n];
        return y;
      },
      nl, m, rs ? rs[m] : 1.f, act);
  float t = fabsf(v);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor(t, o, 32));
  const int sh = gq_fp16_shift(t);
  const int e = nl & 7, to = nib ? (e & 1 ? 4 + (e >> 1) : e >> 1) : e;
  h[(size_t)q * N + n0 + (nl & 24) + to] = (_Float16)(v * gq_pow2(sh));
  if (nl == 0) {
    const int c = (n0 >> 5) & 3;
    float *o = hs + ((size_t)q * ((N + 127) / 128) + (n0 >> 7)) * 4;
    o[2 * (c & 1) + (c >> 1)] = gq_pow2(-sh);
    if (n0 + 32 == N)
      for (int d = c + 1; d < 4; ++d) o[2 * (d & 1) + (d >> 1)] = 0.f;  // (blocks behind the row)
  }
}

// More tokens: a block's rows are its pairs, fp16 rows of x gathered, the scale groups folded into the weights.
template <int FMT, int MT, int R, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_moe_gu_rows(const uint8_t *__restrict__ wg, const uint8_t *__restrict__ wu, size_t sc_off, const _Float16 *__restrict__ a16,
              int lda, const float *__restrict__ rs, MoePlan p, float *__restrict__ h, int M, int N, int C, int units, int act,
              int top) {
  constexpr int T = 2 * R;
  __shared__ gq_f4 red[KS][T][MT][64];
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
  bool row[MT];
  uint32_t xo[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    row[t] = 16 * t + r < blk.count;
    xo[t] = row[t] ? 2u * ((uint32_t)(blk.pair[16 * t + r] / top) * (uint32_t)lda + 16u * (uint32_t)g) : 0u;
  }
  constexpr int G = kGroup<FMT>;
  FUnit<FMT> us[PD][T][G];
  gq_half8 xs[PD][G][MT][4];
  auto request = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < T; ++t) load_group<FMT>(tl[t], group, lane, us[st][t]);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint32_t o = row[t] && G * group < units ? xo[t] + 256u * G * (uint32_t)group : 0xFFFFFC00u;
#pragma unroll
      for (int i = 0; i < 4 * G; ++i) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(xr, o + 128u * (i >> 1) + 16u * (i & 1), 0, 0);
        xs[st][i >> 2][t][i & 3] = __builtin_bit_cast(gq_half8, gq_u4{v[0], v[1], v[2], v[3]});
      }
    }
  };
  gq_f4 acc[T][MT];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[t][m] = gq_f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t mg = gq_nib_magic();
  auto compute = [&](int group, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < G; ++p)
#pragma unroll
      for (int t = 0; t < T; ++t) rows_add<FMT, MT>(us[st][t][p], G * group + p, g, mg, xs[st][p], acc[t]);
  };
  walk_units<PD, KS>(units / G, wave, request, compute);
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) red[wave][t][m][lane] = acc[t][m];
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * R * blk.count; o += 64 * KS) {
    const int nl = o % (16 * R), m = o / (16 * R), n = 16 * R * (int)blockIdx.x + nl, q = blk.pair[m];
    if (n >= N) continue;
    h[(size_t)q * N + n] = moe_gu_h<KS, R>(
        [&](int k, int w, int t, int nn, int mm) {
          return reinterpret_cast<const float *>(&red[k][w * R + t][mm >> 4][4 * (mm & 12) + nn])[mm & 3];
        },
        nl, m, rs[q / top], act);
  }
}

// ---- down ------------------------------------------------------------------------------
// A workgroup owns R row tiles of every expert's W_down (16 R columns of y: one tile with few tokens, two with more); its KS waves take the units
// of all blocks, or of its part of them, in turn (block by block, unit by unit), so that the sum over a token's experts stays in the workgroup,
// in one order, and parts are added in theirs (k_moe_sum).
struct ItemAt {
  int b, u;
  GQ_DEV_M void next(int by, int units) {
    u += by;
    while (u >= units) {
      u -= units;
      ++b;
    }
  }
};
// The items of a wave, PD requested ahead (rq: the next to request), and a group of PD at a time: a group requests the next
// one's unless it is the last.
template <int PD, int KS, typename Request>
GQ_DEV void items_requests(ItemAt &rq, int units, Request request) {
#pragma unroll
  for (int i = 0; i < PD; ++i) {
    request(rq, i);
    rq.next(KS, units);
  }
}
template <int PD, int KS, typename Request, typename Compute>
GQ_DEV void items_computes(ItemAt at, ItemAt rq, int nblk, int units, Request request, Compute compute) {
  while (rq.b < nblk) {
#pragma unroll
    for (int i = 0; i < PD; ++i) {
      compute(at, i);
      at.next(KS, units);
      request(rq, i);
      rq.next(KS, units);
    }
  }
#pragma unroll
  for (int i = 0; i < PD; ++i) {
    if (at.b < nblk) compute(at, i);
    at.next(KS, units);
  }
}

// Up to 4 tokens: rows are the tokens; the scale groups' fp32 sums take the inverse scales of h and the expert's weight.  h and its
// scales go through LDS.
template <int FMT, int MR, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_moe_down_few(const uint8_t *__restrict__ wd, size_t sc_off, const _Float16 *__restrict__ h, const float *__restrict__ hs,
               const int *__restrict__ ids, const float *__restrict__ weights, const void *resid, void *y, int dt, int M, int N, int K,
               int C, int units, int E, int top) {
  constexpr int NG = kFewGroups<FMT>, XT = GQ_DT_F16, MB = kMoeFew * GQ_MOE_MAX_TOP;
  constexpr float OFF = kFewOff<FMT, XT>;
  __shared__ float red[KS][MR][64];
  static_assert(MB <= 64, "a lane a pair");
  __shared__ int p_s[MB][kMoeFew];
  __shared__ float w_s[MB][kMoeFew];
  extern __shared__ __attribute__((aligned(16))) uint8_t xs_s[];  // [pair] rows of h, then [pair][unit][i][m] inverse scales
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, ntiles = K / 16;
  // lane q: its expert's first pair of each token, and that token's weight; lane b then: block b's expert
  int id = lane < M * top ? ids[lane] : -1;
  if (id >= E) id = -1;
  const float weight = lane < M * top ? weights[lane] : 0.f;
  int pair[MR], lead = 64;
  float w[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    pair[m] = -1;
    w[m] = 0.f;
    if (m >= M) continue;
    for (int q = m * top; q < m * top + top; ++q) {
      const bool same = __builtin_amdgcn_readlane(id, q) == id;
      const float f = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(weight), q));
      if (same && pair[m] < 0) pair[m] = q;
      if (same) w[m] += f;
    }
    if (pair[m] >= 0) lead = min(lead, pair[m]);
  }
  const bool leads = id >= 0 && lead == lane;
  const uint64_t all = __ballot(leads);
  const int nblk = __builtin_popcountll(all), b0 = __builtin_popcountll(all & ((1ull << lane) - 1ull));
  // (no two lanes to one place: the others go to the places behind the blocks, whose number is that of the lanes)
  const int expert = __builtin_amdgcn_ds_permute(4 * (leads ? b0 : nblk + lane - b0), id);
  if (tid < 64 && leads)
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      p_s[b0][m] = pair[m];
      w_s[b0][m] = w[m];
    }
  const int np = 128 * units, stride = (int)few_lds_stride(np), P = M * top;
  const bool mine = few_mine<FMT>(lane) && (lane & 3) < M;
  const uint32_t zero_at = (uint32_t)(P * stride);
  const float2 *f_s = reinterpret_cast<const float2 *>(xs_s + P * stride + 160);
  const int gi = NG == 2 ? g & 1 : g >> 1;  // the 32-block of a step that this lane's sums are of
  constexpr int G = kGroup<FMT>;
  FUnit<FMT> us[PD][G];
  auto request = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
    const bool on = at.b < nblk;
    const size_t tile = (size_t)__builtin_amdgcn_readlane(expert, on ? at.b : 0) * (size_t)ntiles + blockIdx.x;
    load_group<FMT>(ftile<FMT>(wd, sc_off, tile, on ? C : 0), at.u, lane, us[st]);
  };
  float acc[MR] = {};
  uint32_t mg;  // (kept in a register)
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(mg));
  const gq_u4 ones = {0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
  const gq_f4 zero = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](int b, int unit, int st, int p) __attribute__((always_inline)) {
    const int q = p_s[b][MR == 1 ? 0 : lane & 3];
    const uint32_t xo = mine && q >= 0 ? (uint32_t)(q * stride + 256 * unit + 32 * g) : zero_at;
    float s[2], mn[2];
    float2 f[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) {
      const int qr = p_s[b][r];
      const float w = w_s[b][r];
      f[r] = f_s[2 * (max(qr, 0) * units + unit) + gi];
      f[r] = qr < 0 ? make_float2(0.f, 0.f) : make_float2(f[r].x * w, f[r].y * w);  // (a token without the expert)
    }
    few_scales<FMT>(us[st][p], unit, g & (NG - 1), s, mn);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const gq_u4 a0 = few_lds(xs_s, xo, m, 0), a1 = few_lds(xs_s, xo, m, 1);
      const gq_f4 sx = few_mfma<XT>(a1, ones, few_mfma<XT>(a0, ones, zero));
      gq_u4 b[2];
      few_codes<FMT, XT>(us[st][p], m, mg, b);
      const gq_f4 d = few_mfma<XT>(a1, b[1], few_mfma<XT>(a0, b[0], zero));
      const float o = FMT == GQ_FMT_Q4_K ? fmaf(s[m], OFF, mn[m]) : s[m] * OFF;
#pragma unroll
      for (int r = 0; r < MR; ++r)
        acc[r] = fmaf(m ? f[r].y : f[r].x, fmaf(s[m], d[r], -o * sx[r]), acc[r]);
    }
  };
  auto compute = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < G; ++p) add(at.b, G * at.u + p, st, p);
  };
  const int groups = units / G;
  ItemAt rq = {0, 0};
  rq.next(wave, groups);
  ItemAt first = rq;
  for (int i = tid; i < P * units; i += 64 * KS)  // (of pairs that name no expert too: not used)
    *reinterpret_cast<gq_f4 *>(xs_s + P * stride + 160 + 16 * i) = *reinterpret_cast<const gq_f4 *>(hs + 4 * (size_t)i);
  few_stage<64 * KS>(h, P, N, np, stride, false, xs_s, tid, [&]() __attribute__((always_inline)) {
    if (nblk > 0) items_requests<PD, KS>(rq, groups, request);
  });
  step_barrier<63>();  // (of LDS alone)
  items_computes<PD, KS>(first, rq, nblk, groups, request, compute);
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
// scale's inverse and the expert's weight, to the wave's own sums of the tokens in LDS.  gridDim.y parts of the blocks: their sums go to part
// [part][M][K] in fp32, which k_moe_sum adds.
template <int FMT, int MT, int R, int KS, int PD>
__global__ void __launch_bounds__(64 * KS)
k_moe_down_rows(const uint8_t *__restrict__ wd, size_t sc_off, const _Float16 *__restrict__ h16, int ldh, const float *__restrict__ hs,
                MoePlan p, const void *resid, void *y, int dt, float *__restrict__ part, int M, int K, int C, int units, int top, int maxblk) {
  extern __shared__ float lds[];
  const int P = M * top;
  float *sum_s = lds;                                                    // [KS][M][16 R]
  float *f_s = sum_s + KS * M * 16 * R;                                    // [P]: weight and scale of a pair
  uint16_t *p_s = reinterpret_cast<uint16_t *>(f_s + P);                 // [maxblk][16 MT]: pairs, 0xFFFF none
  uint16_t *e_s = p_s + 16 * MT * maxblk;                                     // [maxblk]
  uint8_t *t_s = reinterpret_cast<uint8_t *>(e_s + maxblk);              // [P]: token of a pair
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r = lane & 15, ntiles = K / 16;
  const int all = __builtin_amdgcn_readfirstlane(*p.nblk);
  const int b0 = all * (int)blockIdx.y / (int)gridDim.y, nblk = all * ((int)blockIdx.y + 1) / (int)gridDim.y;
  for (int i = tid; i < KS * M * 16 * R; i += 64 * KS) sum_s[i] = 0.f;
  for (int i = tid; i < P; i += 64 * KS) {
    f_s[i] = p.wsum[i] * hs[i];
    t_s[i] = (uint8_t)(i / top);
  }
  for (int i = tid; i < 16 * MT * maxblk; i += 64 * KS) {
    const int at = i % (16 * MT);
    const MoeBlk &b = p.blk[i / (16 * MT)];
    p_s[i] = at < b.count ? (uint16_t)b.pair[at] : (uint16_t)0xFFFF;
    if (at == 0) e_s[i / (16 * MT)] = (uint16_t)b.expert;
  }
  __syncthreads();
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<_Float16 *>(h16), (short)0, (int)(2u * (uint32_t)P * (uint32_t)ldh), 0x00020000);
  constexpr int G = kGroup<FMT>;
  FUnit<FMT> us[PD][R][G];
  gq_half8 xs[PD][G][MT][4];
  auto request = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
    const bool on = at.b < nblk;
    const int b = on ? at.b : b0;
    const size_t tile0 = (size_t)__builtin_amdgcn_readfirstlane((int)e_s[b]) * (size_t)ntiles;
#pragma unroll
    for (int t = 0; t < R; ++t) {
      const int tile = (int)blockIdx.x * R + t;  // (clamped: not stored)
      load_group<FMT>(ftile<FMT>(wd, sc_off, tile0 + (size_t)min(tile, ntiles - 1), on ? C : 0), at.u, lane, us[st][t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint32_t q = p_s[16 * (MT * b + t) + r];
      const uint32_t o = on && q != 0xFFFFu ? 2u * (q * (uint32_t)ldh + 16u * (uint32_t)g) + 256u * G * (uint32_t)at.u : 0xFFFFFC00u;
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
    for (int m = 0; m < MT; ++m) acc[t][m] = gq_f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t mg = gq_nib_magic();
  int cur = -1;
  auto flush = [&]() __attribute__((always_inline)) {
    if (cur < 0) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const uint32_t q = p_s[16 * (MT * cur + m) + 4 * g + v];
        if (q == 0xFFFFu) continue;
        float *s = sum_s + (wave * M + t_s[q]) * (16 * R) + r;  // (a block's tokens differ)
#pragma unroll
        for (int t = 0; t < R; ++t) s[16 * t] += f_s[q] * acc[t][m][v];
      }
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[t][m] = gq_f4{0.f, 0.f, 0.f, 0.f};
  };
  auto compute = [&](const ItemAt &at, int st) __attribute__((always_inline)) {
    if (at.b != cur) {
      flush();
      cur = at.b;
    }
#pragma unroll
    for (int p = 0; p < G; ++p)
#pragma unroll
      for (int t = 0; t < R; ++t) rows_add<FMT, MT>(us[st][t][p], G * at.u + p, g, mg, xs[st][p], acc[t]);
  };
  const int groups = units / G;
  ItemAt rq = {b0, 0};
  rq.next(wave, groups);
  const ItemAt first = rq;
  items_requests<PD, KS>(rq, groups, request);
  items_computes<PD, KS>(first, rq, nblk, groups, request, compute);
  flush();
  __syncthreads();
  for (int i = tid; i < 16 * R * M; i += 64 * KS) {
    const int n = i % (16 * R), m = i / (16 * R), k = 16 * R * (int)blockIdx.x + n;
    if (k >= K) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < KS; ++w) v += sum_s[(w * M + m) * (16 * R) + n];
    const size_t o = (size_t)m * K + k;
    if (part) {
      part[(size_t)blockIdx.y * M * K + o] = v;
      continue;
    }
    if (resid) v += gq_ld_dt(resid, dt, o);
    gq_st_dt(y, dt, o, v);
  }
}
__global__ void __launch_bounds__(256) k_moe_sum(const float *__restrict__ part, const void *resid, void *y, int dt, int n, int parts) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
  for (int p = 0; p < parts; ++p) v += part[(size_t)p * n + i];
  if (resid) v += gq_ld_dt(resid, dt, i);
  gq_st_dt(y, dt, i, v);
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

// Up to 4 tokens whose rows of x, and of h with their scales, fit LDS beside the waves' sums (32 KiB of k_moe_gu_few, 18 of k_moe_down_few)
bool moe_few(const gq_moe &l, size_t M) {
  const size_t P = M * (size_t)l.top_k, nk = (gq_kpad(l.fmt, l.K) + 127) & ~(size_t)127, nn = (gq_kpad(l.fmt_down, l.N) + 127) & ~(size_t)127;
  return M <= (size_t)kMoeFew && few_lds_bytes(M, nk) <= (160 - 34) * 1024 && few_lds_bytes(P, nn) + P * nn / 8 <= (160 - 20) * 1024;
}
// Row tiles of a block: two where an expert has 16 tokens and more if all are taken alike, so that its weights are read and converted for up to 32 of
// them (us the layer by one / two tiles, Q4_K with Q6_K and Q8_0 with Q4_0: 64 tokens, 2 of 8 of 14336 x 4096, 295 / 279 and 311 / 271; 20 tokens, 4 of 4
// of 4096 x 4096, 80 / 68 and 83 / 67; with fewer the second tile's loads and products are for nothing: 48 tokens, 2 of 8 of 14336 x 4096, 231 / 271 and 242 / 256;
// four tiles: 366 - 462 of the first, 212 and 176 of 43 tokens, 4 of 4 of 9984 x 3328, that two do in 189 and 207).
// The mean serves uneven choices too, one expert that every token takes, or experts by their rank's inverse: 64 tokens, 8 of 128 of 768 x 2048,
// 96 / 124 and 93 / 116 (112 / 129 and 106 / 121); 48 tokens, 2 of 8 of 14336 x 4096, 232 / 266 and 226 / 253 (281 / 275 and 273 / 261: 2 and 4 % lost).
int moe_tiles(const gq_moe &l, size_t M) { return M * (size_t)l.top_k >= 16 * l.n_experts ? 2 : 1; }
// Where a call's intermediate values lie in its workspace
struct MoeWs {
  size_t logits, ids, weights, count, nblk, blk, wsum, a16, rs, h, h16, hs, part, bytes;
  int maxblk, parts, tiles;
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
  const bool few = moe_few(l, M);
  // (an expert's last block may be short: at most a block an expert beyond whole ones)
  w.tiles = few ? 1 : moe_tiles(l, M);
  const size_t blocks = few ? std::min(P, l.n_experts) : std::min(P, l.n_experts + P / 16);  // (of one tile: the bytes grow with the tokens)
  w.maxblk = (int)(w.tiles == 1 ? blocks : std::min(P, l.n_experts + P / 32));
  w.logits = take(M * l.n_experts * 8);
  w.ids = take(P * 4);
  w.weights = take(P * 4);
  w.count = take(4);
  w.nblk = take(4);
  w.blk = take(blocks * sizeof(MoeBlk));
  w.wsum = take(P * 4);
  w.a16 = take(M * (gq_kpad(l.fmt, l.K) + 8) * 2);
  w.rs = take((M + 256) * 4);
  w.h = take(few ? 0 : P * l.N * 4);
  w.h16 = take(P * (gq_kpad(l.fmt_down, l.N) + 8) * 2);
  w.hs = take(few ? P * ((l.N + 127) / 128) * 16 : (P + 256) * 4);
  // W_down's row tiles, two a workgroup, in parts as far as a workgroup a CU goes (64 tokens, 128 experts of 768 x 2048, in 2 / 3 / 4
  // parts: 147 / 127 / 117 us the layer; 37 tokens, 61 of 1376 x 2080, whose four are more than that, 100 / 92 / 98)
  w.parts = few ? 1 : (int)std::min(std::max((size_t)1, 256 / ((l.K + 31) / 32)), std::min((size_t)8, blocks));
  w.part = take(w.parts > 1 ? w.parts * M * l.K * 4 : 0);
  w.bytes = at;
  return w;
}

template <int XT, int RT>
int launch_logits_t(const gq_moe &l, const void *x, double *logits, const MoeConv &conv, int *count, int M, hipStream_t s) {
#define GQ_LOG(TOK)                                                                                                       \
  hipLaunchKernelGGL((k_moe_logits<XT, RT, TOK>), dim3((unsigned)(l.n_experts + (conv.a16 != nullptr)),                  \
                                                       (unsigned)((M + (TOK)-1) / (TOK))),                               \
                     dim3(kLogThreads), 0, s, x, l.router, logits, conv, count, M, (int)l.n_experts, (int)l.K)
  if (M == 1) GQ_LOG(1);
  else GQ_LOG(4);
#undef GQ_LOG
  return gq_last_launch();
}
template <int XT>
int launch_logits_x(const gq_moe &l, const void *x, double *logits, const MoeConv &conv, int *count, int M, hipStream_t s) {
  if (l.router_dtype == GQ_DT_F32) return launch_logits_t<XT, GQ_DT_F32>(l, x, logits, conv, count, M, s);
  if (l.router_dtype == GQ_DT_F16) return launch_logits_t<XT, GQ_DT_F16>(l, x, logits, conv, count, M, s);
  return launch_logits_t<XT, GQ_DT_BF16>(l, x, logits, conv, count, M, s);
}
int launch_plan(const gq_moe &l, const RouteArgs &a, const int *ids, const float *weights, const MoePlan &plan, int M,
                hipStream_t s) {
  const int E = (int)l.n_experts;
#define GQ_PLAN(NE)                                                                                                       \
  hipLaunchKernelGGL(k_moe_plan<NE>, dim3((NE) > 0 && M > kPlanThreads / 64 ? (unsigned)M : 1u), dim3(kPlanThreads), 0, s, a, ids, weights, plan, M, E, l.top_k)
  if (!a.logits) GQ_PLAN(0);
  else if (E <= 64) GQ_PLAN(1);
  else if (E <= 128) GQ_PLAN(2);
  else if (E <= 256) GQ_PLAN(4);
  else GQ_PLAN(16);
#undef GQ_PLAN
  return gq_last_launch();
}
int launch_choose(const gq_moe &l, const RouteArgs &a, int M, hipStream_t s) {
  const int E = (int)l.n_experts;
#define GQ_CHOOSE(NE) hipLaunchKernelGGL(k_moe_choose<NE>, dim3((unsigned)M), dim3(64), 0, s, a, E, l.top_k)
  if (E <= 64) GQ_CHOOSE(1);
  else if (E <= 128) GQ_CHOOSE(2);
  else if (E <= 256) GQ_CHOOSE(4);
  else GQ_CHOOSE(16);
#undef GQ_CHOOSE
  return gq_last_launch();
}
int launch_logits(const gq_moe &l, const void *x, int xt, double *logits, const MoeConv &conv, int *count, int M, hipStream_t s) {
  if (xt == GQ_DT_F32) return launch_logits_x<GQ_DT_F32>(l, x, logits, conv, count, M, s);
  if (xt == GQ_DT_F16) return launch_logits_x<GQ_DT_F16>(l, x, logits, conv, count, M, s);
  return launch_logits_x<GQ_DT_BF16>(l, x, logits, conv, count, M, s);
}

// Intermediate values of a call
struct MoeMid {
  _Float16 *a16, *h16;
  float *rs, *h, *hs, *part;
  int lda, ldh, parts;
};
template <int FMT, int XT>
int launch_gu_few_t(const gq_moe &l, const void *x, const float *rs, const RouteArgs *a, const int *ids, const MoeMid &b, int M,
                    hipStream_t s) {
  const int N = (int)l.N, K = (int)l.K, units = (int)(gq_kpad(FMT, K) / 128), nib = l.fmt_down == GQ_FMT_Q4_0 || gq_fmt_is_q4k(l.fmt_down);
#define GQ_GU_R(MR, KS, PD, ROUTE)                                                                                         \
  hipLaunchKernelGGL((k_moe_gu_few<FMT, XT, MR, KS, group_stages<FMT>(PD), ROUTE>), dim3((unsigned)(N / 32), (unsigned)(M * l.top_k)), dim3(64 * (KS)), \
                     few_lds_bytes(M, 128 * (size_t)units), s, (const uint8_t *)l.gate, (const uint8_t *)l.up,            \
                     gq_sc_plane_offset(FMT, l.n_experts * l.N, K), x, rs, a ? *a : RouteArgs{}, ids, b.h16, b.hs, nib, M, N, K,    \
                     (int)gq_chunks(FMT, K), units, l.act, (int)l.n_experts, l.top_k)
#define GQ_GU(MR, KS, PD)                  \
  do {                                     \
    if (a) GQ_GU_R(MR, KS, PD, true);      \
    else GQ_GU_R(MR, KS, PD, false);       \
  } while (0)
  // (one token, Q4_K: 256 workgroups, 64 experts of 1024 x 2048, by 8 waves 20.5 us the layer, by 4 20.8; 896, 8 of 14336 x 4096, 51.7 and 51.1)
  const bool wide = (size_t)(N / 32) * (size_t)(M * l.top_k) > 512;
  if (M == 1) {
    if (wide) GQ_GU(1, 4, 2);
    else GQ_GU(1, 8, 1);
  } else {
    if (wide) GQ_GU(4, 4, 2);
    else GQ_GU(4, 8, 1);
  }
#undef GQ_GU
#undef GQ_GU_R
  return gq_last_launch();
}
template <int FMT>
int launch_gu_t(const gq_moe &l, const void *x, int xt, const float *rs, const RouteArgs *a, const int *ids, const MoePlan &p,
                const MoeMid &b, int M, hipStream_t s) {
  if (moe_few(l, M))
    return xt == GQ_DT_F16 ? launch_gu_few_t<FMT, GQ_DT_F16>(l, x, rs, a, ids, b, M, s)
                           : launch_gu_few_t<FMT, GQ_DT_BF16>(l, x, rs, a, ids, b, M, s);
  const int N = (int)l.N, K = (int)l.K, units = (int)(gq_kpad(FMT, K) / 128), tiles = N / 16;
  // (16 tokens, 8 experts of 14336 x 4096, Q4_0, by one tile 190 us the layer, by two 167; 64 tokens, 128 experts of 768 x 2048, 143 and 128)
  constexpr int R = 2, KS = 4;
#define GQ_GU_ROWS(MT)                                                                                                                      \
  hipLaunchKernelGGL((k_moe_gu_rows<FMT, MT, R, KS, group_stages<FMT>(2)>), dim3((unsigned)((tiles + R - 1) / R), (unsigned)p.maxblk), dim3(64 * KS), 0, s, \
                     (const uint8_t *)l.gate, (const uint8_t *)l.up, gq_sc_plane_offset(FMT, l.n_experts * l.N, K), b.a16, b.lda, rs, p,    \
                     b.h, M, N, (int)gq_chunks(FMT, K), units, l.act, l.top_k)
  if (p.sh == 4) GQ_GU_ROWS(1);
  else GQ_GU_ROWS(2);
#undef GQ_GU_ROWS
  return gq_last_launch();
}
template <int FMT>
int launch_down_t(const gq_moe &l, const int *ids, const float *weights, const MoePlan &p, const MoeMid &b, const void *resid, void *y,
                  int dt, int M, hipStream_t s) {
  const int N = (int)l.N, K = (int)l.K, units = (int)(gq_kpad(FMT, N) / 128), C = (int)gq_chunks(FMT, N);
  const size_t so = gq_sc_plane_offset(FMT, l.n_experts * l.K, N);
  const unsigned tiles = (unsigned)(K / 16);
  if (moe_few(l, M)) {
    const size_t rows = (size_t)M * l.top_k, lds = few_lds_bytes(rows, 128 * (size_t)units) + rows * units * 16;
#define GQ_DOWN(MR, KS, PD)                                                                                              \
  hipLaunchKernelGGL((k_moe_down_few<FMT, MR, KS, group_stages<FMT>(PD)>), dim3(tiles), dim3(64 * (KS)), lds, s, (const uint8_t *)l.down, so, b.h16, b.hs, ids, \
                     weights, resid, y, dt, M, N, K, C, units, (int)l.n_experts, l.top_k)
    if (M == 1) GQ_DOWN(1, 16, 2);
    else GQ_DOWN(4, 16, 2);
#undef GQ_DOWN
    return gq_last_launch();
  }
  // Two tiles a workgroup, which share the rows of h: four of six loads a unit.  (16 tokens, 8 experts of 14336 x 4096, Q4_0, by one tile 167 us
  // the layer, by two in two parts 152, by four in four parts 147 - 149; 64 tokens, 128 experts of 768 x 2048, 127, 117 and 139 - 159.)
  constexpr int R = 2, KS = 8;
  const size_t P = (size_t)M * l.top_k, lds = (size_t)KS * M * 64 * R + P * 4 + (size_t)p.maxblk * ((2u << p.sh) + 2) + P + 16;
#define GQ_DOWN_ROWS(MT)                                                                                                                   \
  hipLaunchKernelGGL((k_moe_down_rows<FMT, MT, R, KS, group_stages<FMT>(2)>), dim3((tiles + R - 1) / R, (unsigned)b.parts), dim3(64 * KS), lds, s, \
                     (const uint8_t *)l.down, so, b.h16, b.ldh, b.hs, p, resid, y, dt, b.parts > 1 ? b.part : nullptr, M, K, C, units,      \
                     l.top_k, p.maxblk)
  if (p.sh == 4) GQ_DOWN_ROWS(1);
  else GQ_DOWN_ROWS(2);
#undef GQ_DOWN_ROWS
  return gq_last_launch();
}

// x goes in as it is: few rows of 16-bit values
bool moe_as_it_is(const gq_moe &l, int xt, int M) { return moe_few(l, M) && xt != GQ_DT_F32; }
MoeMid moe_mid(const gq_moe &l, const MoeWs &w, uint8_t *ws, int M) {
  return MoeMid{(_Float16 *)(ws + w.a16), (_Float16 *)(ws + w.h16), (float *)(ws + w.rs), (float *)(ws + w.h), (float *)(ws + w.hs),
                (float *)(ws + w.part), moe_few(l, M) ? (int)l.K : (int)gq_kpad(l.fmt, l.K) + 8, (int)gq_kpad(l.fmt_down, l.N) + 8, w.parts};
}
int moe_x_order(const gq_moe &l, int M) { return !moe_few(l, M) && (l.fmt == GQ_FMT_Q4_0 || gq_fmt_is_q4k(l.fmt)); }

// The products, x converted already where it has to be.  Few tokens: of the experts ids, or (a) of those that the logits choose, whose ids and
// weights come out in a->ids, a->weights.
int moe_products(const gq_moe &l, const void *x, int xt, const RouteArgs *a, const int *ids, const float *weights, const MoePlan &plan,
                 const MoeMid &b, const void *resid, void *y, int dt, int M, hipStream_t s) {
  const float *rs = nullptr;
  if (!moe_as_it_is(l, xt, M)) {
    x = b.a16;
    xt = GQ_DT_F16;
    rs = b.rs;
  }
#define GQ_GU_F(F) launch_gu_t<F>(l, x, xt, rs, a, ids, plan, b, M, s)
  if (l.fmt == GQ_FMT_Q4_0) GQ_TRY(GQ_GU_F(GQ_FMT_Q4_0));
  else if (l.fmt == GQ_FMT_Q8_0) GQ_TRY(GQ_GU_F(GQ_FMT_Q8_0));
  else if (gq_fmt_is_q6k(l.fmt)) GQ_TRY(GQ_GU_F(GQ_FMT_Q6_K));
  else GQ_TRY(GQ_GU_F(GQ_FMT_Q4_K));
#undef GQ_GU_F
  if (!moe_few(l, M))  // (h as the matrix cores take it, fp16 under a power of two per row: 2.1e-4 of it)
    GQ_TRY(gq_launch_a_to_f16(b.h, GQ_DT_F32, b.h16, b.hs, M * l.top_k, (int)l.N, b.ldh,
                              l.fmt_down == GQ_FMT_Q4_0 || gq_fmt_is_q4k(l.fmt_down), s));
#define GQ_DOWN_F(F) launch_down_t<F>(l, ids, weights, plan, b, resid, y, dt, M, s)
  if (l.fmt_down == GQ_FMT_Q4_0) GQ_TRY(GQ_DOWN_F(GQ_FMT_Q4_0));
  else if (l.fmt_down == GQ_FMT_Q8_0) GQ_TRY(GQ_DOWN_F(GQ_FMT_Q8_0));
  else if (gq_fmt_is_q6k(l.fmt_down)) GQ_TRY(GQ_DOWN_F(GQ_FMT_Q6_K));
  else GQ_TRY(GQ_DOWN_F(GQ_FMT_Q4_K));
#undef GQ_DOWN_F
  if (b.parts == 1) return GQ_OK;
  const int n = M * (int)l.K;
  hipLaunchKernelGGL(k_moe_sum, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, b.part, resid, y, dt, n, b.parts);
  return gq_last_launch();
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
  return MoePlan{(int *)(ws + w.nblk), (MoeBlk *)(ws + w.blk), (float *)(ws + w.wsum), w.maxblk, w.tiles == 1 ? 4 : 5, (int *)(ws + w.count)};
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
  double *logits = (double *)room.ptr;
  GQ_TRY(launch_logits(*l, x, x_dtype, logits, MoeConv{}, nullptr, (int)M, s));
  return launch_choose(*l, RouteArgs{logits, l->router_bias, ids, weights, l->score, l->renorm, l->scale}, (int)M, s);
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
  const MoeMid mid = moe_mid(*l, w, room.ptr, (int)M);
  if (!moe_few(*l, M)) GQ_TRY(launch_plan(*l, RouteArgs{}, ids, weights, plan, (int)M, s));
  if (!moe_as_it_is(*l, x_dtype, (int)M))
    GQ_TRY(gq_launch_a_to_f16(x, x_dtype, mid.a16, mid.rs, (int)M, (int)l->K, mid.lda, moe_x_order(*l, (int)M), s));
  return moe_products(*l, x, x_dtype, nullptr, ids, weights, plan, mid, resid, y, y_dtype, (int)M, s);
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
  const MoeMid mid = moe_mid(*l, w, room.ptr, (int)M);
  const MoeConv conv = moe_as_it_is(*l, x_dtype, (int)M) ? MoeConv{} : MoeConv{mid.a16, mid.rs, mid.lda, moe_x_order(*l, (int)M)};
  if (!ids) ids = (int32_t *)(room.ptr + w.ids);
  if (!weights) weights = (float *)(room.ptr + w.weights);
  RouteArgs a = {(double *)(room.ptr + w.logits), l->router_bias, ids, weights, l->score, l->renorm, l->scale};
  const bool few = moe_few(*l, M), within = few && l->n_experts <= 64 * kFewNE;
  GQ_TRY(launch_logits(*l, x, x_dtype, (double *)(room.ptr + w.logits), conv, few ? nullptr : plan.count, (int)M, s));
  // The choice, a wave a token: few tokens with the gate and up products, else with the plan (four tokens a wave of one workgroup, 64 of 128
  // experts: 22 us; a workgroup a token, the last of them making the plan, 8, in two launches 5 and 5)
  if (!few) GQ_TRY(launch_plan(*l, a, ids, weights, plan, (int)M, s));
  else if (!within) GQ_TRY(launch_choose(*l, a, (int)M, s));
  return moe_products(*l, x, x_dtype, within ? &a : nullptr, ids, weights, plan, mid, resid, y, y_dtype, (int)M, s);
}
