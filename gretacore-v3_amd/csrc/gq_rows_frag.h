// gq_rows_frag.h -- device pieces of the kernels that take few rows of x over T16 weights in units
// of 128 k, and of the tiled kernels' steps and stores.
#pragma once
#include "gq_act.h"
#include "gq_gemv_frag.h"

namespace {

// A unit is 128 k of a row tile: a chunk of Q4_0 / Q8_0, half a super-block of the
// k-quants; it is loaded through buffer resources that end with the tile, so a unit past the
// last one fetches nothing and needs no branch.
template <int FMT>
struct FUnit {
  gq_u4 q[FMT == GQ_FMT_Q8_0 ? 2 : 1];  // codes of the two 64-k steps (lane 16 g + r: row r, k 16 g .. + 15)
  gq_u4 s;  // Q4_0 / Q8_0: d0 d2 | d1 d3; Q4_K: meta; Q6_K: high fields of the steps | their scales
  uint32_t d;  // Q6_K: d
};
template <int FMT>
constexpr bool kSuper = FMT == GQ_FMT_Q4_K || FMT == GQ_FMT_Q6_K;

template <int FMT>
struct FTile {
  __amdgpu_buffer_rsrc_t q, s;
};
template <int FMT>
GQ_DEV FTile<FMT> ftile(const uint8_t *w, size_t sc_off, size_t tile, int C) {
  using F = HFmt<FMT>;
  uint8_t *p = const_cast<uint8_t *>(w);
  return FTile<FMT>{
      __builtin_amdgcn_make_buffer_rsrc(p + tile * (size_t)C * F::QB, (short)0, C * F::QB, 0x00020000),
      __builtin_amdgcn_make_buffer_rsrc(p + sc_off + tile * (size_t)C * F::SB, (short)0, C * F::SB, 0x00020000)};
}
GQ_DEV gq_u4 ld16_r(const __amdgpu_buffer_rsrc_t &r, uint32_t o) {  // (streamed: read once)
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, o, 0, 2);
  return gq_u4{v[0], v[1], v[2], v[3]};
}
template <int FMT>
GQ_DEV void load_unit(const FTile<FMT> &t, int unit, int lane, FUnit<FMT> &u) {
  using F = HFmt<FMT>;
  const uint32_t c = (uint32_t)(kSuper<FMT> ? unit >> 1 : unit), p = kSuper<FMT> ? (uint32_t)unit & 1u : 0u;
  const uint32_t qo = c * F::QB + 1024u * p + 16u * (uint32_t)lane, so = c * F::SB, r = (uint32_t)lane & 15u;
  u.q[0] = ld16_r(t.q, qo);
  if constexpr (FMT == GQ_FMT_Q8_0) u.q[1] = ld16_r(t.q, qo + 1024u);
  if constexpr (FMT == GQ_FMT_Q4_K) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(t.s, so + 16u * r, 0, 0);
    u.s = gq_u4{v[0], v[1], v[2], v[3]};
  } else if constexpr (FMT == GQ_FMT_Q6_K) {
    const auto h = __builtin_amdgcn_raw_buffer_load_b64(t.q, c * F::QB + 2048u + 16u * (uint32_t)lane + 8u * p, 0, 0);
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(t.s, so + 16u * r + 8u * p, 0, 0);
    u.s = gq_u4{h[0], h[1], v[0], v[1]};
    u.d = __builtin_amdgcn_raw_buffer_load_b16(t.s, so + 256u + 2u * r, 0, 0);
  } else {
    const auto v = __builtin_amdgcn_raw_buffer_load_b64(t.s, so + 8u * r, 0, 0);
    u.s[0] = v[0];
    u.s[1] = v[1];
  }
}
// What a wave loads at a time: a unit, of the k-quants both units of a super-block, whose scales come with one load each (Q4_K three loads for
// two units in place of four, Q6_K five of eight; a CU's loads count as much as their bytes).
template <int FMT>
constexpr int kGroup = kSuper<FMT> ? 2 : 1;
// stages of a pipeline `units` deep
template <int FMT>
constexpr int group_stages(int units) {
  return units / kGroup<FMT> > 0 ? units / kGroup<FMT> : 1;
}
template <int FMT>
GQ_DEV void load_group(const FTile<FMT> &t, int group, int lane, FUnit<FMT> (&u)[kGroup<FMT>]) {
  using F = HFmt<FMT>;
  if constexpr (!kSuper<FMT>) {
    load_unit<FMT>(t, group, lane, u[0]);
  } else {
    const uint32_t c = (uint32_t)group, qo = c * F::QB + 16u * (uint32_t)lane, so = c * F::SB, r = (uint32_t)lane & 15u;
    u[0].q[0] = ld16_r(t.q, qo);
    u[1].q[0] = ld16_r(t.q, qo + 1024u);
    if constexpr (FMT == GQ_FMT_Q4_K) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(t.s, so + 16u * r, 0, 0);
      u[0].s = u[1].s = gq_u4{v[0], v[1], v[2], v[3]};
    } else {
      const gq_u4 h = ld16_r(t.q, qo + 2048u);
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(t.s, so + 16u * r, 0, 0);
      u[0].s = gq_u4{h[0], h[1], v[0], v[1]};
      u[1].s = gq_u4{h[2], h[3], v[2], v[3]};
      u[0].d = u[1].d = __builtin_amdgcn_raw_buffer_load_b16(t.s, so + 256u + 2u * r, 0, 0);
    }
  }
}
// Q4_K: scale and min codes of sub-blocks i of the unit's two steps, a byte each (p: the unit's half)
GQ_DEV void unit_codes_q4k(const FUnit<GQ_FMT_Q4_K> &u, uint32_t p, bool i, uint32_t &sc, uint32_t &mn) {
  const uint32_t w = (i ? u.s[2] : u.s[1]) >> (16u * p), m = u.s[3] >> (16u * p + (i ? 4u : 0u));
  sc = w & 0x3F3Fu;
  mn = ((w >> 6) & 0x0303u) | ((m & 0x0F0Fu) << 2);
}
// Q6_K: the 8 codes 8 j .. + 7 of step m as bytes (byte b of the high fields' word holds slot 4 q + b at
// bits 2 q)
GQ_DEV void unit_codes_q6k(const FUnit<GQ_FMT_Q6_K> &u, int m, int j, uint32_t (&o)[2]) {
  const uint32_t w = u.q[0][2 * m + j], h = u.s[m];
  o[0] = (w & 0x0F0F0F0Fu) | ((j ? h : h << 4) & 0x30303030u);
  o[1] = ((w >> 4) & 0x0F0F0F0Fu) | ((j ? h >> 2 : h << 2) & 0x30303030u);
}
// 8 values in the nibbles' order 0 2 4 6 1 3 5 7
GQ_DEV gq_u4 nib_order(const gq_u4 &v) {
  return gq_u4{__builtin_amdgcn_perm(v[1], v[0], 0x05040100u), __builtin_amdgcn_perm(v[3], v[2], 0x05040100u),
               __builtin_amdgcn_perm(v[1], v[0], 0x07060302u), __builtin_amdgcn_perm(v[3], v[2], 0x07060302u)};
}

// The units of a wave: request(unit, stage) and compute(unit, stage), PD stages, the first requests
// apart from the rest.  A group of PD units requests the next one unless it is the last: no branch within a group, around which the
// compiler would wait for every load.
template <int PD, int KS, typename Request>
GQ_DEV void walk_requests(int units, int wave, Request request) {
#pragma unroll
  for (int i = 0; i < PD; ++i) request(min(wave + KS * i, units), i);
}
template <int PD, int KS, typename Request, typename Compute>
GQ_DEV void walk_computes(int units, int wave, Request request, Compute compute) {
  const int n = units > wave ? (units - wave + KS - 1) / KS : 0;
  int j = 0;
  for (; j + PD < n; j += PD) {
#pragma unroll
    for (int i = 0; i < PD; ++i) {
      compute(wave + KS * (j + i), i);
      request(min(wave + KS * (j + i + PD), units), i);
    }
  }
#pragma unroll
  for (int i = 0; i < PD; ++i)
    if (j + i < n) compute(wave + KS * (j + i), i);
}
template <int PD, int KS, typename Request, typename Compute>
GQ_DEV void walk_units(int units, int wave, Request request, Compute compute) {
  walk_requests<PD, KS>(units, wave, request);
  walk_computes<PD, KS>(units, wave, request, compute);
}

struct __attribute__((packed, aligned(2))) FRun16 {  // 8 values at any 2-byte address
  gq_u4 v;
};
// Up to 4 rows: nothing comes before the weights.  x enters the matrix cores as it is (bf16 or
// f16, no conversion launch), and so do the codes, as the 16-bit floats OFF + q; scales and
// minima are applied in fp32 to the sums of each scale group,
//   y += s (sum x (OFF + q) - OFF sum x) - min sum x,  sum x from a product with ones.
// A product of v_mfma_f32_16x16x32 spans NG scale groups (lane groups g / (4 / NG)).  The rows of the
// A operand keep them apart: row 4 i + j holds row j of x masked to group i, and lane group i
// of the result the sums of group i.  One load of x a unit: lane 16 g + 4 b + j takes row j, step b / 2, half
// b % 2 of its 16 k, and moves of whole quads bring a step's half to the operand's rows (four loads
// a unit in the operand's order: 19.4 us against 13.9 without any, 14336 x 4096 Q4_K).  MR: 1 or 4
// rows, the components of the result that are scaled and added.
template <int FMT>
constexpr int kFewGroups = FMT == GQ_FMT_Q6_K ? 4 : 2;
template <int FMT, int XT>
constexpr float kFewOff = (FMT == GQ_FMT_Q8_0 && XT == GQ_DT_BF16 ? 0.f
                           : XT == GQ_DT_BF16                     ? 128.f
                                                                  : 1024.f) +
                          (FMT == GQ_FMT_Q4_0                          ? 8.f
                           : FMT == GQ_FMT_Q6_K                        ? 32.f
                           : FMT == GQ_FMT_Q8_0 && XT == GQ_DT_F16 ? 128.f
                                                                       : 0.f);

typedef __bf16 few_bf8 __attribute__((ext_vector_type(8)));
template <int XT>
GQ_DEV gq_f4 few_mfma(const gq_u4 &a, const gq_u4 &b, const gq_f4 &c) {
  if constexpr (XT == GQ_DT_F16) return gq_mfma16(__builtin_bit_cast(gq_half8, a), __builtin_bit_cast(gq_half8, b), c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(few_bf8, a), __builtin_bit_cast(few_bf8, b), c, 0, 0,
                                                   0);
}
// The lane's 16 codes of step m as B operands of slots 0..7 and 8..15, the 4-bit formats in the
// nibbles' order
template <int FMT, int XT>
GQ_DEV void few_codes(const FUnit<FMT> &u, int m, uint32_t mg, gq_u4 (&o)[2]) {
  if constexpr (FMT == GQ_FMT_Q8_0 && XT == GQ_DT_BF16) {  // whole numbers of 8 bits
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t q = u.q[m][i];
      uint32_t f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __float_as_uint((float)(int8_t)(q >> (8 * e)));
      o[i >> 1][2 * (i & 1)] = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
      o[i >> 1][2 * (i & 1) + 1] = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
    }
  } else if constexpr (FMT == GQ_FMT_Q8_0 || FMT == GQ_FMT_Q6_K) {  // bytes: Q8_0 1024 + 128 + q
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t c[2];
      if constexpr (FMT == GQ_FMT_Q6_K) {
        unit_codes_q6k(u, m, j, c);
      } else {
        c[0] = u.q[m][2 * j] ^ 0x80808080u;
        c[1] = u.q[m][2 * j + 1] ^ 0x80808080u;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        o[j][2 * i] = __builtin_amdgcn_perm(mg, c[i], 0x05010500u);
        o[j][2 * i + 1] = __builtin_amdgcn_perm(mg, c[i], 0x05030502u);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = ((u.q[0][2 * m + j] >> (4 * i)) & 0x000F000Fu) | mg;
  }
}
// Scale and minimum (Q4_K) of the lane's row for scale group i of the two steps
template <int FMT>
GQ_DEV void few_scales(const FUnit<FMT> &u, int unit, int i, float (&s)[2], float (&mn)[2]) {
  if constexpr (FMT == GQ_FMT_Q4_K) {
    uint32_t sc, mc;
    unit_codes_q4k(u, (uint32_t)unit & 1u, i, sc, mc);
    const float d = (float)bits_h(u.s[0]), dm = (float)bits_h(u.s[0] >> 16);
    s[0] = d * (float)(sc & 255u);
    s[1] = d * (float)(sc >> 8);
    mn[0] = dm * (float)(mc & 255u);
    mn[1] = dm * (float)(mc >> 8);
  } else {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      mn[m] = 0.f;
      if constexpr (FMT == GQ_FMT_Q6_K) s[m] = (float)bits_h(u.d) * (float)(int8_t)(u.s[2 + m] >> (8 * i));
      else s[m] = (float)bits_h((i ? u.s[1] : u.s[0]) >> (16 * m));
    }
  }
}
// acc += what a step's product d, of the codes with their offset, and sum sx of x come to under the scale group's scale and minimum
template <int FMT, int XT, int MR>
GQ_DEV void few_scaled(float s, float mn, const gq_f4 &d, const gq_f4 &sx, float (&acc)[MR]) {
  constexpr float OFF = kFewOff<FMT, XT>;
  const float o = FMT == GQ_FMT_Q4_K ? fmaf(s, OFF, mn) : 0.f;
#pragma unroll
  for (int v = 0; v < MR; ++v) {
    if constexpr (FMT == GQ_FMT_Q4_K) acc[v] = fmaf(s, d[v], fmaf(-o, sx[v], acc[v]));
    else acc[v] = fmaf(s, OFF != 0.f ? fmaf(-OFF, sx[v], d[v]) : d[v], acc[v]);
  }
}
// Rows 4 I + j of the operand: quad Q of x in the lane groups of scale group I, the others as in old
template <int NG, int I, int Q>
GQ_DEV uint32_t few_quad(uint32_t old, uint32_t src) {
  constexpr int n = 4 * ((I - Q + 4) % 4), rows = NG == 4 ? 1 << I : 3 << (2 * I);
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)src, n ? 0x120 + n : 0xE4, rows, 1 << I, false);
}
template <int NG, int Q>
GQ_DEV gq_u4 few_operand(const gq_u4 &x) {
  gq_u4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t v = few_quad<NG, 1, Q>(few_quad<NG, 0, Q>(0u, x[e]), x[e]);
    if constexpr (NG == 4) v = few_quad<NG, 3, Q>(few_quad<NG, 2, Q>(v, x[e]), x[e]);
    o[e] = v;
  }
  return o;
}

// The same operands from x in LDS, where the rows fit it: a lane whose row and group do not belong together reads zeros.  Rows of 16-bit
// values (for the 4-bit formats in the nibbles' order) lie `stride` bytes apart, `zero` is the offset of 160 zero bytes behind them.
// (Moves between lanes for every unit: 32 or 64 instructions of 131 to 180 a unit of one row.)
template <int FMT>
GQ_DEV bool few_mine(int lane) {  // row lane % 4 is of this lane's scale group
  const int i = (lane >> 2) & 3, g = lane >> 4;
  return kFewGroups<FMT> == 4 ? i == g : i == g >> 1;
}
// operand of step m, half j of the unit whose 128 values start at offset `at` (of lane group 0)
GQ_DEV gq_u4 few_lds(const uint8_t *xs, uint32_t at, int m, int j) {
  return *reinterpret_cast<const gq_u4 *>(xs + at + 128 * m + 16 * j);
}
// acc += unit `unit` of T tiles, us[t][p], times x at `at` of LDS
template <int FMT, int XT, int T, int MR, int G>
GQ_DEV void few_add(const FUnit<FMT> (&us)[T][G], int p, int unit, int g, const uint8_t *xs, uint32_t at, uint32_t mg, float (&acc)[T][MR]) {
  constexpr uint32_t one = XT == GQ_DT_F16 ? 0x3C003C00u : 0x3F803F80u;
  const gq_u4 ones = {one, one, one, one};
  const gq_f4 zero = {0.f, 0.f, 0.f, 0.f};
  float s[T][2], mn[T][2];
#pragma unroll
  for (int t = 0; t < T; ++t) few_scales<FMT>(us[t][p], unit, g & (kFewGroups<FMT> - 1), s[t], mn[t]);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const gq_u4 a0 = few_lds(xs, at, m, 0), a1 = few_lds(xs, at, m, 1);
    gq_f4 sx = zero;
    if constexpr (kFewOff<FMT, XT> != 0.f || FMT == GQ_FMT_Q4_K) sx = few_mfma<XT>(a1, ones, few_mfma<XT>(a0, ones, zero));
#pragma unroll
    for (int t = 0; t < T; ++t) {
      gq_u4 b[2];
      few_codes<FMT, XT>(us[t][p], m, mg, b);
      few_scaled<FMT, XT>(s[t][m], mn[t][m], few_mfma<XT>(a1, b[1], few_mfma<XT>(a0, b[0], zero)), sx, acc[t]);
    }
  }
}
// Copies rows of `n` 16-bit values (n % 32 == 0, row r at src + r * n) to LDS, zeros up to np, nib: in the nibbles' order, by T threads.
// ahead() is called between the last loads and their stores: what it requests is under way while they are waited for.
template <int T, typename Ahead>
GQ_DEV void few_stage(const void *src, int rows, int n, int np, int stride, bool nib, uint8_t *xs, int tid, Ahead ahead) {
  constexpr int RUNS = 4;
  const int per = np / 8, all = rows * per;  // (below 2^20: i / per from a float is exact)
  const float inv = 1.0f / (float)per;
  auto at = [&](int i, int &r, int &k) __attribute__((always_inline)) {
    r = (int)(((float)i + 0.5f) * inv);
    k = 8 * (i - r * per);
  };
  if (tid < 40) *reinterpret_cast<uint32_t *>(xs + (size_t)rows * stride + 4 * tid) = 0;
  for (int i0 = 0; i0 < all; i0 += T * RUNS) {
    FRun16 v[RUNS];
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
      const int i = i0 + tid + T * u;
      int r, k;
      at(i, r, k);
      v[u] = *reinterpret_cast<const FRun16 *>(reinterpret_cast<const uint16_t *>(src) +
                                               (i < all && k < n ? (size_t)r * (size_t)n + k : 0));
    }
    __builtin_amdgcn_sched_barrier(0);
    if (i0 + T * RUNS >= all) ahead();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
      const int i = i0 + tid + T * u;
      int r, k;
      at(i, r, k);
      gq_u4 o = nib ? nib_order(v[u].v) : v[u].v;
      if (k >= n) o = gq_u4{0, 0, 0, 0};
      if (i < all) *reinterpret_cast<gq_u4 *>(xs + (size_t)r * stride + 2 * k) = o;
    }
  }
}
// bytes of LDS they take
GQ_LHD size_t few_lds_stride(size_t np) { return 2 * np + 16; }
GQ_LHD size_t few_lds_bytes(size_t rows, size_t np) { return rows * few_lds_stride(np) + 160; }

// More rows: the sums of the scale groups would cost more than folding the scale into the
// weights; the matrix cores then add over a unit or all of K.  Q4_0 and Q8_0: d (q - bias), rounded once
// to fp16.  The k-quants keep their d (and dmin) out, one of each to a row and unit, applied in fp32
// to the unit's sums: sc q is exact in fp16, sc (q - 32) but for the few beyond 2048, and the minima
// are a product of their own, of x with their codes.  x comes as fp16 with a power-of-two scale per row (for the
// 4-bit formats in their nibbles' order, where every other pair is x / 16 and its weight 16 x).
template <int FMT>
GQ_DEV void rows_frags(const FUnit<FMT> &u, int unit, int g, uint32_t mg, gq_half8 (&o)[2][2], gq_half8 (&mins)[2]) {
  uint32_t sc = 0, mc = 0;
  if constexpr (FMT == GQ_FMT_Q4_K) unit_codes_q4k(u, (uint32_t)unit & 1u, g >> 1, sc, mc);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    gq_half2 d2, b1;
    if constexpr (FMT == GQ_FMT_Q4_K) {
      const _Float16 s = (_Float16)(float)((sc >> (8 * m)) & 255u), c = (_Float16)(float)((mc >> (8 * m)) & 255u);
      const _Float16 ns = s * (_Float16)-1024.0f, c16 = c * (_Float16)16.0f;
      d2 = gq_half2{s, s};
      b1 = gq_half2{ns, ns};
      mins[m] = gq_half8{c, c, c16, c16, c, c, c16, c16};
    } else if constexpr (FMT == GQ_FMT_Q6_K) {
      const _Float16 s = (_Float16)(float)(int8_t)(u.s[2 + m] >> (8 * g));
      d2 = gq_half2{s, s};
    } else {
      d2 = splat_h((g >> 1 ? u.s[1] : u.s[0]) >> (16 * m));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      gq_half2 p[4];
      if constexpr (FMT == GQ_FMT_Q8_0) {
        magic4(u.q[m][2 * j] ^ 0x80808080u, p[0], p[1]);
        magic4(u.q[m][2 * j + 1] ^ 0x80808080u, p[2], p[3]);
      } else if constexpr (FMT == GQ_FMT_Q6_K) {
        uint32_t c[2];
        unit_codes_q6k(u, m, j, c);
        magic4(c[0], p[0], p[1]);
        magic4(c[1], p[2], p[3]);
      } else {
        gq_nib_halves(u.q[0][2 * m + j], mg, p);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (FMT == GQ_FMT_Q4_K) {
          p[i] = __builtin_elementwise_fma(p[i], d2, b1);  // sc q (or 16 sc q), exact
        } else {
          const float off = FMT == GQ_FMT_Q8_0 ? -1152.f : FMT == GQ_FMT_Q6_K ? -1056.f : i & 1 ? -1152.f : -1032.f;
          p[i] = (p[i] + gq_half2{(_Float16)off, (_Float16)off}) * d2;  // (the sum is exact)
        }
        o[m][j][2 * i] = p[i][0];
        o[m][j][2 * i + 1] = p[i][1];
      }
    }
  }
}
// acc += the unit's products with x (its four fragments xs[t])
template <int FMT, int MT>
GQ_DEV void rows_add(const FUnit<FMT> &u, int unit, int g, uint32_t mg, const gq_half8 (&xs)[MT][4], gq_f4 (&acc)[MT]) {
  gq_half8 b[2][2], mins[2];
  rows_frags<FMT>(u, unit, g, mg, b, mins);
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if constexpr (!kSuper<FMT>) {
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[t] = gq_mfma16(xs[t][f], b[f >> 1][f & 1], acc[t]);
    } else {
      const float d = (float)bits_h(FMT == GQ_FMT_Q4_K ? u.s[0] : u.d);
      gq_f4 y = {0.f, 0.f, 0.f, 0.f}, z = y;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        y = gq_mfma16(xs[t][f], b[f >> 1][f & 1], y);
        if constexpr (FMT == GQ_FMT_Q4_K) z = gq_mfma16(xs[t][f], mins[f >> 1], z);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        acc[t][v] = fmaf(d, y[v], acc[t][v]);
        if constexpr (FMT == GQ_FMT_Q4_K) acc[t][v] = fmaf(-(float)bits_h(u.s[0] >> 16), z[v], acc[t][v]);
      }
    }
  }
}

struct __attribute__((packed, aligned(4))) FRun32 {
  gq_f4 v[2];
};
// a run of 8 values of x as it lies in memory, and as floats (zeros where !in)
template <int XT>
struct FRaw {
  gq_u4 v[XT == GQ_DT_F32 ? 2 : 1];
};
template <int XT>
GQ_DEV void px_load(const void *x, size_t at, FRaw<XT> &r) {
  if constexpr (XT == GQ_DT_F32) {
    const FRun32 t = *reinterpret_cast<const FRun32 *>(reinterpret_cast<const float *>(x) + at);
    r.v[0] = __builtin_bit_cast(gq_u4, t.v[0]);
    r.v[1] = __builtin_bit_cast(gq_u4, t.v[1]);
  } else {
    r.v[0] = reinterpret_cast<const FRun16 *>(reinterpret_cast<const uint16_t *>(x) + at)->v;
  }
}
template <int XT>
GQ_DEV void px_floats(const FRaw<XT> &r, bool in, float (&o)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float f;
    if constexpr (XT == GQ_DT_F32) f = __uint_as_float(r.v[e >> 2][e & 3]);
    else if constexpr (XT == GQ_DT_BF16) f = __uint_as_float(e & 1 ? r.v[0][e >> 1] & 0xFFFF0000u : r.v[0][e >> 1] << 16);
    else f = (float)gq_bits_h2(r.v[0][e >> 1])[e & 1];
    o[e] = in ? f : 0.f;
  }
}

// The tiles of a workgroup: request(tile, slot) ahead, compute(slot), then finish(tile) with the sums
template <int NU, typename Load, typename Request, typename Begin, typename Compute, typename Finish>
GQ_DEV void walk_tiles(int ntiles, Load load_x, Request request, Begin begin, Compute compute, Finish finish) {
  int tile = blockIdx.x;
  load_x();  // (before the first requests: behind them its loads would wait for theirs)
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < NU; ++i) request(tile, i);
  __builtin_amdgcn_sched_barrier(0);
  begin();
  int buf = 0;
  for (; tile < ntiles; tile += gridDim.x) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      compute(i);
      request(tile + (int)gridDim.x, i);  // (past the last tile: nothing is fetched)
    }
    finish(tile, buf);
    buf ^= 1;
  }
}

template <int DT>
GQ_DEV void front_put(const __amdgpu_buffer_rsrc_t &r, uint32_t o, int dt, float v) {
  if constexpr (DT == GQ_DT_F32)
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, o, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b16(
        dt == GQ_DT_BF16 ? gq_f32_to_bf16(v) : __builtin_bit_cast(uint16_t, (_Float16)v), r, o, 0, 0);
}

// A step's end.  Waits for this wave's LDS DMAs but the VM youngest loads (which the caller counts) and for its
// LDS operations, then for the other waves.  __syncthreads would wait for every DMA, those of later
// steps too: its fence counts them as writes to LDS.  (k_front_dx in Q4_K and Q6_K still waits for
// them in some of its steps: the compiler does so between two stores of the scale tables, which lie in the
// DMAs' arrays and are too many for it to tell apart.)
template <int VM>
GQ_DEV void step_barrier() {
  static_assert(VM <= 63, "vmcnt immediate");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (VM & 15) | ((VM >> 4) << 14));  // vmcnt(VM) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// waves per SIMD: what a workgroup brings, at least two
constexpr int front_wpe(int waves) { return waves > 4 ? waves / 4 : 2; }

// Columns n0 .. n0 + COLS - 1 of c, thread (lane, group): GROUPS groups add parts g, g + GROUPS, ... in 64 bits, then the groups in order
template <int COLS, int GROUPS>
GQ_DEV void gq_col_sums(const GqColSums &c, int n0, int lane, int group, double (*red)[COLS]) {
  const int n = n0 + lane;
  double v = 0.0;
  if (n < c.n) {
#pragma unroll 8
    for (int p = group; p < c.parts; p += GROUPS) v += (double)c.part[(size_t)p * (size_t)c.n + n];
  }
  red[group][lane] = v;
  __syncthreads();
  if (group > 0 || n >= c.n) return;
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) v += red[g][lane];
  c.db[n] = (float)v;
}

// 8 values of a row of n from column k on (zeros behind it)
template <int DT>
GQ_DEV void dgu_load(const void *p, size_t row, int k, int n, float (&o)[8]) {
  if (k + 8 <= n) {
    FRaw<DT> r;
    px_load<DT>(p, row + k, r);
    px_floats<DT>(r, true, o);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = k + e < n ? gq_ld_dt(p, DT, row + k + e) : 0.f;
  }
}
template <int DT>
GQ_DEV void dgu_store(void *p, size_t row, int k, int n, const float (&v)[8]) {
  if (k + 8 <= n) {
    if constexpr (DT == GQ_DT_F32) {
      FRun32 r;
      r.v[0] = gq_f4{v[0], v[1], v[2], v[3]};
      r.v[1] = gq_f4{v[4], v[5], v[6], v[7]};
      *reinterpret_cast<FRun32 *>(reinterpret_cast<float *>(p) + row + k) = r;
    } else {
      FRun16 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = DT == GQ_DT_BF16 ? gq_f32_to_bf16(v[2 * e]) : __builtin_bit_cast(uint16_t, (_Float16)v[2 * e]);
        const uint32_t hi =
            DT == GQ_DT_BF16 ? gq_f32_to_bf16(v[2 * e + 1]) : __builtin_bit_cast(uint16_t, (_Float16)v[2 * e + 1]);
        r.v[e] = lo | hi << 16;
      }
      *reinterpret_cast<FRun16 *>(reinterpret_cast<uint16_t *>(p) + row + k) = r;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < n) gq_st_dt(p, DT, row + k + e, v[e]);
  }
}

struct __attribute__((packed, aligned(2))) FRun16h {  // 4 values
  gq_u2 v;
};
struct __attribute__((packed, aligned(4))) FRun32h {
  gq_f4 v;
};

}  // namespace
