// gq_gemv_frag.h -- device pieces of the kernels that stream T16 weights (or fp16 rows)
// chunk by chunk into v_mfma_f32_16x16x32_f16: a chunk's loads and its dequantization into
// B fragments whose 16 columns are the rows of a row tile.
#pragma once
#include "gq_internal.h"

namespace {

template <int FMT>
struct HFmt;
template <>
struct HFmt<GQ_FMT_Q4_0> {
  static constexpr int CK = 128, QB = 1024, SB = 128, STEPS = 2;
};
template <>
struct HFmt<GQ_FMT_Q8_0> {
  static constexpr int CK = 128, QB = 2048, SB = 128, STEPS = 2;
};
template <>
struct HFmt<GQ_FMT_Q4_K> {
  static constexpr int CK = 256, QB = 2048, SB = 256, STEPS = 4;
};
template <>
struct HFmt<GQ_FMT_Q6_K> {
  static constexpr int CK = 256, QB = 3072, SB = 288, STEPS = 4;
};

// fp16 weights, row-major N x K (the reference's FP16 route, no T16 layout):
// a "chunk" is 128 k of one row tile, read straight from the 16 rows
template <>
struct HFmt<GQ_FMT_F16> {
  static constexpr int CK = 128, STEPS = 2;
  [[maybe_unused]] static constexpr int QB = 0, SB = 0;  // (no T16 records or scale plane)
};

template <int FMT>
struct HChunk;
template <>
struct HChunk<GQ_FMT_F16> {
  gq_u4 q[4];  // step m: q[2m], q[2m + 1] = the lane's 16 fp16 weights (halves 0, 1)
};
template <>
struct HChunk<GQ_FMT_Q4_0> {
  gq_u4 q;  // steps 0, 1: 8-byte code groups
  uint32_t d;
};
template <>
struct HChunk<GQ_FMT_Q8_0> {
  gq_u4 q0, q1;
  uint32_t d;
};
template <>
struct HChunk<GQ_FMT_Q4_K> {
  gq_u4 qa, qb;
  gq_u4 meta;
};
template <>
struct HChunk<GQ_FMT_Q6_K> {
  gq_u4 qa, qb;  // low-nibble code groups, steps 0,1 and 2,3
  gq_u4 hi;      // high 2-bit fields, one word per step
  gq_u4 sc;      // the row's 16 int8 scales
  uint32_t d;    // the row's fp16 d (low half)
};

template <int FMT>
GQ_DEV void load_hchunk(const uint8_t *qp, const uint8_t *sp, uint32_t qo, uint32_t so, HChunk<FMT> &ch) {
  if constexpr (FMT == GQ_FMT_Q4_0) {
    ch.q = gq_ld16_nt(qp + qo);
    ch.d = gq_ld4_nt(sp + so);
  } else if constexpr (FMT == GQ_FMT_Q8_0) {
    ch.q0 = gq_ld16_nt(qp + qo);
    ch.q1 = gq_ld16_nt(qp + 1024 + qo);
    ch.d = gq_ld4_nt(sp + so);
  } else if constexpr (FMT == GQ_FMT_Q4_K) {
    ch.qa = gq_ld16_nt(qp + qo);
    ch.qb = gq_ld16_nt(qp + 1024 + qo);
    ch.meta = gq_ld16_nt(sp + so);
  } else {  // Q6_K: so = 16 r
    ch.qa = gq_ld16_nt(qp + qo);
    ch.qb = gq_ld16_nt(qp + 1024 + qo);
    ch.hi = gq_ld16_nt(qp + 2048 + qo);
    ch.sc = gq_ld16_nt(sp + so);
    ch.d = gq_ld4_nt(sp + 256 + 4 * (so >> 5)) >> (16 * ((so >> 4) & 1));
  }
}

// Where a wave's chunks of one row tile come from: T16 records (chunk ci of
// the tile at q + ci * QB, its scales at s + ci * SB, this lane's offsets
// qo / so), or, for row-major fp16 weights, this lane's row (row tile rows
// past N read row N - 1, never stored) with the lane's k offset qo (bytes)
// and the row length K.
template <int FMT>
struct HSrc {
  const uint8_t *q, *s;
  uint32_t qo, so;
  int K;
};
template <int FMT>
GQ_DEV HSrc<FMT> hsrc(const uint8_t *w, size_t sc_off, size_t tile, int C, int N, int K, int lane) {
  const int g = lane >> 4, r = lane & 15;
  if constexpr (FMT == GQ_FMT_F16) {
    size_t n = tile * 16 + (size_t)r;
    n = n < (size_t)N ? n : (size_t)N - 1;
    return HSrc<FMT>{w + n * (size_t)K * 2, nullptr, 32u * (uint32_t)g, 0u, K};
  } else {
    using F = HFmt<FMT>;
    const uint32_t slane = (FMT == GQ_FMT_Q4_K || FMT == GQ_FMT_Q6_K) ? 16u * (uint32_t)r
                                                                      : 8u * (uint32_t)r + 4u * (uint32_t)(g >> 1);
    return HSrc<FMT>{w + tile * (size_t)C * F::QB, w + sc_off + tile * (size_t)C * F::SB, 16u * (uint32_t)lane,
                     slane, K};
  }
}

template <int FMT>
GQ_DEV void load_src(const HSrc<FMT> &src, int ci, HChunk<FMT> &ch) {
  if constexpr (FMT == GQ_FMT_F16) {
    // step m: k = 128 ci + 64 m + 16 g .. + 15 (K % 32 == 0: wholly in or out
    // of the row); a run past K reads the row's start and is zeroed
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint32_t kb = 2u * (uint32_t)(128 * ci + 64 * m) + src.qo;  // byte offset in the row
      const bool in = kb < 2u * (uint32_t)src.K;
      const uint8_t *p = src.q + (in ? kb : 0u);
      gq_u4 a = gq_ld16_nt(p), b = gq_ld16_nt(p + 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = in ? a[e] : 0u;
        b[e] = in ? b[e] : 0u;
      }
      ch.q[2 * m] = a;
      ch.q[2 * m + 1] = b;
    }
  } else {
    using F = HFmt<FMT>;
    load_hchunk<FMT>(src.q + (size_t)ci * F::QB, src.s + (size_t)ci * F::SB, src.qo, src.so, ch);
  }
}

// 4 byte values u (0..255) -> 2 fp16 pairs holding (1024 + u)
GQ_DEV void magic4(uint32_t u, gq_half2 &lo, gq_half2 &hi) {
  lo = gq_bits_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
  hi = gq_bits_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
}

GQ_DEV gq_half2 splat_h(uint32_t b16) { return gq_bits_h2((b16 & 0xFFFFu) * 0x10001u); }

// B fragment element e of a 4-bit format holds slot kQ4Perm[e]; elements with
// kQ4Div16 set are 16 x the weight
constexpr int kQ4Perm[8] = {0, 2, 4, 6, 1, 3, 5, 7};
constexpr bool kQ4Div16[8] = {false, false, true, true, false, false, true, true};
template <int FMT>
constexpr bool kNibOrder = FMT == GQ_FMT_Q4_0 || FMT == GQ_FMT_Q4_K;

GQ_DEV _Float16 bits_h(uint32_t b16) { return __builtin_bit_cast(_Float16, (uint16_t)(b16 & 0xFFFFu)); }

// The 16 weights a lane holds for MFMA step m -> fp16 B fragments (slots
// 0..7, 8..15; for the 4-bit formats in gq_nib_halves order).  g is the lane's
// 16-lane group: its 16 weights are half g & 1 of 32-block 2 m + (g >> 1) of
// the chunk (Q6_K: 16-element scale group 4 m + g).
template <int FMT>
GQ_DEV void dequant_step(const HChunk<FMT> &c, int m, int g, uint32_t mg, gq_half8 &o0, gq_half8 &o1) {
  if constexpr (FMT == GQ_FMT_F16) {
    o0 = __builtin_bit_cast(gq_half8, c.q[2 * m]);
    o1 = __builtin_bit_cast(gq_half8, c.q[2 * m + 1]);
    return;
  } else if constexpr (FMT == GQ_FMT_Q4_0 || FMT == GQ_FMT_Q4_K) {
    uint32_t w0, w1;
    gq_half2 a1, b1, a16, b16;  // (h * a + b) per pair; then * d2 + m2 (Q4_K)
    gq_half2 d2, m1, m16;
    if constexpr (FMT == GQ_FMT_Q4_0) {
      w0 = c.q[2 * m];
      w1 = c.q[2 * m + 1];
      // (q - 8) * d: the subtraction is exact, the product rounds once (and
      // 16 (q - 8) * d is 16 x that rounding)
      const _Float16 d = bits_h(m ? (c.d >> 16) : c.d);
      a1 = gq_half2{(_Float16)1.0f, (_Float16)1.0f};
      b1 = gq_half2{(_Float16)-1032.0f, (_Float16)-1032.0f};
      a16 = a1;
      b16 = gq_half2{(_Float16)-1152.0f, (_Float16)-1152.0f};
      d2 = gq_half2{d, d};
    } else {
      const gq_u4 &q = (m < 2) ? c.qa : c.qb;
      w0 = q[2 * (m & 1)];
      w1 = q[2 * (m & 1) + 1];
      // The lane's sub-blocks of steps 0..3 are 2 m + h (h = g >> 1): their
      // 6-bit scales are the low bits of the 4 bytes of meta word 1 + h, the
      // mins' low 2 bits the top bits of those bytes and their high 4 bits
      // nibble h of the bytes of meta word 3.  All four steps' factors are
      // decoded packed, two per instruction (the same values for every step
      // of a chunk, so the unrolled steps share them).
      const uint32_t h = (uint32_t)(g >> 1);
      const uint32_t wh = h ? c.meta[2] : c.meta[1];
      const uint32_t scb = wh & 0x3F3F3F3Fu;
      const uint32_t mnb = ((wh >> 6) & 0x03030303u) | (((c.meta[3] >> (4u * h)) & 0x0F0F0F0Fu) << 2);
      gq_half2 s01, s23, n01, n23;
      magic4(scb, s01, s23);
      magic4(mnb, n01, n23);
      const gq_half2 k1024 = {(_Float16)-1024.0f, (_Float16)-1024.0f};
      s01 = s01 + k1024;  // sc, exact
      s23 = s23 + k1024;
      n01 = n01 + k1024;  // m, exact
      n23 = n23 + k1024;
      // -(dmin m): the exact product rounded once, as (half)(-(float)dmin * m)
      const _Float16 ndmin = -bits_h(c.meta[0] >> 16);
      const gq_half2 nd2 = {ndmin, ndmin};
      const gq_half2 hm01 = n01 * nd2, hm23 = n23 * nd2;
      const gq_half2 k16 = {(_Float16)16.0f, (_Float16)16.0f};
      // (1024 + q) * sc - 1024 sc = q * sc exactly (<= 945; 16 q sc <= 15120,
      // a multiple of 16: exact too), then one rounding of q sc d - dmin m;
      // -1024 sc and 16 (-dmin m) are exact
      const gq_half2 sp = m < 2 ? s01 : s23, mp = m < 2 ? hm01 : hm23;
      const gq_half2 np = sp * k1024, mp16 = mp * k16;
      if (m & 1) {
        a1 = __builtin_shufflevector(sp, sp, 1, 1);
        b1 = __builtin_shufflevector(np, np, 1, 1);
        m1 = __builtin_shufflevector(mp, mp, 1, 1);
        m16 = __builtin_shufflevector(mp16, mp16, 1, 1);
      } else {
        a1 = __builtin_shufflevector(sp, sp, 0, 0);
        b1 = __builtin_shufflevector(np, np, 0, 0);
        m1 = __builtin_shufflevector(mp, mp, 0, 0);
        m16 = __builtin_shufflevector(mp16, mp16, 0, 0);
      }
      a16 = a1;
      b16 = b1;
      const _Float16 d = bits_h(c.meta[0]);
      d2 = gq_half2{d, d};
    }
#pragma unroll
    for (int hw = 0; hw < 2; ++hw) {
      gq_half2 p[4];
      gq_nib_halves(hw ? w1 : w0, mg, p);
      gq_half8 &o = hw ? o1 : o0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool x16 = q & 1;
        gq_half2 t;
        if constexpr (FMT == GQ_FMT_Q4_0) {
          t = (p[q] + (x16 ? b16 : b1)) * d2;
        } else {
          t = __builtin_elementwise_fma(__builtin_elementwise_fma(p[q], x16 ? a16 : a1, x16 ? b16 : b1), d2,
                                        x16 ? m16 : m1);
        }
        o[2 * q] = t[0];
        o[2 * q + 1] = t[1];
      }
    }
    return;
  } else {
  const int j = 2 * m + (g >> 1);
  (void)j;
  uint32_t regs[4];
  gq_half2 off, d2;
  if constexpr (FMT == GQ_FMT_Q6_K) {
    const gq_u4 &q = (m < 2) ? c.qa : c.qb;
    const uint32_t w0 = q[2 * (m & 1)], w1 = q[2 * (m & 1) + 1], hw = c.hi[m];
    regs[0] = w0 & 0x0F0F0F0Fu;
    regs[1] = (w0 >> 4) & 0x0F0F0F0Fu;
    regs[2] = w1 & 0x0F0F0F0Fu;
    regs[3] = (w1 >> 4) & 0x0F0F0F0Fu;
#pragma unroll
    for (int i = 0; i < 4; ++i) regs[i] |= ((hw >> (2 * i)) & 0x03030303u) << 4;  // codes 0..63
    // (c - 32) * (d * scale): the scale product rounded to fp16, then one
    // rounding of the exact (c - 32) * that
    const float sc = (float)(int8_t)((c.sc[m] >> (8 * g)) & 0xFFu);
    const _Float16 hs = (_Float16)((float)bits_h(c.d) * sc);
    off = gq_half2{(_Float16)-1056.0f, (_Float16)-1056.0f};
    d2 = gq_half2{hs, hs};
  } else {  // Q8_0
    const gq_u4 &q = m ? c.q1 : c.q0;
#pragma unroll
    for (int i = 0; i < 4; ++i) regs[i] = q[i] ^ 0x80808080u;
    off = gq_half2{(_Float16)-1152.0f, (_Float16)-1152.0f};
    d2 = splat_h(m ? (c.d >> 16) : c.d);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    gq_half2 lo, hi;
    magic4(regs[q], lo, hi);
    lo = (lo + off) * d2;  // exact (q - bias), one rounding of the product
    hi = (hi + off) * d2;
    gq_half8 &o = (q < 2) ? o0 : o1;
    const int b = 4 * (q & 1);
    o[b] = lo[0];
    o[b + 1] = lo[1];
    o[b + 2] = hi[0];
    o[b + 3] = hi[1];
  }
  }
}

GQ_DEV gq_f4 mfma16h(const gq_half8 &a, const gq_half8 &b, const gq_f4 &c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

}  // namespace
