// gq_gemm_frag.h -- device pieces of the GEMMs over T16 weights that keep the
// weight operand in registers: tile order, swizzled activation tiles, weight
// records of a K step and their dequantization into MFMA B fragments.
#pragma once
#include "gq_internal.h"

namespace {

constexpr int BK = 64;

GQ_DEV gq_half2 h2_of_bits16(uint32_t b16) {
  uint32_t v = (b16 & 0xFFFFu) * 0x10001u;
  return gq_bits_h2(v);
}

// 4 byte values u (0..255) -> 2 fp16 pairs holding (1024 + u)
GQ_DEV void bytes_to_magic(uint32_t u, gq_half2 &lo, gq_half2 &hi) {
  lo = gq_bits_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
  hi = gq_bits_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
}

// A K step of the tile is BM rows x 8 chunks of 16 B.  One wave instruction
// fills 8 consecutive rows (1 KiB of LDS, lane l at byte 16 l).  Logical chunk
// c of row j sits in physical chunk c ^ swz(j), swz(j) = (j ^ (j >> 3)) & 7 on
// the row index mod 32: any 8 (or 16) consecutive rows then read the same
// logical chunk from 8 (16) different bank groups, for 32 or 64 LDS banks.
GQ_DEV int a_swz(int row) { return (row ^ ((row >> 3) & 3)) & 7; }

GQ_DEV uint16_t f32_to_bf16_rne(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7F800000u) == 0x7F800000u) return (uint16_t)((u >> 16) | ((u & 0xFFFFu) ? 0x40u : 0u));
  u += 0x7FFFu + ((u >> 16) & 1u);
  return (uint16_t)(u >> 16);
}


// Workgroup tile -> (m tile, n tile): ids are spread over the 8 XCDs
// round-robin, so id -> (id mod 8) * (G / 8) + id / 8 gives each XCD a
// contiguous range of tile indices; consecutive indices walk the M tiles of one
// weight column tile.
GQ_DEV void tile_of(int id, int G, int tiles_m, int &mt, int &nt) {
  const int t = (G % 8 == 0) ? (id % 8) * (G / 8) + id / 8 : id;
  nt = t / tiles_m;
  mt = t % tiles_m;
}
// The same with the tile index walked in groups of gm M tiles: within a group,
// consecutive indices walk its M tiles, then the next weight column tile, so
// the workgroups resident on one XCD at a time share fewer activation rows
// (gm <= 0: tile_of).
GQ_DEV void tile_of_g(int id, int G, int tiles_m, int tiles_n, int gm, int &mt, int &nt) {
  if (gm <= 0 || gm >= tiles_m) {
    tile_of(id, G, tiles_m, mt, nt);
    return;
  }
  const int t = (G % 8 == 0) ? (id % 8) * (G / 8) + id / 8 : id;
  const int per = gm * tiles_n, grp = t / per, first = grp * gm;
  const int rows = tiles_m - first < gm ? tiles_m - first : gm;
  const int u = t - grp * per;
  mt = first + u % rows;
  nt = u / rows;
}

// k order inside a 64-k step: MFMA k-step ks (16 k) takes, in lane half kh,
// the 8 k at 32 (ks >> 1) + 16 kh + 8 (ks & 1).  For the weights this is T16
// lane slot g = 2 (ks >> 1) + kh, code-group slots 8 (ks & 1) .. + 7 (one
// dword of the group); for the activations it is 16-byte chunk
// 4 (ks >> 1) + 2 kh + (ks & 1) of the row -- the same k on both sides.  All
// eight k of a fragment lie in 32-block (ks >> 1) of the step.
template <int FMT, int NJ>
struct RStep;
template <int NJ>
struct RStep<GQ_FMT_Q4_0, NJ> {
  gq_u2 q[NJ][2];  // [column block][g = kh or 2 + kh]: the step's 8-byte code groups
  gq_u2 d[NJ];     // d0 d2 | d1 d3 of the column's chunk
};
template <int NJ>
struct RStep<GQ_FMT_Q8_0, NJ> {
  gq_u4 q[NJ][2];  // 16 int8 per lane slot
  gq_u2 d[NJ];
};
template <int NJ>
struct RStep<GQ_FMT_Q4_K, NJ> {
  gq_u2 q[NJ][2];
  gq_u4 meta[NJ];  // d, dmin, W1, W2, W3 of the column's super-block
};
template <int NJ>
struct RStep<GQ_FMT_Q6_K, NJ> {
  gq_u2 q[NJ][2];      // low nibbles: the code groups of slots kh, 2 + kh
  uint32_t hi[NJ][2];  // their high 2-bit fields
  uint32_t sc[NJ];     // the step's four int8 scales (one per 16 k)
  uint32_t d[NJ];      // the super-block's d (fp16 bits)
};
// fp16 weights, row-major N x K (no T16 layout): nothing to dequantize, so they
// go through LDS as the activations do.  A load instruction then takes whole
// 128-byte lines of 8 rows, where fragments loaded straight into registers touch 32
// rows, 32 bytes of each; waves along M share the tile; and no registers are held
// for steps in flight.  Registers / LDS, us: 64 x 4096 x 4096 25.2 / 21.3, 512 x 4096 x
// 4096 45.4 / 40.4, 64 x 4096 x 14336 48.5 / 42.4, 128 x 32000 x 2048 50.7 / 47.1, 512 x
// 32000 x 4096 209 / 203, 2048 x 4096 x 14336 319.5 / 320.5.
template <int NJ>
struct RStep<GQ_FMT_F16, NJ> {};
// loads of one column block and K step
template <int FMT>
constexpr int kRLoads = FMT == GQ_FMT_Q6_K ? 6 : FMT == GQ_FMT_F16 ? 0 : 3;

// Buffer resource over the 4 GiB from p (raw: stride 0, the offset in
// bytes).  The register-B kernel addresses its operands as a 32-bit per-lane
// offset fixed for the whole K walk plus a uniform scalar offset per step, so
// a load costs no vector address arithmetic (the host checks that both the
// packed weights and the activations lie within 4 GiB).
GQ_DEV __amdgpu_buffer_rsrc_t gq_rsrc(const void *p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, -1, 0x00020000);
}
GQ_DEV gq_u2 ld8_b(const void *base, uint32_t vo, uint32_t so) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b64(gq_rsrc(base), vo, so, 0);
  return gq_u2{v[0], v[1]};
}
GQ_DEV gq_u4 ld16_b(const void *base, uint32_t vo, uint32_t so) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(gq_rsrc(base), vo, so, 0);
  return gq_u4{v[0], v[1], v[2], v[3]};
}

GQ_DEV uint32_t ld4_b(const void *base, uint32_t vo, uint32_t so) {
  return __builtin_amdgcn_raw_buffer_load_b32(gq_rsrc(base), vo, so, 0);
}
GQ_DEV uint32_t ld2_b(const void *base, uint32_t vo, uint32_t so) {
  return __builtin_amdgcn_raw_buffer_load_b16(gq_rsrc(base), vo, so, 0);
}

template <int FMT, int NJ>
GQ_DEV void load_rstep(const uint8_t *w, const uint32_t (&qo)[NJ], const uint32_t (&so)[NJ], int step,
                       RStep<FMT, NJ> &st) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if constexpr (FMT == GQ_FMT_Q4_0) {
      const uint32_t b = ((uint32_t)(step >> 1) << 10) + 8u * (uint32_t)(step & 1);
      st.q[j][0] = ld8_b(w, qo[j], b);
      st.q[j][1] = ld8_b(w, qo[j] + 512u, b);
      st.d[j] = ld8_b(w, so[j], (uint32_t)(step >> 1) * 128u);
    } else if constexpr (FMT == GQ_FMT_Q8_0) {
      const uint32_t b = ((uint32_t)(step >> 1) << 11) + ((uint32_t)(step & 1) << 10);
      st.q[j][0] = ld16_b(w, qo[j], b);
      st.q[j][1] = ld16_b(w, qo[j] + 512u, b);
      st.d[j] = ld8_b(w, so[j], (uint32_t)(step >> 1) * 128u);
    } else if constexpr (FMT == GQ_FMT_Q6_K) {
      // (d: from the row's scale bytes at 16 r to its d at 256 + 2 r)
      const uint32_t m = (uint32_t)step & 3u, c = (uint32_t)step >> 2;
      const uint32_t b = c * 3072u + ((m >> 1) << 10) + 8u * (m & 1u), bh = c * 3072u + 2048u + 4u * m;
      const uint32_t r = threadIdx.x & 15u;
      st.q[j][0] = ld8_b(w, qo[j], b);
      st.q[j][1] = ld8_b(w, qo[j] + 512u, b);
      st.hi[j][0] = ld4_b(w, qo[j], bh);
      st.hi[j][1] = ld4_b(w, qo[j] + 512u, bh);
      st.sc[j] = ld4_b(w, so[j], c * 288u + 4u * m);
      st.d[j] = ld2_b(w, so[j] - 14u * r, c * 288u + 256u);
    } else {
      const int m = step & 3;
      const uint32_t b = ((uint32_t)(step >> 2) << 11) + ((uint32_t)(m >> 1) << 10) + 8u * (uint32_t)(m & 1);
      st.q[j][0] = ld8_b(w, qo[j], b);
      st.q[j][1] = ld8_b(w, qo[j] + 512u, b);
      st.meta[j] = ld16_b(w, so[j], (uint32_t)(step >> 2) * 256u);
    }
  }
}

// The register-B kernel's activation tile loads (load_a_lds's rows and
// swizzle): per-lane offsets computed once, the step's columns a scalar offset.
template <int BM, int NW>
GQ_DEV void a_offsets(int lda, int M, int m0, int wave, int lane, uint32_t (&ao)[BM / (8 * NW)]) {
  constexpr int PER_WAVE = BM / (8 * NW);
#pragma unroll
  for (int i = 0; i < PER_WAVE; ++i) {
    const int row0 = 8 * (wave * PER_WAVE + i);
    const int c = (lane & 7) ^ a_swz(row0 + (lane >> 3));
    int m = m0 + row0 + (lane >> 3);
    if (m >= M) m = M - 1;  // clamped; rows >= M are never stored
    ao[i] = 2u * ((uint32_t)m * (uint32_t)lda + 8u * (uint32_t)c);
  }
}
template <int BM, int NW>
GQ_DEV void load_a_lds_b(const _Float16 *a, const uint32_t *ao, int step, int wave,
                         _Float16 *As) {
  constexpr int PER_WAVE = BM / (8 * NW);
#pragma unroll
  for (int i = 0; i < PER_WAVE; ++i) {
    const int row0 = 8 * (wave * PER_WAVE + i);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(gq_rsrc(a), (__attribute__((address_space(3))) void *)(As + row0 * BK), 16, ao[i],
                                             (uint32_t)step * (2u * BK), 0, 0);
  }
}

// Q4_K: the fp16 factors of the sub-block 2 (step & 3) + h of column block j
// (sc, -1024 sc, d, -dmin m), decoded once per K step.
struct QKf {
  gq_half2 sc2, nsc2, d2, mn2, mn16;  // mn16 = 16 mn2 (exact): for the 16 x elements
};
template <int NJ>
GQ_DEV void q4k_factors(const RStep<GQ_FMT_Q4_K, NJ> &st, int step, QKf (&f)[NJ][2]) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const uint32_t mv[4] = {st.meta[j][0], st.meta[j][1], st.meta[j][2], st.meta[j][3]};
    // the fp16 bits as they are (the reference's NaN-to-Inf conversion would
    // compile to branches here)
    const _Float16 hd = __builtin_bit_cast(_Float16, (uint16_t)(mv[0] & 0xFFFFu));
    const _Float16 ndmin = -__builtin_bit_cast(_Float16, (uint16_t)(mv[0] >> 16));
    // the step's two sub-blocks 2 t and 2 t + 1 (t = step & 3): byte t of meta
    // words 1 and 2 (6-bit scale, the min's low 2 bits on top) and of word 3
    // (the mins' high nibbles); both factors of a kind decoded as one fp16
    // pair: 1024 + code from the mantissa bits, minus 1024 (exact)
    const uint32_t sh = 8u * (uint32_t)(step & 3);
    const uint32_t b1 = (mv[1] >> sh) & 0xFFu, b2 = (mv[2] >> sh) & 0xFFu, b3 = (mv[3] >> sh) & 0xFFu;
    const uint32_t scp = (b1 & 63u) | ((b2 & 63u) << 16);
    const uint32_t mnp = ((b1 >> 6) | ((b3 & 15u) << 2)) | (((b2 >> 6) | ((b3 >> 4) << 2)) << 16);
    const gq_half2 k1024 = {(_Float16)-1024.0f, (_Float16)-1024.0f};
    const gq_half2 sc = gq_bits_h2(scp | 0x64006400u) + k1024;   // sc, exact
    const gq_half2 mn = gq_bits_h2(mnp | 0x64006400u) + k1024;   // m, exact
    const gq_half2 nsc = sc * gq_half2{(_Float16)-1024.0f, (_Float16)-1024.0f};  // exact
    const gq_half2 hm = mn * gq_half2{ndmin, ndmin};  // -(dmin m), the exact product rounded once
    const gq_half2 hm16 = hm * gq_half2{(_Float16)16.0f, (_Float16)16.0f};  // exact
    f[j][0] = QKf{__builtin_shufflevector(sc, sc, 0, 0), __builtin_shufflevector(nsc, nsc, 0, 0), gq_half2{hd, hd},
                  __builtin_shufflevector(hm, hm, 0, 0), __builtin_shufflevector(hm16, hm16, 0, 0)};
    f[j][1] = QKf{__builtin_shufflevector(sc, sc, 1, 1), __builtin_shufflevector(nsc, nsc, 1, 1), gq_half2{hd, hd},
                  __builtin_shufflevector(hm, hm, 1, 1), __builtin_shufflevector(hm16, hm16, 1, 1)};
  }
}

// Q6_K: the scales d sc of the step's two 16-element groups this lane holds
// (2 h + kh, h = 0, 1), each product rounded once to fp16.
template <int NJ>
GQ_DEV void q6k_factors(const RStep<GQ_FMT_Q6_K, NJ> &st, int kh, gq_half2 (&f)[NJ][2]) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const float d = (float)__builtin_bit_cast(_Float16, (uint16_t)st.d[j]);
    const uint32_t s = st.sc[j] >> (8 * kh);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const _Float16 hs = (_Float16)(d * (float)(int8_t)((s >> (16 * h)) & 0xFFu));
      f[j][h] = gq_half2{hs, hs};
    }
  }
}

// B fragment of column block j, MFMA k-step ks, K step `step`: 8 fp16 values
// (c - bias) * scale (Q4_K: d sc c - dmin m, factors from q4k_factors; Q6_K:
// factors from q6k_factors), each rounded once.
template <int FMT, int NJ>
GQ_DEV gq_half8 rfrag(const RStep<FMT, NJ> &st, int j, int ks, int step, const QKf *qk, const gq_half2 *q6,
                      uint32_t mg) {
  const int h = ks >> 1;
  gq_half2 p[4];
  if constexpr (FMT == GQ_FMT_Q6_K) {
    // slots 8 (ks & 1) + 0..3 in the low nibbles, + 4..7 in the high ones; the
    // high fields of the first four at bits 4 (ks & 1), of the next at + 2
    const uint32_t w = st.q[j][h][ks & 1], hw = st.hi[j][h];
    const uint32_t h0 = (ks & 1) ? hw : hw << 4, h1 = (ks & 1) ? hw >> 2 : hw << 2;
    bytes_to_magic((w & 0x0F0F0F0Fu) | (h0 & 0x30303030u), p[0], p[1]);
    bytes_to_magic(((w >> 4) & 0x0F0F0F0Fu) | (h1 & 0x30303030u), p[2], p[3]);
    const gq_half2 off = {(_Float16)-1056.0f, (_Float16)-1056.0f};  // codes 0..63, -32
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = (p[i] + off) * q6[h];
  } else if constexpr (FMT == GQ_FMT_Q8_0) {
    const gq_u4 &q = st.q[j][h];
    const uint32_t w0 = q[2 * (ks & 1)] ^ 0x80808080u, w1 = q[2 * (ks & 1) + 1] ^ 0x80808080u;
    const uint32_t db = st.d[j][h];
    const gq_half2 d2 = h2_of_bits16((step & 1) ? (db >> 16) : db);
    const gq_half2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    bytes_to_magic(w0, p[0], p[1]);
    bytes_to_magic(w1, p[2], p[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = (p[i] + off) * d2;
  } else {
    // the 4-bit order (gq_nib_halves): pairs 1 and 3 are 1024 + 16 q, their
    // results 16 x the weight (the activations hold those k divided by 16)
    gq_nib_halves(st.q[j][h][ks & 1], mg, p);
    if constexpr (FMT == GQ_FMT_Q4_0) {
      const uint32_t db = st.d[j][h];
      const gq_half2 d2 = h2_of_bits16((step & 1) ? (db >> 16) : db);
      const gq_half2 off1 = {(_Float16)-1032.0f, (_Float16)-1032.0f};
      const gq_half2 off16 = {(_Float16)-1152.0f, (_Float16)-1152.0f};  // 16 (q - 8), exact
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = (p[i] + ((i & 1) ? off16 : off1)) * d2;
    } else {
      // sc q (or 16 sc q) is exact; then one rounding of d sc q - dmin m
      const QKf &f = qk[h];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[i] = __builtin_elementwise_fma(__builtin_elementwise_fma(p[i], f.sc2, f.nsc2), f.d2, (i & 1) ? f.mn16 : f.mn2);
    }
  }
  gq_half8 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = p[i][0];
    o[2 * i + 1] = p[i][1];
  }
  return o;
}

}  // namespace
