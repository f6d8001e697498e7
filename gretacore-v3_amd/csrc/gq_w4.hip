// gq_w4.hip -- products with 4-bit weights that have a scale and a zero point per group:
// y = x W^T and the gated form act(x W_gate^T) * (x W_up^T), 1 to 16 rows.
//
// Packed layout.  Rows in tiles of 16, K in chunks of 128 (C = ceil(K / 128)); codes
// and scales in two planes, zeros (scale 0) behind N and K:
//   codes [tile][C][64 lanes][4 words], lane 16 g + r, word b: row r, k = 128 c + 32 b + 8 g
//         + 0..7.  One 16-byte load per lane streams a chunk.  Of the word, the codes
//         2 j and 2 j + 1 sit at bits 3 + 4 j and 19 + 4 j (j = 3 wraps around), so that
//         a shift (or rotation) by 4 j brings each pair to bits 3 and 19: the mantissa
//         of two 16-bit floats, 8 steps of the last place each.
//   meta  [tile][C][16 rows][128 / group] one word: the scale as fp32 bits (fp16 and
//         bf16 leave its low 13 bits zero) with the zero point in the low 5.
#include <type_traits>

#include "gq_act.h"
#include "gq_internal.h"

namespace {

constexpr int kW4Chunk = 128, kW4Codes = 1024;  // k and code bytes of a tile's chunk

bool w4_group_valid(int group) { return group == 32 || group == 64 || group == 128; }
size_t w4_chunks(size_t K) { return (K + kW4Chunk - 1) / kW4Chunk; }
size_t w4_meta_off(size_t N, size_t K) { return gq_tiles(N) * w4_chunks(K) * kW4Codes; }
size_t w4_bytes(size_t N, size_t K, int group) {
  return w4_meta_off(N, K) + gq_tiles(N) * w4_chunks(K) * (size_t)(16 * 4 * (kW4Chunk / group));
}

struct __attribute__((packed, aligned(1))) W4Bytes4 {
  uint32_t v;
};
// one word of codes (four bytes of a row in one load: byte by byte 107 us, 4096 x 14336, group 128; so 24), or one
// meta word, a thread
__global__ void __launch_bounds__(256) k_w4_pack(const uint8_t *__restrict__ q, const uint16_t *__restrict__ s, int sbf16,
                                                 const uint8_t *__restrict__ z, size_t N, size_t K, int group,
                                                 uint32_t *__restrict__ codes, uint32_t *__restrict__ meta, size_t n_code,
                                                 size_t n_meta) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t C = (K + kW4Chunk - 1) / kW4Chunk, rb = (K + 1) / 2, ng = (K + group - 1) / group;
  if (i < n_code) {
    const size_t lane = (i >> 2) & 63, tc = i >> 8;
    const size_t n = (tc / C) * 16 + (lane & 15), k = (tc % C) * kW4Chunk + 32 * (i & 3) + 8 * (lane >> 4);
    uint32_t v = 0;  // the row's four bytes, even k in the low nibbles
    if (n < N && k + 8 <= K) {
      v = reinterpret_cast<const W4Bytes4 *>(q + n * rb + k / 2)->v;
    } else if (n < N) {
      for (int e = 0; e < 8; ++e)
        if (k + e < K) v |= (uint32_t)((q[n * rb + ((k + e) >> 1)] >> (4 * (e & 1))) & 15u) << (4 * e);
    }
    // code e to bit 3 + 16 (e % 2) + 4 (e / 2) of 32
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = 3 + 16 * (e & 1) + 4 * (e >> 1);
      w |= __builtin_rotateleft32((v >> (4 * e)) & 15u, at & 31);
    }
    codes[i] = w;
  } else if (i - n_code < n_meta) {
    const size_t j = i - n_code, per = kW4Chunk / group;
    const size_t tc = j / (16 * per), n = (tc / C) * 16 + j / per % 16, gr = (tc % C) * per + j % per;
    uint32_t v = 0;
    if (n < N && gr < ng) {
      const uint32_t b = s[n * ng + gr];
      const float f = sbf16 ? __uint_as_float(b << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
      v = (__float_as_uint(f) & ~31u) | (z ? z[n * ng + gr] & 31u : 8u);
    }
    meta[j] = v;
  }
}

struct W4Mats {
  const uint8_t *w[2];
};

// ---- the product ---------------------------------------------------------------
// v_mfma_f32_16x16x32 on one 32-block: the weights are the B operand (column = row n of
// W, lane 16 g + r holds its codes 8 g .. + 7), x the A operand (row = batch row).  The codes
// enter as they are, as the 16-bit floats 16 + q (bf16) or 128 + q (f16) that one AND-OR
// makes of them; their sum is brought back with the sum of x (a product with ones, shared by
// the tiles of a wave), and scale and zero point are applied once a group, in fp32:
//   y += s (sum x (OFF + q) - (OFF + z) sum x)
// so nothing is rounded but the fp32 sums.  fp32 x goes in as three bf16 parts of 8 bits.
// Bound by the weights' bytes: a workgroup takes R row tiles (of both matrices) with KS waves
// that share K chunk by chunk, PD chunks in flight each.
typedef __bf16 w4_bf8 __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(2))) W4Run16 {  // 8 values at any 2-byte address
  gq_u4 v;
};
struct __attribute__((packed, aligned(4))) W4Run32 {
  gq_u4 v[2];
};

template <int XT>
constexpr int kW4Parts = XT == GQ_DT_F32 ? 3 : 1;
template <int XT>
constexpr float kW4Off = XT == GQ_DT_F16 ? 128.f : 16.f;
template <int XT>
constexpr uint32_t kW4Magic = XT == GQ_DT_F16 ? 0x58005800u : 0x41804180u;
template <int XT>
constexpr uint32_t kW4Ones = XT == GQ_DT_F16 ? 0x3C003C00u : 0x3F803F80u;

template <int XT>
GQ_DEV gq_f4 w4_mfma(const gq_u4 &a, const gq_u4 &b, const gq_f4 &c) {
  if constexpr (XT == GQ_DT_F16)
    return gq_mfma16(__builtin_bit_cast(gq_half8, a), __builtin_bit_cast(gq_half8, b), c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_bf8, a), __builtin_bit_cast(w4_bf8, b), c, 0, 0,
                                                   0);
}
GQ_DEV gq_u4 w4_codes(uint32_t w, uint32_t mg) {
  constexpr uint32_t m = 0x00780078u;
  return gq_u4{(w & m) | mg, ((w >> 4) & m) | mg, ((w >> 8) & m) | mg, (__builtin_rotateright32(w, 12) & m) | mg};
}

// 8 values of a row from k on, as loaded; TAIL: zeros from K on
template <int XT>
struct W4Raw {
  gq_u4 v[XT == GQ_DT_F32 ? 2 : 1];
};
template <int XT, bool TAIL>
GQ_DEV void w4_load_x(const void *x, size_t row, int k, int K, W4Raw<XT> &r) {
  if constexpr (TAIL) {  // (addresses clamped into the row, no branch around a load)
    uint32_t t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const size_t at = row + (k + e < K ? k + e : K - 1);
      if constexpr (XT == GQ_DT_F32) t[e] = reinterpret_cast<const uint32_t *>(x)[at];
      else t[e] = reinterpret_cast<const uint16_t *>(x)[at];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = k + e < K ? t[e] : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (XT == GQ_DT_F32) {
        r.v[0][e] = t[e];
        r.v[1][e] = t[4 + e];
      } else {
        r.v[0][e] = t[2 * e] | t[2 * e + 1] << 16;
      }
    }
  } else if constexpr (XT == GQ_DT_F32) {
    const W4Run32 t = *reinterpret_cast<const W4Run32 *>(reinterpret_cast<const uint32_t *>(x) + row + k);
    r.v[0] = t.v[0];
    r.v[1] = t.v[1];
  } else {
    r.v[0] = reinterpret_cast<const W4Run16 *>(reinterpret_cast<const uint16_t *>(x) + row + k)->v;
  }
}
// The A operand's parts, the smallest first (their sum is the value: 8 bits of it each, cut
// off, not rounded; the differences are exact)
template <int XT>
GQ_DEV void w4_parts(const W4Raw<XT> &r, gq_u4 (&o)[kW4Parts<XT>]) {
  if constexpr (XT != GQ_DT_F32) {
    o[0] = r.v[0];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t p[3][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = 2 * j + h;
        float v = __uint_as_float(r.v[e >> 2][e & 3]);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          p[i][h] = __float_as_uint(v);
          v -= __uint_as_float(p[i][h] & 0xFFFF0000u);
        }
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) o[2 - i][j] = __builtin_amdgcn_perm(p[i][1], p[i][0], 0x07060302u);
    }
  }
}

// FEW: up to 4 rows, and the A operand has 16.  Lane 16 g + 4 b + j then loads row j of
// block b, one load a chunk where the operand's order takes four, and rotations by whole
// quads bring a block to rows 0..3 of the operand; fp32's other parts go to rows 4..7 and 8..11,
// so that they take no product of their own (their sums are added at the end).
template <int I, int B>
GQ_DEV uint32_t w4_quad(uint32_t old, uint32_t src) {  // quad B of each 16 lanes to quad I, the others as in old
  constexpr int n = 4 * ((I - B + 4) % 4);
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)src, n ? 0x120 + n : 0xE4, 0xF, 1 << I, false);
}
template <int XT, bool FEW>
constexpr int kW4Ops = FEW ? 1 : kW4Parts<XT>;  // products of a block
template <int XT, bool FEW, int B>
GQ_DEV void w4_operand(const gq_u4 (&p)[FEW ? 1 : 4][kW4Parts<XT>], gq_u4 (&o)[kW4Ops<XT, FEW>]) {
#pragma unroll
  for (int i = 0; i < kW4Ops<XT, FEW>; ++i)
    if constexpr (!FEW) {
      o[i] = p[B][i];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (XT == GQ_DT_F32) {
          o[0][j] = w4_quad<0, B>(0u, p[0][0][j]);
          o[0][j] = w4_quad<1, B>(o[0][j], p[0][1][j]);
          o[0][j] = w4_quad<2, B>(o[0][j], p[0][2][j]);
        } else {
          o[0][j] = B == 0 ? p[0][0][j] : w4_quad<0, B>(p[0][0][j], p[0][0][j]);
        }
      }
    }
}

template <int MATS, int XT, int GW, int R, int KS, bool FEW>
__global__ void __launch_bounds__(64 * KS)
k_w4(W4Mats mats, size_t meta_off, const void *__restrict__ x, void *__restrict__ y, int ydt, int N, int K, int C,
     int batch, int act) {
  constexpr int T = MATS * R, NP = kW4Parts<XT>, NO = kW4Ops<XT, FEW>, NX = FEW ? 1 : 4;
  constexpr int PD = T == 1 ? (XT == GQ_DT_F32 && !FEW ? 2 : 4) : T == 2 ? 3 : 2;  // (as the registers allow)
  constexpr int BPG = 4 / GW;  // 32-blocks a group
  __shared__ gq_f4 red[KS][T][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int tile0 = (int)blockIdx.x * R, ntiles = (N + 15) >> 4;
  // A tile's codes and meta words through buffer resources of their own, which end with
  // the tile: a load of chunk C or beyond lies out of range and fetches nothing.
  __amdgpu_buffer_rsrc_t wr[T], mr[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    int tile = tile0 + t % R;
    if (tile >= ntiles) tile = ntiles - 1;  // clamped; not stored
    const size_t tc = (size_t)tile * C;
    uint8_t *w = const_cast<uint8_t *>(mats.w[t / R]);
    wr[t] = __builtin_amdgcn_make_buffer_rsrc(w + tc * kW4Codes, (short)0, C * kW4Codes, 0x00020000);
    mr[t] = __builtin_amdgcn_make_buffer_rsrc(w + meta_off + tc * (64 * GW), (short)0, C * (64 * GW), 0x00020000);
  }
  // the row (FEW: and block) of x this lane loads; rows past the batch: any
  const int xr = FEW ? lane & 3 : r;
  const size_t row = (size_t)(xr < batch ? xr : 0) * K;
  const int xk = 8 * g + (FEW ? 32 * ((lane >> 2) & 3) : 0);

  gq_u4 q[PD][T];
  uint32_t meta[PD][T][GW];
  W4Raw<XT> xs[PD][NX];
  auto load = [&](int c, int st) __attribute__((always_inline)) {
    const uint32_t wo = (uint32_t)c * kW4Codes + 16u * (uint32_t)lane, mo = (uint32_t)c * (64 * GW) + 4 * GW * (uint32_t)r;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(wr[t], wo, 0, 2);  // (streamed: read once)
      q[st][t] = gq_u4{v[0], v[1], v[2], v[3]};
      if constexpr (GW == 1) {
        meta[st][t][0] = __builtin_amdgcn_raw_buffer_load_b32(mr[t], mo, 0, 0);
      } else if constexpr (GW == 2) {
        const auto m = __builtin_amdgcn_raw_buffer_load_b64(mr[t], mo, 0, 0);
        meta[st][t][0] = m[0];
        meta[st][t][1] = m[1];
      } else {
        const auto m = __builtin_amdgcn_raw_buffer_load_b128(mr[t], mo, 0, 0);
#pragma unroll
        for (int i = 0; i < GW; ++i) meta[st][t][i] = m[i];
      }
    }
  };
  auto load_x = [&](int c, int st, auto tail) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < NX; ++b)
      w4_load_x<XT, decltype(tail)::value>(x, row, kW4Chunk * c + xk + 32 * b, K, xs[st][b]);
  };

  gq_f4 acc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) acc[t] = gq_f4{0.f, 0.f, 0.f, 0.f};
  uint32_t mg;
  asm volatile("v_mov_b32 %0, %1" : "=v"(mg) : "i"(kW4Magic<XT>));  // (kept in a register)
  const gq_u4 ones = {kW4Ones<XT>, kW4Ones<XT>, kW4Ones<XT>, kW4Ones<XT>};
  auto compute = [&](int st) __attribute__((always_inline)) {
    gq_u4 p[NX][NP];
#pragma unroll
    for (int b = 0; b < NX; ++b) w4_parts<XT>(xs[st][b], p[b]);
    gq_f4 d[T], sx;
    auto block = [&](auto bc) __attribute__((always_inline)) {
      constexpr int B = decltype(bc)::value;
      gq_u4 o[NO];
      w4_operand<XT, FEW, B>(p, o);
      if constexpr (B % BPG == 0) {
        sx = gq_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < T; ++t) d[t] = sx;
      }
#pragma unroll
      for (int i = 0; i < NO; ++i) sx = w4_mfma<XT>(o[i], ones, sx);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const gq_u4 w = w4_codes(q[st][t][B], mg);
#pragma unroll
        for (int i = 0; i < NO; ++i) d[t] = w4_mfma<XT>(o[i], w, d[t]);
      }
      if constexpr (B % BPG == BPG - 1) {
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const uint32_t v = meta[st][t][B / BPG];
          const float s = __uint_as_float(v & ~31u), z = kW4Off<XT> + (float)(v & 31u);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(s, fmaf(-z, sx[i], d[t][i]), acc[t][i]);
        }
      }
    };
    block(std::integral_constant<int, 0>{});
    block(std::integral_constant<int, 1>{});
    block(std::integral_constant<int, 2>{});
    block(std::integral_constant<int, 3>{});
  };

  // this wave's whole chunks: wave, wave + KS, ...; past the last one nothing is fetched of
  // the weights, and x of the last one again
  const int full = K / kW4Chunk, n = full > wave ? (full - wave + KS - 1) / KS : 0;
  if (n > 0) {
    auto request = [&](int j, int st) __attribute__((always_inline)) {
      load(j < n ? wave + KS * j : C, st);
      load_x(wave + KS * (j < n ? j : n - 1), st, std::false_type{});
    };
#pragma unroll
    for (int i = 0; i < PD; ++i) request(i, i);
    for (int j = 0; j < n; j += PD) {
#pragma unroll
      for (int i = 0; i < PD; ++i) {
        if (j + i >= n) break;
        compute(i);
        request(j + i + PD, i);
      }
    }
  }
  if (C > full && full % KS == wave) {  // a chunk that ends behind K
    load(full, 0);
    load_x(full, 0, std::true_type{});
    compute(0);
  }

#pragma unroll
  for (int t = 0; t < T; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  // D layout (16x16): lane l holds column l % 16, rows 4 (l / 16) + i
  for (int o = threadIdx.x; o < 16 * R * batch; o += 64 * KS) {
    const int nl = o % (16 * R), m = o / (16 * R), at = 16 * (m >> 2) + (nl & 15);
    float s[MATS] = {};
#pragma unroll
    for (int k = 0; k < MATS; ++k)
#pragma unroll
      for (int w = 0; w < KS; ++w)
#pragma unroll
        for (int i = 0; i < (FEW ? NP : 1); ++i)
          s[k] += reinterpret_cast<const float *>(&red[w][k * R + (nl >> 4)][at + 16 * i])[m & 3];
    const int nn = 16 * tile0 + nl;
    if (nn < N) gq_st_dt(y, ydt, (size_t)m * N + nn, MATS == 2 ? gq_act_f(act, s[0]) * s[MATS - 1] : s[0]);
  }
}

// Row tiles and waves of a workgroup.  More tiles share one reading of x and its
// conversion, more waves per tile start more loads at once where tiles are few:
//  * one tile while the tiles fit the CUs (8 waves; with more than 4 rows, whose x takes four
//    times the loads, only for long K).  us, tiles 1 / 2 / 4: 4096 x 4096 one row 4.9 / 5.9 / 9.4,
//    8 rows 7.9 / 7.9 / 10.0; 4096 x 14336 one row 9.6 / 13.0 / 26.6, 8 rows 15.5 / 17.2 / 25.8
//  * two tiles, on 8 waves up to 1000 tiles (8192 x 4096 one row 6.5, on 4 waves 7.3; 20000 x 4096 13.1
//    and 12.9); more than 4 rows on 4 waves but for long K (8192 x 4096 8 rows 8.2, on 8 waves 8.5;
//    6000 x 14336 20.1 and 17.8)
//  * four tiles on 4 waves from where two give more than a round of workgroups: 14336 x 4096
//    8 rows 10.7, two tiles 12.1; 32000 x 4096 two rows of fp32 18.9 and 21.1
//  * these on 8 waves where one round of workgroups holds them and a chunk's work is long (groups of 32) or K
//    is: 8 rows of 14336 x 4096, group 32, 11.5, on 4 waves 13.3; 11008 x 8192 17.9 and 21.6, group 64 fp32 22.3 and
//    25.3; but 32000 x 4096 group 32 22.3 and 20.4, 14336 x 4096 group 128 16 rows 11.1 and 10.9
template <int MATS, int XT, int GW, bool FEW>
int launch_w4_shape(W4Mats mats, const void *x, void *y, int ydt, int N, int K, int batch, int act, hipStream_t s) {
  const size_t tiles = gq_tiles(N), tt = tiles * MATS, mo = w4_meta_off(N, K);
  const int C = (int)w4_chunks(K);
  const size_t two = !FEW ? 600 : XT == GQ_DT_F32 ? 800 : 1400;  // the most tiles that go by twos
#define GQ_W4(R, KS)                                                                                               \
  hipLaunchKernelGGL((k_w4<MATS, XT, GW, R, KS, FEW>), dim3((unsigned)((tiles + (R)-1) / (R))), dim3(64 * (KS)), 0, s, mats, \
                     mo, x, y, ydt, N, K, C, batch, act)
  if (MATS == 1 && tt <= 256 && (FEW || C >= 64)) {
    if constexpr (MATS == 1) GQ_W4(1, 8);
  } else if (tt <= two) {
    if (FEW ? tt <= 1000 : C >= 64) GQ_W4(2 / MATS, 8);
    else GQ_W4(2 / MATS, 4);
  } else if (MATS == 1 && !FEW && tt <= 1024 && (GW == 4 || C >= 64)) {
    if constexpr (MATS == 1 && !FEW) GQ_W4(4, 8);
  } else {
    GQ_W4(4 / MATS, 4);
  }
#undef GQ_W4
  return gq_last_launch();
}
template <int MATS, int XT, int GW>
int launch_w4_rows(W4Mats mats, const void *x, void *y, int ydt, int N, int K, int batch, int act, hipStream_t s) {
  return batch <= 4 ? launch_w4_shape<MATS, XT, GW, true>(mats, x, y, ydt, N, K, batch, act, s)
                    : launch_w4_shape<MATS, XT, GW, false>(mats, x, y, ydt, N, K, batch, act, s);
}
template <int MATS, int XT>
int launch_w4_group(W4Mats mats, int group, const void *x, void *y, int ydt, int N, int K, int batch, int act,
                    hipStream_t s) {
  if (group == 128) return launch_w4_rows<MATS, XT, 1>(mats, x, y, ydt, N, K, batch, act, s);
  if (group == 64) return launch_w4_rows<MATS, XT, 2>(mats, x, y, ydt, N, K, batch, act, s);
  return launch_w4_rows<MATS, XT, 4>(mats, x, y, ydt, N, K, batch, act, s);
}

int check_w4(int group, size_t N, size_t K) {
  GQ_CHECK(w4_group_valid(group), GQ_ERR_UNSUPPORTED);
  GQ_CHECK(N <= GQ_MAX_DIM && K <= GQ_MAX_DIM, GQ_ERR_INVALID_ARGS);
  return GQ_OK;
}
template <int MATS>
int launch_w4(W4Mats mats, int group, const void *x, int x_dtype, void *y, int y_dtype, size_t N, size_t K, int batch,
              int act, hipStream_t s) {
  GQ_TRY(check_w4(group, N, K));
  GQ_CHECK(gq_dtype_valid(x_dtype) && gq_dtype_valid(y_dtype), GQ_ERR_UNSUPPORTED);
  GQ_CHECK(MATS == 1 || gq_act_valid(act), GQ_ERR_UNSUPPORTED);
  GQ_CHECK(batch >= 1 && batch <= GQ_MAX_BATCH, GQ_ERR_UNSUPPORTED);
  if (N == 0) return GQ_OK;
  GQ_CHECK(mats.w[0] && mats.w[MATS - 1] && x && y && K > 0, GQ_ERR_INVALID_ARGS);
  GQ_CHECK((((uintptr_t)mats.w[0] | (uintptr_t)mats.w[MATS - 1]) & 15) == 0, GQ_ERR_INVALID_ARGS);  // (16-byte loads)
  const int n = (int)N, k = (int)K;
  if (x_dtype == GQ_DT_F32) return launch_w4_group<MATS, GQ_DT_F32>(mats, group, x, y, y_dtype, n, k, batch, act, s);
  if (x_dtype == GQ_DT_F16) return launch_w4_group<MATS, GQ_DT_F16>(mats, group, x, y, y_dtype, n, k, batch, act, s);
  return launch_w4_group<MATS, GQ_DT_BF16>(mats, group, x, y, y_dtype, n, k, batch, act, s);
}

}  // namespace

extern "C" int gq_w4_packed_size(size_t N, size_t K, int group, size_t *bytes) {
  GQ_TRY(check_w4(group, N, K));
  GQ_CHECK(bytes, GQ_ERR_INVALID_ARGS);
  *bytes = w4_bytes(N, K, group);
  return GQ_OK;
}

extern "C" int gq_w4_pack(const uint8_t *q, const void *scales, int scale_dtype, const uint8_t *zeros, size_t N, size_t K,
                          int group, void *packed, void *stream) {
  GQ_TRY(check_w4(group, N, K));
  // (an fp32 scale would have to be rounded)
  GQ_CHECK(scale_dtype == GQ_DT_F16 || scale_dtype == GQ_DT_BF16, GQ_ERR_UNSUPPORTED);
  if (N == 0 || K == 0) return GQ_OK;
  GQ_CHECK(q && scales && packed && ((uintptr_t)packed & 15) == 0, GQ_ERR_INVALID_ARGS);
  const size_t codes = w4_meta_off(N, K) / 4, meta = w4_bytes(N, K, group) / 4 - codes;
  GQ_CHECK((codes + meta + 255) / 256 <= 0x7FFFFFFFu, GQ_ERR_INVALID_ARGS);
  hipLaunchKernelGGL(k_w4_pack, dim3((unsigned)((codes + meta + 255) / 256)), dim3(256), 0, (hipStream_t)stream, q,
                     (const uint16_t *)scales, scale_dtype == GQ_DT_BF16, zeros, N, K, group, (uint32_t *)packed,
                     (uint32_t *)packed + codes, codes, meta);
  return gq_last_launch();
}

extern "C" int gq_w4_gemv(const void *packed, int group, const void *x, int x_dtype, void *y, int y_dtype, size_t N,
                          size_t K, int batch, void *stream) {
  return launch_w4<1>(W4Mats{{(const uint8_t *)packed, nullptr}}, group, x, x_dtype, y, y_dtype, N, K, batch, GQ_ACT_SILU,
                      (hipStream_t)stream);
}

extern "C" int gq_w4_gate_up(const void *gate, const void *up, int group, const void *x, int x_dtype, void *h, int h_dtype,
                             size_t N, size_t K, int batch, int act, void *stream) {
  return launch_w4<2>(W4Mats{{(const uint8_t *)gate, (const uint8_t *)up}}, group, x, x_dtype, h, h_dtype, N, K, batch, act,
                      (hipStream_t)stream);
}
