// gq_linear_rb.hip -- the tiled product with bias, activation and residual in its epilogue over T16 weights.
#include <algorithm>
#include <type_traits>

#include "gq_gemm_frag.h"
#include "gq_internal.h"
#include "gq_linear.h"
#include "gq_rows_frag.h"

namespace {

// The register-B tile of gq_gemm_frag.h: a wave owns NJ 32-column blocks of W over all BM rows, fp16 activations by LDS DMA PD - 1
// steps of 64 k ahead, weights PD steps ahead in registers, one counted barrier a step.  KG: groups of waves that share the
// tile and take every KG-th step, their sums added through LDS at the end.  gridDim.y parts of the steps: each part's fp32 sums go to
// `part` [part][M][N], and k_lin_sum finishes them.
template <int FMT, int BM, int WN, int NJ, int PD, int KG>
__global__ void __launch_bounds__(64 * WN * KG) __attribute__((amdgpu_waves_per_eu(front_wpe(WN *KG), front_wpe(WN *KG))))
k_lin_rb(const uint8_t *__restrict__ w, uint32_t sc_off, const _Float16 *__restrict__ a16, int lda, const float *__restrict__ rs,
         LinEpi e, float *__restrict__ part, int M, int N, int C, int nsteps, int sps, int tiles_m) {
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
  constexpr int NA = BM / (8 * NW), pend = (PD - 2) * NA + (PD - 1) * kRLoads<FMT> * NJ;
  int mt, nt;
  tile_of_g(blockIdx.x, gridDim.x, tiles_m, (N + BN - 1) / BN, 4, mt, nt);
  const int m0 = mt * BM, n0 = nt * BN;
  // this part's steps s0 .. s1 (whole rounds of the groups)
  const int s0 = (int)blockIdx.y * sps, s1 = s0 + sps < nsteps ? s0 + sps : nsteps, nl = (s1 - s0) / KG;
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
  gq_f16v acc[TM][NJ];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
  RStep<FMT, NJ> st[PD];
  const uint32_t mg = gq_nib_magic();
  uint32_t ao[NA];
  a_offsets<BM, NW>(lda, M, m0, wave, lane, ao);
  const int arow = lane & 31, sw = a_swz(lane & 31);
  auto gstep = [&](int l) { return s0 + (l < nl ? l : nl - 1) * KG + kg; };
  auto run_step = [&](int l, auto buf_c) __attribute__((always_inline)) {
    constexpr int BUF = decltype(buf_c)::value;
    using NB = std::integral_constant<int, (BUF + PD - 1) % PD>;
    const int step = s0 + l * KG + kg, sa = gstep(l + PD - 1), sb = gstep(l + PD);
    load_a_lds_b<BM, NW>(a16, ao, sa, wave, As_of(NB{}));
    __builtin_amdgcn_sched_barrier(0);
    const _Float16 *As = As_of(buf_c) + arow * BK;
    gq_half8 af[2][TM];
    auto read_a = [&](int ks, int fb) __attribute__((always_inline)) {
      const int ch = (4 * (ks >> 1) + 2 * kh + (ks & 1)) ^ sw;
#pragma unroll
      for (int i = 0; i < TM; ++i) af[fb][i] = *reinterpret_cast<const gq_half8 *>(As + 32 * i * BK + 8 * ch);
    };
    read_a(0, 0);
    QKf qk[NJ][2];
    gq_half2 q6[NJ][2];
    if constexpr (FMT == GQ_FMT_Q4_K) q4k_factors<NJ>(st[BUF], step, qk);
    if constexpr (FMT == GQ_FMT_Q6_K) q6k_factors<NJ>(st[BUF], kh, q6);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + 1 < KS) read_a(ks + 1, (ks + 1) & 1);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const gq_half8 bf = rfrag<FMT, NJ>(st[BUF], j, ks, step, qk[j], q6[j], mg);
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i][j] = gq_mfma32(af[ks & 1][i], bf, acc[i][j]);
      }
    }
    load_rstep<FMT, NJ>(w, qo, so, sb, st[BUF]);
    step_barrier<pend>();
  };
  auto prime = [&](auto b) __attribute__((always_inline)) {
    constexpr int i = decltype(b)::value;
    const int s = gstep(i);
    if constexpr (i < PD - 1) load_a_lds_b<BM, NW>(a16, ao, s, wave, As_of(b));
    __builtin_amdgcn_sched_barrier(0);  // (pend counts this order)
    load_rstep<FMT, NJ>(w, qo, so, s, st[i]);
    __builtin_amdgcn_sched_barrier(0);
  };
  // (padded past M)
  const gq_f4 rs4 = rs ? *reinterpret_cast<const gq_f4 *>(rs + m0 + 4 * (tid % (BM / 4))) : gq_f4{1.f, 1.f, 1.f, 1.f};
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
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        gq_f16v &a = acc[i][j];
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
              for (int u = 0; u < 4; ++u) a[4 * q + u] += t[u];
            }
        }
        __syncthreads();
      }
    if (kg > 0) return;
  }
  // D layout (32x32): lane l holds column l % 32, rows 8 (v / 4) + 4 (l / 32) + v % 4.  Rows >= M lie
  // past the resource's end, whose check need not count a scalar offset: all of it is in the lane's
  // (host: a tile's rows span less than 2 GiB).
  auto range = [&](uint32_t es) {
    const size_t left = (size_t)(M - m0) * (size_t)N * es;
    return (int)(uint32_t)(left < 0xFFFFFFFFu ? left : 0xFFFFFFFFu);
  };
  auto row_scales = [&](int i, float (&rsv)[16]) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const gq_f4 t = *reinterpret_cast<const gq_f4 *>(rs_s + 32 * i + 4 * (lane >> 5) + 8 * q);
#pragma unroll
      for (int u = 0; u < 4; ++u) rsv[4 * q + u] = t[u];
    }
  };
  if (part) {
    const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
        part + ((size_t)blockIdx.y * (size_t)M + m0) * (size_t)N, (short)0, range(4u), 0x00020000);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      float rsv[16];
      row_scales(i, rsv);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int n = n0 + 32 * (NJ * wn + j) + (lane & 31);
        if (n >= N) continue;
#pragma unroll
        for (int v = 0; v < 16; ++v)
          front_put<GQ_DT_F32>(pr, ((uint32_t)(32 * i + 4 * (lane >> 5) + 8 * (v >> 2) + (v & 3)) * (uint32_t)N + (uint32_t)n) * 4u,
                               GQ_DT_F32, acc[i][j][v] * rsv[v]);
      }
    }
    return;
  }
  auto store = [&](auto dtc) __attribute__((always_inline)) {
    constexpr int DT = decltype(dtc)::value;
    constexpr uint32_t ES = DT == GQ_DT_F32 ? 4u : 2u;
    auto rsrc = [&](const void *p) {
      return __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t *>(reinterpret_cast<const uint8_t *>(p)) + (p ? (size_t)m0 * N * ES : 0), (short)0,
          p ? range(ES) : 0, 0x00020000);
    };
    const LinAct act = lin_act_of(e.act);
    const __amdgpu_buffer_rsrc_t yr = rsrc(e.y), zr = rsrc(e.z), rr = rsrc(e.resid);  // (none: no range)
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      float rsv[16];
      row_scales(i, rsv);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int n = n0 + 32 * (NJ * wn + j) + (lane & 31);
        if (n >= N) continue;
        const float b = e.bias ? gq_ld_dt(e.bias, e.bias_dt, n) : 0.f;
        const uint32_t vo = ((uint32_t)(32 * i + 4 * (lane >> 5)) * (uint32_t)N + (uint32_t)n) * ES;
        auto at = [&](int v) { return vo + (uint32_t)(8 * (v >> 2) + (v & 3)) * (uint32_t)N * ES; };
        float res[16] = {};
        if (e.resid) {  // (all of it before the first store: resid may be y)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            if constexpr (DT == GQ_DT_F32) {
              res[v] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rr, at(v), 0, 0));
            } else {
              const uint16_t t = __builtin_amdgcn_raw_buffer_load_b16(rr, at(v), 0, 0);
              res[v] = e.dt == GQ_DT_BF16 ? __uint_as_float((uint32_t)t << 16) : (float)__builtin_bit_cast(_Float16, t);
            }
          }
        }
        gq_f16v &z = acc[i][j];
#pragma unroll
        for (int v = 0; v < 16; ++v) z[v] = fmaf(z[v], rsv[v], b);
        if (e.z) {
#pragma unroll
          for (int v = 0; v < 16; ++v) front_put<DT>(zr, at(v), e.dt, z[v]);
        }
        if (e.act != GQ_ACT_NONE) {
#pragma unroll
          for (int v = 0; v < 16; ++v) z[v] = lin_act_f(act, z[v]);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) front_put<DT>(yr, at(v), e.dt, z[v] + res[v]);
      }
    }
  };
  if (e.dt == GQ_DT_F32) store(std::integral_constant<int, GQ_DT_F32>{});
  else store(std::integral_constant<int, GQ_DT_BF16>{});
}

template <int FMT, int BM, int WN, int NJ, int PD, int KG>
int launch_rb(const void *w, const _Float16 *a16, const float *rs, const LinEpi &e, float *part, int parts, int M, int N, int K,
              hipStream_t s) {
  const int tiles_m = (M + BM - 1) / BM, tiles_n = (N + 32 * NJ * WN - 1) / (32 * NJ * WN);
  GQ_CHECK((size_t)tiles_m * (size_t)tiles_n <= 0x7FFFFFFFu, GQ_ERR_INVALID_ARGS);  // (one grid dimension)
  const int nsteps = (int)(gq_kpad(FMT, K) / BK);
  parts = (int)std::min((size_t)parts, kLinPartBytes / ((size_t)M * (size_t)N * 4));  // (what their sums have room for)
  const int sps = parts > 1 ? ((nsteps + parts - 1) / parts + KG - 1) / KG * KG : nsteps;
  const int np = (nsteps + sps - 1) / sps;  // (no part is empty)
  hipLaunchKernelGGL((k_lin_rb<FMT, BM, WN, NJ, PD, KG>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)np), dim3(64 * WN * KG), 0, s,
                     (const uint8_t *)w, (uint32_t)gq_sc_plane_offset(FMT, N, K), a16, (int)gq_kpad(FMT, K), rs, e,
                     np > 1 ? part : (float *)nullptr, M, N, (int)gq_chunks(FMT, K), nsteps, sps, tiles_m);
  GQ_TRY(gq_last_launch());
  return np > 1 ? gq_launch_linear_sum(part, &e, M, N, np, s) : GQ_OK;
}
template <int FMT>
int launch_fmt(const void *w, const _Float16 *a16, const float *rs, const LinEpi &e, float *part, int M, int N, int K, hipStream_t s) {
  const int nsteps = (int)(gq_kpad(FMT, K) / BK);  // (even)
  // The tile and the parts of K whose rounds of the 256 CUs take the least: a round its steps (and what fills its K groups' pipelines) times what
  // a step takes on a full chip; parts a launch more, and their sums' way to memory and back.  us with the conversion of x, Q4_K / Q8_0, against a
  // ladder of tiles that are near one workgroup a CU each:
  //   2048 x 4096 x 14336   239 / -    (250)         128 x 256        900 x 4096 x 14336   120 / 133 (125 / 143; Q4_0, Q6_K)   128 x 128
  //   2048 x 6144 x 4096    113 / 113  (125 / 122)   256 x 256        300 x 14336 x 4096   53 / 63 (67 / 95; Q4_0, Q6_K)       128 x 256
  //   509 x 8191 x 4096     - / 46     (48)          128 x 128        200 x 20000 x 1024   24 / 23 (32 / 34)                   128 x 256
  //   512 x 4096 x 14336    78 / 78    (79 / 77)     in 2, 4 parts    128 x 4096 x 4096    17.7 / 17.1 (19.5 / 20.5)           32 x 64
  //   128 x 14336 x 4096    26 / 34 (Q4_0, Q6_K: the same) 64 x 128   64 x 4096 x 14336    26 / 29 (24 / 31; Q4_0, Q6_K)       64 x 128, 8 parts
  // Loads a lane shares between two column blocks of a wave (64 x 256 by 4 waves): 51 against 47 of 509 x 8191 x 4096.
  float best = 1e30f;
  int parts = 1;
  auto takes = [&](int bm, int bn, int kg, float step) {
    const size_t tiles = (size_t)((M + bm - 1) / bm) * (size_t)((N + bn - 1) / bn);
    bool better = false;
    for (int p = 1; p <= kLinParts && (p == 1 || (nsteps >= 4 * kg * p && (size_t)p * M * N * 4 <= kLinPartBytes)); ++p) {
      const float rounds = (float)((tiles * (size_t)p + 255) / 256);
      const float t = rounds * (float)((nsteps + p - 1) / p + 4 * kg) * step + (p > 1 ? 4.f + (float)p * (float)M * (float)N * 1.6e-6f : 0.f);
      if (t >= best) continue;
      best = t;
      parts = p;
      better = true;
    }
    return better;
  };
  // (4 bits: two K groups of 128 x 256, 2048 x 4096 x 14336 Q4_K 237 us, one group 250; Q8_0, Q6_K 1024 x 8192 x 4096 80, 81 and 72, 78)
  constexpr bool NIB = FMT == GQ_FMT_Q4_0 || FMT == GQ_FMT_Q4_K;
  int tile = 0;
  takes(256, 256, 1, 1.65f);
  if (takes(128, 256, NIB ? 2 : 1, 1.f)) tile = 1;
  if (takes(128, 128, 2, 0.56f)) tile = 2;
  const bool four = nsteps % 4 == 0;  // (whole rounds of the groups)
  if (takes(64, 128, four ? 4 : 2, 0.35f)) tile = 3;
  if (four ? takes(32, 64, 4, 0.16f) : takes(32, 64, 2, 0.2f)) tile = 4;
#define GQ_RB(P, ...) launch_rb<FMT, __VA_ARGS__>(w, a16, rs, e, part, P, M, N, K, s)
  if (tile == 0) return GQ_RB(parts, 256, 8, 1, 3, 1);
  if (tile == 1) {
    if constexpr (NIB) return GQ_RB(parts, 128, 8, 1, 3, 2);
    else return GQ_RB(parts, 128, 8, 1, 4, 1);
  }
  if (tile == 2) return GQ_RB(parts, 128, 4, 1, 3, 2);
  if constexpr (FMT == GQ_FMT_Q4_0 || FMT == GQ_FMT_Q8_0) {  // (K of the k-quants is whole 256s)
    if (!four && tile == 4) return GQ_RB(parts, 32, 2, 1, 3, 2);  // (60 x 633 x 3392 Q8_0 11.4 us, by 128 x 128 in parts 15.0)
    if (!four) return GQ_RB(parts, 64, 4, 1, 4, 2);
  }
  if (tile == 4) return GQ_RB(parts, 32, 2, 1, 4, 4);
  return GQ_RB(parts, 64, 4, 1, 3, 4);
#undef GQ_RB
}

}  // namespace

int gq_launch_linear_rb(int fmt, const void *w, const _Float16 *a16, const float *rs, const void *epi, float *part, int M, int N, int K,
                        hipStream_t s) {
  const LinEpi &e = *reinterpret_cast<const LinEpi *>(epi);
  if (fmt == GQ_FMT_Q4_0) return launch_fmt<GQ_FMT_Q4_0>(w, a16, rs, e, part, M, N, K, s);
  if (fmt == GQ_FMT_Q8_0) return launch_fmt<GQ_FMT_Q8_0>(w, a16, rs, e, part, M, N, K, s);
  if (gq_fmt_is_q6k(fmt)) return launch_fmt<GQ_FMT_Q6_K>(w, a16, rs, e, part, M, N, K, s);
  return launch_fmt<GQ_FMT_Q4_K>(w, a16, rs, e, part, M, N, K, s);
}
