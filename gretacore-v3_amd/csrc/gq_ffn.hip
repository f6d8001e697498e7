// gq_ffn.hip -- the gated feed-forward front h = act(x W_gate^T) * (x W_up^T) over T16
// weights for any number of rows, and its backward pass.
#include "gq_act.h"
#include "gq_gemm_frag.h"
#include "gq_internal.h"

namespace {

// One weight of a T16 tensor, dequantized in fp32.
GQ_DEV float t16_weight(int fmt, const uint8_t *w, size_t sc_off, size_t n, size_t k, size_t C) {
  const uint8_t *sc = w + sc_off;
  const size_t blk = k >> 5;
  const int eh = (int)(k >> 4) & 1, s = (int)k & 15;
  const int b = 4 * (s >> 3) + (s & 3), sh = 4 * ((s >> 2) & 1);  // the slot's byte and nibble in its code group
  if (fmt == GQ_FMT_Q4_0) {
    const int q = (w[gq_q4_0_grp_off(n, blk, eh, C) + b] >> sh) & 15;
    return (float)(q - 8) * gq_h2f(gq_rd16(sc + gq_q4_0_d_off(n, blk, C)));
  }
  if (fmt == GQ_FMT_Q8_0)
    return (float)(int8_t)w[gq_q8_0_half_off(n, blk, eh, C) + s] * gq_h2f(gq_rd16(sc + gq_q4_0_d_off(n, blk, C)));
  const size_t sb = k >> 8;
  const int j = (int)blk & 7;
  if (gq_fmt_is_q6k(fmt)) {
    const uint32_t hw = *reinterpret_cast<const uint32_t *>(w + gq_q6k_hi_off(n, sb, j, eh, C));
    const int q = ((w[gq_q6k_grp_off(n, sb, j, eh, C) + b] >> sh) & 15) | (int)(gq_q6k_hi_of(hw, s) << 4);
    return gq_h2f(gq_rd16(sc + gq_q6k_d_off(n, sb, C))) * (float)(int8_t)sc[gq_q6k_sc_off(n, sb, C) + 2 * j + eh] *
           (float)(q - 32);
  }
  const uint32_t *meta = reinterpret_cast<const uint32_t *>(sc + gq_q4k_meta_off(n, sb, C));
  const uint32_t mv[4] = {meta[0], meta[1], meta[2], meta[3]};
  uint32_t a, m;
  gq_q4k_meta_codes(mv, j, &a, &m);
  const int q = (w[gq_q4k_grp_off(n, sb, j, eh, C) + b] >> sh) & 15;
  return gq_h2f(mv[0]) * (float)a * (float)q - gq_h2f(mv[0] >> 16) * (float)m;
}

// 16 x 16 outputs a workgroup, K in steps of 32 through LDS, fp32 throughout
__global__ void __launch_bounds__(256) k_front(int fmt, const uint8_t *gate, const uint8_t *up, size_t sc_off,
                                               const void *x, int xdt, void *h, int hdt, void *go, void *uo, int M,
                                               int N, int K, int C, int act) {
  __shared__ float xs[16][33], ws[2][16][33];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int n0 = 16 * blockIdx.x;
  for (int m0 = 16 * (int)blockIdx.y; m0 < M; m0 += 16 * (int)gridDim.y) {
    float g = 0.f, u = 0.f;
    for (int k0 = 0; k0 < K; k0 += 32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = ty, k = k0 + tx + 16 * i;
        xs[r][tx + 16 * i] = m0 + r < M ? gq_ld_dt(x, xdt, (size_t)(m0 + r) * K + k) : 0.f;
        ws[0][r][tx + 16 * i] = n0 + r < N ? t16_weight(fmt, gate, sc_off, n0 + r, k, C) : 0.f;
        ws[1][r][tx + 16 * i] = n0 + r < N ? t16_weight(fmt, up, sc_off, n0 + r, k, C) : 0.f;
      }
      __syncthreads();
      for (int k = 0; k < 32; ++k) {
        g += xs[ty][k] * ws[0][tx][k];
        u += xs[ty][k] * ws[1][tx][k];
      }
      __syncthreads();
    }
    if (m0 + ty < M && n0 + tx < N) {
      const size_t i = (size_t)(m0 + ty) * N + n0 + tx;
      gq_st_dt(h, hdt, i, gq_act_f(act, g) * u);
      if (go) gq_st_dt(go, hdt, i, g);
      if (uo) gq_st_dt(uo, hdt, i, u);
    }
  }
}

GQ_DEV void front_grads(int act, float dh, float g, float u, float &dg, float &du) {
  float f, d;
  gq_act_fd(act, g, f, d);
  dg = dh * u * d;
  du = dh * f;
}
__global__ void __launch_bounds__(256) k_front_dx(int fmt, const uint8_t *gate, const uint8_t *up, size_t sc_off,
                                                  const void *dh, const void *g, const void *u, int dt, void *dx,
                                                  int xdt, int M, int N, int K, int C, int act) {
  __shared__ float as[2][16][17], ws[2][16][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int k0 = 16 * blockIdx.x;
  for (int m0 = 16 * (int)blockIdx.y; m0 < M; m0 += 16 * (int)gridDim.y) {
    float s = 0.f;
    for (int n0 = 0; n0 < N; n0 += 16) {
      float dg = 0.f, du = 0.f;
      if (m0 + ty < M && n0 + tx < N) {
        const size_t i = (size_t)(m0 + ty) * N + n0 + tx;
        front_grads(act, gq_ld_dt(dh, dt, i), gq_ld_dt(g, dt, i), gq_ld_dt(u, dt, i), dg, du);
      }
      as[0][ty][tx] = dg;
      as[1][ty][tx] = du;
      ws[0][ty][tx] = n0 + ty < N ? t16_weight(fmt, gate, sc_off, n0 + ty, k0 + tx, C) : 0.f;
      ws[1][ty][tx] = n0 + ty < N ? t16_weight(fmt, up, sc_off, n0 + ty, k0 + tx, C) : 0.f;
      __syncthreads();
      for (int n = 0; n < 16; ++n) s += as[0][ty][n] * ws[0][n][tx] + as[1][ty][n] * ws[1][n][tx];
      __syncthreads();
    }
    if (m0 + ty < M) gq_st_dt(dx, xdt, (size_t)(m0 + ty) * K + k0 + tx, s);
  }
}
__global__ void __launch_bounds__(256) k_front_dgu(const void *dh, const void *g, const void *u, int dt, void *dgo,
                                                   void *duo, size_t mn, int act) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < mn; i += (size_t)gridDim.x * 256) {
    float dg, du;
    front_grads(act, gq_ld_dt(dh, dt, i), gq_ld_dt(g, dt, i), gq_ld_dt(u, dt, i), dg, du);
    if (dgo) gq_st_dt(dgo, dt, i, dg);
    if (duo) gq_st_dt(duo, dt, i, du);
  }
}

int check_front(int fmt, const void *gate, const void *up, size_t M, size_t N, size_t K, int act) {
  GQ_TRY(gq_check_shape(fmt, N, K));
  GQ_CHECK(M <= GQ_MAX_DIM, GQ_ERR_INVALID_ARGS);
  GQ_CHECK(gq_act_valid(act), GQ_ERR_UNSUPPORTED);
  GQ_CHECK(gate && up, GQ_ERR_INVALID_ARGS);
  // the kernels address a packed tensor with 32-bit offsets
  GQ_CHECK(N == 0 || K == 0 || gq_packed_bytes(fmt, N, K) < ((size_t)1 << 32), GQ_ERR_INVALID_ARGS);
  return GQ_OK;
}

}  // namespace

extern "C" size_t gq_ffn_gate_up_workspace_bytes(int fmt, size_t M, size_t N, size_t K) { return 0; }

extern "C" int gq_ffn_gate_up(int fmt, const void *gate, const void *up, const void *x, int x_dtype, void *h,
                              int h_dtype, void *g, void *u, size_t M, size_t N, size_t K, int act, void *ws,
                              size_t ws_bytes, void *stream) {
  GQ_TRY(check_front(fmt, gate, up, M, N, K, act));
  GQ_CHECK(gq_dtype_valid(x_dtype) && gq_dtype_valid(h_dtype), GQ_ERR_UNSUPPORTED);
  GQ_CHECK(x && h, GQ_ERR_INVALID_ARGS);
  if (M == 0 || N == 0) return GQ_OK;
  GQ_CHECK(K > 0, GQ_ERR_INVALID_ARGS);
  const dim3 grid((unsigned)gq_tiles(N), (unsigned)(M < 65536 ? (M + 15) / 16 : 4096));
  hipLaunchKernelGGL(k_front, grid, dim3(256), 0, (hipStream_t)stream, fmt, (const uint8_t *)gate,
                     (const uint8_t *)up, gq_sc_plane_offset(fmt, N, K), x, x_dtype, h, h_dtype, g, u, (int)M, (int)N,
                     (int)K, (int)gq_chunks(fmt, K), act);
  return gq_last_launch();
}

extern "C" size_t gq_ffn_gate_up_bwd_workspace_bytes(int fmt, size_t M, size_t N, size_t K) { return 0; }

extern "C" int gq_ffn_gate_up_bwd(int fmt, const void *gate, const void *up, const void *dh, const void *g,
                                  const void *u, int dtype, void *dg, void *du, void *dx, int dx_dtype, size_t M,
                                  size_t N, size_t K, int act, void *ws, size_t ws_bytes, void *stream) {
  GQ_TRY(check_front(fmt, gate, up, M, N, K, act));
  GQ_CHECK(gq_dtype_valid(dtype) && gq_dtype_valid(dx_dtype), GQ_ERR_UNSUPPORTED);
  GQ_CHECK(dh && g && u, GQ_ERR_INVALID_ARGS);
  if (M == 0 || K == 0) return GQ_OK;
  if (dx) {
    const dim3 grid((unsigned)(K / 16), (unsigned)(M < 65536 ? (M + 15) / 16 : 4096));
    hipLaunchKernelGGL(k_front_dx, grid, dim3(256), 0, (hipStream_t)stream, fmt, (const uint8_t *)gate,
                       (const uint8_t *)up, gq_sc_plane_offset(fmt, N, K), dh, g, u, dtype, dx, dx_dtype, (int)M, (int)N,
                       (int)K, (int)gq_chunks(fmt, K), act);
    GQ_TRY(gq_last_launch());
  }
  if ((dg || du) && N > 0) {
    hipLaunchKernelGGL(k_front_dgu, dim3(4096), dim3(256), 0, (hipStream_t)stream, dh, g, u, dtype, dg, du, M * N, act);
    GQ_TRY(gq_last_launch());
  }
  return GQ_OK;
}
