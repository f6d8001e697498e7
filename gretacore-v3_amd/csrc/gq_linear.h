// gq_linear.h -- what follows a product in its epilogue: z = x W^T + bias, y = act(z) + resid.
#pragma once
#include "gq_act.h"

namespace {

struct LinEpi {
  const void *bias, *resid;  // NULL: none; resid may be y
  void *y, *z;               // z NULL: not kept
  int bias_dt, dt, act;      // dt: of resid, y and z
};

// x / sqrt(2) with the error function: Phi(x) = erfc(-x / sqrt(2)) / 2 keeps its relative accuracy where it is small
GQ_DEV float lin_phi(float x) { return 0.5f * erfcf(-0.7071067811865476f * x); }
GQ_DEV float lin_act(int act, float z) {
  if (act == GQ_ACT_NONE) return z;
  if (act == GQ_ACT_RELU) return z < 0.f ? 0.f : z;  // (a NaN stays one)
  if (act == GQ_ACT_GELU) return z * lin_phi(z);
  return gq_act_f(act, z);
}
GQ_DEV float lin_act_d(int act, float z) {
  if (act == GQ_ACT_NONE) return 1.f;
  if (act == GQ_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
  if (act == GQ_ACT_GELU) {
    // Phi(z) + z phi(z), phi the normal density
    return lin_phi(z) + z * 0.3989422804014327f * __expf(-0.5f * fminf(z * z, 1e30f));
  }
  float f, d;
  gq_act_fd(act, z, f, d);
  return d;
}
// bias and residual of output (m, n), loaded ahead of the sums; the output of a product's sum v
struct LinTail {
  float bias, resid;
};
GQ_DEV LinTail lin_tail(const LinEpi &e, size_t m, int n, int N) {
  return LinTail{e.bias ? gq_ld_dt(e.bias, e.bias_dt, n) : 0.f, e.resid ? gq_ld_dt(e.resid, e.dt, m * (size_t)N + n) : 0.f};
}
GQ_DEV void lin_put(const LinEpi &e, size_t m, int n, int N, float v, const LinTail &t) {
  const size_t i = m * (size_t)N + n;
  v += t.bias;
  if (e.z) gq_st_dt(e.z, e.dt, i, v);
  gq_st_dt(e.y, e.dt, i, lin_act(e.act, v) + t.resid);
}

}  // namespace

// The tiled kernels (gq_linear_rb.hip): a16 fp16 [M][gq_kpad(K)] in the B fragments' order, rs its row scales (padded by 256), part: room for
// parts of K, kLinPartBytes
int gq_launch_linear_rb(int fmt, const void *w, const _Float16 *a16, const float *rs, const void *epi, float *part, int M, int N, int K,
                        hipStream_t s);
// the epilogue epi of the parts' sums [parts][M][N] (gq_linear.hip)
int gq_launch_linear_sum(const float *part, const void *epi, int M, int N, int parts, hipStream_t s);
// Parts are taken only as far as a workgroup a CU goes, each with an fp32 tile of at most 128 x 256 outputs, and at most 8
constexpr int kLinParts = 8;
constexpr size_t kLinPartBytes = (size_t)256 * 128 * 256 * 4;
