// gq_linear.h -- what follows a product in its epilogue: z = x W^T + bias, y = act(z) + resid.
#pragma once
#include "gq_act.h"

namespace {

struct LinEpi {
  const void *bias, *resid;  // NULL: none; resid may be y
  void *y, *z;               // z NULL: not kept
  int bias_dt, dt, act;      // dt: of resid, y and z
};

// act(z) = z gate(z): 1, z > 0, or as in gq_act.h sigmoid(p(z)), p = a z + b z^3 = z for SiLU and 2 sqrt(2 / pi) (z + 0.044715 z^3) for the
// tanh form of GELU, |z| cut at 100, where the sigmoid is 0 or 1 in fp32, so that no power overflows.  One code for
// both sigmoids: a tile's epilogue is unrolled over its outputs, and every case of an activation is fetched with it.
struct LinAct {
  float a, b;
  bool relu;
};
GQ_DEV LinAct lin_act_of(int act) {
  const bool g = act == GQ_ACT_GELU_TANH;
  return LinAct{g ? kGelu1 : 1.f, g ? kGelu1 * kGelu3 : 0.f, act == GQ_ACT_RELU};
}
GQ_DEV float lin_cut(float z) { return fminf(fmaxf(z, -100.f), 100.f); }
// (not GQ_ACT_NONE; a NaN stays one)
GQ_DEV float lin_act_f(const LinAct &t, float z) {
  const float c = lin_cut(z), s = gq_sigmoid(c * fmaf(t.b * c, c, t.a));
  return t.relu ? (z < 0.f ? 0.f : z) : z * s;
}
GQ_DEV float lin_act(int act, float z) { return act == GQ_ACT_NONE ? z : lin_act_f(lin_act_of(act), z); }
// act'(z): s + c p' s (1 - s)
template <int ACT>
GQ_DEV float lin_act_d(float z) {
  if constexpr (ACT == GQ_ACT_NONE) return 1.f;
  if constexpr (ACT == GQ_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
  float f, d;
  gq_act_fd(ACT, z, f, d);
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

// The tiled kernels (gq_linear_rb.hip): a16 fp16 [M][gq_kpad(K)] in the B fragments' order, rs its row scales (padded by 256; NULL: 1), part: room for
// parts of K, kLinPartBytes
int gq_launch_linear_rb(int fmt, const void *w, const _Float16 *a16, const float *rs, const void *epi, float *part, int M, int N, int K,
                        hipStream_t s);
// the epilogue epi of the parts' sums [parts][M][N] (gq_linear.hip)
int gq_launch_linear_sum(const float *part, const void *epi, int M, int N, int parts, hipStream_t s);
// At most 8 parts, chosen by the rounds they make (gq_linear_rb.hip); their sums together fit kLinPartBytes, those of a workgroup a CU with an fp32
// tile of 128 x 256 outputs each
constexpr int kLinParts = 8;
constexpr size_t kLinPartBytes = (size_t)256 * 128 * 256 * 4;
