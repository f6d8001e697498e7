// gq_act.h -- activations of the gated feed-forward block and the values of the
// three activation dtypes.
#pragma once
#include "gq_internal.h"

static inline bool gq_dtype_valid(int dt) { return dt == GQ_DT_F32 || dt == GQ_DT_F16 || dt == GQ_DT_BF16; }
static inline bool gq_act_valid(int act) { return act == GQ_ACT_SILU || act == GQ_ACT_GELU_TANH; }
static inline size_t gq_dtype_size(int dt) { return dt == GQ_DT_F32 ? 4 : 2; }

GQ_DEV uint16_t gq_f32_to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }  // (to nearest even)
GQ_DEV float gq_ld_dt(const void *p, int dt, size_t i) {
  if (dt == GQ_DT_F32) return reinterpret_cast<const float *>(p)[i];
  if (dt == GQ_DT_F16) return (float)reinterpret_cast<const _Float16 *>(p)[i];
  return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p)[i] << 16);
}
GQ_DEV void gq_st_dt(void *p, int dt, size_t i, float v) {
  if (dt == GQ_DT_F32) reinterpret_cast<float *>(p)[i] = v;
  else if (dt == GQ_DT_F16) reinterpret_cast<_Float16 *>(p)[i] = (_Float16)v;
  else reinterpret_cast<uint16_t *>(p)[i] = gq_f32_to_bf16(v);
}

// 1 / (1 + e^-x), the reciprocal of one step's error; e^-x overflows to Inf below -88 and the result is then 0
GQ_DEV float gq_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// Both activations are g * sigmoid(p): p = g for SiLU, and for the tanh form of
// GELU 1/2 (1 + tanh t) = sigmoid(2 t), so p = 2 sqrt(2 / pi) (g + 0.044715 g^3).  There
// |g| is cut at 30, where the sigmoid is 0 or 1 in fp32, so that no power of g overflows
// (a NaN stays one).
constexpr float kGelu1 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGelu3 = 0.044715f;
GQ_DEV float gq_gelu_arg(float g) { return fabsf(g) > 30.f ? copysignf(30.f, g) : g; }
GQ_DEV float gq_act_gate(int act, float g) {
  if (act == GQ_ACT_SILU) return gq_sigmoid(g);
  const float c = gq_gelu_arg(g);
  return gq_sigmoid(kGelu1 * c * (1.0f + kGelu3 * c * c));
}
GQ_DEV float gq_act_f(int act, float g) { return g * gq_act_gate(act, g); }
// act(g) and act'(g) = s + g p' s (1 - s), s = sigmoid(p)
GQ_DEV void gq_act_fd(int act, float g, float &f, float &d) {
  const float s = gq_act_gate(act, g), c = act == GQ_ACT_SILU ? g : gq_gelu_arg(g);
  const float dp = act == GQ_ACT_SILU ? 1.0f : kGelu1 * (1.0f + 3.0f * kGelu3 * c * c);
  f = g * s;
  d = s + s * (1.0f - s) * dp * c;
}
