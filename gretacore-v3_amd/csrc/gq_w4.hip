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

// one word of codes, or one meta word, a thread
__global__ void __launch_bounds__(256) k_w4_pack(const uint8_t *__restrict__ q, const uint16_t *__restrict__ s, int sbf16,
                                                 const uint8_t *__restrict__ z, size_t N, size_t K, int group,
                                                 uint32_t *__restrict__ codes, uint32_t *__restrict__ meta, size_t n_code,
                                                 size_t n_meta) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t C = (K + kW4Chunk - 1) / kW4Chunk, rb = (K + 1) / 2, ng = (K + group - 1) / group;
  if (i < n_code) {
    const size_t lane = (i >> 2) & 63, tc = i >> 8;
    const size_t n = (tc / C) * 16 + (lane & 15), k = (tc % C) * kW4Chunk + 32 * (i & 3) + 8 * (lane >> 4);
    uint32_t w = 0;
    for (int e = 0; e < 8; ++e)
      if (n < N && k + e < K) {
        const uint32_t c = (q[n * rb + ((k + e) >> 1)] >> (4 * (e & 1))) & 15u;
        const int at = 3 + 16 * (e & 1) + 4 * (e >> 1);
        w |= at < 32 ? c << at : 0u;
        w |= at > 28 ? c >> (32 - at) : 0u;
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
GQ_DEV uint32_t w4_code(uint32_t w, int e) { return (__builtin_rotateright32(w, 4 * (e >> 1) + 3 + 16 * (e & 1))) & 15u; }

// One wave a row; lane l takes every 64th run of 8 k.
template <int MATS>
__global__ void __launch_bounds__(256) k_w4(W4Mats mats, size_t meta_off, const void *x, int xdt, void *y, int ydt, int N,
                                            int K, int C, int group, int batch, int act) {
  const int n = 4 * (int)blockIdx.x + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= N) return;
  for (int b = 0; b < batch; ++b) {
    float s[MATS] = {};
    for (int k = 8 * lane; k < K; k += 512) {
      const size_t tc = (size_t)(n >> 4) * C + (k >> 7);
      for (int m = 0; m < MATS; ++m) {
        const uint32_t w = reinterpret_cast<const uint32_t *>(
            mats.w[m])[tc * 256 + 4 * (16 * ((k >> 3) & 3) + (n & 15)) + ((k >> 5) & 3)];
        const uint32_t v = reinterpret_cast<const uint32_t *>(
            mats.w[m] + meta_off)[(tc * 16 + (n & 15)) * (kW4Chunk / group) + (k & 127) / group];
        const float sc = __uint_as_float(v & ~31u), z = (float)(v & 31u);
        for (int e = 0; e < 8 && k + e < K; ++e)
          s[m] += gq_ld_dt(x, xdt, (size_t)b * K + k + e) * (sc * ((float)w4_code(w, e) - z));
      }
    }
    for (int m = 0; m < MATS; ++m)
      for (int o = 32; o > 0; o >>= 1) s[m] += __shfl_xor(s[m], o, 64);
    if (lane == 0) gq_st_dt(y, ydt, (size_t)b * N + n, MATS == 2 ? gq_act_f(act, s[0]) * s[MATS - 1] : s[0]);
  }
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
  GQ_CHECK(mats.w[0] && mats.w[MATS - 1] && x && y, GQ_ERR_INVALID_ARGS);
  if (N == 0) return GQ_OK;
  GQ_CHECK(K > 0, GQ_ERR_INVALID_ARGS);
  hipLaunchKernelGGL(k_w4<MATS>, dim3((unsigned)((N + 3) / 4)), dim3(256), 0, s, mats, w4_meta_off(N, K), x, x_dtype, y,
                     y_dtype, (int)N, (int)K, (int)w4_chunks(K), group, batch, act);
  return gq_last_launch();
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
  GQ_CHECK(q && scales && packed, GQ_ERR_INVALID_ARGS);
  if (N == 0 || K == 0) return GQ_OK;
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
