// A linear layer of few rows on 4-bit weights: y[m, n] = epilogue(sum_g s[n, g] sum_{k in group g} x[m, k] (u[n, k] - 8)), u in 0 .. 15, two to a byte
// (the low nibble holds the even k), s bf16 per group of 32 / 64 / 128 along k.  Epilogue as the GEMM's: + bias, tanh GELU, + residual.
#include "common.hpp"
#include "../../include/avt_hip.h"

namespace {
// One wave per output value: lanes over 8 k at a time (one word of weights).
__global__ __launch_bounds__(256) void w4_row_kernel(const bf16_t* __restrict__ x, long ldx, const uint8_t* __restrict__ q, const bf16_t* __restrict__ s,
                                                     int gshift, const float* __restrict__ bias, int act, const bf16_t* __restrict__ res, long ldres,
                                                     void* __restrict__ out, long ldo, int out_f32, int M, int N, int K) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), m = blockIdx.y;
  if (n >= N) return;
  float acc = 0.f;
  for (int k = lane * 8; k < K; k += 512) {
    const uint32_t w = *(const uint32_t*)(q + (size_t)n * (K / 2) + k / 2);
    const u32x4_t xv = *(const u32x4_t*)(x + (size_t)m * ldx + k);
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) a += bflo(xv[e]) * (float)((int)(w >> (8 * e) & 15) - 8) + bfhi(xv[e]) * (float)((int)(w >> (8 * e + 4) & 15) - 8);
    acc += a * bf2f(s[(size_t)n * (K >> gshift) + (k >> gshift)]);
  }
  acc = wave_sum(acc);
  if (lane == 0) {
    if (bias) acc += bias[n];
    if (act) acc = gelu_tanh(acc);
    if (res) acc += bf2f(res[(size_t)m * ldres + n]);
    if (out_f32) ((float*)out)[(size_t)m * ldo + n] = acc;
    else ((bf16_t*)out)[(size_t)m * ldo + n] = f2bf(acc);
  }
}
}  // namespace

extern "C" int avt_w4_linear(const void* x, long ldx, const void* q, const void* scales, int group, const float* bias, int act, const void* res, long ldres,
                             void* out, long ldo, int out_mode, int M, int N, int K, void* stream) {
  AVT_CHECK(M >= 0 && N >= 1 && K >= 1, "avt_w4_linear: bad sizes (M %d, N %d, K %d)", M, N, K);
  AVT_CHECK(group == 32 || group == 64 || group == 128, "avt_w4_linear: the group must be 32, 64 or 128 (got %d)", group);
  AVT_CHECK(K % group == 0, "avt_w4_linear: K must be a multiple of the group (K %d, group %d)", K, group);
  AVT_CHECK(act == 0 || act == 2, "avt_w4_linear: act must be 0 (none) or 2 (tanh GELU), got %d", act);
  AVT_CHECK(out_mode == 0 || out_mode == 1, "avt_w4_linear: out_mode must be 0 (bf16) or 1 (fp32), got %d", out_mode);
  if (M == 0) return 0;
  AVT_CHECK(x && q && scales && out, "avt_w4_linear: null argument");
  AVT_CHECK(ldx >= K && ldx % 8 == 0 && aligned16(x) && aligned16(q), "avt_w4_linear: 16-byte aligned rows of x and q required");
  AVT_CHECK(ldo >= N && (!res || ldres >= N), "avt_w4_linear: leading dimension below N");
  hipLaunchKernelGGL(w4_row_kernel, dim3((N + 3) / 4, M), dim3(256), 0, (hipStream_t)stream, (const bf16_t*)x, ldx, (const uint8_t*)q, (const bf16_t*)scales,
                     __builtin_ctz(group), bias, act, (const bf16_t*)res, ldres, out, ldo, out_mode, M, N, K);
  AVT_LAUNCH_CHECK();
  return 0;
}
