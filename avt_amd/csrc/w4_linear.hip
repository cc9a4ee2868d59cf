// A linear layer of few rows on 4-bit weights: y[m, n] = epilogue(sum_g s[n, g] sum_{k in group g} x[m, k] (u[n, k] - 8)), u in 0 .. 15, two to a byte
// (the low nibble holds the even k), s bf16 per group of 32 / 64 / 128 along k.  Epilogue as the GEMM's: + bias, tanh GELU, + residual.
#include "common.hpp"
#include "../../include/avt_hip.h"

namespace {
__device__ __forceinline__ f32x4_t mfma16(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

struct W4Args {
  const bf16_t* x; const uint8_t* q; const bf16_t* s; const float* bias; const bf16_t* res; void* out;
  long ldx, ldres, ldo;
  int M, N, K, groups, act, out_f32;                           // groups = K / group
};

// Eight weights of a word as bf16, in pairs (k, k + 4): 16 + u is 0x4180 | u << 3, exact, so a pair costs a shift and one and-or.
__device__ __forceinline__ bf16x8_t unpack8(uint32_t w) {
  const u32x4_t v = {((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u, ((w >> 5) & 0x00780078u) | 0x41804180u,
                     ((w >> 9) & 0x00780078u) | 0x41804180u};
  return __builtin_bit_cast(bf16x8_t, v);
}
// ... and eight values of x in the same pairs
__device__ __forceinline__ bf16x8_t pair8(u32x4_t x) {
  const u32x4_t v = {__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                     __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
  return __builtin_bit_cast(bf16x8_t, v);
}
// Word i of lane group j (16 lanes) <-> word j of lane group i.
__device__ __forceinline__ void transpose4(u32x4_t& w) {
  auto a = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false), b = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
  auto c = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
  w = (u32x4_t){c[0], d[0], c[1], d[1]};
}

// One workgroup (NW waves) per NT * 16 columns and up to MT * 16 rows; the waves take steps of 128 k in turn, and their sums meet in LDS, added in the order of
// the waves.  A lane fetches 16 bytes of one row of weights (a step is 64 contiguous bytes of each of 16 rows), four words are exchanged between the lane groups so
// that one product of the matrix unit covers 32 consecutive k, i.e. stays inside a group; products are of the exact integers 16 + u with the bf16 x, in fp32, and a
// group ends with y += s (sum - 24 sum x): the weights are never rounded.  sum x comes from a product with ones, in the same layout.
template <int MT, int NT, int GS, int NW>
__global__ __launch_bounds__(NW * 64) void w4_linear_kernel(W4Args a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  f32x4_t* part = (f32x4_t*)smem;                              // [NW][NT][MT][64 lanes]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * NT * 16, m0 = blockIdx.y * MT * 16;
  const size_t rowb = (size_t)a.K / 2;
  const int steps = (a.K + 127) / 128;
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, (u32x4_t){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  constexpr int GPS = 4 / GS;                                  // groups of a step
  const uint8_t* qp[NT];
  const bf16_t* sp[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = min(n0 + j * 16 + c16, a.N - 1);             // (columns behind the last one repeat it and are not stored)
    qp[j] = a.q + n * rowb + g * 16;
    sp[j] = a.s + (size_t)n * a.groups;
  }
  const bf16_t* xp[MT];
  bool live[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    live[i] = m0 + i * 16 + c16 < a.M;
    xp[i] = a.x + (size_t)(live[i] ? m0 + i * 16 + c16 : m0) * a.ldx + g * 8;
  }
  f32x4_t y[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) y[j][i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  u32x4_t w[NT];
  bf16_t sc[NT][GPS];
  auto fetch = [&](int st) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      w[j] = (u32x4_t){0u, 0u, 0u, 0u};
      if (st * 128 + g * 32 < a.K) w[j] = AVT_LDG_NT((const u32x4_t*)(qp[j] + (size_t)st * 64));
#pragma unroll
      for (int e = 0; e < GPS; ++e) sc[j][e] = sp[j][min(st * GPS + e, a.groups - 1)];
    }
  };
  if (wave < steps) fetch(wave);
  for (int st = wave; st < steps; st += NW) {
    u32x4_t xv[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        xv[i][e] = (u32x4_t){0u, 0u, 0u, 0u};
        if (live[i] && st * 128 + e * 32 < a.K) xv[i][e] = *(const u32x4_t*)(xp[i] + (size_t)st * 128 + e * 32);
      }
    u32x4_t cw[NT];
    float cs[NT][GPS];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      cw[j] = w[j];
#pragma unroll
      for (int e = 0; e < GPS; ++e) cs[j][e] = bf2f(sc[j][e]);
    }
    if (st + NW < steps) fetch(st + NW);
#pragma unroll
    for (int j = 0; j < NT; ++j) transpose4(cw[j]);
#pragma unroll
    for (int e = 0; e < GPS; ++e) {
      f32x4_t xs[MT];
      bf16x8_t xf[MT][GS];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xs[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < GS; ++q) { xf[i][q] = pair8(xv[i][e * GS + q]); xs[i] = mfma16(xf[i][q], ones, xs[i]); }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        bf16x8_t wf[GS];
#pragma unroll
        for (int q = 0; q < GS; ++q) wf[q] = unpack8(cw[j][e * GS + q]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < GS; ++q) acc = mfma16(xf[i][q], wf[q], acc);
#pragma unroll
          for (int r = 0; r < 4; ++r) y[j][i][r] = fmaf(cs[j][e], fmaf(-24.f, xs[i][r], acc[r]), y[j][i][r]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) part[((wave * NT + j) * MT + i) * 64 + lane] = y[j][i];
  __syncthreads();
  for (int o = tid; o < NT * MT * 64; o += NW * 64) {
    f32x4_t v = part[o];
    for (int z = 1; z < NW; ++z) v += part[z * NT * MT * 64 + o];
    const int ln = o & 63, i = (o >> 6) % MT, j = (o >> 6) / MT;
    const int n = n0 + j * 16 + (ln & 15);
    if (n >= a.N) continue;
    const float b = a.bias ? a.bias[n] : 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + i * 16 + (ln >> 4) * 4 + r;
      if (m >= a.M) continue;
      float t = v[r] + b;
      if (a.act) t = gelu_tanh(t);
      if (a.res) t += bf2f(a.res[(size_t)m * a.ldres + n]);
      if (a.out_f32) ((float*)a.out)[(size_t)m * a.ldo + n] = t;
      else ((bf16_t*)a.out)[(size_t)m * a.ldo + n] = f2bf(t);
    }
  }
}

template <int MT, int NT, int GS, int NW>
int launch(const W4Args& a, hipStream_t st) {
  constexpr int lds = NW * NT * MT * 1024;
  static_assert(lds <= 160 * 1024, "LDS");
  const hipError_t e = hipFuncSetAttribute((const void*)w4_linear_kernel<MT, NT, GS, NW>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  AVT_CHECK(e == hipSuccess, "avt_w4_linear: %s", hipGetErrorString(e));
  hipLaunchKernelGGL((w4_linear_kernel<MT, NT, GS, NW>), dim3((a.N + NT * 16 - 1) / (NT * 16), (a.M + MT * 16 - 1) / (MT * 16)), dim3(NW * 64), lds, st, a);
  return 0;
}
template <int GS>
int launch_rows(const W4Args& a, hipStream_t st) {
  const bool wide = a.N >= 64 * 192;                           // enough workgroups of 64 columns for most of the CUs
  const int mt = a.M > 48 ? 4 : (a.M + 15) / 16;
  if (wide) return mt == 1 ? launch<1, 4, GS, 8>(a, st) : mt == 2 ? launch<2, 4, GS, 8>(a, st) : mt == 3 ? launch<3, 4, GS, 8>(a, st) : launch<4, 4, GS, 8>(a, st);
  return mt == 1 ? launch<1, 1, GS, 16>(a, st) : mt == 2 ? launch<2, 1, GS, 16>(a, st) : mt == 3 ? launch<3, 1, GS, 8>(a, st) : launch<4, 1, GS, 8>(a, st);
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
  AVT_CHECK((M + 63) / 64 <= 65535, "avt_w4_linear: too many rows (%d)", M);
  W4Args a;
  a.x = (const bf16_t*)x; a.q = (const uint8_t*)q; a.s = (const bf16_t*)scales; a.bias = bias; a.res = (const bf16_t*)res; a.out = out;
  a.ldx = ldx; a.ldres = ldres; a.ldo = ldo; a.M = M; a.N = N; a.K = K; a.groups = K / group; a.act = act; a.out_f32 = out_mode;
  const int rc = group == 32 ? launch_rows<1>(a, (hipStream_t)stream) : group == 64 ? launch_rows<2>(a, (hipStream_t)stream) : launch_rows<4>(a, (hipStream_t)stream);
  if (rc) return rc;
  AVT_LAUNCH_CHECK();
  return 0;
}
