// Causal attention of each stream's new tokens over its pages of a shared key / value cache (HF GPT-2 attention with past_key_values, for streams of
// different lengths): query i of a stream with n new tokens and kv cached ones (the new ones among them) sits at position x = kv - n + i and sees the
// keys 0 .. x:  o = sum_{j <= x} softmax_j(scale q k_j) v_j, and 0 where x < 0.
#include "common.hpp"
#include "../../include/avt_hip.h"

namespace {
constexpr int HDMAX = 1024;

// The stream whose new tokens hold row t: the last r with cu[r] <= t, and t < cu[r + 1]; -1 behind the last stream.  All 64 lanes probe at once.
__device__ __forceinline__ int find_stream(const int* __restrict__ cu, int R, int t, int lane) {
  int lo = 0, hi = R;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int p = lo + lane * step;
    const unsigned long long m = __ballot(p < hi && cu[p < hi ? p : lo] <= t);
    const int c = __popcll(m);
    lo += (c > 0 ? c - 1 : 0) * step;
    hi = min(lo + step, hi);
  }
  return cu[lo] <= t && t < cu[lo + 1] ? lo : -1;
}

// One wave per (token, head): keys one after the other, running maximum and sum, everything in fp32.
__global__ __launch_bounds__(256) void paged_attn_row_kernel(const bf16_t* __restrict__ q, long ldq, const bf16_t* __restrict__ kc, const bf16_t* __restrict__ vc,
                                                             long npages, int shift, const int* __restrict__ table, int ldt, int width,
                                                             const int* __restrict__ cu, const int* __restrict__ kv_lens, bf16_t* __restrict__ out, long ldo,
                                                             int T, int R, int H, int Hkv, int hd, float scale) {
  const int lane = threadIdx.x & 63;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (long)T * H) return;
  const int t = (int)(item / H), h = (int)(item % H), hk = h / (H / Hkv);
  const int r = find_stream(cu, R, t, lane);
  if (r < 0) return;
  const int n = min(cu[r + 1], T) - cu[r];
  const long cap = (long)width << shift;
  const int kv = (int)min((long)max(kv_lens[r], 0), cap);
  const int last = kv - n + (t - cu[r]);
  float qv[2][8], acc[2][8];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = (c * 64 + lane) * 8;
      qv[c][e] = d < hd ? bf2f(q[(size_t)t * ldq + h * hd + d + e]) * scale : 0.f;
      acc[c][e] = 0.f;
    }
  float m = -3.0e38f, l = 0.f;
  for (int j = 0; j <= last; ++j) {
    const int pg = table[(size_t)r * ldt + (j >> shift)];
    if (pg < 0 || pg >= npages) continue;                      // an entry that names no page: its keys are not there
    const size_t row = ((((size_t)pg << shift) + (j & ((1 << shift) - 1))) * Hkv + hk) * hd;
    float s = 0.f;
    u32x4_t w[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int d = (c * 64 + lane) * 8;
      if (d < hd) {
        const u32x4_t k = *(const u32x4_t*)(kc + row + d);
        w[c] = *(const u32x4_t*)(vc + row + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) s += qv[c][2 * e] * bflo(k[e]) + qv[c][2 * e + 1] * bfhi(k[e]);
      }
    }
    s = wave_sum(s);
    const float mn = fmaxf(m, s), f = __expf(m - mn), p = __expf(s - mn);
    m = mn;
    l = l * f + p;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int d = (c * 64 + lane) * 8;
      if (d < hd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[c][2 * e] = acc[c][2 * e] * f + p * bflo(w[c][e]);
          acc[c][2 * e + 1] = acc[c][2 * e + 1] * f + p * bfhi(w[c][e]);
        }
      }
    }
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int d = (c * 64 + lane) * 8;
    if (d < hd) {
      u32x4_t w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack2bf(acc[c][2 * e] * inv, acc[c][2 * e + 1] * inv);
      *(u32x4_t*)(out + (size_t)t * ldo + h * hd + d) = w;
    }
  }
}
}  // namespace

extern "C" size_t avt_paged_attn_workspace_bytes(int T, int R, int H, int Hkv, int head_dim, int max_new, int max_kv) { return 16; }

extern "C" int avt_paged_attn_fwd(const void* q, long ldq, const void* kcache, const void* vcache, long npages, int page, const int* table, int ldt, int width,
                                  const int* cu, const int* kv_lens, void* out, long ldo, int T, int R, int H, int Hkv, int head_dim, float scale,
                                  int max_new, int max_kv, void* ws, size_t ws_bytes, void* stream) {
  AVT_CHECK(T >= 0 && R >= 1 && H >= 1 && Hkv >= 1 && H % Hkv == 0, "avt_paged_attn_fwd: bad sizes (T %d, R %d, H %d, Hkv %d)", T, R, H, Hkv);
  AVT_CHECK(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= HDMAX, "avt_paged_attn_fwd: head_dim must be a multiple of 8 in [8, %d] (got %d)", HDMAX, head_dim);
  AVT_CHECK(page >= 8 && page <= 1024 && (page & (page - 1)) == 0, "avt_paged_attn_fwd: the page must be a power of two in [8, 1024] (got %d)", page);
  AVT_CHECK(npages >= 0 && width >= 1 && ldt >= width && (long)width * page <= 0x7fffffffl, "avt_paged_attn_fwd: bad table (width %d, ldt %d, page %d)", width, ldt, page);
  if (T == 0) return 0;
  AVT_CHECK(q && kcache && vcache && table && cu && kv_lens && out, "avt_paged_attn_fwd: null argument");
  AVT_CHECK(ldq >= (long)H * head_dim && ldo >= (long)H * head_dim && ldq % 8 == 0 && ldo % 8 == 0 && aligned16(q) && aligned16(kcache) && aligned16(vcache) && aligned16(out),
            "avt_paged_attn_fwd: 16-byte aligned rows required");
  AVT_CHECK((long)T * H < 0x7f000000l, "avt_paged_attn_fwd: too many rows for one call (%d tokens of %d heads)", T, H);
  hipLaunchKernelGGL(paged_attn_row_kernel, dim3((unsigned)(((long)T * H + 3) / 4)), dim3(256), 0, (hipStream_t)stream, (const bf16_t*)q, ldq, (const bf16_t*)kcache,
                     (const bf16_t*)vcache, npages, __builtin_ctz(page), table, ldt, width, cu, kv_lens, (bf16_t*)out, ldo, T, R, H, Hkv, head_dim, scale);
  AVT_LAUNCH_CHECK();
  return 0;
}
