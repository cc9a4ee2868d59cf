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

// 16 bytes per lane from base + voff + soff straight into LDS (lane l at lds + 16 l)
__device__ __forceinline__ void copy_to_lds(const void* base, char* lds, uint32_t voff, uint32_t soff) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7FFFFFF0u, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, AVT_LDS_PTR(lds), 16, voff, soff, 0, 0);
}

// One workgroup (8 waves) per NT * 16 columns and up to MT * 16 rows; the waves take steps of 128 k in turn, and their sums meet in LDS, added in the order of
// the waves.  Products are of the exact integers 16 + u with the bf16 x, in fp32, and begin at -24 sum x, a product with a matrix of -24, so a group ends with
// y += s sum: the weights are never rounded.
//   1 x 2048 x 2048 3.3 us, 3 x 2048 x 8192 7.8 us, both the launch and one round of loads; 1 x 16384 x 8192 16.1 us, 4.3 TB/s of weights and scales; 33 rows of
// the same 25.1 us among launches on other inputs, 28 to 30 alone: 18.8 of 27.5 without the products, whose operands (weights unpacked, x paired, a wave's 3 x 4 tiles in 250 registers) leave two waves a SIMD.
//   A load whose neighbouring lanes read different rows takes the vector cache 4 cycles per 64 bytes (measured: 59 cycles for 64 x 16 bytes of 16 rows, and these
// loads, not the bytes, set the time: 43 us of 33 x 16384 x 8192 against 24 without those of x), but that is how the matrix unit wants its operands.  So neighbouring
// lanes fetch neighbouring bytes -- weights 64 bytes of each of 16 rows, copied straight into LDS, x 256 bytes of each of 4 rows, through registers -- and a wave
// picks its fragments up from its own piece of LDS, where rows are swizzled over the banks; no wave waits for another before the end.  Four words of weights are then
// exchanged between the lane groups, so that one product of the matrix unit covers 32 consecutive k, i.e. stays inside a group.
template <int MT, int NT, int GS, int XE>
__global__ __launch_bounds__(512) void w4_linear_kernel(W4Args a) {
  constexpr int NW = 8, GPS = 4 / GS, WAVE = 2 * NT * 1024 + 4096;       // GPS: groups of a step; WAVE: bytes of a wave: two steps of weights, 16 rows of x
  constexpr int SC = NT * GPS, SL = (SC + 3) / 4;              // scales of a step per column, loads for them: each lane group fetches another one
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  f32x4_t* part = (f32x4_t*)smem;                              // [NW][NT][MT][64 lanes], at the end
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * NT * 16, m0 = blockIdx.y * MT * 16;
  char* wl = smem + wave * WAVE;
  char* xl = wl + 2 * NT * 1024;
  const size_t rowb = (size_t)a.K / 2;
  const int full = a.K / 128;
  const bf16x8_t minus24 = __builtin_bit_cast(bf16x8_t, (u32x4_t){0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u});
  // (addresses: a uniform base, which moves with the step, and 32-bit lane offsets)
  const uint8_t* qb = a.q + (size_t)n0 * rowb;
  const bf16_t* sb = a.s + (size_t)n0 * a.groups;
  const bf16_t* xb = a.x + (size_t)m0 * a.ldx;
  const int wrow = lane >> 2, wpiece = (lane & 3) ^ (lane >> 4);          // a lane copies piece `wpiece` of row `wrow`: piece p of row r is kept at p ^ (r >> 2)
  uint32_t qo[NT], so[SL];
#pragma unroll
  for (int j = 0; j < NT; ++j) qo[j] = (uint32_t)min(j * 16 + wrow, a.N - 1 - n0) * (uint32_t)rowb;      // (columns behind the last one repeat it and are not stored)
#pragma unroll
  for (int k = 0; k < SL; ++k) so[k] = (uint32_t)min(min(k * 4 + g, SC - 1) / GPS * 16 + c16, a.N - 1 - n0) * a.groups;
  const int xrows = min(a.M - m0, MT * 16);
  f32x4_t y[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) y[j][i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  u32x4_t xr[MT][4];                                           // (of the last row tile only XE: 1 where it has at most 4 rows)
  uint16_t sr[2][SL];
  auto fetch_x = [&](int st, int live) {                       // live: 32-k pieces of the step that exist.  Load e of a tile: rows 4 e + g, 16 bytes per lane
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < (i < MT - 1 ? 4 : XE); ++e)
        xr[i][e] = *(const u32x4_t*)(xb + (size_t)st * 128 + ((uint32_t)min(i * 16 + e * 4 + g, xrows - 1) * (uint32_t)a.ldx + (c16 < live * 4 ? c16 : 0) * 8));
  };
  auto fetch_w = [&](int st, int d, int live) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
      copy_to_lds(qb, wl + (d * NT + j) * 1024, qo[j] + (wpiece < live ? wpiece : 0) * 16, st * 64);
#pragma unroll
    for (int k = 0; k < SL; ++k) sr[d][k] = sb[so[k] + min(st * GPS + min(k * 4 + g, SC - 1) % GPS, a.groups - 1)];
  };
  auto step = [&](int d, int live, auto&& next) {
    u32x4_t w[NT];
    bf16x8_t xf[MT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) w[j] = *(const u32x4_t*)(wl + (d * NT + j) * 1024 + c16 * 64 + ((g ^ (c16 >> 2)) << 4));
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int e = 0; e < (i < MT - 1 ? 4 : XE); ++e) {        // (written by hand: the compiler cannot tell these stores from the copies in flight, and waits for those)
        const int row = e * 4 + g;
        asm volatile("ds_write_b128 %0, %1" ::"v"(lds_addr32(xl) + row * 256 + ((c16 ^ row) << 4)), "v"(xr[i][e]) : "memory");
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) xf[i][e] = *(const bf16x8_t*)(xl + c16 * 256 + (((e * 4 + g) ^ c16) << 4));
    }
    uint32_t sc[SL * 4];                                       // ... and to all four: scale q = (column tile, group of the step)
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      const uint32_t v = sr[d][k];
      auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
      auto even = __builtin_amdgcn_permlane32_swap(p[0], p[0], false, false), odd = __builtin_amdgcn_permlane32_swap(p[1], p[1], false, false);
      sc[k * 4] = even[0]; sc[k * 4 + 1] = odd[0]; sc[k * 4 + 2] = even[1]; sc[k * 4 + 3] = odd[1];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the fragments are in registers: the slot and xr are free
    __builtin_amdgcn_sched_barrier(0);
    next();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NT; ++j) transpose4(w[j]);
#pragma unroll
    for (int e = 0; e < GPS; ++e) {
      if (e * GS >= live) break;
      f32x4_t xs[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xs[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < GS; ++q) {
          xf[i][e * GS + q] = pair8(__builtin_bit_cast(u32x4_t, xf[i][e * GS + q]));
          xs[i] = mfma16(xf[i][e * GS + q], minus24, xs[i]);
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        bf16x8_t wf[GS];
#pragma unroll
        for (int q = 0; q < GS; ++q) wf[q] = unpack8(w[j][e * GS + q]);
        f32x4_t acc[MT];
#pragma unroll
        for (int q = 0; q < GS; ++q)
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i] = mfma16(xf[i][e * GS + q], wf[q], q ? acc[i] : xs[i]);
        const float s = __uint_as_float(sc[j * GPS + e] << 16);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[j][i][r] = fmaf(s, acc[i][r], y[j][i][r]);
      }
    }
  };
  // The order of the requests is x (s + 1), weights (s + 2), and loads come back in order: when x (s) is there, so are the weights of s, and those of s + 1 may still
  // be out.  Requests behind the last step repeat it (a conditional one makes the compiler copy what it loaded, i.e. wait for it).
  const int mine = wave < full ? (full - wave + NW - 1) / NW : 0;
  auto at = [&](int i) { return wave + min(i, mine - 1) * NW; };
  if (mine > 0) {
    fetch_w(at(0), 0, 4);
    __builtin_amdgcn_sched_barrier(0);
    fetch_x(at(0), 4);
    __builtin_amdgcn_sched_barrier(0);
    fetch_w(at(1), 1, 4);
    auto turn = [&](int i, int d) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NT + SL) : "memory");
      step(d, 4, [&] {
        fetch_x(at(i + 1), 4);
        __builtin_amdgcn_sched_barrier(0);
        fetch_w(at(i + 2), d, 4);
      });
    };
    int i = 0;
    for (; i + 2 <= mine; i += 2) { turn(i, 0); turn(i + 1, 1); }
    if (i < mine) turn(i, 0);
  }
  if (a.K % 128 && wave == NW - 1) {                           // a last step of 32, 64 or 96 k
    const int live = (a.K - full * 128) / 32;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    fetch_w(full, 0, live);
    fetch_x(full, live);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    step(0, live, [] {});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // (the requests behind the last step still write into LDS)
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) part[((wave * NT + j) * MT + i) * 64 + lane] = y[j][i];
  __syncthreads();
  for (int o = tid; o < NT * MT * 64; o += 512) {
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

template <int MT, int NT, int GS, int XE>
int launch(const W4Args& a, hipStream_t st) {
  constexpr int ring = 8 * (2 * NT * 1024 + 4096), sums = 8 * NT * MT * 1024, lds = ring > sums ? ring : sums;
  static_assert(lds <= 160 * 1024, "LDS");
  if constexpr (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)w4_linear_kernel<MT, NT, GS, XE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    AVT_CHECK(e == hipSuccess, "avt_w4_linear: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL((w4_linear_kernel<MT, NT, GS, XE>), dim3((a.N + NT * 16 - 1) / (NT * 16), (a.M + MT * 16 - 1) / (MT * 16)), dim3(512), lds, st, a);
  return 0;
}
// (A last tile of at most 4 rows asks for those only: 33 rows of 16384 x 8192 27.9 us, 29.1 with the whole tile; of 2048 x 8192 13.9, 15.1.)
// 33 to 48 rows take three tiles of 16 rows at once and read the weights once; in two blocks of two tiles 33 rows of 6144 x 2048 take 11.6 us instead of 8.0, 48 of 16384 x 8192 44
// instead of 32.7, but 48 of 2048 x 8192 12.5 instead of 16 (one tile of columns each: half of the CUs idle, and two blocks fill them).  From 49 rows on there are two blocks either
// way, and two tiles are the faster up to 64 (64 rows of 16384 x 8192 47.3 us, 55.8 with three); three would be from 65 to 96 (96 rows 67.9, 58.3), and of 6144 x 2048 beyond (1000
// rows 144, 113).  The weights are unpacked again for every block of rows, so that from about 100 rows on (of 2048 x 8192, from about 300) the bf16 product of the unpacked weight is faster: 64
// rows of 6144 x 2048 14.4 us here and 15.2 there, 256 rows 42 and 23, 3000 rows 410 and 102.
template <int NT, int GS>
int launch_cols(const W4Args& a, hipStream_t st) {
  if (a.M <= 4) return launch<1, NT, GS, 1>(a, st);
  if (a.M <= 16) return launch<1, NT, GS, 4>(a, st);
  constexpr int NT3 = (GS < 4 && NT > 2) ? 2 : NT;             // (3 x 4 tiles of small groups do not fit the registers)
  if (a.M > 16 && a.M <= 20) return launch<2, NT, GS, 1>(a, st);
  if (a.M > 32 && a.M <= 36) return launch<3, NT3, GS, 1>(a, st);
  if (a.M > 32 && a.M <= 48) return launch<3, NT3, GS, 4>(a, st);
  return launch<2, NT, GS, 4>(a, st);
}
// As many columns a workgroup as leave three of every four CUs one (more columns share what x costs, fewer workgroups leave CUs idle).  With one / two / four tiles of 16 columns:
// 1 row of 2048 x 8192 6.9 / 9.0 / 12.5 us, of 6144 x 2048 4.9 / 4.4 / 6.4, of 12288 x 2048 7.3 / 7.4 / 7.0; 33 rows of 2048 x 8192 13.6 / 16.9 / 23.9,
// of 6144 x 2048 11.9 / 7.8 / 12.2, of 12288 x 2048 20.1 / 16.9 / 12.6, of 16384 x 8192 52.6 / 37.0 / 29.1.
template <int GS>
int launch_rows(const W4Args& a, hipStream_t st) {
  return a.N >= 64 * 192 ? launch_cols<4, GS>(a, st) : a.N >= 32 * 192 ? launch_cols<2, GS>(a, st) : launch_cols<1, GS>(a, st);
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
  AVT_CHECK(M <= 65535 * 32, "avt_w4_linear: too many rows (%d)", M);
  AVT_CHECK(K < (1 << 24) && ldx < (1 << 24), "avt_w4_linear: K and ldx below 2^24 (K %d, ldx %ld)", K, ldx);
  W4Args a;
  a.x = (const bf16_t*)x; a.q = (const uint8_t*)q; a.s = (const bf16_t*)scales; a.bias = bias; a.res = (const bf16_t*)res; a.out = out;
  a.ldx = ldx; a.ldres = ldres; a.ldo = ldo; a.M = M; a.N = N; a.K = K; a.groups = K / group; a.act = act; a.out_f32 = out_mode;
  const int rc = group == 32 ? launch_rows<1>(a, (hipStream_t)stream) : group == 64 ? launch_rows<2>(a, (hipStream_t)stream) : launch_rows<4>(a, (hipStream_t)stream);
  if (rc) return rc;
  AVT_LAUNCH_CHECK();
  return 0;
}
