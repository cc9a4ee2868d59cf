// Causal attention of each stream's new tokens over its pages of a shared key / value cache (HF GPT-2 attention with past_key_values, for streams of
// different lengths): query i of a stream with n new tokens and kv cached ones (the new ones among them) sits at position x = kv - n + i and sees the
// keys 0 .. x:  o = sum_{j <= x} softmax_j(scale q k_j) v_j, and 0 where x < 0.
#include <type_traits>
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

__device__ const u32x4_t ZERO_CHUNK = {0u, 0u, 0u, 0u};       // what a lane copies where there is no key (behind the last one, no page) or no column

struct AttnArgs {
  const bf16_t* q; const bf16_t* kc; const bf16_t* vc; const int* table; const int* cu; const int* kv_lens;
  bf16_t* out; float* part_o; float* part_ml;                  // part_*: one partial result per split and row ([split][T * H][hd], [split][T * H] (max, sum))
  long ldq, ldo, npages;
  int shift, ldt, width, T, R, H, Hkv, grp, hd, nsplit, cmin;
  float scale_log2;                                            // scale * log2(e): exponentials are powers of two
};

// Keys of one split: a stream's cached tokens are cut into at most nsplit pieces, each a multiple of `cmin` keys (itself a multiple of the tile's).
__device__ __forceinline__ long split_keys(int kv, int nsplit, int cmin) {
  const long c = ((long)kv + nsplit - 1) / nsplit;
  return (c + cmin - 1) / cmin * cmin;
}

// 16-byte piece c of row r of a [keys][HD] tile is kept at c ^ tile_swz(r): a copy into LDS fills whole rows lane by lane, so the swizzle is applied to what a lane
// fetches.  8 consecutive rows land on 8 different 32-byte slots (transposing reads of V: 8 rows x 32 bytes per half wave), 16 rows on 16 different 16-byte slots
// (row fragments of K); rows of 128 bytes pair up in a 256-byte line (the permutation of vit_attention.hip).
template <int HD>
__device__ __forceinline__ int tile_swz(int r) {
  if constexpr (HD == 64) { const int p = (r >> 1) & 7, hi = p >> 2; return (((p & 3) ^ (hi << 1)) << 1) | hi; }
  else return ((r & 7) << 1) | ((r >> 3) & 1);
}

__device__ __forceinline__ f32x4_t mfma16(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float gsum(float v) { v += __shfl_xor(v, 16, 64); return v + __shfl_xor(v, 32, 64); }
__device__ __forceinline__ float gmax(float v) { v = fmaxf(v, __shfl_xor(v, 16, 64)); return fmaxf(v, __shfl_xor(v, 32, 64)); }

// Tile i of a stream's rows (a row = a new token and one of the query heads that share the kv head) is tile cu[r] * grp / BM + r + i of the grid: the tiles of
// two streams never meet, the sum over the streams is known on the host from T and R, and no list of tiles has to be made.
__device__ __forceinline__ int tile_base(const int* __restrict__ cu, int r, int T, int grp, int bm) { return max(0, min(cu[r], T)) * grp / bm + r; }
__device__ __forceinline__ int find_tile(const int* __restrict__ cu, int R, int T, int grp, int bm, int tile, int lane) {
  int lo = 0, hi = R;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int p = lo + lane * step;
    const int c = __popcll(__ballot(p < hi && tile_base(cu, p < hi ? p : lo, T, grp, bm) <= tile));
    lo += (c > 0 ? c - 1 : 0) * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

// One workgroup (4 waves) per (kv head, tile of NQ * 16 rows, split of the keys).  K and V tiles of BN keys come into LDS by direct copies, row by row through the
// page table, two tiles in turn.  S^T = K Q^T: wave w takes 16 keys (w % KT) of the tile and, where the tile has fewer than 64 keys, its share of the head's
// columns (w / KT); the scores pass through LDS (16 bytes per lane, the same lane reads them) and every wave then has all of them in the layout of P^T, the right
// operand of O^T = V^T P^T, and keeps the running maximum and sum (fp32) of every row for itself: no reduction between waves.  Wave w owns a quarter of the head's
// columns of O.  P is rounded to bf16 for the product (the matrix unit's type; half a step 2^-8 of each probability), the sum is of the unrounded ones.
template <int HD, int NQ, int BN>
__global__ __launch_bounds__(256) void paged_attn_tile_kernel(AttnArgs a) {
  constexpr int ROWB = HD * 2, TILEB = BN * ROWB, KT = BN / 16, KS = 4 / KT, DS = HD / KS / 32, DT = HD / 64, TT = BN >= 32 ? BN / 32 : 1, BM = NQ * 16;
  constexpr int NI = TILEB / 4096;                             // copies of 1 KB per wave and tensor
  static_assert(KT * KS == 4 && DS >= 1 && NI >= 1 && 48 * ROWB < 65536 + 32 * ROWB, "tile shape");
  extern __shared__ __attribute__((aligned(1024))) char smem[];          // [2 tiles][K | V], scores, flag
  f32x4_t* sx = (f32x4_t*)(smem + 4 * TILEB);                  // [NQ][4 waves][64 lanes]
  int* odd = (int*)(smem + 4 * TILEB + NQ * 4096);             // some value of V in a partly hidden tile is not finite
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % a.Hkv, tile = (gridDim.x - 1 - blockIdx.x) / a.Hkv, sp = blockIdx.y;      // (the last rows of a chunk see the most keys: first)
  const int r = __builtin_amdgcn_readfirstlane(find_tile(a.cu, a.R, a.T, a.grp, BM, tile, lane));
  const int t0 = max(0, min(a.cu[r], a.T)), n = max(0, min(a.cu[r + 1], a.T) - t0);
  const int row0 = (tile - tile_base(a.cu, r, a.T, a.grp, BM)) * BM, rows = n * a.grp;
  if (row0 < 0 || row0 >= rows) return;
  const int kv = (int)min((long)max(a.kv_lens[r], 0), (long)a.width << a.shift);
  const int first = kv - n + row0 / a.grp, last = kv - n + (min(row0 + BM, rows) - 1) / a.grp;      // positions of the tile's first and last row
  const long chunk = split_keys(kv, a.nsplit, a.cmin);
  const int k0 = (int)min((long)sp * chunk, (long)kv), k1 = (int)min((long)(sp + 1) * chunk, (long)(last + 1));
  if (k0 >= k1 && a.nsplit > 1) return;                        // (the join knows)
  const int* tab = a.table + (size_t)r * a.ldt;
  const int pmask = (1 << a.shift) - 1;

  int pos[NQ];                                                 // this lane's row (column of S^T): its position, -1: no row
  bf16x8_t qf[NQ][DS];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = row0 + i * 16 + c16, tok = row / a.grp;
    const bool ok = row < rows;
    pos[i] = ok ? kv - n + tok : -1;
    const bf16_t* p = a.q + (size_t)(t0 + (ok ? tok : 0)) * a.ldq + (size_t)(hk * a.grp + (ok ? row - tok * a.grp : 0)) * a.hd;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = (wave / KT) * (HD / KS) + s * 32 + g * 8;
      u32x4_t w = {0u, 0u, 0u, 0u};
      if (ok && d < a.hd) w = *(const u32x4_t*)(p + d);
      qf[i][s] = __builtin_bit_cast(bf16x8_t, w);
    }
  }
  bool gap = false;                                            // a table entry of this range names no page
  if (k0 < k1)
    for (int e = (k0 >> a.shift) + lane; e <= (k1 - 1) >> a.shift; e += 64) { const int pg = tab[e]; gap |= pg < 0 || pg >= a.npages; }
  gap = __any(gap);
  if (tid == 0) *odd = 0;

  // copies of one tile: instruction ii of the tile fills bytes [1024 ii, 1024 ii + 1024); its rows lie in one page (a page holds at least 8 tokens)
  auto page_of = [&](int j0, int i) {
    const int jb = j0 + (i * 4 + wave) * 1024 / ROWB;
    return tab[min(jb, k1 - 1) >> a.shift];
  };
  int pg[NI];
  auto issue = [&](int j0, int stage) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int at = (i * 4 + wave) * 1024 + lane * 16, row = at / ROWB, c = ((at % ROWB) >> 4) ^ tile_swz<HD>(row), j = j0 + row;
      const bool ok = j < k1 && pg[i] >= 0 && pg[i] < a.npages && c * 8 < a.hd;
      const size_t off = ((((size_t)(uint32_t)pg[i] << a.shift) + (j & pmask)) * a.Hkv + hk) * a.hd + c * 8;
      const bf16_t* ks = ok ? a.kc + off : (const bf16_t*)&ZERO_CHUNK;
      const bf16_t* vs = ok ? a.vc + off : (const bf16_t*)&ZERO_CHUNK;
      char* dst = smem + stage * 2 * TILEB + (i * 4 + wave) * 1024;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)ks, AVT_LDS_PTR(dst), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)vs, AVT_LDS_PTR(dst + TILEB), 16, 0, 0);
    }
  };
  auto pages = [&](int j0) {
    if (j0 < k1) {
#pragma unroll
      for (int i = 0; i < NI; ++i) pg[i] = page_of(j0, i);
    }
  };

  f32x4_t o[NQ][DT];
  float m[NQ], l[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[i][d] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  const int kswz = tile_swz<HD>(c16);
  const int krow = ((wave % KT) * 16 + c16) * ROWB, kc0 = (wave / KT) * (HD / KS / 8) + g;
  const int vr = 4 * g + (c16 >> 2);
  const uint32_t vaddr0 = lds_addr32(smem) + TILEB + vr * ROWB + (((wave * (HD / 32) + ((c16 & 3) >> 1)) ^ tile_swz<HD>(vr)) << 4) + (c16 & 1) * 8;

  // (Q is waited for here: left to the first product, the compiler's wait for it would sit inside the loop and wait for the copies in flight as well)
#pragma unroll
  for (int i = 0; i < NQ; ++i)
#pragma unroll
    for (int s = 0; s < DS; ++s) asm volatile("" : "+v"(qf[i][s]));
  if (k0 < k1) { pages(k0); issue(k0, 0); pages(k0 + BN); }
  int stage = 0;
  for (int j0 = k0; j0 < k1; j0 += BN, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");       // the tile is there, and every wave is done with the other one and with the scores
    if (j0 + BN < k1) { issue(j0 + BN, stage ^ 1); pages(j0 + 2 * BN); }
    const char* kt = smem + stage * 2 * TILEB;
    f32x4_t s4[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) s4[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const bf16x8_t kf = *(const bf16x8_t*)(kt + krow + (((kc0 + 4 * s) ^ kswz) << 4));
#pragma unroll
      for (int i = 0; i < NQ; ++i) s4[i] = mfma16(kf, qf[i][s], s4[i]);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) sx[(i * 4 + wave) * 64 + lane] = s4[i];
    const bool hide = gap || j0 + BN - 1 > first;              // some row does not see some key of this tile
    const bool uneven = first < last && j0 + BN - 1 > first;   // ... and another one does: a value that is not finite must not pass
    if (uneven) {
      bool bad = false;
      for (int i = tid; i < TILEB / 16; i += 256) {
        const u32x4_t w = *(const u32x4_t*)(kt + TILEB + i * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
      }
      if (__any(bad) && lane == 0) *odd = 1;
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const bool slow = uneven && *odd;
    bf16x8_t pf[NQ][TT];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      f32x4_t p[KT];
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        p[k] = sx[(i * 4 + k) * 64 + lane];
#pragma unroll
        for (int q = 1; q < KS; ++q) p[k] += sx[(i * 4 + q * KT + k) * 64 + lane];
        p[k] *= a.scale_log2;
      }
      if (hide) {
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const int j = j0 + k * 16 + g * 4;
          bool there = true;                                   // (4 keys, one page)
          if (gap && j < k1) { const int e = tab[j >> a.shift]; there = e >= 0 && e < a.npages; }
#pragma unroll
          for (int e = 0; e < 4; ++e) p[k][e] = there && j + e <= pos[i] && j + e < k1 ? p[k][e] : -INFINITY;
        }
      }
#pragma unroll
      for (int k = 0; k < KT; ++k) mx = fmaxf(mx, fmaxf(fmaxf(p[k][0], p[k][1]), fmaxf(p[k][2], p[k][3])));
      mx = gmax(mx);
      const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(m[i] - ms);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) { p[k][e] = __builtin_amdgcn_exp2f(p[k][e] - ms); sum += p[k][e]; }
      l[i] = l[i] * f + sum;
      if (__any(f != 1.f)) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[i][d] *= f;
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        u32x4_t w = {pack2bf(p[2 * t][0], p[2 * t][1]), pack2bf(p[2 * t][2], p[2 * t][3]), 0u, 0u};
        if constexpr (KT > 1) { w[2] = pack2bf(p[2 * t + 1][0], p[2 * t + 1][1]); w[3] = pack2bf(p[2 * t + 1][2], p[2 * t + 1][3]); }
        pf[i][t] = __builtin_bit_cast(bf16x8_t, w);
      }
    }
    const uint32_t va = vaddr0 + stage * 2 * TILEB;
    auto product = [&](auto checked) {
      constexpr int G = DT < 4 ? DT : 4;                         // fragments read ahead of their products
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += G) {
        bf16x8_t vf[G][TT];
#pragma unroll
        for (int d = 0; d < G; ++d) {
          const uint32_t ad = (va ^ (((d0 + d) & 7) * 32)) + ((d0 + d) >> 3) * 256;
          if constexpr (BN == 16) vf[d][0] = tr_join(ds_read_tr_na<0>(ad), (u32x2_t){0u, 0u});
          else vf[d][0] = tr_join(ds_read_tr_na<0>(ad), ds_read_tr_na<16 * ROWB>(ad));
          if constexpr (TT > 1) vf[d][TT - 1] = tr_join(ds_read_tr_na<(BN > 32 ? 32 : 0) * ROWB>(ad), ds_read_tr_na<(BN > 32 ? 48 : 0) * ROWB>(ad));
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int d = 0; d < G; ++d)
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            asm volatile("" : "+v"(vf[d][t]));
            if constexpr (decltype(checked)::value) {
              u32x4_t w = __builtin_bit_cast(u32x4_t, vf[d][t]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
                if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu;
              }
              vf[d][t] = __builtin_bit_cast(bf16x8_t, w);
            }
#pragma unroll
            for (int i = 0; i < NQ; ++i) o[i][d0 + d] = mfma16(vf[d][t], pf[i][t], o[i][d0 + d]);
          }
      }
    };
    if (!slow) product(std::false_type{});
    else product(std::true_type{});
    if (slow) {                                                // the values that are not finite, for the rows that see them
      for (int k = 0; k < BN; ++k) {
        const int j = j0 + k;
        if (j >= k1) break;
        bool there = true;
        if (gap) { const int e = tab[j >> a.shift]; there = e >= 0 && e < a.npages; }
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          const int from = (k & 12) * 4 + c16;                 // the lane that holds this key's scores of this lane's row
          float s = sx[(i * 4 + k / 16) * 64 + from][k & 3];
#pragma unroll
          for (int q = 1; q < KS; ++q) s += sx[(i * 4 + q * KT + k / 16) * 64 + from][k & 3];
          const float p = fmaxf(__builtin_amdgcn_exp2f(s * a.scale_log2 - (m[i] == -INFINITY ? 0.f : m[i])), 1e-30f);
          const bool see = there && j <= pos[i];
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const int col = wave * (HD / 4) + d * 16 + g * 4;
            const u32x2_t w = *(const u32x2_t*)(kt + TILEB + k * ROWB + (((col >> 3) ^ tile_swz<HD>(k)) << 4) + (col & 7) * 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = e & 1 ? bfhi(w[e >> 1]) : bflo(w[e >> 1]);
              if (see && (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[i][d][e] += p * v;
            }
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const float lt = gsum(l[i]);
    const int row = row0 + i * 16 + c16, tok = row / a.grp;
    if (row >= rows) continue;
    const int h = hk * a.grp + row - tok * a.grp;
    const size_t t = t0 + tok;
    if (a.nsplit == 1) {
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int col = wave * (HD / 4) + d * 16 + g * 4;
        if (col < a.hd) *(u32x2_t*)(a.out + t * a.ldo + (size_t)h * a.hd + col) = (u32x2_t){pack2bf(o[i][d][0] * inv, o[i][d][1] * inv), pack2bf(o[i][d][2] * inv, o[i][d][3] * inv)};
      }
    } else {
      const size_t rid = ((size_t)sp * a.T + t) * a.H + h;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int col = wave * (HD / 4) + d * 16 + g * 4;
        if (col < a.hd) *(f32x4_t*)(a.part_o + rid * a.hd + col) = o[i][d];
      }
      if (wave == 0 && g == 0) { a.part_ml[rid * 2] = m[i]; a.part_ml[rid * 2 + 1] = lt; }
    }
  }
}

// The partial results of the splits that a row's keys reach, joined in their order: weights 2^(m_z - max m), fp32.
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  const int r = __builtin_amdgcn_readfirstlane(find_stream(a.cu, a.R, t, lane));
  if (r < 0) return;
  const int t0 = max(0, min(a.cu[r], a.T)), n = max(0, min(a.cu[r + 1], a.T) - t0);
  const int kv = (int)min((long)max(a.kv_lens[r], 0), (long)a.width << a.shift);
  const int pos = kv - n + (t - t0);
  const int nz = pos < 0 ? 0 : (int)(pos / split_keys(kv, a.nsplit, a.cmin)) + 1;
  const int idx = blockIdx.y * 256 + threadIdx.x;
  if (idx >= a.H * a.hd / 4) return;
  const int h = idx * 4 / a.hd;
  const size_t step = (size_t)a.T * a.H, rid = (size_t)t * a.H + h;
  float mx = -INFINITY;
  for (int z = 0; z < nz; ++z) mx = fmaxf(mx, a.part_ml[(rid + z * step) * 2]);
  if (mx == -INFINITY) mx = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int z = 0; z < nz; ++z) {
    const float f = __builtin_amdgcn_exp2f(a.part_ml[(rid + z * step) * 2] - mx);
    l += f * a.part_ml[(rid + z * step) * 2 + 1];
    const f32x4_t p = *(const f32x4_t*)(a.part_o + (rid + z * step) * a.hd + (idx * 4 - h * a.hd));
    if (f != 0.f) o += p * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *(u32x2_t*)(a.out + (size_t)t * a.ldo + idx * 4) = (u32x2_t){pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv)};
}

// ---- choices on the host, from sizes alone -----------------------------------------------------------------------------------------------------------
struct Choice { int hd, nq, bn, nsplit, cmin; long tiles; };

Choice choose(int T, int R, int H, int Hkv, int hd, long max_new, long max_kv, int cu_count) {
  Choice c;
  c.hd = hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : hd <= 512 ? 512 : 1024;
  const int grp = H / Hkv;
  const long rows = (max_new > 0 && max_new < T ? max_new : (T + R - 1) / R) * grp;      // rows of a stream and kv head
  c.nq = rows <= 16 || c.hd == 1024 ? 1 : c.hd == 512 ? 2 : 4;
  c.bn = c.hd <= 128 ? 64 : c.hd <= 512 ? 32 : 16;
  c.tiles = (long)T * grp / (16 * c.nq) + R;
  c.cmin = 256;
  const long items = c.tiles * Hkv;
  long want = (2l * cu_count + items - 1) / items, most = (max_kv + c.cmin - 1) / c.cmin;
  if (want > most) want = most;
  if (want > 128) want = 128;
  c.nsplit = want < 1 ? 1 : (int)want;
  return c;
}

long part_floats(const Choice& c, long T, long H, long hd) { return c.nsplit > 1 ? c.nsplit * T * H * (hd + 2) : 0; }

template <int HD, int NQ, int BN>
int launch_tiles(const AttnArgs& a, const Choice& c, hipStream_t st) {
  constexpr int lds = 4 * BN * HD * 2 + NQ * 4096 + 64;
  static_assert(lds <= 160 * 1024, "LDS");
  if constexpr (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)paged_attn_tile_kernel<HD, NQ, BN>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    AVT_CHECK(e == hipSuccess, "avt_paged_attn_fwd: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL((paged_attn_tile_kernel<HD, NQ, BN>), dim3((unsigned)(c.tiles * a.Hkv), c.nsplit), dim3(256), lds, st, a);
  return 0;
}
constexpr int CUS = 256;
}  // namespace

extern "C" size_t avt_paged_attn_workspace_bytes(int T, int R, int H, int Hkv, int head_dim, int max_new, int max_kv) {
  if (T < 1 || R < 1 || Hkv < 1 || H < Hkv || head_dim < 1) return 16;
  return 16 + 4 * (size_t)part_floats(choose(T, R, H, Hkv, head_dim, max_new, max_kv > 0 ? max_kv : 0x7fffffff, CUS), T, H, head_dim);
}

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
  const Choice c = choose(T, R, H, Hkv, head_dim, max_new, max_kv > 0 ? max_kv : 0x7fffffff, CUS);
  AVT_CHECK(c.tiles * Hkv < 0x7f000000l, "avt_paged_attn_fwd: too many rows for one call (%d tokens of %d streams)", T, R);
  const long pf = part_floats(c, T, H, head_dim);
  AVT_CHECK(pf == 0 || (ws && aligned16(ws) && ws_bytes >= 4 * (size_t)pf), "avt_paged_attn_fwd: workspace of %ld bytes needed", 4 * pf);
  AttnArgs a;
  a.q = (const bf16_t*)q; a.kc = (const bf16_t*)kcache; a.vc = (const bf16_t*)vcache; a.table = table; a.cu = cu; a.kv_lens = kv_lens; a.out = (bf16_t*)out;
  a.part_o = (float*)ws; a.part_ml = (float*)ws + (size_t)c.nsplit * T * H * head_dim;
  a.ldq = ldq; a.ldo = ldo; a.npages = npages; a.shift = __builtin_ctz(page); a.ldt = ldt; a.width = width; a.T = T; a.R = R; a.H = H; a.Hkv = Hkv; a.grp = H / Hkv;
  a.hd = head_dim; a.nsplit = c.nsplit; a.cmin = c.cmin; a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  int rc = 0;
  if (c.nq == 1) rc = c.hd == 64 ? launch_tiles<64, 1, 64>(a, c, st) : c.hd == 128 ? launch_tiles<128, 1, 64>(a, c, st) : c.hd == 256 ? launch_tiles<256, 1, 32>(a, c, st)
                    : c.hd == 512 ? launch_tiles<512, 1, 32>(a, c, st) : launch_tiles<1024, 1, 16>(a, c, st);
  else rc = c.hd == 64 ? launch_tiles<64, 4, 64>(a, c, st) : c.hd == 128 ? launch_tiles<128, 4, 64>(a, c, st) : c.hd == 256 ? launch_tiles<256, 4, 32>(a, c, st)
          : launch_tiles<512, 2, 32>(a, c, st);
  if (rc) return rc;
  AVT_LAUNCH_CHECK();
  if (c.nsplit > 1) {
    hipLaunchKernelGGL(paged_attn_join_kernel, dim3(T, (H * head_dim / 4 + 255) / 256), dim3(256), 0, st, a);
    AVT_LAUNCH_CHECK();
  }
  return 0;
}
