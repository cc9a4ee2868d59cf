// Causal attention of each stream's new tokens over its pages of a shared key / value cache (HF GPT-2 attention with past_key_values, for streams of
// different lengths): query i of a stream with n new tokens and kv cached ones (the new ones among them) sits at position x = kv - n + i and sees the
// keys 0 .. x:  o = sum_{j <= x} softmax_j(scale q k_j) v_j, and 0 where x < 0.
#include <algorithm>
#include "common.hpp"
#include "../../include/avt_hip.h"

namespace {
constexpr int HDMAX = 1024, MAX_SPLITS = 128, FEW_SPLITS = 4;

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

struct AttnArgs {
  const bf16_t* q; const bf16_t* kc; const bf16_t* vc; const int* table; const int* cu; const int* kv_lens;
  bf16_t* out; float* part_o; float* part_ml;                  // part_*: one partial result per split and row ([split][T * H][hd], [split][T * H] (max, sum))
  long ldq, ldo, npages;
  int shift, ldt, width, T, R, H, Hkv, grp, hd, nsplit, cmin;
  float scale_log2;                                            // |scale| log2(e): exponentials are powers of two
  uint32_t rowe;                                               // elements of a token's row in a cache: Hkv hd
  uint32_t q_and, q_xor;                                       // applied to q as it is read: the sign of a negative scale; a scale of 0 is a q of 0
};

// Keys of one split: a stream's cached tokens are cut into at most nsplit pieces of at least `cmin` keys, in steps of 64 (a multiple of every tile).
__device__ __forceinline__ long split_keys(int kv, int nsplit, int cmin) {
  const long c = ((long)kv + nsplit - 1) / nsplit;
  return ((c < cmin ? cmin : c) + 63) / 64 * 64;
}

typedef const __attribute__((address_space(4))) int* table_t;  // (the table does not change while a kernel runs: its entries come through the scalar cache)

// 16-byte piece c of row r of a [keys][HD] tile is kept at c ^ swz(r): a copy into LDS fills whole rows lane by lane, so the swizzle is applied to what a lane
// fetches.  Row fragments of K want 16 rows on 16 different 16-byte slots; the transposing reads of V take 8 rows x 32 bytes per half wave (16-row products) or
// 4 rows x 64 bytes (32-row products), which want 8 rows on 8 different 32-byte slots or 4 rows on 4 different 64-byte ones.  Rows of 128 bytes pair up in a line.
template <int HD>
__device__ __forceinline__ int swz16(int r) {
  if constexpr (HD == 64) { const int p = (r >> 1) & 7, hi = p >> 2; return (((p & 3) ^ (hi << 1)) << 1) | hi; }
  else return ((r & 7) << 1) | ((r >> 3) & 1);
}
template <int HD>
__device__ __forceinline__ int swz32(int r) {
  if constexpr (HD == 64) { const int p = (r >> 1) & 7; return ((p & 1) << 2) | (p >> 1); }
  else return ((r & 3) << 2) | ((r >> 2) & 3);
}

__device__ __forceinline__ f32x4_t mfma16(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float gsum(float v) { v += __shfl_xor(v, 16, 64); return v + __shfl_xor(v, 32, 64); }
__device__ __forceinline__ float gmax(float v) { v = fmaxf(v, __shfl_xor(v, 16, 64)); return fmaxf(v, __shfl_xor(v, 32, 64)); }

// Tile i of a stream's rows (a row = a new token and one of the query heads that share the kv head) is tile cu[r] * grp / BM + r + i of the grid: the tiles of
// two streams never meet, the sum over the streams is known on the host from T and R, and no list of tiles has to be made.
__device__ __forceinline__ int tile_base(const int* __restrict__ cu, int r, int T, int grp, int bm) { return max(0, min(cu[r], T)) * grp / bm + r; }
// q as it was read -> the operand: zeros where there is no row or no column
__device__ __forceinline__ void prepare_q(const AttnArgs& a, bf16x8_t& q, bool there) {
  u32x4_t v = __builtin_bit_cast(u32x4_t, q);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = there ? (v[e] & a.q_and) ^ a.q_xor : 0u;
  q = __builtin_bit_cast(bf16x8_t, v);
  asm volatile("" : "+v"(q));
}

// What a workgroup works on: rows row0 .. of a stream's `rows`, keys k0 .. k1 - 1.
struct Work {
  int hk, sp, t0, n, row0, rows, kv, k0, k1;
  bool gap;                                                    // some table entry of the range names no page
  int entry;                                                   // this lane's entry of the range (its first 64)
  table_t tab;
  const bf16_t *kc, *vc;                                       // the kv head's columns of the caches
};
__device__ __forceinline__ int row_pos(const Work& w, int row, int grp) { return w.kv - w.n + row / grp; }
// (All 64 lanes probe at once, and the last probe brings the stream's numbers with it: what a workgroup waits for before its first copy is this, the page and no more.)
__device__ __forceinline__ bool find_work(const AttnArgs& a, int bm, int lane, Work& w) {
  w.hk = blockIdx.x % a.Hkv;
  w.sp = blockIdx.y;
  const int tile = (gridDim.x - 1 - blockIdx.x) / a.Hkv;       // (the last rows of a chunk see the most keys: first)
  int lo = 0, hi = a.R;
  while (hi - lo > 64) {
    const int step = (hi - lo + 63) / 64;
    const int p = lo + lane * step;
    const int c = __popcll(__ballot(p < hi && tile_base(a.cu, p < hi ? p : lo, a.T, a.grp, bm) <= tile));
    lo += (c > 0 ? c - 1 : 0) * step;
    hi = min(lo + step, hi);
  }
  const int p = min(lo + lane, a.R - 1);
  const int c0 = max(0, min(a.cu[p], a.T)), c1 = max(0, min(a.cu[p + 1], a.T)), len = a.kv_lens[p];
  const int base = c0 * a.grp / bm + p;
  const int hit = max(__popcll(__ballot(lo + lane < hi && base <= tile)) - 1, 0);
  const int r = __builtin_amdgcn_readfirstlane(lo + hit);
  w.t0 = __builtin_amdgcn_readlane(c0, hit);
  w.n = max(0, __builtin_amdgcn_readlane(c1, hit) - w.t0);
  w.row0 = (tile - __builtin_amdgcn_readlane(base, hit)) * bm;
  w.rows = w.n * a.grp;
  if (w.row0 < 0 || w.row0 >= w.rows) return false;
  w.kv = (int)min((long)max(__builtin_amdgcn_readlane(len, hit), 0), (long)a.width << a.shift);
  const int last = row_pos(w, min(w.row0 + bm, w.rows) - 1, a.grp);
  const long chunk = split_keys(w.kv, a.nsplit, a.cmin);
  w.k0 = (int)min((long)w.sp * chunk, (long)w.kv);
  w.k1 = (int)min((long)(w.sp + 1) * chunk, (long)(last + 1));
  if (w.k0 >= w.k1 && a.nsplit > 1) return false;              // (the join knows)
  w.tab = (table_t)(a.table + (size_t)r * a.ldt);
  w.kc = a.kc + (size_t)w.hk * a.hd;
  w.vc = a.vc + (size_t)w.hk * a.hd;
  w.gap = true;                                                // until find_gap, which nothing waits for before the first copies are out
  w.entry = w.tab[max(0, min((w.k0 >> a.shift) + lane, (w.k1 - 1) >> a.shift))];
  return true;
}
__device__ __forceinline__ void find_gap(const AttnArgs& a, int lane, Work& w) {
  bool gap = w.entry < 0 || w.entry >= a.npages;
  for (int e = (w.k0 >> a.shift) + 64 + lane; e <= (w.k1 - 1) >> a.shift; e += 64) { const int pg = w.tab[e]; gap |= pg < 0 || pg >= a.npages; }
  w.gap = __any(gap);
}

// Copies of K and V tiles of BN keys into LDS by NW waves, 1 KB an instruction.  A wave copies its share of the tile's rows, which lie in one page (two, where they
// are 16 and a page may hold 8): the pages' addresses are scalar, and what a lane adds to them does not change from tile to tile, so a copy is little more than its own
// instruction.  Rows behind the last key, rows of no page and columns behind the head's are asked for out of range and arrive as zeros: what is not
// finite in memory that holds no key never meets a probability of 0.
template <int HD, int BN, int NW, int (*SWZ)(int)>
struct Copier {
  static constexpr int ROWB = HD * 2, TILEB = BN * ROWB, NI = TILEB / 1024 / NW, RW = BN / NW, PG = RW > 8 ? 2 : 1, RP = RW / PG;      // rows of a wave, of a page's part
  static constexpr uint32_t NONE = 0xFFFFFFF0u;
  uint32_t off[NI];                                            // of the lane's 16 bytes from its part's first row
  int pg[PG];
  __device__ __forceinline__ void init(const AttnArgs& a, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int at = i * 1024 + lane * 16, row = at / ROWB, c = ((at % ROWB) >> 4) ^ SWZ(wave * RW + row);
      off[i] = c * 8 < a.hd ? (uint32_t)(((row % RP) * a.rowe + c * 8) * 2) : NONE;
    }
  }
  __device__ __forceinline__ void pages(const AttnArgs& a, const Work& w, int j0, int wave) {      // of the tile that is issued next
#pragma unroll
    for (int q = 0; q < PG; ++q) pg[q] = w.tab[max(0, min(j0 + wave * RW + q * RP, w.k1 - 1)) >> a.shift];
  }
  // K: to dst, V: to dst + TILEB; WHICH: 1 K, 2 V, 3 both
  template <int WHICH>
  __device__ __forceinline__ void issue(const AttnArgs& a, const Work& w, int j0, char* dst, int wave, int lane) {
    if (j0 + BN <= w.k1 && !w.gap) put<WHICH, true>(a, w, j0, dst, wave, lane);
    else put<WHICH, false>(a, w, j0, dst, wave, lane);
  }
  template <int WHICH, bool WHOLE>
  __device__ __forceinline__ void put(const AttnArgs& a, const Work& w, int j0, char* dst, int wave, int lane) {
#pragma unroll
    for (int q = 0; q < PG; ++q) {
      const int jb = j0 + wave * RW + q * RP;
      const size_t at = (((size_t)(uint32_t)pg[q] << a.shift) + (jb & ((1 << a.shift) - 1))) * a.rowe;
      const bool there = WHOLE || (pg[q] >= 0 && pg[q] < a.npages);
#pragma unroll
      for (int i = q * NI / PG; i < (q + 1) * NI / PG; ++i) {
        uint32_t v = off[i];
        if constexpr (!WHOLE) { if (jb + (i * 1024 + lane * 16) / ROWB % RP >= w.k1 || !there) v = NONE; }
        if constexpr (WHICH & 1) copy(w.kc + at, dst + wave * (TILEB / NW) + i * 1024, v);
        if constexpr (WHICH & 2) copy(w.vc + at, dst + TILEB + wave * (TILEB / NW) + i * 1024, v);
      }
    }
  }
  __device__ __forceinline__ static void copy(const bf16_t* base, char* lds, uint32_t voff) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7FFFFFF0u, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, AVT_LDS_PTR(lds), 16, voff, 0, 0, 0);
  }
};

// The 64 rows of Q of a workgroup, where the first two tiles of V will be (rows 0 .. 31 in the first one's place): whole rows, neighbouring lanes on neighbouring
// bytes (fetched as a product wants them, 64 lanes on 16 or more rows: 11 x 976 at 42, 8 / 2 heads x 512, 180 us, now 170).  Rows and columns that are not there are zeros.
template <int HD, int NW>
__device__ __forceinline__ void copy_q(const AttnArgs& a, const Work& w, char* smem, int wave, int lane) {
  constexpr int ROWB = HD * 2, TILEB = 32 * ROWB, RPI = 1024 / ROWB, NI = 64 / RPI / NW;      // rows of an instruction, instructions of a wave
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (wave * NI + i) * RPI, row = min(w.row0 + r, w.rows - 1), tok = row / a.grp, h = row - tok * a.grp;
    const bf16_t* base = a.q + (size_t)(w.t0 + tok) * a.ldq + (size_t)(w.hk * a.grp + h) * a.hd;
    const int sub = lane * 16 / ROWB, c = (lane * 16 % ROWB >> 4) ^ swz32<HD>((r + sub) & 31);
    const uint32_t next = (uint32_t)(h + 1 < a.grp ? a.hd : a.ldq - (long)(a.grp - 1) * a.hd);      // from a row to the one behind it
    Copier<HD, 32, NW, swz32<HD>>::copy(base, smem + (r < 32 ? TILEB : 3 * TILEB) + (r & 31) * ROWB,
                                        w.row0 + r + sub < w.rows && c * 8 < a.hd ? (sub * next + c * 8) * 2 : 0xFFFFFFF0u);
  }
}

// A V fragment of a tile that some row sees a part of: values that are not finite are taken out (their rows' probabilities may be 0) and told from `code`, which is
// 1 for a NaN, 2^8 for +inf and 2^16 for -inf: its product with the rows' visibility counts, exactly, what each row sees of them.
__device__ __forceinline__ bool not_finite(bf16x8_t f) {
  const u32x4_t w = __builtin_bit_cast(u32x4_t, f);
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
  return bad;
}
__device__ __forceinline__ void take_out(bf16x8_t& f, bf16x8_t& code) {
  u32x4_t w = __builtin_bit_cast(u32x4_t, f), k = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int sh = (e & 1) * 16;
    const uint32_t v = (w[e >> 1] >> sh) & 0xffffu;
    if ((v & 0x7f80u) == 0x7f80u) {
      w[e >> 1] &= ~(0xffffu << sh);
      k[e >> 1] |= ((v & 0x7fu) ? 0x3f80u : (v & 0x8000u) ? 0x4780u : 0x4380u) << sh;
    }
  }
  f = __builtin_bit_cast(bf16x8_t, w);
  code = __builtin_bit_cast(bf16x8_t, k);
}
__device__ __forceinline__ float put_back(float o, float count) {
  const int c = (int)count;
  if (c & 0xff) o += NAN;
  if (c & 0xff00) o += INFINITY;
  if (c >> 16) o -= INFINITY;
  return o;
}
__device__ __forceinline__ bf16x8_t seen8(uint32_t bits) {     // 8 bits -> 1.0 / 0.0
  u32x4_t w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = ((bits >> (2 * e)) & 1u ? 0x3f80u : 0u) | ((bits >> (2 * e + 1)) & 1u ? 0x3f800000u : 0u);
  return __builtin_bit_cast(bf16x8_t, w);
}
// Four columns of a row: the result, or this split's part of it
__device__ __forceinline__ void put_out(const AttnArgs& a, size_t t, int h, size_t rid, int col, f32x4_t v, float inv) {
  if (col >= a.hd) return;
  if (a.nsplit == 1) *(u32x2_t*)(a.out + t * a.ldo + (size_t)h * a.hd + col) = (u32x2_t){pack2bf(v[0] * inv, v[1] * inv), pack2bf(v[2] * inv, v[3] * inv)};
  else *(f32x4_t*)(a.part_o + rid * a.hd + col) = v;
}
__device__ __forceinline__ bool page_there(const AttnArgs& a, const Work& w, int j) {
  if (!w.gap || j >= w.k1) return true;
  const int e = w.tab[j >> a.shift];
  return e >= 0 && e < a.npages;
}

// ---- few rows: one workgroup (4 waves) per (kv head, tile of 16 rows, split of the keys) ------------------------------------------------------------------------
// K and V tiles of BN keys, two in turn.  S^T = K Q^T: wave w takes 16 keys (w % KT) of the tile and, where the tile has fewer than 64 keys, its share of the head's
// columns (w / KT); the scores pass through LDS (16 bytes per lane, the same lane reads them) and every wave then has all of them in the layout of P^T, the right
// operand of O^T = V^T P^T, and keeps the running maximum and sum (fp32) of every row for itself: no reduction between waves.  Wave w owns a quarter of the head's
// columns of O.  P is rounded to bf16 for the product (the matrix unit's type; half a step 2^-8 of each probability), the sum is of the unrounded ones.
//   Bound by the cache's bytes where there are many streams: 60 x 1 at 9000, 32 / 8 heads x 128, 265 us and 7 of the join, 4.9 TB/s, a large copy's rate; 64 x 1 at
// 1023, 4 heads x 512, 66 us and 4.  Of few short streams, by the chain cu, table, page, key, score, value: 5.6 us for 3 x 1 at 14.
template <int HD, int BN>
__global__ __launch_bounds__(256) void paged_attn_tile_kernel(AttnArgs a) {
  constexpr int ROWB = HD * 2, TILEB = BN * ROWB, KT = BN / 16, KS = 4 / KT, DS = HD / KS / 32, DT = HD / 64, TT = BN >= 32 ? BN / 32 : 1, BM = 16;
  static_assert(KT * KS == 4 && DS >= 1 && TILEB >= 4096, "tile shape");
  extern __shared__ __attribute__((aligned(1024))) char smem[];          // [2 tiles][K | V], scores
  f32x4_t* sx = (f32x4_t*)(smem + 4 * TILEB);                  // [4 waves][64 lanes]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g = lane >> 4;
  Work w;
  if (!find_work(a, BM, lane, w)) return;
  const int first = row_pos(w, w.row0, a.grp), last = row_pos(w, min(w.row0 + BM, w.rows) - 1, a.grp);
  const int row = w.row0 + c16, tok = row / a.grp;             // this lane's row (column of S^T)
  const bool ok = row < w.rows;
  const int pos = ok ? w.kv - w.n + tok : -1;
  bf16x8_t qf[DS];
  {
    const bf16_t* p = a.q + (size_t)(w.t0 + (ok ? tok : 0)) * a.ldq + (size_t)(w.hk * a.grp + (ok ? row - tok * a.grp : 0)) * a.hd;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = (wave / KT) * (HD / KS) + s * 32 + g * 8;
      qf[s] = *(const bf16x8_t*)(p + (d < a.hd ? d : 0));
    }
  }
  f32x4_t o[DT];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const int kswz = swz16<HD>(c16);
  const int krow = ((wave % KT) * 16 + c16) * ROWB, kc0 = (wave / KT) * (HD / KS / 8) + g;
  const int vr = 4 * g + (c16 >> 2);
  const uint32_t vaddr0 = lds_addr32(smem) + TILEB + vr * ROWB + (((wave * (HD / 32) + ((c16 & 3) >> 1)) ^ swz16<HD>(vr)) << 4) + (c16 & 1) * 8;

  Copier<HD, BN, 4, swz16<HD>> cp;
  cp.init(a, wave, lane);
  cp.pages(a, w, w.k0, wave);
  if (w.k0 < w.k1) cp.template issue<3>(a, w, w.k0, smem, wave, lane);
  cp.pages(a, w, w.k0 + BN, wave);
  // (Q is waited for here: left to the first product, the compiler's wait for it would sit inside the loop and wait for the copies in flight as well)
#pragma unroll
  for (int s = 0; s < DS; ++s) prepare_q(a, qf[s], ok && (wave / KT) * (HD / KS) + s * 32 + g * 8 < a.hd);
  find_gap(a, lane, w);
  int stage = 0;
  for (int j0 = w.k0; j0 < w.k1; j0 += BN, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");       // the tile is there, and every wave is done with the other one and with the scores
    if (j0 + BN < w.k1) { cp.template issue<3>(a, w, j0 + BN, smem + (stage ^ 1) * 2 * TILEB, wave, lane); cp.pages(a, w, j0 + 2 * BN, wave); }
    const char* kt = smem + stage * 2 * TILEB;
    f32x4_t s4 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DS; ++s) s4 = mfma16(*(const bf16x8_t*)(kt + krow + (((kc0 + 4 * s) ^ kswz) << 4)), qf[s], s4);
    sx[wave * 64 + lane] = s4;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    f32x4_t p[KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      p[k] = sx[k * 64 + lane];
#pragma unroll
      for (int q = 1; q < KS; ++q) p[k] += sx[(q * KT + k) * 64 + lane];
    }
    uint32_t seen = 0xffffffffu;                               // bit 4 k + e: key 16 k + 4 g + e
    if (w.gap || j0 + BN - 1 > first) {                        // some row does not see some key of this tile
      seen = 0;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const int j = j0 + k * 16 + g * 4;
        const bool there = page_there(a, w, j);                // (4 keys, one page)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool see = there && j + e <= pos && j + e < w.k1;
          p[k][e] = see ? p[k][e] : -INFINITY;
          seen |= (uint32_t)see << (k * 4 + e);
        }
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < KT; ++k) mx = fmaxf(mx, fmaxf(fmaxf(p[k][0], p[k][1]), fmaxf(p[k][2], p[k][3])));
    mx = gmax(mx) * a.scale_log2;
    const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(m - ms);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) { p[k][e] = __builtin_amdgcn_exp2f(fmaf(p[k][e], a.scale_log2, -ms)); sum += p[k][e]; }
    l = l * f + sum;
    if (__any(f != 1.f)) {
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    bf16x8_t pf[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      u32x4_t v = {pack2bf(p[2 * t][0], p[2 * t][1]), pack2bf(p[2 * t][2], p[2 * t][3]), 0u, 0u};
      if constexpr (KT > 1) { v[2] = pack2bf(p[2 * t + 1][0], p[2 * t + 1][1]); v[3] = pack2bf(p[2 * t + 1][2], p[2 * t + 1][3]); }
      pf[t] = __builtin_bit_cast(bf16x8_t, v);
    }
    const uint32_t va = vaddr0 + stage * 2 * TILEB;
    // (a tile of which one row sees a key that another one does not: a value that is not finite must not reach the latter through its probability of 0)
    const bool uneven = first < last && j0 + BN - 1 > first;
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
          if (uneven && __any(not_finite(vf[d][t]))) {
            bf16x8_t code;
            take_out(vf[d][t], code);
            const f32x4_t c = mfma16(code, seen8(KT > 1 ? seen >> (8 * t) : seen & 0xfu), (f32x4_t){0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d0 + d][e] = put_back(o[d0 + d][e], c[e]);
          }
          o[d0 + d] = mfma16(vf[d][t], pf[t], o[d0 + d]);
        }
    }
  }
  l = gsum(l);
  if (!ok) return;
  const int h = w.hk * a.grp + row - tok * a.grp;
  const size_t t = w.t0 + tok, rid = ((size_t)w.sp * a.T + t) * a.H + h;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int d = 0; d < DT; ++d) put_out(a, t, h, rid, wave * (HD / 4) + d * 16 + g * 4, o[d], inv);
  if (a.nsplit > 1 && wave == 0 && g == 0) { a.part_ml[rid * 2] = m; a.part_ml[rid * 2 + 1] = l; }
}

// ---- many rows: one workgroup (4 waves, 128 rows) per (kv head, tile of rows, split of the keys), heads of up to 128 columns -----------------------------------
// Every wave has 32 rows of its own and goes through all keys of a tile with 32 x 32 x 16 products: S^T = K Q^T (a lane has one row and 16 of every 32 keys, so a
// row's maximum and sum are 31 operations and one exchange of the wave's halves), P^T is already the right operand of O^T = V^T P^T.  No wave waits for another but
// for the tile.  The running maximum follows only when a score passes it by more than 2^8: the probabilities then stay below 2^8, where bf16 and the fp32
// sums are as exact as below 1, and the accumulators are rarely rescaled.
//   Two workgroups share a CU, two waves a SIMD, of which one's softmax is to run beside the other's products: chunks of 4099 at 4200, 16 / 4 heads x 128, take
// 362 us among other launches, 372 alone in a graph, 384 under the profiler, 0.83 to 0.88 PFLOP/s, the matrix unit busy 0.46 of its cycles there.  What that cost to reach: half of the score operands read ahead of their products, the products' waves given precedence and V's next
// fragments read ahead (437 -> 414 us); a copy of a whole tile in a path of its own, so that it is eight instructions and their addresses (404 -> 374); a row's
// visible keys in bits of a register, not in 64 scalar registers that pushed the loop's own ones out (4 x 1000 at 1000, 12 heads x 64: 59 -> 54).
template <int HD>
__global__ __launch_bounds__(256, 2) void paged_attn_long_kernel(AttnArgs a) {
  constexpr int BN = 64, BM = 128, ROWB = HD * 2, TILEB = BN * ROWB, DS = HD / 16, DT = HD / 32;
  extern __shared__ __attribute__((aligned(1024))) char smem[];          // [2 tiles][K | V]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, half = lane >> 5;
  Work w;
  if (!find_work(a, BM, lane, w)) return;
  const int wrow = w.row0 + wave * 32, row = wrow + c32, tok = row / a.grp;
  const bool mine = wrow < w.rows, ok = row < w.rows;
  const int pos = ok ? w.kv - w.n + tok : -1;
  const int first = row_pos(w, wrow, a.grp), last = mine ? row_pos(w, min(wrow + 32, w.rows) - 1, a.grp) : -1;      // of this wave's rows
  bf16x8_t qf[DS];
  {
    const bf16_t* p = a.q + (size_t)(w.t0 + (ok ? tok : 0)) * a.ldq + (size_t)(w.hk * a.grp + (ok ? row - tok * a.grp : 0)) * a.hd;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      const int d = s * 16 + half * 8;
      qf[s] = *(const bf16x8_t*)(p + (d < a.hd ? d : 0));
    }
  }
  f32x16_t o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -INFINITY, l = 0.f;                                // m: in units of the scaled scores, what the probabilities are relative to
  const int krow = c32 * ROWB, kswz = swz32<HD>(c32);
  const int vr = 4 * half + ((lane & 15) >> 2);                // row and columns of a lane in a transposing read: 4 rows x 16 columns per 16 lanes
  const int vc = (lane & 16) + (lane & 3) * 4;
  const uint32_t vaddr0 = lds_addr32(smem) + TILEB + vr * ROWB + (((vc >> 3) ^ swz32<HD>(vr)) << 4) + (vc & 7) * 2;

  Copier<HD, BN, 4, swz32<HD>> cp;
  cp.init(a, wave, lane);
  cp.pages(a, w, w.k0, wave);
  if (w.k0 < w.k1) cp.template issue<3>(a, w, w.k0, smem, wave, lane);
  cp.pages(a, w, w.k0 + BN, wave);
#pragma unroll
  for (int s = 0; s < DS; ++s) prepare_q(a, qf[s], ok && s * 16 + half * 8 < a.hd);
  find_gap(a, lane, w);
  int stage = 0;
  for (int j0 = w.k0; j0 < w.k1; j0 += BN, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");       // the tile is there, and every wave is done with the other one
    if (j0 + BN < w.k1) { cp.template issue<3>(a, w, j0 + BN, smem + (stage ^ 1) * 2 * TILEB, wave, lane); cp.pages(a, w, j0 + 2 * BN, wave); }
    if (j0 > last) continue;                                   // none of this wave's rows sees the tile
    const char* kt = smem + stage * 2 * TILEB;
    f32x16_t s[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) s[0][e] = s[1][e] = 0.f;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int q0 = 0; q0 < DS; q0 += 4) {
      bf16x8_t kf[4][2];
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int k = 0; k < 2; ++k) kf[q][k] = *(const bf16x8_t*)(kt + k * 32 * ROWB + krow + (((2 * (q0 + q) + half) ^ kswz) << 4));
      __builtin_amdgcn_sched_barrier(0);                       // (left alone, the compiler reads two fragments ahead of the products and waits for each)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int k = 0; k < 2; ++k) s[k] = mfma32(kf[q][k], qf[q0 + q], s[k]);
    }
    __builtin_amdgcn_s_setprio(0);
    uint32_t seen = 0xffffffffu;                               // bit 16 k + e: key 32 k + 8 (e / 4) + 4 half + e % 4
    if (w.gap || j0 + BN - 1 > first) {
      const int lim = min(pos, w.k1 - 1);
      seen = 0;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int j = j0 + k * 32 + e4 * 8 + half * 4;
          const bool there = page_there(a, w, j);
#pragma unroll
          for (int e = 0; e < 4; ++e) seen |= (uint32_t)(there && j + e <= lim) << (k * 16 + e4 * 4 + e);
          asm volatile("" : "+v"(seen));
#pragma unroll
          for (int e = 0; e < 4; ++e) s[k][e4 * 4 + e] = (seen >> (k * 16 + e4 * 4 + e)) & 1u ? s[k][e4 * 4 + e] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[k][e]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2;
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(m - ms);
      m = mn;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    bf16x8_t pf[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int e = 0; e < 16; ++e) { s[k][e] = __builtin_amdgcn_exp2f(fmaf(s[k][e], a.scale_log2, -ms)); l += s[k][e]; }
#pragma unroll
      for (int t = 0; t < 2; ++t)
        pf[2 * k + t] = __builtin_bit_cast(bf16x8_t, (u32x4_t){pack2bf(s[k][8 * t], s[k][8 * t + 1]), pack2bf(s[k][8 * t + 2], s[k][8 * t + 3]),
                                                               pack2bf(s[k][8 * t + 4], s[k][8 * t + 5]), pack2bf(s[k][8 * t + 6], s[k][8 * t + 7])});
    }
    __builtin_amdgcn_s_setprio(1);
    const uint32_t va = vaddr0 + stage * 2 * TILEB, vb = va ^ 32;       // rows + 8: the swizzle differs by two pieces
    // (a tile that holds a key which some row of this wave does not see -- the wave's rows may be one token's, the tile's keys reach the workgroup's last one: a value
    // that is not finite must not reach that row through its probability of 0)
    const bool uneven = min(j0 + BN, w.k1) - 1 > first;
    bf16x8_t vbuf[2][4];                                       // (the fragments of the next columns are read while these are multiplied)
    const auto read_v = [&](int d) {
      const uint32_t x = va ^ (d * 64), y = vb ^ (d * 64);
      bf16x8_t* v = vbuf[d & 1];
      v[0] = tr_join(ds_read_tr_na<0>(x), ds_read_tr_na<8 * ROWB>(y));
      v[1] = tr_join(ds_read_tr_na<16 * ROWB>(x), ds_read_tr_na<24 * ROWB>(y));
      v[2] = tr_join(ds_read_tr_na<32 * ROWB>(x), ds_read_tr_na<40 * ROWB>(y));
      v[3] = tr_join(ds_read_tr_na<48 * ROWB>(x), ds_read_tr_na<56 * ROWB>(y));
    };
    read_v(0);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      bf16x8_t* vf = vbuf[d & 1];
      if (d + 1 < DT) {
        read_v(d + 1);
        asm volatile("s_waitcnt lgkmcnt(8)" : "+v"(vf[0]), "+v"(vf[1]), "+v"(vf[2]), "+v"(vf[3])::"memory");
      } else {
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(vf[0]), "+v"(vf[1]), "+v"(vf[2]), "+v"(vf[3])::"memory");
      }
      if (uneven) {
        if (__any(not_finite(vf[0]) || not_finite(vf[1]) || not_finite(vf[2]) || not_finite(vf[3]))) {
          f32x16_t c;
#pragma unroll
          for (int e = 0; e < 16; ++e) c[e] = 0.f;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            bf16x8_t code;
            take_out(vf[t], code);
            c = mfma32(code, seen8(seen >> (8 * t)), c);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] = put_back(o[d][e], c[e]);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) o[d] = mfma32(vf[t], pf[t], o[d]);
    }
    __builtin_amdgcn_s_setprio(0);
  }
  l += __shfl_xor(l, 32, 64);
  if (!ok) return;
  const int h = w.hk * a.grp + row - tok * a.grp;
  const size_t t = w.t0 + tok, rid = ((size_t)w.sp * a.T + t) * a.H + h;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) put_out(a, t, h, rid, d * 32 + e * 8 + half * 4, (f32x4_t){o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]}, inv);
  if (a.nsplit > 1 && half == 0) { a.part_ml[rid * 2] = m; a.part_ml[rid * 2 + 1] = l; }
}

// ---- many rows of wide heads (256, 512 columns): one workgroup (NW = 4 or 8 waves, 64 rows) per (kv head, tile of rows, split of the keys) --------------------
// 32 rows of O do not fit one wave's registers, so S^T and O^T are shared out in different ways.  Of S^T = K Q^T (32 keys) a wave has blocks of 16 keys x 16 rows,
// over all of the head's columns (16 x 16 x 32 products: no partial sums to add), which pass through LDS; of O^T it has a quarter of the columns, for all 64 rows
// (4 waves, 256 columns: two workgroups on a CU) or for 32 (8 waves, 512 columns: the LDS holds one).  Either way 2 waves share a SIMD and no accumulator leaves
// the 256 registers that the vector unit reaches (with 4 waves for 512 columns the compiler kept O in the others and moved it to and fro: 8 us a tile).
// The scores of tile i + 1 are made between the same two barriers as the softmax and the products with V of tile i, so that neither unit waits for the other.
// Maximum and sum of a row are kept by every wave that has a part of it, as in the kernel for few rows, and follow as in the one for many.
//   16 chunks of up to 192 at up to 800, 4 heads x 512, take 66 us, 175 TFLOP/s: the longest workgroup has 31 tiles of 2.1 us, where an even share would be 13.3 a CU (180
// workgroups on 256 CUs, of 9 to 31 tiles; 16 chunks that all are the longest take the same, 69 us).  11 x 976 at 42, 8 / 2 heads x 512, are even, 52 tiles a CU, and take 157 us and
// not 110: with one workgroup on a CU nothing runs beside finding the work, fetching Q and the first tiles, and the stores.  Inside a tile it is a wave's own chain, 430
// instructions and four trips to LDS, of which the other wave of its SIMD hides a part: the copies alone take 44 us, the products 10 % of the matrix unit's cycles.
template <int HD, int NW>
__global__ __launch_bounds__(NW * 64, 2) void paged_attn_wide_kernel(AttnArgs a) {
  constexpr int BN = 32, BM = 64, ROWB = HD * 2, TILEB = BN * ROWB, DS = HD / 32, KB = 8 / NW, DT = HD / 128, NB = 8 / NW;      // KB: key blocks of a wave's S, NB: row blocks of its O
  extern __shared__ __attribute__((aligned(1024))) char smem[];          // [2 tiles][K | V], scores of two tiles
  f32x4_t* sx = (f32x4_t*)(smem + 4 * TILEB);                  // [2][2 key blocks][4 row blocks][64 lanes]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g16 = lane >> 4, c32 = lane & 31, half = lane >> 5;
  const int slice = NB == 2 ? wave : wave >> 1, b0 = NB == 2 ? 0 : wave & 1;      // of O: quarter of the columns, first row block
  const int rb = wave & 3, kb0 = KB == 2 ? 0 : wave >> 2;      // of S: row block, first key block
  Work w;
  if (!find_work(a, BM, lane, w)) return;
  const int first = row_pos(w, w.row0, a.grp), last = row_pos(w, min(w.row0 + BM, w.rows) - 1, a.grp);
  int pos[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) { const int row = w.row0 + (b0 + b) * 32 + c32; pos[b] = row < w.rows ? row_pos(w, row, a.grp) : -1; }
  bf16x8_t qf[DS];
  f32x16_t o[NB][DT];
  float m[NB], l[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    m[b] = -INFINITY; l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][d][e] = 0.f;
  }
  const int krow = c16 * ROWB;
  const int vr = 4 * half + ((lane & 15) >> 2), vc = (lane & 16) + (lane & 3) * 4;
  const uint32_t vaddr0 = lds_addr32(smem) + TILEB + vr * ROWB + (((slice * (HD / 32) + (vc >> 3)) ^ swz32<HD>(vr)) << 4) + (vc & 7) * 2;

  const auto scores = [&](const char* kt, int which) {         // of the tile in kt, to sx
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      f32x4_t s = {0.f, 0.f, 0.f, 0.f}, s1 = s;                // (two chains: a product that waits for the one before it would idle the unit half of the time)
      const char* kr = kt + (kb0 + k) * 16 * ROWB + krow;
      const int kswz = swz32<HD>((kb0 + k) * 16 + c16);
#pragma unroll
      for (int q0 = 0; q0 < DS; q0 += 8) {
        bf16x8_t kf[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) kf[q] = *(const bf16x8_t*)(kr + (((g16 * (HD / 32) + q0 + q) ^ kswz) << 4));
        __builtin_amdgcn_sched_barrier(0);                     // (left alone, the compiler reads two fragments ahead of the products and waits for each)
#pragma unroll
        for (int q = 0; q < 8; q += 2) {
          s = mfma16(kf[q], qf[q0 + q], s);
          s1 = mfma16(kf[q + 1], qf[q0 + q + 1], s1);
        }
      }
      sx[((which * 2 + kb0 + k) * 4 + rb) * 64 + lane] = s + s1;
    }
  };
  // K of tile i + 2 and V of tile i + 1 are asked for while tile i is worked on.
  using Copy = Copier<HD, BN, NW, swz32<HD>>;
  Copy ck, cv;
  ck.init(a, wave, lane);
#pragma unroll
  for (int i = 0; i < Copy::NI; ++i) cv.off[i] = ck.off[i];
  if (w.k0 < w.k1) {
    ck.pages(a, w, w.k0, wave);
    cv.pages(a, w, w.k0 + BN, wave);
    ck.template issue<1>(a, w, w.k0, smem, wave, lane);
    if (w.k0 + BN < w.k1) cv.template issue<1>(a, w, w.k0 + BN, smem + 2 * TILEB, wave, lane);
    copy_q<HD, NW>(a, w, smem, wave, lane);
  }
  find_gap(a, lane, w);
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");       // Q and both tiles of K
  {
    const char* qr = smem + (rb < 2 ? TILEB : 3 * TILEB) + ((rb & 1) * 16 + c16) * ROWB;
    const int qswz = swz32<HD>((rb & 1) * 16 + c16);
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      qf[s] = *(const bf16x8_t*)(qr + (((g16 * (HD / 32) + s) ^ qswz) << 4));
      prepare_q(a, qf[s], true);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // every wave has its part of Q: V may take its place
  if (w.k0 < w.k1) {
    ck.template issue<2>(a, w, w.k0, smem, wave, lane);
    ck.pages(a, w, w.k0 + 2 * BN, wave);
    scores(smem, 0);
  }
  int stage = 0;
  for (int j0 = w.k0; j0 < w.k1; j0 += BN, stage ^= 1) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // the scores and V of this tile and K of the next are there, every wave is done with the tile before
    if (j0 + BN < w.k1) cv.template issue<2>(a, w, j0 + BN, smem + (stage ^ 1) * 2 * TILEB, wave, lane);
    if (j0 + 2 * BN < w.k1) ck.template issue<1>(a, w, j0 + 2 * BN, smem + stage * 2 * TILEB, wave, lane);
#pragma unroll
    for (int q = 0; q < Copy::PG; ++q) cv.pg[q] = ck.pg[q];
    ck.pages(a, w, j0 + 3 * BN, wave);
    if (j0 + BN < w.k1) scores(smem + (stage ^ 1) * 2 * TILEB, stage ^ 1);
    const bool hide = w.gap || j0 + BN - 1 > first, uneven = first < last && j0 + BN - 1 > first;
    uint32_t seen[NB];                                         // bit e: key 8 (e / 4) + 4 half + e % 4
    bf16x8_t pf[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      f32x4_t p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = sx[((stage * 2 + (e >> 1)) * 4 + (b0 + b) * 2 + (c32 >> 4)) * 64 + ((e & 1) * 2 + half) * 16 + c16];
      seen[b] = 0xffffu;
      if (hide) {
        const int lim = min(pos[b], w.k1 - 1);
        seen[b] = 0;
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int j = j0 + e4 * 8 + half * 4;
          const bool there = page_there(a, w, j);
#pragma unroll
          for (int e = 0; e < 4; ++e) seen[b] |= (uint32_t)(there && j + e <= lim) << (e4 * 4 + e);
          asm volatile("" : "+v"(seen[b]));
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e4][e] = (seen[b] >> (e4 * 4 + e)) & 1u ? p[e4][e] : -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fmaxf(p[e][0], p[e][1]), fmaxf(p[e][2], p[e][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2;
      if (__any(mx > m[b] + 8.f)) {
        const float mn = fmaxf(m[b], mx), ms = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(m[b] - ms);
        m[b] = mn;
        l[b] *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[b][d] *= f;
      }
      const float ms = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4)
#pragma unroll
        for (int e = 0; e < 4; ++e) { p[e4][e] = __builtin_amdgcn_exp2f(fmaf(p[e4][e], a.scale_log2, -ms)); l[b] += p[e4][e]; }
#pragma unroll
      for (int t = 0; t < 2; ++t)
        pf[b][t] = __builtin_bit_cast(bf16x8_t, (u32x4_t){pack2bf(p[2 * t][0], p[2 * t][1]), pack2bf(p[2 * t][2], p[2 * t][3]), pack2bf(p[2 * t + 1][0], p[2 * t + 1][1]),
                                                          pack2bf(p[2 * t + 1][2], p[2 * t + 1][3])});
    }
    const uint32_t va = vaddr0 + stage * 2 * TILEB, vb = va ^ 32;       // rows + 8: the swizzle differs by two pieces
    constexpr int G = NB == 2 ? 1 : 2;                         // column blocks whose fragments are read at once
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += G) {
      bf16x8_t vf[G][2];
#pragma unroll
      for (int d = 0; d < G; ++d) {
        const uint32_t x = va ^ ((d0 + d) * 64), y = vb ^ ((d0 + d) * 64);
        vf[d][0] = tr_join(ds_read_tr_na<0>(x), ds_read_tr_na<8 * ROWB>(y));
        vf[d][1] = tr_join(ds_read_tr_na<16 * ROWB>(x), ds_read_tr_na<24 * ROWB>(y));
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int d = 0; d < G; ++d) {
        asm volatile("" : "+v"(vf[d][0]), "+v"(vf[d][1]));
        if (uneven && __any(not_finite(vf[d][0]) || not_finite(vf[d][1]))) {
          bf16x8_t code[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) take_out(vf[d][t], code[t]);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            f32x16_t c;
#pragma unroll
            for (int e = 0; e < 16; ++e) c[e] = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t) c = mfma32(code[t], seen8(seen[b] >> (8 * t)), c);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b][d0 + d][e] = put_back(o[b][d0 + d][e], c[e]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int d = 0; d < G; ++d)
#pragma unroll
          for (int b = 0; b < NB; ++b) o[b][d0 + d] = mfma32(vf[d][t], pf[b][t], o[b][d0 + d]);
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float lt = l[b] + __shfl_xor(l[b], 32, 64), inv = lt == 0.f ? 0.f : 1.f / lt;
    const int row = w.row0 + (b0 + b) * 32 + c32, tok = row / a.grp;
    if (row >= w.rows) continue;
    const int h = w.hk * a.grp + row - tok * a.grp;
    const size_t t = w.t0 + tok, rid = ((size_t)w.sp * a.T + t) * a.H + h;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        put_out(a, t, h, rid, slice * (HD / 4) + d * 32 + e * 8 + half * 4, (f32x4_t){o[b][d][4 * e], o[b][d][4 * e + 1], o[b][d][4 * e + 2], o[b][d][4 * e + 3]}, inv);
    if (a.nsplit > 1 && slice == 0 && half == 0) { a.part_ml[rid * 2] = m[b]; a.part_ml[rid * 2 + 1] = lt; }
  }
}

// The partial results of the splits that a row's keys reach, joined in the splits' order with weights 2^(m_z - max m) in fp32.  A weight of 0 does not take a split out:
// the maximum of a split whose scores are all NaN is -inf (a maximum passes over NaN), and 0 NaN is the NaN that the row has without splits.
// What both kernels need of a row: how many splits its keys reach.
__device__ __forceinline__ int splits_of(const AttnArgs& a, int t, int lane) {
  const int r = __builtin_amdgcn_readfirstlane(find_stream(a.cu, a.R, t, lane));
  if (r < 0) return -1;
  const int t0 = max(0, min(a.cu[r], a.T)), n = max(0, min(a.cu[r + 1], a.T) - t0);
  const int kv = (int)min((long)max(a.kv_lens[r], 0), (long)a.width << a.shift);
  const int pos = kv - n + (t - t0);
  return pos < 0 ? 0 : (int)(pos / split_keys(kv, a.nsplit, a.cmin)) + 1;
}
// Few splits (up to FEW_SPLITS; many rows): a thread takes four columns of a row through all of them.  Bound by the partial results' bytes, 8 a column, row and split:
// 8 x 300 at 2000, 8 heads x 256 in two, 10.4 us; 4 us at the least, a launch and two dependent loads.
__global__ __launch_bounds__(256) void paged_attn_join_few_kernel(AttnArgs a) {
  const int t = blockIdx.x, nz = splits_of(a, t, threadIdx.x & 63);
  const int idx = blockIdx.y * 256 + threadIdx.x;
  if (nz < 0 || idx >= a.H * a.hd / 4) return;
  const int h = idx * 4 / a.hd;
  const size_t step = (size_t)a.T * a.H, rid = (size_t)t * a.H + h;
  float mx = -INFINITY;
  for (int z = 0; z < nz; ++z) mx = fmaxf(mx, a.part_ml[(rid + z * step) * 2]);
  if (mx == -INFINITY) mx = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int z = 0; z < nz; ++z) {
    const float f = __builtin_amdgcn_exp2f(a.part_ml[(rid + z * step) * 2] - mx), lz = a.part_ml[(rid + z * step) * 2 + 1];
    const f32x4_t p = *(const f32x4_t*)(a.part_o + (rid + z * step) * a.hd + (idx * 4 - h * a.hd));
    o += p * f;
    l += lz * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *(u32x2_t*)(a.out + (size_t)t * a.ldo + idx * 4) = (u32x2_t){pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv)};
}
// Many splits (few rows): a workgroup per row, the splits taken by hd / 4 lanes each, as many at once as fit.
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
  __shared__ float wt[MAX_SPLITS];
  __shared__ f32x4_t sum[256];
  const int t = blockIdx.x / a.H, h = blockIdx.x % a.H, tid = threadIdx.x, lane = tid & 63;
  const int nz = splits_of(a, t, lane);
  if (nz < 0) return;
  const size_t step = (size_t)a.T * a.H, rid = (size_t)t * a.H + h;
  float mx = -INFINITY, l = 0.f;
  for (int z = lane; z < nz; z += 64) mx = fmaxf(mx, a.part_ml[(rid + z * step) * 2]);      // (every wave for itself)
  mx = wave_max(mx);
  if (mx == -INFINITY) mx = 0.f;
  for (int z = lane; z < nz; z += 64) {
    const float f = __builtin_amdgcn_exp2f(a.part_ml[(rid + z * step) * 2] - mx);
    l += f * a.part_ml[(rid + z * step) * 2 + 1];
    if (tid < 64) wt[z] = f;
  }
  l = wave_sum(l);
  __syncthreads();
  const int d4 = a.hd / 4, groups = 256 / d4, grp = tid / d4, c = tid - grp * d4;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  if (grp < groups)
    for (int z = grp; z < nz; z += groups) {
      const float f = wt[z];
      o += *(const f32x4_t*)(a.part_o + (rid + z * step) * a.hd + c * 4) * f;
    }
  sum[tid] = o;
  __syncthreads();
  if (tid >= d4) return;
  for (int i = 1; i < groups; ++i) o += sum[i * d4 + tid];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *(u32x2_t*)(a.out + (size_t)t * a.ldo + (size_t)h * a.hd + c * 4) = (u32x2_t){pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv)};
}

// ---- choices on the host, from sizes alone -----------------------------------------------------------------------------------------------------------
struct Choice { int hd, bm, nsplit, cmin; long tiles; };

Choice choose(int T, int R, int H, int Hkv, int hd, long max_new, long max_kv, int cu_count) {
  Choice c;
  c.hd = hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : hd <= 512 ? 512 : 1024;
  const int grp = H / Hkv;
  const long rows = (max_new > 0 && max_new < T ? max_new : (T + R - 1) / R) * grp;      // rows of a stream and kv head
  c.bm = rows <= 16 || c.hd == 1024 ? 16 : c.hd <= 128 ? 128 : 64;
  c.tiles = (long)T * grp / c.bm + R;
  c.cmin = c.bm == 16 ? 64 : 256;
  const long items = c.tiles * Hkv;
  // Enough workgroups for two on every CU (one and a half, where 128 rows each make a split's partial results dear), down to 64 keys each of few rows (a tile of 16
  // to 64 keys is 0.9 us of latency, a join 4: 1 x 730, 8 heads x 128, 14 us in splits of 256 keys, 9.4 in splits of 64), 256 of 128 rows and 512 of 64 rows of a
  // wide head (4 heads x 512, 16 chunks of 192 at 800: 67 us whole, 80 in splits of 256 keys, 95 against 69 where all are the longest; 20 x 20 at 3000: 91 in splits of 512,
  // 101 of 256, 176 whole; 8 heads x 256, 8 x 300 at 2000: 111, 112, 125).  With many rows, only to have one on every CU, down to 128 keys (3 x 680 at 1168, one
  // head x 128: 24 us in 8, 21 in 15; 32 x 40 at 500, 8 / 2 heads x 128, which has enough: 21 us in splits of 256 keys, 25 in splits of 128; 4 x 200 at 600, 8 heads x 512:
  // 43, 54 without).
  // And where rows are few and keys many, four times that, so that streams of different lengths even out, but no fewer than 1024 keys each (with many rows the
  // partial results and the join are as much as the keys: 403 against 440 us without it, chunks of 4099 at 4200).
  const long want = c.bm == 128 ? 3l * cu_count / 2 : 2l * cu_count;
  // No splits below 192 keys.  One new token each, in a graph, whole and in splits of 64: 12 heads x 64, 3 x 1 at 150 7.0 and 9.0 us; 8 / 2 heads x 128, 16 x 1 at 150 8.3 and
  // 9.5, 1 x 1 at 190 9.0 and 8.7.  The rule is that of tiles of 32 and 64 keys; heads whose tiles are 16 keys pay for it where streams are few: 4 heads x 256, 3 x 1 at 150 13.5
  // and 11.6 us, 64 x 1 at 150 15.5 and 17.2; 4 heads x 512, 3 x 1 at 100 14.0 and 12.9, at 190 20.5 and 13.8, 64 x 1 at 190 25.0 and 25.4; 2 heads x 1024, 3 x 1 at 190 29.4 and 18.0.
  const bool few = max_kv < 192;
  const long most = few ? 1 : c.bm == 64 ? max_kv / 512 : (max_kv + c.cmin - 1) / c.cmin, one = few ? 1 : std::min(cu_count / items, (max_kv + 127) / 128);
  long fill = std::min((want + items - 1) / items, most);
  if (c.bm > 16 && one > fill) { fill = one; c.cmin = 128; }
  const long even = c.bm == 16 ? std::min((8l * cu_count + items - 1) / items, max_kv / 1024) : 0;
  c.nsplit = (int)std::max(1l, std::min(std::max(fill, even), (long)MAX_SPLITS));
  return c;
}

long part_floats(const Choice& c, long T, long H, long hd) { return c.nsplit > 1 ? c.nsplit * T * H * (hd + 2) : 0; }

template <class F>
int launch(F* kernel, int threads, int lds, const AttnArgs& a, const Choice& c, hipStream_t st) {
  if (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    AVT_CHECK(e == hipSuccess, "avt_paged_attn_fwd: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)(c.tiles * a.Hkv), c.nsplit), dim3(threads), lds, st, a);
  return 0;
}
template <int HD, int BN>
int launch_tiles(const AttnArgs& a, const Choice& c, hipStream_t st) { return launch(paged_attn_tile_kernel<HD, BN>, 256, 4 * BN * HD * 2 + 4096, a, c, st); }
template <int HD>
int launch_long(const AttnArgs& a, const Choice& c, hipStream_t st) { return launch(paged_attn_long_kernel<HD>, 256, 4 * 64 * HD * 2, a, c, st); }
template <int HD, int NW>
int launch_wide(const AttnArgs& a, const Choice& c, hipStream_t st) { return launch(paged_attn_wide_kernel<HD, NW>, NW * 64, 4 * 32 * HD * 2 + 2 * 8192, a, c, st); }
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
  AVT_CHECK(npages >= 0 && width >= 1 && ldt >= width && (long)width * page < 0x7fff0000l, "avt_paged_attn_fwd: bad table (width %d, ldt %d, page %d)", width, ldt, page);
  AVT_CHECK(npages <= (1l << 31) / page, "avt_paged_attn_fwd: a cache may hold 2^31 rows, as many as slots name (%ld pages of %d)", npages, page);
  if (T == 0) return 0;
  AVT_CHECK(q && kcache && vcache && table && cu && kv_lens && out, "avt_paged_attn_fwd: null argument");
  AVT_CHECK(ldq >= (long)H * head_dim && ldo >= (long)H * head_dim && ldq % 8 == 0 && ldo % 8 == 0 && aligned16(q) && aligned16(kcache) && aligned16(vcache) && aligned16(out),
            "avt_paged_attn_fwd: 16-byte aligned rows required");
  AVT_CHECK((long)Hkv * head_dim < (1l << 26), "avt_paged_attn_fwd: a token's row is too long (%d heads of %d)", Hkv, head_dim);
  AVT_CHECK(ldq < (1l << 29), "avt_paged_attn_fwd: rows of q are too far apart (%ld)", ldq);
  AVT_CHECK((long)T * H < 0x7f000000l, "avt_paged_attn_fwd: too many rows for one call (%d tokens of %d heads)", T, H);
  const Choice c = choose(T, R, H, Hkv, head_dim, max_new, max_kv > 0 ? max_kv : 0x7fffffff, CUS);
  AVT_CHECK(c.tiles * Hkv < 0x7f000000l, "avt_paged_attn_fwd: too many rows for one call (%d tokens of %d streams)", T, R);
  const long pf = part_floats(c, T, H, head_dim);
  AVT_CHECK(pf == 0 || (ws && aligned16(ws) && ws_bytes >= 4 * (size_t)pf), "avt_paged_attn_fwd: workspace of %ld bytes needed", 4 * pf);
  AttnArgs a;
  a.q = (const bf16_t*)q; a.kc = (const bf16_t*)kcache; a.vc = (const bf16_t*)vcache; a.table = table; a.cu = cu; a.kv_lens = kv_lens; a.out = (bf16_t*)out;
  a.part_o = (float*)ws; a.part_ml = (float*)ws + (size_t)c.nsplit * T * H * head_dim;
  a.ldq = ldq; a.ldo = ldo; a.npages = npages; a.shift = __builtin_ctz(page); a.ldt = ldt; a.width = width; a.T = T; a.R = R; a.H = H; a.Hkv = Hkv; a.grp = H / Hkv;
  a.hd = head_dim; a.nsplit = c.nsplit; a.cmin = c.cmin; a.scale_log2 = scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f;
  a.rowe = (uint32_t)Hkv * head_dim;
  a.q_and = scale == 0.f ? 0u : 0xffffffffu; a.q_xor = scale < 0.f ? 0x80008000u : 0u;
  hipStream_t st = (hipStream_t)stream;
  int rc = 0;
  if (c.bm == 16) rc = c.hd == 64 ? launch_tiles<64, 64>(a, c, st) : c.hd == 128 ? launch_tiles<128, 32>(a, c, st) : c.hd == 256 ? launch_tiles<256, 16>(a, c, st)
                     : c.hd == 512 ? launch_tiles<512, 16>(a, c, st) : launch_tiles<1024, 16>(a, c, st);
  else rc = c.hd == 64 ? launch_long<64>(a, c, st) : c.hd == 128 ? launch_long<128>(a, c, st) : c.hd == 256 ? launch_wide<256, 4>(a, c, st) : launch_wide<512, 8>(a, c, st);
  if (rc) return rc;
  AVT_LAUNCH_CHECK();
  if (c.nsplit > 1) {
    if (c.nsplit <= FEW_SPLITS) hipLaunchKernelGGL(paged_attn_join_few_kernel, dim3(T, (H * head_dim / 4 + 255) / 256), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(paged_attn_join_kernel, dim3(T * H), dim3(256), 0, st, a);
    AVT_LAUNCH_CHECK();
  }
  return 0;
}
