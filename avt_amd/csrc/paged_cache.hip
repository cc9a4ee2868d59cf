// The pages of a key / value cache that many streams of different lengths share: tables and slots from the lengths, and the rows that go into them.
//   avt_paged_plan      block tables, slots, positions and offsets of a step's new tokens, from the streams' lengths, on the device
//   avt_paged_kv_write  the new tokens' keys and values into their slots
#include "common.hpp"
#include "../../include/avt_hip.h"

namespace {
constexpr int PLAN_RMAX = 4096;       // streams: four LDS words each
constexpr int PLAN_NT = 1024;
constexpr int PLAN_PER = PLAN_RMAX / PLAN_NT;

// inclusive sum over the workgroup's PLAN_NT threads (16 waves): shuffles inside a wave, the waves' totals through LDS
__device__ __forceinline__ long long block_scan(long long v, long long* part, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  long long before = 0;
  for (int w = 0; w < wave; ++w) before += part[w];
  __syncthreads();
  return v + before;
}

// Every workgroup repeats the two sums over the streams (3 R words, from L2 after the first) and then fills its own tokens and pages: no workgroup
// waits for another, one launch, and the result does not depend on any order.  Launch-bound (3 R words in, 3 T + 2 R out): what a call takes is the chain of
// dependent loads, so what the second half needs of a stream is kept in LDS (2000 streams, 96 k tokens: 16.8 us when it was read again, 8.0 us now).
__global__ __launch_bounds__(PLAN_NT) void paged_plan_kernel(const int* __restrict__ lens, const int* __restrict__ fresh, const int* __restrict__ owned,
                                                             int* __restrict__ table, int ldt, int width, const int* __restrict__ free_pages, int nfree_max,
                                                             const int* __restrict__ n_free, int shift, int R, int T, int* __restrict__ cu_out,
                                                             int* __restrict__ kv_out, int* __restrict__ owned_out, int* __restrict__ nfree_out,
                                                             int* __restrict__ slots, int* __restrict__ positions, int* __restrict__ streams) {
  extern __shared__ int lds[];
  int* s_cu = lds;                             // [R + 1] first token row of each stream
  int* s_at = s_cu + R + 1;                    // [R] pages handed out before this stream's, or -1: refused
  int* s_len = s_at + R;                       // [R] cached tokens
  int* s_own = s_len + R;                      // [R] pages owned
  __shared__ long long part[PLAN_NT / 64];
  __shared__ int taken;
  const int tid = threadIdx.x, lane = tid & 63;
  const int per = (R + PLAN_NT - 1) / PLAN_NT, r0 = tid * per;
  const int have = max(0, min(*n_free, nfree_max));
  int n[PLAN_PER], need[PLAN_PER], len[PLAN_PER], own[PLAN_PER];
  long long sum = 0;
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i) {
    const int r = r0 + i;
    const bool in = i < per && r < R;
    n[i] = in ? max(fresh[r], 0) : 0;
    len[i] = in ? max(lens[r], 0) : 0;
    own[i] = in ? owned[r] : 0;
    sum += n[i];
  }
  if (tid == 0) taken = 0;
  long long at = block_scan(sum, part, tid) - sum;
  sum = 0;
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i) {
    const int r = r0 + i;
    need[i] = -1;
    if (i < per && r < R) {
      s_cu[r] = (int)(at < T ? at : T);
      at += n[i];
      if (r == R - 1) s_cu[R] = (int)(at < T ? at : T);
      s_len[r] = len[i];
      s_own[r] = max(own[i], 0);
      const long long pages = ((long long)len[i] + n[i] + (1 << shift) - 1) >> shift;
      if (pages <= width && at <= T) need[i] = max(0, (int)pages - max(own[i], 0));
    }
    sum += max(need[i], 0);
  }
  at = block_scan(sum, part, tid) - sum;
  const bool lead = blockIdx.x == 0;
  int end = 0;                                 // the running sum only grows: the streams that needed pages and got them are the first of those that needed any
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i) {
    const int r = r0 + i;
    if (i < per && r < R) {
      const bool ok = need[i] == 0 || (need[i] > 0 && at + need[i] <= have);      // (a stream that needs no page is never short of one)
      s_at[r] = ok ? (need[i] ? (int)at : 0) : -1;
      at += max(need[i], 0);
      if (ok && need[i] > 0) end = (int)at;
      if (lead) {
        kv_out[r] = ok ? len[i] + n[i] : 0;
        owned_out[r] = ok ? max(own[i], 0) + need[i] : own[i];
      }
    }
  }
  if (lead) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) end = max(end, __shfl_xor(end, o, 64));
    if (lane == 0 && end) atomicMax(&taken, end);
  }
  __syncthreads();
  if (lead) {
    for (int r = tid; r <= R; r += PLAN_NT) cu_out[r] = s_cu[r];
    if (tid == 0) *nfree_out = have - taken;
  }
  const int wave = (blockIdx.x * PLAN_NT + tid) >> 6, nwaves = gridDim.x * (PLAN_NT / 64);
  for (int r = wave; r < R; r += nwaves) {     // new pages into the tables
    if (s_at[r] < 0) continue;
    const int ow = s_own[r], pages = (int)(((long long)s_len[r] + (s_cu[r + 1] - s_cu[r]) + (1 << shift) - 1) >> shift);
    for (int j = lane; ow + j < pages; j += 64) table[(size_t)r * ldt + ow + j] = free_pages[have - 1 - s_at[r] - j];
  }
  for (int t = blockIdx.x * PLAN_NT + tid; t < T; t += gridDim.x * PLAN_NT) {
    int slot = -1, pos = -1, st = -1;
    if (t < s_cu[R]) {
      int lo = 0, hi = R;                      // the last stream that begins at or before t (an empty stream begins where the next one does)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t) lo = mid; else hi = mid;
      }
      st = lo;
      pos = s_len[st] + (t - s_cu[st]);
      if (s_at[st] >= 0) {
        const int ow = s_own[st], p = pos >> shift;
        const int pg = p < ow ? table[(size_t)st * ldt + p] : free_pages[have - 1 - s_at[st] - (p - ow)];
        const long long sl = ((long long)pg << shift) + (pos & ((1 << shift) - 1));
        if (pg >= 0 && sl <= 0x7fffffffll) slot = (int)sl;
      }
    }
    slots[t] = slot;
    positions[t] = pos;
    streams[t] = st;
  }
}

// One thread per 16-byte piece of a token's row; the address is formed in 64 bits (a cache may pass 4 GiB).  Bound by the 4 rows moved per token.
__global__ __launch_bounds__(256) void paged_kv_write_kernel(const bf16_t* __restrict__ k, long ldk, const bf16_t* __restrict__ v, long ldv,
                                                             bf16_t* __restrict__ kc, bf16_t* __restrict__ vc, const int* __restrict__ slots, long nslots,
                                                             int chunks, int total) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < total; i += gridDim.x * 256) {
    const int t = i / chunks, c = i - t * chunks;
    const int s = slots[t];
    if (s < 0 || s >= nslots) continue;
    const size_t to = ((size_t)s * chunks + c) * 8;
    *(u32x4_t*)(kc + to) = *(const u32x4_t*)(k + (size_t)t * ldk + c * 8);
    *(u32x4_t*)(vc + to) = *(const u32x4_t*)(v + (size_t)t * ldv + c * 8);
  }
}
}  // namespace

extern "C" int avt_paged_plan(const int* lens, const int* fresh, const int* owned, int* table, int ldt, int width, const int* free_pages, int nfree_max,
                              const int* n_free, int page, int R, int T, int* cu, int* kv_lens, int* owned_out, int* n_free_out, int* slots, int* positions,
                              int* streams, void* stream) {
  AVT_CHECK(lens && fresh && owned && table && n_free && cu && kv_lens && owned_out && n_free_out, "avt_paged_plan: null argument");
  AVT_CHECK(free_pages || nfree_max == 0, "avt_paged_plan: null free list");
  AVT_CHECK(T == 0 || (slots && positions && streams), "avt_paged_plan: null token output");
  AVT_CHECK(R >= 1 && R <= PLAN_RMAX, "avt_paged_plan: 1 to %d streams (got %d)", PLAN_RMAX, R);
  AVT_CHECK(T >= 0 && nfree_max >= 0 && width >= 1 && ldt >= width, "avt_paged_plan: bad sizes (T %d, free %d, width %d, ldt %d)", T, nfree_max, width, ldt);
  AVT_CHECK(T < 0x7ff00000, "avt_paged_plan: fewer than 2^31 - 2^20 token rows (got %d)", T);      // (a thread's row and the grid's stride stay an int)
  AVT_CHECK(page >= 8 && page <= 1024 && (page & (page - 1)) == 0, "avt_paged_plan: the page must be a power of two in [8, 1024] (got %d)", page);
  AVT_CHECK((long)width * page < 0x7fff0000l, "avt_paged_plan: a stream may hold fewer than 2^31 - 2^16 tokens (width %d, page %d)", width, page);
  const int blocks = T <= PLAN_NT ? 1 : (T + PLAN_NT - 1) / PLAN_NT < 512 ? (T + PLAN_NT - 1) / PLAN_NT : 512, lds = (4 * R + 1) * 4;
  if (lds > 63 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)paged_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    AVT_CHECK(e == hipSuccess, "avt_paged_plan: %s", hipGetErrorString(e));
  }
  hipLaunchKernelGGL(paged_plan_kernel, dim3(blocks), dim3(PLAN_NT), lds, (hipStream_t)stream, lens, fresh, owned, table, ldt, width, free_pages, nfree_max, n_free,
                     __builtin_ctz(page), R, T, cu, kv_lens, owned_out, n_free_out, slots, positions, streams);
  AVT_LAUNCH_CHECK();
  return 0;
}

extern "C" int avt_paged_kv_write(const void* k, long ldk, const void* v, long ldv, void* kcache, void* vcache, const int* slots, long nslots, int T, int width,
                                  void* stream) {
  AVT_CHECK(T >= 0 && width > 0 && width % 8 == 0, "avt_paged_kv_write: a row must be a positive multiple of 8 values (got %d)", width);
  if (T == 0) return 0;
  AVT_CHECK(k && v && kcache && vcache && slots && nslots >= 0, "avt_paged_kv_write: null argument");
  AVT_CHECK(ldk >= width && ldv >= width && ldk % 8 == 0 && ldv % 8 == 0 && aligned16(k) && aligned16(v) && aligned16(kcache) && aligned16(vcache),
            "avt_paged_kv_write: 16-byte aligned rows required");
  AVT_CHECK(nslots <= 1l << 31, "avt_paged_kv_write: a cache may hold 2^31 rows, as many as slots name (got %ld)", nslots);
  const long total = (long)T * (width / 8);
  AVT_CHECK(total < 0x7f000000l, "avt_paged_kv_write: too many values for one call (%ld rows of %d)", (long)T, width);
  const int blocks = (int)((total + 255) / 256 < 8192 ? (total + 255) / 256 : 8192);
  hipLaunchKernelGGL(paged_kv_write_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, (const bf16_t*)k, ldk, (const bf16_t*)v, ldv, (bf16_t*)kcache,
                     (bf16_t*)vcache, slots, nslots, width / 8, (int)total);
  AVT_LAUNCH_CHECK();
  return 0;
}
