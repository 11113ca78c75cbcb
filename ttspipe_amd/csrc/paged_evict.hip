// Eviction from a paged cache by gathered attention weight. For each
// (sequence, kv head) of n > budget rows, the rows are ranked by
//   key = +inf where slot_pos < sinks or slot_pos > position - recent,
//         else the score (NaN counts as -inf),
// ties to the lowest slot; the first `budget` are kept. Attention does not
// care about the order of the slots, so a kept row below `budget` stays where
// it is, and the j-th kept row from slot `budget` on moves into the j-th free
// slot below (K, V, score and position): sources and destinations do not
// overlap, and only the rows that have to move are read and written.
//
// The threshold is the budget-th largest key, found digit by digit (four
// passes over 8 bits of the key's order-preserving integer form, a histogram
// in LDS each); a scan over the slots in order then names the movers and the
// free slots. A second launch moves the K and V rows, a group of lanes each.
#include "paged_common.h"

namespace ttsp {

struct EvictArgs {
  Paged c;
  const long long* SLOT;
  const long long* POS;
  int budget, sinks, recent, max_moves, hd;
  int* work;  // per (sequence, kv head): the count, then max_moves sources and max_moves destinations
};

constexpr int EV_T = 1024;

// Larger keys are larger integers; -0 and +0 are one key.
__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = __float_as_uint(__fadd_rn(f, 0.0f));
  return u >> 31 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t evict_key(const EvictArgs& a, const float* sc, const int* sp, int j, long long pos) {
  const float f = sc[j];
  const int p = sp[j];
  if (p < a.sinks || p > pos - a.recent) return order_of(__uint_as_float(0x7f800000u));
  return order_of(f != f ? __uint_as_float(0xff800000u) : f);
}

// Exclusive prefix over the workgroup of v (0 .. a few), and the total.
__device__ __forceinline__ int block_scan(int v, int* s, int tid, int* total) {
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if ((tid & 63) >= o) x += y;
  }
  __syncthreads();
  if ((tid & 63) == 63) s[tid >> 6] = x;
  __syncthreads();
  int base = 0, all = 0;
  for (int w = 0; w < EV_T / 64; ++w) {
    if (w < (tid >> 6)) base += s[w];
    all += s[w];
  }
  *total = all;
  return base + x - v;
}

__global__ __launch_bounds__(EV_T) void paged_evict_select_kernel(const EvictArgs a) {
  __shared__ int hist[256], scan_s[EV_T / 64], pick[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = a.c.rows(a.SLOT[b]);
  int* work = a.work + ((size_t)b * a.c.nkv + h) * (1 + 2 * (size_t)a.max_moves);
  if (n <= a.budget) {
    if (tid == 0) work[0] = 0;
    return;
  }
  float* sc = a.c.scores + b * a.c.score_seq + h * a.c.score_head;
  int* sp = a.c.slot_pos + b * a.c.pos_seq + h * a.c.pos_head;
  const long long pos = a.POS[b];
  uint32_t prefix = 0;
  int want = a.budget;  // how many of the keys that share the prefix are still kept
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += EV_T) {
      const uint32_t k = evict_key(a, sc, sp, j, pos);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, left = want;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      pick[0] = d;
      pick[1] = left;
    }
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    want = pick[1];
  }
  // keys above `prefix` are kept, and the first `want` equal to it
  int* src = work + 1;
  int* dst = src + a.max_moves;
  int equal = 0, movers = 0, holes = 0;
  for (int j0 = 0; j0 < n; j0 += EV_T) {
    const int j = j0 + tid;
    const uint32_t k = j < n ? evict_key(a, sc, sp, j, pos) : 0;
    int total;
    const int eq = block_scan(j < n && k == prefix, scan_s, tid, &total);
    const bool kept = j < n && (k > prefix || (k == prefix && equal + eq < want));
    equal += total;
    const bool mover = kept && j >= a.budget, hole = j < a.budget && !kept;
    const int m = block_scan(mover, scan_s, tid, &total);
    if (mover && movers + m < a.max_moves) src[movers + m] = j;
    movers += total;
    const int o = block_scan(hole, scan_s, tid, &total);
    if (hole && holes + o < a.max_moves) dst[holes + o] = j;
    holes += total;
  }
  __syncthreads();
  const int moves = min(min(movers, holes), a.max_moves);  // all three are one number
  if (tid == 0) work[0] = moves;
  for (int i = tid; i < moves; i += EV_T) {
    sc[dst[i]] = sc[src[i]];
    sp[dst[i]] = sp[src[i]];
  }
}

template <int D>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(const EvictArgs a) {
  constexpr int LH = D / 8, ROWS = 256 / LH;
  const int h = blockIdx.y, b = blockIdx.z;
  const int* work = a.work + ((size_t)b * a.c.nkv + h) * (1 + 2 * (size_t)a.max_moves);
  const int i = blockIdx.x * ROWS + (int)threadIdx.x / LH, e = (threadIdx.x % LH) * 8;
  if (i >= work[0]) return;
  const int src = work[1 + i], dst = work[1 + a.max_moves + i], mask = (1 << a.c.shift) - 1;
  const int from = a.c.page(b, src), to = a.c.page(b, dst);
  if (from < 0 || to < 0) return;
  *reinterpret_cast<u32x4*>(a.c.K + to * a.c.k_page + h * a.c.k_head + (dst & mask) * a.c.k_row + e) =
      *reinterpret_cast<const u32x4*>(a.c.K + from * a.c.k_page + h * a.c.k_head + (src & mask) * a.c.k_row + e);
  *reinterpret_cast<u32x4*>(a.c.V + to * a.c.v_page + h * a.c.v_head + (dst & mask) * a.c.v_row + e) =
      *reinterpret_cast<const u32x4*>(a.c.V + from * a.c.v_page + h * a.c.v_head + (src & mask) * a.c.v_row + e);
}

}  // namespace ttsp

using namespace ttsp;

extern "C" int ttsp_paged_evict_work_kib(int seqs, int nkv, int cols, int page_size, int budget) {
  if (seqs < 1 || nkv < 1 || cols < 1 || page_size < 1 || budget < 1) return 0;
  const long long cap = (long long)cols * page_size;
  if (cap <= budget) return 0;
  const long long moves = budget < cap - budget ? budget : cap - budget;
  const long long kib = ((long long)seqs * nkv * (1 + 2 * moves) * 4 + 1023) / 1024;
  return kib > 0x7fffffffLL ? -1 : (int)kib;
}

extern "C" int ttsp_paged_evict(const ttsp_paged_cache* cache, const long long* SLOT, const long long* POS,
                                int budget, int sinks, int recent, int* work, hipStream_t stream) {
  EvictArgs a{};
  if (!paged_args(cache, &a.c) || !a.c.scores || !a.c.slot_pos || !SLOT || !POS || budget < 1 || sinks < 0 ||
      recent < 0 || sinks > budget - recent || !a.c.score_seq || !a.c.pos_seq)
    return (int)hipErrorInvalidValue;
  const long long cap = a.c.cap();
  if (cap <= budget) return 0;  // no table row holds more than the budget
  if (!work || (uintptr_t)work % 4) return (int)hipErrorInvalidValue;
  a.SLOT = SLOT;
  a.POS = POS;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.max_moves = (int)(budget < cap - budget ? budget : cap - budget);
  a.hd = cache->head_dim;
  a.work = work;
  hipLaunchKernelGGL(paged_evict_select_kernel, dim3(a.c.nkv, a.c.seqs), dim3(EV_T), 0, stream, a);
  const int rows = 256 / (cache->head_dim / 8);
  const dim3 grid((a.max_moves + rows - 1) / rows, a.c.nkv, a.c.seqs);
  if (cache->head_dim == 128) hipLaunchKernelGGL(paged_evict_move_kernel<128>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(paged_evict_move_kernel<64>, grid, dim3(256), 0, stream, a);
  TTSP_RETURN_LAUNCH();
}
