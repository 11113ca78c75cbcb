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
// The threshold is the budget-th largest key, found digit by digit of the
// key's order-preserving integer form (11, 11 and 10 bits): a histogram in LDS,
// each bin in eight copies that neighbouring lanes spread over (scores share
// their leading bits, and a wave's adds to one word queue up), and a scan from
// the top bin. It ends early where a bin is kept whole. One workgroup ranks a
// (sequence, kv head), its keys read once and held in registers (up to 64 a
// thread; a longer cache's are read again in each pass), a wave's keys
// neighbouring slots, so that ranks among equal keys, movers and free slots are
// counted with ballots and one prefix over the waves each. A second launch
// moves the K and V rows, a group of lanes each; where the cache has little room
// past the budget the first moves them itself. A sequence only a few rows over
// its budget, as after a decode step, has its lowest keys taken out one by one
// instead, while the rows past the budget, which may have to move, are on
// their way already.
#include "paged_common.h"

namespace ttsp {

struct EvictArgs {
  Paged c;
  const long long* SLOT;
  const long long* POS;
  int budget, sinks, recent, max_moves;
  int* work;  // per (sequence, kv head): the count, then max_moves sources and max_moves destinations
};

constexpr int EV_BINS = 2048, EV_COPIES = 8;
// At most this many rows a (sequence, kv head) are moved by the ranking workgroup itself.
constexpr int EV_INLINE = 256;
// Rows over the budget up to which the lowest are taken out one by one.
constexpr int EV_FEW = 4;

// Larger keys are larger integers; -0 and +0 are one key.
__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = __float_as_uint(__fadd_rn(f, 0.0f));
  return u >> 31 ? ~u : u | 0x80000000u;
}

// The key of a row of score f and position p: +inf if protected (p below
// `sinks` or above `newest`, the last position that is not recent).
__device__ __forceinline__ uint32_t evict_key(float f, int p, int sinks, long long newest) {
  if (p < sinks || p > newest) return order_of(__uint_as_float(0x7f800000u));
  return order_of(f != f ? __uint_as_float(0xff800000u) : f);
}

// A row's K and V, eight elements a lane (D / 8 lanes a row).
struct Row {
  u32x4 k, v;
};
// Slot j's row of sequence b, head h, in `page` (not a hole).
__device__ __forceinline__ Row load_row(const Paged& c, int page, int h, int j, int lane) {
  const int row = j & ((1 << c.shift) - 1), e = lane * 8;
  return Row{*reinterpret_cast<const u32x4*>(c.K + page * c.k_page + h * c.k_head + row * c.k_row + e),
             *reinterpret_cast<const u32x4*>(c.V + page * c.v_page + h * c.v_head + row * c.v_row + e)};
}
__device__ __forceinline__ void store_row(const Paged& c, int page, int h, int j, int lane, const Row& r) {
  const int row = j & ((1 << c.shift) - 1), e = lane * 8;
  *reinterpret_cast<u32x4*>(c.K + page * c.k_page + h * c.k_head + row * c.k_row + e) = r.k;
  *reinterpret_cast<u32x4*>(c.V + page * c.v_page + h * c.v_head + row * c.v_row + e) = r.v;
}
__device__ __forceinline__ void move_row(const Paged& c, int b, int h, int src, int dst, int lane) {
  const int from = c.page(b, src), to = c.page(b, dst);
  if (from >= 0 && to >= 0) store_row(c, to, h, dst, lane, load_row(c, from, h, src, lane));
}

// T threads; R: keys a thread holds (0: read again in every pass).
template <int T, int R, int D, bool INLINE>
__global__ __launch_bounds__(T) void paged_evict_select_kernel(const EvictArgs a) {
  constexpr int W = T / 64, PER = EV_BINS / T;  // waves; bins a thread adds up
  __shared__ __align__(16) int hist[EV_BINS * EV_COPIES];
  __shared__ int wsum[2][W], pick[3];
  __shared__ int moves_s[INLINE ? 2 * EV_INLINE : 1];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = a.c.rows(a.SLOT[b]);
  int* const work = INLINE ? nullptr : a.work + ((size_t)b * a.c.nkv + h) * (1 + 2 * (size_t)a.max_moves);
  if (n <= a.budget) {
    if (!INLINE && tid == 0) work[0] = 0;
    return;
  }
  float* const sc = a.c.scores + b * a.c.score_seq + h * a.c.score_head;
  int* const sp = a.c.slot_pos + b * a.c.pos_seq + h * a.c.pos_head;
  const long long newest = a.POS[b] - a.recent;
  const bool few = INLINE && R != 0 && n - a.budget <= EV_FEW;
  constexpr int LH = D / 8;
  // few: group g of LH lanes holds the row of slot budget + g
  const int over = a.budget + tid / LH;
  Row row{};
  int row_page = -1;
  if (few && over < n) {
    row_page = a.c.page(b, over);
    if (row_page >= 0) row = load_row(a.c, row_page, h, over, tid % LH);
  }
  // wave w takes slots w * span .. + span - 1, 64 at a time
  const int steps = (n + T - 1) / T, first = wave * steps * 64 + lane;
  uint32_t held[R ? R : 1];
  if constexpr (R != 0) {
    constexpr int AT_ONCE = R < 8 ? R : 8;  // loads of a lane under way together
#pragma unroll
    for (int i0 = 0; i0 < R; i0 += AT_ONCE) {
      if (i0 >= steps) break;
      float f[AT_ONCE];
      int p[AT_ONCE];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int j = min(first + 64 * (i0 + i), n - 1);
        f[i] = sc[j], p[i] = sp[j];
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) held[i0 + i] = evict_key(f[i], p[i], a.sinks, newest);
    }
  }
  if constexpr (INLINE && R != 0) {
    if (few) {
      __shared__ unsigned long long low_s[EV_FEW][W];
      int out[EV_FEW];  // the slots taken out
#pragma unroll
      for (int r = 0; r < EV_FEW; ++r) {
        out[r] = 0x7fffffff;
        if (r >= n - a.budget) continue;
        // the lowest key, of equal ones the highest slot's; ~0: none of this lane's
        unsigned long long low = ~0ull;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int j = first + 64 * i;
          bool live = i < steps && j < n;
#pragma unroll
          for (int q = 0; q < r; ++q) live = live && j != out[q];
          if (live) low = min(low, (unsigned long long)held[i] << 32 | (uint32_t)~j);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) low = min(low, (unsigned long long)__shfl_xor((long long)low, o, 64));
        if (lane == 0) low_s[r][wave] = low;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) low = min(low, low_s[r][w]);
        out[r] = (int)~(uint32_t)low;
      }
      // this group's slot moves if it stays: to the hole of its rank among the movers
      if (over >= n) return;
      int rank = 0, dst = -1;
      bool stays = true;
#pragma unroll
      for (int r = 0; r < EV_FEW; ++r) stays = stays && out[r] != over;
#pragma unroll
      for (int q = 0; q < EV_FEW; ++q) {
        bool kept = a.budget + q < over;
#pragma unroll
        for (int r = 0; r < EV_FEW; ++r) kept = kept && out[r] != a.budget + q;
        rank += kept;
      }
#pragma unroll
      for (int r = 0; r < EV_FEW; ++r) {
        int below = 0;
#pragma unroll
        for (int q = 0; q < EV_FEW; ++q) below += out[q] < out[r];
        if (below == rank && out[r] < a.budget) dst = out[r];
      }
      if (!stays || dst < 0) return;
      const int to = a.c.page(b, dst);
      if (row_page >= 0 && to >= 0) store_row(a.c, to, h, dst, tid % LH, row);
      if (tid % LH == 0) {
        sc[dst] = sc[over];
        sp[dst] = sp[over];
      }
      return;
    }
  }
  // f(slot, key) for this lane's rows in order; false in `live` for lanes past the last row
  auto each = [&](auto&& f) {
    if constexpr (R != 0) {
      int at = first;
      asm("" : "+v"(at));  // slots worked out anew each time: kept, 64 of them would not fit beside the keys
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i < steps) f(at + 64 * i, held[i], at + 64 * i < n);
    } else {
      for (int i = 0; i < steps; ++i) {
        const int j = first + 64 * i, r = min(j, n - 1);
        f(j, evict_key(sc[r], sp[r], a.sinks, newest), j < n);
      }
    }
  };

  uint32_t limit = 0;   // the digits found so far, the rest 0
  int want = a.budget;  // how many of the keys with these digits are still kept
  bool whole = false;   // all of them
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int above = pass == 1 ? 21 : 10;  // (pass > 0) the bits found lie from here on
    const uint32_t bins = pass == 2 ? 1024 : 2048;
    for (int i = tid * 4; i < EV_BINS * EV_COPIES; i += T * 4) *reinterpret_cast<u32x4*>(hist + i) = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    each([&](int, uint32_t k, bool live) {
      if (live && (pass == 0 || (k >> above) == (limit >> above)))
        atomicAdd(&hist[((k >> shift) & (bins - 1)) * EV_COPIES + (lane & (EV_COPIES - 1))], 1);
    });
    __syncthreads();
    // thread t's bins, from the top: EV_BINS - 1 - PER t and the PER - 1 below it
    int sum[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const u32x4* c = reinterpret_cast<const u32x4*>(hist + (EV_BINS - 1 - PER * tid - i) * EV_COPIES);
      const u32x4 x = c[0], y = c[1];
      sum[i] = (int)(((x[0] + x[1]) + (x[2] + x[3])) + ((y[0] + y[1]) + (y[2] + y[3])));
      mine += sum[i];
    }
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o, 64);
      if (lane >= o) upto += y;
    }
    if (lane == 63) wsum[0][wave] = upto;
    __syncthreads();
    int before = upto - mine;
    for (int w = 0; w < W; ++w) before += w < wave ? wsum[0][w] : 0;
    if (before < want && before + mine >= want) {  // exactly one thread
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (before < want && before + sum[i] >= want) {
          pick[0] = EV_BINS - 1 - PER * tid - i;
          pick[1] = want - before;
          pick[2] = sum[i];
        }
        before += sum[i];
      }
    }
    __syncthreads();
    limit |= (uint32_t)pick[0] << shift;
    want = pick[1];
    whole = pick[2] == want;
    if (whole) break;
  }
  // kept: keys above `limit` and the first `want` equal to it (`whole`: limit's
  // lower digits are 0 and every key from it on is kept; it is not 0 then, as
  // not all keys are kept)
  if (whole) --limit, want = 0;

  // rank of this wave's first key among the equal ones
  auto count_waves = [&](int x, int y, int* xb, int* yb, int* xt) {  // uniform values a wave
    __syncthreads();
    if (lane == 0) wsum[0][wave] = x, wsum[1][wave] = y;
    __syncthreads();
    *xb = *yb = *xt = 0;
    for (int w = 0; w < W; ++w) {
      if (w < wave) *xb += wsum[0][w], *yb += wsum[1][w];
      *xt += wsum[0][w];
    }
  };
  int equal = 0, unused, total;
  if (!whole) {
    int mine = 0;
    each([&](int, uint32_t k, bool live) { mine += __popcll(__ballot(live && k == limit)); });
    count_waves(mine, 0, &equal, &unused, &total);
  }
  // lanes before this one
  auto before_me = [&](uint64_t m) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
  };
  int rank = equal;
  auto keeps = [&](uint32_t k, bool live) {
    const bool eq = live && k == limit && !whole;
    const uint64_t m = __ballot(eq);
    const bool kept = live && (k > limit || (eq && rank + before_me(m) < want));
    rank += __popcll(m);
    return kept;
  };
  int movers = 0, holes = 0;
  each([&](int j, uint32_t k, bool live) {
    const bool kept = keeps(k, live);
    movers += __popcll(__ballot(kept && j >= a.budget));
    holes += __popcll(__ballot(live && !kept && j < a.budget));
  });
  int mb, hb;
  count_waves(movers, holes, &mb, &hb, &total);  // as many holes as movers
  int* const src = INLINE ? moves_s : work + 1;
  const int room = INLINE ? EV_INLINE : a.max_moves;
  int* const dst = src + room;
  rank = equal;
  each([&](int j, uint32_t k, bool live) {
    const bool kept = keeps(k, live), mover = kept && j >= a.budget, hole = live && !kept && j < a.budget;
    const uint64_t mm = __ballot(mover), hm = __ballot(hole);
    const int mi = mb + before_me(mm), hi = hb + before_me(hm);
    if (mover && mi < room) src[mi] = j;
    if (hole && hi < room) dst[hi] = j;
    mb += __popcll(mm);
    hb += __popcll(hm);
  });
  const int moves = min(total, room);
  if (!INLINE && tid == 0) work[0] = moves;
  __syncthreads();
  for (int i = tid; i < moves; i += T) {
    sc[dst[i]] = sc[src[i]];
    sp[dst[i]] = sp[src[i]];
  }
  if constexpr (INLINE)
    for (int i = tid / (D / 8); i < moves; i += T / (D / 8)) move_row(a.c, b, h, src[i], dst[i], tid % (D / 8));
}

template <int D>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(const EvictArgs a) {
  constexpr int LH = D / 8, ROWS = 256 / LH;
  const int h = blockIdx.y, b = blockIdx.z;
  const int* work = a.work + ((size_t)b * a.c.nkv + h) * (1 + 2 * (size_t)a.max_moves);
  const int i = blockIdx.x * ROWS + (int)threadIdx.x / LH;
  if (i >= work[0]) return;
  move_row(a.c, b, h, work[1 + i], work[1 + a.max_moves + i], threadIdx.x % LH);
}

template <int D>
void launch_evict(const EvictArgs& a, hipStream_t stream) {
  const dim3 grid(a.c.nkv, a.c.seqs);
  const int cap = a.c.cap();
#define TTSP_EV(TV, RV, INL) \
  hipLaunchKernelGGL((paged_evict_select_kernel<TV, RV, D, INL>), grid, dim3(TV), 0, stream, a)
  if (a.max_moves <= EV_INLINE) {
    if (cap <= 256 * 8) TTSP_EV(256, 8, true);
    else if (cap <= 1024 * 8) TTSP_EV(1024, 8, true);
    else if (cap <= 1024 * 64) TTSP_EV(1024, 64, true);
    else TTSP_EV(1024, 0, true);
    return;
  }
  if (cap <= 256 * 8) TTSP_EV(256, 8, false);
  else if (cap <= 1024 * 8) TTSP_EV(1024, 8, false);
  else if (cap <= 1024 * 64) TTSP_EV(1024, 64, false);
  else TTSP_EV(1024, 0, false);
#undef TTSP_EV
  const int rows = 256 / (D / 8);
  hipLaunchKernelGGL(paged_evict_move_kernel<D>, dim3((a.max_moves + rows - 1) / rows, a.c.nkv, a.c.seqs), dim3(256), 0,
                     stream, a);
}

}  // namespace ttsp

using namespace ttsp;

extern "C" int ttsp_paged_evict_work_kib(int seqs, int nkv, int cols, int page_size, int budget) {
  if (seqs < 1 || nkv < 1 || cols < 1 || page_size < 1 || budget < 1) return 0;
  const long long cap = (long long)cols * page_size;
  if (cap <= budget) return 0;
  const long long moves = budget < cap - budget ? budget : cap - budget;
  if (moves <= EV_INLINE) return 0;
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
  a.SLOT = SLOT;
  a.POS = POS;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.max_moves = (int)(budget < cap - budget ? budget : cap - budget);
  if (a.max_moves > EV_INLINE && (!work || (uintptr_t)work % 4)) return (int)hipErrorInvalidValue;
  a.work = work;
  if (cache->head_dim == 128) launch_evict<128>(a, stream);
  else launch_evict<64>(a, stream);
  TTSP_RETURN_LAUNCH();
}
