// Eviction from a paged cache by gathered attention weight. For each
// (sequence, kv head) of n > budget rows, the rows are ranked by
//   key = +inf where slot_pos < sinks or slot_pos > position - recent,
//         else the score (NaN counts as -inf; a score of +inf is as good as protected),
// ties to the lowest slot; the first `budget` are kept. Attention does not
// care about the order of the slots, so a kept row below `budget` stays where
// it is, and the j-th kept row from slot `budget` on moves into the j-th free
// slot below (K, V, score and position): sources and destinations do not
// overlap, and only the rows that have to move are read and written.
//
// A row's rank is its key and, below it, its slot counted from the end (so that
// ties go to the lowest slot): no two are equal, and the kept rows are those
// whose rank is at least the budget-th largest. That is found digit by digit
// (11 bits) of the rank's integer form: a histogram in LDS, each bin in eight
// copies that neighbouring lanes spread over (scores share their leading bits,
// and a wave's adds to one word queue up), and a scan from the top bin. It ends
// where a bin is kept whole, as a rule with the key's last digit.
//
// Up to 8192 slots one workgroup ranks a (sequence, kv head), its keys read once
// and held in registers, a wave's keys neighbouring slots, so that movers and
// free slots are listed in order with ballots and one prefix over the waves. A
// second launch moves the rows, a group of lanes each. Where the budget or the
// cache's room past it is at most EV_INLINE rows the first launch moves them
// itself, and there a sequence only a few rows over its budget, as after a decode
// step, has its lowest keys taken out one by one instead, while the rows past the
// budget, which may have to move, are on their way already. A wider cache is ranked
// in full for such a step too: 32 sequences of 1025 rows down to 1024 (8 heads)
// take 4.9 us in tables of 1088 slots, 16.2 in 2304 to 8192, 41 in 16384 and 115 in
// 65536.
//
// In longer caches one workgroup's instructions, not its bytes, set the time
// (65531 rows a head: 74 us, 25 in parts), so they are ranked in parts of a few thousand
// slots: a launch for the parts' histograms of the first digit; one that finds
// that digit and notes the candidates (the rows in its bin, a few per cent, in
// any order: only how many there are of a kind is ever asked); one whose
// workgroups each finish the ranking on all candidates and list their part's
// movers and free slots; and the moving one.
//
// Ranking reads 8 bytes a row, moving reads and writes the moved rows' K and V (256
// bytes at random places): 8 sequences of 1500 to 8192 rows down to 2048 (8 heads
// of 128): 12.7 us of ranking, which one workgroup's chain of passes sets, and
// 20 of moving, about 3.7 TB/s; one of 65531 down to 8192: 5.3 + 9.1 + 12.2 and 14
// us (the second and third launch read their part twice, and each workgroup of the
// third clears and scans its bins for every further digit); 32 of 1025 down to 1024
// in a table of 1088: 5.3 us, a chain of dependent reads.
#include "paged_common.h"

namespace ttsp {

struct EvictArgs {
  Paged c;
  const long long* SLOT;
  const long long* POS;
  int budget, sinks, recent, max_moves;
  int* work;  // per (sequence, kv head), list_ints: the count, then max_moves sources and max_moves destinations
  // long caches: parts of `part` slots; behind the lists, per (sequence, kv
  // head): four words (candidates, the first digit, how many of its rows are
  // kept, whether all), per part two (movers and free slots that are no
  // candidates) and a histogram, then `parts` * `part` candidates of two words
  int parts, part;
  int* heads;
  int* counts;
  int* hists;
  uint2* cands;
  __host__ __device__ size_t list_ints() const { return 1 + 2 * (size_t)max_moves; }
};

constexpr int EV_BINS = 2048, EV_COPIES = 8;
// At most this many rows a (sequence, kv head) are moved by the ranking workgroup itself.
constexpr int EV_INLINE = 256;
// Rows over the budget up to which the lowest are taken out one by one.
constexpr int EV_FEW = 4;

// Slots up to which one workgroup ranks a (sequence, kv head): sequences of up
// to 8192 took 12.7 us in one, 24.0 in the three launches over parts.
constexpr int EV_WHOLE = 8192;
static_assert(EV_WHOLE == 1024 * 8, "eight keys a thread");
constexpr int EV_PT = 512, EV_PART = 4096, EV_PARTS = 64;  // threads, slots (at least) and parts (at most) in parts

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

// A row's rank: 56 bits, taken apart into digits at these shifts.
constexpr int EV_DIGITS = 6;
__device__ __forceinline__ uint64_t rank_of(uint32_t key, int slot) {
  return (uint64_t)key << 24 | (uint32_t)(TTSP_PAGED_MAX_SLOTS - 1 - slot);
}
__device__ __forceinline__ int digit_shift(int i) { return i == 5 ? 0 : 45 - 11 * i; }  // (the last: one bit)
__device__ __forceinline__ uint32_t digit_mask(int i) { return i == 5 ? 1 : EV_BINS - 1; }

// Where the search stands: the digits found (the rest 0), how many of the rows
// that share them are still kept, and whether all of them are.
struct Search {
  uint64_t limit;
  int want;
  bool whole;
};

// One digit: the bin of `hist` (COPIES words each) in which the want-th row from
// the top lies. All T threads; `wsum` of T / 64 words, `pick` of 3.
template <int T, int COPIES>
__device__ __forceinline__ void find_digit(const int* hist, int* wsum, int* pick, int i, int tid, Search* s) {
  constexpr int PER = EV_BINS / T;
  const int lane = tid & 63, wave = tid >> 6;
  // thread t's bins, from the top: EV_BINS - 1 - PER t and the PER - 1 below it
  int sum[PER], mine = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int bin = EV_BINS - 1 - PER * tid - k;
    if constexpr (COPIES == 8) {
      const u32x4* c = reinterpret_cast<const u32x4*>(hist + bin * 8);
      const u32x4 x = c[0], y = c[1];
      sum[k] = (int)(((x[0] + x[1]) + (x[2] + x[3])) + ((y[0] + y[1]) + (y[2] + y[3])));
    } else {
      sum[k] = hist[bin];
    }
    mine += sum[k];
  }
  const int upto = (int)lane_prefix((uint32_t)mine);
  if (lane == 63) wsum[wave] = upto;
  __syncthreads();
  int before = upto - mine;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) before += w < wave ? wsum[w] : 0;
  if (before < s->want && before + mine >= s->want) {  // exactly one thread
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (before < s->want && before + sum[k] >= s->want) {
        pick[0] = EV_BINS - 1 - PER * tid - k;
        pick[1] = s->want - before;
        pick[2] = sum[k];
      }
      before += sum[k];
    }
  }
  __syncthreads();
  s->limit |= (uint64_t)(uint32_t)pick[0] << digit_shift(i);
  s->want = pick[1];
  s->whole = pick[2] == pick[1];
}

template <int T>
__device__ __forceinline__ void clear_bins(int* hist, int words, int tid) {
  for (int i = tid * 4; i < words; i += T * 4) *reinterpret_cast<u32x4*>(hist + i) = u32x4{0u, 0u, 0u, 0u};
}

// Lanes before this one in `m`.
__device__ __forceinline__ int lanes_before(uint64_t m) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
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
// The row of slot src to slot dst with its score and position (sc, sp: the
// sequence's and head's). Nothing of it where either is in a hole.
__device__ __forceinline__ void move_row(const Paged& c, float* sc, int* sp, int b, int h, int src, int dst, int lane) {
  const int from = c.page(b, src), to = c.page(b, dst);
  if (from < 0 || to < 0) return;
  if (lane == 0) {
    sc[dst] = sc[src];
    sp[dst] = sp[src];
  }
  store_row(c, to, h, dst, lane, load_row(c, from, h, src, lane));
}

// T threads holding eight keys each.
template <int T, int D, bool INLINE>
__global__ __launch_bounds__(T) void paged_evict_select_kernel(const EvictArgs a) {
  constexpr int W = T / 64, R = 8;
  __shared__ __align__(16) int hist[EV_BINS * EV_COPIES];
  __shared__ int wsum[2][W], pick[3];
  __shared__ int moves_s[INLINE ? 2 * EV_INLINE : 1];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = a.c.rows(a.SLOT[b]);
  int* const work = INLINE ? nullptr : a.work + ((size_t)b * a.c.nkv + h) * a.list_ints();
  if (n <= a.budget) {
    if (!INLINE && tid == 0) work[0] = 0;
    return;
  }
  float* const sc = a.c.scores + b * a.c.score_seq + h * a.c.score_head;
  int* const sp = a.c.slot_pos + b * a.c.pos_seq + h * a.c.pos_head;
  const long long newest = a.POS[b] - a.recent;
  const bool few = INLINE && n - a.budget <= EV_FEW;
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
  uint32_t held[R];
  {
    float f[R];
    int p[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int j = min(first + 64 * i, n - 1);
      f[i] = sc[j], p[i] = sp[j];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) held[i] = evict_key(f[i], p[i], a.sinks, newest);
  }
  if constexpr (INLINE) {
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
      if (row_page < 0 || to < 0) return;
      store_row(a.c, to, h, dst, tid % LH, row);
      if (tid % LH == 0) {
        sc[dst] = sc[over];
        sp[dst] = sp[over];
      }
      return;
    }
  }
  // f(slot, key, whether there is such a row) for this lane's rows in order
  auto each = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < steps) f(first + 64 * i, held[i], first + 64 * i < n);
  };

  Search s{0, a.budget, false};
  for (int i = 0; i < EV_DIGITS && !s.whole; ++i) {
    clear_bins<T>(hist, EV_BINS * EV_COPIES, tid);
    __syncthreads();
    const int shift = digit_shift(i), done = i ? digit_shift(i - 1) : 0;
    const uint32_t mask = digit_mask(i);
    if (i == 0)
      each([&](int, uint32_t k, bool live) {
        if (live) atomicAdd(&hist[(k >> 21) * EV_COPIES + (lane & (EV_COPIES - 1))], 1);
      });
    else
      each([&](int j, uint32_t k, bool live) {
        const uint64_t r = rank_of(k, j);
        if (live && (r >> done) == (s.limit >> done))
          atomicAdd(&hist[((uint32_t)(r >> shift) & mask) * EV_COPIES + (lane & (EV_COPIES - 1))], 1);
      });
    __syncthreads();
    find_digit<T, EV_COPIES>(hist, wsum[0], pick, i, tid, &s);
  }

  int movers = 0, holes = 0;
  each([&](int j, uint32_t k, bool live) {
    const bool kept = rank_of(k, j) >= s.limit;
    movers += __popcll(__ballot(live && kept && j >= a.budget));
    holes += __popcll(__ballot(live && !kept && j < a.budget));
  });
  __syncthreads();
  if (lane == 0) wsum[0][wave] = movers, wsum[1][wave] = holes;
  __syncthreads();
  int mb = 0, hb = 0, total = 0;  // as many free slots as movers
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < wave) mb += wsum[0][w], hb += wsum[1][w];
    total += wsum[0][w];
  }
  const int room = INLINE ? EV_INLINE : a.max_moves;
  int* const src = INLINE ? moves_s : work + 1;
  int* const dst = src + room;
  each([&](int j, uint32_t k, bool live) {
    const bool kept = rank_of(k, j) >= s.limit, mover = live && kept && j >= a.budget, hole = live && !kept && j < a.budget;
    const uint64_t mm = __ballot(mover), hm = __ballot(hole);
    const int mi = mb + lanes_before(mm), hi = hb + lanes_before(hm);
    if (mover && mi < room) src[mi] = j;
    if (hole && hi < room) dst[hi] = j;
    mb += __popcll(mm);
    hb += __popcll(hm);
  });
  const int moves = min(total, room);
  if (!INLINE) {
    if (tid == 0) work[0] = moves;
    return;
  }
  __syncthreads();
  for (int i = tid / LH; i < moves; i += T / LH) move_row(a.c, sc, sp, b, h, src[i], dst[i], tid % LH);
}

// What the launches over parts share: part blockIdx.x of (kv head blockIdx.y,
// sequence blockIdx.z).
struct Part {
  int b, h, p, n, list, parts, j0, j1;  // parts: those that have rows; slots j0 .. j1 - 1
  const float* sc;
  const int* sp;
  long long newest;
};
__device__ __forceinline__ bool part_of(const EvictArgs& a, Part* q) {
  q->p = blockIdx.x, q->h = blockIdx.y, q->b = blockIdx.z;
  q->n = a.c.rows(a.SLOT[q->b]);
  q->list = q->b * a.c.nkv + q->h;
  q->j0 = q->p * a.part, q->j1 = min(q->j0 + a.part, q->n);
  q->parts = (q->n + a.part - 1) / a.part;
  q->sc = a.c.scores + q->b * a.c.score_seq + q->h * a.c.score_head;
  q->sp = a.c.slot_pos + q->b * a.c.pos_seq + q->h * a.c.pos_head;
  q->newest = a.POS[q->b] - a.recent;
  return q->n > a.budget && q->j0 < q->n;
}

// f(slot, key, whether there is such a row) for this thread's rows of the part,
// a wave's neighbours and in order; eight are read at once.
template <typename F>
__device__ __forceinline__ void part_rows(const EvictArgs& a, const Part& q, int wave, int lane, F&& f) {
  const int steps = (q.j1 - q.j0 + EV_PT - 1) / EV_PT, first = q.j0 + wave * steps * 64 + lane;
  for (int i0 = 0; i0 < steps; i0 += 8) {
    float sc[8];
    int sp[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = min(first + 64 * (i0 + i), q.j1 - 1);
      sc[i] = q.sc[j], sp[i] = q.sp[j];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = first + 64 * (i0 + i);
      if (i0 + i < steps) f(j, evict_key(sc[i], sp[i], a.sinks, q.newest), j < q.j1);
    }
  }
}

// The part's histogram of the first digit.
__global__ __launch_bounds__(EV_PT) void paged_evict_count_kernel(const EvictArgs a) {
  __shared__ __align__(16) int hist[EV_BINS * EV_COPIES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Part q;
  if (!part_of(a, &q)) return;
  if (q.p == 0 && tid == 0) a.heads[q.list * 4] = 0;  // no candidate yet
  clear_bins<EV_PT>(hist, EV_BINS * EV_COPIES, tid);
  __syncthreads();
  part_rows(a, q, wave, lane, [&](int, uint32_t k, bool live) {
    if (live) atomicAdd(&hist[(k >> 21) * EV_COPIES + (lane & (EV_COPIES - 1))], 1);
  });
  __syncthreads();
  int* const out = a.hists + ((size_t)q.list * a.parts + q.p) * EV_BINS;
  for (int i = tid; i < EV_BINS; i += EV_PT) {
    const u32x4* c = reinterpret_cast<const u32x4*>(hist + i * EV_COPIES);
    const u32x4 x = c[0], y = c[1];
    out[i] = (int)(((x[0] + x[1]) + (x[2] + x[3])) + ((y[0] + y[1]) + (y[2] + y[3])));
  }
}

// The first digit, from the parts' histograms (every workgroup by itself); the
// part's candidates, rows with that digit; and how many movers and free slots
// it has besides.
__global__ __launch_bounds__(EV_PT) void paged_evict_split_kernel(const EvictArgs a) {
  static_assert(EV_BINS == 4 * EV_PT, "four bins a thread");
  __shared__ __align__(16) int hist[EV_BINS];
  __shared__ int wsum[EV_PT / 64], pick[3], total[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Part q;
  if (!part_of(a, &q)) return;
  const u32x4* in = reinterpret_cast<const u32x4*>(a.hists + (size_t)q.list * a.parts * EV_BINS) + tid;
  u32x4 sum = {0u, 0u, 0u, 0u};
  for (int p0 = 0; p0 < q.parts; p0 += 8) {
    u32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = in[(size_t)min(p0 + i, q.parts - 1) * (EV_BINS / 4)];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (p0 + i < q.parts) sum += x[i];
  }
  reinterpret_cast<u32x4*>(hist)[tid] = sum;
  if (tid < 2) total[tid] = 0;
  __syncthreads();
  Search s{0, a.budget, false};
  find_digit<EV_PT, 1>(hist, wsum, pick, 0, tid, &s);
  const uint32_t digit = (uint32_t)(s.limit >> 45);
  int* const head = a.heads + q.list * 4;
  if (q.p == 0 && tid == 0) head[1] = (int)digit, head[2] = s.want, head[3] = s.whole;
  uint2* const out = a.cands + (size_t)q.list * a.parts * a.part;
  int movers = 0, holes = 0, mine = 0;
  part_rows(a, q, wave, lane, [&](int j, uint32_t k, bool live) {
    const uint32_t d = k >> 21;
    movers += __popcll(__ballot(live && d > digit && j >= a.budget));
    holes += __popcll(__ballot(live && d < digit && j < a.budget));
    mine += __popcll(__ballot(live && d == digit));
  });
  if (lane == 0) {
    atomicAdd(&total[0], movers);
    atomicAdd(&total[1], holes);
    wsum[wave] = mine;
  }
  __syncthreads();
  if (tid == 0) {  // room for the part's candidates: one add a workgroup (one a wave and step queued up: 40 us)
    int sum = 0;
#pragma unroll
    for (int w = 0; w < EV_PT / 64; ++w) sum += wsum[w];
    pick[0] = sum ? atomicAdd(head, sum) : 0;
  }
  if (tid < 2) a.counts[((size_t)q.list * a.parts + q.p) * 2 + tid] = total[tid];
  __syncthreads();
  int base = pick[0];
#pragma unroll
  for (int w = 0; w < EV_PT / 64; ++w) base += w < wave ? wsum[w] : 0;
  part_rows(a, q, wave, lane, [&](int j, uint32_t k, bool live) {
    const bool cand = live && k >> 21 == digit;
    const uint64_t m = __ballot(cand);
    if (cand) out[base + lanes_before(m)] = make_uint2(k, (uint32_t)j);
    base += __popcll(m);
  });
}

// Finishes the ranking on the list's candidates, and lists the part's movers
// and free slots behind those of the parts before it.
__global__ __launch_bounds__(EV_PT) void paged_evict_list_kernel(const EvictArgs a) {
  constexpr int HELD = 8;  // candidates a thread holds; more are read again in each pass
  __shared__ __align__(16) int hist[EV_BINS * EV_COPIES];
  __shared__ int wsum[2][EV_PT / 64], pick[3], base_s[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Part q;
  if (!part_of(a, &q)) {
    if (tid == 0 && q.p == 0) a.work[q.list * a.list_ints()] = 0;
    return;
  }
  const int* const head = a.heads + q.list * 4;
  const int cands = head[0];
  Search s{(uint64_t)(uint32_t)head[1] << 45, head[2], head[3] != 0};
  const uint2* const c = a.cands + (size_t)q.list * a.parts * a.part;
  uint2 held[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) held[i] = c[min(tid + i * EV_PT, cands - 1)];
  // f(candidate's rank, slot)
  auto each = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (tid + i * EV_PT < cands) f(rank_of(held[i].x, (int)held[i].y), (int)held[i].y);
    for (int i = tid + HELD * EV_PT; i < cands; i += EV_PT) {
      const uint2 x = c[i];
      f(rank_of(x.x, (int)x.y), (int)x.y);
    }
  };
  if (tid < 2) base_s[tid] = 0;
  for (int i = 1; i < EV_DIGITS && !s.whole; ++i) {
    clear_bins<EV_PT>(hist, EV_BINS * EV_COPIES, tid);
    __syncthreads();
    const int shift = digit_shift(i), done = digit_shift(i - 1);
    const uint32_t mask = digit_mask(i);
    each([&](uint64_t r, int) {
      if ((r >> done) == (s.limit >> done))
        atomicAdd(&hist[((uint32_t)(r >> shift) & mask) * EV_COPIES + (lane & (EV_COPIES - 1))], 1);
    });
    __syncthreads();
    find_digit<EV_PT, EV_COPIES>(hist, wsum[0], pick, i, tid, &s);
  }
  __syncthreads();
  // movers and free slots of the parts before this one
  int mb = 0, hb = 0;
  each([&](uint64_t r, int j) {
    mb += j < q.j0 && r >= s.limit && j >= a.budget;
    hb += j < q.j0 && r < s.limit && j < a.budget;
  });
  const int* const counts = a.counts + (size_t)q.list * a.parts * 2;
  if (tid < q.p) mb += counts[tid * 2], hb += counts[tid * 2 + 1];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) mb += __shfl_xor(mb, o, 64), hb += __shfl_xor(hb, o, 64);
  if (lane == 0) {
    atomicAdd(&base_s[0], mb);
    atomicAdd(&base_s[1], hb);
  }
  // the part's own: counted, then listed
  int* const src = a.work + q.list * a.list_ints() + 1;
  int* const dst = src + a.max_moves;
  int movers = 0, holes = 0;
  part_rows(a, q, wave, lane, [&](int j, uint32_t k, bool live) {
    const bool kept = rank_of(k, j) >= s.limit;
    movers += __popcll(__ballot(live && kept && j >= a.budget));
    holes += __popcll(__ballot(live && !kept && j < a.budget));
  });
  if (lane == 0) wsum[0][wave] = movers, wsum[1][wave] = holes;
  __syncthreads();
  mb = base_s[0], hb = base_s[1];
  int all = mb;
#pragma unroll
  for (int w = 0; w < EV_PT / 64; ++w) {
    if (w < wave) mb += wsum[0][w], hb += wsum[1][w];
    all += wsum[0][w];
  }
  if (q.p == q.parts - 1 && tid == 0) src[-1] = min(all, a.max_moves);
  part_rows(a, q, wave, lane, [&](int j, uint32_t k, bool live) {
    const bool kept = rank_of(k, j) >= s.limit, mover = live && kept && j >= a.budget, hole = live && !kept && j < a.budget;
    const uint64_t mm = __ballot(mover), hm = __ballot(hole);
    const int mi = mb + lanes_before(mm), hi = hb + lanes_before(hm);
    if (mover && mi < a.max_moves) src[mi] = j;
    if (hole && hi < a.max_moves) dst[hi] = j;
    mb += __popcll(mm);
    hb += __popcll(hm);
  });
}

// Moves the listed rows with their scores and positions, D / 8 lanes a row.
template <int D>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(const EvictArgs a) {
  constexpr int LH = D / 8, ROWS = 256 / LH;
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x % LH;
  const int* work = a.work + ((size_t)b * a.c.nkv + h) * a.list_ints();
  const int i = blockIdx.x * ROWS + (int)threadIdx.x / LH;
  if (i >= work[0]) return;
  move_row(a.c, a.c.scores + b * a.c.score_seq + h * a.c.score_head, a.c.slot_pos + b * a.c.pos_seq + h * a.c.pos_head,
           b, h, work[1 + i], work[1 + a.max_moves + i], lane);
}

// How a call is done; the workspace in ints.
struct EvictPlan {
  bool in_parts;
  int max_moves, parts, part;
  size_t lists, heads, counts, hists, cands;
};
inline EvictPlan evict_plan(int seqs, int nkv, long long cap, int budget) {
  EvictPlan p{};
  p.max_moves = (int)(budget < cap - budget ? budget : cap - budget);
  // few rows to move: the ranking workgroup moves them, its keys in registers
  p.in_parts = cap > EV_WHOLE;
  const bool inlined = !p.in_parts && p.max_moves <= EV_INLINE;
  if (inlined) return p;
  const size_t n = (size_t)seqs * nkv;
  p.lists = (n * (1 + 2 * (size_t)p.max_moves) + 3) / 4 * 4;
  if (p.in_parts) {
    const long long part = (cap + EV_PARTS - 1) / EV_PARTS;
    p.part = (int)((part > EV_PART ? part : EV_PART) + EV_PT - 1) / EV_PT * EV_PT;
    p.parts = (int)((cap + p.part - 1) / p.part);
    p.heads = n * 4;
    p.counts = (n * p.parts * 2 + 3) / 4 * 4;
    p.hists = n * p.parts * EV_BINS;
    p.cands = n * p.parts * p.part * 2;
  }
  return p;
}

template <int D>
void launch_evict(const EvictArgs& a, const EvictPlan& p, hipStream_t stream) {
  const dim3 grid(a.c.nkv, a.c.seqs), parts(p.parts, a.c.nkv, a.c.seqs);
  const int cap = a.c.cap();
#define TTSP_EV(TV, INL) hipLaunchKernelGGL((paged_evict_select_kernel<TV, D, INL>), grid, dim3(TV), 0, stream, a)
  if (!p.lists) {
    if (cap <= 256 * 8) TTSP_EV(256, true);
    else TTSP_EV(1024, true);
    return;
  }
  if (p.in_parts) {
    hipLaunchKernelGGL(paged_evict_count_kernel, parts, dim3(EV_PT), 0, stream, a);
    hipLaunchKernelGGL(paged_evict_split_kernel, parts, dim3(EV_PT), 0, stream, a);
    hipLaunchKernelGGL(paged_evict_list_kernel, parts, dim3(EV_PT), 0, stream, a);
  } else if (cap <= 256 * 8) {
    TTSP_EV(256, false);
  } else {
    TTSP_EV(1024, false);
  }
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
  if (seqs > 65535 || nkv > 4096 || cap > TTSP_PAGED_MAX_SLOTS) return -1;
  const EvictPlan p = evict_plan(seqs, nkv, cap, budget);
  const size_t kib = ((p.lists + p.heads + p.counts + p.hists + p.cands) * 4 + 1023) / 1024;
  return kib > 0x7fffffffu ? -1 : (int)kib;
}

extern "C" int ttsp_paged_evict(const ttsp_paged_cache* cache, const long long* SLOT, const long long* POS,
                                int budget, int sinks, int recent, int* work, hipStream_t stream) {
  EvictArgs a{};
  if (!paged_args(cache, &a.c) || !a.c.scores || !a.c.slot_pos || !SLOT || !POS || budget < 1 || sinks < 0 ||
      recent < 0 || sinks > budget - recent)
    return (int)hipErrorInvalidValue;
  const long long cap = a.c.cap();
  if (cap <= budget) return 0;  // no table row holds more than the budget
  a.SLOT = SLOT;
  a.POS = POS;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  const EvictPlan p = evict_plan(a.c.seqs, a.c.nkv, cap, budget);
  if (p.lists && (!work || (uintptr_t)work % 16)) return (int)hipErrorInvalidValue;
  a.max_moves = p.max_moves;
  a.parts = p.parts;
  a.part = p.part;
  a.heads = work + p.lists;
  a.counts = a.heads + p.heads;
  a.hists = a.counts + p.counts;
  a.cands = reinterpret_cast<uint2*>(a.hists + p.hists);
  a.work = work;
  if (cache->head_dim == 128) launch_evict<128>(a, p, stream);
  else launch_evict<64>(a, p, stream);
  TTSP_RETURN_LAUNCH();
}
