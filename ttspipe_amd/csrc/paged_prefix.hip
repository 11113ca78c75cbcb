// Attention of one new token per sequence over a prefix that it shares with other
// sequences, and its own rows: softmax over both of scale q . k, times v. The own
// rows take the kernel of paged_attn.h, which leaves partial sums; the prefixes'
// rows are read here once for all the sequences that share them, and a last launch
// joins both.
//
// A workgroup takes a chunk of a prefix's rows, one kv head, and up to 32 RG query
// rows: that kv head's query heads of some of the sequences that have the prefix, one
// sequence's after the other's (tile_attn.h: the same keys for all of them, where a
// sequence by itself has group rows for a key). The chunks are cut on the device from
// the prefixes' lengths and the number of sequences that have each.
//
// The weights go to the matrix cores in two parts (bf16 within 2^-16, fp16 2^-22); the
// products with V are two then, of three in all. In bf16 that takes 3.6 outputs in a
// thousand a step off the nearest one (32 sequences behind 2011 rows), where three parts,
// which the own rows' weights have, take 0.4, as without a prefix; the error's norm is
// 0.00166 of the output's either way, the output's own rounding. The third part would
// cost 0.3 us there, and 98 in place of 87 us for 64 sequences behind 32763 rows.
// 1000 rows for 256 query rows of each of 8 kv heads take 1.36 us more, 1.16 PFLOP/s of
// the matrix cores' work. 64 sequences behind 32763 rows (32 and 8 heads of 128, bf16;
// own rows through a window of 512): 75 us and 9 for the joining launch, the matrix cores
// busy 37 % of the time: a SIMD has 1.6 waves on average, since the own rows'
// workgroups end first, and they wait 39 % of theirs. Few query rows are bound by
// latency: 32 sequences behind 2011 rows, own 20 to 900: 24 and 6 us, 2.9 TB/s. The own
// rows' workgroups are in the same launch (in one of their own before it 36 us a call in
// place of 30).
#include "tile_attn.h"

namespace ttsp {

constexpr int PF_MAX = 256;   // prefixes of a call (one a thread)
// Workgroups the chunks are meant to make: half a round, as the own rows' run beside them (512
// of them: 86 us in place of 77 for 32763 rows, 36 in place of 33 for five prefixes of 500 to 4000).
constexpr int PF_WGS = 256;
constexpr int PF_PARTS = 2;   // parts of a weight (above)

// Item gx of the call: a chunk of a prefix and a tile of its query rows.
struct Item {
  int p, n;          // prefix (-1: there is no such item) and its rows
  int c, count;      // the chunk, and how many the prefix has
  int tile, tiles;   // the tile, and how many the prefix has
  int first;         // the prefix's first item
  int members;       // sequences that have it
};

// All threads; the result is uniform.
__device__ __forceinline__ Item find_item(const AttnArgs& a, int gx, int tid) {
  __shared__ int cnt[TA_T];
  __shared__ uint32_t sums[TA_WAVES];
  __shared__ int found[6];
  static_assert(PF_MAX <= TA_T, "a thread a prefix");
  const int group = a.nh / a.c.nkv;
  const int all = tid < a.prefixes ? a.far_rows(tid) : 0;  // (asked for before what it waits for)
  cnt[tid] = 0;
  __syncthreads();
  for (int b = tid; b < a.seqs; b += TA_T) {
    const int p = a.OF[b];
    if ((unsigned)p < (unsigned)a.prefixes) atomicAdd(&cnt[p], 1);
  }
  __syncthreads();
  const int m = cnt[tid], n = m ? all : 0;
  const uint32_t tiles = n ? (uint32_t)((m * group + a.far_tile - 1) / a.far_tile) : 0;
  uint32_t total;
  block_prefix(tiles * units(n), sums, tid, &total);
  const uint32_t len = min(max((total + a.far_target - 1) / (uint32_t)a.far_target, 1u), PF_CHUNK / PG_STEP);
  const int count = n ? chunk_count(n, len) : 0;
  const int first = (int)block_prefix(tiles * count, sums, tid, &total);
  Item it{-1, 0, 0, 0, 0, 1, 0, 0};
  if ((uint32_t)gx >= total) return it;
  if (gx >= first && gx < first + (int)tiles * count) {  // one thread
    found[0] = tid, found[1] = n, found[2] = count, found[3] = (int)tiles, found[4] = first, found[5] = m;
  }
  __syncthreads();
  it.p = __builtin_amdgcn_readfirstlane(found[0]);
  it.n = __builtin_amdgcn_readfirstlane(found[1]);
  it.count = __builtin_amdgcn_readfirstlane(found[2]);
  it.tiles = __builtin_amdgcn_readfirstlane(found[3]);
  it.first = __builtin_amdgcn_readfirstlane(found[4]);
  it.members = __builtin_amdgcn_readfirstlane(found[5]);
  it.c = (gx - it.first) / it.tiles;
  it.tile = (gx - it.first) % it.tiles;
  return it;
}

// The sequences' own chunks as the own rows' kernel cuts them, for the joining launch
// (one workgroup).
template <int FORM>
__device__ __forceinline__ void describe(const AttnArgs& a, int tid) {
  __shared__ uint32_t sums[TA_WAVES];
  const int per = (a.seqs + TA_T - 1) / TA_T, b0 = tid * per;
  uint32_t mine = 0, total;
  for (int i = 0; i < per; ++i) mine += units(rows_of<FORM>(a, b0 + i));
  block_prefix(mine, sums, tid, &total);
  const uint32_t len = chunk_len(a, total);
  mine = 0;
  for (int i = 0; i < per; ++i) mine += chunk_count(rows_of<FORM>(a, b0 + i), len);
  int first = (int)block_prefix(mine, sums, tid, &total);
  for (int i = 0; i < per && b0 + i < a.seqs; ++i) {
    const int b = b0 + i, count = chunk_count(rows_of<FORM>(a, b), len), p = a.OF[b];
    a.DESC[b] = make_int4(first, count, (unsigned)p < (unsigned)a.prefixes && a.far_rows(p) > 0, 0);
    first += count;
  }
}

template <int DT, int D, int RG, int FORM>
__global__ __launch_bounds__(TA_T, 2) void paged_prefix_kernel(const AttnArgs a, int items) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Tile<D, RG> C;
  constexpr int QT = 32 * RG;
  __shared__ __align__(256) uint8_t ring0[C::STAGE];
  __shared__ __align__(256) uint8_t ring1[C::STAGE];
  __shared__ int seq_s[QT + 2], wcnt[TA_WAVES];
  __shared__ __align__(16) unsigned long long run_s[PF_CHUNK / 16][2];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.nh / a.c.nkv, h = blockIdx.x % a.c.nkv, gx = blockIdx.x / a.c.nkv;
  if ((int)blockIdx.x >= items) {
    const int i = blockIdx.x - items;
    if (i == 0) {
      describe<FORM>(a, tid);
      return;
    }
    __shared__ AttnLds<D> sh;  // the sequences' own rows
    const int wide = a.c.nkv * ((group + PG_HEADS - 1) / PG_HEADS);
    static_assert(PG_T == TA_T && PG_WAVES * AttnLds<D>::REGION <= C::STAGE, "the same waves, and their V rows in a stage");
    attend_chunk<DT, D, FORM>(a, (i - 1) / wide, (i - 1) % wide, tid, ring0, sh);
    return;
  }
  const Item it = find_item(a, gx, tid);
  if (it.p < 0) return;
  const int row0 = it.tile * QT, rows = min(QT, it.members * group - row0);

  // the tile's sequences: the o0-th of the prefix's to the one before the o1-th
  const int o0 = row0 / group, o1 = (row0 + rows - 1) / group + 1;
  for (int b0 = 0, before = 0; b0 < a.seqs && before < o1; b0 += TA_T) {
    const int b = b0 + tid;
    const bool has = b < a.seqs && a.OF[b] == it.p;
    const unsigned long long bits = __ballot(has);
    if (lane == 0) wcnt[wave] = __popcll(bits);
    __syncthreads();
    int at = before + __popcll(bits & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < TA_WAVES; ++w) {
      at += w < wave ? wcnt[w] : 0;
      before += wcnt[w];
    }
    if (has && at >= o0 && at < o1) seq_s[at - o0] = b;
    __syncthreads();
  }
  if (it.c == 0 && h == 0)  // for the joining launch: where a sequence's parts are
    for (int i = tid; i < o1 - o0; i += TA_T)
      if ((o0 + i) * group >= row0)
        a.DESC[a.seqs + seq_s[i]] = make_int4(it.first, it.count, it.tiles, (o0 + i) * group);

  const int rg = wave % RG, kg = wave / RG;
  const int myrow = 32 * rg + (lane & 31);  // this lane's query row of the tile
  TaWave<DT, D, PF_PARTS> w;
  w.init(lane);
  {
    const int r = row0 + min(myrow, rows - 1);  // (rows past the tile's: its last one's, not written)
    const uint16_t* const q = a.Q + seq_s[r / group - o0] * a.q_seq + (size_t)(h * group + r % group) * D + 8 * (lane >> 5);
    const uint32_t flip = a.scale2 < 0.0f ? 0x80008000u : 0u;  // (a negative scale: -q and its absolute value)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) w.q[i] = *reinterpret_cast<const u32x4*>(q + 16 * i) ^ flip;
  }
  const float scale2 = a.scale2 == 0.0f ? 1e-30f : fabsf(a.scale2);  // (0: -inf times it is to stay so)

  const int size = chunk_size(it.n, it.count), k0 = min(it.c * size, it.n), k1 = min(k0 + size, it.n);
  // Where the chunk's runs of 16 rows lie (bit 0 of V's address: a hole, for which page 0's are read).
  const int mask = (1 << a.c.shift) - 1, runs = (k1 - k0 + 15) / 16;
  bool holes = false;
  for (int i = tid; i < runs; i += TA_T) {
    const int j = k0 + 16 * i, page = a.far_table[it.p * a.far_stride + (j >> a.c.shift)];
    const bool hole = (unsigned)page >= (unsigned)a.c.pages;
    const long long q = hole ? 0 : page, r = j & mask;
    run_s[i][0] = (unsigned long long)(a.c.K + q * a.c.k_page + h * a.c.k_head + r * a.c.k_row);
    run_s[i][1] = (unsigned long long)(a.c.V + q * a.c.v_page + h * a.c.v_head + r * a.c.v_row) | hole;
    holes = holes || hole;
  }
  holes = __syncthreads_or(holes);
  // this wave's loads of a tile: PER of RPI rows from row PER RPI wave on, all in one run
  uint32_t ko[C::PER], vo[C::PER];
#pragma unroll
  for (int i = 0; i < C::PER; ++i) {
    const int lrow = lane / C::PPR, row = (wave * C::PER + i) * C::RPI;
    const int piece = (lane % C::PPR) ^ ta_swz<D>(row + lrow);
    ko[i] = (uint32_t)((row % 16 + lrow) * (int)a.c.k_row) * 2 + piece * 16;
    vo[i] = (uint32_t)((row % 16 + lrow) * (int)a.c.v_row) * 2 + piece * 16;
  }
  static_assert(C::PER * C::RPI <= 16, "a wave's rows of a tile lie in one run");
  const int lr0 = wave * C::PER * C::RPI, last = max(runs - 1, 0);
  auto run_at = [&](int t) { return *reinterpret_cast<const u32x4*>(run_s[min((t * C::KEYS + lr0) / 16, last)]); };
  u32x4 next = run_at(0);  // (asked for a tile ahead)
  auto load = [&](int t, uint8_t* ring) {
    uint32_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = __builtin_amdgcn_readfirstlane(next[i]);
    const void* const kp = (const void*)((unsigned long long)at[1] << 32 | at[0]);
    const void* const vp = (const void*)((unsigned long long)at[3] << 32 | (at[2] & ~1u));
#pragma unroll
    for (int i = 0; i < C::PER; ++i) {
      ta_load(kp, ko[i], ring + (wave * C::PER + i) * 1024);
      ta_load(vp, vo[i], ring + C::HALF + (wave * C::PER + i) * 1024);
    }
    next = run_at(t + 1);
  };
  auto hole_at = [&](int r) { return holes && (run_s[min(r / 16, last)][1] & 1); };  // row r of the chunk
  const int n = k1 - k0;
  // V rows that are no keys are zeros (what they hold may be NaN)
  auto landed = [&](int t, uint8_t* ring) {
    const int r0 = t * C::KEYS + lr0;
    if (!holes && r0 + C::PER * C::RPI <= n) return;
    const bool hole = hole_at(r0);
#pragma unroll
    for (int i = 0; i < C::PER; ++i)
      if (hole || r0 + i * C::RPI + lane / C::PPR >= n)
        *reinterpret_cast<u32x4*>(ring + C::HALF + (wave * C::PER + i) * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
  };
  bool seen = false;
  auto compute = [&](int t, uint8_t* ring) {
    const int row = 32 * C::SB * kg, r0 = t * C::KEYS + row;
    if (r0 >= n) return;
    uint32_t gone = 0;  // the holes among its runs of 16 rows
    if (holes)
      for (int i = 0; i < 2 * C::SB; ++i) {
        const bool hole = hole_at(r0 + 16 * i);
        gone |= hole << i;
        seen = seen || (!hole && r0 + 16 * i < n);
      }
    else
      seen = true;
    w.template run<C::SB>(ring + row * C::ROWB, ring + C::HALF + row * C::ROWB, scale2, gone || r0 + 32 * C::SB > n, n - 1 - r0, 0,
                          0, gone);
  };
#pragma unroll
  for (int i = 0; i < D / 16; ++i) asm volatile("" ::"v"(w.q[i]));  // (waited for here, not among the loop's loads)
  ta_tiles<C>((n + C::KEYS - 1) / C::KEYS, ring0, ring1, load, landed, compute);
  ta_join<C>(w, seen, ring0, ring1, rg, kg, lane);

  if (kg == 0 && myrow < rows) {
    const size_t at = a.far_base + ((size_t)gx * a.c.nkv + h) * QT + myrow;
    const int h4 = 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(a.PACC + at * D + 32 * d + 8 * g + h4) =
            f32x4{w.o[d][4 * g], w.o[d][4 * g + 1], w.o[d][4 * g + 2], w.o[d][4 * g + 3]};
    if (lane < 32) {
      a.PM[at] = w.m;
      a.PL[at] = seen ? w.l : -1.0f;
    }
  }
#endif
}

// How the prefixes' part of a call is cut up; false where it is more than is counted.
struct PrefixPlan {
  int tile, target, items;
  size_t rows;  // of partial sums
};
inline bool prefix_plan(int seqs, int nh, int nkv, int prefixes, long long far_cap, PrefixPlan* p) {
  const long long group = nh / nkv, rows = seqs * group;
  p->tile = rows <= 64 ? 64 : 128;
  p->target = nkv < PF_WGS ? PF_WGS / nkv : 1;
  // each prefix that a sequence has may end with a tile that is not full
  const long long tiles = rows / p->tile + (prefixes < seqs ? prefixes : seqs);
  const long long units = (far_cap + PG_STEP - 1) / PG_STEP;
  if (tiles * units > 0x3fffffff) return false;
  // chunks of the length that makes `target` of them, or of the longest
  const long long most = tiles + (p->target > tiles * units / (PF_CHUNK / PG_STEP) ? p->target : tiles * units / (PF_CHUNK / PG_STEP));
  const long long items = most < tiles * units ? most : tiles * units;
  if (items * nkv > PG_MAX_GRID) return false;
  p->items = (int)items;
  p->rows = (size_t)items * nkv * p->tile;
  return true;
}

}  // namespace ttsp

using namespace ttsp;

// The workspace: own and prefix rows of partial sums, the sequences' places in the
// latter, scores; in floats, false where there is no such call.
struct PrefixWork {
  AttnPlan own;
  PrefixPlan far;
  size_t rows, desc, scores, total;
};
static bool prefix_work(int seqs, int nh, int nkv, int hd, long long cap, long long rows, int prefixes, long long far_cap,
                        bool tracked, PrefixWork* w) {
  if (!attn_plan(seqs, nh, nkv, hd, cap, rows, tracked, true, &w->own) ||
      !prefix_plan(seqs, nh, nkv, prefixes, far_cap, &w->far) ||
      (long long)w->far.items * nkv + 1 + (long long)w->own.chunks * nkv * w->own.hgs > PG_MAX_GRID)
    return false;
  w->rows = (size_t)w->own.chunks * nh + w->far.rows;
  w->desc = (w->rows * (2 + hd) + 3) / 4 * 4;
  w->scores = w->desc + (size_t)seqs * 8;
  w->total = w->scores + w->own.scores;
  return (w->total + 255) / 256 <= 0x7fffffff;
}

extern "C" int ttsp_paged_attention_prefix_work_kib(int seqs, int nh, int nkv, int head_dim, int cols, int page_size,
                                                    int prefixes, int prefix_cols, int window, int sinks, int tracked) {
  if (seqs < 1 || nkv < 1 || nh < nkv || cols < 1 || page_size < 1 || head_dim < 1 || prefixes < 1 || prefix_cols < 1 ||
      window < 0 || sinks < 0)
    return -1;
  PrefixWork w;
  const long long cap = (long long)cols * page_size, far_cap = (long long)prefix_cols * page_size;
  if (seqs > 65535 || nh > 65535 || nkv > 4096 || head_dim > 128 || cap > TTSP_PAGED_MAX_SLOTS ||
      far_cap > TTSP_PAGED_MAX_SLOTS || prefixes > PF_MAX ||
      !prefix_work(seqs, nh, nkv, head_dim, cap, window ? window_rows(cap, window, sinks) : cap, prefixes, far_cap,
                   tracked != 0, &w))
    return -1;
  return (int)((w.total + 255) / 256);
}

template <int FORM>
static int prefix_launch(const AttnArgs& a, const PrefixWork& w, int hd, int dtype, hipStream_t stream) {
  const int items = w.far.items * a.c.nkv;
  const dim3 grid((unsigned)(items + 1 + w.own.chunks * a.c.nkv * w.own.hgs));
  const int gathers = w.own.chunks * a.c.nkv;
#define TTSP_PFX(DTV, DV)                                                                                              \
  do {                                                                                                                 \
    if (w.far.tile == 64) hipLaunchKernelGGL((paged_prefix_kernel<DTV, DV, 2, FORM>), grid, dim3(TA_T), 0, stream, a, items);         \
    else hipLaunchKernelGGL((paged_prefix_kernel<DTV, DV, 4, FORM>), grid, dim3(TA_T), 0, stream, a, items);            \
    if (FORM & PG_TRACK)                                                                                               \
      hipLaunchKernelGGL((paged_gather_kernel<DTV, DV, FORM>), dim3(gathers + a.seqs * a.nh), dim3(256), 0, stream, a,  \
                         gathers);                                                                                     \
    else                                                                                                               \
      hipLaunchKernelGGL((paged_join_kernel<DTV, DV, FORM>), dim3(a.nh, a.seqs), dim3(256), 0, stream, a);              \
  } while (0)
  if (dtype == DT_F16) {
    if (hd == 128) TTSP_PFX(DT_F16, 128);
    else TTSP_PFX(DT_F16, 64);
  } else {
    if (hd == 128) TTSP_PFX(DT_BF16, 128);
    else TTSP_PFX(DT_BF16, 64);
  }
#undef TTSP_PFX
  TTSP_RETURN_LAUNCH();
}

extern "C" int ttsp_paged_attention_prefix(const ttsp_paged_cache* cache, const ttsp_paged_prefix* prefix, const void* Q,
                                           long long q_seq_stride, const long long* SLOT, void* Y, int nh, float scale,
                                           int window, int sinks, float* work, hipStream_t stream) {
  AttnArgs a{};
  PrefixWork w;
  if (!paged_args(cache, &a.c) || !Q || !SLOT || !Y || nh < 1 || nh > 65535 || nh % a.c.nkv || (uintptr_t)Q % 16 ||
      (uintptr_t)Y % 16 || q_seq_stride % 8 || q_seq_stride < (long long)nh * cache->head_dim || window < 0 || sinks < 0)
    return (int)hipErrorInvalidValue;
  if (!prefix || !prefix->table || !prefix->SLOT || !prefix->OF || (uintptr_t)prefix->table % 4 ||
      (uintptr_t)prefix->SLOT % 8 || (uintptr_t)prefix->OF % 4 || prefix->count < 1 || prefix->count > PF_MAX ||
      prefix->cols < 1 || prefix->table_stride < prefix->cols ||
      (long long)prefix->cols * cache->page_size > TTSP_PAGED_MAX_SLOTS)
    return (int)hipErrorInvalidValue;
  const int hd = cache->head_dim, cap = a.c.cap();
  const bool tracked = a.c.scores != nullptr;
  if (window) {
    a.window = window < cap ? window : cap;
    a.sinks = sinks < cap ? sinks : cap;
  }
  if (!prefix_work(a.c.seqs, nh, a.c.nkv, hd, cap, window ? window_rows(cap, a.window, a.sinks) : cap, prefix->count,
                   (long long)prefix->cols * cache->page_size, tracked, &w) ||
      !work || (uintptr_t)work % 16)
    return (int)hipErrorInvalidValue;
  a.Q = (const uint16_t*)Q;
  a.q_seq = q_seq_stride;
  a.SLOT = SLOT;
  a.Y = (uint16_t*)Y;
  a.PACC = work;
  a.PM = work + w.rows * hd;
  a.PL = a.PM + w.rows;
  a.DESC = reinterpret_cast<int4*>(work + w.desc);
  a.S = tracked ? work + w.scores : nullptr;
  a.scale2 = scale * 1.4426950408889634f;
  a.nh = nh;
  a.seqs = a.c.seqs;
  a.target = w.own.target;
  a.far_table = prefix->table;
  a.far_stride = prefix->table_stride;
  a.FAR_SLOT = prefix->SLOT;
  a.OF = prefix->OF;
  a.prefixes = prefix->count;
  a.far_cols = prefix->cols;
  a.far_target = w.far.target;
  a.far_tile = w.far.tile;
  a.far_base = (size_t)w.own.chunks * nh;
  if (window)
    return tracked ? prefix_launch<PG_PREFIX | PG_WINDOW | PG_TRACK>(a, w, hd, cache->dtype, stream)
                   : prefix_launch<PG_PREFIX | PG_WINDOW>(a, w, hd, cache->dtype, stream);
  return tracked ? prefix_launch<PG_PREFIX | PG_TRACK>(a, w, hd, cache->dtype, stream)
                 : prefix_launch<PG_PREFIX>(a, w, hd, cache->dtype, stream);
}
