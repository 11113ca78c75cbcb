// Attention of one new token per sequence over a prefix that it shares with other
// sequences, and its own rows: softmax over both of scale q . k, times v. The own
// rows take the kernel of paged_attn.h, which leaves partial sums; the prefixes'
// rows are read here once for all the sequences that share them, and a last launch
// joins both.
//
// A workgroup takes a chunk of a prefix's rows, one kv head, and 16 T query rows:
// the query heads of the kv head of T 16 / group sequences that have the prefix.
// The same rows for every column of the matrix cores' tiles: that is a matrix
// product with 16 T columns where a sequence by itself has group of them. Four waves
// each take every fourth run of 32 rows as in paged_attn.h, each with all the
// workgroup's query rows, so every row of K and V goes from memory into one wave's
// registers, and once through its LDS to be transposed, for 16 T query rows.
#include "paged_attn.h"

namespace ttsp {

constexpr int PF_MAX = 256;   // prefixes of a call (one a thread)
constexpr int PF_WGS = 512;   // workgroups the chunks are meant to make

// Item gx of the call: a chunk of a prefix and a tile of its query rows.
struct Item {
  int p, n;          // prefix (-1: there is no such item) and its rows
  int c, count;      // the chunk, and how many the prefix has
  int tile, tiles;   // the tile, and how many the prefix has
  int first;         // the prefix's first item
  int members;       // sequences that have it
};

// All 256 threads; the result is uniform.
__device__ __forceinline__ Item find_item(const AttnArgs& a, int gx, int tid) {
  __shared__ int cnt[PF_MAX];
  __shared__ uint32_t sums[PG_T / 64];
  __shared__ int found[8];
  const int group = a.nh / a.c.nkv;
  cnt[tid] = 0;
  __syncthreads();
  for (int b = tid; b < a.seqs; b += PG_T) {
    const int p = a.OF[b];
    if ((unsigned)p < (unsigned)a.prefixes) atomicAdd(&cnt[p], 1);
  }
  __syncthreads();
  const int m = cnt[tid], n = m ? a.far_rows(tid) : 0;
  const uint32_t tiles = n ? (uint32_t)((m * group + a.far_tile - 1) / a.far_tile) : 0;
  uint32_t total;
  block_prefix(tiles * units(n), sums, tid, &total);
  const uint32_t len = max((total + a.far_target - 1) / (uint32_t)a.far_target, 1u);
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

template <int DT, int D, int T>
__global__ __launch_bounds__(64 * PG_WAVES, 2) void paged_prefix_kernel(const AttnArgs a) {
  constexpr int QT = 16 * T;                    // query rows of the workgroup
  constexpr int QROW = D + 8;                   // their stride in LDS (elements)
  constexpr int KC = D / 32, DC = D / 16, VPL = PG_KEYS * D * 2 / 1024, VR = 1024 / (D * 2);
  constexpr int REGION = PG_KEYS * D * 2;       // a wave's LDS: V rows, at the end 16 fp32 rows of O
  __shared__ __align__(16) uint8_t lds[PG_WAVES * REGION];
  __shared__ __align__(16) uint16_t qs[QT * QROW];
  __shared__ float m_s[PG_WAVES][16], l_s[PG_WAVES][16];
  __shared__ int seq_s[QT + 2], wcnt[PG_WAVES];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int group = a.nh / a.c.nkv, h = blockIdx.x % a.c.nkv, gx = blockIdx.x / a.c.nkv;
  const Item it = find_item(a, gx, tid);
  if (it.p < 0) return;
  const int row0 = it.tile * QT, rows = min(QT, it.members * group - row0);

  // the tile's sequences: the o0-th of the prefix's to the one before the o1-th
  const int o0 = row0 / group, o1 = (row0 + rows - 1) / group + 1;
  for (int b0 = 0, before = 0; b0 < a.seqs && before < o1; b0 += PG_T) {
    const int b = b0 + tid;
    const bool has = b < a.seqs && a.OF[b] == it.p;
    const unsigned long long bits = __ballot(has);
    if (lane == 0) wcnt[wave] = __popcll(bits);
    __syncthreads();
    int at = before + __popcll(bits & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) {
      at += w < wave ? wcnt[w] : 0;
      before += wcnt[w];
    }
    if (has && at >= o0 && at < o1) seq_s[at - o0] = b;
    __syncthreads();
  }
  if (it.c == 0 && h == 0)  // for the joining launch: where a sequence's parts are
    for (int i = tid; i < o1 - o0; i += PG_T)
      if ((o0 + i) * group >= row0)
        a.DESC[seq_s[i]] = make_int4(it.first, it.count, it.tiles, (o0 + i) * group);
  for (int i = tid; i < QT * (D / 8); i += PG_T) {
    const int r = i / (D / 8), e = (i % (D / 8)) * 8;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (r < rows)
      v = *reinterpret_cast<const u32x4*>(a.Q + seq_s[(row0 + r) / group - o0] * a.q_seq +
                                          (size_t)(h * group + (row0 + r) % group) * D + e);
    *reinterpret_cast<u32x4*>(qs + r * QROW + e) = v;
  }
  __syncthreads();

  const int size = chunk_size(it.n, it.count), k0 = it.c * size, k1 = min(k0 + size, it.n);
  const int mask = (1 << a.c.shift) - 1;
  const int* const trow = a.far_table + it.p * a.far_stride;
  auto page_at = [&](int j) {
    const int p = j < k1 ? trow[j >> a.c.shift] : -1;
    return (unsigned)p < (unsigned)a.c.pages ? p : -1;
  };
  uint8_t* const vs = lds + wave * REGION;
  const uint32_t ko = (uint32_t)(lr * (int)a.c.k_row + 8 * lg) * 2;
  const uint32_t vo = (uint32_t)((lane / (64 / VR)) * (int)a.c.v_row + (lane % (64 / VR)) * 8) * 2;
  u32x4 kf[2][KC], vf[VPL];
  auto load = [&](int j, int p0, int p1) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int p = max(s ? p1 : p0, 0), row = (j + 16 * s) & mask;
      const uint8_t* kb = (const uint8_t*)(a.c.K + p * a.c.k_page + h * a.c.k_head + row * a.c.k_row);
#pragma unroll
      for (int i = 0; i < KC; ++i) kf[s][i] = *reinterpret_cast<const u32x4*>(kb + 64 * i + ko);
      const uint8_t* vb = (const uint8_t*)(a.c.V + p * a.c.v_page + h * a.c.v_head + row * a.c.v_row);
#pragma unroll
      for (int i = 0; i < VPL / 2; ++i)
        vf[s * (VPL / 2) + i] = *reinterpret_cast<const u32x4*>(vb + (size_t)i * VR * a.c.v_row * 2 + vo);
    }
  };
  auto vaddr = [&](int row, int blk) {
    const int sw = D == 128 ? row & 7 : (row >> 1) & 3;
    return row * (D * 2) + ((blk ^ sw) << 5);
  };

  f32x4 o[T][DC];
  float mref[T], lsum[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    mref[t] = PG_NONE, lsum[t] = 0.0f;
#pragma unroll
    for (int d = 0; d < DC; ++d) o[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  bool seen = false;

  int j = k0 + PG_KEYS * wave;
  int p0 = page_at(j), p1 = page_at(j + 16);
  if (j < k1) load(j, p0, p1);
  int n0 = page_at(j + PG_STEP), n1 = page_at(j + PG_STEP + 16);
  for (; j < k1; j += PG_STEP) {
    const bool whole = j + PG_KEYS <= k1 && p0 >= 0 && p1 >= 0;
    seen = seen || p0 >= 0 || p1 >= 0;
    f32x4 s[T][2];
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
      for (int u = 0; u < 2; ++u) s[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const u32x4 qf = *reinterpret_cast<const u32x4*>(qs + (16 * t + lr) * QROW + 32 * i + 8 * lg);
#pragma unroll
        for (int u = 0; u < 2; ++u) s[t][u] = pg_mfma<DT>(kf[u][i], qf, s[t][u]);
      }
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int row = i * VR + lane / (64 / VR), c16 = lane % (64 / VR);
      *reinterpret_cast<u32x4*>(vs + vaddr(row, c16 >> 1) + (c16 & 1) * 16) = vf[i];
    }
    if (!whole) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int row = i * VR + lane / (64 / VR), c16 = lane % (64 / VR);
        if (j + row >= k1 || (row < 16 ? p0 : p1) < 0)
          *reinterpret_cast<u32x4*>(vs + vaddr(row, c16 >> 1) + (c16 & 1) * 16) = u32x4{0u, 0u, 0u, 0u};
      }
    }
    const int c0 = p0, c1 = p1;
    p0 = n0, p1 = n1;
    if (j + PG_STEP < k1) load(j + PG_STEP, p0, p1);
    n0 = page_at(j + 2 * PG_STEP), n1 = page_at(j + 2 * PG_STEP + 16);

    u32x4 pf[T][pg_parts<DT>];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      bool over = false;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = s[t][u][r] * a.scale2;
          if (!whole && (j + 16 * u + 4 * lg + r >= k1 || (u ? c1 : c0) < 0)) x = -__builtin_inff();
          s[t][u][r] = x;
          over = over || x > mref[t] + pg_above<DT>;
        }
      if (__any(over)) {
        float bm = fmaxf(fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3])),
                         fmaxf(fmaxf(s[t][1][0], s[t][1][1]), fmaxf(s[t][1][2], s[t][1][3])));
        bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
        bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
        const float mnew = bm > mref[t] + pg_above<DT> ? bm - pg_below<DT> : mref[t];
        const float alpha = __builtin_amdgcn_exp2f(mref[t] - mnew);
        mref[t] = mnew;
        lsum[t] *= alpha;
#pragma unroll
        for (int d = 0; d < DC; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[t][d][r] *= alpha;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = __builtin_amdgcn_exp2f(s[t][u][r] - mref[t]);
          lsum[t] += p[r];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t parts[pg_parts<DT>];
          pg_split<DT>(p[2 * r], p[2 * r + 1], parts);
#pragma unroll
          for (int i = 0; i < pg_parts<DT>; ++i) pf[t][i][2 * u + r] = parts[i];
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int d = 0; d < DC; ++d) {
      const int row = 4 * lg + (lr >> 2);
      const uint2 lo = pg_ld_tr(vs + vaddr(row, d) + 8 * (lr & 3));
      const uint2 hi = pg_ld_tr(vs + vaddr(row + 16, d) + 8 * (lr & 3));
      const u32x4 vt = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int i = 0; i < pg_parts<DT>; ++i) o[t][d] = pg_mfma<DT>(vt, pf[t][i], o[t][d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  // the waves' parts, 16 query rows at a time
  float* const os = reinterpret_cast<float*>(vs);
  const float* const all = reinterpret_cast<const float*>(lds);
  const size_t out0 = a.far_base + ((size_t)gx * a.c.nkv + h) * QT;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    float l = lsum[t];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < 16) {
      m_s[wave][lane] = mref[t];
      l_s[wave][lane] = seen ? l : -1.0f;
    }
#pragma unroll
    for (int d = 0; d < DC; ++d) *reinterpret_cast<f32x4*>(os + lr * D + 16 * d + 4 * lg) = o[t][d];
    __syncthreads();
    for (int i = tid; i < min(16, rows - 16 * t) * D; i += PG_T) {
      const int g = i / D, d = i % D;
      float m = PG_NONE;
#pragma unroll
      for (int w = 0; w < PG_WAVES; ++w) m = fmaxf(m, m_s[w][g]);
      float num = 0.0f, den = 0.0f;
      bool any = false;
#pragma unroll
      for (int w = 0; w < PG_WAVES; ++w) {
        const float lw = l_s[w][g], e = __builtin_amdgcn_exp2f(m_s[w][g] - m);
        const bool none = lw < 0.0f;
        den += (none ? 0.0f : lw) * e;
        num += all[(size_t)w * (REGION / 4) + g * D + d] * e;
        any = any || !none;
      }
      const size_t at = out0 + 16 * t + g;
      a.PACC[at * D + d] = num;
      if (d == 0) {
        a.PM[at] = m;
        a.PL[at] = any ? den : -1.0f;
      }
    }
    __syncthreads();
  }
}

// How the prefixes' part of a call is cut up; false where it is more than is counted.
struct PrefixPlan {
  int tile, target, items;
  size_t rows;  // of partial sums
};
inline bool prefix_plan(int seqs, int nh, int nkv, int prefixes, long long far_cap, PrefixPlan* p) {
  const long long group = nh / nkv, rows = seqs * group;
  p->tile = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  p->target = nkv < PF_WGS ? PF_WGS / nkv : 1;
  // each prefix that a sequence has may end with a tile that is not full
  const long long tiles = rows / p->tile + (prefixes < seqs ? prefixes : seqs);
  const long long units = (far_cap + PG_STEP - 1) / PG_STEP;
  if (tiles * units > 0x3fffffff) return false;
  const long long items = p->target + tiles < tiles * units ? p->target + tiles : tiles * units;
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
      !prefix_plan(seqs, nh, nkv, prefixes, far_cap, &w->far))
    return false;
  w->rows = (size_t)w->own.chunks * nh + w->far.rows;
  w->desc = (w->rows * (2 + hd) + 3) / 4 * 4;
  w->scores = w->desc + (size_t)seqs * 4;
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
  const dim3 far((unsigned)(w.far.items * a.c.nkv)), own((unsigned)(w.own.chunks * a.c.nkv * w.own.hgs));
  const int gathers = w.own.chunks * a.c.nkv;
#define TTSP_PFX(DTV, DV)                                                                                              \
  do {                                                                                                                 \
    if (w.far.tile == 16) hipLaunchKernelGGL((paged_prefix_kernel<DTV, DV, 1>), far, dim3(PG_T), 0, stream, a);         \
    else if (w.far.tile == 32) hipLaunchKernelGGL((paged_prefix_kernel<DTV, DV, 2>), far, dim3(PG_T), 0, stream, a);    \
    else hipLaunchKernelGGL((paged_prefix_kernel<DTV, DV, 4>), far, dim3(PG_T), 0, stream, a);                          \
    hipLaunchKernelGGL((paged_attn_kernel<DTV, DV, FORM>), own, dim3(64 * PG_WAVES), 0, stream, a);                     \
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
