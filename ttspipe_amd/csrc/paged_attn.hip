// Attention of one new token per sequence over a paged key-value cache:
//   s_j = scale q . k_j over the sequence's slots j with a page,
//   y = sum_j p_j v_j,  p = softmax(s),
// query head h reading kv head h / (nh / nkv); a sequence without a row gives
// zeros. With scores, sum over the kv head's query heads of p_j is added to
// the sequence's score of slot j.
//
// Memory bound: every cached row is read once for all the query heads of its
// kv head (G = nh / nkv flop a byte), so what counts is how many bytes are under
// way at once. One sequence of 130995 rows (8 kv heads of 128): the first launch
// 84 us, 6.4 TB/s, the rate of a plain streaming read; 64 of 2048 to 5119: 163 us,
// 5.8 TB/s; 32 of 200 to 2304, where a workgroup has only three rounds between its
// first dependent reads and its merge: 36 us, 4.7 TB/s. Cached rows are read past
// the caches (plain loads: 97 and 181 us for the first two).
//
// The work. The sequences' rows are cut into chunks of about equal length,
// enough of them to fill the GPU whatever the batch looks like (one long
// sequence, many short ones): each workgroup reads all the slots, adds up the
// rows, derives the chunk length and finds its own (sequence, chunk), so the
// split follows the lengths on the device and a captured call keeps working as
// they grow. Workgroup = (chunk, kv head or 16 of its query heads), four waves
// that each take every fourth run of 32 keys and merge at the end; chunks of a
// sequence join in a second launch. A sequence of one chunk is finished in the
// first. A chunk's kv heads are neighbouring workgroups: their rows are
// neighbours in the pages (171 against 167 us for 64 sequences of 2048 to 5119
// rows where its chunks were, 43.5 against 41.2 for 32 of 200 to 2304).
//
// A wave's 32 keys: S^T = K Q^T on the matrix cores (16 keys x 16 query heads a
// tile; K straight from memory into the operand's layout, Q^T stays in
// registers), so a lane holds 8 keys of one query head. The exponentials
// subtract a reference that moves only when a score outgrows it (pg_above), so the
// running maximum needs no exchange between lanes but a vote. P^T goes to the
// matrix cores in parts of the cache's type: bf16 in three, which hold a weight
// whole, fp16 in two, together within 2^-22 of it; the sums stay in fp32. (bf16 in
// two parts, within 2^-16: 300 rows of one sequence 8.0 against 8.3 us, the larger
// calls the same within 1 %; one output in a thousand off by a step.) It feeds
// O^T += V^T P^T from the registers it is in: the contraction takes the keys in the order the score
// tiles hold them, and V^T comes from V's rows in LDS through the transposing
// read. Each wave has its own 32 rows of LDS and never waits for another. K and
// V rows of the next 32 keys are loaded while these are computed.
//
// MFMA 16x16x32: lane l supplies row (l % 16) of A and column (l % 16) of B at
// k = 8 (l / 16) .. + 7; accumulator r of lane l is D[4 (l / 16) + r][l % 16].
#include "paged_common.h"

namespace ttsp {

typedef __bf16 pg_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_f16x8 __attribute__((ext_vector_type(8)));
typedef short pg_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pg_s16x4 pg_lds_s16x4;

constexpr int PG_WAVES = 4, PG_KEYS = 32;      // waves a workgroup, keys a wave takes at once
constexpr int PG_STEP = PG_WAVES * PG_KEYS;    // chunk lengths are multiples of this
// Workgroups the chunks are meant to make, two rounds of the two that fit a CU.
// Per call, 1024 / 1536 / 2048 of them: 32 sequences of 200 to 2304 rows 41.1 / 42.2 /
// 42.5 us; 64 of 2048 to 5119 167 / 166 / 165; one of 130995 90 / 96 / 96 (32 query
// and 8 kv heads of 128, bf16; 512 of them, one round: 49 / 200 / 88).
constexpr int PG_WGS = 1024;
// Caches of up to this many slots: a sequence is one chunk, and there is no
// joining launch (300 rows, alone: 8.3 us; in three chunks and joined: 10.2).
constexpr int PG_SHORT = 512;
constexpr int PG_HEADS = 16;                   // query heads a workgroup takes
constexpr float PG_NONE = -3.0e38f;            // the reference before any score
// A moved reference lies `pg_below` under the largest score and moves again when a
// score is `pg_above` over it. bf16 weights have room on both sides. fp16 ones end
// at 2^-24: a largest weight of 2^13 to 2^15 lets those 2^-38 of it count, where one
// of 1 to 2^8 would round a long tail of weights around 2^-24 to 0 or to double.
template <int DT> constexpr float pg_below = DT == DT_F16 ? 13.0f : 0.0f;
template <int DT> constexpr float pg_above = DT == DT_F16 ? 15.0f : 8.0f;

struct AttnArgs {
  Paged c;
  const uint16_t* Q;  // [seqs][nh][D] by q_seq
  long long q_seq;
  const long long* SLOT;
  uint16_t* Y;   // [seqs][nh][D]
  float* PM;     // [chunks][nh]: the chunk's reference (log2 units)
  float* PL;     // [chunks][nh]: its sum of exp2(s - reference), -1: no key seen
  float* PACC;   // [chunks][nh][D]: its sum of exp2(s - reference) v
  float* S;      // scores in log2 units [seqs][nh][cap] (with scores to gather)
  float scale2;  // scale * log2(e)
  int nh, seqs, target;  // target: chunks that fill the GPU (0: chunk b is the whole sequence b)
};

template <int DT>
__device__ __forceinline__ f32x4 pg_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == DT_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf16x8, a), __builtin_bit_cast(pg_bf16x8, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_f16x8, a), __builtin_bit_cast(pg_f16x8, b), c, 0,
                                                  0, 0);
}

// 16-bit parts a weight goes to the matrix cores in.
template <int DT> constexpr int pg_parts = DT == DT_F16 ? 2 : 3;

// Two weights (not negative) as packed pairs of DT. bf16: three parts of eight
// bits each, their sum the weight itself (the lower ones are kept above 0, so that
// a weight's parts times an infinite value have one sign). fp16: what it holds of
// the weight, rounded towards zero, and the rest, rounded to nearest, together
// within 2^-22 of it.
template <int DT>
__device__ __forceinline__ void pg_split(float p, float q, uint32_t* parts) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == DT_BF16) {
    constexpr float least = 1.17549435e-38f;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t up = __float_as_uint(p), uq = __float_as_uint(q);
      parts[i] = __builtin_amdgcn_perm(uq, up, 0x07060302u);
      p = fmaxf(p - __uint_as_float(up & 0xffff0000u), least);
      q = fmaxf(q - __uint_as_float(uq & 0xffff0000u), least);
    }
  } else {
    typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
    const h16x2 h = __builtin_bit_cast(h16x2, __builtin_amdgcn_cvt_pkrtz(p, q));
    parts[0] = __builtin_bit_cast(uint32_t, h);
    parts[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p - (float)h[0], q - (float)h[1]}, h16x2));
  }
}

// ds_read_b64_tr_b16: in each group of 16 lanes, lane j's element k is element
// j % 4 of the 8 bytes that lane 4 k + j / 4 addresses.
__device__ __forceinline__ uint2 pg_ld_tr(const uint8_t* p) {
  const pg_lds_s16x4* q = (const pg_lds_s16x4*)(__attribute__((address_space(3))) const uint8_t*)p;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(const_cast<pg_lds_s16x4*>(q)));
}

// y from its sums. den == 0: every score is -inf, whose softmax is NaN (num then
// holds what pg_split keeps above 0).
__device__ __forceinline__ float quotient(float num, float den) { return (den == 0.0f ? 0.0f : num) / den; }

// Where chunk `gx` of the call lies.
struct Chunk {
  int b, n;       // its sequence (-1: there is no such chunk) and the sequence's rows
  int c, count;   // its number in the sequence, and how many the sequence has
  int first;      // the number in the call of the sequence's first chunk
  int size;       // rows a chunk of this sequence
};

// Rows in units of PG_STEP, the steps that chunks are cut in.
__device__ __forceinline__ uint32_t units(int n) { return (uint32_t)(n + PG_STEP - 1) / PG_STEP; }

// A sequence's chunk count from the call's chunk length (units).
__device__ __forceinline__ int chunk_count(int n, uint32_t len) { return (int)((units(n) + len - 1) / len); }
// The rows a chunk then has: the sequence's, evenly.
__device__ __forceinline__ int chunk_size(int n, int count) {
  return count < 2 ? n : (int)((units(n) + count - 1) / count * PG_STEP);
}

// Rows of sequence b, 0 past the last.
__device__ __forceinline__ int rows_of(const AttnArgs& a, int b) { return b < a.seqs ? a.c.rows(a.SLOT[b]) : 0; }

// The call's chunk length (units): its rows over the chunks wanted. (attn_plan
// keeps all units within 31 bits.)
__device__ __forceinline__ uint32_t chunk_len(const AttnArgs& a, uint32_t total) {
  return max((total + a.target - 1) / (uint32_t)a.target, 1u);
}

// Up to 64 sequences a wave counts by itself, one a lane; more are counted by the
// workgroup, a run of neighbours a thread (all 256 threads, with barriers). Sequences
// of up to 1000 rows, where each wave counts all by itself and where the workgroup
// does: 65 of them 41 and 42 us, 256 of them 115 and 108, 1024 of them 548 and 425.
constexpr int PG_T = 64 * PG_WAVES;
static_assert(PG_T == 256, "the launches that look for chunks have 256 threads");

// The sum of v over the workgroup, and over the threads before this one.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* sums, int tid, uint32_t* total) {
  const uint32_t upto = lane_prefix(v);
  __syncthreads();
  if ((tid & 63) == 63) sums[tid >> 6] = upto;
  __syncthreads();
  uint32_t before = upto - v, all = 0;
#pragma unroll
  for (int w = 0; w < PG_T / 64; ++w) {
    if (w < (tid >> 6)) before += sums[w];
    all += sums[w];
  }
  *total = all;
  return before;
}

// Chunk `gx` of the call; the result is uniform.
__device__ __forceinline__ Chunk find_chunk(const AttnArgs& a, int gx, int tid) {
  __shared__ uint32_t sums[PG_T / 64];
  __shared__ int found[4];
  const int lane = tid & 63;
  if (a.target == 0) {
    const int n = a.c.rows(a.SLOT[gx]);
    return Chunk{gx, n, 0, 1, gx, n};
  }
  Chunk k{-1, 0, 0, 0, 0, 0};
  if (a.seqs <= 64) {
    const int n = rows_of(a, lane);
    const uint32_t len = chunk_len(a, __builtin_amdgcn_readlane(lane_prefix(units(n)), 63));
    const int count = chunk_count(n, len), upto = (int)lane_prefix(count);
    const uint64_t past = __ballot(upto > gx);
    if (!past) return k;
    const int l = __builtin_ctzll(past);
    k.b = l;
    k.n = __builtin_amdgcn_readlane(n, l);
    k.count = __builtin_amdgcn_readlane(count, l);
    k.first = __builtin_amdgcn_readlane(upto, l) - k.count;
  } else {
    const int per = (a.seqs + PG_T - 1) / PG_T, b0 = tid * per;
    uint32_t mine = 0, total;
    for (int i = 0; i < per; ++i) mine += units(rows_of(a, b0 + i));
    block_prefix(mine, sums, tid, &total);
    const uint32_t len = chunk_len(a, total);
    mine = 0;
    for (int i = 0; i < per; ++i) mine += chunk_count(rows_of(a, b0 + i), len);
    int first = (int)block_prefix(mine, sums, tid, &total);
    if ((uint32_t)gx >= total) return k;
    if (gx >= first && gx < first + (int)mine)  // one thread
      for (int i = 0; i < per; ++i) {
        const int n = rows_of(a, b0 + i), count = chunk_count(n, len);
        if (gx < first + count) {
          found[0] = b0 + i, found[1] = n, found[2] = count, found[3] = first;
          break;
        }
        first += count;
      }
    __syncthreads();
    k.b = __builtin_amdgcn_readfirstlane(found[0]);
    k.n = __builtin_amdgcn_readfirstlane(found[1]);
    k.count = __builtin_amdgcn_readfirstlane(found[2]);
    k.first = __builtin_amdgcn_readfirstlane(found[3]);
  }
  k.c = gx - k.first;
  k.size = chunk_size(k.n, k.count);
  return k;
}

// The chunks of sequence b (its rows and the numbers `c`, `size` left out).
__device__ __forceinline__ Chunk sequence_chunks(const AttnArgs& a, int b, int tid) {
  __shared__ uint32_t sums[PG_T / 64];
  Chunk k{b, 0, 0, 1, b, 0};
  if (a.target == 0) return k;
  if (a.seqs <= 64) {
    const int n = rows_of(a, tid & 63);
    const uint32_t len = chunk_len(a, __builtin_amdgcn_readlane(lane_prefix(units(n)), 63));
    const int count = chunk_count(n, len), upto = (int)lane_prefix(count);
    k.count = __builtin_amdgcn_readlane(count, b);
    k.first = __builtin_amdgcn_readlane(upto, b) - k.count;
    return k;
  }
  const int per = (a.seqs + PG_T - 1) / PG_T, b0 = tid * per;
  uint32_t mine = 0, total;
  for (int i = 0; i < per; ++i) mine += units(rows_of(a, b0 + i));
  block_prefix(mine, sums, tid, &total);
  const uint32_t len = chunk_len(a, total);
  mine = 0;
  for (int i = 0; i < per && b0 + i < b; ++i) mine += chunk_count(rows_of(a, b0 + i), len);
  block_prefix(mine, sums, tid, &total);
  k.first = (int)total;
  k.count = chunk_count(rows_of(a, b), len);
  return k;
}

template <int DT, int D, bool TRACK>
__global__ __launch_bounds__(64 * PG_WAVES) void paged_attn_kernel(const AttnArgs a) {
  constexpr int KC = D / 32, DC = D / 16;       // 32-wide steps of q . k, 16-wide tiles of V^T
  constexpr int VPL = PG_KEYS * D * 2 / 1024;   // 16-byte pieces of the 32 V rows a lane
  constexpr int VR = 1024 / (D * 2);            // V rows a load of the wave covers
  constexpr int REGION = PG_KEYS * D * 2;       // a wave's LDS: V rows, at the end 16 fp32 rows of O
  static_assert(REGION == PG_HEADS * D * 4, "the output tile takes the V rows' place");
  __shared__ __align__(16) uint8_t lds[PG_WAVES * REGION];
  __shared__ float m_s[PG_WAVES][PG_HEADS], l_s[PG_WAVES][PG_HEADS];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int group = a.nh / a.c.nkv, hgs = (group + PG_HEADS - 1) / PG_HEADS;
  const int wide = a.c.nkv * hgs, part = blockIdx.x % wide, gx = blockIdx.x / wide;
  const int h = part / hgs, head0 = h * group + (part % hgs) * PG_HEADS;
  const int heads = min(PG_HEADS, (h + 1) * group - head0);
  const Chunk ck = find_chunk(a, gx, tid);
  if (ck.b < 0) return;  // (a sequence without a row has no chunk; with target == 0 an empty one)
  const int b = __builtin_amdgcn_readfirstlane(ck.b);
  const int k0 = ck.c * ck.size, k1 = min(k0 + ck.size, ck.n);
  const int mask = (1 << a.c.shift) - 1;
  uint8_t* const vs = lds + wave * REGION;

  // Q^T: column = query head lr, dims 32 i + 8 lg .. + 7
  u32x4 qf[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i)
    qf[i] = lr < heads ? *reinterpret_cast<const u32x4*>(a.Q + b * a.q_seq + (size_t)(head0 + lr) * D + 32 * i + 8 * lg)
                       : u32x4{0u, 0u, 0u, 0u};

  // pages of the two 16-key halves of the run at j (uniform; past the chunk: holes)
  const int* const trow = a.c.table + b * a.c.table_stride;
  auto page_at = [&](int j) {
    const int p = j < k1 ? trow[j >> a.c.shift] : -1;
    return (unsigned)p < (unsigned)a.c.pages ? p : -1;
  };
  // a lane's place in a 16-key half: 32-bit byte offsets from a uniform base
  const uint32_t ko = (uint32_t)(lr * (int)a.c.k_row + 8 * lg) * 2;
  const uint32_t vo = (uint32_t)((lane / (64 / VR)) * (int)a.c.v_row + (lane % (64 / VR)) * 8) * 2;
  u32x4 kf[2][KC], vf[VPL];
  // A hole reads page 0's rows, which are masked; a page's 16-row runs are whole.
  auto load = [&](int j, int p0, int p1) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int p = max(s ? p1 : p0, 0), row = (j + 16 * s) & mask;
      const uint8_t* kb = (const uint8_t*)(a.c.K + p * a.c.k_page + h * a.c.k_head + row * a.c.k_row);
#pragma unroll
      for (int i = 0; i < KC; ++i) kf[s][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kb + 64 * i + ko));
      const uint8_t* vb = (const uint8_t*)(a.c.V + p * a.c.v_page + h * a.c.v_head + row * a.c.v_row);
#pragma unroll
      for (int i = 0; i < VPL / 2; ++i)
        vf[s * (VPL / 2) + i] =
            __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vb + (size_t)i * VR * a.c.v_row * 2 + vo));
    }
  };
  // V's 32-byte blocks lie swizzled by row, so that the transposing reads of
  // eight rows touch all banks
  auto vaddr = [&](int row, int blk) {
    const int sw = D == 128 ? row & 7 : (row >> 1) & 3;
    return row * (D * 2) + ((blk ^ sw) << 5);
  };

  f32x4 o[DC];
#pragma unroll
  for (int d = 0; d < DC; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float mref = PG_NONE, lsum = 0.0f;
  bool seen = false;
  float* const srow = TRACK ? a.S + ((size_t)b * a.nh + head0 + lr) * a.c.cap() : nullptr;

  int j = k0 + PG_KEYS * wave;
  int p0 = page_at(j), p1 = page_at(j + 16);
  if (j < k1) load(j, p0, p1);
  int n0 = page_at(j + PG_STEP), n1 = page_at(j + PG_STEP + 16);
  for (; j < k1; j += PG_STEP) {
    const bool whole = j + PG_KEYS <= k1 && p0 >= 0 && p1 >= 0;
    seen = seen || p0 >= 0 || p1 >= 0;
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < KC; ++i) s[t] = pg_mfma<DT>(kf[t][i], qf[i], s[t]);
    }
    // V rows into LDS; rows that are no keys as zeros (what they hold may be NaN)
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
    // the next run's rows
    const int c0 = p0, c1 = p1;
    p0 = n0, p1 = n1;
    if (j + PG_STEP < k1) load(j + PG_STEP, p0, p1);
    n0 = page_at(j + 2 * PG_STEP), n1 = page_at(j + 2 * PG_STEP + 16);

    // scores in log2 units; keys 16 t + 4 lg + r of the run
    bool over = false;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = s[t][r] * a.scale2;
        if (!whole && (j + 16 * t + 4 * lg + r >= k1 || (t ? c1 : c0) < 0)) x = -__builtin_inff();
        s[t][r] = x;
        over = over || x > mref + pg_above<DT>;
      }
    if constexpr (TRACK) {
      if (lr < heads)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (j + 16 * t < k1) *reinterpret_cast<f32x4*>(srow + j + 16 * t + 4 * lg) = s[t];
    }
    if (__any(over)) {
      float bm = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
      bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
      const float mnew = bm > mref + pg_above<DT> ? bm - pg_below<DT> : mref;
      const float alpha = __builtin_amdgcn_exp2f(mref - mnew);
      mref = mnew;
      lsum *= alpha;
#pragma unroll
      for (int d = 0; d < DC; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[d][r] *= alpha;
    }
    u32x4 pf[pg_parts<DT>];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = __builtin_amdgcn_exp2f(s[t][r] - mref);
        lsum += p[r];
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t parts[pg_parts<DT>];
        pg_split<DT>(p[2 * r], p[2 * r + 1], parts);
#pragma unroll
        for (int i = 0; i < pg_parts<DT>; ++i) pf[i][2 * t + r] = parts[i];
      }
    }
    // V^T: row = dim 16 d + lr at keys 4 lg .. + 3 and 16 + 4 lg .. + 3
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
      for (int i = 0; i < pg_parts<DT>; ++i) o[d] = pg_mfma<DT>(vt, pf[i], o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  // The waves' parts: each leaves its reference, sum and O [head][D] in LDS.
  lsum += __shfl_xor(lsum, 16, 64);
  lsum += __shfl_xor(lsum, 32, 64);
  if (lane < PG_HEADS) {
    m_s[wave][lane] = mref;
    l_s[wave][lane] = seen ? lsum : -1.0f;
  }
  float* const os = reinterpret_cast<float*>(vs);
#pragma unroll
  for (int d = 0; d < DC; ++d) *reinterpret_cast<f32x4*>(os + lr * D + 16 * d + 4 * lg) = o[d];
  __syncthreads();
  const float* const all = reinterpret_cast<const float*>(lds);
  const bool alone = ck.count == 1;
  for (int i = tid; i < heads * D; i += 64 * PG_WAVES) {
    const int g = i / D, d = i % D;
    float m = PG_NONE;
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) m = fmaxf(m, m_s[w][g]);
    float num = 0.0f, den = 0.0f;
    bool any = false;
#pragma unroll
    for (int w = 0; w < PG_WAVES; ++w) {  // (a wave without a key has a sum of -1 and zeros in O)
      const float l = l_s[w][g], e = __builtin_amdgcn_exp2f(m_s[w][g] - m);
      const bool none = l < 0.0f;
      den += (none ? 0.0f : l) * e;
      num += all[(size_t)w * (REGION / 4) + g * D + d] * e;
      any = any || !none;
    }
    const int head = head0 + g;
    if (alone) {
      a.Y[((size_t)b * a.nh + head) * D + d] = Elem<DT>::store(any ? quotient(num, den) : 0.0f);
      continue;
    }
    const size_t at = (size_t)gx * a.nh + head;
    a.PACC[at * D + d] = num;
    if (d == 0) {
      a.PM[at] = m;
      a.PL[at] = any ? den : -1.0f;
    }
  }
  if (!TRACK || !alone) {
    return;
  }
  if (group > PG_HEADS) {  // several workgroups share the kv head: the second launch adds their weights up
    const int g = tid;
    if (g < heads) {
      float m = PG_NONE, den = 0.0f;
      bool any = false;
      for (int w = 0; w < PG_WAVES; ++w) m = fmaxf(m, m_s[w][g]);
      for (int w = 0; w < PG_WAVES; ++w)
        if (!(l_s[w][g] < 0.0f)) den += l_s[w][g] * __builtin_amdgcn_exp2f(m_s[w][g] - m), any = true;
      const size_t at = (size_t)gx * a.nh + head0 + g;
      a.PM[at] = m;
      a.PL[at] = any ? den : -1.0f;
    }
    return;
  }
  // the weights of a sequence of one chunk
  for (int k = k0 + tid; k < k1; k += 64 * PG_WAVES) {
    if (a.c.page(b, k) < 0) continue;
    float w = 0.0f;
    for (int g = 0; g < heads; ++g) {
      float m = PG_NONE, den = 0.0f;
      for (int v = 0; v < PG_WAVES; ++v) m = fmaxf(m, m_s[v][g]);
      for (int v = 0; v < PG_WAVES; ++v)
        if (!(l_s[v][g] < 0.0f)) den += l_s[v][g] * __builtin_amdgcn_exp2f(m_s[v][g] - m);
      w += __builtin_amdgcn_exp2f(a.S[((size_t)b * a.nh + head0 + g) * a.c.cap() + k] - m) / den;
    }
    a.c.scores[b * a.c.score_seq + h * a.c.score_head + k] += w;
  }
}

// The reference and sum of one query head over a sequence's chunks, by a wave;
// uniform. den < 0: no key.
__device__ __forceinline__ void join_sums(const AttnArgs& a, const Chunk& ck, int head, int lane, float* m, float* den) {
  float mx = PG_NONE;
  for (int c = lane; c < ck.count; c += 64) mx = fmaxf(mx, a.PM[(size_t)(ck.first + c) * a.nh + head]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  float l = 0.0f;
  bool any = false;
  for (int c = lane; c < ck.count; c += 64) {
    const size_t at = (size_t)(ck.first + c) * a.nh + head;
    const float x = a.PL[at];
    if (x < 0.0f) continue;
    l += x * __builtin_amdgcn_exp2f(a.PM[at] - mx);
    any = true;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
  *m = mx;
  *den = __any(any) ? l : -1.0f;
}

// One query head's output from its sequence's chunks (two or more); all 256
// threads. The chunks' sums of the first round are on their way before the
// joined reference is known.
template <int DT, int D>
__device__ __forceinline__ void join_head(const AttnArgs& a, const Chunk& ck, int head, int tid) {
  constexpr int ROWS = 256 / (D / 4);  // chunks read at once, four elements a lane
  constexpr int AHEAD = 8;             // reads of a lane under way together
  __shared__ f32x4 part[256];
  __shared__ float w_s[PG_WGS];        // the chunks' weights (chunk_len: a sequence has at most `target` chunks)
  const int e = tid % (D / 4), r0 = tid / (D / 4);
  f32x4 x[AHEAD];
  auto load = [&](int c0) {  // past the last chunk: the last one's, not used
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const size_t at = (size_t)(ck.first + min(c0 + r0 + i * ROWS, ck.count - 1)) * a.nh + head;
      x[i] = reinterpret_cast<const f32x4*>(a.PACC + at * D)[e];
    }
  };
  load(0);
  float m, den;
  join_sums(a, ck, head, tid & 63, &m, &den);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = tid; c < ck.count; c += 256)  // (a chunk without a key: weight times zeros)
    w_s[c] = __builtin_amdgcn_exp2f(a.PM[(size_t)(ck.first + c) * a.nh + head] - m);
  __syncthreads();
  for (int c0 = 0; c0 < ck.count; c0 += ROWS * AHEAD) {
    if (c0) load(c0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int c = c0 + r0 + i * ROWS;
      if (c < ck.count) {
        const float w = w_s[c];
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] += x[i][k] * w;
      }
    }
  }
  part[tid] = acc;
  __syncthreads();
  if (tid < D / 4) {
    for (int r = 1; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += part[r * (D / 4) + tid][i];
    uint2 out;
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = den < 0.0f ? 0.0f : quotient(acc[i], den);
    out.x = Elem<DT>::store(q[0]) | (uint32_t)Elem<DT>::store(q[1]) << 16;
    out.y = Elem<DT>::store(q[2]) | (uint32_t)Elem<DT>::store(q[3]) << 16;
    reinterpret_cast<uint2*>(a.Y + ((size_t)ck.b * a.nh + head) * D)[tid] = out;
  }
}

// Query head `head` of sequence b, where the first launch has not finished it.
template <int DT, int D>
__device__ __forceinline__ void join_sequence(const AttnArgs& a, int b, int head, int tid) {
  const Chunk ck = sequence_chunks(a, b, tid);
  if (ck.count > 1)
    join_head<DT, D>(a, ck, head, tid);
  else if (ck.count == 0)  // no row, so no chunk. (In the first launch, stores that never ran took 10 % off its speed.)
    for (int i = tid; i < D / 8; i += 256)
      reinterpret_cast<u32x4*>(a.Y + ((size_t)b * a.nh + head) * D)[i] = u32x4{0u, 0u, 0u, 0u};
}

// Joins the sequences' chunks: workgroup (query head, sequence).
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const AttnArgs a) {
  join_sequence<DT, D>(a, blockIdx.y, blockIdx.x, threadIdx.x);
}

// With scores to gather: workgroups (kv head, chunk) add the weights of their
// chunk's slots to their scores; behind them, workgroups (query head, sequence)
// join the chunks.
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_gather_kernel(const AttnArgs a, int gathers) {
  constexpr int HG = 64;  // query heads whose sums are held at once
  __shared__ float m_s[HG], l_s[HG];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x >= gathers) {
    const int i = blockIdx.x - gathers;
    join_sequence<DT, D>(a, i / a.nh, i % a.nh, tid);
    return;
  }
  const int h = blockIdx.x % a.c.nkv, group = a.nh / a.c.nkv;
  const Chunk ck = find_chunk(a, blockIdx.x / a.c.nkv, tid);
  if (ck.b < 0 || (ck.count == 1 && group <= PG_HEADS)) return;  // (finished by the first launch)
  const int k0 = ck.c * ck.size, k1 = min(k0 + ck.size, ck.n);
  for (int g0 = 0; g0 < group; g0 += HG) {
    const int gs = min(HG, group - g0);
    const size_t step = a.c.cap();
    const float* const s0 = a.S + ((size_t)ck.b * a.nh + h * group + g0) * step;
    __syncthreads();
    for (int g = wave; g < gs; g += 4) {
      float m, den;
      join_sums(a, ck, h * group + g0 + g, lane, &m, &den);
      if (lane == 0) m_s[g] = m, l_s[g] = den;
    }
    __syncthreads();
    for (int k = k0 + tid; k < k1; k += 256) {
      if (a.c.page(ck.b, k) < 0) continue;
      float w = 0.0f;
#pragma unroll 4
      for (int g = 0; g < gs; ++g) w += __builtin_amdgcn_exp2f(s0[g * step + k] - m_s[g]) / l_s[g];
      a.c.scores[ck.b * a.c.score_seq + h * a.c.score_head + k] += w;
    }
  }
}

// How a call is cut up; false where the workspace, the rows or the launch are more than are counted.
struct AttnPlan {
  int target, chunks, hgs;
  size_t parts, scores;  // floats
};
inline bool attn_plan(int seqs, int nh, int nkv, int hd, long long cap, bool tracked, AttnPlan* p) {
  const int group = nh / nkv;
  p->hgs = (group + PG_HEADS - 1) / PG_HEADS;
  const long long wide = (long long)nkv * p->hgs;
  p->target = (int)(wide < PG_WGS ? PG_WGS / wide : 1);
  p->parts = p->scores = 0;
  if ((long long)seqs * ((cap + PG_STEP - 1) / PG_STEP) > 0x3fffffff) return false;  // (more rows than any memory holds)
  const bool one = cap <= PG_SHORT;
  if (one) p->target = 0;
  // a sequence adds at most one partly filled chunk to those the rows fill
  const long long most = (long long)seqs * ((cap + PG_STEP - 1) / PG_STEP);
  const long long chunks = p->target + (long long)seqs;
  p->chunks = one ? seqs : (int)(most < chunks ? most : chunks);
  // several workgroups of a kv head leave their sums for the gathering launch even so
  if (!one || (tracked && p->hgs > 1)) p->parts = (((size_t)p->chunks * nh * (2 + hd)) + 3) / 4 * 4;
  p->scores = tracked ? (size_t)seqs * nh * cap : 0;
  return (p->parts + p->scores + 255) / 256 <= 0x7fffffff && p->chunks * wide + (long long)seqs * nh <= PG_MAX_GRID;
}

}  // namespace ttsp

using namespace ttsp;

extern "C" int ttsp_paged_attention_work_kib(int seqs, int nh, int nkv, int head_dim, int cols, int page_size,
                                             int tracked) {
  if (seqs < 1 || nkv < 1 || nh < nkv || cols < 1 || page_size < 1 || head_dim < 1) return 0;
  AttnPlan p;
  const long long cap = (long long)cols * page_size;
  if (seqs > 65535 || nh > 65535 || nkv > 4096 || head_dim > 128 || cap > TTSP_PAGED_MAX_SLOTS ||
      !attn_plan(seqs, nh, nkv, head_dim, cap, tracked != 0, &p))
    return -1;
  return (int)((p.parts + p.scores + 255) / 256);
}

extern "C" int ttsp_paged_attention(const ttsp_paged_cache* cache, const void* Q, long long q_seq_stride,
                                    const long long* SLOT, void* Y, int nh, float scale, float* work,
                                    hipStream_t stream) {
  AttnArgs a{};
  AttnPlan p;
  if (!paged_args(cache, &a.c) || !Q || !SLOT || !Y || nh < 1 || nh > 65535 || nh % a.c.nkv ||
      (uintptr_t)Q % 16 || (uintptr_t)Y % 16 || q_seq_stride % 8 ||
      q_seq_stride < (long long)nh * cache->head_dim)
    return (int)hipErrorInvalidValue;
  const int hd = cache->head_dim;
  const bool tracked = a.c.scores != nullptr;
  if (!attn_plan(a.c.seqs, nh, a.c.nkv, hd, a.c.cap(), tracked, &p)) return (int)hipErrorInvalidValue;
  if (p.parts + p.scores && (!work || (uintptr_t)work % 16)) return (int)hipErrorInvalidValue;
  a.Q = (const uint16_t*)Q;
  a.q_seq = q_seq_stride;
  a.SLOT = SLOT;
  a.Y = (uint16_t*)Y;
  a.PACC = work;
  a.PM = work + (size_t)p.chunks * nh * hd;
  a.PL = a.PM + (size_t)p.chunks * nh;
  a.S = tracked ? work + p.parts : nullptr;
  a.scale2 = scale * 1.4426950408889634f;
  a.nh = nh;
  a.seqs = a.c.seqs;
  a.target = p.target;
  const dim3 grid((unsigned)p.chunks * a.c.nkv * p.hgs);
  const int gathers = p.chunks * a.c.nkv;
#define TTSP_PATT(DTV, DV)                                                                                       \
  do {                                                                                                           \
    if (tracked) hipLaunchKernelGGL((paged_attn_kernel<DTV, DV, true>), grid, dim3(64 * PG_WAVES), 0, stream, a); \
    else hipLaunchKernelGGL((paged_attn_kernel<DTV, DV, false>), grid, dim3(64 * PG_WAVES), 0, stream, a);        \
    if (tracked && (p.target || p.hgs > 1))                                                                       \
      hipLaunchKernelGGL((paged_gather_kernel<DTV, DV>), dim3(gathers + a.seqs * nh), dim3(256), 0, stream, a, gathers); \
    else if (p.target)                                                                                            \
      hipLaunchKernelGGL((paged_join_kernel<DTV, DV>), dim3(nh, a.seqs), dim3(256), 0, stream, a);                \
  } while (0)
  if (cache->dtype == DT_F16) {
    if (hd == 128) TTSP_PATT(DT_F16, 128);
    else TTSP_PATT(DT_F16, 64);
  } else {
    if (hd == 128) TTSP_PATT(DT_BF16, 128);
    else TTSP_PATT(DT_BF16, 64);
  }
#undef TTSP_PATT
  TTSP_RETURN_LAUNCH();
}
