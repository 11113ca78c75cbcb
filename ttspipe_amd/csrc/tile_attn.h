// Attention of many query rows over the same keys, the core of the kernels that have
// such rows: sequences that share a prefix (paged_prefix.hip) and a prompt's rows
// through a window (prefill_window.hip).
//
// A workgroup of four waves takes 32 RG query rows of one kv head. Its keys come in
// tiles of 64 through a ring of two in LDS, straight from memory (buffer loads to LDS,
// so that no register holds what is on its way): RG waves take 32 rows each of the same
// keys, and with two row groups (RG 2) the other two waves take the other half of a
// tile's keys and join their sums through LDS at the end. Two workgroups fit a CU: one
// waits at its barrier while the other computes (64 sequences behind 32763 rows: 111 us
// with eight waves in one workgroup, 100 so, and 84 since a prefix's chunks are longer). A ring of four tiles is slower for few
// tiles: twice the code to be fetched before it has run once (2 to 5 us).
//
// A wave's 32 keys: S^T = K Q^T on the matrix cores (Q stays in registers), so that a
// lane holds 16 keys of one query row; the exponentials subtract a reference that
// moves only when a score outgrows it (pg_above), so the running maximum needs no
// exchange between lanes but a vote; P^T goes back to the matrix cores from the
// registers it is in, in PARTS of the cache's type: O^T += V^T P^T, V^T through the
// transposing LDS read.
//
// K and V rows lie in LDS as in memory, their 16-byte pieces swizzled by row (ta_swz):
// sixteen rows' same piece lies in sixteen different bank groups (K's reads), and the
// same 64 bytes of four neighbouring rows in four (V's transposing reads).
//
// MFMA 32x32x16: lane l supplies row (l % 32) of A and column (l % 32) of B at
// k = 8 (l / 32) .. + 7; accumulator r of lane l is D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32].
#pragma once

#include "nf4_mfma.h"
#include "paged_attn.h"

namespace ttsp {

constexpr int TA_WAVES = 4, TA_T = 64 * TA_WAVES;

template <int D, int RG>
struct Tile {
  static constexpr int KG = TA_WAVES / RG, SB = 2 / KG;  // key groups; runs of 32 keys a wave takes of a tile
  static constexpr int KEYS = 64, ROWB = D * 2, PPR = ROWB / 16;
  static constexpr int HALF = KEYS * ROWB, STAGE = 2 * HALF;  // K, then V
  static constexpr int RPI = 1024 / ROWB, PER = KEYS / RPI / TA_WAVES;  // rows a load covers, loads of K (and of V) a wave
};

// The swizzle of row r: its 16-byte piece p lies at piece p ^ ta_swz(r).
template <int D>
__device__ __forceinline__ int ta_swz(int r) {
  return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Two weights (not negative) in PARTS of DT as packed pairs. One part: rounded to
// nearest. Two: fp16 as pg_split, within 2^-22; bf16 the upper eight bits and the rest
// rounded to eight, within 2^-16 (the lower part is kept above 0, as in pg_split).
template <int DT, int PARTS>
__device__ __forceinline__ void ta_split(float p, float q, uint32_t* parts) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
  if constexpr (PARTS == 1) {
    if constexpr (DT == DT_BF16) parts[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p, q}, b16x2));
    else parts[0] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){p, q}, h16x2));
  } else if constexpr (DT == DT_F16) {
    pg_split<DT>(p, q, parts);
  } else {
    constexpr float least = 1.17549435e-38f;
    const uint32_t up = __float_as_uint(p), uq = __float_as_uint(q);
    parts[0] = __builtin_amdgcn_perm(uq, up, 0x07060302u);
    const f32x2 rest = {fmaxf(p - __uint_as_float(up & 0xffff0000u), least), fmaxf(q - __uint_as_float(uq & 0xffff0000u), least)};
    parts[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, b16x2));
  }
}

// A wave's 32 query rows.
template <int DT, int D, int PARTS>
struct TaWave {
  u32x4 q[D / 16];      // Q^T: column = query row lane % 32, dims 16 i + 8 (lane / 32) .. + 7
  f32x16_v o[D / 32];   // O^T
  float m, l;           // reference (log2 units) and this lane's keys' sum of exp2(s - m)
  uint32_t kb, vb;      // this lane's first bytes of K and of V in a run of 32 keys

  __device__ __forceinline__ void init(int lane) {
    const int h = lane >> 5, ql = lane & 31, g = lane >> 4, li = lane & 15;
    m = PG_NONE, l = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    kb = ql * (D * 2) + ((h ^ ta_swz<D>(ql)) << 4);
    const int row = 4 * (g >> 1) + (li >> 2), piece = 2 * (g & 1) + ((li & 3) >> 1);
    vb = row * (D * 2) + ((piece ^ ta_swz<D>(row)) << 4) + (li & 1) * 8;
  }

  // K's rows of 32 keys in the operand's layout
  __device__ __forceinline__ void keys(const uint8_t* k, u32x4 (&kf)[D / 16]) const {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) kf[i] = *reinterpret_cast<const u32x4*>(k + (kb ^ (i << 5)));
  }
  __device__ __forceinline__ f32x16_v score(const u32x4 (&kf)[D / 16]) const {
    f32x16_v s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) s = mfma32<DT>(kf[i], q[i], s);
    return s;
  }
  // Weights by the reference as it is; their sum.
  __device__ __forceinline__ float weigh(const f32x16_v& s, float scale2, f32x16_v& p) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale2, -m));
    return (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]))) +
           (((p[8] + p[9]) + (p[10] + p[11])) + ((p[12] + p[13]) + (p[14] + p[15])));
  }
  // The reference above the scores. fp16 weights in two parts use their type's whole
  // range (pg_below) and have no room for larger ones, so their maximum is looked at
  // first. The others are weighed as the reference is, and only where they come out too
  // large (sixteen of 2^8 and less sum up to no more than 4096) it moves, and they are
  // weighed again; fp16's largest is 2^4 then, which keeps those down to 2^-28 of it
  // (a prompt of 8111 rows in fp16: 295 us with the maximum of every run, 261 so).
  static constexpr bool FIRST = DT == DT_F16 && PARTS > 1;
  static constexpr float above = FIRST ? pg_above<DT> : 8.0f, below = FIRST ? pg_below<DT> : DT == DT_F16 ? 4.0f : 0.0f;
  __device__ __forceinline__ void move(const f32x16_v& s, float scale2) {
    float bm = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) bm = fmaxf(bm, s[r]);
    bm *= scale2;
    if (FIRST && !__any(bm > m + above)) return;
    bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
    const float mnew = bm > m + above ? bm - below : m;
    const float alpha = __builtin_amdgcn_exp2f(m - mnew);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
  }
  // V^T of 16 keys at v, and O^T += V^T P^T of them
  __device__ __forceinline__ void values(const uint8_t* v, u32x4 (&vt)[D / 32]) const {
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      const uint2 lo = pg_ld_tr(v + (vb ^ (d << 6))), hi = pg_ld_tr(v + 8 * (D * 2) + (vb ^ (d << 6) ^ 32));
      vt[d] = u32x4{lo.x, lo.y, hi.x, hi.y};
    }
  }
  __device__ __forceinline__ void split(const f32x16_v& p, int c, u32x4 (&pf)[PARTS]) const {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t parts[PARTS];
      ta_split<DT, PARTS>(p[8 * c + 2 * u], p[8 * c + 2 * u + 1], parts);
#pragma unroll
      for (int i = 0; i < PARTS; ++i) pf[i][u] = parts[i];
    }
  }
  __device__ __forceinline__ void add(const u32x4 (&vt)[D / 32], const u32x4 (&pf)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) o[d] = mfma32<DT>(vt[d], pf[i], o[d]);
  }

  // 32 NB keys, K and V rows at k and v. masked (uniform): those behind key `after` of them
  // are none, nor the `hidden` ones from key `from` on, nor 16-key run i where bit i of
  // `gone` (uniform) is set.
  template <int NB>
  __device__ __forceinline__ void run(const uint8_t* k, const uint8_t* v, float scale2, bool masked, int after, int from,
                                      uint32_t hidden, uint32_t gone) {
    constexpr int RB = 32 * D * 2;  // bytes of 32 rows
    const int h4 = (threadIdx.x & 63) >> 5 << 2;
    auto mask = [&](int b, f32x16_v& s) {
      int last = after - (32 * b + h4), first = from - (32 * b + h4);
      asm volatile("" : "+v"(last), "+v"(first));  // (what follows from them would be computed ahead, and spilled)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = 8 * (r / 4) + r % 4;
        if ((j > last) | ((uint32_t)(j - first) < hidden)) s[r] = -__builtin_inff();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (gone >> (2 * b + i) & 1)
#pragma unroll
          for (int r = 0; r < 8; ++r) s[8 * i + r] = -__builtin_inff();
    };
    u32x4 kf[NB][D / 16];
#pragma unroll
    for (int b = 0; b < NB; ++b) keys(k + b * RB, kf[b]);
    __builtin_amdgcn_sched_barrier(0);
    f32x16_v s[NB], p;
    s[0] = score(kf[0]);
    if (masked) mask(0, s[0]);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      // the weights of run b beside the scores of run b + 1 or the products of run b - 1
      if constexpr (FIRST) move(s[b], scale2);
      if (b + 1 < NB) s[b + 1] = score(kf[b + 1]);
      float sum = weigh(s[b], scale2, p);
      if (b + 1 < NB)
        for (int i = 0; i < D / 16; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
        }
      if (b + 1 < NB && masked) mask(b + 1, s[b + 1]);
      if constexpr (!FIRST)
        if (__any(!(sum <= 4096.0f))) {
          move(s[b], scale2);
          sum = weigh(s[b], scale2, p);
        }
      l += sum;
      u32x4 vt[2][D / 32], pf[2][PARTS];
      values(v + b * RB, vt[0]);
      values(v + b * RB + RB / 2, vt[1]);
      split(p, 0, pf[0]);
      add(vt[0], pf[0]);
      split(p, 1, pf[1]);
      add(vt[1], pf[1]);
    }
  }
};

// n tiles through a ring of two: load(t, ring) issues this wave's 2 PER loads of tile t (any
// t: past the last it may load what it likes), landed(t, ring) may touch up the rows
// that this wave loaded, compute(t, ring) reads tile t.
template <typename C, typename F, typename G, typename H>
__device__ __forceinline__ void ta_tiles(int n, uint8_t* ring0, uint8_t* ring1, F load, G landed, H compute) {
  if (n <= 0) return;
  load(0, ring0);
  // step t: tile t has landed and every wave is past tile t - 1, whose place tile t + 1 takes
  auto one = [&](int t, uint8_t* rd, uint8_t* dst) {
    TTSP_WAIT_VM_LGKM0(0);
    landed(t, rd);
    TTSP_WAIT_LGKM0();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    load(t + 1, dst);
    compute(t, rd);
  };
#pragma unroll 1
  for (int t = 0; t < n; t += 2) {
    one(t, ring0, ring1);
    if (t + 1 < n) one(t + 1, ring1, ring0);
  }
  TTSP_WAIT_VM_LGKM0(0);
  __syncthreads();
}

// The key groups' sums joined into the first group's waves (the ring is free). seen:
// whether the wave has had a key; the first group's get the groups'.
template <typename C, int DT, int D, int PARTS>
__device__ __forceinline__ void ta_join(TaWave<DT, D, PARTS>& w, bool& seen, uint8_t* ring0, uint8_t* ring1, int rg, int kg, int lane) {
  w.l += __shfl_xor(w.l, 32, 64);
  if constexpr (C::KG == 2) {
    static_assert((TA_WAVES / 2) * (D / 32) * 4096 <= C::STAGE, "the givers' O in a stage");
    float* const part = reinterpret_cast<float*>(ring0) + rg * (D / 32) * 1024 + lane;
    float* const ml = reinterpret_cast<float*>(ring1) + rg * 192 + lane;
    if (kg) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) part[(16 * d + r) * 64] = w.o[d][r];
      ml[0] = w.m, ml[64] = w.l, ml[128] = seen ? 1.0f : 0.0f;
    }
    __syncthreads();
    if (!kg) {
      const float m2 = ml[0], mm = fmaxf(w.m, m2);
      const float f1 = __builtin_amdgcn_exp2f(w.m - mm), f2 = __builtin_amdgcn_exp2f(m2 - mm);
      w.l = w.l * f1 + ml[64] * f2;
      w.m = mm;
      seen = seen || ml[128] != 0.0f;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) w.o[d][r] = w.o[d][r] * f1 + part[(16 * d + r) * 64] * f2;
    }
  }
}

// One load of 1024 bytes of rows from base into LDS at dst, lane l's 16 bytes from byte voff.
__device__ __forceinline__ void ta_load(const void* base, uint32_t voff, uint8_t* dst) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, -1, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 16, voff, 0, 0, 0);
}

}  // namespace ttsp
