// New rows of a paged cache: head norms, rotary and the write into the pages
// (a decode step's token of every sequence, or a ragged batch of prompt rows),
// and the plain copy of rows that are finished already.
//
// A row's q and k heads are x -> rotate(x / sqrt(mean(x^2) + eps) * w): rotary
// on interleaved pairs (a, b) -> (a c - b s, b c + a s) at the row's position,
// computed in fp32 and rounded to the activation type once, at the end. (The
// contiguous cache's kernel rounds after the norm as well, as the module it
// replaces does; here one rounding keeps the result nearer to the formula.
// Without head norms both give the same bits: the sums, products and their
// order are the same.)
//
// Memory bound: (nh + 2 nkv) heads of a row are read and written once. Eight
// elements (16 bytes) a lane, so a head is 16 lanes (8 of a 64-wide one), its
// pairs lie within a lane and its sum of squares needs only the group's lanes.
// 2011 rows of 48 heads of 128 (50 MB): 12.5 us, 4.0 TB/s; 32 rows: 3.1 us, the
// launch and three dependent reads (slot, page, row's factors).
#include "paged_common.h"

namespace ttsp {

struct RowsArgs {
  Paged c;
  const uint16_t* Q;  // (nh == 0: none)
  const uint16_t* K;
  const uint16_t* V;
  long long q_rs, q_hs, k_rs, k_hs, v_rs, v_hs;  // row and head strides, elements
  uint16_t* QO;                                  // [rows][nh][D]
  const uint16_t* QW;
  const uint16_t* KW;
  float eps;
  const void* F;  // rotary table [n_freqs][D / 2][2]
  int ftype, n_freqs;
  const long long* POS;   // positions (NULL: row t has rotary row t and no position is noted)
  const int* SEQ;         // sequences (NULL: row t is sequence t)
  const long long* SLOT;  // slots
  int rows, nh;
};

// Eight 16-bit elements as fp32.
template <int DT>
__device__ __forceinline__ void unpack8(u32x4 u, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Elem<DT>::load(u[i]);
    x[2 * i + 1] = Elem<DT>::load(u[i] >> 16);
  }
}

// (cos, sin) of four neighbouring pairs, from element `at` of the table.
__device__ __forceinline__ void load_turn(const void* F, int ftype, size_t at, float* f) {
  if (ftype == DT_F32) {
    const f32x4* p = reinterpret_cast<const f32x4*>((const float*)F + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
    return;
  }
  const u32x4 u = *reinterpret_cast<const u32x4*>((const uint16_t*)F + at);
  if (ftype == DT_F16) unpack8<DT_F16>(u, f);
  else unpack8<DT_BF16>(u, f);
}

// A lane group a head of a row. (Two or four heads a group share the row's slot,
// position and factors, and leave fewer loads under way: 2011 rows of 48 heads took
// 13.1 and 13.7 us so, 12.5 with one.)
template <int DT, int D, bool ROPE>
__global__ __launch_bounds__(256) void paged_rows_kernel(const RowsArgs a) {
  constexpr int LH = D / 8;  // lanes a head
  const int lane = threadIdx.x & (LH - 1), e = lane * 8;
  const int heads = a.nh + 2 * a.c.nkv;
  const long long item = ((long long)blockIdx.x * 256 + threadIdx.x) / LH;
  if (item >= (long long)a.rows * heads) return;  // whole groups of LH lanes
  const int t = (int)(item / heads), head = (int)(item % heads), k = head - a.nh, v = k - a.c.nkv;
  const long long pos = a.POS ? a.POS[t] : t;
  const long long slot = a.SLOT[t];
  const int b = a.SEQ ? a.SEQ[t] : t;
  const uint16_t* src = k < 0 ? a.Q + t * a.q_rs + head * a.q_hs : v < 0 ? a.K + t * a.k_rs + k * a.k_hs
                                                                       : a.V + t * a.v_rs + v * a.v_hs;
  u32x4 u = *reinterpret_cast<const u32x4*>(src + e);
  const bool turns = !ROPE || (pos >= 0 && pos < a.n_freqs);  // else the row is left out
  float f[8];
  if constexpr (ROPE) load_turn(a.F, a.ftype, (size_t)(turns ? pos : 0) * D + e, f);
  // the page and row a k or v head goes to (-1: none)
  int page = -1, off = 0;
  if (k >= 0 && turns && (unsigned)b < (unsigned)a.c.seqs && slot >= 0 && slot < a.c.cap()) {
    page = a.c.page(b, (int)slot);
    off = (int)slot & ((1 << a.c.shift) - 1);
  }
  if (ROPE && v < 0) {
    float x[8];
    unpack8<DT>(u, x);
    const uint16_t* w = k < 0 ? a.QW : a.KW;
    if (w) {
      float wt[8];
      unpack8<DT>(*reinterpret_cast<const u32x4*>(w + e), wt);
      // the sum over neighbours, pairs of neighbours, and so on: within the
      // lane, then over the group (the mirrored steps pair what xor 4 and 8 do)
      float s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = __fmul_rn(x[i], x[i]);
      float ss = __fadd_rn(__fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3])),
                           __fadd_rn(__fadd_rn(s[4], s[5]), __fadd_rn(s[6], s[7])));
      ss = dpp_add<0xB1, 0xF>(ss);
      ss = dpp_add<0x4E, 0xF>(ss);
      ss = dpp_add<0x141, 0xF>(ss);
      if constexpr (LH == 16) ss = dpp_add<0x140, 0xF>(ss);
      const float r = rsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)D), a.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], r), wt[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = x[2 * i], y = x[2 * i + 1], c = f[2 * i], s = f[2 * i + 1];
      const uint32_t lo = Elem<DT>::store(__fsub_rn(__fmul_rn(p, c), __fmul_rn(y, s)));
      const uint32_t hi = Elem<DT>::store(__fadd_rn(__fmul_rn(y, c), __fmul_rn(p, s)));
      u[i] = lo | hi << 16;
    }
  }
  if (k < 0) {
    if (!turns) u = u32x4{0u, 0u, 0u, 0u};
    *reinterpret_cast<u32x4*>(a.QO + ((size_t)t * a.nh + head) * D + e) = u;
    return;
  }
  if (page < 0) return;
  uint16_t* dst = v < 0 ? a.c.K + page * a.c.k_page + k * a.c.k_head + off * a.c.k_row
                        : a.c.V + page * a.c.v_page + v * a.c.v_head + off * a.c.v_row;
  *reinterpret_cast<u32x4*>(dst + e) = u;
  if (v < 0 && lane == 0) {
    if (a.c.scores) a.c.scores[b * a.c.score_seq + k * a.c.score_head + slot] = 0.0f;
    if (a.c.slot_pos) a.c.slot_pos[b * a.c.pos_seq + k * a.c.pos_head + slot] = (int)pos;
  }
}

template <bool ROPE>
int launch_rows(const RowsArgs& a, int hd, int dtype, hipStream_t stream) {
  const int heads = a.nh + 2 * a.c.nkv;
  const long long groups = ((long long)a.rows * heads * (hd / 8) + 255) / 256;
  if (groups > PG_MAX_GRID) return (int)hipErrorInvalidValue;
#define TTSP_ROWS(DTV, DV) \
  hipLaunchKernelGGL((paged_rows_kernel<DTV, DV, ROPE>), dim3((unsigned)groups), dim3(256), 0, stream, a)
  if (dtype == DT_F16) {
    if (hd == 128) TTSP_ROWS(DT_F16, 128);
    else TTSP_ROWS(DT_F16, 64);
  } else {
    if (hd == 128) TTSP_ROWS(DT_BF16, 128);
    else TTSP_ROWS(DT_BF16, 64);
  }
#undef TTSP_ROWS
  TTSP_RETURN_LAUNCH();
}

}  // namespace ttsp

using namespace ttsp;

extern "C" int ttsp_paged_qk_rope_kv(const ttsp_paged_cache* cache, const void* QKV, long long qkv_row_stride,
                                     const void* QW, const void* KW, float eps, const void* F, int ftype, int n_freqs,
                                     const long long* POS, const int* SEQ, const long long* SLOT, void* Q, int nh,
                                     int rows, hipStream_t stream) {
  RowsArgs a{};
  if (!paged_args(cache, &a.c) || !QKV || !F || !SLOT || !Q || nh < 1 || nh > 4096 || rows < 0 || rows > (1 << 24) ||
      ftype < 0 || ftype > 2 || n_freqs < 1)
    return (int)hipErrorInvalidValue;
  const int hd = cache->head_dim;
  if (qkv_row_stride < (long long)(nh + 2 * a.c.nkv) * hd || qkv_row_stride % 8 || (uintptr_t)QKV % 16 ||
      (uintptr_t)F % 16 || (uintptr_t)Q % 16 || (uintptr_t)QW % 16 || (uintptr_t)KW % 16 ||
      (!POS && (n_freqs < rows || a.c.slot_pos)) || (!SEQ && rows > a.c.seqs))
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  a.Q = (const uint16_t*)QKV;
  a.K = a.Q + (size_t)nh * hd;
  a.V = a.K + (size_t)a.c.nkv * hd;
  a.q_rs = a.k_rs = a.v_rs = qkv_row_stride;
  a.q_hs = a.k_hs = a.v_hs = hd;
  a.QO = (uint16_t*)Q;
  a.QW = (const uint16_t*)QW;
  a.KW = (const uint16_t*)KW;
  a.eps = eps;
  a.F = F;
  a.ftype = ftype;
  a.n_freqs = n_freqs;
  a.POS = POS;
  a.SEQ = SEQ;
  a.SLOT = SLOT;
  a.rows = rows;
  a.nh = nh;
  return launch_rows<true>(a, hd, cache->dtype, stream);
}

extern "C" int ttsp_paged_store(const ttsp_paged_cache* cache, const void* K, long long k_row_stride,
                                long long k_head_stride, const void* V, long long v_row_stride,
                                long long v_head_stride, const long long* POS, const int* SEQ, const long long* SLOT,
                                int rows, hipStream_t stream) {
  RowsArgs a{};
  if (!paged_args(cache, &a.c) || !K || !V || !SLOT || rows < 0 || rows > (1 << 24) || (uintptr_t)K % 16 ||
      (uintptr_t)V % 16 || (a.c.slot_pos && !POS) || (!SEQ && rows > a.c.seqs))
    return (int)hipErrorInvalidValue;
  const long long strides[] = {k_row_stride, k_head_stride, v_row_stride, v_head_stride};
  for (long long s : strides)
    if (s < 0 || s % 8) return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  a.K = (const uint16_t*)K;
  a.V = (const uint16_t*)V;
  a.k_rs = k_row_stride;
  a.k_hs = k_head_stride;
  a.v_rs = v_row_stride;
  a.v_hs = v_head_stride;
  a.POS = POS;
  a.SEQ = SEQ;
  a.SLOT = SLOT;
  a.rows = rows;
  return launch_rows<false>(a, cache->head_dim, cache->dtype, stream);
}
