// Attention of one new token per sequence over a paged cache: the entry points
// (the kernels and their reasons are in paged_attn.h).
#include "paged_attn.h"

using namespace ttsp;

// The window (-1: none) and sinks cut to the table.
static int attention_kib(int seqs, int nh, int nkv, int head_dim, int cols, int page_size, long long window,
                         long long sinks, int tracked) {
  if (seqs < 1 || nkv < 1 || nh < nkv || cols < 1 || page_size < 1 || head_dim < 1) return 0;
  AttnPlan p;
  const long long cap = (long long)cols * page_size;
  if (seqs > 65535 || nh > 65535 || nkv > 4096 || head_dim > 128 || cap > TTSP_PAGED_MAX_SLOTS ||
      !attn_plan(seqs, nh, nkv, head_dim, cap, window < 0 ? cap : window_rows(cap, window, sinks), tracked != 0, false, &p))
    return -1;
  return (int)((p.parts + p.scores + 255) / 256);
}

template <int FORM>
static int attention_launch(const ttsp_paged_cache* cache, const void* Q, long long q_seq_stride, const long long* SLOT,
                            void* Y, int nh, float scale, int window, int sinks, float* work, hipStream_t stream) {
  AttnArgs a{};
  AttnPlan p;
  if (!paged_args(cache, &a.c) || !Q || !SLOT || !Y || nh < 1 || nh > 65535 || nh % a.c.nkv ||
      (uintptr_t)Q % 16 || (uintptr_t)Y % 16 || q_seq_stride % 8 ||
      q_seq_stride < (long long)nh * cache->head_dim)
    return (int)hipErrorInvalidValue;
  const int hd = cache->head_dim;
  const bool tracked = a.c.scores != nullptr;
  const int cap = a.c.cap();
  if (FORM & PG_WINDOW) {
    if (window < 1 || sinks < 0) return (int)hipErrorInvalidValue;
    a.window = window < cap ? window : cap;
    a.sinks = sinks < cap ? sinks : cap;
  }
  if (!attn_plan(a.c.seqs, nh, a.c.nkv, hd, cap, FORM & PG_WINDOW ? window_rows(cap, a.window, a.sinks) : cap, tracked,
                 false, &p))
    return (int)hipErrorInvalidValue;
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
    if (tracked) hipLaunchKernelGGL((paged_attn_kernel<DTV, DV, FORM | PG_TRACK>), grid, dim3(64 * PG_WAVES), 0, stream, a); \
    else hipLaunchKernelGGL((paged_attn_kernel<DTV, DV, FORM>), grid, dim3(64 * PG_WAVES), 0, stream, a);        \
    if (tracked && (p.target || p.hgs > 1))                                                                       \
      hipLaunchKernelGGL((paged_gather_kernel<DTV, DV, FORM>), dim3(gathers + a.seqs * nh), dim3(256), 0, stream, a, gathers); \
    else if (p.target)                                                                                            \
      hipLaunchKernelGGL((paged_join_kernel<DTV, DV, FORM>), dim3(nh, a.seqs), dim3(256), 0, stream, a);                \
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

extern "C" int ttsp_paged_attention_work_kib(int seqs, int nh, int nkv, int head_dim, int cols, int page_size,
                                             int tracked) {
  return attention_kib(seqs, nh, nkv, head_dim, cols, page_size, -1, 0, tracked);
}

extern "C" int ttsp_paged_attention(const ttsp_paged_cache* cache, const void* Q, long long q_seq_stride,
                                    const long long* SLOT, void* Y, int nh, float scale, float* work,
                                    hipStream_t stream) {
  return attention_launch<0>(cache, Q, q_seq_stride, SLOT, Y, nh, scale, 0, 0, work, stream);
}

extern "C" int ttsp_paged_attention_window_work_kib(int seqs, int nh, int nkv, int head_dim, int cols, int page_size,
                                                    int window, int sinks, int tracked) {
  if (window < 1 || sinks < 0) return -1;
  return attention_kib(seqs, nh, nkv, head_dim, cols, page_size, window, sinks, tracked);
}

extern "C" int ttsp_paged_attention_window(const ttsp_paged_cache* cache, const void* Q, long long q_seq_stride,
                                           const long long* SLOT, void* Y, int nh, float scale, int window, int sinks,
                                           float* work, hipStream_t stream) {
  return attention_launch<PG_WINDOW>(cache, Q, q_seq_stride, SLOT, Y, nh, scale, window, sinks, work, stream);
}
