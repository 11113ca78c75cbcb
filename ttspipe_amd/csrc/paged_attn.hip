// Attention of one new token per sequence over a paged key-value cache:
//   s_j = scale q . k_j over the sequence's slots j with a page,
//   y = sum_j p_j v_j,  p = softmax(s),
// query head h reading kv head h / (nh / nkv); a sequence without a row gives
// zeros. With scores, sum over the kv head's query heads of p_j is added to
// the sequence's score of slot j.
//
// Workgroup = (kv head, sequence), one query head after the other: a thread a
// key for the scores, a thread an output element for the sum over the values.
#include "paged_common.h"

namespace ttsp {

struct AttnArgs {
  Paged c;
  const uint16_t* Q;  // [seqs][nh][D] by q_seq
  long long q_seq;
  const long long* SLOT;
  uint16_t* Y;  // [seqs][nh][D]
  float* work;  // scores in log2 units [seqs][nh][cap]
  float scale2;  // scale * log2(e)
  int nh, seqs;
};

__device__ __forceinline__ float block_max(float v, float* s, int tid) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((tid & 63) == 0) s[tid >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}
__device__ __forceinline__ float block_sum(float v, float* s, int tid) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((tid & 63) == 0) s[tid >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <int DT, int D>
__global__ __launch_bounds__(256) void paged_attn_kernel(const AttnArgs a) {
  __shared__ float q_s[D], red[4], y_s[256];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = a.c.rows(a.SLOT[b]), group = a.nh / a.c.nkv, mask = (1 << a.c.shift) - 1;
  for (int g = 0; g < group; ++g) {
    const int head = h * group + g;
    float* w = a.work + ((size_t)b * a.nh + head) * a.c.cap();
    uint16_t* y = a.Y + ((size_t)b * a.nh + head) * D;
    __syncthreads();
    if (tid < D) q_s[tid] = Elem<DT>::load(a.Q[b * a.q_seq + head * D + tid]);
    __syncthreads();
    float m = -3.0e38f, l = 0.0f, any = 0.0f;
    for (int j = tid; j < n; j += 256) {
      const int page = a.c.page(b, j);
      float s = __uint_as_float(0xff800000u);
      if (page >= 0) {
        const uint16_t* k = a.c.K + page * a.c.k_page + h * a.c.k_head + (j & mask) * a.c.k_row;
        s = 0.0f;
        for (int d = 0; d < D; ++d) s = __builtin_fmaf(q_s[d], Elem<DT>::load(k[d]), s);
        s *= a.scale2;
        m = fmaxf(m, s);
        any = 1.0f;
      }
      w[j] = s;
    }
    m = block_max(m, red, tid);
    any = block_max(any, red, tid);
    for (int j = tid; j < n; j += 256) {
      const float p = a.c.page(b, j) < 0 ? 0.0f : __builtin_amdgcn_exp2f(w[j] - m);
      w[j] = p;
      l += p;
    }
    l = block_sum(l, red, tid);
    if (any == 0.0f) {
      if (tid < D) y[tid] = 0;
      continue;
    }
    for (int j = tid; j < n; j += 256) w[j] /= l;
    __syncthreads();
    constexpr int KS = 256 / D;
    float acc = 0.0f;
    for (int j = tid / D; j < n; j += KS) {
      const int page = a.c.page(b, j);
      if (page < 0) continue;
      acc = __builtin_fmaf(w[j], Elem<DT>::load(a.c.V[page * a.c.v_page + h * a.c.v_head + (j & mask) * a.c.v_row + tid % D]), acc);
    }
    y_s[tid] = acc;
    __syncthreads();
    if (tid < D) {
      for (int k = 1; k < KS; ++k) acc += y_s[tid + k * D];
      y[tid] = Elem<DT>::store(acc);
    }
  }
  __syncthreads();
  if (a.c.scores)
    for (int j = tid; j < n; j += 256) {
      if (a.c.page(b, j) < 0) continue;
      float s = 0.0f;
      for (int g = 0; g < group; ++g) s += a.work[((size_t)b * a.nh + h * group + g) * a.c.cap() + j];
      a.c.scores[b * a.c.score_seq + h * a.c.score_head + j] += s;
    }
}

}  // namespace ttsp

using namespace ttsp;

extern "C" int ttsp_paged_attention_work_kib(int seqs, int nh, int nkv, int head_dim, int cols, int page_size,
                                             int tracked) {
  (void)nkv, (void)head_dim, (void)tracked;
  if (seqs < 1 || nh < 1 || cols < 1 || page_size < 1) return 0;
  const long long kib = ((long long)seqs * nh * cols * page_size * 4 + 1023) / 1024;
  return kib > 0x7fffffffLL ? -1 : (int)kib;
}

extern "C" int ttsp_paged_attention(const ttsp_paged_cache* cache, const void* Q, long long q_seq_stride,
                                    const long long* SLOT, void* Y, int nh, float scale, float* work,
                                    hipStream_t stream) {
  AttnArgs a{};
  if (!paged_args(cache, &a.c) || !Q || !SLOT || !Y || !work || nh < 1 || nh > 65535 || nh % a.c.nkv ||
      (uintptr_t)Q % 16 || (uintptr_t)Y % 16 || (uintptr_t)work % 16 || q_seq_stride % 8 ||
      q_seq_stride < (long long)nh * cache->head_dim)
    return (int)hipErrorInvalidValue;
  a.Q = (const uint16_t*)Q;
  a.q_seq = q_seq_stride;
  a.SLOT = SLOT;
  a.Y = (uint16_t*)Y;
  a.work = work;
  a.scale2 = scale * 1.4426950408889634f;
  a.nh = nh;
  a.seqs = a.c.seqs;
#define TTSP_PATT(DTV, DV) \
  hipLaunchKernelGGL((paged_attn_kernel<DTV, DV>), dim3(a.c.nkv, a.seqs), dim3(256), 0, stream, a)
  if (cache->dtype == DT_F16) {
    if (cache->head_dim == 128) TTSP_PATT(DT_F16, 128);
    else TTSP_PATT(DT_F16, 64);
  } else {
    if (cache->head_dim == 128) TTSP_PATT(DT_BF16, 128);
    else TTSP_PATT(DT_BF16, 64);
  }
#undef TTSP_PATT
  TTSP_RETURN_LAUNCH();
}
