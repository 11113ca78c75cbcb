// Penalties, biases and a grammar's mask on rows of logits, before they are
// sampled. With c the number of times token t occurs in the row's history:
//   x = logit;  c > 0: x = x > 0 ? x / r : x r, then x -= f c + p
//   x += bias;  x = -inf where bit t % 32 of word t / 32 of the mask is 0
// in fp32, one rounding an operation in this order, and one to the row's type.
//
// A workgroup takes a slice of a row: it counts the history's tokens that fall
// into the slice in LDS (integer adds, so their order does not matter) while the
// slice's logits are on their way, and applies the counts as it writes. So there
// is no count array in memory and no second pass. 256 rows of 131001 logits in fp32
// after up to 4096 tokens: 63 us, 4.4 TB/s, where a copy of as many bytes runs at 5.1;
// a row of 4096 after 16 tokens 3.5 us, a launch and two reads one after the other.
#define TTSP_HIP_TYPES_ONLY
#include "../../include/ttsp_hip.h"
#include "ttsp_common.h"

namespace ttsp {

constexpr int LG_FULL = 256;  // workgroups from which on the slices are large

struct PenaltyArgs {
  const void* X;
  void* Y;
  long long x_row, y_row;  // row strides, elements
  int rows, vocab, slices;
  const void* HIST;  // int32 or int64 [rows][hist] by hist_row; null: no history
  long long hist_row;
  int hist, hist64;
  const void* LEN;  // int32 or int64: entries of each row that count; null: all
  int len64;
  const float *REP, *FREQ, *PRES;  // per row by scalar_row; null: none
  int rep_row, freq_row, pres_row;  // 1, or 0: one value for all rows
  const void* BIAS;
  long long bias_row;
  int bias_f32;
  const uint32_t* MASK;
  long long mask_row;
};

// 16 bytes at any address that their elements allow.
template <int A> struct Vec16;
template <> struct Vec16<2> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Vec16<4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4))); };

// T threads of NV 16-byte vectors.
template <int DT, int T, int NV>
__global__ __launch_bounds__(T) void penalize_kernel(const PenaltyArgs a) {
  constexpr int ES = DT == DT_F32 ? 4 : 2, VE = 16 / ES;  // bytes an element, elements a vector
  constexpr int SL = T * NV * VE;                // elements a slice
  typedef typename Vec16<ES>::type vec;
  __shared__ __align__(16) uint32_t cnt[SL];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / a.slices, base = (blockIdx.x % a.slices) * SL;
  const int n = min(SL, a.vocab - base);  // elements of this slice
  const uint8_t* const x = (const uint8_t*)a.X + ((size_t)row * a.x_row + base) * ES;
  uint8_t* const y = (uint8_t*)a.Y + ((size_t)row * a.y_row + base) * ES;

  u32x4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * T + tid) * VE;
    v[i] = u32x4{0u, 0u, 0u, 0u};
    if (e + VE <= n) {
      v[i] = *reinterpret_cast<const vec*>(x + (size_t)e * ES);
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k)
        if (e + k < n) {
          if constexpr (ES == 4) v[i][k] = reinterpret_cast<const uint32_t*>(x)[e + k];
          else v[i][k / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(x)[e + k] << (16 * (k % 2));
        }
    }
  }
  const float rep = a.REP ? a.REP[row * a.rep_row] : 1.0f;
  const float freq = a.FREQ ? a.FREQ[row * a.freq_row] : 0.0f, pres = a.PRES ? a.PRES[row * a.pres_row] : 0.0f;
  const bool additive = a.FREQ || a.PRES;

  if (a.HIST) {
    long long len = a.hist;
    if (a.LEN) len = a.len64 ? ((const long long*)a.LEN)[row] : (long long)((const int*)a.LEN)[row];
    len = min(len, (long long)a.hist);
#pragma unroll
    for (int i = 0; i < SL / 4 / T; ++i)
      reinterpret_cast<u32x4*>(cnt)[i * T + tid] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    auto count = [&](auto* hist) {
      constexpr int AHEAD = 4;  // tokens of a thread under way together
      for (long long i0 = tid; i0 < len; i0 += AHEAD * T) {
        unsigned long long at[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const long long i = i0 + k * T;
          at[k] = i < len ? (unsigned long long)(long long)hist[i] - (unsigned long long)base : ~0ull;
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (at[k] < (unsigned long long)n) atomicAdd(&cnt[at[k]], 1u);
      }
    };
    if (a.hist64) count((const long long*)a.HIST + (size_t)row * a.hist_row);
    else count((const int*)a.HIST + (size_t)row * a.hist_row);
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = (i * T + tid) * VE;
    if (e >= n) break;
    float f[VE];
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      if constexpr (ES == 4) f[k] = __uint_as_float(v[i][k]);
      else f[k] = Elem<DT>::load(v[i][k / 2] >> (16 * (k % 2)));
    }
    if (a.HIST) {
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        const uint32_t c = cnt[e + k];
        if (c) {
          if (a.REP) f[k] = f[k] > 0.0f ? __fdiv_rn(f[k], rep) : __fmul_rn(f[k], rep);
          if (additive) f[k] = __fsub_rn(f[k], __fadd_rn(__fmul_rn(freq, (float)c), pres));
        }
      }
    }
    if (a.BIAS) {
      const size_t b0 = (size_t)row * a.bias_row + base + e;
#pragma unroll
      for (int k = 0; k < VE; ++k)
        if (e + k < n)
          f[k] = __fadd_rn(f[k], a.bias_f32 || ES == 4 ? ((const float*)a.BIAS)[b0 + k]
                                                       : Elem<DT == DT_F32 ? DT_F16 : DT>::load(((const uint16_t*)a.BIAS)[b0 + k]));
    }
    if (a.MASK) {  // (a vector's elements lie in one word)
      const uint32_t bits = a.MASK[(size_t)row * a.mask_row + (base + e) / 32] >> ((base + e) % 32);
#pragma unroll
      for (int k = 0; k < VE; ++k)
        if (!(bits >> k & 1u)) f[k] = -__builtin_inff();
    }
    u32x4 o = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      if constexpr (ES == 4) o[k] = __float_as_uint(f[k]);
      else o[k / 2] |= (uint32_t)Elem<DT == DT_F32 ? DT_F16 : DT>::store(f[k]) << (16 * (k % 2));
    }
    if (e + VE <= n) {
      *reinterpret_cast<vec*>(y + (size_t)e * ES) = o;
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k)
        if (e + k < n) {
          if constexpr (ES == 4) reinterpret_cast<uint32_t*>(y)[e + k] = o[k];
          else reinterpret_cast<uint16_t*>(y)[e + k] = (uint16_t)(o[k / 2] >> (16 * (k % 2)));
        }
    }
  }
}

}  // namespace ttsp

using namespace ttsp;

extern "C" int ttsp_penalize(const ttsp_penalties* p, const void* X, long long x_row_stride, void* Y,
                             long long y_row_stride, int rows, int vocab, int dtype, hipStream_t stream) {
  if (!p || !X || !Y || rows < 0 || vocab < 1 || vocab > (1 << 30)) return (int)hipErrorInvalidValue;
  if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32) return (int)hipErrorInvalidValue;
  const uintptr_t es = dtype == DT_F32 ? 4 : 2;
  if ((uintptr_t)X % es || (uintptr_t)Y % es || x_row_stride < 0 ||
      y_row_stride < (rows > 1 ? vocab : 0))
    return (int)hipErrorInvalidValue;
  if (p->hist < 0 || p->hist_row_stride < 0 || p->bias_row_stride < 0 || p->mask_row_stride < 0)
    return (int)hipErrorInvalidValue;
  if (p->HIST && (uintptr_t)p->HIST % (p->hist_64 ? 8 : 4)) return (int)hipErrorInvalidValue;
  if (p->LEN && (uintptr_t)p->LEN % (p->len_64 ? 8 : 4)) return (int)hipErrorInvalidValue;
  if ((uintptr_t)p->REP % 4 || (uintptr_t)p->FREQ % 4 || (uintptr_t)p->PRES % 4 || (uintptr_t)p->MASK % 4)
    return (int)hipErrorInvalidValue;
  if (p->BIAS && ((p->bias_dtype != dtype && p->bias_dtype != DT_F32) || (uintptr_t)p->BIAS % (p->bias_dtype == DT_F32 ? 4 : 2)))
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  PenaltyArgs a{X, Y, x_row_stride, y_row_stride, rows, vocab, 0, p->hist ? p->HIST : nullptr, p->hist_row_stride, p->hist,
                p->hist_64 != 0, p->LEN, p->len_64 != 0, p->REP, p->FREQ, p->PRES, p->rep_rows != 0, p->freq_rows != 0,
                p->pres_rows != 0, p->BIAS, p->bias_row_stride, p->bias_dtype == DT_F32, (const uint32_t*)p->MASK,
                p->mask_row_stride};
  // Every workgroup reads its row's history, so long ones (of enough rows to fill the GPU
  // all the same) go with large slices: 256 rows of 131001 in fp32 after 4096 tokens
  // 66 us in slices of 2048 and 56 in those of 16384, 1500 tokens 53 and 53, 50 tokens 47
  // and 52 (the same inputs again and again, which the caches then hold in part).
  constexpr int WIDE = 16384, SMALL = 2048;
  const bool wide = p->hist > 1024 && (long long)rows * ((vocab + WIDE - 1) / WIDE) >= LG_FULL;
  const int slice = wide ? WIDE : SMALL;
  a.slices = (vocab + slice - 1) / slice;
  if ((long long)rows * a.slices > 0xffffff >> 2) return (int)hipErrorInvalidValue;  // (threads are counted in 32 bits)
  const dim3 grid((unsigned)(rows * a.slices));
#define TTSP_LG(DTV, VE)                                                                                            \
  do {                                                                                                              \
    if (wide) hipLaunchKernelGGL((penalize_kernel<DTV, 1024, WIDE / 1024 / VE>), grid, dim3(1024), 0, stream, a);    \
    else hipLaunchKernelGGL((penalize_kernel<DTV, 256, SMALL / 256 / VE>), grid, dim3(256), 0, stream, a);           \
  } while (0)
  if (dtype == DT_F32) TTSP_LG(DT_F32, 4);
  else if (dtype == DT_F16) TTSP_LG(DT_F16, 8);
  else TTSP_LG(DT_BF16, 8);
#undef TTSP_LG
  TTSP_RETURN_LAUNCH();
}
