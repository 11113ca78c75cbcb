// A prompt's attention through a sliding window with sinks: the query row at position p
// sees keys j <= p with j < sinks or j > p - window; softmax over them of scale q . k,
// times v.
//
// A workgroup takes 32 RG rows of one kv head (tile_attn.h): position after position, and
// of each the query heads that share the kv head, so a tile of keys serves as many rows
// whatever the grouping, and the rows of a workgroup see nearly the same keys. Tiles of
// 64 keys that none of its rows sees are left out: of those behind the sinks, the ones
// before the first row's window. A run of keys that a wave's rows see whole is not
// masked, one that they do not see at all is not computed. Where there are few rows and
// many keys, the tiles are split over workgroups, whose sums a second launch joins. The
// weights go to the matrix cores rounded to the cache's type once, as the causal
// attention's do: bf16 within 2^-9, less than the output's own rounding in sum.
//
// 8111 rows, window 2048, 32 and 8 heads of 128, bf16: 255 us, 0.93 PFLOP/s of the keys
// that the mask leaves, bound by the exponentials' instructions beside the matrix cores'.
// 512 rows over 2000 keys, window 1024: 22 us a call (24 replayed in a graph), bound by
// latency (256 workgroups of 17 tiles one after the other). The matrix cores are busy 52 and
// 18 % of the time; LDS 28 and 12, of which 2 to 3 % bank conflicts.
#include "attn_common.h"
#include "prefill_merge.h"
#include "tile_attn.h"

namespace ttsp {

struct PromptArgs {
  const uint16_t *Q, *K, *V;  // [S][nh][128], [L][nkv][128] by strides
  uint16_t* Y;                // [S][nh][128]
  long long q_ss, q_sh, k_ss, k_sh, v_ss, v_sh;
  const long long* POS;
  int S, nh, nkv, L, window, sinks;
  float scale2;
  float* WO;   // SPLIT: as prefill_merge takes them
  int splits;
};

template <int DT, int RG, bool SPLIT>
__global__ __launch_bounds__(TA_T, 2) void prompt_window_kernel(const PromptArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Tile<HD, RG> C;
  constexpr int QT = 32 * RG, NB = C::SB;
  __shared__ __align__(256) uint8_t ring0[C::STAGE];
  __shared__ __align__(256) uint8_t ring1[C::STAGE];
  __shared__ int lim_s[2][TA_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wave % RG, kg = wave / RG, ql = lane & 31;
  // the last rows' workgroups first: they see most keys
  const int group = a.nh / a.nkv, wide = SPLIT ? a.nkv * a.splits : a.nkv, tiles = gridDim.x / wide;
  const int h = blockIdx.x % a.nkv, z = SPLIT ? blockIdx.x % wide / a.nkv : 0;
  const int row0 = (tiles - 1 - (int)blockIdx.x / wide) * QT, rows = min(QT, a.S * group - row0);
  const int r = row0 + min(32 * rg + ql, rows - 1);  // (rows past the last: that one's, not written)
  const int at = r / group, head = h * group + r % group;

  const long long pos = a.POS[at];
  TaWave<DT, HD, 1> w;
  w.init(lane);
  {
    const uint16_t* const q = a.Q + at * a.q_ss + head * a.q_sh + 8 * (lane >> 5);
    const uint32_t flip = a.scale2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) w.q[i] = *reinterpret_cast<const u32x4*>(q + 16 * i) ^ flip;
  }
  const float scale2 = a.scale2 == 0.0f ? 1e-30f : fabsf(a.scale2);

  // the last key this lane's row sees (-1: none) and the first of its window; over the
  // wave's rows the largest and smallest of both
  const int klast = (int)max(min(pos, (long long)a.L - 1), -1LL);
  const int klow = (int)min(max(pos, (long long)a.window - 1) - (a.window - 1), (long long)a.L);
  int last = klast, whole = klast, low = klow, first = klow;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    last = max(last, __shfl_xor(last, o, 64)), whole = min(whole, __shfl_xor(whole, o, 64));
    low = max(low, __shfl_xor(low, o, 64)), first = min(first, __shfl_xor(first, o, 64));
  }
  last = __builtin_amdgcn_readfirstlane(last), whole = __builtin_amdgcn_readfirstlane(whole);
  low = __builtin_amdgcn_readfirstlane(low), first = __builtin_amdgcn_readfirstlane(first);
  if (lane == 0) lim_s[0][wave] = last, lim_s[1][wave] = first;
  __syncthreads();
  int wlast = lim_s[0][0], wfirst = lim_s[1][0];  // over the workgroup's
#pragma unroll
  for (int i = 1; i < TA_WAVES; ++i) wlast = max(wlast, lim_s[0][i]), wfirst = min(wfirst, lim_s[1][i]);
  wlast = __builtin_amdgcn_readfirstlane(wlast), wfirst = __builtin_amdgcn_readfirstlane(wfirst);
  const int sink_tiles = (a.sinks + C::KEYS - 1) / C::KEYS, gap = max(wfirst / C::KEYS - sink_tiles, 0);
  // the workgroup's tiles: n from t0 on
  int n = max((wlast + C::KEYS) / C::KEYS - gap, 0), t0 = 0;
  if constexpr (SPLIT) {
    const int each = (n + a.splits - 1) / a.splits;
    t0 = z * each;
    n = max(min(n - t0, each), 0);
  }
  auto key_of = [&](int t) { return (t0 + t < sink_tiles ? t0 + t : t0 + t + gap) * C::KEYS; };

  const uint32_t hidden = (uint32_t)max(klow - a.sinks, 0);  // keys between the sinks and this lane's row's window
  uint32_t ko[C::PER], vo[C::PER];
  const int lrow0 = wave * C::PER * C::RPI + lane / C::PPR;
#pragma unroll
  for (int i = 0; i < C::PER; ++i) {
    const int row = lrow0 + i * C::RPI, piece = (lane % C::PPR) ^ ta_swz<HD>(row);
    ko[i] = (uint32_t)row * (uint32_t)a.k_ss * 2 + piece * 16;
    vo[i] = (uint32_t)row * (uint32_t)a.v_ss * 2 + piece * 16;
  }
  auto load = [&](int t, uint8_t* ring) {
    const int key = min(key_of(t), (a.L - 1) / C::KEYS * C::KEYS);
    const uint16_t* const kp = a.K + h * a.k_sh + key * a.k_ss;
    const uint16_t* const vp = a.V + h * a.v_sh + key * a.v_ss;
    const bool tail = key + C::KEYS > a.L;  // (rows past the keys: the last one's)
#pragma unroll
    for (int i = 0; i < C::PER; ++i) {
      uint32_t k = ko[i], v = vo[i];
      if (tail) {
        const uint32_t over = max(lrow0 + i * C::RPI - (a.L - 1 - key), 0);
        k -= over * (uint32_t)a.k_ss * 2, v -= over * (uint32_t)a.v_ss * 2;
      }
      ta_load(kp, k, ring + (wave * C::PER + i) * 1024);
      ta_load(vp, v, ring + C::HALF + (wave * C::PER + i) * 1024);
    }
  };
  // V rows that no row of the workgroup sees are zeros (what they hold may be NaN)
  auto landed = [&](int t, uint8_t* ring) {
    const int key = key_of(t);
    if (key + C::KEYS <= wlast + 1 && (key >= wfirst || key + C::KEYS <= a.sinks)) return;
#pragma unroll
    for (int i = 0; i < C::PER; ++i)
      if (const int j = key + lrow0 + i * C::RPI; j > wlast || (j >= a.sinks && j < wfirst))
        *reinterpret_cast<u32x4*>(ring + C::HALF + (wave * C::PER + i) * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
  };
  auto compute = [&](int t, uint8_t* ring) {
    const int row = 32 * NB * kg, k0 = key_of(t) + row, k1 = k0 + 32 * NB - 1;
    if (k0 > last || (k0 >= a.sinks && k1 < first)) return;
    const bool masked = k1 > whole || (k0 < low && k1 >= a.sinks);
    w.template run<NB>(ring + row * C::ROWB, ring + C::HALF + row * C::ROWB, scale2, masked, klast - k0, a.sinks - k0, hidden, 0);
  };
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) asm volatile("" ::"v"(w.q[i]));
  ta_tiles<C>(n, ring0, ring1, load, landed, compute);
  bool seen = true;
  ta_join<C>(w, seen, ring0, ring1, rg, kg, lane);
  if (kg) return;

  if constexpr (SPLIT) {
    const int row = 32 * rg + ql;
    if (row < rows) {
      const size_t to = ((size_t)z * a.S + at) * a.nh + head;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(a.WO + to * HD + 32 * d + 8 * g + 4 * (lane >> 5)) =
              f32x4{w.o[d][4 * g], w.o[d][4 * g + 1], w.o[d][4 * g + 2], w.o[d][4 * g + 3]};
      if (lane < 32)
        *reinterpret_cast<float2*>(a.WO + (size_t)a.splits * a.S * a.nh * HD + to * 2) = make_float2(w.m, w.l);
    }
    return;
  }
  // y = O / l (a row without a key: 0 / 0), the wave's 32 rows through its own LDS, so
  // that a store writes whole rows
  constexpr int PITCH = HD + 8;
  static_assert(32 * PITCH * 2 <= C::STAGE / 2, "two waves' rows in a stage");
  uint16_t* const os = reinterpret_cast<uint16_t*>((wave < 2 ? ring0 : ring1) + wave % 2 * (C::STAGE / 2));
  const float inv = 1.0f / w.l;
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint2 v;
      v.x = pack2<DT>(w.o[d][4 * g] * inv, w.o[d][4 * g + 1] * inv);
      v.y = pack2<DT>(w.o[d][4 * g + 2] * inv, w.o[d][4 * g + 3] * inv);
      *reinterpret_cast<uint2*>(os + ql * PITCH + 32 * d + 8 * g + 4 * (lane >> 5)) = v;
    }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 64 * i, row = e >> 4, c = (e & 15) * 8, y = 32 * rg + row;
    if (y < rows) {
      const int p = (row0 + y) / group, g = (row0 + y) % group;
      *reinterpret_cast<u32x4*>(a.Y + ((size_t)p * a.nh + h * group + g) * HD + c) =
          *reinterpret_cast<const u32x4*>(os + row * PITCH + c);
    }
  }
#endif
}

// Rows a workgroup takes, and over how many workgroups their tiles of keys are split.
//
// 128 rows where that makes two workgroups a CU, else 64 (1024 rows of 32 and 8 heads,
// window 1024: 26.1 us with 256 workgroups of 128 rows, 22.2 with 512 of 64).
// Splits: the joining launch costs about as much as six tiles, so not below twelve of
// them, and none once the workgroups are one a CU (9 rows over 2000 keys, window 1024:
// 20.8 us in one, 11.5 in eight; 512 rows: 24.4 in one, 30.1 in two; all in graphs).
struct PromptPlan {
  int rg, splits;
  long long wgs;
};
static PromptPlan prompt_plan(int S, int nh, int nkv, int L, int window, int sinks) {
  const long long rows = (long long)S * (nh / nkv);
  PromptPlan p{4, 1, (rows + 127) / 128 * nkv};
  if (p.wgs < 512) p = PromptPlan{2, 1, (rows + 63) / 64 * nkv};
  const long long seen = (long long)window + sinks + 64, tiles = ((seen < L ? seen : L) + 63) / 64;
  while (tiles >= 12 && p.wgs * p.splits < 256 && p.splits < 16 && tiles / (2 * p.splits) >= 2) p.splits *= 2;
  return p;
}

}  // namespace ttsp

using namespace ttsp;

extern "C" int ttsp_prefill_attention_window_splits(int S, int nh, int nkv, int L, int window, int sinks) {
  if (S <= 0 || nkv <= 0 || nh < nkv || L <= 0 || window <= 0 || sinks < 0) return 1;
  return prompt_plan(S, nh, nkv, L, window < L ? window : L, sinks < L ? sinks : L).splits;
}

extern "C" int ttsp_prefill_attention_window(const void* Q, long long q_seq_stride, long long q_head_stride,
                                             const void* K, long long k_seq_stride, long long k_head_stride,
                                             const void* V, long long v_seq_stride, long long v_head_stride,
                                             const long long* pos, void* Y, int S, int nh, int nkv, int L, int window,
                                             int sinks, float scale, int dtype, float* work, int splits,
                                             hipStream_t stream) {
  if (!Q || !K || !V || !pos || !Y || S <= 0 || S > (1 << 20) || nkv <= 0 || nh <= 0 || nh % nkv || nh > 65535 || L <= 0 ||
      window < 1 || sinks < 0 || splits < 1 || splits > 16 || (dtype != DT_F16 && dtype != DT_BF16))
    return (int)hipErrorInvalidValue;
  const long long st[6] = {q_seq_stride, q_head_stride, k_seq_stride, k_head_stride, v_seq_stride, v_head_stride};
  for (long long s : st)
    if (s < 0 || s % 8) return (int)hipErrorInvalidValue;
  if ((uintptr_t)Q % 16 || (uintptr_t)K % 16 || (uintptr_t)V % 16 || (uintptr_t)Y % 16 || (uintptr_t)pos % 8 ||
      (splits > 1 && (!work || (uintptr_t)work % 16)))
    return (int)hipErrorInvalidValue;
  // a tile's rows are addressed with 32-bit byte offsets from its first one
  const long long lim = (1LL << 31) - 1;
  if (L > lim - 127 ||  // (tiles are counted to the one behind the last, in keys)
      (L > 1 && (k_seq_stride > lim || v_seq_stride > lim)) || ((L - 1) * k_seq_stride + 128) * 2 > lim || ((L - 1) * v_seq_stride + 128) * 2 > lim)
    return (int)hipErrorInvalidValue;
  window = window < L ? window : L, sinks = sinks < L ? sinks : L;
  const PromptPlan p = prompt_plan(S, nh, nkv, L, window, sinks);
  if (p.wgs * splits > PG_MAX_GRID) return (int)hipErrorInvalidValue;
  const PromptArgs a{(const uint16_t*)Q, (const uint16_t*)K, (const uint16_t*)V, (uint16_t*)Y, q_seq_stride, q_head_stride,
                     k_seq_stride, k_head_stride, v_seq_stride, v_head_stride, pos, S, nh, nkv, L, window, sinks,
                     scale * 1.4426950408889634f, work, splits};
  const dim3 grid((unsigned)(p.wgs * splits));
#define TTSP_PW_(DTV, RGV, SPV) hipLaunchKernelGGL((prompt_window_kernel<DTV, RGV, SPV>), grid, dim3(TA_T), 0, stream, a)
#define TTSP_PW(DTV)                                     \
  do {                                                   \
    if (p.rg == 4 && splits > 1) TTSP_PW_(DTV, 4, true); \
    else if (p.rg == 4) TTSP_PW_(DTV, 4, false);         \
    else if (splits > 1) TTSP_PW_(DTV, 2, true);         \
    else TTSP_PW_(DTV, 2, false);                        \
  } while (0)
  if (dtype == DT_F16) TTSP_PW(DT_F16);
  else TTSP_PW(DT_BF16);
#undef TTSP_PW
#undef TTSP_PW_
  if (splits > 1) prefill_merge(work, splits, S, nh, Y, dtype, stream);
  TTSP_RETURN_LAUNCH();
}
