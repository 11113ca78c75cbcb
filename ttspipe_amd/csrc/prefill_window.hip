// A prompt's attention through a sliding window with sinks: the query row at position p
// sees keys j <= p with j < sinks or j > p - window; softmax over them of scale q . k,
// times v.
//
// A workgroup takes 32 RG rows of one kv head (tile_attn.h): position after position, and
// of each the query heads that share the kv head, so a tile of keys serves as many rows
// whatever the grouping, and the rows of a workgroup see nearly the same keys. Tiles of
// 64 keys that none of its rows sees are left out: of those behind the sinks, the ones
// before the first row's window. A run of keys that a wave's rows see whole is not
// masked, one that they do not see at all is not computed. The weights go to the matrix
// cores rounded to the cache's type once, as the causal attention's do.
#include "attn_common.h"
#include "prefill_window.h"
#include "tile_attn.h"

namespace ttsp {

struct PromptArgs {
  const uint16_t *Q, *K, *V;  // [S][nh][128], [L][nkv][128] by strides
  uint16_t* Y;                // [S][nh][128]
  long long q_ss, q_sh, k_ss, k_sh, v_ss, v_sh;
  const long long* POS;
  int S, nh, nkv, L, window, sinks;
  float scale2;
};

template <int DT, int RG>
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
  const int group = a.nh / a.nkv, h = blockIdx.x % a.nkv, tiles = gridDim.x / a.nkv;
  const int row0 = (tiles - 1 - (int)blockIdx.x / a.nkv) * QT, rows = min(QT, a.S * group - row0);
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
  const int n = max((wlast + C::KEYS) / C::KEYS - gap, 0);
  auto key_of = [&](int t) { return (t < sink_tiles ? t : t + gap) * C::KEYS; };

  uint32_t ko[C::PER], vo[C::PER];
  const int lrow0 = wave * C::PER * C::RPI + lane / C::PPR;
#pragma unroll
  for (int i = 0; i < C::PER; ++i) {
    const int row = lrow0 + i * C::RPI, piece = (lane % C::PPR) ^ ta_swz<HD>(row);
    ko[i] = (uint32_t)(row * (int)a.k_ss) * 2 + piece * 16;
    vo[i] = (uint32_t)(row * (int)a.v_ss) * 2 + piece * 16;
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
        const int over = max(lrow0 + i * C::RPI - (a.L - 1 - key), 0);
        k -= (uint32_t)(over * (int)a.k_ss) * 2, v -= (uint32_t)(over * (int)a.v_ss) * 2;
      }
      ta_load(kp, k, ring + (wave * C::PER + i) * 1024);
      ta_load(vp, v, ring + C::HALF + (wave * C::PER + i) * 1024);
    }
  };
  // V rows behind the last key that any row sees are zeros (what they hold may be NaN)
  auto landed = [&](int t, uint8_t* ring) {
    const int key = key_of(t);
    if (key + C::KEYS <= wlast + 1) return;
#pragma unroll
    for (int i = 0; i < C::PER; ++i)
      if (key + lrow0 + i * C::RPI > wlast)
        *reinterpret_cast<u32x4*>(ring + C::HALF + (wave * C::PER + i) * 1024 + lane * 16) = u32x4{0u, 0u, 0u, 0u};
  };
  auto compute = [&](int t, uint8_t* ring) {
    const int row = 32 * NB * kg, k0 = key_of(t) + row, k1 = k0 + 32 * NB - 1;
    if (k0 > last || (k0 >= a.sinks && k1 < first)) return;
    const bool masked = k1 > whole || (k0 < low && k1 >= a.sinks);
    w.template run<NB>(ring + row * C::ROWB, ring + C::HALF + row * C::ROWB, scale2, masked,
                       [&](int i) { return k0 + i > klast || (k0 + i >= a.sinks && k0 + i < klow); });
  };
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) asm volatile("" ::"v"(w.q[i]));
  ta_tiles<C>(n, ring0, ring1, load, landed, compute);
  bool seen = true;
  ta_join<C>(w, seen, ring0, ring1, rg, kg, lane);
  if (kg) return;

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

int prompt_window_tiles(int S, int nh, int nkv) {
  const long long rows = (long long)S * (nh / nkv);
  if ((rows + 127) / 128 * nkv >= PW_FULL) return 4;
  return (rows + 63) / 64 * nkv >= PW_LEAST ? 2 : 0;
}

int prompt_window_launch(const void* Q, long long q_ss, long long q_sh, const void* K, long long k_ss, long long k_sh,
                         const void* V, long long v_ss, long long v_sh, const long long* pos, void* Y, int S, int nh,
                         int nkv, int L, int window, int sinks, float scale, int dtype, int tiles, hipStream_t stream) {
  const PromptArgs a{(const uint16_t*)Q, (const uint16_t*)K, (const uint16_t*)V, (uint16_t*)Y, q_ss, q_sh, k_ss, k_sh, v_ss, v_sh,
                     pos, S, nh, nkv, L, window, sinks, scale * 1.4426950408889634f};
  const long long rows = (long long)S * (nh / nkv), wgs = (rows + 32 * tiles - 1) / (32 * tiles) * nkv;
  if (wgs > PG_MAX_GRID) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs);
#define TTSP_PW(DTV)                                                                                              \
  do {                                                                                                            \
    if (tiles == 4) hipLaunchKernelGGL((prompt_window_kernel<DTV, 4>), grid, dim3(TA_T), 0, stream, a);            \
    else hipLaunchKernelGGL((prompt_window_kernel<DTV, 2>), grid, dim3(TA_T), 0, stream, a);                       \
  } while (0)
  if (dtype == DT_F16) TTSP_PW(DT_F16);
  else TTSP_PW(DT_BF16);
#undef TTSP_PW
  return 0;
}

}  // namespace ttsp
