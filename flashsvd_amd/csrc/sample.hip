// The next token drawn from filtered logits, one launch.  With the logits in descending order, equal ones by their index, and weights
// w_i = exp((l_i - l_0) / T), C_n = w_0 + .. + w_{n-1}:
//   n_k = top_k, n_p = the smallest n with C_n > top_p C_{n_k}, n_m = how many w >= min_p, N = the least of them; the token is the first whose
//   C exceeds u C_N.
// Every filter keeps a prefix of that order, and 16-bit logits have few distinct values, so nothing is sorted: the values of a row are counted in a
// histogram over their 65536 patterns in LDS, and an exponential is taken for each value that occurs, once, in 64 bits, as the sums are (a boundary between
// two of 10^5 nearly equal tokens is 10^-5 of the sum wide; with 32-bit sums one draw in a thousand lands on the wrong side of it).
#include "common.hpp"
#include "../../include/flashsvd_hip.h"

namespace fsvd {

constexpr int kDrawThreads = 1024, kDrawWaves = kDrawThreads / kWave, kDrawRow = 1 << 24;
constexpr int kHistWords = 32768, kSegs = 1024, kSegBins = 64;      // two 16-bit counts a word; bins of one wave's look
constexpr int kMostExtra = kDrawRow / 32768;

struct SampleArgs {
  const uint16_t* logits; int64_t ld;
  const float* uniforms;
  int64_t* tokens; int64_t ldt;
  int32_t* positions;
  double temperature, top_p, min_p; int top_k;
  const float *temperatures, *top_ps, *min_ps; const int32_t* top_ks;      // per row, in place of the numbers
  int V;
};

// patterns as whole numbers in the order of their values, NaN above everything, the two zeros equal; and back
template <int DT>
__device__ __forceinline__ uint32_t draw_key(uint32_t p) {
  constexpr uint32_t kInf = DT == 1 ? 0x7c00u : 0x7f80u;
  const uint32_t mag = p & 0x7fffu;
  if (mag > kInf) return 0xffffu;                       // above the key of the infinity
  if (mag == 0) return 0x8000u;
  return (p & 0x8000u) ? 0x7fffu - mag : 0x8000u + mag;
}
template <int DT>
__device__ __forceinline__ float key_value(uint32_t k) {
  return E16<DT>::val(k >= 0x8000u ? k - 0x8000u : 0xffffu - k);          // 0x7fff - k is the magnitude, the sign bit above it
}

template <class T>
__device__ __forceinline__ T wave_scan(T v, int lane) {                   // inclusive, towards higher lanes
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const T x = __shfl_up(v, o);
    if (lane >= o) v += x;
  }
  return v;
}
template <class T>
__device__ __forceinline__ T wave_total(T v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <int DT>
__global__ __launch_bounds__(kDrawThreads) void sample_token_kernel(SampleArgs a) {
  constexpr uint32_t kInf = DT == 1 ? 0x7c00u : 0x7f80u, kLowest = 0x7fffu - kInf + 1, kHighest = 0x8000u + kInf - 1;     // keys of the finite values
  extern __shared__ __align__(16) uint32_t hist[];                       // [kHistWords]
  __shared__ double seg_mass[kSegs], wave_mass[kDrawWaves], at_mass;
  __shared__ uint32_t seg_count[kSegs], wave_count[kDrawWaves], wave_most[kDrawWaves], wave_kept[kDrawWaves], at_seg, at_count, rank_key, rank_in, rank_n;
  __shared__ uint16_t extra[kMostExtra];                                  // keys that hold 32768 more than their bin says, once for each
  __shared__ uint32_t n_extra;
  __shared__ double rank_mass;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint16_t* row = a.logits + (int64_t)b * a.ld;
  const int V = a.V, pieces = (V + 7) >> 3;
  // eight logits; behind the row's end stands -inf, which is never counted
  const auto fetch = [&](int c) {
    if (c * 8 + 8 <= V) return __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(row + (int64_t)c * 8));
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t p = c * 8 + e < V ? row[c * 8 + e] : 0x8000u | kInf;
      w[e >> 1] = e & 1 ? w[e >> 1] | p << 16 : p;
    }
    return u32x4_t{w[0], w[1], w[2], w[3]};
  };
  const auto each = [&](u32x4_t v, auto f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) f(draw_key<DT>((w[e >> 1] >> (16 * (e & 1))) & 0xffffu), e);
  };

  // the largest
  uint32_t most = 0;
  for (int c = tid; c < pieces; c += kDrawThreads) each(fetch(c), [&](uint32_t k, int) { most = max(most, k); });
#pragma unroll
  for (int o = 32; o; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
  if (lane == 0) wave_most[wave] = most;
  for (int i = tid; i < kHistWords; i += kDrawThreads) hist[i] = 0;
  if (tid == 0) n_extra = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kDrawWaves; ++i) most = max(most, wave_most[i]);

  const double temp = a.temperatures ? (double)a.temperatures[b] : a.temperature;
  uint32_t key = most, rank = 0;                        // the token: this occurrence of this key
  if (temp > 0. && most >= kLowest && most <= kHighest) {
    const double top_p = a.top_ps ? (double)a.top_ps[b] : a.top_p, min_p = a.min_ps ? (double)a.min_ps[b] : a.min_p;
    const int top_k = a.top_ks ? a.top_ks[b] : a.top_k;
    const float high = key_value<DT>(most);
    // what is below e^-80 of the largest changes no sum of 64 bits and is not counted
    const double floor_ = (double)high - 80. * temp;
    uint32_t least = kLowest;
    if (floor_ > (double)key_value<DT>(kLowest)) least = max(kLowest, draw_key<DT>(E16<DT>::bits((float)floor_)));
    const auto count_up = [&](int c) {
      each(fetch(c), [&](uint32_t k, int) { if (k >= least) atomicAdd(&hist[k >> 1], 1u << (16 * (k & 1))); });
    };
    uint32_t mine = 0;
    for (int c = tid; c < pieces; c += kDrawThreads) {
      count_up(c);
      each(fetch(c), [&](uint32_t k, int) { mine += k >= least; });
    }
    const auto bin = [&](uint32_t k) {
      uint32_t n = (hist[k >> 1] >> (16 * (k & 1))) & 0xffffu;
      for (uint32_t i = 0; i < n_extra; ++i) n += extra[i] == k ? 32768u : 0u;
      return n;
    };
    const auto weight = [&](uint32_t k) { return exp(((double)key_value<DT>(k) - (double)high) / temp); };
    mine = wave_total(mine);
    uint32_t counted = 0, in_all = 0;
    for (int round = 0; round < 2; ++round) {
      __syncthreads();
      for (int s = tid; s < kSegs; s += kDrawThreads) { seg_mass[s] = 0.; seg_count[s] = 0; }
      if (lane == 0) wave_count[wave] = mine;
      __syncthreads();
      uint32_t kept = 0;
      for (int s = (int)(least / kSegBins) + wave; s <= (int)(most / kSegBins); s += kDrawWaves) {
        const uint32_t k = s * kSegBins + lane, n = k <= most ? bin(k) : 0;
        if (!__any(n != 0)) continue;
        const double w = n ? weight(k) : 0.;
        const double m = wave_total(n * w);
        const uint32_t c = wave_total(n);
        kept += w >= min_p ? n : 0;
        if (lane == 0) { seg_mass[s] = m; seg_count[s] = c; }
      }
      kept = wave_total(kept);
      if (lane == 0) wave_kept[wave] = kept;
      __syncthreads();
      counted = 0;
      in_all = 0;
      for (int i = 0; i < kDrawWaves; ++i) counted += wave_count[i];
      uint32_t c = wave_total(seg_count[tid]);
      __syncthreads();
      if (lane == 0) wave_most[wave] = c;
      __syncthreads();
      for (int i = 0; i < kDrawWaves; ++i) in_all += wave_most[i];
      if (in_all == counted) break;
      // A 16-bit count has run over (more than 65535 equal logits): the row is counted again in steps that cannot, and after each what exceeds 32767 is
      // set aside.
      __syncthreads();
      for (int i = tid; i < kHistWords; i += kDrawThreads) hist[i] = 0;
      for (int c0 = 0; c0 < pieces; c0 += 4095) {
        __syncthreads();
        for (int c = c0 + tid; c < min(c0 + 4095, pieces); c += kDrawThreads) count_up(c);
        __syncthreads();
        for (int i = tid; i < kHistWords; i += kDrawThreads) {
          const uint32_t w = hist[i];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (w & (0x8000u << (16 * h))) extra[atomicAdd(&n_extra, 1u)] = (uint16_t)(2 * i + h);
          hist[i] = w & 0x7fff7fffu;
        }
      }
    }
    // running sums over the segments, from the largest values down: thread t has segment kSegs - 1 - t
    const int seg = kSegs - 1 - tid;
    double mass = seg_mass[seg];
    uint32_t count = seg_count[seg];
    const double own_mass = mass;
    const uint32_t own_count = count;
    mass = wave_scan(mass, lane);
    count = wave_scan(count, lane);
    if (lane == 63) { wave_mass[wave] = mass; wave_count[wave] = count; }
    __syncthreads();
    double mass0 = 0., all = 0.;
    uint32_t count0 = 0;
    for (int i = 0; i < kDrawWaves; ++i) {
      if (i < wave) { mass0 += wave_mass[i]; count0 += wave_count[i]; }
      all += wave_mass[i];
    }
    mass += mass0;
    count += count0;
    // The n-th of the order, where n is the smallest with C_n > target (by_mass) or given: its key, how many of its key are up to it, n and C_n
    const auto locate = [&](bool by_mass, double target, uint32_t n) {
      __syncthreads();
      const bool here = by_mass ? mass > target && mass - own_mass <= target : count >= n && count - own_count < n;
      if (tid == 0) at_seg = 0xffffffffu;
      __syncthreads();
      if (here && own_count) atomicMin(&at_seg, (uint32_t)tid);           // rounding may leave two neighbours, or none
      __syncthreads();
      uint32_t t = at_seg;
      __syncthreads();
      if (t == 0xffffffffu) {                                            // none: the last that has any
        if (tid == 0) at_seg = 0;
        __syncthreads();
        if (own_count) atomicMax(&at_seg, (uint32_t)tid);
        __syncthreads();
        t = at_seg;
      }
      if ((uint32_t)tid == t) { at_mass = mass - own_mass; at_count = count - own_count; }
      __syncthreads();
      if (wave == 0) {
        const uint32_t k = (kSegs - 1 - t) * kSegBins + kSegBins - 1 - lane, c = k <= most && k >= least ? bin(k) : 0;
        const double w = c ? weight(k) : 0., m = c * w;
        const double ms = at_mass + wave_scan(m, lane);
        const uint32_t cs = at_count + wave_scan(c, lane);
        const uint64_t hit = __ballot(c && (by_mass ? ms > target : cs >= n)), some = __ballot(c != 0);
        const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
        if (lane == l) {
          uint32_t j = c;
          const double before = ms - m;
          if (hit) j = by_mass ? (uint32_t)fmin(fmax(floor((target - before) / w), 0.) + 1., (double)c) : n - (cs - c);
          rank_key = k;
          rank_in = j;
          rank_n = cs - c + j;
          rank_mass = before + j * w;
        }
      }
      __syncthreads();
    };
    uint32_t keep = top_k > 0 && (uint32_t)top_k < in_all ? (uint32_t)top_k : in_all;
    double z = all;
    if (keep < in_all) { locate(false, 0., keep); z = rank_mass; }
    uint32_t n = keep;
    if (top_p < 1.) { locate(true, top_p * z, 0); n = min(n, rank_n); }
    uint32_t likely = 0;
    for (int i = 0; i < kDrawWaves; ++i) likely += wave_kept[i];
    if (min_p > 0.) n = min(n, likely);
    n = max(n, 1u);
    if (n < in_all) { locate(false, 0., n); z = rank_mass; }
    locate(true, (double)a.uniforms[b] * z, 0);
    if (rank_n > n) locate(false, 0., n);
    key = rank_key;
    rank = rank_in - 1;
  }

  // that occurrence, by index: how many a wave has in each of its pieces, then the piece, then the element
  __syncthreads();
  const int rounds = (pieces + kDrawThreads - 1) / kDrawThreads;
  for (int r = 0; r < rounds; ++r) {
    const int c = r * kDrawThreads + tid;
    uint32_t n = 0;
    if (c < pieces) each(fetch(c), [&](uint32_t k, int) { n += k == key; });
    n = wave_total(n);
    if (lane == 0) hist[r * kDrawWaves + wave] = n;
  }
  __syncthreads();
  if (wave != 0) return;
  uint32_t before = 0;
  for (int i0 = 0; i0 < rounds * kDrawWaves; i0 += kWave) {
    const uint32_t n = i0 + lane < rounds * kDrawWaves ? hist[i0 + lane] : 0, s = before + wave_scan(n, lane);
    const uint64_t hit = __ballot(s > rank);
    if (hit == 0) { before = __shfl(s, 63); continue; }
    const int l = __builtin_ctzll(hit), c = (i0 + l) * kWave + lane;
    before = __shfl(s - n, l);
    const u32x4_t v = fetch(min(c, pieces - 1));
    uint32_t m = 0;
    if (c < pieces) each(v, [&](uint32_t k, int) { m += k == key; });
    uint32_t at = before + wave_scan(m, lane) - m;
    if (c < pieces && at <= rank && rank < at + m) {
      each(v, [&](uint32_t k, int e) {
        if (k == key) { if (at == rank) a.tokens[(int64_t)b * a.ldt] = c * 8 + e; ++at; }
      });
      if (a.positions) a.positions[b] += 1;
    }
    return;
  }
}

template <int DT>
static int launch_sample(const char* fn, const SampleArgs& a, int B, hipStream_t st) {
  static bool granted = false;
  if (!granted) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&sample_token_kernel<DT>), hipFuncAttributeMaxDynamicSharedMemorySize, kHistWords * 4);
    if (e != hipSuccess) { set_last_error("%s: cannot reserve %d bytes of LDS: %s", fn, kHistWords * 4, hipGetErrorString(e)); return kErrLaunch; }
    granted = true;
  }
  hipLaunchKernelGGL(sample_token_kernel<DT>, dim3(B), dim3(kDrawThreads), kHistWords * 4, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

}  // namespace fsvd

using namespace fsvd;

extern "C" int fsvd_sample_token(const void* logits, int64_t ld, const float* uniforms, int64_t* tokens, int64_t ldt, int32_t* positions, double temperature,
                                 const float* temperatures, int top_k, const int32_t* top_ks, double top_p, const float* top_ps, double min_p,
                                 const float* min_ps, int B, int V, int dtype, void* stream) {
  const char* fn = "fsvd_sample_token";
  if (logits == nullptr || uniforms == nullptr || tokens == nullptr) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (B <= 0 || V <= 0 || V > kDrawRow) { set_last_error("%s: B = %d, V = %d (1 to %d logits are served)", fn, B, V, kDrawRow); return kErrBadShape; }
  if (dtype != 0 && dtype != 1) { set_last_error("%s: dtype code %d (bf16 = 0 and fp16 = 1 are served)", fn, dtype); return kErrBadDtype; }
  if ((reinterpret_cast<uintptr_t>(logits) & 1) != 0) { set_last_error("%s: logits must be 2-byte aligned", fn); return kErrBadAlign; }
  const SampleArgs a{static_cast<const uint16_t*>(logits), ld, uniforms, tokens, ldt, positions, temperature, top_p, min_p, top_k,
                     temperatures, top_ps, min_ps, top_ks, V};
  return dtype == 1 ? launch_sample<1>(fn, a, B, static_cast<hipStream_t>(stream)) : launch_sample<0>(fn, a, B, static_cast<hipStream_t>(stream));
}
