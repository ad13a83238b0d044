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
constexpr int kHistWords = 32768, kSegs = 1024, kSegBins = 64;      // two 16-bit counts a word; keys of a segment
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

// 16-bit patterns as unsigned numbers in the order of their values, two to a word: a negative pattern inverted, a positive one above all of them.  -0 comes
// out next below +0 (its count is moved there), a NaN beyond the infinity of its sign.
typedef double f64x4_t __attribute__((ext_vector_type(4)));
typedef short i16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
constexpr uint32_t kMinusZero = 0x7fffu, kZero = 0x8000u;
__device__ __forceinline__ uint32_t order_pair(uint32_t w) {
  const i16x2_t p = __builtin_bit_cast(i16x2_t, w);
  return __builtin_bit_cast(uint32_t, (i16x2_t)(p ^ ((p >> 15) | (short)0x8000)));
}
template <int DT>
__device__ __forceinline__ float key_value(uint32_t k) { return E16<DT>::val(k >= kZero ? k - kZero : 0xffffu - k); }

// running sums over the lanes of a wave (each lane with all before it), by register moves
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) { return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
  const u32x2_t w = __builtin_bit_cast(u32x2_t, v);
  return v + __builtin_bit_cast(double, u32x2_t{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, CTRL, ROWS, 0xf, false),
                                                (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, CTRL, ROWS, 0xf, false)});
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
  v = dpp_add<0x111, 0xf>(v);      // row_shr 1, 2, 4, 8, then the last lane of a row into the next rows
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);
  return dpp_add<0x143, 0xc>(v);
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ double lane_value(double v, int l) {
  const u32x2_t w = __builtin_bit_cast(u32x2_t, v);
  return __builtin_bit_cast(double, u32x2_t{(uint32_t)__builtin_amdgcn_readlane(w.x, l), (uint32_t)__builtin_amdgcn_readlane(w.y, l)});
}
// e^x for -746 < x <= 0, to a few 2^-53: x = n ln 2 + r, the series of e^r to r^13 (|r| <= 0.347: the next term is 4e-18)
__device__ __forceinline__ double exp_below(double x) {
  const double n = rint(x * 1.4426950408889634074);
  double r = fma(n, -6.93147180369123816490e-01, x);      // ln 2 in two parts, the first of 32 bits
  r = fma(n, -1.90821492927058770002e-10, r);
  double y = 1. / 6227020800.;
#pragma unroll
  for (const double c : {1. / 479001600., 1. / 39916800., 1. / 3628800., 1. / 362880., 1. / 40320., 1. / 5040., 1. / 720., 1. / 120., 1. / 24., 1. / 6., .5, 1., 1.})
    y = fma(y, r, c);
  return ldexp(y, (int)n);
}
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

// R: 16-byte pieces of the row that a thread keeps in registers; 0: longer rows, read once for each pass.
template <int DT, int R>
__global__ __launch_bounds__(kDrawThreads) void sample_token_kernel(SampleArgs a) {
  constexpr uint32_t kInf = DT == 1 ? 0x7c00u : 0x7f80u, kNegInf = kMinusZero - kInf, kLowest = kNegInf + 1, kHighest = kZero + kInf - 1;
  extern __shared__ __align__(16) uint32_t hist[];                       // [kHistWords]
  __shared__ double seg_mass[kSegs], group_mass[kDrawWaves];             // from the largest values down
  __shared__ uint32_t seg_count[kSegs], group_count[kDrawWaves], wave_a[kDrawWaves], wave_b[kDrawWaves], wave_kept[kDrawWaves], drawn_key, drawn_rank;
  __shared__ uint16_t extra[kMostExtra];                                  // keys that hold 32768 more than their bin says, once for each
  __shared__ uint32_t n_extra;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint16_t* row = a.logits + (int64_t)b * a.ld;
  const int V = a.V, pieces = (V + 7) >> 3, rounds = R > 0 ? R : (pieces + kDrawThreads - 1) / kDrawThreads;
  // eight logits as ordered numbers; behind the row's end stands -inf, which is never counted
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
  const auto ordered = [](u32x4_t v) { return u32x4_t{order_pair(v.x), order_pair(v.y), order_pair(v.z), order_pair(v.w)}; };
  u32x4_t held[R > 0 ? R : 1];
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) held[r] = fetch(r * kDrawThreads + tid);
  }
  const auto all_pieces = [&](auto f) {                                   // f(round, piece)
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) f(r, held[r]);
    } else {
      for (int r = 0; r < rounds; ++r) f(r, ordered(fetch(r * kDrawThreads + tid)));
    }
  };
  for (int i = tid; i < kHistWords / 4; i += kDrawThreads) reinterpret_cast<u32x4_t*>(hist)[i] = u32x4_t{0u, 0u, 0u, 0u};
  for (int i = tid; i < kSegs; i += kDrawThreads) { seg_mass[i] = 0.; seg_count[i] = 0; }
  if (tid == 0) n_extra = 0;
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) held[r] = ordered(held[r]);
  }

  // the largest, and the smallest: a NaN lies beyond the infinity of its sign
  u16x2_t up = {0, 0}, down = {0xffff, 0xffff};
  all_pieces([&](int, u32x4_t v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = v[i];                          // a bit cast of an element of a vector would take the first one
      up = __builtin_elementwise_max(up, __builtin_bit_cast(u16x2_t, w));
      down = __builtin_elementwise_min(down, __builtin_bit_cast(u16x2_t, w));
    }
  });
  {
    const uint32_t x = wave_most(max((uint32_t)up.x, (uint32_t)up.y)), y = wave_most(0xffffu - min((uint32_t)down.x, (uint32_t)down.y));
    if (lane == 0) { wave_a[wave] = x; wave_b[wave] = y; }
  }
  __syncthreads();
  uint32_t most = 0, deep = 0;
#pragma unroll
  for (int i = 0; i < kDrawWaves; ++i) { most = max(most, wave_a[i]); deep = max(deep, wave_b[i]); }
  const bool nan = most > kHighest + 1 || 0xffffu - deep < kNegInf;
  if (most == kMinusZero) most = kZero;

  const double temp = a.temperatures ? (double)a.temperatures[b] : a.temperature;
  uint32_t key = most, rank = 0;                        // the token: this occurrence of this key
  if (temp > 0. && !nan && most >= kLowest && most <= kHighest) {
    const double top_p = a.top_ps ? (double)a.top_ps[b] : a.top_p, min_p = a.min_ps ? (double)a.min_ps[b] : a.min_p, u = (double)a.uniforms[b];
    const int top_k = a.top_ks ? a.top_ks[b] : a.top_k;
    const double high = (double)key_value<DT>(most);
    // what is below e^-80 of the largest changes no sum of 64 bits and is not counted
    const double floor_ = high - 80. * temp;
    uint32_t least = kLowest;
    if (floor_ > (double)key_value<DT>(kLowest)) least = max(kLowest, order_pair(E16<DT>::bits((float)floor_)) & 0xffffu);
    uint32_t mine = 0;                                  // counted by this thread
    const auto count_up = [&](u32x4_t v) {
      u16x2_t low = {0xffff, 0xffff};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = v[i];
        low = __builtin_elementwise_min(low, __builtin_bit_cast(u16x2_t, w));
      }
      const auto add = [&](uint32_t k) { atomicAdd(&hist[k >> 1], 1u + (k & 1u) * 0xffffu); };
      if (__all(min((uint32_t)low.x, (uint32_t)low.y) >= least)) {        // nothing of the wave's pieces is left out
        mine += 8;
#pragma unroll
        for (int i = 0; i < 4; ++i) { add(v[i] & 0xffffu); add(v[i] >> 16); }
      } else {
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = e < 4 ? (e < 2 ? v[0] : v[1]) : (e < 6 ? v[2] : v[3]), k = e & 1 ? w >> 16 : w & 0xffffu;
          if (k >= least) { add(k); ++mine; }
        }
      }
    };
    all_pieces([&](int, u32x4_t v) { count_up(v); });
    if (R == 0 || R > 8) {
      mine = wave_scan(mine);
      if (lane == 63) wave_a[wave] = mine;
    }
    __syncthreads();
    constexpr bool kMayRunOver = R == 0 || R > 8;        // rows of more than 65535
    uint32_t extras = 0;
    const auto counts = [&](uint32_t k, uint32_t n) {     // of key k whose bin holds n
      for (uint32_t i = 0; kMayRunOver && i < extras; ++i) n += extra[i] == k ? 32768u : 0u;
      return n;
    };
    const auto bin = [&](uint32_t k) { return counts(k, (hist[k >> 1] >> (16 * (k & 1))) & 0xffffu); };
    // the count of -0 belongs to 0
    const auto merged = [&](uint32_t s, uint32_t k, uint32_t n) {
      if (s == kMinusZero / kSegBins) return k == kMinusZero ? 0u : n;
      if (s == kZero / kSegBins) return k == kZero ? n + bin(kMinusZero) : n;
      return n;
    };
    const double per = 1. / fmax(temp, 1e-280);
    const auto weight = [&](uint32_t k) { return exp_below(((double)key_value<DT>(k) - high) * per); };
    if (kMayRunOver) {
      // A 16-bit count runs over where more than 65535 logits are equal, and all of them come to less then than there are.  The row is counted again in
      // steps that cannot, and after each what exceeds 32767 is set aside.
      uint32_t there = 0, sum = 0, counted = 0;
#pragma unroll
      for (int i = 0; i < kHistWords / 4; i += kDrawThreads) {
        const u32x4_t w = reinterpret_cast<const u32x4_t*>(hist)[i + tid];
        sum += (w.x & 0xffffu) + (w.x >> 16) + (w.y & 0xffffu) + (w.y >> 16) + (w.z & 0xffffu) + (w.z >> 16) + (w.w & 0xffffu) + (w.w >> 16);
      }
      sum = lane_value(wave_scan(sum), 63);
      if (lane == 0) wave_b[wave] = sum;
      __syncthreads();
      for (int i = 0; i < kDrawWaves; ++i) { there += wave_b[i]; counted += wave_a[i]; }
      if (there != counted) {
        for (int i = tid; i < kHistWords; i += kDrawThreads) hist[i] = 0;
        for (int c0 = 0; c0 < pieces; c0 += 4095) {
          __syncthreads();
          for (int c = c0 + tid; c < min(c0 + 4095, pieces); c += kDrawThreads) count_up(ordered(fetch(c)));
          __syncthreads();
          for (int i = tid; i < kHistWords; i += kDrawThreads) {
            const uint32_t w = hist[i];
            if (w & 0x8000u) extra[atomicAdd(&n_extra, 1u)] = (uint16_t)(2 * i);
            if (w & 0x80000000u) extra[atomicAdd(&n_extra, 1u)] = (uint16_t)(2 * i + 1);
            hist[i] = w & 0x7fff7fffu;
          }
        }
        __syncthreads();
        extras = n_extra;
      }
    }
    // Sums over segments of 64 keys.  A wave asks for the counts of every 16th of 256 segments at once (those that hold something stand side by side, so
    // the waves share them); the sums over the lanes come from the matrix cores, in 64 bits: a segment's masses are the rows, and a column of ones puts
    // their sums into the segment's own column.
    uint32_t kept = 0;
    constexpr int kAsk = 16, kStep = kAsk * kDrawWaves;
    const int last_seg = (int)(most / kSegBins);
    for (int s0 = (int)(least / kSegBins) / kStep * kStep + wave; s0 <= last_seg; s0 += kStep) {
      const uint16_t* counts16 = reinterpret_cast<const uint16_t*>(hist) + s0 * kSegBins + lane;
      constexpr int kNext = kDrawWaves * kSegBins;
      uint32_t raw[kAsk];
#pragma unroll
      for (int i = 0; i < kAsk; ++i) raw[i] = counts16[i * kNext];
      uint32_t some = 0;                                  // segments with a count, and those whose counts are not all in their bins
#pragma unroll
      for (int i = 0; i < kAsk; ++i) some |= __any(raw[i] != 0) ? 1u << i : 0u;
      const auto also = [&](int s) {
        s -= s0;
        if (s >= 0 && s < kStep && s % kDrawWaves == 0) some |= 1u << (s / kDrawWaves);
      };
      also(kZero / kSegBins);
      for (uint32_t i = 0; kMayRunOver && i < extras; ++i) also(extra[i] / kSegBins);
      f64x4_t mass = {0., 0., 0., 0.};
      f32x4_t count = {0.f, 0.f, 0.f, 0.f};               // whole numbers up to 2^24
      while (some) {
        const int i = __builtin_ctz(some), s = s0 + i * kDrawWaves;
        some &= some - 1;
        const uint32_t k = s * kSegBins + lane, n = merged(s, k, counts(k, counts16[i * kNext]));
        const bool own = (lane & 15) == i;
        const double w = n ? weight(k) : 0.;
        if (min_p > 0.) kept += w >= min_p ? n : 0;
        mass = __builtin_amdgcn_mfma_f64_16x16x4f64(n * w, own ? 1. : 0., mass, 0, 0, 0);
        count = __builtin_amdgcn_mfma_f32_16x16x4f32((float)n, own ? 1.f : 0.f, count, 0, 0, 0);
      }
      double m = (mass[0] + mass[1]) + (mass[2] + mass[3]);
      float c = (count[0] + count[1]) + (count[2] + count[3]);
      m += __shfl_xor(m, 16); c += __shfl_xor(c, 16);
      m += __shfl_xor(m, 32); c += __shfl_xor(c, 32);
      if (lane < kAsk) {
        const int at = kSegs - 1 - (s0 + lane * kDrawWaves);
        seg_mass[at] = m;
        seg_count[at] = (uint32_t)c;
      }
    }
    kept = wave_scan(kept);
    if (lane == 63) wave_kept[wave] = kept;
    __syncthreads();
    // running sums of groups of 64 segments, a wave each
    const double gm = wave_scan(seg_mass[tid]);
    const uint32_t gc = wave_scan(seg_count[tid]);
    seg_mass[tid] = gm;
    seg_count[tid] = gc;
    if (lane == 63) { group_mass[wave] = gm; group_count[wave] = gc; }
    __syncthreads();
    if (wave == 0) {
      double run_m = 0., to_m = 0.;                     // lane i: up to group i
      uint32_t run_c = 0, to_c = 0, likely = 0;
#pragma unroll
      for (int i = 0; i < kDrawWaves; ++i) {
        run_m += group_mass[i];
        run_c += group_count[i];
        likely += wave_kept[i];
        if (lane == i) { to_m = run_m; to_c = run_c; }
      }
      // The n-th of the order, where n is the smallest with C_n > target (by_mass) or given: its key, how many of its key are up to it, n and C_n.  Where
      // rounding leaves no C above the target, the last that there is.
      uint32_t at_key = 0, at_rank = 0, at_n = 0;
      double at_mass = 0.;
      const auto locate = [&](bool by_mass, double target, uint32_t n) {
        const auto first = [&](bool in, double m, uint32_t c, uint32_t before) {
          const uint64_t hit = __ballot(in && (by_mass ? m > target : c >= n)), some = __ballot(in && c > before);
          return hit ? __builtin_ctzll(hit) : some ? 63 - __builtin_clzll(some) : 0;
        };
        const auto shifted = [&](uint32_t c) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)c, 0x138, 0xf, 0xf, false); };      // from the lane before
        const int g = first(lane < kDrawWaves, to_m, to_c, shifted(to_c));
        const double m0 = g ? lane_value(to_m, g - 1) : 0.;
        const uint32_t c0 = g ? lane_value(to_c, g - 1) : 0;
        const double ms = m0 + seg_mass[g * kWave + lane];
        const uint32_t cs = c0 + seg_count[g * kWave + lane], cp = shifted(cs);
        const int t = first(true, ms, cs, lane ? cp : c0);
        const double m1 = t ? lane_value(ms, t - 1) : m0;
        const uint32_t c1 = t ? lane_value(cs, t - 1) : c0;
        const uint32_t k = (kSegs - 1 - (g * kWave + t)) * kSegBins + kSegBins - 1 - lane, c = k >= least ? merged(k / kSegBins, k, bin(k)) : 0;
        const double w = c ? weight(k) : 0., m = c * w, mk = m1 + wave_scan(m);
        const uint32_t ck = c1 + wave_scan(c);
        const bool found = __any(c && (by_mass ? mk > target : ck >= n));
        const int l = first(c != 0, mk, ck, ck - c);
        uint32_t j = c;
        if (found) j = by_mass ? (uint32_t)fmin(fmax(floor((target - (mk - m)) / w), 0.) + 1., (double)c) : n - (ck - c);
        at_key = lane_value(k, l);
        at_rank = lane_value(j, l);
        at_n = lane_value(ck - c + j, l);
        at_mass = lane_value(mk - m + j * w, l);
      };
      uint32_t keep = top_k > 0 && (uint32_t)top_k < run_c ? (uint32_t)top_k : run_c;
      double z = run_m;
      if (keep < run_c) { locate(false, 0., keep); z = at_mass; }
      uint32_t n = keep;
      if (top_p < 1.) { locate(true, top_p * z, 0); n = min(n, at_n); }
      if (min_p > 0.) n = min(n, likely);
      n = max(n, 1u);
      if (n < run_c) { if (n != at_n) locate(false, 0., n); z = at_mass; }
      locate(true, u * z, 0);
      if (at_n > n) locate(false, 0., n);
      if (lane == 0) { drawn_key = at_key; drawn_rank = at_rank - 1; }
    }
    __syncthreads();
    key = drawn_key;
    rank = drawn_rank;
  }

  // that occurrence, by index: how many a wave has in each of its pieces, then the piece, then the element
  __syncthreads();
  const uint32_t lo = nan ? kHighest + 2 : key == kZero ? kMinusZero : key, span = nan ? 0xffffu - (kHighest + 2) + kNegInf : key == kZero ? 1 : 0;
  const auto hits = [&](u32x4_t v, auto f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (((v[i] - lo) & 0xffffu) <= span) f(2 * i);
      if ((((v[i] >> 16) - lo) & 0xffffu) <= span) f(2 * i + 1);
    }
  };
  const u16x2_t first = {(unsigned short)lo, (unsigned short)lo};
  uint32_t sums = 0;                                      // of up to three rounds, ten bits each (512 of a wave at most)
  all_pieces([&](int r, u32x4_t v) {
    uint32_t n = 0;
    u16x2_t least_off = {0xffff, 0xffff};                 // distance from the key, two elements to an instruction
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = v[i];
      least_off = __builtin_elementwise_min(least_off, (u16x2_t)(__builtin_bit_cast(u16x2_t, w) - first));
    }
    if (__any(min((uint32_t)least_off.x, (uint32_t)least_off.y) <= span)) hits(v, [&](int) { ++n; });
    sums |= n << (10 * (r % 3));
    if (r % 3 == 2 || r == rounds - 1) {
      sums = wave_scan(sums);
      if (lane == 63)
        for (int q = r - r % 3; q <= r; ++q) hist[q * kDrawWaves + wave] = (sums >> (10 * (q % 3))) & 0x3ffu;
      sums = 0;
    }
  });
  __syncthreads();
  if (wave != 0) return;
  uint32_t before = 0;
  for (int i0 = 0; i0 < rounds * kDrawWaves; i0 += kWave) {
    const uint32_t n = i0 + lane < rounds * kDrawWaves ? hist[i0 + lane] : 0, s = before + wave_scan(n);
    const uint64_t hit = __ballot(s > rank);
    if (hit == 0) { before = lane_value(s, 63); continue; }
    const int l = __builtin_ctzll(hit), c = (i0 + l) * kWave + lane;
    before = lane_value(s - n, l);
    const u32x4_t v = ordered(fetch(c));
    uint32_t m = 0;
    hits(v, [&](int) { ++m; });
    uint32_t at = before + wave_scan(m) - m;
    if (at <= rank && rank < at + m) {
      hits(v, [&](int e) { if (at++ == rank) a.tokens[(int64_t)b * a.ldt] = (int64_t)c * 8 + e; });
      if (a.positions) a.positions[b] += 1;
    }
    return;
  }
}

template <int DT, int R>
static int launch_sample(const char* fn, const SampleArgs& a, int B, hipStream_t st) {
  static bool granted = false;
  if (!granted) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&sample_token_kernel<DT, R>), hipFuncAttributeMaxDynamicSharedMemorySize, kHistWords * 4);
    if (e != hipSuccess) { set_last_error("%s: cannot reserve %d bytes of LDS: %s", fn, kHistWords * 4, hipGetErrorString(e)); return kErrLaunch; }
    granted = true;
  }
  hipLaunchKernelGGL((sample_token_kernel<DT, R>), dim3(B), dim3(kDrawThreads), kHistWords * 4, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

template <int DT>
static int launch_sample_row(const char* fn, const SampleArgs& a, int B, hipStream_t st) {
  constexpr int kRound = kDrawThreads * 8;
  if (a.V <= 2 * kRound) return launch_sample<DT, 2>(fn, a, B, st);
  if (a.V <= 4 * kRound) return launch_sample<DT, 4>(fn, a, B, st);
  if (a.V < 8 * kRound) return launch_sample<DT, 8>(fn, a, B, st);       // at most 65535: no count can run over
  if (a.V <= 16 * kRound) return launch_sample<DT, 16>(fn, a, B, st);
  return launch_sample<DT, 0>(fn, a, B, st);
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
  return dtype == 1 ? launch_sample_row<1>(fn, a, B, static_cast<hipStream_t>(stream)) : launch_sample_row<0>(fn, a, B, static_cast<hipStream_t>(stream));
}
