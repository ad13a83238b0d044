// The next token drawn from filtered logits, one launch.  With the logits in descending order, equal ones by their index, and weights
// w_i = exp((l_i - l_0) / T), C_n = w_0 + .. + w_{n-1}:
//   n_k = top_k, n_p = the smallest n with C_n > top_p C_{n_k}, n_m = how many w >= min_p, N = the least of them; the token is the first whose
//   C exceeds u C_N.
// Every filter keeps a prefix of that order, and 16-bit logits have few distinct values, so nothing is sorted: the values of a row are counted in a
// histogram over their 65536 patterns in LDS, and an exponential is taken for each value that occurs, once, in 64 bits, as the sums are (a boundary between
// two of 10^5 nearly equal tokens is 10^-5 of the sum wide; with 32-bit sums one draw in a thousand lands on the wrong side of it).
// A row is one workgroup's, so latency bounds it.  Of the 12.3 us of 32000 logits with every filter on, reading and the largest take 1.9, counting 2.5 (LDS
// additions), the list of segments 1.1, their masses 2.1, the search by one wave 2.7, the token's place 0.7; 64 rows take 13.2, 16 rows of 128256 logits 28.
#include "common.hpp"
#include "../../include/flashsvd_hip.h"

namespace fsvd {

constexpr int kDrawThreads = 1024, kDrawWaves = kDrawThreads / kWave, kDrawRow = 1 << 24;
constexpr int kHistWords = 32768, kSegs = 1024, kSegBins = 64, kBatch = 8;      // two 16-bit counts a word; keys of a segment; segments of a wave
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
// e^x for -746 < x <= 0, to a few 2^-53, by the reduction of Cody and Waite: x = n ln 2 + r with ln 2 in two parts, the first of 41 bits (n has eleven), and
// the series of e^r to r^13 (|r| <= 0.347: the next term is 4e-18)
__device__ __forceinline__ double exp_below(double x) {
  const double n = rint(x * 1.4426950408889634074);
  double r = fma(n, -0.693147180559663, x);
  r = fma(n, -2.8235290563031577e-13, r);
  double y = 1. / 6227020800.;
#pragma unroll
  for (const double c : {1. / 479001600., 1. / 39916800., 1. / 3628800., 1. / 362880., 1. / 40320., 1. / 5040., 1. / 720., 1. / 120., 1. / 24., 1. / 6., .5, 1., 1.})
    y = fma(y, r, c);
  return ldexp(y, (int)n);
}
// the halves (or rows of 16 lanes, by pairs) of two values change places and are added
template <int LANES>
__device__ __forceinline__ double swap_add(double x, double y) {
  const u32x2_t a = __builtin_bit_cast(u32x2_t, x), b = __builtin_bit_cast(u32x2_t, y);
  const uint32_t al = a.x, ah = a.y, bl = b.x, bh = b.y;
  if constexpr (LANES == 32) {
    const auto l = __builtin_amdgcn_permlane32_swap(al, bl, false, false), h = __builtin_amdgcn_permlane32_swap(ah, bh, false, false);
    return __builtin_bit_cast(double, u32x2_t{l[0], h[0]}) + __builtin_bit_cast(double, u32x2_t{l[1], h[1]});
  } else {
    const auto l = __builtin_amdgcn_permlane16_swap(al, bl, false, false), h = __builtin_amdgcn_permlane16_swap(ah, bh, false, false);
    return __builtin_bit_cast(double, u32x2_t{l[0], h[0]}) + __builtin_bit_cast(double, u32x2_t{l[1], h[1]});
  }
}
__device__ __forceinline__ double row_sum(double v) {      // of 16 lanes, in each of them: rotations by 8, 4, 2, 1
  v = dpp_add<0x128, 0xf>(v);
  v = dpp_add<0x124, 0xf>(v);
  v = dpp_add<0x122, 0xf>(v);
  return dpp_add<0x121, 0xf>(v);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_most(uint32_t v) { return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false)); }
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {      // the steps of a running sum
  v = dpp_most<0x111, 0xf>(v);
  v = dpp_most<0x112, 0xf>(v);
  v = dpp_most<0x114, 0xf>(v);
  v = dpp_most<0x118, 0xf>(v);
  v = dpp_most<0x142, 0xa>(v);
  return lane_value(dpp_most<0x143, 0xc>(v), 63);
}

// R: 16-byte pieces of the row that a thread keeps in registers; 0: longer rows, read once for each pass (32000 logits: 13.1 us from registers, 16.3 read again;
// 128256: 28.1 and 33.3).  The smallest R that holds the row: 32000 logits with R = 16 take 30.8.
template <int DT, int R>
__global__ __launch_bounds__(kDrawThreads) void sample_token_kernel(SampleArgs a) {
  constexpr uint32_t kInf = DT == 1 ? 0x7c00u : 0x7f80u, kNegInf = kMinusZero - kInf, kLowest = kNegInf + 1, kHighest = kZero + kInf - 1;
  extern __shared__ __align__(16) uint32_t hist[];                       // [kHistWords]
  // the segments that hold something, from the largest values down: which, their masses, their counts with all before them
  __shared__ __align__(16) uint16_t seg_at[kSegs + kBatch];
  __shared__ double seg_mass[kSegs], group_mass[kDrawWaves];
  __shared__ uint32_t seg_count[kSegs], wave_a[kDrawWaves], wave_b[kDrawWaves], wave_kept[kDrawWaves], drawn_key, drawn_rank;
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
  // the row's numbers: asked for here, as a load that is waited for further down costs a round trip to memory
  const double temp = a.temperatures ? (double)a.temperatures[b] : a.temperature, top_p = a.top_ps ? (double)a.top_ps[b] : a.top_p;
  const double min_p = a.min_ps ? (double)a.min_ps[b] : a.min_p, u = (double)a.uniforms[b];
  const int top_k = a.top_ks ? a.top_ks[b] : a.top_k;
  for (int i = tid; i < kHistWords / 4; i += kDrawThreads) reinterpret_cast<u32x4_t*>(hist)[i] = u32x4_t{0u, 0u, 0u, 0u};
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

  uint32_t key = most, rank = 0;                        // the token: this occurrence of this key
  if (temp > 0. && !nan && most >= kLowest && most <= kHighest) {
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
    all_pieces([&](int r, u32x4_t v) {
      if (r * kDrawThreads + wave * kWave < pieces) count_up(v);          // not all behind the row
    });
    if (R == 0 || R > 8) {
      mine = wave_scan(mine);
      if (lane == 63) wave_kept[wave] = mine;
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
      if (s - kMinusZero / kSegBins <= 1) n = k == kMinusZero ? 0u : k == kZero ? n + bin(kMinusZero) : n;
      return n;
    };
    const double per = 1. / fmax(temp, 1e-280);
    const auto weight = [&](uint32_t k) { return exp_below(((double)key_value<DT>(k) - high) * per); };
    // what a thread's segment holds, read in an order that spreads the lanes over the banks
    const int last_seg = (int)(most / kSegBins), seg = kSegs - 1 - tid;
    const bool in_range = kSegs - wave * kWave > (int)(least / kSegBins) && kSegs - wave * kWave - kWave <= last_seg;
    const auto counted_here = [&] {
      uint32_t n = 0;
      if (in_range) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const u32x4_t w = reinterpret_cast<const u32x4_t*>(hist)[seg * 8 + ((j + (seg >> 1)) & 7)];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = w[e];
            n = __builtin_amdgcn_udot2(__builtin_bit_cast(u16x2_t, x), u16x2_t{1, 1}, n, false);
          }
        }
      }
      return n;
    };
    uint32_t here = counted_here();
    if (kMayRunOver) {
      // A 16-bit count runs over where more than 65535 logits are equal, and all of them come to less then than there are.  The row is counted again in
      // steps that cannot, and after each what exceeds 32767 is set aside.
      const uint32_t sum = lane_value(wave_scan(here), 63);
      if (lane == 0) wave_b[wave] = sum;
      __syncthreads();
      uint32_t there = 0, counted = 0;
      for (int i = 0; i < kDrawWaves; ++i) { there += wave_b[i]; counted += wave_kept[i]; }
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
        here = counted_here();
        for (uint32_t i = 0; i < extras; ++i) here += extra[i] / kSegBins == seg ? 32768u : 0u;
      }
    }
    if (seg == kMinusZero / kSegBins) here -= bin(kMinusZero);
    if (seg == kZero / kSegBins) here += bin(kMinusZero);
    const uint64_t some = __ballot(here != 0);
    const uint32_t run_here = wave_scan(here);
    if (kMayRunOver) __syncthreads();                     // all have read wave_b
    if (lane == 63) { wave_a[wave] = __popcll(some); wave_b[wave] = run_here; }
    __syncthreads();
    uint32_t segs = 0, run_c = 0, seg_before = 0, c_before = 0;
#pragma unroll
    for (int i = 0; i < kDrawWaves; ++i) {
      if (i == wave) { seg_before = segs; c_before = run_c; }
      segs += wave_a[i];
      run_c += wave_b[i];
    }
    if (here) {
      const uint32_t at = seg_before + __popcll(some & ((1ull << lane) - 1));
      seg_at[at] = (uint16_t)seg;
      seg_count[at] = c_before + run_here;
    }
    if (tid < kBatch) seg_at[segs + tid] = 0;             // a segment that is never counted
    __syncthreads();
    // Masses of the segments, eight at a time for a wave.  The values of a segment are evenly spaced, and those of all segments of an exponent alike, so a
    // key's weight is that of its segment's last one times what the way there makes: one exponential of a wave for its eight segments, and one for the lanes
    // at each exponent.  (In the segment of the largest, that one stands in for the last: its weight is 1 as it has to be, and nothing runs over.)
    uint32_t kept = 0;
    constexpr int kExponent = (DT == 1 ? 1024 : 128) / kSegBins;
    const auto below = [&](uint32_t k, double top) { return exp_below(fmin(fmax(((double)key_value<DT>(k) - top) * per, -700.), 0.)); };
    const auto last_key = [&](int s) { return s == last_seg ? most : (uint32_t)s * kSegBins + kSegBins - 1; };
    const int my = 2 * (lane >> 4) + (lane & 1);          // whose sum ends in this lane
    for (uint32_t b0 = wave * kBatch; b0 < segs; b0 += kDrawWaves * kBatch) {
      const uint16_t* counts16 = reinterpret_cast<const uint16_t*>(hist) + lane;
      int s[kBatch];
      uint32_t n[kBatch];
      const u32x4_t at = *reinterpret_cast<const u32x4_t*>(seg_at + b0);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t w = at[i >> 1];
        s[i] = __builtin_amdgcn_readfirstlane(i & 1 ? w >> 16 : w & 0xffffu);
        n[i] = counts16[s[i] * kSegBins];
      }
      const double seg_weight = below(last_key(seg_at[b0 + my]), high);
      double lane_weight = 0., m[kBatch];
      int exponent = -1;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t k = s[i] * kSegBins + lane;
        const int e = s[i] == last_seg ? kSegs : s[i] / kExponent;
        if (e != exponent) {
          exponent = e;
          lane_weight = below(k, (double)key_value<DT>(last_key(s[i])));
        }
        const uint32_t c = merged(s[i], k, counts(k, n[i]));
        if (min_p > 0.) kept += lane_weight * lane_value(seg_weight, (i >> 1) * 16 + (i & 1)) >= min_p ? c : 0;
        m[i] = c * lane_weight;
      }
      // sums over the lanes: halves, then rows of 16 lanes change places with those of another segment and are added; a row adds up by rotations
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = swap_add<32>(m[i], m[i + 4]);
#pragma unroll
      for (int i = 0; i < 2; ++i) m[i] = row_sum(swap_add<16>(m[i], m[i + 2]));
      if ((lane & 15) < 2 && b0 + my < segs) seg_mass[b0 + my] = (lane & 1 ? m[1] : m[0]) * seg_weight;
    }
    kept = wave_scan(kept);
    if (lane == 63) wave_kept[wave] = kept;
    __syncthreads();
    // running sums of groups of 64 segments, a wave each
    const double gm = wave_scan((uint32_t)tid < segs ? seg_mass[tid] : 0.);
    seg_mass[tid] = gm;
    if (lane == 63) group_mass[wave] = gm;
    __syncthreads();
    if (wave == 0) {
      double run_m = 0., to_m = 0.;                     // lane i: up to group i
      uint32_t likely = 0;
#pragma unroll
      for (int i = 0; i < kDrawWaves; ++i) {
        run_m += group_mass[i];
        likely += wave_kept[i];
        if (lane == i) to_m = run_m;
      }
      const bool is_group = lane * kWave < (int)segs;
      const uint32_t to_c = is_group ? seg_count[min(lane * kWave + kWave, (int)segs) - 1] : 0;
      // The n-th of the order, where n is the smallest with C_n > target (by_mass) or given: its key, how many of its key are up to it, n and C_n.  Where
      // rounding leaves no C above the target, the last that there is.
      uint32_t at_key = 0, at_rank = 0, at_n = 0;
      double at_mass = 0., w = 0., m = 0., to_mk = 0.;
      uint32_t k = 0, c = 0, to_ck = 0;
      int held = -1;
      const auto locate = [&](bool by_mass, double target, uint32_t n) {
        const auto first = [&](bool in, double m, uint32_t c) {
          const uint64_t hit = __ballot(in && (by_mass ? m > target : c >= n)), some = __ballot(in);
          return hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some | 1);
        };
        const int g = first(is_group, to_m, to_c);
        const double m0 = g ? lane_value(to_m, g - 1) : 0.;
        const uint32_t c0 = g ? lane_value(to_c, g - 1) : 0;
        const bool is_seg = (uint32_t)(g * kWave + lane) < segs;
        const double ms = m0 + seg_mass[g * kWave + lane];
        const uint32_t cs = is_seg ? seg_count[g * kWave + lane] : 0;
        const int t = first(is_seg, ms, cs);
        const double m1 = t ? lane_value(ms, t - 1) : m0;
        const uint32_t c1 = t ? lane_value(cs, t - 1) : c0;
        if (held != g * kWave + t) {                    // its keys from the largest down; the next search often ends in the same segment
          held = g * kWave + t;
          const uint32_t s = seg_at[held];
          k = s * kSegBins + kSegBins - 1 - lane;
          c = k >= least ? merged(s, k, bin(k)) : 0;
          w = c ? weight(k) : 0.;
          m = c * w;
          to_mk = wave_scan(m);
          to_ck = wave_scan(c);
        }
        const double mk = m1 + to_mk;
        const uint32_t ck = c1 + to_ck;
        const bool found = __any(c && (by_mass ? mk > target : ck >= n));
        const int l = first(c != 0, mk, ck);
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
  static std::atomic<uint32_t> granted{0};
  if (const int rc = grant_lds(fn, reinterpret_cast<const void*>(&sample_token_kernel<DT, R>), kHistWords * 4, granted)) return rc;
  set_last_form(R == 0 ? "draw" : R == 2 ? "draw 2" : R == 4 ? "draw 4" : R == 8 ? "draw 8" : "draw 16");
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
  if (B > 1 && ldt == 0) { set_last_error("%s: tokens must not be expanded", fn); return kErrBadShape; }
  if (dtype != 0 && dtype != 1) { set_last_error("%s: dtype code %d (bf16 = 0 and fp16 = 1 are served)", fn, dtype); return kErrBadDtype; }
  if ((reinterpret_cast<uintptr_t>(logits) & 1) != 0) { set_last_error("%s: logits must be 2-byte aligned", fn); return kErrBadAlign; }
  const SampleArgs a{static_cast<const uint16_t*>(logits), ld, uniforms, tokens, ldt, positions, temperature, top_p, min_p, top_k,
                     temperatures, top_ps, min_ps, top_ks, V};
  return dtype == 1 ? launch_sample_row<1>(fn, a, B, static_cast<hipStream_t>(stream)) : launch_sample_row<0>(fn, a, B, static_cast<hipStream_t>(stream));
}
