// Log probabilities of given tokens, the entropy of their distributions and the likeliest alternatives: with x_i = l_i - max l and Z = sum e^(x_i),
//   log p_t = x_t - log Z,  H = log Z - sum e^(x_i) x_i / Z,  and the `top` largest logits, equal ones by index.
// A row is read once, into the registers of a workgroup (from 2097153 logits on twice, by parts that no registers hold).  Each thread sums against the largest of its own logits, so that the sums need no maximum of the row;
// one exchange joins them and gives, as the k-th largest of the maxima of groups of the row's logits, a bound below which no alternative lies.  What is not below it is
// collected and ranked by counting.  Rows in which that is much (many equal logits, most of them masked) or that hold a NaN are gone over again, see below.
// All times here are of a call in a captured graph of six over three sets of inputs.  4096 rows of 32000 logits in bf16: 56 to 61 us on different machines, 4.3 to 4.7
// TB/s of the 5.4 that a copy reaches; 64 rows of 128256, in parts, 12.4 us; 1 row of 32000 with 20 alternatives 8.9 us, with 5 8.0.
#include "common.hpp"
#include "../../include/flashsvd_hip.h"

namespace fsvd {

struct LogprobArgs {
  const uint16_t* logits; int64_t sl_b, sl_t;
  const int64_t* tokens;
  float* logprobs; float* entropy; int64_t* top_tokens; float* top_logprobs;
  int B, T, V, top;
  int parts, part;                     // workgroups of a row, 8-logit pieces of each
  f32x4_t* sums; uint64_t* cands;      // of the parts: (largest, Z, sum e^x x); `top` candidates [row][part][top], 0: none
};
constexpr int kMostTop = 64, kMostCands = 512, kMostParts = 16, kMostHeld = 16;       // kMostHeld: pieces that a thread keeps

// 16-bit patterns as unsigned numbers in the order of their values, two to a word: -0 comes out next below +0, a NaN beyond the infinity of its sign
typedef short i16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
constexpr uint32_t kMinusZero = 0x7fffu, kZero = 0x8000u;
__device__ __forceinline__ uint32_t order_pair(uint32_t w) {
  const i16x2_t p = __builtin_bit_cast(i16x2_t, w);
  return __builtin_bit_cast(uint32_t, (i16x2_t)(p ^ ((p >> 15) | (short)0x8000)));
}
template <int DT>
__device__ __forceinline__ float key_value(uint32_t k) { return E16<DT>::val(k >= kZero ? k - kZero : 0xffffu - k); }
// the same with the zeros equal and every NaN above all else
template <int DT>
__device__ __forceinline__ uint32_t rank_key(uint32_t k) {
  constexpr uint32_t inf = DT == 1 ? 0x7c00u : 0x7f80u;
  return k > kZero + inf || k < kMinusZero - inf ? 0xffffu : k == kMinusZero ? kZero : k;
}

// Sums against their own largest, m, as sums against another.  Where the distance is beyond the numbers (logits at the type's lowest value, the usual mask, below others)
// it counts as 200, whose power is nothing already: 0 times its product with z would be a NaN.
__device__ __forceinline__ void move_sums(float m, float& z, float& zx, float to) {
  constexpr float kLog2e = 1.4426950408889634f;
  const float d = fmaxf(m - to, -200.f), f = __builtin_amdgcn_exp2f(d * kLog2e);        // a NaN of m, or of m - to at infinity, is in z too
  zx = f * fmaf(d, z, zx);
  z *= f;
}
__device__ __forceinline__ void join_lanes(float& m, float& z, float& zx) {
  const float to = wave_max(m);
  move_sums(m, z, zx, to == -INFINITY ? 0.f : to);
  m = to;
  z = wave_sum(z);
  zx = wave_sum(zx);
}
// how many of n candidates are above one; zeros stand behind them, eight at a time are read
constexpr int kRanked = 8;
__device__ __forceinline__ int rank_of(const uint64_t* cand, int n, uint64_t mine) {
  typedef uint64_t u64x2_t __attribute__((ext_vector_type(2)));
  int rank = 0;
  for (int j = 0; j < n; j += kRanked) {
    u64x2_t c[kRanked / 2];
#pragma unroll
    for (int i = 0; i < kRanked / 2; ++i) c[i] = *reinterpret_cast<const u64x2_t*>(cand + j + 2 * i);
#pragma unroll
    for (int i = 0; i < kRanked / 2; ++i) rank += (c[i].x > mine) + (c[i].y > mine);
  }
  return rank;
}
template <int DT>
__device__ __forceinline__ float put_sums(const LogprobArgs& a, int64_t r, int64_t token, float given, float m, float z, float zx, bool& finite, bool writes) {
  finite = fabsf(m) < INFINITY && z == z;
  const float lz = logf(z), none = __builtin_nanf("");
  if (writes) {
    a.logprobs[r] = token < 0 ? 0.f : token >= a.V || !finite ? none : (given - m) - lz;
    a.entropy[r] = finite ? lz - zx / z : none;
  }
  return lz;
}

// THREADS: of a workgroup; R: 16-byte pieces of the row that a thread keeps, 0: longer rows, which are read twice.  PART: a workgroup has a part of the row and leaves
// its sums and candidates.
template <int DT, int THREADS, int R, bool PART>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(LogprobArgs a) {
  typedef E16<DT> E;
  constexpr int WAVES = THREADS / kWave;
  constexpr uint32_t kNegInf2 = DT == 1 ? 0xfc00fc00u : 0xff80ff80u;
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ __align__(16) uint64_t cand[kMostCands + kRanked];      // rank key, then the index from the largest down
  __shared__ uint32_t part_top[WAVES][kWave], counts[WAVES], n_cand;
  __shared__ float wave_m[WAVES], wave_z[WAVES], wave_zx[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = PART ? blockIdx.x / (uint32_t)a.parts : blockIdx.x;
  const int first = PART ? (int)(blockIdx.x - r * a.parts) * a.part * 8 : 0, V = PART ? min(a.V - first, a.part * 8) : a.V, pieces = (V + 7) >> 3;
  const int top = PART ? min(a.top, V) : a.top;
  const uint16_t* row = a.logits + r / a.T * a.sl_b + r % a.T * a.sl_t + first;
  // eight logits; behind the row's end stands -inf
  const auto fetch = [&](int c) {
    if (c * 8 + 8 <= V) {
      const u32x4_any_t* p = reinterpret_cast<const u32x4_any_t*>(row + (int64_t)c * 8);
      return __builtin_bit_cast(u32x4_t, R > 0 ? __builtin_nontemporal_load(p) : *p);       // read once: past the caches (64 rows of 128256 12.4 us, 13.0 through them; 4096 of 32000 and 300 of 6000 within 4 % either way)
    }
    uint32_t w[4] = {kNegInf2, kNegInf2, kNegInf2, kNegInf2};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c * 8 + e < V) w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | (uint32_t)row[c * 8 + e] << 16 : (w[e >> 1] & 0xffff0000u) | row[c * 8 + e];
    return u32x4_t{w[0], w[1], w[2], w[3]};
  };
  const int64_t token = !PART && tid == 0 ? a.tokens[r] : 0;
  const float given = !PART && tid == 0 && token >= 0 && token < V ? E::val(row[token]) : 0.f;
  u32x4_t held[R > 0 ? R : 1];
  float m = -INFINITY, z = 0.f, zx = 0.f;
  uint32_t most = 0;
  const auto largest = [&](u32x4_t v) {
    u16x2_t up = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) up = __builtin_elementwise_max(up, __builtin_bit_cast(u16x2_t, order_pair(v[i])));
    return max((uint32_t)up.x, (uint32_t)up.y);
  };
  const auto add = [&](u32x4_t v, float base) {           // a logit of -inf has weight zero and counts for nothing in zx; a NaN makes NaN of both
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = (e & 1 ? E::hi(v[e >> 1]) : E::lo(v[e >> 1])) - base, w = __builtin_amdgcn_exp2f(d * kLog2e);
      z += w;
      zx = fmaf(w, fmaxf(d, -200.f), zx);
    }
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) held[i] = i * THREADS + tid < pieces ? fetch(i * THREADS + tid) : u32x4_t{kNegInf2, kNegInf2, kNegInf2, kNegInf2};
#pragma unroll
    for (int i = 0; i < R; ++i) most = max(most, largest(held[i]));
    m = key_value<DT>(most);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      asm volatile("" : "+v"(held[i]));                   // the logits alone stay in registers, not what was made of them
      add(held[i], base);
      asm volatile("" : "+v"(held[i]));
    }
  } else {
    for (int c = tid; c < pieces; c += THREADS) {
      const u32x4_t v = fetch(c);
      const uint32_t k = largest(v);
      if (k > most) {
        const float to = key_value<DT>(k);
        if (m > -INFINITY) move_sums(m, z, zx, to);
        most = k;
        m = to;
      }
      add(v, m == -INFINITY ? 0.f : m);
    }
  }
  // joined over the wave, then over the waves, against the largest of all; lanes without a weight stay out
  join_lanes(m, z, zx);
  if (lane == 0) { wave_m[wave] = m; wave_z[wave] = z; wave_zx[wave] = zx; }
  part_top[wave][lane] = most;
  if (tid == 0) n_cand = 0;
  for (int i = tid; i < kMostCands + kRanked; i += THREADS) cand[i] = 0;
  __syncthreads();
  const bool one = lane < WAVES;
  m = one ? wave_m[lane] : -INFINITY; z = one ? wave_z[lane] : 0.f; zx = one ? wave_zx[lane] : 0.f;
  join_lanes(m, z, zx);
  bool finite;
  float lz = 0.f;
  if constexpr (PART) {
    finite = z == z;                                      // of a part of -inf alone too: its keys are in order
    if (tid == 0) a.sums[blockIdx.x] = f32x4_t{m, z, zx, 0.f};
  } else {
    lz = put_sums<DT>(a, r, token, given, m, z, zx, finite, tid == 0);
  }
  if (a.top == 0) return;

  // the bound: the k-th largest of the maxima of 64 groups, the lanes', or, of many alternatives, of four times as many: fewer logits are above it then
  const int sets = top > 32 ? 4 : 1;
  uint32_t best[4] = {0, 0, 0, 0}, bound = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (sets == 1) best[0] = max(best[0], part_top[w][lane]);
    else best[w & 3] = max(best[w & 3], part_top[w][lane]);
  }
#pragma unroll
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t t = bound | 1u << bit;
    int n = __popcll(__ballot(best[0] >= t));
    if (sets > 1) n += __popcll(__ballot(best[1] >= t)) + __popcll(__ballot(best[2] >= t)) + __popcll(__ballot(best[3] >= t));
    if (n >= top) bound = t;
  }
  if (bound == kZero) bound = kMinusZero;
  const auto put = [&](uint32_t key, int i) {
    const uint32_t at = atomicAdd(&n_cand, 1u);
    if (at < kMostCands) cand[at] = (uint64_t)rank_key<DT>(key) << 32 | (uint32_t)~i;
  };
  const auto collect = [&](u32x4_t v, int c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t w = order_pair(v[e >> 1]), k = e & 1 ? w >> 16 : w & 0xffffu;
      if (k >= bound && c * 8 + e < V) put(k, c * 8 + e);
    }
  };
  if (finite && most >= bound) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i * THREADS + tid < pieces && largest(held[i]) >= bound) collect(held[i], i * THREADS + tid);
    } else {
      for (int c = tid; c < pieces; c += THREADS) {
        const u32x4_t v = fetch(c);
        if (largest(v) >= bound) collect(v, c);
      }
    }
  }
  __syncthreads();
  int n = (int)n_cand;
  if (!finite || n > kMostCands) {
    // Gone over again: the k-th largest key by bisection (mostly the bound is it), what lies above it in any order, and of those equal to it the first ones, piece
    // after piece.
    const auto count = [&](uint32_t least) {
      uint32_t mine = 0;
      for (int c = tid; c < pieces; c += THREADS) {
        const u32x4_t v = fetch(c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = order_pair(v[e >> 1]);
          mine += rank_key<DT>(e & 1 ? w >> 16 : w & 0xffffu) >= least && c * 8 + e < V;
        }
      }
      mine = (uint32_t)wave_sum((float)mine);             // up to 2^24 in all
      __syncthreads();
      if (lane == 0) counts[wave] = mine;
      __syncthreads();
      uint32_t all = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) all += counts[w];
      return (int)all;
    };
    uint32_t low = finite ? rank_key<DT>(bound) : 0, high = 0x10000u;     // the k-th largest is at least `low` and below `high`
    if (finite && count(low + 1) < top) high = low + 1;
#pragma unroll 1
    while (high - low > 1) {
      const uint32_t mid = (low + high) >> 1;
      if (count(mid) >= top) low = mid;
      else high = mid;
    }
    __syncthreads();
    if (tid == 0) n_cand = 0;
    __syncthreads();
    int equal = 0, above = -1;                            // taken so far; how many lie above
#pragma unroll 1
    for (int c0 = 0; c0 < pieces; c0 += THREADS) {
      const int c = c0 + tid;
      uint32_t mine = 0, which = 0;
      if (c < pieces) {
        const u32x4_t v = fetch(c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = order_pair(v[e >> 1]), k = e & 1 ? w >> 16 : w & 0xffffu, q = rank_key<DT>(k);
          if (c * 8 + e < V) {
            if (q > low) put(k, c * 8 + e);
            if (q == low) { ++mine; which |= 1u << e; }
          }
        }
      }
      if (equal < top) {                                // of the first pieces that hold any; uniform over the workgroup
        uint32_t before = mine;                           // with those of the lanes before
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
          const uint32_t o = __shfl_up(before, d);
          if (lane >= d) before += o;
        }
        __syncthreads();
        if (lane == 63) counts[wave] = before;
        __syncthreads();
        uint32_t at = equal + before - mine, all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          if (w < wave) at += counts[w];
          all += counts[w];
        }
        for (; which && at < (uint32_t)top; ++at) {     // from the list's end, where there is room behind those above
          const int e = __ffs(which) - 1;
          which &= which - 1;
          cand[kMostCands - 1 - at] = (uint64_t)low << 32 | (uint32_t)~(c * 8 + e);
        }
        equal += (int)all;
      }
    }
    __syncthreads();
    above = (int)n_cand;                                  // fewer than top
    n = top;
    for (int i = above + tid; i < n; i += THREADS) cand[i] = cand[kMostCands - 1 - (i - above)];
    __syncthreads();
    if (tid < kRanked) cand[n + tid] = 0;
    __syncthreads();
  }
  uint64_t* out = PART ? a.cands + (int64_t)blockIdx.x * a.top : nullptr;
  for (int i = tid; i < n; i += THREADS) {
    const uint64_t mine = cand[i];
    const int rank = rank_of(cand, n, mine);
    if (rank >= top) continue;
    const int at = (int)~(uint32_t)mine;
    if constexpr (PART) {
      out[rank] = (mine >> 32 << 32) | (uint32_t)~(first + at);
    } else {
      a.top_tokens[r * a.top + rank] = at;
      a.top_logprobs[r * a.top + rank] = finite ? (key_value<DT>((uint32_t)(mine >> 32)) - m) - lz : __builtin_nanf("");
    }
  }
  if constexpr (PART)
    for (int i = top + tid; i < a.top; i += THREADS) out[i] = 0;
}

// The parts' sums and candidates.
template <int DT>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
  __shared__ __align__(16) uint64_t cand[kMostParts * kMostTop + kRanked];
  const int tid = threadIdx.x, lane = tid & 63, n = a.parts * a.top;
  const int64_t r = blockIdx.x, token = a.tokens[r];
  const uint16_t* row = a.logits + r / a.T * a.sl_b + r % a.T * a.sl_t;
  const float given = token >= 0 && token < a.V ? E16<DT>::val(row[token]) : 0.f;
  for (int i = tid; i < n + kRanked; i += 256) cand[i] = i < n ? a.cands[r * n + i] : 0;
  const f32x4_t part = lane < a.parts ? a.sums[r * a.parts + lane] : f32x4_t{-INFINITY, 0.f, 0.f, 0.f};
  float m = part[0], z = part[1], zx = part[2];
  join_lanes(m, z, zx);
  bool finite;
  const float lz = put_sums<DT>(a, r, token, given, m, z, zx, finite, tid == 0);
  __syncthreads();
  for (int i = tid; i < n; i += 256) {
    const uint64_t mine = cand[i];
    const int rank = rank_of(cand, n, mine);
    if (rank >= a.top || mine == 0) continue;
    a.top_tokens[r * a.top + rank] = (int)~(uint32_t)mine;
    a.top_logprobs[r * a.top + rank] = finite ? (key_value<DT>((uint32_t)(mine >> 32)) - m) - lz : __builtin_nanf("");
  }
}

template <int DT, int THREADS, bool PART>
static void launch_rows(const LogprobArgs& a, int pieces, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.T * a.parts));
  if (pieces <= THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 1, PART>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= 2 * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 2, PART>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= 4 * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 4, PART>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= 8 * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 8, PART>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= kMostHeld * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, kMostHeld, PART>), grid, dim3(THREADS), 0, st, a);
  else if constexpr (PART) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 0, true>), grid, dim3(THREADS), 0, st, a);
}
// Workgroups of a row.  A row of more than 4 pieces a thread has more work than one compute unit should do while others are idle: up to one workgroup for each, of
// 2000 pieces at least, whose join is a launch of its own (64 rows of 128256 logits: 19.1 us in one, 12.4 in 4; 1 row 16.3 and 9.1 in 8; 1 of 50000 10.6 and 10.1 in
// 3; of 32000, four a thread, 8.9 and 9.8 in 2, 64 of them 9.0 and 10.3).  And so many that a part stays in registers (200 rows of 500000 in 4: 73 us, 89 read twice).
static int row_parts(int64_t rows, int V) {
  const int pieces = (V + 7) / 8;
  if (pieces <= 4 * 1024) return 1;
  const int idle = (int)min((int64_t)(256 / rows), (int64_t)pieces / 2000), held = (pieces + kMostHeld * 1024 - 1) / (kMostHeld * 1024);
  return max(1, min(kMostParts, max(idle, held)));
}
static size_t part_bytes(int64_t rows, int parts, int top) { return parts == 1 ? 0 : rows * parts * (sizeof(f32x4_t) + top * sizeof(uint64_t)); }
template <int DT>
static void launch_logprobs(const LogprobArgs& a, hipStream_t st) {
  if (a.parts > 1) {
    set_last_form(a.part > kMostHeld * 1024 ? "logprobs long parts" : "logprobs parts");
    launch_rows<DT, 1024, true>(a, a.part, st);
    hipLaunchKernelGGL((logprobs_join_kernel<DT>), dim3((unsigned)(a.B * a.T)), dim3(256), 0, st, a);
    return;
  }
  // More rows than compute units: workgroups of four waves, several to a unit, whose phases overlap (4096 rows of 32000 logits 61 us, in sixteen waves 105; 300 of 6000
  // 7.2 and 9.8; but 256 of 32000 11.0 and 10.1).  So few logits that four waves hold them in two pieces a thread: less to join (8 rows of 1000: 5.0 and 5.8 us).
  const bool narrow = ((int64_t)a.B * a.T > 256 || a.part <= 512) && a.part <= kMostHeld * 256;
  set_last_form(narrow ? "logprobs 256" : "logprobs 1024");
  narrow ? launch_rows<DT, 256, false>(a, a.part, st) : launch_rows<DT, 1024, false>(a, a.part, st);
}

}  // namespace fsvd

using namespace fsvd;

extern "C" size_t fsvd_token_logprobs_scratch_bytes(int B, int T, int V, int top) {
  if (B <= 0 || T <= 0 || V <= 0 || V > (1 << 24) || top < 0 || top > kMostTop || (int64_t)B * T > 0x7fffffff) return 0;
  return part_bytes((int64_t)B * T, row_parts((int64_t)B * T, V), top);
}

extern "C" int fsvd_token_logprobs(const void* logits, int64_t sl_b, int64_t sl_t, const int64_t* tokens, float* logprobs, float* entropy, int64_t* top_tokens,
                                   float* top_logprobs, void* scratch, size_t scratch_bytes, int B, int T, int V, int top, int dtype, void* stream) {
  const char* fn = "fsvd_token_logprobs";
  if (B < 0 || T < 0 || V <= 0 || V > (1 << 24) || top < 0 || top > kMostTop || top > V || (int64_t)B * T > 0x7fffffff) {
    set_last_error("%s: %d x %d rows of %d logits, %d alternatives (up to 2^24 logits and 64 alternatives)", fn, B, T, V, top);
    return kErrBadShape;
  }
  if (dtype != 0 && dtype != 1) { set_last_error("%s: dtype code %d (bf16 = 0 and fp16 = 1 are served)", fn, dtype); return kErrBadDtype; }
  if (B == 0 || T == 0) return kOk;
  if (logits == nullptr || tokens == nullptr || logprobs == nullptr || entropy == nullptr || (top > 0 && (top_tokens == nullptr || top_logprobs == nullptr))) {
    set_last_error("%s: a buffer is NULL", fn);
    return kErrNullPtr;
  }
  if (reinterpret_cast<uintptr_t>(logits) & 1) { set_last_error("%s: logits at an odd address", fn); return kErrBadAlign; }
  const int64_t rows = (int64_t)B * T;
  const int pieces = (V + 7) / 8, want = row_parts(rows, V), part = (pieces + want - 1) / want, parts = (pieces + part - 1) / part;
  if (rows * parts >= 1 << 22) {                           // 2^32 threads of a launch
    set_last_error("%s: %lld rows in %d parts (fewer than 4194304 of both are served)", fn, (long long)rows, parts);
    return kErrBadShape;
  }
  const size_t need = part_bytes(rows, parts, top);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15))) {
    set_last_error("%s: %zu bytes of scratch for %d parts of a row, %zu needed", fn, scratch ? scratch_bytes : (size_t)0, parts, need);
    return kErrWorkspace;
  }
  f32x4_t* sums = static_cast<f32x4_t*>(scratch);
  const LogprobArgs a{static_cast<const uint16_t*>(logits), sl_b, sl_t, tokens, logprobs, entropy, top_tokens, top_logprobs, B, T, V, top, parts, part, sums,
                      parts > 1 ? reinterpret_cast<uint64_t*>(sums + rows * parts) : nullptr};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  dtype == 1 ? launch_logprobs<1>(a, st) : launch_logprobs<0>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}
