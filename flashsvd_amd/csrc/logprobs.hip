// Log probabilities of given tokens, the entropy of their distributions and the likeliest alternatives: with x_i = l_i - max l and Z = sum e^(x_i),
//   log p_t = x_t - log Z,  H = log Z - sum e^(x_i) x_i / Z,  and the `top` largest logits, equal ones by index.
// A row is read once, into the registers of a workgroup.  Each thread sums against the largest of its own logits, so that the sums need no maximum of the row;
// one exchange joins them and gives, as the k-th largest of the maxima of 64 parts of the row, a bound below which no alternative lies.  What is not below it is
// collected and ranked by counting.  Rows in which that is much (many equal logits, most of them masked) or that hold a NaN are gone over again, see below.
#include "common.hpp"
#include "../../include/flashsvd_hip.h"

namespace fsvd {

struct LogprobArgs {
  const uint16_t* logits; int64_t sl_b, sl_t;
  const int64_t* tokens;
  float* logprobs; float* entropy; int64_t* top_tokens; float* top_logprobs;
  int B, T, V, top;
};
constexpr int kMostTop = 64, kMostCands = 512;

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

// THREADS: of a workgroup; R: 16-byte pieces of the row that a thread keeps, 0: longer rows, which are read twice.
template <int DT, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(LogprobArgs a) {
  typedef E16<DT> E;
  constexpr int WAVES = THREADS / kWave;
  constexpr uint32_t kNegInf2 = DT == 1 ? 0xfc00fc00u : 0xff80ff80u;
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ uint64_t cand[kMostCands];                  // rank key, then the index from the largest down
  __shared__ uint32_t part_top[WAVES][kWave], counts[WAVES], n_cand;
  __shared__ float wave_m[WAVES], wave_z[WAVES], wave_zx[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.V, pieces = (V + 7) >> 3;
  const int64_t r = blockIdx.x;
  const uint16_t* row = a.logits + r / a.T * a.sl_b + r % a.T * a.sl_t;
  // eight logits; behind the row's end stands -inf
  const auto fetch = [&](int c) {
    if (c * 8 + 8 <= V) return __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(row + (int64_t)c * 8));
    uint32_t w[4] = {kNegInf2, kNegInf2, kNegInf2, kNegInf2};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c * 8 + e < V) w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | (uint32_t)row[c * 8 + e] << 16 : (w[e >> 1] & 0xffff0000u) | row[c * 8 + e];
    return u32x4_t{w[0], w[1], w[2], w[3]};
  };
  const int64_t token = tid == 0 ? a.tokens[r] : 0;
  const float given = tid == 0 && token >= 0 && token < V ? E::val(row[token]) : 0.f;
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
        if (m > -INFINITY) {                              // the sums move to the new largest
          const float d = m - to, f = __builtin_amdgcn_exp2f(d * kLog2e);
          zx = f * fmaf(d, z, zx);
          z *= f;
        }
        most = k;
        m = to;
      }
      add(v, m == -INFINITY ? 0.f : m);
    }
  }
  // joined over the wave, then over the waves, against the largest of all; parts without a weight stay out
  const auto join = [](float m, float& z, float& zx, float to) {
    const float d = fmaxf(m - to, -200.f), f = __builtin_amdgcn_exp2f(d * kLog2e);      // a NaN of m, or of m - to at infinity, is in z too
    zx = f * fmaf(d, z, zx);
    z *= f;
  };
  float to = wave_max(m);
  join(m, z, zx, to == -INFINITY ? 0.f : to);
  z = wave_sum(z);
  zx = wave_sum(zx);
  if (lane == 0) { wave_m[wave] = to; wave_z[wave] = z; wave_zx[wave] = zx; }
  part_top[wave][lane] = most;
  if (tid == 0) n_cand = 0;
  __syncthreads();
  const bool one = lane < WAVES;
  m = one ? wave_m[lane] : -INFINITY; z = one ? wave_z[lane] : 0.f; zx = one ? wave_zx[lane] : 0.f;
  to = wave_max(m);
  join(m, z, zx, to == -INFINITY ? 0.f : to);
  z = wave_sum(z);
  zx = wave_sum(zx);
  const bool finite = fabsf(to) < INFINITY && z == z;
  const float lz = finite ? to + logf(z) : __builtin_nanf("");            // log of the sum of all e^l
  if (tid == 0) {
    a.logprobs[r] = token < 0 ? 0.f : token >= V ? __builtin_nanf("") : finite ? (given - to) - logf(z) : lz;
    a.entropy[r] = finite ? logf(z) - zx / z : lz;
  }
  if (a.top == 0) return;

  // the bound: the k-th largest of the 64 parts' maxima
  uint32_t best = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) best = max(best, part_top[w][lane]);
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t t = bound | 1u << bit;
    if (__popcll(__ballot(best >= t)) >= a.top) bound = t;
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
    if (finite && count(low + 1) < a.top) high = low + 1;
#pragma unroll 1
    while (high - low > 1) {
      const uint32_t mid = (low + high) >> 1;
      if (count(mid) >= a.top) low = mid;
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
      if (equal < a.top) {                                // of the first pieces that hold any; uniform over the workgroup
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
        for (; which && at < (uint32_t)a.top; ++at) {     // from the list's end, where there is room behind those above
          const int e = __ffs(which) - 1;
          which &= which - 1;
          cand[kMostCands - 1 - at] = (uint64_t)low << 32 | (uint32_t)~(c * 8 + e);
        }
        equal += (int)all;
      }
    }
    __syncthreads();
    above = (int)n_cand;                                  // fewer than top
    n = a.top;
    for (int i = above + tid; i < n; i += THREADS) cand[i] = cand[kMostCands - 1 - (i - above)];
    __syncthreads();
  }
  for (int i = tid; i < n; i += THREADS) {
    const uint64_t mine = cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > mine;
    if (rank < a.top) {
      const int at = (int)~(uint32_t)mine;
      a.top_tokens[r * a.top + rank] = at;
      a.top_logprobs[r * a.top + rank] = finite ? (E::val(row[at]) - to) - logf(z) : __builtin_nanf("");
    }
  }
}

template <int DT, int THREADS>
static void launch_rows(const LogprobArgs& a, int pieces, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.T));
  if (pieces <= THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 1>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= 2 * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 2>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= 4 * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 4>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= 8 * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 8>), grid, dim3(THREADS), 0, st, a);
  else if (pieces <= 16 * THREADS) hipLaunchKernelGGL((token_logprobs_kernel<DT, THREADS, 16>), grid, dim3(THREADS), 0, st, a);
  else hipLaunchKernelGGL((token_logprobs_kernel<DT, 1024, 0>), grid, dim3(1024), 0, st, a);
}
template <int DT>
static void launch_logprobs(const LogprobArgs& a, hipStream_t st) {
  const int pieces = (a.V + 7) / 8;
  const bool narrow = (int64_t)a.B * a.T >= 512 && pieces <= 16 * 256;
  set_last_form(narrow ? "logprobs 256" : pieces <= 16 * 1024 ? "logprobs 1024" : "logprobs long");
  narrow ? launch_rows<DT, 256>(a, pieces, st) : launch_rows<DT, 1024>(a, pieces, st);
}

}  // namespace fsvd

using namespace fsvd;

extern "C" int fsvd_token_logprobs(const void* logits, int64_t sl_b, int64_t sl_t, const int64_t* tokens, float* logprobs, float* entropy, int64_t* top_tokens,
                                   float* top_logprobs, int B, int T, int V, int top, int dtype, void* stream) {
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
  const LogprobArgs a{static_cast<const uint16_t*>(logits), sl_b, sl_t, tokens, logprobs, entropy, top_tokens, top_logprobs, B, T, V, top};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  dtype == 1 ? launch_logprobs<1>(a, st) : launch_logprobs<0>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}
