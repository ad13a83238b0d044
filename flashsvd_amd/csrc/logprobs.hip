// Log probabilities of given tokens, the entropy of their distributions and the likeliest alternatives: with x_i = l_i - max l and Z = sum e^(x_i),
//   log p_t = x_t - log Z,  H = log Z - sum e^(x_i) x_i / Z,  and the `top` largest logits, equal ones by index.
#include "common.hpp"
#include "../../include/flashsvd_hip.h"

namespace fsvd {

struct LogprobArgs {
  const uint16_t* logits; int64_t sl_b, sl_t;
  const int64_t* tokens;
  float* logprobs; float* entropy; int64_t* top_tokens; float* top_logprobs;
  int B, T, V, top;
};
// patterns as numbers in the order of their values: the two zeros equal, every NaN above all else
template <int DT>
__device__ __forceinline__ uint32_t logit_key(uint32_t p) {
  const uint32_t mag = p & 0x7fffu;
  if (mag > (DT == 1 ? 0x7c00u : 0x7f80u)) return 0xffffu;
  if (mag == 0) return 0x8000u;
  return (p & 0x8000u) ? 0xffffu - p : p | 0x8000u;
}
constexpr int kLpThreads = 256;

template <int DT>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(LogprobArgs a) {
  typedef E16<DT> E;
  __shared__ float red[2][4];
  __shared__ unsigned long long best[4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t r = blockIdx.x;
  const uint16_t* row = a.logits + r / a.T * a.sl_b + r % a.T * a.sl_t;
  float top = -INFINITY;
  bool nan = false;
  for (int i = tid; i < a.V; i += kLpThreads) { const float x = E::val(row[i]); top = fmaxf(top, x); nan = nan || x != x; }
  top = wave_max(nan ? INFINITY : top);
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  __syncthreads();
  float z = 0.f, zx = 0.f;
  for (int i = tid; i < a.V; i += kLpThreads) {
    const float x = E::val(row[i]) - top, w = expf(x);
    z += w;
    zx += w > 0.f ? w * x : 0.f;
  }
  z = wave_sum(z); zx = wave_sum(zx);
  if (lane == 0) { red[0][wave] = z; red[1][wave] = zx; }
  __syncthreads();
  z = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
  zx = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const bool finite = fabsf(top) < INFINITY;
  const float lz = finite ? logf(z) : __builtin_nanf("");
  if (tid == 0) {
    const int64_t t = a.tokens[r];
    a.logprobs[r] = t < 0 ? 0.f : t >= a.V ? __builtin_nanf("") : E::val(row[t]) - top - lz;
    a.entropy[r] = lz - zx / z;
  }
  unsigned long long last = ~0ull;
  for (int n = 0; n < a.top; ++n) {
    unsigned long long mine = 0;
    for (int i = tid; i < a.V; i += kLpThreads) {
      const unsigned long long c = ((unsigned long long)logit_key<DT>(row[i]) << 32) | (0xffffffffu - (uint32_t)i);
      if (c < last && c > mine) mine = c;
    }
    for (int o = 32; o; o >>= 1) { const unsigned long long other = __shfl_xor(mine, o); mine = other > mine ? other : mine; }
    __syncthreads();
    if (lane == 0) best[wave] = mine;
    __syncthreads();
    for (int w = 0; w < 4; ++w) mine = best[w] > mine ? best[w] : mine;
    last = mine;
    if (tid == 0) {
      const uint32_t i = 0xffffffffu - (uint32_t)mine;
      a.top_tokens[r * a.top + n] = i;
      a.top_logprobs[r * a.top + n] = E::val(row[i]) - top - lz;
    }
  }
}

}  // namespace fsvd

using namespace fsvd;

extern "C" int fsvd_token_logprobs(const void* logits, int64_t sl_b, int64_t sl_t, const int64_t* tokens, float* logprobs, float* entropy, int64_t* top_tokens,
                                   float* top_logprobs, int B, int T, int V, int top, int dtype, void* stream) {
  const char* fn = "fsvd_token_logprobs";
  if (B < 0 || T < 0 || V <= 0 || V > (1 << 24) || top < 0 || top > 64 || top > V || (int64_t)B * T > 0x7fffffff) {
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
  if (dtype == 1) hipLaunchKernelGGL((token_logprobs_kernel<1>), dim3((unsigned)(B * T)), dim3(kLpThreads), 0, st, a);
  else hipLaunchKernelGGL((token_logprobs_kernel<0>), dim3((unsigned)(B * T)), dim3(kLpThreads), 0, st, a);
  set_last_form("logprobs");
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}
