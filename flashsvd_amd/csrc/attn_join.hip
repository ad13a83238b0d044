// The results of key ranges joined.
#include "attn_join.hpp"

namespace fsvd {

// Weight of a range, below zero where it has no keys and so has written no values.  One that fp32 does not hold is 0: nothing of a number, and a NaN among the values stays one.
constexpr float kNoKeys = -1.f;
__device__ __forceinline__ float range_weight(float reference, float top) { return reference > -INFINITY ? __builtin_amdgcn_exp2f(reference - top) : kNoKeys; }
// The ranges of a row joined in their order, WPR waves for a row, each with every WPR-th range.  Rows of a decode call are (b, h), those of a chunk (b, kv head,
// token, head of the group).  Nothing that a load needs comes from another load: what it takes is a round trip to memory and its launch.
template <int DT, int DH, int WPR>
__global__ __launch_bounds__(256) void join_ranges_kernel(JoinArgs a, int ranges, bool decode, float* scratch) {
  typedef E16<DT> E;
  constexpr int D = DH / kWave, U = 8;
  __shared__ float vs[4][DH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part_of = wave % WPR, G = a.H / a.Hk;
  const int64_t rows = (int64_t)a.B * a.M * a.H, row = (int64_t)blockIdx.x * (4 / WPR) + wave / WPR;
  const bool live = row < rows;
  const int64_t at = live ? row : rows - 1;
  const RangeParts part{scratch, rows, ranges, DH};
  float v[D], sum = 0.f, top = -INFINITY;
#pragma unroll
  for (int i = 0; i < D; ++i) v[i] = 0.f;
  if (ranges > kWave)
    for (int s0 = 0; s0 < ranges; s0 += kWave) top = fmaxf(top, s0 + lane < ranges ? (*part.stats(at, s0 + lane))[0] : -INFINITY);
  for (int s0 = 0; s0 < ranges; s0 += kWave) {
    const int n = min(kWave, ranges - s0);
    const f32x2_t st = *part.stats(at, s0 + min(lane, n - 1));
    float w = kNoKeys;
    for (int s = part_of; s < n; s += WPR * U) {
      float x[U][D];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < D; ++i) x[u][i] = part.values(at, s0 + min(s + u * WPR, n - 1))[lane * D + i];
      if (s == part_of) {                                  // the weights, with the first values on their way
        if (s0 == 0) top = wave_max(fmaxf(top, lane < n ? st[0] : -INFINITY));
        w = lane < n ? range_weight(st[0], top) : kNoKeys;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float f = s + u * WPR < n ? __shfl(w, s + u * WPR) : kNoKeys;
#pragma unroll
        for (int i = 0; i < D; ++i) v[i] += f >= 0.f ? f * x[u][i] : 0.f;
      }
    }
    if (part_of >= n) {                                    // more waves than ranges: the sum all the same
      if (s0 == 0) top = wave_max(fmaxf(top, lane < n ? st[0] : -INFINITY));
      w = lane < n ? range_weight(st[0], top) : kNoKeys;
    }
    sum += fmaxf(w, 0.f) * st[1];
  }
  sum = wave_sum(sum);
  if (WPR > 1) {
#pragma unroll
    for (int i = 0; i < D; ++i) vs[wave][lane * D + i] = v[i];
    __syncthreads();
    if (part_of == 0) {
#pragma unroll
      for (int i = 0; i < D; ++i)
#pragma unroll
        for (int w = 1; w < WPR; ++w) v[i] += vs[wave + w][lane * D + i];
    }
  }
  const int b = (int)(at / ((int64_t)a.M * a.H)), in = (int)(at - (int64_t)b * a.M * a.H), hk = in / (a.M * G), r = in - hk * a.M * G;
  const int m = decode ? 0 : r / G, h = decode ? in : hk * G + r - m * G;
  if (!live || part_of || (a.rows && m >= a.rows[b])) return;
  uint16_t* o = a.out + (int64_t)b * a.so_b + (int64_t)m * a.so_m + (int64_t)h * a.so_h + lane * D;
#pragma unroll
  for (int i = 0; i < D; ++i) o[i] = (uint16_t)E::bits(sum == 0.f ? 0.f : v[i] / sum);
}
template <int DT, int DH>
static void launch_form(const JoinArgs& a, int ranges, bool decode, float* scratch, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.M * a.H;
  // 63 ranges of 32 rows: 13.9 us with the attention before it, 15.2 by one wave a row; 8 ranges of 512 rows: 27.5 by one wave, 28.5 by four
  if (ranges > 8) hipLaunchKernelGGL((join_ranges_kernel<DT, DH, 4>), dim3((unsigned)rows), dim3(256), 0, st, a, ranges, decode, scratch);
  else hipLaunchKernelGGL((join_ranges_kernel<DT, DH, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, ranges, decode, scratch);
}

void launch_join(const JoinArgs& a, int ranges, bool decode, float* scratch, hipStream_t st) {
  if (a.dt == 1) a.Dh == 128 ? launch_form<1, 128>(a, ranges, decode, scratch, st) : launch_form<1, 64>(a, ranges, decode, scratch, st);
  else a.Dh == 128 ? launch_form<0, 128>(a, ranges, decode, scratch, st) : launch_form<0, 64>(a, ranges, decode, scratch, st);
}

}  // namespace fsvd
