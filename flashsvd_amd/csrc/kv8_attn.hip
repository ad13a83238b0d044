// Attention over the KV cache in 8 bits.
#include "kv8.hpp"

namespace fsvd {

// One wave for a query row of one head: every key's score by a sum over the lanes, the running maximum and sum of the softmax.
template <int DT>
__global__ __launch_bounds__(64) void kv8_attend_kernel(Kv8AttnArgs a) {
  typedef E16<DT> E;
  const int m = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x, half = a.c.Dh >> 1;
  if (a.rows && m >= a.rows[b]) return;
  const int hk = h / (a.H / a.c.Hk), pos = a.positions[b] + m;
  const int keys = max(0, min(pos + a.key_add, a.c.S));
  const uint16_t* q = a.q + (int64_t)b * a.sq_b + (int64_t)m * a.sq_m + (int64_t)h * a.sq_h;
  // dimensions lane and lane + half of this lane (the first half lanes alone where half is 32)
  float q0 = 0.f, q1 = 0.f;
  const bool in = lane < half;
  if (in) {
    q0 = E::val(q[lane]); q1 = E::val(q[lane + half]);
    if (a.cos) {
      const int64_t tp = min(max(pos, 0), a.rope_len - 1);
      const float c = E::val(a.cos[tp * half + lane]), n = E::val(a.sin[tp * half + lane]);
      const float y0 = q0 * c - q1 * n, y1 = q0 * n + q1 * c;
      q0 = y0; q1 = y1;
    }
  }
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h + (in ? lane : 0);
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h + (in ? lane : 0);
  const float* ks = a.c.k_scale + b * a.c.ss_b + hk * a.c.ss_h;
  const float* vs = a.c.v_scale + b * a.c.ss_b + hk * a.c.ss_h;
  float top = -INFINITY, sum = 0.f, o0 = 0.f, o1 = 0.f;
  for (int n = 0; n < keys; ++n) {
    const uint8_t* k = kb + (int64_t)n * a.c.sc_s;
    const auto kk = codes_lo((uint32_t)k[0] | (uint32_t)k[half] << 8);
    const float s = wave_sum(q0 * kk[0] + q1 * kk[1]) * ks[(int64_t)(n / a.c.block) * a.c.ss_n] * a.scale;
    const float now = fmaxf(top, s), w = __expf(s - now), keep = __expf(top - now);
    const uint8_t* v = vb + (int64_t)n * a.c.sc_s;
    const auto vv = codes_lo((uint32_t)v[0] | (uint32_t)v[half] << 8);
    const float f = w * vs[(int64_t)(n / a.c.block) * a.c.ss_n];
    o0 = o0 * keep + f * vv[0];
    o1 = o1 * keep + f * vv[1];
    sum = sum * keep + w;
    top = now;
  }
  if (!in) return;
  uint16_t* o = a.out + (int64_t)b * a.so_b + (int64_t)m * a.so_m + (int64_t)h * a.so_h;
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  o[lane] = (uint16_t)E::bits(o0 * inv);
  o[lane + half] = (uint16_t)E::bits(o1 * inv);
}

int launch_kv8_attend(const char* fn, const Kv8AttnArgs& a, hipStream_t st) {
  if (a.H > 65535) { set_last_error("%s: %d query heads", fn, a.H); return kErrBadShape; }
  const dim3 grid(a.M, a.H, a.B);
  if (a.dt == 1) hipLaunchKernelGGL(kv8_attend_kernel<1>, grid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL(kv8_attend_kernel<0>, grid, dim3(64), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

}  // namespace fsvd
