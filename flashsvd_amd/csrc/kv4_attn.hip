// Attention over the KV cache in 4 bits.
#include "kv4.hpp"

namespace fsvd {

// One query row of a head for a workgroup: scores of 256 keys at a time, one a thread, their weights against a running maximum, and the values of those keys by
// DH-fold threads.  Everything in fp32.
template <int DT, int DH>
__global__ __launch_bounds__(256) void kv4_attend_kernel(Kv4AttnArgs a) {
  typedef E16<DT> E;
  constexpr int HALF = DH / 2, GROUPS = DH / kGroup4, PARTS = 256 / DH;
  __shared__ float qs[DH], ws[256], red[4], os[PARTS][DH];
  const int tid = threadIdx.x, h = blockIdx.x, m = blockIdx.y, b = blockIdx.z, hk = h / (a.H / a.c.Hk);
  if (a.rows && m >= a.rows[b]) return;
  const int64_t at = (int64_t)a.positions[b] + m;
  const int keys = (int)max((int64_t)0, min(at + a.key_add, (int64_t)a.c.S));
  const uint16_t* q = a.q + (int64_t)b * a.sq_b + (int64_t)m * a.sq_m + (int64_t)h * a.sq_h;
  if (tid < DH) {
    float x = E::val(q[tid]);
    if (a.cos) {
      const int64_t tp = min(max(at, (int64_t)0), (int64_t)a.rope_len - 1) * HALF + tid % HALF;
      const float c = E::val(a.cos[tp]), s = E::val(a.sin[tp]), y = E::val(q[tid < HALF ? tid + HALF : tid - HALF]);
      x = x * c + (tid < HALF ? -y : y) * s;
    }
    qs[tid] = x * a.scale;
  }
  __syncthreads();
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* ks = static_cast<const uint8_t*>(a.c.k_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const uint8_t* vs = static_cast<const uint8_t*>(a.c.v_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const int d = tid % DH, part = tid / DH;
  float top = -INFINITY, sum = 0.f, o = 0.f;
  for (int n0 = 0; n0 < keys; n0 += 256) {
    const int n = n0 + tid;
    float s = -INFINITY;
    if (n < keys) {
      s = 0.f;
      for (int g = 0; g < GROUPS; ++g) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(kb + n * a.c.sc_s + 16 * g);
        const uint32_t byte = ks[g * a.c.ss_g + n];
        const float f = scale_of(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x2_t x[4] = {pair4_f32<0>(w[i], f), pair4_f32<1>(w[i], f), pair4_f32<2>(w[i], f), pair4_f32<3>(w[i], f)};
#pragma unroll
          for (int e = 0; e < 8; ++e) s += x[e >> 1][e & 1] * qs[32 * g + 8 * i + e];
        }
        if (byte == kNanByte) s = __builtin_nanf("");
      }
    }
    float most = wave_max(s);
    if ((tid & 63) == 0) red[tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), top);
    const float base = most == -INFINITY ? 0.f : most, keep = __expf(top - base);
    ws[tid] = n < keys ? __expf(s - base) : 0.f;
    top = most;
    __syncthreads();
    o *= keep; sum *= keep;
    for (int i = part; i < 256 && n0 + i < keys; i += PARTS) {
      const uint32_t byte = vs[d / kGroup4 * a.c.ss_g + n0 + i], code = vb[(int64_t)(n0 + i) * a.c.sc_s + d / 2];
      const f32x2_t x = pair4_f32<0>(code, scale_of(byte));
      o += ws[i] * (byte == kNanByte ? __builtin_nanf("") : d & 1 ? x[1] : x[0]);
      sum += ws[i];
    }
  }
  os[part][d] = o;
  __syncthreads();
  if (d == 0) ws[part] = sum;
  __syncthreads();
  if (part == 0) {
    for (int p = 1; p < PARTS; ++p) { o += os[p][d]; sum += ws[p]; }
    a.out[(int64_t)b * a.so_b + (int64_t)m * a.so_m + (int64_t)h * a.so_h + d] = (uint16_t)E::bits(keys == 0 ? 0.f : o / sum);
  }
}

int launch_kv4_attend(const char* fn, const Kv4AttnArgs& a, hipStream_t st) {
  if (a.M > 65535) { set_last_error("%s: %d rows", fn, a.M); return kErrBadShape; }
  const dim3 grid(a.H, a.M, a.B);
  if (a.dt == 1) {
    if (a.c.Dh == 128) hipLaunchKernelGGL((kv4_attend_kernel<1, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv4_attend_kernel<1, 64>), grid, dim3(256), 0, st, a);
  } else {
    if (a.c.Dh == 128) hipLaunchKernelGGL((kv4_attend_kernel<0, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv4_attend_kernel<0, 64>), grid, dim3(256), 0, st, a);
  }
  set_last_form("kv4 attend");
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

}  // namespace fsvd
