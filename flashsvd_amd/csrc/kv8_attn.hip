// Attention over the KV cache in 8 bits.
#include "kv8.hpp"

namespace fsvd {

// ---------------------------------------------------------------------------------------------
// One query token per sequence.  A workgroup takes a range of the keys of one kv head for up to 16 of its query heads, a wave every fourth step of 32
// keys, on the matrix cores: S^T = K Q^T, O^T = V^T P^T (16 x 16 x 32).
//   K: lane (n, g) = (lane % 16, lane / 16) loads 16-byte pieces of key n: the order of the products' k axis is free as long as q is laid out the same.
//   S^T leaves lane (n, g) the scores of query n and keys 4 g .. 4 g + 3 of the two 16-key tiles: eight weights that are one operand of the second product.
//   V: lane (n, g) loads those eight keys' dimensions DH / 16 n .. of the row, and byte permutes put two keys of a dimension next to each other.
// Codes become 16-bit elements exactly; a scale multiplies what one tile of 16 keys has in common, the scores and the weights.
// ---------------------------------------------------------------------------------------------
constexpr int kMinRange = 256;                            // keys of a range, but for the last
__host__ __device__ __forceinline__ int kv8_range(int keys, int ranges) {
  const int per = (keys + ranges - 1) / ranges;
  return per < kMinRange ? kMinRange : (per + 127) / 128 * 128;
}
constexpr int kDecWaves = 4, kDecStep = 32, kDecGroup = 16;

template <int DT, int DH>
__global__ __launch_bounds__(kDecWaves * kWave) void kv8_decode_kernel(Kv8AttnArgs a, int ranges, float* scratch) {
  typedef E16<DT> E;
  typedef typename E::frag_t frag_t;
  typedef E16<0>::frag_t pfrag_t;
  constexpr int J = DH / 64, ST = DH / 32, NT = DH / 16, VW = DH / 64;      // 16-byte pieces of a key; products a tile; output tiles; words of a value piece
  __shared__ float os[kDecWaves][kDecGroup][DH + 4], ms[kDecWaves][kDecGroup], ls[kDecWaves][kDecGroup];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  const int G = a.H / a.c.Hk, GG = (G + kDecGroup - 1) / kDecGroup;
  int id = blockIdx.x;
  const int s = id % ranges; id /= ranges;
  const int gg = id % GG; id /= GG;
  const int hk = id % a.c.Hk, b = id / a.c.Hk;
  const int pos = a.positions[b], keys = max(0, min(pos + a.key_add, a.c.S));
  const int per = kv8_range(keys, ranges), k0 = min(s * per, keys), k1 = min(k0 + per, keys);
  if (k0 >= k1 && s > 0) return;
  const int h0 = hk * G + gg * kDecGroup, heads = min(kDecGroup, G - gg * kDecGroup);

  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h + g * 16;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h + n * NT;
  const float* ksp = a.c.k_scale + b * a.c.ss_b + hk * a.c.ss_h;
  const float* vsp = a.c.v_scale + b * a.c.ss_b + hk * a.c.ss_h;
  const int shift = 31 - __builtin_clz(a.c.block);
  u32x4_t kr[2][J];
  uint32_t vr[8][VW];
  float ks[2], vs[2];
  const auto fetch_k = [&](int c0) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* p = kb + (int64_t)min(c0 + 16 * t + n, k1 - 1) * a.c.sc_s;
#pragma unroll
      for (int j = 0; j < J; ++j) kr[t][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p + 64 * j));
      ks[t] = ksp[(int64_t)(min(c0 + 16 * t, k1 - 1) >> shift) * a.c.ss_n];
    }
  };
  const auto fetch_v = [&](int c0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t* p = vb + (int64_t)min(c0 + 16 * (e >> 2) + 4 * g + (e & 3), k1 - 1) * a.c.sc_s;
      if constexpr (VW == 2) {
        const u32x2_t w = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(p));
        vr[e][0] = w.x; vr[e][1] = w.y;
      } else {
        vr[e][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) vs[t] = vsp[(int64_t)(min(c0 + 16 * t, k1 - 1) >> shift) * a.c.ss_n];
  };
  int c0 = k0 + wave * kDecStep;
  if (c0 < k1) { fetch_k(c0); fetch_v(c0); }

  // q: element e of piece (j, h) is dimension 64 j + 16 g + 8 h + e of query n, rotated in fp32 and rounded to the type of the products
  frag_t qf[ST];
  {
    const uint16_t* qp = a.q + (int64_t)b * a.sq_b + (int64_t)(h0 + min(n, heads - 1)) * a.sq_h;
    constexpr int HALF = DH / 2;
    const int64_t tp = a.cos ? (int64_t)min(max(pos, 0), a.rope_len - 1) * HALF : 0;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      const int d = 64 * (st >> 1) + 16 * g + 8 * (st & 1);
      u32x4_t x = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(qp + d));
      if (a.cos) {
        const bool up = d >= HALF;
        const int dt = up ? d - HALF : d;
        const u32x4_t y = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(qp + (up ? d - HALF : d + HALF)));
        const u32x4_t cw = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(a.cos + tp + dt));
        const u32x4_t sw = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(a.sin + tp + dt));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sl = up ? E::lo(sw[i]) : -E::lo(sw[i]), sh = up ? E::hi(sw[i]) : -E::hi(sw[i]);
          x[i] = E::pack2(E::lo(x[i]) * E::lo(cw[i]) + E::lo(y[i]) * sl, E::hi(x[i]) * E::hi(cw[i]) + E::hi(y[i]) * sh);
        }
      }
      if (n >= heads) x = u32x4_t{0u, 0u, 0u, 0u};
      qf[st] = __builtin_bit_cast(frag_t, x);
    }
  }

  const float scale = a.scale * 1.4426950408889634f;      // weights are powers of two of the scores' differences
  float m = -INFINITY, l = 0.f;
  f32x4_t o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (; c0 < k1; c0 += kDecWaves * kDecStep) {
    const int next = c0 + kDecWaves * kDecStep;
    float x[2][4], f[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w0 = kr[t][j][2 * h], w1 = kr[t][j][2 * h + 1];
          const u32x4_t kk{Code16<DT>::template pair<false>(w0), Code16<DT>::template pair<true>(w0), Code16<DT>::template pair<false>(w1),
                           Code16<DT>::template pair<true>(w1)};
          acc = E::mfma(__builtin_bit_cast(frag_t, kk), qf[2 * j + h], acc);
        }
      const float by = ks[t] * scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[t][i] = acc[i] * by;
      f[t] = vs[t];
    }
    if (next < k1) fetch_k(next);
    if (c0 + kDecStep > k1) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = c0 + 16 * t + 4 * g + i < k1 ? x[t][i] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    top = fmaxf(m, column_max(top));
    if (__any(top > m)) {
      const float keep = __builtin_amdgcn_exp2f(m - top);                  // 0 in front of the first step
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] *= keep;
      l *= keep;
      m = top;
    }
    uint32_t ph[4], pl[4];                                // the weights as a 16-bit part and what it leaves
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float w0 = __builtin_amdgcn_exp2f(x[t][2 * i] - m), w1 = __builtin_amdgcn_exp2f(x[t][2 * i + 1] - m);
        l += w0 + w1;
        w0 *= f[t]; w1 *= f[t];
        ph[2 * t + i] = pack_bf16x2(w0, w1);
        pl[2 * t + i] = pack_bf16x2(w0 - bf16_lo(ph[2 * t + i]), w1 - bf16_hi(ph[2 * t + i]));
      }
    const pfrag_t hi = __builtin_bit_cast(pfrag_t, u32x4_t{ph[0], ph[1], ph[2], ph[3]}), lo = __builtin_bit_cast(pfrag_t, u32x4_t{pl[0], pl[1], pl[2], pl[3]});
#pragma unroll
    for (int w = 0; w < VW; ++w)
#pragma unroll
      for (int c = 0; c < 2; ++c) {                       // dimensions 4 w + 2 c and + 1 of the piece
        uint32_t two[4];                                  // keys 2 i, 2 i + 1 of the first, then of the second
#pragma unroll
        for (int i = 0; i < 4; ++i) two[i] = __builtin_amdgcn_perm(vr[2 * i + 1][w], vr[2 * i][w], c ? 0x07030602u : 0x05010400u);
        const u32x4_t v0{Code16<0>::pair<false>(two[0]), Code16<0>::pair<false>(two[1]), Code16<0>::pair<false>(two[2]), Code16<0>::pair<false>(two[3])};
        const u32x4_t v1{Code16<0>::pair<true>(two[0]), Code16<0>::pair<true>(two[1]), Code16<0>::pair<true>(two[2]), Code16<0>::pair<true>(two[3])};
        const int t = 4 * w + 2 * c;
        o[t] = E16<0>::mfma(__builtin_bit_cast(pfrag_t, v0), hi, o[t]);
        o[t] = E16<0>::mfma(__builtin_bit_cast(pfrag_t, v0), lo, o[t]);
        o[t + 1] = E16<0>::mfma(__builtin_bit_cast(pfrag_t, v1), hi, o[t + 1]);
        o[t + 1] = E16<0>::mfma(__builtin_bit_cast(pfrag_t, v1), lo, o[t + 1]);
      }
    if (next < k1) fetch_v(next);
  }
  // the waves' results through LDS: element i of tile t is dimension NT (4 g + i) + t of query n
  l = column_sum(l);
  if (g == 0) { ms[wave][n] = m; ls[wave][n] = l; }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) os[wave][n][NT * (4 * g + i) + t] = o[t][i];
  __syncthreads();
  const bool whole = per >= keys;                          // a single range
  for (int e = tid; e < heads * DH; e += kDecWaves * kWave) {
    const int q = e / DH, d = e % DH;
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) top = fmaxf(top, ms[w][q]);
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
      const float f = ms[w][q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[w][q] - top);
      sum += f * ls[w][q];
      v += f * os[w][q][d];
    }
    if (whole) {
      a.out[(int64_t)b * a.so_b + (int64_t)(h0 + q) * a.so_h + d] = (uint16_t)E::bits(sum > 0.f ? v / sum : 0.f);
    } else {
      float* part = scratch + ((int64_t)(b * a.H + h0 + q) * ranges + s) * (DH + 2);
      part[d] = v;
      if (d == 0) { part[DH] = top; part[DH + 1] = sum; }
    }
  }
}

// The ranges of a head joined, in their order.
template <int DT, int DH>
__global__ __launch_bounds__(DH) void kv8_join_kernel(Kv8AttnArgs a, int ranges, const float* scratch) {
  typedef E16<DT> E;
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const int keys = max(0, min(a.positions[b] + a.key_add, a.c.S)), per = kv8_range(keys, ranges);
  if (per >= keys) return;                                 // written by its only workgroup
  const int used = (keys + per - 1) / per;
  const float* part = scratch + (int64_t)(b * a.H + h) * ranges * (DH + 2);
  float top = -INFINITY, sum = 0.f, v = 0.f;
  for (int s = 0; s < used; ++s) top = fmaxf(top, part[s * (DH + 2) + DH]);
  for (int s = 0; s < used; ++s) {
    const float f = __builtin_amdgcn_exp2f(part[s * (DH + 2) + DH] - top);
    sum += f * part[s * (DH + 2) + DH + 1];
    v += f * part[s * (DH + 2) + d];
  }
  a.out[(int64_t)b * a.so_b + (int64_t)h * a.so_h + d] = (uint16_t)E::bits(sum > 0.f ? v / sum : 0.f);
}

int kv8_ranges(int B, int H, int Hk, int S, int nsplit) {
  const int most = (S + kMinRange - 1) / kMinRange;
  if (nsplit <= 0) {
    const int64_t pairs = (int64_t)B * Hk * ((H / Hk + kDecGroup - 1) / kDecGroup);
    nsplit = (int)((1024 + pairs - 1) / pairs);
  }
  return max(1, min(nsplit, most));
}
size_t kv8_scratch_bytes(int B, int H, int Dh, int ranges) { return ranges > 1 ? (size_t)B * H * ranges * (Dh + 2) * sizeof(float) : 0; }

template <int DT, int DH>
static void decode_form(const Kv8AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  const int groups = (a.H / a.c.Hk + kDecGroup - 1) / kDecGroup;
  hipLaunchKernelGGL((kv8_decode_kernel<DT, DH>), dim3((unsigned)a.B * a.c.Hk * groups * ranges), dim3(kDecWaves * kWave), 0, st, a, ranges, scratch);
  if (ranges > 1) hipLaunchKernelGGL((kv8_join_kernel<DT, DH>), dim3(a.H, a.B), dim3(DH), 0, st, a, ranges, scratch);
}
int launch_kv8_decode(const char* fn, const Kv8AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  if (a.dt == 1) a.c.Dh == 128 ? decode_form<1, 128>(a, ranges, scratch, st) : decode_form<1, 64>(a, ranges, scratch, st);
  else a.c.Dh == 128 ? decode_form<0, 128>(a, ranges, scratch, st) : decode_form<0, 64>(a, ranges, scratch, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

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
