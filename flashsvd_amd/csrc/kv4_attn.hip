// Attention over the KV cache in 4 bits.
#include "attn_join.hpp"
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


static JoinArgs join_args(const Kv4AttnArgs& a) { return {a.out, a.so_b, a.so_m, a.so_h, a.rows, a.B, a.M, a.H, a.c.Hk, a.c.Dh, a.dt}; }

// Eight elements of a query row, rotated in fp32 (y: those half a head away; sign: -1 in the lower half; not rotated: cosines 1, y and sines 0), as two bf16 parts:
// 16 significant bits.
template <class E>
__device__ __forceinline__ void query_parts(u32x4_t x, u32x4_t y, u32x4_t cos, u32x4_t sin, float sign, u32x4_t& high, u32x4_t& rest) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float l = E::lo(x[i]) * E::lo(cos[i]) + E::lo(y[i]) * (sign * E::lo(sin[i])), h = E::hi(x[i]) * E::hi(cos[i]) + E::hi(y[i]) * (sign * E::hi(sin[i]));
    const uint32_t w = pack_bf16x2(l, h);
    high[i] = w;
    rest[i] = pack_bf16x2(l - bf16_lo(w), h - bf16_hi(w));
  }
}

// Keys of a decode range, but for the last: a step of every wave.
constexpr int kDec4Waves = 4, kDec4Step = 64, kDec4Group = 16, kMinRange4 = kDec4Waves * kDec4Step;
__host__ __device__ __forceinline__ int kv4_range(int keys, int ranges) {
  const int per = (keys + ranges - 1) / ranges;
  return (max(per, 1) + kMinRange4 - 1) / kMinRange4 * kMinRange4;
}

// ---------------------------------------------------------------------------------------------
// One query token per sequence.  A workgroup takes a range of the keys of one kv head for up to 16 of its query heads, a wave every fourth step of 64
// keys, on the matrix cores in bf16: S^T = K Q^T, O^T = V^T P^T (16 x 16 x 32).
//   K: lane (n, g) = (lane % 16, lane / 16) loads the Dh / 4 channels from Dh / 4 g on of keys 4 n .. 4 n + 3, one for each of four tiles: its scales are four
//   bytes next to each other.  S^T then leaves it the scores of query n and keys 16 g .. 16 g + 15.
//   V: the lane loads channels Dh / 16 n .. of those 16 keys, whose scales are 16 bytes next to each other; a pair of codes becomes a pair of elements, scale
//   included, and byte permutes put two keys of a channel next to each other.
// q and the weights go into the products as two bf16 parts, 16 significant bits: of up to eight heads (HALVES) the second parts are columns 8 to 15 of the same
// products, of more they are products of their own.  The cache's rooms are whole steps, so nothing is clamped: rows behind the last
// key are read and their codes and scores replaced.
// ---------------------------------------------------------------------------------------------
template <int DT, int DH, bool HALVES>
__global__ __launch_bounds__(kDec4Waves * kWave, 3) void kv4_decode_kernel(Kv4AttnArgs a, int ranges, float* scratch) {
  typedef E16<DT> E;
  typedef E16<0> P;
  typedef P::frag_t frag_t;
  constexpr int CH = DH / 4, KW = CH / 8, ST = DH / 32, NT = DH / 16, HALF = DH / 2;      // channels and words of a lane's key; products a tile; output tiles
  extern __shared__ __align__(16) float os[];                               // [kDec4Waves][heads of a workgroup][DH + 4]
  __shared__ float ms[kDec4Waves][kDec4Group], ls[kDec4Waves][kDec4Group];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  const int G = a.H / a.c.Hk, GG = (G + kDec4Group - 1) / kDec4Group;
  // the heads of a sequence, whose ranges are alike, on different XCDs; the last range of every sequence, which may hold the new row, first
  const int pairs = a.B * a.c.Hk * GG, turn = __builtin_amdgcn_readfirstlane(blockIdx.x / pairs), of = blockIdx.x - turn * pairs;
  const int id = __builtin_amdgcn_readfirstlane(of / GG), gg = of - id * GG, b = __builtin_amdgcn_readfirstlane(id / a.c.Hk), hk = id - b * a.c.Hk;
  const int pos = a.positions[b], keys = (int)max((int64_t)0, min((int64_t)pos + a.key_add, (int64_t)a.c.S));
  const int per = __builtin_amdgcn_readfirstlane(kv4_range(keys, ranges)), used = __builtin_amdgcn_readfirstlane(max(1, (keys + per - 1) / per)), s = turn < used ? used - 1 - turn : turn;
  const int k0 = min(s * per, keys), k1 = min(k0 + per, keys);
  const int h0 = hk * G + gg * kDec4Group, heads = min(kDec4Group, G - gg * kDec4Group);
  const RangeParts part{scratch, (int64_t)a.B * a.H, ranges, DH};
  if (s >= used) {
    if (tid < heads) *part.stats((int64_t)b * a.H + h0 + tid, s) = f32x2_t{-INFINITY, 0.f};
    return;
  }

  // an address is the wave's (a step's row, 64 bits) and an offset of the lane's that stays the same
  const uint32_t row = (uint32_t)a.c.sc_s;
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* ksp = static_cast<const uint8_t*>(a.c.k_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const uint8_t* vsp = static_cast<const uint8_t*>(a.c.v_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  uint32_t klane = 4 * n * row + CH / 2 * g, vlane = 16 * g * row + NT / 2 * n;
  uint32_t kslane = CH * g / kGroup4 * (uint32_t)a.c.ss_g + 4 * n, vslane = NT * n / kGroup4 * (uint32_t)a.c.ss_g + 16 * g;
  asm volatile("" : "+v"(klane), "+v"(vlane), "+v"(kslane), "+v"(vslane));      // made by 64-bit products, each would take two registers
  uint32_t kr[4][KW], vr[16], ks, vs[4];
  const auto fetch_k = [&](int c0) {
    const Rows4 r = rows4(kb + (int64_t)c0 * a.c.sc_s);
#pragma unroll
    for (int t = 0; t < 4; ++t) load4<4 * KW, kOnce>(r, klane, t * row, kr[t]);
    load4<4, 0>(rows4(ksp + c0), kslane, 0, &ks);
  };
  const auto fetch_v = [&](int c0) {
    const Rows4 r = rows4(vb + (int64_t)c0 * a.c.sc_s);
#pragma unroll
    for (int j = 0; j < 16; ++j) load4<NT / 2, kOnce>(r, vlane, j * row, vr + j);
    load4<16, 0>(rows4(vsp + c0), vslane, 0, vs);
  };
  int c0 = k0 + wave * kDec4Step;
  // The new row is the last key, and this workgroup alone reads it.  One wave writes it while the others begin, and the step that holds it comes behind a barrier.
  const bool appends = a.k_new != nullptr && pos >= k0 && pos < k1;
  const int before = appends ? pos / kDec4Step * kDec4Step : k1;
  if (appends && wave == kDec4Waves - 1)
    append_row4<DT, DH>(a.c, a.k_new + (int64_t)b * a.sk_b + (int64_t)hk * a.sk_h, a.v_new + (int64_t)b * a.sv_b + (int64_t)hk * a.sv_h, a.cos, a.sin, a.rope_len,
                        b, hk, pos, lane);
  if (c0 < before) { fetch_k(c0); fetch_v(c0); }

  frag_t qf[ST], qr[HALVES ? 1 : ST];                     // element e of product st is channel CH g + 8 st + e
  {
    const int head = HALVES ? n & 7 : n;
    const uint16_t* qp = a.q + (int64_t)b * a.sq_b + (int64_t)(h0 + min(head, heads - 1)) * a.sq_h;
    const int64_t tp = (int64_t)min(max(pos, 0), a.rope_len - 1) * HALF;
    const float sign = CH * g < HALF ? -1.f : 1.f;
    u32x4_t x[ST], y[ST], cw[ST], sw[ST];
#pragma unroll
    for (int st = 0; st < ST; ++st) x[st] = eight4(qp + CH * g + 8 * st);
    if (a.cos) {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int d = CH * g + 8 * st;
        y[st] = eight4(qp + (d ^ HALF));
        cw[st] = eight4(a.cos + tp + (d & (HALF - 1)));
        sw[st] = eight4(a.sin + tp + (d & (HALF - 1)));
      }
    } else {
#pragma unroll
      for (int st = 0; st < ST; ++st) { y[st] = sw[st] = u32x4_t{0u, 0u, 0u, 0u}; cw[st] = u32x4_t{E::one2, E::one2, E::one2, E::one2}; }
    }
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      u32x4_t high, rest;
      query_parts<E>(x[st], y[st], cw[st], sw[st], sign, high, rest);
      if (HALVES && n >= 8) high = rest;
      if (head >= heads) high = rest = u32x4_t{0u, 0u, 0u, 0u};
      qf[st] = __builtin_bit_cast(frag_t, high);
      if constexpr (!HALVES) qr[st] = __builtin_bit_cast(frag_t, rest);
    }
  }

  const float scale = a.scale * 1.4426950408889634f;      // weights are powers of two of the scores' differences
  const float second = n < 8 ? 0.f : -1.f;                // the columns of the second parts take what the first leave
  float m = -INFINITY, l = 0.f;
  f32x4_t o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const auto walk = [&](int stop) {
    for (; c0 < stop; c0 += kDec4Waves * kDec4Step) {
      const int next = c0 + kDec4Waves * kDec4Step, left = k1 - c0 - 16 * g;      // of the lane's 16 keys
      float x[4][4];                                      // key 16 g + 4 i + t
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
        const float f = scale_at(ks, t);
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const uint32_t w = kr[t][st];
          const frag_t kk = __builtin_bit_cast(frag_t, u32x4_t{pair4<0>(w, f), pair4<1>(w, f), pair4<2>(w, f), pair4<3>(w, f)});
          acc = P::mfma(kk, qf[st], acc);
          if constexpr (!HALVES) acc = P::mfma(kk, qr[st], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][i] = (HALVES ? acc[i] + dpp_f32<0x128>(acc[i]) : acc[i]) * scale;
      }
      if (next < stop) fetch_k(next);
      if (c0 + kDec4Step > k1) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = 4 * i + t;
            x[t][i] = j < left ? x[t][i] : -INFINITY;
            vr[j] = j < left ? vr[j] : 0u;
            if (j >= left) vs[i] &= ~(0x80u << (8 * t));   // no byte of a row behind the last key is that of a NaN or beyond the numbers: zeros stay zeros
          }
      }
      float top = x[0][0];
#pragma unroll
      for (int t = 0; t < 4; ++t) top = fmaxf(top, fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
      top = fmaxf(m, column_max(top));
      if (__any(top > m)) {
        const float keep = __builtin_amdgcn_exp2f(m - top);                // 0 in front of the first step
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t] *= keep;
        l *= keep;
        m = top;
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) asm volatile("" : "+v"(o[t]));           // the sums stay in their registers whether they were rescaled or not
      frag_t hi[2], lo[2];                                // the weights of the lane's keys 8 u .. 8 u + 7 as a 16-bit part and what it leaves
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = 2 * u + (i >> 1), t = 2 * (i & 1);
          const float w0 = __builtin_amdgcn_exp2f(x[t][c] - m), w1 = __builtin_amdgcn_exp2f(x[t + 1][c] - m);
          l += w0 + w1;
          ph[i] = pack_bf16x2(w0, w1);
          if constexpr (HALVES) ph[i] = pack_bf16x2(fmaf(bf16_lo(ph[i]), second, w0), fmaf(bf16_hi(ph[i]), second, w1));
          else pl[i] = pack_bf16x2(w0 - bf16_lo(ph[i]), w1 - bf16_hi(ph[i]));
        }
        hi[u] = __builtin_bit_cast(frag_t, u32x4_t{ph[0], ph[1], ph[2], ph[3]});
        if constexpr (!HALVES) lo[u] = __builtin_bit_cast(frag_t, u32x4_t{pl[0], pl[1], pl[2], pl[3]});
      }
      __builtin_amdgcn_sched_barrier(0);                  // left to itself the compiler converts far ahead, and three waves a SIMD do not fit
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int c = 0; c < NT / 2; ++c) {               // channels 2 c and 2 c + 1 of the lane's
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = pair4_at(c, vr[8 * u + e], scale_at(vs[2 * u + (e >> 2)], e & 3));
          u32x4_t v0, v1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v0[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
            v1[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
          }
          o[2 * c] = P::mfma(__builtin_bit_cast(frag_t, v0), hi[u], o[2 * c]);
          if constexpr (!HALVES) o[2 * c] = P::mfma(__builtin_bit_cast(frag_t, v0), lo[u], o[2 * c]);
          o[2 * c + 1] = P::mfma(__builtin_bit_cast(frag_t, v1), hi[u], o[2 * c + 1]);
          if constexpr (!HALVES) o[2 * c + 1] = P::mfma(__builtin_bit_cast(frag_t, v1), lo[u], o[2 * c + 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (next < stop) fetch_v(next);
    }
  };
  walk(before);
  if (appends) {
    wait_stores_acked();
    __syncthreads();
    if (c0 < k1) { fetch_k(c0); fetch_v(c0); }
    walk(k1);
  }
  // the waves' results through LDS: element i of tile t is channel NT (4 g + i) + t of query n.  A sum that is NaN takes the largest reference, so that it is kept.
  if constexpr (HALVES) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][i] += dpp_f32<0x128>(o[t][i]);
  }
  l = column_sum(l);
  if (g == 0) { ms[wave][n] = l != l ? INFINITY : m; ls[wave][n] = l; }
  if (n < heads) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < NT; t += 4)
        *reinterpret_cast<f32x4_t*>(os + (wave * heads + n) * (DH + 4) + NT * (4 * g + i) + t) = f32x4_t{o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]};
  }
  __syncthreads();
  for (int e = tid; e < heads * DH; e += kDec4Waves * kWave) {
    const int q = e / DH, d = e % DH;
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kDec4Waves; ++w) top = fmaxf(top, ms[w][q]);
#pragma unroll
    for (int w = 0; w < kDec4Waves; ++w) {
      const float f = ms[w][q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[w][q] - top);
      sum += f * ls[w][q];
      v += f * os[(w * heads + q) * (DH + 4) + d];
    }
    if (ranges == 1) {
      a.out[(int64_t)b * a.so_b + (int64_t)(h0 + q) * a.so_h + d] = (uint16_t)E::bits(sum == 0.f ? 0.f : v / sum);
    } else {
      const int64_t at = (int64_t)b * a.H + h0 + q;
      part.values(at, s)[d] = v;
      if (d == 0) *part.stats(at, s) = f32x2_t{top, sum};
    }
  }
}

int kv4_ranges(int B, int H, int Hk, int S, int nsplit) {
  const int most = S < 384 ? 1 : (S + kMinRange4 - 1) / kMinRange4;
  if (nsplit <= 0) {
    const int64_t pairs = (int64_t)B * Hk * ((H / Hk + kDec4Group - 1) / kDec4Group);
    nsplit = max((int)((512 + pairs - 1) / pairs), (S + 2047) / 2048);
  }
  return max(1, min(nsplit, most));
}
size_t kv4_decode_scratch_bytes(int B, int H, int Dh, int ranges) { return ranges > 1 ? RangeParts::bytes((int64_t)B * H, ranges, Dh) : 0; }

template <int DT, int DH>
static void decode_form(const Kv4AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  const int groups = (a.H / a.c.Hk + kDec4Group - 1) / kDec4Group;
  const dim3 grid((unsigned)a.B * a.c.Hk * groups * ranges);
  const size_t lds = kDec4Waves * min(a.H / a.c.Hk, kDec4Group) * (DH + 4) * sizeof(float);
  if (a.H / a.c.Hk <= 8) hipLaunchKernelGGL((kv4_decode_kernel<DT, DH, true>), grid, dim3(kDec4Waves * kWave), lds, st, a, ranges, scratch);
  else hipLaunchKernelGGL((kv4_decode_kernel<DT, DH, false>), grid, dim3(kDec4Waves * kWave), lds, st, a, ranges, scratch);
  if (ranges > 1) launch_join(join_args(a), ranges, true, scratch, st);
  set_last_form(ranges == 1 ? "kv4 decode" : "kv4 decode ranges");
}
int launch_kv4_decode(const char* fn, const Kv4AttnArgs& args, int ranges, float* scratch, hipStream_t st) {
  Kv4AttnArgs a = args;
  if ((int64_t)a.B * a.H * ranges > (1 << 23)) { set_last_error("%s: %d sequences of %d heads in %d ranges", fn, a.B, a.H, ranges); return kErrBadShape; }
  if (a.k_new != nullptr && a.H / a.c.Hk > kDec4Group) {   // several workgroups read the keys of a kv head: the rows in a launch before them
    const Kv4AppendArgs n{a.c, a.k_new, a.sk_b, 0, a.sk_h, a.v_new, a.sv_b, 0, a.sv_h, a.positions, nullptr, a.cos, a.sin, a.rope_len, a.B, 1, a.dt};
    if (const int rc = launch_kv4_append(fn, n, st)) return rc;
    a.k_new = nullptr;
  }
  if (a.dt == 1) a.c.Dh == 128 ? decode_form<1, 128>(a, ranges, scratch, st) : decode_form<1, 64>(a, ranges, scratch, st);
  else a.c.Dh == 128 ? decode_form<0, 128>(a, ranges, scratch, st) : decode_form<0, 64>(a, ranges, scratch, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

}  // namespace fsvd
