// Attention over the KV cache in 4 bits.
#include <type_traits>

#include "attn_join.hpp"
#include "kv4.hpp"

namespace fsvd {

typedef uint32_t u32x2_any_t __attribute__((ext_vector_type(2), aligned(2)));
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

// The largest of three numbers, in one instruction: what fmaxf compiles to first makes quiet NaNs of each product's result, which has no others.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// The maximum of a row that has seen no score yet.  A score may be -infinity where fp32 does not hold it, and has no weight against this, where its distance from
// another -infinity is no number.
constexpr float kLowest4 = -__FLT_MAX__;

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
// products, of more they are products of their own.  K's rows are read for once only, but V's, whose lines several loads of a lane take parts of, stay in the caches
// (32 heads of 64, 16 x 4000 keys: 37.5 us, 46.2 read for once too; heads of 128 56 either way, 57.4 with K's kept as well).  The cache's rooms are whole steps, so nothing is clamped: rows behind the last
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
  const int pos = a.positions[b], keys = (int)max((int64_t)0, min((int64_t)pos + a.key_add, (int64_t)a.c.limit));
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
    for (int j = 0; j < 16; ++j) load4<NT / 2, 0>(r, vlane, j * row, vr + j);
    load4<16, 0>(rows4(vsp + c0), vslane, 0, vs);
  };
  int c0 = k0 + wave * kDec4Step;
  // The new row is the last key, and this workgroup alone reads it.  One wave writes it while the others begin, and the step that holds it comes behind a barrier (in a
  // captured graph, us without a new row / with one / with a launch of its own for it: 1 x 137 keys of 8 heads of 64 5.4 / 6.3 / 8.1, 1 x 512 of 32 heads 9.3 / 10.3 / 12.9, 16 x 1000 to 4001
  // of 8 21.8 / 21.3 / 25.2, 16 x 4090 of 32 54.8 / 55.9 / 57.0).
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
  float m = kLowest4, l = 0.f;
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
      float top = m;
#pragma unroll
      for (int t = 0; t < 4; ++t) top = max3(max3(top, x[t][0], x[t][1]), x[t][2], x[t][3]);
      top = column_max(top);
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
  if (g == 0) { ms[wave][n] = l != l ? INFINITY : m == kLowest4 ? -INFINITY : m; ls[wave][n] = l; }
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

// Key ranges: two workgroups for each compute unit, where a range then has 512 keys at least, else one for each and up to 16 ranges of any length.  Times of a call with
// its join, us: 8 kv heads of 16000 keys in 16 ranges 16.3, 32 12.9 (taken), 63 14.3; 128 kv heads of 4000 in 2 22.8, 4 21.1 (taken), 8 23.9; 32 of 1000 in 2 10.3, 4
// 9.1 (taken); 512 of 4090 in 1 56.3 (taken), 2 58.0, with lengths down to a quarter 42.1 and 44.2; 384 of 4000 in 1 52.5, 2 46.2 (taken), 3 50.8; 2048 of 1000 in 1
// 60.2 (taken), 2 71.6.
int kv4_ranges(int B, int H, int Hk, int S, int nsplit) {
  const int most = S < 384 ? 1 : (S + kMinRange4 - 1) / kMinRange4;
  if (nsplit <= 0) {
    const int64_t pairs = (int64_t)B * Hk * ((H / Hk + kDec4Group - 1) / kDec4Group);
    nsplit = (int)min((512 + pairs - 1) / pairs, max(min((256 + pairs - 1) / pairs, (int64_t)16), ((int64_t)S + 511) / 512));
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

// ---------------------------------------------------------------------------------------------
// A chunk of a prompt.  The query rows of the heads that share a kv head are one list, row r = query token r / G of head r % G, so that grouped heads share
// the tiles of keys too.  A workgroup of four waves takes 16 rows for each; tiles of 64 keys go through LDS as bf16, converted once for the workgroup,
// scales included: K row by row, V transposed (two keys of a channel next to each other by byte permutes), two buffers and one barrier a tile.
//   S^T = K Q^T leaves a lane four consecutive keys of one query in every 16-key block, O^T = V^T P^T takes them as they stand (the V columns of 32 keys
//   follow the order 16 (e / 4) + 4 g + e % 4 of the products' k axis).
//   The weights go into the second product as two bf16 parts, 16 significant bits, and into their sums as they are; a q that the call rotates, or of float16, is
//   two parts too (TWO).
// V columns: 16-byte pieces of the 128-byte rows are XOR-ed with a number of the row, which keeps the fragments' 16-byte reads and the 8-byte transposing writes off
// each other's banks (found by enumeration).
// ---------------------------------------------------------------------------------------------
constexpr int kTile4 = 64, kPrompt4Waves = 4;
constexpr float kSlack4 = 8.f;
constexpr int kLeastTiles = 4;           // of a range: the room may be longer than what it holds, and ranges without keys only say so
__device__ __forceinline__ int v_piece4(int d) { return ((d >> 2) & 7) ^ (d & 6); }

template <int DT, int DH, int KG, bool TWO>
__global__ __launch_bounds__(kWave * kPrompt4Waves * KG, 2) void kv4_prompt_kernel(Kv4AttnArgs a, int ranges, float* scratch) {
  typedef E16<DT> E;
  typedef E16<0> P;
  typedef P::frag_t frag_t;
  constexpr int ST = DH / 32, NT = DH / 16, KSTR = DH + 16, TH = kWave * kPrompt4Waves, QW = 16, BM = QW * kPrompt4Waves, HALF = DH / 2;
  constexpr int KB = DH / 8, VD = DH / 16;               // bytes of a key, channels of four values that a thread stages
  extern __shared__ __align__(16) unsigned char smem[];
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0;
  uint16_t* Ks = reinterpret_cast<uint16_t*>(smem) + kg * 2 * kTile4 * (KSTR + DH);      // [2][kTile4][KSTR]
  uint16_t* Vt = Ks + 2 * kTile4 * KSTR;                                    // [2][DH][kTile4]
  __shared__ int nan_at[DH / kGroup4];                                      // the first NaN of a group among the values that not every row sees
  __shared__ int any_nan;

  const int G = a.H / a.c.Hk, HB = a.c.Hk * a.B, MT = gridDim.x / HB;
  int mt, hb;
  // the row tiles of a kv head on one XCD, the ones with the most keys first
  if (HB % 8 == 0) {
    const int per = HB >> 3, r = blockIdx.x >> 3;
    mt = r / per;
    hb = (blockIdx.x & 7) * per + r - mt * per;
  } else {
    const int t = xcd_run_index(blockIdx.x, MT * HB);
    hb = t / MT;
    mt = t - hb * MT;
  }
  mt = MT - 1 - mt;
  const int hk = hb / a.B, b = hb - hk * a.B, range = blockIdx.y;
  const int tid = threadIdx.x % TH, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 15, lg = lane >> 4;
  const int M = a.rows ? max(0, min(a.rows[b], a.M)) : a.M, rows = M * G, row0 = mt * BM;
  if (row0 >= rows) return;
  const int pos = min(a.positions[b], 0x7ffffffe - a.M);
  const auto seen_by = [&](int r) { return max(0, min(pos + r / G + a.key_add, a.c.limit)); };     // keys of row r
  const int all_end = seen_by(min(row0 + BM, rows) - 1);
  const int tiles = (all_end + kTile4 - 1) / kTile4, per = max((tiles + ranges - 1) / ranges, kLeastTiles);
  const int n_begin = range * per * kTile4, n_end = min(all_end, (range + 1) * per * kTile4);
  if (range > 0 && n_begin >= all_end) {
    const RangeParts part{scratch, (int64_t)HB * a.M * G, ranges, DH};
    if (threadIdx.x < BM && row0 + threadIdx.x < rows) *part.stats((int64_t)(b * a.c.Hk + hk) * a.M * G + row0 + threadIdx.x, range) = f32x2_t{-INFINITY, 0.f};
    return;
  }
  const int w0 = row0 + wave * QW;
  const int wave_end = w0 < rows ? min(n_end, seen_by(min(w0 + QW, rows) - 1)) : 0;             // keys past it are unseen by the wave

  const float scale = a.scale * 1.4426950408889634f;
  float m_run = -INFINITY, l_run = 0.f;                                     // l_run: a lane's own sum of the weights, not rounded
  f32x4_t o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // K: four lanes a row; V: sixteen lanes with VD channels each for four adjacent keys.  The rooms are whole tiles: nothing is clamped.
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* ksp = static_cast<const uint8_t*>(a.c.k_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const uint8_t* vsp = static_cast<const uint8_t*>(a.c.v_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const int krow = tid >> 2, kc = tid & 3, vq = tid >> 4, vc = tid & 15;
  const uint32_t row = (uint32_t)a.c.sc_s;
  const uint32_t koff = krow * row + KB * kc, voff = 4 * vq * row + VD / 2 * vc;
  const uint32_t ksoff = 2 * KB * kc / kGroup4 * (uint32_t)a.c.ss_g + krow, vsoff = VD * vc / kGroup4 * (uint32_t)a.c.ss_g + 4 * vq;
  uint32_t kreg[KB / 4], vreg[4], kbyte, vbyte;
  const auto request = [&](int n0) {
    load4<KB, 0>(rows4(kb + (int64_t)n0 * a.c.sc_s), koff, 0, kreg);
    const Rows4 v = rows4(vb + (int64_t)n0 * a.c.sc_s);
#pragma unroll
    for (int e = 0; e < 4; ++e) load4<VD / 2, 0>(v, voff, e * row, vreg + e);
    kbyte = ksp[n0 + ksoff];
    load4<4, 0>(rows4(vsp + n0), vsoff, 0, &vbyte);
  };
  const auto at = [&](int i) { return n_begin + (i * KG + kg) * kTile4; };
  const int all = n_begin < n_end ? (n_end - n_begin + kTile4 - 1) / kTile4 : 0, n = (all - kg + KG - 1) / KG;      // of the workgroup, of this half
  if (n > 0) request(at(0));             // the first tile is on its way while q is turned

  frag_t qf[ST], qr[ST];                                  // qr: what the first part leaves
  const int r = min(w0 + lr, rows - 1), m = r / G, h = hk * G + r - m * G, seen = seen_by(r);
  const uint16_t* qp = a.q + (int64_t)b * a.sq_b + (int64_t)m * a.sq_m + (int64_t)h * a.sq_h;
  u32x4_t x[ST];
#pragma unroll
  for (int st = 0; st < ST; ++st) x[st] = eight4(qp + 32 * st + 8 * lg);
  if constexpr (TWO) {
    u32x4_t cw[ST / 2], sw[ST / 2];
    const int64_t tp = (int64_t)min(max(pos + m, 0), a.rope_len - 1) * HALF + 8 * lg;
#pragma unroll
    for (int st = 0; st < ST / 2; ++st) {
      cw[st] = a.cos ? eight4(a.cos + tp + 32 * st) : u32x4_t{E::one2, E::one2, E::one2, E::one2};
      sw[st] = a.cos ? eight4(a.sin + tp + 32 * st) : u32x4_t{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int st = 0; st < ST / 2; ++st) {
      const u32x4_t none = {0u, 0u, 0u, 0u};
      u32x4_t h0, r0, h1, r1;
      query_parts<E>(x[st], a.cos ? x[st + ST / 2] : none, cw[st], sw[st], -1.f, h0, r0);
      query_parts<E>(x[st + ST / 2], a.cos ? x[st] : none, cw[st], sw[st], 1.f, h1, r1);
      asm volatile("" : "+v"(r0), "+v"(r1), "+v"(h0), "+v"(h1));         // made here: put off, they spill
      qf[st] = __builtin_bit_cast(frag_t, h0);
      qf[st + ST / 2] = __builtin_bit_cast(frag_t, h1);
      qr[st] = __builtin_bit_cast(frag_t, r0);
      qr[st + ST / 2] = __builtin_bit_cast(frag_t, r1);
    }
  } else {
#pragma unroll
    for (int st = 0; st < ST; ++st) qf[st] = __builtin_bit_cast(frag_t, x[st]);
  }
  const auto stage_k = [&](int buf) {
    uint16_t* to = Ks + buf * kTile4 * KSTR + krow * KSTR + 2 * KB * kc;
    const float f = scale_of(kbyte);
#pragma unroll
    for (int i = 0; i < KB / 4; ++i)
      *reinterpret_cast<u32x4_t*>(to + 8 * i) = u32x4_t{pair4<0>(kreg[i], f), pair4<1>(kreg[i], f), pair4<2>(kreg[i], f), pair4<3>(kreg[i], f)};
  };
  // A masked key has weight zero, and zero times a NaN is one: where not every row sees the whole tile, a group that is NaN is staged as numbers and put into the
  // rows that see it at the end; so is what stands behind the last key, whatever its bytes.
  const int all_see = seen_by(row0);
  const auto set_nans_aside = [&](int n0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + 4 * vq + e;
      const bool none = n >= n_end, nan = !none && (vbyte >> (8 * e) & 0xff) == kNanByte;
      if (nan) {
        any_nan = 1;
        atomicMin(&nan_at[VD * vc / kGroup4], n);
      }
      if (none || nan) vbyte &= ~(0xffu << (8 * e));
    }
  };
  const auto stage_v = [&](int buf) {
    const int ko = (4 * vq) & 31, col = ((4 * vq) & 32) + 8 * ((ko & 15) >> 2) + 4 * (ko >> 4);
    uint16_t* to = Vt + buf * DH * kTile4 + VD * vc * kTile4;
#pragma unroll
    for (int c = 0; c < VD / 2; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pair4_at(c, vreg[e], scale_at(vbyte, e));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = 2 * c + i;
        const uint32_t lohi = i ? 0x07060302u : 0x05040100u;
        *reinterpret_cast<u32x2_t*>(to + d * kTile4 + (col ^ (8 * v_piece4(VD * vc + d)))) =
            u32x2_t{__builtin_amdgcn_perm(w[1], w[0], lohi), __builtin_amdgcn_perm(w[3], w[2], lohi)};
      }
    }
  };
  const auto k_frags = [&](frag_t (&kf)[2][ST], int buf, int half) {       // of 32 of the tile's keys
    const uint16_t* ks = Ks + buf * kTile4 * KSTR;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int st = 0; st < ST; ++st) kf[j][st] = __builtin_bit_cast(frag_t, *reinterpret_cast<const u32x4_t*>(ks + (32 * half + 16 * j + lr) * KSTR + 32 * st + 8 * lg));
  };
  const auto scores = [&](f32x4_t (&s)[4], const frag_t (&kf)[2][ST], int half) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        s[2 * half + j] = P::mfma(kf[j][st], qf[st], st ? s[2 * half + j] : f32x4_t{0.f, 0.f, 0.f, 0.f});
        if constexpr (TWO) s[2 * half + j] = P::mfma(kf[j][st], qr[st], s[2 * half + j]);
      }
  };
  // row d = 16 t + lr of V: its piece is turned by (lr / 4) ^ (lr & 6) ^ 4 (t % 2), so two addresses and constants reach all of them
  const uint32_t vread = lr * kTile4 + 8 * (lg ^ (lr >> 2) ^ (lr & 6));
  const auto v_frags = [&](frag_t (&vf)[NT], int buf, int st) {
    const uint16_t* vt = Vt + buf * DH * kTile4;
#pragma unroll
    for (int t = 0; t < NT; ++t) vf[t] = __builtin_bit_cast(frag_t, *reinterpret_cast<const u32x4_t*>(vt + ((st ^ t) & 1 ? vread ^ 32 : vread) + 16 * t * kTile4));
  };
  frag_t ph[2], pl[2];
  const auto values = [&](const frag_t (&vf)[NT], int st) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      o[t] = P::mfma(vf[t], ph[st], o[t]);
      o[t] = P::mfma(vf[t], pl[st], o[t]);
    }
  };
  const int wave_sees = seen_by(min(w0, rows - 1));                  // keys of the wave's first row; the others see more from one to the next
  const auto weights = [&](f32x4_t (&s)[4], int n0) {
    const bool plain = n0 + kTile4 <= wave_sees;                     // every row of the wave sees the whole tile
    if (!plain) {
      const int vis = seen - n0 - 4 * lg;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[j][i] = 16 * j + i < vis ? s[j][i] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max3(max3(top, s[j][0], s[j][1]), s[j][2], s[j][3]);
    top *= scale;
    // m_run moves only where a score is kSlack4 over it, and the lanes of a column need not agree on a maximum until then; weights are taken 2^-kSlack4 of
    // what they are over it, at most 1, which changes no rounding, so that no value becomes infinite on its way.
    if (__any(top > m_run + kSlack4)) {
      top = fmaxf(m_run, column_max(top));
      const float keep = top > m_run ? __builtin_amdgcn_exp2f(m_run - top) : 1.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t] *= keep;
      l_run *= keep;
      m_run = top;
    }
    const float base = m_run == -INFINITY ? 0.f : m_run + kSlack4;  // a row that has seen nothing yet: exp2(-inf - 0)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[j][i] = __builtin_amdgcn_exp2f(fmaf(s[j][i], scale, -base));
        l_run += s[j][i];
      }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint32_t hw[4], lw[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float x0 = s[2 * st + (c >> 1)][2 * (c & 1)], x1 = s[2 * st + (c >> 1)][2 * (c & 1) + 1];
        hw[c] = pack_bf16x2(x0, x1);
        lw[c] = pack_bf16x2(x0 - bf16_lo(hw[c]), x1 - bf16_hi(hw[c]));
      }
      ph[st] = __builtin_bit_cast(frag_t, u32x4_t{hw[0], hw[1], hw[2], hw[3]});
      pl[st] = __builtin_bit_cast(frag_t, u32x4_t{lw[0], lw[1], lw[2], lw[3]});
    }
  };

  if (tid < DH / kGroup4) nan_at[tid] = 0x7fffffff;
  if (tid == 0) any_nan = 0;
  __syncthreads();
  for (int i = 0; i * KG < all; ++i) {
    const int buf = i & 1;
    if (KG == 1 || i < n) {
      stage_k(buf);
      if (at(i) + kTile4 > all_see) set_nans_aside(at(i));
      stage_v(buf);
    }
    if (i + 1 < n) request(at(i + 1));
    __syncthreads();                   // this buffer is written; the other one is read by nobody any more
    if (at(i) >= wave_end || (KG > 1 && i >= n)) continue;
    // All fragments of K are read at once, those of V before and behind the weights, so that no product waits for one: 512 tokens of 32 heads 13.9 us (14.5 with a half of
    // K's and of V's at a time), 2 x 512 in groups of 4 18.5 (19.8).
    f32x4_t s[4];
    frag_t kf0[2][ST], kf1[2][ST], vf0[NT], vf1[NT];
    k_frags(kf0, buf, 0);
    k_frags(kf1, buf, 1);
    __builtin_amdgcn_sched_barrier(0);
    scores(s, kf0, 0);
    scores(s, kf1, 1);
    __builtin_amdgcn_sched_barrier(0);
    v_frags(vf0, buf, 0);
    __builtin_amdgcn_sched_barrier(0);
    weights(s, at(i));
    v_frags(vf1, buf, 1);
    __builtin_amdgcn_sched_barrier(0);
    values(vf0, 0);
    values(vf1, 1);
  }
  if constexpr (KG > 1) {                // the halves' results
    static_assert(KG == 2, "one exchange");
    f32x4_t* part = reinterpret_cast<f32x4_t*>(smem) + wave * (NT + 1) * kWave + lane;
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t) part[t * kWave] = o[t];
      part[NT * kWave] = f32x4_t{m_run, l_run, 0.f, 0.f};
    }
    __syncthreads();
    if (kg == 1) return;
    const f32x4_t other = part[NT * kWave];
    const float top = fmaxf(m_run, other[0]);
    // a half whose sum is NaN keeps it, whatever its reference
    const float f0 = m_run > -INFINITY ? __builtin_amdgcn_exp2f(m_run - top) : l_run == 0.f ? 0.f : 1.f;
    const float f1 = other[0] > -INFINITY ? __builtin_amdgcn_exp2f(other[0] - top) : other[1] == 0.f ? 0.f : 1.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = o[t] * f0 + part[t * kWave] * f1;
    l_run = l_run * f0 + other[1] * f1;
    m_run = top;
  }
  // element i of tile t is channel 16 t + 4 lg + i of row lr
  const float l = column_sum(l_run);
  if (w0 + lr >= rows) return;
  if (any_nan) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (nan_at[t / 2] < seen)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] = __builtin_nanf("");
  }
  if (ranges > 1) {
    const RangeParts part{scratch, (int64_t)HB * a.M * G, ranges, DH};
    const int64_t at = (int64_t)(b * a.c.Hk + hk) * a.M * G + r;
    if (lg == 0) *part.stats(at, range) = f32x2_t{l != l ? INFINITY : m_run, l};
    float* v = part.values(at, range) + 4 * lg;
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4_t*>(v + 16 * t) = o[t];
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* op = a.out + (int64_t)b * a.so_b + (int64_t)m * a.so_m + (int64_t)h * a.so_h + 4 * lg;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const u32x2_t w{E::pack2(o[t][0] * inv, o[t][1] * inv), E::pack2(o[t][2] * inv, o[t][3] * inv)};
    *reinterpret_cast<u32x2_any_t*>(op + 16 * t) = w;      // at any element's address: of a row's bits nothing depends on where it goes
  }
}

// ---------------------------------------------------------------------------------------------
// The same for long chunks: 128 rows of a workgroup, 32 of a wave, in products of 32 x 32 x 16.  These hold up the vector unit for 14 cycles of their 38, those of
// 16 x 16 x 32 for 12 of 19 (a loop of both kinds of work with two waves a SIMD; an exponential takes 9 cycles, a conversion of two codes 4.5), and the vector unit is
// what this path needs most.
//   S^T = K Q^T leaves lane (n, h) = (lane % 32, lane / 32) keys 8 b + 4 h + j of a 32-key block of query n; O^T = V^T P^T takes keys 16 u + 4 h + j and 16 u + 8 + 4 h + j
//   of it in product u, and the V columns stand in that order.
// For outputs in bf16 the weights and V are float16 where it holds V exactly (the codes do, their scales nearly always): eleven bits of a weight, each off by 2^-11 of itself
// at most, where the output is rounded by 2^-8; of 8 x 2048 random tokens the error against 64 bits is 0.001655 of the output (root mean square), 0.001646 with sixteen bits in 427 us instead of 335.
// From the first tile on whose values it does not hold, and for outputs in float16, they are two bf16 parts, sixteen bits, and V bf16.
// K rows are an odd number of 16-byte pieces long and V's pieces XOR-ed with a number of the channel, so that 16 lanes read 16 different pieces of 256 bytes.
// 8 chunks of 2048 tokens, 32 heads of 128, causal: 320 to 337 us on different machines, up to 855 TFLOP/s of scores and outputs
// (before the maxima, its reads and its stores were what they are now 344; with weights in two bf16 parts then 412, 414 in products of 16 x 16 x 32); with rotation, whose q is two parts, 403
// us; in float16 464 us.
// ---------------------------------------------------------------------------------------------
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
constexpr uint16_t kLeastHalf = 127 - 23, kMostHalf = 127 + 13;            // bytes whose values float16 holds, the least of them as subnormals
constexpr float kLift4 = 7.f;                                               // weights in float16 are taken 2^7 larger: none above 2^-32 of the largest is lost
__device__ __forceinline__ int wide_piece(int c) { return ((c >> 1) ^ (c >> 4)) & 7; }

template <int DT, int DH, bool TWO>
__global__ __launch_bounds__(kWave * kPrompt4Waves, 2) void kv4_wide_kernel(Kv4AttnArgs a, int ranges, float* scratch) {
  typedef E16<DT> E;
  typedef E16<0> P;
  typedef P::frag_t frag_t;
  constexpr int SQ = DH / 16, NB = DH / 32, KSTR = DH + 8, BM = 32 * kPrompt4Waves, HALF = DH / 2;      // products of a key block; output blocks
  constexpr int KB = DH / 8, VD = DH / 16;               // bytes of a key, channels of four values that a thread stages
  constexpr int kAhead = 4, kAheadV = 4;                 // of the products, fragments on their way
  extern __shared__ __align__(16) unsigned char smem[];
  uint16_t* Ks = reinterpret_cast<uint16_t*>(smem);                         // [2][kTile4][KSTR]
  uint16_t* Vt = Ks + 2 * kTile4 * KSTR;                                    // [2][DH][kTile4]
  __shared__ int nan_at[DH / kGroup4];                                      // the first NaN of a group among the values that not every row sees
  __shared__ int any_nan, odd_tile, has_nan;

  const int G = a.H / a.c.Hk, HB = a.c.Hk * a.B, MT = gridDim.x / HB;
  int mt, hb;
  // the row tiles of a kv head on one XCD, the ones with the most keys first
  if (HB % 8 == 0) {
    const int per = HB >> 3, r = blockIdx.x >> 3;
    mt = r / per;
    hb = (blockIdx.x & 7) * per + r - mt * per;
  } else {
    const int t = xcd_run_index(blockIdx.x, MT * HB);
    hb = t / MT;
    mt = t - hb * MT;
  }
  mt = MT - 1 - mt;
  const int hk = hb / a.B, b = hb - hk * a.B, range = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, lh = lane >> 5;
  const int M = a.rows ? max(0, min(a.rows[b], a.M)) : a.M, rows = M * G, row0 = mt * BM;
  if (row0 >= rows) return;
  const int pos = min(a.positions[b], 0x7ffffffe - a.M);
  const auto seen_by = [&](int r) { return max(0, min(pos + r / G + a.key_add, a.c.limit)); };     // keys of row r
  const int all_end = seen_by(min(row0 + BM, rows) - 1), all_tiles = (all_end + kTile4 - 1) / kTile4, per = max((all_tiles + ranges - 1) / ranges, kLeastTiles);
  const int t0 = range * per, tiles = min(all_tiles, t0 + per), n_end = min(all_end, tiles * kTile4);        // the range: tiles t0 .. tiles - 1
  if (range > 0 && t0 >= all_tiles) {
    const RangeParts part{scratch, (int64_t)HB * a.M * G, ranges, DH};
    if (tid < BM && row0 + tid < rows) *part.stats((int64_t)(b * a.c.Hk + hk) * a.M * G + row0 + tid, range) = f32x2_t{-INFINITY, 0.f};
    return;
  }
  const int w0 = row0 + wave * 32;
  const int wave_end = w0 < rows ? min(n_end, seen_by(min(w0 + 32, rows) - 1)) : 0;             // keys past it are unseen by the wave
  const int r = min(w0 + lr, rows - 1), m = r / G, head = hk * G + r - m * G, seen = seen_by(r);

  frag_t qf[SQ], qr[TWO ? SQ : 1];                                          // qr: what the first part leaves
  {
    const uint16_t* qp = a.q + (int64_t)b * a.sq_b + (int64_t)m * a.sq_m + (int64_t)head * a.sq_h + 8 * lh;
    u32x4_t x[SQ];
#pragma unroll
    for (int st = 0; st < SQ; ++st) x[st] = eight4(qp + 16 * st);
    if constexpr (TWO) {
      const int64_t tp = (int64_t)min(max(pos + m, 0), a.rope_len - 1) * HALF + 8 * lh;
#pragma unroll
      for (int st = 0; st < SQ / 2; ++st) {
        const u32x4_t none = {0u, 0u, 0u, 0u}, cw = a.cos ? eight4(a.cos + tp + 16 * st) : u32x4_t{E::one2, E::one2, E::one2, E::one2};
        const u32x4_t sw = a.cos ? eight4(a.sin + tp + 16 * st) : none;
        u32x4_t h0, r0, h1, r1;
        query_parts<E>(x[st], a.cos ? x[st + SQ / 2] : none, cw, sw, -1.f, h0, r0);
        query_parts<E>(x[st + SQ / 2], a.cos ? x[st] : none, cw, sw, 1.f, h1, r1);
        asm volatile("" : "+v"(r0), "+v"(r1), "+v"(h0), "+v"(h1));         // made here: put off, they spill
        qf[st] = __builtin_bit_cast(frag_t, h0);
        qf[st + SQ / 2] = __builtin_bit_cast(frag_t, h1);
        qr[st] = __builtin_bit_cast(frag_t, r0);
        qr[st + SQ / 2] = __builtin_bit_cast(frag_t, r1);
      }
    } else {
#pragma unroll
      for (int st = 0; st < SQ; ++st) qf[st] = __builtin_bit_cast(frag_t, x[st]);
    }
  }
  const float scale = a.scale * 1.4426950408889634f;
  float m_run = -INFINITY, l_run = 0.f;                                     // l_run: a lane's own sum of the weights, not rounded
  f32x16_t o[NB];
#pragma unroll
  for (int t = 0; t < NB; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;

  // K: four lanes a row; V: sixteen lanes with VD channels each for four adjacent keys.  The rooms are whole tiles: nothing is clamped.
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* ksp = static_cast<const uint8_t*>(a.c.k_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const uint8_t* vsp = static_cast<const uint8_t*>(a.c.v_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const int krow = tid >> 2, kc = tid & 3, vq = tid >> 4, vc = tid & 15;
  const uint32_t row = (uint32_t)a.c.sc_s;
  const uint32_t koff = krow * row + KB * kc, voff = 4 * vq * row + VD / 2 * vc;
  const uint32_t ksoff = 2 * KB * kc / kGroup4 * (uint32_t)a.c.ss_g + krow, vsoff = VD * vc / kGroup4 * (uint32_t)a.c.ss_g + 4 * vq;
  uint32_t kreg[KB / 4], vreg[4], kbyte, vbyte;
  const auto request = [&](int n0) {
    load4<KB, 0>(rows4(kb + (int64_t)n0 * a.c.sc_s), koff, 0, kreg);
    load4<1, 0>(rows4(ksp + n0), ksoff, 0, &kbyte);
    const Rows4 v = rows4(vb + (int64_t)n0 * a.c.sc_s);
#pragma unroll
    for (int e = 0; e < 4; ++e) load4<VD / 2, 0>(v, voff, e * row, vreg + e);
    load4<4, 0>(rows4(vsp + n0), vsoff, 0, &vbyte);
  };
  const auto stage_k = [&](int buf) {
    uint16_t* to = Ks + buf * kTile4 * KSTR + krow * KSTR + 2 * KB * kc;
    const float f = scale_of(kbyte);
#pragma unroll
    for (int i = 0; i < KB / 4; ++i)
      *reinterpret_cast<u32x4_t*>(to + 8 * i) = u32x4_t{pair4<0>(kreg[i], f), pair4<1>(kreg[i], f), pair4<2>(kreg[i], f), pair4<3>(kreg[i], f)};
  };
  // a masked key has weight zero, and zero times a NaN is one: see kv4_prompt_kernel; a NaN among values in float16 is set aside wherever it stands
  const int all_see = seen_by(row0);
  const auto set_nans_aside = [&](int n0, uint32_t to) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + 4 * vq + e;
      const bool none = n >= n_end, nan = !none && (vbyte >> (8 * e) & 0xff) == kNanByte;
      if (nan) {
        any_nan = 1;
        atomicMin(&nan_at[VD * vc / kGroup4], n);
      }
      if (none || nan) vbyte = (vbyte & ~(0xffu << (8 * e))) | to << (8 * e);
    }
  };
  // V as bf16, or (half) as float16
  const auto stage_v = [&](int i, auto half) {
    const int piece = 2 * (vq >> 2) + (vq & 1), part = vq >> 1 & 1;
    uint16_t* to = Vt + (i & 1) * DH * kTile4 + VD * vc * kTile4 + 4 * part;
#pragma unroll
    for (int c = 0; c < VD / 2; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = half ? pair4_half_at(c, vreg[e], scale_at(vbyte, e)) : pair4_at(c, vreg[e], scale_at(vbyte, e));
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = 2 * c + k;
        const uint32_t sel = k ? 0x07060302u : 0x05040100u;
        *reinterpret_cast<u32x2_t*>(to + d * kTile4 + 8 * (piece ^ wide_piece(VD * vc + d))) =
            u32x2_t{__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel)};
      }
    }
  };
  const int wave_sees = seen_by(min(w0, rows - 1));                  // keys of the wave's first row; the others see more from one to the next
  const uint16_t* kread = Ks + lr * KSTR + 8 * lh;
  // channel 32 d + lr of V: its piece 2 u + lh is turned by (lr / 2) ^ (lr / 16) ^ 2 d, so four addresses and constants reach all of them
  const uint32_t vread = lr * kTile4 + 8 * ((lh ^ (lr >> 1) ^ (lr >> 4)) & 7);
  const auto attend = [&](int i, auto half) {
    const int buf = i & 1, n0 = i * kTile4;
    f32x16_t s[2];
    // Fragments of K are read four products ahead, the first of V before the weights are made: left to itself the compiler has two on their way (2 x 1024 tokens of 32
    // heads 36.6 us, 34.6 so, six ahead 34.2; 8 chunks of 128 behind 2000 60.8, 56.4 and 57.1; 8 x 2048 348, 342 and 340).
    const auto k_frag = [&](int p) { return __builtin_bit_cast(frag_t, *reinterpret_cast<const u32x4_t*>(kread + buf * kTile4 * KSTR + 32 * (p / SQ) * KSTR + 16 * (p % SQ))); };
    frag_t kf[kAhead];
#pragma unroll
    for (int p = 0; p < kAhead; ++p) kf[p] = k_frag(p);
#pragma unroll
    for (int p = 0; p < 2 * SQ; ++p) {
      const int k = p / SQ, st = p % SQ;
      if (st == 0) s[k] = f32x16_t{};
      s[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[p % kAhead], qf[st], s[k], 0, 0, 0);
      if constexpr (TWO) s[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[p % kAhead], qr[st], s[k], 0, 0, 0);
      if (p + kAhead < 2 * SQ) kf[p % kAhead] = k_frag(p + kAhead);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (n0 + kTile4 > wave_sees) {       // not every row of the wave sees the whole tile
      const int vis = seen - n0 - 4 * lh;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[k][e] = 32 * k + 8 * (e >> 2) + (e & 3) < vis ? s[k][e] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 16; e += 2) top = max3(top, s[k][e], s[k][e + 1]);
    top *= scale;
    // m_run moves only where a score is kSlack4 over it.  Weights in bf16 are taken 2^-kSlack4 of what they are over it, at most 1, so that no value becomes
    // infinite on its way; those in float16, whose values are small, 2^kLift4, at most 2^15.
    if (__any(top > m_run + kSlack4)) {
      const uint32_t u = __float_as_uint(top);
      const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
      top = fmaxf(m_run, fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
      const float keep = top > m_run ? __builtin_amdgcn_exp2f(m_run - top) : 1.f;
#pragma unroll
      for (int t = 0; t < NB; ++t) o[t] *= keep;
      l_run *= keep;
      m_run = top;
    }
    const float base = m_run == -INFINITY ? 0.f : half ? m_run - kLift4 : m_run + kSlack4;       // a row that has seen nothing yet: exp2(-inf - 0)
    const auto v_frag = [&](int p) { return *reinterpret_cast<const u32x4_t*>(Vt + buf * DH * kTile4 + (vread ^ (16 * (p / NB ^ p % NB))) + 32 * (p % NB) * kTile4); };
    u32x4_t vf[kAheadV];
#pragma unroll
    for (int p = 0; p < kAheadV; ++p) vf[p] = v_frag(p);
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t ph[4], pl[half ? 1 : 4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float x0 = __builtin_amdgcn_exp2f(fmaf(s[u >> 1][8 * (u & 1) + 2 * c], scale, -base));
        const float x1 = __builtin_amdgcn_exp2f(fmaf(s[u >> 1][8 * (u & 1) + 2 * c + 1], scale, -base));
        l_run += x0 + x1;
        if constexpr (half) {
          ph[u][c] = E16<1>::pack2(x0, x1);
        } else {
          const uint32_t w = pack_bf16x2(x0, x1);
          ph[u][c] = w;
          pl[u][c] = pack_bf16x2(x0 - bf16_lo(w), x1 - bf16_hi(w));
        }
      }
#pragma unroll
    for (int p = 0; p < 4 * NB; ++p) {
      const int u = p / NB, t = p % NB;
      const u32x4_t v = vf[p % kAheadV];
      if constexpr (half) {
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, v), __builtin_bit_cast(f16x8_t, ph[u]), o[t], 0, 0, 0);
      } else {
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(frag_t, v), __builtin_bit_cast(frag_t, ph[u]), o[t], 0, 0, 0);
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(frag_t, v), __builtin_bit_cast(frag_t, pl[u]), o[t], 0, 0, 0);
      }
      if (p + kAheadV < 4 * NB) vf[p % kAheadV] = v_frag(p + kAheadV);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (t0 < tiles) request(t0 * kTile4);
  if (tid < DH / kGroup4) nan_at[tid] = 0x7fffffff;
  if (tid == 0) { any_nan = has_nan = 0; odd_tile = tiles; }
  __syncthreads();
  if constexpr (DT == 0) {               // the first tile that float16 does not hold: waves in turn have the bytes of a group
    for (int n = t0 * kTile4 + 16 * (lane + kWave * (wave / NB)); n < n_end && wave / NB < kPrompt4Waves / NB; n += 16 * kWave * (kPrompt4Waves / NB)) {
      uint32_t w[4];
      load4<16, 0>(rows4(vsp), wave % NB * (uint32_t)a.c.ss_g + n, 0, w);
      u16x2_t far = {0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int left = n_end - n - 4 * e;                                 // bytes of the word that count
        const uint32_t inv = ~w[e];                                         // a byte of 0 is that of a NaN
        if ((inv - 0x01010101u) & ~inv & 0x80808080u) {                     // which moves no tile to the other form
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((w[e] >> (8 * i) & 0xff) == kNanByte) {
              w[e] = (w[e] & ~(0xffu << (8 * i))) | (uint32_t)kLeastHalf << (8 * i);
              if (i < left) has_nan = 1;
            }
        }
        if (left < 4) w[e] = left <= 0 ? 0x01010101u * kLeastHalf : (w[e] & ~(~0u << (8 * left))) | (0x01010101u * kLeastHalf & (~0u << (8 * left)));
        const u16x2_t first = {kLeastHalf, kLeastHalf};
        far = __builtin_elementwise_max(far, (u16x2_t)(__builtin_bit_cast(u16x2_t, w[e] & 0x00ff00ffu) - first));
        far = __builtin_elementwise_max(far, (u16x2_t)(__builtin_bit_cast(u16x2_t, w[e] >> 8 & 0x00ff00ffu) - first));
      }
      if (max((uint32_t)far.x, (uint32_t)far.y) > kMostHalf - kLeastHalf) {
        // A group of zeros is held whatever its scale (an append's has the least, a new cache's 0): the codes say, up to the first that is none.  8 x 2048 tokens of 32
        // heads whose every 16th row is zero: 351 us, 430 in two bf16 parts; none is 340, every scale below float16 435 (430 without this look).
        bool odd = false;
#pragma unroll 1
        for (int j = n; j < min(n + 16, n_end) && !odd; ++j) {
          const int byte = vsp[wave % NB * a.c.ss_g + j];
          if ((byte >= kLeastHalf && byte <= kMostHalf) || byte == kNanByte) continue;
          const u32x4_t c = *reinterpret_cast<const u32x4_t*>(vb + j * a.c.sc_s + wave % NB * (kGroup4 / 2));
          odd = ((c.x | c.y | c.z | c.w) & 0x77777777u) != 0;
        }
        if (odd) atomicMin(&odd_tile, n / kTile4);
      }
    }
    __syncthreads();
  }
  // the wave's own tiles; every wave stages and passes every barrier
  const int halves = DT == 0 ? __builtin_amdgcn_readfirstlane(odd_tile) : 0, nans = __builtin_amdgcn_readfirstlane(has_nan), own = (wave_end + kTile4 - 1) / kTile4;
  int i = t0;
  const auto stage = [&](auto half) {
    stage_k(i & 1);
    if ((i + 1) * kTile4 > all_see || (half && nans)) set_nans_aside(i * kTile4, half ? kLeastHalf : 0);
    stage_v(i, half);
    if (i + 1 < tiles) request((i + 1) * kTile4);
    __syncthreads();                     // this buffer is written; the other one is read by nobody any more
  };
  if constexpr (DT == 0) {
    for (; i < min(halves, own); ++i) {
      stage(std::true_type{});
      attend(i, std::true_type{});
    }
    for (; i < halves; ++i) stage(std::true_type{});
    if (i < own) {                       // from the reference of float16 weights to the other
      constexpr float f = 1.f / (1 << (int)(kLift4 + kSlack4));
#pragma unroll
      for (int t = 0; t < NB; ++t) o[t] *= f;
      l_run *= f;
    }
  }
  for (; i < own; ++i) {
    stage(std::false_type{});
    attend(i, std::false_type{});
  }
  for (; i < tiles; ++i) stage(std::false_type{});
  // element i of block t is channel 32 t + 8 (i / 4) + 4 lh + i % 4 of row lr
  {
    const uint32_t u = __float_as_uint(l_run);
    const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    l_run = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (w0 + lr >= rows) return;
  if (any_nan) {
#pragma unroll
    for (int t = 0; t < NB; ++t)
      if (nan_at[t] < seen)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = __builtin_nanf("");
  }
  if (ranges > 1) {
    const RangeParts part{scratch, (int64_t)HB * a.M * G, ranges, DH};
    const int64_t at = (int64_t)(b * a.c.Hk + hk) * a.M * G + r;
    // the reference that the weights were taken to in the end
    if (lh == 0) *part.stats(at, range) = f32x2_t{l_run != l_run ? INFINITY : DT == 0 && own <= halves ? m_run - kLift4 : m_run + kSlack4, l_run};
    float* v = part.values(at, range) + 4 * lh;
#pragma unroll
    for (int t = 0; t < NB; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) *reinterpret_cast<f32x4_t*>(v + 32 * t + 2 * i) = f32x4_t{o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]};
    return;
  }
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
  // the two lanes of a row change words, so that either has eight channels next to each other (stores of four: 8 x 2048 tokens 325 us)
  uint16_t* op = a.out + (int64_t)b * a.so_b + (int64_t)m * a.so_m + (int64_t)head * a.so_h + 8 * lh;
#pragma unroll
  for (int t = 0; t < NB; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      const auto x = __builtin_amdgcn_permlane32_swap(E::pack2(o[t][i] * inv, o[t][i + 1] * inv), E::pack2(o[t][i + 4] * inv, o[t][i + 5] * inv), false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(E::pack2(o[t][i + 2] * inv, o[t][i + 3] * inv), E::pack2(o[t][i + 6] * inv, o[t][i + 7] * inv), false, false);
      *reinterpret_cast<u32x4_any_t*>(op + 32 * t + 2 * i) = u32x4_any_t{x[0], y[0], x[1], y[1]};
    }
}

// Rows of a workgroup, its halves and key ranges, by the room's length S, as what it holds is known to the device alone.  Times are of bf16 without a rotation, in us; where q is
// two parts (float16, or rotated by the call) the borders between the forms are taken over from these and but for the one case below not measured.
//   128 rows where they make up 3/2 workgroups for each compute unit (heads of 64: two), and 3/4 where the room is twice the chunk or more: what a workgroup of a chunk at
// the start sees varies, and more of them level it out.  32 heads of 1500 tokens 43 (64 rows 47); 16 heads of 1500, with a rotation, 45 (35, therefore 64 rows); 32 of 1024
// behind 2000 others 70 (82); 8 chunks of 128 tokens, groups of 4, behind 2000 56 (72); 6 of 32 heads 54 (67); heads of 64: 32 of 1500 28.7 (28.1, therefore 64).  In two
// key ranges where each has 32 tiles: 1024 tokens, groups of 4, behind 16000 301 (341), but 32 heads behind 2000 75 (70).
//   128 rows in more key ranges where these make up a workgroup for each compute unit, up to two, and have 6 tiles each (heads of 64: 12, as ranges of 10 took 35.1 for
// 29.1): 128 tokens, groups of 4, behind 16000 in 16 ranges 56 (64 rows 68); 512 behind 8000 in 4 92 (118); 300 behind 2000 in 6 36 (38); but 500 tokens of 8 heads on
// one behind 3000 in 16 33 (26).
//   64 rows else: 2 of 512 tokens, groups of 4, 18.0 (with halves 20.9); 32 heads of 768 in halves 21.0 (23.1); 77 tokens behind 1411 in halves and 3 ranges 21.6
// (without ranges 26.9, without halves in 3 22.9, halves in 4 29.7).
struct Prompt4Form { int rows, halves, ranges; };
static Prompt4Form prompt_form(int B, int M, int H, int Hk, int Dh, int S) {
  const int64_t pairs = (int64_t)B * Hk, list = (int64_t)M * (H / Hk), cu = 256, wide = (list + 127) / 128 * pairs, tiles = S / kTile4;
  const int64_t ranges = max((int64_t)1, min(2 * cu / wide, (int64_t)16)), least = 4 * wide >= 3 * cu ? 32 : Dh == 128 ? 6 : 12;
  if (ranges > 1 && ranges * wide >= cu && tiles >= least * ranges) return {128, 1, (int)ranges};
  if (Dh == 64 ? wide >= 2 * cu : (S >= 2 * (int64_t)M ? 4 : 2) * wide >= 3 * cu) return {128, 1, 1};
  const int64_t n = (list + 63) / 64 * pairs;
  if (n * 2 > 3 * cu) return {64, 1, 1};
  return {64, 2, (int)max((int64_t)1, min(cu / n, (int64_t)S / ((n * 4 > cu ? 8 : 4) * kTile4)))};
}
size_t kv4_prompt_scratch_bytes(int B, int M, int H, int Hk, int Dh, int S) {
  const Prompt4Form f = prompt_form(B, M, H, Hk, Dh, S);
  return f.ranges > 1 ? RangeParts::bytes((int64_t)B * M * H, f.ranges, Dh) : 0;
}

template <int DT, int DH, int KG, bool TWO>
static int prompt_launch_form(const char* fn, const Kv4AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  constexpr size_t lds = KG * 2 * ((size_t)kTile4 * (DH + 16) * 2 + (size_t)DH * kTile4 * 2);
  static std::atomic<uint32_t> granted{0};
  if (const int rc = lds > 65536 ? grant_lds(fn, reinterpret_cast<const void*>(&kv4_prompt_kernel<DT, DH, KG, TWO>), lds, granted) : kOk) return rc;
  const int64_t list = (int64_t)a.M * (a.H / a.c.Hk), groups = (list + 16 * kPrompt4Waves - 1) / (16 * kPrompt4Waves) * a.B * a.c.Hk;
  if (list > 0x7fffffff - 256 || groups > 0x7fffffff) { set_last_error("%s: %d rows of %d heads", fn, a.M, a.H); return kErrBadShape; }
  hipLaunchKernelGGL((kv4_prompt_kernel<DT, DH, KG, TWO>), dim3((unsigned)groups, ranges), dim3(kPrompt4Waves * KG * kWave), lds, st, a, ranges, scratch);
  if (ranges > 1) launch_join(join_args(a), ranges, false, scratch, st);
  return kOk;
}
template <int DT, int DH, int KG>
static int prompt_launch(const char* fn, const Kv4AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  if constexpr (DT == 1) return prompt_launch_form<DT, DH, KG, true>(fn, a, ranges, scratch, st);
  else return a.cos ? prompt_launch_form<DT, DH, KG, true>(fn, a, ranges, scratch, st) : prompt_launch_form<DT, DH, KG, false>(fn, a, ranges, scratch, st);
}
template <int DT, int DH, bool TWO>
static int wide_launch(const char* fn, const Kv4AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  constexpr size_t lds = 2 * ((size_t)kTile4 * (DH + 8) * 2 + (size_t)DH * kTile4 * 2);
  static std::atomic<uint32_t> granted{0};
  if (const int rc = lds > 65536 ? grant_lds(fn, reinterpret_cast<const void*>(&kv4_wide_kernel<DT, DH, TWO>), lds, granted) : kOk) return rc;
  const int64_t list = (int64_t)a.M * (a.H / a.c.Hk), groups = (list + 32 * kPrompt4Waves - 1) / (32 * kPrompt4Waves) * a.B * a.c.Hk;
  if (list > 0x7fffffff - 256 || groups > 0x7fffffff) { set_last_error("%s: %d rows of %d heads", fn, a.M, a.H); return kErrBadShape; }
  hipLaunchKernelGGL((kv4_wide_kernel<DT, DH, TWO>), dim3((unsigned)groups, ranges), dim3(kPrompt4Waves * kWave), lds, st, a, ranges, scratch);
  if (ranges > 1) launch_join(join_args(a), ranges, false, scratch, st);
  return kOk;
}
template <int DT, int DH>
static int prompt_launch_rows(const char* fn, const Kv4AttnArgs& a, Prompt4Form f, float* scratch, hipStream_t st) {
  set_last_form(f.rows == 128 ? (f.ranges == 1 ? "kv4 prompt 128" : "kv4 prompt 128 ranges") : f.halves == 1 ? "kv4 prompt 64" : f.ranges == 1 ? "kv4 prompt 64 halves" : "kv4 prompt 64 halves ranges");
  if (f.rows == 128) {
    if constexpr (DT == 1) return wide_launch<DT, DH, true>(fn, a, f.ranges, scratch, st);
    else return a.cos ? wide_launch<DT, DH, true>(fn, a, f.ranges, scratch, st) : wide_launch<DT, DH, false>(fn, a, f.ranges, scratch, st);
  }
  if (f.halves == 1) return prompt_launch<DT, DH, 1>(fn, a, f.ranges, scratch, st);
  return prompt_launch<DT, DH, 2>(fn, a, f.ranges, scratch, st);
}
int launch_kv4_prompt(const char* fn, const Kv4AttnArgs& a, float* scratch, size_t scratch_bytes, hipStream_t st) {
  const Prompt4Form f = prompt_form(a.B, a.M, a.H, a.c.Hk, a.c.Dh, a.c.S);
  const size_t need = kv4_prompt_scratch_bytes(a.B, a.M, a.H, a.c.Hk, a.c.Dh, a.c.S);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15))) {
    set_last_error("%s: %zu bytes of scratch for %d key ranges, %zu needed", fn, scratch ? scratch_bytes : (size_t)0, f.ranges, need);
    return kErrWorkspace;
  }
  const int rc = a.dt == 1 ? (a.c.Dh == 128 ? prompt_launch_rows<1, 128>(fn, a, f, scratch, st) : prompt_launch_rows<1, 64>(fn, a, f, scratch, st))
                           : (a.c.Dh == 128 ? prompt_launch_rows<0, 128>(fn, a, f, scratch, st) : prompt_launch_rows<0, 64>(fn, a, f, scratch, st));
  if (rc != kOk) return rc;
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

}  // namespace fsvd
