// Attention over the KV cache in 8 bits.
#include "attn_join.hpp"
#include "kv8.hpp"

namespace fsvd {

// eight elements x of a query row in the lower or upper half of the head, rotated with their partners y half a head away, in fp32 and rounded to the type of
// the products; rest: what that rounding leaves.  A pair of large float16 elements may turn to one beyond the type's range (up to 1.42 times its end): the first
// part stops at the end, the rest has the remainder.
template <class E>
__device__ __forceinline__ u32x4_t rotated(u32x4_t x, u32x4_t y, u32x4_t cos, u32x4_t sin, bool upper, u32x4_t& rest) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float sl = upper ? E::lo(sin[i]) : -E::lo(sin[i]), sh = upper ? E::hi(sin[i]) : -E::hi(sin[i]);
    const float l = E::lo(x[i]) * E::lo(cos[i]) + E::lo(y[i]) * sl, h = E::hi(x[i]) * E::hi(cos[i]) + E::hi(y[i]) * sh;
    constexpr float kEnd = 65504.f;
    const uint32_t w = E::code == 1 ? E::pack2(__builtin_amdgcn_fmed3f(l, -kEnd, kEnd), __builtin_amdgcn_fmed3f(h, -kEnd, kEnd)) : E::pack2(l, h);
    x[i] = w;
    rest[i] = E::pack2(l - E::lo(w), h - E::hi(w));
  }
  return x;
}
__device__ __forceinline__ u32x4_t eight(const uint16_t* p) { return __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(p)); }
static JoinArgs join_args(const Kv8AttnArgs& a) { return {a.out, a.so_b, a.so_m, a.so_h, a.rows, a.B, a.M, a.H, a.c.Hk, a.c.Dh, a.dt}; }

// The maximum of a row that has seen no score yet.  A score may be -infinity where fp32 does not hold it, and has no weight against this, where its distance from
// another -infinity is no number.
constexpr float kLowest8 = -__FLT_MAX__;

// Keys of a decode range, but for the last: a step of every wave, and whole blocks.
constexpr int kMinRange = 128;
__host__ __device__ __forceinline__ int kv8_range(int keys, int ranges) {
  const int per = (keys + ranges - 1) / ranges;
  return (max(per, 1) + kMinRange - 1) / kMinRange * kMinRange;
}

// ---------------------------------------------------------------------------------------------
// One query token per sequence.  A workgroup takes a range of the keys of one kv head for up to 16 of its query heads, a wave every fourth step of 32
// keys, on the matrix cores: S^T = K Q^T, O^T = V^T P^T (16 x 16 x 32).
//   K: lane (n, g) = (lane % 16, lane / 16) loads 16-byte pieces of key n: the order of the products' k axis is free as long as q is laid out the same.
//   S^T leaves lane (n, g) the scores of query n and keys 4 g .. 4 g + 3 of the two 16-key tiles: eight weights that are one operand of the second product.
//   V: lane (n, g) loads those eight keys' dimensions DH / 16 n .. of the row, and byte permutes put two keys of a dimension next to each other.
// Codes become 16-bit elements exactly; a scale multiplies what one tile of 16 keys has in common, the scores and the weights.  The weights go
// into the second product as two bf16 parts, 16 significant bits.
// Bound by the bytes of the cache: 16 x 4090 keys of 32 heads of 128 (537 MB) in 93 us and a join of 5, 5.5 TB/s, 16 x 1000 to 4001 keys of 8 kv heads (92 MB) in 25 and a
// join of 4; small calls by the latency of a few dependent loads (137 keys of 8 heads of 64: 5.7 us).  A rotated q goes into the first product as
// two parts of its type: one rounding of it would be the largest error of the output (0.0036 of its size against 0.0016 in bf16, the output's own rounding) and
// saves 2 to 3 % of a call.  Three waves a SIMD hold that; four spill (stress call: 131 us against 102).
// ---------------------------------------------------------------------------------------------
constexpr int kDecWaves = 4, kDecStep = 32, kDecGroup = 16;

template <int DT, int DH>
__global__ __launch_bounds__(kDecWaves * kWave, 3) void kv8_decode_kernel(Kv8AttnArgs a, int ranges, float* scratch) {
  typedef E16<DT> E;
  typedef typename E::frag_t frag_t;
  typedef E16<0>::frag_t pfrag_t;
  constexpr int J = DH / 64, ST = DH / 32, NT = DH / 16, VW = DH / 64;      // 16-byte pieces of a key; products a tile; output tiles; words of a value piece
  extern __shared__ __align__(16) float os[];                               // [kDecWaves][heads of a workgroup][DH + 4]
  __shared__ float ms[kDecWaves][kDecGroup], ls[kDecWaves][kDecGroup];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  const int G = a.H / a.c.Hk, GG = (G + kDecGroup - 1) / kDecGroup;
  // The heads of a sequence, whose ranges are alike, on different XCDs; the last range of every sequence, which may hold the new row, first.
  const int pairs = a.B * a.c.Hk * GG, turn = blockIdx.x / pairs;
  int id = blockIdx.x - turn * pairs;
  const int gg = id % GG; id /= GG;
  const int b = id / a.c.Hk, hk = id - b * a.c.Hk;
  const int pos = a.positions[b], keys = (int)max((int64_t)0, min((int64_t)pos + a.key_add, (int64_t)a.c.S));
  const int per = kv8_range(keys, ranges), used = max(1, (keys + per - 1) / per), s = turn < used ? used - 1 - turn : turn;
  const int k0 = min(s * per, keys), k1 = min(k0 + per, keys);
  const int h0 = hk * G + gg * kDecGroup, heads = min(kDecGroup, G - gg * kDecGroup);
  const RangeParts part{scratch, (int64_t)a.B * a.H, ranges, DH};
  if (s >= used) {
    if (tid < heads) *part.stats((int64_t)b * a.H + h0 + tid, s) = f32x2_t{-INFINITY, 0.f};
    return;
  }

  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint32_t row = (uint32_t)a.c.sc_s;                                  // a step's first row is the wave's, 64 bits; from there on 32 do
  const float* ksp = a.c.k_scale + b * a.c.ss_b + hk * a.c.ss_h;
  const float* vsp = a.c.v_scale + b * a.c.ss_b + hk * a.c.ss_h;
  const int shift = 31 - __builtin_clz(a.c.block);
  u32x4_t kr[2][J];
  uint32_t vr[8][VW];
  float ks[2], vs[2];
  const auto fetch_k = [&](int c0) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t off = (uint32_t)min(16 * t + n, k1 - 1 - c0) * row + 16 * g;
#pragma unroll
      for (int j = 0; j < J; ++j) kr[t][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(kb + (int64_t)c0 * a.c.sc_s + off + 64 * j));
      ks[t] = ksp[(int64_t)(min(c0 + 16 * t, k1 - 1) >> shift) * a.c.ss_n];
    }
  };
  const auto fetch_v = [&](int c0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t* p = vb + (int64_t)c0 * a.c.sc_s + ((uint32_t)min(16 * (e >> 2) + 4 * g + (e & 3), k1 - 1 - c0) * row + n * NT);
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
  // The new row is the last key.  Ranges are whole blocks, so this workgroup alone reads the block that the row may change; one wave writes the row while the
  // others begin, and the steps that touch its block come behind a barrier.
  const bool appends = a.k_new != nullptr && pos >= k0 && pos < k1;
  const int before = appends ? (pos >> shift << shift) - (kDecStep - 1) : k1;
  if (appends && wave == kDecWaves - 1)
    append_row<DT, DH>(a.c, a.k_new + (int64_t)b * a.sk_b + (int64_t)hk * a.sk_h, a.v_new + (int64_t)b * a.sv_b + (int64_t)hk * a.sv_h, a.cos, a.sin, a.rope_len,
                       b, hk, pos, lane);
  if (c0 < before) { fetch_k(c0); fetch_v(c0); }

  // q: element e of piece (j, h) is dimension 64 j + 16 g + 8 h + e of query n, rotated in fp32, as two parts of the type of the products then
  frag_t qf[ST], qr[ST];
  {
    const uint16_t* qp = a.q + (int64_t)b * a.sq_b + (int64_t)(h0 + min(n, heads - 1)) * a.sq_h;
    constexpr int HALF = DH / 2;
    const auto dim = [&](int st) { return 64 * (st >> 1) + 16 * g + 8 * (st & 1); };
    u32x4_t x[ST], z[ST], y[2], cw[2], sw[2];
#pragma unroll
    for (int st = 0; st < ST; ++st) z[st] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int st = 0; st < ST; ++st) x[st] = eight(qp + dim(st));
    if (a.cos) {
      const int64_t tp = (int64_t)min(max(pos, 0), a.rope_len - 1) * HALF;
#pragma unroll
      for (int h = 0; h < 2; ++h) {                       // of 128 dimensions the partner is the lane's own, of 64 another lane has it
        if constexpr (DH == 64) y[h] = eight(qp + (dim(h) ^ HALF));
        cw[h] = eight(a.cos + tp + dim(h) % HALF);
        sw[h] = eight(a.sin + tp + dim(h) % HALF);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (DH == 64) {
          x[h] = rotated<E>(x[h], y[h], cw[h], sw[h], dim(h) >= HALF, z[h]);
        } else {
          const u32x4_t low = x[h];
          x[h] = rotated<E>(low, x[h + 2], cw[h], sw[h], false, z[h]);
          x[h + 2] = rotated<E>(x[h + 2], low, cw[h], sw[h], true, z[h + 2]);
        }
      }
    }
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      qf[st] = __builtin_bit_cast(frag_t, n < heads ? x[st] : u32x4_t{0u, 0u, 0u, 0u});
      qr[st] = __builtin_bit_cast(frag_t, n < heads ? z[st] : u32x4_t{0u, 0u, 0u, 0u});
    }
  }

  const float scale = a.scale * 1.4426950408889634f;      // weights are powers of two of the scores' differences
  float m = kLowest8, l = 0.f;
  f32x4_t o[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const auto walk = [&](int stop) {
  for (; c0 < stop; c0 += kDecWaves * kDecStep) {
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
          acc = E::mfma(__builtin_bit_cast(frag_t, kk), qr[2 * j + h], acc);
        }
      const float by = ks[t] * scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[t][i] = acc[i] * by;
      f[t] = vs[t];
    }
    if (next < stop) fetch_k(next);
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
  // the waves' results through LDS: element i of tile t is dimension NT (4 g + i) + t of query n
  l = column_sum(l);
  if (g == 0) { ms[wave][n] = l != l ? INFINITY : m == kLowest8 ? -INFINITY : m; ls[wave][n] = l; }
  if (n < heads) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < NT; t += 4)
        *reinterpret_cast<f32x4_t*>(os + (wave * heads + n) * (DH + 4) + NT * (4 * g + i) + t) = f32x4_t{o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]};
  }
  __syncthreads();
  for (int e = tid; e < heads * DH; e += kDecWaves * kWave) {
    const int q = e / DH, d = e % DH;
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) top = fmaxf(top, ms[w][q]);
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
      const float f = ms[w][q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[w][q] - top);
      sum += f * ls[w][q];
      v += f * os[(w * heads + q) * (DH + 4) + d];
    }
    if (ranges == 1) {
      a.out[(int64_t)b * a.so_b + (int64_t)(h0 + q) * a.so_h + d] = (uint16_t)E::bits(sum == 0.f ? 0.f : v / sum);
    } else {
      const int64_t row = (int64_t)b * a.H + h0 + q;
      part.values(row, s)[d] = v;
      if (d == 0) *part.stats(row, s) = f32x2_t{top, sum};
    }
  }
}

// Ranges of a decode call (times in us from a captured graph, 32 heads of 128 over 8).  S is the room of the cache: what it holds is known on the device only,
// so short sequences in a long cache are cut too (without an append, 137 keys of 8 heads of 64 in room for 160: 4.5, for 4096: 6.3; 16 sequences of 4090 keys with 32 kv heads in
// room for 4091: 96, for 32768: 101).
//  - About two workgroups for each compute unit: with 512 / 640 / 1024 in all one sequence of 30000 keys takes 20.3 / 22.2 / 23.1, 64 of 2000 49.5 / 52.9 / 52.4;
//    with 384 one sequence of 16001 takes 16.4 against 14.3.
//  - Ranges of 2048 keys at most: 16 sequences of 4090 keys with 32 kv heads take 105 in one range, 97 to 102 in three, 114 in six.
//  - One range below 384 keys (137 keys of 8 heads of 64: 5.7, in two 7.5), else down to 128 keys (one sequence of 400 keys 8.3, with 256 at least 9.5; of 4000
//    9.5 and 10.9; of 8000 12.4 and 11.4).
int kv8_ranges(int B, int H, int Hk, int S, int nsplit) {
  const int most = S < 384 ? 1 : (S + kMinRange - 1) / kMinRange;
  if (nsplit <= 0) {
    const int64_t pairs = (int64_t)B * Hk * ((H / Hk + kDecGroup - 1) / kDecGroup);
    nsplit = max((int)((512 + pairs - 1) / pairs), (S + 2047) / 2048);
  }
  return max(1, min(nsplit, most));
}
size_t kv8_decode_scratch_bytes(int B, int H, int Dh, int ranges) { return ranges > 1 ? RangeParts::bytes((int64_t)B * H, ranges, Dh) : 0; }

template <int DT, int DH>
static void decode_form(const Kv8AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  const int groups = (a.H / a.c.Hk + kDecGroup - 1) / kDecGroup;
  hipLaunchKernelGGL((kv8_decode_kernel<DT, DH>), dim3((unsigned)a.B * a.c.Hk * groups * ranges), dim3(kDecWaves * kWave),
                     kDecWaves * min(a.H / a.c.Hk, kDecGroup) * (DH + 4) * sizeof(float), st, a, ranges, scratch);
  if (ranges > 1) launch_join(join_args(a), ranges, true, scratch, st);
  set_last_form(ranges == 1 ? "kv8 decode" : ranges <= 8 ? "kv8 decode ranges" : ranges <= kWave ? "kv8 decode ranges 9" : "kv8 decode ranges 65");
}
int launch_kv8_decode(const char* fn, const Kv8AttnArgs& args, int ranges, float* scratch, hipStream_t st) {
  Kv8AttnArgs a = args;
  if ((int64_t)a.B * a.H * ranges > (1 << 23)) { set_last_error("%s: %d sequences of %d heads in %d ranges", fn, a.B, a.H, ranges); return kErrBadShape; }
  if (a.k_new != nullptr && a.H / a.c.Hk > kDecGroup) {    // several workgroups read the keys of a kv head: the rows in a launch before them
    const Kv8AppendArgs n{a.c, a.k_new, a.sk_b, 0, a.sk_h, a.v_new, a.sv_b, 0, a.sv_h, a.positions, nullptr, a.cos, a.sin, a.rope_len, a.B, 1, a.dt};
    if (const int rc = launch_kv8_append(fn, n, st)) return rc;
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
// the tiles of keys too.  A workgroup of four waves takes 16 MI rows for each; tiles of 64 keys go through LDS as 16-bit elements, converted once for
// the workgroup: K row by row, V transposed (two keys of a dimension next to each other by byte permutes), two buffers and one barrier a tile.
//   S^T = K Q^T leaves a lane four consecutive keys of one query in every 16-key block, O^T = V^T P^T takes them as they stand (the V columns of 32 keys
//   follow the order 16 (e / 4) + 4 g + e % 4 of the products' k axis).
//   The key scale of a block multiplies its maximum and goes into the multiply-add in front of the exponential; the power of two of the value scale into the
//   conversion.
//   The weights go into the second product as two bf16 parts, 16 significant bits, and into their sums as they are: rounded to one, outputs in bf16 are off by
//   0.0020 of their size instead of 0.0016 (their own rounding), and 8 x 2048 tokens take four fifths of the time.  A q that the call rotates
//   is two parts of its type: rounded once, float16 outputs are off by 0.0004 of their size instead of 0.0002, 77 tokens behind 1411 take 4 % less and 8 x 2048,
//   whose workgroups of 128 rows have registers for the fragments of 32 keys at a time only, 12 %.
// V columns: 16-byte pieces of the 128-byte rows are XOR-ed with (d / 4 % 8) ^ (d & 6), which keeps the fragments' 16-byte reads and the 8-byte transposing
// writes off each other's banks (found by enumeration).
// ---------------------------------------------------------------------------------------------
// Two halves of waves (KG = 2) take every other tile and add up at the end, in a workgroup of its own for a compute unit, where there are few.
// 8 x 2048 tokens, 32 heads of 128: 445 us, 618 TFLOP/s of the formula's operations and half as many again for the second parts, 927 in all, where a large
// product of the library reaches 1189.  The vector unit (conversion, softmax, parts of the weights) is busy half of the time, the matrix cores 40 %, LDS a third; they
// overlap in part.  Short chunks are bound by the time of a tile.
constexpr int kTile = 64, kPromptWaves = 4;
constexpr float kSlack = 8.f;                             // with a reference that moves with every larger score 8 x 2048 tokens take 1.3 % more
__device__ __forceinline__ int v_piece(int d) { return ((d >> 2) & 7) ^ (d & 6); }
// A value scale as a power of two, which goes into the conversion of the codes to bf16 exactly, and the factor that it leaves, which is multiplied to the
// weights in front of their rounding: 1 for the scales that kv8_append makes (looking for others costs 1 to 4 %).  A zero, a subnormal, an infinity and a NaN are
// all factor.
__device__ __forceinline__ bool is_power(float scale) {
  const uint32_t u = __float_as_uint(scale);
  return (u & 0x807fffffu) == 0 && u != 0 && u != 0x7f800000u;
}
__device__ __forceinline__ float power_of(float scale) {
  const uint32_t e = __float_as_uint(scale) & 0x7f800000u;
  return e == 0 || e == 0x7f800000u ? 1.f : __uint_as_float(e);
}
__device__ __forceinline__ float factor_of(float scale) {
  const uint32_t u = __float_as_uint(scale), e = u & 0x7f800000u;
  return e == 0 || e == 0x7f800000u ? scale : __uint_as_float((u & 0x807fffffu) | 0x3f800000u);
}
template <bool HI>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t w, float power) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, HI));
}

template <int DT, int DH, int MI, int KG, bool TURN>
__global__ __launch_bounds__(kWave * kPromptWaves * KG, 2) void kv8_prompt_kernel(Kv8AttnArgs a, int ranges, float* scratch) {
  typedef E16<DT> E;
  typedef typename E::frag_t frag_t;
  typedef E16<0>::frag_t pfrag_t;
  constexpr int ST = DH / 32, NT = DH / 16, KSTR = DH + 16, TH = kWave * kPromptWaves, QW = 16 * MI, BM = QW * kPromptWaves;
  constexpr int KL = DH / 16, KP = kTile * KL / TH;              // lanes of a key row; passes of the workgroup over the tile's keys
  constexpr int VL = DH / 4, VP = kTile / 4 * VL / TH;
  extern __shared__ __align__(16) unsigned char smem[];
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TH) : 0;
  uint16_t* Ks = reinterpret_cast<uint16_t*>(smem) + kg * 2 * kTile * (KSTR + DH);      // [2][kTile][KSTR]
  uint16_t* Vt = Ks + 2 * kTile * KSTR;                                     // [2][DH][kTile]
  __shared__ __align__(16) int nan_at[DH];                                  // the first NaN of a dimension among the values that not every row sees
  __shared__ int any_nan;
  __shared__ int odd_tile[KG][2];                                           // the last tile of a buffer with a value scale that is no power of two

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
  const auto seen_by = [&](int r) { return max(0, min(pos + r / G + a.key_add, a.c.S)); };     // keys of row r
  const int all_end = seen_by(min(row0 + BM, rows) - 1);
  const int tiles = (all_end + kTile - 1) / kTile, per = (tiles + ranges - 1) / ranges;
  const int n_begin = range * per * kTile, n_end = min(all_end, (range + 1) * per * kTile);
  const int w0 = row0 + wave * QW;
  const int wave_end = w0 < rows ? min(n_end, seen_by(min(w0 + QW, rows) - 1)) : 0;             // keys past it are unseen by the wave

  constexpr bool kTight = TURN && MI == 2 && DH == 128;                     // fragments of 32 keys at a time: the registers hold no more beside both parts of q
  frag_t qf[MI][ST], qr[TURN ? MI : 1][ST];                                 // qr: what the rounding of a rotated q leaves
  int seen[MI];
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int r = min(w0 + 16 * mi + lr, rows - 1), m = r / G, h = hk * G + r - m * G;
    seen[mi] = seen_by(r);
    const uint16_t* qp = a.q + (int64_t)b * a.sq_b + (int64_t)m * a.sq_m + (int64_t)h * a.sq_h;
    constexpr int HALF = DH / 2, SH = ST / 2;
    u32x4_t x[ST], cw[SH], sw[SH];
#pragma unroll
    for (int st = 0; st < ST; ++st) x[st] = eight(qp + 32 * st + 8 * lg);
    if constexpr (TURN) {
      const int64_t tp = (int64_t)min(max(pos + m, 0), a.rope_len - 1) * HALF + 8 * lg;
#pragma unroll
      for (int st = 0; st < SH; ++st) { cw[st] = eight(a.cos + tp + 32 * st); sw[st] = eight(a.sin + tp + 32 * st); }
#pragma unroll
      for (int st = 0; st < SH; ++st) {
        const u32x4_t low = x[st];
        u32x4_t r0, r1;
        x[st] = rotated<E>(low, x[st + SH], cw[st], sw[st], false, r0);
        x[st + SH] = rotated<E>(x[st + SH], low, cw[st], sw[st], true, r1);
        if constexpr (kTight) asm volatile("" : "+v"(r0), "+v"(r1), "+v"(x[st]), "+v"(x[st + SH]));       // made here: put off, they spill
        qr[mi][st] = __builtin_bit_cast(frag_t, r0);
        qr[mi][st + SH] = __builtin_bit_cast(frag_t, r1);
      }
    }
#pragma unroll
    for (int st = 0; st < ST; ++st) qf[mi][st] = __builtin_bit_cast(frag_t, x[st]);
  }
  const float scale = a.scale * 1.4426950408889634f;
  float m_run[MI];
  float l_run[MI];                                                          // a lane's own sum of the weights, not rounded
  f32x4_t o[MI][NT];
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    m_run[mi] = -INFINITY; l_run[mi] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[mi][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + b * a.c.sc_b + hk * a.c.sc_h;
  const float* ksp = a.c.k_scale + b * a.c.ss_b + hk * a.c.ss_h;
  const float* vsp = a.c.v_scale + b * a.c.ss_b + hk * a.c.ss_h;
  const int shift = 31 - __builtin_clz(a.c.block);
  // K: KL lanes with 16 codes each for a row; V: VL lanes with 4 codes each for four adjacent keys
  const int krow = tid / KL, kd = tid % KL * 16, vrow = tid / VL, vd = tid % VL * 4;
  u32x4_t kreg[KP];
  uint32_t vreg[VP][4];
  float vscale[VP];
  // a tile's first row is the workgroup's, 64 bits; from there on 32 do (and stay the same from tile to tile, but for one that the range ends in)
  const uint32_t line = (uint32_t)a.c.sc_s;
  uint32_t koff[KP], voff[VP][4], kso, vso[VP];
  const uint32_t step = (uint32_t)a.c.ss_n * 4;
  const auto k_offset = [&](int p, int left) { return (uint32_t)min(krow + p * (TH / KL), left - 1) * line + kd; };
  const auto v_offset = [&](int p, int e, int left) { return (uint32_t)min(4 * (vrow + p * (TH / VL)) + e, left - 1) * line + vd; };
  const auto s_offset = [&](int row, int left) { return (uint32_t)(min(row, left - 1) >> shift) * step; };      // of a tile's row, tiles begin with blocks or lie in one
  const auto scale_at = [&](const float* base, int n0, uint32_t off) {
    return *reinterpret_cast<const float*>(reinterpret_cast<const char*>(base + (int64_t)(n0 >> shift) * a.c.ss_n) + off);
  };
  const auto request_k = [&](int n0) {
    if (n0 + kTile > n_end) {
#pragma unroll
      for (int p = 0; p < KP; ++p) koff[p] = k_offset(p, n_end - n0);
    }
    const uint8_t* kt = kb + (int64_t)n0 * a.c.sc_s;
#pragma unroll
    for (int p = 0; p < KP; ++p) kreg[p] = *reinterpret_cast<const u32x4_t*>(kt + koff[p]);
  };
  const auto request_v = [&](int n0) {
    if (n0 + kTile > n_end) {
#pragma unroll
      for (int p = 0; p < VP; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) voff[p][e] = v_offset(p, e, n_end - n0);
#pragma unroll
      for (int p = 0; p < VP; ++p) vso[p] = s_offset(4 * (vrow + p * (TH / VL)), n_end - n0);
    }
    const uint8_t* vt = vb + (int64_t)n0 * a.c.sc_s;
#pragma unroll
    for (int p = 0; p < VP; ++p) {
#pragma unroll
      for (int e = 0; e < 4; ++e) vreg[p][e] = *reinterpret_cast<const uint32_t*>(vt + voff[p][e]);
      vscale[p] = scale_at(vsp, n0, vso[p]);
    }
  };
  float fs;                              // the key scale of block lane % 4 of a tile's four blocks of 16 keys (by a vector load: a scalar one would be waited for here)
  const auto request_f = [&](int n0) {
    if (n0 + kTile > n_end) kso = s_offset(16 * (lane & 3), n_end - n0);
    fs = scale_at(ksp, n0, kso);
  };
  const auto stage_k = [&](int buf) {
    uint16_t* ks = Ks + buf * kTile * KSTR;
#pragma unroll
    for (int p = 0; p < KP; ++p)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = kreg[p][2 * h], y = kreg[p][2 * h + 1];
        *reinterpret_cast<u32x4_t*>(ks + (krow + p * (TH / KL)) * KSTR + kd + 8 * h) = u32x4_t{
            Code16<DT>::template pair<false>(x), Code16<DT>::template pair<true>(x), Code16<DT>::template pair<false>(y), Code16<DT>::template pair<true>(y)};
      }
  };
  // A masked key has weight zero, and zero times a NaN is one: where not every row sees the whole tile, a NaN is staged as zero and put into the rows that see
  // it at the end.
  const int all_see = seen_by(row0);
  const auto set_nans_aside = [&](int n0) {
#pragma unroll
    for (int p = 0; p < VP; ++p) {
      const int row = 4 * (vrow + p * (TH / VL));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t nan = ((vreg[p][e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        if (__builtin_expect(!__any(nan != 0), 1)) continue;
        any_nan = 1;
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
          if (nan >> (8 * i + 7) & 1) atomicMin(&nan_at[vd + i], n0 + row + e);
        vreg[p][e] &= ~((nan >> 7) * 0xffu);
      }
    }
  };
  const auto stage_v = [&](int buf, int tile) {
    uint16_t* vt = Vt + buf * DH * kTile;
#pragma unroll
    for (int p = 0; p < VP; ++p) {
      const int row4 = vrow + p * (TH / VL);
      const int ko = (4 * row4) & 31, col = ((4 * row4) & 32) + 8 * ((ko & 15) >> 2) + 4 * (ko >> 4);
      uint16_t* to = vt + vd * kTile;
      const uint32_t turned = col ^ (8 * v_piece(vd));          // of rows vd and vd + 1; of the next two the piece two further
      float power = vscale[p];
      if (__builtin_expect(!__all(is_power(power)), 0)) {
        power = power_of(power);
        odd_tile[kg][buf] = tile;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t lo = __builtin_amdgcn_perm(vreg[p][1], vreg[p][0], c ? 0x07030602u : 0x05010400u);
        const uint32_t hi = __builtin_amdgcn_perm(vreg[p][3], vreg[p][2], c ? 0x07030602u : 0x05010400u);
        uint16_t* at = to + (c ? turned ^ 16 : turned) + 2 * c * kTile;
        *reinterpret_cast<u32x2_t*>(at) = u32x2_t{scaled_pair<false>(lo, power), scaled_pair<false>(hi, power)};
        *reinterpret_cast<u32x2_t*>(at + kTile) = u32x2_t{scaled_pair<true>(lo, power), scaled_pair<true>(hi, power)};
      }
    }
  };
  // Fragments are asked for ahead of the products: left to itself the compiler asks for each in front of its use.
  const auto k_frags = [&](frag_t (&kf)[2][ST], int buf, int half) {       // of 32 of the tile's keys
    const uint16_t* ks = Ks + buf * kTile * KSTR;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int st = 0; st < ST; ++st) kf[j][st] = __builtin_bit_cast(frag_t, *reinterpret_cast<const u32x4_t*>(ks + (32 * half + 16 * j + lr) * KSTR + 32 * st + 8 * lg));
  };
  const auto scores = [&](f32x4_t (&s)[MI][4], const frag_t (&kf)[2][ST], int half) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
          s[mi][2 * half + j] = E::mfma(kf[j][st], qf[mi][st], st ? s[mi][2 * half + j] : f32x4_t{0.f, 0.f, 0.f, 0.f});
          if constexpr (TURN) s[mi][2 * half + j] = E::mfma(kf[j][st], qr[mi][st], s[mi][2 * half + j]);
        }
  };
  // row d = 16 t + lr of V: its piece is turned by (lr / 4) ^ (lr & 6) ^ 4 (t % 2), so two addresses and constants reach all of them
  const uint32_t vread = lr * kTile + 8 * (lg ^ (lr >> 2) ^ (lr & 6));
  const auto v_frags = [&](pfrag_t (&vf)[NT], int buf, int st) {
    const uint16_t* vt = Vt + buf * DH * kTile;
#pragma unroll
    for (int t = 0; t < NT; ++t) vf[t] = __builtin_bit_cast(pfrag_t, *reinterpret_cast<const u32x4_t*>(vt + ((st ^ t) & 1 ? vread ^ 32 : vread) + 16 * t * kTile));
  };
  pfrag_t ph[MI][2], pl[MI][2];
  const auto values = [&](const pfrag_t (&vf)[NT], int st) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) {
        o[mi][t] = E16<0>::mfma(vf[t], ph[mi][st], o[mi][t]);
        o[mi][t] = E16<0>::mfma(vf[t], pl[mi][st], o[mi][t]);
      }
  };
  const int wave_sees = seen_by(min(w0, rows - 1));                  // keys of the wave's first row; the others see more from one to the next
  const auto weights = [&](f32x4_t (&s)[MI][4], int n0, float by, bool odd) {
    float f[4];
    by *= scale;
    const bool plain = n0 + kTile <= wave_sees;                      // every row of the wave sees the whole tile
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(by), j));
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      float top = -INFINITY;
      if (plain) {
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, f[j] * fmaxf(fmaxf(s[mi][j][0], s[mi][j][1]), fmaxf(s[mi][j][2], s[mi][j][3])));
      } else {
        const int vis = seen[mi] - n0 - 4 * lg;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[mi][j][i] = 16 * j + i < vis ? s[mi][j][i] * f[j] : -INFINITY;
            top = fmaxf(top, s[mi][j][i]);
          }
      }
      // The reference of the weights moves only where a score is kSlack over it: until then weights are up to 2^kSlack, which changes no rounding, and the
      // lanes of a column need not agree on a maximum.
      if (__any(top > m_run[mi] + kSlack)) {
        top = fmaxf(m_run[mi], column_max(top));
        const float keep = top > m_run[mi] ? __builtin_amdgcn_exp2f(m_run[mi] - top) : 1.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[mi][t] *= keep;
        l_run[mi] *= keep;
        m_run[mi] = top;
      }
      const float base = m_run[mi] == -INFINITY ? 0.f : m_run[mi];  // a row that has seen nothing yet: exp2(-inf - 0)
      if (plain) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mi][j][i] = fmaf(s[mi][j][i], f[j], -base);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mi][j][i] -= base;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[mi][j][i] = __builtin_amdgcn_exp2f(s[mi][j][i]);
          l_run[mi] += s[mi][j][i];
        }
    }
    if (__builtin_expect(odd, 0)) {
      const float mine = factor_of(scale_at(vsp, n0, s_offset(16 * (lane & 3), n_end - n0)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float left = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), j));
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) s[mi][j] *= left;
      }
    }
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        uint32_t hw[4], lw[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x0 = s[mi][2 * st + (c >> 1)][2 * (c & 1)], x1 = s[mi][2 * st + (c >> 1)][2 * (c & 1) + 1];
          hw[c] = pack_bf16x2(x0, x1);
          lw[c] = pack_bf16x2(x0 - bf16_lo(hw[c]), x1 - bf16_hi(hw[c]));
        }
        ph[mi][st] = __builtin_bit_cast(pfrag_t, u32x4_t{hw[0], hw[1], hw[2], hw[3]});
        pl[mi][st] = __builtin_bit_cast(pfrag_t, u32x4_t{lw[0], lw[1], lw[2], lw[3]});
      }
  };

#pragma unroll
  for (int p = 0; p < KP; ++p) koff[p] = k_offset(p, kTile);
#pragma unroll
  for (int p = 0; p < VP; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) voff[p][e] = v_offset(p, e, kTile);
  kso = s_offset(16 * (lane & 3), kTile);
#pragma unroll
  for (int p = 0; p < VP; ++p) vso[p] = s_offset(4 * (vrow + p * (TH / VL)), kTile);
  const auto at = [&](int i) { return n_begin + (i * KG + kg) * kTile; };
  const int all = n_begin < n_end ? (n_end - n_begin + kTile - 1) / kTile : 0, n = (all - kg + KG - 1) / KG;      // of the workgroup, of this half
  if (n > 0) { request_k(at(0)); request_v(at(0)); request_f(at(0)); }
  for (int d = tid; d < DH; d += TH) nan_at[d] = 0x7fffffff;
  if (tid == 0) any_nan = 0;
  if (tid < 2) odd_tile[kg][tid] = -1;
  __syncthreads();
  for (int i = 0; i * KG < all; ++i) {
    const int buf = i & 1;
    if (KG == 1 || i < n) {
      stage_k(buf);
      if (at(i) + kTile > all_see) set_nans_aside(at(i));
      stage_v(buf, i);
    }
    const float g = fs;
    if (i + 1 < n) { request_k(at(i + 1)); request_v(at(i + 1)); request_f(at(i + 1)); }
    __syncthreads();                   // this buffer is written; the other one is read by nobody any more
    if (at(i) >= wave_end || (KG > 1 && i >= n)) continue;
    f32x4_t s[MI][4];
    const bool odd = __builtin_amdgcn_readfirstlane(odd_tile[kg][buf]) == i;
    if constexpr (kTight) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        frag_t kf[2][ST];
        k_frags(kf, buf, half);
        scores(s, kf, half);
        __builtin_amdgcn_sched_barrier(0);
      }
      weights(s, at(i), g, odd);
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        __builtin_amdgcn_sched_barrier(0);
        pfrag_t vf[NT];
        v_frags(vf, buf, st);
        values(vf, st);
      }
    } else {
      frag_t kf[2][2][ST];
      k_frags(kf[0], buf, 0);
      k_frags(kf[1], buf, 1);
      __builtin_amdgcn_sched_barrier(0);
      scores(s, kf[0], 0);
      scores(s, kf[1], 1);
      pfrag_t vf[2][NT];               // those of V's first half during the softmax, of its second during the products with the first
      v_frags(vf[0], buf, 0);
      __builtin_amdgcn_sched_barrier(0);
      weights(s, at(i), g, odd);
      v_frags(vf[1], buf, 1);
      __builtin_amdgcn_sched_barrier(0);
      values(vf[0], 0);
      values(vf[1], 1);
    }
  }
  if constexpr (KG > 1) {                // the halves' results
    static_assert(KG == 2 && MI == 1, "one exchange");
    f32x4_t* part = reinterpret_cast<f32x4_t*>(smem) + wave * (NT + 1) * kWave + lane;
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t) part[t * kWave] = o[0][t];
      part[NT * kWave] = f32x4_t{m_run[0], l_run[0], 0.f, 0.f};
    }
    __syncthreads();
    if (kg == 1) return;
    const f32x4_t other = part[NT * kWave];
    const float top = fmaxf(m_run[0], other[0]);
    const float f0 = m_run[0] > -INFINITY ? __builtin_amdgcn_exp2f(m_run[0] - top) : 0.f, f1 = other[0] > -INFINITY ? __builtin_amdgcn_exp2f(other[0] - top) : 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) o[0][t] = o[0][t] * f0 + part[t * kWave] * f1;
    l_run[0] = l_run[0] * f0 + other[1] * f1;
    m_run[0] = top;
  }
  // element i of tile t is dimension 16 t + 4 lg + i of row lr
  const bool out8 = (reinterpret_cast<uintptr_t>(a.out) & 7) == 0 && (a.so_b % 4) == 0 && (a.so_m % 4) == 0 && (a.so_h % 4) == 0;
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int r = w0 + 16 * mi + lr;
    const float l = column_sum(l_run[mi]);
    if (r >= rows) continue;
    if (any_nan) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (nan_at[16 * t + 4 * lg + i] < seen[mi]) o[mi][t][i] = __builtin_nanf("");
    }
    if (ranges > 1) {
      const RangeParts part{scratch, (int64_t)HB * a.M * G, ranges, DH};
      const int64_t row = (int64_t)(b * a.c.Hk + hk) * a.M * G + r;
      if (lg == 0) *part.stats(row, range) = f32x2_t{m_run[mi], l};
      float* v = part.values(row, range) + 4 * lg;
#pragma unroll
      for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4_t*>(v + 16 * t) = o[mi][t];
      continue;
    }
    const int m = r / G, h = hk * G + r - m * G;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint16_t* op = a.out + (int64_t)b * a.so_b + (int64_t)m * a.so_m + (int64_t)h * a.so_h + 4 * lg;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const u32x2_t w{E::pack2(o[mi][t][0] * inv, o[mi][t][1] * inv), E::pack2(o[mi][t][2] * inv, o[mi][t][3] * inv)};
      if (out8) {
        *reinterpret_cast<u32x2_t*>(op + 16 * t) = w;
      } else {
        op[16 * t] = (uint16_t)w.x; op[16 * t + 1] = (uint16_t)(w.x >> 16);
        op[16 * t + 2] = (uint16_t)w.y; op[16 * t + 3] = (uint16_t)(w.y >> 16);
      }
    }
  }
}

// Rows of a workgroup, its halves and key ranges of a chunk (times in us from a captured graph of chunks without a past, 32 heads of 128, bf16, and of 64 tokens
// behind cached ones, 32 heads over 8).
//  - 128 rows share a tile better, 64 fill the chip and end evenly: 128 from two workgroups for each compute unit on (2 x 1024 tokens: 46.6 against 47.2;
//    8 x 2048: 443 against 542), else 64 (1500 tokens: 47.3 against 61.1).
//  - Up to one and a half workgroups of 64 rows for each compute unit, two halves of waves with every other tile (700 tokens: 17.7 against 21.9; 512: 13.9
//    against 16.5; 2 x 512, which are two for each: 19.8 against 18.2).
//  - Where these leave compute units idle, the keys in as many ranges as fill them once (64 behind 4800: 22.4 against 76.5 in one range and 31.5 in twice as
//    many), each of four tiles at least (64 behind 600: 14.6 against 16.2; behind 300: 12.2 against 11.2), of eight where the partial results are many (256
//    tokens without a past in ranges of two tiles: 16.8 against 9.6).
//  - S is the room of the cache, and ranges go by it: what the cache holds is known on the device only.  A chunk without a past in a long cache pays for empty
//    ranges and the join (256 tokens in room for 256: 9.9, for 1024 and more: 17.0; 64 tokens of 32 heads over 8: 6.7 and 13.3).
struct PromptForm { int rows, halves, ranges; };
static PromptForm prompt_form(int B, int M, int H, int Hk, int S) {
  const int64_t pairs = (int64_t)B * Hk, list = (int64_t)M * (H / Hk), cu = 256;
  if ((list + 127) / 128 * pairs >= 2 * cu) return {128, 1, 1};
  const int64_t n = (list + 63) / 64 * pairs;
  if (n * 2 > 3 * cu) return {64, 1, 1};
  return {64, 2, (int)max((int64_t)1, min(cu / n, (int64_t)S / ((n * 4 > cu ? 8 : 4) * kTile)))};
}
size_t kv8_prompt_scratch_bytes(int B, int M, int H, int Hk, int Dh, int S) {
  const PromptForm f = prompt_form(B, M, H, Hk, S);
  return f.ranges > 1 ? RangeParts::bytes((int64_t)B * M * H, f.ranges, Dh) : 0;
}

template <int DT, int DH, int MI, int KG, bool TURN>
static int prompt_launch_form(const char* fn, const Kv8AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  constexpr size_t lds = KG * 2 * ((size_t)kTile * (DH + 16) * 2 + (size_t)DH * kTile * 2);
  static std::atomic<uint32_t> granted{0};
  if (const int rc = lds > 65536 ? grant_lds(fn, reinterpret_cast<const void*>(&kv8_prompt_kernel<DT, DH, MI, KG, TURN>), lds, granted) : kOk) return rc;
  const int64_t list = (int64_t)a.M * (a.H / a.c.Hk), groups = (list + 16 * MI * kPromptWaves - 1) / (16 * MI * kPromptWaves) * a.B * a.c.Hk;
  if (list > 0x7fffffff - 256 || groups > 0x7fffffff) { set_last_error("%s: %d rows of %d heads", fn, a.M, a.H); return kErrBadShape; }
  hipLaunchKernelGGL((kv8_prompt_kernel<DT, DH, MI, KG, TURN>), dim3((unsigned)groups, ranges), dim3(kPromptWaves * KG * kWave), lds, st, a, ranges, scratch);
  if (ranges > 1) launch_join(join_args(a), ranges, false, scratch, st);
  return kOk;
}
template <int DT, int DH, int MI, int KG>
static int prompt_launch(const char* fn, const Kv8AttnArgs& a, int ranges, float* scratch, hipStream_t st) {
  return a.cos ? prompt_launch_form<DT, DH, MI, KG, true>(fn, a, ranges, scratch, st) : prompt_launch_form<DT, DH, MI, KG, false>(fn, a, ranges, scratch, st);
}
template <int DT, int DH>
static int prompt_launch_rows(const char* fn, const Kv8AttnArgs& a, PromptForm f, float* scratch, hipStream_t st) {
  set_last_form(f.rows == 128 ? "kv8 prompt 128" : f.halves == 1 ? "kv8 prompt 64" : f.ranges == 1 ? "kv8 prompt 64 halves" : "kv8 prompt 64 halves ranges");
  if (f.rows == 128) return prompt_launch<DT, DH, 2, 1>(fn, a, f.ranges, scratch, st);
  if (f.halves == 1) return prompt_launch<DT, DH, 1, 1>(fn, a, f.ranges, scratch, st);
  return prompt_launch<DT, DH, 1, 2>(fn, a, f.ranges, scratch, st);
}
int launch_kv8_prompt(const char* fn, const Kv8AttnArgs& a, float* scratch, size_t scratch_bytes, hipStream_t st) {
  const PromptForm f = prompt_form(a.B, a.M, a.H, a.c.Hk, a.c.S);
  const size_t need = kv8_prompt_scratch_bytes(a.B, a.M, a.H, a.c.Hk, a.c.Dh, a.c.S);
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
