// The KV cache in 4 bits: e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign) [B, S, Hk, Dh / 2] of keys (rotated) and values, two a byte with the even channel in
// the low bits, and one byte for each token, kv head and 32 channels [B, Hk, Dh / 32, S], value = code * 2^(byte - 127): the hardware's own form of 4 bits, so a
// pair of codes becomes a pair of bf16 elements, scale included, in one instruction and exactly.
#pragma once
#include "../../include/flashsvd_hip.h"
#include "common.hpp"

namespace fsvd {

constexpr int kGroup4 = 32, kNanByte = 255;
// Exponents that a scale may have: 6 * 2^125 is the largest that bf16 holds, 2^-126 (a code of 1/2) its smallest normal number.
constexpr int kLeastExp4 = -125, kMostExp4 = 125;

// p + q rounded to fp32 such that comparing with or rounding to fewer bits gives what the exact sum gives: towards zero, the last bit set where that is not exact.
// p and q are products of 16-bit elements, exact in fp32.
__device__ __forceinline__ float odd_sum(float p, float q) {
  const float s = p + q, t = s - p, r = (p - (s - t)) + (q - t);          // r: what the rounding left
  const uint32_t u = __float_as_uint(s), inexact = __builtin_islessgreater(r, 0.f) ? ~0u : 0u;      // neither of an infinity nor of a NaN
  const uint32_t away = (uint32_t)((int)(__float_as_uint(r) ^ u) >> 31) & inexact;                 // -1 where s lies beyond the sum
  return __uint_as_float((u + away) | (inexact & 1u));
}
// Byte of the scale of a group whose largest magnitude is amax = m * 2^E, 1 <= m < 2: the smallest 2^e whose 7-fold covers it, 7 = 1.75 * 2^2.
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  return min(max((int)(u >> 23) - 127 - 2 + ((u & 0x7fffffu) > 0x600000u), kLeastExp4), kMostExp4) + 127;
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }       // of a byte that is no NaN
// The nearest codes of x0 and x1 (ties to even, the largest beyond it; infinities too) into byte AT of w.
template <int AT>
__device__ __forceinline__ uint32_t codes4_of(uint32_t w, float x0, float x1, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x0, x1, scale, AT);
}
// the pair of codes in byte AT of w as a pair of bf16 or fp32 elements
template <int AT>
__device__ __forceinline__ uint32_t pair4(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, AT));
}
template <int AT>
__device__ __forceinline__ f32x2_t pair4_f32(uint32_t w, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, AT); }

// the same with the position known after unrolling only
__device__ __forceinline__ uint32_t pair4_at(int at, uint32_t w, float scale) { return at == 0 ? pair4<0>(w, scale) : at == 1 ? pair4<1>(w, scale) : at == 2 ? pair4<2>(w, scale) : pair4<3>(w, scale); }
// two elements of float16, rounded where it does not hold them
__device__ __forceinline__ uint32_t pair4_half_at(int at, uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, at == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)
                                      : at == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)
                                      : at == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)
                                                : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
}
// Byte i of four scales as a scale: the conversions read the exponent alone, so what stands around it may stay.  Byte 255 makes NaN of every code.
__device__ __forceinline__ float scale_at(uint32_t four, int i) { return __uint_as_float(i == 0 ? four << 23 : i == 1 ? four << 15 : i == 2 ? four << 7 : four >> 1); }

// A row of a kv head into the cache: the lane has dimensions 8 part .. 8 part + 7 in x[0] and those half a head further in x[1], Dh / 16 lanes a row, four of
// them a group of 32 channels in either half (of 64 dimensions the halves are the groups).  codes: the row's; scales: its byte of group 0.  All lanes of the wave
// call it, `in` says which write.
template <int DH>
__device__ __forceinline__ void put_row(const float (&x)[2][8], uint8_t* codes, uint8_t* scales, int64_t ss_g, int part, bool in) {
  uint32_t word[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float amax = 0.f, bad = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      amax = fmaxf(amax, fmaxf(fabsf(x[h][e]), fabsf(x[h][e + 1])));
      bad = __builtin_isunordered(x[h][e], x[h][e + 1]) ? 1.f : bad;
    }
    if (__builtin_expect(__any(amax == INFINITY), 0)) {    // neither a NaN, which no maximum takes, nor an infinity decides a scale
      amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[h][e]) < INFINITY ? fabsf(x[h][e]) : 0.f);
    }
    amax = fmaxf(amax, dpp_f32<0xB1>(amax));               // over the four lanes
    amax = fmaxf(amax, dpp_f32<0x4E>(amax));
    bad = fmaxf(bad, dpp_f32<0xB1>(bad));
    bad = fmaxf(bad, dpp_f32<0x4E>(bad));
    const int byte = scale_byte(amax);
    const float scale = scale_of(byte);
    uint32_t w = codes4_of<0>(0u, x[h][0], x[h][1], scale);
    w = codes4_of<1>(w, x[h][2], x[h][3], scale);
    w = codes4_of<2>(w, x[h][4], x[h][5], scale);
    w = codes4_of<3>(w, x[h][6], x[h][7], scale);
    word[h] = w;
    if (in && part % 4 == 0) scales[(h * (DH / 64) + part / 4) * ss_g] = (uint8_t)(bad > 0.f ? kNanByte : byte);
  }
  // lanes 2 i and 2 i + 1 change words, so that the first has eight bytes of the lower half and the second of the upper
  const bool odd = part & 1;
  const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(odd ? word[0] : word[1]), 0xB1, 0xF, 0xF, true);
  if (in) *reinterpret_cast<u32x2_t*>(codes + (odd ? DH / 4 : 0) + part / 2 * 8) = odd ? u32x2_t{other, word[1]} : u32x2_t{word[0], other};
}
// Eight elements and those half a head further as numbers, rotated where `turn` says, for comparisons and roundings as the exact values.  The borders of exponents
// and codes have two bits behind the first: a rotated value that rounding to fp32 has not put on such a number lies on the side of them where the exact one does, and the
// others (few but for the first positions, whose cosines are 1) are made again by odd_sum.  All of them by it, 8 x 2048 rows of 32 heads take 80 us instead of 75, 1 x 2048 16.9 instead of 14.6.
template <class E>
__device__ __forceinline__ void row_numbers(u32x4_t lo, u32x4_t hi, bool turn, u32x4_t cw, u32x4_t sw, float (&x)[2][8]) {
  float c[8], s[8];
  uint32_t least = 1;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t wl = lo[e >> 1], wh = hi[e >> 1], wc = cw[e >> 1], ws = sw[e >> 1];
    const float u = e & 1 ? E::hi(wl) : E::lo(wl), v = e & 1 ? E::hi(wh) : E::lo(wh);
    c[e] = e & 1 ? E::hi(wc) : E::lo(wc); s[e] = e & 1 ? E::hi(ws) : E::lo(ws);
    const float y0 = fmaf(u, c[e], -(v * s[e])), y1 = fmaf(u, s[e], v * c[e]);
    least = min(least, min(__float_as_uint(y0) & 0x1fffffu, __float_as_uint(y1) & 0x1fffffu));
    x[0][e] = turn ? y0 : u; x[1][e] = turn ? y1 : v;
  }
  if (__builtin_expect(__any(turn && least == 0), 0) && turn) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t wl = lo[e >> 1], wh = hi[e >> 1];
      const float u = e & 1 ? E::hi(wl) : E::lo(wl), v = e & 1 ? E::hi(wh) : E::lo(wh);
      x[0][e] = odd_sum(u * c[e], -(v * s[e])); x[1][e] = odd_sum(u * s[e], v * c[e]);
      // beyond fp32, but no infinity (which has no bit behind the first either, so it comes here): decides the scale as the largest number
      const bool numbers = fabsf(u) < INFINITY && fabsf(v) < INFINITY && fabsf(c[e]) < INFINITY && fabsf(s[e]) < INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (numbers && fabsf(x[h][e]) == INFINITY) x[h][e] = copysignf(__FLT_MAX__, x[h][e]);
    }
  }
}
__device__ __forceinline__ u32x4_t eight4(const uint16_t* p) { return __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(p)); }

// Loads at a base of the wave's, an offset of the wave's and one of the lane's (each below 2^31): nothing of the address but the lane's offset is in vector registers.
#if defined(__HIP_DEVICE_COMPILE__)
typedef __amdgpu_buffer_rsrc_t Rows4;
constexpr int kOnce = 2;                                  // read once: not kept in the caches
__device__ __forceinline__ Rows4 rows4(const uint8_t* base) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, 0xffffffffu, 0x00020000u); }
template <int BYTES, int AUX>
__device__ __forceinline__ void load4(Rows4 r, uint32_t lane, uint32_t off, uint32_t* w) {
  if constexpr (BYTES == 16) {
    const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane, (int)off, AUX);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const u32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(r, (int)lane, (int)off, AUX);
    w[0] = v.x; w[1] = v.y;
  } else if constexpr (BYTES == 4) {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)lane, (int)off, AUX);
  } else if constexpr (BYTES == 2) {
    w[0] = __builtin_amdgcn_raw_buffer_load_b16(r, (int)lane, (int)off, AUX);
  } else {
    w[0] = __builtin_amdgcn_raw_buffer_load_b8(r, (int)lane, (int)off, AUX);
  }
}
#else
struct Rows4 {};
constexpr int kOnce = 2;
__device__ Rows4 rows4(const uint8_t* base);
template <int BYTES, int AUX> __device__ void load4(Rows4 r, uint32_t lane, uint32_t off, uint32_t* w);
#endif

struct Kv4AppendArgs {
  fsvd_kv4_cache c;                                    // limit: 1 to S
  const uint16_t* k; int64_t sk_b, sk_t, sk_h;         // [B, T, Hk, Dh]
  const uint16_t* v; int64_t sv_b, sv_t, sv_h;
  const int32_t* positions;                            // [B]
  const int32_t* rows;                                 // [B] or null: T rows each
  const uint16_t* cos; const uint16_t* sin; int rope_len;
  int B, T, dt;
};
struct Kv4AttnArgs {
  fsvd_kv4_cache c;                                    // limit: 1 to S
  const uint16_t* q; int64_t sq_b, sq_m, sq_h;         // [B, M, H, Dh]
  const int32_t* positions;                            // [B]: position of a sequence's first query row
  const int32_t* rows;                                 // [B] or null: M query rows each
  const uint16_t* cos; const uint16_t* sin; int rope_len;
  uint16_t* out; int64_t so_b, so_m, so_h;
  int B, M, H;
  int key_add;                                         // query row m sees the keys below positions[b] + m + key_add
  float scale;
  int dt;
  // decode: the rows [B, Hk, Dh] that the call appends at positions[b], or null
  const uint16_t* k_new = nullptr; int64_t sk_b = 0, sk_h = 0;
  const uint16_t* v_new = nullptr; int64_t sv_b = 0, sv_h = 0;
};

// One row of a kv head (k, v [Dh]) into its place at position pos, 0 <= pos < limit, by one wave: the first Dh / 16 lanes hold the key, as many behind them the value.
template <int DT, int DH>
__device__ __forceinline__ void append_row4(const fsvd_kv4_cache& c, const uint16_t* k, const uint16_t* v, const uint16_t* cos, const uint16_t* sin, int rope_len,
                                            int b, int hk, int pos, int lane) {
  constexpr int LPR = DH / 16, HALF = DH / 2;
  const int value = lane / LPR & 1, part = lane % LPR;
  const uint16_t* x = (value ? v : k) + 8 * part;
  const u32x4_t lo = eight4(x), hi = eight4(x + HALF);
  u32x4_t cw = {0u, 0u, 0u, 0u}, sw = cw;
  if (cos != nullptr) {
    const int64_t tp = (int64_t)min(pos, rope_len - 1) * HALF + 8 * part;
    cw = eight4(cos + tp); sw = eight4(sin + tp);
  }
  float y[2][8];
  row_numbers<E16<DT>>(lo, hi, cos != nullptr && !value, cw, sw, y);
  put_row<DH>(y, static_cast<uint8_t*>(value ? c.v : c.k) + b * c.sc_b + hk * c.sc_h + pos * c.sc_s,
              static_cast<uint8_t*>(value ? c.v_scale : c.k_scale) + b * c.ss_b + hk * c.ss_h + pos, c.ss_g, part, lane < 2 * LPR);
}

int launch_kv4_append(const char* fn, const Kv4AppendArgs& a, hipStream_t st);
// ranges of keys that a sequence may be cut into, and the scratch for their partial results
int kv4_ranges(int B, int H, int Hk, int S, int nsplit);
size_t kv4_decode_scratch_bytes(int B, int H, int Dh, int ranges);
size_t kv4_prompt_scratch_bytes(int B, int M, int H, int Hk, int Dh, int S);
int launch_kv4_decode(const char* fn, const Kv4AttnArgs& a, int ranges, float* scratch, hipStream_t st);
int launch_kv4_prompt(const char* fn, const Kv4AttnArgs& a, float* scratch, size_t scratch_bytes, hipStream_t st);

}  // namespace fsvd
