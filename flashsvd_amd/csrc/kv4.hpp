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

// p + q rounded to fp32 such that comparing with or rounding to fewer bits gives what the exact sum gives: towards the odd neighbour where it is not exact.
// p and q are products of 16-bit elements, exact in fp32.
__device__ __forceinline__ float odd_sum(float p, float q) {
  const float s = p + q, t = s - p, r = (p - (s - t)) + (q - t);          // r: what the rounding left
  const uint32_t u = __float_as_uint(s);
  if ((r > 0.f || r < 0.f) && !(u & 1)) return __uint_as_float((r > 0.f) == (s > 0.f) ? u + 1 : u - 1);
  return s;
}
// magnitude that counts towards a scale: neither a NaN nor an infinity decides it
__device__ __forceinline__ float finite_mag4(float x) {
  const float m = fabsf(x);
  return m < INFINITY ? m : 0.f;
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

struct Kv4AppendArgs {
  fsvd_kv4_cache c;
  const uint16_t* k; int64_t sk_b, sk_t, sk_h;         // [B, T, Hk, Dh]
  const uint16_t* v; int64_t sv_b, sv_t, sv_h;
  const int32_t* positions;                            // [B]
  const int32_t* rows;                                 // [B] or null: T rows each
  const uint16_t* cos; const uint16_t* sin; int rope_len;
  int B, T, dt;
};
struct Kv4AttnArgs {
  fsvd_kv4_cache c;
  const uint16_t* q; int64_t sq_b, sq_m, sq_h;         // [B, M, H, Dh]
  const int32_t* positions;                            // [B]: position of a sequence's first query row
  const int32_t* rows;                                 // [B] or null: M query rows each
  const uint16_t* cos; const uint16_t* sin; int rope_len;
  uint16_t* out; int64_t so_b, so_m, so_h;
  int B, M, H;
  int key_add;                                         // query row m sees the keys below positions[b] + m + key_add
  float scale;
  int dt;
};

int launch_kv4_append(const char* fn, const Kv4AppendArgs& a, hipStream_t st);
int launch_kv4_attend(const char* fn, const Kv4AttnArgs& a, hipStream_t st);

}  // namespace fsvd
