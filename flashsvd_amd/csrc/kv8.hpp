// The KV cache in 8 bits: e4m3 codes [B, S, Hk, Dh] of keys (rotated) and values, one fp32 scale for each sequence, block of tokens and kv head,
// value = code * scale.  Scales are powers of two, 2^e with the smallest e for which 448 * 2^e covers the block (not below 2^-126): the product of
// a code and its scale is exact then, and so is the step of held codes to a larger scale, but for codes that become subnormal.
#pragma once
#include "../../include/flashsvd_hip.h"
#include "common.hpp"

namespace fsvd {

constexpr float kCodeMax = 448.f;

// four codes at once, and back
__device__ __forceinline__ f32x2_t codes_lo(uint32_t w) { return __builtin_amdgcn_cvt_pk_f32_fp8(w, false); }
__device__ __forceinline__ f32x2_t codes_hi(uint32_t w) { return __builtin_amdgcn_cvt_pk_f32_fp8(w, true); }
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {
  const uint32_t lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// what a code may be made of: a NaN stays one, an infinity becomes the largest code
__device__ __forceinline__ float in_code_range(float x) { return x != x ? x : fminf(fmaxf(x, -kCodeMax), kCodeMax); }
// magnitude that counts towards a scale: neither a NaN nor an infinity decides it
__device__ __forceinline__ float finite_mag(float x) {
  const float m = fabsf(x);
  return m < INFINITY ? m : 0.f;
}
// exponent e of the scale 2^e of a block whose largest magnitude is amax = m * 2^E, 1 <= m < 2: 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  return max((int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u), -126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }     // -126 <= e <= 127

// a pair of codes (low or high half of a word) as a pair of 16-bit elements, exact in both types
template <int DT> struct Code16;
template <> struct Code16<0> {
  template <bool HI> static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
  }
};
template <> struct Code16<1> {
  template <bool HI> static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
  }
};

struct Kv8AppendArgs {
  fsvd_kv8_cache c;
  const uint16_t* k; int64_t sk_b, sk_t, sk_h;         // [B, T, Hk, Dh]
  const uint16_t* v; int64_t sv_b, sv_t, sv_h;
  const int32_t* positions;                            // [B]
  const int32_t* rows;                                 // [B] or null: T rows each
  const uint16_t* cos; const uint16_t* sin; int rope_len;
  int B, T, dt;
};
struct Kv8AttnArgs {
  fsvd_kv8_cache c;
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
int check_kv8_cache(const char* fn, const fsvd_kv8_cache* c);
int launch_kv8_append(const char* fn, const Kv8AppendArgs& a, hipStream_t st);
// ranges of keys that a sequence may be cut into, and the scratch for their partial results
int kv8_ranges(int B, int H, int Hk, int S, int nsplit);
size_t kv8_decode_scratch_bytes(int B, int H, int Dh, int ranges);
size_t kv8_prompt_scratch_bytes(int B, int M, int H, int Hk, int Dh, int S);
int launch_kv8_decode(const char* fn, const Kv8AttnArgs& a, int ranges, float* scratch, hipStream_t st);
int launch_kv8_prompt(const char* fn, const Kv8AttnArgs& a, float* scratch, size_t scratch_bytes, hipStream_t st);

}  // namespace fsvd
