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
  // decode: the rows [B, Hk, Dh] that the call appends at positions[b], or null
  const uint16_t* k_new = nullptr; int64_t sk_b = 0, sk_h = 0;
  const uint16_t* v_new = nullptr; int64_t sv_b = 0, sv_h = 0;
};
// four held codes at another scale, `move` times their own
__device__ __forceinline__ uint32_t moved(uint32_t w, float move) {
  const f32x2_t lo = codes_lo(w), hi = codes_hi(w);
  return codes_of(lo[0] * move, lo[1] * move, hi[0] * move, hi[1] * move);
}

// One row of a kv head (k, v [Dh]) into its place at position pos, 0 <= pos < S, by one wave: lanes 0 to 15 hold the key, 16 to 31 the value, each lane DH / 32
// dimensions of either half of the head.  The rows of the block before it are moved where the row needs a larger scale.
template <int DT, int DH>
__device__ __forceinline__ void append_row(const fsvd_kv8_cache& c, const uint16_t* k, const uint16_t* v, const uint16_t* cos, const uint16_t* sin, int rope_len,
                                           int b, int hk, int pos, int lane) {
  typedef E16<DT> E;
  constexpr int HALF = DH / 2, N = HALF / 16;
  const int part = (lane >> 4) & 1, d = (lane & 15) * N, at = pos % c.block;
  const int64_t base = b * c.sc_b + hk * c.sc_h;
  uint8_t* codes = static_cast<uint8_t*>(part ? c.v : c.k) + base;
  float* scale = (part ? c.v_scale : c.k_scale) + b * c.ss_b + (int64_t)(pos / c.block) * c.ss_n + hk * c.ss_h;
  const uint16_t* x = (part ? v : k) + d;
  const float old = at > 0 ? *scale : 0.f;
  uint32_t w0[N], w1[N], wc[N], ws[N];                   // everything is asked for at once
  const bool turn = part == 0 && cos != nullptr;
  const int64_t tp = (int64_t)min(pos, rope_len - 1) * HALF + d;
#pragma unroll
  for (int e = 0; e < N; ++e) { w0[e] = x[e]; w1[e] = x[e + HALF]; }
  if (turn) {
#pragma unroll
    for (int e = 0; e < N; ++e) { wc[e] = cos[tp + e]; ws[e] = sin[tp + e]; }
  }
  float x0[N], x1[N], amax = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    x0[e] = E::val(w0[e]); x1[e] = E::val(w1[e]);
    if (turn) {
      const float c1 = E::val(wc[e]), s1 = E::val(ws[e]), y0 = x0[e] * c1 - x1[e] * s1, y1 = x0[e] * s1 + x1[e] * c1;
      x0[e] = y0; x1[e] = y1;
    }
    amax = fmaxf(amax, fmaxf(finite_mag(x0[e]), finite_mag(x1[e])));
  }
  amax = row16_max(amax);
  const float now = fmaxf(old, power_of_two(scale_exponent(amax))), inv = 1.f / now;
  if (lane < 32) {
    uint8_t* y = codes + (int64_t)pos * c.sc_s + d;
#pragma unroll
    for (int e = 0; e < N; ++e) { x0[e] = in_code_range(x0[e] * inv); x1[e] = in_code_range(x1[e] * inv); }
    if constexpr (N == 4) {
      *reinterpret_cast<uint32_t*>(y) = codes_of(x0[0], x0[1], x0[2], x0[3]);
      *reinterpret_cast<uint32_t*>(y + HALF) = codes_of(x1[0], x1[1], x1[2], x1[3]);
    } else {
      *reinterpret_cast<uint16_t*>(y) = (uint16_t)codes_of(x0[0], x0[1], 0.f, 0.f);
      *reinterpret_cast<uint16_t*>(y + HALF) = (uint16_t)codes_of(x1[0], x1[1], 0.f, 0.f);
    }
    if ((lane & 15) == 0) *scale = now;
  }
  // rare: lanes 0 to 31 go over the rows before it, each word by word of its part
  if (__any(at > 0 && now > old) && lane < 32 && now > old) {
    const float move = old * inv;
    for (int i = lane & 15; i < at * (DH / 4); i += 16) {
      uint32_t* w = reinterpret_cast<uint32_t*>(codes + (int64_t)(pos - at + i / (DH / 4)) * c.sc_s) + i % (DH / 4);
      *w = moved(*w, move);
    }
  }
}

int check_kv8_cache(const char* fn, const fsvd_kv8_cache* c);
int launch_kv8_append(const char* fn, const Kv8AppendArgs& a, hipStream_t st);
// ranges of keys that a sequence may be cut into, and the scratch for their partial results
int kv8_ranges(int B, int H, int Hk, int S, int nsplit);
size_t kv8_decode_scratch_bytes(int B, int H, int Dh, int ranges);
size_t kv8_prompt_scratch_bytes(int B, int M, int H, int Hk, int Dh, int S);
int launch_kv8_decode(const char* fn, const Kv8AttnArgs& a, int ranges, float* scratch, hipStream_t st);
int launch_kv8_prompt(const char* fn, const Kv8AttnArgs& a, float* scratch, size_t scratch_bytes, hipStream_t st);

}  // namespace fsvd
