// The KV cache in 4 bits: rows written to it, what it holds, and its entry points.
#include "kv4.hpp"

namespace fsvd {

// A workgroup has 256 / (Dh / 16) rows of the keys or the values of HEADS kv heads, which share the rows of the rotation tables and have all their loads in
// flight.  Bound by its bytes: every row is read once and written once.  8 x 2048 rows of 32 heads of 128 (339 MB) take 73 to 75 us, 4.6 TB/s, where a copy reaches
// 5.4; rows that come rotated 59 to 60.  Times are of a call in a captured graph of six over three sets of inputs.
template <int DT, int DH, int HEADS>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendArgs a) {
  constexpr int HALF = DH / 2, LPR = DH / 16, PER = 256 / LPR;
  const int value = blockIdx.x & 1, h0 = (blockIdx.x >> 1) * HEADS, b = blockIdx.z, part = threadIdx.x % LPR, t = (int)blockIdx.y * PER + threadIdx.x / LPR;
  const int rows = a.rows ? min(a.rows[b], a.T) : a.T;
  const int64_t pos = (int64_t)a.positions[b] + t, sh = value ? a.sv_h : a.sk_h;
  const bool in = t < rows && pos >= 0 && pos < a.c.limit, turn = !value && a.cos != nullptr;
  const uint16_t* x = (value ? a.v + (int64_t)b * a.sv_b + (in ? t : 0) * a.sv_t : a.k + (int64_t)b * a.sk_b + (in ? t : 0) * a.sk_t) + h0 * sh + 8 * part;
  u32x4_t lo[HEADS], hi[HEADS], cw = {0u, 0u, 0u, 0u}, sw = cw;
  // Many rows are read past the caches, which they would only empty (8 x 2048 rows of 32 heads that come rotated 60.3 us, 63.3 through them; to be rotated 75 either
  // way); of few it costs more than it gives (2 x 2048 rows 24.2 us, 26.6 so).
  const auto once = [](const uint16_t* p) {
    if constexpr (HEADS == 1) return eight4(p);
    else return __builtin_bit_cast(u32x4_t, __builtin_nontemporal_load(reinterpret_cast<const u32x4_any_t*>(p)));
  };
#pragma unroll
  for (int i = 0; i < HEADS; ++i) { lo[i] = once(x + i * sh); hi[i] = once(x + i * sh + HALF); }
  if (turn) {
    const int64_t tp = min(max(pos, (int64_t)0), (int64_t)a.rope_len - 1) * HALF + 8 * part;
    cw = eight4(a.cos + tp); sw = eight4(a.sin + tp);
  }
  uint8_t* codes = static_cast<uint8_t*>(value ? a.c.v : a.c.k) + b * a.c.sc_b + h0 * a.c.sc_h + pos * a.c.sc_s;
  uint8_t* scales = static_cast<uint8_t*>(value ? a.c.v_scale : a.c.k_scale) + b * a.c.ss_b + h0 * a.c.ss_h + pos;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    float y[2][8];
    row_numbers<E16<DT>>(lo[i], hi[i], turn, cw, sw, y);
    put_row<DH>(y, codes + i * a.c.sc_h, scales + i * a.c.ss_h, a.c.ss_g, part, in);
  }
}
// One row for each sequence: a wave for a kv head.  Nothing but latency.
template <int DT, int DH>
__global__ __launch_bounds__(kWave) void kv4_append_one_kernel(Kv4AppendArgs a) {
  const int b = blockIdx.x / a.c.Hk, hk = blockIdx.x % a.c.Hk, pos = a.positions[b];
  if (pos < 0 || pos >= a.c.limit || (a.rows && a.rows[b] <= 0)) return;
  append_row4<DT, DH>(a.c, a.k + (int64_t)b * a.sk_b + (int64_t)hk * a.sk_h, a.v + (int64_t)b * a.sv_b + (int64_t)hk * a.sv_h, a.cos, a.sin, a.rope_len, b, hk, pos,
                      threadIdx.x);
}
template <int DT, int DH>
static void append_form(const Kv4AppendArgs& a, hipStream_t st) {
  constexpr int rows = 256 / (DH / 16);
  // us with one head / with four, rows of 32 heads of 128: 1 x 128 4.4 / 7.5, 1 x 2048 14.5 / 16.4, 2 x 2048 23.9 / 24.8, 4 x 2048 47.6 / 41.5, 8 x 2048 87.3 / 75.2
  const int64_t tiles = (a.T + rows - 1) / rows;
  const bool four = a.c.Hk % 4 == 0 && 2 * a.c.Hk * tiles * a.B >= 16384;
  set_last_form(a.T == 1 ? "kv4 row" : four ? "kv4 rows of 4 heads" : "kv4 rows");
  if (a.T == 1) hipLaunchKernelGGL((kv4_append_one_kernel<DT, DH>), dim3((unsigned)(a.B * a.c.Hk)), dim3(kWave), 0, st, a);
  else if (four) hipLaunchKernelGGL((kv4_append_kernel<DT, DH, 4>), dim3(2 * a.c.Hk / 4, (unsigned)tiles, a.B), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((kv4_append_kernel<DT, DH, 1>), dim3(2 * a.c.Hk, (unsigned)tiles, a.B), dim3(256), 0, st, a);
}

int launch_kv4_append(const char* fn, const Kv4AppendArgs& a, hipStream_t st) {
  if (a.T == 0) return kOk;
  if ((int64_t)a.B * a.c.Hk > 0x7fffffff || a.T > (1 << 20)) { set_last_error("%s: %d rows of %d heads for %d sequences", fn, a.T, a.c.Hk, a.B); return kErrBadShape; }
  if (a.dt == 1) a.c.Dh == 128 ? append_form<1, 128>(a, st) : append_form<1, 64>(a, st);
  else a.c.Dh == 128 ? append_form<0, 128>(a, st) : append_form<0, 64>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

// What the first L rows hold, [B, L, Hk, Dh] each: a thread has eight channels of four rows, whose scales are four bytes next to each other.  What it makes goes past
// the caches: 8 x 2048 rows of 32 heads of 128 (339 MB) take 49 us, 6.9 TB/s (64 through them), 512 rows 4.0 (4.6).
struct Kv4ReadArgs {
  fsvd_kv4_cache c;
  uint16_t* k; uint16_t* v;
  int64_t so_b, so_t, so_h;
  int L;
};
template <int DT, int DH>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4ReadArgs a) {
  typedef E16<DT> E;
  constexpr int LPR = DH / 8;
  const int value = blockIdx.x & 1, hk = blockIdx.x >> 1, b = blockIdx.z, part = threadIdx.x % LPR;
  const int64_t pos = 4 * ((int64_t)blockIdx.y * (256 / LPR) + threadIdx.x / LPR);
  if (pos >= a.L) return;
  const uint8_t* codes = static_cast<const uint8_t*>(value ? a.c.v : a.c.k) + b * a.c.sc_b + hk * a.c.sc_h + pos * a.c.sc_s + 4 * part;
  const uint8_t* scales = static_cast<const uint8_t*>(value ? a.c.v_scale : a.c.k_scale) + b * a.c.ss_b + hk * a.c.ss_h + part / 4 * a.c.ss_g + pos;
  uint16_t* out = (value ? a.v : a.k) + b * a.so_b + pos * a.so_t + hk * a.so_h + 8 * part;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(codes + i * a.c.sc_s);       // rooms are multiples of four rows
  const uint32_t four = *reinterpret_cast<const uint32_t*>(scales);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float f = scale_at(four, i);
    u32x4_t x;
    if constexpr (DT == 0) {
      x = u32x4_t{pair4<0>(w[i], f), pair4<1>(w[i], f), pair4<2>(w[i], f), pair4<3>(w[i], f)};
    } else {
      const f32x2_t y[4] = {pair4_f32<0>(w[i], f), pair4_f32<1>(w[i], f), pair4_f32<2>(w[i], f), pair4_f32<3>(w[i], f)};
      x = u32x4_t{E::pack2(y[0][0], y[0][1]), E::pack2(y[1][0], y[1][1]), E::pack2(y[2][0], y[2][1]), E::pack2(y[3][0], y[3][1])};
    }
    if (pos + i < a.L) __builtin_nontemporal_store(__builtin_bit_cast(u32x4_any_t, x), reinterpret_cast<u32x4_any_t*>(out + i * a.so_t));
  }
}

static int check_kv4_cache(const char* fn, const fsvd_kv4_cache* c) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) {
    set_last_error("%s: a buffer of the cache is NULL", fn);
    return kErrNullPtr;
  }
  if (c->S <= 0 || c->S % 64 || c->Hk <= 0 || (c->Dh != 64 && c->Dh != 128)) {
    set_last_error("%s: bad cache: S=%d Hk=%d Dh=%d (a multiple of 64 rows; 64 and 128 dimensions are served)", fn, c->S, c->Hk, c->Dh);
    return kErrBadShape;
  }
  if (c->limit < 0 || c->limit > c->S) { set_last_error("%s: limit of %d rows of a cache of %d", fn, c->limit, c->S); return kErrBadShape; }
  if (c->sc_b < 0 || c->sc_s < c->Dh / 2 || c->sc_s > (1 << 24) || c->sc_h < 0 || c->ss_b < 0 || c->ss_h < 0 || c->ss_g < c->S || c->ss_g > (1 << 28)) { set_last_error("%s: bad cache strides", fn); return kErrBadShape; }
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 15) ||
      ((c->sc_b | c->sc_s | c->sc_h | c->ss_b | c->ss_h | c->ss_g) & 15)) {
    set_last_error("%s: cache pointers and strides must be 16-byte aligned", fn);
    return kErrBadAlign;
  }
  return kOk;
}

}  // namespace fsvd

using namespace fsvd;

static int check_call(const char* fn, int B, int dtype, const void* cos, const void* sin, int rope_len) {
  if (B <= 0 || B > 65535) { set_last_error("%s: batch of %d (1 to 65535 are served)", fn, B); return kErrBadShape; }
  if (dtype != 0 && dtype != 1) { set_last_error("%s: dtype code %d (bf16 = 0 and fp16 = 1 are served)", fn, dtype); return kErrBadDtype; }
  if ((cos == nullptr) != (sin == nullptr) || (cos != nullptr && rope_len <= 0)) { set_last_error("%s: cos and sin go together, with rope_len rows", fn); return kErrNullPtr; }
  return kOk;
}
// rows that a call writes must not lie in each other
static int check_written(const char* fn, const fsvd_kv4_cache* c, int B) {
  if ((B > 1 && (c->sc_b == 0 || c->ss_b == 0)) || (c->Hk > 1 && (c->sc_h == 0 || c->ss_h == 0))) {
    set_last_error("%s: a cache that is written to must not be expanded over its sequences or heads", fn);
    return kErrBadShape;
  }
  return kOk;
}
static int check_out(const char* fn, int B, int M, int H, int64_t so_b, int64_t so_m, int64_t so_h) {
  if ((B > 1 && so_b == 0) || (M > 1 && so_m == 0) || (H > 1 && so_h == 0)) { set_last_error("%s: out must not be expanded", fn); return kErrBadShape; }
  return kOk;
}
static fsvd_kv4_cache with_limit(const fsvd_kv4_cache* c) {
  fsvd_kv4_cache r = *c;
  if (r.limit == 0) r.limit = r.S;
  return r;
}
static const uint16_t* in16(const void* p) { return static_cast<const uint16_t*>(p); }

extern "C" {

int fsvd_kv4_append(const fsvd_kv4_cache* cache, const void* k, int64_t sk_b, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_b, int64_t sv_t,
                    int64_t sv_h, const int32_t* positions, const int32_t* rows, const void* cos, const void* sin, int rope_len, int B, int T, int dtype,
                    void* stream) {
  const char* fn = "fsvd_kv4_append";
  if (const int rc = check_kv4_cache(fn, cache)) return rc;
  if (const int rc = check_call(fn, B, dtype, cos, sin, rope_len)) return rc;
  if (positions == nullptr || (T != 0 && (k == nullptr || v == nullptr))) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (T < 0) { set_last_error("%s: %d rows", fn, T); return kErrBadShape; }
  if (const int rc = check_written(fn, cache, B)) return rc;
  const Kv4AppendArgs a{with_limit(cache), in16(k), sk_b, sk_t, sk_h, in16(v), sv_b, sv_t, sv_h, positions, rows, in16(cos), in16(sin), rope_len, B, T, dtype};
  return launch_kv4_append(fn, a, static_cast<hipStream_t>(stream));
}

int fsvd_kv4_dequantize(const fsvd_kv4_cache* cache, void* k, void* v, int64_t so_b, int64_t so_t, int64_t so_h, int B, int L, int dtype, void* stream) {
  const char* fn = "fsvd_kv4_dequantize";
  if (const int rc = check_kv4_cache(fn, cache)) return rc;
  if (const int rc = check_call(fn, B, dtype, nullptr, nullptr, 0)) return rc;
  if (L < 0 || L > cache->S) { set_last_error("%s: %d rows of a cache of %d", fn, L, cache->S); return kErrBadShape; }
  if (L == 0) return kOk;
  if (k == nullptr || v == nullptr) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (const int rc = check_out(fn, B, L, cache->Hk, so_b, so_t, so_h)) return rc;
  const Kv4ReadArgs a{*cache, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v), so_b, so_t, so_h, L};
  const int per = 4 * 256 / (cache->Dh / 8);
  const dim3 grid(2 * cache->Hk, (L + per - 1) / per, B);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == 1) {
    if (cache->Dh == 128) hipLaunchKernelGGL((kv4_read_kernel<1, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv4_read_kernel<1, 64>), grid, dim3(256), 0, st, a);
  } else {
    if (cache->Dh == 128) hipLaunchKernelGGL((kv4_read_kernel<0, 128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv4_read_kernel<0, 64>), grid, dim3(256), 0, st, a);
  }
  set_last_form("kv4 read");
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

size_t fsvd_attn_decode_kv4_scratch_bytes(int B, int H, int Hk, int Dh, int S, int nsplit) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk || S <= 0) return 0;
  return kv4_decode_scratch_bytes(B, H, Dh, kv4_ranges(B, H, Hk, S, nsplit));
}

int fsvd_attn_decode_kv4(const fsvd_kv4_cache* cache, const void* q, int64_t sq_b, int64_t sq_h, const void* k_new, int64_t sk_b, int64_t sk_h,
                         const void* v_new, int64_t sv_b, int64_t sv_h, const int32_t* cache_seqlens, int seqlen_add, const void* cos, const void* sin,
                         int rope_len, void* out, int64_t so_b, int64_t so_h, void* scratch, size_t scratch_bytes, int B, int H, int nsplit, float scale,
                         int dtype, void* stream) {
  const char* fn = "fsvd_attn_decode_kv4";
  if (const int rc = check_kv4_cache(fn, cache)) return rc;
  if (const int rc = check_call(fn, B, dtype, cos, sin, rope_len)) return rc;
  if (q == nullptr || out == nullptr || cache_seqlens == nullptr || (k_new == nullptr) != (v_new == nullptr)) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (H <= 0 || H % cache->Hk) { set_last_error("%s: %d query heads over %d", fn, H, cache->Hk); return kErrBadShape; }
  if (const int rc = k_new ? check_written(fn, cache, B) : kOk) return rc;
  if (const int rc = check_out(fn, B, 1, H, so_b, 0, so_h)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int ranges = kv4_ranges(B, H, cache->Hk, cache->S, nsplit);
  const size_t need = kv4_decode_scratch_bytes(B, H, cache->Dh, ranges);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15))) {
    set_last_error("%s: %zu bytes of scratch for %d key ranges, %zu needed", fn, scratch ? scratch_bytes : (size_t)0, ranges, need);
    return kErrWorkspace;
  }
  const Kv4AttnArgs a{with_limit(cache), in16(q), sq_b, 0, sq_h, cache_seqlens, nullptr, in16(cos), in16(sin), rope_len, static_cast<uint16_t*>(out), so_b, 0, so_h,
                      B, 1, H, k_new ? 1 : seqlen_add, scale > 0.f ? scale : 1.f / sqrtf((float)cache->Dh), dtype,
                      in16(k_new), sk_b, sk_h, in16(v_new), sv_b, sv_h};
  return launch_kv4_decode(fn, a, ranges, static_cast<float*>(scratch), st);
}

size_t fsvd_attn_prefill_kv4_scratch_bytes(int B, int M, int H, int Hk, int Dh, int S) {
  if (B <= 0 || M <= 0 || H <= 0 || Hk <= 0 || H % Hk || S <= 0) return 0;
  return kv4_prompt_scratch_bytes(B, M, H, Hk, Dh, S);
}

int fsvd_attn_prefill_kv4(const fsvd_kv4_cache* cache, const void* q, int64_t sq_b, int64_t sq_m, int64_t sq_h, const int32_t* q_pos0, const int32_t* rows,
                          const void* cos, const void* sin, int rope_len, void* out, int64_t so_b, int64_t so_m, int64_t so_h, void* scratch,
                          size_t scratch_bytes, int B, int M, int H, float scale, int dtype, void* stream) {
  const char* fn = "fsvd_attn_prefill_kv4";
  if (const int rc = check_kv4_cache(fn, cache)) return rc;
  if (const int rc = check_call(fn, B, dtype, cos, sin, rope_len)) return rc;
  if (q_pos0 == nullptr || (M != 0 && (q == nullptr || out == nullptr))) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (M < 0 || H <= 0 || H % cache->Hk) { set_last_error("%s: %d rows of %d query heads over %d", fn, M, H, cache->Hk); return kErrBadShape; }
  if (const int rc = check_out(fn, B, M, H, so_b, so_m, so_h)) return rc;
  const Kv4AttnArgs a{with_limit(cache), in16(q), sq_b, sq_m, sq_h, q_pos0, rows, in16(cos), in16(sin), rope_len, static_cast<uint16_t*>(out), so_b, so_m, so_h,
                      B, M, H, 1, scale > 0.f ? scale : 1.f / sqrtf((float)cache->Dh), dtype};
  return M == 0 ? kOk : launch_kv4_prompt(fn, a, static_cast<float*>(scratch), scratch_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
