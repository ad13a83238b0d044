// The KV cache in 8 bits: rows written to it, and its entry points.
#include "kv8.hpp"

namespace fsvd {

// One workgroup for a block of one kv head of one sequence, keys and values one after the other.  The scale of a block comes from the new rows, and
// where rows stand before the first of them, from the scale that those have: they are moved to the larger one.
template <int DT>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a) {
  typedef E16<DT> E;
  const int b = blockIdx.z, hk = blockIdx.y, tid = threadIdx.x;
  const int p = a.positions[b], rows = a.rows ? min(a.rows[b], a.T) : a.T;
  const int64_t end = (int64_t)p + rows;
  const int first = max(p, 0), last = (int)(end < a.c.S ? end : a.c.S);          // the rows that are written
  const int64_t blk = (int64_t)(first / a.c.block) + blockIdx.x, r0 = blk * a.c.block;
  if (first >= last || r0 >= last) return;
  const int n0 = (int)(r0 > first ? r0 : first), n1 = (int)(r0 + a.c.block < last ? r0 + a.c.block : last);
  const int half = a.c.Dh >> 1;
  __shared__ float red[4];
  for (int part = 0; part < 2; ++part) {
    const uint16_t* src = part ? a.v + (int64_t)b * a.sv_b + (int64_t)hk * a.sv_h : a.k + (int64_t)b * a.sk_b + (int64_t)hk * a.sk_h;
    const int64_t st = part ? a.sv_t : a.sk_t;
    uint8_t* dst = static_cast<uint8_t*>(part ? a.c.v : a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
    float* scale = (part ? a.c.v_scale : a.c.k_scale) + b * a.c.ss_b + blk * a.c.ss_n + hk * a.c.ss_h;
    const auto pair = [&](int row, int d, float& x0, float& x1) {
      const uint16_t* s = src + (int64_t)(row - p) * st;
      x0 = E::val(s[d]); x1 = E::val(s[d + half]);
      if (part == 0 && a.cos) {
        const int64_t tp = min(row, a.rope_len - 1);
        const float c = E::val(a.cos[tp * half + d]), n = E::val(a.sin[tp * half + d]);
        const float y0 = x0 * c - x1 * n, y1 = x0 * n + x1 * c;
        x0 = y0; x1 = y1;
      }
    };
    float amax = 0.f;
    for (int i = tid; i < (n1 - n0) * half; i += 256) {
      float x0, x1;
      pair(n0 + i / half, i % half, x0, x1);
      amax = fmaxf(amax, fmaxf(finite_mag(x0), finite_mag(x1)));
    }
    amax = wave_max(amax);
    if ((tid & 63) == 0) red[tid >> 6] = amax;
    const float old = n0 > r0 ? *scale : 0.f;
    __syncthreads();
    amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float fresh = power_of_two(scale_exponent(amax)), now = fmaxf(old, fresh), inv = 1.f / now;
    if (n0 > r0 && now > old) {
      const float move = old * inv;
      for (int i = tid; i < (int)(n0 - r0) * (a.c.Dh / 4); i += 256) {
        uint32_t* w = reinterpret_cast<uint32_t*>(dst + (r0 + i / (a.c.Dh / 4)) * a.c.sc_s) + i % (a.c.Dh / 4);
        const auto lo = codes_lo(*w), hi = codes_hi(*w);
        *w = codes_of(lo[0] * move, lo[1] * move, hi[0] * move, hi[1] * move);
      }
    }
    for (int i = tid; i < (n1 - n0) * half; i += 256) {
      float x0, x1;
      const int row = n0 + i / half, d = i % half;
      pair(row, d, x0, x1);
      const uint32_t w = codes_of(in_code_range(x0 * inv), in_code_range(x1 * inv), 0.f, 0.f);
      dst[row * a.c.sc_s + d] = (uint8_t)w;
      dst[row * a.c.sc_s + d + half] = (uint8_t)(w >> 8);
    }
    __syncthreads();
    if (tid == 0) *scale = now;
  }
}

int launch_kv8_append(const char* fn, const Kv8AppendArgs& a, hipStream_t st) {
  if (a.T == 0) return kOk;
  const dim3 grid((a.T + a.c.block - 2) / a.c.block + 1, a.c.Hk, a.B);
  if (a.dt == 1) hipLaunchKernelGGL(kv8_append_kernel<1>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(kv8_append_kernel<0>, grid, dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) { set_last_error("%s: launch failed: %s", fn, hipGetErrorString(e)); return kErrLaunch; }
  return kOk;
}

int check_kv8_cache(const char* fn, const fsvd_kv8_cache* c) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) {
    set_last_error("%s: a buffer of the cache is NULL", fn);
    return kErrNullPtr;
  }
  if (c->S <= 0 || c->Hk <= 0 || (c->Dh != 64 && c->Dh != 128)) { set_last_error("%s: bad cache: S=%d Hk=%d Dh=%d (64 and 128 are served)", fn, c->S, c->Hk, c->Dh); return kErrBadShape; }
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) { set_last_error("%s: block of %d tokens (16, 32, 64 and 128 are served)", fn, c->block); return kErrBadShape; }
  if (c->sc_b < 0 || c->sc_s < c->Dh || c->sc_h < 0 || c->ss_b < 0 || c->ss_n < 0 || c->ss_h < 0) { set_last_error("%s: bad cache strides", fn); return kErrBadShape; }
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) || ((c->sc_b | c->sc_s | c->sc_h) & 15)) {
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
static const uint16_t* in16(const void* p) { return static_cast<const uint16_t*>(p); }

extern "C" {

int fsvd_kv8_append(const fsvd_kv8_cache* cache, const void* k, int64_t sk_b, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_b, int64_t sv_t,
                    int64_t sv_h, const int32_t* positions, const int32_t* rows, const void* cos, const void* sin, int rope_len, int B, int T, int dtype,
                    void* stream) {
  const char* fn = "fsvd_kv8_append";
  if (const int rc = check_kv8_cache(fn, cache)) return rc;
  if (const int rc = check_call(fn, B, dtype, cos, sin, rope_len)) return rc;
  if (k == nullptr || v == nullptr || positions == nullptr) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (T < 0) { set_last_error("%s: %d rows", fn, T); return kErrBadShape; }
  const Kv8AppendArgs a{*cache, in16(k), sk_b, sk_t, sk_h, in16(v), sv_b, sv_t, sv_h, positions, rows, in16(cos), in16(sin), rope_len, B, T, dtype};
  return launch_kv8_append(fn, a, static_cast<hipStream_t>(stream));
}

size_t fsvd_attn_decode_kv8_scratch_bytes(int B, int H, int Hk, int Dh, int S, int nsplit) {
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk || S <= 0) return 0;
  return kv8_decode_scratch_bytes(B, H, Dh, kv8_ranges(B, H, Hk, S, nsplit));
}

int fsvd_attn_decode_kv8(const fsvd_kv8_cache* cache, const void* q, int64_t sq_b, int64_t sq_h, const void* k_new, int64_t sk_b, int64_t sk_h,
                         const void* v_new, int64_t sv_b, int64_t sv_h, const int32_t* cache_seqlens, int seqlen_add, const void* cos, const void* sin,
                         int rope_len, void* out, int64_t so_b, int64_t so_h, void* scratch, size_t scratch_bytes, int B, int H, int nsplit, float scale,
                         int dtype, void* stream) {
  const char* fn = "fsvd_attn_decode_kv8";
  if (const int rc = check_kv8_cache(fn, cache)) return rc;
  if (const int rc = check_call(fn, B, dtype, cos, sin, rope_len)) return rc;
  if (q == nullptr || out == nullptr || cache_seqlens == nullptr || (k_new == nullptr) != (v_new == nullptr)) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (H <= 0 || H % cache->Hk) { set_last_error("%s: %d query heads over %d", fn, H, cache->Hk); return kErrBadShape; }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int ranges = kv8_ranges(B, H, cache->Hk, cache->S, nsplit);
  const size_t need = kv8_decode_scratch_bytes(B, H, cache->Dh, ranges);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15))) {
    set_last_error("%s: %zu bytes of scratch for %d key ranges, %zu needed", fn, scratch ? scratch_bytes : (size_t)0, ranges, need);
    return kErrWorkspace;
  }
  if (k_new) {
    const Kv8AppendArgs n{*cache, in16(k_new), sk_b, 0, sk_h, in16(v_new), sv_b, 0, sv_h, cache_seqlens, nullptr, in16(cos), in16(sin), rope_len, B, 1, dtype};
    if (const int rc = launch_kv8_append(fn, n, st)) return rc;
    seqlen_add = 1;
  }
  const Kv8AttnArgs a{*cache, in16(q), sq_b, 0, sq_h, cache_seqlens, nullptr, in16(cos), in16(sin), rope_len, static_cast<uint16_t*>(out), so_b, 0, so_h,
                      B, 1, H, seqlen_add, scale > 0.f ? scale : 1.f / sqrtf((float)cache->Dh), dtype};
  return launch_kv8_decode(fn, a, ranges, static_cast<float*>(scratch), st);
}

size_t fsvd_attn_prefill_kv8_scratch_bytes(int B, int M, int H, int Hk, int Dh, int S) {
  if (B <= 0 || M <= 0 || H <= 0 || Hk <= 0 || H % Hk || S <= 0) return 0;
  return kv8_prompt_scratch_bytes(B, M, H, Hk, Dh, S);
}

int fsvd_attn_prefill_kv8(const fsvd_kv8_cache* cache, const void* q, int64_t sq_b, int64_t sq_m, int64_t sq_h, const int32_t* q_pos0, const int32_t* rows,
                          const void* cos, const void* sin, int rope_len, void* out, int64_t so_b, int64_t so_m, int64_t so_h, void* scratch,
                          size_t scratch_bytes, int B, int M, int H, float scale, int dtype, void* stream) {
  const char* fn = "fsvd_attn_prefill_kv8";
  if (const int rc = check_kv8_cache(fn, cache)) return rc;
  if (const int rc = check_call(fn, B, dtype, cos, sin, rope_len)) return rc;
  if (q == nullptr || out == nullptr || q_pos0 == nullptr) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (M < 0 || H <= 0 || H % cache->Hk) { set_last_error("%s: %d rows of %d query heads over %d", fn, M, H, cache->Hk); return kErrBadShape; }
  const Kv8AttnArgs a{*cache, in16(q), sq_b, sq_m, sq_h, q_pos0, rows, in16(cos), in16(sin), rope_len, static_cast<uint16_t*>(out), so_b, so_m, so_h,
                      B, M, H, 1, scale > 0.f ? scale : 1.f / sqrtf((float)cache->Dh), dtype};
  return M == 0 ? kOk : launch_kv8_prompt(fn, a, static_cast<float*>(scratch), scratch_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
