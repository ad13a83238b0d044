// The KV cache in 8 bits: rows written to it, and its entry points.
#include "kv8.hpp"

namespace fsvd {

// Rows of a call in registers: a lane holds dimensions d .. d + 7 and the eight half a head further of a row (the pairs of the rotation), LPR lanes a row; a
// workgroup has P times 256 / LPR rows of the keys or the values of one kv head, that is one block or, of small blocks, several.  The scale of a block is the
// largest magnitude of its new rows, and where rows stand before the first of them, that of the scale that those have: they are moved to the larger one.
// Bound by its bytes: every row is read once and written once.  8 x 2048 rows of 32 heads of 128 (403 MB) take 83 us, 4.8 TB/s; a copy reaches 5.2.
template <int DT, int DH, int P>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a) {
  typedef E16<DT> E;
  constexpr int HALF = DH / 2, LPR = HALF / 8;
  __shared__ float red[4];
  const int part = blockIdx.x & 1, hk = blockIdx.x >> 1, b = blockIdx.z, tid = threadIdx.x;
  const int p = a.positions[b], rows = a.rows ? min(a.rows[b], a.T) : a.T, block = a.c.block;
  const int64_t end = (int64_t)p + rows;
  const int first = max(p, 0), last = (int)(end < a.c.S ? end : a.c.S);          // the rows that are written
  const int64_t row0 = (int64_t)(first / block) * block + (int64_t)blockIdx.y * (P * 256 / LPR);
  if (first >= last || row0 >= last) return;
  const uint16_t* src = part ? a.v + (int64_t)b * a.sv_b + (int64_t)hk * a.sv_h : a.k + (int64_t)b * a.sk_b + (int64_t)hk * a.sk_h;
  const int64_t st = part ? a.sv_t : a.sk_t;
  uint8_t* dst = static_cast<uint8_t*>(part ? a.c.v : a.c.k) + b * a.c.sc_b + hk * a.c.sc_h;
  float* scales = (part ? a.c.v_scale : a.c.k_scale) + b * a.c.ss_b + hk * a.c.ss_h;
  const int d = tid % LPR * 8;
  const bool turn = part == 0 && a.cos != nullptr;
  u32x4_t lo[P], hi[P], cw[P], sw[P];
  int64_t row[P];
  bool in[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    row[i] = row0 + (i * 256 + tid) / LPR;
    in[i] = row[i] >= first && row[i] < last;
    const int64_t r = in[i] ? row[i] : first;
    const uint16_t* x = src + (r - p) * st + d;
    lo[i] = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(x));
    hi[i] = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(x + HALF));
    if (turn) {
      const int64_t tp = (r < a.rope_len ? r : a.rope_len - 1) * HALF + d;
      cw[i] = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(a.cos + tp));
      sw[i] = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_any_t*>(a.sin + tp));
    }
  }
  const int64_t blk = row[0] / block;                     // of this thread's rows: one block, whatever P (more than one pass means a larger block)
  const bool open = blk * block < first;                  // rows stand before the first new one
  const float old = open ? scales[blk * a.c.ss_n] : 0.f;
  float x0[P][8], x1[P][8], amax = 0.f;
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t wl = lo[i][e >> 1], wh = hi[i][e >> 1];
      float u = e & 1 ? E::hi(wl) : E::lo(wl), v = e & 1 ? E::hi(wh) : E::lo(wh);
      if (turn) {
        const uint32_t wc = cw[i][e >> 1], ws = sw[i][e >> 1];
        const float c = e & 1 ? E::hi(wc) : E::lo(wc), s = e & 1 ? E::hi(ws) : E::lo(ws), y0 = u * c - v * s, y1 = u * s + v * c;
        u = y0; v = y1;
      }
      x0[i][e] = u; x1[i][e] = v;
      amax = fmaxf(amax, in[i] ? fmaxf(finite_mag(u), finite_mag(v)) : 0.f);
    }
  amax = wave_max(amax);
  if ((tid & 63) == 0) red[tid >> 6] = amax;
  __syncthreads();
  const int waves = min(4, block * LPR / kWave), w0 = (tid >> 6) / waves * waves;        // that hold the block
  for (int i = 0; i < waves; ++i) amax = fmaxf(amax, red[w0 + i]);
  if (blk * block >= last || (blk + 1) * block <= first) return;
  const float now = fmaxf(old, power_of_two(scale_exponent(amax))), inv = 1.f / now;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    uint8_t* y = dst + row[i] * a.c.sc_s + d;
    if (in[i]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) { x0[i][e] = in_code_range(x0[i][e] * inv); x1[i][e] = in_code_range(x1[i][e] * inv); }
      *reinterpret_cast<u32x2_t*>(y) = u32x2_t{codes_of(x0[i][0], x0[i][1], x0[i][2], x0[i][3]), codes_of(x0[i][4], x0[i][5], x0[i][6], x0[i][7])};
      *reinterpret_cast<u32x2_t*>(y + HALF) = u32x2_t{codes_of(x1[i][0], x1[i][1], x1[i][2], x1[i][3]), codes_of(x1[i][4], x1[i][5], x1[i][6], x1[i][7])};
    } else if (row[i] < first && now > old) {
      u32x2_t held[2] = {*reinterpret_cast<const u32x2_t*>(y), *reinterpret_cast<const u32x2_t*>(y + HALF)};
      const float move = old * inv;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) held[h][q] = moved(held[h][q], move);
      *reinterpret_cast<u32x2_t*>(y) = held[0];
      *reinterpret_cast<u32x2_t*>(y + HALF) = held[1];
    }
  }
  if (row[0] == blk * block && d == 0) scales[blk * a.c.ss_n] = now;
}

// One row for each sequence: one wave for a kv head, its lanes 0 to 15 with the key's dimensions, 16 to 31 with the value's.  Nothing but latency: 2.9 us for 16
// rows of 8 heads of 128 (3.6 in the kernel above).
template <int DT, int DH>
__global__ __launch_bounds__(kWave) void kv8_append_one_kernel(Kv8AppendArgs a) {
  const int b = blockIdx.x / a.c.Hk, hk = blockIdx.x % a.c.Hk, pos = a.positions[b];
  if (pos < 0 || pos >= a.c.S || (a.rows && a.rows[b] <= 0)) return;
  append_row<DT, DH>(a.c, a.k + (int64_t)b * a.sk_b + (int64_t)hk * a.sk_h, a.v + (int64_t)b * a.sv_b + (int64_t)hk * a.sv_h, a.cos, a.sin, a.rope_len, b, hk, pos,
                     threadIdx.x);
}

template <int DT, int DH>
static void append_form(const Kv8AppendArgs& a, hipStream_t st) {
  if (a.T == 1) {
    set_last_form("kv8 row");
    hipLaunchKernelGGL((kv8_append_one_kernel<DT, DH>), dim3((unsigned)(a.B * a.c.Hk)), dim3(kWave), 0, st, a);
    return;
  }
  constexpr int LPR = DH / 16;
  const int passes = max(1, a.c.block * LPR / 256), rows = passes * 256 / LPR;       // rows of a workgroup: whole blocks
  set_last_form(passes == 1 ? "kv8 rows 1" : passes == 2 ? "kv8 rows 2" : "kv8 rows 4");
  const dim3 grid(2 * a.c.Hk, (unsigned)((a.T + a.c.block - 1 + (int64_t)rows - 1) / rows), a.B);
  if (passes == 1) hipLaunchKernelGGL((kv8_append_kernel<DT, DH, 1>), grid, dim3(256), 0, st, a);
  else if (passes == 2) hipLaunchKernelGGL((kv8_append_kernel<DT, DH, 2>), grid, dim3(256), 0, st, a);
  else if constexpr (DH == 128) hipLaunchKernelGGL((kv8_append_kernel<DT, DH, 4>), grid, dim3(256), 0, st, a);      // blocks of 128
}
int launch_kv8_append(const char* fn, const Kv8AppendArgs& a, hipStream_t st) {
  if (a.T == 0) return kOk;
  if ((int64_t)a.B * a.c.Hk > 0x7fffffff || a.T > (1 << 20)) { set_last_error("%s: %d rows of %d heads for %d sequences", fn, a.T, a.c.Hk, a.B); return kErrBadShape; }
  if (a.dt == 1) a.c.Dh == 128 ? append_form<1, 128>(a, st) : append_form<1, 64>(a, st);
  else a.c.Dh == 128 ? append_form<0, 128>(a, st) : append_form<0, 64>(a, st);
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
  if (c->sc_b < 0 || c->sc_s < c->Dh || c->sc_s > (1 << 26) || c->sc_h < 0 || c->ss_b < 0 || c->ss_n < 0 || c->ss_n > (1 << 26) || c->ss_h < 0) { set_last_error("%s: bad cache strides", fn); return kErrBadShape; }
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
// rows that a call writes must not lie in each other
static int check_written(const char* fn, const fsvd_kv8_cache* c, int B) {
  if ((B > 1 && (c->sc_b == 0 || c->ss_b == 0)) || (c->Hk > 1 && (c->sc_h == 0 || c->ss_h == 0)) || (c->S > c->block && c->ss_n == 0)) {
    set_last_error("%s: a cache that is written to must not be expanded over its sequences, blocks or heads", fn);
    return kErrBadShape;
  }
  return kOk;
}
static int check_out(const char* fn, int B, int M, int H, int64_t so_b, int64_t so_m, int64_t so_h) {
  if ((B > 1 && so_b == 0) || (M > 1 && so_m == 0) || (H > 1 && so_h == 0)) { set_last_error("%s: out must not be expanded", fn); return kErrBadShape; }
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
  if (positions == nullptr || (T != 0 && (k == nullptr || v == nullptr))) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (T < 0) { set_last_error("%s: %d rows", fn, T); return kErrBadShape; }
  if (const int rc = check_written(fn, cache, B)) return rc;
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
  if (const int rc = k_new ? check_written(fn, cache, B) : kOk) return rc;
  if (const int rc = check_out(fn, B, 1, H, so_b, 0, so_h)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int ranges = kv8_ranges(B, H, cache->Hk, cache->S, nsplit);
  const size_t need = kv8_decode_scratch_bytes(B, H, cache->Dh, ranges);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15))) {
    set_last_error("%s: %zu bytes of scratch for %d key ranges, %zu needed", fn, scratch ? scratch_bytes : (size_t)0, ranges, need);
    return kErrWorkspace;
  }
  const Kv8AttnArgs a{*cache, in16(q), sq_b, 0, sq_h, cache_seqlens, nullptr, in16(cos), in16(sin), rope_len, static_cast<uint16_t*>(out), so_b, 0, so_h,
                      B, 1, H, k_new ? 1 : seqlen_add, scale > 0.f ? scale : 1.f / sqrtf((float)cache->Dh), dtype,
                      in16(k_new), sk_b, sk_h, in16(v_new), sv_b, sv_h};
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
  if (q_pos0 == nullptr || (M != 0 && (q == nullptr || out == nullptr))) { set_last_error("%s: a buffer is NULL", fn); return kErrNullPtr; }
  if (M < 0 || H <= 0 || H % cache->Hk) { set_last_error("%s: %d rows of %d query heads over %d", fn, M, H, cache->Hk); return kErrBadShape; }
  if (const int rc = check_out(fn, B, M, H, so_b, so_m, so_h)) return rc;
  const Kv8AttnArgs a{*cache, in16(q), sq_b, sq_m, sq_h, q_pos0, rows, in16(cos), in16(sin), rope_len, static_cast<uint16_t*>(out), so_b, so_m, so_h,
                      B, M, H, 1, scale > 0.f ? scale : 1.f / sqrtf((float)cache->Dh), dtype};
  return M == 0 ? kOk : launch_kv8_prompt(fn, a, static_cast<float*>(scratch), scratch_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
