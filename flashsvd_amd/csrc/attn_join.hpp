// Attention over key ranges: what every range of a row leaves, and the launch that joins them.
#pragma once
#include "common.hpp"

namespace fsvd {

// Partial results of key ranges: values [rows][ranges][Dh], not divided by their sums, and behind them (maximum, sum) [rows][ranges].
struct RangeParts {
  float* base;
  int64_t rows;
  int ranges, dh;
  static size_t bytes(int64_t rows, int ranges, int dh) { return (size_t)rows * ranges * (dh + 2) * sizeof(float); }
  __device__ __forceinline__ float* values(int64_t row, int s) const { return base + (row * ranges + s) * dh; }
  __device__ __forceinline__ f32x2_t* stats(int64_t row, int s) const { return reinterpret_cast<f32x2_t*>(base + rows * ranges * dh) + row * ranges + s; }
};

// The output [B, M, H, Dh] that the joined rows go to; rows [B] or null: so many of a sequence's M rows are real.
struct JoinArgs {
  uint16_t* out; int64_t so_b, so_m, so_h;
  const int32_t* rows;
  int B, M, H, Hk, Dh, dt;
};
// decode: rows of scratch are (b, h), else (b, kv head, token, head of the group)
void launch_join(const JoinArgs& a, int ranges, bool decode, float* scratch, hipStream_t st);

}  // namespace fsvd
