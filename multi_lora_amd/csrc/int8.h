// Products in 8-bit integers: argument structs shared by csrc/int8.hip and the
// C entry points (the layouts callers see are in include/mlora_hip.h).
#pragma once

#include "common.h"

namespace mlora {

// Codes lie in blocks of 16 rows (a band) by 64 columns, 1 KB each: the 16 bytes
// at 16 (16 c + r) of a block are columns 16 c to 16 c + 15 of row r.  That is how
// lane 16 c + r of a wave holds an operand of the matrix units.  Blocks of the
// same columns lie side by side, band after band: what a tile, or all tiles at
// work at one time, read is one run of memory.
// Columns are padded with zeros to a multiple of 128, rows to one of 16.
constexpr int kInt8Pad = 128;
constexpr int kInt8Block = 1024;
__host__ __device__ constexpr int64_t int8_padded(int64_t k) { return (k + kInt8Pad - 1) / kInt8Pad * kInt8Pad; }
__host__ __device__ constexpr int64_t int8_bands(int64_t rows) { return (rows + 15) / 16; }
constexpr int64_t int8_bytes(int64_t rows, int64_t k) { return int8_bands(rows) * 16 * int8_padded(k); }

// 128^2 * (2^17 - 1) < 2^31: sums of this many products fit 32 bits (codes
// quantised elsewhere may be -128).
constexpr int kInt8MaxK = (1 << 17) - 1;

struct QuantArgs {
  const void* x;
  int64_t x_stride;
  int rows, k;
  int8_t* codes;      // of these rows alone
  float* scales;
};
hipError_t launch_quantize_rows(const QuantArgs& a, int dtype, bool aligned, hipStream_t stream);

struct Int8Args {
  // Activations: codes and scales, or (of calls with few of them) the 16-bit
  // rows themselves.
  const int8_t* a;
  int64_t a_step;     // bytes from a block to that of the next columns
  const float* a_scales;
  const void* x;
  int64_t x_stride;
  int x_aligned;
  int m;
  // Weight.
  const int8_t* b;
  int64_t b_step;
  const float* b_scales;
  int n;
  int k;              // of x; the codes have int8_padded(k)
  const void* bias;   // [n] of the data type, or nullptr
  void* out;
  int64_t out_stride;
  int vec;            // four outputs of a row can be stored at once
  int wide;           // eight can
};
// Whether a call of 16-bit rows is quantised inside the product's own launch.
bool int8_fused(int m, int k);
hipError_t launch_int8_matmul(const Int8Args& a, int dtype, int cus, hipStream_t stream);

}  // namespace mlora
