// Launch interface of the 8-bit products (csrc/hip/fp8.hip): e4m3 values
// with a power-of-two scale (e8m0) for each block of 128, which is what the
// matrix instructions of gfx950 take. Host-compilable header: no device
// code. Launches are asynchronous on `stream` of `device`, check their
// arguments (EnforceNotMet) and leave the current device as it was.
#pragma once

#include <cstddef>
#include <cstdint>

#include "collectives/reduce_fns.h"

struct ihipStream_t;
typedef struct ihipStream_t* hipStream_t;

namespace glooamd {
namespace hip {

constexpr int kFp8Block = 128; // elements along a row that share a scale

// q[r, c] = e4m3(x[r, c] / 2^e) and the scales' e of each 1 x 128 block
// (scales [rows, ceil(cols / 128)]). x has any strides. q's rows are qStride
// bytes apart, a multiple of 16; the bytes between are zeros (NaN where the
// last block's are).
void launchQuantizeFp8(
    const void* x,
    int64_t rowStride,
    int64_t colStride,
    DType dtype,
    int64_t rows,
    int64_t cols,
    void* q,
    int64_t qStride,
    void* scales,
    int device,
    hipStream_t stream);

// The same with a scale for each 128 x 128 tile of each expert's matrix:
// q [experts, rows, qStride], scales [experts, ceil(rows / 128),
// ceil(cols / 128)].
void launchQuantizeFp8Tiles(
    const void* x,
    int64_t expertStride,
    int64_t rowStride,
    int64_t colStride,
    DType dtype,
    int64_t experts,
    int64_t rows,
    int64_t cols,
    void* q,
    int64_t qStride,
    void* scales,
    int device,
    hipStream_t stream);

struct Fp8ProductArgs {
  const void* a = nullptr; // [rows, inner], aStride bytes a row
  int64_t aStride = 0;
  const void* aScale = nullptr; // [rows, ceil(inner / 128)]
  const void* b = nullptr; // [experts, n, inner]
  int64_t bStride = 0; // bytes from one row to the next
  int64_t bExpertStride = 0; // bytes from one expert to the next
  const void* bScale = nullptr; // [experts, ceil(n / 128), ceil(inner / 128)]
  const int32_t* offsets = nullptr; // [experts + 1], null: one expert
  int64_t rows = 0;
  int64_t n = 0;
  int64_t inner = 0;
  int experts = 1;
  void* out = nullptr; // [rows, n], begins on 16 bytes
  DType dtype = DType::BF16; // of out: F32, F16 or BF16
};
// out[r] = b[e] a[r] for the rows of each expert; zeros for rows before the
// first expert's and behind the last one's. Sums are fp32's; for BF16 groups
// of eight products lose their bits below 2^-13 of the largest first.
void launchFp8Matmul(
    const Fp8ProductArgs& args,
    int device,
    hipStream_t stream);

struct Fp8WeightGradArgs {
  const void* dy = nullptr; // [m, rows], dyStride bytes a row
  int64_t dyStride = 0;
  const void* dyScale = nullptr; // [m, ceil(rows / 128)]
  const void* x = nullptr; // [n, rows]
  int64_t xStride = 0;
  const void* xScale = nullptr; // [n, ceil(rows / 128)]
  const int32_t* offsets = nullptr; // [experts + 1], null: one expert
  int64_t m = 0;
  int64_t n = 0;
  int64_t rows = 0;
  int experts = 1;
  void* out = nullptr; // [experts, m, n], begins on 16 bytes
  DType dtype = DType::F32;
};
// out[e] = sum over the expert's rows r of dy[:, r] x[:, r]^T.
void launchFp8WeightGrad(
    const Fp8WeightGradArgs& args,
    int device,
    hipStream_t stream);

} // namespace hip
} // namespace glooamd
