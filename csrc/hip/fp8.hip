// 8-bit products for gfx950: quantisation to e4m3 with a power of two for
// each block of 128, dense and grouped products, and the weight gradient.
// Interface and formulas: hip/fp8.h.
//
// The scales are e8m0 bytes because the matrix instructions of gfx950
// (v_mfma_scale_f32_*_f8f6f4) multiply their operands by such scales as they
// read them: a product of blocks then accumulates in one fp32 register over
// all of the inner dimension, with no multiply-add for each result and block.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "hip/device_types.h"
#include "hip/fp8.h"

namespace glooamd {
namespace hip {

namespace {

constexpr int kWave = 64;
constexpr int kQuant = kFp8Block;

using Int8 = int __attribute__((ext_vector_type(8)));
using Bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using Bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using Float16 = float __attribute__((ext_vector_type(16)));

__device__ inline uint32_t absBits(float v) {
  return __float_as_uint(v) & 0x7fffffffu;
}

__device__ inline uint32_t maxBits(uint32_t a, uint32_t b) {
  return a > b ? a : b;
}

template <int kWidth>
__device__ inline uint32_t laneMax(uint32_t v) {
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) {
    v = maxBits(v, __shfl_xor(v, o));
  }
  return v;
}

template <int N>
__device__ inline void storeFp8(uint8_t* to, const float* v, float inv) {
  static_assert(N % 16 == 0, "16 bytes a store");
#pragma unroll
  for (int c = 0; c < N / 16; c++) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float* f = v + c * 16 + i * 4;
      w[i] = fp8Pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
    }
    reinterpret_cast<uint4*>(to)[c] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// --- quantisation ------------------------------------------------------------

struct QuantShape {
  int64_t rowStride;
  int64_t colStride;
  int64_t rows;
  int64_t cols;
  int64_t qStride;
};

// Adjacent columns: eight lanes take a block of 128, 16 elements each.
template <typename T, bool kVec>
__global__ __launch_bounds__(256) void quantizeRowsKernel(
    const T* __restrict__ x,
    uint8_t* __restrict__ q,
    uint8_t* __restrict__ scales,
    QuantShape p) {
  constexpr int kEach = 16;
  const int64_t perRow = (p.qStride + kQuant - 1) / kQuant * 8;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = id / perRow; // eight lanes never part: perRow % 8 == 0
  const int64_t at = id % perRow * kEach;
  float v[kEach];
  const T* from = x + row * p.rowStride + at;
  const bool in = row < p.rows;
  if (kVec && in && at + kEach <= p.cols) {
    constexpr int kSize = Vec16<T>::kSize;
#pragma unroll
    for (int i = 0; i < kEach / kSize; i++) {
      const Vec16<T> part = reinterpret_cast<const Vec16<T>*>(from)[i];
#pragma unroll
      for (int c = 0; c < kSize; c++) {
        v[i * kSize + c] = toFloat(part.v[c]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      v[i] = in && at + i < p.cols ? toFloat(from[i]) : 0.0f;
    }
  }
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    amax = maxBits(amax, absBits(v[i]));
  }
  amax = laneMax<8>(amax);
  if (!in || at >= p.qStride) {
    return;
  }
  const uint32_t byte = fp8ScaleByte(amax);
  storeFp8<kEach>(q + row * p.qStride + at, v, fp8InverseScale(byte));
  if (at % kQuant == 0 && at < p.cols) {
    scales[row * ((p.cols + kQuant - 1) / kQuant) + at / kQuant] =
        static_cast<uint8_t>(byte);
  }
}

// Any strides, and adjacent rows above all: a transposed matrix. 64 rows x
// 128 columns go through LDS, so that lanes run along the rows for the loads
// and along the columns for the stores.
template <typename T>
__global__ __launch_bounds__(256) void quantizeColumnsKernel(
    const T* __restrict__ x,
    uint8_t* __restrict__ q,
    uint8_t* __restrict__ scales,
    QuantShape p) {
  constexpr int kRows = 64;
  __shared__ float tile[kRows][kQuant + 1];
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int64_t col0 = static_cast<int64_t>(blockIdx.y) * kQuant;
  const int lane = threadIdx.x % kRows;
  for (int c = threadIdx.x / kRows; c < kQuant; c += 256 / kRows) {
    const int64_t row = row0 + lane;
    const int64_t col = col0 + c;
    tile[lane][c] = row < p.rows && col < p.cols
        ? toFloat(x[row * p.rowStride + col * p.colStride])
        : 0.0f;
  }
  __syncthreads();
  constexpr int kEach = 32; // four lanes a row
  const int r = threadIdx.x / 4;
  const int c0 = threadIdx.x % 4 * kEach;
  float v[kEach];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    v[i] = tile[r][c0 + i];
    amax = maxBits(amax, absBits(v[i]));
  }
  amax = laneMax<4>(amax);
  const int64_t row = row0 + r;
  if (row >= p.rows) {
    return;
  }
  const uint32_t byte = fp8ScaleByte(amax);
  const float inv = fp8InverseScale(byte);
  uint8_t* to = q + row * p.qStride + col0 + c0;
  if (col0 + c0 + 16 <= p.qStride) {
    storeFp8<16>(to, v, inv);
  }
  if (col0 + c0 + 32 <= p.qStride) {
    storeFp8<16>(to + 16, v + 16, inv);
  }
  if (c0 == 0) {
    scales[row * gridDim.y + blockIdx.y] = static_cast<uint8_t>(byte);
  }
}

// One scale for 128 x 128. Weights: laid out once, so any strides will do.
template <typename T>
__global__ __launch_bounds__(256) void quantizeTilesKernel(
    const T* __restrict__ x,
    uint8_t* __restrict__ q,
    uint8_t* __restrict__ scales,
    QuantShape p) {
  constexpr int kEach = 16;
  __shared__ uint32_t most[4];
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kQuant;
  const int64_t col0 = static_cast<int64_t>(blockIdx.y) * kQuant;
  const int c0 = threadIdx.x % 8 * kEach;
  float v[4][kEach];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t row = row0 + i * 32 + threadIdx.x / 8;
#pragma unroll
    for (int c = 0; c < kEach; c++) {
      const int64_t col = col0 + c0 + c;
      v[i][c] = row < p.rows && col < p.cols
          ? toFloat(x[row * p.rowStride + col * p.colStride])
          : 0.0f;
      amax = maxBits(amax, absBits(v[i][c]));
    }
  }
  amax = laneMax<64>(amax);
  if (threadIdx.x % kWave == 0) {
    most[threadIdx.x / kWave] = amax;
  }
  __syncthreads();
  amax = maxBits(maxBits(most[0], most[1]), maxBits(most[2], most[3]));
  const uint32_t byte = fp8ScaleByte(amax);
  const float inv = fp8InverseScale(byte);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t row = row0 + i * 32 + threadIdx.x / 8;
    if (row < p.rows && col0 + c0 + kEach <= p.qStride) {
      storeFp8<kEach>(q + row * p.qStride + col0 + c0, v[i], inv);
    }
  }
  if (threadIdx.x == 0) {
    scales[blockIdx.x * static_cast<int64_t>(gridDim.y) + blockIdx.y] =
        static_cast<uint8_t>(byte);
  }
}

// --- products ----------------------------------------------------------------

struct ProductShape {
  const uint8_t* a; // the result's rows
  const uint8_t* b; // the result's columns
  const uint8_t* aScale;
  const uint8_t* bScale;
  const int32_t* offsets;
  int64_t aStride;
  int64_t bStride;
  int64_t bExpertStride;
  int64_t m; // product: rows of a, weight gradient: dy's
  int64_t n;
  int64_t inner;
  int experts;
  int tilesN;
  bool aWhole; // rows begin on borders of 16 bytes
  bool bWhole;
};

// Part of an expert's rows: [begin, end) of `of`, kBM at most. of ==
// experts: the rows behind the last one.
struct RowTile {
  int of;
  int64_t begin;
  int64_t end;
};

__device__ inline int64_t clampOffset(
    const int32_t* offsets,
    int e,
    int64_t rows) {
  const int64_t v = offsets[e];
  return v < 0 ? 0 : (v > rows ? rows : v);
}

// The tile-th tile of kBM rows when each expert's rows begin a new one. All
// lanes of a wave look at 64 experts at a time. of = -1: there are fewer.
__device__ inline RowTile findTile(
    const ProductShape& p,
    int64_t tile,
    int size) {
  if (p.offsets == nullptr) {
    const int64_t begin = tile * size;
    const int64_t end = begin + size < p.m ? begin + size : p.m;
    return RowTile{begin < p.m ? 0 : -1, begin, end};
  }
  const int lane = threadIdx.x % kWave;
  int64_t base = 0;
  for (int from = 0; from <= p.experts; from += kWave) {
    const int e = from + lane;
    int64_t begin = 0;
    int64_t end = 0;
    if (e <= p.experts) {
      begin = clampOffset(p.offsets, e, p.m);
      end = e < p.experts ? clampOffset(p.offsets, e + 1, p.m) : p.m;
    }
    const int count =
        end > begin ? static_cast<int>((end - begin + size - 1) / size) : 0;
    int sum = count;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int other = __shfl_up(sum, o);
      sum += lane >= o ? other : 0;
    }
    const int64_t first = base + sum - count;
    const uint64_t here =
        __ballot(tile >= first && tile < first + count);
    if (here != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(here)) - 1;
      const int64_t from2 =
          __shfl(begin + (tile - first) * size, at);
      const int64_t to = __shfl(end, at);
      return RowTile{
          from + at, from2, from2 + size < to ? from2 + size : to};
    }
    base += __shfl(sum, kWave - 1);
  }
  return RowTile{-1, 0, 0};
}

// One operand of a product: rows of bytes, `rows` of them from `p` on.
struct Operand {
  const uint8_t* p;
  int64_t stride;
  int64_t rows;
  int64_t inner; // bytes of a row that belong to it
  bool whole; // rows begin on borders of 16 bytes
};

// Bytes k to k + 15 of a row, zeros in place of those outside [lo, hi).
// Bytes that are masked may hold anything, NaN too, and are never used.
__device__ inline uint4 load16(
    const Operand& o,
    int64_t row,
    int64_t k,
    int64_t lo,
    int64_t hi) {
  if (k >= hi || k + 16 <= lo) {
    return make_uint4(0, 0, 0, 0);
  }
  const uint8_t* at = o.p + row * o.stride + k;
  uint32_t w[4] = {0, 0, 0, 0};
  const bool inside = row * o.stride + k + 16 <=
      (o.rows - 1) * o.stride + o.inner;
  if (o.whole && inside) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
    if (k < lo || k + 16 > hi) {
      const int first = static_cast<int>(lo > k ? lo - k : 0);
      const int last = static_cast<int>(hi < k + 16 ? hi - k : 16);
#pragma unroll
      for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          if (i * 4 + c < first || i * 4 + c >= last) {
            w[i] &= ~(0xffu << (c * 8));
          }
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; i++) {
      if (k + i >= lo && k + i < hi) {
        w[i / 4] |= static_cast<uint32_t>(at[i]) << (i % 4 * 8);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Four results of a row, as one store where that is possible.
template <typename O>
__device__ inline void store4(
    O* row,
    int64_t n,
    int64_t count,
    const float* v,
    bool whole) {
  if (whole && n + 4 <= count) {
    struct alignas(4 * sizeof(O)) V {
      O v[4];
    };
    V o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      o.v[i] = fromFloat<O>(v[i]);
    }
    *reinterpret_cast<V*>(row + n) = o;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (n + i < count) {
      row[n + i] = fromFloat<O>(v[i]);
    }
  }
}

// How products add up.
//
// Native: v_mfma_scale_f32_32x32x64_f8f6f4 takes bytes and scales as they
// are, at twice the rate of 16-bit operands. It adds groups of eight products
// whose bits below 2^-13 of the group's largest one are cut (measured with
// single products of known size; the groups' sums are added in full fp32).
// That is finer than a result of 16 bits by itself, so those take it.
// Exact: fp32 results show the cut. The bytes become bf16 with the scale
// applied (no rounding: e4m3 has four bits, bf16 eight, and their exponents
// are fp32's; below 2^-126 bits are lost) and the bf16 instruction, whose
// groups are added with 24 bits, multiplies those.
template <bool kExact>
struct Fragment;

template <>
struct Fragment<false> {
  Int8 v;
  int scale;
  __device__ void set(uint4 lo, uint4 hi, int byte) {
    reinterpret_cast<uint4*>(&v)[0] = lo;
    reinterpret_cast<uint4*>(&v)[1] = hi;
    scale = byte;
  }
};

template <>
struct Fragment<true> {
  Bf16x8 v[4];
  __device__ void set(uint4 lo, uint4 hi, int byte) {
    // 2^(byte - 127) in fp32; 255 is NaN
    const uint32_t bits = byte == 0 ? 0x00400000u
        : byte == 255             ? 0x7fc00000u
                                  : static_cast<uint32_t>(byte) << 23;
    const float s = __uint_as_float(bits);
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const Bf16x2 a =
          __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, false);
      const Bf16x2 b =
          __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, true);
      v[i / 2][i % 2 * 4] = a[0];
      v[i / 2][i % 2 * 4 + 1] = a[1];
      v[i / 2][i % 2 * 4 + 2] = b[0];
      v[i / 2][i % 2 * 4 + 3] = b[1];
    }
  }
};

// c += a b^T over 64 bytes. Which lane holds which byte of them does not
// matter as long as a and b agree and a row's bytes have one scale.
__device__ inline Float16 multiply(
    const Fragment<false>& a,
    const Fragment<false>& b,
    Float16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
      a.v, b.v, c, 0, 0, 0, a.scale, 0, b.scale);
}

__device__ inline Float16 multiply(
    const Fragment<true>& a,
    const Fragment<true>& b,
    Float16 c) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v[i], b.v[i], c, 0, 0, 0);
  }
  return c;
}

// What a workgroup computes: rows [m0, mEnd) by columns from n0 on, over
// bytes [k0, k1) of the inner dimension.
struct Job {
  Operand a;
  Operand b;
  const uint8_t* aScale;
  const uint8_t* bScale;
  int64_t blocks; // scales of a row
  int64_t m0;
  int64_t mEnd;
  int64_t n0;
  int64_t k0;
  int64_t k1;
};

// A tile of results, TM x TN of the 32 x 32 instruction for each of WM x WN
// waves, kQuant bytes of the inner dimension a step through LDS. The
// result's columns are the instruction's rows: a lane then holds four
// adjacent columns of one row, and its row's scale is its own.
//
// LDS rows are 128 bytes; a row's 16-byte chunks are permuted by (row & 7),
// so that eight rows' equal chunks lie in different banks.
template <int TM, int TN, int WM, int WN>
struct Tile {
  static constexpr int kM = TM * WM * 32;
  static constexpr int kN = TN * WN * 32;
  static constexpr int kThreads = WM * WN * kWave;
};

template <int kRows, int kThreads>
__device__ inline void stage(
    const Operand& o,
    int64_t row0,
    int64_t rowEnd,
    int64_t k,
    int64_t lo,
    int64_t hi,
    uint4* lds) {
#pragma unroll
  for (int i = 0; i < kRows * 8 / kThreads; i++) {
    const int chunk = i * kThreads + threadIdx.x;
    const int row = chunk / 8;
    const int c = chunk % 8;
    const int64_t r = row0 + row < rowEnd ? row0 + row : rowEnd - 1;
    lds[row * 8 + (c ^ (row & 7))] = load16(o, r, k + c * 16, lo, hi);
  }
}

template <typename O, bool kWeightGrad, int TM, int TN, int WM, int WN>
__device__ inline void
computeTile(const Job& job, int64_t n, O* __restrict__ out) {
  using T = Tile<TM, TN, WM, WN>;
  constexpr bool kExact = std::is_same<O, float>::value;
  __shared__ uint4 la[T::kM * 8];
  __shared__ uint4 lb[T::kN * 8];
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  const int waveM = wave / WN * TM * 32;
  const int waveN = wave % WN * TN * 32;
  Float16 acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; i++) {
#pragma unroll
    for (int j = 0; j < TM; j++) {
      acc[i][j] = 0.0f;
    }
  }
  const int64_t kb1 =
      job.k1 > job.k0 ? (job.k1 + kQuant - 1) / kQuant : 0;
  for (int64_t kb = job.k0 / kQuant; kb < kb1; kb++) {
    __syncthreads();
    stage<T::kM, T::kThreads>(
        job.a, job.m0, job.mEnd, kb * kQuant, job.k0, job.k1, la);
    stage<T::kN, T::kThreads>(
        job.b, job.n0, n, kb * kQuant, job.k0, job.k1, lb);
    int sa[TM];
    int sb[TN];
#pragma unroll
    for (int j = 0; j < TM; j++) {
      const int64_t m = job.m0 + waveM + j * 32 + lane % 32;
      sa[j] =
          job.aScale[(m < job.mEnd ? m : job.mEnd - 1) * job.blocks + kb];
    }
#pragma unroll
    for (int i = 0; i < TN; i++) {
      int64_t r = job.n0 + waveN + i * 32 + lane % 32;
      r = r < n ? r : n - 1;
      sb[i] = job.bScale[(kWeightGrad ? r : r / kQuant) * job.blocks + kb];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; s++) {
      Fragment<kExact> fa[TM];
      Fragment<kExact> fb[TN];
      const int c = s * 4 + lane / 32 * 2;
#pragma unroll
      for (int j = 0; j < TM; j++) {
        const int r = waveM + j * 32 + lane % 32;
        fa[j].set(la[r * 8 + (c ^ (r & 7))],
                  la[r * 8 + ((c + 1) ^ (r & 7))], sa[j]);
      }
#pragma unroll
      for (int i = 0; i < TN; i++) {
        const int r = waveN + i * 32 + lane % 32;
        fb[i].set(lb[r * 8 + (c ^ (r & 7))],
                  lb[r * 8 + ((c + 1) ^ (r & 7))], sb[i]);
      }
#pragma unroll
      for (int i = 0; i < TN; i++) {
#pragma unroll
        for (int j = 0; j < TM; j++) {
          acc[i][j] = multiply(fb[i], fa[j], acc[i][j]);
        }
      }
    }
  }
  const bool whole = n % 4 == 0;
#pragma unroll
  for (int j = 0; j < TM; j++) {
    const int64_t m = job.m0 + waveM + j * 32 + lane % 32;
    if (m >= job.mEnd) {
      continue;
    }
#pragma unroll
    for (int i = 0; i < TN; i++) {
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int64_t col =
            job.n0 + waveN + i * 32 + g * 8 + lane / 32 * 4;
        const float v[4] = {acc[i][j][g * 4], acc[i][j][g * 4 + 1],
                            acc[i][j][g * 4 + 2], acc[i][j][g * 4 + 3]};
        store4(out + m * n, col, n, v, whole);
      }
    }
  }
}

template <typename O, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * kWave) void
matmulKernel(ProductShape p, O* __restrict__ out) {
  using T = Tile<TM, TN, WM, WN>;
  const RowTile tile = findTile(p, blockIdx.x / p.tilesN, T::kM);
  if (tile.of < 0) {
    return;
  }
  Job job;
  job.a = Operand{p.a, p.aStride, p.m, p.inner, p.aWhole};
  job.b = Operand{p.b, p.bStride, p.n, p.inner, p.bWhole};
  job.aScale = p.aScale;
  job.bScale = p.bScale;
  job.blocks = (p.inner + kQuant - 1) / kQuant;
  job.m0 = tile.begin;
  job.mEnd = tile.end;
  job.n0 = static_cast<int64_t>(blockIdx.x % p.tilesN) * T::kN;
  job.k0 = 0;
  job.k1 = p.inner;
  if (tile.of == p.experts) {
    job.k1 = 0; // no expert's rows: zeros
  } else {
    job.b.p += tile.of * p.bExpertStride;
    job.bScale += tile.of * ((p.n + kQuant - 1) / kQuant) * job.blocks;
  }
  computeTile<O, false, TM, TN, WM, WN>(job, p.n, out);
}

template <typename O, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * kWave) void
weightGradKernel(ProductShape p, O* __restrict__ out) {
  using T = Tile<TM, TN, WM, WN>;
  const int64_t tilesM = (p.m + T::kM - 1) / T::kM;
  const int64_t rest = blockIdx.x / p.tilesN;
  const int e = static_cast<int>(rest / tilesM);
  Job job;
  job.a = Operand{p.a, p.aStride, p.m, p.inner, p.aWhole};
  job.b = Operand{p.b, p.bStride, p.n, p.inner, p.bWhole};
  job.aScale = p.aScale;
  job.bScale = p.bScale;
  job.blocks = (p.inner + kQuant - 1) / kQuant;
  job.m0 = rest % tilesM * T::kM;
  job.mEnd = job.m0 + T::kM < p.m ? job.m0 + T::kM : p.m;
  job.n0 = static_cast<int64_t>(blockIdx.x % p.tilesN) * T::kN;
  job.k0 = 0;
  job.k1 = p.inner;
  if (p.offsets != nullptr) {
    job.k0 = clampOffset(p.offsets, e, p.inner);
    job.k1 = clampOffset(p.offsets, e + 1, p.inner);
  }
  computeTile<O, true, TM, TN, WM, WN>(
      job, p.n, out + e * p.m * p.n);
}

bool whole16(const void* p, int64_t stride) {
  return aligned16(p) && stride % 16 == 0;
}

void checkProduct(const ProductShape& p) {
  GA_ENFORCE_GE(p.m, 0);
  GA_ENFORCE_GT(p.n, 0);
  GA_ENFORCE_GE(p.inner, 0);
  GA_ENFORCE_LE(p.m, INT32_MAX);
  GA_ENFORCE_LE(p.n, INT32_MAX);
  GA_ENFORCE_LE(p.inner, INT32_MAX);
  GA_ENFORCE_GT(p.experts, 0);
  GA_ENFORCE_GE(p.aStride, 0);
  GA_ENFORCE_GE(p.bStride, 0);
}

} // namespace

void launchQuantizeFp8(
    const void* x,
    int64_t rowStride,
    int64_t colStride,
    DType dtype,
    int64_t rows,
    int64_t cols,
    bool tile,
    void* q,
    int64_t qStride,
    void* scales,
    int device,
    hipStream_t stream) {
  GA_ENFORCE_GE(rows, 0);
  GA_ENFORCE_GE(cols, 0);
  GA_ENFORCE_GE(qStride, cols);
  GA_ENFORCE_EQ(qStride % 16, 0);
  GA_ENFORCE(aligned16(q), "quantize_fp8: q must begin on 16 bytes");
  if (rows == 0 || cols == 0) {
    return;
  }
  DeviceGuard guard(device);
  const QuantShape p{rowStride, colStride, rows, cols, qStride};
  const int64_t blocks = (cols + kQuant - 1) / kQuant;
  GA_ENFORCE_LE((rows + 63) / 64, INT32_MAX);
  GA_ENFORCE_LE(blocks, 65535);
  GA_ENFORCE_LE(qStride, blocks * kQuant);
  auto* to = static_cast<uint8_t*>(q);
  auto* sc = static_cast<uint8_t*>(scales);
  dispatchFloat(dtype, "quantize_fp8", [&](auto t) {
    using T = decltype(t);
    const T* from = static_cast<const T*>(x);
    if (tile) {
      const dim3 grid(
          static_cast<unsigned>((rows + kQuant - 1) / kQuant),
          static_cast<unsigned>(blocks));
      hipLaunchKernelGGL(
          (quantizeTilesKernel<T>), grid, dim3(256), 0, stream, from, to, sc,
          p);
    } else if (colStride == 1) {
      const int64_t lanes =
          rows * ((qStride + kQuant - 1) / kQuant * 8);
      GA_ENFORCE_LE((lanes + 255) / 256, INT32_MAX);
      const dim3 grid(static_cast<unsigned>((lanes + 255) / 256));
      if (aligned16(x) && rowStride % Vec16<T>::kSize == 0) {
        hipLaunchKernelGGL(
            (quantizeRowsKernel<T, true>), grid, dim3(256), 0, stream, from,
            to, sc, p);
      } else {
        hipLaunchKernelGGL(
            (quantizeRowsKernel<T, false>), grid, dim3(256), 0, stream, from,
            to, sc, p);
      }
    } else {
      const dim3 grid(
          static_cast<unsigned>((rows + 63) / 64),
          static_cast<unsigned>(blocks));
      hipLaunchKernelGGL(
          (quantizeColumnsKernel<T>), grid, dim3(256), 0, stream, from, to,
          sc, p);
    }
  });
  GA_HIP_CHECK(hipGetLastError());
}

void launchFp8Matmul(
    const Fp8ProductArgs& a,
    int device,
    hipStream_t stream) {
  ProductShape p{};
  p.a = static_cast<const uint8_t*>(a.a);
  p.b = static_cast<const uint8_t*>(a.b);
  p.aScale = static_cast<const uint8_t*>(a.aScale);
  p.bScale = static_cast<const uint8_t*>(a.bScale);
  p.offsets = a.offsets;
  p.aStride = a.aStride;
  p.bStride = a.bStride;
  p.bExpertStride = a.bExpertStride;
  p.m = a.rows;
  p.n = a.n;
  p.inner = a.inner;
  p.experts = a.experts;
  checkProduct(p);
  GA_ENFORCE(a.offsets != nullptr || a.experts == 1);
  if (p.m == 0) {
    return;
  }
  DeviceGuard guard(device);
  p.aWhole = whole16(p.a, p.aStride);
  p.bWhole = whole16(p.b, p.bStride) && p.bExpertStride % 16 == 0;
  dispatchFloat(a.dtype, "fp8_matmul", [&](auto t) {
    using O = decltype(t);
    auto go = [&](auto kernel, auto tile) {
      using T = decltype(tile);
      p.tilesN = static_cast<int>((p.n + T::kN - 1) / T::kN);
      // every expert's last tile may be a part of one, and so may the
      // rows' behind the last expert
      const int64_t tilesM = a.offsets == nullptr
          ? (p.m + T::kM - 1) / T::kM
          : p.m / T::kM + std::min<int64_t>(p.experts + 1, p.m);
      GA_ENFORCE_LE(tilesM * p.tilesN, INT32_MAX);
      hipLaunchKernelGGL(
          kernel, dim3(static_cast<unsigned>(tilesM * p.tilesN)),
          dim3(T::kThreads), 0, stream, p, static_cast<O*>(a.out));
    };
    go(matmulKernel<O, 2, 2, 2, 2>, Tile<2, 2, 2, 2>{});
  });
  GA_HIP_CHECK(hipGetLastError());
}

void launchFp8WeightGrad(
    const Fp8WeightGradArgs& a,
    int device,
    hipStream_t stream) {
  ProductShape p{};
  p.a = static_cast<const uint8_t*>(a.dy);
  p.b = static_cast<const uint8_t*>(a.x);
  p.aScale = static_cast<const uint8_t*>(a.dyScale);
  p.bScale = static_cast<const uint8_t*>(a.xScale);
  p.offsets = a.offsets;
  p.aStride = a.dyStride;
  p.bStride = a.xStride;
  p.m = a.m;
  p.n = a.n;
  p.inner = a.rows;
  p.experts = a.experts;
  checkProduct(p);
  GA_ENFORCE_GT(a.m, 0);
  GA_ENFORCE(a.offsets != nullptr || a.experts == 1);
  DeviceGuard guard(device);
  p.aWhole = whole16(p.a, p.aStride);
  p.bWhole = whole16(p.b, p.bStride);
  dispatchFloat(a.dtype, "fp8_weight_grad", [&](auto t) {
    using O = decltype(t);
    auto go = [&](auto kernel, auto tile) {
      using T = decltype(tile);
      p.tilesN = static_cast<int>((p.n + T::kN - 1) / T::kN);
      const int64_t tiles =
          (p.m + T::kM - 1) / T::kM * p.tilesN * p.experts;
      GA_ENFORCE_LE(tiles, INT32_MAX);
      hipLaunchKernelGGL(
          kernel, dim3(static_cast<unsigned>(tiles)), dim3(T::kThreads), 0,
          stream, p, static_cast<O*>(a.out));
    };
    go(weightGradKernel<O, 2, 2, 2, 2>, Tile<2, 2, 2, 2>{});
  });
  GA_HIP_CHECK(hipGetLastError());
}

} // namespace hip
} // namespace glooamd
