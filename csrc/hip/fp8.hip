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

using Int4 = int __attribute__((ext_vector_type(4)));
using Int8 = int __attribute__((ext_vector_type(8)));
using Bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using Bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using Float4 = float __attribute__((ext_vector_type(4)));
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

// Any strides, and adjacent rows above all: a transposed matrix. A workgroup
// takes 256 bytes of each of 128 columns through LDS, so that lanes run along
// the rows for loads and scales, and the bytes through LDS again, so that
// they run along the columns for stores. 16384 x 4096 bf16, transposed, 201 MB,
// take 46 us, 4.3 TB/s, one after another on inputs that alternate (57 with
// bytes stored by lanes that run along the rows), and 56 between other kernels,
// with nothing of the input in the caches and their results on their way out.
template <typename T, bool kVec>
__global__ __launch_bounds__(256) void quantizeColumnsKernel(
    const T* __restrict__ x,
    uint8_t* __restrict__ q,
    uint8_t* __restrict__ scales,
    QuantShape p) {
  constexpr int kSize = Vec16<T>::kSize;
  constexpr int kRows = 16 * kSize; // 256 bytes
  constexpr int kParts = 256 / kRows; // lanes that share a row
  constexpr int kEach = kQuant / kParts; // columns of one of them
  constexpr int kWords = kQuant / 4 + 1; // of a row of bytes in LDS
  __shared__ Vec16<T> tile[kQuant][16];
  __shared__ uint32_t most[kParts][kRows];
  auto* bytes = reinterpret_cast<uint32_t*>(tile); // [kRows][kWords]
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
  const int64_t col0 = static_cast<int64_t>(blockIdx.y) * kQuant;
  const int chunk = threadIdx.x % 16;
  const int64_t from = row0 + chunk * kSize;
#pragma unroll
  for (int i = 0; i < kQuant / 16; i++) {
    const int c = i * 16 + threadIdx.x / 16;
    const int64_t col = col0 + c;
    Vec16<T> v;
    if (kVec && col < p.cols && from + kSize <= p.rows) {
      v = *reinterpret_cast<const Vec16<T>*>(x + from + col * p.colStride);
    } else {
#pragma unroll
      for (int j = 0; j < kSize; j++) {
        v.v[j] = col < p.cols && from + j < p.rows
            ? x[(from + j) * p.rowStride + col * p.colStride]
            : fromFloat<T>(0.0f);
      }
    }
    tile[c][chunk] = v;
  }
  __syncthreads();
  const int r = threadIdx.x % kRows;
  const int part = threadIdx.x / kRows;
  float v[kEach];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    v[i] = toFloat(
        reinterpret_cast<const T*>(tile[part * kEach + i])[r]);
    amax = maxBits(amax, absBits(v[i]));
  }
  most[part][r] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kParts; i++) {
    amax = maxBits(amax, most[i][r]);
  }
  const uint32_t byte = fp8ScaleByte(amax);
  const float inv = fp8InverseScale(byte);
#pragma unroll
  for (int i = 0; i < kEach / 4; i++) {
    bytes[r * kWords + part * (kEach / 4) + i] = fp8Pack4(
        v[i * 4] * inv, v[i * 4 + 1] * inv, v[i * 4 + 2] * inv,
        v[i * 4 + 3] * inv);
  }
  if (part == 0 && row0 + r < p.rows) {
    scales[(row0 + r) * gridDim.y + blockIdx.y] = static_cast<uint8_t>(byte);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRows / 32; i++) {
    const int at = i * 32 + threadIdx.x / 8;
    const int64_t row = row0 + at;
    const int64_t col = col0 + threadIdx.x % 8 * 16;
    if (row < p.rows && col + 16 <= p.qStride) {
      const uint32_t* w = bytes + at * kWords + threadIdx.x % 8 * 4;
      *reinterpret_cast<uint4*>(q + row * p.qStride + col) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// One scale for 128 x 128 of each expert. A lane has 64 elements in registers,
// kRows: 16 adjacent ones of four rows, loaded whole; kColumns, a transposed
// matrix: 16 bytes along the rows of each of four columns, so that the bytes
// of a row's four columns are one word of LDS, through which they change
// lanes; kAny: any strides, as kRows one by one. Bound by memory: 64 x 4096 x
// 2048 bf16, 1.6 GB, take 321 us, 5.0 TB/s, and transposed 415 (1415 and 1484
// element by element with an expert a launch).
enum class Order { kRows, kColumns, kAny };

struct QuantTileShape {
  QuantShape m; // of one expert
  int64_t expertStride;
  int rowTiles;
};

template <typename T, Order kOrder>
__global__ __launch_bounds__(256) void quantizeTilesKernel(
    const T* __restrict__ x,
    uint8_t* __restrict__ q,
    uint8_t* __restrict__ scales,
    QuantTileShape shape) {
  constexpr int kEach = 16;
  constexpr int kSize = Vec16<T>::kSize;
  constexpr int kWords = kQuant / 4 + 1; // of a row in LDS
  __shared__ uint32_t most[4];
  __shared__ uint32_t turned[kOrder == Order::kColumns ? kQuant * kWords : 1];
  const QuantShape& p = shape.m;
  const int64_t e = blockIdx.x / shape.rowTiles;
  const int64_t rowTile = blockIdx.x % shape.rowTiles;
  const int64_t row0 = rowTile * kQuant;
  const int64_t col0 = static_cast<int64_t>(blockIdx.y) * kQuant;
  x += e * shape.expertStride;
  q += e * p.rows * p.qStride;
  scales += e * shape.rowTiles * gridDim.y;
  const int c0 = threadIdx.x % 8 * kEach;
  float v[4 * kEach]; // kColumns: [pass][row][four columns], else [row][column]
  constexpr int kChunks = kQuant / kSize; // along the rows
  constexpr int kPasses = kChunks / 8;
  const int r0 = threadIdx.x % kChunks * kSize;
  const int quad = threadIdx.x / kChunks;
  if constexpr (kOrder == Order::kColumns) {
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const int64_t row = row0 + r0;
        const int64_t col =
            col0 + (i * (256 / kChunks) + quad) * 4 + c;
        Vec16<T> part;
        const T* from = x + row + col * p.colStride;
        if (col < p.cols && row + kSize <= p.rows) {
          part = *reinterpret_cast<const Vec16<T>*>(from);
        } else {
#pragma unroll
          for (int k = 0; k < kSize; k++) {
            part.v[k] = col < p.cols && row + k < p.rows
                ? from[k]
                : fromFloat<T>(0.0f);
          }
        }
#pragma unroll
        for (int k = 0; k < kSize; k++) {
          v[(i * kSize + k) * 4 + c] = toFloat(part.v[k]);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int64_t row = row0 + i * 32 + threadIdx.x / 8;
      const int64_t col = col0 + c0;
      const T* from = x + row * p.rowStride + col * p.colStride;
      if (kOrder == Order::kRows && row < p.rows && col + kEach <= p.cols) {
#pragma unroll
        for (int k = 0; k < kEach / kSize; k++) {
          const Vec16<T> part = reinterpret_cast<const Vec16<T>*>(from)[k];
#pragma unroll
          for (int c = 0; c < kSize; c++) {
            v[i * kEach + k * kSize + c] = toFloat(part.v[c]);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < kEach; c++) {
          v[i * kEach + c] = row < p.rows && col + c < p.cols
              ? toFloat(from[c * p.colStride])
              : 0.0f;
        }
      }
    }
  }
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 4 * kEach; i++) {
    amax = maxBits(amax, absBits(v[i]));
  }
  amax = laneMax<64>(amax);
  if (threadIdx.x % kWave == 0) {
    most[threadIdx.x / kWave] = amax;
  }
  __syncthreads();
  amax = maxBits(maxBits(most[0], most[1]), maxBits(most[2], most[3]));
  const uint32_t byte = fp8ScaleByte(amax);
  const float inv = fp8InverseScale(byte);
  if constexpr (kOrder == Order::kColumns) {
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
#pragma unroll
      for (int k = 0; k < kSize; k++) {
        const float* f = v + (i * kSize + k) * 4;
        turned[(r0 + k) * kWords + i * (256 / kChunks) + quad] =
            fp8Pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = i * 32 + threadIdx.x / 8;
    const int64_t row = row0 + r;
    if (row < p.rows && col0 + c0 + kEach <= p.qStride) {
      uint8_t* to = q + row * p.qStride + col0 + c0;
      if constexpr (kOrder == Order::kColumns) {
        const uint32_t* w = turned + r * kWords + c0 / 4;
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        storeFp8<kEach>(to, v + i * kEach, inv);
      }
    }
  }
  if (threadIdx.x == 0) {
    scales[rowTile * gridDim.y + blockIdx.y] = static_cast<uint8_t>(byte);
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
  bool stream; // results are stored past the caches
};

// Part of an expert's rows: [begin, end) of `of`. of == experts: the rows
// behind the last one's, experts + 1: those before the first one's.
struct RowTile {
  int of;
  int64_t begin;
  int64_t end;
};

// The same value in every lane, told to the compiler: what follows from it
// is held once a wave.
__device__ inline int uniform(int v) {
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ inline int64_t uniform(int64_t v) {
  const uint32_t lo = uniform(static_cast<int>(v));
  const uint32_t hi = uniform(static_cast<int>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ inline int64_t clampOffset(
    const int32_t* offsets,
    int e,
    int64_t rows) {
  const int64_t v = offsets[e];
  return v < 0 ? 0 : (v > rows ? rows : v);
}

// Rows [begin, end) of expert e, or those of none (see RowTile).
__device__ inline void rowsOf(
    const ProductShape& p,
    int e,
    int64_t& begin,
    int64_t& end) {
  begin = 0;
  end = 0;
  if (e <= p.experts) {
    begin = clampOffset(p.offsets, e, p.m);
    end = e < p.experts ? clampOffset(p.offsets, e + 1, p.m) : p.m;
  } else if (e == p.experts + 1) {
    end = clampOffset(p.offsets, 0, p.m);
  }
}

__device__ inline int waveScan(int v) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int other = __shfl_up(v, o);
    v += lane >= o ? other : 0;
  }
  return v;
}

// How many tiles of `size` rows there are when each expert's rows begin a
// new one. All lanes of a wave look at 64 experts at a time.
__device__ inline int countTiles(const ProductShape& p, int size) {
  if (p.offsets == nullptr) {
    return static_cast<int>((p.m + size - 1) / size);
  }
  int base = 0;
  for (int from = 0; from < p.experts + 2; from += kWave) {
    int64_t begin;
    int64_t end;
    rowsOf(p, from + static_cast<int>(threadIdx.x) % kWave, begin, end);
    const int count =
        end > begin ? static_cast<int>((end - begin + size - 1) / size) : 0;
    base += uniform(__shfl(waveScan(count), kWave - 1));
  }
  return base;
}

// The tile-th of them. of = -1: there are fewer.
__device__ inline RowTile findTile(
    const ProductShape& p,
    int tile,
    int size) {
  if (p.offsets == nullptr) {
    const int64_t begin = static_cast<int64_t>(tile) * size;
    const int64_t end = begin + size < p.m ? begin + size : p.m;
    return RowTile{begin < p.m ? 0 : -1, begin, end};
  }
  int base = 0;
  for (int from = 0; from < p.experts + 2; from += kWave) {
    int64_t begin;
    int64_t end;
    rowsOf(p, from + static_cast<int>(threadIdx.x) % kWave, begin, end);
    const int count =
        end > begin ? static_cast<int>((end - begin + size - 1) / size) : 0;
    const int sum = waveScan(count);
    const int first = base + sum - count;
    const uint64_t here = __ballot(tile >= first && tile < first + count);
    if (here != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(here)) - 1;
      const int64_t start = uniform(
          __shfl(begin + static_cast<int64_t>(tile - first) * size, at));
      const int64_t to = uniform(__shfl(end, at));
      return RowTile{
          uniform(from + at), start, start + size < to ? start + size : to};
    }
    base += uniform(__shfl(sum, kWave - 1));
  }
  return RowTile{-1, 0, 0};
}

// Which tile this workgroup computes. Workgroups go to the card's eight dies
// in turn, and each die has a cache of its own: a die takes tiles that lie
// together, kBand rows of tiles at a time, column by column, so that the
// workgroups that run at once on it read the same few bands of both operands.
constexpr int kDies = 8;
constexpr int kBand = 8;

struct TileAt {
  int m;
  int n;
};

__device__ inline TileAt inBands(int64_t id, int tilesM, int tilesN) {
  const int band =
      static_cast<int>(id / (static_cast<int64_t>(kBand) * tilesN));
  const int inBand =
      static_cast<int>(id - static_cast<int64_t>(band) * kBand * tilesN);
  const int left = tilesM - band * kBand;
  const int height = left < kBand ? left : kBand;
  return TileAt{band * kBand + inBand % height, inBand / height};
}

__device__ inline bool tileAt(int tilesM, int tilesN, TileAt& at) {
  const int64_t total = static_cast<int64_t>(tilesM) * tilesN;
  const int die = blockIdx.x % kDies;
  const int64_t begin = total * die / kDies;
  const int64_t id = begin + blockIdx.x / kDies;
  if (id >= total * (die + 1) / kDies) {
    return false;
  }
  at = inBands(id, tilesM, tilesN);
  return true;
}

unsigned gridOf(int64_t tiles, int threads) {
  return groupsOf((tiles + kDies - 1) / kDies * kDies, threads);
}

// One operand of a product: rows of bytes, `rows` of them from `p` on.
struct Operand {
  const uint8_t* p;
  int64_t stride;
  int64_t rows;
  int64_t inner; // bytes of a row that belong to it
  bool whole; // rows begin on borders of 16 bytes
};

// Bytes k to k + 15, zeros in place of those outside [lo, hi). What is
// masked may hold anything, NaN too.
__device__ inline uint4 maskOf(uint4 v, int64_t k, int64_t lo, int64_t hi) {
  const int first = static_cast<int>(lo > k ? (lo - k < 16 ? lo - k : 16) : 0);
  const int last = static_cast<int>(hi < k + 16 ? (hi > k ? hi - k : 0) : 16);
  uint64_t w[2] = {static_cast<uint64_t>(v.y) << 32 | v.x,
                   static_cast<uint64_t>(v.w) << 32 | v.z};
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int f = first - i * 8;
    const int l = last - i * 8;
    w[i] = f > 7 || l < 1 ? 0
                          : w[i] & ~0ull << (f > 0 ? f * 8 : 0) &
            ~0ull >> (l < 8 ? 64 - l * 8 : 0);
  }
  return make_uint4(
      static_cast<uint32_t>(w[0]), static_cast<uint32_t>(w[0] >> 32),
      static_cast<uint32_t>(w[1]), static_cast<uint32_t>(w[1] >> 32));
}

// The same of a row in memory, of any alignment: none but its own bytes and
// those of its operand are read.
__device__ inline uint4 load16(
    const Operand& o,
    int64_t row,
    int64_t k,
    int64_t lo,
    int64_t hi) {
  const int64_t at = row * o.stride + k;
  if (k >= hi || k + 16 <= lo) {
    return make_uint4(0, 0, 0, 0);
  }
  if (o.whole && at + 16 <= (o.rows - 1) * o.stride + o.inner) {
    return maskOf(*reinterpret_cast<const uint4*>(o.p + at), k, lo, hi);
  }
  uint64_t w[2] = {0, 0};
  const int first = static_cast<int>(lo > k ? lo - k : 0);
  const int last = static_cast<int>(hi < k + 16 ? hi - k : 16);
#pragma unroll 1
  for (int i = first; i < last; i++) {
    const uint64_t byte = static_cast<uint64_t>(o.p[at + i]) << (i % 8 * 8);
    w[0] |= i < 8 ? byte : 0;
    w[1] |= i < 8 ? 0 : byte;
  }
  return make_uint4(
      static_cast<uint32_t>(w[0]), static_cast<uint32_t>(w[0] >> 32),
      static_cast<uint32_t>(w[1]), static_cast<uint32_t>(w[1] >> 32));
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

// The same for 16 bytes of results.
template <typename O>
__device__ inline void store16(
    O* row,
    int64_t n,
    int64_t count,
    const uint32_t (&w)[4],
    bool whole,
    bool stream) {
  constexpr int kEach = 16 / sizeof(O);
  const Int4 v = {
      static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]),
      static_cast<int>(w[3])};
  if (whole && n + kEach <= count) {
    if (stream) {
      __builtin_nontemporal_store(v, reinterpret_cast<Int4*>(row + n));
    } else {
      *reinterpret_cast<Int4*>(row + n) = v;
    }
    return;
  }
  const auto parts = __builtin_bit_cast(Vec16<O>, v);
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    if (n + i < count) {
      row[n + i] = parts.v[i];
    }
  }
}

// The upper 32 lanes of a and the lower ones of b change places.
__device__ inline void swapHalves(uint32_t& a, uint32_t& b) {
  const auto v = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = v[0];
  b = v[1];
}

// Lanes 16 to 31 and 48 to 63 of a and the 16 before them of b.
__device__ inline void swapQuarters(uint32_t& a, uint32_t& b) {
  const auto v = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = v[0];
  b = v[1];
}

// How products add up.
//
// Native: v_mfma_scale_f32_32x32x64_f8f6f4 takes bytes and scales as they
// are, at twice the rate of 16-bit operands. It adds groups of eight products
// whose bits below 2^-13 of the group's largest one are cut (measured with
// single products of known size; the groups' sums are added in full fp32):
// seven of a group lose up to 7 * 2^-13 < 2^-10 of the largest. bf16 results
// take it: that is a quarter of half their step, 2^-8 (with random operands it
// is 1.5e-5 of the result's norm). fp16 results, half a step of which is 2^-11,
// do not, at the cost of time: 4095 x 8192 x 4096 242 us, bf16 117.
// Exact: fp32 and fp16 results show the cut. The bytes become bf16 with the
// scale applied (no rounding: e4m3 has four bits, bf16 eight, and their
// exponents are fp32's; below 2^-126 bits are lost) and the bf16 instruction,
// whose groups are added with 24 bits, multiplies those.
template <typename O>
constexpr bool kExactSums = !std::is_same<O, __hip_bfloat16>::value;

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

// 2^(byte - 127) in fp32; 255 is NaN
__device__ inline float scaleOf(int byte) {
  return __uint_as_float(
      byte == 0         ? 0x00400000u
          : byte == 255 ? 0x7fc00000u
                        : static_cast<uint32_t>(byte) << 23);
}

// Eight bytes as bf16, with their scale.
__device__ inline Bf16x8 toBf16(uint32_t lo, uint32_t hi, float s) {
  Bf16x8 v;
  const uint32_t w[2] = {lo, hi};
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const Bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, false);
    const Bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], s, true);
    v[i * 4] = a[0];
    v[i * 4 + 1] = a[1];
    v[i * 4 + 2] = b[0];
    v[i * 4 + 3] = b[1];
  }
  return v;
}

template <>
struct Fragment<true> {
  Bf16x8 v[4];
  __device__ void set(uint4 lo, uint4 hi, int byte) {
    const float s = scaleOf(byte);
    v[0] = toBf16(lo.x, lo.y, s);
    v[1] = toBf16(lo.z, lo.w, s);
    v[2] = toBf16(hi.x, hi.y, s);
    v[3] = toBf16(hi.z, hi.w, s);
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

// The same for 16 x 16 results, over 128 bytes.
__device__ inline Float4 multiply(
    const Fragment<false>& a,
    const Fragment<false>& b,
    Float4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      a.v, b.v, c, 0, 0, 0, a.scale, 0, b.scale);
}

__device__ inline Float4 multiply(
    const Fragment<true>& a,
    const Fragment<true>& b,
    Float4 c) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
  }
  return c;
}

// The widest tiles keep two stages of LDS and a third of half a block in
// registers (see Product::run).
constexpr int kWideStages = 4;

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
// waves, kQuant bytes of the inner dimension at a time through LDS. The
// result's columns are the instruction's rows: a lane then holds four
// adjacent columns of one row, and its row's scale is its own.
//
// LDS rows are 128 bytes, half of its 64 banks. A row's 16-byte chunks are
// permuted by (row / 2) % 8, so that equal chunks of the 16 rows that one
// cycle of a 16-byte read serves lie in 16 different places.
constexpr int kChunks = kQuant / 16;

__device__ inline int chunkOf(int row, int c) {
  return c ^ (row >> 1 & 7);
}

template <int TM, int TN, int WM, int WN>
struct Tile {
  static constexpr int kM = TM * WM * 32;
  static constexpr int kN = TN * WN * 32;
  static constexpr int kThreads = WM * WN * kWave;
};

// Rows row0 to row0 + kRows - 1 of an operand on their way into LDS; those
// from rowEnd on are copies of the last one, and their results are dropped.
template <int kRows, int kThreads>
struct Stager {
  static constexpr int kEach = kRows * kChunks / kThreads; // chunks a lane
  const Operand& o;
  int64_t row0;
  int64_t rowEnd;
  int64_t lo; // bytes of the inner dimension that count: [lo, hi)
  int64_t hi;
  bool direct;
  __amdgpu_buffer_rsrc_t buffer;
  int offset[kEach];

  __device__ Stager(
      const Operand& operand,
      int64_t first,
      int64_t end,
      int64_t low,
      int64_t high)
      : o(operand), row0(first), rowEnd(end), lo(low), hi(high) {
    // Offsets from row0 on are 32 bits wide.
    const int64_t room = (o.rows - 1 - row0) * o.stride + o.inner;
    direct = o.whole && o.stride <= (1 << 22) && o.inner < (1 << 28);
    buffer = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(o.p + row0 * o.stride), 0,
        static_cast<int>(room < (1ll << 31) - 1 ? room : (1ll << 31) - 1),
        0x00027000);
    // The wave writes 64 chunks to adjacent places: the permutation of a
    // row's chunks is one of the lanes' addresses.
    const int last = static_cast<int>(rowEnd - row0) - 1;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      const int chunk = i * kThreads + threadIdx.x;
      const int row = chunk / kChunks;
      const int c = chunkOf(row, chunk % kChunks);
      offset[i] = (row < last ? row : last) * static_cast<int>(
                      direct ? o.stride : 0) + c * 16;
    }
  }

  // Bytes k on, all of which count, straight into LDS: no registers and no
  // wait until they are needed.
  __device__ void loadDirect(int k, uint4* lds) const {
    k = uniform(k);
    const int wave = uniform(static_cast<int>(threadIdx.x / kWave));
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          buffer,
          (__attribute__((address_space(3))) void*)(
              lds + i * kThreads + wave * kWave),
          16, offset[i], k, 0, 0);
    }
  }

  // Bytes k on through masks.
  __device__ void loadMasked(int64_t k, uint4* lds) const {
#pragma unroll 1
    for (int i = 0; i < kEach; i++) {
      const int chunk = i * kThreads + threadIdx.x;
      const int row = chunk / kChunks;
      const int c = chunkOf(row, chunk % kChunks);
      const int64_t r = row0 + row < rowEnd ? row0 + row : rowEnd - 1;
      lds[chunk] = load16(o, r, k + c * 16, lo, hi);
    }
  }
};

// The scales of a step's rows and columns, one a lane, on their way into
// LDS. Bytes that are far apart take a cycle each to load: a wave's 64 lanes
// fetch them once for the workgroup and not for every wave's fragments.
template <bool kWeightGrad, typename T>
struct ScaleStager {
  static_assert(T::kM + T::kN <= T::kThreads, "one scale a lane");
  static_assert(T::kM % kWave == 0, "a wave's scales are of one operand");
  const uint8_t* p; // of the wave's operand
  int64_t blocks;
  int row;
  int offset;
  __amdgpu_buffer_rsrc_t buffer;

  __device__ ScaleStager(const Job& job, int64_t n) : blocks(job.blocks) {
    const int wave = uniform(static_cast<int>(threadIdx.x / kWave));
    const bool ofA = wave < T::kM / kWave;
    const int last = static_cast<int>(
        ofA ? job.mEnd - 1 - job.m0
            : (n - 1 - job.n0 < T::kN ? n - 1 - job.n0 : T::kN - 1));
    row = static_cast<int>(threadIdx.x) - (ofA ? 0 : T::kM);
    row = row < last ? row : last;
    if (ofA) {
      p = job.aScale + job.m0 * job.blocks;
    } else if (kWeightGrad) {
      p = job.bScale + job.n0 * job.blocks;
    } else {
      p = job.bScale + job.n0 / kQuant * job.blocks;
      row /= kQuant;
    }
    offset = row * static_cast<int>(job.blocks);
    buffer = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p), 0, 0x7fffffff, 0x00027000);
  }

  __device__ void loadDirect(int kb, int* ls) const {
    const int wave = uniform(static_cast<int>(threadIdx.x / kWave));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        buffer,
        (__attribute__((address_space(3))) void*)(ls + wave * kWave), 1,
        offset, uniform(kb), 0, 0);
  }

  __device__ void load(int kb, int* ls) const {
    ls[threadIdx.x] = p[row * blocks + kb];
  }
};

// The wave's loads into LDS but the last kLater have arrived, its reads are
// done, and so have and are all other waves'. A plain barrier and not
// __syncthreads(), which would wait for every load into LDS.
template <int kLater>
__device__ inline void arrived() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLater) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename O, bool kWeightGrad, int TM, int TN, int WM, int WN, int S>
struct Product {
  using T = Tile<TM, TN, WM, WN>;
  static constexpr bool kExact = kExactSums<O>;
  const Job& job;
  int64_t n;
  int lane;
  int waveM;
  int waveN;
  int sa[TM];
  int sb[TN];
  Float16 acc[TN][TM];

  __device__ Product(const Job& j, int64_t columns) : job(j), n(columns) {
    const int wave = threadIdx.x / kWave;
    lane = threadIdx.x % kWave;
    waveM = wave / WN * TM * 32;
    waveN = wave % WN * TN * 32;
#pragma unroll
    for (int i = 0; i < TN; i++) {
#pragma unroll
      for (int k = 0; k < TM; k++) {
        acc[i][k] = 0.0f;
      }
    }
  }

  // A lane of the instruction's result has four times four adjacent columns
  // of a row. Stored like that, 32 rows would get 32 bytes each (16 of 16-bit
  // results) at a time; lanes exchange them first, within the vector unit,
  // and a store is 64 bytes of each of 16 rows. 16384 x 4096 x 2048 for 16
  // experts, bf16: 258 us against 288.
  __device__ void write(O* __restrict__ out, bool stream) const {
    constexpr int kEach = 16 / sizeof(O); // a lane's columns
    constexpr int kParts = 8 / kEach; // of 32 columns
    constexpr bool kFull = sizeof(O) == 4;
    const bool whole = n % kEach == 0;
    const int quarter = lane / 16;
#pragma unroll
    for (int j = 0; j < TM; j++) {
#pragma unroll
      for (int i = 0; i < TN; i++) {
#pragma unroll
        for (int c = 0; c < kParts; c++) {
          uint32_t v[2][4]; // rows 0 to 15, and 16 to 31
          if constexpr (kFull) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
              v[0][r] = __float_as_uint(acc[i][j][c * 8 + r]);
              v[1][r] = __float_as_uint(acc[i][j][c * 8 + 4 + r]);
              swapHalves(v[0][r], v[1][r]);
              swapQuarters(v[0][r], v[1][r]);
            }
          } else {
#pragma unroll
            for (int r = 0; r < 4; r++) {
              v[0][r] = pack2(acc[i][j][r * 2], acc[i][j][r * 2 + 1]);
              v[1][r] = pack2(acc[i][j][8 + r * 2], acc[i][j][9 + r * 2]);
            }
#pragma unroll
            for (int r = 0; r < 2; r++) {
              swapHalves(v[0][r], v[0][2 + r]);
              swapHalves(v[1][r], v[1][2 + r]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
              swapQuarters(v[0][r], v[1][r]);
            }
          }
          const int64_t col = job.n0 + waveN + i * 32 +
              (kFull ? c * 16 + quarter * 4
                      : quarter % 2 * 16 + quarter / 2 * 8);
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const int64_t m = job.m0 + waveM + j * 32 + r * 16 + lane % 16;
            if (m < job.mEnd) {
              store16(out + m * n, col, n, v[r], whole, stream);
            }
          }
        }
      }
    }
  }

  static __device__ uint32_t pack2(float lo, float hi) {
    struct Two {
      O v[2];
    };
    return __builtin_bit_cast(
        uint32_t, Two{{fromFloat<O>(lo), fromFloat<O>(hi)}});
  }

  __device__ void readScales(const int* ls) {
#pragma unroll
    for (int j = 0; j < TM; j++) {
      sa[j] = ls[waveM + j * 32 + lane % 32];
    }
#pragma unroll
    for (int i = 0; i < TN; i++) {
      sb[i] = ls[T::kM + waveN + i * 32 + lane % 32];
    }
  }

  // The operands of half a block, 64 bytes of the inner dimension.
  struct Half {
    Fragment<false> a[TM];
    Fragment<false> b[TN];
  };

  __device__ void
  read(const uint4* la, const uint4* lb, int h, Half& f) const {
    const int c = h * 4 + lane / 32 * 2;
#pragma unroll
    for (int j = 0; j < TM; j++) {
      const int r = waveM + j * 32 + lane % 32;
      f.a[j].set(la[r * kChunks + chunkOf(r, c)],
                 la[r * kChunks + chunkOf(r, c + 1)], sa[j]);
    }
#pragma unroll
    for (int i = 0; i < TN; i++) {
      const int r = waveN + i * 32 + lane % 32;
      f.b[i].set(lb[r * kChunks + chunkOf(r, c)],
                 lb[r * kChunks + chunkOf(r, c + 1)], sb[i]);
    }
  }

  __device__ void add(const Half& f) {
#pragma unroll
    for (int i = 0; i < TN; i++) {
#pragma unroll
      for (int j = 0; j < TM; j++) {
        acc[i][j] = multiply(f.b[i], f.a[j], acc[i][j]);
      }
    }
  }

  // A quarter of half a block as bf16: 16 bytes of the inner dimension, eight
  // of which a lane holds.
  struct Piece {
    Bf16x8 a[TM];
    Bf16x8 b[TN];
  };

  static __device__ uint32_t word(const Fragment<false>& f, int i) {
    return static_cast<uint32_t>(f.v[i]);
  }

  __device__ void convert(
      const Half& f,
      int i,
      const float (&fa)[TM],
      const float (&fb)[TN],
      Piece& to) const {
#pragma unroll
    for (int j = 0; j < TM; j++) {
      to.a[j] =
          toBf16(word(f.a[j], i * 2), word(f.a[j], i * 2 + 1), fa[j]);
    }
#pragma unroll
    for (int j = 0; j < TN; j++) {
      to.b[j] =
          toBf16(word(f.b[j], i * 2), word(f.b[j], i * 2 + 1), fb[j]);
    }
  }

  __device__ void scales(float (&fa)[TM], float (&fb)[TN]) const {
#pragma unroll
    for (int j = 0; j < TM; j++) {
      fa[j] = scaleOf(sa[j]);
    }
#pragma unroll
    for (int i = 0; i < TN; i++) {
      fb[i] = scaleOf(sb[i]);
    }
  }

  __device__ void add(const Piece& f) {
#pragma unroll
    for (int i = 0; i < TN; i++) {
#pragma unroll
      for (int j = 0; j < TM; j++) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            f.b[i], f.a[j], acc[i][j], 0, 0, 0);
      }
    }
  }

  // Exact: while one piece is multiplied the next one is converted, which the
  // groups ask of the compiler: left alone it converts first and multiplies
  // then, and the matrix unit waits.
  __device__ void stepExact(const Half (&f)[2]) {
    float fa[TM];
    float fb[TN];
    scales(fa, fb);
    Piece piece[2];
    convert(f[0], 0, fa, fb, piece[0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 8; u++) {
      if (u < 7) {
        convert(f[(u + 1) / 4], (u + 1) % 4, fa, fb, piece[(u + 1) % 2]);
      }
      add(piece[u % 2]);
#pragma unroll
      for (int i = 0; i < TN * TM; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0); // one product
        __builtin_amdgcn_sched_group_barrier(
            0x2, (TM + TN) * 4 / (TM * TN), 0); // conversions
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  __device__ void step(const uint4* la, const uint4* lb, const int* ls) {
    readScales(ls);
    if constexpr (kExact) {
      Half f[2];
      read(la, lb, 0, f[0]);
      read(la, lb, 1, f[1]);
      stepExact(f);
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        Half f;
        read(la, lb, h, f);
        add(f);
      }
    }
  }

  // A block of which only bytes [k0, k1) count, zeros in place of the others:
  // they may be NaN. Half a block that has none is left out.
  __device__ void
  stepEdge(const uint4* la, const uint4* lb, const int* ls, int k) {
    readScales(ls);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int first = k + h * 64;
      if (first + 64 <= job.k0 || first >= job.k1) {
        continue;
      }
      Half f;
      read(la, lb, h, f);
      const int own = first + lane / 32 * 32;
      Int8 mask;
#pragma unroll
      for (int w = 0; w < 8; w++) {
        mask[w] = bytesFrom(job.k0 - own - w * 4) &
            ~bytesFrom(job.k1 - own - w * 4);
      }
#pragma unroll
      for (int j = 0; j < TM; j++) {
        f.a[j].v &= mask;
      }
#pragma unroll
      for (int i = 0; i < TN; i++) {
        f.b[i].v &= mask;
      }
      if constexpr (kExact) {
        float fa[TM];
        float fb[TN];
        scales(fa, fb);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          Piece piece;
          convert(f, i, fa, fb, piece);
          add(piece);
        }
      } else {
        add(f);
      }
    }
  }

  // The bytes of a word from the n-th on.
  static __device__ int bytesFrom(int n) {
    return n <= 0 ? -1 : (n >= 4 ? 0 : static_cast<int>(~0u << n * 8));
  }

  // A ring of three stages of LDS, two on their way while one is multiplied,
  // or of two, one on its way. Arrays of their own and not parts of one: the
  // compiler sees that a read of one does not wait for loads into another.
  __device__ void run() {
    constexpr int kSizeA = T::kM * kChunks;
    constexpr int kSizeB = T::kN * kChunks;
    constexpr bool kThree = S == 3;
    constexpr bool kWide = S == kWideStages;
    __shared__ uint4 la0[kSizeA];
    __shared__ uint4 lb0[kSizeB];
    __shared__ uint4 la1[kSizeA];
    __shared__ uint4 lb1[kSizeB];
    __shared__ uint4 la2[kThree ? kSizeA : 1];
    __shared__ uint4 lb2[kThree ? kSizeB : 1];
    __shared__ int ls0[T::kThreads];
    __shared__ int ls1[T::kThreads];
    __shared__ int ls2[kThree ? T::kThreads : 1];
    if (job.k1 <= job.k0) {
      return;
    }
    // A wave none of whose rows are the expert's brings its part into LDS and
    // multiplies nothing: the others have the matrix units to themselves. 256
    // rows for 64 experts, 4096 x 2048, fp32: 112 us against 131, 16384 rows
    // for 32 experts, 4096 x 4096, bf16: 309 against 314.
    const bool live = job.m0 + uniform(waveM) < job.mEnd;
    using StageA = Stager<T::kM, T::kThreads>;
    using StageB = Stager<T::kN, T::kThreads>;
    const StageA a(job.a, job.m0, job.mEnd, job.k0, job.k1);
    const StageB b(job.b, job.n0, n, job.k0, job.k1);
    const ScaleStager<kWeightGrad, T> s(job, n);
    const int first = uniform(static_cast<int>(job.k0 / kQuant));
    const int last =
        uniform(static_cast<int>((job.k1 + kQuant - 1) / kQuant));
    // Blocks that lie within the rows, [first, direct), are loaded directly.
    // An expert's first and last one in a weight gradient may hold bytes of
    // its neighbours: those come behind the others, [whole0, whole1), and are
    // masked.
    const int full = static_cast<int>(job.a.inner / kQuant);
    const int direct = uniform(
        a.direct && b.direct ? (last < full ? last : full) : first);
    if (first < direct) {
      int whole0 = uniform(
          static_cast<int>((job.k0 + kQuant - 1) / kQuant));
      int whole1 = uniform(static_cast<int>(job.k1 / kQuant));
      whole1 = whole1 < direct ? whole1 : direct;
      whole0 = whole0 < whole1 ? whole0 : whole1;
      const int whole = whole1 - whole0;
      const int total = direct - first;
      // The t-th block in this order. Behind the last the loads go on with
      // that one again: every step then has as many loads on their way.
      const auto nth = [&](int t) {
        t = t < total ? t : total - 1;
        const int edge = first + t - whole;
        return uniform(
            t < whole ? whole0 + t : (edge < whole0 ? edge : edge + whole));
      };
      constexpr int kLater =
          kThree ? StageA::kEach + StageB::kEach + 1 : 0;
      const auto begin = [&](int t, uint4* la, uint4* lb, int* ls) {
        const int kb = nth(t);
        a.loadDirect(kb * kQuant, la);
        b.loadDirect(kb * kQuant, lb);
        s.loadDirect(kb, ls);
      };
      const auto rest = [&](int t, uint4* la, uint4* lb, const int* ls,
                            auto live) {
        if (t < total) {
          if constexpr (decltype(live)::value) {
            if (!kWeightGrad || t < whole) {
              step(la, lb, ls);
            } else {
              stepEdge(la, lb, ls, nth(t) * kQuant);
            }
          }
        }
      };
      const auto all = [&](auto live) {
        constexpr bool kLive = decltype(live)::value;
        int t = 0;
        begin(0, la0, lb0, ls0);
        if constexpr (kWide) {
          // While half a block is multiplied the next half is read. A stage is
          // free in the middle of its step, and one barrier says both that and
          // that the next stage has arrived. (Whole blocks alone: the rows of
          // a product do not part the inner dimension.)
          begin(1, la1, lb1, ls1);
          Half f0;
          Half f1;
          arrived<StageA::kEach + StageB::kEach + 1>();
          if constexpr (kLive) {
            readScales(ls0);
            read(la0, lb0, 0, f0);
          }
          for (; t + 1 < total; t += 2) {
            if constexpr (kLive) {
              read(la0, lb0, 1, f1);
              add(f0);
            }
            __builtin_amdgcn_sched_barrier(0);
            arrived<0>();
            begin(t + 2, la0, lb0, ls0);
            if constexpr (kLive) {
              readScales(ls1);
              read(la1, lb1, 0, f0);
              add(f1);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kLive) {
              read(la1, lb1, 1, f1);
              add(f0);
            }
            __builtin_amdgcn_sched_barrier(0);
            arrived<0>();
            begin(t + 3, la1, lb1, ls1);
            if constexpr (kLive) {
              readScales(ls0);
              read(la0, lb0, 0, f0);
              add(f1);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if (t < total) {
            if constexpr (kLive) {
              read(la0, lb0, 1, f1);
              add(f0);
              add(f1);
            }
          }
        } else if constexpr (kThree) {
          begin(1, la1, lb1, ls1);
          for (; t + 2 < whole; t += 3) {
            arrived<kLater>();
            begin(t + 2, la2, lb2, ls2);
            if constexpr (kLive) {
              step(la0, lb0, ls0);
            }
            arrived<kLater>();
            begin(t + 3, la0, lb0, ls0);
            if constexpr (kLive) {
              step(la1, lb1, ls1);
            }
            arrived<kLater>();
            begin(t + 4, la1, lb1, ls1);
            if constexpr (kLive) {
              step(la2, lb2, ls2);
            }
          }
          // at most two whole blocks and two edges are left
          arrived<kLater>();
          begin(t + 2, la2, lb2, ls2);
          rest(t, la0, lb0, ls0, live);
          arrived<kLater>();
          begin(t + 3, la0, lb0, ls0);
          rest(t + 1, la1, lb1, ls1, live);
          arrived<0>();
          rest(t + 2, la2, lb2, ls2, live);
          rest(t + 3, la0, lb0, ls0, live);
        } else {
          for (; t + 1 < whole; t += 2) {
            arrived<0>();
            begin(t + 1, la1, lb1, ls1);
            if constexpr (kLive) {
              step(la0, lb0, ls0);
            }
            arrived<0>();
            begin(t + 2, la0, lb0, ls0);
            if constexpr (kLive) {
              step(la1, lb1, ls1);
            }
          }
          // at most one whole block and two edges are left
          arrived<0>();
          begin(t + 1, la1, lb1, ls1);
          rest(t, la0, lb0, ls0, live);
          arrived<0>();
          begin(t + 2, la0, lb0, ls0);
          rest(t + 1, la1, lb1, ls1, live);
          arrived<0>();
          rest(t + 2, la0, lb0, ls0, live);
        }
        arrived<0>();
      };
      if (live) {
        all(std::true_type{});
      } else {
        all(std::false_type{});
      }
    }
    // the block in which the rows end, and rows that begin on odd borders
#pragma unroll 1
    for (int kb = direct; kb < last; kb++) {
      const int64_t k = static_cast<int64_t>(kb) * kQuant;
      __syncthreads();
      a.loadMasked(k, la0);
      b.loadMasked(k, lb0);
      s.load(kb, ls0);
      __syncthreads();
      if (live) {
        step(la0, lb0, ls0);
      }
    }
  }
};

template <typename O, bool kWeightGrad, int TM, int TN, int WM, int WN, int S>
__device__ inline void
computeTile(const Job& job, int64_t n, bool stream, O* __restrict__ out) {
  Product<O, kWeightGrad, TM, TN, WM, WN, S> p(job, n);
  p.run();
  p.write(out, stream);
}

template <typename O, int TM, int TN, int WM, int WN, int S = 3>
__global__ __launch_bounds__(WM * WN * kWave, S == 3 ? WM * WN / 4 : 2) void
matmulKernel(ProductShape p, O* __restrict__ out) {
  using T = Tile<TM, TN, WM, WN>;
  TileAt at;
  if (!tileAt(countTiles(p, T::kM), p.tilesN, at)) {
    return;
  }
  const RowTile tile = findTile(p, at.m, T::kM);
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
  job.n0 = static_cast<int64_t>(at.n) * T::kN;
  job.k0 = 0;
  job.k1 = p.inner;
  if (p.offsets != nullptr && tile.of >= p.experts) {
    job.k1 = 0; // no expert's rows: zeros
  } else {
    job.b.p += tile.of * p.bExpertStride;
    job.bScale += tile.of * ((p.n + kQuant - 1) / kQuant) * job.blocks;
  }
  computeTile<O, false, TM, TN, WM, WN, S>(job, p.n, p.stream, out);
}

// Few rows: the weights are read once and multiplied by few bytes, so what
// counts is how many of them are on their way. A workgroup takes 16 columns;
// its kWaves waves part the inner dimension, load their fragments from memory
// as the 16 x 16 instruction wants them (16 rows of 128 bytes, whole lines)
// and add their results up in LDS, in the order of the waves. An expert's
// rows are taken MT * 16 at a time.
template <typename O, int MT, int kWaves>
__global__ __launch_bounds__(kWaves * kWave) void fewRowsKernel(
    ProductShape p,
    O* __restrict__ out) {
  constexpr bool kExact = kExactSums<O>;
  constexpr int kAhead = MT == 1 ? 4 : 2; // blocks on their way
  __shared__ float4 partial[kWaves][MT][kWave];
  const int lane = threadIdx.x % kWave;
  const int wave = uniform(static_cast<int>(threadIdx.x / kWave));
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int e = blockIdx.y;
  int64_t begin = 0;
  int64_t end = p.m;
  if (p.offsets != nullptr) {
    rowsOf(p, e, begin, end);
  }
  const bool whole = p.n % 4 == 0;
  if (p.offsets != nullptr && e >= p.experts) { // no expert's: zeros
    const float zero[4] = {0, 0, 0, 0};
    for (int64_t i = threadIdx.x; i < (end - begin) * 4;
         i += kWaves * kWave) {
      store4(out + (begin + i / 4) * p.n, n0 + i % 4 * 4, p.n, zero, whole);
    }
    return;
  }
  const int blocks = static_cast<int>((p.inner + kQuant - 1) / kQuant);
  const Operand a{p.a, p.aStride, p.m, p.inner, true};
  const Operand b{
      p.b + e * p.bExpertStride, p.bStride, p.n, p.inner, true};
  const int64_t n = n0 + lane % 16 < p.n ? n0 + lane % 16 : p.n - 1;
  const uint8_t* bScale = p.bScale +
      (e * ((p.n + kQuant - 1) / kQuant) + n0 / kQuant) * blocks;
  const auto load = [&](const Operand& o, int64_t row, int kb, uint4* v) {
    const int64_t k =
        static_cast<int64_t>(kb) * kQuant + lane / 16 * 32;
    if (static_cast<int64_t>(kb + 1) * kQuant <= p.inner) {
      const auto* from =
          reinterpret_cast<const uint4*>(o.p + row * o.stride + k);
      v[0] = from[0];
      v[1] = from[1];
    } else {
      v[0] = load16(o, row, k, 0, p.inner);
      v[1] = load16(o, row, k + 16, 0, p.inner);
    }
  };
  for (int64_t m0 = begin; m0 < end; m0 += MT * 16) {
    Float4 acc[MT];
    int64_t m[MT];
#pragma unroll
    for (int j = 0; j < MT; j++) {
      acc[j] = 0.0f;
      const int64_t r = m0 + j * 16 + lane % 16;
      m[j] = r < end ? r : end - 1;
    }
    for (int kb0 = wave; kb0 < blocks; kb0 += kWaves * kAhead) {
      uint4 vb[kAhead][2];
      uint4 va[kAhead][MT][2];
      int sb[kAhead];
      int sa[kAhead][MT];
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int kb = kb0 + u * kWaves;
        if (kb < blocks) {
          load(b, n, kb, vb[u]);
          sb[u] = bScale[kb];
#pragma unroll
          for (int j = 0; j < MT; j++) {
            load(a, m[j], kb, va[u][j]);
            sa[u][j] = p.aScale[m[j] * blocks + kb];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        if (kb0 + u * kWaves < blocks) {
          Fragment<kExact> fb;
          fb.set(vb[u][0], vb[u][1], sb[u]);
#pragma unroll
          for (int j = 0; j < MT; j++) {
            Fragment<kExact> fa;
            fa.set(va[u][j][0], va[u][j][1], sa[u][j]);
            acc[j] = multiply(fb, fa, acc[j]);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < MT; j++) {
      partial[wave][j][lane] =
          make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < MT * kWave; i += kWaves * kWave) {
      const int j = i / kWave;
      const int l = i % kWave;
      float v[4] = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float4 f = partial[w][j][l];
        v[0] += f.x;
        v[1] += f.y;
        v[2] += f.z;
        v[3] += f.w;
      }
      const int64_t r = m0 + j * 16 + l % 16;
      if (r < end) {
        store4(out + r * p.n, n0 + l / 16 * 4, p.n, v, whole);
      }
    }
    __syncthreads();
  }
}

// A weight gradient's tiles take as long as their expert has rows, so that
// dies with experts of their own would end one after the other. An expert's
// tiles, if they are enough, are parted in eight or, with many experts, in
// four, and the dies take the parts in turn. Ragged rows, 16384 in all, whole
// experts and parts, in us: 4 experts of 4096 x 2048 274 / 244, 8 of 1408 x
// 2048 134 / 103; 16 of 4096 x 2048 411 to 485 / 396 to 411, bf16 273 to 347 /
// 276 to 288, 32 of 2048 x 1408 188 to 203 / 198 to 201, bf16 121 to 131 / 116
// to 120, 64 of 1024 x 2048 242 to 250 / 224 to 226.
__host__ __device__ inline int partsOf(int64_t tiles, int experts) {
  return tiles < kDies * kBand ? 0 : (experts < 2 * kDies ? kDies : kDies / 2);
}

int64_t weightTiles(int64_t tiles, int experts) {
  const int parts = partsOf(tiles, experts);
  if (parts == 0) {
    return tiles * experts;
  }
  const int64_t units =
      (static_cast<int64_t>(experts) * parts + kDies - 1) / kDies * kDies;
  return (tiles + parts - 1) / parts * units;
}

// False: fewer tiles than workgroups.
__device__ inline bool
weightTileAt(const ProductShape& p, int tilesM, int& e, TileAt& at) {
  const int64_t tiles = static_cast<int64_t>(tilesM) * p.tilesN;
  const int parts = partsOf(tiles, p.experts);
  if (parts == 0) {
    if (!tileAt(tilesM * p.experts, p.tilesN, at)) {
      return false;
    }
    e = at.m / tilesM;
    at.m %= tilesM;
    return true;
  }
  const int each = static_cast<int>((tiles + parts - 1) / parts);
  const int id = blockIdx.x / kDies;
  const int unit = id / each * kDies + blockIdx.x % kDies;
  e = unit / parts;
  const int part = unit % parts;
  const int64_t in = tiles * part / parts + id % each;
  if (e >= p.experts || in >= tiles * (part + 1) / parts) {
    return false;
  }
  at = inBands(in, tilesM, p.tilesN);
  return true;
}

template <typename O, int TM, int TN, int WM, int WN, int S = 3>
__global__ __launch_bounds__(WM * WN * kWave, S == 3 ? WM * WN / 4 : 2) void
weightGradKernel(ProductShape p, O* __restrict__ out) {
  using T = Tile<TM, TN, WM, WN>;
  const int tilesM = static_cast<int>((p.m + T::kM - 1) / T::kM);
  TileAt at;
  int e;
  if (!weightTileAt(p, tilesM, e, at)) {
    return;
  }
  Job job;
  job.a = Operand{p.a, p.aStride, p.m, p.inner, p.aWhole};
  job.b = Operand{p.b, p.bStride, p.n, p.inner, p.bWhole};
  job.aScale = p.aScale;
  job.bScale = p.bScale;
  job.blocks = (p.inner + kQuant - 1) / kQuant;
  job.m0 = static_cast<int64_t>(at.m) * T::kM;
  job.mEnd = job.m0 + T::kM < p.m ? job.m0 + T::kM : p.m;
  job.n0 = static_cast<int64_t>(at.n) * T::kN;
  job.k0 = 0;
  job.k1 = p.inner;
  if (p.offsets != nullptr) {
    job.k0 = clampOffset(p.offsets, e, p.inner);
    job.k1 = clampOffset(p.offsets, e + 1, p.inner);
  }
  computeTile<O, true, TM, TN, WM, WN, S>(
      job, p.n, p.stream, out + e * p.m * p.n);
}

// Large tiles read each operand's bytes less often, small ones are more of
// them: the largest is taken of which there are enough, most of the 256
// compute units having one. Measured for bf16 results, in us:
//                       128 x 256  128 x 128  64 x 128  64 x 64
//   8192 x 8192 x 8192     478       590        652      864
//   1024 x 4096 x 4096      28.7      22.0      24.8     30.6
//    512 x 4096 x 4096      26.5      19.3      14.6     16.7
//    256 x 4096 x 4096      25.4      18.2      11.9      9.8
//   1024 x 2048 x 2048      16.1      12.1       9.0      9.8
// weight gradient of 16384 rows, 2048 x 2048 and 1024 x 1024:
//                          139        92.8     108.9    136.1
//                          136        86.9      57.1     39.2
// Wider ones still, for bf16 results: 256 x 256 424 for the first of these,
// for 32 experts 16384 x 4096 x 4096 318 against 356 us with 128 x 256, if
// experts have rows for them (each has a part of a tile that is empty).
using WideTile = Tile<2, 4, 4, 2>;
constexpr int64_t kWideRows = 128;
using LargeTile = Tile<2, 2, 2, 4>;
using SmallTile = Tile<2, 2, 2, 2>;
using HalfTile = Tile<1, 2, 2, 2>;
using QuarterTile = Tile<1, 1, 2, 2>;
constexpr int64_t kEnough = 192;
// A weight gradient of experts with few rows is done with a tile after a few
// steps: two workgroups with small tiles on a compute unit, with two stages of
// LDS each, store and multiply at the same time. 16 experts, 16384 x 4096 x
// 2048 (about eight steps): 367 us against 414 with the large tile for fp32
// results, 250 / 290 for bf16; 4 experts, some 32 steps, are even.
constexpr int kShort = 32;
// So are products with fp32 or fp16 results and a short inner dimension: 8192 x
// 4096 x 512 48 us against 50, 8741 x 4096 x 512 of 8 experts 62 / 72, 16384 x
// 2048 x 1024 of 16 84 / 95, 8192 x 8192 x 2048 244 / 255 (279 on inputs that
// alternate); from there on even.
constexpr int kShortInner = 16;

// Tiles of rows, at most: every expert's last one may be a part of one, and
// so may those of the rows of no expert, before the first and behind the last.
template <typename T>
int64_t tilesOf(T, const ProductShape& p, bool grouped) {
  return grouped ? p.m / T::kM + std::min<int64_t>(p.experts + 2, p.m)
                 : (p.m + T::kM - 1) / T::kM;
}

// How many times 16 rows fewRowsKernel takes at a time, 0 where tiles are
// better. Measured by 8192 x 4096, this kernel and tiles in us, for bf16
// results: 1 row 7 / 10.4, 4 rows 8.2 / 10.2, 16 rows 10.8 / 10.6; for fp32
// (and fp16) ones, whose tiles take longer: 16 rows 13.6 / 15.2, 32 rows 18.1 /
// 15.4 (by 4096 x 4096 10.4 / 15.5).
// Of several experts each has workgroups for all of its columns, without rows
// too, and with many of them those cost what the others save: from some 4096 on
// (64 experts with 1024 columns, 16 with 4096), for one or two rows from 8192.
// 4 rows, bf16 and fp32: 32 experts of 1024 x 4096 8.3 / 8.4 and 8.6 / 15.3, 64
// of them 9.9 / 8.7 and 11.2 / 15.7, 128 of them 12.0 / 9.8 and 17.7 / 16.7; 16
// experts of 4096 x 2048 8.1 / 8.2 and 9.5 / 10.5, 32 of them 9.7 / 8.1 and
// 11.2 / 10.4. 1 row: 32 of those 5.1 / 6.4 and 5.7 / 9.9, 64 of them 8.0 / 6.8
// and 8.6 / 10.1. 8 rows: bf16, 8 experts of 1024 x 4096 7.6 / 8.5, 16 of 4096 x
// 2048 13.7 / 13.7; fp32, 32 of 4096 x 2048 18.8 / 15.7.
constexpr int64_t kFewWorkgroups = 4096;

int fewRows(const ProductShape& p, bool grouped, bool exact) {
  if (!p.aWhole || !p.bWhole) {
    return 0;
  }
  if (grouped) {
    const int64_t most = p.m <= 2 ? 2 * kFewWorkgroups : kFewWorkgroups;
    return p.m <= (exact ? 4 : 8) && p.experts * ((p.n + 15) / 16) <= most
        ? 1
        : 0;
  }
  if (exact) {
    return p.m <= 16 ? 1 : p.m <= 32 ? 2 : 0;
  }
  return p.m <= 8 ? 1 : 0;
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
  GA_ENFORCE_LT(p.experts, 65534);
  GA_ENFORCE_GE(p.aStride, 0);
  GA_ENFORCE_GE(p.bStride, 0);
}

} // namespace

namespace {

QuantShape checkQuantize(
    int64_t rowStride,
    int64_t colStride,
    int64_t rows,
    int64_t cols,
    const void* q,
    int64_t qStride) {
  GA_ENFORCE_GE(rows, 0);
  GA_ENFORCE_GE(cols, 0);
  GA_ENFORCE_GE(qStride, cols);
  GA_ENFORCE_EQ(qStride % 16, 0);
  GA_ENFORCE(aligned16(q), "quantize_fp8: q must begin on 16 bytes");
  const int64_t blocks = (cols + kQuant - 1) / kQuant;
  GA_ENFORCE_LE(blocks, 65535);
  GA_ENFORCE_LE(qStride, blocks * kQuant);
  return QuantShape{rowStride, colStride, rows, cols, qStride};
}

} // namespace

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
    hipStream_t stream) {
  const QuantShape p =
      checkQuantize(rowStride, colStride, rows, cols, q, qStride);
  if (rows == 0 || cols == 0) {
    return;
  }
  DeviceGuard guard(device);
  dispatchFloat(dtype, "quantize_fp8", [&](auto t) {
    using T = decltype(t);
    const auto go = [&](auto kernel, dim3 grid) {
      hipLaunchKernelGGL(
          kernel, grid, dim3(256), 0, stream, static_cast<const T*>(x),
          static_cast<uint8_t*>(q), static_cast<uint8_t*>(scales), p);
    };
    if (colStride == 1) {
      const int64_t lanes =
          rows * ((qStride + kQuant - 1) / kQuant * 8);
      const dim3 grid(groupsOf((lanes + 255) / 256, 256));
      if (aligned16(x) && rowStride % Vec16<T>::kSize == 0) {
        go(quantizeRowsKernel<T, true>, grid);
      } else {
        go(quantizeRowsKernel<T, false>, grid);
      }
    } else {
      constexpr int kRows = 16 * Vec16<T>::kSize;
      const dim3 grid(
          groupsOf((rows + kRows - 1) / kRows, 256),
          static_cast<unsigned>((cols + kQuant - 1) / kQuant));
      if (rowStride == 1 && aligned16(x) &&
          colStride % Vec16<T>::kSize == 0) {
        go(quantizeColumnsKernel<T, true>, grid);
      } else {
        go(quantizeColumnsKernel<T, false>, grid);
      }
    }
  });
  GA_HIP_CHECK(hipGetLastError());
}

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
    hipStream_t stream) {
  QuantTileShape p;
  p.m = checkQuantize(rowStride, colStride, rows, cols, q, qStride);
  GA_ENFORCE_GE(experts, 0);
  if (experts == 0 || rows == 0 || cols == 0) {
    return;
  }
  const int64_t rowTiles = (rows + kQuant - 1) / kQuant;
  GA_ENFORCE_LE(rowTiles, INT32_MAX);
  GA_ENFORCE_LE(experts, INT32_MAX);
  p.rowTiles = static_cast<int>(rowTiles);
  p.expertStride = expertStride;
  DeviceGuard guard(device);
  const dim3 grid(
      groupsOf(experts * rowTiles, 256),
      static_cast<unsigned>((cols + kQuant - 1) / kQuant));
  dispatchFloat(dtype, "quantize_fp8", [&](auto t) {
    using T = decltype(t);
    constexpr int kSize = Vec16<T>::kSize;
    const auto go = [&](auto kernel) {
      hipLaunchKernelGGL(
          kernel, grid, dim3(256), 0, stream, static_cast<const T*>(x),
          static_cast<uint8_t*>(q), static_cast<uint8_t*>(scales), p);
    };
    const bool whole = aligned16(x) && expertStride % kSize == 0;
    if (whole && colStride == 1 && rowStride % kSize == 0) {
      go(quantizeTilesKernel<T, Order::kRows>);
    } else if (whole && rowStride == 1 && colStride % kSize == 0) {
      go(quantizeTilesKernel<T, Order::kColumns>);
    } else {
      go(quantizeTilesKernel<T, Order::kAny>);
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
  GA_ENFORCE(aligned16(a.out), "fp8_matmul: out must begin on 16 bytes");
  if (p.m == 0) {
    return;
  }
  DeviceGuard guard(device);
  p.aWhole = whole16(p.a, p.aStride);
  p.bWhole = whole16(p.b, p.bStride) && p.bExpertStride % 16 == 0;
  dispatchFloat(a.dtype, "fp8_matmul", [&](auto t) {
    using O = decltype(t);
    p.stream = p.m * p.n * static_cast<int64_t>(sizeof(O)) >= kStreamFrom;
    auto go = [&](auto kernel, auto tile) {
      using T = decltype(tile);
      p.tilesN = static_cast<int>((p.n + T::kN - 1) / T::kN);
      const int64_t tilesM = tilesOf(tile, p, a.offsets != nullptr);
      hipLaunchKernelGGL(
          kernel, dim3(gridOf(tilesM * p.tilesN, T::kThreads)),
          dim3(T::kThreads), 0, stream, p, static_cast<O*>(a.out));
    };
    const auto tiles = [&](auto tile) {
      return tilesOf(tile, p, a.offsets != nullptr) *
          ((p.n + decltype(tile)::kN - 1) / decltype(tile)::kN);
    };
    const int few = fewRows(p, a.offsets != nullptr, kExactSums<O>);
    if (few != 0) {
      const auto goFew = [&](auto rows, auto waves) {
        constexpr int kRows = decltype(rows)::value;
        constexpr int kWaves = decltype(waves)::value;
        const dim3 grid(
            groupsOf((p.n + 15) / 16, kWaves * kWave),
            a.offsets != nullptr ? p.experts + 2 : 1);
        hipLaunchKernelGGL(
            (fewRowsKernel<O, kRows, kWaves>), grid, dim3(kWaves * kWave), 0,
            stream, p, static_cast<O*>(a.out));
      };
      // Eight waves where each still has four blocks.
      const auto goWaves = [&](auto rows) {
        if (p.inner >= 32 * kQuant) {
          goFew(rows, std::integral_constant<int, 8>{});
        } else {
          goFew(rows, std::integral_constant<int, 4>{});
        }
      };
      if constexpr (kExactSums<O>) {
        if (few == 2) {
          goWaves(std::integral_constant<int, 2>{});
          return;
        }
      }
      goWaves(std::integral_constant<int, 1>{});
      return;
    }
    if constexpr (!kExactSums<O>) {
      if (tiles(WideTile{}) >= kEnough && p.m >= kWideRows * p.experts) {
        go(matmulKernel<O, 2, 4, 4, 2, kWideStages>, WideTile{});
        return;
      }
    }
    if constexpr (kExactSums<O>) {
      if (tiles(LargeTile{}) >= kEnough && p.inner <= kShortInner * kQuant) {
        go(matmulKernel<O, 2, 2, 2, 2, 2>, SmallTile{});
        return;
      }
    }
    if (tiles(LargeTile{}) >= kEnough) {
      go(matmulKernel<O, 2, 2, 2, 4>, LargeTile{});
    } else if (tiles(SmallTile{}) >= kEnough) {
      go(matmulKernel<O, 2, 2, 2, 2>, SmallTile{});
    } else if (tiles(HalfTile{}) >= kEnough) {
      go(matmulKernel<O, 1, 2, 2, 2>, HalfTile{});
    } else {
      go(matmulKernel<O, 1, 1, 2, 2>, QuarterTile{});
    }
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
  GA_ENFORCE(
      aligned16(a.out), "fp8_weight_grad: out must begin on 16 bytes");
  DeviceGuard guard(device);
  p.aWhole = whole16(p.a, p.aStride);
  p.bWhole = whole16(p.b, p.bStride);
  dispatchFloat(a.dtype, "fp8_weight_grad", [&](auto t) {
    using O = decltype(t);
    p.stream = p.experts * p.m * p.n * static_cast<int64_t>(sizeof(O)) >=
        kStreamFrom;
    auto go = [&](auto kernel, auto tile) {
      using T = decltype(tile);
      p.tilesN = static_cast<int>((p.n + T::kN - 1) / T::kN);
      const int64_t tiles =
          weightTiles((p.m + T::kM - 1) / T::kM * p.tilesN, p.experts);
      hipLaunchKernelGGL(
          kernel, dim3(gridOf(tiles, T::kThreads)), dim3(T::kThreads), 0,
          stream, p, static_cast<O*>(a.out));
    };
    const auto tiles = [&](auto tile) {
      using T = decltype(tile);
      return (p.m + T::kM - 1) / T::kM * ((p.n + T::kN - 1) / T::kN) *
          p.experts;
    };
    if (tiles(LargeTile{}) >= kEnough &&
        p.inner / p.experts < kShort * kQuant) {
      go(weightGradKernel<O, 2, 2, 2, 2, 2>, SmallTile{});
    } else if (tiles(LargeTile{}) >= kEnough) {
      go(weightGradKernel<O, 2, 2, 2, 4>, LargeTile{});
    } else if (tiles(SmallTile{}) >= kEnough) {
      go(weightGradKernel<O, 2, 2, 2, 2>, SmallTile{});
    } else if (tiles(HalfTile{}) >= kEnough) {
      go(weightGradKernel<O, 1, 2, 2, 2>, HalfTile{});
    } else {
      go(weightGradKernel<O, 1, 1, 2, 2>, QuarterTile{});
    }
  });
  GA_HIP_CHECK(hipGetLastError());
}

} // namespace hip
} // namespace glooamd
