// Expert-parallel operators for gfx950: the router, the stable sort of token
// copies by expert, and the moves of rows into and out of that order.
// Interface and formulas: hip/experts.h.
#include <hip/hip_runtime.h>

#include <cfloat>

#include "hip/device_types.h"
#include "hip/experts.h"

namespace glooamd {
namespace hip {

namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4; // waves of a workgroup
constexpr int kBlock = kWave * kWaves;

// LDS written by some lanes of a wave and read by others of the same wave:
// the hardware keeps the order, this keeps the compiler's.
__device__ inline void waveFence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ inline double waveSum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v += __shfl_xor(v, o);
  }
  return v;
}

__device__ inline float waveMax(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v = fmaxf(v, __shfl_xor(v, o));
  }
  return v;
}

// --- router ------------------------------------------------------------------

struct RouteShape {
  int64_t stride;
  int64_t tokens;
  int experts;
  int k;
  int groups;
  int topkGroups;
  bool sigmoid;
  bool groupTop2;
  bool renormalize;
  float scale;
};

// One wave a token; a lane holds the experts lane, lane + 64, ... What is
// compared is held in 64 bits: the k chosen experts change with the last bit
// of a score, and 32 bits round different scores to the same one.
template <typename T, int kPer>
__global__ __launch_bounds__(kBlock) void routeKernel(
    const T* __restrict__ logits,
    const float* __restrict__ bias,
    float* __restrict__ weights,
    int32_t* __restrict__ ids,
    RouteShape p) {
  extern __shared__ double shared[];
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
  if (row >= p.tokens) {
    return;
  }
  const double none = -HUGE_VAL;
  const T* x = logits + row * p.stride;
  float logit[kPer];
  float top = -HUGE_VALF;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int e = i * kWave + lane;
    float v = e < p.experts ? toFloat(x[e]) : -HUGE_VALF;
    v = v > -HUGE_VALF ? fminf(v, FLT_MAX) : -HUGE_VALF; // NaN: no expert
    logit[i] = v;
    top = fmaxf(top, v);
  }
  double score[kPer];
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      score[i] = 1.0 / (1.0 + exp(-static_cast<double>(logit[i])));
    }
  } else {
    top = waveMax(top);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      score[i] = logit[i] > -HUGE_VALF
          ? exp(static_cast<double>(logit[i]) - static_cast<double>(top))
          : 0.0;
      sum += score[i];
    }
    sum = waveSum(sum);
    const double inv = sum > 0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      score[i] *= inv;
    }
  }
  // What ranks the experts; without a bias the logits rank them as the
  // scores would, and keep apart what the scores round together.
  double rank[kPer];
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int e = i * kWave + lane;
    double r = none;
    if (logit[i] > -HUGE_VALF) {
      r = bias == nullptr ? static_cast<double>(logit[i])
                          : score[i] + static_cast<double>(bias[e]);
      r = r > none ? r : none;
    }
    rank[i] = r;
  }
  if (p.groups > 1) {
    double* value = shared + static_cast<size_t>(wave) * p.experts;
    const bool two = p.groupTop2;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int e = i * kWave + lane;
      if (e < p.experts) {
        value[e] = two && bias == nullptr && rank[i] > none ? score[i]
                                                            : rank[i];
      }
    }
    waveFence();
    const int per = p.experts / p.groups;
    double of = none;
    if (lane < p.groups) {
      double first = none;
      double second = none;
      for (int i = 0; i < per; i++) {
        const double v = value[lane * per + i];
        second = v > first ? first : (v > second ? v : second);
        first = v > first ? v : first;
      }
      of = two && second > none ? first + second : first;
    }
    int before = 0;
    for (int g = 0; g < p.groups; g++) {
      const double other = __shfl(of, g);
      before += other > of || (other == of && g < lane);
    }
    const uint64_t kept =
        __ballot(lane < p.groups && before < p.topkGroups);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int e = i * kWave + lane;
      if (e < p.experts && !(kept >> (e / per) & 1)) {
        rank[i] = none;
      }
    }
  }
  int mine = -1;
  double w = 0;
  for (int j = 0; j < p.k; j++) {
    double best = none;
    int at = p.experts;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (rank[i] > best) {
        best = rank[i];
        at = i * kWave + lane;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double b = __shfl_xor(best, o);
      const int a = __shfl_xor(at, o);
      if (b > best || (b == best && a < at)) {
        best = b;
        at = a;
      }
    }
    if (!(best > none)) {
      break; // the same in every lane
    }
    double s = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (at == i * kWave + lane) {
        s = score[i];
        rank[i] = none;
      }
    }
    s = __shfl(s, at % kWave);
    if (lane == j) {
      mine = at;
      w = s;
    }
  }
  double scale = p.scale;
  if (p.renormalize) {
    const double sum = waveSum(w);
    scale = sum > 0 ? scale / sum : scale;
  }
  if (lane < p.k) {
    weights[row * p.k + lane] = static_cast<float>(w * scale);
    ids[row * p.k + lane] = mine;
  }
}

// One wave a token. Renormalised softmax weights are a softmax over the
// chosen logits, sigmoid scores have no sum over all experts: only softmax
// without renormalisation reads all of a token's logits.
template <typename T, int kPer>
__global__ __launch_bounds__(kBlock) void routeBackwardKernel(
    const T* __restrict__ logits,
    const int32_t* __restrict__ ids,
    const float* __restrict__ grad,
    T* __restrict__ dlogits,
    RouteShape p) {
  const int lane = threadIdx.x % kWave;
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
  if (row >= p.tokens) {
    return;
  }
  const T* x = logits + row * p.stride;
  int id = -1;
  double g = 0;
  float logit = -HUGE_VALF;
  if (lane < p.k) {
    id = ids[row * p.k + lane];
    if (id >= 0 && id < p.experts) {
      g = grad[row * p.k + lane];
      logit = fminf(toFloat(x[id]), FLT_MAX);
    } else {
      id = -1;
    }
  }
  double d = 0; // this lane's chosen expert's gradient
  double shift = 0; // softmax without renormalisation: sum of g * score
  float top = -HUGE_VALF;
  double inv = 0;
  float all[kPer];
  const bool dense = !p.sigmoid && !p.renormalize;
  if (dense) {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int e = i * kWave + lane;
      const float v = e < p.experts ? toFloat(x[e]) : -HUGE_VALF;
      all[i] = v > -HUGE_VALF ? fminf(v, FLT_MAX) : -HUGE_VALF;
      top = fmaxf(top, all[i]);
    }
    top = waveMax(top);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      sum += all[i] > -HUGE_VALF
          ? exp(static_cast<double>(all[i]) - static_cast<double>(top))
          : 0.0;
    }
    sum = waveSum(sum);
    inv = sum > 0 ? 1.0 / sum : 0.0;
    g *= p.scale;
    const double s = id >= 0
        ? exp(static_cast<double>(logit) - static_cast<double>(top)) * inv
        : 0.0;
    shift = waveSum(g * s);
    d = s * (g - shift);
  } else if (p.sigmoid) {
    const double s =
        id >= 0 ? 1.0 / (1.0 + exp(-static_cast<double>(logit))) : 0.0;
    if (p.renormalize) {
      const double sum = waveSum(s);
      const double over = sum > 0 ? 1.0 / sum : 1.0;
      g = (g - waveSum(g * s) * over) * over;
    }
    d = p.scale * g * s * (1.0 - s);
  } else {
    const float most = waveMax(logit);
    double s = id >= 0
        ? exp(static_cast<double>(logit) - static_cast<double>(most))
        : 0.0;
    const double sum = waveSum(s);
    s = sum > 0 ? s / sum : 0.0;
    d = p.scale * s * (g - waveSum(g * s));
  }
  double out[kPer];
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    out[i] = dense && all[i] > -HUGE_VALF
        ? -shift * inv *
            exp(static_cast<double>(all[i]) - static_cast<double>(top))
        : 0.0;
  }
  for (int j = 0; j < p.k; j++) {
    const int e = __shfl(id, j);
    const double v = __shfl(d, j);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (e == i * kWave + lane) {
        out[i] = v;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int e = i * kWave + lane;
    if (e < p.experts) {
      dlogits[row * p.experts + e] = fromFloat<T>(static_cast<float>(out[i]));
    }
  }
}

template <typename F>
void withPerLane(int experts, F&& f) {
  const int per = (experts + kWave - 1) / kWave;
  if (per <= 1) {
    f(std::integral_constant<int, 1>{});
  } else if (per <= 2) {
    f(std::integral_constant<int, 2>{});
  } else if (per <= 4) {
    f(std::integral_constant<int, 4>{});
  } else if (per <= 8) {
    f(std::integral_constant<int, 8>{});
  } else {
    f(std::integral_constant<int, 16>{});
  }
}

RouteShape checkRoute(const RouteArgs& a) {
  GA_ENFORCE_GE(a.tokens, 0);
  GA_ENFORCE_GT(a.experts, 0);
  GA_ENFORCE_LE(a.experts, kMaxExperts);
  GA_ENFORCE_GT(a.k, 0);
  GA_ENFORCE_LE(a.k, kMaxTopK);
  GA_ENFORCE_LE(a.k, a.experts);
  GA_ENFORCE_GT(a.groups, 0);
  GA_ENFORCE_LE(a.groups, kMaxExpertGroups);
  GA_ENFORCE_EQ(a.experts % a.groups, 0);
  GA_ENFORCE_GT(a.topkGroups, 0);
  GA_ENFORCE_LE(a.topkGroups, a.groups);
  GA_ENFORCE_GE(a.stride, 0);
  GA_ENFORCE_LE((a.tokens + kWaves - 1) / kWaves, INT32_MAX);
  return RouteShape{a.stride,    a.tokens,     a.experts, a.k,
                    a.groups,    a.topkGroups, a.sigmoid, a.groupTop2,
                    a.renormalize, a.scale};
}

// --- sort of token copies by expert ------------------------------------------

// A workgroup ranks the ids of one chunk. kPlanMaxBlocks bounds the counts
// that each workgroup adds up over the chunks before its own.
constexpr int kPlanMinChunk = 2048;
constexpr int kPlanMaxBlocks = 128;

struct PlanShape {
  int64_t n;
  int64_t chunk; // ids a workgroup, a multiple of kBlock
  int blocks;
  int experts;
};

PlanShape planShape(int64_t n, int experts) {
  int64_t chunk = (n + kPlanMaxBlocks - 1) / kPlanMaxBlocks;
  chunk = chunk < kPlanMinChunk ? kPlanMinChunk : chunk;
  chunk = (chunk + kBlock - 1) / kBlock * kBlock;
  const int64_t blocks = n == 0 ? 1 : (n + chunk - 1) / chunk;
  return PlanShape{n, chunk, static_cast<int>(blocks), experts};
}

__device__ inline int bucketOf(int32_t id, int experts) {
  return id < 0 || id >= experts ? experts : id;
}

// Counts of each wave's part of this workgroup's chunk, in LDS: [kWaves]
// [experts + 1]. Adding whole numbers: the order does not matter.
__device__ inline void countChunk(
    const int32_t* __restrict__ ids,
    const PlanShape& p,
    int64_t begin,
    int64_t end,
    int* counts) {
  const int buckets = p.experts + 1;
  for (int i = threadIdx.x; i < kWaves * buckets; i += kBlock) {
    counts[i] = 0;
  }
  __syncthreads();
  const int wave = threadIdx.x / kWave;
  const int64_t part = p.chunk / kWaves;
  const int64_t from = begin + wave * part;
  const int64_t to = from + part < end ? from + part : end;
  for (int64_t i = from + threadIdx.x % kWave; i < to; i += kWave) {
    atomicAdd(&counts[wave * buckets + bucketOf(ids[i], p.experts)], 1);
  }
  __syncthreads();
}

__global__ __launch_bounds__(kBlock) void planCountKernel(
    const int32_t* __restrict__ ids,
    int32_t* __restrict__ chunkCounts,
    PlanShape p) {
  extern __shared__ int counts[];
  const int buckets = p.experts + 1;
  const int64_t begin = blockIdx.x * p.chunk;
  const int64_t end = begin + p.chunk < p.n ? begin + p.chunk : p.n;
  countChunk(ids, p, begin, end, counts);
  for (int e = threadIdx.x; e < buckets; e += kBlock) {
    int sum = 0;
    for (int w = 0; w < kWaves; w++) {
      sum += counts[w * buckets + e];
    }
    chunkCounts[static_cast<int64_t>(blockIdx.x) * buckets + e] = sum;
  }
}

// Places of a chunk's ids: where its expert begins, the copies of earlier
// chunks, of earlier waves of this one, and of earlier lanes, which a wave
// finds by comparing the bits of its 64 buckets with ballots.
__global__ __launch_bounds__(kBlock) void planPlaceKernel(
    const int32_t* __restrict__ ids,
    const int32_t* __restrict__ chunkCounts,
    int32_t* __restrict__ position,
    int32_t* __restrict__ countsOut,
    int32_t* __restrict__ offsetsOut,
    PlanShape p,
    int bits) {
  extern __shared__ int counts[]; // [kWaves][buckets], then [buckets] twice
  const int buckets = p.experts + 1;
  int* total = counts + kWaves * buckets;
  int* start = total + buckets;
  const int64_t begin = blockIdx.x * p.chunk;
  const int64_t end = begin + p.chunk < p.n ? begin + p.chunk : p.n;
  countChunk(ids, p, begin, end, counts);
  for (int e = threadIdx.x; e < buckets; e += kBlock) {
    int sum = 0;
    int before = 0;
    if (p.blocks == 1) {
      for (int w = 0; w < kWaves; w++) {
        sum += counts[w * buckets + e];
      }
    } else {
      for (int b = 0; b < p.blocks; b++) {
        before = b == static_cast<int>(blockIdx.x) ? sum : before;
        sum += chunkCounts[static_cast<int64_t>(b) * buckets + e];
      }
    }
    total[e] = sum;
    start[e] = before;
  }
  __syncthreads();
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  if (wave == 0) { // where each expert begins: a scan over the totals
    int base = 0;
    for (int from = 0; from < buckets; from += kWave) {
      const int e = from + lane;
      const int own = e < buckets ? total[e] : 0;
      int sum = own;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int other = __shfl_up(sum, o);
        sum += lane >= o ? other : 0;
      }
      if (e < buckets) {
        const int at = base + sum - own;
        if (blockIdx.x == 0) {
          offsetsOut[e] = at;
          if (e < p.experts) {
            countsOut[e] = own;
          }
        }
        start[e] += at;
      }
      base += __shfl(sum, kWave - 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < buckets; e += kBlock) {
    int at = start[e];
    for (int w = 0; w < kWaves; w++) {
      const int own = counts[w * buckets + e];
      counts[w * buckets + e] = at;
      at += own;
    }
  }
  __syncthreads();
  int* next = counts + wave * buckets;
  const int64_t part = p.chunk / kWaves;
  const int64_t from = begin + wave * part;
  const int64_t to = from + part < end ? from + part : end;
  for (int64_t i = from; i < to; i += kWave) {
    const bool in = i + lane < to;
    const int bucket = in ? bucketOf(ids[i + lane], p.experts) : 0;
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; b++) {
      const uint64_t set = __ballot(bucket >> b & 1);
      same &= bucket >> b & 1 ? set : ~set;
    }
    const int before = __popcll(same & ((1ull << lane) - 1));
    int place = 0;
    if (in) {
      place = next[bucket] + before;
    }
    waveFence();
    if (in && before == 0) {
      next[bucket] += __popcll(same);
    }
    waveFence();
    if (in) {
      position[i + lane] = bucket == p.experts ? ~place : place;
    }
  }
}

// --- rows --------------------------------------------------------------------

struct RowsShape {
  int64_t tokens;
  int64_t hidden;
  int64_t rows; // tokens * k
  int k;
};

// A position as a row, or -1 where it is none of the rows (a plan's never
// is: this keeps a caller's wrong plan inside its buffers).
__device__ inline int64_t rowOf(int32_t position, int64_t rows) {
  const int64_t row = position < 0 ? ~position : position;
  return row < rows ? row : -1;
}

// A workgroup copies one part of a token's row to its k places: the row is
// read once. kVec elements a lane and step.
template <typename T, int kVec>
__global__ __launch_bounds__(kBlock) void packKernel(
    const T* __restrict__ x,
    int64_t xStride,
    const int32_t* __restrict__ position,
    T* __restrict__ rows,
    RowsShape p) {
  struct alignas(kVec * sizeof(T)) V {
    T v[kVec];
  };
  const int64_t t = blockIdx.x;
  const int64_t at =
      (static_cast<int64_t>(blockIdx.y) * kBlock + threadIdx.x) * kVec;
  if (at >= p.hidden) {
    return;
  }
  const V v = *reinterpret_cast<const V*>(x + t * xStride + at);
  V zero;
#pragma unroll
  for (int i = 0; i < kVec; i++) {
    zero.v[i] = fromFloat<T>(0.0f);
  }
  for (int j = 0; j < p.k; j++) {
    const int32_t to = position[t * p.k + j];
    const int64_t row = rowOf(to, p.rows);
    if (row >= 0) {
      *reinterpret_cast<V*>(rows + row * p.hidden + at) = to < 0 ? zero : v;
    }
  }
}

// Eight lanes quantise a block of 128 (16 elements each) and write it to its
// k places.
template <typename T, bool kVec>
__global__ __launch_bounds__(kBlock) void packFp8Kernel(
    const T* __restrict__ x,
    int64_t xStride,
    const int32_t* __restrict__ position,
    uint8_t* __restrict__ q,
    int64_t qStride,
    uint8_t* __restrict__ scales,
    RowsShape p) {
  constexpr int kEach = 16;
  const int64_t t = blockIdx.x;
  const int64_t at =
      (static_cast<int64_t>(blockIdx.y) * kBlock + threadIdx.x) * kEach;
  float v[kEach];
  uint32_t amax = 0;
  const T* from = x + t * xStride + at;
  if (kVec && at + kEach <= p.hidden) {
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
      v[i] = at + i < p.hidden ? toFloat(from[i]) : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kEach; i++) {
    const uint32_t bits = __float_as_uint(v[i]) & 0x7fffffffu;
    amax = bits > amax ? bits : amax;
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(amax, o);
    amax = other > amax ? other : amax;
  }
  if (at >= qStride) {
    return;
  }
  const uint32_t byte = fp8ScaleByte(amax);
  const float inv = fp8InverseScale(byte);
  uint4 packed;
  uint32_t* word = &packed.x;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    word[i] = fp8Pack4(v[i * 4] * inv, v[i * 4 + 1] * inv,
                       v[i * 4 + 2] * inv, v[i * 4 + 3] * inv);
  }
  const int64_t blocks = (p.hidden + 127) / 128;
  const bool first = at % 128 == 0 && at < p.hidden;
  for (int j = 0; j < p.k; j++) {
    const int32_t to = position[t * p.k + j];
    const int64_t row = rowOf(to, p.rows);
    if (row < 0) {
      continue;
    }
    *reinterpret_cast<uint4*>(q + row * qStride + at) =
        to < 0 ? make_uint4(0, 0, 0, 0) : packed;
    if (first) {
      scales[row * blocks + at / 128] =
          static_cast<uint8_t>(to < 0 ? 127u : byte);
    }
  }
}

// The weighted sum of a token's rows, added in the order of its copies in
// 32 bits and rounded once.
template <typename T, int kVec>
__global__ __launch_bounds__(kBlock) void combineKernel(
    const T* __restrict__ rows,
    int64_t rowStride,
    const int32_t* __restrict__ position,
    const float* __restrict__ weights,
    T* __restrict__ out,
    RowsShape p) {
  struct alignas(kVec * sizeof(T)) V {
    T v[kVec];
  };
  const int64_t t = blockIdx.x;
  const int64_t at =
      (static_cast<int64_t>(blockIdx.y) * kBlock + threadIdx.x) * kVec;
  if (at >= p.hidden) {
    return;
  }
  float sum[kVec] = {};
  for (int j = 0; j < p.k; j++) {
    const int32_t from = position[t * p.k + j];
    if (from < 0 || from >= p.rows) {
      continue;
    }
    const float w = weights == nullptr ? 1.0f : weights[t * p.k + j];
    const V v =
        *reinterpret_cast<const V*>(rows + from * rowStride + at);
#pragma unroll
    for (int i = 0; i < kVec; i++) {
      sum[i] = fmaf(w, toFloat(v.v[i]), sum[i]);
    }
  }
  V o;
#pragma unroll
  for (int i = 0; i < kVec; i++) {
    o.v[i] = fromFloat<T>(sum[i]);
  }
  *reinterpret_cast<V*>(out + t * p.hidden + at) = o;
}

// A workgroup takes a token: its gradient times each weight goes to the
// rows, its product with each row to the weights. kCopies copies share one
// pass over the gradient.
template <typename T, int kVec, int kCopies>
__global__ __launch_bounds__(kBlock) void combineBackwardKernel(
    const T* __restrict__ rows,
    int64_t rowStride,
    const int32_t* __restrict__ position,
    const float* __restrict__ weights,
    const T* __restrict__ grad,
    int64_t gradStride,
    T* __restrict__ drows,
    float* __restrict__ dweights,
    RowsShape p) {
  struct alignas(kVec * sizeof(T)) V {
    T v[kVec];
  };
  __shared__ float partial[kWaves][kCopies];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  for (int from = 0; from < p.k; from += kCopies) {
    float dot[kCopies] = {};
    int64_t row[kCopies];
    bool real[kCopies];
    float w[kCopies];
#pragma unroll
    for (int j = 0; j < kCopies; j++) {
      row[j] = -1;
      real[j] = false;
      w[j] = 0;
      if (from + j < p.k) {
        const int32_t to = position[t * p.k + from + j];
        row[j] = rowOf(to, p.rows);
        real[j] = to >= 0 && row[j] >= 0;
        w[j] = real[j] ? weights[t * p.k + from + j] : 0.0f;
      }
    }
    for (int64_t at = threadIdx.x * kVec; at < p.hidden;
         at += kBlock * kVec) {
      const V g = *reinterpret_cast<const V*>(grad + t * gradStride + at);
#pragma unroll
      for (int j = 0; j < kCopies; j++) {
        if (row[j] < 0) {
          continue;
        }
        V d;
        if (real[j]) {
          const V y = *reinterpret_cast<const V*>(
              rows + row[j] * rowStride + at);
#pragma unroll
          for (int i = 0; i < kVec; i++) {
            const float gv = toFloat(g.v[i]);
            dot[j] = fmaf(gv, toFloat(y.v[i]), dot[j]);
            d.v[i] = fromFloat<T>(w[j] * gv);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kVec; i++) {
            d.v[i] = fromFloat<T>(0.0f);
          }
        }
        *reinterpret_cast<V*>(drows + row[j] * p.hidden + at) = d;
      }
    }
#pragma unroll
    for (int j = 0; j < kCopies; j++) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        dot[j] += __shfl_xor(dot[j], o);
      }
    }
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < kCopies; j++) {
        partial[wave][j] = dot[j];
      }
    }
    __syncthreads();
    if (threadIdx.x < kCopies && from + static_cast<int>(threadIdx.x) < p.k) {
      float sum = 0;
#pragma unroll
      for (int i = 0; i < kWaves; i++) {
        sum += partial[i][threadIdx.x];
      }
      dweights[t * p.k + from + threadIdx.x] = sum;
    }
    __syncthreads();
  }
}

RowsShape checkRows(const ExpertRowsArgs& a) {
  GA_ENFORCE_GE(a.tokens, 0);
  GA_ENFORCE_GT(a.k, 0);
  GA_ENFORCE_GT(a.hidden, 0);
  GA_ENFORCE_LE(a.tokens, INT32_MAX / a.k);
  GA_ENFORCE_LE(a.hidden, 1 << 24);
  return RowsShape{a.tokens, a.hidden, a.tokens * a.k, a.k};
}

// 16 bytes a lane where every row begins and ends on such a border, else
// one element: a row that does not start on one cannot be loaded whole.
template <typename T>
bool wholeVectors(int64_t hidden, int64_t stride, int64_t stride2) {
  constexpr int kSize = Vec16<T>::kSize;
  return hidden % kSize == 0 && stride % kSize == 0 && stride2 % kSize == 0;
}

dim3 rowsGrid(const RowsShape& p, int64_t width, int each) {
  const int64_t span = static_cast<int64_t>(kBlock) * each;
  return dim3(
      static_cast<unsigned>(p.tokens),
      static_cast<unsigned>((width + span - 1) / span));
}

} // namespace

void launchRoute(const RouteArgs& a, int device, hipStream_t stream) {
  const RouteShape p = checkRoute(a);
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  const dim3 grid(static_cast<unsigned>((p.tokens + kWaves - 1) / kWaves));
  const size_t lds =
      p.groups > 1 ? sizeof(double) * kWaves * p.experts : 0;
  dispatchFloat(a.dtype, "route", [&](auto t) {
    using T = decltype(t);
    withPerLane(p.experts, [&](auto per) {
      hipLaunchKernelGGL(
          (routeKernel<T, decltype(per)::value>), grid, dim3(kBlock), lds,
          stream, static_cast<const T*>(a.logits), a.bias, a.weights, a.ids,
          p);
    });
  });
  GA_HIP_CHECK(hipGetLastError());
}

void launchRouteBackward(
    const RouteArgs& a,
    const float* grad,
    void* dlogits,
    int device,
    hipStream_t stream) {
  const RouteShape p = checkRoute(a);
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  const dim3 grid(static_cast<unsigned>((p.tokens + kWaves - 1) / kWaves));
  dispatchFloat(a.dtype, "route", [&](auto t) {
    using T = decltype(t);
    withPerLane(p.experts, [&](auto per) {
      hipLaunchKernelGGL(
          (routeBackwardKernel<T, decltype(per)::value>), grid, dim3(kBlock),
          0, stream, static_cast<const T*>(a.logits), a.ids, grad,
          static_cast<T*>(dlogits), p);
    });
  });
  GA_HIP_CHECK(hipGetLastError());
}

size_t expertPlanWorkspace(int64_t n, int experts) {
  const PlanShape p = planShape(n, experts);
  return p.blocks == 1 ? 0
                       : sizeof(int32_t) * p.blocks *
          static_cast<size_t>(experts + 1);
}

void launchExpertPlan(
    const int32_t* ids,
    int64_t n,
    int experts,
    int32_t* position,
    int32_t* counts,
    int32_t* offsets,
    void* workspace,
    size_t workspaceBytes,
    int device,
    hipStream_t stream) {
  GA_ENFORCE_GE(n, 0);
  GA_ENFORCE_LE(n, INT32_MAX);
  GA_ENFORCE_GT(experts, 0);
  GA_ENFORCE_LE(experts, kMaxExperts);
  GA_ENFORCE_GE(workspaceBytes, expertPlanWorkspace(n, experts));
  const PlanShape p = planShape(n, experts);
  DeviceGuard guard(device);
  const size_t buckets = experts + 1;
  int bits = 1;
  while ((1 << bits) < static_cast<int>(buckets)) {
    bits++;
  }
  auto* chunkCounts = static_cast<int32_t*>(workspace);
  if (p.blocks > 1) {
    hipLaunchKernelGGL(
        planCountKernel, dim3(p.blocks), dim3(kBlock),
        sizeof(int) * kWaves * buckets, stream, ids, chunkCounts, p);
    GA_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(
      planPlaceKernel, dim3(p.blocks), dim3(kBlock),
      sizeof(int) * (kWaves + 2) * buckets, stream, ids, chunkCounts,
      position, counts, offsets, p, bits);
  GA_HIP_CHECK(hipGetLastError());
}

void launchExpertPack(
    const ExpertRowsArgs& a,
    const void* x,
    int64_t xStride,
    void* rows,
    int device,
    hipStream_t stream) {
  const RowsShape p = checkRows(a);
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  dispatchFloat(a.dtype, "pack", [&](auto t) {
    using T = decltype(t);
    const bool whole = wholeVectors<T>(p.hidden, xStride, 0) &&
        aligned16(x) && aligned16(rows);
    auto go = [&](auto vec) {
      constexpr int kVec = decltype(vec)::value;
      hipLaunchKernelGGL(
          (packKernel<T, kVec>), rowsGrid(p, p.hidden, kVec), dim3(kBlock),
          0, stream, static_cast<const T*>(x), xStride, a.position,
          static_cast<T*>(rows), p);
    };
    if (whole) {
      go(std::integral_constant<int, Vec16<T>::kSize>{});
    } else {
      go(std::integral_constant<int, 1>{});
    }
  });
  GA_HIP_CHECK(hipGetLastError());
}

void launchExpertPackFp8(
    const ExpertRowsArgs& a,
    const void* x,
    int64_t xStride,
    void* q,
    int64_t qStride,
    void* scales,
    int device,
    hipStream_t stream) {
  const RowsShape p = checkRows(a);
  GA_ENFORCE_GE(qStride, p.hidden);
  GA_ENFORCE_EQ(qStride % 16, 0);
  GA_ENFORCE(aligned16(q), "pack_fp8: rows must begin on 16 bytes");
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  dispatchFloat(a.dtype, "pack_fp8", [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto vec) {
      hipLaunchKernelGGL(
          (packFp8Kernel<T, decltype(vec)::value>), rowsGrid(p, qStride, 16),
          dim3(kBlock), 0, stream, static_cast<const T*>(x), xStride,
          a.position, static_cast<uint8_t*>(q), qStride,
          static_cast<uint8_t*>(scales), p);
    };
    if (aligned16(x) && xStride % Vec16<T>::kSize == 0) {
      go(std::true_type{});
    } else {
      go(std::false_type{});
    }
  });
  GA_HIP_CHECK(hipGetLastError());
}

void launchExpertCombine(
    const ExpertRowsArgs& a,
    const void* rows,
    int64_t rowStride,
    const float* weights,
    void* out,
    int device,
    hipStream_t stream) {
  const RowsShape p = checkRows(a);
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  dispatchFloat(a.dtype, "combine", [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto vec) {
      constexpr int kVec = decltype(vec)::value;
      hipLaunchKernelGGL(
          (combineKernel<T, kVec>), rowsGrid(p, p.hidden, kVec),
          dim3(kBlock), 0, stream, static_cast<const T*>(rows), rowStride,
          a.position, weights, static_cast<T*>(out), p);
    };
    if (wholeVectors<T>(p.hidden, rowStride, 0) && aligned16(rows) &&
        aligned16(out)) {
      go(std::integral_constant<int, Vec16<T>::kSize>{});
    } else {
      go(std::integral_constant<int, 1>{});
    }
  });
  GA_HIP_CHECK(hipGetLastError());
}

void launchExpertCombineBackward(
    const ExpertRowsArgs& a,
    const void* rows,
    int64_t rowStride,
    const float* weights,
    const void* grad,
    int64_t gradStride,
    void* drows,
    float* dweights,
    int device,
    hipStream_t stream) {
  const RowsShape p = checkRows(a);
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  dispatchFloat(a.dtype, "combine", [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto vec) {
      constexpr int kVec = decltype(vec)::value;
      hipLaunchKernelGGL(
          (combineBackwardKernel<T, kVec, 8>),
          dim3(static_cast<unsigned>(p.tokens)), dim3(kBlock), 0, stream,
          static_cast<const T*>(rows), rowStride, a.position, weights,
          static_cast<const T*>(grad), gradStride, static_cast<T*>(drows),
          dweights, p);
    };
    if (wholeVectors<T>(p.hidden, rowStride, gradStride) &&
        aligned16(rows) && aligned16(grad) && aligned16(drows)) {
      go(std::integral_constant<int, Vec16<T>::kSize>{});
    } else {
      go(std::integral_constant<int, 1>{});
    }
  });
  GA_HIP_CHECK(hipGetLastError());
}

} // namespace hip
} // namespace glooamd
