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
  bool whole; // a token's logits fill the lanes and may be loaded as vectors
};

// A lane holds kPer adjacent experts, so that a token's logits come in wide
// loads and the lowest lane of several has the lowest number.
template <typename T, int kPer>
__device__ inline void loadLogits(
    const T* __restrict__ x,
    int experts,
    bool whole,
    float (&logit)[kPer]) {
  const int first = (threadIdx.x % kWave) * kPer;
  if (whole) {
    struct alignas(kPer * sizeof(T) < 16 ? kPer * sizeof(T) : 16) V {
      T v[kPer];
    };
    const V v = *reinterpret_cast<const V*>(x + first);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      logit[i] = toFloat(v.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      logit[i] = first + i < experts ? toFloat(x[first + i]) : -HUGE_VALF;
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; i++) { // NaN and -inf: no expert; -0 is 0
    logit[i] = logit[i] > -HUGE_VALF ? fminf(logit[i], FLT_MAX) + 0.0f
                                     : -HUGE_VALF;
  }
}

// Whole numbers in the order of the floats, all of them above 0.
__device__ inline uint32_t orderOf(float v) {
  const uint32_t bits = __float_as_uint(v);
  return bits ^ (bits >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ inline float valueOf(uint32_t order) {
  return __uint_as_float(
      order ^ (order >> 31 ? 0x80000000u : 0xffffffffu));
}

// The largest of a wave's numbers, in every lane: six steps within the
// vector unit, where shuffles would go through LDS.
__device__ inline uint32_t waveMaxOrder(uint32_t v) {
#define GA_DPP_MAX(ctrl)                                                    \
  {                                                                         \
    const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(   \
        0, static_cast<int>(v), ctrl, 0xf, 0xf, false));                    \
    v = v > o ? v : o;                                                      \
  }
  GA_DPP_MAX(0x111) // row_shr:1
  GA_DPP_MAX(0x112) // row_shr:2
  GA_DPP_MAX(0x114) // row_shr:4
  GA_DPP_MAX(0x118) // row_shr:8
  GA_DPP_MAX(0x142) // row_bcast:15
  GA_DPP_MAX(0x143) // row_bcast:31
#undef GA_DPP_MAX
  return static_cast<uint32_t>(
      __builtin_amdgcn_readlane(static_cast<int>(v), kWave - 1));
}

__device__ inline float laneOf(float v, int lane) {
  return __int_as_float(
      __builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ inline double laneOf(double v, int lane) {
  const int lo = __builtin_amdgcn_readlane(__double2loint(v), lane);
  const int hi = __builtin_amdgcn_readlane(__double2hiint(v), lane);
  return __hiloint2double(hi, lo);
}

// e^x to some 2^-51 of itself, in half the instructions of the library's
// function (64-bit ones take twice the time of others): x = n ln 2 + r with
// |r| <= ln 2 / 2, and the first 13 terms of e^r's series, whose rest is
// below r^13 / 13! < 2^-52. Beyond +-800 the result is infinite or 0 anyhow.
// N of them side by side share the constants' loads.
template <int N>
__device__ inline void expOf(double (&x)[N]) {
  constexpr double kTerms[] = {
      1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0,
      1.0 / 5040.0,     1.0 / 720.0,     1.0 / 120.0,    1.0 / 24.0,
      1.0 / 6.0,        0.5,             1.0,            1.0};
  int power[N];
  double e[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    const double v = fmin(fmax(x[i], -800.0), 800.0);
    const double n = rint(v * 1.4426950408889634);
    const double r = fma(n, -0.6931471805599453, v); // ln 2 to 53 bits,
    x[i] = fma(n, -2.3190468138462996e-17, r); // and what is left of it
    power[i] = static_cast<int>(n);
    e[i] = 1.0 / 479001600.0; // 12!
  }
#pragma unroll
  for (double term : kTerms) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      e[i] = fma(e[i], x[i], term);
    }
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    x[i] = ldexp(e[i], power[i]);
  }
}

__device__ inline double expOf(double x) {
  double v[1] = {x};
  expOf(v);
  return v[0];
}

// 1 / v for v >= 1, infinity included: the unit's estimate and two of
// Newton's steps, each of which doubles its bits.
__device__ inline double reciprocalOf(double v) {
  double y = __builtin_amdgcn_rcp(v);
  y = fma(fma(-v, y, 1.0), y, y);
  y = fma(fma(-v, y, 1.0), y, y);
  return v < HUGE_VAL ? y : 0.0;
}

__device__ inline double sigmoidOf(float logit) {
  return reciprocalOf(1.0 + expOf(-static_cast<double>(logit)));
}

// The two largest of two pairs.
__device__ inline void mergeTwo(
    double& first,
    double& second,
    double f,
    double s) {
  const double low = first > f ? f : first;
  first = first > f ? first : f;
  second = second > s ? second : s;
  second = second > low ? second : low;
}

// One wave a token. What decides is compared in 64 bits: the chosen experts
// change with the last bit of a score, and 32 bits round different scores to
// the same one. Without a bias the logits decide, as their scores would.
//
// The k best are taken one after the other by a 32-bit number in the scores'
// order, the largest of which six instructions find; where several scores
// share it, the 64-bit values are compared. Bound by the vector unit's some
// 700 instructions a token: 16381 tokens of 256 experts with bias and groups
// take 27 us, 8 tokens 6.3 us.
template <typename T, int kPer, bool kBias>
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
  const int first = lane * kPer;
  float logit[kPer];
  loadLogits<T, kPer>(logits + row * p.stride, p.experts, p.whole, logit);
  // scores are wanted of all experts, or of the chosen ones alone
  const bool two = p.groups > 1 && p.groupTop2;
  const bool all = kBias || two;
  const bool summed = !p.sigmoid && (all || !p.renormalize);
  double top = 0;
  double inv = 1;
  double score[kPer];
  if (summed) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint32_t o = orderOf(logit[i]);
      most = most > o ? most : o;
    }
    most = waveMaxOrder(most);
    top = valueOf(most);
  }
  if (summed || all) {
    // the arguments of what cannot be chosen give 0 either way
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const double v = logit[i];
      score[i] = p.sigmoid ? -v
          : logit[i] > -HUGE_VALF ? v - top : -HUGE_VAL;
    }
    expOf(score);
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        score[i] = reciprocalOf(1.0 + score[i]);
      }
    } else {
      double sum = 0;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        sum += score[i];
      }
      sum = waveSum(sum);
      inv = sum > 0 ? 1.0 / sum : 0.0;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        score[i] *= inv;
      }
    }
  }
  double rank[kPer]; // with a bias: score + bias
  uint32_t order[kPer]; // 0: cannot be chosen
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const bool alive = logit[i] > -HUGE_VALF;
    if (!kBias) {
      rank[i] = alive ? static_cast<double>(logit[i]) : none;
      order[i] = alive ? orderOf(logit[i]) : 0;
    } else {
      const double r =
          alive ? score[i] + static_cast<double>(bias[first + i]) : none;
      rank[i] = r > none ? r : none;
      order[i] = r > none ? orderOf(static_cast<float>(r)) : 0;
    }
  }
  if (p.groups > 1) {
    const int per = p.experts / p.groups;
    const int lanes = per / kPer; // of a group, where they are whole ones
    if (lanes * kPer == per && (lanes & (lanes - 1)) == 0) {
      double one = none;
      double next = none;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const double v = two && !kBias && order[i] != 0 ? score[i]
                                                                 : rank[i];
        mergeTwo(one, next, v, none);
      }
      for (int o = 1; o < lanes; o <<= 1) {
        mergeTwo(one, next, __shfl_xor(one, o), __shfl_xor(next, o));
      }
      const double of = two && next > none ? one + next : one;
      const int group = lane / lanes;
      int before = 0;
      for (int g = 0; g < p.groups; g++) {
        const double other = laneOf(of, g * lanes);
        before += other > of || (other == of && g < group);
      }
      if (before >= p.topkGroups) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
          order[i] = 0;
        }
      }
    } else {
      double* value = shared + static_cast<size_t>(wave) * p.experts;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (first + i < p.experts) {
          value[first + i] =
              two && !kBias && order[i] != 0 ? score[i] : rank[i];
        }
      }
      waveFence();
      double one = none;
      double next = none;
      if (lane < p.groups) {
        for (int i = 0; i < per; i++) {
          mergeTwo(one, next, value[lane * per + i], none);
        }
      }
      const double of = two && next > none ? one + next : one;
      int before = 0;
      for (int g = 0; g < p.groups; g++) {
        const double other = laneOf(of, g);
        before += other > of || (other == of && g < lane);
      }
      const uint64_t kept =
          __ballot(lane < p.groups && before < p.topkGroups);
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (first + i < p.experts && !(kept >> ((first + i) / per) & 1)) {
          order[i] = 0;
        }
      }
    }
  }
  int mine = -1;
  float chosen = -HUGE_VALF;
  for (int j = 0; j < p.k; j++) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      most = most > order[i] ? most : order[i];
    }
    const uint32_t best = waveMaxOrder(most);
    if (best == 0) {
      break; // none is left
    }
    // Who has it, as masks: what follows from them is the scalar unit's work.
    uint64_t have[kPer];
    uint64_t any = 0;
    int count = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      have[i] = __ballot(order[i] == best);
      any |= have[i];
      count += kBias ? __popcll(have[i]) : 0;
    }
    int winner = __ffsll(static_cast<unsigned long long>(any)) - 1;
    int at = 0;
#pragma unroll
    for (int i = kPer - 1; i >= 0; i--) {
      at = have[i] >> winner & 1 ? i : at;
    }
    if (kBias && count > 1) {
      double r = none;
      int own = 0;
#pragma unroll
      for (int i = kPer - 1; i >= 0; i--) {
        const bool is = order[i] == best && rank[i] >= r;
        own = is ? i : own;
        r = is ? rank[i] : r;
      }
      double highest = none;
      for (uint64_t rest = any; rest != 0; rest &= rest - 1) {
        const int of = __ffsll(static_cast<unsigned long long>(rest)) - 1;
        const double other = laneOf(r, of);
        winner = other > highest ? of : winner;
        highest = other > highest ? other : highest;
      }
      at = __builtin_amdgcn_readlane(own, winner);
    }
    const int expert = winner * kPer + at;
    float value = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (at == i) { // the same in every lane
        value = laneOf(logit[i], winner);
        order[i] = lane == winner ? 0 : order[i];
      }
    }
    if (lane == j) {
      mine = expert;
      chosen = value;
    }
  }
  // Renormalised softmax weights are a softmax over the chosen logits: below
  // their own largest one, since a bias may have kept the token's largest out,
  // and all of them may lie so far below that one that their scores are 0.
  // Without a bias the first one chosen is the largest.
  if (!p.sigmoid && p.renormalize) {
    top = kBias ? valueOf(waveMaxOrder(orderOf(chosen))) : laneOf(chosen, 0);
    inv = 1;
  }
  double w = 0;
  if (mine >= 0) {
    w = p.sigmoid ? sigmoidOf(chosen)
                  : expOf(static_cast<double>(chosen) - top) * inv;
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
  float d = 0; // this lane's chosen expert's gradient
  float out[kPer];
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    out[i] = 0;
  }
  if (p.sigmoid) {
    const double s = id >= 0 ? sigmoidOf(logit) : 0.0;
    if (p.renormalize) {
      const double sum = waveSum(s);
      const double over = sum > 0 ? 1.0 / sum : 1.0;
      g = (g - waveSum(g * s) * over) * over;
    }
    d = static_cast<float>(p.scale * g * s * (1.0 - s));
  } else if (p.renormalize) {
    const float most = waveMax(logit);
    double s = id >= 0
        ? expOf(static_cast<double>(logit) - static_cast<double>(most))
        : 0.0;
    const double sum = waveSum(s);
    s = sum > 0 ? s / sum : 0.0;
    d = static_cast<float>(p.scale * s * (g - waveSum(g * s)));
  } else {
    float all[kPer];
    loadLogits<T, kPer>(x, p.experts, p.whole, all);
    float top = -HUGE_VALF;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      top = fmaxf(top, all[i]);
    }
    top = waveMax(top);
    double score[kPer];
    double sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      score[i] = all[i] > -HUGE_VALF
          ? static_cast<double>(all[i]) - static_cast<double>(top)
          : -HUGE_VAL;
    }
    expOf(score);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      sum += score[i];
    }
    sum = waveSum(sum);
    const double inv = sum > 0 ? 1.0 / sum : 0.0;
    g *= p.scale;
    const double s = id >= 0
        ? expOf(static_cast<double>(logit) - static_cast<double>(top)) * inv
        : 0.0;
    const double shift = waveSum(g * s);
    d = static_cast<float>(s * (g - shift));
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      out[i] = static_cast<float>(-shift * inv * score[i]);
    }
  }
  const int first = lane * kPer;
  for (int j = 0; j < p.k; j++) {
    const int e = __builtin_amdgcn_readlane(id, j);
    const float v = laneOf(d, j);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      out[i] = e == first + i ? v : out[i];
    }
  }
  T* to = dlogits + row * p.experts + first;
  if (p.experts == kWave * kPer) {
    struct alignas(kPer * sizeof(T) < 16 ? kPer * sizeof(T) : 16) V {
      T v[kPer];
    };
    V v;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      v.v[i] = fromFloat<T>(out[i]);
    }
    *reinterpret_cast<V*>(to) = v;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (first + i < p.experts) {
        to[i] = fromFloat<T>(out[i]);
      }
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

template <typename T, int kPer>
bool wholeLogits(const RouteArgs& a) {
  constexpr size_t kBytes = kPer * sizeof(T) < 16 ? kPer * sizeof(T) : 16;
  return a.experts == kWave * kPer &&
      reinterpret_cast<uintptr_t>(a.logits) % kBytes == 0 &&
      a.stride * sizeof(T) % kBytes == 0;
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
  return RouteShape{a.stride,    a.tokens,     a.experts, a.k,
                    a.groups,    a.topkGroups, a.sigmoid, a.groupTop2,
                    a.renormalize, a.scale, false};
}

// --- sort of token copies by expert ------------------------------------------

// Two passes. In the first each workgroup ranks the ids of one chunk among
// the chunk's ids of the same expert and counts them; in the second it adds up
// the counts of the chunks before its own and where each expert begins. One
// chunk needs no second pass. Chunks are short, so that a small batch has many
// workgroups, and at most kPlanMaxBlocks, which bounds the counts that each
// adds up. 65536 ids of 64 experts: 11 us for both; 256 of 256: 4.3 us.
constexpr int kPlanWaves = 8;
constexpr int kPlanBlock = kPlanWaves * kWave;
constexpr int kPlanMinChunk = 1024;
constexpr int kPlanMaxBlocks = 128;

struct PlanShape {
  int64_t n;
  int64_t chunk; // ids a workgroup, a multiple of kPlanBlock
  int blocks;
  int experts;
  int bits; // of a bucket's number
};

PlanShape planShape(int64_t n, int experts) {
  int64_t chunk = (n + kPlanMaxBlocks - 1) / kPlanMaxBlocks;
  chunk = chunk < kPlanMinChunk ? kPlanMinChunk : chunk;
  chunk = (chunk + kPlanBlock - 1) / kPlanBlock * kPlanBlock;
  const int64_t blocks = n == 0 ? 1 : (n + chunk - 1) / chunk;
  int bits = 1;
  while ((1 << bits) < experts + 1) {
    bits++;
  }
  return PlanShape{n, chunk, static_cast<int>(blocks), experts, bits};
}

// The last bucket is the ids' that are no expert.
__device__ inline int bucketOf(int32_t id, int experts) {
  return id < 0 || id >= experts ? experts : id;
}

// Sums of what stands before each of `count` numbers in LDS, by the whole
// workgroup; `total` is of one wave's numbers each.
__device__ inline void
scanBuckets(int* values, int count, int* total) {
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  int base = 0;
  for (int from = 0; from < count; from += kPlanBlock) {
    const int at = from + threadIdx.x;
    const int own = at < count ? values[at] : 0;
    int sum = own;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int other = __shfl_up(sum, o);
      sum += lane >= o ? other : 0;
    }
    if (lane == kWave - 1) {
      total[wave] = sum;
    }
    __syncthreads();
    int before = base;
    int all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) {
      before += w < wave ? total[w] : 0;
      all += total[w];
    }
    if (at < count) {
      values[at] = before + sum - own;
    }
    base += all;
    __syncthreads();
  }
}

// Each wave takes a part of the chunk, 64 ids at a time; a lane's rank among
// equal ids is what the wave has counted, and the lanes before it that agree
// in all bits of the bucket's number.
__global__ __launch_bounds__(kPlanBlock) void planRankKernel(
    const int32_t* __restrict__ ids,
    int32_t* __restrict__ position,
    int32_t* __restrict__ chunkCounts,
    int32_t* __restrict__ countsOut,
    int32_t* __restrict__ offsetsOut,
    PlanShape p) {
  extern __shared__ int bucketSpace[]; // [kPlanWaves][buckets], [buckets]
  __shared__ int total[kPlanWaves];
  const int buckets = p.experts + 1;
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  int* counts = bucketSpace + wave * buckets;
  int* sums = bucketSpace + kPlanWaves * buckets;
  for (int i = threadIdx.x; i < kPlanWaves * buckets; i += kPlanBlock) {
    bucketSpace[i] = 0;
  }
  __syncthreads();
  const int64_t begin = blockIdx.x * p.chunk;
  const int64_t end = begin + p.chunk < p.n ? begin + p.chunk : p.n;
  const int64_t part = p.chunk / kPlanWaves;
  const int64_t from = begin + wave * part;
  const int64_t to = from + part < end ? from + part : end;
  for (int64_t i = from; i < to; i += kWave) {
    const bool in = i + lane < to;
    const int bucket = in ? bucketOf(ids[i + lane], p.experts) : 0;
    uint64_t same = __ballot(in);
    for (int b = 0; b < p.bits; b++) {
      const uint64_t set = __ballot(bucket >> b & 1);
      same &= bucket >> b & 1 ? set : ~set;
    }
    const int before = __popcll(same & ((1ull << lane) - 1));
    int rank = 0;
    if (in) {
      rank = counts[bucket] + before;
    }
    waveFence();
    if (in && before == 0) {
      counts[bucket] += __popcll(same);
    }
    waveFence();
    if (in) {
      position[i + lane] = rank;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < buckets; e += kPlanBlock) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; w++) {
      const int own = bucketSpace[w * buckets + e];
      bucketSpace[w * buckets + e] = sum;
      sum += own;
    }
    if (p.blocks > 1) {
      chunkCounts[static_cast<int64_t>(blockIdx.x) * buckets + e] = sum;
    } else {
      sums[e] = sum;
      if (e < p.experts) {
        countsOut[e] = sum;
      }
    }
  }
  __syncthreads();
  if (p.blocks == 1) {
    scanBuckets(sums, buckets, total);
    for (int e = threadIdx.x; e < buckets; e += kPlanBlock) {
      offsetsOut[e] = sums[e];
    }
  }
  for (int64_t i = from + lane; i < to; i += kWave) {
    const int bucket = bucketOf(ids[i], p.experts);
    int place = position[i] + counts[bucket];
    if (p.blocks == 1) {
      place += sums[bucket];
      place = bucket == p.experts ? ~place : place;
    }
    position[i] = place;
  }
}

__global__ __launch_bounds__(kPlanBlock) void planPlaceKernel(
    const int32_t* __restrict__ ids,
    const int32_t* __restrict__ chunkCounts,
    int32_t* __restrict__ position,
    int32_t* __restrict__ countsOut,
    int32_t* __restrict__ offsetsOut,
    PlanShape p) {
  extern __shared__ int bucketSpace[]; // [buckets] twice
  __shared__ int total[kPlanWaves];
  const int buckets = p.experts + 1;
  int* start = bucketSpace;
  int* earlier = bucketSpace + buckets;
  for (int e = threadIdx.x; e < buckets; e += kPlanBlock) {
    int sum = 0;
    int before = 0;
#pragma unroll 8
    for (int b = 0; b < p.blocks; b++) {
      before = b == static_cast<int>(blockIdx.x) ? sum : before;
      sum += chunkCounts[static_cast<int64_t>(b) * buckets + e];
    }
    start[e] = sum;
    earlier[e] = before;
    if (blockIdx.x == 0 && e < p.experts) {
      countsOut[e] = sum;
    }
  }
  __syncthreads();
  scanBuckets(start, buckets, total);
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < buckets; e += kPlanBlock) {
      offsetsOut[e] = start[e];
    }
  }
  const int64_t begin = blockIdx.x * p.chunk;
  const int64_t end = begin + p.chunk < p.n ? begin + p.chunk : p.n;
  for (int64_t i = begin + threadIdx.x; i < end; i += kPlanBlock) {
    const int bucket = bucketOf(ids[i], p.experts);
    const int place = position[i] + start[bucket] + earlier[bucket];
    position[i] = bucket == p.experts ? ~place : place;
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

// 2, 4 or 16 bytes as one register value, so that masking it takes no
// memory.
template <int kBytes>
struct RawOf;
template <>
struct RawOf<2> {
  using type = uint16_t;
};
template <>
struct RawOf<4> {
  using type = uint32_t;
};
template <>
struct RawOf<16> {
  using type = uint32_t __attribute__((ext_vector_type(4)));
};

template <bool kStream, typename V>
__device__ inline void store(V* to, V v) {
  if (kStream) {
    __builtin_nontemporal_store(v, to);
  } else {
    *to = v;
  }
}

// A workgroup copies one part of a token's row to its k places: the row is
// read once. kBytes a lane and step. Bound by memory: 16384 tokens of 4096
// bf16 to 4 places, 671 MB, take 126 us, 5.3 TB/s, what a copy reaches (204
// us with stores that stay in the caches).
template <int kBytes, bool kStream>
__global__ __launch_bounds__(kBlock) void packKernel(
    const char* __restrict__ x,
    int64_t xStride, // bytes
    const int32_t* __restrict__ position,
    char* __restrict__ rows,
    int64_t width, // bytes of a row
    RowsShape p) {
  using V = typename RawOf<kBytes>::type;
  const int64_t t = blockIdx.x;
  const int64_t at =
      (static_cast<int64_t>(blockIdx.y) * kBlock + threadIdx.x) * kBytes;
  if (at >= width) {
    return;
  }
  const V v = *reinterpret_cast<const V*>(x + t * xStride + at);
  const V zero = 0;
#pragma unroll 4
  for (int j = 0; j < p.k; j++) {
    const int32_t to = position[t * p.k + j];
    const int64_t row = rowOf(to, p.rows);
    if (row >= 0) {
      store<kStream>(
          reinterpret_cast<V*>(rows + row * width + at), to < 0 ? zero : v);
    }
  }
}

// Eight lanes quantise a block of 128 (16 elements each) and write it to its
// k places: a token is read and rounded once. 8190 tokens of 5120 bf16 to 8
// places, 430 MB: 69 us, 6.2 TB/s.
template <typename T, bool kVec, bool kStream>
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
  using V = typename RawOf<16>::type;
  V packed;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    packed[i] = fp8Pack4(v[i * 4] * inv, v[i * 4 + 1] * inv,
                       v[i * 4 + 2] * inv, v[i * 4 + 3] * inv);
  }
  const int64_t blocks = (p.hidden + 127) / 128;
  const bool first = at % 128 == 0 && at < p.hidden;
#pragma unroll 4
  for (int j = 0; j < p.k; j++) {
    const int32_t to = position[t * p.k + j];
    const int64_t row = rowOf(to, p.rows);
    if (row < 0) {
      continue;
    }
    const V zero = 0;
    store<kStream>(
        reinterpret_cast<V*>(q + row * qStride + at), to < 0 ? zero : packed);
    if (first) {
      scales[row * blocks + at / 128] =
          static_cast<uint8_t>(to < 0 ? 127u : byte);
    }
  }
}

// The weighted sum of a token's rows, added in the order of its copies in
// 32 bits and rounded once. Bound by memory: 16384 tokens of 4 rows of 4096
// bf16, 671 MB, take 123 to 135 us.
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
// pass over the gradient. Bound by memory: 16384 tokens of 4 rows of 4096
// bf16, 1.2 GB, take 229 us, 5.3 TB/s.
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
  GA_ENFORCE_LE(a.hidden, 1 << 23);
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
      groupsOf(p.tokens, kBlock),
      static_cast<unsigned>((width + span - 1) / span));
}

} // namespace

void launchRoute(const RouteArgs& a, int device, hipStream_t stream) {
  RouteShape p = checkRoute(a);
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  const dim3 grid(groupsOf((p.tokens + kWaves - 1) / kWaves, kBlock));
  const size_t lds =
      p.groups > 1 ? sizeof(double) * kWaves * p.experts : 0;
  dispatchFloat(a.dtype, "route", [&](auto t) {
    using T = decltype(t);
    withPerLane(p.experts, [&](auto per) {
      p.whole = wholeLogits<T, decltype(per)::value>(a);
      const auto go = [&](auto withBias) {
        hipLaunchKernelGGL(
            (routeKernel<T, decltype(per)::value, decltype(withBias)::value>),
            grid, dim3(kBlock), lds, stream, static_cast<const T*>(a.logits),
            a.bias, a.weights, a.ids, p);
      };
      if (a.bias != nullptr) {
        go(std::true_type{});
      } else {
        go(std::false_type{});
      }
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
  RouteShape p = checkRoute(a);
  GA_ENFORCE(
      aligned16(dlogits), "route: the gradient must begin on 16 bytes");
  if (p.tokens == 0) {
    return;
  }
  DeviceGuard guard(device);
  const dim3 grid(groupsOf((p.tokens + kWaves - 1) / kWaves, kBlock));
  dispatchFloat(a.dtype, "route", [&](auto t) {
    using T = decltype(t);
    withPerLane(p.experts, [&](auto per) {
      p.whole = wholeLogits<T, decltype(per)::value>(a);
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
  auto* chunkCounts = static_cast<int32_t*>(workspace);
  hipLaunchKernelGGL(
      planRankKernel, dim3(p.blocks), dim3(kPlanBlock),
      sizeof(int) * (kPlanWaves + 1) * buckets, stream, ids, position,
      chunkCounts, counts, offsets, p);
  GA_HIP_CHECK(hipGetLastError());
  if (p.blocks > 1) {
    hipLaunchKernelGGL(
        planPlaceKernel, dim3(p.blocks), dim3(kPlanBlock),
        sizeof(int) * 2 * buckets, stream, ids, chunkCounts, position,
        counts, offsets, p);
    GA_HIP_CHECK(hipGetLastError());
  }
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
    constexpr int kSize = sizeof(T);
    auto go = [&](auto bytes) {
      constexpr int kBytes = decltype(bytes)::value;
      const int64_t width = p.hidden * kSize;
      const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(
            kernel, rowsGrid(p, width, kBytes), dim3(kBlock), 0, stream,
            static_cast<const char*>(x), xStride * kSize, a.position,
            static_cast<char*>(rows), width, p);
      };
      if (p.rows * width >= kStreamFrom) {
        launch(packKernel<kBytes, true>);
      } else {
        launch(packKernel<kBytes, false>);
      }
    };
    if (wholeVectors<T>(p.hidden, xStride, 0) && aligned16(x) &&
        aligned16(rows)) {
      go(std::integral_constant<int, 16>{});
    } else {
      go(std::integral_constant<int, kSize>{});
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
      const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(
            kernel, rowsGrid(p, qStride, 16), dim3(kBlock), 0, stream,
            static_cast<const T*>(x), xStride, a.position,
            static_cast<uint8_t*>(q), qStride, static_cast<uint8_t*>(scales),
            p);
      };
      if (p.rows * qStride >= kStreamFrom) {
        launch(packFp8Kernel<T, decltype(vec)::value, true>);
      } else {
        launch(packFp8Kernel<T, decltype(vec)::value, false>);
      }
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
          dim3(groupsOf(p.tokens, kBlock)), dim3(kBlock), 0, stream,
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
