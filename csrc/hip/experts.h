// Launch interface of the expert-parallel operators (csrc/hip/experts.hip):
// routing, the sort of token copies by expert, and the moves of rows into
// and out of that order, which are an alltoallv's send and receive buffers.
// Host-compilable header: no device code. All launches are asynchronous on
// `stream` of `device`, check their arguments (EnforceNotMet) and leave the
// calling thread's current device as it was.
#pragma once

#include <cstddef>
#include <cstdint>

#include "collectives/reduce_fns.h"

struct ihipStream_t;
typedef struct ihipStream_t* hipStream_t;

namespace glooamd {
namespace hip {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 64;
constexpr int kMaxExpertGroups = 64;

struct RouteArgs {
  const void* logits = nullptr; // [tokens, experts], experts adjacent
  int64_t stride = 0; // elements from one token's logits to the next
  DType dtype = DType::F32; // F32, F16 or BF16
  const float* bias = nullptr; // [experts] or null
  int64_t tokens = 0;
  int experts = 0;
  int k = 0;
  bool sigmoid = false; // else softmax
  int groups = 1;
  int topkGroups = 1;
  bool groupTop2 = false; // a group's value: sum of its two best, else max
  bool renormalize = true;
  float scale = 1.0f;
  float* weights = nullptr; // [tokens, k]
  int32_t* ids = nullptr; // [tokens, k]
};
void launchRoute(const RouteArgs& args, int device, hipStream_t stream);

// dlogits [tokens, experts] (contiguous, the logits' type, begins on 16
// bytes) of `grad` [tokens, k]; args.ids are the forward pass's.
void launchRouteBackward(
    const RouteArgs& args,
    const float* grad,
    void* dlogits,
    int device,
    hipStream_t stream);

// Bytes of workspace that launchExpertPlan needs for n ids.
size_t expertPlanWorkspace(int64_t n, int experts);
// Stable sort of n ids by expert. An id outside [0, experts) stands behind
// all others, and its place p is told as ~p.
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
    hipStream_t stream);

struct ExpertRowsArgs {
  const int32_t* position = nullptr; // [tokens, k]
  int64_t tokens = 0;
  int k = 0;
  int64_t hidden = 0;
  DType dtype = DType::F32; // of tokens and rows: F32, F16 or BF16
};
// rows[position[t, j]] = x[t]; zeros where the position is negative.
void launchExpertPack(
    const ExpertRowsArgs& args,
    const void* x,
    int64_t xStride,
    void* rows,
    int device,
    hipStream_t stream);
// The same in e4m3 with a power of two (e8m0) for each 128 elements. q's
// rows are qStride bytes apart, a multiple of 16 that is at least hidden;
// the bytes between are zeros (NaN where the last block's are). scales: [tokens * k, ceil(hidden / 128)].
void launchExpertPackFp8(
    const ExpertRowsArgs& args,
    const void* x,
    int64_t xStride,
    void* q,
    int64_t qStride,
    void* scales,
    int device,
    hipStream_t stream);
// out[t] = sum over j of weights[t, j] * rows[position[t, j]], without the
// negative positions; all weights are 1 where weights is null.
void launchExpertCombine(
    const ExpertRowsArgs& args,
    const void* rows,
    int64_t rowStride,
    const float* weights,
    void* out,
    int device,
    hipStream_t stream);
// drows[position[t, j]] = weights[t, j] * grad[t], dweights[t, j] = rows[
// position[t, j]] . grad[t]; both zero for negative positions.
void launchExpertCombineBackward(
    const ExpertRowsArgs& args,
    const void* rows,
    int64_t rowStride,
    const float* weights,
    const void* grad,
    int64_t gradStride,
    void* drows,
    float* dweights,
    int device,
    hipStream_t stream);

} // namespace hip
} // namespace glooamd
