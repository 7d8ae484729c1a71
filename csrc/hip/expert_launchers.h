// The expert operators' launches, handed from the extension that holds the
// kernels (gloo_amd._C, which does without torch) to the one that links torch
// (gloo_amd._operators) as one pointer.
#pragma once

#include "hip/experts.h"
#include "hip/fp8.h"

namespace glooamd {
namespace hip {

struct ExpertLaunchers {
  decltype(&launchRoute) route;
  decltype(&launchRouteBackward) routeBackward;
  decltype(&expertPlanWorkspace) planWorkspace;
  decltype(&launchExpertPlan) plan;
  decltype(&launchExpertPack) pack;
  decltype(&launchExpertPackFp8) packFp8;
  decltype(&launchExpertCombine) combine;
  decltype(&launchExpertCombineBackward) combineBackward;
  decltype(&launchQuantizeFp8) quantize;
  decltype(&launchQuantizeFp8Tiles) quantizeTiles;
  decltype(&launchFp8Matmul) matmul;
  decltype(&launchFp8WeightGrad) weightGrad;
};

constexpr const char* kExpertLaunchers = "gloo_amd.ExpertLaunchers";

} // namespace hip
} // namespace glooamd
