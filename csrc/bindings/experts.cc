#include "bindings/experts.h"

#include <string>

#include "common/logging.h"
#include "hip/expert_launchers.h"
#include "hip/experts.h"
#include "hip/fp8.h"

namespace py = pybind11;

namespace glooamd {

namespace {

template <typename T>
T* ptr(uintptr_t p) {
  return reinterpret_cast<T*>(p);
}

hipStream_t toStream(uintptr_t s) {
  return reinterpret_cast<hipStream_t>(s);
}

bool isSigmoid(const std::string& score) {
  GA_ENFORCE(
      score == "softmax" || score == "sigmoid", "score: ", score);
  return score == "sigmoid";
}

bool isTop2(const std::string& groupScore) {
  GA_ENFORCE(
      groupScore == "max" || groupScore == "top2",
      "group_score: ", groupScore);
  return groupScore == "top2";
}

hip::ExpertRowsArgs rowsArgs(
    uintptr_t position,
    int64_t tokens,
    int k,
    int64_t hidden,
    DType dtype) {
  hip::ExpertRowsArgs a;
  a.position = ptr<const int32_t>(position);
  a.tokens = tokens;
  a.k = k;
  a.hidden = hidden;
  a.dtype = dtype;
  return a;
}

} // namespace

void bindExperts(py::module_& m) {
  m.attr("MAX_EXPERTS") = hip::kMaxExperts;
  m.attr("MAX_TOPK") = hip::kMaxTopK;
  m.attr("MAX_EXPERT_GROUPS") = hip::kMaxExpertGroups;

  // For gloo_amd._operators, which does not link the kernels.
  m.def("expert_launchers", [] {
    static hip::ExpertLaunchers launchers{
        &hip::launchRoute, &hip::launchRouteBackward,
        &hip::expertPlanWorkspace, &hip::launchExpertPlan,
        &hip::launchExpertPack, &hip::launchExpertPackFp8,
        &hip::launchExpertCombine, &hip::launchExpertCombineBackward,
        &hip::launchQuantizeFp8, &hip::launchQuantizeFp8Tiles,
        &hip::launchFp8Matmul, &hip::launchFp8WeightGrad};
    return py::capsule(&launchers, hip::kExpertLaunchers);
  });

  m.def(
      "hip_expert_route",
      [](uintptr_t logits, int64_t stride, DType dtype, uintptr_t bias,
         int64_t tokens, int experts, int k, const std::string& score,
         int groups, int topkGroups, const std::string& groupScore,
         bool renormalize, float scale, uintptr_t weights, uintptr_t ids,
         int device, uintptr_t stream) {
        hip::RouteArgs a;
        a.logits = ptr<const void>(logits);
        a.stride = stride;
        a.dtype = dtype;
        a.bias = ptr<const float>(bias);
        a.tokens = tokens;
        a.experts = experts;
        a.k = k;
        a.sigmoid = isSigmoid(score);
        a.groups = groups;
        a.topkGroups = topkGroups;
        a.groupTop2 = isTop2(groupScore);
        a.renormalize = renormalize;
        a.scale = scale;
        a.weights = ptr<float>(weights);
        a.ids = ptr<int32_t>(ids);
        py::gil_scoped_release rel;
        hip::launchRoute(a, device, toStream(stream));
      });

  m.def(
      "hip_expert_route_backward",
      [](uintptr_t logits, int64_t stride, DType dtype, int64_t tokens,
         int experts, int k, const std::string& score, bool renormalize,
         float scale, uintptr_t ids, uintptr_t grad, uintptr_t dlogits,
         int device, uintptr_t stream) {
        hip::RouteArgs a;
        a.logits = ptr<const void>(logits);
        a.stride = stride;
        a.dtype = dtype;
        a.tokens = tokens;
        a.experts = experts;
        a.k = k;
        a.sigmoid = isSigmoid(score);
        a.renormalize = renormalize;
        a.scale = scale;
        a.ids = ptr<int32_t>(ids);
        py::gil_scoped_release rel;
        hip::launchRouteBackward(
            a, ptr<const float>(grad), ptr<void>(dlogits), device,
            toStream(stream));
      });

  m.def("hip_expert_plan_workspace", &hip::expertPlanWorkspace);
  m.def(
      "hip_expert_plan",
      [](uintptr_t ids, int64_t n, int experts, uintptr_t position,
         uintptr_t counts, uintptr_t offsets, uintptr_t workspace,
         size_t workspaceBytes, int device, uintptr_t stream) {
        py::gil_scoped_release rel;
        hip::launchExpertPlan(
            ptr<const int32_t>(ids), n, experts, ptr<int32_t>(position),
            ptr<int32_t>(counts), ptr<int32_t>(offsets),
            ptr<void>(workspace), workspaceBytes, device, toStream(stream));
      });

  m.def(
      "hip_expert_pack",
      [](uintptr_t position, int64_t tokens, int k, int64_t hidden,
         DType dtype, uintptr_t x, int64_t xStride, uintptr_t rows,
         int device, uintptr_t stream) {
        const auto a = rowsArgs(position, tokens, k, hidden, dtype);
        py::gil_scoped_release rel;
        hip::launchExpertPack(
            a, ptr<const void>(x), xStride, ptr<void>(rows), device,
            toStream(stream));
      });

  m.def(
      "hip_expert_pack_fp8",
      [](uintptr_t position, int64_t tokens, int k, int64_t hidden,
         DType dtype, uintptr_t x, int64_t xStride, uintptr_t q,
         int64_t qStride, uintptr_t scales, int device, uintptr_t stream) {
        const auto a = rowsArgs(position, tokens, k, hidden, dtype);
        py::gil_scoped_release rel;
        hip::launchExpertPackFp8(
            a, ptr<const void>(x), xStride, ptr<void>(q), qStride,
            ptr<void>(scales), device, toStream(stream));
      });

  m.def(
      "hip_expert_combine",
      [](uintptr_t position, int64_t tokens, int k, int64_t hidden,
         DType dtype, uintptr_t rows, int64_t rowStride, uintptr_t weights,
         uintptr_t out, int device, uintptr_t stream) {
        const auto a = rowsArgs(position, tokens, k, hidden, dtype);
        py::gil_scoped_release rel;
        hip::launchExpertCombine(
            a, ptr<const void>(rows), rowStride, ptr<const float>(weights),
            ptr<void>(out), device, toStream(stream));
      });

  m.def(
      "hip_expert_combine_backward",
      [](uintptr_t position, int64_t tokens, int k, int64_t hidden,
         DType dtype, uintptr_t rows, int64_t rowStride, uintptr_t weights,
         uintptr_t grad, int64_t gradStride, uintptr_t drows,
         uintptr_t dweights, int device, uintptr_t stream) {
        const auto a = rowsArgs(position, tokens, k, hidden, dtype);
        py::gil_scoped_release rel;
        hip::launchExpertCombineBackward(
            a, ptr<const void>(rows), rowStride, ptr<const float>(weights),
            ptr<const void>(grad), gradStride, ptr<void>(drows),
            ptr<float>(dweights), device, toStream(stream));
      });

  m.def(
      "hip_quantize_fp8",
      [](uintptr_t x, int64_t rowStride, int64_t colStride, DType dtype,
         int64_t rows, int64_t cols, bool tile, uintptr_t q, int64_t qStride,
         uintptr_t scales, int device, uintptr_t stream) {
        py::gil_scoped_release rel;
        if (tile) {
          hip::launchQuantizeFp8Tiles(
              ptr<const void>(x), 0, rowStride, colStride, dtype, 1, rows,
              cols, ptr<void>(q), qStride, ptr<void>(scales), device,
              toStream(stream));
        } else {
          hip::launchQuantizeFp8(
              ptr<const void>(x), rowStride, colStride, dtype, rows, cols,
              ptr<void>(q), qStride, ptr<void>(scales), device,
              toStream(stream));
        }
      });

  m.def(
      "hip_fp8_matmul",
      [](uintptr_t a, int64_t aStride, uintptr_t aScale, uintptr_t b,
         int64_t bStride, int64_t bExpertStride, uintptr_t bScale,
         uintptr_t offsets, int64_t rows, int64_t n, int64_t inner,
         int experts, uintptr_t out, DType dtype, int device,
         uintptr_t stream) {
        hip::Fp8ProductArgs p;
        p.a = ptr<const void>(a);
        p.aStride = aStride;
        p.aScale = ptr<const void>(aScale);
        p.b = ptr<const void>(b);
        p.bStride = bStride;
        p.bExpertStride = bExpertStride;
        p.bScale = ptr<const void>(bScale);
        p.offsets = ptr<const int32_t>(offsets);
        p.rows = rows;
        p.n = n;
        p.inner = inner;
        p.experts = experts;
        p.out = ptr<void>(out);
        p.dtype = dtype;
        py::gil_scoped_release rel;
        hip::launchFp8Matmul(p, device, toStream(stream));
      });

  m.def(
      "hip_fp8_weight_grad",
      [](uintptr_t dy, int64_t dyStride, uintptr_t dyScale, uintptr_t x,
         int64_t xStride, uintptr_t xScale, uintptr_t offsets, int64_t mm,
         int64_t n, int64_t rows, int experts, uintptr_t out, DType dtype,
         int device, uintptr_t stream) {
        hip::Fp8WeightGradArgs p;
        p.dy = ptr<const void>(dy);
        p.dyStride = dyStride;
        p.dyScale = ptr<const void>(dyScale);
        p.x = ptr<const void>(x);
        p.xStride = xStride;
        p.xScale = ptr<const void>(xScale);
        p.offsets = ptr<const int32_t>(offsets);
        p.m = mm;
        p.n = n;
        p.rows = rows;
        p.experts = experts;
        p.out = ptr<void>(out);
        p.dtype = dtype;
        py::gil_scoped_release rel;
        hip::launchFp8WeightGrad(p, device, toStream(stream));
      });
}

} // namespace glooamd
