// The tensors' side of gloo_amd.experts: outputs, launches and autograd nodes
// of the operators, whose arguments the Python module has checked.
//
// In C++ because calls on small batches are bound by the host. A call takes 6
// to 7 us here, of which HIP's launch is 3, and 9 to 10 us where Python
// allocates. A backward pass over device tensors runs on a thread of its own:
// a node in Python hands the interpreter's lock over to it and back, and a
// forward and backward pass of route takes 41 to 84 us, by where the threads
// run, with the nodes here 31 to 55.
//
// A backward pass runs on its forward pass's stream, as the engine has it, so
// nodes keep that stream's handle.
#include <ATen/ATen.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <exception>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "common/error.h"
#include "hip/expert_launchers.h"

namespace py = pybind11;

namespace glooamd {

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

hip::ExpertLaunchers launchers;

DType typeOf(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return DType::F32;
    case at::kHalf:
      return DType::F16;
    default:
      return DType::BF16; // the callers allow no other type
  }
}

hipStream_t toStream(int64_t s) {
  return reinterpret_cast<hipStream_t>(s);
}

// What a tensor's memory holds is its values: not those of a view with the
// negative bit set (the imaginary part of a conjugate is one), and not a zero
// that has no memory. Data pointers are taken behind torch's dispatcher, which
// would see to both. Differentiable.
Tensor plain(const Tensor& t) {
  if (t.defined() && (t.is_neg() || t._is_zerotensor())) {
    return t.is_neg() ? t.resolve_neg() : at::zeros(t.sizes(), t.options());
  }
  return t;
}

std::optional<Tensor> plain(const std::optional<Tensor>& t) {
  return t.has_value() ? std::optional<Tensor>(plain(*t)) : t;
}

Tensor adjacent(const Tensor& given) {
  const Tensor t = plain(given);
  return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

Tensor contiguous(const Tensor& t) {
  return plain(t).contiguous();
}

// Operators have no forward-mode gradient, and a dual tensor's tangent would be
// lost without a word.
void noTangent(const char* name, const std::optional<Tensor>& t) {
  if (t.has_value() && t->defined() && t->_fw_grad(/*level=*/0).defined()) {
    throw py::value_error(
        std::string(name) +
        " has no forward-mode gradient: detach() its inputs");
  }
}

template <typename... Ts>
void noTangents(const char* name, const Ts&... ts) {
  (noTangent(name, ts), ...);
}

bool differentiated(const Tensor& t) {
  return at::GradMode::is_enabled() && t.defined() && t.requires_grad();
}

// Backward passes run in grad mode only where they are to be differentiated
// themselves.
void once() {
  TORCH_CHECK(
      !at::GradMode::is_enabled(),
      "the expert operators' gradients cannot be differentiated again "
      "(create_graph=True)");
}

// Arguments of nodes that may be absent are optional: a node takes no
// undefined tensor.
Tensor orNone(const std::optional<Tensor>& t) {
  return t.has_value() ? *t : Tensor();
}

// --- router ------------------------------------------------------------------

struct RouteOptions {
  int64_t k;
  bool sigmoid;
  int64_t groups;
  int64_t topkGroups;
  bool top2;
  bool renormalize;
  double scale;
};

hip::RouteArgs routeArgs(const Tensor& x, const RouteOptions& o) {
  hip::RouteArgs a;
  a.logits = x.const_data_ptr();
  a.stride = x.stride(0);
  a.dtype = typeOf(x);
  a.tokens = x.size(0);
  a.experts = static_cast<int>(x.size(1));
  a.k = static_cast<int>(o.k);
  a.sigmoid = o.sigmoid;
  a.groups = static_cast<int>(o.groups);
  a.topkGroups = static_cast<int>(o.topkGroups);
  a.groupTop2 = o.top2;
  a.renormalize = o.renormalize;
  a.scale = static_cast<float>(o.scale);
  return a;
}

variable_list routeForward(
    const Tensor& logits,
    const Tensor& bias,
    const RouteOptions& o,
    int64_t stream) {
  const Tensor x = adjacent(logits);
  Tensor weights =
      at::empty({x.size(0), o.k}, x.options().dtype(at::kFloat));
  Tensor ids = at::empty({x.size(0), o.k}, x.options().dtype(at::kInt));
  auto a = routeArgs(x, o);
  a.bias = bias.defined() ? bias.const_data_ptr<float>() : nullptr;
  a.weights = weights.mutable_data_ptr<float>();
  a.ids = ids.mutable_data_ptr<int32_t>();
  launchers.route(a, x.get_device(), toStream(stream));
  return {weights, ids};
}

struct RouteNode : public torch::autograd::Function<RouteNode> {
  static variable_list forward(
      AutogradContext* ctx,
      const Tensor& logits,
      const std::optional<Tensor>& bias,
      const RouteOptions& o,
      int64_t stream) {
    auto out = routeForward(logits, orNone(bias), o, stream);
    ctx->mark_non_differentiable({out[1]});
    ctx->save_for_backward({logits, out[1]});
    ctx->saved_data["options"] = o.k << 2 | o.sigmoid << 1 | o.renormalize;
    ctx->saved_data["scale"] = o.scale;
    ctx->saved_data["stream"] = stream;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const auto saved = ctx->get_saved_variables();
    const Tensor x = adjacent(saved[0]);
    const Tensor grad = contiguous(grads[0]);
    const int64_t bits = ctx->saved_data["options"].toInt();
    RouteOptions o{};
    o.k = bits >> 2;
    o.sigmoid = bits >> 1 & 1;
    o.renormalize = bits & 1;
    o.groups = 1;
    o.topkGroups = 1;
    o.scale = ctx->saved_data["scale"].toDouble();
    auto a = routeArgs(x, o);
    a.ids = saved[1].mutable_data_ptr<int32_t>();
    Tensor dx = at::empty(x.sizes(), x.options());
    launchers.routeBackward(
        a, grad.const_data_ptr<float>(), dx.mutable_data_ptr(),
        x.get_device(), toStream(ctx->saved_data["stream"].toInt()));
    return {dx, Tensor(), Tensor(), Tensor()};
  }
};

// --- plan --------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor>
plan(const Tensor& experts, int64_t numExperts, int64_t stream) {
  const Tensor ids = contiguous(experts);
  Tensor position = at::empty(ids.sizes(), ids.options());
  Tensor counts = at::empty({numExperts}, ids.options());
  Tensor offsets = at::empty({numExperts + 1}, ids.options());
  const size_t size =
      launchers.planWorkspace(ids.numel(), static_cast<int>(numExperts));
  Tensor work;
  if (size != 0) {
    work = at::empty(
        {static_cast<int64_t>(size)}, ids.options().dtype(at::kByte));
  }
  launchers.plan(
      ids.const_data_ptr<int32_t>(), ids.numel(),
      static_cast<int>(numExperts), position.mutable_data_ptr<int32_t>(),
      counts.mutable_data_ptr<int32_t>(), offsets.mutable_data_ptr<int32_t>(),
      size != 0 ? work.mutable_data_ptr() : nullptr, size, ids.get_device(),
      toStream(stream));
  return {position, counts, offsets};
}

// --- pack and combine --------------------------------------------------------

hip::ExpertRowsArgs rowsArgs(const Tensor& position, const Tensor& like) {
  hip::ExpertRowsArgs a;
  a.position = position.const_data_ptr<int32_t>();
  a.tokens = position.size(0);
  a.k = static_cast<int>(position.size(1));
  a.hidden = like.size(1);
  a.dtype = typeOf(like);
  return a;
}

Tensor packForward(
    const Tensor& tokens,
    const Tensor& position,
    int64_t stream) {
  const Tensor x = adjacent(tokens);
  Tensor rows = at::empty({position.numel(), x.size(1)}, x.options());
  if (rows.numel() != 0) {
    launchers.pack(
        rowsArgs(position, x), x.const_data_ptr(), x.stride(0),
        rows.mutable_data_ptr(), x.get_device(), toStream(stream));
  }
  return rows;
}

Tensor combineForward(
    const Tensor& all,
    const Tensor& position,
    const Tensor& weights,
    int64_t stream) {
  const Tensor rows = adjacent(all);
  Tensor out = at::empty({position.size(0), rows.size(1)}, rows.options());
  if (out.numel() != 0) {
    launchers.combine(
        rowsArgs(position, rows), rows.const_data_ptr(), rows.stride(0),
        weights.defined() ? weights.const_data_ptr<float>() : nullptr,
        out.mutable_data_ptr(), rows.get_device(), toStream(stream));
  }
  return out;
}

struct PackNode : public torch::autograd::Function<PackNode> {
  static Tensor forward(
      AutogradContext* ctx,
      const Tensor& x,
      const Tensor& position,
      int64_t stream) {
    ctx->save_for_backward({position});
    ctx->saved_data["stream"] = stream;
    return packForward(x, position, stream);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const auto saved = ctx->get_saved_variables();
    return {combineForward(grads[0], saved[0], Tensor(),
                           ctx->saved_data["stream"].toInt()),
            Tensor(), Tensor()};
  }
};

struct CombineNode : public torch::autograd::Function<CombineNode> {
  static Tensor forward(
      AutogradContext* ctx,
      const Tensor& rows,
      const Tensor& position,
      const std::optional<Tensor>& given,
      int64_t stream) {
    const Tensor weights = orNone(given);
    // Without weights the gradient needs no rows: they are free to change.
    ctx->save_for_backward(
        {weights.defined() ? rows : Tensor(), position, weights});
    ctx->saved_data["stream"] = stream;
    return combineForward(rows, position, weights, stream);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const auto saved = ctx->get_saved_variables();
    const Tensor& position = saved[1];
    const Tensor& weights = saved[2];
    const int64_t stream = ctx->saved_data["stream"].toInt();
    if (!weights.defined()) {
      return {packForward(grads[0], position, stream), Tensor(), Tensor(),
              Tensor()};
    }
    const Tensor rows = adjacent(saved[0]);
    const Tensor grad = adjacent(grads[0]);
    Tensor drows = at::empty(rows.sizes(), rows.options());
    Tensor dw = at::empty(weights.sizes(), weights.options());
    if (drows.numel() != 0) {
      launchers.combineBackward(
          rowsArgs(position, rows), rows.const_data_ptr(), rows.stride(0),
          weights.const_data_ptr<float>(), grad.const_data_ptr(),
          grad.stride(0), drows.mutable_data_ptr(),
          dw.mutable_data_ptr<float>(), rows.get_device(), toStream(stream));
    } else {
      dw.zero_();
    }
    return {drows, Tensor(), dw, Tensor()};
  }
};

// --- 8-bit rows and products -------------------------------------------------

constexpr int64_t kBlock = hip::kFp8Block;

int64_t blocksOf(int64_t n) {
  return (n + kBlock - 1) / kBlock;
}

// Room for rows of `width` 8-bit values that begin on borders of 128 bytes,
// so that products can load them whole: the values, and bytes from one row to
// the next.
std::pair<Tensor, int64_t>
fp8Rows(std::vector<int64_t> shape, int64_t width, const Tensor& like) {
  const int64_t pitch = blocksOf(width) * kBlock;
  shape.push_back(pitch);
  Tensor q = at::empty(shape, like.options().dtype(at::kFloat8_e4m3fn));
  return {pitch == width ? q : q.narrow(-1, 0, width), pitch};
}

Tensor fp8Scales(at::IntArrayRef shape, const Tensor& like) {
  return at::empty(shape, like.options().dtype(at::kFloat8_e8m0fnu));
}

std::pair<Tensor, Tensor>
packFp8(const Tensor& tokens, const Tensor& positions, int64_t stream) {
  noTangents("pack_fp8", tokens);
  const Tensor x = adjacent(tokens);
  const Tensor position = plain(positions);
  const int64_t n = position.numel();
  auto [q, pitch] = fp8Rows({n}, x.size(1), x);
  Tensor scales = fp8Scales({n, blocksOf(x.size(1))}, x);
  if (q.numel() != 0) {
    launchers.packFp8(
        rowsArgs(position, x), x.const_data_ptr(), x.stride(0),
        q.mutable_data_ptr(), pitch, scales.mutable_data_ptr(),
        x.get_device(), toStream(stream));
  }
  return {q, scales};
}

std::pair<Tensor, Tensor>
quantize(const Tensor& given, bool tile, int64_t stream) {
  noTangents("quantize_fp8", given);
  const Tensor x = plain(given);
  const int64_t rows = x.size(-2);
  const int64_t cols = x.size(-1);
  const bool many = x.dim() == 3;
  std::vector<int64_t> shape;
  if (many) {
    shape.push_back(x.size(0));
  }
  std::vector<int64_t> blocks = shape;
  shape.push_back(rows);
  blocks.push_back(tile ? blocksOf(rows) : rows);
  blocks.push_back(blocksOf(cols));
  auto [q, pitch] = fp8Rows(std::move(shape), cols, x);
  Tensor scales = fp8Scales(blocks, x);
  if (x.numel() == 0) {
    return {q, scales};
  }
  if (tile) {
    launchers.quantizeTiles(
        x.const_data_ptr(), many ? x.stride(0) : 0, x.stride(-2),
        x.stride(-1), typeOf(x), many ? x.size(0) : 1, rows, cols,
        q.mutable_data_ptr(), pitch, scales.mutable_data_ptr(),
        x.get_device(), toStream(stream));
  } else {
    launchers.quantize(
        x.const_data_ptr(), x.stride(0), x.stride(1), typeOf(x), rows, cols,
        q.mutable_data_ptr(), pitch, scales.mutable_data_ptr(),
        x.get_device(), toStream(stream));
  }
  return {q, scales};
}

// Bytes from one row to the next; a single row has none, whatever its stride
// says, and begins where the tensor does.
int64_t pitchOf(const Tensor& q) {
  return q.size(-2) > 1 ? q.stride(-2) : 0;
}

Tensor matmul(
    const Tensor& aGiven,
    const Tensor& aScaleGiven,
    const Tensor& bGiven,
    const Tensor& bScaleGiven,
    const std::optional<Tensor>& offsetsGiven,
    at::ScalarType dtype,
    int64_t stream) {
  const auto offsets = plain(offsetsGiven);
  noTangents("fp8_matmul", aGiven, aScaleGiven, bGiven, bScaleGiven);
  const Tensor a = adjacent(aGiven);
  const Tensor b = adjacent(bGiven);
  const Tensor aScale = contiguous(aScaleGiven);
  const Tensor bScale = contiguous(bScaleGiven);
  Tensor out =
      at::empty({a.size(0), b.size(-2)}, a.options().dtype(dtype));
  if (a.size(0) == 0) {
    return out;
  }
  hip::Fp8ProductArgs p;
  p.a = a.const_data_ptr();
  p.aStride = pitchOf(a);
  p.aScale = aScale.const_data_ptr();
  p.b = b.const_data_ptr();
  p.bStride = pitchOf(b);
  p.bScale = bScale.const_data_ptr();
  if (offsets.has_value()) {
    p.offsets = offsets->const_data_ptr<int32_t>();
    p.experts = static_cast<int>(b.size(0));
    p.bExpertStride = b.size(0) > 1 ? b.stride(0) : 0;
  }
  p.rows = a.size(0);
  p.n = b.size(-2);
  p.inner = a.size(1);
  p.out = out.mutable_data_ptr();
  p.dtype = typeOf(out);
  launchers.matmul(p, a.get_device(), toStream(stream));
  return out;
}

Tensor weightGrad(
    const Tensor& dyGiven,
    const Tensor& dyScaleGiven,
    const Tensor& xGiven,
    const Tensor& xScaleGiven,
    const std::optional<Tensor>& offsetsGiven,
    at::ScalarType dtype,
    int64_t stream) {
  const auto offsets = plain(offsetsGiven);
  noTangents(
      "fp8_weight_grad", dyGiven, dyScaleGiven, xGiven, xScaleGiven);
  const Tensor dy = adjacent(dyGiven);
  const Tensor x = adjacent(xGiven);
  const Tensor dyScale = contiguous(dyScaleGiven);
  const Tensor xScale = contiguous(xScaleGiven);
  hip::Fp8WeightGradArgs p;
  p.m = dy.size(0);
  p.n = x.size(0);
  p.rows = dy.size(1);
  std::vector<int64_t> shape{p.m, p.n};
  if (offsets.has_value()) {
    p.offsets = offsets->const_data_ptr<int32_t>();
    p.experts = static_cast<int>(offsets->size(0) - 1);
    shape.insert(shape.begin(), p.experts);
  }
  Tensor out = at::empty(shape, dy.options().dtype(dtype));
  p.dy = dy.const_data_ptr();
  p.dyStride = pitchOf(dy);
  p.dyScale = dyScale.const_data_ptr();
  p.x = x.const_data_ptr();
  p.xStride = pitchOf(x);
  p.xScale = xScale.const_data_ptr();
  p.out = out.mutable_data_ptr();
  p.dtype = typeOf(out);
  launchers.weightGrad(p, dy.get_device(), toStream(stream));
  return out;
}

} // namespace

} // namespace glooamd

PYBIND11_MODULE(_operators, m) {
  using namespace glooamd;
  using Unlocked = py::call_guard<py::gil_scoped_release>;
  m.doc() = "The tensors' side of gloo_amd.experts";

  // What a launch refuses (a grid that it cannot hold) is a wrong argument.
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      std::rethrow_exception(p);
    } catch (const EnforceNotMet& e) {
      PyErr_SetString(PyExc_ValueError, e.what());
    }
  });

  m.def("set_launchers", [](const py::capsule& c) {
    const auto* given = static_cast<hip::ExpertLaunchers*>(
        PyCapsule_GetPointer(c.ptr(), hip::kExpertLaunchers));
    if (given == nullptr) {
      throw py::error_already_set();
    }
    launchers = *given;
  });

  m.def(
      "route",
      [](const Tensor& given, const std::optional<Tensor>& biasGiven,
         int64_t k, bool sigmoid, int64_t groups, int64_t topkGroups, bool top2,
         bool renormalize, double scale, int64_t stream) {
        noTangents("route", given);
        const Tensor logits = plain(given);
        const auto bias = plain(biasGiven);
        const RouteOptions o{k,    sigmoid,     groups, topkGroups,
                             top2, renormalize, scale};
        const auto out = differentiated(logits)
            ? RouteNode::apply(logits, bias, o, stream)
            : routeForward(logits, orNone(bias), o, stream);
        return std::make_pair(out[0], out[1]);
      },
      Unlocked());

  m.def(
      "pack",
      [](const Tensor& given, const Tensor& positionGiven, int64_t stream) {
        noTangents("pack", given);
        const Tensor x = plain(given);
        const Tensor position = plain(positionGiven);
        return differentiated(x) ? PackNode::apply(x, position, stream)
                                 : packForward(x, position, stream);
      },
      Unlocked());

  m.def(
      "combine",
      [](const Tensor& given, const Tensor& positionGiven,
         const std::optional<Tensor>& weightsGiven, int64_t stream) {
        noTangents("combine", given, weightsGiven);
        const Tensor rows = plain(given);
        const Tensor position = plain(positionGiven);
        const auto weights = plain(weightsGiven);
        return differentiated(rows) || differentiated(orNone(weights))
            ? CombineNode::apply(rows, position, weights, stream)
            : combineForward(rows, position, orNone(weights), stream);
      },
      Unlocked());

  m.def("plan", &plan, Unlocked());
  m.def("pack_fp8", &packFp8, Unlocked());
  m.def("quantize_fp8", &quantize, Unlocked());
  m.def("fp8_matmul", &matmul, Unlocked());
  m.def("fp8_weight_grad", &weightGrad, Unlocked());
}
