// torch operators of the training kernels, with their gradients (namespace disentangled_flash).
//
// The kernels are libdflash's, called through its C ABI; here tensors are allocated and the
// autograd nodes made.  They are C++ because a training step calls them dozens of times:
// as Python functions one LayerNorm tail of few rows, forward and backward, took about 130 us
// of host time for 15 us of kernels, most of it in the backward pass, which torch runs on
// a thread of its own.
//
// Host code only, built against torch's headers; the Python side (training.py) checks the
// arguments, registers the fake implementations and binds the library.

#include <ATen/core/Tensor.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>

#include "dflash.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct Library {
  decltype(&dflash_dropout) dropout;
  decltype(&dflash_dropout_layernorm_fwd) layernorm_fwd;
  decltype(&dflash_dropout_layernorm_bwd) layernorm_bwd;
  decltype(&dflash_dropout_layernorm_bwd_workspace_bytes) layernorm_bwd_workspace_bytes;
  decltype(&dflash_embedding_fwd) embedding_fwd;
  decltype(&dflash_embedding_bwd) embedding_bwd;
  decltype(&dflash_embedding_bwd_workspace_bytes) embedding_bwd_workspace_bytes;
  decltype(&dflash_error_string) error_string;
} lib;

template <typename F>
void find(void* handle, const char* name, F& function) {
  function = reinterpret_cast<F>(dlsym(handle, name));
  TORCH_CHECK(function, "libdflash has no ", name);
}

// The library at `path`, which the process has loaded already (it stays loaded).
void bind_library(std::string path) {
  void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(handle, "cannot load ", path, ": ", dlerror());
  find(handle, "dflash_dropout", lib.dropout);
  find(handle, "dflash_dropout_layernorm_fwd", lib.layernorm_fwd);
  find(handle, "dflash_dropout_layernorm_bwd", lib.layernorm_bwd);
  find(handle, "dflash_dropout_layernorm_bwd_workspace_bytes", lib.layernorm_bwd_workspace_bytes);
  find(handle, "dflash_embedding_fwd", lib.embedding_fwd);
  find(handle, "dflash_embedding_bwd", lib.embedding_bwd);
  find(handle, "dflash_embedding_bwd_workspace_bytes", lib.embedding_bwd_workspace_bytes);
  find(handle, "dflash_error_string", lib.error_string);
}

void check(int code, const char* name) {
  TORCH_CHECK(code == DFLASH_OK, name, " failed with code ", code, ": ", lib.error_string(code));
}

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return DFLASH_DTYPE_FP16;
    case at::kBFloat16: return DFLASH_DTYPE_BF16;
    case at::kFloat: return DFLASH_DTYPE_FP32;
    default: TORCH_CHECK_TYPE(false, "dtype is not fp16, bf16 or fp32");
  }
}

// The tensor's device made current, and torch's current stream there.
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
};

// Uninitialised memory, past the dispatcher (five of them in a backward pass).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }

// The LayerNorm's rows start on 16-byte boundaries.
bool is_aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
Tensor aligned(const Tensor& t) { return is_aligned(t) ? t : t.clone(); }
MaybeTensor aligned(const MaybeTensor& t) { return t && !is_aligned(*t) ? t->clone() : t; }

void* data(const Tensor& t) { return t.data_ptr(); }
void* data(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }
const int64_t* words(const MaybeTensor& rng) {
  return rng ? static_cast<const int64_t*>(rng->data_ptr()) : nullptr;
}

// What the C calls take on trust.  training.py refuses more, and says more; but the operators can
// be called past it, from a traced graph or by their names.
void expect(bool good, const char* name) {
  TORCH_CHECK_VALUE(good, name, " does not fit the call: shape, dtype, device or strides");
}
bool fits(const Tensor& t, const Tensor& x) { return t.device() == x.device() && t.is_contiguous(); }
bool same_form(const Tensor& t, const Tensor& x) {
  return fits(t, x) && t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type();
}
bool vector_of(const Tensor& t, int64_t n, const Tensor& x) {
  return fits(t, x) && t.dim() == 1 && t.size(0) == n;
}
void expect_dropout(const MaybeTensor& rng, int64_t site, const Tensor& x) {
  expect(!rng || (vector_of(*rng, 2, x) && rng->scalar_type() == at::kLong), "rng");
  expect(site >= 0 && site <= UINT32_MAX, "site");
}
void expect_rows(const Tensor& x) {
  expect(x.is_contiguous() && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= INT32_MAX, "x");
}

// ---- the calls ----------------------------------------------------------------------

Tensor dropout(const Tensor& x, const Tensor& rng, double p, int64_t site) {
  expect(x.is_contiguous(), "x");
  expect_dropout(rng, site, x);
  Tensor out = fresh_like(x);
  On on(x);
  check(lib.dropout(data(x), data(out), x.numel(), p, words(rng), site, code_of(x), on.stream),
        "dflash_dropout");
  return out;
}

Tensor layernorm(const Tensor& given, const MaybeTensor& given_residual, const Tensor& weight,
                 const Tensor& bias, const MaybeTensor& rng, double eps, double p, int64_t site,
                 float* statistics) {
  expect_rows(given);
  expect(!given_residual || same_form(*given_residual, given), "residual");
  expect(vector_of(weight, given.size(-1), given), "weight");
  expect(same_form(bias, weight), "bias");
  expect_dropout(rng, site, given);
  const Tensor x = aligned(given);
  const MaybeTensor residual = aligned(given_residual);
  Tensor y = fresh_like(x);
  const int64_t hidden = x.size(-1), rows = x.numel() / hidden;
  On on(x);
  check(lib.layernorm_fwd(data(x), data(residual), data(weight), data(bias), data(y), statistics,
                          statistics ? statistics + rows : nullptr, rows, hidden, eps, p,
                          words(rng), site, code_of(x), code_of(weight), on.stream),
        "dflash_dropout_layernorm_fwd");
  return y;
}

Tensor dropout_layernorm(const Tensor& x, const MaybeTensor& residual, const Tensor& weight,
                         const Tensor& bias, const MaybeTensor& rng, double eps, double p,
                         int64_t site) {
  return layernorm(x, residual, weight, bias, rng, eps, p, site, nullptr);
}

// (y, [mean, rstd])
std::tuple<Tensor, Tensor> dropout_layernorm_train(const Tensor& x, const MaybeTensor& residual,
                                                   const Tensor& weight, const Tensor& bias,
                                                   const MaybeTensor& rng, double eps, double p,
                                                   int64_t site) {
  expect_rows(x);
  Tensor statistics = fresh({2, x.numel() / x.size(-1)}, at::kFloat, x);
  Tensor y = layernorm(x, residual, weight, bias, rng, eps, p, site,
                       static_cast<float*>(data(statistics)));
  return {y, statistics};
}

// (dx, dresidual, dweight, dbias); those not wanted are empty.
std::tuple<Tensor, Tensor, Tensor, Tensor> dropout_layernorm_backward(
    const Tensor& given_dy, const Tensor& given, const MaybeTensor& given_residual,
    const Tensor& weight, const Tensor& statistics, const MaybeTensor& rng, double p, int64_t site,
    bool want_x, bool want_residual, bool want_weights) {
  expect_rows(given);
  expect(same_form(given_dy, given), "dy");
  expect(!given_residual || same_form(*given_residual, given), "residual");
  expect(vector_of(weight, given.size(-1), given), "weight");
  expect(fits(statistics, given) && statistics.scalar_type() == at::kFloat &&
             statistics.numel() == given.numel() / given.size(-1) * 2,
         "statistics");
  expect_dropout(rng, site, given);
  const Tensor dy = aligned(given_dy), x = aligned(given);
  const MaybeTensor residual = aligned(given_residual);
  const int64_t hidden = x.size(-1), rows = x.numel() / hidden;
  auto made = [](bool wanted, const Tensor& like) {
    return wanted ? fresh_like(like) : fresh({0}, like.scalar_type(), like);
  };
  Tensor dx = made(want_x, x), dresidual = made(want_residual, x);
  Tensor dweight = made(want_weights, weight), dbias = made(want_weights, weight);
  const size_t bytes = want_weights ? lib.layernorm_bwd_workspace_bytes(rows, hidden) : 0;
  Tensor workspace;
  if (bytes) workspace = fresh({static_cast<int64_t>(bytes)}, at::kByte, x);
  const float* mean = static_cast<const float*>(data(statistics));
  On on(x);
  check(lib.layernorm_bwd(data(dy), data(x), data(residual), data(weight), mean, mean + rows,
                          want_x ? data(dx) : nullptr, want_residual ? data(dresidual) : nullptr,
                          want_weights ? data(dweight) : nullptr,
                          want_weights ? data(dbias) : nullptr, rows, hidden, p, words(rng), site,
                          code_of(x), code_of(weight), bytes ? data(workspace) : nullptr, bytes,
                          on.stream),
        "dflash_dropout_layernorm_bwd");
  return {dx, dresidual, dweight, dbias};
}

void expect_ids(const Tensor& ids, const Tensor& like) {
  expect(fits(ids, like) && (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong),
         "ids");
}

Tensor embedding_lookup(const Tensor& ids, const Tensor& table, double scale,
                        int64_t /*padding*/) {
  expect(table.dim() == 2 && table.is_contiguous() && table.size(0) < INT32_MAX &&
             table.size(1) <= INT32_MAX,
         "table");
  expect_ids(ids, table);
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  Tensor out = fresh(shape, table.scalar_type(), table);
  On on(table);
  check(lib.embedding_fwd(data(ids), data(table), data(out), ids.numel(), table.size(0),
                          table.size(1), scale, ids.element_size(), code_of(table), on.stream),
        "dflash_embedding_fwd");
  return out;
}

Tensor embedding_gradient(const Tensor& dy, const Tensor& ids, c10::SymInt table_rows,
                          double scale, int64_t padding) {
  expect(dy.is_contiguous() && dy.dim() >= 1, "dy");
  expect_ids(ids, dy);
  const int64_t hidden = dy.size(-1), rows = table_rows.expect_int();
  expect(dy.numel() == ids.numel() * hidden, "dy");
  expect(rows >= 1 && rows < INT32_MAX && hidden <= INT32_MAX, "the table");
  Tensor out = fresh({rows, hidden}, dy.scalar_type(), dy);
  const size_t bytes = lib.embedding_bwd_workspace_bytes(ids.numel(), hidden);
  Tensor workspace;
  if (bytes) workspace = fresh({static_cast<int64_t>(bytes)}, at::kByte, dy);
  On on(dy);
  check(lib.embedding_bwd(data(ids), data(dy), data(out), ids.numel(), rows, hidden, scale, padding,
                          ids.element_size(), code_of(dy), bytes ? data(workspace) : nullptr,
                          bytes, on.stream),
        "dflash_embedding_bwd");
  return out;
}

// ---- autograd ------------------------------------------------------------------------

template <typename F>
auto operator_of(const char* name) {
  return c10::Dispatcher::singleton()
      .findSchemaOrThrow((std::string("disentangled_flash::") + name).c_str(), "")
      .typed<F>();
}

const auto& dropout_op() {
  static const auto op = operator_of<decltype(dropout)>("dropout");
  return op;
}
const auto& layernorm_op() {
  static const auto op = operator_of<decltype(dropout_layernorm)>("dropout_layernorm");
  return op;
}
const auto& layernorm_train_op() {
  static const auto op =
      operator_of<decltype(dropout_layernorm_train)>("dropout_layernorm_train");
  return op;
}
const auto& layernorm_backward_op() {
  static const auto op =
      operator_of<decltype(dropout_layernorm_backward)>("dropout_layernorm_backward");
  return op;
}
const auto& lookup_op() {
  static const auto op = operator_of<decltype(embedding_lookup)>("embedding_lookup");
  return op;
}
const auto& gradient_op() {
  static const auto op = operator_of<decltype(embedding_gradient)>("embedding_gradient");
  return op;
}

// Forward-mode derivatives are not implemented; below autograd a tangent would be lost unseen.
void no_tangent(const Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name,
                              ": forward-mode derivatives are not implemented");
}
void no_tangent(const MaybeTensor& t, const char* name) {
  if (t) no_tangent(*t, name);
}

// Gradients whose own gradient is not implemented: differentiating them raises.
variable_list only_once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) defined.push_back(g.detach().requires_grad_());
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + ": trying to differentiate twice a gradient that can only be taken once",
      static_cast<int64_t>(defined.size()));
  variable_list out = (*error)(std::move(defined));
  size_t next = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[next++];
  return grads;
}

struct DropoutNode : Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& rng, double p,
                        int64_t site) {
    ctx->save_for_backward({rng});
    ctx->saved_data["p"] = p;
    ctx->saved_data["site"] = site;
    at::AutoDispatchBelowADInplaceOrView below;
    return dropout_op().call(x, rng, p, site);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor rng = ctx->get_saved_variables()[0];
    // (The same elements of dy: differentiable again.)
    return {dropout_op().call(grads[0].contiguous(), rng, ctx->saved_data["p"].toDouble(),
                              ctx->saved_data["site"].toInt()),
            Tensor(), Tensor(), Tensor()};
  }
};

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

struct LayerNormNode : Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual,
                        const Tensor& weight, const Tensor& bias, const MaybeTensor& rng,
                        double eps, double p, int64_t site) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, statistics] = layernorm_train_op().call(x, residual, weight, bias, rng, eps, p, site);
    ctx->save_for_backward({x, residual.value_or(Tensor()), weight, statistics,
                            rng.value_or(Tensor())});
    ctx->saved_data["p"] = p;
    ctx->saved_data["site"] = site;
    ctx->saved_data["wanted"] = static_cast<int64_t>(
        x.requires_grad() | (residual && residual->requires_grad()) << 1 |
        weight.requires_grad() << 2 | bias.requires_grad() << 3);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const double p = ctx->saved_data["p"].toDouble();
    const int64_t wanted = ctx->saved_data["wanted"].toInt();
    const bool want_x = wanted & 1, want_residual = wanted & 2, want_weight = wanted & 4,
               want_bias = wanted & 8;
    no_tangent(grads[0], "layer_norm");
    // Without dropout the gradients of x and of the residual are the same tensor.
    const bool shared = p == 0.0 && want_residual;
    Tensor dx, dresidual, dweight, dbias;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(dx, dresidual, dweight, dbias) = layernorm_backward_op().call(
          grads[0].contiguous(), saved[0], maybe(saved[1]), saved[2], saved[3], maybe(saved[4]), p,
          ctx->saved_data["site"].toInt(), want_x || shared, want_residual && !shared,
          want_weight || want_bias);
    }
    if (shared) dresidual = dx;
    const Tensor none;
    return only_once({want_x ? dx : none, want_residual ? dresidual : none,
                      want_weight ? dweight : none, want_bias ? dbias : none, none, none, none,
                      none},
                     "layer_norm");
  }
};

struct EmbeddingNode : Function<EmbeddingNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale,
                        int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.sym_size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    at::AutoDispatchBelowADInplaceOrView below;
    return lookup_op().call(ids, table, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor ids = ctx->get_saved_variables()[0];
    no_tangent(grads[0], "embedding");
    Tensor grad;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      grad = gradient_op().call(grads[0].contiguous(), ids, ctx->saved_data["rows"].toSymInt(),
                                ctx->saved_data["scale"].toDouble(),
                                ctx->saved_data["padding"].toInt());
    }
    return only_once({Tensor(), grad, Tensor(), Tensor()}, "embedding");
  }
};

bool records(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

Tensor dropout_autograd(const Tensor& x, const Tensor& rng, double p, int64_t site) {
  no_tangent(x, "dropout");
  if (records(x)) return DropoutNode::apply(x, rng, p, site);
  at::AutoDispatchBelowADInplaceOrView below;
  return dropout_op().call(x, rng, p, site);
}

Tensor dropout_layernorm_autograd(const Tensor& x, const MaybeTensor& residual,
                                  const Tensor& weight, const Tensor& bias, const MaybeTensor& rng,
                                  double eps, double p, int64_t site) {
  for (const Tensor* t : {&x, &weight, &bias}) no_tangent(*t, "layer_norm");
  no_tangent(residual, "layer_norm");
  if (records(x) || records(weight) || records(bias) || (residual && records(*residual)))
    return LayerNormNode::apply(x, residual, weight, bias, rng, eps, p, site);
  at::AutoDispatchBelowADInplaceOrView below;
  return layernorm_op().call(x, residual, weight, bias, rng, eps, p, site);
}

Tensor embedding_lookup_autograd(const Tensor& ids, const Tensor& table, double scale,
                                 int64_t padding) {
  no_tangent(table, "embedding");
  if (records(table)) return EmbeddingNode::apply(ids, table, scale, padding);
  at::AutoDispatchBelowADInplaceOrView below;
  return lookup_op().call(ids, table, scale, padding);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(disentangled_flash, m) {
  m.def("bind_library(str path) -> ()", &bind_library);
  m.def("dropout(Tensor x, Tensor rng, float p, int site) -> Tensor");
  m.def(
      "dropout_layernorm(Tensor x, Tensor? residual, Tensor weight, Tensor bias, Tensor? rng, "
      "float eps, float p, int site) -> Tensor");
  m.def(
      "dropout_layernorm_train(Tensor x, Tensor? residual, Tensor weight, Tensor bias, "
      "Tensor? rng, float eps, float p, int site) -> (Tensor, Tensor)");
  m.def(
      "dropout_layernorm_backward(Tensor dy, Tensor x, Tensor? residual, Tensor weight, "
      "Tensor statistics, Tensor? rng, float p, int site, bool want_x, bool want_residual, "
      "bool want_weights) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("embedding_lookup(Tensor ids, Tensor table, float scale, int padding) -> Tensor");
  m.def(
      "embedding_gradient(Tensor dy, Tensor ids, SymInt rows, float scale, int padding) -> Tensor");
}

TORCH_LIBRARY_IMPL(disentangled_flash, CUDA, m) {
  m.impl("dropout", &dropout);
  m.impl("dropout_layernorm", &dropout_layernorm);
  m.impl("dropout_layernorm_train", &dropout_layernorm_train);
  m.impl("dropout_layernorm_backward", &dropout_layernorm_backward);
  m.impl("embedding_lookup", &embedding_lookup);
  m.impl("embedding_gradient", &embedding_gradient);
}

TORCH_LIBRARY_IMPL(disentangled_flash, Autograd, m) {
  m.impl("dropout", &dropout_autograd);
  m.impl("dropout_layernorm", &dropout_layernorm_autograd);
  m.impl("embedding_lookup", &embedding_lookup_autograd);
}
