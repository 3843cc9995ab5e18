// Tensors and gradients for the operators of include/spnc_hip_rows.h: the native half of spnc/mixture.py. Argument checks,
// outputs from PyTorch's allocator, the current stream of the tensors' device and autograd nodes; all arithmetic is behind the
// C-ABI. In C++ because a call of a few microseconds of GPU time is otherwise dominated by the interpreter, twice so where
// the backward pass runs on PyTorch's own thread.
#include <ATen/MemoryOverlap.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/spnc_hip_rows.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t ROWS_LIMIT = int64_t(1) << 31;

// Failures are RuntimeErrors with the bare message, as everywhere in spnc.
template <typename... Args>
void refuse(bool condition, const Args&... args) {
  if (C10_UNLIKELY(condition)) throw std::runtime_error(c10::str(args...));
}

// Behind the C-ABI an error that an earlier, foreign call left behind is not touched. PyTorch would raise it from whichever operation comes
// next; here, where the call it belongs to can still be guessed, it is told as a warning.
void check(int rc) {
  refuse(rc != 0, spnc_hip_last_error());
  if (C10_LIKELY(hipPeekAtLastError() == hipSuccess)) return;
  TORCH_WARN("a HIP call before this one of spnc.mixture left an error behind: ", hipGetErrorString(hipGetLastError()));
}

int elementType(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SPNC_HIP_FLOAT32;
    case at::kDouble: return SPNC_HIP_FLOAT64;
    case at::kHalf: return SPNC_HIP_FLOAT16;
    case at::kBFloat16: return SPNC_HIP_BFLOAT16;
    default: return -1;
  }
}

// All defined tensors on one GPU.
void onGpu(std::initializer_list<const Tensor*> tensors) {
  const at::Device device = (*tensors.begin())->device();
  for (const Tensor* t : tensors)
    if (t->defined()) {
      refuse(!t->is_cuda(), "Tensors must be on a GPU, got one on ", t->device());
      refuse(t->device() != device, "Tensors must be on one GPU, got ", device, " and ", t->device());
    }
}

void* streamOf(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool wantsGrad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The kernels are reached without PyTorch's dispatcher, so what it would do on the way is not done: a tangent would be dropped, and a trace
// would hold the allocation of a result that nothing computes. Such calls are refused.
void checkRecorded(std::initializer_list<const Tensor*> tensors) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  refuse(torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
             (TorchDispatchModeTLS::any_modes_set() && TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value()),
         "spnc.mixture cannot be traced");
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors) refuse(t->defined() && t->_fw_grad(0).defined(), "spnc.mixture has no forward-mode derivatives");
}

// Views of a conjugate's imaginary part, which autograd hands out as gradients too, hold their numbers with the other sign. Memory that
// holds a tensor's own numbers, a copy for such a view:
Tensor plain(const Tensor& t) { return C10_UNLIKELY(t.is_neg()) ? t.resolve_neg() : t; }
Tensor flat(const Tensor& t) { return plain(t).contiguous(); }

// A 2-D tensor whose rows are contiguous and do not overlap; a copy where they are not.
Tensor rowsOf(const Tensor& given) {
  const Tensor t = plain(given);
  const int64_t n = t.size(0), width = t.size(1);
  if ((width <= 1 || t.stride(1) == 1) && (n <= 1 || t.stride(0) >= width)) return t;
  return t.contiguous();
}

int64_t rowStride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const int32_t* ints(const Tensor& t) { return t.const_data_ptr<int32_t>(); }

// Gradients of first order: what comes out of a backward pass cannot be differentiated again, and says so when it is tried.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();  // the error node is only reached through tensors that want a gradient
  auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of spnc.mixture cannot be differentiated again", int64_t(grads.size()));
  return (*error)(std::move(grads));
}

struct Plan {
  Tensor position, starts, counts;
  int64_t capacity;
  int64_t rows() const { return position.size(0); }
  unsigned k() const { return unsigned(position.size(1)); }
  unsigned experts() const { return unsigned(counts.size(0)); }
};

void checkExperts(int64_t experts) {
  refuse(experts < 1 || experts > int64_t(SPNC_HIP_MAX_EXPERTS), "The number of experts must be between 1 and ", SPNC_HIP_MAX_EXPERTS, ", got ", experts);
}

Plan planOf(const Tensor& position, const Tensor& starts, const Tensor& counts, int64_t capacity) {
  auto shaped = [](const Tensor& t, int64_t dim, const char* name) {
    refuse(t.scalar_type() != at::kInt || t.dim() != dim || !t.is_contiguous(), name, " must be a contiguous int32 tensor of ", dim, " dimensions");
  };
  shaped(position, 2, "position");
  shaped(starts, 1, "starts");
  shaped(counts, 1, "counts");
  refuse(position.size(1) < 1, "A row must have at least one slot");
  refuse(starts.size(0) != counts.size(0) + 1, "starts must have one entry more than counts");
  checkExperts(counts.size(0));
  refuse(capacity < 0 || capacity >= ROWS_LIMIT, "The capacity must be below 2^31, got ", capacity);
  return {position, starts, counts, capacity};
}

// ---- gate -----------------------------------------------------------------------------------------------------------

// Rows of logits a million elements and more apart are copied.
Tensor logitsOf(const Tensor& t) {
  const Tensor rows = rowsOf(t);
  return rowStride(rows) < 1 << 20 ? rows : rows.contiguous();
}

std::pair<Tensor, Tensor> gateForward(const Tensor& given, int64_t k, int64_t flags) {
  c10::DeviceGuard guard(given.device());
  const Tensor logits = logitsOf(given);
  const int64_t n = logits.size(0);
  Tensor index = at::empty({n, k}, logits.options().dtype(at::kInt).requires_grad(false));
  Tensor weight = at::empty({n, k}, index.options().dtype(logits.scalar_type() == at::kDouble ? at::kDouble : at::kFloat));
  check(spnc_hip_gate(data(logits), elementType(logits.scalar_type()), n, unsigned(logits.size(1)), rowStride(logits), unsigned(k), unsigned(flags),
                      index.mutable_data_ptr<int32_t>(), out(weight), streamOf(logits)));
  return {index, weight};
}

struct Gate : torch::autograd::Function<Gate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k, int64_t flags) {
    auto [index, weight] = gateForward(logits, k, flags);
    ctx->saved_data["flags"] = flags;
    ctx->saved_data["experts"] = logits.size(1);
    ctx->saved_data["type"] = int64_t(logits.scalar_type());
    ctx->save_for_backward({(flags & SPNC_HIP_GATE_ALL) ? logits : Tensor(), index, weight});
    ctx->mark_non_differentiable({index});
    return {index, weight};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    checkRecorded({&grads[1]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &index = saved[1], &weight = saved[2];
    c10::DeviceGuard guard(index.device());
    const Tensor logits = saved[0].defined() ? logitsOf(saved[0]) : Tensor(), grad = flat(grads[1]);
    const int64_t flags = ctx->saved_data["flags"].toInt(), experts = ctx->saved_data["experts"].toInt();
    const auto type = at::ScalarType(ctx->saved_data["type"].toInt());
    Tensor result = at::empty({index.size(0), experts}, weight.options().dtype(type).requires_grad(false));
    check(spnc_hip_gate_backward(data(logits), elementType(type), index.size(0), unsigned(experts), logits.defined() ? rowStride(logits) : experts,
                                 unsigned(index.size(1)), unsigned(flags), ints(index), data(weight), data(grad), out(result), streamOf(index)));
    return once({result, Tensor(), Tensor()});
  }
};

std::pair<Tensor, Tensor> gate(const Tensor& logits, int64_t k, int64_t flags) {
  refuse(logits.dim() != 2, "Logits must have shape [rows, experts], got ", logits.sizes());
  refuse(elementType(logits.scalar_type()) < 0, "Logits must be float32, float64, float16 or bfloat16, got ", logits.scalar_type());
  const int64_t experts = logits.size(1), most = std::min<int64_t>(experts, SPNC_HIP_MAX_CHOICES);
  checkExperts(experts);
  refuse(k < 1 || k > most, "k must be between 1 and ", most, ", got ", k);
  checkRecorded({&logits});
  onGpu({&logits});
  if (!wantsGrad({&logits})) return gateForward(logits, k, flags);
  auto r = Gate::apply(logits, k, flags);
  return {r[0], r[1]};
}

// ---- routing --------------------------------------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor, int64_t> route(const Tensor& given, int64_t experts, int64_t align) {
  refuse(given.dim() != 2 || given.scalar_type() != at::kInt || given.size(1) < 1, "The index must be int32 [rows, choices], got ", given.scalar_type(),
         " ", given.sizes());
  checkExperts(experts);
  refuse(align < 1, "align must be at least 1, got ", align);
  const int64_t slots = given.numel();
  refuse(slots >= ROWS_LIMIT || align > ROWS_LIMIT || slots + experts * (align - 1) >= ROWS_LIMIT, slots, " slots and ", experts, " segments aligned to ",
         align, " rows exceed 2^31 rows");
  checkRecorded({});
  onGpu({&given});
  c10::DeviceGuard guard(given.device());
  const Tensor index = given.contiguous();
  const auto options = index.options();
  Tensor position = at::empty(index.sizes(), options), starts = at::empty({experts + 1}, options), counts = at::empty({experts}, options), workspace;
  const size_t bytes = spnc_hip_route_workspace(slots, unsigned(experts));
  if (bytes) workspace = at::empty({int64_t(bytes)}, options.dtype(at::kByte));
  check(spnc_hip_route(ints(index), slots, unsigned(experts), unsigned(align), position.mutable_data_ptr<int32_t>(), starts.mutable_data_ptr<int32_t>(),
                       counts.mutable_data_ptr<int32_t>(), out(workspace), bytes, streamOf(index)));
  return {position, starts, counts, slots + experts * (align - 1)};
}

Tensor dispatchForward(const Tensor& given, const Plan& plan, Tensor result, bool clear) {
  c10::DeviceGuard guard(given.device());
  const Tensor rows = rowsOf(given);
  const int64_t size = int64_t(rows.element_size()), width = rows.size(1);
  if (!result.defined()) result = at::empty({plan.capacity, width}, rows.options().requires_grad(false));
  check(spnc_hip_dispatch(data(rows), rows.size(0), width * size, rowStride(rows) * size, ints(plan.position), plan.k(), plan.capacity, ints(plan.starts),
                          ints(plan.counts), plan.experts(), clear, out(result), streamOf(rows)));
  return result;
}

Tensor combineForward(const Tensor& given, const Plan& plan, const Tensor& weights) {
  c10::DeviceGuard guard(given.device());
  const Tensor values = rowsOf(given);
  Tensor result = at::empty({plan.rows(), values.size(1)}, values.options().requires_grad(false));
  check(spnc_hip_combine(data(values), elementType(values.scalar_type()), plan.capacity, values.size(1), rowStride(values), ints(plan.position),
                         plan.rows(), plan.k(), data(weights), weights.defined() ? elementType(weights.scalar_type()) : 0, out(result), streamOf(values)));
  return result;
}

// The plan's tensors are saved with the others: writing to them between the passes is an error, not another gradient.
variable_list savedWith(const Plan& plan, variable_list tensors) {
  tensors.insert(tensors.end(), {plan.position, plan.starts, plan.counts});
  return tensors;
}

Plan savedPlan(AutogradContext* ctx, const variable_list& saved) {
  const size_t n = saved.size();
  return {saved[n - 3], saved[n - 2], saved[n - 1], ctx->saved_data["capacity"].toInt()};
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Plan& plan) {
    ctx->saved_data["capacity"] = plan.capacity;
    ctx->save_for_backward(savedWith(plan, {}));
    return dispatchForward(rows, plan, Tensor(), true);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    checkRecorded({&grads[0]});
    return once({combineForward(grads[0], savedPlan(ctx, ctx->get_saved_variables()), Tensor()), Tensor()});
  }
};

Tensor dispatch(const Tensor& rows, const Tensor& position, const Tensor& starts, const Tensor& counts, int64_t capacity,
                const std::optional<Tensor>& result) {
  const Plan plan = planOf(position, starts, counts, capacity);
  refuse(rows.dim() != 2, "Rows must have shape [rows, width], got ", rows.sizes());
  refuse(rows.size(0) != plan.rows(), "The plan is for ", plan.rows(), " rows, got ", rows.size(0));
  refuse(rows.element_size() > 8 || rows.is_complex(), "Rows of ", rows.scalar_type(), " are not supported");
  checkRecorded({&rows});
  if (result) {
    checkRecorded({&*result});
    refuse(result->dim() != 2 || result->size(0) != capacity || result->size(1) != rows.size(1) || result->scalar_type() != rows.scalar_type() ||
               !result->is_contiguous() || result->is_neg(),
           "out must be a contiguous ", rows.scalar_type(), " tensor of shape [", capacity, ", ", rows.size(1), "]");
    // views that this cannot tell are either told apart behind the C-ABI, which knows the rows' strides, or copied first
    for (const Tensor* read : {&rows, &position, &starts, &counts}) {
      const auto status = at::get_overlap_status(*result, *read);
      refuse(status == at::MemOverlapStatus::Full || status == at::MemOverlapStatus::Partial, "out must not share memory with the rows or the plan");
    }
    refuse(wantsGrad({&rows, &*result}), "dispatch with out= has no gradient; call it without");
    onGpu({&rows, &position, &starts, &counts, &*result});
    torch::autograd::impl::bump_version(*result);  // whoever saved the buffer for a backward pass learns that it was written to
    return dispatchForward(rows, plan, *result, false);
  }
  onGpu({&rows, &position, &starts, &counts});
  if (!wantsGrad({&rows})) return dispatchForward(rows, plan, Tensor(), true);
  refuse(elementType(rows.scalar_type()) < 0, "Rows of ", rows.scalar_type(), " have no gradient");
  return Dispatch::apply(rows, plan);
}

// ---- combination ----------------------------------------------------------------------------------------------------

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& values, const std::optional<Tensor>& given, const Plan& plan) {
    const Tensor weights = given.value_or(Tensor());
    ctx->saved_data["capacity"] = plan.capacity;
    ctx->save_for_backward(savedWith(plan, {values, weights}));
    return combineForward(values, plan, weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    checkRecorded({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Plan plan = savedPlan(ctx, saved);
    const Tensor& weights = saved[1];
    c10::DeviceGuard guard(grads[0].device());
    const Tensor values = rowsOf(saved[0]), grad = rowsOf(grads[0]);
    if (!weights.defined()) return once({dispatchForward(grad, plan, Tensor(), true), Tensor(), Tensor()});
    Tensor gradValues, gradWeights;
    if (ctx->needs_input_grad(0)) gradValues = at::empty({plan.capacity, values.size(1)}, values.options().requires_grad(false));
    if (ctx->needs_input_grad(1)) gradWeights = at::empty(weights.sizes(), weights.options().requires_grad(false));
    check(spnc_hip_combine_backward(data(values), elementType(values.scalar_type()), plan.capacity, values.size(1), rowStride(values), ints(plan.position),
                                    plan.rows(), plan.k(), data(weights), elementType(weights.scalar_type()), data(grad), rowStride(grad), ints(plan.starts),
                                    ints(plan.counts), plan.experts(), out(gradValues), out(gradWeights), streamOf(values)));
    return once({gradValues, gradWeights, Tensor()});
  }
};

void checkWeights(const Tensor& weights, const Plan& plan, bool doubles) {
  refuse(weights.sizes() != plan.position.sizes(), "Weights must have shape ", plan.position.sizes(), ", got ", weights.sizes());
  refuse(weights.scalar_type() != at::kFloat && !(doubles && weights.scalar_type() == at::kDouble), "Weights must be float32",
         doubles ? " or float64" : "", ", got ", weights.scalar_type());
}

Tensor combine(const Tensor& values, const Tensor& position, const Tensor& starts, const Tensor& counts, int64_t capacity,
               const std::optional<Tensor>& given) {
  const Plan plan = planOf(position, starts, counts, capacity);
  refuse(values.dim() != 2 || values.size(0) != capacity, "Values must have shape [", capacity, ", width], got ", values.sizes());
  refuse(elementType(values.scalar_type()) < 0, "Values must be float32, float64, float16 or bfloat16, got ", values.scalar_type());
  checkRecorded({&values});
  Tensor weights;
  if (given) {
    checkRecorded({&*given});
    checkWeights(*given, plan, values.scalar_type() == at::kDouble);
    onGpu({&values, &position, &starts, &counts, &*given});
    weights = flat(*given);
  } else {
    onGpu({&values, &position, &starts, &counts});
  }
  if (!wantsGrad({&values, &weights})) return combineForward(values, plan, weights);
  return Combine::apply(values, weights.defined() ? std::optional<Tensor>(weights) : std::nullopt, plan);
}

Tensor combineLogForward(const Tensor& values, const Plan& plan, const Tensor& weights, const Tensor& share) {
  c10::DeviceGuard guard(values.device());
  Tensor result = at::empty({plan.rows()}, values.options().requires_grad(false));
  check(spnc_hip_combine_log(data(values), elementType(values.scalar_type()), plan.capacity, ints(plan.position), plan.rows(), plan.k(), data(weights),
                             elementType(weights.scalar_type()), out(result), out(share), streamOf(values)));
  return result;
}

struct CombineLog : torch::autograd::Function<CombineLog> {
  static Tensor forward(AutogradContext* ctx, const Tensor& values, const Tensor& weights, const Plan& plan) {
    c10::DeviceGuard guard(values.device());
    const Tensor share = at::empty(weights.sizes(), values.options().requires_grad(false));
    ctx->saved_data["capacity"] = plan.capacity;
    ctx->saved_data["weights"] = int64_t(weights.scalar_type());
    ctx->save_for_backward(savedWith(plan, {share}));
    return combineLogForward(values, plan, weights, share);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    checkRecorded({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Plan plan = savedPlan(ctx, saved);
    const Tensor& share = saved[0];
    c10::DeviceGuard guard(share.device());
    const auto type = at::ScalarType(ctx->saved_data["weights"].toInt());
    const Tensor grad = flat(grads[0]);
    Tensor gradValues, gradWeights;
    if (ctx->needs_input_grad(0)) gradValues = at::empty({plan.capacity}, share.options());
    if (ctx->needs_input_grad(1)) gradWeights = at::empty(share.sizes(), share.options().dtype(type));
    check(spnc_hip_combine_log_backward(data(share), elementType(share.scalar_type()), plan.capacity, ints(plan.position), plan.rows(), plan.k(),
                                        elementType(type), data(grad), ints(plan.starts), ints(plan.counts), plan.experts(), out(gradValues),
                                        out(gradWeights), streamOf(share)));
    return once({gradValues, gradWeights, Tensor()});
  }
};

Tensor combineLog(const Tensor& given, const Tensor& position, const Tensor& starts, const Tensor& counts, int64_t capacity, const Tensor& logWeights) {
  const Plan plan = planOf(position, starts, counts, capacity);
  refuse(given.dim() != 1 || given.size(0) != capacity, "Values must have shape [", capacity, "], got ", given.sizes());
  refuse(given.scalar_type() != at::kFloat && given.scalar_type() != at::kDouble, "Values must be float32 or float64, got ", given.scalar_type());
  checkWeights(logWeights, plan, true);
  checkRecorded({&given, &logWeights});
  onGpu({&given, &position, &starts, &counts, &logWeights});
  const Tensor values = flat(given), weights = flat(logWeights);
  if (!wantsGrad({&values, &weights})) return combineLogForward(values, plan, weights, Tensor());
  return CombineLog::apply(values, weights, plan);
}

// ---- dropout --------------------------------------------------------------------------------------------------------

struct Mask {
  double p;
  int64_t mode;
  uint64_t seed, offset;
  Tensor offsetDevice;
};

Tensor dropoutForward(const Tensor& given, const Mask& mask) {
  if (given.numel() == 0) return at::empty(given.sizes(), given.options().requires_grad(false));
  c10::DeviceGuard guard(given.device());
  const Tensor x = rowsOf(given.dim() == 2 ? given : given.dim() < 2 ? given.reshape({1, -1}) : given.reshape({-1, given.size(-1)}));
  Tensor result = at::empty(given.sizes(), given.options().requires_grad(false));
  check(spnc_hip_dropout(data(x), elementType(x.scalar_type()), x.size(0), x.size(1), rowStride(x), out(result), x.size(1), mask.p, int(mask.mode), mask.seed,
                         mask.offset, static_cast<const uint64_t*>(data(mask.offsetDevice)), streamOf(x)));
  return result;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Mask& mask) {
    ctx->saved_data["p"] = mask.p;
    ctx->saved_data["mode"] = mask.mode;
    ctx->saved_data["seed"] = int64_t(mask.seed);
    ctx->saved_data["offset"] = int64_t(mask.offset);
    if (mask.offsetDevice.defined()) ctx->save_for_backward({mask.offsetDevice});  // the mask must be the same: a change in between is an error
    return dropoutForward(x, mask);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    checkRecorded({&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const int64_t mode = ctx->saved_data["mode"].toInt();
    const Mask mask{ctx->saved_data["p"].toDouble(), mode == SPNC_HIP_DROPOUT_MARGINAL ? int64_t(SPNC_HIP_DROPOUT_MASK) : mode,
                    uint64_t(ctx->saved_data["seed"].toInt()), uint64_t(ctx->saved_data["offset"].toInt()), saved.empty() ? Tensor() : saved[0]};
    return once({dropoutForward(grads[0], mask), Tensor()});
  }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const std::optional<Tensor>& offsetDevice, bool marginal) {
  refuse(elementType(x.scalar_type()) < 0, "x must be float32, float64, float16 or bfloat16, got ", x.scalar_type());
  checkRecorded({&x});
  Mask mask{p, marginal ? SPNC_HIP_DROPOUT_MARGINAL : SPNC_HIP_DROPOUT_ZERO, seed, offset, Tensor()};
  if (offsetDevice) {
    refuse(offsetDevice->scalar_type() != at::kLong || offsetDevice->numel() != 1, "An offset on the device must be a one-element int64 tensor");
    mask.offsetDevice = *offsetDevice;
    onGpu({&x, &mask.offsetDevice});
  } else {
    onGpu({&x});
  }
  if (!wantsGrad({&x})) return dropoutForward(x, mask);
  return Dropout::apply(x, mask);
}

}  // namespace

PYBIND11_MODULE(_mixture_ops, m) {
  m.def("check_recorded", [](const Tensor& t) { checkRecorded({&t}); });
  m.def("gate", &gate);
  m.def("route", &route);
  m.def("check_plan", [](const Tensor& position, const Tensor& starts, const Tensor& counts, int64_t capacity) { planOf(position, starts, counts, capacity); });
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("combine_log", &combineLog);
  m.def("dropout", &dropout);
}
