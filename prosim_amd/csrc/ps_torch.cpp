// prosim_amd/_finetune.so -- the fine-tuning operators (include/prosim_hip.h) on torch tensors, with their gradients.
//
// Host code only.  The engine's entry points take numpy arrays and run for milliseconds, so engine.py binds them with ctypes; these run for
// microseconds inside an autograd step, where a Python binding costs more than the kernels.  Everything a wrong argument can do is refused here,
// before a launch; what passes goes to the C ABI on the current stream of the tensors' device.
#include <torch/extension.h>

#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "prosim_hip.h"

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

const char* type_name(const Tensor& t) { return c10::toString(t.scalar_type()); }

// Is the tensor's memory what the tensor says?  (the imaginary part of a conjugate is a view whose sign is a flag; torch's efficient zeros have no memory)
bool as_stored(const Tensor& t) { return !t.is_neg() && !t._is_zerotensor(); }
void check_gpu(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.layout() == at::kStrided, name, ": expected a dense tensor on the GPU, got one on ", t.device(), " (", t.layout(), ")");
  TORCH_CHECK_VALUE(as_stored(t), name, ": a lazily negated or zero tensor: clone() it");
}
// an incoming gradient as dense memory
Tensor incoming(const Tensor& g) { return (as_stored(g) ? g : g.clone()).contiguous(); }
void check_gpu(const Tensor& t, const char* name, const Tensor& like) {
  check_gpu(t, name);
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", the other tensors are on ", like.device());
}
int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PS_F32;
    case at::kBFloat16: return PS_BF16;
    case at::kHalf: return PS_F16;
    default: return -1;
  }
}
Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type = at::kFloat) { return at::empty(sizes, at::TensorOptions().device(like.device()).dtype(type)); }
template <typename T> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check(int rc) {
  if (rc == PS_OK) return;
  if (rc == PS_E_ARG) TORCH_CHECK_VALUE(false, "prosim_hip error ", rc, ": ", ps_last_error());
  TORCH_CHECK(false, "prosim_hip error ", rc, ": ", ps_last_error());
}

// A float32 constant of the rows' shape as dense memory.
Tensor constant(const Tensor& t, const char* name, at::IntArrayRef shape, const Tensor& like, bool broadcast = false) {
  check_gpu(t, name, like);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, ": expected float32, got ", type_name(t));
  const bool same = t.sizes() == shape;
  TORCH_CHECK_VALUE(same || (broadcast && at::is_expandable_to(t.sizes(), shape)), name, ": expected shape ", shape, ", got ", t.sizes());
  if (same && t.is_contiguous()) return t;
  const at::NoGradGuard quiet;      // (a layout copy is no part of the graph)
  return t.expand(shape).contiguous();
}
Tensor mask_of(const Maybe& m, const char* name, at::IntArrayRef shape, const Tensor& like) {
  if (!m) return Tensor();
  check_gpu(*m, name, like);
  TORCH_CHECK_TYPE(m->scalar_type() == at::kBool || m->scalar_type() == at::kByte, name, ": expected bool or uint8, got ", type_name(*m));
  TORCH_CHECK_VALUE(m->sizes() == shape, name, ": expected shape ", shape, ", got ", m->sizes());
  return m->contiguous();
}

// The one stride at which the rows of [..., K] lie, or -1: they have to be copied.
int64_t row_stride(const Tensor& t) {
  const int64_t k = t.size(-1);
  if (t.is_contiguous()) return k;
  if (t.stride(-1) != 1 && k != 1) return -1;
  int64_t step = -1, span = 0;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (step < 0) {
      if (t.stride(d) < k) return -1;
      step = t.stride(d);
      span = step;
    } else if (t.stride(d) != span) {
      return -1;
    }
    span *= t.size(d);
  }
  return step < 0 ? k : step;
}

// Rows of decisions that have passed the checks.  `held` keeps a copy of the rows alive until the launch is enqueued.
struct Decisions {
  Tensor held, choice, mask;
  ps_decisions d;
  Decisions(const Tensor& logits, const Tensor& choice_, const Tensor& mask_) : held(logits), choice(choice_), mask(mask_) {
    int64_t stride = row_stride(held);
    if (stride < 0) {
      held = held.contiguous();
      stride = held.size(-1);
    }
    d = ps_decisions{held.data_ptr(), choice.numel(), held.size(-1), stride, dtype_of(held), choice.scalar_type() == at::kLong ? 64 : 32, choice.data_ptr(), ptr<uint8_t>(mask)};
  }
};
// (choice, mask) as dense memory
std::pair<Tensor, Tensor> check_decisions(const Tensor& logits, const Tensor& choice, const Maybe& mask) {
  check_gpu(logits, "logits");
  TORCH_CHECK_TYPE(dtype_of(logits) >= 0, "logits: expected float32, bfloat16 or float16, got ", type_name(logits));
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) < (1LL << 31), "logits: expected [..., choices] with at least one choice, got shape ", logits.sizes());
  const at::IntArrayRef shape = logits.sizes().slice(0, logits.dim() - 1);
  check_gpu(choice, "choice", logits);
  TORCH_CHECK_TYPE(choice.scalar_type() == at::kInt || choice.scalar_type() == at::kLong, "choice: expected int32 or int64, got ", type_name(choice));
  TORCH_CHECK_VALUE(choice.sizes() == shape, "choice: expected shape ", shape, ", got ", choice.sizes());
  return {choice.contiguous(), mask_of(mask, "mask", shape, logits)};
}
int reduction_of(const std::string& name) {
  TORCH_CHECK_VALUE(name == "mean" || name == "sum", "reduction: expected 'mean' or 'sum', got '", name, "'");
  return name == "mean";
}

// A gradient of a gradient is an error, not a silent zero.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  return (*std::make_shared<torch::autograd::DelayedError>("prosim_amd.finetune: the operators are differentiable once", (int64_t)grads.size()))(std::move(grads));
}

// What a call keeps on the device besides its results, in one piece: workspace | (maximum, 1 / sum) per row | coefficient per row
struct Space {
  Tensor all;
  int64_t bytes;
  float *stat = nullptr, *coef = nullptr;
  Space(const Decisions& r, bool keep) : bytes((ps_choice_workspace(&r.d) + 7) / 8 * 8) {
    const int64_t n = r.d.rows;
    all = empty({bytes + (keep ? 12 * n : 0)}, r.held, at::kByte);
    if (keep) {
      stat = (float*)((char*)all.data_ptr() + bytes);
      coef = stat + 2 * n;
    }
  }
};

Tensor choice_grad(const Tensor& logits, const Tensor& choice, const Tensor& mask, const float* stat, const float* coef, const float* gain, Tensor done) {
  const Decisions r(logits, choice, mask);
  const bool ready = done.defined();
  Tensor grad = ready ? std::move(done) : empty(logits.sizes(), logits, logits.scalar_type());
  check(ps_choice_grad(&r.d, coef, stat, gain, ready, grad.data_ptr(), stream_of(logits)));
  return grad;
}

// What travels beside the differentiable inputs (torch's function objects take no undefined tensors as inputs).
struct Rest { Tensor choice, mask; };

// ---- log-probability of a choice ----
Tensor logp_forward(const Decisions& r, const Space& space) {
  Tensor logp = empty(r.choice.sizes(), r.held);
  check(ps_choice_logp(&r.d, ptr<float>(logp), space.stat, space.all.data_ptr(), space.bytes, stream_of(r.held)));
  return logp;
}
struct ChoiceLogp : torch::autograd::Function<ChoiceLogp> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Rest& rest) {
    const Decisions r(logits, rest.choice, rest.mask);
    const Space space(r, true);
    Tensor logp = logp_forward(r, space);
    ctx->save_for_backward({logits, rest.choice, rest.mask, space.all});
    return logp;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    const Tensor coef = incoming(grads[0]);
    const int64_t n = s[1].numel();
    return once({choice_grad(s[0], s[1], s[2], (float*)((char*)s[3].data_ptr() + s[3].numel() - 12 * n), ptr<float>(coef), nullptr, Tensor()), Tensor()});
  }
};
Tensor choice_logp(const Tensor& logits, const Tensor& choice, const Maybe& mask) {
  const auto [c, m] = check_decisions(logits, choice, mask);
  const c10::DeviceGuard guard(logits.device());
  if (logits.requires_grad() && at::GradMode::is_enabled()) return ChoiceLogp::apply(logits, Rest{c, m});
  const Decisions r(logits, c, m);
  return logp_forward(r, Space(r, false));
}

// ---- clipped policy loss ----
variable_list policy_forward(const Decisions& r, const ps_policy_terms& terms, const Space& space, const Tensor& grad) {
  Tensor loss = empty({}, r.held), kl = empty({}, r.held), frac = empty({}, r.held), logp = empty(r.choice.sizes(), r.held);
  check(ps_policy_loss(&r.d, &terms, ptr<float>(loss), ptr<float>(kl), ptr<float>(frac), ptr<float>(logp), space.stat, space.coef, ptr<void>(grad), space.all.data_ptr(), space.bytes,
                       stream_of(r.held)));
  return {loss, logp, kl, frac};
}
// The gradient is written by the forward pass, which has the row at hand once its sum is known (one read of the logits instead of two); the backward
// pass finds it ready when the incoming gradient is 1 and computes it afresh from the rows' statistics otherwise.
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Rest& rest, const ps_policy_terms& terms) {
    const Decisions r(logits, rest.choice, rest.mask);
    const Space space(r, true);
    const Tensor grad = empty(logits.sizes(), logits, logits.scalar_type());
    variable_list out = policy_forward(r, terms, space, grad);
    ctx->saved_data["ready"] = grad;
    ctx->save_for_backward({logits, rest.choice, rest.mask, space.all});
    ctx->mark_non_differentiable({out[1], out[2], out[3]});
    ctx->set_materialize_grads(false);        // (no zeros for the three numbers that carry no gradient)
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    Tensor ready;
    const auto it = ctx->saved_data.find("ready");
    if (it != ctx->saved_data.end()) {        // (handed out once: a second backward pass of a retained graph computes its own)
      ready = it->second.toTensor();
      ctx->saved_data.erase(it);
    }
    const Tensor gain = incoming(grads[0]);
    const int64_t n = s[1].numel();
    const float* stat = (float*)((char*)s[3].data_ptr() + s[3].numel() - 12 * n);
    return once({choice_grad(s[0], s[1], s[2], stat, stat + 2 * n, ptr<float>(gain), ready), Tensor(), Tensor()});
  }
};
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& choice, const Tensor& old_logp, const Tensor& advantage, const Maybe& ref_logp, const Maybe& mask,
                                                       double clip_low, std::optional<double> clip_high, double kl_coef, const std::string& reduction, double scale) {
  const auto [c, m] = check_decisions(logits, choice, mask);
  const Tensor old_ = constant(old_logp, "old_logp", c.sizes(), logits), adv = constant(advantage, "advantage", c.sizes(), logits, true);
  const Tensor ref = ref_logp ? constant(*ref_logp, "ref_logp", c.sizes(), logits) : Tensor();
  TORCH_CHECK_VALUE(!(kl_coef > 0) || ref.defined(), "kl_coef > 0 needs ref_logp");
  const ps_policy_terms terms{ptr<float>(old_), ptr<float>(adv), ptr<float>(ref), clip_low, clip_high.value_or(clip_low), kl_coef, scale, reduction_of(reduction)};
  const c10::DeviceGuard guard(logits.device());
  variable_list out;
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    out = PolicyLoss::apply(logits, Rest{c, m}, terms);
  } else {
    const Decisions r(logits, c, m);
    out = policy_forward(r, terms, Space(r, false), Tensor());
  }
  return {out[0], out[1], out[2], out[3]};
}

// ---- preference loss ----
struct Side { Tensor logp, ref, mask; };
struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& better, const Tensor& worse, const Side& b, const Side& w, const ps_preference& q) {
    Tensor loss = empty({}, better), margin = empty({q.pairs}, better);
    const int64_t bytes = ps_preference_loss_workspace(q.pairs);
    const Tensor space = empty({bytes + 4 * q.pairs}, better, at::kByte);       // workspace | d loss / d h per pair
    float* coef = (float*)((char*)space.data_ptr() + bytes);
    check(ps_preference_loss(&q, ptr<float>(loss), ptr<float>(margin), coef, space.data_ptr(), bytes, stream_of(better)));
    ctx->save_for_backward({space, b.mask, w.mask});
    ctx->saved_data["shapes"] = std::vector<int64_t>{q.pairs, better.dim() == 2 ? q.better_steps : -1, worse.dim() == 2 ? q.worse_steps : -1};      // (-1: [pairs])
    ctx->mark_non_differentiable({margin});
    ctx->set_materialize_grads(false);
    return {loss, margin};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    const std::vector<int64_t> shapes = ctx->saved_data["shapes"].toIntVector();
    const int64_t pairs = shapes[0];
    Tensor out[2];
    for (int i = 0; i < 2; ++i)
      if (ctx->needs_input_grad(i)) out[i] = shapes[1 + i] < 0 ? empty({pairs}, s[0]) : empty({pairs, shapes[1 + i]}, s[0]);
    ps_preference q{};
    q.better_mask = ptr<uint8_t>(s[1]);
    q.worse_mask = ptr<uint8_t>(s[2]);
    q.pairs = pairs;
    q.better_steps = shapes[1] < 0 ? 1 : shapes[1];
    q.worse_steps = shapes[2] < 0 ? 1 : shapes[2];
    const Tensor gain = incoming(grads[0]);
    check(ps_preference_grad(&q, (float*)((char*)s[0].data_ptr() + s[0].numel() - 4 * pairs), ptr<float>(gain), ptr<float>(out[0]), ptr<float>(out[1]), stream_of(s[0])));
    return once({out[0], out[1], Tensor(), Tensor(), Tensor()});
  }
};
std::tuple<Tensor, Tensor> preference_loss(const Tensor& better, const Tensor& worse, const Maybe& better_ref, const Maybe& worse_ref, const Maybe& better_mask, const Maybe& worse_mask,
                                           double beta, double label_smoothing, const std::string& reduction, double scale) {
  check_gpu(better, "better");
  check_gpu(worse, "worse", better);
  TORCH_CHECK_VALUE((better.dim() == 1 || better.dim() == 2) && (worse.dim() == 1 || worse.dim() == 2) && better.size(0) == worse.size(0) && better.size(0) >= 1,
                    "better / worse: expected [pairs, steps] or [pairs] with the same pairs >= 1, got ", better.sizes(), " and ", worse.sizes());
  const Side b{constant(better, "better", better.sizes(), better), better_ref ? constant(*better_ref, "better_ref", better.sizes(), better) : Tensor(),
               mask_of(better_mask, "better_mask", better.sizes(), better)};
  const Side w{constant(worse, "worse", worse.sizes(), better), worse_ref ? constant(*worse_ref, "worse_ref", worse.sizes(), better) : Tensor(),
               mask_of(worse_mask, "worse_mask", worse.sizes(), better)};
  const ps_preference q{ptr<float>(b.logp), ptr<float>(b.ref), ptr<float>(w.logp), ptr<float>(w.ref), ptr<uint8_t>(b.mask), ptr<uint8_t>(w.mask), better.size(0),
                        better.dim() == 2 ? better.size(1) : 1, worse.dim() == 2 ? worse.size(1) : 1, beta, label_smoothing, scale, reduction_of(reduction)};
  const c10::DeviceGuard guard(better.device());
  const variable_list out = PreferenceLoss::apply(better, worse, b, w, q);
  return {out[0], out[1]};
}

// ---- gradient clipping ----
// Every element of the tensor's stretch of memory belongs to it exactly once, in whatever order of dimensions.
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

Tensor clip_grads(const py::list& list, double max_norm, double eps) {
  std::vector<const Tensor*> ts;      // (the list keeps them)
  ts.reserve(list.size());
  for (Py_ssize_t i = 0, n = PyList_GET_SIZE(list.ptr()); i < n; ++i) {
    PyObject* o = PyList_GET_ITEM(list.ptr(), i);
    if (o == Py_None) continue;
    TORCH_CHECK_TYPE(THPVariable_Check(o), "grads: expected tensors, got ", Py_TYPE(o)->tp_name);
    ts.push_back(&THPVariable_Unpack(o));
  }
  TORCH_CHECK_VALUE(!ts.empty(), "clip_grads_: no gradients");
  const Tensor& like = *ts[0];
  check_gpu(like, "grads");
  // Ranges of memory, by address: that finds tensors on top of each other, and makes one range of neighbours -- data-parallel training keeps its
  // gradients as views of a few flat buffers, hundreds of tensors that are then a handful of ranges.
  struct Range { uintptr_t begin, end; int32_t dtype; };
  std::vector<Range> used;
  used.reserve(ts.size());
  bool sorted = true;
  for (const Tensor* p : ts) {
    const Tensor& t = *p;
    if (t.device() != like.device() || t.layout() != at::kStrided || !as_stored(t)) check_gpu(t, "grads", like);
    const int dtype = dtype_of(t);
    TORCH_CHECK_TYPE(dtype >= 0, "grads: expected float32, bfloat16 or float16, got ", type_name(t));
    TORCH_CHECK_VALUE(!t.requires_grad(), "grads: a tensor requires a gradient itself (parameters instead of their gradients?)");
    TORCH_CHECK_VALUE(dense(t), "grads: a tensor of shape ", t.sizes(), " and strides ", t.strides(), " is not dense");
    if (!t.numel()) continue;
    const uintptr_t begin = (uintptr_t)t.data_ptr();
    sorted = sorted && (used.empty() || used.back().begin <= begin);
    used.push_back(Range{begin, begin + t.numel() * t.element_size(), dtype});
  }
  if (!sorted) std::sort(used.begin(), used.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  std::vector<void*> at;
  std::vector<int64_t> numel;
  std::vector<int32_t> dtypes;
  for (size_t i = 0; i < used.size(); ++i) {
    const Range& r = used[i];
    const int64_t n = (r.end - r.begin) / (r.dtype == PS_F32 ? 4 : 2);
    TORCH_CHECK_VALUE(!i || used[i - 1].end <= r.begin, "grads: two tensors share memory");
    if (i && used[i - 1].end == r.begin && dtypes.back() == r.dtype) {
      numel.back() += n;
    } else {
      at.push_back((void*)r.begin);
      numel.push_back(n);
      dtypes.push_back(r.dtype);
    }
  }
  const int32_t n = (int32_t)at.size();
  const c10::DeviceGuard guard(like.device());
  const Tensor norm = empty({}, like), space = empty({ps_clip_grads_workspace(n, numel.data(), dtypes.data())}, like, at::kByte);
  check(ps_clip_grads(n, at.data(), numel.data(), dtypes.data(), max_norm, eps, ptr<float>(norm), space.data_ptr(), space.numel(), stream_of(like)));
  for (const Tensor* t : ts)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return norm;
}
}  // namespace

PYBIND11_MODULE(_finetune, m) {
  m.def("choice_logp", &choice_logp);
  m.def("policy_loss", &policy_loss);
  m.def("preference_loss", &preference_loss);
  m.def("clip_grads", &clip_grads);
  m.def("row_stride", &row_stride);
  m.def("dense", &dense);
}
