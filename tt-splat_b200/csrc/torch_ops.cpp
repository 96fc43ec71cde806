// The row lookup and the label scores as torch functions: argument checks, allocation on the current stream and
// the autograd nodes, over the C entry points.  In C++ because small training calls are bound by the host: a
// backward that torch's engine thread runs without Python takes half the time (4000 lookups of 16 fp32 and
// their gradient: 101 us by Python autograd functions, 61 us here, of which an empty C++ function takes 41).
#include <torch/extension.h>

#include <algorithm>
#include <string>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/ttsplat_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void check(int rc, const char* what) {
  if (rc == TTS_OK) return;
  TORCH_CHECK_VALUE(rc != TTS_ERR_INVALID, what, ": ", tts_last_error());
  TORCH_CHECK(false, what, ": ", tts_last_error(), " (code ", rc, ")");
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
void need_cuda(const Tensor& t) { TORCH_CHECK(t.is_cuda(), "tt-splat B200 ops need CUDA tensors (no CPU fallback)"); }
void same_device(const Tensor& t, const Tensor& as, const char* what) {
  need_cuda(t);
  TORCH_CHECK_VALUE(t.device() == as.device(), what, " is on ", t.device(), ", expected ", as.device());
}
// There are no forward-mode formulas: a tangent that went unseen would read as a derivative of zero.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what,
                              " has a forward-mode tangent: this function is differentiable in reverse mode only");
}
int row_type(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return TTS_ROW_F32;
    case at::kBFloat16: return TTS_ROW_BF16;
    case at::kHalf: return TTS_ROW_F16;
    default: TORCH_CHECK_TYPE(false, what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}
int index_type(const Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, what, " must be int32 or int64, got ",
                   t.scalar_type());
  return t.scalar_type() == at::kLong;
}
std::string shape_text(at::IntArrayRef s) {
  std::string text = "(";
  for (size_t i = 0; i < s.size(); ++i) text += (i ? ", " : "") + std::to_string(s[i]);
  return text + ")";
}
bool same_shape(at::IntArrayRef a, at::IntArrayRef b) {
  return a.size() == b.size() && std::equal(a.begin(), a.end(), b.begin());
}
Tensor of(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
template <class T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// The kernels read memory as it is: a tensor that only says that its numbers are negated (the imaginary part of
// a conjugate, and such gradients) is copied with them negated.
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// [n, width] view of a tensor's rows with unit stride along them (the kernels take any distance between rows
// below 2^30, an expanded row's included); a copy where no such view exists.
Tensor rows2d(const Tensor& t, int64_t n, int64_t width) {
  const Tensor r = t.dim() == 2 && t.size(0) == n && t.size(1) == width ? t : t.reshape({n, width});
  return (width <= 1 || r.stride(1) == 1) && (n <= 1 || r.stride(0) < (1ll << 30)) ? r : r.contiguous();
}
int64_t row_stride(const Tensor& rows) { return rows.size(0) <= 1 ? rows.size(1) : rows.stride(0); }
int64_t width_of(const Tensor& table) {
  int64_t w = 1;
  for (int64_t i = 1; i < table.dim(); ++i) w *= table.size(i);
  return w;
}

// Results of a backward that a graph was asked for: differentiating them again raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list live;
  for (Tensor& g : grads)
    if (g.defined()) live.push_back(g.detach().requires_grad_(true));
  if (live.empty()) return grads;
  auto refuse = std::make_shared<torch::autograd::DelayedError>("this function is differentiable once only",
                                                                 static_cast<int64_t>(live.size()));
  variable_list out = (*refuse)(std::move(live));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

// ---- rows ------------------------------------------------------------------------------------------

Tensor rows_forward(const Tensor& table, const Tensor& idx, const Tensor& valid, const Tensor& weight, double scale) {
  const c10::cuda::CUDAGuard guard(table.device());
  const int64_t R = table.size(0), C = width_of(table);
  const Tensor rows = rows2d(table, R, C);
  std::vector<int64_t> shape = idx.sizes().vec();
  for (int64_t i = 1; i < table.dim(); ++i) shape.push_back(table.size(i));
  Tensor out = at::empty(shape, table.options().requires_grad(false));
  check(tts_gather_rows(ptr<void>(rows), R, C, row_stride(rows), row_type(table, "table"), ptr<void>(idx),
                        index_type(idx, "idx"), ptr<uint8_t>(valid), ptr<float>(weight), static_cast<float>(scale),
                        idx.numel(), ptr<void>(out), stream()),
        "tts_gather_rows");
  return out;
}

// gtable [R, C] in gout's type and gweight in idx's shape, each undefined when not wanted.
std::tuple<Tensor, Tensor> rows_backward(const Tensor& table, int64_t R, int64_t C, const Tensor& idx, const Tensor& valid,
                                         const Tensor& weight, double scale, const Tensor& gout, bool want_table,
                                         bool want_weight) {
  const c10::cuda::CUDAGuard guard(gout.device());
  const int64_t N = idx.numel();
  const Tensor go = rows2d(gout, N, C);
  const Tensor rows = table.defined() ? rows2d(table, R, C) : Tensor();
  Tensor gtable, gweight, ws;
  size_t bytes = 0;
  if (want_table) {
    gtable = at::empty({R, C}, gout.options().requires_grad(false));
    bytes = tts_gather_rows_bwd_workspace_bytes(N, R, C);
    ws = at::empty({static_cast<int64_t>(bytes)}, gout.options().dtype(at::kByte).requires_grad(false));
  }
  if (want_weight) gweight = at::empty(idx.sizes(), idx.options().dtype(at::kFloat));
  check(tts_gather_rows_bwd(ptr<void>(rows), R, C, rows.defined() ? row_stride(rows) : 0, row_type(gout, "gout"),
                            ptr<void>(idx), index_type(idx, "idx"), ptr<uint8_t>(valid), ptr<float>(weight),
                            static_cast<float>(scale), N, ptr<void>(go), row_stride(go), ptr<void>(gtable),
                            ptr<float>(gweight), ptr<void>(ws), bytes, stream()),
        "tts_gather_rows_bwd");
  return {gtable, gweight};
}

struct GatherRows : torch::autograd::Function<GatherRows> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const OptTensor& weight_, const Tensor& idx,
                        const OptTensor& valid_, double scale) {
    const Tensor weight = of(weight_), valid = of(valid_);
    const bool gw = weight.defined() && weight.requires_grad();
    ctx->save_for_backward({gw ? table : Tensor(), weight, idx, valid});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["shape"] = table.sizes().vec();
    return rows_forward(table, idx, valid, weight, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    // what this call asks for, not all that could be asked for (an absent weight has no place among the inputs)
    const bool want_table = ctx->needs_input_grad(0), want_weight = s[1].defined() && ctx->needs_input_grad(1);
    int64_t C = 1;
    for (size_t i = 1; i < shape.size(); ++i) C *= shape[i];
    variable_list out(5);
    if (!grads[0].defined()) return out;
    no_tangent(grads[0], "the rows' gradient");
    std::tie(out[0], out[1]) = rows_backward(s[0], shape[0], C, s[2], s[3], s[1], ctx->saved_data["scale"].toDouble(),
                                             plain(grads[0]), want_table, want_weight);
    if (out[0].defined() && shape.size() != 2) out[0] = out[0].view(shape);
    return once(std::move(out));
  }
};

Tensor gather_rows(const Tensor& table_, const Tensor& idx_, const OptTensor& valid_, const OptTensor& weight_, double scale) {
  TORCH_CHECK_VALUE(table_.dim() >= 1, "table must have at least one dimension");
  row_type(table_, "table");
  index_type(idx_, "idx");
  Tensor valid = of(valid_), weight = of(weight_);
  if (valid.defined()) {
    TORCH_CHECK_TYPE(valid.scalar_type() == at::kBool || valid.scalar_type() == at::kByte,
                     "valid must be bool or uint8, got ", valid.scalar_type());
    TORCH_CHECK_VALUE(same_shape(valid.sizes(), idx_.sizes()), "valid must have the shape of idx ",
                      shape_text(idx_.sizes()), ", got ", shape_text(valid.sizes()));
  }
  if (weight.defined()) {
    TORCH_CHECK_TYPE(weight.scalar_type() == at::kFloat, "weight must be float32, got ", weight.scalar_type());
    TORCH_CHECK_VALUE(same_shape(weight.sizes(), idx_.sizes()), "weight must have the shape of idx ",
                      shape_text(idx_.sizes()), ", got ", shape_text(weight.sizes()));
  }
  no_tangent(table_, "table");
  no_tangent(weight, "weight");
  need_cuda(table_);
  same_device(idx_, table_, "idx");
  if (valid.defined()) same_device(valid, table_, "valid");
  if (weight.defined()) same_device(weight, table_, "weight");
  const Tensor table = plain(table_), idx = plain(idx_).contiguous();
  if (valid.defined()) valid = valid.contiguous();
  if (weight.defined()) weight = plain(weight).contiguous();
  if (at::GradMode::is_enabled() && (table.requires_grad() || (weight.defined() && weight.requires_grad())))
    return GatherRows::apply(table, weight.defined() ? OptTensor(weight) : OptTensor(), idx,
                             valid.defined() ? OptTensor(valid) : OptTensor(), scale);
  return rows_forward(table, idx, valid, weight, scale);
}

// ---- labels ----------------------------------------------------------------------------------------

struct Scores {
  Tensor logp, entropy, top_logp, top_ids, stats;
};

Scores scores_forward(const Tensor& logits, const Tensor& labels, int64_t top, bool want_stats) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t C = logits.size(-1), P = labels.numel();
  const Tensor x = rows2d(logits, P, C);
  const auto f32 = labels.options().dtype(at::kFloat);
  std::vector<int64_t> shape = labels.sizes().vec();
  Scores s;
  s.logp = at::empty(shape, f32);
  s.entropy = at::empty(shape, f32);
  shape.push_back(top);
  s.top_logp = at::empty(shape, f32);
  s.top_ids = at::empty(shape, labels.options().dtype(at::kLong));
  if (want_stats) s.stats = at::empty({P, 2}, f32);
  check(tts_label_log_probs(ptr<void>(x), P, C, row_stride(x), row_type(logits, "logits"), ptr<void>(labels),
                            index_type(labels, "labels"), static_cast<int>(top), ptr<float>(s.logp),
                            ptr<float>(s.entropy), ptr<float>(s.top_logp), ptr<int64_t>(s.top_ids),
                            ptr<float>(s.stats), stream()),
        "tts_label_log_probs");
  return s;
}

struct LabelLogProbs : torch::autograd::Function<LabelLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t top) {
    const Scores s = scores_forward(logits, labels, top, true);
    ctx->save_for_backward({logits, labels, s.stats, s.entropy, s.top_ids});
    ctx->mark_non_differentiable({s.top_ids});
    ctx->set_materialize_grads(false);
    return {s.logp, s.entropy, s.top_logp, s.top_ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor& logits = s[0];
    variable_list out(3);
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t C = logits.size(-1), P = s[1].numel();
    const Tensor x = rows2d(logits, P, C);
    for (int i = 0; i < 3; ++i) {
      no_tangent(grads[i], "a gradient of the scores");
      if (grads[i].defined()) grads[i] = plain(grads[i]).contiguous();
    }
    out[0] = at::empty(logits.sizes(), logits.options().requires_grad(false));
    check(tts_label_log_probs_bwd(ptr<void>(x), P, C, row_stride(x), row_type(logits, "logits"), ptr<void>(s[1]),
                                  index_type(s[1], "labels"), static_cast<int>(s[4].size(-1)), ptr<float>(s[2]),
                                  ptr<float>(s[3]), ptr<int64_t>(s[4]), ptr<float>(grads[0]), ptr<float>(grads[1]),
                                  ptr<float>(grads[2]), ptr<void>(out[0]), stream()),
          "tts_label_log_probs_bwd");
    return once(std::move(out));
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> label_log_probs(const Tensor& logits_, const Tensor& labels_, int64_t top) {
  TORCH_CHECK_VALUE(logits_.dim() >= 1 && logits_.size(-1) >= 1, "logits must be [..., C] with at least one label, got ",
                    shape_text(logits_.sizes()));
  row_type(logits_, "logits");
  index_type(labels_, "labels");
  const at::IntArrayRef rows = logits_.sizes().slice(0, logits_.dim() - 1);
  TORCH_CHECK_VALUE(same_shape(labels_.sizes(), rows), "labels must have the shape ", shape_text(rows), ", got ",
                    shape_text(labels_.sizes()));
  TORCH_CHECK_VALUE(top >= 0 && top <= 16, "top must be 0 to 16, got ", top);
  no_tangent(logits_, "logits");
  need_cuda(logits_);
  same_device(labels_, logits_, "labels");
  const Tensor logits = plain(logits_), labels = plain(labels_).contiguous();
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    variable_list v = LabelLogProbs::apply(logits, labels, top);
    return {v[0], v[1], v[2], v[3]};
  }
  const Scores s = scores_forward(logits, labels, top, false);
  return {s.logp, s.entropy, s.top_logp, s.top_ids};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // without the interpreter's lock, as torch's own functions run: a launch may wait for room in the GPU's queue
  namespace py = pybind11;
  m.def("gather_rows", &gather_rows, py::call_guard<py::gil_scoped_release>());
  m.def("label_log_probs", &label_log_probs, py::call_guard<py::gil_scoped_release>());
}
