// train_ops.cpp -- PyTorch operators of the training step around the Muon
// update: distillation from a teacher's top logits, the norms around a
// residual block, routing to experts.  CUDA kernels through the C ABI
// (include/muon_train_sm100.h); gradients on the Autograd key.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <array>
#include <cfloat>
#include <cmath>
#include <cstdlib>
#include <optional>
#include <tuple>

#include "muon_train_sm100.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// Of a launch on the current device.  With MUON_POLAR_DEBUG_SYNC set (read on
// every call) it also synchronises, and raises if a wait of a kernel ran out.
void CheckStatus(int rc, const char* who) {
  TORCH_CHECK(rc == MUON_POLAR_OK, who, " failed, status=", rc,
              ", detail=", muon_polar_status_string(rc));
  if (std::getenv("MUON_POLAR_DEBUG_SYNC") == nullptr) return;
  uint32_t flags = 0;
  const int read = muon_train_read_device_status(c10::cuda::current_device(), &flags, /*clear=*/1);
  TORCH_CHECK(read == MUON_POLAR_OK, who, " failed, status=", read,
              ", detail=", muon_polar_status_string(read));
  TORCH_CHECK(flags == 0, who, " gave up on a bounded wait, status word=", flags);
}

int Dtype(const Tensor& t, const char* who, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return MUON_TRAIN_F32;
    case at::kBFloat16: return MUON_TRAIN_BF16;
    case at::kHalf: return MUON_TRAIN_F16;
    default: TORCH_CHECK_TYPE(false, who, ": ", name, " must be float32, bfloat16 or float16, got ",
                              t.scalar_type());
  }
}

void CheckCuda(const Tensor& t, const char* who, const char* name) {
  TORCH_CHECK_VALUE(t.device().is_cuda(), who, ": ", name, " must be a CUDA tensor, got ", t.device());
}
void CheckDevice(const Tensor& t, const Tensor& like, const char* who, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device(), who, ": ", name, " must be on ", like.device(),
                    ", got ", t.device());
}

// An uninitialised contiguous CUDA tensor, without the dispatcher's way there:
// small calls are bound by the host.
Tensor Empty(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}

void* Ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const Tensor& Given(const OptTensor& t) {
  static const Tensor none;
  return t.has_value() && t->defined() ? *t : none;
}
void* Stream(const Tensor& t) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// Tangents are not carried on, nor is a gradient of a gradient computed: say
// so instead of returning a result that autograd would take for a constant.
void NoTangents(std::initializer_list<const Tensor*> inputs, const char* who) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), who,
                                ": forward-mode differentiation (jvp) is not supported");
}
void NoSecondOrder(const variable_list& grads, const char* who) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), who,
                              ": the gradient cannot be differentiated again (create_graph=True)");
  for (const Tensor& g : grads) NoTangents({&g}, who);
}

// ------------------------------------------------------------ distillation
// [..., n] as [rows, n], read in place when the elements of a row are
// contiguous and the rows are evenly spaced and apart (a slice of padded
// logits), else copied.
Tensor Rows2d(const Tensor& t) {
  const int64_t n = t.size(-1);
  const Tensor rows = t.dim() == 2 ? t : t.reshape({n > 0 ? t.numel() / n : 0, n});
  const bool in_place = (n <= 1 || rows.stride(1) == 1) && (rows.size(0) <= 1 || rows.stride(0) >= n);
  return in_place ? rows : rows.contiguous();
}
int64_t RowStride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// The gradient in the logits' own layout, their padding and their offset from
// a 16-byte boundary included, so that its rows are written in the vectors
// that the logits' are read in.
Tensor GradLike(const Tensor& z) {
  const int64_t ld = RowStride(z), rows = z.size(0), cols = z.size(1);
  if (rows == 0 || ld > 2 * cols) return Empty({rows, cols}, z.scalar_type(), z);
  const int64_t item = z.element_size();
  const int64_t shift = static_cast<int64_t>(reinterpret_cast<uintptr_t>(z.data_ptr()) % 16) / item;
  if (ld == cols && shift == 0) return Empty({rows, cols}, z.scalar_type(), z);
  const int64_t used = (rows - 1) * ld + cols;
  return Empty({used + shift}, z.scalar_type(), z).as_strided({rows, cols}, {ld, 1}, shift);
}

at::IntArrayRef Lead(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

// One fp32 value for each row.
Tensor RowValues(const OptTensor& t, const Tensor& like, const char* who, const char* name) {
  if (!Given(t).defined()) return Tensor();
  CheckDevice(*t, like, who, name);
  TORCH_CHECK_VALUE(t->sizes() == Lead(like), who, ": ", name, " must have shape ", Lead(like),
                    ", got ", t->sizes());
  TORCH_CHECK_TYPE(t->is_floating_point(), who, ": ", name, " must be a floating tensor");
  return t->to(at::kFloat).contiguous();
}

struct DistillInputs {
  Tensor student, values, indices, lse;
  muon_train_distill_args args{};
};

DistillInputs CheckDistill(const Tensor& student, const Tensor& values, const Tensor& indices,
                           const OptTensor& teacher_lse, double temperature, const char* who) {
  CheckCuda(student, who, "student_logits");
  TORCH_CHECK_VALUE(student.dim() >= 1 && student.size(-1) > 0, who,
                    ": student_logits must have shape [..., vocab], got ", student.sizes());
  TORCH_CHECK_VALUE(values.dim() == student.dim() && indices.sizes() == values.sizes() &&
                        Lead(values) == Lead(student),
                    who, ": teacher_logits and teacher_indices must both have shape [..., top] with "
                    "student_logits' leading sizes, got ", values.sizes(), " and ", indices.sizes());
  const int64_t top = values.size(-1);
  TORCH_CHECK_VALUE(top >= 1 && top <= MUON_TRAIN_MAX_TOP, who, ": a list must have 1 to ",
                    MUON_TRAIN_MAX_TOP, " entries, got ", top);
  CheckDevice(values, student, who, "teacher_logits");
  CheckDevice(indices, student, who, "teacher_indices");
  TORCH_CHECK_TYPE(indices.scalar_type() == at::kLong || indices.scalar_type() == at::kInt, who,
                   ": teacher_indices must be int64 or int32, got ", indices.scalar_type());
  TORCH_CHECK_VALUE(static_cast<float>(temperature) >= FLT_MIN && std::isfinite(static_cast<float>(temperature)), who,
                    ": temperature must be positive (2^-126 or more) and finite, got ", temperature);
  DistillInputs in;
  in.args.dtype = Dtype(student, who, "student_logits");
  in.args.teacher_dtype = Dtype(values, who, "teacher_logits");
  in.lse = RowValues(teacher_lse, student, who, "teacher_lse");
  in.student = Rows2d(student);
  in.values = values.contiguous();
  in.indices = indices.contiguous();
  in.args.logits = Ptr(in.student);
  in.args.rows = in.student.size(0);
  in.args.vocab = in.student.size(1);
  in.args.ld = RowStride(in.student);
  in.args.teacher_logits = Ptr(in.values);
  in.args.teacher_indices = Ptr(in.indices);
  in.args.teacher_lse = static_cast<const float*>(Ptr(in.lse));
  in.args.top = top;
  in.args.temperature = static_cast<float>(temperature);
  in.args.index_bytes = indices.scalar_type() == at::kLong ? 8 : 4;
  return in;
}

std::tuple<Tensor, Tensor> DistillCuda(const Tensor& student, const Tensor& values,
                                       const Tensor& indices, const OptTensor& teacher_lse,
                                       double temperature) {
  const char* who = "distill_topk";
  DistillInputs in = CheckDistill(student, values, indices, teacher_lse, temperature, who);
  const c10::cuda::CUDAGuard guard(student.device());
  Tensor loss = Empty(Lead(student), at::kFloat, student), stats = Empty({in.args.rows, 2}, at::kFloat, student);
  in.args.loss = static_cast<float*>(Ptr(loss));
  in.args.stats = static_cast<float*>(Ptr(stats));
  CheckStatus(muon_train_distill_sm100(&in.args, Stream(student)), who);
  return {loss, stats};
}

Tensor DistillBackwardCuda(const Tensor& grad_loss, const Tensor& student, const Tensor& values,
                           const Tensor& indices, const OptTensor& teacher_lse, const Tensor& stats,
                           double temperature) {
  const char* who = "distill_topk_backward";
  DistillInputs in = CheckDistill(student, values, indices, teacher_lse, temperature, who);
  TORCH_CHECK_VALUE(stats.dim() == 2 && stats.size(0) == in.args.rows && stats.size(1) == 2, who,
                    ": stats must have shape [rows, 2]");
  CheckDevice(stats, student, who, "stats");
  TORCH_CHECK_TYPE(stats.scalar_type() == at::kFloat, who, ": stats must be float32");
  const c10::cuda::CUDAGuard guard(student.device());
  const Tensor scale = RowValues(grad_loss, student, who, "grad_loss"), kept = stats.contiguous();
  Tensor grad = GradLike(in.student);
  in.args.row_scale = static_cast<const float*>(Ptr(scale));
  in.args.stats = static_cast<float*>(Ptr(kept));
  in.args.grad = Ptr(grad);
  in.args.ld_grad = RowStride(grad);
  CheckStatus(muon_train_distill_backward_sm100(&in.args, Stream(student)), who);
  return student.dim() == 2 ? grad : grad.view(student.sizes());
}

std::tuple<Tensor, Tensor> DistillGradCuda(const Tensor& student, const Tensor& values,
                                           const Tensor& indices, const OptTensor& row_scale,
                                           const OptTensor& teacher_lse, double temperature) {
  const char* who = "distill_topk_grad";
  DistillInputs in = CheckDistill(student, values, indices, teacher_lse, temperature, who);
  const c10::cuda::CUDAGuard guard(student.device());
  const Tensor scale = RowValues(row_scale, student, who, "row_scale");
  Tensor loss = Empty(Lead(student), at::kFloat, student), stats = Empty({in.args.rows, 2}, at::kFloat, student);
  Tensor grad = GradLike(in.student);
  in.args.row_scale = static_cast<const float*>(Ptr(scale));
  in.args.loss = static_cast<float*>(Ptr(loss));
  in.args.stats = static_cast<float*>(Ptr(stats));
  in.args.grad = Ptr(grad);
  in.args.ld_grad = RowStride(grad);
  CheckStatus(muon_train_distill_sm100(&in.args, Stream(student)), who);
  return {loss, student.dim() == 2 ? grad : grad.view(student.sizes())};
}

// ------------------------------------------------------------ residual norm
struct NormInputs {
  Tensor block_out, residual, post, pre, gate, scale;
  muon_train_norm_args args{};
};

// Rows of the gate: its leading sizes are block_out's up to some axis and 1
// from there on, or it is one row; -1 for any other shape.
int64_t GateRows(const Tensor& gate, const Tensor& block_out) {
  const int64_t n = gate.dim() - 1;
  if (n < 0 || gate.size(-1) != block_out.size(-1)) return -1;
  int64_t rows = 1, same = 0;
  for (int64_t i = 0; i < n; ++i) rows *= gate.size(i);
  const auto ones_from = [&](int64_t i) {
    while (i < n && gate.size(i) == 1) ++i;
    return i == n;
  };
  if (ones_from(0)) return 1;
  if (n != block_out.dim() - 1) return -1;
  while (same < n && gate.size(same) == block_out.size(same)) ++same;
  return ones_from(same) ? rows : -1;
}

NormInputs CheckNorm(const Tensor& block_out, const Tensor& residual, const OptTensor& post,
                     const OptTensor& pre, const OptTensor& gate, const OptTensor& scale,
                     double eps, const char* who) {
  CheckCuda(block_out, who, "block_out");
  CheckDevice(residual, block_out, who, "residual");
  TORCH_CHECK_VALUE(block_out.dim() >= 1 && block_out.size(-1) > 0, who,
                    ": block_out must have shape [..., width], got ", block_out.sizes());
  TORCH_CHECK_VALUE(residual.sizes() == block_out.sizes(), who, ": residual must have block_out's shape ",
                    block_out.sizes(), ", got ", residual.sizes());
  TORCH_CHECK_TYPE(residual.scalar_type() == block_out.scalar_type(), who,
                   ": residual must have block_out's dtype ", block_out.scalar_type(), ", got ",
                   residual.scalar_type());
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), who, ": eps must be finite and not negative, got ", eps);
  const int64_t width = block_out.size(-1);
  NormInputs in;
  auto& a = in.args;
  const auto weight = [&](const OptTensor& w, const char* name, Tensor* to, int* dtype) {
    const Tensor& t = Given(w);
    if (!t.defined()) return;
    CheckDevice(t, block_out, who, name);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == width, who, ": ", name, " must have shape [", width,
                      "], got ", t.sizes());
    *dtype = Dtype(t, who, name);
    *to = t.contiguous();
  };
  a.dtype = Dtype(block_out, who, "block_out");
  weight(post, "post_weight", &in.post, &a.post_dtype);
  weight(pre, "pre_weight", &in.pre, &a.pre_dtype);
  if (Given(gate).defined()) {
    CheckDevice(*gate, block_out, who, "gate");
    a.gate_rows = GateRows(*gate, block_out);
    TORCH_CHECK_VALUE(a.gate_rows >= 0, who, ": gate must have shape [", width, "] or ", block_out.sizes(),
                      " with trailing leading sizes of 1, got ", gate->sizes());
    a.gate_dtype = Dtype(*gate, who, "gate");
    in.gate = gate->contiguous();
  }
  if (Given(scale).defined()) {
    CheckDevice(*scale, block_out, who, "residual_scale");
    TORCH_CHECK_VALUE(scale->numel() == 1 || (scale->dim() == 1 && scale->size(0) == width), who,
                      ": residual_scale must have one element or shape [", width, "], got ", scale->sizes());
    a.scale_dtype = Dtype(*scale, who, "residual_scale");
    in.scale = scale->contiguous();
    a.scale_count = scale->numel();
  }
  in.block_out = block_out.contiguous();
  in.residual = residual.contiguous();
  a.block_out = Ptr(in.block_out);
  a.residual = Ptr(in.residual);
  a.post_weight = Ptr(in.post);
  a.pre_weight = Ptr(in.pre);
  a.gate = Ptr(in.gate);
  a.residual_scale = Ptr(in.scale);
  a.rows = block_out.numel() / width;
  a.width = width;
  a.eps = static_cast<float>(eps);
  return in;
}

// (hidden, normed, rstd): rstd holds the two statistics of each row, [2,
// rows], 1 and 0 of a norm that there is not.  Without pre_weight normed is empty.
std::tuple<Tensor, Tensor, Tensor> ResidualNormCuda(
    const Tensor& block_out, const Tensor& residual, const OptTensor& post, const OptTensor& pre,
    const OptTensor& gate, const OptTensor& scale, double eps) {
  const char* who = "residual_norm";
  NormInputs in = CheckNorm(block_out, residual, post, pre, gate, scale, eps, who);
  const c10::cuda::CUDAGuard guard(block_out.device());
  const auto dtype = block_out.scalar_type();
  const int64_t rows = in.args.rows;
  Tensor hidden = Empty(block_out.sizes(), dtype, block_out);
  Tensor normed = in.pre.defined() ? Empty(block_out.sizes(), dtype, block_out) : Empty({0}, dtype, block_out);
  Tensor rstd = Empty({2, rows}, at::kFloat, block_out);
  in.args.hidden = Ptr(hidden);
  in.args.normed = in.pre.defined() ? Ptr(normed) : nullptr;
  in.args.rstd_post = static_cast<float*>(Ptr(rstd));
  in.args.rstd_pre = in.args.rstd_post + rows;
  CheckStatus(muon_train_residual_norm_sm100(&in.args, Stream(block_out)), who);
  return {hidden, normed, rstd};
}

// Gradients of (block_out, residual, post_weight, pre_weight, gate,
// residual_scale); those not asked for by `wanted` are empty.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> ResidualNormBackwardCuda(
    const OptTensor& grad_hidden, const OptTensor& grad_normed, const Tensor& block_out,
    const Tensor& residual, const OptTensor& post, const OptTensor& pre, const OptTensor& gate,
    const OptTensor& scale, const Tensor& rstd, double eps, std::array<bool, 6> wanted) {
  const char* who = "residual_norm_backward";
  NormInputs in = CheckNorm(block_out, residual, post, pre, gate, scale, eps, who);
  const c10::cuda::CUDAGuard guard(block_out.device());
  const int64_t rows = in.args.rows;
  const auto upstream = [&](const OptTensor& g, const char* name) -> Tensor {
    if (!Given(g).defined()) return Tensor();
    CheckDevice(*g, block_out, who, name);
    TORCH_CHECK_VALUE(g->sizes() == block_out.sizes(), who, ": ", name, " must have block_out's shape");
    TORCH_CHECK_TYPE(g->scalar_type() == block_out.scalar_type(), who, ": ", name,
                     " must have block_out's dtype");
    return g->contiguous();
  };
  const Tensor dh = upstream(grad_hidden, "grad_hidden"), dn = upstream(grad_normed, "grad_normed");
  CheckDevice(rstd, block_out, who, "rstd");
  TORCH_CHECK_TYPE(rstd.scalar_type() == at::kFloat, who, ": rstd must be float32");
  TORCH_CHECK_VALUE(rstd.dim() == 2 && rstd.size(0) == 2 && rstd.size(1) == rows, who,
                    ": rstd must have shape [2, rows]");
  const Tensor kept = rstd.contiguous();
  in.args.rstd_post = static_cast<float*>(Ptr(kept));
  in.args.rstd_pre = in.args.rstd_post + rows;
  const Tensor* like[6] = {&in.block_out, &in.residual, &in.post, &in.pre, &in.gate, &in.scale};
  std::array<Tensor, 6> out;
  const bool none = rows == 0 || (!dh.defined() && !dn.defined());
  for (int i = 0; i < 6; ++i) {
    if (!wanted[i] || !like[i]->defined())
      out[i] = Empty({0}, block_out.scalar_type(), block_out);
    else
      out[i] = none ? at::zeros(like[i]->sizes(), like[i]->options())
                    : Empty(like[i]->sizes(), like[i]->scalar_type(), block_out);
  }
  if (!none) {
    muon_train_norm_grads g{};
    g.grad_hidden = Ptr(dh);
    g.grad_normed = Ptr(dn);
    void** to[6] = {&g.grad_block_out, &g.grad_residual, &g.grad_post_weight,
                    &g.grad_pre_weight, &g.grad_gate, &g.grad_residual_scale};
    for (int i = 0; i < 6; ++i) *to[i] = wanted[i] && like[i]->defined() ? Ptr(out[i]) : nullptr;
    g.workspace_bytes = muon_train_residual_norm_workspace_bytes(&in.args);
    const Tensor workspace = Empty({static_cast<int64_t>(g.workspace_bytes)}, at::kByte, block_out);
    g.workspace = Ptr(workspace);
    CheckStatus(muon_train_residual_norm_backward_sm100(&in.args, &g, Stream(block_out)), who);
  }
  return {out[0], out[1], out[2], out[3], out[4], out[5]};
}

// ------------------------------------------------------------ routing
muon_train_route_args CheckRoute(const Tensor& logits, int64_t k, int64_t score, int64_t groups,
                                 int64_t top_groups, int64_t group_top, bool renormalize,
                                 double scale, Tensor* rows, const char* who) {
  CheckCuda(logits, who, "logits");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) > 0, who,
                    ": logits must have shape [..., experts], got ", logits.sizes());
  const int64_t experts = logits.size(-1);
  TORCH_CHECK_VALUE(experts >= 1 && experts <= MUON_TRAIN_MAX_EXPERTS, who, ": 1 to ",
                    MUON_TRAIN_MAX_EXPERTS, " experts are supported, got ", experts);
  TORCH_CHECK_VALUE(score == 0 || score == 1, who, ": score must be 0 (softmax) or 1 (sigmoid)");
  TORCH_CHECK_VALUE(groups >= 1 && experts % groups == 0, who,
                    ": groups must divide the experts, got ", groups, " and ", experts);
  TORCH_CHECK_VALUE(top_groups >= 1 && top_groups <= groups, who,
                    ": top_groups must be 1 to groups, got ", top_groups);
  TORCH_CHECK_VALUE(group_top == 1 || (group_top == 2 && (groups == 1 || experts / groups >= 2)), who,
                    ": group_top must be 1, or 2 with groups of two experts or more");
  TORCH_CHECK_VALUE(k >= 1 && k <= MUON_TRAIN_MAX_ROUTES && k <= top_groups * (experts / groups),
                    who, ": k must be 1 to ", MUON_TRAIN_MAX_ROUTES,
                    " and at most the experts of the chosen groups, got ", k);
  TORCH_CHECK_VALUE(std::isfinite(scale), who, ": scale must be finite, got ", scale);
  *rows = Rows2d(logits);
  muon_train_route_args a{};
  a.logits = Ptr(*rows);
  a.tokens = rows->size(0);
  a.experts = experts;
  a.ld = RowStride(*rows);
  a.dtype = Dtype(logits, who, "logits");
  a.score = static_cast<int>(score);
  a.k = static_cast<int>(k);
  a.groups = static_cast<int>(groups);
  a.top_groups = static_cast<int>(top_groups);
  a.group_top = static_cast<int>(group_top);
  a.renormalize = renormalize ? 1 : 0;
  a.scale = static_cast<float>(scale);
  return a;
}

std::tuple<Tensor, Tensor, Tensor> RouteCuda(const Tensor& logits, const OptTensor& bias, int64_t k,
                                             int64_t score, int64_t groups, int64_t top_groups,
                                             int64_t group_top, bool renormalize, double scale) {
  const char* who = "route_experts";
  Tensor rows, b;
  muon_train_route_args a =
      CheckRoute(logits, k, score, groups, top_groups, group_top, renormalize, scale, &rows, who);
  const c10::cuda::CUDAGuard guard(logits.device());
  if (Given(bias).defined()) {
    CheckDevice(*bias, logits, who, "bias");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == a.experts, who,
                      ": bias must have shape [", a.experts, "], got ", bias->sizes());
    TORCH_CHECK_TYPE(bias->is_floating_point(), who, ": bias must be a floating tensor");
    b = bias->to(at::kFloat).contiguous();
    a.bias = static_cast<const float*>(Ptr(b));
  }
  at::DimVector shape(Lead(logits));
  shape.push_back(k);
  Tensor weights = Empty(shape, at::kFloat, logits), indices = Empty(shape, at::kLong, logits);
  Tensor counts = Empty({a.experts}, at::kLong, logits);
  a.weights = static_cast<float*>(Ptr(weights));
  a.indices = static_cast<int64_t*>(Ptr(indices));
  a.counts = static_cast<int64_t*>(Ptr(counts));
  CheckStatus(muon_train_route_sm100(&a, Stream(logits)), who);
  return {weights, indices, counts};
}

Tensor RouteBackwardCuda(const Tensor& grad_weights, const Tensor& logits, const Tensor& indices,
                         int64_t score, bool renormalize, double scale) {
  const char* who = "route_experts_backward";
  TORCH_CHECK_VALUE(logits.dim() >= 1 && indices.dim() == logits.dim() && Lead(indices) == Lead(logits) &&
                        grad_weights.sizes() == indices.sizes(),
                    who, ": indices and grad_weights must have shape [..., k]");
  TORCH_CHECK_TYPE(indices.scalar_type() == at::kLong, who, ": indices must be int64");
  Tensor rows;
  muon_train_route_args a = CheckRoute(logits, indices.size(-1), score, 1, 1, 1, renormalize, scale, &rows, who);
  CheckDevice(grad_weights, logits, who, "grad_weights");
  CheckDevice(indices, logits, who, "indices");
  const c10::cuda::CUDAGuard guard(logits.device());
  const Tensor g = grad_weights.to(at::kFloat).contiguous(), chosen = indices.contiguous();
  a.indices = static_cast<int64_t*>(Ptr(chosen));
  Tensor grad = Empty(logits.sizes(), logits.scalar_type(), logits);
  CheckStatus(muon_train_route_backward_sm100(&a, static_cast<const float*>(Ptr(g)), Ptr(grad),
                                              Stream(logits)), who);
  return grad;
}

// ------------------------------------------------------------ autograd
template <typename Fn>
auto Op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}

// Whether autograd records a call: otherwise it goes to the kernels directly.
bool Recorded(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A node of the graph whose next edges are `inputs`, in order.
template <typename N, typename... Inputs>
std::shared_ptr<N> MakeNode(const Inputs&... inputs) {
  auto node = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return node;
}

OptTensor Optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct DistillBackward : public torch::autograd::Node {
  SavedVariable student, values, indices, lse, stats;
  double temperature = 1.0;

  std::string name() const override { return "DistillTopkBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&student, &values, &indices, &lse, &stats}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    NoSecondOrder(grads, "distill_topk");
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    static auto op = Op<decltype(DistillBackwardCuda)>("muon_ascend950::distill_topk_backward");
    return {op.call(grads[0], student.unpack(), values.unpack(), indices.unpack(), Optional(lse.unpack()),
                    stats.unpack(), temperature)};
  }
};

std::tuple<Tensor, Tensor> DistillAutograd(const Tensor& student, const Tensor& values,
                                           const Tensor& indices, const OptTensor& lse,
                                           double temperature) {
  static auto op = Op<decltype(DistillCuda)>("muon_ascend950::distill_topk");
  const auto call = [&] {
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(student, values, indices, lse, temperature);
  };
  NoTangents({&student, &values, &Given(lse)}, "distill_topk");
  if (!Recorded({&student})) return call();
  auto node = MakeNode<DistillBackward>(student);
  auto out = call();
  node->student = SavedVariable(student, false);
  node->values = SavedVariable(values, false);
  node->indices = SavedVariable(indices, false);
  node->lse = SavedVariable(Given(lse), false);
  node->stats = SavedVariable(std::get<1>(out), false);
  node->temperature = temperature;
  torch::autograd::set_history(std::get<0>(out), node);
  return out;
}

// The loss with its gradient is not recorded: nothing flows back through it.
std::tuple<Tensor, Tensor> DistillGradAutograd(const Tensor& student, const Tensor& values,
                                               const Tensor& indices, const OptTensor& row_scale,
                                               const OptTensor& lse, double temperature) {
  NoTangents({&student, &values, &Given(row_scale), &Given(lse)}, "distill_topk_grad");
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = Op<decltype(DistillGradCuda)>("muon_ascend950::distill_topk_grad");
  return op.call(student, values, indices, row_scale, lse, temperature);
}

struct ResidualNormBackward : public torch::autograd::Node {
  std::array<SavedVariable, 6> inputs;
  SavedVariable rstd;
  double eps = 0.0;

  std::string name() const override { return "ResidualNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable& v : inputs) v.reset_data();
    rstd.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    NoSecondOrder(grads, "residual_norm");
    std::lock_guard<std::mutex> lock(mutex_);
    std::array<Tensor, 6> s;
    std::array<bool, 6> wanted;
    for (size_t i = 0; i < 6; ++i) {
      s[i] = inputs[i].unpack();
      wanted[i] = s[i].defined() && task_should_compute_output(i);
    }
    const OptTensor dn = grads.size() > 1 ? Optional(grads[1]) : OptTensor();
    static auto op = Op<decltype(ResidualNormBackwardCuda)>("muon_ascend950::residual_norm_backward");
    auto [d0, d1, d2, d3, d4, d5] =
        op.call(Optional(grads[0]), dn, s[0], s[1], Optional(s[2]), Optional(s[3]), Optional(s[4]),
                Optional(s[5]), rstd.unpack(), eps, wanted);
    Tensor* all[6] = {&d0, &d1, &d2, &d3, &d4, &d5};
    variable_list out(6);
    for (size_t i = 0; i < 6; ++i)
      if (wanted[i]) out[i] = std::move(*all[i]);
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> ResidualNormAutograd(
    const Tensor& block_out, const Tensor& residual, const OptTensor& post, const OptTensor& pre,
    const OptTensor& gate, const OptTensor& scale, double eps) {
  static auto op = Op<decltype(ResidualNormCuda)>("muon_ascend950::residual_norm");
  const auto call = [&] {
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(block_out, residual, post, pre, gate, scale, eps);
  };
  const Tensor* inputs[6] = {&block_out, &residual, &Given(post), &Given(pre), &Given(gate), &Given(scale)};
  NoTangents({inputs[0], inputs[1], inputs[2], inputs[3], inputs[4], inputs[5]}, "residual_norm");
  if (!Recorded({inputs[0], inputs[1], inputs[2], inputs[3], inputs[4], inputs[5]})) return call();
  auto node = MakeNode<ResidualNormBackward>(*inputs[0], *inputs[1], *inputs[2], *inputs[3], *inputs[4],
                                             *inputs[5]);
  auto out = call();
  for (size_t i = 0; i < 6; ++i) node->inputs[i] = SavedVariable(*inputs[i], false);
  node->rstd = SavedVariable(std::get<2>(out), false);
  node->eps = eps;
  torch::autograd::set_history(std::get<0>(out), node);
  if (Given(pre).defined()) torch::autograd::set_history(std::get<1>(out), node);
  return out;
}

struct RouteBackward : public torch::autograd::Node {
  SavedVariable logits, indices;
  int64_t score = 0;
  bool renormalize = true;
  double scale = 1.0;

  std::string name() const override { return "RouteExpertsBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits.reset_data();
    indices.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    NoSecondOrder(grads, "route_experts");
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    static auto op = Op<decltype(RouteBackwardCuda)>("muon_ascend950::route_experts_backward");
    return {op.call(grads[0], logits.unpack(), indices.unpack(), score, renormalize, scale)};
  }
};

std::tuple<Tensor, Tensor, Tensor> RouteAutograd(const Tensor& logits, const OptTensor& bias, int64_t k,
                                                 int64_t score, int64_t groups, int64_t top_groups,
                                                 int64_t group_top, bool renormalize, double scale) {
  static auto op = Op<decltype(RouteCuda)>("muon_ascend950::route_experts");
  const auto call = [&] {
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(logits, bias, k, score, groups, top_groups, group_top, renormalize, scale);
  };
  NoTangents({&logits, &Given(bias)}, "route_experts");
  if (!Recorded({&logits})) return call();
  auto node = MakeNode<RouteBackward>(logits);
  auto out = call();
  node->logits = SavedVariable(logits, false);
  node->indices = SavedVariable(std::get<1>(out), false);
  node->score = score;
  node->renormalize = renormalize;
  node->scale = scale;
  torch::autograd::set_history(std::get<0>(out), node);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(muon_ascend950, m) {
  m.def("distill_topk(Tensor student_logits, Tensor teacher_logits, Tensor teacher_indices, "
        "Tensor? teacher_lse, float temperature) -> (Tensor loss, Tensor stats)");
  m.def("distill_topk_backward(Tensor grad_loss, Tensor student_logits, Tensor teacher_logits, "
        "Tensor teacher_indices, Tensor? teacher_lse, Tensor stats, float temperature) -> Tensor");
  m.def("distill_topk_grad(Tensor student_logits, Tensor teacher_logits, Tensor teacher_indices, "
        "Tensor? row_scale, Tensor? teacher_lse, float temperature) -> (Tensor loss, Tensor grad)");
  m.def("residual_norm(Tensor block_out, Tensor residual, Tensor? post_weight, Tensor? pre_weight, "
        "Tensor? gate, Tensor? residual_scale, float eps) -> (Tensor hidden, Tensor normed, Tensor rstd)");
  m.def("residual_norm_backward(Tensor? grad_hidden, Tensor? grad_normed, Tensor block_out, "
        "Tensor residual, Tensor? post_weight, Tensor? pre_weight, Tensor? gate, "
        "Tensor? residual_scale, Tensor rstd, float eps, bool[6] wanted) -> "
        "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("route_experts(Tensor logits, Tensor? bias, int k, int score, int groups, int top_groups, "
        "int group_top, bool renormalize, float scale) -> (Tensor weights, Tensor indices, Tensor counts)");
  m.def("route_experts_backward(Tensor grad_weights, Tensor logits, Tensor indices, int score, "
        "bool renormalize, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(muon_ascend950, CUDA, m) {
  m.impl("distill_topk", &DistillCuda);
  m.impl("distill_topk_backward", &DistillBackwardCuda);
  m.impl("distill_topk_grad", &DistillGradCuda);
  m.impl("residual_norm", &ResidualNormCuda);
  m.impl("residual_norm_backward", &ResidualNormBackwardCuda);
  m.impl("route_experts", &RouteCuda);
  m.impl("route_experts_backward", &RouteBackwardCuda);
}

TORCH_LIBRARY_IMPL(muon_ascend950, Autograd, m) {
  m.impl("distill_topk", &DistillAutograd);
  m.impl("distill_topk_grad", &DistillGradAutograd);
  m.impl("residual_norm", &ResidualNormAutograd);
  m.impl("route_experts", &RouteAutograd);
}
