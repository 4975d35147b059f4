// block_ops.cpp -- PyTorch operators of a transformer block and of the clipping
// before the update: attention, rotary positions, gradient norm and clipping.
// CUDA kernels through the C ABI (include/muon_train_sm100.h); gradients on the
// Autograd key.
#include <algorithm>
#include <array>
#include <cmath>
#include <limits>
#include <tuple>
#include <vector>

#include "train_ops_common.h"

namespace {

using namespace muon_train_ops;

// ------------------------------------------------------------ attention
// [batch, rows, heads, dim], read in place where the heads' elements are
// contiguous, all strides and the address are multiples of 16 bytes and nothing
// overlaps (a slice of one projection), else copied.
Tensor Heads4d(const Tensor& t) {
  bool in_place = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.size(3) <= 1 || t.stride(3) == 1);
  for (int i = 0; i < 3; ++i)
    in_place = in_place && (t.size(i) <= 1 || (t.stride(i) >= t.size(3) && t.stride(i) % 8 == 0));
  return in_place ? t : t.clone(at::MemoryFormat::Contiguous);
}
muon_train_strides Strides(const Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }

struct AttentionInputs {
  Tensor q, k, v, offsets, lengths;
  muon_train_attention_args args{};
};

Tensor Counts(const Tensor& t, const Tensor& like, const char* who, const char* name) {
  CheckDevice(t, like, who, name);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, who, ": ", name,
                   " must be int32 or int64, got ", t.scalar_type());
  if (t.scalar_type() == at::kInt) return t.contiguous();
  // what is beyond 32 bits is beyond the tensors too, and stays there
  constexpr int64_t kMost = std::numeric_limits<int32_t>::max();
  return t.clamp(int64_t{0}, kMost).to(at::kInt).contiguous();
}

AttentionInputs CheckAttention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& offsets,
                               const OptTensor& lengths, bool causal, int64_t window, double scale,
                               const char* who) {
  CheckCuda(q, who, "query");
  CheckDevice(k, q, who, "key");
  CheckDevice(v, q, who, "value");
  const bool packed = Given(offsets).defined();
  const int64_t n = packed ? 3 : 4;
  TORCH_CHECK_VALUE(q.dim() == n && k.dim() == n && v.dim() == n, who, ": query, key and value must have shape ",
                    packed ? "[tokens, heads, dim]" : "[batch, length, heads, dim]", ", got ", q.sizes(), ", ",
                    k.sizes(), " and ", v.sizes());
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(n - 1) == q.size(n - 1) &&
                        k.size(0) == q.size(0),
                    who, ": key and value must have one shape, with query's ", packed ? "tokens" : "batch",
                    " and dim, got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  const int64_t dim = q.size(n - 1), heads = q.size(n - 2), kv_heads = k.size(n - 2);
  TORCH_CHECK_VALUE(dim >= 8 && dim <= MUON_TRAIN_MAX_HEAD_DIM && dim % 8 == 0, who, ": dim must be 8 to ",
                    MUON_TRAIN_MAX_HEAD_DIM, " in steps of 8, got ", dim);
  TORCH_CHECK_VALUE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads <= 65535, who,
                    ": the key heads must divide the query heads, got ", kv_heads, " and ", heads);
  TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, who,
                   ": query must be bfloat16 or float16, got ", q.scalar_type());
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), who,
                   ": key and value must have query's dtype ", q.scalar_type(), ", got ", k.scalar_type(), " and ",
                   v.scalar_type());
  TORCH_CHECK_VALUE(window >= 0, who, ": window must be positive, got ", window);
  TORCH_CHECK_VALUE(static_cast<float>(scale) > 0.0f && std::isfinite(static_cast<float>(scale)), who,
                    ": scale must be positive and finite, got ", scale);
  AttentionInputs in;
  auto& a = in.args;
  a.batch = packed ? 1 : q.size(0);
  a.length = q.size(n - 3);
  a.keys = k.size(n - 3);
  constexpr int64_t kMost = int64_t{1} << 30;
  TORCH_CHECK_VALUE(a.batch <= 65535 && a.batch * a.length <= kMost && a.batch * a.keys <= kMost, who,
                    ": at most 65535 sequences and 2^30 tokens are supported");
  if (packed) {
    TORCH_CHECK_VALUE(!Given(lengths).defined(), who, ": offsets and lengths exclude each other");
    TORCH_CHECK_VALUE(offsets->dim() == 1 && offsets->size(0) >= 1, who,
                      ": offsets must have shape [sequences + 1], got ", offsets->sizes());
    in.offsets = Counts(*offsets, q, who, "offsets");
    a.sequences = offsets->size(0) - 1;
  }
  if (Given(lengths).defined()) {
    TORCH_CHECK_VALUE(a.keys == a.length, who, ": lengths need as many keys as queries, got ", a.keys, " and ",
                      a.length);
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == a.batch, who, ": lengths must have shape [",
                      a.batch, "], got ", lengths->sizes());
    in.lengths = Counts(*lengths, q, who, "lengths");
  }
  in.q = Heads4d(packed ? q.unsqueeze(0) : q);
  in.k = Heads4d(packed ? k.unsqueeze(0) : k);
  in.v = Heads4d(packed ? v.unsqueeze(0) : v);
  a.q = Ptr(in.q);
  a.k = Ptr(in.k);
  a.v = Ptr(in.v);
  a.q_stride = Strides(in.q);
  a.k_stride = Strides(in.k);
  a.v_stride = Strides(in.v);
  a.offsets = static_cast<const int32_t*>(Ptr(in.offsets));
  a.lengths = static_cast<const int32_t*>(Ptr(in.lengths));
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  // a window over all places is none
  a.window = window >= kMost * 2 ? 0 : window;
  a.scale = static_cast<float>(scale);
  a.causal = causal ? 1 : 0;
  a.dtype = Dtype(q, who, "query");
  return in;
}

// (out, lse, rest): with `keep`, rest is what rounding took from out, for the
// backward pass; else it is empty.
std::tuple<Tensor, Tensor, Tensor> AttentionCuda(const Tensor& q, const Tensor& k, const Tensor& v,
                                                 const OptTensor& offsets, const OptTensor& lengths, bool causal,
                                                 int64_t window, double scale, bool keep) {
  const char* who = "attention";
  const c10::cuda::OptionalCUDAGuard guard(q.device().is_cuda() ? std::make_optional(q.device()) : std::nullopt);
  AttentionInputs in = CheckAttention(q, k, v, offsets, lengths, causal, window, scale, who);
  Tensor out = Empty(q.sizes(), q.scalar_type(), q);
  Tensor lse = Empty({in.args.heads, in.args.batch * in.args.length}, at::kFloat, q);
  Tensor rest = keep ? Empty(q.sizes(), q.scalar_type(), q) : Empty({0}, q.scalar_type(), q);
  in.args.out = Ptr(out);
  in.args.out_rest = keep ? Ptr(rest) : nullptr;
  in.args.lse = static_cast<float*>(Ptr(lse));
  CheckStatus(muon_train_attention_sm100(&in.args, Stream(q)), who);
  return {out, lse, rest};
}

std::tuple<Tensor, Tensor, Tensor> AttentionBackwardCuda(
    const Tensor& grad_out, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
    const Tensor& lse, const Tensor& rest, const OptTensor& offsets, const OptTensor& lengths, bool causal, int64_t window,
    double scale) {
  const char* who = "attention_backward";
  const c10::cuda::OptionalCUDAGuard guard(q.device().is_cuda() ? std::make_optional(q.device()) : std::nullopt);
  AttentionInputs in = CheckAttention(q, k, v, offsets, lengths, causal, window, scale, who);
  for (const auto& [t, name] :
       {std::pair<const Tensor&, const char*>{grad_out, "grad_out"}, {out, "out"}, {rest, "rest"}}) {
    if (&t == &rest && t.numel() == 0) continue;
    CheckDevice(t, q, who, name);
    TORCH_CHECK_VALUE(t.sizes() == q.sizes(), who, ": ", name, " must have query's shape ", q.sizes(), ", got ",
                      t.sizes());
    TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(), who, ": ", name, " must have query's dtype");
  }
  CheckDevice(lse, q, who, "lse");
  TORCH_CHECK_TYPE(lse.scalar_type() == at::kFloat, who, ": lse must be float32");
  TORCH_CHECK_VALUE(lse.dim() == 2 && lse.size(0) == in.args.heads && lse.size(1) == in.args.batch * in.args.length,
                    who, ": lse must have shape [heads, batch * length]");
  const Tensor kept_out = out.contiguous(), kept_lse = lse.contiguous(), kept_rest = rest.contiguous();
  const Tensor g = Heads4d(in.offsets.defined() ? grad_out.unsqueeze(0) : grad_out);
  in.args.out = Ptr(kept_out);
  in.args.out_rest = kept_rest.numel() > 0 ? Ptr(kept_rest) : nullptr;
  in.args.lse = static_cast<float*>(Ptr(kept_lse));
  Tensor dq = Empty(q.sizes(), q.scalar_type(), q), dk = Empty(k.sizes(), q.scalar_type(), q);
  Tensor dv = Empty(v.sizes(), q.scalar_type(), q);
  muon_train_attention_grads grads{};
  grads.grad_out = Ptr(g);
  grads.grad_out_stride = Strides(g);
  grads.grad_q = Ptr(dq);
  grads.grad_k = Ptr(dk);
  grads.grad_v = Ptr(dv);
  grads.workspace_bytes = muon_train_attention_workspace_bytes(&in.args);
  const Tensor workspace = Empty({static_cast<int64_t>(grads.workspace_bytes)}, at::kByte, q);
  grads.workspace = Ptr(workspace);
  CheckStatus(muon_train_attention_backward_sm100(&in.args, &grads, Stream(q)), who);
  return {dq, dk, dv};
}

// ------------------------------------------------------------ rotary
// Leading sizes as [batch, length]: the row before the heads, and all before it.
void RotaryTensor(const Tensor& t, int which, Tensor* kept, muon_train_rotary_args* a) {
  const int64_t n = t.dim(), length = n >= 3 ? t.size(n - 3) : 1;
  int64_t batch = 1;
  for (int64_t i = 0; i + 3 < n; ++i) batch *= t.size(i);
  Tensor x = n == 4 ? t : t.reshape({batch, length, t.size(n - 2), t.size(n - 1)});
  if (x.size(3) > 1 && x.stride(3) != 1) x = x.contiguous();
  *kept = x;
  a->x[which] = Ptr(x);
  a->x_batch[which] = x.stride(0);
  a->x_row[which] = x.stride(1);
  a->x_head[which] = x.stride(2);
  a->heads[which] = x.size(2);
  a->batch = x.size(0);
  a->length = x.size(1);
  a->dim = x.size(3);
}

std::tuple<Tensor, Tensor> RotaryCuda(const Tensor& q, const OptTensor& key, const Tensor& positions,
                                      const Tensor& frequencies, bool interleaved, double scale, bool inverse) {
  const char* who = inverse ? "rotary_backward" : "rotary";
  const Tensor& k = Given(key);
  CheckCuda(q, who, "query");
  const c10::cuda::CUDAGuard guard(q.device());
  TORCH_CHECK_VALUE(q.dim() >= 2, who, ": query must have shape [..., heads, dim], got ", q.sizes());
  muon_train_rotary_args a{};
  a.dtype = Dtype(q, who, "query");
  if (k.defined()) {
    CheckDevice(k, q, who, "key");
    TORCH_CHECK_VALUE(k.dim() == q.dim() && k.size(-1) == q.size(-1) &&
                          k.sizes().slice(0, k.dim() - 2) == q.sizes().slice(0, q.dim() - 2),
                      who, ": key must have query's shape but for the heads, got ", k.sizes(), " and ", q.sizes());
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), who, ": key must have query's dtype ", q.scalar_type(),
                     ", got ", k.scalar_type());
  }
  CheckDevice(positions, q, who, "positions");
  CheckDevice(frequencies, q, who, "frequencies");
  TORCH_CHECK_TYPE(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, who,
                   ": positions must be int64 or int32, got ", positions.scalar_type());
  TORCH_CHECK_TYPE(frequencies.scalar_type() == at::kFloat || frequencies.scalar_type() == at::kDouble, who,
                   ": frequencies must be float32 or float64, got ", frequencies.scalar_type());
  const at::IntArrayRef lead = q.sizes().slice(0, q.dim() - 2);
  const bool shared = lead.size() > 1 && positions.sizes() == lead.slice(lead.size() - 1);
  TORCH_CHECK_VALUE(positions.sizes() == lead || shared, who, ": positions must have shape ", lead,
                    lead.size() > 1 ? " or its last size" : "", ", got ", positions.sizes());
  const int64_t dim = q.size(-1);
  TORCH_CHECK_VALUE(dim >= 1 && dim <= MUON_TRAIN_MAX_ROTARY_DIM, who, ": dim must be 1 to ",
                    MUON_TRAIN_MAX_ROTARY_DIM, ", got ", dim);
  TORCH_CHECK_VALUE(frequencies.dim() == 1 && 2 * frequencies.size(0) <= dim, who,
                    ": frequencies must have shape [pairs] of at most dim / 2 = ", dim / 2, " pairs, got ",
                    frequencies.sizes());
  TORCH_CHECK_VALUE(std::isfinite(static_cast<float>(scale)), who, ": scale must be finite, got ", scale);
  Tensor kept_q, kept_k;
  if (k.defined()) RotaryTensor(k, 1, &kept_k, &a);
  RotaryTensor(q, 0, &kept_q, &a);
  TORCH_CHECK_VALUE(a.batch * a.length < (int64_t{1} << 31) && (a.heads[0] + a.heads[1]) * dim < (int64_t{1} << 24),
                    who, ": fewer than 2^31 tokens, and 2^24 elements a token, are supported");
  const Tensor at = positions.contiguous(), f = frequencies.contiguous();
  Tensor yq = Empty(q.sizes(), q.scalar_type(), q);
  Tensor yk = k.defined() ? Empty(k.sizes(), k.scalar_type(), k) : Empty({0}, q.scalar_type(), q);
  a.y[0] = Ptr(yq);
  a.y[1] = Ptr(yk);
  a.positions = Ptr(at);
  a.frequencies = Ptr(f);
  a.pairs = f.size(0);
  a.position_rows = shared ? 1 : a.batch;
  a.position_bytes = static_cast<int>(at.element_size());
  a.frequency_bytes = static_cast<int>(f.element_size());
  a.interleaved = interleaved ? 1 : 0;
  a.inverse = inverse ? 1 : 0;
  a.scale = static_cast<float>(scale);
  CheckStatus(muon_train_rotary_sm100(&a, Stream(q)), who);
  return {yq, yk};
}

// ------------------------------------------------------------ clipping
// Whether `t` is a run of memory without gaps, in some order of its axes.
bool Dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

// Bytes [begin, end) of memory, in the order of their addresses where they came
// in that order; sorted on the first question otherwise.
class Ranges {
 public:
  explicit Ranges(size_t n) { ranges_.reserve(n); }
  void Add(uintptr_t begin, uintptr_t end) {
    sorted_ = sorted_ && (ranges_.empty() || ranges_.back().first <= begin);
    ranges_.emplace_back(begin, end);
  }
  // Whether two of them have bytes in common.
  bool Overlap() {
    Sort();
    for (size_t i = 1; i < ranges_.size(); ++i)
      if (ranges_[i - 1].second > ranges_[i].first) return true;
    return false;
  }
  // Whether [begin, end) has bytes in common with one of them; they do not overlap themselves.
  bool Touches(uintptr_t begin, uintptr_t end) {
    Sort();
    // questions come in the order of addresses too, as a rule: the answer is near the last one
    if (at_ >= ranges_.size() || !(at_ == 0 || ranges_[at_ - 1].first <= begin) || ranges_[at_].first <= begin)
      at_ = std::upper_bound(ranges_.begin(), ranges_.end(), std::make_pair(begin, UINTPTR_MAX)) - ranges_.begin();
    return (at_ > 0 && ranges_[at_ - 1].second > begin) || (at_ < ranges_.size() && ranges_[at_].first < end);
  }

 private:
  void Sort() {
    if (!sorted_) std::sort(ranges_.begin(), ranges_.end());
    sorted_ = true;
  }
  std::vector<std::pair<uintptr_t, uintptr_t>> ranges_;
  bool sorted_ = true;
  size_t at_ = 0;
};

}  // namespace

// A call with hundreds of tensors is bound by the host: what cannot be wrong is
// not asked twice.
void muon_train_ops::clip_gradients(TensorPointers grads, TensorPointers out, double max_norm, bool largest,
                                    const Tensor& norm) {
  const char* who = "clip_gradients";
  TORCH_CHECK_VALUE(!grads.empty(), who, ": no gradients");
  TORCH_CHECK_VALUE(out.empty() || out.size() == grads.size(), who, ": out must have a tensor for each gradient, got ",
                    out.size(), " and ", grads.size());
  TORCH_CHECK_VALUE(max_norm >= 0.0, who, ": max_norm must not be negative, got ", max_norm);
  const Tensor& first = *grads[0];
  CheckCuda(first, who, "gradients");
  const c10::cuda::CUDAGuard guard(first.device());
  const size_t n = grads.size();
  std::vector<muon_train_clip_tensor> list(n);
  Ranges written(n);
  const auto check = [&](const Tensor& t, const char* name) {
    CheckDevice(t, first, who, name);
    if (t.unsafeGetTensorImpl()->autograd_meta() == nullptr) return;  // never seen by autograd
    NoTangents({&t}, who);
    TORCH_CHECK_VALUE(!t.requires_grad(), who,
                      ": parameters and recorded tensors are not clipped (pass their gradients, detached)");
  };
  for (size_t i = 0; i < n; ++i) {
    const Tensor& g = *grads[i];
    const Tensor& o = out.empty() ? g : *out[i];
    check(g, "every gradient");
    TORCH_CHECK_VALUE(Dense(g), who, ": gradients must be dense, got strides ", g.strides(), " for ", g.sizes());
    muon_train_clip_tensor& t = list[i];
    t.count = g.numel();
    t.dtype = t.out_dtype = Dtype(g, who, "every gradient");
    if (!out.empty()) {
      check(o, "out");
      TORCH_CHECK_VALUE(o.sizes() == g.sizes() && (o.strides() == g.strides() || (o.is_contiguous() && g.is_contiguous())),
                        who, ": out must have its gradient's shape and layout, got ", o.sizes(), " for ", g.sizes());
      t.out_dtype = Dtype(o, who, "out");
    }
    if (t.count == 0) continue;
    t.out = o.unsafeGetTensorImpl()->mutable_data();  // a lazy clone gets memory of its own here
    const uintptr_t begin = reinterpret_cast<uintptr_t>(t.out);
    written.Add(begin, begin + static_cast<uintptr_t>(t.count) * o.element_size());
  }
  for (size_t i = 0; i < n; ++i)  // where they are when all that is written has its memory
    if (list[i].count > 0) list[i].grad = grads[i]->unsafeGetTensorImpl()->data();
  TORCH_CHECK_VALUE(!written.Overlap(), who,
                    ": the same memory would be scaled twice (a gradient listed twice, or views of one another)");
  if (!out.empty()) {  // what is written may not be read as another gradient
    for (const muon_train_clip_tensor& t : list) {
      const uintptr_t begin = reinterpret_cast<uintptr_t>(t.grad);
      const bool itself = t.grad == t.out && t.dtype == t.out_dtype;
      TORCH_CHECK_VALUE(t.count == 0 || itself ||
                            !written.Touches(begin, begin + static_cast<uintptr_t>(t.count) * (t.dtype == MUON_TRAIN_F32 ? 4 : 2)),
                        who, ": out may be its gradient, of the same type, but not overlap one otherwise");
    }
  }
  TORCH_CHECK_VALUE(norm.device() == first.device() && norm.scalar_type() == at::kFloat && norm.numel() == 1, who,
                    ": norm must be one float32 element on ", first.device());
  const size_t bytes = muon_train_clip_workspace_bytes(static_cast<int64_t>(n));
  const Tensor workspace = Empty({static_cast<int64_t>(bytes)}, at::kByte, first);
  CheckStatus(muon_train_clip_sm100(list.data(), static_cast<int64_t>(n), max_norm, largest ? 0 : 2,
                                    static_cast<float*>(Ptr(norm)), Ptr(workspace), bytes, Stream(first)),
              who);
  for (const Tensor* t : out.empty() ? grads : out)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

namespace {

Tensor ClipCuda(at::TensorList grads, at::TensorList out, double max_norm, bool largest) {
  TORCH_CHECK_VALUE(!grads.empty(), "clip_gradients: no gradients");
  CheckCuda(grads[0], "clip_gradients", "gradients");
  Tensor norm = Empty({}, at::kFloat, grads[0]);
  std::vector<const Tensor*> g(grads.size()), o(out.size());
  for (size_t i = 0; i < g.size(); ++i) g[i] = &grads[i];
  for (size_t i = 0; i < o.size(); ++i) o[i] = &out[i];
  muon_train_ops::clip_gradients(g, o, max_norm, largest, norm);
  return norm;
}
Tensor ClipInPlaceCuda(at::TensorList grads, double max_norm, bool largest) {
  return ClipCuda(grads, {}, max_norm, largest);
}
Tensor ClipOutCuda(at::TensorList grads, at::TensorList out, double max_norm, bool largest) {
  TORCH_CHECK_VALUE(out.size() == grads.size(), "clip_gradients: out must have a tensor for each gradient, got ",
                    out.size(), " and ", grads.size());
  return ClipCuda(grads, out, max_norm, largest);
}

// ------------------------------------------------------------ autograd
struct AttentionBackward : public torch::autograd::Node {
  SavedVariable q, k, v, out, lse, rest, offsets, lengths;
  bool causal = false;
  int64_t window = 0;
  double scale = 1.0;

  std::string name() const override { return "AttentionBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &v, &out, &lse, &rest, &offsets, &lengths}) s->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    NoSecondOrder(grads, "attention");
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(3);
    static auto op = Op<decltype(AttentionBackwardCuda)>("muon_ascend950::attention_backward");
    auto [dq, dk, dv] = op.call(grads[0], q.unpack(), k.unpack(), v.unpack(), out.unpack(shared_from_this()),
                                lse.unpack(), rest.unpack(), Optional(offsets.unpack()),
                                Optional(lengths.unpack()), causal, window, scale);
    variable_list all(3);
    Tensor* made[3] = {&dq, &dk, &dv};
    for (size_t i = 0; i < 3; ++i)
      if (task_should_compute_output(i)) all[i] = std::move(*made[i]);
    return all;
  }
};

std::tuple<Tensor, Tensor, Tensor> AttentionAutograd(const Tensor& q, const Tensor& k, const Tensor& v,
                                                     const OptTensor& offsets, const OptTensor& lengths, bool causal,
                                                     int64_t window, double scale, bool keep) {
  static auto op = Op<decltype(AttentionCuda)>("muon_ascend950::attention");
  const bool recorded = Recorded({&q, &k, &v});
  const auto call = [&] {
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(q, k, v, offsets, lengths, causal, window, scale, keep || recorded);
  };
  NoTangents({&q, &k, &v}, "attention");
  if (!recorded) return call();
  auto node = MakeNode<AttentionBackward>(q, k, v);
  auto result = call();
  node->q = SavedVariable(q, false);
  node->k = SavedVariable(k, false);
  node->v = SavedVariable(v, false);
  node->lse = SavedVariable(std::get<1>(result), false);
  node->rest = SavedVariable(std::get<2>(result), false);
  node->offsets = SavedVariable(Given(offsets), false);
  node->lengths = SavedVariable(Given(lengths), false);
  node->causal = causal;
  node->window = window;
  node->scale = scale;
  torch::autograd::set_history(std::get<0>(result), node);
  node->out = SavedVariable(std::get<0>(result), true);
  return result;
}

struct RotaryBackward : public torch::autograd::Node {
  SavedVariable positions, frequencies;
  bool interleaved = false;
  double scale = 1.0;

  std::string name() const override { return "RotaryBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    positions.reset_data();
    frequencies.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    NoSecondOrder(grads, "rotary");
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list all(2);
    static auto op = Op<decltype(RotaryCuda)>("muon_ascend950::rotary_backward");
    const bool want_q = grads[0].defined() && task_should_compute_output(0);
    const bool want_k = grads.size() > 1 && grads[1].defined() && task_should_compute_output(1);
    if (!want_q && !want_k) return all;
    const Tensor& first = want_q ? grads[0] : grads[1];
    auto [d0, d1] = op.call(first, want_q && want_k ? OptTensor(grads[1]) : OptTensor(), positions.unpack(),
                            frequencies.unpack(), interleaved, scale, true);
    if (want_q) all[0] = std::move(d0);
    if (want_k) all[1] = want_q ? std::move(d1) : std::move(d0);
    return all;
  }
};

std::tuple<Tensor, Tensor> RotaryAutograd(const Tensor& q, const OptTensor& key, const Tensor& positions,
                                          const Tensor& frequencies, bool interleaved, double scale) {
  static auto op = Op<std::tuple<Tensor, Tensor>(const Tensor&, const OptTensor&, const Tensor&, const Tensor&,
                                                 bool, double)>("muon_ascend950::rotary");
  const auto call = [&] {
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(q, key, positions, frequencies, interleaved, scale);
  };
  const Tensor& k = Given(key);
  NoTangents({&q, &k, &frequencies}, "rotary");
  TORCH_CHECK_NOT_IMPLEMENTED(!Recorded({&frequencies}),
                              "rotary: frequencies have no gradient (pass them detached, or without recording)");
  if (!Recorded({&q, &k})) return call();
  auto node = MakeNode<RotaryBackward>(q, k);
  auto result = call();
  node->positions = SavedVariable(positions, false);
  node->frequencies = SavedVariable(frequencies, false);
  node->interleaved = interleaved;
  node->scale = scale;
  torch::autograd::set_history(std::get<0>(result), node);
  if (k.defined()) torch::autograd::set_history(std::get<1>(result), node);
  return result;
}
std::tuple<Tensor, Tensor> RotaryForwardCuda(const Tensor& q, const OptTensor& key, const Tensor& positions,
                                             const Tensor& frequencies, bool interleaved, double scale) {
  return RotaryCuda(q, key, positions, frequencies, interleaved, scale, false);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(muon_ascend950, m) {
  m.def("attention(Tensor query, Tensor key, Tensor value, Tensor? offsets, Tensor? lengths, bool causal, "
        "int window, float scale, bool keep) -> (Tensor out, Tensor lse, Tensor rest)");
  m.def("attention_backward(Tensor grad_out, Tensor query, Tensor key, Tensor value, Tensor out, Tensor lse, "
        "Tensor rest, Tensor? offsets, Tensor? lengths, bool causal, int window, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("rotary(Tensor query, Tensor? key, Tensor positions, Tensor frequencies, bool interleaved, "
        "float scale) -> (Tensor, Tensor)");
  m.def("rotary_backward(Tensor grad_query, Tensor? grad_key, Tensor positions, Tensor frequencies, "
        "bool interleaved, float scale, bool inverse) -> (Tensor, Tensor)");
  m.def("clip_gradients_(Tensor(a!)[] gradients, float max_norm, bool largest) -> Tensor");
  m.def("clip_gradients(Tensor[] gradients, Tensor(a!)[] out, float max_norm, bool largest) -> Tensor");
}

TORCH_LIBRARY_IMPL(muon_ascend950, CUDA, m) {
  m.impl("attention", &AttentionCuda);
  m.impl("attention_backward", &AttentionBackwardCuda);
  m.impl("rotary", &RotaryForwardCuda);
  m.impl("rotary_backward", &RotaryCuda);
  m.impl("clip_gradients_", &ClipInPlaceCuda);
  m.impl("clip_gradients", &ClipOutCuda);
}

TORCH_LIBRARY_IMPL(muon_ascend950, Autograd, m) {
  m.impl("attention", &AttentionAutograd);
  m.impl("rotary", &RotaryAutograd);
}
