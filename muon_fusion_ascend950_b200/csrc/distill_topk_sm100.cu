// distill_topk_sm100.cu -- distillation loss over a teacher's top logits, and
// its gradient in the student's logits.
//
//   q_j  = softmax over the row's counted teacher entries (or with the
//          teacher's own normaliser), lse = log sum_v exp(z_v / tau)
//   loss = sum_j q_j (log q_j - z_{i_j} / tau + lse)
//   dz_v = g / tau (Q exp(z_v / tau - lse) - sum_{i_j = v} q_j),  Q = sum q
//
// Bound by memory: the vocabulary is read once (and the gradient written
// once); the lists are a thousandth of it.
#include "train_common.cuh"

namespace muon_train {

std::atomic<uint64_t>& launch_counter() {
  static std::atomic<uint64_t> count{0};
  return count;
}

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// A row's list in shared memory: index (-1: not counted), q, log q and the
// student's logit.
struct List {
  int index[MUON_TRAIN_MAX_TOP];
  float q[MUON_TRAIN_MAX_TOP];
  float log_q[MUON_TRAIN_MAX_TOP];
  float z[MUON_TRAIN_MAX_TOP];
};

template <typename T>
__device__ __forceinline__ float logit(const T* row, int64_t i) { return to_float(row[i]); }

// Fills the list (z only for the loss) and returns Q; one whole warp, each
// lane its own entries.  The differences to the largest entry are taken
// before the division by tau, so that entries of the type's lowest value stay
// finite.
template <typename T>
__device__ float load_list(const muon_train_distill_args& a, int64_t row, const T* z, List* list) {
  const int lane = threadIdx.x & 31;
  const int top = static_cast<int>(a.top);
  const float inv_tau = 1.0f / a.temperature;
  const int64_t base = row * a.top;
  float best = -INFINITY;
  for (int j = lane; j < top; j += 32) {
    const int64_t i = a.index_bytes == 8
                          ? static_cast<const int64_t*>(a.teacher_indices)[base + j]
                          : static_cast<const int32_t*>(a.teacher_indices)[base + j];
    const float t = load_any(a.teacher_logits, a.teacher_dtype, base + j);
    const bool counted = i >= 0 && i < a.vocab && t > -INFINITY;
    list->index[j] = counted ? static_cast<int>(i) : -1;
    list->log_q[j] = t;
    if (counted) {
      best = fmaxf(best, t);
      if (a.loss != nullptr) list->z[j] = logit(z, i);
    }
  }
  best = warp_max(best);
  // log q = (t - shift) / tau - log_norm
  float shift = 0.f, log_norm = 0.f;
  if (a.teacher_lse != nullptr) {
    log_norm = a.teacher_lse[row];
  } else if (best > -INFINITY) {
    shift = best;
    float s = 0.f;
    for (int j = lane; j < top; j += 32)
      if (list->index[j] >= 0) s += expf((list->log_q[j] - shift) * inv_tau);
    log_norm = logf(warp_sum(s));
  }
  float total = 0.f;
  for (int j = lane; j < top; j += 32) {
    const float log_q = (list->log_q[j] - shift) * inv_tau - log_norm;
    const float q = list->index[j] >= 0 ? expf(log_q) : 0.f;
    list->log_q[j] = log_q;
    list->q[j] = q;
    total += q;
  }
  return warp_sum(total);
}

// The row's loss from its largest logit and the sum of exponentials relative
// to it: sum_j q_j (log q_j - (z_j - max) / tau + log sum).  One whole warp.
__device__ float row_loss(const List& list, int top, float inv_tau, float max, float sum) {
  const float log_sum = logf(sum);
  float loss = 0.f;
  for (int j = threadIdx.x & 31; j < top; j += 32) {
    const float q = list.q[j];  // a NaN q counts: it must reach the loss
    if (q != 0.f) loss += q * (list.log_q[j] - (list.z[j] - max) * inv_tau + log_sum);
  }
  return warp_sum(loss);
}

// Sum of the q of every entry that has entry j's index, in list order: the
// entries of one index all find the same value.
__device__ __forceinline__ float q_of_index(const List& list, int top, int index) {
  float q = 0.f;
  for (int l = 0; l < top; ++l)
    if (list.index[l] == index) q += list.q[l];
  return q;
}

// (max, sum of exp2((z - max) c)) of two parts of a row.  A part without a
// finite element has max -inf and sum 0.
__device__ __forceinline__ float2 join(float2 x, float2 y, float c) {
  const float m = fmaxf(x.x, y.x);
  const float base = m == -INFINITY ? 0.f : m;
  return make_float2(m, x.y * fast_exp2((x.x - base) * c) + y.y * fast_exp2((y.x - base) * c));
}
__device__ __forceinline__ float2 warp_join(float2 v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = join(v, make_float2(__shfl_xor_sync(kFullMask, v.x, o), __shfl_xor_sync(kFullMask, v.y, o)),
             c);
  return v;
}

// One block a row, any vocabulary: reads the row for its statistics (unless
// `from_stats`), then, for the gradient, once more.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    distill_row_kernel(const __grid_constant__ muon_train_distill_args a, bool from_stats) {
  __shared__ List list;
  __shared__ float total_shared;
  __shared__ float2 part[kWarps];
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float c = kLog2e / a.temperature;
  if (warp == 0) {
    const float total = load_list(a, row, z, &list);
    if (lane == 0) total_shared = total;
  }
  float2 v = make_float2(-INFINITY, 0.f);
  if (!from_stats) {
    for (int64_t i = threadIdx.x; i < a.vocab; i += kThreads) v = join(v, make_float2(logit(z, i), 1.f), c);
    v = warp_join(v, c);
    if (lane == 0) part[warp] = v;
  }
  __syncthreads();
  if (from_stats) {
    v = make_float2(a.stats[2 * row], a.stats[2 * row + 1]);
  } else {
    v = part[0];
    for (int w = 1; w < kWarps; ++w) v = join(v, part[w], c);
  }
  const float total = total_shared;
  if (warp == 0 && a.loss != nullptr) {
    const float loss = row_loss(list, static_cast<int>(a.top), 1.0f / a.temperature, v.x, v.y);
    if (lane == 0) a.loss[row] = loss;
  }
  if (threadIdx.x == 0) {
    if (a.stats != nullptr && !from_stats) {
      a.stats[2 * row] = v.x;
      a.stats[2 * row + 1] = v.y;
    }
  }
  if (a.grad == nullptr) return;
  T* dz = static_cast<T*>(a.grad) + row * a.ld_grad;
  const float g = (a.row_scale != nullptr ? a.row_scale[row] : 1.f) / a.temperature;
  const bool none = g == 0.f || total == 0.f;  // zero whatever the logits hold
  const float p_scale = g * total / v.y;
  for (int64_t i = threadIdx.x; i < a.vocab; i += kThreads)
    dz[i] = from_float<T>(none ? 0.f : p_scale * fast_exp2((logit(z, i) - v.x) * c));
  if (none) return;
  __syncthreads();  // the listed elements are written again, with their q
  for (int j = threadIdx.x; j < a.top; j += kThreads) {
    const int i = list.index[j];
    if (i < 0) continue;
    const float q = q_of_index(list, static_cast<int>(a.top), i);
    dz[i] = from_float<T>(p_scale * fast_exp2((logit(z, i) - v.x) * c) - g * q);
  }
}

template <typename T>
int run(const muon_train_distill_args& a, bool from_stats, void* stream) {
  return launch(distill_row_kernel<T>, dim3(static_cast<unsigned>(a.rows)), kThreads, 0, 1, stream,
                a, from_stats);
}

int check(const muon_train_distill_args* a) {
  if (a == nullptr || a->rows < 0 || a->vocab < 1 || a->top < 1 || a->top > MUON_TRAIN_MAX_TOP ||
      a->rows > 0x7fffffff / 8 || a->vocab > 0x7fffff00 || !(a->temperature > 0.f) ||
      (a->rows > 1 && a->ld < a->vocab) || !valid_dtype(a->dtype) ||
      !valid_dtype(a->teacher_dtype) || (a->index_bytes != 4 && a->index_bytes != 8))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->rows > 0 && (a->logits == nullptr || a->teacher_logits == nullptr ||
                      a->teacher_indices == nullptr || a->grad == a->logits ||
                      (a->grad != nullptr && a->rows > 1 && a->ld_grad < a->vocab)))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}

int dispatch(const muon_train_distill_args& a, bool from_stats, void* stream) {
  if (a.rows == 0) return MUON_POLAR_OK;
  switch (a.dtype) {
    case MUON_TRAIN_F32: return run<float>(a, from_stats, stream);
    case MUON_TRAIN_BF16: return run<__nv_bfloat16>(a, from_stats, stream);
    default: return run<__half>(a, from_stats, stream);
  }
}

}  // namespace
}  // namespace muon_train

extern "C" {

uint64_t muon_train_launch_count(void) {
  return muon_train::launch_counter().load(std::memory_order_relaxed);
}

int muon_train_distill_sm100(const muon_train_distill_args* args, void* stream) {
  const int rc = muon_train::check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->rows > 0 && args->loss == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return muon_train::dispatch(*args, false, stream);
}

int muon_train_distill_backward_sm100(const muon_train_distill_args* args, void* stream) {
  const int rc = muon_train::check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->rows > 0 && (args->stats == nullptr || args->grad == nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  muon_train_distill_args a = *args;
  a.loss = nullptr;
  return muon_train::dispatch(a, true, stream);
}

}  // extern "C"
