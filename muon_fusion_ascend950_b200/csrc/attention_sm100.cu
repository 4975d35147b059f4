// attention_sm100.cu -- attention of training sequences, forward and backward.
//
//   s_ij = scale q_i . k_j over the keys that query i sees
//   p_ij = exp(s_ij - lse_i), out_i = sum_j p_ij v_j
//   delta_i = dout_i . out_i, dp_ij = dout_i . v_j, ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij dout_i
// (dk and dv also over the query heads that share the key head).
//
// A warp a row: each lane holds four elements of the head, products are summed
// over the warp, and the softmax goes by a running maximum and sum.  The
// backward pass computes the probabilities again from lse: one kernel for the
// queries' rows, one for the keys' rows, so that no sum needs atomics.
#include "train_common.cuh"

namespace muon_train {
namespace {

constexpr int kWarps = 8;
constexpr int kDims = 4;  // of a lane

struct Rows {  // a row's sequence: its first row, its length, whether it counts
  int64_t first;
  int length;
};

// The sequence of row `r` (packed: of all tokens; else of batch entry b).
__device__ __forceinline__ Rows sequence_of(const muon_train_attention_args& a, int64_t b, int64_t r) {
  Rows s{0, static_cast<int>(a.length)};
  if (a.lengths != nullptr) {
    const int n = a.lengths[b];
    s.length = n < 0 ? 0 : n < a.length ? n : static_cast<int>(a.length);
  }
  if (a.offsets != nullptr) {
    int64_t low = 0, high = a.sequences + 1;  // offsets up to r: [0, low)
    while (low < high) {
      const int64_t mid = (low + high) / 2;
      if (a.offsets[mid] <= r)
        low = mid + 1;
      else
        high = mid;
    }
    s.first = r;
    s.length = 0;
    if (low > 0 && low <= a.sequences) {
      s.first = a.offsets[low - 1] < 0 ? 0 : a.offsets[low - 1];
      const int64_t end = a.offsets[low] < a.length ? a.offsets[low] : a.length;
      s.length = static_cast<int>(end - s.first);
    }
  }
  return s;
}

__device__ __forceinline__ int clip(int64_t v, int high) {
  return v < 0 ? 0 : v > high ? high : static_cast<int>(v);
}

template <typename T>
__device__ __forceinline__ void load_dims(const T* p, int dim, float (&v)[kDims]) {
  const int lane = threadIdx.x % 32;
  if (lane * kDims < dim) {
    Elements<T, kDims>::unpack(Elements<T, kDims>::load(p + lane * kDims), v);
  } else {
#pragma unroll
    for (int i = 0; i < kDims; ++i) v[i] = 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_dims(T* p, int dim, const float (&v)[kDims], float by) {
  const int lane = threadIdx.x % 32;
  if (lane * kDims >= dim) return;
  float w[kDims];
#pragma unroll
  for (int i = 0; i < kDims; ++i) w[i] = v[i] * by;
  Elements<T, kDims>::store(p + lane * kDims, Elements<T, kDims>::pack(w));
}
__device__ __forceinline__ float dot(const float (&a)[kDims], const float (&b)[kDims]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kDims; ++i) s = fmaf(a[i], b[i], s);
  return warp_sum(s);
}

template <typename T>
__device__ __forceinline__ const T* row_of(const void* p, const muon_train_strides& s, int64_t b, int64_t r,
                                           int64_t h) {
  return static_cast<const T*>(p) + b * s.batch + r * s.row + h * s.head;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    forward_kernel(const __grid_constant__ muon_train_attention_args a) {
  begin_kernel();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32, h = blockIdx.y;
  if (row >= a.batch * a.length) return;
  const int64_t b = row / a.length, r = row % a.length, kh = h / (a.heads / a.kv_heads);
  const int dim = static_cast<int>(a.dim);
  const Rows s = sequence_of(a, b, r);
  const int keys = a.lengths != nullptr || a.offsets != nullptr ? s.length : static_cast<int>(a.keys);
  const int64_t i = r - s.first, place = i + keys - s.length;
  int low = 0, high = i < s.length ? keys : 0;
  if (a.causal) high = clip(place + 1, high);
  if (a.window > 0) {
    low = clip(place - a.window + 1, high);
    high = clip(place + a.window, high);
  }
  float q[kDims], acc[kDims] = {};
  load_dims(row_of<T>(a.q, a.q_stride, b, r, h), dim, q);
  float top = -INFINITY, sum = 0.0f;
  for (int j = low; j < high; ++j) {
    float k[kDims], v[kDims];
    load_dims(row_of<T>(a.k, a.k_stride, b, s.first + j, kh), dim, k);
    load_dims(row_of<T>(a.v, a.v_stride, b, s.first + j, kh), dim, v);
    const float score = dot(q, k) * a.scale, next = fmaxf(top, score);
    const float old = expf(top - next), p = expf(score - next);
    sum = sum * old + p;
    top = next;
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] = acc[d] * old + p * v[d];
  }
  store_dims(static_cast<T*>(a.out) + (row * a.heads + h) * dim, dim, acc, sum > 0.0f ? 1.0f / sum : high > low ? NAN : 0.0f);
  if (threadIdx.x % 32 == 0) a.lse[h * a.batch * a.length + row] = high > low ? top + logf(sum) : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    query_grad_kernel(const __grid_constant__ muon_train_attention_args a,
                      const __grid_constant__ muon_train_attention_grads g) {
  begin_kernel();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32, h = blockIdx.y;
  if (row >= a.batch * a.length) return;
  const int64_t b = row / a.length, r = row % a.length, kh = h / (a.heads / a.kv_heads);
  const int dim = static_cast<int>(a.dim);
  const Rows s = sequence_of(a, b, r);
  const int keys = a.lengths != nullptr || a.offsets != nullptr ? s.length : static_cast<int>(a.keys);
  const int64_t i = r - s.first, place = i + keys - s.length;
  int low = 0, high = i < s.length ? keys : 0;
  if (a.causal) high = clip(place + 1, high);
  if (a.window > 0) {
    low = clip(place - a.window + 1, high);
    high = clip(place + a.window, high);
  }
  float q[kDims], o[kDims], go[kDims], acc[kDims] = {};
  load_dims(row_of<T>(a.q, a.q_stride, b, r, h), dim, q);
  load_dims(static_cast<const T*>(a.out) + (row * a.heads + h) * dim, dim, o);
  load_dims(row_of<T>(g.grad_out, g.grad_out_stride, b, r, h), dim, go);
  const float delta = dot(o, go), lse = a.lse[h * a.batch * a.length + row];
  if (threadIdx.x % 32 == 0) static_cast<float*>(g.workspace)[h * a.batch * a.length + row] = delta;
  for (int j = low; j < high; ++j) {
    float k[kDims], v[kDims];
    load_dims(row_of<T>(a.k, a.k_stride, b, s.first + j, kh), dim, k);
    load_dims(row_of<T>(a.v, a.v_stride, b, s.first + j, kh), dim, v);
    const float p = expf(dot(q, k) * a.scale - lse), ds = p * (dot(go, v) - delta);
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[d] = fmaf(ds, k[d], acc[d]);
  }
  store_dims(static_cast<T*>(g.grad_q) + (row * a.heads + h) * dim, dim, acc, a.scale);
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    key_grad_kernel(const __grid_constant__ muon_train_attention_args a,
                    const __grid_constant__ muon_train_attention_grads g) {
  begin_kernel();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + threadIdx.x / 32, kh = blockIdx.y;
  if (row >= a.batch * a.keys) return;
  const int64_t b = row / a.keys, r = row % a.keys, group = a.heads / a.kv_heads;
  const int dim = static_cast<int>(a.dim);
  const Rows s = sequence_of(a, b, r);
  const int keys = a.lengths != nullptr || a.offsets != nullptr ? s.length : static_cast<int>(a.keys);
  const int64_t j = r - s.first, place = j - (keys - s.length);  // the query that stands where this key does
  int low = 0, high = j < keys ? s.length : 0;
  if (a.causal) low = clip(place, high);
  if (a.window > 0) {
    low = clip(place - a.window + 1 > low ? place - a.window + 1 : low, high);
    high = clip(place + a.window, high);
  }
  float k[kDims], v[kDims], dk[kDims] = {}, dv[kDims] = {};
  load_dims(row_of<T>(a.k, a.k_stride, b, r, kh), dim, k);
  load_dims(row_of<T>(a.v, a.v_stride, b, r, kh), dim, v);
  for (int64_t h = kh * group; h < (kh + 1) * group; ++h) {
    for (int i = low; i < high; ++i) {
      const int64_t at = s.first + i, stat = h * a.batch * a.length + b * a.length + at;
      float q[kDims], go[kDims];
      load_dims(row_of<T>(a.q, a.q_stride, b, at, h), dim, q);
      load_dims(row_of<T>(g.grad_out, g.grad_out_stride, b, at, h), dim, go);
      const float p = expf(dot(q, k) * a.scale - a.lse[stat]);
      const float ds = p * (dot(go, v) - static_cast<const float*>(g.workspace)[stat]);
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        dk[d] = fmaf(ds, q[d], dk[d]);
        dv[d] = fmaf(p, go[d], dv[d]);
      }
    }
  }
  const int64_t to = (row * a.kv_heads + kh) * dim;
  store_dims(static_cast<T*>(g.grad_k) + to, dim, dk, a.scale);
  store_dims(static_cast<T*>(g.grad_v) + to, dim, dv, 1.0f);
}

// ------------------------------------------------------------ host side
int check(const muon_train_attention_args* a) {
  constexpr int64_t kMost = int64_t{1} << 30;
  if (a == nullptr || a->batch < 0 || a->length < 0 || a->keys < 0 || a->heads < 1 || a->kv_heads < 1 ||
      a->heads % a->kv_heads != 0 || a->dim < 8 || a->dim > MUON_TRAIN_MAX_HEAD_DIM || a->dim % 8 != 0 ||
      a->window < 0 || !(a->scale > 0.0f && a->scale < INFINITY) ||
      (a->dtype != MUON_TRAIN_BF16 && a->dtype != MUON_TRAIN_F16))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->batch > 65535 || a->length > kMost || a->keys > kMost || a->batch * a->length > kMost ||
      a->batch * a->keys > kMost || a->heads > 65535)
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if ((a->lengths != nullptr || a->offsets != nullptr) && a->keys != a->length) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->offsets != nullptr &&
      (a->lengths != nullptr || a->batch != 1 || a->sequences < 0 || a->sequences > kMost))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}
bool strided(const void* p, const muon_train_strides& s, int64_t batch, int64_t rows, int64_t heads) {
  const auto fits = [](int64_t n, int64_t stride) { return n <= 1 || (stride >= 8 && stride % 8 == 0); };
  return p != nullptr && aligned16(p) && fits(batch, s.batch) && fits(rows, s.row) && fits(heads, s.head);
}
int check_forward(const muon_train_attention_args& a) {
  if (a.batch * a.length > 0 && !strided(a.q, a.q_stride, a.batch, a.length, a.heads)) return MUON_POLAR_ERR_ALIGNMENT;
  if (a.batch * a.keys > 0 && (!strided(a.k, a.k_stride, a.batch, a.keys, a.kv_heads) ||
                               !strided(a.v, a.v_stride, a.batch, a.keys, a.kv_heads)))
    return MUON_POLAR_ERR_ALIGNMENT;
  if (a.batch * a.length > 0 && (a.out == nullptr || !aligned16(a.out) || a.lse == nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}

dim3 grid_for(int64_t rows, int64_t heads) {
  return dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps), static_cast<unsigned>(heads));
}

template <typename T>
int backward(const muon_train_attention_args& a, const muon_train_attention_grads& g, void* stream) {
  if (a.batch * a.length > 0) {
    const int rc = launch(query_grad_kernel<T>, grid_for(a.batch * a.length, a.heads), kWarps * 32, 0, 1, true, stream, a, g);
    if (rc != MUON_POLAR_OK) return rc;
  }
  if (a.batch * a.keys == 0) return MUON_POLAR_OK;
  return launch(key_grad_kernel<T>, grid_for(a.batch * a.keys, a.kv_heads), kWarps * 32, 0, 1, true, stream, a, g);
}

}  // namespace
}  // namespace muon_train

extern "C" {

int muon_train_attention_sm100(const muon_train_attention_args* args, void* stream) {
  using namespace muon_train;
  int rc = check(args);
  if (rc == MUON_POLAR_OK) rc = check_forward(*args);
  if (rc != MUON_POLAR_OK || args->batch * args->length == 0) return rc;
  const dim3 grid = grid_for(args->batch * args->length, args->heads);
  return args->dtype == MUON_TRAIN_BF16
             ? launch(forward_kernel<__nv_bfloat16>, grid, kWarps * 32, 0, 1, true, stream, *args)
             : launch(forward_kernel<__half>, grid, kWarps * 32, 0, 1, true, stream, *args);
}

size_t muon_train_attention_workspace_bytes(const muon_train_attention_args* args) {
  using namespace muon_train;
  if (check(args) != MUON_POLAR_OK) return 0;
  return static_cast<size_t>(args->heads * args->batch * args->length + 4) * sizeof(float);
}

int muon_train_attention_backward_sm100(const muon_train_attention_args* args,
                                        const muon_train_attention_grads* grads, void* stream) {
  using namespace muon_train;
  int rc = check(args);
  if (rc == MUON_POLAR_OK) rc = check_forward(*args);
  if (rc != MUON_POLAR_OK) return rc;
  if (grads == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  const muon_train_attention_args& a = *args;
  const muon_train_attention_grads& g = *grads;
  if (a.batch * a.length > 0) {
    if (!strided(g.grad_out, g.grad_out_stride, a.batch, a.length, a.heads)) return MUON_POLAR_ERR_ALIGNMENT;
    if (g.grad_q == nullptr || !aligned16(g.grad_q)) return MUON_POLAR_ERR_INVALID_ARGUMENT;
    if (g.workspace == nullptr || !aligned16(g.workspace) ||
        g.workspace_bytes < muon_train_attention_workspace_bytes(args))
      return MUON_POLAR_ERR_WORKSPACE;
  }
  if (a.batch * a.keys > 0 && (g.grad_k == nullptr || g.grad_v == nullptr || !aligned16(g.grad_k) || !aligned16(g.grad_v)))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return a.dtype == MUON_TRAIN_BF16 ? backward<__nv_bfloat16>(a, g, stream) : backward<__half>(a, g, stream);
}

}  // extern "C"
