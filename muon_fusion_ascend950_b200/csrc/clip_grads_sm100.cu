// clip_grads_sm100.cu -- the norm of many tensors taken as one vector, and the
// tensors times min(1, max_norm / (norm + 1e-6)).
//
// Two launches over the same work, a share of the elements for each block: the
// first leaves each block's sum of squares (or largest magnitude) in the
// workspace, the second adds them up, every block in the same order, and
// scales.  Bound by memory: the gradients are read once for the norm and once
// more to be scaled, where the second pass begins with what the first read
// last, which L2 still holds.  In place, gradients within the limit would be
// written back as they are: the second pass then only gives the norm.
//
// Squares are added up in 64 bits: those of fp32 gradients leave fp32's range
// from 10^19 and under 10^-19 on.
#include "train_common.cuh"

namespace muon_train {
namespace {

constexpr int kThreads = 512;
constexpr int kBlocksPerSm = 2;
constexpr int64_t kLeast = 8192;  // elements of a block
constexpr int kUnroll = 4;        // 16-byte loads in flight a thread

// The tensors of one launch travel as a kernel's parameters (at most 32764 bytes).
constexpr int kMost = 1024;
template <int kEntries>
struct Table {
  const void* in[kEntries];
  void* out[kEntries];
  int64_t end[kEntries];    // elements of the tensors up to and with this one
  uint8_t types[kEntries];  // of in, and 4 times of out
  int count;
};

// Element at which block `b` begins, in whole runs of 64.
__device__ __forceinline__ int64_t share(int64_t n, int64_t b, int64_t blocks) {
  const int64_t at = (n + 63) / 64 * b / blocks * 64;
  return at < n ? at : n;
}

// Of the sum of squares, or of the bits of the largest magnitude (those of NaN
// are above infinity's, so that a NaN stays).
template <bool kLargest>
struct Total {
  double v = 0.0;
  __device__ __forceinline__ void add(float x) {
    if constexpr (kLargest)
      v = fmax(v, static_cast<double>(__float_as_uint(x) & 0x7fffffffu));
    else
      v = fma(static_cast<double>(x), static_cast<double>(x), v);
  }
  __device__ __forceinline__ static double join(double a, double b) { return kLargest ? fmax(a, b) : a + b; }
  __device__ __forceinline__ double norm() const {
    return kLargest ? static_cast<double>(__uint_as_float(static_cast<uint32_t>(v))) : sqrt(v);
  }
};

// Joins a block's values in a fixed order; every thread gets the result.
template <bool kLargest>
__device__ __forceinline__ double block_total(double v) {
  __shared__ double of_warp[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = Total<kLargest>::join(v, __shfl_xor_sync(kFullMask, v, o));
  if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = v;
  __syncthreads();
  v = of_warp[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = Total<kLargest>::join(v, of_warp[w]);
  return v;
}

template <int kEntries>
__device__ __forceinline__ int64_t begin_of(const Table<kEntries>& t, int i) { return i > 0 ? t.end[i - 1] : 0; }
// The tensor that holds element `at`.
template <int kEntries>
__device__ __forceinline__ int find(const Table<kEntries>& t, int64_t at) {
  int low = 0, high = t.count - 1;
  while (low < high) {
    const int mid = (low + high) / 2;
    if (t.end[mid] > at)
      high = mid;
    else
      low = mid + 1;
  }
  return low;
}

// Elements before the first 16-byte boundary of p, at most n.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* p, int64_t n) {
  const int64_t h = (16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T);
  return h < n ? h : n;
}

template <typename T, bool kLargest>
__device__ __forceinline__ void total_of(const T* p, int64_t n, Total<kLargest>& total) {
  constexpr int kN = kVec<T>;
  const int64_t head = head_of(p, n), vectors = (n - head) / kN, tail = head + vectors * kN;
  for (int64_t i = threadIdx.x; i < head; i += kThreads) total.add(to_float(p[i]));
  for (int64_t i = tail + threadIdx.x; i < n; i += kThreads) total.add(to_float(p[i]));
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
  for (int64_t v0 = threadIdx.x; v0 < vectors; v0 += kThreads * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)  // beyond the end: zeros, which add nothing
      raw[u] = v0 + u * kThreads < vectors ? q[v0 + u * kThreads] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float x[kN];
      unpack<T>(raw[u], x);
#pragma unroll
      for (int j = 0; j < kN; ++j) total.add(x[j]);
    }
  }
}

template <int kEntries, bool kLargest>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    total_kernel(const __grid_constant__ Table<kEntries> t, double* partial) {
  begin_kernel();
  const int64_t all = t.end[t.count - 1];
  int64_t at = share(all, blockIdx.x, gridDim.x);
  const int64_t end = share(all, blockIdx.x + 1, gridDim.x);
  Total<kLargest> total;
  for (int i = find(t, at); at < end; ++i) {
    const int64_t begin = begin_of(t, i), stop = t.end[i] < end ? t.end[i] : end;
    const int64_t from = at - begin, n = stop - at;
    switch (t.types[i] & 3) {
      case MUON_TRAIN_F32: total_of(static_cast<const float*>(t.in[i]) + from, n, total); break;
      case MUON_TRAIN_BF16: total_of(static_cast<const __nv_bfloat16*>(t.in[i]) + from, n, total); break;
      default: total_of(static_cast<const __half*>(t.in[i]) + from, n, total); break;
    }
    at = stop;
  }
  const double v = block_total<kLargest>(total.v);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// out = factor * in, from the end to the beginning.
template <typename In, typename Out>
__device__ __forceinline__ void scale_run(const In* p, Out* out, int64_t n, float factor) {
  constexpr int kN = kVec<In>;
  const int64_t head = head_of(p, n), vectors = (n - head) / kN, tail = head + vectors * kN;
  constexpr uintptr_t kStore = kN * sizeof(Out) < 16 ? kN * sizeof(Out) : 16;
  const bool whole = reinterpret_cast<uintptr_t>(out + head) % kStore == 0;
  for (int64_t i = tail + threadIdx.x; i < n; i += kThreads) out[i] = from_float<Out>(to_float(p[i]) * factor);
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
  for (int64_t v0 = threadIdx.x; v0 < vectors; v0 += kThreads * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v0 + u * kThreads < vectors) raw[u] = q[vectors - 1 - v0 - u * kThreads];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (v0 + u * kThreads >= vectors) continue;
      const int64_t i = head + (vectors - 1 - v0 - u * kThreads) * kN;
      float x[kN];
      unpack<In>(raw[u], x);
#pragma unroll
      for (int j = 0; j < kN; ++j) x[j] *= factor;
      if (whole) {
        store_run<Out, kN>(out, i, x);
      } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) out[i + j] = from_float<Out>(x[j]);
      }
    }
  }
  for (int64_t i = threadIdx.x; i < head; i += kThreads) out[i] = from_float<Out>(to_float(p[i]) * factor);
}
template <typename In>
__device__ __forceinline__ void scale_into(const void* in, void* out, int dtype, int64_t from, int64_t n,
                                           float factor) {
  const In* p = static_cast<const In*>(in) + from;
  if (dtype == MUON_TRAIN_F32)
    scale_run(p, static_cast<float*>(out) + from, n, factor);
  else if (dtype == MUON_TRAIN_BF16)
    scale_run(p, static_cast<__nv_bfloat16*>(out) + from, n, factor);
  else
    scale_run(p, static_cast<__half*>(out) + from, n, factor);
}

template <int kEntries, bool kLargest>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    scale_kernel(const __grid_constant__ Table<kEntries> t, const double* partial, int partials,
                 double max_norm, float* norm) {
  begin_kernel();
  double v = 0.0;
  for (int i = threadIdx.x; i < partials; i += kThreads) v = Total<kLargest>::join(v, partial[i]);
  Total<kLargest> total;
  total.v = block_total<kLargest>(v);
  const double n = total.norm(), c = max_norm / (n + 1e-6);
  const float factor = c > 1.0 ? 1.0f : static_cast<float>(c);  // NaN stays
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  if (t.count == 0) return;
  const int64_t all = t.end[t.count - 1];
  const int64_t first = share(all, blockIdx.x, gridDim.x);
  int64_t end = share(all, blockIdx.x + 1, gridDim.x);
  if (first == end) return;
  for (int i = find(t, end - 1); end > first; --i) {
    const int64_t begin = begin_of(t, i), at = begin > first ? begin : first;
    const int in = t.types[i] & 3, out = t.types[i] >> 2;
    if (!(t.in[i] == t.out[i] && factor == 1.0f)) {
      if (in == MUON_TRAIN_F32)
        scale_into<float>(t.in[i], t.out[i], out, at - begin, end - at, factor);
      else if (in == MUON_TRAIN_BF16)
        scale_into<__nv_bfloat16>(t.in[i], t.out[i], out, at - begin, end - at, factor);
      else
        scale_into<__half>(t.in[i], t.out[i], out, at - begin, end - at, factor);
    }
    end = at;
  }
}

// ------------------------------------------------------------ host side
int blocks_for(int64_t elements, int sms) {
  const int64_t want = (elements + kLeast - 1) / kLeast, most = static_cast<int64_t>(sms) * kBlocksPerSm;
  return static_cast<int>(want < 1 ? 1 : want < most ? want : most);
}

// The next tensors of the list that are not empty, from *at on.
template <int kEntries>
int64_t fill(Table<kEntries>* t, const muon_train_clip_tensor* tensors, int64_t n, int64_t* at) {
  t->count = 0;
  int64_t end = 0;
  for (; *at < n && t->count < kEntries; ++*at) {
    const muon_train_clip_tensor& e = tensors[*at];
    if (e.count == 0) continue;
    t->in[t->count] = e.grad;
    t->out[t->count] = e.out;
    t->types[t->count] = static_cast<uint8_t>(e.dtype + 4 * e.out_dtype);
    t->end[t->count++] = end += e.count;
  }
  return end;
}

template <int kEntries, bool kLargest>
int run(const muon_train_clip_tensor* tensors, int64_t n, double max_norm, float* norm, double* partial,
        size_t slots, int sms, void* stream) {
  Table<kEntries> t;
  int partials = 0;
  for (int64_t at = 0; at < n;) {
    const int64_t elements = fill(&t, tensors, n, &at);
    if (t.count == 0) break;
    const int blocks = blocks_for(elements, sms);
    if (partials + static_cast<size_t>(blocks) > slots) return MUON_POLAR_ERR_WORKSPACE;
    const int rc = launch(total_kernel<kEntries, kLargest>, dim3(blocks), kThreads, 0, 1, true, stream, t,
                          partial + partials);
    if (rc != MUON_POLAR_OK) return rc;
    partials += blocks;
  }
  int64_t at = 0;
  do {
    const int64_t elements = fill(&t, tensors, n, &at);
    const int rc = launch(scale_kernel<kEntries, kLargest>, dim3(blocks_for(elements, sms)), kThreads, 0, 1, true,
                          stream, t, static_cast<const double*>(partial), partials, max_norm, norm);
    if (rc != MUON_POLAR_OK) return rc;
    norm = nullptr;
  } while (at < n);
  return MUON_POLAR_OK;
}

template <bool kLargest>
int run(const muon_train_clip_tensor* tensors, int64_t n, double max_norm, float* norm, double* partial,
        size_t slots, int sms, void* stream) {
  // A launch takes longer the more parameters it has.
  if (n <= 64) return run<64, kLargest>(tensors, n, max_norm, norm, partial, slots, sms, stream);
  if (n <= 256) return run<256, kLargest>(tensors, n, max_norm, norm, partial, slots, sms, stream);
  return run<kMost, kLargest>(tensors, n, max_norm, norm, partial, slots, sms, stream);
}

}  // namespace
}  // namespace muon_train

extern "C" {

size_t muon_train_clip_workspace_bytes(int64_t tensors) {
  using namespace muon_train;
  int sms = 0;
  if (tensors < 0 || sm_count(&sms) != MUON_POLAR_OK) return 0;
  const int64_t launches = tensors / kMost + 1;
  return static_cast<size_t>(launches) * sms * kBlocksPerSm * sizeof(double);
}

int muon_train_clip_sm100(const muon_train_clip_tensor* tensors, int64_t n, double max_norm, int norm_type,
                          float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace muon_train;
  if (n < 0 || (n > 0 && tensors == nullptr) || !(max_norm >= 0.0) || (norm_type != 0 && norm_type != 2) ||
      norm == nullptr)
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  int64_t all = 0;
  for (int64_t i = 0; i < n; ++i) {
    const muon_train_clip_tensor& t = tensors[i];
    if (t.count < 0 || t.count > (int64_t{1} << 48) || !valid_dtype(t.dtype) || !valid_dtype(t.out_dtype))
      return MUON_POLAR_ERR_INVALID_ARGUMENT;
    if (t.count == 0) continue;
    if (t.grad == nullptr || t.out == nullptr || (t.grad == t.out && t.dtype != t.out_dtype))
      return MUON_POLAR_ERR_INVALID_ARGUMENT;
    if (reinterpret_cast<uintptr_t>(t.grad) % dtype_size(t.dtype) != 0 ||
        reinterpret_cast<uintptr_t>(t.out) % dtype_size(t.out_dtype) != 0)
      return MUON_POLAR_ERR_ALIGNMENT;
    all += t.count;
    if (all > (int64_t{1} << 48)) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  }
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 8 != 0) return MUON_POLAR_ERR_WORKSPACE;
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != MUON_POLAR_OK) return rc;
  double* partial = static_cast<double*>(workspace);
  const size_t slots = workspace_bytes / sizeof(double);
  return norm_type == 2 ? run<false>(tensors, n, max_norm, norm, partial, slots, sms, stream)
                        : run<true>(tensors, n, max_norm, norm, partial, slots, sms, stream);
}

}  // extern "C"
