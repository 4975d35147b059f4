// route_experts_sm100.cu -- routing of tokens to experts and its gradient.
//
//   s = softmax(l) or sigmoid(l), key = s + bias; the best groups by the sum
//   of their one or two largest keys, then the k largest keys in them; the
//   weights are the chosen s, renormalised or not, times a scale.
//
// A choice between experts must not depend on a kernel's order of summation
// or contraction, so the sigmoid is 1 / (1 + expf(-l)) with each operation
// rounded by itself, the softmax's sum is held in 64 bits, and a softmax
// without bias is ordered by its logits.
#include "train_common.cuh"

namespace muon_train {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kSoftmax = 0;
constexpr float kTiny = 1e-20f;

__device__ __forceinline__ float sigmoid(float x) {
  return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-x)));
}

// Order-preserving unsigned image of a key: 0 is kept for "taken", 1 for NaN
// (below -inf); -0 and +0 are one key.
__device__ __forceinline__ uint32_t ordered(float key) {
  if (key != key) return 1u;
  const uint32_t b = __float_as_uint(key + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

// Scores of one token in shared memory, by one warp; returns nothing.
template <typename T>
__device__ void scores(const T* l, int experts, int score, float* s) {
  const int lane = threadIdx.x & 31;
  if (score != kSoftmax) {
    for (int e = lane; e < experts; e += 32) s[e] = sigmoid(to_float(l[e]));
  } else {
    float m = -INFINITY;
    for (int e = lane; e < experts; e += 32) m = fmaxf(m, to_float(l[e]));
    m = warp_max(m);
    double sum = 0.0;
    for (int e = lane; e < experts; e += 32) {
      const float x = m == -INFINITY && !(to_float(l[e]) != to_float(l[e]))
                          ? 0.f
                          : expf(__fsub_rn(to_float(l[e]), m));
      s[e] = x;
      sum += x;
    }
    const float total = static_cast<float>(warp_sum64(sum));
    for (int e = lane; e < experts; e += 32) s[e] = total == 0.f ? 0.f : __fdiv_rn(s[e], total);
  }
  __syncwarp();
}

// The largest key in s_key[0 .. n) of the warp's lanes: its lowest index, or
// -1 when all are taken.
__device__ int best_of(const uint32_t* keys, int n) {
  const int lane = threadIdx.x & 31;
  uint32_t best = 0;
  int at = n;
  for (int e = lane; e < n; e += 32)
    if (keys[e] > best) {
      best = keys[e];
      at = e;
    }
  const uint32_t top = __reduce_max_sync(kFullMask, best);
  const int index = __reduce_min_sync(kFullMask, best == top ? at : n);
  return top == 0 ? -1 : index;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    route_kernel(const __grid_constant__ muon_train_route_args a) {
  extern __shared__ float smem[];
  const int experts = static_cast<int>(a.experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s = smem + warp * 3 * experts;
  uint32_t* keys = reinterpret_cast<uint32_t*>(s + experts);
  uint32_t* group_keys = keys + experts;
  const bool by_logit = a.score == kSoftmax && a.bias == nullptr &&
                        (a.groups == 1 || a.group_top == 1);
  for (int64_t token = static_cast<int64_t>(blockIdx.x) * kWarps + warp; token < a.tokens;
       token += static_cast<int64_t>(gridDim.x) * kWarps) {
    const T* l = static_cast<const T*>(a.logits) + token * a.ld;
    scores(l, experts, a.score, s);
    for (int e = lane; e < experts; e += 32) {
      const float key = by_logit ? to_float(l[e])
                                 : (a.bias != nullptr ? __fadd_rn(s[e], a.bias[e]) : s[e]);
      keys[e] = ordered(key);
    }
    __syncwarp();
    if (a.groups > 1) {
      const int size = experts / a.groups;
      for (int g = lane; g < a.groups; g += 32) {
        float first = -INFINITY, second = -INFINITY;
        for (int e = g * size; e < (g + 1) * size; ++e) {
          const float key = by_logit ? to_float(l[e])
                                     : (a.bias != nullptr ? __fadd_rn(s[e], a.bias[e]) : s[e]);
          if (key > first) {
            second = first;
            first = key;
          } else if (key > second) {
            second = key;
          }
        }
        group_keys[g] = ordered(a.group_top == 2 ? __fadd_rn(first, second) : first);
      }
      __syncwarp();
      // the chosen groups' keys become 0: taken
      for (int j = 0; j < a.top_groups; ++j) {
        const int g = best_of(group_keys, a.groups);
        __syncwarp();
        if (lane == 0) group_keys[g] = 0;
        __syncwarp();
      }
      for (int e = lane; e < experts; e += 32)
        if (group_keys[e / size] != 0) keys[e] = 0;
      __syncwarp();
    }
    float total = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const int e = best_of(keys, experts);
      __syncwarp();
      if (lane == 0) {
        keys[e] = 0;
        a.indices[token * a.k + j] = e;
        if (a.counts != nullptr)
          atomicAdd(reinterpret_cast<unsigned long long*>(a.counts) + e, 1ull);
      }
      total += s[e];
      __syncwarp();
      if (!a.renormalize && lane == 0) a.weights[token * a.k + j] = s[e] * a.scale;
      if (a.renormalize && lane == 0) group_keys[j] = e;
    }
    __syncwarp();
    if (a.renormalize)
      for (int j = lane; j < a.k; j += 32)
        a.weights[token * a.k + j] = __fdiv_rn(s[group_keys[j]], total + kTiny) * a.scale;
    __syncwarp();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    route_backward_kernel(const __grid_constant__ muon_train_route_args a,
                          const float* __restrict__ grad_weights, T* __restrict__ grad) {
  extern __shared__ float smem[];
  const int experts = static_cast<int>(a.experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s = smem + warp * 2 * experts;
  float* d = s + experts;
  for (int64_t token = static_cast<int64_t>(blockIdx.x) * kWarps + warp; token < a.tokens;
       token += static_cast<int64_t>(gridDim.x) * kWarps) {
    scores(static_cast<const T*>(a.logits) + token * a.ld, experts, a.score, s);
    for (int e = lane; e < experts; e += 32) d[e] = 0.f;
    __syncwarp();
    float total = 0.f, dot = 0.f;  // over the chosen: s, and dw s
    for (int j = lane; j < a.k; j += 32) {
      const int64_t e = a.indices[token * a.k + j];
      if (e < 0 || e >= experts) continue;
      total += s[e];
      dot += grad_weights[token * a.k + j] * s[e];
    }
    total = warp_sum(total) + kTiny;
    dot = warp_sum(dot);
    for (int j = lane; j < a.k; j += 32) {
      const int64_t e = a.indices[token * a.k + j];
      if (e < 0 || e >= experts) continue;
      const float g = grad_weights[token * a.k + j];
      d[e] = a.scale * (a.renormalize ? (g - dot / total) / total : g);
    }
    __syncwarp();
    float shared = 0.f;  // softmax: sum of d s
    if (a.score == kSoftmax) {
      for (int e = lane; e < experts; e += 32) shared += d[e] * s[e];
      shared = warp_sum(shared);
    }
    T* out = grad + token * a.experts;
    for (int e = lane; e < experts; e += 32) {
      const float v = a.score == kSoftmax ? s[e] * (d[e] - shared) : d[e] * s[e] * (1.0f - s[e]);
      out[e] = from_float<T>(v);
    }
    __syncwarp();
  }
}

int check(const muon_train_route_args* a) {
  if (a == nullptr || a->tokens < 0 || a->experts < 1 || a->experts > MUON_TRAIN_MAX_EXPERTS ||
      a->k < 1 || a->k > MUON_TRAIN_MAX_ROUTES || a->groups < 1 || a->experts % a->groups != 0 ||
      a->top_groups < 1 || a->top_groups > a->groups ||
      a->k > a->top_groups * (a->experts / a->groups) ||
      (a->group_top != 1 && a->group_top != 2) ||
      (a->groups > 1 && a->group_top > a->experts / a->groups) || (a->score != 0 && a->score != 1) ||
      !valid_dtype(a->dtype) || (a->tokens > 1 && a->ld < a->experts))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->tokens > 0 && (a->logits == nullptr || a->indices == nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}

int grid_for(int64_t tokens, unsigned* grid) {
  int sms = 0;
  const int rc = sm_count(&sms);
  const int64_t want = (tokens + kWarps - 1) / kWarps;
  *grid = static_cast<unsigned>(want < sms * 8 ? want : sms * 8);
  return rc;
}

// Shared memory above 48 KB needs the kernel's leave.
template <typename Kernel>
int allow_smem(Kernel kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return MUON_POLAR_OK;
  return static_cast<int>(cudaFuncSetAttribute(
      kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
}

template <typename T>
int forward(const muon_train_route_args& a, void* stream) {
  unsigned grid = 0;
  const size_t smem = kWarps * 3 * a.experts * sizeof(float);
  int rc = grid_for(a.tokens, &grid);
  if (rc == MUON_POLAR_OK) rc = allow_smem(route_kernel<T>, smem);
  if (rc != MUON_POLAR_OK) return rc;
  return launch(route_kernel<T>, dim3(grid), kThreads, smem, 1, stream, a);
}

template <typename T>
int backward(const muon_train_route_args& a, const float* grad_weights, void* grad, void* stream) {
  unsigned grid = 0;
  const size_t smem = kWarps * 2 * a.experts * sizeof(float);
  int rc = grid_for(a.tokens, &grid);
  if (rc == MUON_POLAR_OK) rc = allow_smem(route_backward_kernel<T>, smem);
  if (rc != MUON_POLAR_OK) return rc;
  return launch(route_backward_kernel<T>, dim3(grid), kThreads, smem, 1, stream, a, grad_weights,
                static_cast<T*>(grad));
}

}  // namespace
}  // namespace muon_train

extern "C" {

int muon_train_route_sm100(const muon_train_route_args* args, void* stream) {
  using namespace muon_train;
  const int rc = check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->tokens > 0 && args->weights == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (args->counts != nullptr) {
    const cudaError_t e = cudaMemsetAsync(args->counts, 0, args->experts * sizeof(int64_t),
                                          static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  if (args->tokens == 0) return MUON_POLAR_OK;
  switch (args->dtype) {
    case MUON_TRAIN_F32: return forward<float>(*args, stream);
    case MUON_TRAIN_BF16: return forward<__nv_bfloat16>(*args, stream);
    default: return forward<__half>(*args, stream);
  }
}

int muon_train_route_backward_sm100(const muon_train_route_args* args, const float* grad_weights,
                                    void* grad_logits, void* stream) {
  using namespace muon_train;
  const int rc = check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->tokens == 0) return MUON_POLAR_OK;
  if (grad_weights == nullptr || grad_logits == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  switch (args->dtype) {
    case MUON_TRAIN_F32: return backward<float>(*args, grad_weights, grad_logits, stream);
    case MUON_TRAIN_BF16: return backward<__nv_bfloat16>(*args, grad_weights, grad_logits, stream);
    default: return backward<__half>(*args, grad_weights, grad_logits, stream);
  }
}

}  // extern "C"
