// train_common.cuh -- what the training-step kernels share: element types,
// 16-byte vectors of them, reductions in a fixed order, the launch helper.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "muon_train_sm100.h"
#include "sm100_ptx.cuh"

namespace muon_train {

constexpr unsigned kFullMask = 0xffffffffu;

// ------------------------------------------------------------ elements
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Element i of an array whose type is known at run time only: parameters and
// short lists, read once a row or once a block.
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == MUON_TRAIN_F32) return static_cast<const float*>(p)[i];
  if (dtype == MUON_TRAIN_BF16) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == MUON_TRAIN_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == MUON_TRAIN_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(v);
  else
    static_cast<__half*>(p)[i] = from_float<__half>(v);
}

// ------------------------------------------------------------ 16-byte vectors
template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ void unpack(const uint4& u, float (&v)[4], float) {
  v[0] = __uint_as_float(u.x);
  v[1] = __uint_as_float(u.y);
  v[2] = __uint_as_float(u.z);
  v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of its fp32
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[8], __half) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[kVec<T>]) {
  unpack(u, v, T());
}

__device__ __forceinline__ uint4 pack(const float (&v)[4], float) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                    __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], __nv_bfloat16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], __half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[kVec<T>]) {
  return pack(v, T());
}

// N elements as one load or store of N * sizeof(T) bytes: 16 bytes where rows
// keep that alignment, else pairs or single elements.
template <int kBytes>
struct RawOf;
template <>
struct RawOf<16> { using type = uint4; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<2> { using type = uint16_t; };

template <typename T, int N>
struct Elements {
  using Raw = typename RawOf<N * static_cast<int>(sizeof(T))>::type;
  static __device__ __forceinline__ Raw load(const T* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ void store(T* p, const Raw& r) { *reinterpret_cast<Raw*>(p) = r; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[N]) {
    if constexpr (sizeof(Raw) == 16) {
      muon_train::unpack<T>(r, v);
    } else {
      const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = to_float(e[i]);
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&v)[N]) {
    if constexpr (sizeof(Raw) == 16) {
      return muon_train::pack<T>(v);
    } else {
      Raw r;
      T* e = reinterpret_cast<T*>(&r);
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = from_float<T>(v[i]);
      return r;
    }
  }
};

// N elements from index i on of a parameter whose type is known at run time;
// i is a multiple of N and the array aligned to 16 bytes (N > 1).
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, int64_t i, float (&v)[N]) {
  constexpr int kPart = N * sizeof(T) > 16 ? 16 / static_cast<int>(sizeof(T)) : N;
#pragma unroll
  for (int j = 0; j < N; j += kPart) {
    float part[kPart];
    Elements<T, kPart>::unpack(Elements<T, kPart>::load(p + i + j), part);
#pragma unroll
    for (int l = 0; l < kPart; ++l) v[j + l] = part[l];
  }
}
template <int N>
__device__ __forceinline__ void load_any(const void* p, int dtype, int64_t i, float (&v)[N]) {
  if (dtype == MUON_TRAIN_F32)
    load_run<float, N>(static_cast<const float*>(p), i, v);
  else if (dtype == MUON_TRAIN_BF16)
    load_run<__nv_bfloat16, N>(static_cast<const __nv_bfloat16*>(p), i, v);
  else
    load_run<__half, N>(static_cast<const __half*>(p), i, v);
}
template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, int64_t i, const float (&v)[N]) {
  constexpr int kPart = N * sizeof(T) > 16 ? 16 / static_cast<int>(sizeof(T)) : N;
#pragma unroll
  for (int j = 0; j < N; j += kPart) {
    float part[kPart];
#pragma unroll
    for (int l = 0; l < kPart; ++l) part[l] = v[j + l];
    Elements<T, kPart>::store(p + i + j, Elements<T, kPart>::pack(part));
  }
}
template <int N>
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, const float (&v)[N]) {
  if (dtype == MUON_TRAIN_F32)
    store_run<float, N>(static_cast<float*>(p), i, v);
  else if (dtype == MUON_TRAIN_BF16)
    store_run<__nv_bfloat16, N>(static_cast<__nv_bfloat16*>(p), i, v);
  else
    store_run<__half, N>(static_cast<__half*>(p), i, v);
}

// First in every kernel, by every thread: lets the next kernel of the stream be
// set up, and waits until the one before has ended and its writes are seen.
__device__ __forceinline__ void begin_kernel() {
  muon_sm100::grid_launch_dependents();
  muon_sm100::grid_dependency_wait();
}

// ------------------------------------------------------------ arithmetic
// 2^x in one instruction (ex2.approx: at most 2 ulp; 2^-inf = 0).
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// Two fp32 operations in one instruction, each rounded as alone.  The pairs
// pass as 64-bit registers, so that they need not be put together again.
__device__ __forceinline__ uint64_t bits(float2 v) { return reinterpret_cast<const uint64_t&>(v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(bits(a)), "l"(bits(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(bits(a)), "l"(bits(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The largest element of a vector, joined to m; NaN elements are passed over.
__device__ __forceinline__ float vector_max(const uint4& u, float m, float) {
  return fmaxf(fmaxf(fmaxf(m, __uint_as_float(u.x)), fmaxf(__uint_as_float(u.y), __uint_as_float(u.z))),
               __uint_as_float(u.w));
}
template <typename Pair>
__device__ __forceinline__ Pair vector_max2(const uint4& u) {
  const Pair* p = reinterpret_cast<const Pair*>(&u);
  return __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
}
__device__ __forceinline__ float vector_max(const uint4& u, float m, __nv_bfloat16) {
  const float2 f = __bfloat1622float2(vector_max2<__nv_bfloat162>(u));
  return fmaxf(m, fmaxf(f.x, f.y));
}
__device__ __forceinline__ float vector_max(const uint4& u, float m, __half) {
  const float2 f = __half22float2(vector_max2<__half2>(u));
  return fmaxf(m, fmaxf(f.x, f.y));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}

// ------------------------------------------------------------ bounded waits
// Each translation unit has its own status word; the read call joins them.
static __device__ uint32_t g_status = 0;

// Waits for the phase of `bar`; false if it gave up after the wait limit, or
// (unless `alone`) once another thread of the block has.  The device status
// then tells, and the block runs on without waiting: its results are void.
// What it gave up on may still be in flight, so its barrier must not be armed
// again, and the block waits for it (drain_ring) before it ends.
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, volatile int* failed,
                                          bool alone = false) {
  if (muon_sm100::mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = muon_sm100::global_timer_ns();
  for (uint32_t spins = 1;; ++spins) {
    if (muon_sm100::mbar_try_wait(bar, parity)) return true;
    if (!alone && *failed) return false;
    if ((spins & 63u) != 0) continue;
    if (muon_sm100::global_timer_ns() - t0 > muon_sm100::g_wait_limit_ns) {
      *failed = 1;
      atomicOr(&g_status, MUON_TRAIN_STATUS_WAIT);
      return false;
    }
  }
}

// Before a block ends: waits for what is in flight to `n` barriers in a row of a
// ring, from its `stage` with `parity` on, whatever the limit of the other waits
// is set to.
__device__ __forceinline__ void drain_ring(uint64_t* bars, int stages, int stage, uint32_t parity, int n) {
  const uint64_t t0 = muon_sm100::global_timer_ns();
  while (n > 0) {
    if (!muon_sm100::mbar_try_wait(&bars[stage], parity)) {
      if (muon_sm100::global_timer_ns() - t0 > muon_sm100::kDefaultWaitLimitNs) return;
      continue;
    }
    --n;
    if (++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
  }
}

// Joins this translation unit's status to *flags, and zeroes it if asked.
static inline cudaError_t take_status(uint32_t* flags, int clear) {
  uint32_t v = 0;
  const uint32_t zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(g_status, &zero, sizeof(zero));
  *flags |= v;
  return e;
}

// This translation unit's wait limit on the current device.
static inline cudaError_t put_wait_limit(uint64_t limit_ns) {
  return cudaMemcpyToSymbol(muon_sm100::g_wait_limit_ns, &limit_ns, sizeof(limit_ns));
}
static inline cudaError_t get_wait_limit(uint64_t* limit_ns) {
  return cudaMemcpyFromSymbol(limit_ns, muon_sm100::g_wait_limit_ns, sizeof(*limit_ns));
}

// ------------------------------------------------------------ host side
std::atomic<uint64_t>& launch_counter();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool valid_dtype(int d) { return d >= MUON_TRAIN_F32 && d <= MUON_TRAIN_F16; }
inline size_t dtype_size(int d) { return d == MUON_TRAIN_F32 ? 4 : 2; }

// SMs of the current device, asked once for each.
inline int sm_count(int* sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const bool kept = dev >= 0 && dev < 64;
  *sms = kept ? known[dev].load(std::memory_order_relaxed) : 0;
  if (*sms > 0) return MUON_POLAR_OK;
  e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && kept) known[dev].store(*sms, std::memory_order_relaxed);
  return static_cast<int>(e);
}

// Lets a kernel have up to `bytes` of dynamic shared memory, once for each
// device.
template <auto kKernel>
int allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return MUON_POLAR_OK;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) return static_cast<int>(e);
  done.fetch_or(bit, std::memory_order_relaxed);
  return MUON_POLAR_OK;
}

// One launch, as clusters of `cluster` blocks along x when that is over 1.
// With `early`, by programmatic dependent launch: the kernel may be set up
// while its predecessor in the stream ends, and waits for it (begin_kernel)
// before it touches memory.
template <typename Kernel, typename... Args>
int launch(Kernel kernel, dim3 grid, int threads, size_t smem, int cluster, bool early, void* stream,
           Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return static_cast<int>(e);
  launch_counter().fetch_add(1, std::memory_order_relaxed);
  return MUON_POLAR_OK;
}

}  // namespace muon_train
