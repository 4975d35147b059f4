// clip_grads_sm100.cu -- the norm of many tensors taken as one vector, and the
// tensors times min(1, max_norm / (norm + 1e-6)).
//
// Two launches over the same work, chunks of the tensors dealt out to the blocks
// in turn: the first leaves each block's sum of squares (or largest magnitude)
// in the workspace, the second adds them up, every block in the same order, and
// scales.  (With one run of neighbouring elements a block, all the short
// tensors of a model, which stand together, fell to one of them: 57 us for 40
// MB.)  Bound by memory: the gradients are read once for the norm and once
// more to be scaled, where the second pass begins with what the first read
// last, which L2 still holds.  In place, gradients within the limit would be
// written back as they are: the second pass then only gives the norm (640 M
// bf16: 202 to 214 us, 6.0 to 6.3 TB/s).  160 M fp32 into bf16: 253 us for 1.6
// GB, of which 0.6 are the second reading.
//
// A few small tensors take one launch: a cluster of blocks, which exchange their
// sums through shared memory.
//
// Squares are added up in fp32 over the elements of one 16-byte load and in 64
// bits from there on: converting every element to 64 bits is what bounded the
// first pass before (640 M bf16: 3.8 TB/s).  A load whose sum leaves the range
// in which that is exact to a few roundings (squares of 10^19, or of 10^-12
// alone) is added up again in 64 bits.
//
// Tensors lie at any element, and so do the outputs: the second pass stores
// whole aligned vectors and puts each one's elements together from the two
// aligned 16-byte granules that hold them.
#include "train_common.cuh"

namespace muon_train {
namespace {

constexpr int kThreads = 512;
constexpr int kBlocksPerSm = 2;
constexpr int kUnroll = 4;     // 16-byte loads in flight a thread that scales
constexpr int kUnrollSum = 8;  // and one that adds up (4: 228 us for 1.28 GB)
// Elements of a chunk: as many as a block has in flight, of 16-bit types, or
// fewer where there are not two for each block.
constexpr int64_t kMostChunk = kThreads * kUnrollSum * 8, kLeastChunk = kThreads * 4;

// The tensors of one launch travel as a kernel's parameters (at most 32764 bytes).
constexpr int kMost = 1024;
template <int kEntries>
struct Table {
  const void* in[kEntries];
  void* out[kEntries];
  int64_t elements[kEntries];
  int32_t end[kEntries];    // chunks of the tensors up to and with this one
  uint8_t types[kEntries];  // of in, and 4 times of out
  int64_t chunk;            // elements of one
  int count;
  int in_place;             // all of them
};

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

// The tensor that chunk `c` belongs to, from tensor `low` on.
template <int kEntries>
__device__ __forceinline__ int find(const Table<kEntries>& t, int c, int low, int high) {
  while (low < high) {
    const int mid = (low + high) / 2;
    if (t.end[mid] > c)
      high = mid;
    else
      low = mid + 1;
  }
  return low;
}
// First element of chunk `c` of tensor `i`, and how many there are.
template <int kEntries>
__device__ __forceinline__ int64_t run_of(const Table<kEntries>& t, int i, int c, int64_t* n) {
  const int64_t from = (c - (i > 0 ? t.end[i - 1] : 0)) * t.chunk, left = t.elements[i] - from;
  *n = left < t.chunk ? left : t.chunk;
  return from;
}

// Elements before the first 16-byte boundary of p, at most n.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* p, int64_t n) {
  const int64_t h = (16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T);
  return h < n ? h : n;
}

// The elements of one load.
template <typename T, bool kLargest>
__device__ __forceinline__ void add_load(const uint4& raw, Total<kLargest>& total) {
  constexpr int kN = kVec<T>;
  float x[kN];
  unpack<T>(raw, x);
  if constexpr (kLargest) {
#pragma unroll
    for (int j = 0; j < kN; ++j) total.add(x[j]);
  } else {
    float2 s = mul2(make_float2(x[0], x[1]), make_float2(x[0], x[1]));
#pragma unroll
    for (int j = 2; j < kN; j += 2) s = fma2(make_float2(x[j], x[j + 1]), make_float2(x[j], x[j + 1]), s);
    const float sum = s.x + s.y;
    if (sum >= 0x1p-80f && sum <= 0x1p120f) {
      total.v += static_cast<double>(sum);
    } else if ((raw.x | raw.y | raw.z | raw.w) != 0) {
#pragma unroll
      for (int j = 0; j < kN; ++j) total.add(x[j]);
    }
  }
}

// By kGroup threads, of which this is thread `rank`.
template <int kGroup, typename T, bool kLargest>
__device__ __forceinline__ void total_of(const T* p, int64_t n, int rank, Total<kLargest>& total) {
  constexpr int kN = kVec<T>;
  const int64_t head = head_of(p, n), vectors = (n - head) / kN, tail = head + vectors * kN;
  for (int64_t i = rank; i < head; i += kGroup) total.add(to_float(p[i]));
  for (int64_t i = tail + rank; i < n; i += kGroup) total.add(to_float(p[i]));
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
  int64_t v = rank;
  for (; v + (kUnrollSum - 1) * kGroup < vectors; v += kGroup * kUnrollSum) {
    uint4 raw[kUnrollSum];
#pragma unroll
    for (int u = 0; u < kUnrollSum; ++u) raw[u] = q[v + u * kGroup];
#pragma unroll
    for (int u = 0; u < kUnrollSum; ++u) add_load<T>(raw[u], total);
  }
  for (; v < vectors; v += kGroup) add_load<T>(q[v], total);
}

// The share of group `group` of `groups` of kGroup threads.
template <int kGroup, int kEntries, bool kLargest>
__device__ __forceinline__ double share_total(const Table<kEntries>& t, int group, int groups, int rank) {
  const int chunks = t.count > 0 ? t.end[t.count - 1] : 0;
  Total<kLargest> total;
  int i = 0;
  for (int c = group; c < chunks; c += groups) {
    i = find(t, c, i, t.count - 1);
    int64_t n;
    const int64_t from = run_of(t, i, c, &n);
    switch (t.types[i] & 3) {
      case MUON_TRAIN_F32: total_of<kGroup>(static_cast<const float*>(t.in[i]) + from, n, rank, total); break;
      case MUON_TRAIN_BF16: total_of<kGroup>(static_cast<const __nv_bfloat16*>(t.in[i]) + from, n, rank, total); break;
      default: total_of<kGroup>(static_cast<const __half*>(t.in[i]) + from, n, rank, total); break;
    }
  }
  return total.v;
}

template <int kEntries, bool kLargest>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    total_kernel(const __grid_constant__ Table<kEntries> t, double* partial) {
  begin_kernel();
  const double mine = share_total<kThreads, kEntries, kLargest>(t, blockIdx.x, gridDim.x, threadIdx.x);
  const double v = block_total<kLargest>(mine);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// A granule's bytes from byte `shift` (even) on of two side by side.
__device__ __forceinline__ uint4 joined(const uint4& a, const uint4& b, int shift) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (shift & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (shift & 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint2 joined(const uint2& a, const uint2& b, int shift) {
  uint32_t w[4] = {a.x, a.y, b.x, b.y};
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 3; ++i) w[i] = w[i + 1];
  }
  if (shift & 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint2(w[0], w[1]);
}

// out = factor * in by kGroup threads, from the end to the beginning, in
// vectors that are 16 bytes of the wider type: neighbouring threads then load
// and store neighbouring bytes (16-bit types into fp32 by eight elements a
// thread stored every other 16 bytes at a time).
template <int kGroup, typename In, typename Out>
__device__ __noinline__ void scale_run(const In* p, Out* out, int64_t n, float factor, int rank) {
  constexpr int kN = 16 / static_cast<int>(sizeof(In) > sizeof(Out) ? sizeof(In) : sizeof(Out));
  constexpr int kLoad = kN * static_cast<int>(sizeof(In)), kStore = kN * static_cast<int>(sizeof(Out));  // bytes
  constexpr int kFlight = kLoad == 16 ? kUnroll : 2 * kUnroll;
  using E = Elements<In, kN>;
  using Raw = typename E::Raw;
  // vectors begin where a store of the output may; those whose input needs two granules stay clear of both ends
  int64_t head = (kStore - reinterpret_cast<uintptr_t>(out) % kStore) % kStore / sizeof(Out);
  if (head > n) head = n;
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(p + head) % kLoad);
  if (shift != 0) head = head + kN < n ? head + kN : n;
  int64_t vectors = (n - head) / kN;
  if (shift != 0 && vectors > 0) --vectors;
  const int64_t tail = head + vectors * kN;
  for (int64_t i = tail + rank; i < n; i += kGroup) out[i] = from_float<Out>(to_float(p[i]) * factor);
  const Raw* q = reinterpret_cast<const Raw*>(reinterpret_cast<uintptr_t>(p + head) - shift);
  const auto put = [&](int64_t v, const Raw& raw) {
    float x[kN];
    E::unpack(raw, x);
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] *= factor;
    Elements<Out, kN>::store(out + head + v * kN, Elements<Out, kN>::pack(x));
  };
  int64_t v = vectors - 1 - rank;
  if (shift == 0) {
    for (; v >= (kFlight - 1) * kGroup; v -= kGroup * kFlight) {
      Raw raw[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) raw[u] = q[v - u * kGroup];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) put(v - u * kGroup, raw[u]);
    }
    for (; v >= 0; v -= kGroup) put(v, q[v]);
  } else {
    for (; v >= (kFlight - 1) * kGroup; v -= kGroup * kFlight) {
      Raw a[kFlight], b[kFlight];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) a[u] = q[v - u * kGroup], b[u] = q[v - u * kGroup + 1];
#pragma unroll
      for (int u = 0; u < kFlight; ++u) put(v - u * kGroup, joined(a[u], b[u], shift));
    }
    for (; v >= 0; v -= kGroup) put(v, joined(q[v], q[v + 1], shift));
  }
  for (int64_t i = rank; i < head; i += kGroup) out[i] = from_float<Out>(to_float(p[i]) * factor);
}
template <int kGroup, typename In>
__device__ __forceinline__ void scale_into(const void* in, void* out, int dtype, int64_t from, int64_t n,
                                           float factor, int rank) {
  const In* p = static_cast<const In*>(in) + from;
  if (dtype == MUON_TRAIN_F32)
    scale_run<kGroup>(p, static_cast<float*>(out) + from, n, factor, rank);
  else if (dtype == MUON_TRAIN_BF16)
    scale_run<kGroup>(p, static_cast<__nv_bfloat16*>(out) + from, n, factor, rank);
  else
    scale_run<kGroup>(p, static_cast<__half*>(out) + from, n, factor, rank);
}

// The share of group `group` of `groups` of kGroup threads, from the end on.
template <int kGroup, int kEntries>
__device__ __forceinline__ void scale_share(const Table<kEntries>& t, float factor, int group, int groups, int rank) {
  if (t.count == 0 || (t.in_place && factor == 1.0f)) return;
  int i = t.count - 1;
  for (int c = t.end[i] - 1 - group; c >= 0; c -= groups) {
    i = find(t, c, 0, i);
    int64_t n;
    const int64_t from = run_of(t, i, c, &n);
    const int in = t.types[i] & 3, out = t.types[i] >> 2;
    if (t.in[i] == t.out[i] && factor == 1.0f) continue;
    if (in == MUON_TRAIN_F32)
      scale_into<kGroup, float>(t.in[i], t.out[i], out, from, n, factor, rank);
    else if (in == MUON_TRAIN_BF16)
      scale_into<kGroup, __nv_bfloat16>(t.in[i], t.out[i], out, from, n, factor, rank);
    else
      scale_into<kGroup, __half>(t.in[i], t.out[i], out, from, n, factor, rank);
  }
}
// Without a limit nothing is scaled, whatever the norm is: inf / inf is none.
__device__ __forceinline__ float factor_of(double norm, double max_norm) {
  if (max_norm == static_cast<double>(INFINITY)) return 1.0f;
  const double c = max_norm / (norm + 1e-6);
  return c > 1.0 ? 1.0f : static_cast<float>(c);  // NaN stays
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
  const double n = total.norm();
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  scale_share<kThreads>(t, factor_of(n, max_norm), blockIdx.x, gridDim.x, threadIdx.x);
}

// Both passes by one cluster, whose blocks are the whole grid; a warp a chunk, so
// that many tensors are on their way at once.
constexpr int kCluster = 8;
template <int kEntries, bool kLargest>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    small_kernel(const __grid_constant__ Table<kEntries> t, double max_norm, float* norm) {
  __shared__ double of_block;
  begin_kernel();
  const int warp = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x % 32;
  const double mine = block_total<kLargest>(share_total<32, kEntries, kLargest>(t, warp, kCluster * kThreads / 32, lane));
  if (threadIdx.x == 0) of_block = mine;
  muon_sm100::cluster_sync();
  Total<kLargest> total;
#pragma unroll
  for (int b = 0; b < kCluster; ++b) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];"
                 : "=d"(v)
                 : "r"(muon_sm100::map_to_cta(muon_sm100::smem_addr(&of_block), b))
                 : "memory");
    total.v = Total<kLargest>::join(total.v, v);
  }
  muon_sm100::cluster_sync();  // a block's memory stays until all have read it
  const double n = total.norm();
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  scale_share<32>(t, factor_of(n, max_norm), warp, kCluster * kThreads / 32, lane);
}

// ------------------------------------------------------------ host side
// What one cluster takes: one launch less, which a call bound by the host notices
// (24 tensors of 200000 fp32 in all: 5.7 us on the device), but eight blocks have
// to read it all (500000: 17 us, 7 with two launches).
constexpr int kFew = 64;
constexpr int64_t kSmall = int64_t{1} << 18;

int blocks_for(int chunks, int sms) {
  const int most = sms * kBlocksPerSm;
  return chunks < 1 ? 1 : chunks < most ? chunks : most;
}

// Elements of a chunk of tensors of `elements` in all.
int64_t chunk_for(int64_t elements, int sms) {
  int64_t chunk = elements / (2 * kBlocksPerSm * sms) / kLeastChunk * kLeastChunk;
  chunk = chunk < kLeastChunk ? kLeastChunk : chunk < kMostChunk ? chunk : kMostChunk;
  while (elements / chunk > (int64_t{1} << 30)) chunk *= 2;
  return chunk;
}

// The next tensors of the list that are not empty, from *at on; their chunks.
template <int kEntries>
int fill(Table<kEntries>* t, const muon_train_clip_tensor* tensors, int64_t n, int64_t* at, int64_t chunk) {
  t->count = 0;
  t->chunk = chunk;
  t->in_place = 1;
  int64_t end = 0;
  for (; *at < n && t->count < kEntries; ++*at) {
    const muon_train_clip_tensor& e = tensors[*at];
    if (e.count == 0) continue;
    t->in[t->count] = e.grad;
    t->out[t->count] = e.out;
    t->elements[t->count] = e.count;
    t->types[t->count] = static_cast<uint8_t>(e.dtype + 4 * e.out_dtype);
    t->in_place = t->in_place && e.grad == e.out;
    end += (e.count + chunk - 1) / chunk;
    t->end[t->count++] = static_cast<int32_t>(end);
  }
  return static_cast<int>(end);
}

template <int kEntries, bool kLargest>
int run(const muon_train_clip_tensor* tensors, int64_t n, int64_t all, double max_norm, float* norm, double* partial,
        size_t slots, int sms, void* stream) {
  const int64_t chunk = chunk_for(all, sms);
  Table<kEntries> t;
  int partials = 0;
  if constexpr (kEntries == kFew) {
    if (all <= kSmall) {
      int64_t at = 0;
      fill(&t, tensors, n, &at, chunk);
      return launch(small_kernel<kFew, kLargest>, dim3(kCluster), kThreads, 0, kCluster, true, stream, t, max_norm, norm);
    }
  }
  for (int64_t at = 0; at < n;) {
    const int blocks = blocks_for(fill(&t, tensors, n, &at, chunk), sms);
    if (t.count == 0) break;
    if (partials + static_cast<size_t>(blocks) > slots) return MUON_POLAR_ERR_WORKSPACE;
    const int rc = launch(total_kernel<kEntries, kLargest>, dim3(blocks), kThreads, 0, 1, true, stream, t,
                          partial + partials);
    if (rc != MUON_POLAR_OK) return rc;
    partials += blocks;
  }
  int64_t at = 0;
  do {
    const int blocks = blocks_for(fill(&t, tensors, n, &at, chunk), sms);
    const int rc = launch(scale_kernel<kEntries, kLargest>, dim3(blocks), kThreads, 0, 1, true, stream, t,
                          static_cast<const double*>(partial), partials, max_norm, norm);
    if (rc != MUON_POLAR_OK) return rc;
    norm = nullptr;
  } while (at < n);
  return MUON_POLAR_OK;
}

template <bool kLargest>
int run(const muon_train_clip_tensor* tensors, int64_t n, int64_t all, double max_norm, float* norm, double* partial,
        size_t slots, int sms, void* stream) {
  // A launch takes longer the more parameters it has.
  if (n <= kFew) return run<kFew, kLargest>(tensors, n, all, max_norm, norm, partial, slots, sms, stream);
  if (n <= 256) return run<256, kLargest>(tensors, n, all, max_norm, norm, partial, slots, sms, stream);
  return run<kMost, kLargest>(tensors, n, all, max_norm, norm, partial, slots, sms, stream);
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
  return norm_type == 2 ? run<false>(tensors, n, all, max_norm, norm, partial, slots, sms, stream)
                        : run<true>(tensors, n, all, max_norm, norm, partial, slots, sms, stream);
}

}  // extern "C"
