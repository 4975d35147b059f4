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
#include <algorithm>
#include <cfloat>

#include "sm100_ptx.cuh"
#include "train_common.cuh"

namespace muon_train {

cudaError_t norm_status(uint32_t* flags, int clear);  // residual_norm_sm100.cu
cudaError_t norm_put_wait_limit(uint64_t limit_ns);
cudaError_t norm_get_wait_limit(uint64_t* limit_ns);
cudaError_t attention_status(uint32_t* flags, int clear);  // attention_sm100.cu
cudaError_t attention_put_wait_limit(uint64_t limit_ns);
cudaError_t attention_get_wait_limit(uint64_t* limit_ns);

cudaError_t set_wait_limit(uint64_t limit_ns) {  // called by muon_polar_set_wait_limit_ns
  cudaError_t e = put_wait_limit(limit_ns);
  if (e == cudaSuccess) e = norm_put_wait_limit(limit_ns);
  return e != cudaSuccess ? e : attention_put_wait_limit(limit_ns);
}

std::atomic<uint64_t>& launch_counter() {
  static std::atomic<uint64_t> count{0};
  return count;
}

namespace {

// A row's list in shared memory: index (-1: not counted), q, log q and the
// student's logit.
struct List {
  int* index;
  float *q, *log_q, *z;
  static __host__ __device__ size_t bytes(int64_t top) { return static_cast<size_t>(top) * 16; }
  __device__ List(void* at, int top)
      : index(static_cast<int*>(at)), q(reinterpret_cast<float*>(index + top)), log_q(q + top), z(log_q + top) {}
};

template <typename T>
__device__ __forceinline__ float logit(const T* row, int64_t i) { return to_float(row[i]); }

// An index of 4 or 8 bytes and a value of 2 or 4, without branches on the
// type: several entries' loads can then be on their way together.
__device__ __forceinline__ int64_t load_index(const uint8_t* p, int bytes) {
  const int32_t low = *reinterpret_cast<const int32_t*>(p);
  const int32_t high = *reinterpret_cast<const int32_t*>(p + (bytes - 4));
  return bytes == 8 ? static_cast<int64_t>(high) << 32 | static_cast<uint32_t>(low) : static_cast<int64_t>(low);
}
__device__ __forceinline__ float load_value(const uint8_t* p, int dtype) {
  const uint32_t low = *reinterpret_cast<const uint16_t*>(p);
  const uint32_t high = *reinterpret_cast<const uint16_t*>(p + (dtype == MUON_TRAIN_F32 ? 2 : 0));
  const float half = __half2float(__ushort_as_half(static_cast<unsigned short>(low)));
  const float other = __uint_as_float(high << 16 | (dtype == MUON_TRAIN_F32 ? low : 0u));
  return dtype == MUON_TRAIN_F16 ? half : other;
}

// A row's list from memory, four entries a lane at a time: the indices and
// teacher logits first, then the student's logits at the indices, so that four
// entries wait for memory twice, and not each of them.  Returns the largest
// counted teacher logit of the lane's.
template <typename T>
__device__ __forceinline__ float load_entries(const muon_train_distill_args& a, int64_t row, const T* z,
                                              const List& list) {
  constexpr int kBatch = 4;
  const int lane = threadIdx.x & 31, top = static_cast<int>(a.top), value_bytes = a.teacher_dtype == MUON_TRAIN_F32 ? 4 : 2;
  const uint8_t* indices = static_cast<const uint8_t*>(a.teacher_indices) + row * a.top * a.index_bytes;
  const uint8_t* values = static_cast<const uint8_t*>(a.teacher_logits) + row * a.top * value_bytes;
  float best = -INFINITY;
  for (int base = lane; base < top; base += 32 * kBatch) {
    int64_t index[kBatch];
    float t[kBatch], zi[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int j = min(base + b * 32, top - 1);  // the last entry again, past the end
      index[b] = load_index(indices + static_cast<int64_t>(j) * a.index_bytes, a.index_bytes);
      t[b] = load_value(values + static_cast<int64_t>(j) * value_bytes, a.teacher_dtype);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const bool counted = index[b] >= 0 && index[b] < a.vocab && t[b] > -INFINITY;
      index[b] = counted ? index[b] : -1;
      zi[b] = logit(z, counted ? index[b] : 0);
      best = counted ? fmaxf(best, t[b]) : best;
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int j = base + b * 32;
      if (j >= top) break;
      list.index[j] = static_cast<int>(index[b]);
      list.log_q[j] = t[b];
      list.z[j] = zi[b];
    }
  }
  return best;
}

// Fills the list and returns Q; one whole warp, each lane its own entries.
// The differences to the largest entry are taken before the division by tau,
// so that entries of the type's lowest value stay finite.
template <typename T>
__device__ float load_list(const muon_train_distill_args& a, int64_t row, const T* z, const List& list) {
  const int lane = threadIdx.x & 31;
  const int top = static_cast<int>(a.top);
  const float inv_tau = 1.0f / a.temperature;
  float best = load_entries(a, row, z, list);
  best = warp_max(best);
  // log q = (t - shift) / tau - log_norm
  float shift = 0.f, log_norm = 0.f;
  if (a.teacher_lse != nullptr) {
    log_norm = a.teacher_lse[row];
  } else if (best > -INFINITY) {
    shift = best;
    float s = 0.f;
    for (int j = lane; j < top; j += 32)
      if (list.index[j] >= 0) s += expf((list.log_q[j] - shift) * inv_tau);
    log_norm = logf(warp_sum(s));
  }
  float total = 0.f;
  for (int j = lane; j < top; j += 32) {
    const float log_q = (list.log_q[j] - shift) * inv_tau - log_norm;
    const float q = list.index[j] >= 0 ? expf(log_q) : 0.f;
    list.log_q[j] = log_q;
    list.q[j] = q;
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
#pragma unroll 8
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

// ------------------------------------------------------------ rows in registers
// A row is held in registers by the threads of one block, or of a cluster of
// up to 8, so that the loss and its gradient read it once.  It is cut into
// granules of 16 bytes on 16-byte boundaries, whatever the row's own
// alignment; a thread has kVectors of them, and the elements of the first and
// last granule outside the row count as -inf.  A further warp loads the list
// meanwhile and makes the loss.
constexpr int kBlockThreads = 256;  // that hold granules, at most
constexpr int kMaxCluster = 8;

enum Mode { kLoss, kLossGrad, kGradFromStats };

struct Cut {
  int parts;       // blocks of a row
  bool same_phase; // the gradient's rows begin as far off a 16-byte boundary as the logits'
};

// exp2((e - base) c) of two elements.
__device__ __forceinline__ float2 exp2_of(float x, float y, float2 minus_base, float2 c) {
  const float2 t = mul2(add2(make_float2(x, y), minus_base), c);
  return make_float2(fast_exp2(t.x), fast_exp2(t.y));
}

template <typename T, int kVectors, Mode kMode>
__global__ void __launch_bounds__(kBlockThreads + 32, 4)
    distill_kernel(const __grid_constant__ muon_train_distill_args a, Cut cut) {
  constexpr int kN = kVec<T>;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ float total_shared;
  __shared__ float2 warp_part[kBlockThreads / 32];
  __shared__ float2 block_part[kMaxCluster];
  const List list(dynamic, static_cast<int>(a.top));
  begin_kernel();
  const int64_t row = blockIdx.x / cut.parts;
  const int part = static_cast<int>(blockIdx.x - row * cut.parts);
  const int threads = blockDim.x - 32;  // that hold granules
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = threads >> 5;
  const bool list_warp = warp == warps;
  const int vocab = static_cast<int>(a.vocab);
  const float c = kLog2e / a.temperature;
  const float2 cc = make_float2(c, c);
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  if constexpr (kMode != kGradFromStats)
    if (cut.parts > 1) muon_sm100::cluster_sync();  // every block has begun

  // this block's granules of the row: [first, last)
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(z) & 15u) / static_cast<int>(sizeof(T));
  const int granules = (vocab + shift + kN - 1) / kN;
  const int each = (granules + cut.parts - 1) / cut.parts;
  const int first = part * each, last = min(granules, first + each);
  const int mine = first + static_cast<int>(threadIdx.x);
  const auto inside = [&](int element) { return element >= 0 && element + kN <= vocab; };
  uint4 raw[kVectors];
  float max, sum;
  if (list_warp) {
    const float total = load_list(a, row, z, list);
    if (lane == 0) total_shared = total;
  } else {
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      const int granule = mine + v * threads, element = granule * kN - shift;
      if (granule < last && inside(element)) {
        raw[v] = *reinterpret_cast<const uint4*>(z + element);
      } else {
        float e[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j)
          e[j] = granule < last && element + j >= 0 && element + j < vocab ? logit(z, element + j) : -INFINITY;
        raw[v] = pack<T>(e);
      }
    }
    if constexpr (kMode != kGradFromStats) {
      float m = -INFINITY;
#pragma unroll
      for (int v = 0; v < kVectors; ++v) m = vector_max(raw[v], m, T());
      m = warp_max(m);
      const float base = m == -INFINITY ? 0.f : m;  // nothing finite: a sum of 0
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        float e[kN];
        unpack<T>(raw[v], e);
#pragma unroll
        for (int j = 0; j < kN; j += 2)
          s = add2(s, exp2_of(e[j], e[j + 1], make_float2(-base, -base), cc));
      }
      const float all = warp_sum(s.x + s.y);
      if (lane == 0) warp_part[warp] = make_float2(m, all);
    }
  }
  __syncthreads();
  if constexpr (kMode == kGradFromStats) {
    max = a.stats[2 * row];
    sum = a.stats[2 * row + 1];
  } else {
    float2 both = warp_join(lane < warps ? warp_part[lane] : make_float2(-INFINITY, 0.f), c);
    if (cut.parts > 1) {
      if (warp == 0 && lane < cut.parts) {
        const uint32_t to = muon_sm100::map_to_cta(muon_sm100::smem_addr(&block_part[part]),
                                                   static_cast<uint32_t>(lane));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(both.x), "f"(both.y) : "memory");
      }
      muon_sm100::cluster_sync();
      both = block_part[0];
      for (int i = 1; i < cut.parts; ++i) both = join(both, block_part[i], c);
    }
    max = both.x;
    sum = both.y;
    if (part == 0 && list_warp) {
      const float loss = row_loss(list, static_cast<int>(a.top), 1.0f / a.temperature, max, sum);
      if (lane == 0) {
        a.loss[row] = loss;
        if (a.stats != nullptr) {
          a.stats[2 * row] = max;
          a.stats[2 * row + 1] = sum;
        }
      }
    }
  }
  if constexpr (kMode != kLoss) {
    const float total = total_shared;
    const float g = (a.row_scale != nullptr ? a.row_scale[row] : 1.f) / a.temperature;
    const bool none = g == 0.f || total == 0.f;  // zero whatever the logits hold
    const float p_scale = none ? 0.f : g * total / sum;
    const float2 scale2 = make_float2(p_scale, p_scale), minus_max = make_float2(-max, -max);
    T* dz = static_cast<T*>(a.grad) + row * a.ld_grad;
    if (!list_warp) {
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        const int granule = mine + v * threads, element = granule * kN - shift;
        if (granule >= last) continue;
        float e[kN];
        if (none) {
#pragma unroll
          for (int j = 0; j < kN; ++j) e[j] = 0.f;
        } else {
          unpack<T>(raw[v], e);
#pragma unroll
          for (int j = 0; j < kN; j += 2) {
            const float2 p = mul2(scale2, exp2_of(e[j], e[j + 1], minus_max, cc));
            e[j] = p.x;
            e[j + 1] = p.y;
          }
        }
        if (cut.same_phase && inside(element)) {
          *reinterpret_cast<uint4*>(dz + element) = pack<T>(e);
        } else {
#pragma unroll
          for (int j = 0; j < kN; ++j)
            if (element + j >= 0 && element + j < vocab) dz[element + j] = from_float<T>(e[j]);
        }
      }
    }
    if (none) return;
    __syncthreads();  // the listed elements are written again, with their q
    for (int j = threadIdx.x; j < static_cast<int>(a.top); j += blockDim.x) {
      const int i = list.index[j];
      const int granule = (i + shift) / kN;
      if (i < 0 || granule < first || granule >= last) continue;
      const float q = q_of_index(list, static_cast<int>(a.top), i);
      dz[i] = from_float<T>(p_scale * fast_exp2((list.z[j] - max) * c) - g * q);
    }
  }
}

// ------------------------------------------------------------ rows through a ring
// Long rows: persistent blocks, two an SM, or clusters of them a row.  A
// producer warp streams the block's slices of row after row into a ring of
// stages with bulk copies; eight consumer warps take the statistics from the
// stages as they land.  For the loss with its gradient the slice is then
// streamed a second time, from L2, where the first copy asked it to stay.  A
// list warp makes the lists one row ahead, adds up the block's and the
// cluster's sums and makes the loss.  So the next stages are on their way while
// one is worked on, and while one block waits for its sums the other one of
// the SM computes.
//
// Where a wait runs out, no barrier is armed while copies to it are in flight,
// and none are in flight when the block ends: a consumer warp that gave a stage
// up releases none any more, so that the producer refills only stages that all
// have seen land, and comes to a stop; at its end it waits for what it issued.
// A list warp that gave up neither expects nor sends any more.
//
// Measured for the loss with its gradient, 4096 x 131072 bf16 (333 us at the
// copy rate): rows in registers of 8-block clusters 783 us (4 blocks an SM
// 616), slices held in the ring between the passes 504 us, streamed twice
// 403 us (394 now).  8192 x 65536: 372 us.  The loss alone: 172 us of 167.
constexpr int kConsumers = 256;
constexpr int kConsumerWarps = kConsumers / 32;
constexpr int kPerStage = 4;  // granules of a thread in a stage
constexpr int kBlocksPerSm = 2;
constexpr int kStageGranules = kPerStage * kConsumers;
constexpr int kStageBytes = kStageGranules * 16;
constexpr int kMaxStages = 6;
constexpr size_t kRingBytes = 111 * 1024;  // of dynamic shared memory
// Measured: bytes/ns of an SM at the copy rate; what a row costs a block besides
// its bytes, and more with every doubling of a cluster; the bytes of rows in
// flight that L2 holds until their second reading; and what rows in registers
// reach (600 x 65536 bf16 loss with gradient: 51 us, ring 44; 150 rows: 14 and
// 26; 600 x 131072: 94, and 145 with a cluster of 4, 83 of 2).
constexpr double kSmBytesPerNs = 43.0, kRowNs = 1500.0, kClusterNs = 3000.0, kHeldBytes = 60e6;
constexpr double kRegisterBytesPerNs = 3200.0;

struct Ring {
  Cut cut;
  int stages;
};

// Arrives at a named barrier without waiting for the others.
__device__ __forceinline__ void named_arrive(uint32_t id, uint32_t count) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(count) : "memory");
}

// Bulk copy into shared memory with an L2 eviction policy.
__device__ __forceinline__ void bulk_load_hint(void* dst, const void* src, uint32_t bytes, uint64_t* bar,
                                               uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, "
      "[%3], %4;" ::"r"(muon_sm100::smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(muon_sm100::smem_addr(bar)), "l"(policy)
      : "memory");
}

// A block's slice of one row.
template <typename T>
struct Slice {
  const T* z;
  int shift, first, last;  // granules [first, last), the row beginning `shift` elements into granule 0
  __device__ Slice(const muon_train_distill_args& a, const Cut& cut, int64_t row, int part) {
    constexpr int kN = kVec<T>;
    z = static_cast<const T*>(a.logits) + row * a.ld;
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(z) & 15u) / static_cast<int>(sizeof(T));
    const int granules = static_cast<int>((a.vocab + shift + kN - 1) / kN);
    const int each = (granules + cut.parts - 1) / cut.parts;
    first = min(granules, part * each);
    last = min(granules, first + each);
  }
};

template <typename T, Mode kMode>
__global__ void __launch_bounds__(kConsumers + 64, kBlocksPerSm)
    distill_ring_kernel(const __grid_constant__ muon_train_distill_args a, Ring ring) {
  using namespace muon_sm100;
  constexpr int kN = kVec<T>;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], heard[2];
  __shared__ float2 warp_part[2][kConsumerWarps];
  __shared__ float2 block_part[2][kMaxCluster];
  __shared__ float2 row_part[2];  // the row's statistics
  __shared__ float4 row_info[2];  // Q, g, and the statistics of an earlier call
  __shared__ volatile int failed;
  const int parts = ring.cut.parts, stages = ring.stages;
  const int part = static_cast<int>(blockIdx.x % parts);
  const int64_t workers = gridDim.x / parts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vocab = static_cast<int>(a.vocab), top = static_cast<int>(a.top);
  const float c = kLog2e / a.temperature;
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumerWarps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&heard[i], 1);
    failed = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (parts > 1) cluster_sync();  // every block has begun, its barriers are there
  begin_kernel();

  int stage = 0;
  uint32_t phase = 0;
  const auto advance = [&] {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  };
  // For the list warp: the row's statistics from the parts of this block's
  // warps, and of the cluster's blocks; `turn` counts the worker's rows.  Each
  // block sends its part to every block, and goes on to the next row only
  // after it has heard all of them: so no block is ever more than one row ahead
  // of another, and two slots are enough.
  bool deaf = false;  // it gave up, at this turn
  uint32_t deaf_turn = 0;
  const auto drain_heard = [&] {
    if (lane == 0) drain_ring(&heard[deaf_turn & 1], 1, 0, (deaf_turn >> 1) & 1, 1);
  };
  const auto statistics = [&](uint32_t turn) {
    const uint32_t slot = turn & 1;
    float2 v = warp_join(lane < kConsumerWarps ? warp_part[slot][lane] : make_float2(-INFINITY, 0.f), c);
    if (parts > 1 && !deaf) {
      if (lane == 0) mbar_arrive_expect_tx(&heard[slot], static_cast<uint32_t>(parts * sizeof(float2)));
      __syncwarp();
      if (lane < parts) {
        const uint32_t peer = static_cast<uint32_t>(lane);
        asm volatile(
            "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(
                map_to_cta(smem_addr(&block_part[slot][part]), peer)),
            "f"(v.x), "f"(v.y), "r"(map_to_cta(smem_addr(&heard[slot]), peer)) : "memory");
      }
      deaf = !__all_sync(kFullMask, ring_wait(&heard[slot], (turn >> 1) & 1, &failed, /*alone=*/true));
      if (deaf) {  // by the time that this takes, what it sent has landed
        deaf_turn = turn;
        drain_heard();
      }
      v = block_part[slot][0];
      for (int i = 1; i < parts; ++i) v = join(v, block_part[slot][i], c);
    }
    return v;
  };

  if (warp == kConsumerWarps) {  // producer
    // with the gradient, what is read again stays in L2, the rest need not
    [[maybe_unused]] uint64_t keep = 0, drop = 0;
    if constexpr (kMode == kLossGrad) {
      asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));
      asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(drop));
    }
    bool stopped = false;
    for (int64_t row = blockIdx.x / parts; row < a.rows && !stopped; row += workers) {
      const Slice<T> slice(a, ring.cut, row, part);
      for (int pass = 0; pass < (kMode == kLossGrad ? 2 : 1) && !stopped; ++pass)
      for (int g0 = slice.first; g0 < slice.last; g0 += kStageGranules) {
        const int g1 = min(slice.last, g0 + kStageGranules);
        // whole granules [lo, hi); at most one more at either end of the row
        const int lo = g0 * kN < slice.shift ? g0 + 1 : g0;
        const int hi = g1 * kN - slice.shift > vocab ? g1 - 1 : g1;
        uint8_t* to = dynamic + stage * kStageBytes;
        stopped = __any_sync(kFullMask, lane == 0 && !ring_wait(&empty[stage], phase ^ 1, &failed));
        if (stopped) break;
        if (lane < 2 * kN) {
          const bool left = lane < kN;
          const int granule = left ? g0 : g1 - 1, j = lane % kN;
          if (left ? lo > g0 : (hi < g1 && g1 - 1 >= lo)) {
            const int element = granule * kN - slice.shift + j;
            reinterpret_cast<T*>(to)[(granule - g0) * kN + j] =
                element >= 0 && element < vocab ? slice.z[element] : from_float<T>(-INFINITY);
          }
        }
        __syncwarp();
        if (lane == 0) {
          const uint32_t bytes = hi > lo ? static_cast<uint32_t>(hi - lo) * 16u : 0u;
          mbar_arrive_expect_tx(&full[stage], bytes);
          const T* from = slice.z + (static_cast<int64_t>(lo) * kN - slice.shift);
          if (bytes > 0) {
            if constexpr (kMode == kLossGrad)
              bulk_load_hint(to + (lo - g0) * 16, from, bytes, &full[stage], pass == 0 ? keep : drop);
            else
              bulk_load(to + (lo - g0) * 16, from, bytes, &full[stage]);
          }
        }
        advance();
      }
    }
    // the stages' last fillings, from the oldest on: the consumers may have given them up
    if (lane == 0) drain_ring(full, stages, stage, phase ^ 1, stages);
  } else if (warp == kConsumerWarps + 1) {  // lists
    uint32_t turn = 0;
    for (int64_t row = blockIdx.x / parts; row < a.rows; row += workers, ++turn) {
      const List list(dynamic + stages * kStageBytes + (turn & 1) * List::bytes(top), top);
      const float total = load_list(a, row, static_cast<const T*>(a.logits) + row * a.ld, list);
      if (lane == 0) {
        float4 info = make_float4(total, 1.f, 0.f, 0.f);
        if (a.row_scale != nullptr) info.y = a.row_scale[row];
        info.y /= a.temperature;
        if constexpr (kMode == kGradFromStats) {
          info.z = a.stats[2 * row];
          info.w = a.stats[2 * row + 1];
        }
        row_info[turn & 1] = info;
      }
      named_barrier(1, kConsumers + 32);
      if constexpr (kMode != kGradFromStats) {
        const float2 v = statistics(turn);
        if constexpr (kMode == kLossGrad) {
          if (lane == 0) row_part[turn & 1] = v;
          __syncwarp();
          named_arrive(3, kConsumers + 32);
        }
        if (part == 0) {
          const float loss = row_loss(list, top, 1.0f / a.temperature, v.x, v.y);
          if (lane == 0) {
            a.loss[row] = loss;
            if (a.stats != nullptr) {
              a.stats[2 * row] = v.x;
              a.stats[2 * row + 1] = v.y;
            }
          }
        }
      }
    }
  } else {  // consumers
    const float2 cc = make_float2(c, c);
    const int tid = static_cast<int>(threadIdx.x);
    uint32_t turn = 0;
    bool lost = false;  // gave a stage up
    for (int64_t row = blockIdx.x / parts; row < a.rows; row += workers, ++turn) {
      const Slice<T> slice(a, ring.cut, row, part);
      uint4 u[kPerStage];
      const auto at = [&](int i) { return tid + i * kConsumers; };
      const auto read = [&](int i) {
        return *reinterpret_cast<const uint4*>(dynamic + stage * kStageBytes + at(i) * 16);
      };
      const auto wait = [&] {
        if (!lost) lost = !ring_wait(&full[stage], phase, &failed);
      };
      const auto release = [&] {
        __syncwarp();
        if (lane == 0 && !lost) mbar_arrive(&empty[stage]);
      };
      if constexpr (kMode != kGradFromStats) {
        float m = -INFINITY;
        float2 s = make_float2(0.f, 0.f);
        for (int g0 = slice.first; g0 < slice.last; g0 += kStageGranules) {
          wait();
          // past the slice's end: -inf
          if (g0 + kStageGranules <= slice.last) {
#pragma unroll
            for (int i = 0; i < kPerStage; ++i) u[i] = read(i);
          } else {
            float none[kN];
#pragma unroll
            for (int j = 0; j < kN; ++j) none[j] = -INFINITY;
#pragma unroll
            for (int i = 0; i < kPerStage; ++i) u[i] = g0 + at(i) < slice.last ? read(i) : pack<T>(none);
          }
          release();
          float largest = m;
#pragma unroll
          for (int i = 0; i < kPerStage; ++i) largest = vector_max(u[i], largest, T());
          const float base = largest == -INFINITY ? 0.f : largest;  // nothing finite yet: a sum of 0
          const float down = fast_exp2((m - base) * c);
          s = mul2(s, make_float2(down, down));
          m = largest;
#pragma unroll
          for (int i = 0; i < kPerStage; ++i) {
            float e[kN];
            unpack<T>(u[i], e);
#pragma unroll
            for (int j = 0; j < kN; j += 2)
              s = add2(s, exp2_of(e[j], e[j + 1], make_float2(-base, -base), cc));
          }
          advance();
        }
        const float2 v = warp_join(make_float2(m, s.x + s.y), c);
        if (lane == 0) warp_part[turn & 1][warp] = v;
        __syncwarp();
      }
      if constexpr (kMode == kLossGrad) {  // the list warp answers
        named_arrive(1, kConsumers + 32);
        named_barrier(3, kConsumers + 32);
      } else {
        named_barrier(1, kConsumers + 32);
      }
      if constexpr (kMode != kLoss) {
        const float4 info = row_info[turn & 1];
        const float2 v = kMode == kLossGrad ? row_part[turn & 1] : make_float2(info.z, info.w);
        const float g = info.y;
        const bool none = g == 0.f || info.x == 0.f;  // zero whatever the logits hold
        const float p_scale = none ? 0.f : g * info.x / v.y;
        const float2 scale2 = make_float2(p_scale, p_scale), minus_max = make_float2(-v.x, -v.x);
        T* dz = static_cast<T*>(a.grad) + row * a.ld_grad;
        for (int g0 = slice.first; g0 < slice.last; g0 += kStageGranules) {
          wait();
          const int element0 = g0 * kN - slice.shift;
          if (ring.cut.same_phase && !none && g0 + kStageGranules <= slice.last && element0 >= 0 &&
              element0 + kStageGranules * kN <= vocab) {  // whole vectors throughout
#pragma unroll
            for (int i = 0; i < kPerStage; ++i) u[i] = read(i);
            release();
            T* to = dz + element0 + tid * kN;
#pragma unroll
            for (int i = 0; i < kPerStage; ++i) {
              float e[kN];
              unpack<T>(u[i], e);
#pragma unroll
              for (int j = 0; j < kN; j += 2) {
                const float2 p = mul2(scale2, exp2_of(e[j], e[j + 1], minus_max, cc));
                e[j] = p.x;
                e[j + 1] = p.y;
              }
              uint4* at_vector = reinterpret_cast<uint4*>(to + i * kConsumers * kN);
              if constexpr (kMode == kLossGrad)
                __stcs(at_vector, pack<T>(e));
              else
                *at_vector = pack<T>(e);
            }
          } else {
            for (int i = 0; i < kPerStage; ++i) {
              if (g0 + at(i) >= slice.last) break;
              const int element = element0 + at(i) * kN;
              float e[kN];
              unpack<T>(read(i), e);
#pragma unroll
              for (int j = 0; j < kN; ++j)
                e[j] = none ? 0.f : p_scale * fast_exp2((e[j] - v.x) * c);
              if (ring.cut.same_phase && element >= 0 && element + kN <= vocab) {
                *reinterpret_cast<uint4*>(dz + element) = pack<T>(e);
              } else {
#pragma unroll
                for (int j = 0; j < kN; ++j)
                  if (element + j >= 0 && element + j < vocab) dz[element + j] = from_float<T>(e[j]);
              }
            }
            release();
          }
          advance();
        }
        named_barrier(2, kConsumers);  // the listed elements are written again, with their q
        const List list(dynamic + stages * kStageBytes + (turn & 1) * List::bytes(top), top);
        for (int j = threadIdx.x; j < top && !none; j += kConsumers) {
          const int i = list.index[j], granule = (i + slice.shift) / kN;
          if (i < 0 || granule < slice.first || granule >= slice.last) continue;
          const float q = q_of_index(list, top, i);
          dz[i] = from_float<T>(p_scale * fast_exp2((list.z[j] - v.x) * c) - g * q);
        }
      }
    }
  }
  __syncwarp();
  if (parts > 1) {
    cluster_sync();  // no block leaves while another may still write to it
    if (deaf) drain_heard();
  }
}

// ------------------------------------------------------------ host side
bool same_phase(const muon_train_distill_args& a, size_t item) {
  return a.grad != nullptr &&
         ((reinterpret_cast<uintptr_t>(a.grad) ^ reinterpret_cast<uintptr_t>(a.logits)) & 15u) == 0 &&
         (a.rows == 1 || ((a.ld_grad - a.ld) * static_cast<int64_t>(item)) % 16 == 0);
}

template <typename T, int kVectors>
int run_vectors(const muon_train_distill_args& a, Mode mode, int threads, int parts, void* stream) {
  const Cut cut{parts, same_phase(a, sizeof(T))};
  const dim3 grid(static_cast<unsigned>(a.rows * parts));
  const size_t smem = List::bytes(a.top);
  threads += 32;
  if (mode == kGradFromStats)
    return launch(distill_kernel<T, kVectors, kGradFromStats>, grid, threads, smem, 1, true, stream, a, cut);
  if (mode == kLossGrad)
    return launch(distill_kernel<T, kVectors, kLossGrad>, grid, threads, smem, parts, true, stream, a, cut);
  return launch(distill_kernel<T, kVectors, kLoss>, grid, threads, smem, parts, true, stream, a, cut);
}

template <typename T, Mode kMode>
int run_ring(const muon_train_distill_args& a, int parts, int stages, int64_t workers, void* stream) {
  const size_t smem = static_cast<size_t>(stages) * kStageBytes + 2 * List::bytes(a.top);
  const int rc = allow_smem<distill_ring_kernel<T, kMode>>(kRingBytes);
  if (rc != MUON_POLAR_OK) return rc;
  const Ring ring{Cut{parts, same_phase(a, sizeof(T))}, stages};
  return launch(distill_ring_kernel<T, kMode>, dim3(static_cast<unsigned>(workers * parts)),
                kConsumers + 64, smem, kMode == kGradFromStats ? 1 : parts, true, stream, a, ring);
}

template <typename T>
int run(const muon_train_distill_args& a, Mode mode, void* stream) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != MUON_POLAR_OK) return rc;
  // granules of a row: one more where a row can begin off a boundary
  const bool aligned = aligned16(a.logits) && (a.rows == 1 || a.ld % kVec<T> == 0);
  const int64_t granules = (a.vocab + kVec<T> - 1) / kVec<T> + (aligned ? 0 : 1);
  const int64_t register_row = static_cast<int64_t>(kBlockThreads) * 8;  // of one block

  // The ring's parts of a row by the smallest estimate: rounds of rows, each
  // of a slice at a block's share of the measured copy rate and what a row
  // costs besides.
  const int64_t blocks = static_cast<int64_t>(sms) * kBlocksPerSm;
  const double row_bytes = static_cast<double>(granules) * 16.0, passes = mode == kLoss ? 1.0 : 2.0;
  int parts = 1;
  double ring_ns = 0.0;
  for (int p = 1, steps = 0; p <= kMaxCluster && p <= blocks; p *= 2, ++steps) {
    const int64_t workers = std::min<int64_t>(a.rows, blocks / p);
    const double rounds = static_cast<double>((a.rows + workers - 1) / workers);
    const bool again = mode == kLossGrad && static_cast<double>(workers) * row_bytes > kHeldBytes;
    const double slice_ns = row_bytes / p * kBlocksPerSm / kSmBytesPerNs * (again ? 2.7 : passes);
    const double cluster_ns = mode == kGradFromStats ? 0.0 : mode == kLoss ? kClusterNs / 2 : kClusterNs;
    const double estimate = rounds * (slice_ns + kRowNs + steps * cluster_ns);
    if (p == 1 || estimate < ring_ns) {
      parts = p;
      ring_ns = estimate;
    }
  }
  // Rows of one block's registers never pay for a ring; longer ones do where
  // there are rows enough.
  const double register_ns = row_bytes * static_cast<double>(a.rows) * passes / kRegisterBytesPerNs;
  if (granules <= register_row || (granules <= kMaxCluster * register_row && register_ns <= ring_ns)) {
    // Parts of a row: as many as keep a thread at 8 vectors; more, down to one
    // vector a thread, while the device is not full.
    parts = 1;
    while (parts < kMaxCluster &&
           (granules > parts * register_row || (a.rows * parts < 2 * sms && granules > parts * kBlockThreads)))
      parts *= 2;
    const int64_t each = (granules + parts - 1) / parts;
    // Threads: 8 vectors each when there are blocks enough, else one each.
    const int64_t want = a.rows * parts >= 4 * sms ? (each + 7) / 8 : each;
    const int threads = static_cast<int>(want >= kBlockThreads ? kBlockThreads : want <= 64 ? 64 : (want + 31) / 32 * 32);
    const int64_t vectors = (each + threads - 1) / threads;
    if (vectors <= 1) return run_vectors<T, 1>(a, mode, threads, parts, stream);
    if (vectors <= 2) return run_vectors<T, 2>(a, mode, threads, parts, stream);
    if (vectors <= 4) return run_vectors<T, 4>(a, mode, threads, parts, stream);
    return run_vectors<T, 8>(a, mode, threads, parts, stream);
  }
  const int stages = static_cast<int>(
      std::min<size_t>(kMaxStages, (kRingBytes - 2 * List::bytes(a.top)) / kStageBytes));
  const int64_t workers = std::min<int64_t>(a.rows, blocks / parts);
  if (mode == kLossGrad) return run_ring<T, kLossGrad>(a, parts, stages, workers, stream);
  if (mode == kLoss) return run_ring<T, kLoss>(a, parts, stages, workers, stream);
  return run_ring<T, kGradFromStats>(a, parts, stages, workers, stream);
}

int check(const muon_train_distill_args* a) {
  if (a == nullptr || a->rows < 0 || a->vocab < 1 || a->top < 1 || a->top > MUON_TRAIN_MAX_TOP ||
      a->rows > 0x7fffffff / 8 || a->vocab > 0x7fffff00 || !(a->temperature >= FLT_MIN) ||
      (a->rows > 1 && a->ld < a->vocab) || !valid_dtype(a->dtype) ||
      !valid_dtype(a->teacher_dtype) || (a->index_bytes != 4 && a->index_bytes != 8))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->rows > 0 && (a->logits == nullptr || a->teacher_logits == nullptr ||
                      a->teacher_indices == nullptr || a->grad == a->logits ||
                      (a->grad != nullptr && a->rows > 1 && a->ld_grad < a->vocab)))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}

int dispatch(const muon_train_distill_args& a, Mode mode, void* stream) {
  if (a.rows == 0) return MUON_POLAR_OK;
  switch (a.dtype) {
    case MUON_TRAIN_F32: return run<float>(a, mode, stream);
    case MUON_TRAIN_BF16: return run<__nv_bfloat16>(a, mode, stream);
    default: return run<__half>(a, mode, stream);
  }
}

}  // namespace
}  // namespace muon_train

extern "C" {

uint64_t muon_train_launch_count(void) {
  return muon_train::launch_counter().load(std::memory_order_relaxed);
}

int muon_train_read_device_status(int device, uint32_t* flags, int clear) {
  if (flags == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  int prev = 0;
  cudaError_t e = cudaGetDevice(&prev);
  if (e == cudaSuccess && device != prev) e = cudaSetDevice(device);
  if (e != cudaSuccess) return static_cast<int>(e);
  uint32_t v = 0;
  e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = muon_train::take_status(&v, clear);
  if (e == cudaSuccess) e = muon_train::norm_status(&v, clear);
  if (e == cudaSuccess) e = muon_train::attention_status(&v, clear);
  if (device != prev) cudaSetDevice(prev);
  if (e != cudaSuccess) return static_cast<int>(e);
  *flags = v;
  return MUON_POLAR_OK;
}

int muon_train_wait_limit_ns(uint64_t* limit_ns) {
  if (limit_ns == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  uint64_t limit[3] = {};
  cudaError_t e = muon_train::get_wait_limit(&limit[0]);
  if (e == cudaSuccess) e = muon_train::norm_get_wait_limit(&limit[1]);
  if (e == cudaSuccess) e = muon_train::attention_get_wait_limit(&limit[2]);
  if (e != cudaSuccess) return static_cast<int>(e);
  *limit_ns = std::max({limit[0], limit[1], limit[2]});
  return MUON_POLAR_OK;
}

int muon_train_distill_sm100(const muon_train_distill_args* args, void* stream) {
  using namespace muon_train;
  const int rc = check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->rows > 0 && (args->loss == nullptr || (args->grad != nullptr && args->stats == nullptr)))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return dispatch(*args, args->grad != nullptr ? kLossGrad : kLoss, stream);
}

int muon_train_distill_backward_sm100(const muon_train_distill_args* args, void* stream) {
  using namespace muon_train;
  const int rc = check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->rows > 0 && (args->stats == nullptr || args->grad == nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return dispatch(*args, kGradFromStats, stream);
}

}  // extern "C"
