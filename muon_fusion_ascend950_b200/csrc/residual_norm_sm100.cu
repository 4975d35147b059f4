// residual_norm_sm100.cu -- the norms before and after a residual block, with
// its gate and residual scale, in one pass, and their gradients.
//
//   r = rsqrt(mean y^2 + eps), u = y r w, h = s x + g u,
//   R = rsqrt(mean h^2 + eps), n = h R p
//
// With the normed rows v = y r and m = h R, a = dn p, A = sum a m,
// B1 = sum g w v (dh + R a), B2 = sum g w v m and k = R A / width:
//   dH = dh + R a - k m         dx = s dH        ds = sum dH x
//   dy = r (g w dH - v (B1 - k B2) / width)
//   C  = sum dH v               dg = w C         dw = g C
//   dp = sum dn m
// so that a row needs one reduction of three sums, and h is made again from
// x and y instead of being kept.  No power of r or R is formed: their cubes
// leave fp32's range from rows of rms 5e12 on, and below 1e-13 when eps allows.
//
// Bound by memory: forward reads x, y and writes h, n; backward reads x, y,
// dh, dn and writes dx, dy.  Parameter gradients: each block adds up its rows
// in order, a second kernel adds up the blocks in order.
#include <initializer_list>

#include "sm100_ptx.cuh"
#include "train_common.cuh"

namespace muon_train {
namespace {

// ------------------------------------------------------------ parameters
// One column's parameters; the gate's row is chosen by the caller.
struct Params {
  const muon_train_norm_args& a;
  __device__ float post(int64_t c) const {
    return a.post_weight != nullptr ? load_any(a.post_weight, a.post_dtype, c) : 1.f;
  }
  __device__ float pre(int64_t c) const {
    return a.pre_weight != nullptr ? load_any(a.pre_weight, a.pre_dtype, c) : 0.f;
  }
  __device__ float gate(int64_t gate_row, int64_t c) const {
    return a.gate != nullptr ? load_any(a.gate, a.gate_dtype, gate_row * a.width + c) : 1.f;
  }
  __device__ float scale(int64_t c) const {
    return a.residual_scale != nullptr
               ? load_any(a.residual_scale, a.scale_dtype, a.scale_count == 1 ? 0 : c)
               : 1.f;
  }
};

// Sums of N values over a block of `threads` threads, in a fixed order; every
// thread gets them.  `red` holds N x 32 floats and may be used again after
// the next barrier.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float* red, int threads) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = threads / 32;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? red[i * 32 + lane] : 0.f);
}

__device__ __forceinline__ float rms_rstd(float sum, float width, float eps) {
  return rsqrtf(sum / width + eps);
}

// ------------------------------------------------------------ rows in registers
// A row of up to 16384 elements is held in registers: each thread has kE = 8
// or 16 of its columns, the same ones in every row, as kE / N loads of N
// elements.  A row belongs to one warp (up to 256 columns, no barrier), to a
// block of up to 512 threads, or to a cluster of such blocks, which add up
// their sums over distributed shared memory.  Rows of whole 16-byte vectors
// have 8 columns a thread up to 4096, 16 above, and a cluster of 2 above
// 8192: 16384 x 8192 bf16 backward took 436 us so when it was chosen (402 now),
// 568 with 8 columns in a cluster, whose barrier holds up every row.  Other
// rows have 8 columns a thread and clusters of 2 and 4: 16 would not fit the
// registers (4098 columns: 716 us when it was chosen, with 16 a thread 1219;
// 567 now).
constexpr int kMaxThreads = 512;
constexpr int kWarpRowWarps = 8;   // rows in flight of a block, one a warp
constexpr int kMaxCluster = 4;

enum RowOwner { kWarpRow, kBlockRow, kClusterRow };

// Shared memory of the sums of one row's parts, twice: a buffer is written
// again only after a barrier that follows its last reading.
struct SumSlots {
  float warp[2][4][16];
  float block[2][kMaxCluster][4];
};

// Four sums over a warp with 6 shuffles: each step halves the values that a
// lane carries on.  Lane l ends with the sum of value (l >> 3) & 3 .. in the
// order 0, 1, 2, 3 of its upper two bits.
__device__ __forceinline__ float warp_sum4(const float (&v)[4]) {
  const int lane = threadIdx.x & 31;
  const bool high = lane & 16, odd = lane & 8;
  const float a0 = high ? v[2] : v[0], a1 = high ? v[3] : v[1];
  const float b0 = high ? v[0] : v[2], b1 = high ? v[1] : v[3];
  const float c0 = a0 + __shfl_xor_sync(kFullMask, b0, 16);
  const float c1 = a1 + __shfl_xor_sync(kFullMask, b1, 16);
  float d = (odd ? c1 : c0) + __shfl_xor_sync(kFullMask, odd ? c0 : c1, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) d += __shfl_xor_sync(kFullMask, d, o);
  return d;
}

// Sums of four values over a row's threads, in a fixed order; every thread
// gets them.  `turn` begins at 0 and alternates from call to call.
template <RowOwner kOwner>
__device__ __forceinline__ void row_sums(float (&v)[4], SumSlots& slots, int& turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float d = warp_sum4(v);
  if constexpr (kOwner != kWarpRow) {
    if ((lane & 7) == 0) slots.warp[turn][lane >> 3][warp] = d;
    __syncthreads();
    const float* from = slots.warp[turn][lane >> 3];
    d = ((lane & 7) < warps ? from[lane & 7] : 0.f) + ((lane & 7) + 8 < warps ? from[(lane & 7) + 8] : 0.f);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) d += __shfl_xor_sync(kFullMask, d, o);
  }
  if constexpr (kOwner == kClusterRow) {
    const int rank = static_cast<int>(muon_sm100::cluster_cta_rank());
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    // each block puts its sums into every block's slots, by rank
    if (warp < static_cast<int>(n) && (lane & 7) == 0) {
      const uint32_t to = muon_sm100::map_to_cta(
          muon_sm100::smem_addr(&slots.block[turn][rank][lane >> 3]), static_cast<uint32_t>(warp));
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(d) : "memory");
    }
    muon_sm100::cluster_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float sum = 0.f;
      for (uint32_t k = 0; k < n; ++k) sum += slots.block[turn][k][i];
      v[i] = sum;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __shfl_sync(kFullMask, d, i * 8);
  }
  turn ^= 1;
}

// Which rows and columns a thread has.
template <int N, RowOwner kOwner>
struct Place {
  int64_t worker, workers;  // rows go to workers: a warp, a block or a cluster
  int tid, threads;         // of the row's threads
  __device__ Place() {
    if constexpr (kOwner == kWarpRow) {
      tid = threadIdx.x & 31;
      threads = 32;
      worker = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
      workers = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
    } else if constexpr (kOwner == kBlockRow) {
      tid = threadIdx.x;
      threads = blockDim.x;
      worker = blockIdx.x;
      workers = gridDim.x;
    } else {
      uint32_t n;
      asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
      tid = static_cast<int>(muon_sm100::cluster_cta_rank() * blockDim.x + threadIdx.x);
      threads = static_cast<int>(n * blockDim.x);
      worker = blockIdx.x / n;
      workers = gridDim.x / n;
    }
  }
  __device__ int column(int i) const { return (i * threads + tid) * N; }
};

// A thread's columns of one row, in pairs for the packed fp32 instructions.
template <int kE>
struct Columns {
  float2 v[kE / 2];
  __device__ __forceinline__ float& at(int i) { return (i & 1) ? v[i / 2].y : v[i / 2].x; }
  __device__ __forceinline__ float at(int i) const { return (i & 1) ? v[i / 2].y : v[i / 2].x; }
};

// One parameter's values in a thread's columns, on their way: N elements are
// loaded as two halves of the bytes that N fp32 have; of 16-bit types the
// first half is all of them.  No branch on the type stands between the loads,
// so that those of several parameters wait for memory together.
template <int N, int kE>
struct ParamColumns {
  using Raw = typename RawOf<2 * N>::type;
  Raw low[kE / N], high[kE / N];
  const void* p;
  int dtype;
  template <typename P>
  __device__ __forceinline__ void load(const P& place, int width, const void* param, int type, int64_t offset) {
    p = param;
    dtype = type;
    const int size = type == MUON_TRAIN_F32 ? 4 : 2;
    const uint8_t* from = static_cast<const uint8_t*>(param) + offset * size;
#pragma unroll
    for (int i = 0; i < kE / N; ++i) {
      const int c = place.column(i);
      low[i] = high[i] = Raw();
      if (param != nullptr && c < width) {
        const uint8_t* at = from + static_cast<int64_t>(c) * size;
        low[i] = *reinterpret_cast<const Raw*>(at);
        high[i] = *reinterpret_cast<const Raw*>(at + (size - 2) * N);
      }
    }
  }
  // `none` outside the row, and everywhere when there is no such parameter
  template <typename P>
  __device__ __forceinline__ void values(Columns<kE>& v, const P& place, int width, float none) const {
#pragma unroll
    for (int i = 0; i < kE / N; ++i) {
      const uint16_t* l = reinterpret_cast<const uint16_t*>(&low[i]);
      const uint16_t* h = reinterpret_cast<const uint16_t*>(&high[i]);
      const bool there = p != nullptr && place.column(i) < width;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        // 16-bit words 2 j and 2 j + 1 of the N fp32, word j of the N others
        const uint32_t w0 = 2 * j < N ? l[2 * j] : h[2 * j - N];
        const uint32_t w1 = 2 * j + 1 < N ? l[2 * j + 1] : h[2 * j + 1 - N];
        const float f32 = __uint_as_float(w1 << 16 | w0), bf16 = __uint_as_float(static_cast<uint32_t>(l[j]) << 16);
        const float f16 = __half2float(__ushort_as_half(l[j]));
        const float value = dtype == MUON_TRAIN_F32 ? f32 : dtype == MUON_TRAIN_BF16 ? bf16 : f16;
        v.at(i * N + j) = there ? value : none;
      }
    }
  }
};
template <int N, int kE, typename P>
__device__ __forceinline__ void load_columns(Columns<kE>& v, const P& place, int width, const void* p, int dtype,
                                             int64_t offset, float none) {
  ParamColumns<N, kE> raw;
  raw.load(place, width, p, dtype, offset);
  raw.values(v, place, width, none);
}
// A gate row times the post weight.
template <int N, int kE, typename P>
__device__ __forceinline__ void load_gain(Columns<kE>& v, const P& place, int width, const muon_train_norm_args& a,
                                          int64_t gate_row) {
  ParamColumns<N, kE> gate, post;
  gate.load(place, width, a.gate, a.gate_dtype, gate_row * width);
  post.load(place, width, a.post_weight, a.post_dtype, 0);
  Columns<kE> w;
  gate.values(v, place, width, 1.f);
  post.values(w, place, width, 1.f);
#pragma unroll
  for (int i = 0; i < kE / 2; ++i) v.v[i] = mul2(v.v[i], w.v[i]);
}

template <typename T, int N, int kE>
struct RowVectors {
  using E = Elements<T, N>;
  typename E::Raw raw[kE / N];
  template <typename P>
  __device__ __forceinline__ void load(const T* row, const P& place, int width) {
#pragma unroll
    for (int i = 0; i < kE / N; ++i)
      raw[i] = place.column(i) < width ? E::load(row + place.column(i)) : typename E::Raw();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kE / N; ++i) raw[i] = typename E::Raw();
  }
  __device__ __forceinline__ void values(Columns<kE>& v) const {
#pragma unroll
    for (int i = 0; i < kE / N; ++i) {
      float part[N];
      E::unpack(raw[i], part);
#pragma unroll
      for (int j = 0; j < N; ++j) v.at(i * N + j) = part[j];
    }
  }
  template <typename P>
  static __device__ __forceinline__ void store(T* row, const P& place, int width, const Columns<kE>& v) {
#pragma unroll
    for (int i = 0; i < kE / N; ++i) {
      float part[N];
#pragma unroll
      for (int j = 0; j < N; ++j) part[j] = v.at(i * N + j);
      if (place.column(i) < width) E::store(row + place.column(i), E::pack(part));
    }
  }
};

__device__ __forceinline__ float pair_sum(float2 v) { return v.x + v.y; }

// Rows of a block (or of its part of a cluster's rows) on their way through
// shared memory: bulk copies of kArrays tensors' rows into `stages` stages,
// issued by the warps' first lanes.  A stage is free again once every thread has it in
// registers, which the barrier of the row's sums tells.
//
// If a thread's wait ran out, nothing more is issued from the next barrier on:
// all issuing lanes find it in failed_in[turn], which like the sums of `turn`
// is written before the barrier and again only after the next but one, and set
// the other turn's too.  So a stage is armed only when every thread has seen
// its copies land, and the rows in flight are the next ones of the ring.
constexpr int kMaxStages = 16;
constexpr size_t kRingMost = 222 * 1024;  // bytes of an SM's rings
struct RingState {
  uint64_t full[kMaxStages];
  volatile int failed, failed_in[2];
  // Kept by thread 0: where in the ring the rows in flight begin, and what
  // tells how many they are (forward: rows left; backward: row and chunk).
  volatile int stopped, stage, phase;
  volatile int64_t row, chunk;
};
template <typename T, int N, int kE, int kArrays>
struct Ring {
  RingState* state;
  T* data;
  int stages, stage;
  uint32_t phase;

  // By every thread; each barrier expects `copies` arrivals.
  __device__ void init(uint32_t copies) const {
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) muon_sm100::mbar_init(&state->full[i], copies);
      state->failed = state->failed_in[0] = state->failed_in[1] = state->stopped = 0;
      muon_sm100::fence_mbar_init();
    }
    __syncthreads();
  }
  // For an issuing lane after the barrier that follows the waits of `turn`, for
  // rows from `back` stages ago on: whether it issues no more.
  __device__ __forceinline__ bool stopped(int turn, int back, int64_t row, int64_t chunk) const {
    if (!state->failed_in[turn]) return false;
    state->failed_in[turn ^ 1] = 1;
    if (threadIdx.x == 0 && !state->stopped) {
      state->stopped = 1;
      state->stage = stage < back ? stage - back + stages : stage - back;
      state->phase = stage < back ? phase ^ 1 : phase;
      state->row = row;
      state->chunk = chunk;
    }
    return true;
  }
  // By thread 0 if it stopped, with the rows that were left: waits for those in flight.
  __device__ void drain(int64_t left) const {
    drain_ring(state->full, stages, state->stage, state->phase, static_cast<int>(left < stages ? left : stages));
  }
  __device__ T* at(int stage_, int array, int run) const {
    return data + ((stage_ * kArrays + array) * kE / N + run) * static_cast<int>(blockDim.x) * N;
  }
  // By one thread: this block's columns of a row of one tensor.  The stage's
  // barrier expects one such call for each tensor.
  template <typename P>
  __device__ void issue(int stage_, int array, const T* from, int64_t row, int width, const P& place) const {
    const int span = static_cast<int>(blockDim.x) * N;
    const int first = place.tid - static_cast<int>(threadIdx.x);  // the block's first thread of the row
    uint32_t bytes = 0;
#pragma unroll
    for (int i = 0; i < kE / N; ++i)
      bytes += static_cast<uint32_t>(max(0, min(span, width - (i * place.threads + first) * N))) * sizeof(T);
    muon_sm100::mbar_arrive_expect_tx(&state->full[stage_], bytes);
#pragma unroll
    for (int i = 0; i < kE / N; ++i) {
      const int c = (i * place.threads + first) * N;
      const int n = min(span, width - c);
      if (n > 0)
        muon_sm100::bulk_load(at(stage_, array, i), from + row * width + c, static_cast<uint32_t>(n) * sizeof(T),
                              &state->full[stage_]);
    }
  }
  __device__ void wait(int turn) const {
    if (!ring_wait(&state->full[stage], phase, &state->failed)) state->failed_in[turn] = 1;
  }
  template <typename P>
  __device__ void read(RowVectors<T, N, kE>& v, int array, int width, const P& place) const {
#pragma unroll
    for (int i = 0; i < kE / N; ++i)
      v.raw[i] = place.column(i) < width
                     ? Elements<T, N>::load(at(stage, array, i) + static_cast<int>(threadIdx.x) * N)
                     : typename Elements<T, N>::Raw();
  }
  __device__ void advance() {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// Which row of the gate a row uses.
__device__ __forceinline__ int64_t gate_row_of(const muon_train_norm_args& a, int64_t row) {
  return a.gate_rows > 1 ? row / (a.rows / a.gate_rows) : 0;
}

// Forward.  Four rows (of 8 columns a thread) at a time: their sums share the
// shuffles and barriers, whose latency else held up every row.  16384 x 4096
// bf16: 93 us, 83 at the copy rate (one row at a time, two blocks an SM: 116;
// with all copies issued by one thread, on whose warp the next sums wait: 103).
template <typename T, int N, int kE, RowOwner kOwner>
__global__ void __launch_bounds__(kOwner == kWarpRow ? kWarpRowWarps * 32 : kMaxThreads,
                                  kOwner == kWarpRow ? 2 : 1)
    norm_forward_kernel(const __grid_constant__ muon_train_norm_args a, int stages) {
  constexpr int kRowsAtOnce = 32 / kE, kPairs = kE / 2;
  constexpr bool kRing = N * sizeof(T) == 16 && kOwner != kWarpRow;
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ SumSlots slots;
  __shared__ RingState ring_state;
  int turn = 0;
  if constexpr (kOwner == kClusterRow) muon_sm100::cluster_sync();  // every block has begun
  begin_kernel();
  const Place<N, kOwner> place;
  // Neighbouring rows, which mostly share a gate row (100 x 150 rows of 4096
  // with a gate row for each 150: 184 us dealt out in turn, 103 so), and which a
  // block with 8 columns a thread streams better (2050 columns: 122 and 107);
  // other rows are dealt out in turn (200 columns: 8.9 us as neighbours, 7.6 so;
  // 8192 without such a gate: 179 and 170).
  const bool neighbours = (kOwner == kBlockRow && kE == 8) || a.gate_rows > 1;
  const int64_t stride = neighbours ? 1 : place.workers;
  const int64_t begin = neighbours ? place.worker * a.rows / place.workers : place.worker;
  const int64_t end = neighbours ? (place.worker + 1) * a.rows / place.workers : a.rows;
  const int width = static_cast<int>(a.width);
  const float inv_width = 1.0f / static_cast<float>(width);
  const T* y_all = static_cast<const T*>(a.block_out);
  const T* x_all = static_cast<const T*>(a.residual);
  Ring<T, N, kE, 2> ring{&ring_state, reinterpret_cast<T*>(dynamic), stages, 0, 0};
  // `rows` rows from `row` on into the stages from `stage` on; a warp's first
  // lane issues every so many of the 2 rows copies, since the next sums wait
  // for the slowest warp
  const auto issue = [&](int stage, int64_t row, int rows) {
    if ((threadIdx.x & 31) != 0) return;
    for (int i = threadIdx.x >> 5; i < 2 * rows; i += blockDim.x >> 5) {
      const int64_t r = row + (i >> 1) * stride;
      const int to = stage + (i >> 1);
      if (r < end) ring.issue(to < stages ? to : to - stages, i & 1, (i & 1) == 0 ? y_all : x_all, r, width, place);
    }
  };
  if constexpr (kRing) {
    ring.init(2);
    issue(0, begin, stages);
  }
  Columns<kE> gain, scale, pre;
  int64_t gate_row = begin < end ? gate_row_of(a, begin) : 0;
  {
    ParamColumns<N, kE> gate_raw, post_raw, pre_raw, scale_raw;
    gate_raw.load(place, width, a.gate, a.gate_dtype, gate_row * width);
    post_raw.load(place, width, a.post_weight, a.post_dtype, 0);
    pre_raw.load(place, width, a.pre_weight, a.pre_dtype, 0);
    scale_raw.load(place, width, a.scale_count > 1 ? a.residual_scale : nullptr, a.scale_dtype, 0);
    const float one = a.scale_count == 1 ? load_any(a.residual_scale, a.scale_dtype, 0) : 1.f;
    gate_raw.values(gain, place, width, 1.f);
    post_raw.values(scale, place, width, 1.f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) gain.v[i] = mul2(gain.v[i], scale.v[i]);
    pre_raw.values(pre, place, width, 0.f);
    scale_raw.values(scale, place, width, one);
  }
  for (int64_t first = begin; first < end; first += kRowsAtOnce * stride) {
    const int64_t left = (end - first + stride - 1) / stride;  // rows of this worker
    const int rows = left < kRowsAtOnce ? static_cast<int>(left) : kRowsAtOnce;
    // After a barrier that follows the rows' reading: their stages take later ones.
    const auto refill = [&] {
      if constexpr (kRing) {
        if ((threadIdx.x & 31) != 0 || ring.stopped(turn ^ 1, rows, left, 0)) return;
        const int stage = ring.stage - rows;
        issue(stage < 0 ? stage + stages : stage, first + stages * stride, rows);
      }
    };
    Columns<kE> y[kRowsAtOnce], h[kRowsAtOnce];
    {
      RowVectors<T, N, kE> ry[kRowsAtOnce], rx[kRowsAtOnce];
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        ry[j].clear();
        rx[j].clear();
        if (j < rows) {
          if constexpr (kRing) {
            ring.wait(turn);
            ring.read(ry[j], 0, width, place);
            ring.read(rx[j], 1, width, place);
            ring.advance();
          } else {
            const int64_t row = first + j * stride;
            ry[j].load(y_all + row * width, place, width);
            rx[j].load(x_all + row * width, place, width);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        ry[j].values(y[j]);
        rx[j].values(h[j]);
      }
    }
    float r[4] = {1.f, 1.f, 1.f, 1.f};
    if (a.post_weight != nullptr) {
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        float2 s = both(0.f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) s = fma2(y[j].v[i], y[j].v[i], s);
        r[j] = pair_sum(s);
      }
      row_sums<kOwner>(r, slots, turn);
      refill();
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j) {
        r[j] = rsqrtf(r[j] * inv_width + a.eps);
        if (place.tid == 0 && j < rows && a.rstd_post != nullptr) a.rstd_post[first + j * stride] = r[j];
      }
    }
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kRowsAtOnce; ++j) {
      const int64_t row = first + j * stride;
      if (j < rows) {
        if (const int64_t g = gate_row_of(a, row); g != gate_row) {
          gate_row = g;
          load_gain<N>(gain, place, width, a, gate_row);
        }
      }
      float2 s = both(0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        h[j].v[i] = fma2(scale.v[i], h[j].v[i], mul2(gain.v[i], mul2(y[j].v[i], both(r[j]))));
        s = fma2(h[j].v[i], h[j].v[i], s);
      }
      sums[j] = pair_sum(s);
      if (j < rows) RowVectors<T, N, kE>::store(static_cast<T*>(a.hidden) + row * width, place, width, h[j]);
    }
    if (a.pre_weight == nullptr) {
      if (a.post_weight == nullptr) {
        if constexpr (kRing) {
          __syncthreads();
          turn ^= 1;
        }
        refill();
      }
      continue;
    }
    row_sums<kOwner>(sums, slots, turn);
    if (a.post_weight == nullptr) refill();
#pragma unroll
    for (int j = 0; j < kRowsAtOnce; ++j) {
      if (j >= rows) break;
      const int64_t row = first + j * stride;
      const float rh = rsqrtf(sums[j] * inv_width + a.eps);
      if (place.tid == 0 && a.rstd_pre != nullptr) a.rstd_pre[row] = rh;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) h[j].v[i] = mul2(mul2(h[j].v[i], both(rh)), pre.v[i]);
      RowVectors<T, N, kE>::store(static_cast<T*>(a.normed) + row * width, place, width, h[j]);
    }
  }
  // the statistics of a norm that there is not
  if (a.post_weight == nullptr && a.rstd_post != nullptr)
    for (int64_t row = begin + place.tid * stride; row < end; row += place.threads * stride) a.rstd_post[row] = 1.f;
  if (a.pre_weight == nullptr && a.rstd_pre != nullptr)
    for (int64_t row = begin + place.tid * stride; row < end; row += place.threads * stride) a.rstd_pre[row] = 0.f;
  if constexpr (kRing)
    if (threadIdx.x == 0 && ring_state.stopped) ring.drain(ring_state.row);
  if constexpr (kOwner == kClusterRow) muon_sm100::cluster_sync();  // peers' stores have landed
}

// ------------------------------------------------------------ any width
constexpr int kThreads = 256;

// One block a row; the row is read again from L1 / L2 for each step.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_row_kernel(const __grid_constant__ muon_train_norm_args a) {
  __shared__ float red[2 * 32];
  begin_kernel();
  const Params p{a};
  const int64_t row = blockIdx.x, base = row * a.width;
  const int64_t gate_row = a.gate_rows > 0 ? row / (a.rows / a.gate_rows) : 0;
  const T* y = static_cast<const T*>(a.block_out) + base;
  const T* x = static_cast<const T*>(a.residual) + base;
  const float width = static_cast<float>(a.width);
  float r = 1.f;
  if (a.post_weight != nullptr) {
    float sum[1] = {0.f};
    for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
      const float v = to_float(y[c]);
      sum[0] = fmaf(v, v, sum[0]);
    }
    block_sums(sum, red, kThreads);
    r = rms_rstd(sum[0], width, a.eps);
  }
  if (threadIdx.x == 0 && a.rstd_post != nullptr) a.rstd_post[row] = r;
  float sum[1] = {0.f};
  T* hidden = static_cast<T*>(a.hidden) + base;
  for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
    const float h = fmaf(p.scale(c), to_float(x[c]), p.gate(gate_row, c) * (to_float(y[c]) * r * p.post(c)));
    hidden[c] = from_float<T>(h);
    sum[0] = fmaf(h, h, sum[0]);
  }
  if (a.pre_weight == nullptr) {
    if (threadIdx.x == 0 && a.rstd_pre != nullptr) a.rstd_pre[row] = 0.f;
    return;
  }
  block_sums(sum, red + 32, kThreads);
  const float rh = rms_rstd(sum[0], width, a.eps);
  if (threadIdx.x == 0 && a.rstd_pre != nullptr) a.rstd_pre[row] = rh;
  T* normed = static_cast<T*>(a.normed) + base;
  for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
    const float h = fmaf(p.scale(c), to_float(x[c]), p.gate(gate_row, c) * (to_float(y[c]) * r * p.post(c)));
    normed[c] = from_float<T>(h * rh * p.pre(c));
  }
}

// ------------------------------------------------------------ backward plan
// Rows are cut into chunks that do not cross a gate row's rows (unless every
// row has its own gate row); a block takes chunks blockIdx.x, + gridDim.x, ..
// Partial sums in the workspace, fp32:
//   gain  [chunks][width]  C (times the gate when every row has its own)
//   pre   [blocks][width]  dp
//   scale [blocks][width]  ds, or one fp64 of each block for one value
struct Plan {
  int64_t groups, chunks_per_group, chunks, blocks;
  int gate_per_row;
  size_t gain_off, pre_off, scale_off, bytes;
};

Plan make_plan(const muon_train_norm_args& a, int64_t target) {
  Plan p;
  p.gate_per_row = a.gate != nullptr && a.gate_rows == a.rows && a.rows > 1;
  p.groups = (a.gate != nullptr && !p.gate_per_row) ? a.gate_rows : 1;
  const int64_t per_group = a.rows / p.groups;
  // Workers take chunks in rounds: of the counts that fill k rounds the one
  // with the least time in rows, where a chunk costs kChunkRows besides its own
  // (one chunk more than workers, in place of a few less, doubled the time: 5
  // sequences of 3288 x 2050 with a gate row each: 150 chunks 347 us, 145 183).
  constexpr int64_t kChunkRows = 2;
  int64_t least_rows = INT64_MAX;
  for (int64_t k = 1; k <= 8; ++k) {
    int64_t n = k * target / p.groups;
    n = n < 1 ? 1 : n > per_group ? per_group : n;
    const int64_t rounds = (p.groups * n + target - 1) / target;
    const int64_t rows = rounds * ((per_group + n - 1) / n + kChunkRows);
    if (rows < least_rows) {
      least_rows = rows;
      p.chunks_per_group = n;
    }
  }
  p.chunks = p.groups * p.chunks_per_group;
  p.blocks = p.chunks < target ? p.chunks : target;
  const auto align = [](size_t v) { return (v + 255) / 256 * 256; };
  p.gain_off = 0;
  p.pre_off = align(static_cast<size_t>(p.chunks * a.width) * sizeof(float));
  p.scale_off = p.pre_off + align(static_cast<size_t>(p.blocks * a.width) * sizeof(float));
  // (one value: an fp64 of every block of a worker's cluster)
  const int64_t least = 2 * kMaxCluster;
  p.bytes = p.scale_off + align(static_cast<size_t>(p.blocks * (a.width < least ? least : a.width)) * sizeof(float));
  return p;
}

// The block's sum of one value a thread, in a fixed order: of a scalar
// parameter's gradient, which adds up every element of every row, with both
// signs, and is held in 64 bits therefore.
__device__ __forceinline__ void store_block_sum(double v, double* to) {
  __shared__ double part[32];
  v = warp_sum64(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double sum = 0.0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) sum += part[w];
  *to = sum;
}

struct Backward {
  muon_train_norm_args a;
  muon_train_norm_grads g;
  Plan plan;
  int64_t scale_rows;         // partial rows of `scale`
  float *gain, *pre, *scale;  // partial sums; NULL: not wanted
};

__device__ __forceinline__ void chunk_rows(const Backward& b, int64_t chunk, int64_t* r0,
                                           int64_t* r1, int64_t* group) {
  const int64_t per_group = b.a.rows / b.plan.groups, n = b.plan.chunks_per_group;
  *group = chunk / n;
  const int64_t i = chunk - *group * n;
  *r0 = *group * per_group + i * per_group / n;
  *r1 = *group * per_group + (i + 1) * per_group / n;
}

// Sums over a block's warps of each warp's columns (kWarpRow), written to a
// partial row.
__device__ __forceinline__ void store_warp_columns(float* to, int width, const Columns<8>& v, int n,
                                                   float (*columns)[256]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) columns[warp][((i / n) * 32 + lane) * n + i % n] = v.at(i);
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    float sum = 0.f;
    for (int w = 0; w < kWarpRowWarps; ++w) sum += columns[w][c];
    to[c] = sum;
  }
}

// Columns that a thread keeps for the whole kernel: in registers, or in shared
// memory, where only the thread itself reads and writes them.
template <int kE, bool kShared>
struct Held {
  Columns<kE> c;
  __device__ Held(float4*, int) {}
  __device__ void set(const Columns<kE>& v) { c = v; }
  __device__ void pairs(int q, float2 (&p)[2]) const {  // columns 4 q .. 4 q + 3
    p[0] = c.v[2 * q];
    p[1] = c.v[2 * q + 1];
  }
  __device__ void set_pairs(int q, const float2 (&p)[2]) {
    c.v[2 * q] = p[0];
    c.v[2 * q + 1] = p[1];
  }
};
template <int kE>
struct Held<kE, true> {
  float4* at;
  int stride;
  __device__ Held(float4* area, int index)
      : at(area + index * (kE / 4) * blockDim.x + threadIdx.x), stride(static_cast<int>(blockDim.x)) {}
  __device__ void set(const Columns<kE>& v) {
#pragma unroll
    for (int q = 0; q < kE / 4; ++q)
      at[q * stride] = make_float4(v.v[2 * q].x, v.v[2 * q].y, v.v[2 * q + 1].x, v.v[2 * q + 1].y);
  }
  __device__ void pairs(int q, float2 (&p)[2]) const {
    const float4 v = at[q * stride];
    p[0] = make_float2(v.x, v.y);
    p[1] = make_float2(v.z, v.w);
  }
  __device__ void set_pairs(int q, const float2 (&p)[2]) {
    at[q * stride] = make_float4(p[0].x, p[0].y, p[1].x, p[1].y);
  }
};
// Which of a thread's held columns are in shared memory, and how many there are.
// With 16 columns: gain, pre weight and the sums of a residual scale with
// columns (the scale itself would take the ring's second stage, and is loaded
// for every row).  With 8 columns registers would do, but the fewer they hold
// the less a row waits: that scale and its sums (16384 x 4096 bf16 174 us when
// that was chosen, 179 now; the sums in registers 228, and the scale loaded for
// every row 272); of rows through the ring the pre weight (174 us then, 178 in
// registers), of fp32 the gain too (291 us then, 334; bf16 181).  Single
// elements have no registers for the addresses (2049 columns: 377 us, the scale
// loaded for every row 326, and 317 now).
template <typename T, int N, int kE, bool kRing, bool kScaleColumns>
struct Holds {
  static constexpr bool kScale = kScaleColumns && kE == 8 && N > 1;
  static constexpr bool kScaleSums = kScaleColumns && (kE == 16 || kScale);
  static constexpr bool kPre = kE == 16 || kRing;
  static constexpr bool kGain = kE == 16 || (kRing && sizeof(T) == 4);
  static constexpr int kFloats = (kScale + kScaleSums + kPre + kGain) * kE;
};

// Backward.  16384 x 4096 bf16: 167 us, 125 at the copy rate; 59% of the issue
// slots are used, the rest goes into each row's sums and barrier (two rows at
// a time, read from their stages again, took 202 against 183 then: more
// instructions than the waits were worth).
// A worker (block or cluster) takes whole chunks; with one warp a
// row, the block's warps take every 8th row of the chunk and are added up
// where the chunk ends.  kScaleColumns: residual_scale has a value for each
// column (else one value, or none).
template <typename T, int N, int kE, RowOwner kOwner, bool kScaleColumns>
__global__ void __launch_bounds__(kOwner == kWarpRow ? kWarpRowWarps * 32 : kMaxThreads, 1)
    norm_backward_kernel(const __grid_constant__ Backward b, int stages) {
  extern __shared__ __align__(128) uint8_t dynamic[];
  __shared__ SumSlots slots;
  __shared__ float columns[kOwner == kWarpRow ? kWarpRowWarps : 1][256];
  __shared__ RingState ring_state;
  // whole vectors come through a ring; else the next row is loaded while this
  // one is worked on where registers allow
  constexpr int kPairs = kE / 2;
  constexpr bool kRing = N * sizeof(T) == 16 && kOwner != kWarpRow;
  constexpr bool kAhead = !kRing && sizeof(T) == 2 && N > 1;
  constexpr bool kAgain = kRing && sizeof(T) == 2;
  using Hold = Holds<T, N, kE, kRing, kScaleColumns>;
  const muon_train_norm_args& a = b.a;
  const Place<N, kOwner> place;
  const int width = static_cast<int>(a.width);
  const float inv_width = 1.0f / static_cast<float>(width);
  int turn = 0;
  if constexpr (kOwner == kClusterRow) muon_sm100::cluster_sync();  // every block has begun
  begin_kernel();
  const int64_t worker = kOwner == kWarpRow ? blockIdx.x : place.worker;
  const int64_t workers = kOwner == kWarpRow ? gridDim.x : place.workers;
  const int step = kOwner == kWarpRow ? kWarpRowWarps : 1;
  const int first = kOwner == kWarpRow ? threadIdx.x >> 5 : 0;

  const T* y_all = static_cast<const T*>(a.block_out);
  const T* x_all = static_cast<const T*>(a.residual);
  const T* dh_all = static_cast<const T*>(b.g.grad_hidden);
  const T* dn_all = static_cast<const T*>(b.g.grad_normed);
  const bool has_pre = a.pre_weight != nullptr && dn_all != nullptr;
  RowVectors<T, N, kE> ry, rx, rdh, rdn;
  const auto load_row = [&](int64_t row) {
    ry.load(y_all + row * width, place, width);
    rx.load(x_all + row * width, place, width);
    if (dh_all != nullptr) rdh.load(dh_all + row * width, place, width);
    if (dn_all != nullptr) rdn.load(dn_all + row * width, place, width);
  };
  rdh.clear();
  rdn.clear();
  float4* const held = reinterpret_cast<float4*>(dynamic);
  Ring<T, N, kE, 4> ring{&ring_state, reinterpret_cast<T*>(dynamic + Hold::kFloats * sizeof(float) * blockDim.x),
                         stages, 0, 0};
  // Each warp's first lane: the row that goes into the ring next.  It issues
  // every so many of the row's copies, since the next sums wait for the slowest
  // warp.
  int64_t ahead_chunk = worker, ahead_row = 0, ahead_end = 0;
  const auto issue_next = [&](int stage) {
    while (ahead_row >= ahead_end) {
      if (ahead_chunk >= b.plan.chunks) return;
      int64_t group;
      chunk_rows(b, ahead_chunk, &ahead_row, &ahead_end, &group);
      ahead_chunk += workers;
    }
    for (int t = threadIdx.x >> 5; t < 4; t += blockDim.x >> 5) {
      const T* from = t == 0 ? y_all : t == 1 ? x_all : t == 2 ? dh_all : dn_all;
      if (from != nullptr) ring.issue(stage, t, from, ahead_row, width, place);
    }
    ++ahead_row;
  };
  if constexpr (kRing) {
    ring.init(2 + (dh_all != nullptr) + (dn_all != nullptr));
    if ((threadIdx.x & 31) == 0 && threadIdx.x < 4 * 32)
      for (int i = 0; i < stages; ++i) issue_next(i);
  }

  Held<kE, Hold::kGain> gain(held, 0);  // gate times post weight
  Held<kE, Hold::kPre> pre(held, Hold::kGain);
  Held<kE, Hold::kScaleSums> sum_scale(held, Hold::kGain + Hold::kPre);
  Held<kE, Hold::kScale> scale_held(held, Hold::kGain + Hold::kPre + Hold::kScaleSums);
  Columns<kE> scale_columns{};
  float2 scale_one = both(1.f);
  double sum_scale_one = 0.0;  // over all of a thread's elements: in 64 bits, an addition a row
  {
    Columns<kE> v;
    load_columns<N>(v, place, width, a.post_weight, a.post_dtype, 0, 1.f);
    gain.set(v);
    load_columns<N>(v, place, width, a.pre_weight, a.pre_dtype, 0, 0.f);
    pre.set(v);
    if constexpr (kScaleColumns) sum_scale.set(Columns<kE>{});
    if constexpr (Hold::kScale) {
      load_columns<N>(v, place, width, a.residual_scale, a.scale_dtype, 0, 1.f);
      scale_held.set(v);
    }
  }
  if (!kScaleColumns && a.residual_scale != nullptr)
    scale_one = both(load_any(a.residual_scale, a.scale_dtype, 0));
  const auto load_scale = [&] {
    if constexpr (kScaleColumns && !Hold::kScale)
      load_columns<N>(scale_columns, place, width, a.residual_scale, a.scale_dtype, 0, 1.f);
  };
  const auto scale_pairs = [&](int q, float2 (&p)[2]) {
    if constexpr (Hold::kScale) {
      scale_held.pairs(q, p);
    } else {
      p[0] = kScaleColumns ? scale_columns.v[2 * q] : scale_one;
      p[1] = kScaleColumns ? scale_columns.v[2 * q + 1] : scale_one;
    }
  };
  const auto hold_gain = [&](int64_t gate_row) {
    Columns<kE> v;
    load_gain<N>(v, place, width, a, gate_row);
    gain.set(v);
  };

  Columns<kE> sum_gain, sum_pre;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) sum_gain.v[i] = sum_pre.v[i] = both(0.f);

  const auto store_columns = [&](float* to, const Columns<kE>& v) {
    if constexpr (kOwner == kWarpRow) {
      store_warp_columns(to, width, v, N, columns);
    } else {
#pragma unroll
      for (int i = 0; i < kE / N; ++i) {
        if (place.column(i) >= width) continue;
#pragma unroll
        for (int j = 0; j < N; ++j) to[place.column(i) + j] = v.at(i * N + j);
      }
    }
  };

  for (int64_t chunk = worker; chunk < b.plan.chunks; chunk += workers) {
    int64_t r0, r1, group;
    chunk_rows(b, chunk, &r0, &r1, &group);
    if (a.gate != nullptr && !b.plan.gate_per_row) hold_gain(group);
    if (kAhead && r0 + first < r1) load_row(r0 + first);
    // the statistics of the next row are loaded a row ahead too
    float next_r = 1.f, next_rh = 0.f;
    const auto load_rstd = [&](int64_t row) {
      if (row >= r1) return;
      if (a.post_weight != nullptr) next_r = a.rstd_post[row];
      if (has_pre) next_rh = a.rstd_pre[row];
    };
    load_rstd(r0 + first);
    for (int64_t row = r0 + first; row < r1; row += step) {
      if constexpr (kRing) {
        ring.wait(turn);
        ring.read(ry, 0, width, place);
        ring.read(rx, 1, width, place);
        if (dh_all != nullptr) ring.read(rdh, 2, width, place);
        if (dn_all != nullptr) ring.read(rdn, 3, width, place);
      } else if constexpr (!kAhead) {
        load_row(row);
      }
      if (b.plan.gate_per_row) hold_gain(row);
      const float r = next_r, rh = next_rh;
      load_rstd(row + step);
      Columns<kE> m, u;  // m: hidden, normed; u: dh + rh dn pre
      rdh.values(u);
      float2 s0 = both(0.f), s1 = both(0.f), s2 = both(0.f);
      Columns<kE> y, x, dn;
      ry.values(y);
      rx.values(x);
      rdn.values(dn);
      if constexpr (kAhead) {
        if (row + step < r1) load_row(row + step);
      }
      load_scale();
#pragma unroll
      for (int q = 0; q < kE / 4; ++q) {
        float2 g[2], p[2], s[2];
        gain.pairs(q, g);
        pre.pairs(q, p);
        scale_pairs(q, s);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = 2 * q + j;
          const float2 gv = mul2(g[j], mul2(y.v[i], both(r))), an = mul2(dn.v[i], p[j]);
          m.v[i] = mul2(fma2(s[j], x.v[i], gv), both(rh));
          u.v[i] = fma2(both(rh), an, u.v[i]);
          s0 = fma2(an, m.v[i], s0);
          s1 = fma2(gv, u.v[i], s1);
          s2 = fma2(gv, m.v[i], s2);
        }
      }
      float sums[4] = {pair_sum(s0), pair_sum(s1), pair_sum(s2), 0.f};
      row_sums<kOwner>(sums, slots, turn);
      if constexpr (kRing) {  // every thread has the row in registers
        if ((threadIdx.x & 31) == 0 && threadIdx.x < 4 * 32 && !ring.stopped(turn ^ 1, 0, row, chunk))
          issue_next(ring.stage);
        ring.advance();
      }
      const float k = rh * (sums[0] * inv_width);
      const float ky = a.post_weight != nullptr ? r * ((sums[1] - k * sums[2]) * inv_width) : 0.f;
      if constexpr (kAgain) {  // out of the packed registers: fewer are held over the barrier
        ry.values(y);
        rx.values(x);
        rdn.values(dn);
        load_scale();
      }
      Columns<kE> gained;
      float2 row_scale = both(0.f);
#pragma unroll
      for (int q = 0; q < kE / 4; ++q) {
        float2 g[2], s[2], sc[2];
        gain.pairs(q, g);
        scale_pairs(q, s);
        if constexpr (kScaleColumns) sum_scale.pairs(q, sc);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = 2 * q + j;
          const float2 d = fma2(both(-k), m.v[i], u.v[i]), v = mul2(y.v[i], both(r));
          gained.v[i] = mul2(d, v);
          sum_pre.v[i] = fma2(dn.v[i], m.v[i], sum_pre.v[i]);
          if constexpr (kScaleColumns)
            sc[j] = fma2(d, x.v[i], sc[j]);
          else
            row_scale = fma2(d, x.v[i], row_scale);
          x.v[i] = mul2(d, s[j]);
          y.v[i] = fma2(both(-ky), v, mul2(mul2(g[j], both(r)), d));
        }
        if constexpr (kScaleColumns) sum_scale.set_pairs(q, sc);
      }
      if constexpr (!kScaleColumns) sum_scale_one += pair_sum(row_scale);
      if (b.g.grad_residual != nullptr)
        RowVectors<T, N, kE>::store(static_cast<T*>(b.g.grad_residual) + row * width, place, width, x);
      if (b.g.grad_block_out != nullptr)
        RowVectors<T, N, kE>::store(static_cast<T*>(b.g.grad_block_out) + row * width, place, width, y);
      if (!b.plan.gate_per_row) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) sum_gain.v[i] = add2(sum_gain.v[i], gained.v[i]);
        continue;
      }
      // a gate row of its own: its gradient leaves with the row
      Columns<kE> gate, post;
      load_columns<N>(gate, place, width, a.gate, a.gate_dtype, row * width, 1.f);
      load_columns<N>(post, place, width, a.post_weight, a.post_dtype, 0, 1.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        sum_gain.v[i] = fma2(gained.v[i], gate.v[i], sum_gain.v[i]);
        gained.v[i] = mul2(gained.v[i], post.v[i]);
      }
      if (b.g.grad_gate == nullptr) continue;
#pragma unroll
      for (int i = 0; i < kE / N; ++i) {
        if (place.column(i) >= width) continue;
        float part[N];
#pragma unroll
        for (int j = 0; j < N; ++j) part[j] = gained.at(i * N + j);
        store_any<N>(b.g.grad_gate, a.gate_dtype, row * width + place.column(i), part);
      }
    }
    if (b.gain != nullptr) {
      store_columns(b.gain + chunk * width, sum_gain);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) sum_gain.v[i] = both(0.f);
    }
  }
  if (b.pre != nullptr) store_columns(b.pre + worker * width, sum_pre);
  if (b.scale != nullptr) {
    if constexpr (kScaleColumns) {
      Columns<kE> v;
#pragma unroll
      for (int q = 0; q < kE / 4; ++q) {
        float2 sc[2];
        sum_scale.pairs(q, sc);
        v.v[2 * q] = sc[0];
        v.v[2 * q + 1] = sc[1];
      }
      store_columns(b.scale + worker * width, v);
    } else {  // one value of each block
      store_block_sum(sum_scale_one, reinterpret_cast<double*>(b.scale) + blockIdx.x);
    }
  }
  if constexpr (kRing) {
    if (threadIdx.x == 0 && ring_state.stopped) {
      int64_t left = 0, from, to, group;
      for (int64_t chunk = ring_state.chunk; chunk < b.plan.chunks && left < stages; chunk += workers) {
        chunk_rows(b, chunk, &from, &to, &group);
        left += to - (chunk == ring_state.chunk ? ring_state.row : from);
      }
      ring.drain(left);
    }
  }
  if constexpr (kOwner == kClusterRow) muon_sm100::cluster_sync();  // peers' stores have landed
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_backward_row_kernel(const __grid_constant__ Backward b) {
  __shared__ float red[3 * 32];
  begin_kernel();
  const muon_train_norm_args& a = b.a;
  const Params p{a};
  const float width = static_cast<float>(a.width);
  const T* dh_all = static_cast<const T*>(b.g.grad_hidden);
  const T* dn_all = static_cast<const T*>(b.g.grad_normed);
  float* pre = b.pre != nullptr ? b.pre + blockIdx.x * a.width : nullptr;
  float* scale = b.scale != nullptr
                     ? b.scale + (a.scale_count == 1 ? 0 : blockIdx.x * a.width)
                     : nullptr;
  bool first_row = true;
  double scale_sum = 0.0;
  for (int64_t chunk = blockIdx.x; chunk < b.plan.chunks; chunk += gridDim.x) {
    int64_t r0, r1, group;
    chunk_rows(b, chunk, &r0, &r1, &group);
    float* gain = b.gain != nullptr ? b.gain + chunk * a.width : nullptr;
    for (int64_t row = r0; row < r1; ++row) {
      const int64_t base = row * a.width;
      const int64_t gate_row = b.plan.gate_per_row ? row : group;
      const T* y = static_cast<const T*>(a.block_out) + base;
      const T* x = static_cast<const T*>(a.residual) + base;
      const float r = a.post_weight != nullptr ? a.rstd_post[row] : 1.f;
      const float rh = a.pre_weight != nullptr && dn_all != nullptr ? a.rstd_pre[row] : 0.f;
      float sums[3] = {0.f, 0.f, 0.f};
      for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
        const float gv = p.gate(gate_row, c) * p.post(c) * (to_float(y[c]) * r);
        const float m = fmaf(p.scale(c), to_float(x[c]), gv) * rh;
        const float dh = dh_all != nullptr ? to_float(dh_all[base + c]) : 0.f;
        const float an = dn_all != nullptr ? to_float(dn_all[base + c]) * p.pre(c) : 0.f;
        sums[0] = fmaf(an, m, sums[0]);
        sums[1] = fmaf(gv, fmaf(rh, an, dh), sums[1]);
        sums[2] = fmaf(gv, m, sums[2]);
      }
      __syncthreads();  // the last row's sums have been read
      block_sums(sums, red, kThreads);
      const float k = rh * (sums[0] / width);
      const float ky = a.post_weight != nullptr ? r * ((sums[1] - k * sums[2]) / width) : 0.f;
      for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
        const float v = to_float(y[c]) * r, xv = to_float(x[c]);
        const float gate = p.gate(gate_row, c), post = p.post(c), sc = p.scale(c);
        const float m = fmaf(sc, xv, gate * post * v) * rh;
        const float dh = dh_all != nullptr ? to_float(dh_all[base + c]) : 0.f;
        const float dn = dn_all != nullptr ? to_float(dn_all[base + c]) : 0.f;
        const float d = fmaf(-k, m, fmaf(rh, dn * p.pre(c), dh));
        if (b.g.grad_residual != nullptr)
          static_cast<T*>(b.g.grad_residual)[base + c] = from_float<T>(d * sc);
        if (b.g.grad_block_out != nullptr)
          static_cast<T*>(b.g.grad_block_out)[base + c] = from_float<T>(fmaf(-ky, v, r * (gate * post) * d));
        const float gained = d * v;
        if (b.plan.gate_per_row && b.g.grad_gate != nullptr)
          store_any(b.g.grad_gate, a.gate_dtype, base + c, gained * post);
        if (gain != nullptr)
          gain[c] = (row == r0 ? 0.f : gain[c]) + (b.plan.gate_per_row ? gained * gate : gained);
        if (pre != nullptr) pre[c] = (first_row ? 0.f : pre[c]) + dn * m;
        if (scale != nullptr) {
          if (a.scale_count == 1)
            scale_sum += d * xv;
          else
            scale[c] = (first_row ? 0.f : scale[c]) + d * xv;
        }
      }
      first_row = false;
    }
  }
  if (scale != nullptr && a.scale_count == 1) {
    store_block_sum(scale_sum, reinterpret_cast<double*>(b.scale) + blockIdx.x);
  }
}

// Adds up partial sums: blockIdx.y = 0 pre weight, 1 residual scale, 2 post
// weight, from 3 on gate rows (blockIdx.y - 3, + gridDim.y - 3, ..).  A warp
// reads 32 columns of a partial row; the block's 16 warps take every 16th row
// and are added in order.
constexpr int kSumWarps = 16;
constexpr int kGateRowBlocks = 4096;

// Sum of partial rows first, first + step, .. below last in one column, eight
// loads on their way at a time.
__device__ __forceinline__ float rows_sum(const float* from, int64_t width, int64_t column, int64_t first,
                                          int64_t last, int step) {
  float sum = 0.f;
  int64_t i = first;
  for (; i + 7 * step < last; i += 8 * step) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = from[(i + j * step) * width + column];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j];
  }
  for (; i < last; i += step) sum += from[i * width + column];
  return sum;
}

// The block's 16 warps' sums of its 32 columns, added up in order in warp 0.
__device__ float warps_sum(float sum, float (*part)[32]) {
  __syncthreads();  // part has been read
  part[threadIdx.x >> 5][threadIdx.x & 31] = sum;
  __syncthreads();
  sum = 0.f;
  if (threadIdx.x < 32)
    for (int w = 0; w < kSumWarps; ++w) sum += part[w][threadIdx.x];
  return sum;
}

__global__ void __launch_bounds__(kSumWarps * 32)
    norm_sums_kernel(const __grid_constant__ Backward b) {
  __shared__ float part[kSumWarps][32];
  begin_kernel();
  const muon_train_norm_args& a = b.a;
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const bool inside = column < a.width, writes = threadIdx.x < 32 && inside;
  const int what = blockIdx.y, warp = threadIdx.x >> 5;
  const Params p{a};
  if (what == 0) {
    if (b.pre == nullptr) return;
    const float v = warps_sum(inside ? rows_sum(b.pre, a.width, column, warp, b.plan.blocks, kSumWarps) : 0.f, part);
    if (writes) store_any(b.g.grad_pre_weight, a.pre_dtype, column, v);
  } else if (what == 1) {
    if (b.scale == nullptr || static_cast<int64_t>(blockIdx.x) * 32 >= a.scale_count) return;
    if (a.scale_count == 1) {  // by the first warp
      if (warp != 0) return;
      const double* from = reinterpret_cast<const double*>(b.scale);
      double sum = 0.0;
      for (int64_t i = threadIdx.x; i < b.scale_rows; i += 32) sum += from[i];
      sum = warp_sum64(sum);
      if (threadIdx.x == 0) store_any(b.g.grad_residual_scale, a.scale_dtype, 0, static_cast<float>(sum));
      return;
    }
    const float v = warps_sum(column < a.scale_count ? rows_sum(b.scale, a.scale_count, column, warp, b.scale_rows, kSumWarps)
                                                     : 0.f, part);
    if (writes && column < a.scale_count)
      store_any(b.g.grad_residual_scale, a.scale_dtype, column, v);
  } else if (what == 2) {
    if (b.g.grad_post_weight == nullptr) return;
    float sum = 0.f;
    const int64_t n = b.plan.chunks_per_group;
    if (!inside) {
    } else if (a.gate == nullptr || b.plan.gate_per_row) {
      sum = rows_sum(b.gain, a.width, column, warp, b.plan.chunks, kSumWarps);
    } else if (n >= kSumWarps) {  // the warps share each gate row's chunks
      for (int64_t g = 0; g < b.plan.groups; ++g)
        sum = fmaf(rows_sum(b.gain, a.width, column, g * n + warp, (g + 1) * n, kSumWarps), p.gate(g, column), sum);
    } else {  // each has gate rows of its own
#pragma unroll 4
      for (int64_t g = warp; g < b.plan.groups; g += kSumWarps)
        sum = fmaf(rows_sum(b.gain, a.width, column, g * n, (g + 1) * n, 1), p.gate(g, column), sum);
    }
    const float v = warps_sum(sum, part);
    if (writes) store_any(b.g.grad_post_weight, a.post_dtype, column, v);
  } else {
    for (int64_t g = what - 3; g < b.plan.groups; g += gridDim.y - 3) {
      const int64_t first = g * b.plan.chunks_per_group;
      const float v = warps_sum(
          inside ? rows_sum(b.gain, a.width, column, first + warp, first + b.plan.chunks_per_group, kSumWarps) : 0.f, part);
      if (writes) store_any(b.g.grad_gate, a.gate_dtype, g * a.width + column, v * p.post(column));
    }
  }
}

// ------------------------------------------------------------ host side
int check(const muon_train_norm_args* a) {
  if (a == nullptr || a->rows < 0 || a->width < 1 || a->rows > 0x7fffffff ||
      a->width > (1 << 24) || !(a->eps >= 0.f) || !valid_dtype(a->dtype))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if ((a->post_weight != nullptr && !valid_dtype(a->post_dtype)) ||
      (a->pre_weight != nullptr && !valid_dtype(a->pre_dtype)))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->gate != nullptr &&
      (!valid_dtype(a->gate_dtype) || a->gate_rows < 1 || a->rows % a->gate_rows != 0))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->residual_scale != nullptr &&
      (!valid_dtype(a->scale_dtype) || (a->scale_count != 1 && a->scale_count != a->width)))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a->rows > 0 && (a->block_out == nullptr || a->residual == nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}

// The gate of no rows, and gate_rows without a gate, are normalised to none.
muon_train_norm_args normalised(const muon_train_norm_args& args) {
  muon_train_norm_args a = args;
  if (a.gate == nullptr) a.gate_rows = 0;
  if (a.residual_scale == nullptr) a.scale_count = 0;
  return a;
}

// How a call's rows are laid out: the vectors they are read in, who has a row.
struct Layout {
  int elements;  // N: 16 bytes, two 16-bit elements, or one; 0: any width (one block a row)
  RowOwner owner;
  int columns;   // of a thread: 8 or 16
  int threads, cluster;
  int per_sm;    // blocks that an SM holds: 512 threads of up to 128 registers
};

bool all_aligned16(std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (!aligned16(p)) return false;
  return true;
}

// Vectors of 16 bytes need rows, and so a width, of whole vectors, and every
// pointer on a 16-byte boundary; pairs an even width.
Layout make_layout(const muon_train_norm_args& a, const muon_train_norm_grads* g) {
  Layout l{};
  const int vec = static_cast<int>(16 / dtype_size(a.dtype));
  bool aligned = all_aligned16({a.block_out, a.residual, a.hidden, a.normed, a.post_weight, a.pre_weight,
                                a.gate, a.residual_scale});
  if (g != nullptr)
    aligned = aligned && all_aligned16({g->grad_hidden, g->grad_normed, g->grad_block_out,
                                        g->grad_residual, g->grad_gate});
  l.elements = !aligned ? 1 : a.width % vec == 0 ? vec : (vec == 8 && a.width % 2 == 0) ? 2 : 1;
  l.cluster = 1;
  l.columns = 8;
  // With 16 columns a thread, backward's three held arrays and one stage of
  // four rows have to fit the shared memory: 512 threads of 16-bit types, 480
  // of fp32.
  const int most_columns = l.elements == vec ? 16 : 8;
  const bool wide = a.width > kMaxThreads * 8;
  const int most_threads =
      wide && most_columns == 16 && a.dtype == MUON_TRAIN_F32 && g != nullptr ? 480 : kMaxThreads;
  const int most_cluster = l.elements == vec ? 2 : kMaxCluster;
  if (a.width <= 32 * 8) {
    l.owner = kWarpRow;
    l.threads = kWarpRowWarps * 32;
  } else if (a.width <= most_cluster * most_threads * most_columns) {
    if (wide) l.columns = most_columns;
    while (a.width > l.cluster * most_threads * l.columns) l.cluster *= 2;
    l.owner = l.cluster > 1 ? kClusterRow : kBlockRow;
    const int64_t each = 32 * l.columns * l.cluster;
    l.threads = static_cast<int>((a.width + each - 1) / each * 32);
  } else {
    l.elements = 0;
    l.owner = kBlockRow;
    l.threads = kThreads;
  }
  l.per_sm = l.columns == 16 ? 1 : kMaxThreads / l.threads;  // 16: for their shared memory
  return l;
}

// Blocks (of all clusters) that the device works on at once in backward.
int target_workers(const Layout& l, int64_t* target) {
  int sms = 0;
  const int rc = sm_count(&sms);
  *target = static_cast<int64_t>(sms) * l.per_sm / l.cluster;
  return rc;
}

// Shared memory of a ring of `arrays` tensors' rows, and its stages: what the
// `per_sm` blocks of an SM have between them, besides `held` bytes each.
template <typename T, int N>
size_t ring_bytes(const Layout& l, int arrays, int per_sm, size_t held, int* stages) {
  *stages = 0;
  if (N * sizeof(T) != 16 || l.owner == kWarpRow) return 0;
  const size_t stage = static_cast<size_t>(l.threads) * l.columns * sizeof(T) * arrays;
  const size_t most = ((kRingMost + 2048) / per_sm - 2048 - held) / stage;
  *stages = static_cast<int>(most < kMaxStages ? most : kMaxStages);
  return *stages * stage;
}

template <typename T, int N, int kE, RowOwner kOwner>
int launch_forward(const muon_train_norm_args& a, const Layout& l, int sms, void* stream) {
  if (l.columns != kE || l.owner != kOwner) return MUON_POLAR_ERR_INVALID_ARGUMENT;  // not make_layout's
  const int64_t rows_a_block = kOwner == kWarpRow ? kWarpRowWarps : 1;
  const int64_t most = static_cast<int64_t>(sms) * l.per_sm / l.cluster;
  const int64_t want = (a.rows + rows_a_block - 1) / rows_a_block, workers = want < most ? want : most;
  int stages = 0;
  const size_t smem = ring_bytes<T, N>(l, 2, l.per_sm, 0, &stages);
  if (N * sizeof(T) == 16 && kOwner != kWarpRow && stages < 1)
    return MUON_POLAR_ERR_INVALID_ARGUMENT;  // not with make_layout's sizes
  const int rc = smem == 0 ? MUON_POLAR_OK : allow_smem<norm_forward_kernel<T, N, kE, kOwner>>(kRingMost);
  if (rc != MUON_POLAR_OK) return rc;
  return launch(norm_forward_kernel<T, N, kE, kOwner>, dim3(static_cast<unsigned>(workers * l.cluster)),
                l.threads, smem, l.cluster, true, stream, a, stages);
}

template <typename T, int N>
int forward_rows(const muon_train_norm_args& a, const Layout& l, int sms, void* stream) {
  if (l.owner == kWarpRow) return launch_forward<T, N, 8, kWarpRow>(a, l, sms, stream);
  if constexpr (N * sizeof(T) == 16) {
    if (l.owner == kClusterRow) return launch_forward<T, N, 16, kClusterRow>(a, l, sms, stream);
    if (l.columns == 16) return launch_forward<T, N, 16, kBlockRow>(a, l, sms, stream);
  } else {
    if (l.owner == kClusterRow) return launch_forward<T, N, 8, kClusterRow>(a, l, sms, stream);
  }
  return launch_forward<T, N, 8, kBlockRow>(a, l, sms, stream);
}

template <typename T>
int forward(const muon_train_norm_args& a, void* stream) {
  const Layout l = make_layout(a, nullptr);
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != MUON_POLAR_OK) return rc;
  if (l.elements == 0)
    return launch(norm_row_kernel<T>, dim3(static_cast<unsigned>(a.rows)), kThreads, 0, 1, true, stream, a);
  if (l.elements == kVec<T>) return forward_rows<T, kVec<T>>(a, l, sms, stream);
  if constexpr (sizeof(T) == 2)
    if (l.elements == 2) return forward_rows<T, 2>(a, l, sms, stream);
  return forward_rows<T, 1>(a, l, sms, stream);
}

template <typename T, int N, int kE, RowOwner kOwner, bool kScaleColumns>
int launch_backward(const Backward& b, const Layout& l, void* stream) {
  if (l.columns != kE || l.owner != kOwner) return MUON_POLAR_ERR_INVALID_ARGUMENT;  // not make_layout's
  int stages = 0;
  constexpr bool kRing = N * sizeof(T) == 16 && kOwner != kWarpRow;
  const size_t held =
      static_cast<size_t>(l.threads) * Holds<T, N, kE, kRing, kScaleColumns>::kFloats * sizeof(float);
  const size_t ring = ring_bytes<T, N>(l, 4, l.per_sm, held, &stages), smem = held + ring;
  if (N * sizeof(T) == 16 && kOwner != kWarpRow && stages < 1)
    return MUON_POLAR_ERR_INVALID_ARGUMENT;  // not with make_layout's sizes
  const int rc =
      smem <= 32 * 1024 ? MUON_POLAR_OK : allow_smem<norm_backward_kernel<T, N, kE, kOwner, kScaleColumns>>(kRingMost);
  if (rc != MUON_POLAR_OK) return rc;
  return launch(norm_backward_kernel<T, N, kE, kOwner, kScaleColumns>,
                dim3(static_cast<unsigned>(b.plan.blocks * l.cluster)), l.threads, smem, l.cluster, true, stream,
                b, stages);
}

template <typename T, int N, bool kScaleColumns>
int backward_rows(const Backward& b, const Layout& l, void* stream) {
  if (l.owner == kWarpRow) return launch_backward<T, N, 8, kWarpRow, kScaleColumns>(b, l, stream);
  if constexpr (N * sizeof(T) == 16) {
    if (l.owner == kClusterRow) return launch_backward<T, N, 16, kClusterRow, kScaleColumns>(b, l, stream);
    if (l.columns == 16) return launch_backward<T, N, 16, kBlockRow, kScaleColumns>(b, l, stream);
  } else {
    if (l.owner == kClusterRow) return launch_backward<T, N, 8, kClusterRow, kScaleColumns>(b, l, stream);
  }
  return launch_backward<T, N, 8, kBlockRow, kScaleColumns>(b, l, stream);
}

template <typename T, int N>
int backward_rows(const Backward& b, const Layout& l, void* stream) {
  return b.a.scale_count > 1 ? backward_rows<T, N, true>(b, l, stream)
                             : backward_rows<T, N, false>(b, l, stream);
}

template <typename T>
int backward(const Backward& b, const Layout& l, void* stream) {
  if (l.elements == 0)
    return launch(norm_backward_row_kernel<T>, dim3(static_cast<unsigned>(b.plan.blocks)), kThreads,
                  0, 1, true, stream, b);
  if (l.elements == kVec<T>) return backward_rows<T, kVec<T>>(b, l, stream);
  if constexpr (sizeof(T) == 2)
    if (l.elements == 2) return backward_rows<T, 2>(b, l, stream);
  return backward_rows<T, 1>(b, l, stream);
}

}  // namespace

cudaError_t norm_status(uint32_t* flags, int clear) { return take_status(flags, clear); }
cudaError_t norm_put_wait_limit(uint64_t limit_ns) { return put_wait_limit(limit_ns); }
cudaError_t norm_get_wait_limit(uint64_t* limit_ns) { return get_wait_limit(limit_ns); }

}  // namespace muon_train

extern "C" {

int muon_train_residual_norm_sm100(const muon_train_norm_args* args, void* stream) {
  using namespace muon_train;
  const int rc = check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->rows == 0) return MUON_POLAR_OK;
  if (args->hidden == nullptr || (args->pre_weight != nullptr && args->normed == nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  const muon_train_norm_args a = normalised(*args);
  switch (a.dtype) {
    case MUON_TRAIN_F32: return forward<float>(a, stream);
    case MUON_TRAIN_BF16: return forward<__nv_bfloat16>(a, stream);
    default: return forward<__half>(a, stream);
  }
}

size_t muon_train_residual_norm_workspace_bytes(const muon_train_norm_args* args) {
  using namespace muon_train;
  int64_t target = 0;
  if (check(args) != MUON_POLAR_OK || args->rows == 0) return 0;
  muon_train_norm_args a = normalised(*args);
  a.hidden = a.normed = nullptr;  // as in the backward call
  // over what the layout may be, which also depends on the gradients' alignment
  size_t bytes = 0;
  for (int aligned = 0; aligned < 2; ++aligned) {
    muon_train_norm_grads g = {};
    if (!aligned) g.grad_residual = reinterpret_cast<void*>(2);
    if (target_workers(make_layout(a, &g), &target) != MUON_POLAR_OK) return 0;
    const size_t b = make_plan(a, target).bytes;
    if (b > bytes) bytes = b;
  }
  return bytes;
}

int muon_train_residual_norm_backward_sm100(const muon_train_norm_args* args,
                                            const muon_train_norm_grads* grads, void* stream) {
  using namespace muon_train;
  int rc = check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->rows == 0) return MUON_POLAR_OK;
  if (grads == nullptr || (grads->grad_hidden == nullptr && grads->grad_normed == nullptr) ||
      (args->post_weight != nullptr && args->rstd_post == nullptr) ||
      (args->pre_weight != nullptr && grads->grad_normed != nullptr && args->rstd_pre == nullptr) ||
      (args->pre_weight == nullptr && grads->grad_normed != nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  Backward b;
  b.a = normalised(*args);
  b.g = *grads;
  if (b.a.post_weight == nullptr) b.g.grad_post_weight = nullptr;
  if (b.a.pre_weight == nullptr) b.g.grad_pre_weight = nullptr;
  if (b.a.gate == nullptr) b.g.grad_gate = nullptr;
  if (b.a.residual_scale == nullptr) b.g.grad_residual_scale = nullptr;
  b.a.hidden = b.a.normed = nullptr;
  const Layout layout = make_layout(b.a, &b.g);
  int64_t target = 0;
  rc = target_workers(layout, &target);
  if (rc != MUON_POLAR_OK) return rc;
  b.plan = make_plan(b.a, target);
  b.scale_rows = b.plan.blocks * (b.a.scale_count == 1 ? layout.cluster : 1);
  if (grads->workspace == nullptr || !aligned16(grads->workspace) ||
      grads->workspace_bytes < b.plan.bytes)
    return MUON_POLAR_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(grads->workspace);
  const bool want_gate_sums = b.g.grad_gate != nullptr && !b.plan.gate_per_row;
  b.gain = b.g.grad_post_weight != nullptr || want_gate_sums
               ? reinterpret_cast<float*>(ws + b.plan.gain_off) : nullptr;
  b.pre = b.g.grad_pre_weight != nullptr ? reinterpret_cast<float*>(ws + b.plan.pre_off) : nullptr;
  b.scale = b.g.grad_residual_scale != nullptr ? reinterpret_cast<float*>(ws + b.plan.scale_off)
                                               : nullptr;
  switch (b.a.dtype) {
    case MUON_TRAIN_F32: rc = backward<float>(b, layout, stream); break;
    case MUON_TRAIN_BF16: rc = backward<__nv_bfloat16>(b, layout, stream); break;
    default: rc = backward<__half>(b, layout, stream); break;
  }
  if (rc != MUON_POLAR_OK || (b.gain == nullptr && b.pre == nullptr && b.scale == nullptr)) return rc;
  const unsigned columns = static_cast<unsigned>((b.a.width + 31) / 32);
  const int64_t gate_rows = want_gate_sums ? b.plan.groups : 0;
  const unsigned what = 3 + static_cast<unsigned>(gate_rows < kGateRowBlocks ? gate_rows : kGateRowBlocks);
  return launch(norm_sums_kernel, dim3(columns, what), kSumWarps * 32, 0, 1, true, stream, b);
}

}  // extern "C"
