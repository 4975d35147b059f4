// rotary_sm100.cu -- rotary positions of queries and keys in one launch.
//
// For a head of `dim` elements with `pairs` frequencies f, at position n:
//   angle_i = n f_i,  c = scale cos(angle_i),  s = scale sin(angle_i)
//   (a, b) -> (a c - b s, b c + a s)
// with (a, b) = (x[i], x[i + pairs]) or, interleaved, (x[2i], x[2i + 1]).  The
// elements from 2 pairs on are copied.  The gradient is the same with -s.
//
// The angle is taken in turns, n (f / 2 pi), in 64 bits and reduced to half a
// turn before it is rounded to 32: at position 10^7 a 32-bit angle is off by
// half a radian.  The operator is bound by memory: every element is read and
// written once.  A block takes a few tokens, computes their cosines and sines
// into shared memory once for all heads, and turns all heads of both tensors
// from there, in vectors of up to 16 bytes.
#include "train_common.cuh"

namespace muon_train {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;          // vectors (pairs of them, by halves) in flight a thread
constexpr int kTableBytes = 16384;  // cosines and sines of a block's tokens

struct Plan {
  int tokens;        // of a block
  int vectors;       // items of a head: rotated vectors (pairs of them, by halves), then copied ones
  int turned;        // of these, rotated
};

__device__ __forceinline__ double frequency(const muon_train_rotary_args& a, int i) {
  return a.frequency_bytes == 8 ? static_cast<const double*>(a.frequencies)[i]
                                : static_cast<double>(static_cast<const float*>(a.frequencies)[i]);
}
__device__ __forceinline__ double position(const muon_train_rotary_args& a, int64_t batch, int64_t row) {
  const int64_t i = (a.position_rows > 1 ? batch * a.length : 0) + row;
  return a.position_bytes == 8 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[i])
                               : static_cast<double>(static_cast<const int32_t*>(a.positions)[i]);
}

// N elements a load.  kInterleaved: pairs side by side, both in one load where
// N > 1; else, and by halves, the partners are two loads.
template <typename T, int N, bool kInterleaved>
__global__ void __launch_bounds__(kThreads)
    rotary_kernel(const __grid_constant__ muon_train_rotary_args a, Plan plan) {
  using E = Elements<T, N>;
  using Raw = typename E::Raw;
  constexpr bool kInside = kInterleaved && N > 1;
  extern __shared__ float2 table[];  // [token][pair]
  begin_kernel();
  const uint32_t length = static_cast<uint32_t>(a.length), all = static_cast<uint32_t>(a.batch) * length;
  const uint32_t first = blockIdx.x * plan.tokens;
  const int tokens = static_cast<int>(min(all - first, static_cast<uint32_t>(plan.tokens)));
  const int pairs = static_cast<int>(a.pairs);
  for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
    const uint32_t token = first + i / pairs;
    const double turns = position(a, token / length, token % length) *
                         (frequency(a, i % pairs) * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    table[i] = make_float2(c * a.scale, a.inverse ? -s * a.scale : s * a.scale);
  }
  __syncthreads();
  const int heads = static_cast<int>(a.heads[0] + a.heads[1]);
  const int each = heads * plan.vectors, items = tokens * each;
  for (int i0 = threadIdx.x; i0 < items; i0 += kThreads * kUnroll) {
    Raw low[kUnroll], high[kUnroll];
    T* to[kUnroll];
    int cell[kUnroll];  // first pair in the table; -1: copied
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * kThreads;
      to[u] = nullptr;
      if (i >= items) continue;
      const int t = i / each, rest = i - t * each, head = rest / plan.vectors, v = rest - head * plan.vectors;
      const int which = head >= a.heads[0] ? 1 : 0;
      const int64_t h = head - (which ? a.heads[0] : 0);
      const uint32_t token = first + t, b = token / length, r = token - b * length;
      const bool turn = v < plan.turned;
      int column = v * N;  // of the head
      if (!kInside) column = !turn ? column + pairs : kInterleaved ? 2 * v : column;
      const T* from = static_cast<const T*>(a.x[which]) + b * a.x_batch[which] + r * a.x_row[which] +
                      h * a.x_head[which] + column;
      to[u] = static_cast<T*>(a.y[which]) + (token * a.heads[which] + h) * a.dim + column;
      cell[u] = turn ? t * pairs + (kInterleaved ? column / 2 : column) : -1;
      low[u] = E::load(from);
      if (!kInside && turn) high[u] = E::load(from + (kInterleaved ? 1 : pairs));
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (to[u] == nullptr) continue;
      if (cell[u] < 0) {
        E::store(to[u], low[u]);
        continue;
      }
      float x[N], z[N];
      E::unpack(low[u], x);
      if constexpr (kInside) {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          const float2 cs = table[cell[u] + j];
          z[2 * j] = x[2 * j] * cs.x - x[2 * j + 1] * cs.y;
          z[2 * j + 1] = x[2 * j + 1] * cs.x + x[2 * j] * cs.y;
        }
        E::store(to[u], E::pack(z));
      } else {
        float y[N], w[N];
        E::unpack(high[u], y);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float2 cs = table[cell[u] + j];
          z[j] = x[j] * cs.x - y[j] * cs.y;
          w[j] = y[j] * cs.x + x[j] * cs.y;
        }
        E::store(to[u], E::pack(z));
        E::store(to[u] + (kInterleaved ? 1 : pairs), E::pack(w));
      }
    }
  }
}

// Whether all loads and stores may take n elements at once.
bool fits(const muon_train_rotary_args& a, int n) {
  const int64_t bytes = n * static_cast<int64_t>(dtype_size(a.dtype));
  if (a.dim % n != 0 || (a.interleaved ? 2 * a.pairs : a.pairs) % n != 0) return false;
  for (int w = 0; w < 2; ++w) {
    if (a.heads[w] == 0) continue;
    if ((reinterpret_cast<uintptr_t>(a.x[w]) | reinterpret_cast<uintptr_t>(a.y[w])) % bytes != 0) return false;
    if ((a.batch > 1 && a.x_batch[w] % n != 0) || (a.length > 1 && a.x_row[w] % n != 0) ||
        (a.heads[w] > 1 && a.x_head[w] % n != 0))
      return false;
  }
  return true;
}

template <typename T, int N, bool kInterleaved>
int run(const muon_train_rotary_args& a, void* stream) {
  Plan p;
  p.turned = static_cast<int>((kInterleaved && N > 1 ? 2 * a.pairs : a.pairs) / N);
  p.vectors = p.turned + static_cast<int>((a.dim - 2 * a.pairs) / N);
  const int64_t heads = a.heads[0] + a.heads[1], items = heads * p.vectors;
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc != MUON_POLAR_OK) return rc;
  // two rounds of unrolled vectors a block, but blocks for every SM first, and a table that fits
  const int64_t all = a.batch * a.length;
  int64_t tokens = (2 * kUnroll * kThreads + items - 1) / items;
  const int64_t spread = (all + 4 * sms - 1) / (4 * sms);
  const int64_t room = kTableBytes / (static_cast<int64_t>(sizeof(float2)) * (a.pairs > 0 ? a.pairs : 1));
  tokens = tokens < spread ? tokens : spread;
  tokens = tokens < room ? tokens : room;
  p.tokens = static_cast<int>(tokens < 1 ? 1 : tokens);
  const int64_t blocks = (all + p.tokens - 1) / p.tokens;
  return launch(rotary_kernel<T, N, kInterleaved>, dim3(static_cast<unsigned>(blocks)), kThreads,
                p.tokens * a.pairs * sizeof(float2), 1, true, stream, a, p);
}

template <typename T, bool kInterleaved>
int run(const muon_train_rotary_args& a, void* stream) {
  if constexpr (sizeof(T) == 2)
    if (fits(a, 8)) return run<T, 8, kInterleaved>(a, stream);
  if (fits(a, 4)) return run<T, 4, kInterleaved>(a, stream);
  if (fits(a, 2)) return run<T, 2, kInterleaved>(a, stream);
  return run<T, 1, kInterleaved>(a, stream);
}

template <typename T>
int run(const muon_train_rotary_args& a, void* stream) {
  return a.interleaved ? run<T, true>(a, stream) : run<T, false>(a, stream);
}

}  // namespace
}  // namespace muon_train

extern "C" {

int muon_train_rotary_sm100(const muon_train_rotary_args* args, void* stream) {
  using namespace muon_train;
  if (args == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  const muon_train_rotary_args& a = *args;
  if (a.batch < 0 || a.length < 0 || a.dim < 1 || a.dim > MUON_TRAIN_MAX_ROTARY_DIM || a.pairs < 0 ||
      2 * a.pairs > a.dim || !valid_dtype(a.dtype) || a.heads[0] < 0 || a.heads[1] < 0 ||
      (a.frequency_bytes != 4 && a.frequency_bytes != 8) || (a.position_bytes != 4 && a.position_bytes != 8) ||
      (a.position_rows != 1 && a.position_rows != a.batch))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  const int64_t rows = a.batch * a.length, heads = a.heads[0] + a.heads[1];
  if (a.batch > (int64_t{1} << 31) || a.length > (int64_t{1} << 31) || rows >= (int64_t{1} << 31) ||
      heads * a.dim >= (int64_t{1} << 24))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (rows == 0 || heads == 0) return MUON_POLAR_OK;
  for (int w = 0; w < 2; ++w)
    if (a.heads[w] > 0 && (a.x[w] == nullptr || a.y[w] == nullptr)) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (a.positions == nullptr || (a.pairs > 0 && a.frequencies == nullptr)) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  switch (a.dtype) {
    case MUON_TRAIN_F32: return run<float>(a, stream);
    case MUON_TRAIN_BF16: return run<__nv_bfloat16>(a, stream);
    default: return run<__half>(a, stream);
  }
}

}  // extern "C"
