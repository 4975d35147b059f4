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
// One vector (two, by halves) in flight a thread, but every thread that an SM
// has: four a thread in 57 registers took 79 us for 16384 tokens of 40 heads of
// 128 bf16, two 67, one 65 in 40 registers and 58 in 32 (floor 51; 5.8 TB/s).
constexpr int kBlocksPerSm = 8;
constexpr int kRounds = 4;          // vectors of a thread
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

// a c - b s and b c + a s, rounded the same way in every form of the kernel.
__device__ __forceinline__ float2 turned(float a, float b, float2 cs) {
  return make_float2(fmaf(-b, cs.y, __fmul_rn(a, cs.x)), fmaf(a, cs.y, __fmul_rn(b, cs.x)));
}

// kN entries of the table, two at a time where their number is even: then it
// divides the pairs, and every place.
template <int kN>
__device__ __forceinline__ void load_turns(float2 (&to)[kN], const float2* from) {
  if constexpr (kN % 2 == 0) {
#pragma unroll
    for (int j = 0; j < kN; j += 2) {
      const float4 v = *reinterpret_cast<const float4*>(from + j);
      to[j] = make_float2(v.x, v.y);
      to[j + 1] = make_float2(v.z, v.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; ++j) to[j] = from[j];
  }
}

// N elements a load.  kInterleaved: pairs side by side, both in one load where
// N > 1; else, and by halves, the partners are two loads.
template <typename T, int N, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    rotary_kernel(const __grid_constant__ muon_train_rotary_args a, Plan plan) {
  using E = Elements<T, N>;
  using Raw = typename E::Raw;
  constexpr bool kInside = kInterleaved && N > 1;
  extern __shared__ __align__(16) float2 table[];  // [token][pair]
  begin_kernel();
  const uint32_t length = static_cast<uint32_t>(a.length), all = static_cast<uint32_t>(a.batch) * length;
  const uint32_t first = blockIdx.x * plan.tokens;
  const int tokens = static_cast<int>(min(all - first, static_cast<uint32_t>(plan.tokens)));
  const int pairs = static_cast<int>(a.pairs);
  const int heads = static_cast<int>(a.heads[0] + a.heads[1]);
  const int each = heads * plan.vectors, items = tokens * each;
  Raw low, high;
  T* to;
  int cell;  // first pair in the table; -1: copied
  const auto load = [&](int i) {
    const int t = i / each, rest = i - t * each, head = rest / plan.vectors, v = rest - head * plan.vectors;
    const int which = head >= a.heads[0] ? 1 : 0;
    const int64_t h = head - (which ? a.heads[0] : 0);
    const uint32_t token = first + t, b = token / length, r = token - b * length;
    const bool turn = v < plan.turned;
    int column = v * N;  // of the head
    if (!kInside) column = !turn ? column + pairs : kInterleaved ? 2 * v : column;
    const T* from = static_cast<const T*>(a.x[which]) + b * a.x_batch[which] + r * a.x_row[which] +
                    h * a.x_head[which] + column;
    to = static_cast<T*>(a.y[which]) + (token * a.heads[which] + h) * a.dim + column;
    cell = turn ? t * pairs + (kInterleaved ? column / 2 : column) : -1;
    low = E::load(from);
    if (!kInside && turn) high = E::load(from + (kInterleaved ? 1 : pairs));
  };
  int item = threadIdx.x;
  if (item < items) load(item);  // in flight while the table is made
  for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
    const uint32_t token = first + i / pairs;
    const double turns = position(a, token / length, token % length) *
                         (frequency(a, i % pairs) * 0.15915494309189533577);  // 1 / (2 pi)
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    table[i] = make_float2(c * a.scale, a.inverse ? -s * a.scale : s * a.scale);
  }
  __syncthreads();
  while (item < items) {
    if (cell < 0) {
      E::store(to, low);
    } else {
      float x[N], z[N];
      E::unpack(low, x);
      float2 turn[kInside ? N / 2 : N];
      load_turns(turn, table + cell);
      if constexpr (kInside) {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          const float2 p = turned(x[2 * j], x[2 * j + 1], turn[j]);
          z[2 * j] = p.x;
          z[2 * j + 1] = p.y;
        }
        E::store(to, E::pack(z));
      } else {
        float y[N], w[N];
        E::unpack(high, y);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float2 p = turned(x[j], y[j], turn[j]);
          z[j] = p.x;
          w[j] = p.y;
        }
        E::store(to, E::pack(z));
        E::store(to + (kInterleaved ? 1 : pairs), E::pack(w));
      }
    }
    item += kThreads;
    if (item < items) load(item);
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
  // a few vectors a thread, but blocks for every SM first, and a table that fits
  const int64_t all = a.batch * a.length;
  int64_t tokens = (kRounds * kThreads + items - 1) / items;
  const int64_t spread = (all + kBlocksPerSm * sms - 1) / (kBlocksPerSm * sms);
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
