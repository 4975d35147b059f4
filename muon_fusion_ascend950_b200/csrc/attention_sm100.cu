// attention_sm100.cu -- attention of training sequences, forward and backward,
// on the tensor cores.
//
//   s_ij = scale q_i . k_j over the keys that query i sees
//   p_ij = exp(s_ij - lse_i), out_i = sum_j p_ij v_j
//   delta_i = dout_i . out_i, dp_ij = dout_i . v_j, ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j, dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij dout_i
// (dk and dv also over the query heads that share the key head).
//
// Tiles of 128 queries and 128 keys.  All products are tcgen05 ones with fp32
// results in tensor memory; tiles of the inputs come by TMA into swizzled
// shared memory.  The scores are read from tensor memory into registers, a row
// a thread, and the probabilities go back there as 16-bit values, in place of
// the scores, as the next product's left operand: neither is ever in shared or
// global memory.  Eight warps of a block work on the scores, one loads and one
// issues the products.
//
// The backward pass computes the scores again.  It is two kernels, one for a
// tile of keys (dk, dv: four products a pair of tiles) and one for a tile of
// queries (dq: three): seven products in place of five, but every sum is held
// in tensor memory from its first term to its last, without atomics or partial
// sums in memory, and its order is fixed.
//
// Rounding: p and ds are rounded to the inputs' type as operands of the second
// products, as the inputs were; everything else is fp32.  delta is taken from
// the output and from what rounding took from it (out_rest), so that it has the
// scores' precision.  fp16 operands are scaled by powers of two: p by 2^7
// (forward; at most 2^15) and 2^10 (backward), so that small ones do not fall
// below fp16's range, and ds by a factor for each query (dq) or key (dk), of what
// its own row can reach (ds_exponent).
//
// What bounds it (heads of 128, bf16): the latency of scores, probabilities and
// product one after another, which two tiles in flight cover in part (the tensor
// pipe is busy in 53 to 67% of the cycles), and in the backward pass two more
// products than needed.  Long sequences also draw 1000 W, which brings the clock
// to 1.57-1.7 GHz (2 x 8192 both ways, 16 heads: forward 1000 us, 1100 TFLOP/s;
// backward 3320, 1160 TFLOP/s of its seven products; plain products sustain 1382
// at that power); shorter ones do not (4096 causal, 37 heads: 167 and 529 us, 950
// and 750 TFLOP/s of the products needed).  With heads of 64 the exponentials and
// the issue slots come first (2 x 8192, 16 heads: 750 and 2240 us, 733 and 614
// TFLOP/s).
#include <cuda.h>

#include <type_traits>

#include "tcgen05_attention.cuh"
#include "train_common.cuh"

namespace muon_train {
namespace {

using namespace muon_sm100;

constexpr int kTileShift = 7, kTile = 1 << kTileShift;  // queries, or keys, of a tile
constexpr int kThreads = 384;  // warps 0-7: scores, 8: loads, 9: products; 10 and 11 only give registers
constexpr int kLoadWarp = 8, kMmaWarp = 9;
// Registers of a thread at launch, and then of the two warpgroups that work on
// scores and of the third.
constexpr int kLaunchRegisters = 168, kScoreRegisters = 208, kOtherRegisters = 88;
static_assert(2 * kScoreRegisters + kOtherRegisters <= 3 * kLaunchRegisters, "no more than there are at launch");
constexpr uint32_t kTmemColumns = 512;
constexpr int kAtom = kTile * 128;  // bytes of 64 columns of a tile, the swizzle's width

template <typename T>
constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same_v<T, __half>;
// Binary exponents that p is raised by.
template <typename T>
constexpr float kRaise = kBf16<T> ? 0.0f : 7.0f;
template <typename T>
constexpr float kRaiseBack = kBf16<T> ? 0.0f : 10.0f;
// The running maximum may lag behind by this many binary exponents before the
// sums so far are scaled again: nearly all rows then keep their first maximum.
constexpr float kLag = 8.0f;

// ------------------------------------------------------------ sequences
struct Problem {
  void* out;                // forward: out; backward: see there
  void* out2;
  float* lse;
  const float* stats;       // backward: [2][heads][rows]: -lse (binary), -delta
  const float* grad_norm;   // backward, fp16: [rows][heads]: |dout|
  const float* value_norm;  // [batch * keys][kv_heads]: |v|
  const float2* query_top;  // the largest |dout| and |delta| of each tile of queries, of the heads that share a key head
  const float* key_top;     // the largest |v| of each tile of keys
  const int32_t* lengths;
  const int32_t* offsets;
  int64_t rows;             // batch * length
  int length, keys, heads, kv_heads, dim, sequences, batch, window, causal;
  int section;              // heads (pairs of them: by_heads) whose tiles are worked on together
  int by_heads;             // forward: 1, pairs of tiles are of two heads; 0, of one
  int blind;                // kernel for keys: queries from the first on that see no key, and that its maps leave out
  float scale;
};

// One tile of rows of one sequence.
struct Tile {
  int batch;      // coordinate of the tensors
  int row0;       // first row of the sequence
  int first;      // of the tile, in the sequence
  int stored;     // rows of the sequence that are written
  int queries;    // rows that count, as queries
  int keys;       // and as keys
  int number;     // of the sequence's first tile
  bool found;
};

__device__ __forceinline__ int clamp_int(int v, int low, int high) { return v < low ? low : v > high ? high : v; }

// Item `item`: a tile of 2^shift rows of one of `heads` heads, of `rows` rows a
// batch entry; packed, of `tiles` tiles of all sequences, the tokens before the
// first and behind the last among them as sequences that see nothing.  Heads of
// all entries go in sections, and those of a section tile by tile, with
// `backwards` from the last, which has the most keys under a causal mask.
//
// The tiles of packed sequence s, which begins at token b, are numbered from
// (b >> shift) + s on.  That leaves room for all of the sequences before it, and
// some numbers without a tile, but the sequence of a number is found by
// bisection.  Every warp looks for itself.
__device__ __forceinline__ Tile find_tile(const Problem& p, int item, int rows, int heads, int shift, int tiles,
                                          bool backwards, int* head) {
  Tile t;
  const int size = 1 << shift, per = p.offsets == nullptr ? (rows + size - 1) >> shift : tiles;
  const int section = item / (p.section * per), in_it = item - section * p.section * per;
  const int columns = min(p.section, p.batch * heads - section * p.section);
  const int rank = in_it / columns, at = section * p.section + in_it - rank * columns;
  const int index = backwards ? per - 1 - rank : rank;
  *head = at % heads;
  if (p.offsets == nullptr) {
    t.found = true;
    t.batch = at / heads;
    t.first = index << shift;
    t.row0 = 0;
    t.number = 0;
    t.stored = rows;
    t.queries = p.length;
    t.keys = p.keys;
    if (p.lengths != nullptr) t.queries = t.keys = clamp_int(p.lengths[t.batch], 0, p.length);
    return t;
  }
  const int lane = threadIdx.x % 32, count = p.sequences + 2;
  // the last sequence that starts at this index or before, 32 of them at a time
  int begin, end, low = 0, span = count, step, pick;
  do {
    step = (span + 31) / 32;
    const int s = low + lane * step;
    const bool in = lane * step < span;
    begin = end = 0;
    if (in) {
      begin = s == 0 ? 0 : clamp_int(p.offsets[s - 1], 0, p.length);
      end = s == count - 1 ? p.length : clamp_int(p.offsets[s], 0, p.length);
    }
    pick = max(__popc(__ballot_sync(kFullMask, in && (begin >> shift) + s <= index)) - 1, 0);  // below 0: descending offsets
    low += pick * step;
    span = min(step, span - pick * step);
  } while (step > 1);
  t.batch = 0;
  t.row0 = __shfl_sync(kFullMask, begin, pick);
  t.stored = max(__shfl_sync(kFullMask, end, pick) - t.row0, 0);
  t.queries = t.keys = low > 0 && low < count - 1 ? t.stored : 0;
  t.number = (t.row0 >> shift) + low;
  const int local = index - t.number;
  t.found = local >= 0 && local < (t.stored + size - 1) >> shift;
  t.first = t.found ? local << shift : 0;
  return t;
}

// The place of the first of a key head's tiles of 128 rows in an array of a value
// a tile: of all sequences' together where they are packed.
__device__ __forceinline__ int64_t tile_slot(const Problem& p, const Tile& t, int rows, int tiles, int kv_head) {
  const int per = p.offsets == nullptr ? (rows + kTile - 1) >> kTileShift : tiles;
  return (static_cast<int64_t>(t.batch) * p.kv_heads + kv_head) * per + t.number;
}

// Keys [low, high) that queries [i0, i1) of the sequence see at least in part.
__device__ __forceinline__ void keys_of(const Problem& p, const Tile& t, int i0, int i1, int* low, int* high) {
  const int shift = t.keys - t.queries;
  *low = 0;
  *high = i0 < i1 ? t.keys : 0;
  if (p.causal) *high = min(*high, i1 + shift);
  if (p.window > 0) {
    *low = max(0, i0 + shift - p.window + 1);
    *high = min(*high, i1 - 1 + shift + p.window);
  }
  *high = max(*high, 0);
  *low = min(*low, *high);
}
// Queries [low, high) that see keys [j0, j1) at least in part.
__device__ __forceinline__ void queries_of(const Problem& p, const Tile& t, int j0, int j1, int* low, int* high) {
  const int shift = t.keys - t.queries;
  *low = 0;
  *high = j0 < j1 ? t.queries : 0;
  if (p.causal) *low = max(0, j0 - shift);
  if (p.window > 0) {
    if (!p.causal) *low = max(*low, j0 - shift - p.window + 1);
    *high = min(*high, j1 - 1 - shift + p.window);
  }
  *high = max(*high, 0);
  *low = min(*low, *high);
}

// ------------------------------------------------------------ shared pieces
// All lanes of a warp wait; false for all if one gave up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  return __all_sync(kFullMask, ring_wait(bar, parity, failed));
}

// The items of a block, a tile of a head each.  The grid has a block for each
// item; one that runs takes over those that have not begun, in the order of
// their indices, which goes from the items with the most tiles to those with
// the fewest.  The warp that loads asks, every warp takes the answer for itself.
// (Dealt out in fixed turns, two padded batch entries of 8192 and some 5000
// tokens took 804 us forward, 699 with a block an item, whose start and end
// stand alone.)
constexpr int kAnswers = 4;
struct Items {
  __align__(16) uint4 answer[kAnswers];
  uint64_t full[kAnswers], empty[kAnswers];

  __device__ __forceinline__ void init() {
    for (int i = 0; i < kAnswers; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 10);  // warps that take it
    }
  }
  // The item behind item k; -1: there is none.
  __device__ __forceinline__ int take(int k, volatile int* failed) {
    if (!warp_wait(&full[k % kAnswers], (k / kAnswers) & 1, failed)) return -1;
    const int item = cancelled_block(&answer[k % kAnswers]);
    fence_proxy_async_smem();
    __syncwarp();
    if (threadIdx.x % 32 == 0) mbar_arrive(&empty[k % kAnswers]);
    return item;
  }
  // The same for the loading warp, which asks: when it has asked for the last
  // tile of its item and not before, so that the blocks that end first get the
  // items that are left.
  __device__ __forceinline__ int next(int* asked, volatile int* failed) {
    const int k = *asked;
    if (k >= kAnswers && !warp_wait(&empty[k % kAnswers], (k / kAnswers - 1) & 1, failed)) return -1;
    if (threadIdx.x % 32 == 0) {
      mbar_arrive_expect_tx(&full[k % kAnswers], 16);
      try_cancel_block(&answer[k % kAnswers], &full[k % kAnswers]);
    }
    __syncwarp();
    ++*asked;
    return take(k, failed);
  }
};

// Rows from `valid` on of a tile in shared memory become zeros: they belong to
// another sequence or to padding, and 0 * NaN would reach the sums.
template <int kCols>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int valid) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int a = 0; a < kCols / 64; ++a)
    for (int i = valid * 128 + lane * 16; i < kAtom; i += 512)
      *reinterpret_cast<uint4*>(tile + a * kAtom + i) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// Boxes of 64 columns of 128 rows.
template <int kCols>
__device__ __forceinline__ void load_tile(uint8_t* to, const CUtensorMap* map, uint64_t* bar, int row, int head,
                                          int batch) {
#pragma unroll
  for (int a = 0; a < kCols / 64; ++a) tma_load_4d(to + a * kAtom, map, bar, a * 64, row, head, batch);
}

// Operand descriptors of a tile as their two words: the upper one is the same
// for all tiles, and a step along the summed axis adds to the lower one.  The
// warp that issues the products shares its scheduler with two that work on
// scores: behind a branch of one thread, with its operands in plain registers,
// a product that runs in 64 cycles took 100 to 125 to issue beside busy warps,
// by a whole warp with the elected lane's predicate 68 to 80.
struct Operand {
  uint32_t low, high;
  __device__ __forceinline__ Operand(const uint8_t* tile, uint32_t lbo) {
    const uint64_t d = smem_desc_sw128(smem_addr(tile), lbo, 1024);
    low = static_cast<uint32_t>(d);
    high = static_cast<uint32_t>(d >> 32);
  }
  __device__ __forceinline__ uint64_t at(uint32_t bytes) const {
    return static_cast<uint64_t>(high) << 32 | (low + (bytes >> 4));
  }
};

// D[128 x 128] = A B^T over the first `dim` of kCols columns of both tiles.
template <int kCols>
__device__ __forceinline__ void scores(uint32_t d, const uint8_t* a, const uint8_t* b, uint32_t idesc, int dim,
                                       uint32_t el) {
  const Operand oa(a, 16), ob(b, 16);
#pragma unroll
  for (int k = 0; k < kCols / 16; ++k)
    if (k * 16 < dim) {
      const uint32_t at = (k / 4) * kAtom + (k % 4) * 32;
      umma_ss(d, oa.at(at), ob.at(at), idesc, k > 0, el);
    }
}
// D[128 x n] (+)= A[tmem: 128 x 64] B, B's rows summed over: four products, of
// the tile's first 64 rows or its last.
__device__ __forceinline__ void weighted(uint32_t d, uint32_t a, const uint8_t* b, int half, uint32_t idesc, bool more,
                                         uint32_t el) {
  const Operand ob(b + half * 64 * 128, kAtom);
#pragma unroll
  for (int k = 0; k < 4; ++k) umma_ts(d, a + k * 8, ob.at(k * 2048), idesc, more || k > 0, el);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float low, float high) {
  if constexpr (kBf16<T>) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

__device__ __forceinline__ float as_float(uint32_t v) { return __uint_as_float(v); }

// Four vectors of a row a lane, turned among each four lanes: afterwards x[r] is
// vector (lane % 4) of the row of lane (lane & ~3) + r.
__device__ __forceinline__ void turn(uint4 (&x)[4]) {
#pragma unroll
  for (int b = 1; b < 4; b *= 2) {
    const bool odd = threadIdx.x & b;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q & b) continue;
      uint32_t *u = &x[q].x, *v = &x[q + b].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t got = __shfl_xor_sync(kFullMask, odd ? u[i] : v[i], b);
        u[i] = odd ? got : u[i];
        v[i] = odd ? v[i] : got;
      }
    }
  }
}

// A warp's rows of a result in tensor memory times `by` to memory, lane by lane
// at `to` and `stride` elements apart; with `rest` also what the rounding took.
// kTurned: four lanes write 64 bytes of a row together, eight rows a store;
// else each lane its own row, 16 bytes and 32 rows a store.  Those stores hold
// the two tiles of a pair up where rows have 256 bytes: 128 x 256 causal, 16
// heads of 128 over 4, 191 us with own rows, 121 turned; 8 x 4096 651 and 556.
// With 128 bytes a row they gain where tiles are full (256: 109 and 100 us;
// 4096: 423 and 413), and lose by their exchange where sequences end inside
// (1024 packed ones of 64, 16 heads of 64 over 4: 442 and 462 us; backward 995
// and 1050).
template <typename T, int kCols, bool kTurned>
__device__ __forceinline__ void store_rows(T* to, T* rest, int64_t stride, uint32_t taddr, int dim, float by, bool write) {
  const unsigned rows = __ballot_sync(kFullMask, write);
  const int lane = threadIdx.x % 32, m = lane % 4;
  const auto store = [&](T* own, uint4 (&x)[4], int column) {
    if constexpr (kTurned) {
      turn(x);
      T* row0 = own - m * stride;
      column += 8 * m;
      if (column >= dim) return;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (rows >> (lane - m + r) & 1) *reinterpret_cast<uint4*>(row0 + r * stride + column) = x[r];
    } else if (write) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (column + 8 * q < dim) *reinterpret_cast<uint4*>(own + column + 8 * q) = x[q];
    }
  };
#pragma unroll 1
  for (int c = 0; c < kCols; c += 32) {
    if (c >= dim) return;
    uint32_t t[32];
    tmem_ld_32x32b_x32(taddr + c, t);
    tmem_wait_ld(t);
    uint4 x[4], y[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[8], w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = as_float(t[8 * q + i]) * by;
      x[q] = pack<T>(v);
      unpack<T>(x[q], w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] -= w[i];
      y[q] = pack<T>(v);
    }
    store(to, x, c);
    if (rest != nullptr) store(rest, y, c);
    __syncwarp();
  }
}
template <typename T>
__device__ __forceinline__ void zero_row(T* to, int dim) {
  for (int c = 0; c < dim; c += 8) *reinterpret_cast<uint4*>(to + c) = make_uint4(0, 0, 0, 0);
}

// After a wait that gave up: the copies in flight to the last fills of a ring.
__device__ __forceinline__ void drain_fills(uint64_t* full, int stages, int fills) {
  const int first = fills > stages ? fills - stages : 0;
  drain_ring(full, stages, first % stages, (first / stages) & 1, fills - first);
}

// The end of a block, by all threads: tensor memory is given back.  After a wait
// that gave up, only when the copies and products in flight have ended: those
// to a ring after `fills` of its tiles, and the last of `loads` to `once` and
// `again` each.
__device__ __forceinline__ void finish(uint32_t tmem, volatile int* failed, int fills, uint64_t* full, int stages,
                                       uint64_t* once, int loads, uint64_t* again, int loads_again,
                                       Items& queue, int asked, uint64_t* drained) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  tc_fence_before();
  __syncthreads();
  if (*failed && warp == kLoadWarp && lane == 0) {
    drain_fills(full, stages, fills);
    if (loads > 0) drain_ring(once, 1, 0, (loads - 1) & 1, 1);
    if (loads_again > 0) drain_ring(again, 1, 0, (loads_again - 1) & 1, 1);
    drain_fills(queue.full, kAnswers, asked);
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    if (*failed) {
      umma_commit(drained, elect_one());
      __syncwarp();
      drain_ring(drained, 1, 0, 0, 1);
      __syncwarp();
    }
    tmem_relinquish();
    tmem_dealloc(tmem, kTmemColumns);
  }
}

// ------------------------------------------------------------ forward
template <int kCols>
struct Forward {
  static constexpr int kTileBytes = kTile * kCols * 2;
  static constexpr int kStages = kCols == 128 ? 5 : 8;  // tiles of keys or values
  static constexpr int kBytes = (2 + kStages) * kTileBytes + 1024;
};

// An item is two tiles of queries, which take turns: while the scores of one are
// worked on, the products of the other run.  They are those of two heads at the
// same rows where an even number of heads shares a key head, else neighbours of
// one head, of which one has more keys under a causal mask, and a short sequence
// may have one only (16 heads over 4, 1024 packed sequences of 64 tokens: 667 us
// with neighbours, 441 with two heads; 8 x 4096 causal of 128: 585 and 562).
// Keys and values pass through a ring of tiles, keys j, values j, keys j + 1 and
// so on.  Loads and products go on to the next item while the results of the last
// are written.
struct Pair {
  int head, heads_on, rows_on;  // of the first tile; from it to the second
  Tile t;
  int from[2], to[2];  // key tiles of the two query tiles
  int first, last;     // of both

  __device__ __forceinline__ Pair(const Problem& p, int item, int tiles) {
    heads_on = p.by_heads;
    rows_on = p.by_heads ? 0 : kTile;
    t = find_tile(p, item, p.length, p.heads >> heads_on, kTileShift + 1 - heads_on, tiles, true, &head);
    head <<= heads_on;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int i0 = t.first + i * rows_on;
      int low = 0, high = 0;
      if (t.found) keys_of(p, t, min(i0, t.queries), min(i0 + kTile, t.queries), &low, &high);
      from[i] = low / kTile;
      to[i] = (high + kTile - 1) / kTile;
      if (low >= high) from[i] = to[i] = 0;
    }
    first = from[0], last = to[0];
    if (from[0] == to[0]) first = from[1], last = to[1];
    if (from[0] < to[0] && from[1] < to[1]) first = min(from[0], from[1]), last = max(to[0], to[1]);
  }
};

template <typename T, int kCols, bool kTurned>
__global__ void __launch_bounds__(kThreads, 1)
    forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Problem p, int tiles) {
  using C = Forward<kCols>;
  extern __shared__ __align__(1024) uint8_t dynamic[];
  __shared__ uint64_t q_full[2], q_empty[2], s_full[2], p_full[2][2], o_done[2], drained, full[C::kStages],
      empty[C::kStages];
  __shared__ Items queue;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed_word;
  volatile int* failed = &failed_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dynamic) + 1023) & ~uintptr_t{1023});
  uint8_t* ring = smem + 2 * C::kTileBytes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i][0], kTile);
      mbar_init(&p_full[i][1], kTile);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(&drained, 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    queue.init();
    fence_mbar_init();
    failed_word = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_slot, kTmemColumns);
  tc_fence_before();
  begin_kernel();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const bool foreign = p.offsets != nullptr || p.lengths != nullptr;

  int fills = 0, loads[2] = {0, 0}, asked = 0;
  if (warp >= kLoadWarp) {
    give_registers<kOtherRegisters>();
    if (warp == kLoadWarp) {
      bool ok = true;
      for (int item = blockIdx.x; ok && item >= 0; item = queue.next(&asked, failed)) {
        const Pair w(p, item, tiles);
        const int kv_head = w.head / (p.heads / p.kv_heads);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (w.from[i] == w.to[i]) continue;
          if (loads[i] > 0) ok = ok && warp_wait(&q_empty[i], (loads[i] - 1) & 1, failed);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[i], C::kTileBytes);
            load_tile<kCols>(smem + i * C::kTileBytes, &map_q, &q_full[i], w.t.row0 + w.t.first + i * w.rows_on,
                             w.head + i * w.heads_on, w.t.batch);
          }
          ++loads[i];
        }
        for (int j = w.first; j < w.last && ok; ++j) {
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const int s = fills % C::kStages;
            if (fills >= C::kStages) ok = ok && warp_wait(&empty[s], (fills / C::kStages - 1) & 1, failed);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&full[s], C::kTileBytes);
              load_tile<kCols>(ring + s * C::kTileBytes, which ? &map_v : &map_k, &full[s], w.t.row0 + j * kTile, kv_head,
                               w.t.batch);
            }
            ++fills;
          }
        }
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      const uint32_t id_s = idesc_16bit(kBf16<T>, kTile, 0), id_o = idesc_16bit(kBf16<T>, (p.dim + 15) / 16 * 16, 1);
      const uint32_t el = elect_one();
      int fill = 0, used[2] = {0, 0}, done[2] = {0, 0};  // tiles of queries, and of keys with them, in all items
      bool ok = true;
      for (int k = 0, item = blockIdx.x; ok && item >= 0; item = queue.take(k, failed), ++k) {
        const Pair w(p, item, tiles);
        if (w.first == w.last) continue;
        // scores of query tile i with keys j in `slot`
        const auto ask = [&](int i, int j, int slot) {
          if (j == w.from[i]) ok = ok && warp_wait(&q_full[i], used[i]++ & 1, failed);
          if (!ok) return;
          scores<kCols>(tmem + i * kTile, smem + i * C::kTileBytes, ring + slot * C::kTileBytes, id_s, p.dim, el);
          umma_commit(&s_full[i], el);
          if (j + 1 == w.to[i]) umma_commit(&q_empty[i], el);
        };
        ok = warp_wait(&full[fill % C::kStages], (fill / C::kStages) & 1, failed);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (ok && w.from[i] <= w.first && w.first < w.to[i]) ask(i, w.first, fill % C::kStages);
        if (ok) umma_commit(&empty[fill % C::kStages], el);
        for (int j = w.first; j < w.last && ok; ++j) {
          const int v_slot = (fill + 1) % C::kStages, k_slot = (fill + 2) % C::kStages;
          ok = warp_wait(&full[v_slot], ((fill + 1) / C::kStages) & 1, failed);
          if (!ok) break;
          if (foreign && (j + 1) * kTile > w.t.keys)
            zero_rows<kCols>(ring + v_slot * C::kTileBytes, w.t.keys - j * kTile);
          const bool more = j + 1 < w.last;
          if (more) ok = warp_wait(&full[k_slot], ((fill + 2) / C::kStages) & 1, failed);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (ok && w.from[i] <= j && j < w.to[i]) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                ok = ok && warp_wait(&p_full[i][half], done[i] & 1, failed);
                if (!ok) break;
                tc_fence_after();
                weighted(tmem + 2 * kTile + i * kCols, tmem + i * kTile + half * 32, ring + v_slot * C::kTileBytes, half,
                         id_o, j > w.from[i] || half > 0, el);
              }
              if (ok) umma_commit(&o_done[i], el);
              ++done[i];
            }
            if (ok && more && w.from[i] <= j + 1 && j + 1 < w.to[i]) ask(i, j + 1, k_slot);
          }
          if (ok) {
            umma_commit(&empty[v_slot], el);
            if (more) umma_commit(&empty[k_slot], el);
          }
          fill += 2;
        }
      }
    }
  } else {
    take_registers<kScoreRegisters>();
    const int i = warp / 4;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp % 4) << 21);
    const uint32_t s_at = lanes + i * kTile, o_at = lanes + 2 * kTile + i * kCols;
    const float c = p.scale * kLog2e;
    int done = 0;  // tiles of keys in all items
    bool ok = true;
    Pair w(p, blockIdx.x, tiles);
    for (int k = 0, item = blockIdx.x; ok && item >= 0; ++k) {
      const Tile t = w.t;
      const int head = w.head + i * w.heads_on, first = t.first + i * w.rows_on;
      const int row = first + threadIdx.x % kTile;  // of the sequence
      const int from = i == 0 ? w.from[0] : w.from[1], to = i == 0 ? w.to[0] : w.to[1];
      int low = 0, high = 0, all_low = 0, all_high = 0;
      if (t.found) {
        keys_of(p, t, min(row, t.queries), min(row + 1, t.queries), &low, &high);
        // what every row of the tile sees
        const int last = min(first + kTile, t.queries) - 1;
        int unused;
        if (first <= last) {
          keys_of(p, t, last, last + 1, &all_low, &unused);
          keys_of(p, t, first, first + 1, &unused, &all_high);
        }
      }
      float top = -INFINITY, sum = 0.0f;
      for (int j = from; j < to; ++j, ++done) {
        ok = warp_wait(&s_full[i], done & 1, failed);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[4][32];
        float best[4];
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_ld_32x32b_x32(s_at + q * 32, s[q]);
        tmem_wait_ld(s[0]);
        tmem_wait_ld(s[1]);
#pragma unroll
        for (int q = 2; q < 4; ++q) tmem_ld_32x32b_x32(s_at + q * 32, s[q]);
        const int k0 = j * kTile, a = low - k0, b = high - k0;
        const bool partial = k0 < all_low || k0 + kTile > all_high;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1) {
            tmem_wait_ld(s[2]);
            tmem_wait_ld(s[3]);
          }
          if (partial) {
#pragma unroll
            for (int e = 0; e < 64; ++e)
              if (h * 64 + e < a || h * 64 + e >= b) s[2 * h + e / 32][e % 32] = 0xff800000u;
          }
          // the largest in four chains: one is as long as its 128 latencies
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int at = 2 * h + q / 2, e0 = q % 2 * 16;
            float m = as_float(s[at][e0]);
#pragma unroll
            for (int e = 1; e < 16; ++e) m = fmaxf(m, as_float(s[at][e0 + e]));
            best[q] = h == 0 ? m : fmaxf(best[q], m);
          }
        }
        const float most = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
        if (j == from) {
          top = most;
        } else {
          const bool grow = (most - top) * c > kLag;
          if (__any_sync(kFullMask, grow)) {
            const float next = grow ? most : top, by = grow ? fast_exp2((top - next) * c) : 1.0f;
            sum *= by;
            top = next;
            ok = warp_wait(&o_done[i], (done - 1) & 1, failed);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < kCols; q += 32) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(o_at + q, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(as_float(o[e]) * by);
              tmem_st_32x32b_x32(o_at + q, o);
            }
          }
        }
        const float base = top == -INFINITY ? kRaise<T> : kRaise<T> - top * c;
        float2 sums[4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 64 keys each: the product of the first begins while the others are worked on
          uint32_t w[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int at = h * 64 + 2 * e;
            const float2 x = fma2(make_float2(as_float(s[at / 32][at % 32]), as_float(s[at / 32][at % 32 + 1])), both(c),
                                  both(base));
            const float2 v = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            sums[e % 4] = add2(sums[e % 4], v);
            w[e] = pack2<T>(v.x, v.y);
          }
          tmem_st_32x32b_x32(s_at + h * 32, w);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&p_full[i][h]);
        }
        const float2 s01 = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
        sum += s01.x + s01.y;
      }
      // the next item is looked up while the last products of this one run
      item = ok ? queue.take(k, failed) : -1;
      if (item >= 0) w = Pair(p, item, tiles);
      if (ok && from < to) ok = warp_wait(&o_done[i], (done - 1) & 1, failed);
      tc_fence_after();
      const int64_t at = static_cast<int64_t>(t.batch) * p.length + t.row0 + row;
      const bool write = ok && t.found && row < t.stored, some = low < high;
      const int64_t stride = static_cast<int64_t>(p.heads) * p.dim;
      T* out = static_cast<T*>(p.out) + at * stride + head * p.dim;
      T* rest = p.out2 != nullptr ? static_cast<T*>(p.out2) + at * stride + head * p.dim : nullptr;
      if (from < to)
        store_rows<T, kCols, kTurned>(out, rest, stride, o_at, p.dim, some ? 1.0f / sum : 0.0f, write && some);
      if (write && (from >= to || !some)) {
        zero_row(out, p.dim);
        if (rest != nullptr) zero_row(rest, p.dim);
      }
      if (write)
        p.lse[head * p.rows + at] = some ? top * p.scale + logf(sum) - kRaise<T> * 0.6931471805599453f : -INFINITY;
      __syncwarp();
    }
  }
  finish(tmem, failed, fills, full, C::kStages, &q_full[0], loads[0], &q_full[1], loads[1], queue, asked, &drained);
}

// ------------------------------------------------------------ backward: statistics
// -lse in binary exponents (so that p = 2^(s scale log2 e - it); -inf where
// nothing is seen: p = 0) and -delta of each row and head; for fp16 also the
// norms of dout's rows, 0 where nothing is seen, and of v's, of their finite
// elements.  A lane has 8 columns.  Bound by memory: 117 MB in 23 us, cold.
struct Stats {
  const void* out;
  const void* rest;
  const void* grad;
  const void* v;
  const float* lse;
  float* stats;
  float* grad_norm;
  float* value_norm;
  muon_train_strides grad_stride, v_stride;
  int64_t rows, v_rows;
  int length, keys, heads, kv_heads, dim;
};
constexpr int kStatRows = 2;  // a thread's, in flight together

template <typename T>
__device__ __forceinline__ const T* row_of(const void* x, const muon_train_strides& s, uint32_t row, uint32_t length,
                                           uint32_t head) {
  const uint32_t b = row / length, r = row - b * length;
  return static_cast<const T*>(x) + b * s.batch + r * s.row + head * s.head;
}

// x^2 added to n, where it is a number.
__device__ __forceinline__ float add_square(float x, float n) { return fabsf(x) < INFINITY ? fmaf(x, x, n) : n; }

template <typename T, int kCols>
__global__ void __launch_bounds__(256, 6) stats_kernel(const __grid_constant__ Stats a) {
  constexpr int kLanes = kCols / 8, kGroups = 256 / kLanes;
  begin_kernel();
  const int lane = threadIdx.x % kLanes, dim = a.dim;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups * kStatRows;
  const auto join = [](float v) {  // of a row's lanes
#pragma unroll
    for (int q = kLanes / 2; q > 0; q >>= 1) v += __shfl_xor_sync(kFullMask, v, q, kLanes);
    return v;
  };
  // items are heads of rows; the first of the block is divided in 64 bits, the others' distances in 32
  const uint32_t heads = a.heads, row0 = static_cast<uint32_t>(base / heads),
                 h0 = static_cast<uint32_t>(base - static_cast<int64_t>(row0) * heads);
  uint32_t row[kStatRows], head[kStatRows];
  uint4 o[kStatRows], e[kStatRows], g[kStatRows];
  float l[kStatRows];
#pragma unroll
  for (int u = 0; u < kStatRows; ++u) {
    const uint32_t in_it = h0 + u * kGroups + threadIdx.x / kLanes, down = in_it / heads;
    row[u] = row0 + down;
    head[u] = in_it - down * heads;
    o[u] = e[u] = g[u] = make_uint4(0, 0, 0, 0);
    l[u] = -INFINITY;
    if (row[u] >= a.rows) continue;
    l[u] = a.lse[head[u] * a.rows + row[u]];
    if (lane * 8 >= dim) continue;
    const int64_t at = (row[u] * static_cast<int64_t>(heads) + head[u]) * dim + lane * 8;
    o[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.out) + at);
    if (a.rest != nullptr) e[u] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.rest) + at);
    g[u] = *reinterpret_cast<const uint4*>(row_of<T>(a.grad, a.grad_stride, row[u], a.length, head[u]) + lane * 8);
  }
#pragma unroll
  for (int u = 0; u < kStatRows; ++u) {
    // a row that sees nothing has no gradient, whatever dout holds there
    const bool none = l[u] == -INFINITY;
    float x[8], y[8], z[8], d = 0.0f, n = 0.0f;
    unpack<T>(o[u], x);
    unpack<T>(e[u], y);
    unpack<T>(g[u], z);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      d = fmaf(x[i], z[i], d);
      d = fmaf(y[i], z[i], d);
      if constexpr (!kBf16<T>) n = add_square(z[i], n);
    }
    d = join(d);
    if constexpr (!kBf16<T>) n = join(n);
    if (row[u] < a.rows && lane == 0) {
      const int64_t at = head[u] * a.rows + row[u];
      a.stats[at] = none ? -INFINITY : kRaiseBack<T> - l[u] * kLog2e;
      a.stats[a.heads * a.rows + at] = none ? 0.0f : -d;
      if constexpr (!kBf16<T>) a.grad_norm[row[u] * static_cast<int64_t>(heads) + head[u]] = none ? 0.0f : sqrtf(n);
    }
  }
  if constexpr (!kBf16<T>) {
    const int64_t v_items = a.v_rows * a.kv_heads;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups * kStatRows;
    for (int64_t first = base + threadIdx.x / kLanes; first - threadIdx.x / kLanes < v_items; first += step) {
      uint4 v[kStatRows];
#pragma unroll
      for (int u = 0; u < kStatRows; ++u) {
        const int64_t at = first + u * kGroups;
        v[u] = make_uint4(0, 0, 0, 0);
        if (at >= v_items || lane * 8 >= dim) continue;
        const uint32_t r = static_cast<uint32_t>(at / a.kv_heads);
        const uint32_t h = static_cast<uint32_t>(at - static_cast<int64_t>(r) * a.kv_heads);
        v[u] = *reinterpret_cast<const uint4*>(row_of<T>(a.v, a.v_stride, r, a.keys, h) + lane * 8);
      }
#pragma unroll
      for (int u = 0; u < kStatRows; ++u) {
        float x[8], n = 0.0f;
        unpack<T>(v[u], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) n = add_square(x[i], n);
        n = join(n);
        if (first + u * kGroups < v_items && lane == 0) a.value_norm[first + u * kGroups] = sqrtf(n);
      }
    }
  }
}

// The largest of a warp's values, none below 0, whose bits are ordered as they are.
__device__ __forceinline__ float warp_top(float v) {
  return __uint_as_float(__reduce_max_sync(kFullMask, __float_as_uint(v)));
}

// fp16: the largest |dout| and |delta| of each tile of queries, over the heads
// that share a key head, and the largest |v| of each tile of keys, over the rows
// that count: what others hold reaches nothing.  A block a tile, a row a thread.
__global__ void __launch_bounds__(kTile)
    tops_kernel(const __grid_constant__ Problem p, float2* query_top, float* key_top, int query_tiles, int key_tiles) {
  __shared__ float2 of_warp[kTile / 32];
  begin_kernel();
  const bool queries = blockIdx.y == 0;
  const int rows = queries ? p.length : p.keys, tiles = queries ? query_tiles : key_tiles;
  if (blockIdx.x >= static_cast<uint32_t>(tiles) * p.kv_heads) return;
  int kv_head;
  const Tile t = find_tile(p, blockIdx.x, rows, p.kv_heads, kTileShift, tiles, false, &kv_head);
  if (!t.found) return;
  const int row = t.first + threadIdx.x;
  const int64_t at = static_cast<int64_t>(t.batch) * rows + t.row0 + row;
  float norm = 0.0f, delta = 0.0f;
  if (!queries) {
    if (row < t.keys) norm = p.value_norm[at * p.kv_heads + kv_head];
  } else if (row < t.queries) {
    const int group = p.heads / p.kv_heads;
#pragma unroll 4
    for (int head = kv_head * group; head < (kv_head + 1) * group; ++head) {
      norm = fmaxf(norm, p.grad_norm[at * p.heads + head]);
      const float d = fabsf(p.stats[(p.heads + head) * p.rows + at]);
      if (d < INFINITY) delta = fmaxf(delta, d);
    }
  }
  norm = warp_top(norm);
  delta = warp_top(delta);
  if (threadIdx.x % 32 == 0) of_warp[threadIdx.x / 32] = make_float2(norm, delta);
  __syncthreads();
  if (threadIdx.x > 0) return;
  for (int w = 1; w < kTile / 32; ++w) norm = fmaxf(norm, of_warp[w].x), delta = fmaxf(delta, of_warp[w].y);
  const int64_t to = tile_slot(p, t, rows, tiles, kv_head) + (t.first >> kTileShift);
  if (queries)
    query_top[to] = make_float2(norm, delta);
  else
    key_top[to] = norm;
}

// The binary exponent that brings ds, of at most `bound` (|dp| <= |dout| |v|), to
// 2^14 to 2^15.  A ds below fp16's normal range is then off by half of its last
// place, 2^-25, which is 2^-39 of the bound or less.  Query rows have one each, of
// the row's own |dout| and |delta| and the largest |v| of the keys' tiles; keys one
// each, of the key's |v| and the largest |dout| and |delta| of the queries' tiles:
// what is large elsewhere takes nothing from them.  (One for the whole call, of
// its largest elements, lost up to all of dq and dk beside large padding or
// another sequence 10^3 as large.  The bounds cost 8191 packed tokens, 16 heads of
// 64, window 512: 169 -> 178 us; 4 x 4096, 16 over 4: 981 -> 997.)
__device__ __forceinline__ int ds_exponent(float bound) {
  return bound > 0.0f && bound < INFINITY ? clamp_int(14 - ilogbf(bound), -60, 100) : 0;
}

// ------------------------------------------------------------ backward: keys and values
template <int kCols>
struct KeyGrads {
  static constexpr int kTileBytes = kTile * kCols * 2;
  static constexpr int kStages = kCols == 128 ? 5 : 8;  // tiles
  static constexpr int kBytes = (2 + kStages) * kTileBytes + 1024;
};
// What the kernel for keys has beside the tiles; in dynamic shared memory, so
// that the tiles begin on their boundary without room to move them there: there
// is none (232448 bytes, of which seven tiles take 229376).
struct KeyShared {
  Items queue;
  uint64_t kv_full, kv_empty, s_full, dp_full, p_done[2], ds_done[2], finished, drained;
  uint64_t stat_full[2], stat_read[2], full[8], empty[8];
  __align__(16) float stat[2][2][kTile];  // of two tiles of queries: -lse and -delta
  uint32_t tmem_slot;
  int failed_word;
};

// An item is one tile of keys with all query heads that share them.
struct Keys {
  int kv_head;
  Tile t;
  int from, to, per;  // tiles of queries, of one head

  __device__ __forceinline__ Keys(const Problem& p, int item, int tiles) {
    t = find_tile(p, item, p.keys, p.kv_heads, kTileShift, tiles, false, &kv_head);
    int low = 0, high = 0;
    if (t.found) queries_of(p, t, min(t.first, t.keys), min(t.first + kTile, t.keys), &low, &high);
    from = low / kTile;
    to = low < high ? (high + kTile - 1) / kTile : from;
    per = to - from;
  }
};

// Scores stand the other way round, a key a thread: p^T and ds^T are left
// operands as they are.  The warps 0-3 take queries 0 to 63 of each tile, 4-7 the
// others.  While the scores of the next tile are computed ds is worked on, while
// dp is computed the next p.  4096 both ways, 37 heads of 128: 492 us alone, with
// the tensor pipe busy in 67% of the cycles.
template <typename T, int kCols>
__global__ void __launch_bounds__(kThreads, 1)
    key_grad_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                    const __grid_constant__ Problem p, int tiles) {
  using C = KeyGrads<kCols>;
  extern __shared__ __align__(1024) uint8_t dynamic[];
  uint8_t* smem = dynamic;
  uint8_t* tile_k = smem;
  uint8_t* tile_v = smem + C::kTileBytes;
  uint8_t* ring = smem + 2 * C::kTileBytes;
  KeyShared& m = *reinterpret_cast<KeyShared*>(smem + (2 + C::kStages) * C::kTileBytes);
  volatile int* failed = &m.failed_word;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    mbar_init(&m.kv_full, 1);
    mbar_init(&m.kv_empty, 1);
    mbar_init(&m.s_full, 1);
    mbar_init(&m.dp_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m.p_done[i], 128);
      mbar_init(&m.ds_done[i], 128);
    }
    mbar_init(&m.finished, 1);
    mbar_init(&m.drained, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&m.stat_full[i], 32);
      mbar_init(&m.stat_read[i], 8);
    }
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&m.full[i], 1);
      mbar_init(&m.empty[i], 1);
    }
    m.queue.init();
    fence_mbar_init();
    m.failed_word = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(&m.tmem_slot, kTmemColumns);
  tc_fence_before();
  begin_kernel();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = m.tmem_slot, tmem_s = tmem, tmem_dp = tmem + kTile, tmem_dv = tmem + 2 * kTile,
                 tmem_dk = tmem + 2 * kTile + kCols;
  const int group = p.heads / p.kv_heads;
  const bool foreign = p.offsets != nullptr || p.lengths != nullptr;
  // `g` counts the tiles of queries of all items: fill 2 g of the ring is the queries of one, 2 g + 1 their dout

  int fills = 0, loads = 0, asked = 0;
  if (warp >= kLoadWarp) {
    give_registers<kOtherRegisters>();
    if (warp == kLoadWarp) {
      bool ok = true;
      int g = 0;
      for (int item = blockIdx.x; ok && item >= 0; item = m.queue.next(&asked, failed)) {
        const Keys w(p, item, tiles);
        if (w.per == 0) continue;
        if (loads > 0) ok = warp_wait(&m.kv_empty, (loads - 1) & 1, failed);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&m.kv_full, 2 * C::kTileBytes);
          load_tile<kCols>(tile_k, &map_k, &m.kv_full, w.t.row0 + w.t.first, w.kv_head, w.t.batch);
          load_tile<kCols>(tile_v, &map_v, &m.kv_full, w.t.row0 + w.t.first, w.kv_head, w.t.batch);
        }
        ++loads;
        int head = w.kv_head * group, i = w.from;
        for (int it = 0; it < w.per * group && ok; ++it, ++g) {
          const int row = w.t.row0 + i * kTile;
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const int s = fills % C::kStages;
            if (fills >= C::kStages) ok = ok && warp_wait(&m.empty[s], (fills / C::kStages - 1) & 1, failed);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&m.full[s], C::kTileBytes);
              load_tile<kCols>(ring + s * C::kTileBytes, which ? &map_g : &map_q, &m.full[s], row - p.blind, head, w.t.batch);
            }
            ++fills;
            if (which == 0) {
              if (g >= 2) ok = warp_wait(&m.stat_read[g % 2], (g / 2 - 1) & 1, failed);
              if (!ok) break;
              const int64_t from = head * p.rows + static_cast<int64_t>(w.t.batch) * p.length + row;
#pragma unroll
              for (int e = lane; e < kTile; e += 32) {
                const bool counts = i * kTile + e < w.t.queries;
                m.stat[g % 2][0][e] = counts ? p.stats[from + e] : -INFINITY;
                m.stat[g % 2][1][e] = counts ? p.stats[p.heads * p.rows + from + e] : 0.0f;
              }
              mbar_arrive(&m.stat_full[g % 2]);
            }
          }
          if (++i == w.to) i = w.from, ++head;
        }
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      const uint32_t id_s = idesc_16bit(kBf16<T>, kTile, 0), id_o = idesc_16bit(kBf16<T>, (p.dim + 15) / 16 * 16, 1);
      const uint32_t el = elect_one();
      bool ok = true;
      int g = 0, used = 0;
      for (int at = 0, item = blockIdx.x; ok && item >= 0; item = m.queue.take(at, failed), ++at) {
        const Keys w(p, item, tiles);
        const int n = w.per * group;
        if (n == 0) continue;
        // waits for fill `f`, a tile from query `first` on, and clears what is not the sequence's
        const auto arrived = [&](int f, int first) {
          if (!warp_wait(&m.full[f % C::kStages], (f / C::kStages) & 1, failed)) return false;
          if (foreign && w.t.queries - first < kTile)
            zero_rows<kCols>(ring + f % C::kStages * C::kTileBytes, w.t.queries - first);
          return true;
        };
        ok = warp_wait(&m.kv_full, used++ & 1, failed) && arrived(2 * g, w.from * kTile);
        if (!ok) break;
        scores<kCols>(tmem_s, tile_k, ring + 2 * g % C::kStages * C::kTileBytes, id_s, p.dim, el);
        umma_commit(&m.s_full, el);
        ok = arrived(2 * g + 1, w.from * kTile);
        if (!ok) break;
        scores<kCols>(tmem_dp, tile_v, ring + (2 * g + 1) % C::kStages * C::kTileBytes, id_s, p.dim, el);
        umma_commit(&m.dp_full, el);
        if (n == 1) umma_commit(&m.kv_empty, el);
        int next = w.from + 1 == w.to ? w.from : w.from + 1;  // the next iteration's tile of queries
        for (int it = 0; it < n && ok; ++it, ++g) {
          const int q_slot = 2 * g % C::kStages, g_slot = (2 * g + 1) % C::kStages;
          const bool more = it + 1 < n;
          if (more) ok = arrived(2 * g + 2, next * kTile);  // there before p is, as a rule
          if (!ok) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && warp_wait(&m.p_done[h], g & 1, failed);
            if (!ok) break;
            tc_fence_after();
            weighted(tmem_dv, tmem_s + h * 64, ring + g_slot * C::kTileBytes, h, id_o, it > 0 || h > 0, el);
          }
          if (!ok) break;
          if (more) {
            scores<kCols>(tmem_s, tile_k, ring + (2 * g + 2) % C::kStages * C::kTileBytes, id_s, p.dim, el);
            umma_commit(&m.s_full, el);
          }
          umma_commit(&m.empty[g_slot], el);
          if (more) ok = arrived(2 * g + 3, next * kTile);
          if (!ok) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && warp_wait(&m.ds_done[h], g & 1, failed);
            if (!ok) break;
            tc_fence_after();
            weighted(tmem_dk, tmem_dp + h * 64, ring + q_slot * C::kTileBytes, h, id_o, it > 0 || h > 0, el);
          }
          if (!ok) break;
          if (more) {
            scores<kCols>(tmem_dp, tile_v, ring + (2 * g + 3) % C::kStages * C::kTileBytes, id_s, p.dim, el);
            umma_commit(&m.dp_full, el);
            if (it + 2 == n) umma_commit(&m.kv_empty, el);
            if (++next == w.to) next = w.from;
          } else {
            umma_commit(&m.finished, el);
          }
          umma_commit(&m.empty[q_slot], el);
        }
      }
    }
  } else {
    take_registers<kScoreRegisters>();
    const int w = warp / 4;  // both halves have all keys
    const uint32_t lanes = static_cast<uint32_t>(warp % 4) << 21;
    const float c = p.scale * kLog2e;
    bool ok = true;
    int g = 0, used = 0;
    const auto factor_of = [&](const Keys& item) {
      if constexpr (kBf16<T>) return 1.0f;
      const float2* top = p.query_top + tile_slot(p, item.t, p.length, tiles, item.kv_head) + item.from;
      float grad = 0.0f, delta = 0.0f, value = 0.0f;
      const int row = item.t.first + threadIdx.x % 128;
      if (item.per > 0 && row < item.t.keys)
        value = p.value_norm[(static_cast<int64_t>(item.t.batch) * p.keys + item.t.row0 + row) * p.kv_heads + item.kv_head];
      for (int x = lane; x < item.per; x += 32) {
        const float2 most = top[x];
        grad = fmaxf(grad, most.x);
        delta = fmaxf(delta, most.y);
      }
      return scalbnf(1.0f, ds_exponent(warp_top(grad) * value + warp_top(delta)));
    };
    Keys next(p, blockIdx.x, tiles);
    float next_factor = factor_of(next);
    for (int k = 0, number = blockIdx.x; ok && number >= 0; ++k) {
      const Keys item = next;
      const Tile& t = item.t;
      const float factor = next_factor, raise = factor * (kBf16<T> ? 1.0f : 0x1p-10f);
      const int row = t.first + threadIdx.x % 128, n = item.per * group;  // the thread's key
      int mine_low = 0, mine_high = 0, all_low = 0, all_high = 0;
      if (t.found) {
        queries_of(p, t, min(row, t.keys), min(row + 1, t.keys), &mine_low, &mine_high);
        const int j1 = min(t.first + kTile, t.keys);
        int unused;
        if (t.first < j1) {
          queries_of(p, t, j1 - 1, j1, &all_low, &unused);
          queries_of(p, t, t.first, t.first + 1, &unused, &all_high);
        }
      }
      int i = item.from;
      for (int it = 0; it < n; ++it, ++g) {
        const int first = i * kTile;
        if (++i == item.to) i = item.from;
        const bool partial = first < all_low || first + kTile > all_high;
        const int a = mine_low - first - w * 64, b = mine_high - first - w * 64;
        ok = warp_wait(&m.stat_full[g % 2], (g / 2) & 1, failed);
        if (!ok) break;
        // the statistics are in registers before the scores are there: loads from shared memory wait behind the products'
        float4 l[16];
        const float4* l4 = reinterpret_cast<const float4*>(&m.stat[g % 2][0][w * 64]);
#pragma unroll
        for (int e = 0; e < 16; ++e) l[e] = l4[e];
        ok = warp_wait(&m.s_full, g & 1, failed);
        if (!ok) break;
        tc_fence_after();
        uint32_t x[2][32];
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_ld_32x32b_x32(tmem_s + lanes + w * 64 + q * 32, x[q]);
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_wait_ld(x[q]);
        uint32_t packed[32];
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 u = fma2(make_float2(as_float(x[e / 32][e % 32]), as_float(x[e / 32][e % 32 + 1])), both(c),
                                e % 4 == 0 ? make_float2(l[e / 4].x, l[e / 4].y) : make_float2(l[e / 4].z, l[e / 4].w));
          x[e / 32][e % 32] = __float_as_uint(fast_exp2(u.x));
          x[e / 32][e % 32 + 1] = __float_as_uint(fast_exp2(u.y));
        }
        if (partial) {
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (e < a || e >= b) x[e / 32][e % 32] = 0;
        }
#pragma unroll
        for (int e = 0; e < 64; e += 2)
          packed[e / 2] = pack2<T>(as_float(x[e / 32][e % 32]), as_float(x[e / 32][e % 32 + 1]));
        tmem_st_32x32b_x32(tmem_s + lanes + w * 64, packed);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&m.p_done[w]);

        const float4* d4 = reinterpret_cast<const float4*>(&m.stat[g % 2][1][w * 64]);
#pragma unroll
        for (int e = 0; e < 16; ++e) l[e] = d4[e];
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.stat_read[g % 2]);
        ok = warp_wait(&m.dp_full, g & 1, failed);
        if (!ok) break;
        tc_fence_after();
        uint32_t y[2][32];
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_ld_32x32b_x32(tmem_dp + lanes + w * 64 + q * 32, y[q]);
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_wait_ld(y[q]);
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          float2 v = add2(make_float2(as_float(y[e / 32][e % 32]), as_float(y[e / 32][e % 32 + 1])),
                          e % 4 == 0 ? make_float2(l[e / 4].x, l[e / 4].y) : make_float2(l[e / 4].z, l[e / 4].w));
          if constexpr (!kBf16<T>) v = mul2(v, both(raise));
          v = mul2(v, make_float2(as_float(x[e / 32][e % 32]), as_float(x[e / 32][e % 32 + 1])));
          y[e / 32][e % 32] = __float_as_uint(v.x);
          y[e / 32][e % 32 + 1] = __float_as_uint(v.y);
        }
        if (partial) {  // p is 0 there, but dp may be no number
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (e < a || e >= b) y[e / 32][e % 32] = 0;
        }
#pragma unroll
        for (int e = 0; e < 64; e += 2)
          packed[e / 2] = pack2<T>(as_float(y[e / 32][e % 32]), as_float(y[e / 32][e % 32 + 1]));
        tmem_st_32x32b_x32(tmem_dp + lanes + w * 64, packed);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&m.ds_done[w]);
      }
      number = ok ? m.queue.take(k, failed) : -1;
      if (number >= 0) {
        next = Keys(p, number, tiles);
        next_factor = factor_of(next);
      }
      if (ok && n > 0) ok = warp_wait(&m.finished, used++ & 1, failed);
      tc_fence_after();
      // the first half writes dv, the other dk
      const int64_t at = static_cast<int64_t>(t.batch) * p.keys + t.row0 + row;
      T* grad = static_cast<T*>(w == 0 ? p.out2 : p.out) + (at * p.kv_heads + item.kv_head) * p.dim;
      const bool write = ok && t.found && row < t.stored, some = mine_low < mine_high;
      const float by = w == 0 ? (kBf16<T> ? 1.0f : 0x1p-10f) : p.scale / factor;
      if (n > 0)
        store_rows<T, kCols, kCols == 128>(grad, nullptr, static_cast<int64_t>(p.kv_heads) * p.dim,
                                           (w == 0 ? tmem_dv : tmem_dk) + lanes, p.dim, by, write && some);
      if (write && (n == 0 || !some)) zero_row(grad, p.dim);
      __syncwarp();
    }
  }
  finish(tmem, failed, fills, m.full, C::kStages, &m.kv_full, loads, nullptr, 0, m.queue, asked, &m.drained);
}

// ------------------------------------------------------------ backward: queries
// An item is one tile of queries.
struct Queries {
  int head;
  Tile t;
  int from, to;  // tiles of keys

  __device__ __forceinline__ Queries(const Problem& p, int item, int tiles) {
    t = find_tile(p, item, p.length, p.heads, kTileShift, tiles, true, &head);
    int low = 0, high = 0;
    if (t.found) keys_of(p, t, min(t.first, t.queries), min(t.first + kTile, t.queries), &low, &high);
    from = low / kTile;
    to = low < high ? (high + kTile - 1) / kTile : from;
  }
};

// Two tiles of scores in tensor memory, one of dp: the products of the next keys
// run while ds is worked on, which takes the place of its scores.  Half of the
// warps may be done with the next ds before the product with the present one has
// been issued, so those barriers are two.  4096 both ways, 37 heads of 128: 447 us
// alone, tensor pipe 53%.
template <typename T, int kCols>
__global__ void __launch_bounds__(kThreads, 1)
    query_grad_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                      const __grid_constant__ Problem p, int tiles) {
  using C = KeyGrads<kCols>;
  extern __shared__ __align__(1024) uint8_t dynamic[];
  __shared__ uint64_t q_full, q_empty, s_full[2], dp_full, dp_read, ds_done[2][2], finished, drained;
  __shared__ uint64_t full[C::kStages], empty[C::kStages];
  __shared__ Items queue;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed_word;
  volatile int* failed = &failed_word;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dynamic) + 1023) & ~uintptr_t{1023});
  uint8_t* tile_q = smem;
  uint8_t* tile_g = smem + C::kTileBytes;
  uint8_t* ring = smem + 2 * C::kTileBytes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(&dp_full, 1);
    mbar_init(&dp_read, 256);
    for (int i = 0; i < 4; ++i) mbar_init(&ds_done[i / 2][i % 2], 128);
    mbar_init(&finished, 1);
    mbar_init(&drained, 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    queue.init();
    fence_mbar_init();
    failed_word = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_slot, kTmemColumns);
  tc_fence_before();
  begin_kernel();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, tmem_dp = tmem + 2 * kTile, tmem_dq = tmem + 3 * kTile;
  const bool foreign = p.offsets != nullptr || p.lengths != nullptr;
  // `g` counts the tiles of keys of all items: fill 2 g of the ring is the keys of one, 2 g + 1 their values

  int fills = 0, loads = 0, asked = 0;
  if (warp >= kLoadWarp) {
    give_registers<kOtherRegisters>();
    if (warp == kLoadWarp) {
      bool ok = true;
      for (int item = blockIdx.x; ok && item >= 0; item = queue.next(&asked, failed)) {
        const Queries w(p, item, tiles);
        if (w.from == w.to) continue;
        const int kv_head = w.head / (p.heads / p.kv_heads);
        if (loads > 0) ok = warp_wait(&q_empty, (loads - 1) & 1, failed);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full, 2 * C::kTileBytes);
          load_tile<kCols>(tile_q, &map_q, &q_full, w.t.row0 + w.t.first, w.head, w.t.batch);
          load_tile<kCols>(tile_g, &map_g, &q_full, w.t.row0 + w.t.first, w.head, w.t.batch);
        }
        ++loads;
        for (int j = w.from; j < w.to && ok; ++j) {
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const int s = fills % C::kStages;
            if (fills >= C::kStages) ok = ok && warp_wait(&empty[s], (fills / C::kStages - 1) & 1, failed);
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&full[s], C::kTileBytes);
              load_tile<kCols>(ring + s * C::kTileBytes, which ? &map_v : &map_k, &full[s], w.t.row0 + j * kTile, kv_head,
                               w.t.batch);
            }
            ++fills;
          }
        }
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      const uint32_t id_s = idesc_16bit(kBf16<T>, kTile, 0), id_o = idesc_16bit(kBf16<T>, (p.dim + 15) / 16 * 16, 1);
      const uint32_t el = elect_one();
      bool ok = true;
      int g = 0, used = 0;
      for (int at = 0, item = blockIdx.x; ok && item >= 0; item = queue.take(at, failed), ++at) {
        const Queries w(p, item, tiles);
        const int n = w.to - w.from;
        if (n == 0) continue;
        // scores of this item's iteration `it`; its keys' rows that are not the sequence's are cleared: ds is
        // multiplied with them
        const auto ask = [&](int it, int number) {
          const int f = 2 * number, valid = w.t.keys - (w.from + it) * kTile;
          uint8_t* tile = ring + f % C::kStages * C::kTileBytes;
          if (!warp_wait(&full[f % C::kStages], (f / C::kStages) & 1, failed)) return false;
          if (foreign && valid < kTile) zero_rows<kCols>(tile, valid);
          scores<kCols>(tmem + (number & 1) * kTile, tile_q, tile, id_s, p.dim, el);
          umma_commit(&s_full[number & 1], el);
          return true;
        };
        const auto ask_dp = [&](int it, int number) {
          const int f = 2 * number + 1;
          if (!warp_wait(&full[f % C::kStages], (f / C::kStages) & 1, failed)) return false;
          // the dp before has been read
          if (number > 0 && !warp_wait(&dp_read, (number - 1) & 1, failed)) return false;
          tc_fence_after();
          scores<kCols>(tmem_dp, tile_g, ring + f % C::kStages * C::kTileBytes, id_s, p.dim, el);
          umma_commit(&dp_full, el);
          umma_commit(&empty[f % C::kStages], el);
          if (it + 1 == n) umma_commit(&q_empty, el);
          return true;
        };
        ok = warp_wait(&q_full, used++ & 1, failed) && ask(0, g) && ask_dp(0, g);
        for (int it = 0; it < n && ok; ++it, ++g) {
          const bool more = it + 1 < n;
          if (more) ok = ask(it + 1, g + 1) && ask_dp(it + 1, g + 1);
          if (!ok) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ok = ok && warp_wait(&ds_done[h][g & 1], (g / 2) & 1, failed);
            if (!ok) break;
            tc_fence_after();
            weighted(tmem_dq, tmem + (g & 1) * kTile + h * 64, ring + 2 * g % C::kStages * C::kTileBytes, h, id_o,
                     it > 0 || h > 0, el);
          }
          if (!ok) break;
          umma_commit(&empty[2 * g % C::kStages], el);
          if (!more) umma_commit(&finished, el);
        }
      }
    }
  } else {
    take_registers<kScoreRegisters>();
    const int w = warp / 4;  // both halves have all queries
    const uint32_t lanes = static_cast<uint32_t>(warp % 4) << 21;
    const float c = p.scale * kLog2e;
    bool ok = true;
    int g = 0, used = 0;
    // the row's -lse, with ds's factor, and -delta; the factor's exponent
    float next_lse, next_delta;
    int next_exponent;
    const auto look_up = [&](const Queries& item) {
      next_lse = -INFINITY, next_delta = 0.0f, next_exponent = 0;
      const int64_t at = static_cast<int64_t>(item.t.batch) * p.length + item.t.row0 + item.t.first + threadIdx.x % 128;
      const bool counts = item.t.found && item.t.first + static_cast<int>(threadIdx.x % 128) < item.t.queries;
      if (counts) {
        next_lse = p.stats[item.head * p.rows + at];
        next_delta = p.stats[(p.heads + item.head) * p.rows + at];
      }
      if constexpr (!kBf16<T>) {
        const float* top = p.key_top + tile_slot(p, item.t, p.keys, tiles, item.head / (p.heads / p.kv_heads)) + item.from;
        const float grad = counts ? p.grad_norm[at * p.heads + item.head] : 0.0f;
        float value = 0.0f;
        for (int x = lane; x < item.to - item.from; x += 32) value = fmaxf(value, top[x]);
        next_exponent = ds_exponent(grad * warp_top(value) + fabsf(next_delta));
        next_lse += static_cast<float>(next_exponent) - kRaiseBack<T>;
      }
    };
    Queries next(p, blockIdx.x, tiles);
    look_up(next);
    for (int k = 0, number = blockIdx.x; ok && number >= 0; ++k) {
      const Queries item = next;
      const Tile& t = item.t;
      const float lse = next_lse, delta = next_delta;
      const int exponent = next_exponent;
      const int row = t.first + threadIdx.x % 128, n = item.to - item.from;
      int mine_low = 0, mine_high = 0, all_low = 0, all_high = 0;
      if (t.found) {
        keys_of(p, t, min(row, t.queries), min(row + 1, t.queries), &mine_low, &mine_high);
        const int i1 = min(t.first + kTile, t.queries);
        int unused;
        if (t.first < i1) {
          keys_of(p, t, i1 - 1, i1, &all_low, &unused);
          keys_of(p, t, t.first, t.first + 1, &unused, &all_high);
        }
      }
      const int64_t at = static_cast<int64_t>(t.batch) * p.length + t.row0 + row;
      for (int it = 0; it < n; ++it, ++g) {
        const int first = (item.from + it) * kTile;
        const bool partial = first < all_low || first + kTile > all_high;
        const int a = mine_low - first - w * 64, b = mine_high - first - w * 64;
        const uint32_t s_at = tmem + (g & 1) * kTile + lanes + w * 64;
        ok = warp_wait(&s_full[g & 1], (g / 2) & 1, failed);
        if (!ok) break;
        tc_fence_after();
        uint32_t x[2][32], y[2][32];
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_ld_32x32b_x32(s_at + q * 32, x[q]);
        ok = warp_wait(&dp_full, g & 1, failed);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_ld_32x32b_x32(tmem_dp + lanes + w * 64 + q * 32, y[q]);
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_wait_ld(x[q]);
#pragma unroll
        for (int q = 0; q < 2; ++q) tmem_wait_ld(y[q]);
        tc_fence_before();
        mbar_arrive(&dp_read);
        uint32_t packed[32];
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float2 u = fma2(make_float2(as_float(x[e / 32][e % 32]), as_float(x[e / 32][e % 32 + 1])), both(c), both(lse));
          float2 v = add2(make_float2(as_float(y[e / 32][e % 32]), as_float(y[e / 32][e % 32 + 1])), both(delta));
          v = mul2(v, make_float2(fast_exp2(u.x), fast_exp2(u.y)));
          y[e / 32][e % 32] = __float_as_uint(v.x);
          y[e / 32][e % 32 + 1] = __float_as_uint(v.y);
        }
        if (partial) {
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (e < a || e >= b) y[e / 32][e % 32] = 0;
        }
#pragma unroll
        for (int e = 0; e < 64; e += 2)
          packed[e / 2] = pack2<T>(as_float(y[e / 32][e % 32]), as_float(y[e / 32][e % 32 + 1]));
        tmem_st_32x32b_x32(s_at, packed);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ds_done[w][g & 1]);
      }
      number = ok ? queue.take(k, failed) : -1;
      if (number >= 0) {
        next = Queries(p, number, tiles);
        look_up(next);
      }
      if (ok && n > 0) ok = warp_wait(&finished, used++ & 1, failed);
      tc_fence_after();
      if (w == 0) {
        T* grad = static_cast<T*>(p.out) + (at * p.heads + item.head) * p.dim;
        const bool write = ok && t.found && row < t.stored, some = mine_low < mine_high;
        if (n > 0)
          store_rows<T, kCols, kCols == 128>(grad, nullptr, static_cast<int64_t>(p.heads) * p.dim, tmem_dq + lanes, p.dim,
                                             scalbnf(p.scale, -exponent), write && some);
        if (write && (n == 0 || !some)) zero_row(grad, p.dim);
      }
      __syncwarp();
    }
  }
  finish(tmem, failed, fills, full, C::kStages, &q_full, loads, nullptr, 0, queue, asked, &drained);
}

// ------------------------------------------------------------ host side
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static std::atomic<EncodeTiled> known{nullptr};
  EncodeTiled fn = known.load(std::memory_order_relaxed);
  if (fn != nullptr) return fn;
  void* f = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
      q == cudaDriverEntryPointSuccess)
    fn = reinterpret_cast<EncodeTiled>(f);
  known.store(fn, std::memory_order_relaxed);
  return fn;
}

// [dim, rows, heads, batch] in boxes of 64 columns of 128 rows; what is outside
// reads as zeros.
int encode(CUtensorMap* map, const void* base, const muon_train_strides& s, int64_t rows, int64_t heads, int64_t batch,
           int64_t dim, int dtype) {
  const EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return MUON_POLAR_ERR_DRIVER;
  // the stride of an axis of one element is never used, but has to be a legal one
  const auto stride = [](int64_t n, int64_t v) { return static_cast<cuuint64_t>(n > 1 ? v * 2 : 16); };
  const cuuint64_t sizes[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads),
                               static_cast<cuuint64_t>(batch)};
  const cuuint64_t strides[3] = {stride(rows, s.row), stride(heads, s.head), stride(batch, s.batch)};
  const cuuint32_t box[4] = {64, kTile, 1, 1}, step[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, dtype == MUON_TRAIN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        4, const_cast<void*>(base), sizes, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MUON_POLAR_OK : MUON_POLAR_ERR_TENSOR_MAP;
}

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
  if (a->offsets != nullptr && (a->lengths != nullptr || a->batch != 1 || a->sequences < 0 || a->sequences > kMost))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  // tiles times heads number the blocks
  const int64_t most = (a->length > a->keys ? a->length : a->keys) / kTile + 1;
  if ((most * a->batch + (a->offsets != nullptr ? a->sequences + 2 : 0)) * a->heads >= (int64_t{1} << 31))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}
bool strided(const void* p, const muon_train_strides& s, int64_t batch, int64_t rows, int64_t heads) {
  const auto fits = [](int64_t n, int64_t stride) {
    return n <= 1 || (stride >= 8 && stride % 8 == 0 && stride < (int64_t{1} << 38));
  };
  return p != nullptr && aligned16(p) && fits(batch, s.batch) && fits(rows, s.row) && fits(heads, s.head);
}
int check_forward(const muon_train_attention_args& a) {
  if (a.batch * a.length > 0 && !strided(a.q, a.q_stride, a.batch, a.length, a.heads)) return MUON_POLAR_ERR_ALIGNMENT;
  if (a.batch * a.keys > 0 && (!strided(a.k, a.k_stride, a.batch, a.keys, a.kv_heads) ||
                               !strided(a.v, a.v_stride, a.batch, a.keys, a.kv_heads)))
    return MUON_POLAR_ERR_ALIGNMENT;
  if (a.batch * a.length > 0 &&
      (a.out == nullptr || !aligned16(a.out) || !aligned16(a.out_rest) || a.lse == nullptr))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return MUON_POLAR_OK;
}

// Tiles of `size` rows of all sequences, at most.
int64_t tiles_of(const muon_train_attention_args& a, int64_t rows, int64_t size) {
  if (a.offsets != nullptr) return rows / size + a.sequences + 2;
  return a.batch * ((rows + size - 1) / size);
}

// A backward call's workspace: its arrays' first elements, in floats.
struct Workspace {
  int64_t stats, query_top, grad_norm, value_norm, key_top, end;
};
Workspace workspace_of(const muon_train_attention_args& a) {
  const bool half = a.dtype == MUON_TRAIN_F16;
  const int64_t rows = a.heads * a.batch * a.length;
  Workspace w;
  w.stats = 0;
  w.query_top = w.stats + 2 * rows;  // pairs
  w.grad_norm = w.query_top + (half ? 2 * a.kv_heads * tiles_of(a, a.length, kTile) : 0);
  w.value_norm = w.grad_norm + (half ? rows : 0);
  w.key_top = w.value_norm + (half ? a.kv_heads * a.batch * a.keys : 0);
  w.end = w.key_top + (half ? a.kv_heads * tiles_of(a, a.keys, kTile) : 0);
  return w;
}

struct Maps {
  CUtensorMap q, k, v;
};
int encode_inputs(const muon_train_attention_args& a, Maps* m) {
  // a thread that has made no CUDA call yet (autograd's) has no context, which the encoder needs
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  int rc = encode(&m->q, a.q, a.q_stride, a.length, a.heads, a.batch, a.dim, a.dtype);
  // without keys no tile of them is loaded: any legal map will do
  if (a.keys == 0) {
    m->k = m->v = m->q;
    return rc;
  }
  if (rc == MUON_POLAR_OK) rc = encode(&m->k, a.k, a.k_stride, a.keys, a.kv_heads, a.batch, a.dim, a.dtype);
  if (rc == MUON_POLAR_OK) rc = encode(&m->v, a.v, a.v_stride, a.keys, a.kv_heads, a.batch, a.dim, a.dtype);
  return rc;
}

Problem problem_of(const muon_train_attention_args& a) {
  Problem p{};
  p.lse = a.lse;
  p.lengths = a.lengths;
  p.offsets = a.offsets;
  p.rows = a.batch * a.length;
  p.length = static_cast<int>(a.length);
  p.keys = static_cast<int>(a.keys);
  p.heads = static_cast<int>(a.heads);
  p.kv_heads = static_cast<int>(a.kv_heads);
  p.dim = static_cast<int>(a.dim);
  p.sequences = static_cast<int>(a.sequences);
  p.batch = static_cast<int>(a.batch);
  // no two places are further apart than there are queries or keys
  const int64_t span = a.length > a.keys ? a.length : a.keys;
  p.window = a.window >= span ? 0 : static_cast<int>(a.window);
  p.causal = a.causal != 0;
  p.scale = a.scale;
  return p;
}

// Lets a kernel have its shared memory, and checks once that it is launched with
// the registers that its warpgroups share out among them, or it would wait for
// them forever.
template <auto kKernel>
int prepare(size_t bytes) {
  static std::atomic<bool> checked{false};
  if (!checked.load(std::memory_order_relaxed)) {
    cudaFuncAttributes attributes;
    const cudaError_t e = cudaFuncGetAttributes(&attributes, kKernel);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (attributes.numRegs != kLaunchRegisters) return MUON_POLAR_ERR_UNSUPPORTED_DEVICE;
    checked.store(true, std::memory_order_relaxed);
  }
  return allow_smem<kKernel>(bytes);
}

// Heads, of all batch entries, of a section: as many as stay in L2 together
// with `bytes` of streamed tiles each, but enough for a few items a block, so
// that a section's large items do not come at the end of all.  8192 keys both
// ways, 32 heads of 4 MB: backward 3400 us with 8 heads a section, 3600 with 16;
// 37 heads of 4096 causal, 2 MB each: forward 190 us, 212 with one round of the
// blocks, and a head at a time 366 us where 64 heads together took 301.
constexpr int64_t kSectionBytes = int64_t{32} << 20;
constexpr int kSectionRounds = 2;
int section_of(int64_t heads, int64_t bytes, int64_t tiles, int* section) {
  int sms = 0;
  const int rc = sm_count(&sms);
  int64_t n = kSectionBytes / (bytes > 0 ? bytes : 1);
  const int64_t least = (kSectionRounds * static_cast<int64_t>(sms) + tiles - 1) / (tiles > 0 ? tiles : 1);
  n = n > least ? n : least;
  n = n < 1 ? 1 : n;
  const int64_t sections = (heads + n - 1) / n;  // of about the same size
  *section = static_cast<int>((heads + sections - 1) / sections);
  return rc;
}

template <typename T, int kCols, bool kTurned>
int forward(const muon_train_attention_args& a, void* stream) {
  Maps m;
  int rc = encode_inputs(a, &m);
  if (rc != MUON_POLAR_OK) return rc;
  Problem p = problem_of(a);
  p.out = a.out;
  p.out2 = a.out_rest;
  constexpr int kBytes = Forward<kCols>::kBytes;
  rc = prepare<forward_kernel<T, kCols, kTurned>>(kBytes);
  if (rc != MUON_POLAR_OK) return rc;
  const int64_t group = a.heads / a.kv_heads, pair_bytes = 2 * a.dim * static_cast<int64_t>(sizeof(T));
  p.by_heads = group % 2 == 0;
  const int64_t tiles = tiles_of(a, a.length, p.by_heads ? kTile : 2 * kTile), columns = a.heads >> p.by_heads;
  rc = section_of(a.batch * columns, a.keys * pair_bytes / (group >> p.by_heads), tiles / a.batch, &p.section);
  if (rc != MUON_POLAR_OK) return rc;
  return launch(forward_kernel<T, kCols, kTurned>, dim3(static_cast<unsigned>(tiles * columns)), kThreads, kBytes, 1, true,
                stream, m.q, m.k, m.v, p, static_cast<int>(tiles));
}

template <typename T, int kCols>
int backward(const muon_train_attention_args& a, const muon_train_attention_grads& g, void* stream) {
  const int64_t rows = a.batch * a.length;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {  // keys that nothing looks at
    const size_t bytes = static_cast<size_t>(a.batch * a.keys * a.kv_heads * a.dim) * sizeof(T);
    if (bytes == 0) return MUON_POLAR_OK;
    cudaError_t e = cudaMemsetAsync(g.grad_k, 0, bytes, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(g.grad_v, 0, bytes, s);
    return static_cast<int>(e);
  }
  Maps m;
  CUtensorMap map_g;
  int rc = encode_inputs(a, &m);
  if (rc == MUON_POLAR_OK) rc = encode(&map_g, g.grad_out, g.grad_out_stride, a.length, a.heads, a.batch, a.dim, a.dtype);
  if (rc != MUON_POLAR_OK) return rc;
  Problem p = problem_of(a);
  float* workspace = static_cast<float*>(g.workspace);
  const Workspace w = workspace_of(a);
  p.stats = workspace + w.stats;
  p.grad_norm = workspace + w.grad_norm;
  p.value_norm = workspace + w.value_norm;
  p.query_top = reinterpret_cast<float2*>(workspace + w.query_top);
  p.key_top = workspace + w.key_top;
  const Stats st{a.out, a.out_rest, g.grad_out, a.v, a.lse, workspace + w.stats, workspace + w.grad_norm,
                 workspace + w.value_norm, g.grad_out_stride, a.v_stride, rows, a.batch * a.keys, p.length, p.keys, p.heads,
                 p.kv_heads, p.dim};
  const int64_t per = 256 / (kCols / 8) * kStatRows;
  const dim3 grid(static_cast<unsigned>((rows * a.heads + per - 1) / per));
  rc = launch(stats_kernel<T, kCols>, grid, 256, 0, 1, true, stream, st);
  if (rc != MUON_POLAR_OK) return rc;
  if constexpr (!kBf16<T>) {
    const int64_t query_tiles = tiles_of(a, a.length, kTile), key_tiles = tiles_of(a, a.keys, kTile);
    p.section = static_cast<int>(a.batch * a.kv_heads);  // all
    rc = launch(tops_kernel, dim3(static_cast<unsigned>((query_tiles > key_tiles ? query_tiles : key_tiles) * a.kv_heads), 2),
                kTile, 0, 1, true, stream, p, reinterpret_cast<float2*>(workspace + w.query_top), workspace + w.key_top,
                static_cast<int>(query_tiles), static_cast<int>(key_tiles));
    if (rc != MUON_POLAR_OK) return rc;
  }
  const int64_t group = a.heads / a.kv_heads, pair_bytes = 2 * a.dim * static_cast<int64_t>(sizeof(T));
  constexpr int kBytes = KeyGrads<kCols>::kBytes;
  if (a.keys > 0) {
    constexpr int kBytes =
        (2 + KeyGrads<kCols>::kStages) * KeyGrads<kCols>::kTileBytes + static_cast<int>(sizeof(KeyShared));
    rc = prepare<key_grad_kernel<T, kCols>>(kBytes);
    if (rc != MUON_POLAR_OK) return rc;
    p.out = g.grad_k;
    p.out2 = g.grad_v;
    const int64_t tiles = tiles_of(a, a.keys, kTile);
    rc = section_of(a.batch * a.kv_heads, a.length * pair_bytes * group, tiles / a.batch, &p.section);
    if (rc != MUON_POLAR_OK) return rc;
    // Queries before the first key's place, which see none, share tiles with others: maps that begin behind them
    // give zeros for what they and their gradients hold.
    const int64_t blind = a.causal ? a.length - a.keys : a.window > 0 ? a.length - a.keys - a.window + 1 : 0;
    CUtensorMap seeing_q = m.q, seeing_g = map_g;
    if (blind > 0 && blind < a.length) {
      p.blind = static_cast<int>(blind);
      rc = encode(&seeing_q, static_cast<const T*>(a.q) + blind * a.q_stride.row, a.q_stride, a.length - blind, a.heads,
                  a.batch, a.dim, a.dtype);
      if (rc == MUON_POLAR_OK)
        rc = encode(&seeing_g, static_cast<const T*>(g.grad_out) + blind * g.grad_out_stride.row, g.grad_out_stride,
                    a.length - blind, a.heads, a.batch, a.dim, a.dtype);
      if (rc != MUON_POLAR_OK) return rc;
    }
    rc = launch(key_grad_kernel<T, kCols>, dim3(static_cast<unsigned>(tiles * a.kv_heads)), kThreads, kBytes, 1, true,
                stream, seeing_q, m.k, m.v, seeing_g, p, static_cast<int>(tiles));
    if (rc != MUON_POLAR_OK) return rc;
  }
  rc = prepare<query_grad_kernel<T, kCols>>(kBytes);
  if (rc != MUON_POLAR_OK) return rc;
  p.out = g.grad_q;
  p.out2 = nullptr;
  const int64_t tiles = tiles_of(a, a.length, kTile);
  rc = section_of(a.batch * a.heads, a.keys * pair_bytes / group, tiles / a.batch, &p.section);
  if (rc != MUON_POLAR_OK) return rc;
  return launch(query_grad_kernel<T, kCols>, dim3(static_cast<unsigned>(tiles * a.heads)), kThreads, kBytes, 1, true,
                stream, m.q, m.k, m.v, map_g, p, static_cast<int>(tiles));
}

template <typename T>
int forward(const muon_train_attention_args& a, void* stream) {
  if (a.dim > 64) return forward<T, 128, true>(a, stream);
  return a.offsets == nullptr ? forward<T, 64, true>(a, stream) : forward<T, 64, false>(a, stream);
}
template <typename T>
int backward(const muon_train_attention_args& a, const muon_train_attention_grads& g, void* stream) {
  return a.dim <= 64 ? backward<T, 64>(a, g, stream) : backward<T, 128>(a, g, stream);
}

}  // namespace

cudaError_t attention_status(uint32_t* flags, int clear) { return take_status(flags, clear); }
cudaError_t attention_put_wait_limit(uint64_t limit_ns) { return put_wait_limit(limit_ns); }
cudaError_t attention_get_wait_limit(uint64_t* limit_ns) { return get_wait_limit(limit_ns); }

}  // namespace muon_train

extern "C" {

int muon_train_attention_sm100(const muon_train_attention_args* args, void* stream) {
  using namespace muon_train;
  int rc = check(args);
  if (rc == MUON_POLAR_OK) rc = check_forward(*args);
  if (rc != MUON_POLAR_OK || args->batch * args->length == 0) return rc;
  return args->dtype == MUON_TRAIN_BF16 ? forward<__nv_bfloat16>(*args, stream) : forward<__half>(*args, stream);
}

size_t muon_train_attention_workspace_bytes(const muon_train_attention_args* args) {
  using namespace muon_train;
  if (check(args) != MUON_POLAR_OK) return 0;
  return static_cast<size_t>(workspace_of(*args).end) * sizeof(float);
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
  if (a.batch * a.keys > 0 &&
      (g.grad_k == nullptr || g.grad_v == nullptr || !aligned16(g.grad_k) || !aligned16(g.grad_v)))
    return MUON_POLAR_ERR_INVALID_ARGUMENT;
  return a.dtype == MUON_TRAIN_BF16 ? backward<__nv_bfloat16>(a, g, stream) : backward<__half>(a, g, stream);
}

}  // extern "C"
