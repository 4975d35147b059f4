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

constexpr int kWarps = 16;  // tokens in flight of a block, one a warp
constexpr int kThreads = kWarps * 32;
constexpr int kBlocksPerSm = 2;
constexpr int kSoftmax = 0;
constexpr float kTiny = 1e-20f;
// few_best pays from 3 choices on (32768 x 256, one group: 1 of them 23.1 us, by
// argmaxes 19.0; 2: 23.8 and 22.9; 8: 27 and 40; 16: 34 and 63); with more than
// half of the lanes chosen from, the bound lets too many keys through.
constexpr int kFewFrom = 3, kFewTo = 16;
constexpr int kSlots = MUON_TRAIN_MAX_ROUTES / 32;  // chosen experts a lane keeps

__device__ __forceinline__ float sigmoid(float x) {
  return __frcp_rn(__fadd_rn(1.0f, expf(-x)));
}

// Keys are compared as they are, which makes -0 and +0 one key.  A NaN counts
// as -inf; NaN itself then marks a key that can no longer be chosen, since a
// maximum passes over it and it equals nothing.
__device__ __forceinline__ float number(float key) { return fmaxf(key, -INFINITY); }
__device__ __forceinline__ float taken() { return __int_as_float(0x7fffffff); }

__device__ __forceinline__ float lanes_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, %2;" : "=f"(m) : "f"(v), "r"(kFullMask));
  return m;
}

// A lane has up to kPer neighbouring experts of a token, e0 the first, and a
// higher lane higher ones, so that the lowest lane holds the lowest index.
// With groups, each group has lanes of its own.
struct Lanes {
  int e0, count;
  __device__ Lanes(int experts, int groups, int lanes_a_group, int per) {
    const int lane = threadIdx.x & 31, group = lane / lanes_a_group, size = experts / groups;
    const int inside = (lane % lanes_a_group) * per;
    e0 = group * size + inside;
    count = group < groups ? max(0, min(per, size - inside)) : 0;
  }
};

// A lane's logits.  They are loaded in runs of up to 16 bytes where rows and
// groups keep that alignment (whole), else one by one.
template <typename T, int kPer>
struct Row {
  static constexpr int kRun = kPer * static_cast<int>(sizeof(T)) > 16 ? 16 / static_cast<int>(sizeof(T)) : kPer;
  float v[kPer];
  __device__ __forceinline__ void load(const T* l, const Lanes& at, bool whole) {
#pragma unroll
    for (int i = 0; i < kPer; i += kRun) {
      if (whole && i < at.count) {
        if constexpr (kRun * sizeof(T) >= 4) {
          float part[kRun];
          Elements<T, kRun>::unpack(Elements<T, kRun>::load(l + at.e0 + i), part);
#pragma unroll
          for (int j = 0; j < kRun; ++j) v[i + j] = part[j];
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < kRun; ++j) v[i + j] = i + j < at.count ? to_float(l[at.e0 + i + j]) : -INFINITY;
    }
  }
};

// Scores of a lane's experts (0 beyond the last).
template <int kPer>
__device__ __forceinline__ void scores(const float (&l)[kPer], const Lanes& at, int score, float (&s)[kPer]) {
  if (score != kSoftmax) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s[i] = i < at.count ? sigmoid(l[i]) : 0.f;
    return;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) m = fmaxf(m, l[i]);
  m = warp_max(m);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    // a row of -inf has no scores; a NaN stays one
    s[i] = i >= at.count || (m == -INFINITY && l[i] == l[i]) ? 0.f : expf(__fsub_rn(l[i], m));
    sum += s[i];
  }
  const float total = static_cast<float>(warp_sum64(sum));
#pragma unroll
  for (int i = 0; i < kPer; ++i) s[i] = total == 0.f ? 0.f : __fdiv_rn(s[i], total);
}

// How a call's rows are laid out and its groups ranked.
struct Plan {
  bool whole;         // runs of a row can be loaded at once
  bool few;           // the best keys may come from few_best
  bool by_logit;      // the logits are the keys
  bool ranked;        // each group has lanes of its own; else groups go through shared memory
  int lanes_a_group;  // a power of two; 32 for one group, and when not ranked
};

// The two largest of (first, second, key), a number.
__device__ __forceinline__ void best_two(float key, float& first, float& second) {
  second = fmaxf(second, fminf(first, key));
  first = fmaxf(first, key);
}

// The k best keys of a lane's and its warp's, best first, the lowest index of
// equal ones: lane j < k receives the index of the j-th.  best is the lane's
// largest key, none a NaN.  The k-th largest of the lanes' best keys is a bound
// that k keys reach, so only the few keys from it on, the candidates, are put
// side by side, a lane each, and each counts the better ones.  Returns false
// with nothing chosen if there are not k such lanes, or too many candidates.
template <int kPer>
__device__ __forceinline__ bool few_best(const float (&key)[kPer], float best, const Lanes& at, int k,
                                         float2* found, int& chosen) {
  const int lane = threadIdx.x & 31;
  float bound = taken();
  for (int j = 0; j < k; ++j) {  // equal ones go at once, which lowers the bound
    bound = lanes_max(best);
    if (best == bound) best = taken();
  }
  int count = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) count += key[i] >= bound;
  int before = count;  // the candidates of this lane and lower ones, then of these alone
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(kFullMask, before, o);
    if (lane >= o) before += other;
  }
  const int total = __shfl_sync(kFullMask, before, 31);
  if (total < k || total > 32) return false;  // (no bound: no candidate)
  before -= count;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (key[i] >= bound) found[before++] = make_float2(key[i], __int_as_float(at.e0 + i));
  __syncwarp();
  const float2 mine = lane < total ? found[lane] : make_float2(taken(), 0.f);
  int better = lane < total ? 0 : 32;
#pragma unroll 4
  for (int j = 0; j < total; ++j) {
    const float other = __shfl_sync(kFullMask, mine.x, j);
    better += other > mine.x || (other == mine.x && j < lane);
  }
  __syncwarp();  // found is read
  int* sorted = reinterpret_cast<int*>(found);
  if (better < k) sorted[better] = __float_as_int(mine.y);
  __syncwarp();
  if (lane < k) chosen = sorted[lane];
  return true;
}

// Forward: one warp a token.  The time goes into instructions, not memory (256
// sigmoid scores in 8 groups: about 840 a token against 1 KB read, 79% of the
// issue slots used), so keys and scores stay in registers, and kFull, rows of
// exactly 32 kPer experts, leaves out every check for a lane's last one.  The
// best keys come from few_best where the plan allows it, else one by one: an
// argmax is one redux of the lanes' best keys, and only the winning lane looks
// for its next one.  32768 tokens of 256 experts, 8 of 8 groups' 4 best, fp32:
// 33 us (45 with argmaxes alone, 53 without kFull too; the bytes take 5.5).
template <typename T, int kPer, bool kFull>
__global__ void __launch_bounds__(kThreads, kPer <= 8 ? kBlocksPerSm : 1)
    route_kernel(const __grid_constant__ muon_train_route_args a, Plan plan) {
  extern __shared__ __align__(16) float smem[];
  const int experts = static_cast<int>(a.experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Lanes at(experts, plan.ranked ? a.groups : 1, plan.lanes_a_group, kPer);
  if constexpr (kFull) at.count = kPer;
  __shared__ float2 candidates[kPer >= 2 ? kWarps : 1][32];
  float2* found = candidates[kPer >= 2 ? warp : 0];
  uint32_t* histogram = reinterpret_cast<uint32_t*>(smem);  // of the block's tokens
  float* row = smem + experts + warp * (plan.ranked ? 1 : 2) * experts;
  float* row_keys = row + experts;  // when not ranked
  for (int e = threadIdx.x; e < experts; e += kThreads) histogram[e] = 0;
  __syncthreads();
  float bias[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) bias[i] = a.bias != nullptr && i < at.count ? a.bias[at.e0 + i] : 0.f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
  int64_t token = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  Row<T, kPer> l;
  if (token < a.tokens) l.load(static_cast<const T*>(a.logits) + token * a.ld, at, plan.whole);
  for (; token < a.tokens; token += step) {
    float s[kPer], key[kPer];
    scores(l.v, at, a.score, s);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float k = plan.by_logit ? l.v[i] : a.bias != nullptr ? __fadd_rn(s[i], bias[i]) : s[i];
      key[i] = i < at.count ? number(k) : taken();
      if (kFull && kPer % 4 == 0) {
        if (i % 4 == 3) *reinterpret_cast<float4*>(row + at.e0 + i - 3) = make_float4(s[i - 3], s[i - 2], s[i - 1], s[i]);
      } else if (i < at.count) {
        row[at.e0 + i] = s[i];
      }
    }
    if (token + step < a.tokens)
      l.load(static_cast<const T*>(a.logits) + (token + step) * a.ld, at, plan.whole);
    if (a.groups > 1) {
      if (plan.ranked) {
        float first = -INFINITY, second = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPer; ++i) best_two(i < at.count ? key[i] : -INFINITY, first, second);
        for (int o = 1; o < plan.lanes_a_group; o <<= 1) {
          const float f = __shfl_xor_sync(kFullMask, first, o), g = __shfl_xor_sync(kFullMask, second, o);
          second = fmaxf(fminf(first, f), fmaxf(second, g));
          first = fmaxf(first, f);
        }
        const float mine = number(a.group_top == 2 ? __fadd_rn(first, second) : first);
        const int group = lane / plan.lanes_a_group;
        int better = 0;
        for (int g = 0; g < a.groups; ++g) {
          const float other = __shfl_sync(kFullMask, mine, g * plan.lanes_a_group);
          better += other > mine || (other == mine && g < group);
        }
        if (better >= a.top_groups) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) key[i] = taken();
        }
      } else {
        const int size = experts / a.groups;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (i < at.count) row_keys[at.e0 + i] = key[i];
        __syncwarp();
        // each lane ranks its groups g = lane, + 32, ..
        float mine[MUON_TRAIN_MAX_EXPERTS / 32];
        const int rounds = (a.groups + 31) / 32;
        for (int r = 0; r < rounds; ++r) {
          const int g = r * 32 + lane;
          float first = -INFINITY, second = -INFINITY;
          if (g < a.groups)
            for (int e = g * size; e < (g + 1) * size; ++e) best_two(row_keys[e], first, second);
          mine[r] = g < a.groups ? number(a.group_top == 2 ? __fadd_rn(first, second) : first) : taken();
        }
        __syncwarp();
        // the best groups one by one; row_keys now says which groups stay
        for (int g = lane; g < a.groups; g += 32) row_keys[g] = 0.f;
        __syncwarp();
        for (int j = 0; j < a.top_groups; ++j) {
          float best = taken();
          for (int r = 0; r < rounds; ++r) best = fmaxf(best, mine[r]);
          best = lanes_max(best);
          int g = 0x7fffffff;
          for (int r = rounds - 1; r >= 0; --r)
            if (mine[r] == best) g = r * 32 + lane;
          g = __reduce_min_sync(kFullMask, g);
          if ((g & 31) == lane) {
            mine[g >> 5] = taken();
            row_keys[g] = 1.f;
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (i < at.count && row_keys[(at.e0 + i) / size] == 0.f) key[i] = taken();
      }
    }
    // the k best; of equal ones the lowest lane, and in
    // it the first
    float best = taken();
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = fmaxf(best, key[i]);
    int chosen[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) chosen[i] = 0;
    bool done = false;
    if constexpr (kPer >= 2) {
      if (plan.few) done = few_best<kPer>(key, best, at, a.k, found, chosen[0]);
    }
    if (!done) {
      for (int j = 0; j < a.k; ++j) {
        const float top = lanes_max(best);
        const int who = __ffs(__ballot_sync(kFullMask, best == top)) - 1;
        int e = 0;
        if (lane == who) {
          int which = 0;
#pragma unroll
          for (int i = kPer - 1; i >= 0; --i)
            if (key[i] == top) which = i;
          best = taken();
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            if (i == which) key[i] = taken();
            best = fmaxf(best, key[i]);
          }
          e = at.e0 + which;
        }
        e = __shfl_sync(kFullMask, e, who);
        if (lane == (j & 31)) {
#pragma unroll
          for (int i = 0; i < kSlots; ++i)
            if (i == (j >> 5)) chosen[i] = e;
        }
      }
    }
    __syncwarp();  // row is written
    float w[kSlots], total = 0.f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (i * 32 >= a.k) break;
      w[i] = i * 32 + lane < a.k ? row[chosen[i]] : 0.f;
      total += w[i];
    }
    total = a.renormalize ? warp_sum(total) + kTiny : 1.f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int j = i * 32 + lane;
      if (i * 32 >= a.k) break;
      if (j >= a.k) continue;
      a.weights[token * a.k + j] = (a.renormalize ? __fdiv_rn(w[i], total) : w[i]) * a.scale;
      a.indices[token * a.k + j] = chosen[i];
      atomicAdd(&histogram[chosen[i]], 1u);
    }
    __syncwarp();  // row is read before the next token's is written
  }
  if (a.counts == nullptr) return;
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kThreads) {
    if (gridDim.x == 1)
      a.counts[e] = histogram[e];
    else if (histogram[e] != 0)
      atomicAdd(reinterpret_cast<unsigned long long*>(a.counts) + e,
                static_cast<unsigned long long>(histogram[e]));
  }
}

// Backward, one warp a token.  With the renormalised weights v = s / (S + tiny),
// S the chosen scores' sum, and c = sum g v, a chosen score's gradient is
// scale (g_j - c) / (S + tiny).  The sigmoid's logits get s (1 - s) times that,
// the others nothing and are not read: zeros, and then the chosen.  A softmax
// reaches every expert (kWholeRow): dl = s (ds - sum s ds), whose last sum is
// scale c tiny / (S + tiny) renormalised, and scale sum g s otherwise.  The
// whole row's maximum and sum are needed even where the others' part vanishes:
// a bias may choose experts whose scores vanish beside the row's.
// 32768 x 256 fp32, 8 chosen: softmax 24.5 us (from the chosen logits alone
// 17, which is no gradient of such a choice), sigmoid 15.
template <typename T, int kPer, bool kWholeRow>
__global__ void __launch_bounds__(kThreads)
    route_backward_kernel(const __grid_constant__ muon_train_route_args a, Plan plan,
                          const float* __restrict__ grad_weights, T* __restrict__ grad) {
  using Logits = Row<T, kPer>;
  const int experts = static_cast<int>(a.experts);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lanes at(experts, 1, 32, kPer);
  for (int64_t token = static_cast<int64_t>(blockIdx.x) * kWarps + warp; token < a.tokens;
       token += static_cast<int64_t>(gridDim.x) * kWarps) {
    const T* l = static_cast<const T*>(a.logits) + token * a.ld;
    T* out = grad + token * a.experts;
    int chosen[kSlots];
    float g[kSlots];
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int j = i * 32 + lane;
      chosen[i] = -1;
      g[i] = 0.f;
      if (j < a.k) {
        const int64_t e = a.indices[token * a.k + j];
        if (e >= 0 && e < experts) {
          chosen[i] = static_cast<int>(e);
          g[i] = grad_weights[token * a.k + j];
        }
      }
    }
    const auto store_row = [&](const float(&v)[kPer]) {
#pragma unroll
      for (int i = 0; i < kPer; i += Logits::kRun) {
        if (plan.whole && i < at.count) {
          if constexpr (Logits::kRun * sizeof(T) >= 4) {
            float part[Logits::kRun];
#pragma unroll
            for (int j = 0; j < Logits::kRun; ++j) part[j] = v[i + j];
            Elements<T, Logits::kRun>::store(out + at.e0 + i, Elements<T, Logits::kRun>::pack(part));
            continue;
          }
        }
#pragma unroll
        for (int j = 0; j < Logits::kRun; ++j)
          if (i + j < at.count) out[at.e0 + i + j] = from_float<T>(v[i + j]);
      }
    };
    if constexpr (!kWholeRow) store_row({});
    const int slots = (a.k + 31) / 32;  // of chosen experts that a lane has
    float s[kSlots], total = 0.f;
    [[maybe_unused]] float all[kPer];  // the row's scores
    if constexpr (kWholeRow) {
      Logits logits;
      logits.load(l, at, plan.whole);
      scores(logits.v, at, kSoftmax, all);
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (i >= slots) break;
      s[i] = 0.f;
      if constexpr (kWholeRow) {  // from the lane that has the expert
        const int e = max(chosen[i], 0);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const float other = __shfl_sync(kFullMask, all[j], e / kPer);
          if (j == e % kPer && chosen[i] >= 0) s[i] = other;
        }
      } else if (chosen[i] >= 0) {
        s[i] = sigmoid(to_float(l[chosen[i]]));
      }
      total += s[i];
    }
    total = a.renormalize ? warp_sum(total) + kTiny : 1.f;
    float v[kSlots], c = 0.f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (i >= slots) break;
      v[i] = a.renormalize ? __fdiv_rn(s[i], total) : s[i];
      c = fmaf(g[i], v[i], c);
    }
    if (kWholeRow || a.renormalize) c = warp_sum(c);
    // every expert's part, and what the chosen ones' g is relative to
    const float others = a.scale * c * (a.renormalize ? kTiny / total : 1.f), base = a.renormalize ? c : 0.f;
    if constexpr (kWholeRow) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) all[i] = -all[i] * others;
      store_row(all);
    }
    __syncwarp();  // the row is written
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (i >= slots || chosen[i] < 0) continue;
      const float own = a.scale * v[i] * (g[i] - base);
      out[chosen[i]] = from_float<T>(kWholeRow ? fmaf(-s[i], others, own) : own * (1.0f - s[i]));
    }
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
  const int64_t want = (tokens + kWarps - 1) / kWarps, most = static_cast<int64_t>(sms) * kBlocksPerSm;
  *grid = static_cast<unsigned>(want < most ? want : most);
  return rc;
}

// Shared memory of a block with the most experts; above 48 KB it needs the
// kernel's leave.
constexpr size_t kMostSmem = (1 + kWarps * 2) * MUON_TRAIN_MAX_EXPERTS * sizeof(float);

// Lanes of each group: the most, a power of two, that all groups can have.
int lanes_for(int groups) {
  int lanes = 32;
  while (lanes > 1 && lanes * groups > 32) lanes /= 2;
  return lanes;
}
// Whether every group can have lanes of its own, up to 32 experts a lane; its
// experts a lane are then *per, else those of one row of all experts.
bool ranked_groups(const muon_train_route_args& a, int64_t* per) {
  const int64_t size = a.experts / a.groups, lanes = lanes_for(a.groups);
  *per = (size + lanes - 1) / lanes;
  if (a.groups <= 32 && *per <= 32) return true;
  *per = (a.experts + 31) / 32;
  return false;
}

template <typename T, int kPer, bool kFull>
int forward_as(const muon_train_route_args& a, bool ranked, void* stream) {
  constexpr int kRun = Row<T, kPer>::kRun;
  const int64_t ld = a.tokens > 1 ? a.ld : a.experts;
  Plan plan{};
  plan.ranked = ranked;
  plan.lanes_a_group = ranked ? lanes_for(a.groups) : 32;
  plan.whole = (ranked ? a.experts / a.groups : a.experts) % kRun == 0 && ld % kRun == 0 && aligned16(a.logits);
  const int64_t size = ranked ? a.experts / a.groups : a.experts;
  // every choice needs a lane with keys
  plan.few = a.k >= kFewFrom && a.k <= kFewTo && a.k <= (ranked ? a.top_groups : 1) * ((size + kPer - 1) / kPer);
  plan.by_logit = a.score == kSoftmax && a.bias == nullptr && (a.groups == 1 || a.group_top == 1);
  const size_t smem = (1 + kWarps * (ranked ? 1 : 2)) * a.experts * sizeof(float);
  unsigned grid = 0;
  int rc = grid_for(a.tokens, &grid);
  if (rc == MUON_POLAR_OK && smem > 40 * 1024) rc = allow_smem<route_kernel<T, kPer, kFull>>(kMostSmem);
  if (rc != MUON_POLAR_OK) return rc;
  if (a.counts != nullptr && grid > 1) {  // one block writes its counts, more add them up
    const cudaError_t e = cudaMemsetAsync(a.counts, 0, a.experts * sizeof(int64_t),
                                          static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return launch(route_kernel<T, kPer, kFull>, dim3(grid), kThreads, smem, 1, false, stream, a, plan);
}

template <typename T, int kPer>
int forward(const muon_train_route_args& a, bool ranked, void* stream) {
  if (a.experts == 32 * kPer) return forward_as<T, kPer, true>(a, ranked, stream);
  return forward_as<T, kPer, false>(a, ranked, stream);
}

template <typename T, int kPer>
int backward(const muon_train_route_args& a, const float* grad_weights, void* grad, void* stream) {
  constexpr int kRun = Row<T, kPer>::kRun;
  const int64_t ld = a.tokens > 1 ? a.ld : a.experts;
  Plan plan{};
  plan.whole = a.experts % kRun == 0 && ld % kRun == 0 && aligned16(a.logits) && aligned16(grad);
  unsigned grid = 0;
  const int rc = grid_for(a.tokens, &grid);
  if (rc != MUON_POLAR_OK) return rc;
  if (a.score == kSoftmax)
    return launch(route_backward_kernel<T, kPer, true>, dim3(grid), kThreads, 0, 1, false, stream, a, plan,
                  grad_weights, static_cast<T*>(grad));
  return launch(route_backward_kernel<T, kPer, false>, dim3(grid), kThreads, 0, 1, false, stream, a, plan,
                grad_weights, static_cast<T*>(grad));
}

// kPer: the power of two that covers a lane's experts.
template <typename T>
int forward(const muon_train_route_args& a, void* stream) {
  int64_t per = 0;
  const bool ranked = ranked_groups(a, &per);
  if (per <= 1) return forward<T, 1>(a, ranked, stream);
  if (per <= 2) return forward<T, 2>(a, ranked, stream);
  if (per <= 4) return forward<T, 4>(a, ranked, stream);
  if (per <= 8) return forward<T, 8>(a, ranked, stream);
  if (per <= 16) return forward<T, 16>(a, ranked, stream);
  return forward<T, 32>(a, ranked, stream);
}
template <typename T>
int backward(const muon_train_route_args& a, const float* grad_weights, void* grad, void* stream) {
  if (a.experts <= 32) return backward<T, 1>(a, grad_weights, grad, stream);
  if (a.experts <= 64) return backward<T, 2>(a, grad_weights, grad, stream);
  if (a.experts <= 128) return backward<T, 4>(a, grad_weights, grad, stream);
  if (a.experts <= 256) return backward<T, 8>(a, grad_weights, grad, stream);
  if (a.experts <= 512) return backward<T, 16>(a, grad_weights, grad, stream);
  return backward<T, 32>(a, grad_weights, grad, stream);
}

}  // namespace
}  // namespace muon_train

extern "C" {

int muon_train_route_sm100(const muon_train_route_args* args, void* stream) {
  using namespace muon_train;
  const int rc = check(args);
  if (rc != MUON_POLAR_OK) return rc;
  if (args->tokens > 0 && args->weights == nullptr) return MUON_POLAR_ERR_INVALID_ARGUMENT;
  if (args->tokens == 0) {
    if (args->counts == nullptr) return MUON_POLAR_OK;
    return static_cast<int>(cudaMemsetAsync(args->counts, 0, args->experts * sizeof(int64_t),
                                            static_cast<cudaStream_t>(stream)));
  }
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
