// residual_norm_sm100.cu -- the norms before and after a residual block, with
// its gate and residual scale, in one pass, and their gradients.
//
//   r = rsqrt(mean y^2 + eps), u = y r w, h = s x + g u,
//   R = rsqrt(mean h^2 + eps), n = h R p
//
// With a = dn p, b0 = g w (dh + R a), A = sum a h, B1 = sum b0 y,
// B2 = sum g w y h and k = R^3 A / width:
//   dH = dh + R a - k h         dx = s dH        ds = sum dH x
//   dy = r g w dH - y r^3 (B1 - k B2) / width
//   C  = sum dH y r             dg = w C         dw = g C
//   dp = sum dn h R
// so that a row needs one reduction of three sums, and h is made again from
// x and y instead of being kept.
//
// Bound by memory: forward reads x, y and writes h, n; backward reads x, y,
// dh, dn and writes dx, dy.  Parameter gradients: each block adds up its rows
// in order, a second kernel adds up the blocks in order.
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

// ------------------------------------------------------------ any width
constexpr int kThreads = 256;

// One block a row; the row is read again from L1 / L2 for each step.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_row_kernel(const __grid_constant__ muon_train_norm_args a) {
  __shared__ float red[2 * 32];
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
    if (threadIdx.x == 0 && a.rstd_post != nullptr) a.rstd_post[row] = r;
  }
  float sum[1] = {0.f};
  T* hidden = static_cast<T*>(a.hidden) + base;
  for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
    const float h = fmaf(p.scale(c), to_float(x[c]), p.gate(gate_row, c) * (to_float(y[c]) * r * p.post(c)));
    hidden[c] = from_float<T>(h);
    sum[0] = fmaf(h, h, sum[0]);
  }
  if (a.pre_weight == nullptr) return;
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
//   scale [blocks][width or 1]  ds
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
  int64_t want = (target + p.groups - 1) / p.groups;
  if (want > per_group) want = per_group;
  p.chunks_per_group = want < 1 ? 1 : want;
  p.chunks = p.groups * p.chunks_per_group;
  p.blocks = p.chunks < target ? p.chunks : target;
  const auto align = [](size_t v) { return (v + 255) / 256 * 256; };
  p.gain_off = 0;
  p.pre_off = align(static_cast<size_t>(p.chunks * a.width) * sizeof(float));
  p.scale_off = p.pre_off + align(static_cast<size_t>(p.blocks * a.width) * sizeof(float));
  p.bytes = p.scale_off + align(static_cast<size_t>(p.blocks * a.width) * sizeof(float));
  return p;
}

struct Backward {
  muon_train_norm_args a;
  muon_train_norm_grads g;
  Plan plan;
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

template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_backward_row_kernel(const __grid_constant__ Backward b) {
  __shared__ float red[3 * 32];
  const muon_train_norm_args& a = b.a;
  const Params p{a};
  const float width = static_cast<float>(a.width);
  const T* dh_all = static_cast<const T*>(b.g.grad_hidden);
  const T* dn_all = static_cast<const T*>(b.g.grad_normed);
  float* pre = b.pre != nullptr ? b.pre + blockIdx.x * a.width : nullptr;
  float* scale = b.scale != nullptr
                     ? b.scale + blockIdx.x * (a.scale_count == 1 ? 1 : a.width)
                     : nullptr;
  bool first_row = true;
  float scale_sum = 0.f;
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
        const float yv = to_float(y[c]), gw = p.gate(gate_row, c) * p.post(c);
        const float h = fmaf(p.scale(c), to_float(x[c]), gw * (yv * r));
        const float dh = dh_all != nullptr ? to_float(dh_all[base + c]) : 0.f;
        const float an = dn_all != nullptr ? to_float(dn_all[base + c]) * p.pre(c) : 0.f;
        sums[0] = fmaf(an, h, sums[0]);
        sums[1] = fmaf(gw * fmaf(rh, an, dh), yv, sums[1]);
        sums[2] = fmaf(gw * yv, h, sums[2]);
      }
      __syncthreads();  // the last row's sums have been read
      block_sums(sums, red, kThreads);
      const float k = rh * rh * rh * sums[0] / width;
      const float ky = a.post_weight != nullptr ? r * r * r * (sums[1] - k * sums[2]) / width : 0.f;
      for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
        const float yv = to_float(y[c]), xv = to_float(x[c]);
        const float gate = p.gate(gate_row, c), post = p.post(c), sc = p.scale(c);
        const float h = fmaf(sc, xv, gate * post * (yv * r));
        const float dh = dh_all != nullptr ? to_float(dh_all[base + c]) : 0.f;
        const float dn = dn_all != nullptr ? to_float(dn_all[base + c]) : 0.f;
        const float d = fmaf(-k, h, fmaf(rh, dn * p.pre(c), dh));
        if (b.g.grad_residual != nullptr)
          static_cast<T*>(b.g.grad_residual)[base + c] = from_float<T>(d * sc);
        if (b.g.grad_block_out != nullptr)
          static_cast<T*>(b.g.grad_block_out)[base + c] = from_float<T>(fmaf(-ky, yv, r * (gate * post) * d));
        const float gained = d * (yv * r);
        if (b.plan.gate_per_row && b.g.grad_gate != nullptr)
          store_any(b.g.grad_gate, a.gate_dtype, base + c, gained * post);
        if (gain != nullptr)
          gain[c] = (row == r0 ? 0.f : gain[c]) + (b.plan.gate_per_row ? gained * gate : gained);
        if (pre != nullptr) pre[c] = (first_row ? 0.f : pre[c]) + dn * h * rh;
        if (scale != nullptr) {
          if (a.scale_count == 1)
            scale_sum = fmaf(d, xv, scale_sum);
          else
            scale[c] = (first_row ? 0.f : scale[c]) + d * xv;
        }
      }
      first_row = false;
    }
  }
  if (scale != nullptr && a.scale_count == 1) {
    __syncthreads();
    float sums[1] = {scale_sum};
    block_sums(sums, red, kThreads);
    if (threadIdx.x == 0) scale[0] = sums[0];
  }
}

// Adds up partial sums: blockIdx.y = 0 pre weight, 1 residual scale, 2 post
// weight, from 3 on gate rows (blockIdx.y - 3, + gridDim.y - 3, ..).  A warp
// reads 32 columns of a partial row; the block's 16 warps take every 16th row
// and are added in order.
constexpr int kSumWarps = 16;
constexpr int kGateRowBlocks = 4096;

// Sum over partial rows [first, last) of this block's 32 columns, in warp 0.
// With `gate`, row i is multiplied by the gate row of its chunk.
__device__ float column_sum(const float* from, int64_t width, int64_t first, int64_t last,
                            const Backward* gate, float (*part)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.f;
  if (column < width) {
    for (int64_t i = first + warp; i < last; i += kSumWarps) {
      const float v = from[i * width + column];
      sum = gate != nullptr ? fmaf(v, Params{gate->a}.gate(i / gate->plan.chunks_per_group, column), sum)
                            : sum + v;
    }
  }
  __syncthreads();  // part has been read
  part[warp][lane] = sum;
  __syncthreads();
  sum = 0.f;
  if (warp == 0)
    for (int w = 0; w < kSumWarps; ++w) sum += part[w][lane];
  return sum;
}

__global__ void __launch_bounds__(kSumWarps * 32)
    norm_sums_kernel(const __grid_constant__ Backward b) {
  __shared__ float part[kSumWarps][32];
  const muon_train_norm_args& a = b.a;
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const bool writes = threadIdx.x < 32 && column < a.width;
  const int what = blockIdx.y;
  if (what == 0) {
    if (b.pre == nullptr) return;
    const float v = column_sum(b.pre, a.width, 0, b.plan.blocks, nullptr, part);
    if (writes) store_any(b.g.grad_pre_weight, a.pre_dtype, column, v);
  } else if (what == 1) {
    if (b.scale == nullptr || static_cast<int64_t>(blockIdx.x) * 32 >= a.scale_count) return;
    const float v = column_sum(b.scale, a.scale_count, 0, b.plan.blocks, nullptr, part);
    if (writes && column < a.scale_count)
      store_any(b.g.grad_residual_scale, a.scale_dtype, column, v);
  } else if (what == 2) {
    if (b.g.grad_post_weight == nullptr) return;
    const bool times_gate = a.gate != nullptr && !b.plan.gate_per_row;
    const float v = column_sum(b.gain, a.width, 0, b.plan.chunks, times_gate ? &b : nullptr, part);
    if (writes) store_any(b.g.grad_post_weight, a.post_dtype, column, v);
  } else {
    for (int64_t g = what - 3; g < b.plan.groups; g += gridDim.y - 3) {
      const int64_t first = g * b.plan.chunks_per_group;
      const float v = column_sum(b.gain, a.width, first, first + b.plan.chunks_per_group, nullptr, part);
      if (writes) store_any(b.g.grad_gate, a.gate_dtype, g * a.width + column, v * Params{a}.post(column));
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

int target_blocks(int64_t* target) {
  int sms = 0;
  const int rc = sm_count(&sms);
  *target = static_cast<int64_t>(sms) * 2;
  return rc;
}

template <typename T>
int forward(const muon_train_norm_args& a, void* stream) {
  return launch(norm_row_kernel<T>, dim3(static_cast<unsigned>(a.rows)), kThreads, 0, 1, stream, a);
}

template <typename T>
int backward(const Backward& b, void* stream) {
  return launch(norm_backward_row_kernel<T>, dim3(static_cast<unsigned>(b.plan.blocks)), kThreads,
                0, 1, stream, b);
}

}  // namespace
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
  if (check(args) != MUON_POLAR_OK || args->rows == 0 || target_blocks(&target) != MUON_POLAR_OK)
    return 0;
  return make_plan(normalised(*args), target).bytes;
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
  int64_t target = 0;
  rc = target_blocks(&target);
  if (rc != MUON_POLAR_OK) return rc;
  Backward b;
  b.a = normalised(*args);
  b.g = *grads;
  if (b.a.post_weight == nullptr) b.g.grad_post_weight = nullptr;
  if (b.a.pre_weight == nullptr) b.g.grad_pre_weight = nullptr;
  if (b.a.gate == nullptr) b.g.grad_gate = nullptr;
  if (b.a.residual_scale == nullptr) b.g.grad_residual_scale = nullptr;
  b.plan = make_plan(b.a, target);
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
    case MUON_TRAIN_F32: rc = backward<float>(b, stream); break;
    case MUON_TRAIN_BF16: rc = backward<__nv_bfloat16>(b, stream); break;
    default: rc = backward<__half>(b, stream); break;
  }
  if (rc != MUON_POLAR_OK || (b.gain == nullptr && b.pre == nullptr && b.scale == nullptr)) return rc;
  const unsigned columns = static_cast<unsigned>((b.a.width + 31) / 32);
  const int64_t gate_rows = want_gate_sums ? b.plan.groups : 0;
  const unsigned what = 3 + static_cast<unsigned>(gate_rows < kGateRowBlocks ? gate_rows : kGateRowBlocks);
  return launch(norm_sums_kernel, dim3(columns, what), kSumWarps * 32, 0, 1, stream, b);
}

}  // extern "C"
