// Distillation from a teacher's top logits: loss and gradient in one pass over the student's logits.
//
// Student logits l [M, V] (after the softcap where cap > 0), and per row up to K teacher entries (token id, logit
// u_k); an id of -1 is an unused place. With temperature t, weight a and hard target y (ignored when -1):
//   q_k = softmax over the row's entries of u_k / t,   P = softmax(l / t),   p = softmax(l)
//   kl  = sum_k q_k (log q_k - log P[id_k])            (an entry of q_k = 0 adds nothing)
//   ce  = -log(p_y + 1e-10)                            (the form of softcap_ce)
//   row = a t^2 kl + (1 - a) ce,                       loss = scale * sum of the rows
//   dz_j = scale [a t (P_j - sum of q_k with id_k = j) + (1 - a) p_y / (p_y + 1e-10) (p_j - [j == y])] c_j
// with c_j = 1 - (l_j / cap)^2, the softcap's derivative (1 without one). A row without entries has kl 0 and no
// gradient from it; a row whose logits are all -inf has no softmax: its gradient is zero.
// The K + 1 columns of a row that the teacher or the target names get their value from the entries' own fp32
// terms after the dense part is written, so every value of dz is rounded once; entries that name the same
// column add up in the order of their places, so results do not depend on the schedule.
//
// One block per row; the row is read twice (the second time from L2).
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <string>
#include <tuple>

#include "common.cuh"
#include "status.h"

namespace br {
namespace {

constexpr int kMaxTop = 1024;
constexpr int kDistThreads = 256;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f32(float x, float& y) { y = x; }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& y) { y = __float2bfloat16(x); }
__device__ __forceinline__ void from_f32(float x, __half& y) { y = __float2half(x); }

struct DistillParams {
  int64_t ld, ldg;  // row strides of the logits and of the gradient
  int V, K;
  const int* ids;     // [M, K]
  int64_t ld_ids, ld_teacher;
  const int* targets;  // [M] or null
  float inv_cap, inv_t, t, alpha, scale;
  float* rows;  // [M]
  int* status;
};

template <int N>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int w = 1; w < N / 32; ++w) s += red[w];
  return s;
}
template <int N>
__device__ __forceinline__ float block_max_f(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int w = 1; w < N / 32; ++w) s = fmaxf(s, red[w]);
  return s;
}

template <typename T, typename U, bool HARD, bool GRAD>
__global__ void __launch_bounds__(kDistThreads) distill_kernel(const T* logits, const U* __restrict__ teacher, T* grad,
                                                               DistillParams p) {
  extern __shared__ float sm[];  // q [K], l at the ids [K], ids [K]
  __shared__ float red[kDistThreads / 32];
  float* s_q = sm;
  float* s_l = sm + p.K;
  int* s_id = reinterpret_cast<int*>(sm + 2 * p.K);
  const int64_t row = blockIdx.x;
  const T* L = logits + row * p.ld;
  const int tid = threadIdx.x;

  float m = -INFINITY;
  bool nan = false;
  for (int j = tid; j < p.V; j += kDistThreads) {
    const float x = to_f32(L[j]);
    m = fmaxf(m, x);
    nan |= x != x;
  }
  m = block_max_f<kDistThreads>(m, red);
  if (__syncthreads_or(nan)) m = NAN;
  const bool dead = m == -INFINITY;
  const float mref = dead ? 0.f : m;
  float s1 = 0.f, st = 0.f;
  for (int j = tid; j < p.V; j += kDistThreads) {
    const float x = to_f32(L[j]) - mref;
    st += __expf(x * p.inv_t);
    if constexpr (HARD) s1 += __expf(x);
  }
  st = block_sum<kDistThreads>(st, red);
  if constexpr (HARD) s1 = block_sum<kDistThreads>(s1, red);

  // the teacher's distribution over the row's entries
  float um = -INFINITY;
  bool unan = false;
  for (int k = tid; k < p.K; k += kDistThreads) {
    const int raw = p.ids[row * p.ld_ids + k];
    const bool ok = raw == -1 ? false : index_ok(raw, p.V, p.status);
    const float u = ok ? to_f32(teacher[row * p.ld_teacher + k]) * p.inv_t : -INFINITY;
    s_id[k] = ok ? raw : -1;
    s_q[k] = u;
    s_l[k] = ok ? to_f32(L[raw]) : 0.f;
    um = fmaxf(um, u);
    unan |= u != u;
  }
  um = block_max_f<kDistThreads>(um, red);
  if (__syncthreads_or(unan)) um = NAN;
  const bool some = um != -INFINITY;
  float us = 0.f;
  for (int k = tid; k < p.K; k += kDistThreads)
    if (some && s_id[k] >= 0) us += __expf(s_q[k] - um);
  us = block_sum<kDistThreads>(us, red);
  const float log_us = __logf(us), log_st = __logf(st);
  float kl = 0.f;
  for (int k = tid; k < p.K; k += kDistThreads) {
    float q = 0.f;
    if (some && s_id[k] >= 0) {
      const float lq = s_q[k] - um - log_us;
      q = __expf(lq);
      const float lp = s_l[k] == -INFINITY ? -INFINITY : (s_l[k] - mref) * p.inv_t - log_st;
      if (q != 0.f) kl += q * (lq - lp);
    }
    s_q[k] = q;
  }
  kl = block_sum<kDistThreads>(kl, red);  // also orders s_q and s_id for the loop over duplicates

  int y = -1;
  float ly = 0.f, py = 0.f, r = 0.f, loss = p.alpha * p.t * p.t * kl;
  if constexpr (HARD) {
    y = p.targets[row];
    if (y != -1 && !index_ok(y, p.V, p.status)) y = -1;
    if (y >= 0) {
      ly = to_f32(L[y]);
      py = dead ? 0.f : __expf(ly - mref) / s1;
      loss += (1.f - p.alpha) * -__logf(py + 1e-10f);
      r = (1.f - p.alpha) * (py / (py + 1e-10f));
    }
  }
  if (tid == 0) p.rows[row] = loss;
  if constexpr (GRAD) {
    T* G = grad + row * p.ldg;
    __syncthreads();  // in place: every thread has read the columns named by the teacher and the target
    const float ct = dead || !some ? 0.f : p.scale * p.alpha * p.t, cs = ct == 0.f ? 0.f : ct / st;
    const float ch = dead ? 0.f : p.scale * r, c1 = ch == 0.f ? 0.f : ch / s1;
    auto dense = [&](float l) {
      const float x = l - mref;
      float g = cs * __expf(x * p.inv_t);
      if constexpr (HARD) g = fmaf(c1, __expf(x), g);
      return g;
    };
    auto slope = [&](float l) {
      const float c = p.inv_cap > 0.f ? l * p.inv_cap : 0.f;  // without a softcap a logit may be -inf
      return 1.f - c * c;
    };
    for (int j = tid; j < p.V; j += kDistThreads) {
      const float l = to_f32(L[j]);
      from_f32(dead ? 0.f : dense(l) * slope(l), G[j]);
    }
    __syncthreads();
    if (!dead) {
      for (int k = tid; k < p.K + (HARD ? 1 : 0); k += kDistThreads) {
        const int id = k < p.K ? s_id[k] : y;
        if (id < 0) continue;
        const float l = k < p.K ? s_l[k] : ly;
        float q = 0.f;
        for (int i = 0; i < p.K; ++i) q += s_id[i] == id ? s_q[i] : 0.f;
        float g = dense(l) - ct * q;
        if (HARD && id == y) g -= ch;
        from_f32(g * slope(l), G[id]);
      }
    }
  }
}

// loss = scale * sum of the rows, in one fixed order: one block, each thread's rows in order in 64 bits
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) sum_rows_kernel(const float* __restrict__ rows, int64_t M, float scale,
                                                               float* __restrict__ loss) {
  __shared__ double red[kSumThreads];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < M; i += kSumThreads) s += (double)rows[i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = kSumThreads / 2; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *loss = (float)(red[0] * (double)scale);
}

template <typename F>
void by_float(at::ScalarType t, F&& f) {
  if (t == at::kFloat) return f(float{});
  if (t == at::kBFloat16) return f(__nv_bfloat16{});
  f(__half{});
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor, c10::optional<torch::Tensor>> distill_topk(
    const torch::Tensor& logits, const torch::Tensor& ids, const torch::Tensor& teacher,
    c10::optional<torch::Tensor> targets, double cap, double temperature, double alpha, double scale, bool need_grad,
    c10::optional<torch::Tensor> grad_) {
  const char* what = "distill_topk: ";
  auto real = [](const torch::Tensor& t) {
    return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf;
  };
  TORCH_CHECK_VALUE(logits.dim() == 2 && real(logits), what, "logits must be [M, V] in float32, bfloat16 or float16");
  const int64_t M = logits.size(0), V = logits.size(1);
  TORCH_CHECK_VALUE(V >= 1 && V < (int64_t(1) << 31) && M < (int64_t(1) << 31), what, "logits out of range");
  TORCH_CHECK_VALUE(V == 1 || logits.stride(1) == 1, what, "logits need contiguous rows");
  TORCH_CHECK_VALUE(M <= 1 || logits.stride(0) >= V, what, "rows of the logits overlap");
  TORCH_CHECK_VALUE(ids.dim() == 2 && ids.size(0) == M && ids.scalar_type() == at::kInt, what,
                    "teacher_ids must be int32 [M, K]");
  const int64_t K = ids.size(1);
  TORCH_CHECK_VALUE(K >= 1 && K <= kMaxTop, what, "1 to ", std::to_string(kMaxTop),
                    " teacher entries per row, got ", std::to_string(K));
  TORCH_CHECK_VALUE(K == 1 || ids.stride(1) == 1, what, "teacher_ids need contiguous rows");
  TORCH_CHECK_VALUE(teacher.dim() == 2 && teacher.size(0) == M && teacher.size(1) == K && real(teacher), what,
                    "teacher_logits must be [M, K] in float32, bfloat16 or float16");
  TORCH_CHECK_VALUE(K == 1 || teacher.stride(1) == 1, what, "teacher_logits need contiguous rows");
  TORCH_CHECK_VALUE(std::isfinite(cap) && cap >= 0, what, "cap must not be negative (0: no softcap)");
  TORCH_CHECK_VALUE(std::isfinite(temperature) && temperature > 0, what, "temperature must be positive");
  TORCH_CHECK_VALUE(alpha >= 0 && alpha <= 1, what, "alpha must be in [0, 1]");
  TORCH_CHECK_VALUE(std::isfinite(scale), what, "scale must be finite");
  const bool hard = alpha < 1;
  const bool has_targets = targets.has_value() && targets->defined();
  TORCH_CHECK_VALUE(!hard || has_targets, what, "alpha < 1 needs targets");
  if (has_targets) {
    TORCH_CHECK_VALUE(targets->scalar_type() == at::kInt && targets->dim() == 1 && targets->size(0) == M &&
                          targets->is_contiguous(), what, "targets must be contiguous int32 [M]");
    TORCH_CHECK_VALUE(targets->device() == logits.device(), what, "targets are on another device");
  }
  TORCH_CHECK_VALUE(ids.device() == logits.device() && teacher.device() == logits.device(), what,
                    "the teacher's entries are on another device");
  c10::optional<torch::Tensor> grad;
  if (need_grad) {
    if (grad_.has_value() && grad_->defined()) {
      TORCH_CHECK_VALUE(grad_->dim() == 2 && grad_->size(0) == M && grad_->size(1) == V &&
                            grad_->scalar_type() == logits.scalar_type() && grad_->device() == logits.device() &&
                            (V == 1 || grad_->stride(1) == 1) && (M <= 1 || grad_->stride(0) >= V), what,
                        "grad must be [M, V] like the logits, with contiguous rows");
      // the logits themselves (in place), or apart from them
      if (!(grad_->data_ptr() == logits.data_ptr() && grad_->strides() == logits.strides()))
        at::assert_no_overlap(*grad_, logits);
      grad = *grad_;
    } else {
      grad = torch::empty({M, V}, logits.options());
    }
  } else {
    TORCH_CHECK_VALUE(!grad_.has_value() || !grad_->defined(), what, "grad is given but not wanted");
  }
  TORCH_CHECK_VALUE(logits.is_cuda(), what, "logits must be on a CUDA device");
  c10::cuda::CUDAGuard g(logits.device());
  auto st = at::cuda::getCurrentCUDAStream();
  torch::Tensor rows = torch::empty({M}, logits.options().dtype(at::kFloat));
  torch::Tensor loss = torch::empty({}, logits.options().dtype(at::kFloat));
  DistillParams p{};
  p.ld = M > 1 ? logits.stride(0) : V;
  p.ldg = need_grad && M > 1 ? grad->stride(0) : V;
  p.V = (int)V;
  p.K = (int)K;
  p.ids = ids.data_ptr<int>();
  p.ld_ids = M > 1 ? ids.stride(0) : K;
  p.ld_teacher = M > 1 ? teacher.stride(0) : K;
  p.targets = hard ? targets->data_ptr<int>() : nullptr;
  p.inv_cap = cap > 0 ? (float)(1.0 / cap) : 0.f;
  p.inv_t = (float)(1.0 / temperature);
  p.t = (float)temperature;
  p.alpha = (float)alpha;
  p.scale = (float)scale;
  p.rows = rows.data_ptr<float>();
  p.status = status_ptr(logits.device().index());
  if (M > 0) {
    by_float(logits.scalar_type(), [&](auto lt) {
      using T = decltype(lt);
      by_float(teacher.scalar_type(), [&](auto ut) {
        using U = decltype(ut);
        auto launch = [&](auto h, auto w) {
          distill_kernel<T, U, decltype(h)::value, decltype(w)::value>
              <<<(unsigned)M, kDistThreads, K * 12, st>>>(reinterpret_cast<const T*>(logits.data_ptr()),
                                                          reinterpret_cast<const U*>(teacher.data_ptr()),
                                                          need_grad ? reinterpret_cast<T*>(grad->data_ptr()) : nullptr, p);
        };
        if (hard) {
          need_grad ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
        } else {
          need_grad ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
        }
      });
    });
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  sum_rows_kernel<<<1, kSumThreads, 0, st>>>(rows.data_ptr<float>(), M, p.scale, loss.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {loss, rows, grad};
}

}  // namespace br
