// Attention inside the sequences of a packed batch (forward and backward), causal, with an optional sliding
// window and grouped heads.
//
// q [N, H, D], k and v [N, KV, D] hold N rows (tokens) of any number of sequences one behind the other;
// start[i] and end[i] give the span of row i's sequence (bounds.cu). With head h reading kv head
// g = h / (H / KV), scale s and window w (w = N without one), row i sees the keys
//   j in [max(start[i], i - w + 1), min(i + 1, end[i])):
//   x_ij = s q_i.k_j,  lse_i = log sum_j exp(x_ij),  p_ij = exp(x_ij - lse_i),  o_i = sum_j p_ij v_j
// and with do the gradient of o and delta_i = do_i.o_i
//   dS_ij = p_ij (do_i.v_j - delta_i),  dq_i = s sum_j dS_ij k_j,  dk_j = s sum_i,h dS_ij q_i,  dv_j = sum_i,h p_ij do_i.
// Key row j is seen by the queries [j, min(j + w, end[j])). Rows of no sequence (empty span) are neither read
// as keys nor written. Spans are clamped to the rows that exist, so a bad span reads nothing outside.
//
// One warp per row and head: a lane holds D / 32 of the row's values in fp32, a score is a warp-wide sum.
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <string>
#include <tuple>

#include "half_types.cuh"
#include "status.h"

namespace br {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Rows {  // a [N, heads, D] tensor: element (i, h, d) at p + i * row + h * head + d
  void* p;
  int64_t row, head;
};

struct PackedParams {
  int N, H, KV, window;
  float scale, scale_log2;
  Rows q, k, v, o, dout, dq, dk, dv;
  const int* start;
  const int* end;
  float* lse;    // [H, N], natural log
  float* delta;  // [H, N]
};

// ---------------------------------------------------------------------------------------- row by row
template <typename T, int D>
__device__ __forceinline__ void load_row(const Rows& r, int64_t i, int h, int lane, float (&x)[D / 32]) {
  const T* p = reinterpret_cast<const T*>(r.p) + i * r.row + h * r.head + lane * (D / 32);
  if constexpr (D == 128) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    const float2 a = Half16<T>::unpack(u.x), b = Half16<T>::unpack(u.y);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  } else {
    const float2 a = Half16<T>::unpack(__ldg(reinterpret_cast<const uint32_t*>(p)));
    x[0] = a.x, x[1] = a.y;
  }
}
template <typename T, int D>
__device__ __forceinline__ void store_row(const Rows& r, int64_t i, int h, int lane, const float (&x)[D / 32]) {
  T* p = reinterpret_cast<T*>(r.p) + i * r.row + h * r.head + lane * (D / 32);
  if constexpr (D == 128) {
    *reinterpret_cast<uint2*>(p) = make_uint2(Half16<T>::pack(x[0], x[1]), Half16<T>::pack(x[2], x[3]));
  } else {
    *reinterpret_cast<uint32_t*>(p) = Half16<T>::pack(x[0], x[1]);
  }
}
template <int E>
__device__ __forceinline__ float dot(const float (&a)[E], const float (&b)[E]) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s = fmaf(a[e], b[e], s);
  return warp_sum(s);
}

// the keys that row i sees, [lo, hi)
__device__ __forceinline__ int2 keys_of(const PackedParams& p, int i) {
  const int lo = max(max(__ldg(p.start + i), 0), i - p.window + 1);
  const int hi = min(i + 1, __ldg(p.end + i));
  return make_int2(lo, hi);
}
// the queries that see key row j, [j, hi)
__device__ __forceinline__ int queries_of(const PackedParams& p, int j) {
  const int64_t by_window = (int64_t)j + p.window;
  return (int)min((int64_t)min(__ldg(p.end + j), p.N), by_window);
}

template <typename T, int D>
__device__ __forceinline__ void fwd_row(const PackedParams& p, int i, int h, int lane) {
  constexpr int E = D / 32;
  const int2 key = keys_of(p, i);
  if (key.y <= key.x) return;
  const int g = h / (p.H / p.KV);
  float q[E], acc[E] = {};
  load_row<T, D>(p.q, i, h, lane, q);
  float m = -INFINITY, l = 0.f;
  for (int j = key.x; j < key.y; ++j) {
    float k[E], v[E];
    load_row<T, D>(p.k, j, g, lane, k);
    load_row<T, D>(p.v, j, g, lane, v);
    const float x = dot(q, k) * p.scale_log2;
    if (x > m) {  // the same in every lane
      const float a = exp2f(m - x);
      l *= a;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= a;
      m = x;
    }
    const float w = exp2f(x - (m == -INFINITY ? 0.f : m));  // a score of -inf has weight 0 also before any other
    l += w;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, v[e], acc[e]);
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] *= inv;
  store_row<T, D>(p.o, i, h, lane, acc);
  if (lane == 0) p.lse[(int64_t)h * p.N + i] = (m + log2f(l)) * kLn2;
}

template <typename T, int D>
__device__ __forceinline__ void dq_row(const PackedParams& p, int i, int h, int lane, float delta) {
  constexpr int E = D / 32;
  const int2 key = keys_of(p, i);
  if (key.y <= key.x) return;
  const int g = h / (p.H / p.KV);
  float q[E], d[E], acc[E] = {};
  load_row<T, D>(p.q, i, h, lane, q);
  load_row<T, D>(p.dout, i, h, lane, d);
  const float lse2 = p.lse[(int64_t)h * p.N + i] * kLog2e;
  for (int j = key.x; j < key.y; ++j) {
    float k[E], v[E];
    load_row<T, D>(p.k, j, g, lane, k);
    load_row<T, D>(p.v, j, g, lane, v);
    const float w = exp2f(dot(q, k) * p.scale_log2 - lse2);
    const float ds = w * (dot(d, v) - delta);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(ds, k[e], acc[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] *= p.scale;
  store_row<T, D>(p.dq, i, h, lane, acc);
}

template <typename T, int D>
__device__ __forceinline__ void dkv_row(const PackedParams& p, int j, int g, int lane) {
  constexpr int E = D / 32;
  const int hi = queries_of(p, j), group = p.H / p.KV;
  if (hi <= j || __ldg(p.start + j) > j) return;
  float k[E], v[E], dk[E] = {}, dv[E] = {};
  load_row<T, D>(p.k, j, g, lane, k);
  load_row<T, D>(p.v, j, g, lane, v);
  for (int h = g * group; h < (g + 1) * group; ++h) {
    for (int i = j; i < hi; ++i) {
      float q[E], d[E];
      load_row<T, D>(p.q, i, h, lane, q);
      load_row<T, D>(p.dout, i, h, lane, d);
      const int64_t at = (int64_t)h * p.N + i;
      const float w = exp2f(dot(q, k) * p.scale_log2 - __ldg(p.lse + at) * kLog2e);
      const float ds = w * (dot(d, v) - p.delta[at]);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        dv[e] = fmaf(w, d[e], dv[e]);
        dk[e] = fmaf(ds, q[e], dk[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) dk[e] *= p.scale;
  store_row<T, D>(p.dk, j, g, lane, dk);
  store_row<T, D>(p.dv, j, g, lane, dv);
}

constexpr int kRowWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32) fwd_rows_kernel(PackedParams p) {
  const int i = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (i < p.N) fwd_row<T, D>(p, i, blockIdx.y, threadIdx.x & 31);
}
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32) dq_rows_kernel(PackedParams p) {
  const int i = blockIdx.x * kRowWarps + (threadIdx.x >> 5), h = blockIdx.y, lane = threadIdx.x & 31;
  if (i >= p.N) return;
  float o[D / 32], d[D / 32];
  load_row<T, D>(p.o, i, h, lane, o);
  load_row<T, D>(p.dout, i, h, lane, d);
  const float delta = dot(o, d);
  if (lane == 0) p.delta[(int64_t)h * p.N + i] = delta;
  dq_row<T, D>(p, i, h, lane, delta);
}
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32) dkv_rows_kernel(PackedParams p) {
  const int j = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (j < p.N) dkv_row<T, D>(p, j, blockIdx.y, threadIdx.x & 31);
}

// ---------------------------------------------------------------------------------------- host side
void check_rows(const torch::Tensor& t, const char* what, const char* name, int64_t N, int64_t heads, int64_t D,
                const torch::Tensor& like) {
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(0) == N && t.size(1) == heads && t.size(2) == D, what, ": ", name,
                    " must be [", std::to_string(N), ", ", std::to_string(heads), ", ", std::to_string(D), "]");
  TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type(), what, ": ", name, " has another type than q");
  TORCH_CHECK_VALUE(t.device() == like.device(), what, ": ", name, " is on another device than q");
  TORCH_CHECK_VALUE(t.stride(2) == 1, what, ": ", name, " needs contiguous heads (stride 1 in the last dimension)");
  // 16-byte rows for vector and TMA access; a stride of a dimension of one entry is never used
  TORCH_CHECK_VALUE((N <= 1 || (t.stride(0) >= D && t.stride(0) % 8 == 0)) &&
                        (heads <= 1 || (t.stride(1) >= D && t.stride(1) % 8 == 0)),
                    what, ": ", name, " needs row and head strides that are multiples of 8 elements and at least ", std::to_string(D));
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, what, ": ", name,
                    " must start on a 16-byte boundary");
}

Rows rows_of(const torch::Tensor& t) {
  return Rows{t.data_ptr(), t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2),
              t.size(1) > 1 ? t.stride(1) : t.size(2)};
}

torch::Tensor out_rows(const c10::optional<torch::Tensor>& t, const char* what, const char* name, int64_t heads,
                       const torch::Tensor& like) {
  // rows of no sequence are left as they were: in a new tensor they are zero
  if (!t.has_value() || !t->defined()) return torch::zeros({like.size(0), heads, like.size(2)}, like.options());
  check_rows(*t, what, name, like.size(0), heads, like.size(2), like);
  at::assert_no_internal_overlap(*t);
  return *t;
}

torch::Tensor stat_rows(const c10::optional<torch::Tensor>& t, const char* what, const char* name, int64_t heads,
                        const torch::Tensor& like, bool zero) {
  if (!t.has_value() || !t->defined()) {
    auto opt = like.options().dtype(at::kFloat);
    return zero ? torch::zeros({heads, like.size(0)}, opt) : torch::empty({heads, like.size(0)}, opt);
  }
  TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == heads &&
                        t->size(1) == like.size(0) && t->is_contiguous(),
                    what, ": ", name, " must be contiguous float32 [", std::to_string(heads), ", ", std::to_string(like.size(0)), "]");
  TORCH_CHECK_VALUE(t->device() == like.device(), what, ": ", name, " is on another device than q");
  return *t;
}

PackedParams common_params(const char* what, const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                           const torch::Tensor& start, const torch::Tensor& end, int64_t window, double scale) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3, what, ": q, k and v must be [rows, heads, dim]");
  const int64_t N = q.size(0), H = q.size(1), D = q.size(2), KV = k.size(1);
  TORCH_CHECK_VALUE(D == 64 || D == 128, what, ": head dim must be 64 or 128, got ", std::to_string(D));
  TORCH_CHECK_VALUE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, what,
                    ": q must be bfloat16 or float16");
  TORCH_CHECK_VALUE(H >= 1 && KV >= 1 && H % KV == 0, what, ": ", std::to_string(H), " heads cannot share ", std::to_string(KV),
                    " kv heads");
  TORCH_CHECK_VALUE(H <= 65535 && N < (int64_t(1) << 30), what, ": too many rows or heads");
  check_rows(q, what, "q", N, H, D, q);
  check_rows(k, what, "k", N, KV, D, q);
  check_rows(v, what, "v", N, KV, D, q);
  for (const torch::Tensor* b : {&start, &end}) {
    TORCH_CHECK_VALUE(b->scalar_type() == at::kInt && b->dim() == 1 && b->size(0) == N && b->is_contiguous(), what,
                      ": start and end must be contiguous int32 [", std::to_string(N), "]");
    TORCH_CHECK_VALUE(b->device() == q.device(), what, ": start and end must be on q's device");
  }
  TORCH_CHECK_VALUE(window >= 0, what, ": window must not be negative (0: none)");
  TORCH_CHECK_VALUE(std::isfinite(scale) && scale > 0, what, ": scale must be a positive number");
  PackedParams p{};
  p.N = (int)N;
  p.H = (int)H;
  p.KV = (int)KV;
  p.window = (int)(window == 0 ? N : std::min(window, N));
  p.scale = (float)scale;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.q = rows_of(q);
  p.k = rows_of(k);
  p.v = rows_of(v);
  p.start = start.data_ptr<int>();
  p.end = end.data_ptr<int>();
  return p;
}

template <typename F>
void by_type(const torch::Tensor& q, F&& f) {
  const bool wide = q.size(2) == 128;
  if (q.scalar_type() == at::kBFloat16) {
    wide ? f(__nv_bfloat16{}, std::integral_constant<int, 128>{}) : f(__nv_bfloat16{}, std::integral_constant<int, 64>{});
  } else {
    wide ? f(__half{}, std::integral_constant<int, 128>{}) : f(__half{}, std::integral_constant<int, 64>{});
  }
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor> packed_attn_fwd(const torch::Tensor& q, const torch::Tensor& k,
                                                         const torch::Tensor& v, const torch::Tensor& start,
                                                         const torch::Tensor& end, int64_t window, double scale,
                                                         c10::optional<torch::Tensor> out_,
                                                         c10::optional<torch::Tensor> lse_) {
  const char* what = "packed attention_fwd";
  PackedParams p = common_params(what, q, k, v, start, end, window, scale);
  torch::Tensor out = out_rows(out_, what, "out", p.H, q);
  torch::Tensor lse = stat_rows(lse_, what, "lse", p.H, q, true);
  for (const torch::Tensor* t : {&q, &k, &v}) at::assert_no_overlap(out, *t);
  TORCH_CHECK_VALUE(q.is_cuda(), what, ": q must be on a CUDA device");
  if (p.N == 0) return {out, lse};
  p.o = rows_of(out);
  p.lse = lse.data_ptr<float>();
  c10::cuda::CUDAGuard g(q.device());
  auto st = at::cuda::getCurrentCUDAStream();
  by_type(q, [&](auto t, auto d) {
    fwd_rows_kernel<decltype(t), d()><<<dim3((unsigned)((p.N + kRowWarps - 1) / kRowWarps), (unsigned)p.H), kRowWarps * 32, 0, st>>>(p);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {out, lse};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> packed_attn_bwd(
    const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& out,
    const torch::Tensor& lse, const torch::Tensor& dout, const torch::Tensor& start, const torch::Tensor& end,
    int64_t window, double scale, c10::optional<torch::Tensor> dq_, c10::optional<torch::Tensor> dk_,
    c10::optional<torch::Tensor> dv_, c10::optional<torch::Tensor> delta_) {
  const char* what = "packed attention_bwd";
  PackedParams p = common_params(what, q, k, v, start, end, window, scale);
  const int64_t N = p.N, H = p.H, KV = p.KV, D = q.size(2);
  check_rows(out, what, "out", N, H, D, q);
  check_rows(dout, what, "dout", N, H, D, q);
  stat_rows(lse, what, "lse", H, q, false);
  torch::Tensor dq = out_rows(dq_, what, "dq", H, q), dk = out_rows(dk_, what, "dk", KV, q),
                dv = out_rows(dv_, what, "dv", KV, q);
  torch::Tensor delta = stat_rows(delta_, what, "delta", H, q, false);
  for (const torch::Tensor* r : {&dq, &dk, &dv})
    for (const torch::Tensor* t : {&q, &k, &v, &out, &dout}) at::assert_no_overlap(*r, *t);
  TORCH_CHECK_VALUE(q.is_cuda(), what, ": q must be on a CUDA device");
  if (N == 0) return {dq, dk, dv};
  p.o = rows_of(out);
  p.dout = rows_of(dout);
  p.dq = rows_of(dq);
  p.dk = rows_of(dk);
  p.dv = rows_of(dv);
  p.lse = lse.data_ptr<float>();
  p.delta = delta.data_ptr<float>();
  c10::cuda::CUDAGuard g(q.device());
  auto st = at::cuda::getCurrentCUDAStream();
  by_type(q, [&](auto t, auto d) {
    const unsigned x = (unsigned)((N + kRowWarps - 1) / kRowWarps);
    dq_rows_kernel<decltype(t), d()><<<dim3(x, (unsigned)H), kRowWarps * 32, 0, st>>>(p);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    dkv_rows_kernel<decltype(t), d()><<<dim3(x, (unsigned)KV), kRowWarps * 32, 0, st>>>(p);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dq, dk, dv};
}

}  // namespace br
