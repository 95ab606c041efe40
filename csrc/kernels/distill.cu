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
// The row is read once and kept in registers, as 16-byte vectors of the type it came in: by one block of 256
// threads up to 16 KB, else by 512 threads per 64 KB in a cluster of up to 8 blocks, which exchange their partial
// maxima and sums through distributed shared memory; longer rows are read once per pass, again from L2. Bytes
// bound the call (each logit in and out once); next to that is the exponential unit, 16 results per SM and
// cycle: a value that both passes need costs two of them. p and P therefore come from one exponential where t is
// 1 (they are the same) or 2 (exp(x) is the square of exp(x / 2), which doubles a relative error of 2^-22).
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

constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

enum Mode : int {
  kSoft,    // alpha = 1: the teacher alone
  kSame,    // teacher and target, t = 1
  kSquare,  // teacher and target, t = 2
  kHard,    // teacher and target, any other t
};

struct DistillParams {
  int64_t ld, ldg;  // row strides of the logits and of the gradient
  int V, K;
  const int* ids;  // [M, K]
  const void* teacher;
  int teacher_type;  // 0 fp32, 1 bf16, 2 fp16
  int64_t ld_ids, ld_teacher;
  const int* targets;  // [M] or null
  float cap, inv_cap, inv_t, t, alpha, scale;
  int use_cap;     // the softcap bounds the logits: exponentials are taken relative to it, without a maximum
  int cluster;     // blocks of a row
  float* rows;     // [M]
  int* status;
};

// ---- 16-byte vectors of logits
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static constexpr uint32_t kMinusInf = 0xff800000u;
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float round(float x) { return x; }
};
template <typename T>
struct Vec {
  static constexpr int E = 8;
  static constexpr uint32_t kMinusInf = Half16<T>::kFormat ? 0xff80ff80u : 0xfc00fc00u;
  static __device__ __forceinline__ float one(T x) { return static_cast<float>(x); }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = Half16<T>::unpack(w[k]);
      f[2 * k] = a.x, f[2 * k + 1] = a.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(Half16<T>::pack(f[0], f[1]), Half16<T>::pack(f[2], f[3]), Half16<T>::pack(f[4], f[5]),
                      Half16<T>::pack(f[6], f[7]));
  }
  static __device__ __forceinline__ T round(float x) { return static_cast<T>(x); }
};

template <typename T>
__device__ __forceinline__ void store_vec(T* at, bool aligned, const float (&f)[Vec<T>::E]) {
  if (aligned) {
    __stcs(reinterpret_cast<uint4*>(at), Vec<T>::pack(f));
  } else {
#pragma unroll
    for (int e = 0; e < Vec<T>::E; ++e) at[e] = Vec<T>::round(f[e]);
  }
}

__device__ __forceinline__ float load_teacher(const DistillParams& p, int64_t i) {
  if (p.teacher_type == 0) return reinterpret_cast<const float*>(p.teacher)[i];
  if (p.teacher_type == 1) return static_cast<float>(reinterpret_cast<const __nv_bfloat16*>(p.teacher)[i]);
  return static_cast<float>(reinterpret_cast<const __half*>(p.teacher)[i]);
}

__device__ __forceinline__ float2 peer_pair(const float2* mine, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(cluster_map(mine, rank))
               : "memory");
  return v;
}

// NV > 0: NT x NV vectors per block, kept in registers. NV = 0: any number, read in each pass.
template <typename T, int NT, int NV, int MODE>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_kernel(const T* logits, T* grad, const DistillParams p) {
  constexpr int E = Vec<T>::E, kHeld = NV > 0 ? NV : 1;
  extern __shared__ float sm[];  // q [K], l at the ids [K], ids [K]
  __shared__ float2 red[NT / 32];
  __shared__ float2 part[2];  // this block's maximum, and its sums; read by the other blocks of the cluster
  __shared__ float head[6];   // from warp 0: q's part of kl, sum of q, target's logit; target id, entries there
  float* s_q = sm;
  float* s_l = sm + p.K;
  int* s_id = reinterpret_cast<int*>(sm + 2 * p.K);
  asm volatile("griddepcontrol.launch_dependents;");
  const int cs = p.cluster, rank = cs > 1 ? (int)cluster_rank() : 0;
  const int64_t row = blockIdx.x / cs;
  const T* L = logits + row * p.ld;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the row: edge elements before its first 16-byte boundary, nvec whole vectors, edge elements behind them
  const int before = (int)((16 - (reinterpret_cast<uintptr_t>(L) & 15)) % 16 / sizeof(T)), n_head = min(before, p.V);
  const int nvec = (p.V - n_head) / E, tail = n_head + nvec * E;
  const int edges = n_head + p.V - tail;  // at most 2 (E - 1): one for each of the first threads of the row
  const bool has_edge = rank == 0 && tid < edges;
  const int edge_at = tid < n_head ? tid : tail + tid - n_head;
  const float edge = has_edge ? Vec<T>::one(L[edge_at]) : -INFINITY;

  // vectors of this thread: the v-th is (rank NV + v) NT + tid, or every cs NT-th. f(vector, its first element)
  uint4 held[kHeld];
  auto each = [&](auto&& f) {
    if constexpr (NV > 0) {
#pragma unroll
      for (int v = 0; v < NV; ++v) f(held[v], ((rank * NV + v) * NT + tid) * E + n_head);
    } else {
      for (int64_t i = (int64_t)rank * NT + tid; i < nvec; i += (int64_t)cs * NT)
        f(__ldcs(reinterpret_cast<const uint4*>(L + i * E + n_head)), (int)(i * E + n_head));
    }
  };
  if constexpr (NV > 0) {
    constexpr uint32_t kInf = Vec<T>::kMinusInf;  // no weight in any sum
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = (rank * NV + v) * NT + tid;
      held[v] = make_uint4(kInf, kInf, kInf, kInf);
      if (i < nvec) held[v] = __ldcs(reinterpret_cast<const uint4*>(L + (int64_t)i * E + n_head));
    }
  }
  // over the row: pairs of sums or maxima, in the order of warps and blocks
  auto over_row = [&](float a, float b, bool is_max, float2* mine) {
    a = is_max ? warp_max(a) : warp_sum(a);
    b = is_max ? b : warp_sum(b);
    if (lane == 0) red[warp] = make_float2(a, b);
    __syncthreads();
    float2 s = red[0];
#pragma unroll
    for (int w = 1; w < NT / 32; ++w) s = is_max ? make_float2(fmaxf(s.x, red[w].x), 0.f) : make_float2(s.x + red[w].x, s.y + red[w].y);
    if (cs > 1) {
      if (tid == 0) *mine = s;
      cluster_sync_all();
      s = peer_pair(mine, 0);
      for (int r = 1; r < cs; ++r) {
        const float2 o = peer_pair(mine, r);
        s = is_max ? make_float2(fmaxf(s.x, o.x), 0.f) : make_float2(s.x + o.x, s.y + o.y);
      }
    } else {
      __syncthreads();  // red is written again
    }
    return s;
  };

  float m = p.cap;
  if (!p.use_cap) {
    m = edge;
    each([&](const uint4& u, int) {
      float f[E];
      Vec<T>::unpack(u, f);
#pragma unroll
      for (int e = 0; e < E; ++e) m = fmaxf(m, f[e]);
    });
    m = over_row(m, 0.f, true, &part[0]).x;
    if (m == -INFINITY) m = 0.f;  // nothing to take them relative to
  }
  const float k1 = kLog2e * p.inv_t;
  // exp((l - m) / t) and exp(l - m) of two logits; the difference comes first, so that neither large logits nor
  // the lowest finite ones lose it
  const uint64_t m2 = f32x2(m, m), k12 = f32x2(k1, k1), k22 = f32x2(kLog2e, kLog2e);
  auto soft = [&](float a, float b) {
    const float2 x = f32x2_split(mul_f32x2(sub_f32x2(f32x2(a, b), m2), k12));
    return f32x2(exp2f(x.x), exp2f(x.y));
  };
  auto hard = [&](float a, float b, uint64_t e) {
    if constexpr (MODE == kSame) {
      return e;
    } else if constexpr (MODE == kSquare) {
      return mul_f32x2(e, e);
    } else {
      const float2 x = f32x2_split(mul_f32x2(sub_f32x2(f32x2(a, b), m2), k22));
      return f32x2(exp2f(x.x), exp2f(x.y));
    }
  };

  if (warp == 0) {
    // the teacher's distribution over the row's entries, and the target, while the other warps begin their sums
    float um = -INFINITY;
    bool some = false;
    for (int k = lane; k < p.K; k += 32) {
      const int raw = p.ids[row * p.ld_ids + k];
      const bool ok = raw == -1 ? false : index_ok(raw, p.V, p.status);
      const float u = ok ? load_teacher(p, row * p.ld_teacher + k) * p.inv_t : -INFINITY;
      s_id[k] = ok ? raw : -1;
      s_q[k] = u;
      s_l[k] = ok ? Vec<T>::one(L[raw]) : 0.f;
      um = fmaxf(um, u);
      some |= u != -INFINITY;
    }
    um = warp_max(um);
    some = __any_sync(0xffffffffu, some);
    float us = 0.f, a = 0.f, qs = 0.f;
    if (some)
      for (int k = lane; k < p.K; k += 32)
        if (s_id[k] >= 0) us += exp2f((s_q[k] - um) * kLog2e);
    const float log_us = log2f(warp_sum(us)) * kLn2;
    for (int k = lane; k < p.K; k += 32) {
      float q = 0.f;
      if (some && s_id[k] >= 0) {
        const float lq = s_q[k] - um - log_us;
        q = exp2f(lq * kLog2e);
        if (q != 0.f) a += q * (lq - (s_l[k] - m) * p.inv_t);  // log P = (l - m) / t - log of the row's sum
        qs += q;
      }
      s_q[k] = q;
    }
    a = warp_sum(a);
    qs = warp_sum(qs);
    if (lane == 0) {
      int y = -1;
      if constexpr (MODE != kSoft) {
        y = p.targets[row];
        if (y != -1 && !index_ok(y, p.V, p.status)) y = -1;
      }
      head[0] = a;
      head[1] = qs;
      head[2] = y >= 0 ? Vec<T>::one(L[y]) : 0.f;
      head[3] = __int_as_float(y);
      head[4] = some ? 1.f : 0.f;
    }
  }
  uint64_t st2 = soft(edge, -INFINITY), s12 = 0;
  if constexpr (MODE != kSoft) s12 = hard(edge, -INFINITY, st2);
  each([&](const uint4& u, int) {
    float f[E];
    Vec<T>::unpack(u, f);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const uint64_t x = soft(f[e], f[e + 1]);
      st2 = add_f32x2(st2, x);
      if constexpr (MODE != kSoft) s12 = add_f32x2(s12, hard(f[e], f[e + 1], x));
    }
  });
  float st = f32x2_split(st2).x + f32x2_split(st2).y, s1 = f32x2_split(s12).x + f32x2_split(s12).y;
  // in place too: every block of the row has read the columns that the teacher and the target name
  const float2 sums = over_row(st, s1, false, &part[1]);
  if (cs > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // the others' sums are read
  st = sums.x;
  s1 = sums.y;
  const bool dead = st == 0.f, some = head[4] != 0.f;
  float py = 0.f, r = 0.f, loss = 0.f;
  if (some) loss = dead ? INFINITY : p.alpha * p.t * p.t * fmaf(log2f(st) * kLn2, head[1], head[0]);
  if (p.alpha == 0.f) loss = 0.f;
  const int y = __float_as_int(head[3]);
  const float ly = head[2];
  if constexpr (MODE != kSoft) {
    if (y >= 0) {
      py = dead ? 0.f : f32x2_split(hard(ly, ly, soft(ly, ly))).x / s1;
      loss += (1.f - p.alpha) * -(log2f(py + 1e-10f) * kLn2);
      r = (1.f - p.alpha) * (py / (py + 1e-10f));
    }
  }
  if (tid == 0 && rank == 0) p.rows[row] = loss;
  if (grad) {
    T* G = grad + row * p.ldg;
    const bool aligned = ((reinterpret_cast<uintptr_t>(G) ^ reinterpret_cast<uintptr_t>(L)) & 15) == 0;
    const float ct = dead || !some ? 0.f : p.scale * p.alpha * p.t, cs1 = ct == 0.f ? 0.f : ct / st;
    const float ch = dead ? 0.f : p.scale * r, ch1 = ch == 0.f ? 0.f : ch / s1;
    const uint64_t cs12 = f32x2(cs1, cs1), ch12 = f32x2(ch1, ch1);
    auto dense = [&](float a, float b) {
      const uint64_t x = soft(a, b);
      uint64_t g = mul_f32x2(cs12, x);
      if constexpr (MODE != kSoft) g = fma_f32x2(ch12, hard(a, b, x), g);
      return g;
    };
    if constexpr (NV > 0) {
      // the exponentials are taken again: kept from the first pass they would cost twice the logits' registers
#pragma unroll
      for (int v = 0; v < NV; ++v) asm volatile("" : "+r"(held[v].x), "+r"(held[v].y), "+r"(held[v].z), "+r"(held[v].w));
    }
    const uint64_t ic2 = f32x2(p.inv_cap, p.inv_cap), one2 = f32x2(1.f, 1.f);
    auto write = [&](auto capped) {
      auto slope = [&](float a, float b, uint64_t g) {
        if constexpr (decltype(capped)::value) {
          const uint64_t c = mul_f32x2(f32x2(a, b), ic2);
          g = mul_f32x2(g, sub_f32x2(one2, mul_f32x2(c, c)));
        }
        return g;
      };
      each([&](const uint4& u, int e0) {
        float f[E];
        Vec<T>::unpack(u, f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 o = f32x2_split(slope(f[e], f[e + 1], dense(f[e], f[e + 1])));
          f[e] = o.x;
          f[e + 1] = o.y;
        }
        if (e0 < tail) store_vec(G + e0, aligned, f);
      });
      if (has_edge) G[edge_at] = Vec<T>::round(f32x2_split(slope(edge, edge, dense(edge, edge))).x);
    };
    if (p.inv_cap > 0.f) {
      write(std::true_type{});
    } else {
      write(std::false_type{});  // a logit may be -inf, which has no slope
    }
    __syncthreads();
    if (!dead) {
      for (int k = tid; k < p.K + (MODE != kSoft ? 1 : 0); k += NT) {
        const int id = k < p.K ? s_id[k] : y;
        if (id < 0) continue;
        const int vec = (id - n_head) / E;  // the block that wrote the column, of the row's blocks
        const int by = id < n_head || id >= tail ? 0 : NV > 0 ? vec / (NT * kHeld) : vec / NT % cs;
        if (by != rank) continue;
        const float l = k < p.K ? s_l[k] : ly;
        float q = 0.f;
        for (int i = 0; i < p.K; ++i) q += s_id[i] == id ? s_q[i] : 0.f;
        float g = f32x2_split(dense(l, l)).x - ct * q;
        if (MODE != kSoft && id == y) g -= ch;
        const float c = p.inv_cap > 0.f ? l * p.inv_cap : 0.f;
        G[id] = Vec<T>::round(g * fmaf(-c, c, 1.f));
      }
    }
  }
  if (cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // shared memory stays until then
}

// loss = scale * sum of the rows, in one fixed order: one block, each thread's rows in order in 64 bits. Launched
// while the rows' kernel still runs (programmatic dependent launch), so only its own work comes after it.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) sum_rows_kernel(const float* __restrict__ rows, int64_t M, float scale,
                                                               float* __restrict__ loss) {
  __shared__ double red[kSumThreads];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows' kernel has finished
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

// a launch with cluster blocks per cluster, or as a dependent of the launch before it
template <typename... P, typename... A>
void launch(void (*kernel)(P...), int64_t blocks, int threads, size_t smem, cudaStream_t st, int cluster, bool dependent,
            A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim = {(unsigned)cluster, 1, 1};
    ++n;
  }
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

template <typename T, int MODE>
void launch_rows(int64_t M, int64_t V, const T* logits, T* grad, DistillParams& p, int sms, cudaStream_t st) {
  const int64_t vecs = std::max<int64_t>(1, V / Vec<T>::E);
  const size_t smem = (size_t)p.K * 12;
  // a row's blocks: as few as hold it; more while the GPU has SMs to spare and each keeps 256 vectors (4 KB)
  p.cluster = 1;
  while (p.cluster < 8 && (vecs > p.cluster * 4096 || (M * p.cluster * 2 <= sms && vecs > p.cluster * 512))) p.cluster *= 2;
  const int64_t blocks = M * p.cluster;
  TORCH_CHECK_VALUE(blocks < (int64_t(1) << 31), "distill_topk: too many rows");
  if (vecs <= p.cluster * 1024) {
    launch(distill_kernel<T, 256, 4, MODE>, blocks, 256, smem, st, p.cluster, false, logits, grad, p);
  } else if (vecs <= p.cluster * 4096) {
    launch(distill_kernel<T, 512, 8, MODE>, blocks, 512, smem, st, p.cluster, false, logits, grad, p);
  } else {
    launch(distill_kernel<T, 512, 0, MODE>, blocks, 512, smem, st, p.cluster, false, logits, grad, p);
  }
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
  TORCH_CHECK_VALUE(V >= 1 && V < (int64_t(1) << 30) && M < (int64_t(1) << 31), what, "logits out of range");
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
  p.teacher = teacher.data_ptr();
  p.teacher_type = teacher.scalar_type() == at::kFloat ? 0 : teacher.scalar_type() == at::kBFloat16 ? 1 : 2;
  p.cap = (float)cap;
  p.inv_cap = cap > 0 ? (float)(1.0 / cap) : 0.f;
  p.inv_t = (float)(1.0 / temperature);
  p.t = (float)temperature;
  p.alpha = (float)alpha;
  p.scale = (float)scale;
  // exponentials relative to the softcap span e^(-2 cap / t): far above fp32's smallest number up to 2 cap / t = 60
  p.use_cap = cap > 0 && 2 * cap <= 60 * std::min(1.0, temperature);
  p.rows = rows.data_ptr<float>();
  p.status = status_ptr(logits.device().index());
  if (M > 0) {
    int sms = 0;
    C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, logits.device().index()));
    by_float(logits.scalar_type(), [&](auto lt) {
      using T = decltype(lt);
      const T* l = reinterpret_cast<const T*>(logits.data_ptr());
      T* dz = need_grad ? reinterpret_cast<T*>(grad->data_ptr()) : nullptr;
      if (!hard) {
        launch_rows<T, kSoft>(M, V, l, dz, p, sms, st);
      } else if (p.t == 1.f) {
        launch_rows<T, kSame>(M, V, l, dz, p, sms, st);
      } else if (p.t == 2.f) {
        launch_rows<T, kSquare>(M, V, l, dz, p, sms, st);
      } else {
        launch_rows<T, kHard>(M, V, l, dz, p, sms, st);
      }
    });
  }
  launch(sum_rows_kernel, 1, kSumThreads, 0, st, 1, M > 0, rows.data_ptr<float>(), M, p.scale, loss.data_ptr<float>());
  return {loss, rows, grad};
}

}  // namespace br
