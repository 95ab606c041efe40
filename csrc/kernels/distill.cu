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
// Persistent blocks, each with every so-manieth row. Three roles run side by side, so that the row's bytes, the
// entries' chain of dependent loads (ids, then the logits they name) and the arithmetic overlap:
//   producer warp   bulk copies of the coming rows into a ring in shared memory;
//   holding warps   a row from the ring into registers (as it came: 16-byte vectors), its sums, and its gradient;
//   entries' warps  taking the rows in turn, so that each has several rows' time: the teacher's distribution, the target,
//                   their logits; then the row's loss, and once the dense gradient is written the columns that
//                   the entries name.
// Rows of more than 128 KB, and few rows, are split over a cluster of up to 8 blocks, which exchange their partial
// maxima and sums through distributed shared memory. Bytes bound the call (each logit in and out once); next to
// that is the exponential unit, 16 results per SM and cycle: a value that both passes need costs two of them. p
// and P therefore come from one exponential where t is 1 (they are the same) or 2 (exp(x) is the square of
// exp(x / 2), which doubles a relative error of 2^-22).
// On B200: 8191 x 65536 bf16 408 us (5.3 TB/s, 0.80 of the measured copy); 32768 x 8192 bf16 with targets at t = 2
// 302 us (3.6 TB/s; 22 instructions per logit, a row's fixed part among them, fill half of the issue slots, and a
// barrier per row is among the leading stalls), at t = 1.5 415 us (four exponentials per logit), the loss alone 153
// us, the same rows in fp32 607 us. With one block per row, no ring and no entries' warps it was 378 us at t = 2, and
// 690 us for the wide rows.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <string>
#include <tuple>

#include "half_types.cuh"
#include "overlap.h"
#include "status.h"

namespace br {
namespace {

constexpr int kMaxTop = 1024, kMaxTable = 2048;
constexpr int64_t kMaxRowBytes = 1 << 20;  // 8 blocks of 128 KB
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
  int64_t M;
  int V, K;
  const int* ids;  // [M, K]
  const void* teacher;
  int teacher_type;  // 0 fp32, 1 bf16, 2 fp16
  int64_t ld_ids, ld_teacher;
  const int* targets;  // [M] or null
  float cap, inv_cap, inv_t, t, alpha, scale;
  int use_cap;     // the softcap bounds the logits: exponentials are taken relative to it, without a maximum
  int cluster;     // blocks of a row
  int table;       // places of the hash table, a power of two of at least 2 K
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
__device__ __forceinline__ void bulk_row(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

constexpr uint64_t kBudgetNs = 2000000000ull;

// NT threads hold NT x NV vectors of a row, S of them wait in the ring, TW warps see to the entries; MINB blocks per
// SM. CAP: cap > 0.
template <typename T, int NT, int NV, int S, int TW, int MINB, int MODE, bool CAP>
__global__ void __launch_bounds__(NT + 32 * TW + 32, MINB) distill_kernel(const T* logits, T* grad, const DistillParams p) {
  constexpr int E = Vec<T>::E, kWarps = NT / 32, kPiece = NT * NV;  // vectors of a block
  constexpr bool kTwoSums = MODE == kSquare || MODE == kHard;
  extern __shared__ __align__(16) uint8_t smem[];  // [S][kPiece] vectors; per entries' warp q, l, id [K] and a hash table
  __shared__ uint64_t full[S], empty[S], written[TW];
  // A row's sums and maximum, read by the holding warps and by the row's entries' warp after both(n). That warp may still
  // read them while the holding warps go on as far as row n + TW, whose both() it has to reach first: TW + 1 places.
  constexpr int kPlaces = TW + 1;
  __shared__ float red[kPlaces][2][kWarps], s_m[kPlaces];
  __shared__ float redm[2][kWarps];     // by parity of the row: only the holding warps', which meet twice in between
  __shared__ float2 part[2], partm[2];  // this block's sums and maximum, read by the cluster's others
  __shared__ struct { int some, y; float ly; } info[TW];
  __shared__ int s_gave_up;
  volatile int* gave_up = &s_gave_up;
  asm volatile("griddepcontrol.launch_dependents;");
  const int cs = p.cluster, rank = cs > 1 ? (int)cluster_rank() : 0;
  const int64_t first = blockIdx.x / cs, stride = gridDim.x / cs;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    for (int i = 0; i < TW; ++i) mbar_init(&written[i], kWarps);
    s_gave_up = 0;
    fence_barrier_init();
  }
  __syncthreads();
  // A wait that runs out records it and its thread goes on, so that every thread still meets every barrier; no further
  // wait of the block spends its budget then. The device's status word ends no wait: it may hold a bad id, of this
  // launch's own rows among others, and all rows but that one are to come out right.
  auto wait = [&](uint64_t* bar, int64_t phase) {
    if (mbar_wait(bar, phase & 1, kBudgetNs, gave_up)) return true;
    *gave_up = 1;
    atomicCAS(p.status, 0, (int)kErrTimeoutProducer);
    return false;
  };
  // a row: edge elements before its first 16-byte boundary, nvec whole vectors, edge elements behind them
  struct Row {
    const T* L;
    int n_head, nvec, tail;
  };
  auto row_of = [&](int64_t row) {
    Row r;
    r.L = logits + row * p.ld;
    r.n_head = min((int)((16 - (reinterpret_cast<uintptr_t>(r.L) & 15)) % 16 / sizeof(T)), p.V);
    r.nvec = (p.V - r.n_head) / E;
    r.tail = r.n_head + r.nvec * E;
    return r;
  };
  // the barrier's instructions want the whole warp at once, and it comes here from branches for one lane
  auto cluster_barrier = [] {
    __syncwarp();
    cluster_sync_all();
  };
  // with max: the cluster's maximum; else its sums. Every thread of the cluster comes here once per row (and kind)
  auto meet = [&](bool is_max, int par, float2 s) {
    cluster_barrier();
    const float2* mine = is_max ? &partm[par] : &part[par];
    s = peer_pair(mine, 0);
    for (int r = 1; r < cs; ++r) {
      const float2 o = peer_pair(mine, r);
      s = is_max ? make_float2(fmaxf(s.x, o.x), 0.f) : make_float2(s.x + o.x, s.y + o.y);
    }
    return s;
  };
  const bool need_max = !CAP || !p.use_cap;
  const float k1 = kLog2e * p.inv_t;
  const uint64_t k12 = f32x2(k1, k1), k22 = f32x2(kLog2e, kLog2e);
  // exp((l - m) / t) of two logits, and exp(l - m). Behind a softcap the exponent is one multiply-add (its rounding,
  // 2^-24 of at most cap / t log2 e, is that small an error of the result); without one the difference comes first,
  // so that neither large logits nor the lowest finite ones lose it
  auto power = [&](float a, float b, float m, uint64_t k, float kf) {
    const uint64_t l = f32x2(a, b);
    const float2 x = f32x2_split(CAP ? fma_f32x2(l, k, f32x2(-m * kf, -m * kf)) : mul_f32x2(sub_f32x2(l, f32x2(m, m)), k));
    return f32x2(exp2f(x.x), exp2f(x.y));
  };
  auto soft = [&](float a, float b, float m) { return power(a, b, m, k12, k1); };
  auto hard = [&](float a, float b, float m, uint64_t e) {  // e: soft of the same
    if constexpr (MODE == kHard) return power(a, b, m, k22, kLog2e);
    if constexpr (MODE == kSquare) return mul_f32x2(e, e);
    return e;
  };
  // a row's factors of the gradient, from its maximum and sums
  struct Factors {
    float m, ct, ch, cs1, ch1, loss;
    bool dead;
  };
  auto factors = [&](float m, float2 sums, int some, int y, float ly) {
    Factors f;
    const float st = sums.x, s1 = kTwoSums ? sums.y : sums.x;
    f.m = m;
    f.dead = st == 0.f;  // every logit is -inf
    f.ct = f.dead || !some ? 0.f : p.scale * p.alpha * p.t;
    f.cs1 = f.ct == 0.f ? 0.f : f.ct / st;
    f.ch = f.ch1 = f.loss = 0.f;
    if (MODE != kSoft && y >= 0) {
      const float py = f.dead ? 0.f : f32x2_split(hard(ly, ly, m, soft(ly, ly, m))).x / s1;
      f.loss = (1.f - p.alpha) * -(log2f(py + 1e-10f) * kLn2);
      f.ch = p.scale * (1.f - p.alpha) * (py / (py + 1e-10f));
      f.ch1 = f.dead ? 0.f : f.ch / s1;
    }
    return f;
  };
  const uint64_t ic2 = f32x2(-p.inv_cap * p.inv_cap, -p.inv_cap * p.inv_cap), one2 = f32x2(1.f, 1.f);
  // the dense part of the gradient: cs1 exp((l - m) / t) + ch1 exp(l - m), times the softcap's slope (without a softcap
  // a logit may be -inf, which has none)
  auto dense = [&](float a, float b, const Factors& f) {
    const uint64_t x = soft(a, b, f.m), c = f32x2(f.cs1, f.cs1), h = f32x2(f.ch1, f.ch1);
    if constexpr (MODE == kSoft) return mul_f32x2(c, x);
    if constexpr (MODE == kSame) return mul_f32x2(f32x2(f.cs1 + f.ch1, f.cs1 + f.ch1), x);
    if constexpr (MODE == kSquare) return mul_f32x2(x, fma_f32x2(h, x, c));
    return fma_f32x2(h, hard(a, b, f.m, x), mul_f32x2(c, x));
  };
  auto slope = [&](float a, float b) {
    const uint64_t l = f32x2(a, b);
    return CAP ? fma_f32x2(mul_f32x2(l, l), ic2, one2) : one2;
  };
  // the holding warps and the entries' warp of row n: its sums and its entries are there
  auto both = [](int n) {
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(2 + n % TW), "n"(NT + 32) : "memory");
  };  // holding warps and entries' warp

  if (warp < kWarps) {
    int n = 0;
    for (int64_t row = first; row < p.M; row += stride, ++n) {
      const int par = n & 1, place = n % kPlaces;
      const Row r = row_of(row);
      // edge elements: one for each of the first threads of the row's first block
      const bool has_edge = rank == 0 && tid < r.n_head + p.V - r.tail;
      const int edge_at = tid < r.n_head ? tid : r.tail + tid - r.n_head;
      const float edge = has_edge ? Vec<T>::one(r.L[edge_at]) : -INFINITY;
      uint4 held[NV];
      // each pass unpacks the logits and takes the exponentials anew: kept from the pass before (as the compiler would)
      // they cost two to four times the registers of the logits as they came
      auto again = [&] {
#pragma unroll
        for (int v = 0; v < NV; ++v) asm volatile("" : "+r"(held[v].x), "+r"(held[v].y), "+r"(held[v].z), "+r"(held[v].w));
      };
      const int mine = r.nvec - rank * kPiece - warp * 32;  // vectors of this block from this warp's first on
      wait(&full[n % S], n / S);
      {
        constexpr uint32_t kInf = Vec<T>::kMinusInf;  // no weight in any sum
        const uint4* ring = reinterpret_cast<const uint4*>(smem) + n % S * kPiece;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          held[v] = make_uint4(kInf, kInf, kInf, kInf);
          if (v * NT + lane < mine) held[v] = ring[v * NT + tid];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[n % S]);
      }
      float m = p.cap;
      if (need_max) {
        m = edge;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          float f[E];
          Vec<T>::unpack(held[v], f);
#pragma unroll
          for (int e = 0; e < E; ++e) m = fmaxf(m, f[e]);
        }
        m = warp_max(m);
        if (lane == 0) redm[par][warp] = m;
        asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, redm[par][w]);
        if (cs > 1) {
          if (tid == 0) partm[par] = make_float2(m, 0.f);
          m = meet(true, par, make_float2(m, 0.f)).x;
        }
        if (m == -INFINITY) m = 0.f;  // nothing to take them relative to
        again();
        if (tid == 0) s_m[place] = m;
      }
      uint64_t st2 = soft(edge, -INFINITY, m), s12 = 0;
      if constexpr (kTwoSums) s12 = hard(edge, -INFINITY, m, st2);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (v * NT >= mine) break;  // the rest of the warp's vectors are empty
        float f[E];
        Vec<T>::unpack(held[v], f);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const uint64_t x = soft(f[e], f[e + 1], m);
          st2 = add_f32x2(st2, x);
          if constexpr (MODE == kSquare) s12 = fma_f32x2(x, x, s12);
          if constexpr (MODE == kHard) s12 = add_f32x2(s12, hard(f[e], f[e + 1], m, x));
        }
      }
      {
        const float2 a = f32x2_split(st2), b = f32x2_split(s12);
        const float st = warp_sum(a.x + a.y), s1 = kTwoSums ? warp_sum(b.x + b.y) : 0.f;
        if (lane == 0) red[place][0][warp] = st, red[place][1][warp] = s1;
      }
      both(n);
      float2 sums = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sums = make_float2(sums.x + red[place][0][w], sums.y + red[place][1][w]);
      if (cs > 1) {
        if (tid == 0) part[par] = sums;
        sums = meet(false, par, sums);
      }
      if (!grad) continue;
      const Factors f = factors(m, sums, info[n % TW].some, info[n % TW].y, info[n % TW].ly);
      T* G = grad + row * p.ldg;
      const bool aligned = ((reinterpret_cast<uintptr_t>(G) ^ reinterpret_cast<uintptr_t>(r.L)) & 15) == 0;
      again();
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (v * NT >= mine) break;
        float x[E];
        Vec<T>::unpack(held[v], x);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          uint64_t g = dense(x[e], x[e + 1], f);
          if constexpr (CAP) g = mul_f32x2(g, slope(x[e], x[e + 1]));
          const float2 o = f32x2_split(g);
          x[e] = o.x;
          x[e + 1] = o.y;
        }
        if (v * NT + lane < mine) store_vec(G + r.n_head + (int64_t)(rank * kPiece + v * NT + tid) * E, aligned, x);
      }
      if (has_edge) {
        const float g = f32x2_split(dense(edge, edge, f)).x;
        G[edge_at] = Vec<T>::round(CAP ? g * f32x2_split(slope(edge, edge)).x : g);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&written[n % TW]);
    }
  } else if (warp < kWarps + TW) {
    const int turn = warp - kWarps;
    float* s_q = reinterpret_cast<float*>(smem + (size_t)S * kPiece * 16) + (3 * p.K + p.table) * turn;
    float* s_l = s_q + p.K;
    int* s_id = reinterpret_cast<int*>(s_l + p.K);
    int* table = s_id + p.K;
    // the columns that the entries and the target of a row name, once its dense gradient is written
    auto patch = [&](int64_t row, const Factors& f, int y, float ly) {
      if (f.dead) return;
      const Row r = row_of(row);
      T* G = grad + row * p.ldg;
      for (int k = lane; k < p.K + (MODE != kSoft ? 1 : 0); k += 32) {
        const int id = k < p.K ? s_id[k] : y;
        if (id < 0) continue;
        const int by = id < r.n_head || id >= r.tail ? 0 : (id - r.n_head) / E / kPiece;  // the block that has the column
        if (by != rank) continue;
        const float l = k < p.K ? s_l[k] : ly;
        float q = k < p.K ? s_q[k] : 0.f;
        if (k == p.K) {  // the target's own column: an entry that names it has all the column's mass
          for (int i = 0; i < p.K; ++i)
            if (s_id[i] == id) q = s_q[i];
        }
        float g = f32x2_split(dense(l, l, f)).x;
        if (f.ct != 0.f) g -= f.ct * q;  // without weight the teacher may hold anything
        if (MODE != kSoft && id == y) g -= f.ch;
        G[id] = Vec<T>::round(g * f32x2_split(slope(l, l)).x);
      }
      __syncwarp();
    };
    int n = 0;
    for (int64_t row = first; row < p.M; row += stride, ++n) {
      const int par = n & 1, place = n % kPlaces;
      if (n % TW != turn) {
        if (cs > 1) {  // every thread of the cluster meets
          if (need_max) meet(true, par, make_float2(0.f, 0.f));
          meet(false, par, make_float2(0.f, 0.f));
        }
        continue;
      }
      // ---- the row's entries
      const T* L = logits + row * p.ld;
      int y = -1;
      float ly = 0.f;
      if constexpr (MODE != kSoft) {
        y = p.targets[row];
        if (y != -1 && !index_ok(y, p.V, p.status)) y = -1;
        ly = y >= 0 ? Vec<T>::one(L[y]) : 0.f;
      }
      float um = -INFINITY, lm = -INFINITY;
      bool some = false;
      for (int k = lane; k < p.K; k += 32) {
        const int raw = p.ids[row * p.ld_ids + k];
        const float teacher = load_teacher(p, row * p.ld_teacher + k);
        const bool ok = raw == -1 ? false : index_ok(raw, p.V, p.status);
        const float u = ok ? teacher * p.inv_t : -INFINITY;
        const float l = ok ? Vec<T>::one(L[raw]) : -INFINITY;
        s_id[k] = ok ? raw : -1;
        s_q[k] = u;
        s_l[k] = l;
        um = fmaxf(um, u);
        lm = fmaxf(lm, l);
        some |= u != -INFINITY;
      }
      um = warp_max(um);
      lm = warp_max(lm);
      if (lm == -INFINITY) lm = 0.f;
      some = __any_sync(0xffffffffu, some);
      float us = 0.f;
      if (some)
        for (int k = lane; k < p.K; k += 32)
          if (s_id[k] >= 0) us += exp2f((s_q[k] - um) * kLog2e);
      const float log_us = log2f(warp_sum(us)) * kLn2;
      // kl = sum of q (log q - (l - lm) / t) + sum of q ((m - lm) / t + log of the row's sum)
      float ent = 0.f, qs = 0.f;
      for (int k = lane; k < p.K; k += 32) {
        float q = 0.f;
        if (some && s_id[k] >= 0) {
          const float lq = s_q[k] - um - log_us;
          q = exp2f(lq * kLog2e);
          if (q != 0.f) ent += q * (lq - (s_l[k] - lm) * p.inv_t);
          qs += q;
        }
        s_q[k] = q;
      }
      ent = warp_sum(ent);
      qs = warp_sum(qs);
      // do two entries name the same column? each id goes into an open-addressed table, where it meets its like
      bool twice = false;
      for (int k = lane; k < p.table; k += 32) table[k] = -1;
      __syncwarp();
      for (int k = lane; k < p.K; k += 32) {
        const int id = s_id[k];
        if (id < 0) continue;
        for (int at = (int)((uint32_t)id * 2654435761u >> 7) & (p.table - 1);; at = (at + 1) & (p.table - 1)) {
          const int was = atomicCAS(&table[at], -1, id);
          twice |= was == id;
          if (was == -1 || was == id) break;  // at most half of the places are taken
        }
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, twice)) {
        // give each entry the mass of all that name its column, added in the order of their places
        for (int k = lane; k < p.K; k += 32) {
          float q = 0.f;
          for (int i = 0; i < p.K; ++i) q += s_id[i] == s_id[k] ? s_q[i] : 0.f;
          reinterpret_cast<float*>(table)[k] = q;
        }
        __syncwarp();
        for (int k = lane; k < p.K; k += 32) s_q[k] = reinterpret_cast<float*>(table)[k];
      }
      if (lane == 0) info[turn].some = some, info[turn].y = y, info[turn].ly = ly;
      // ---- its sums
      if (need_max && cs > 1) meet(true, par, make_float2(0.f, 0.f));
      both(n);
      float2 sums = make_float2(0.f, 0.f);
      for (int w = 0; w < kWarps; ++w) sums = make_float2(sums.x + red[place][0][w], sums.y + red[place][1][w]);
      if (cs > 1) sums = meet(false, par, sums);
      const float m = need_max ? s_m[place] : p.cap;
      const Factors f = factors(m, sums, some, y, ly);
      if (lane == 0 && rank == 0) {
        float loss = f.loss;
        if (some && p.alpha != 0.f)
          loss += f.dead ? INFINITY : p.alpha * p.t * p.t * fmaf((m - lm) * p.inv_t + log2f(sums.x) * kLn2, qs, ent);
        p.rows[row] = loss;
      }
      if (grad) {
        wait(&written[turn], n / TW);
        patch(row, f, y, ly);
      }
    }
  } else {
    // the producer: this block's whole vectors of each row, S rows ahead; none any more once a wait has run out
    int issued = 0;
    auto load = [&](int64_t row, int n) {
      issued = n + 1;
      const Row r = row_of(row);
      const int count = max(0, min(r.nvec - rank * kPiece, kPiece));
      mbar_arrive_expect_tx(&full[n % S], count * 16);
      if (count > 0)
        bulk_row(smem + (size_t)(n % S) * kPiece * 16, r.L + r.n_head + (int64_t)rank * kPiece * E, count * 16, &full[n % S]);
    };
    if (lane == 0)
      for (int n = 0; n < S; ++n)
        if (first + n * stride < p.M) load(first + n * stride, n);
    int n = 0;
    for (int64_t row = first; row < p.M; row += stride, ++n) {
      if (cs > 1) {
        if (need_max) cluster_barrier();
        cluster_barrier();
      }
      if (lane == 0 && row + S * stride < p.M && !*gave_up && wait(&empty[n % S], n / S)) load(row + S * stride, n + S);
      __syncwarp();
    }
    // the block's shared memory stays until the last copies have landed
    if (lane == 0)
      for (int n = max(0, issued - S); n < issued; ++n) mbar_wait(&full[n % S], (n / S) & 1, kBudgetNs, nullptr);
    __syncwarp();
  }
  if (cs > 1) cluster_barrier();  // the others may still read this block's sums
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

// a kernel's attributes belong to a device: f runs once for each device that the kernel is used on
template <auto kernel, typename F>
void once_per_device(int device, F&& f) {
  static std::atomic<uint64_t> done{0};
  TORCH_CHECK(device >= 0 && device < 64, "bad device index");
  if (!(done.load(std::memory_order_acquire) >> device & 1)) {
    f();
    done.fetch_or(uint64_t(1) << device, std::memory_order_release);
  }
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

template <typename T, int NT, int NV, int S, int TW, int MINB, int MODE, bool CAP>
void launch_held(const T* logits, T* grad, const DistillParams& p, int device, int sms, cudaStream_t st) {
  auto* kernel = distill_kernel<T, NT, NV, S, TW, MINB, MODE, CAP>;
  const size_t smem = (size_t)S * NT * NV * 16 + TW * ((size_t)p.K * 12 + (size_t)p.table * 4);
  once_per_device<distill_kernel<T, NT, NV, S, TW, MINB, MODE, CAP>>(device, [&] {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        S * NT * NV * 16 + TW * (kMaxTop * 12 + kMaxTable * 4)));
  });
  // persistent: as many blocks as run at once, whole clusters, no more than rows
  const int64_t groups = std::max<int64_t>(1, (int64_t)sms * MINB / p.cluster);
  launch(kernel, std::min<int64_t>(p.M, groups) * p.cluster, NT + 32 * TW + 32, smem, st, p.cluster, false, logits, grad, p);
}

template <typename T, int MODE, bool CAP>
void launch_rows(const T* logits, T* grad, DistillParams& p, int device, int sms, cudaStream_t st) {
  const int64_t vecs = std::max(1, p.V / Vec<T>::E);
  // a row's blocks: as few as hold it in 128 KB each; more while the GPU has SMs to spare and each keeps 512 vectors (8 KB)
  p.cluster = 1;
  while (p.cluster < 8 && (vecs > p.cluster * 8192 || (p.M * p.cluster * 2 <= sms && vecs > p.cluster * 1024)))
    p.cluster *= 2;
  if (vecs <= p.cluster * 1024) {  // 16 KB per block
    launch_held<T, 128, 8, 3, 3, 4, MODE, CAP>(logits, grad, p, device, sms, st);
  } else if (vecs <= p.cluster * 4096) {  // 64 KB
    launch_held<T, 512, 8, 2, 2, 1, MODE, CAP>(logits, grad, p, device, sms, st);
  } else {  // 128 KB
    launch_held<T, 512, 16, 1, 2, 1, MODE, CAP>(logits, grad, p, device, sms, st);
  }
}

template <typename T>
void launch_rows_mode(bool hard, const T* logits, T* grad, DistillParams& p, int device, int sms, cudaStream_t st) {
  auto with = [&](auto cap) {
    constexpr bool C = decltype(cap)::value;
    if (!hard) {
      launch_rows<T, kSoft, C>(logits, grad, p, device, sms, st);
    } else if (p.t == 1.f) {
      launch_rows<T, kSame, C>(logits, grad, p, device, sms, st);
    } else if (p.t == 2.f) {
      launch_rows<T, kSquare, C>(logits, grad, p, device, sms, st);
    } else {
      launch_rows<T, kHard, C>(logits, grad, p, device, sms, st);
    }
  };
  p.cap > 0 ? with(std::true_type{}) : with(std::false_type{});
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
  TORCH_CHECK_VALUE(V >= 1 && M < (int64_t(1) << 31), what, "logits out of range");
  TORCH_CHECK_VALUE(V * logits.element_size() <= kMaxRowBytes, what, "rows of the logits of up to 1 MB, got ",
                    std::to_string(V * logits.element_size()), " bytes");
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
      grad = *grad_;
      // the logits themselves (in place), or apart from them
      if (grad->data_ptr() != logits.data_ptr() || (M > 1 && grad->stride(0) != logits.stride(0)))
        check_output("distill_topk", {"grad", &*grad}, {{"logits", &logits}});
      check_output("distill_topk", {"grad", &*grad}, {{"teacher_ids", &ids}, {"teacher_logits", &teacher}});
      if (has_targets) check_output("distill_topk", {"grad", &*grad}, {{"targets", &*targets}});
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
  p.M = M;
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
  p.table = 32;
  while (p.table < 2 * p.K) p.table *= 2;
  p.rows = rows.data_ptr<float>();
  p.status = status_ptr(logits.device().index());
  if (M > 0) {
    int sms = 0;
    C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, logits.device().index()));
    by_float(logits.scalar_type(), [&](auto lt) {
      using T = decltype(lt);
      const T* l = reinterpret_cast<const T*>(logits.data_ptr());
      T* dz = need_grad ? reinterpret_cast<T*>(grad->data_ptr()) : nullptr;
      launch_rows_mode<T>(hard, l, dz, p, logits.device().index(), sms, st);
    });
  }
  launch(sum_rows_kernel, 1, kSumThreads, 0, st, 1, M > 0, rows.data_ptr<float>(), M, p.scale, loss.data_ptr<float>());
  return {loss, rows, grad};
}

}  // namespace br
