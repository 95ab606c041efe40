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
// Forward: tcgen05 tiles of 128 packed rows by 64 packed keys (described at the kernel). A tile may hold the end of
// one sequence and the start of the next: the tiles are cut by row number, not by sequence, so a batch of
// short sequences fills them as well as one long sequence does, no work list has to be built, and the sequences
// appear only as each row's range of keys. A matrix product multiplies hidden keys by a weight of exactly 0,
// which does nothing unless such a key holds a value that is no number. Keys before the first sequence of a
// work item are overwritten with zeros in shared memory; what else a row does not see is within the item's own
// tiles' rows: a row that came out as no number, and has foreign keys or hidden ones of its own sequence that are
// no numbers there, has those columns computed alone, from its own keys (fwd_row). A row's hidden keys of its own
// sequence are less than 256 rows away, and where the keys that it sees make it no number the computation ends with
// the first that does in all those columns, so the cost stays bounded also where all values are none.
//
// Backward: dQ, then dK/dV, on tcgen05 tiles of the same kind (described at the kernels).
//
// Row by row (the rows that a tile's product spoils): one warp per row and head, 32 keys (or queries) at a time: each
// lane takes the dot products of one of them with the row's vectors, which lie in shared memory, then each lane adds up
// D / 32 columns of all 32. Only columns that came out as no numbers are written again.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <climits>
#include <string>
#include <tuple>
#include <utility>

#include "half_types.cuh"
#include "overlap.h"
#include "status.h"
#include "tma_host.h"

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
  float2* stat;  // backward scratch [H, Np]: (kUp - lse in log2 units, -delta) of each row; (-inf, 0) for rows of no sequence
  // fp16 backward scratch, each value the largest of the row's sequence among the 32 rows that hold it
  float* v_most;   // [KV, Np]: |v|
  float2* d_most;  // [H, Np]: |do| and |delta|
  int Np;        // N rounded up to whole tiles
  uint64_t wait_ns;  // how long a wait of the forward may take: rows by themselves hold a tile up
};

// Powers of two that keep the fp16 backward's 16-bit factors in the normal range. P of a long sequence is far below
// fp16's smallest normal number (2^-14), and dS = P (dP - delta) is as small as the gradients make it; bf16 has fp32's
// range and needs none of this. P goes to its product times 2^kUp (it is at most 1, but for its fp32 error). dS goes to
// its product times 2^up_for(b), where b is at least |dP - delta|: below 2^14 P, so normal down to P = 2^-24 where |dP
// - delta| is b / 16 (dP is a sum of D products, |do| |v| its largest possible value). The factor is undone, exactly,
// on the fp32 sums. It belongs to a row of the output, so that it follows what that row sees and nothing of other
// sequences: in dQ b = |do_i| max |v_j| + |delta_i| over the row's keys, in dK/dV b = max |do_i| |v_j| + max |delta_i|
// over the queries that see the row (and others of its sequence). Rows that are no numbers count as zero there: what
// sees them is no number anyway.
template <typename T>
constexpr bool kScaled = Half16<T>::kFormat == 0;
template <typename T>
constexpr float kUp = kScaled<T> ? 14.f : 0.f;
// The forward's P is exp2(x - m + kRaise) with m the running maximum, which is replaced once it is exceeded by more than
// kGrow in log2 units: rarely, with kGrow far above what the maximum of a block's scores usually gains on the first
// block's. In fp16 P is then at most 2^15 and normal down to 2^-25 of the row's largest weight (with m alone and 2^8
// of room weights below 2^-14 lost bits, and those below 2^-25, as beside one key that takes nearly all, vanished). The
// smaller kGrow costs fp16 8% on 65536 rows in documents (122 -> 132 us) and nothing on longer ones or 64-wide heads.
template <typename T>
constexpr float kRaise = kScaled<T> ? 11.f : 0.f;
template <typename T>
constexpr float kGrow = kScaled<T> ? 4.f : 8.f;
__device__ __forceinline__ float power_of_2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int up_for(float b) {
  const int e = (__float_as_int(b) >> 23) - 127;  // b < 2^(e + 1)
  return b > 0.f ? 13 - max(e, -87) : 0;
}

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
__device__ __forceinline__ bool is_number(float x) { return fabsf(x) < INFINITY; }
// the columns of a row that the tiles' product left as no numbers, and the row as it stands. Its values were written by
// other lanes before a __syncwarp (by bulk copies: before lane 0 had waited for them)
template <typename T, int D>
__device__ __forceinline__ uint32_t spoilt_columns(const Rows& r, int64_t i, int h, int lane, float (&x)[D / 32]) {
  const T* p = reinterpret_cast<const T*>(r.p) + i * r.row + h * r.head + lane * (D / 32);
  uint32_t u[D / 64], need = 0;
  if constexpr (D == 128) {
    const uint2 w = __ldcg(reinterpret_cast<const uint2*>(p));
    u[0] = w.x, u[1] = w.y;
  } else {
    u[0] = __ldcg(reinterpret_cast<const uint32_t*>(p));
  }
#pragma unroll
  for (int e = 0; e < D / 32; e += 2) {
    const float2 f = Half16<T>::unpack(u[e / 2]);
    x[e] = f.x, x[e + 1] = f.y;
    need |= (uint32_t)!is_number(f.x) << e | (uint32_t)!is_number(f.y) << (e + 1);
  }
  return need;
}
// every column that is needed is no number, which nothing that is added to it changes (it may still turn from infinite
// to NaN: which of them such a column holds is not said)
template <int E>
__device__ __forceinline__ bool all_lost(const float (&acc)[E], uint32_t need) {
  bool lost = true;
#pragma unroll
  for (int e = 0; e < E; ++e) lost &= !((need >> e) & 1u) || !is_number(acc[e]);
  return __all_sync(0xffffffffu, lost);
}
// The first and the last of the rows [lo, hi) that hold a value that is no number in one of the heads [h0, h1)
// ((INT_MAX, -1): none). The whole warp.
template <typename T, int D>
__device__ __noinline__ int2 odd_rows(const Rows& r, int h0, int h1, int lo, int hi, int lane) {
  constexpr uint32_t kExp = Half16<T>::kFormat ? 0x7f80u : 0x7c00u;
  int first = INT_MAX, last = -1;
  // lo may be any number where the spans are none; hi is a row
  for (int i = lo < hi ? lo + lane : hi; i < hi; i += 32) {
    bool odd = false;
    for (int h = h0; h < h1; ++h) {
      const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(r.p) + (int64_t)i * r.row + h * r.head);
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 a = __ldg(p + c);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (w[e] & kExp) == kExp || ((w[e] >> 16) & kExp) == kExp;
      }
    }
    if (odd) first = min(first, i), last = i;
  }
  return make_int2(__reduce_min_sync(0xffffffffu, first), __reduce_max_sync(0xffffffffu, last));
}
template <int E>
__device__ __forceinline__ float dot(const float (&a)[E], const float (&b)[E]) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s = fmaf(a[e], b[e], s);
  return warp_sum(s);
}

// x[0..D) in shared memory, as fp32 times f, from the lanes' parts of a row
template <int E>
__device__ __forceinline__ void keep_row(float* x, int lane, const float (&v)[E], float f) {
#pragma unroll
  for (int e = 0; e < E; ++e) x[lane * E + e] = v[e] * f;
}
// one lane's dot product of row (i, h) with x
template <typename T, int D>
__device__ __forceinline__ float dot_row(const Rows& r, int64_t i, int h, const float* x) {
  const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(r.p) + i * r.row + h * r.head);
  float s[2] = {};
#pragma unroll
  for (int c = 0; c < D / 8; ++c) {
    const uint4 a = __ldg(p + c);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = Half16<T>::unpack(w[e]), y = *reinterpret_cast<const float2*>(x + c * 8 + 2 * e);
      s[e & 1] = fmaf(f.x, y.x, fmaf(f.y, y.y, s[e & 1]));
    }
  }
  return s[0] + s[1];
}
// acc += sum of w_u times row (first + u step) of r, w_u lane u's, over the rows u < count
template <typename T, int D>
__device__ __forceinline__ void add_rows(const Rows& r, int first, int step, int count, int h, float w, int lane,
                                         float (&acc)[D / 32]) {
  auto add = [&](int u) {
    float v[D / 32];
    load_row<T, D>(r, first + u * step, h, lane, v);
    const float wu = __shfl_sync(0xffffffffu, w, u);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(wu, v[e], acc[e]);
  };
  if (count == 32) {
#pragma unroll
    for (int u = 0; u < 32; ++u) add(u);  // their loads overlap
  } else {
    for (int u = 0; u < count; ++u) add(u);
  }
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
__device__ __noinline__ void fwd_row(const PackedParams& p, int i, int h, int lane, float* buf) {
  constexpr int E = D / 32;
  const int2 key = keys_of(p, i);
  if (key.y <= key.x) return;
  const int g = h / (p.H / p.KV);
  float q[E], old[E], acc[E] = {};
  const uint32_t need = spoilt_columns<T, D>(p.o, i, h, lane, old);
  load_row<T, D>(p.q, i, h, lane, q);
  keep_row(buf, lane, q, p.scale_log2);
  __syncwarp();
  float m = -INFINITY, l = 0.f;  // l: this lane's keys
  // from the last key on: behind one that is no number there usually are more
  for (int last = key.y - 1; last >= key.x && !all_lost(acc, need); last -= 32) {
    const int j = last - lane, count = min(32, last - key.x + 1);
    const float x = lane < count ? dot_row<T, D>(p.k, j, g, buf) : -INFINITY, most = warp_max(x);
    if (most > m) {
      const float a = exp2f(m - most);
      l *= a;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= a;
      m = most;
    }
    const float w = exp2f(x - (m == -INFINITY ? 0.f : m));  // a score of -inf has weight 0 also before any other
    l += w;
    add_rows<T, D>(p.v, last, -1, count, g, w, lane, acc);
  }
  const float inv = 1.f / warp_sum(l);
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = (need >> e) & 1u ? acc[e] * inv : old[e];
  store_row<T, D>(p.o, i, h, lane, acc);  // its lse is right: hidden scores are not added up
  __syncwarp();
}

template <typename T, int D>
__device__ __noinline__ void dq_row(const PackedParams& p, int i, int h, int half, int lane, float2 stat, float* buf) {
  constexpr int E = D / 32;
  const int2 key = keys_of(p, i);
  if (key.y <= key.x) return;
  const int g = h / (p.H / p.KV);
  float x[E], old[E], acc[E] = {};
  // the other half of the row is the other warp's
  const uint32_t need = lane / 16 == half ? spoilt_columns<T, D>(p.dq, i, h, lane, old) : 0u;
  load_row<T, D>(p.q, i, h, lane, x);
  keep_row(buf, lane, x, p.scale_log2);
  load_row<T, D>(p.dout, i, h, lane, x);
  keep_row(buf + D, lane, x, 1.f);
  __syncwarp();
  for (int last = key.y - 1; last >= key.x && !all_lost(acc, need); last -= 32) {
    const int j = last - lane, count = min(32, last - key.x + 1);
    float ds = 0.f;
    if (lane < count) ds = exp2f(dot_row<T, D>(p.k, j, g, buf) - stat.x) * (dot_row<T, D>(p.v, j, g, buf + D) - stat.y);
    add_rows<T, D>(p.k, last, -1, count, g, ds, lane, acc);
  }
  __syncwarp();
  if (lane / 16 != half) return;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = (need >> e) & 1u ? acc[e] * p.scale : old[e];
  store_row<T, D>(p.dq, i, h, lane, acc);
}

template <typename T, int D>
__device__ __noinline__ void dkv_row(const PackedParams& p, int j, int g, bool want_dk, int lane, float* buf) {
  constexpr int E = D / 32;
  const int hi = queries_of(p, j), group = p.H / p.KV;
  const Rows& to = want_dk ? p.dk : p.dv;
  float x[E], old[E], acc[E] = {};
  const uint32_t need = spoilt_columns<T, D>(to, j, g, lane, old);
  load_row<T, D>(p.k, j, g, lane, x);
  keep_row(buf, lane, x, p.scale_log2);
  load_row<T, D>(p.v, j, g, lane, x);
  keep_row(buf + D, lane, x, 1.f);
  __syncwarp();
  for (int first = j; first < hi && !all_lost(acc, need); first += 32) {
    const int i = first + lane, count = min(32, hi - first);
    for (int h = g * group; h < (g + 1) * group; ++h) {
      float w = 0.f;
      if (lane < count) {
        const float2 st = p.stat[(int64_t)h * p.Np + i];
        w = exp2f(dot_row<T, D>(p.q, i, h, buf) + st.x);
        if (want_dk) w *= dot_row<T, D>(p.dout, i, h, buf + D) + st.y;
      }
      add_rows<T, D>(want_dk ? p.q : p.dout, first, 1, count, h, w, lane, acc);
    }
  }
  const float f = (want_dk ? p.scale : 1.f) * power_of_2(-(int)kUp<T>);  // stat raised the weights
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = (need >> e) & 1u ? acc[e] * f : old[e];
  store_row<T, D>(to, j, g, lane, acc);
  __syncwarp();
}

// the largest of the values (none negative) of a warp's lanes that have the same seq
__device__ __forceinline__ float most_of_seq(float x, int seq) {
  return __uint_as_float(__reduce_max_sync(__match_any_sync(0xffffffffu, seq), __float_as_uint(x)));
}

// v_most: one warp per 32 rows of a kv head. It reads V once; before dQ, in fp16 alone.
constexpr int kNormThreads = 256;
template <typename T, int D>
__global__ void __launch_bounds__(kNormThreads) v_most_kernel(const __grid_constant__ PackedParams p) {
  constexpr int E = D / 32;
  const int groups = p.Np / 32, lane = lane_id();
  const int64_t at = (int64_t)blockIdx.x * (kNormThreads / 32) + warp_id();
  if (at >= (int64_t)groups * p.KV) return;
  const int g = (int)(at / groups), j0 = (int)(at % groups) * 32, j = j0 + lane;
  const int first = j < p.N ? __ldg(p.start + j) : 0;
  const bool real = j < p.N && first <= j && queries_of(p, j) > j;
  const uint32_t read = __ballot_sync(0xffffffffu, real);  // a row of no sequence is not read
  float m = 0.f;
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    if (!((read >> r) & 1u)) continue;
    float v[E];
    load_row<T, D>(p.v, j0 + r, g, lane, v);
    const float s = dot(v, v);
    if (lane == r && s < INFINITY) m = sqrtf(s);
  }
  p.v_most[(int64_t)g * p.Np + j] = most_of_seq(m, real ? first : -1 - lane);
}

// ---------------------------------------------------------------------------------------- forward, tcgen05
// Persistent, one CTA per SM, 384 threads. A work item is two 128-row query tiles A and B that share their keys: two
// heads of one kv head over the same rows where the group of query heads is even, else two neighbouring row
// tiles of one head. The grid has one block per item; a running CTA takes over blocks that have not started
// (clc_request), so items of uneven cost balance over the SMs without a counter in memory that two launches
// would share. Items go from the last rows to the first: in a long sequence the late rows cost most.
//   warp 0     takes items, hands them to the other warps through a two-slot ring, and loads K and V tiles (TMA) into
//              rings;
//   warps 1, 2 issue the MMAs of tile A and of B, by blocks of 64 keys with two score sets (set s = t % 2): S_X = Q_X K_t^T
//              -> TMEM [256X + 64s, +64) fp32; P_X, written there by the softmax warps as 16-bit pairs over S_X, is
//              the A operand of O_X += P_X V_t -> TMEM [256X + 128, +D). Order: PV_X(t), S_X(t+2), so the scores of
//              block t + 1 stand ready while t's softmax runs. One thread for both
//              tiles took 600 to 1000 cycles for a block's twelve MMAs, its waits and commits, twice what they run;
//   warp 3     loads the Q tiles, one lane each;
//   warps 4-11 softmax, one query row per thread (4-7 tile A, 8-11 tile B), and the output through shared memory.
// The two tiles meet only in the K and V rings (a slot is free when both have passed it), so one may be in its next
// item while the other finishes. What an item costs to start and to end (loads, output) hides behind the other tile's
// work only where their blocks differ: two heads over the same rows have the same ones and start and end together,
// and two row tiles' differ by two or so; with short sequences, where an item is few blocks, most of it lies open.
// P is rounded to 16 bits for the product (half a step, relative to each weight, see kRaise); the row sum l adds the
// unrounded fp32 values, the maximum, l and O stay in fp32.
// Bounds: 4 D operations per pair on the tensor core, one exponential per pair (16 per SM and cycle, as long as the
// pair's products at D = 128), and for the 64-key score products 6 KB of shared memory per 128 x 64 x 16 step. On
// B200, several inputs in turn: one prompt of 16384 rows, 8 heads of 128 on 2, 537 us (1024 TFLOP/s); 65536 rows in
// documents of 512 on average, window 1024, 4 x 128, 121 us (2.2 TB/s; an item's start, end and masks weigh as much as
// its nine blocks). 32 rows of 2048, 4 x 128: 163 us, 193 with the fixed-length kernel of attention_tc.cu. On one input
// over and over 128-key blocks with one score set took 482 us instead of 466, and 148 instead of 113 us.
constexpr uint64_t kBudgetNs = 2000000000ull, kDrainNs = 100000000ull;
constexpr int BT = 128;  // rows of a query tile (forward, dQ), keys of a tile (dK/dV)
constexpr int BB = 64;   // keys (forward, dQ) or queries (dK/dV) of a block
constexpr int kAtom = BT * 128;   // 128 rows x 128 bytes, one 128-byte-swizzle atom column of a tile
constexpr int kAtom64 = BB * 128;  // and of a block

// 32 columns of 32 rows on their way to memory: each lane writes its row into the warp's buffer (64-byte rows, 16-byte
// pieces swizzled as the tensor map has it), then one lane sends it off. Rows behind the tensor's end are cut off.
constexpr int kOutBytes = 32 * 64;
__device__ __forceinline__ void out_piece(uint8_t* buf, int lane, int piece, uint4 v) {
  *reinterpret_cast<uint4*>(buf + lane * 64 + ((piece ^ ((lane >> 1) & 3)) << 4)) = v;
}
__device__ __forceinline__ void out_send(const CUtensorMap* m, bool swap, const uint8_t* buf, int col, int head, int row) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(smem_u32(buf)), "r"(col), "r"(swap ? row : head), "r"(swap ? head : row)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void out_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void out_wait_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int D>
struct FwdCfg {
  static constexpr int kTile = BT * D * 2, kBlock = BB * D * 2;
  static constexpr int kK = 5, kV = 4;  // ring depths: K runs two blocks ahead of V
  static constexpr int oQ = 0, oK = 2 * kTile, oV = oK + kK * kBlock;
  static constexpr int oOut = oV + kV * kBlock;  // [8 warps] 32 rows x 32 columns of output on their way
  static constexpr int oBar = oOut + 8 * kOutBytes;
  static constexpr int kSmem = oBar + 448 + 1024;
  static_assert(kSmem <= 232448, "forward shared memory");
};

struct FwdMaps {
  CUtensorMap q, k, v, o;
  int swap;    // bit 0: q's map has its coordinates as (d, row, head), bit 1: k's, bit 2: v's
  int swap_o;  // the same of o's map, whose boxes are 32 rows
};

__device__ __forceinline__ void load_tile(const CUtensorMap* m, bool swap, uint64_t* bar, uint8_t* dst, int head, int row,
                                          int atoms, int atom_bytes) {
  for (int c = 0; c < atoms; ++c)
    tma_load_3d(m, bar, dst + c * atom_bytes, 64 * c, swap ? row : head, swap ? head : row);
}

constexpr int kThreads = 384;
// The backward's blocks are three warpgroups, launched with 168 registers a thread (64512 of an SM's 65536): the first
// one, which loads and issues, gives a part of its share up and the two that hold score rows take it:
// 128 x (104 + 200 + 200) = 64512.
__device__ __forceinline__ void few_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 104;"); }
__device__ __forceinline__ void many_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 200;"); }

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory descriptors of a tile whose rows run along the product's free index (K-major: a step of 16 along D
// is 32 bytes inside an atom) or along its summed one (MN-major: 16 rows are 2048 bytes; atom: bytes of an atom
// column). The address field counts 16 bytes and has no carry into the next, so steps are added to it.
__device__ __forceinline__ uint64_t k_major(const void* tile) { return umma_desc_sw128(smem_u32(tile), 16, 1024); }
__device__ __forceinline__ uint64_t mn_major(const void* tile, uint32_t atom) {
  return umma_desc_sw128(smem_u32(tile), atom, 1024);
}

struct FwdItem {
  int h[2], q0[2];  // head and first row of the query tiles A and B
  int lo[2], hi[2];  // key blocks [lo, hi) of each (empty: no such query tile)
  int kvh;
  __device__ int first() const { return hi[1] > lo[1] ? min(lo[0], lo[1]) : lo[0]; }
  __device__ int last() const { return max(hi[0], hi[1]); }  // one past the last key block
};

// where an item's query tiles are; the key ranges follow from the spans (item_keys) or the ring
__device__ __forceinline__ FwdItem item_rows(int block, int n_blocks, const PackedParams& p) {
  FwdItem I;
  const int item = n_blocks - 1 - block;
  const int group = p.H / p.KV;
  if (group % 2 == 0) {
    const int hp = p.H / 2, tile = item / hp;
    I.h[0] = 2 * (item % hp);
    I.h[1] = I.h[0] + 1;
    I.q0[0] = I.q0[1] = tile * BT;
  } else {
    I.h[0] = I.h[1] = item % p.H;
    I.q0[0] = item / p.H * (2 * BT);
    I.q0[1] = I.q0[0] + BT;
  }
  I.kvh = I.h[0] / group;
  for (int x = 0; x < 2; ++x) {
    I.hi[x] = I.q0[x] < p.N ? (min(I.q0[x] + BT, p.N) - 1) / BB + 1 : 0;
    I.lo[x] = 0;
  }
  return I;
}
// spans never decrease along the rows, so a tile's first row has its first key; returns the first row of the first
// sequence: keys before it are foreign to every row of the item
__device__ __forceinline__ int item_keys(FwdItem& I, const PackedParams& p) {
  for (int x = 0; x < 2; ++x) I.lo[x] = I.hi[x] > 0 ? min(max(keys_of(p, I.q0[x]).x, 0) / BB, I.q0[x] / BB) : 0;
  return __ldg(p.start + I.q0[0]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) fwd_tc_kernel(const __grid_constant__ FwdMaps maps,
                                                        const __grid_constant__ PackedParams p, int* status) {
  using C = FwdCfg<D>;
  constexpr int kAtoms = D / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::oBar);
  uint64_t* q_full = bars + 0;      // [2] per query tile
  uint64_t* q_empty = bars + 2;     // [2]
  uint64_t* s_full = bars + 4;      // [2][2] per query tile and score set
  uint64_t* p_full = bars + 8;      // [2][2]
  uint64_t* pv_done = bars + 12;    // [2] after each block's product with V
  uint64_t* o_done = bars + 48;     // [2] after an item's last one
  uint64_t* o_empty = bars + 14;    // [2]
  uint64_t* item_full = bars + 16;  // [2] ring slots
  uint64_t* item_empty = bars + 18;
  uint64_t* drain = bars + 50;      // [2]
  uint64_t* clc_full = bars + 21;
  uint64_t* k_full = bars + 22;
  uint64_t* k_empty = k_full + C::kK;
  uint64_t* v_full = k_empty + C::kK;
  uint64_t* v_empty = v_full + C::kV;
  static_assert(22 + 2 * (C::kK + C::kV) <= 40, "barrier region");
  // [2][4]: block (-1: the end), first key block of A and of B, first row of A's first sequence
  volatile int* ring = reinterpret_cast<volatile int*>(bars + 40);
  uint8_t* clc_resp = reinterpret_cast<uint8_t*>(bars + 44);  // 16 bytes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 46);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id();
  if (__syncthreads_or(device_failed(status))) return;  // all threads or none: the word may change meanwhile
  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 1);
      mbar_init(&q_empty[x], 1);
      for (int s = 0; s < 2; ++s) {
        mbar_init(&s_full[2 * x + s], 1);
        mbar_init(&p_full[2 * x + s], 128);
      }
      mbar_init(&pv_done[x], 1);
      mbar_init(&o_done[x], 1);
      mbar_init(&o_empty[x], 128);
      mbar_init(&item_full[x], 1);
      mbar_init(&item_empty[x], 12);  // the MMA thread for each tile, two Q loaders, one lane of each softmax warp
    }
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    mbar_init(clc_full, 1);
    for (int i = 0; i < C::kK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);  // both query tiles have passed
    }
    for (int i = 0; i < C::kV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 3) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&](int code) {
    *abort_flag = 1;
    if (status) atomicCAS(status, 0, code);
  };
  auto wait = [&](uint64_t* bar, int phase) { return mbar_wait(bar, phase & 1, p.wait_ns, abort_flag, status); };
  auto item_of = [&](int slot) {
    FwdItem I = item_rows(ring[slot * 4], gridDim.x, p);
    I.lo[0] = ring[slot * 4 + 1];
    I.lo[1] = ring[slot * 4 + 2];
    return I;
  };

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
      int ik = 0, iv = 0, nc = 0;  // K and V blocks loaded so far (ring positions), requests for work
      bool ok = true;
      auto publish = [&](int n, int block, FwdItem& I) {
        volatile int* slot = ring + (n & 1) * 4;
        slot[0] = block;
        if (block >= 0) {
          I = item_rows(block, gridDim.x, p);
          slot[3] = item_keys(I, p);
          slot[1] = I.lo[0];
          slot[2] = I.lo[1];
        }
        mbar_arrive(&item_full[n & 1]);
      };
      FwdItem I, next;
      int block = blockIdx.x;
      publish(0, block, I);
      for (int n = 0; ok && block >= 0; ++n, I = next) {
        fence_async_smem();  // the last answer has been read before the next one is written over it
        clc_request(clc_resp, clc_full);
        ++nc;
        // the next item is handed out as soon as it is known, between this item's loads: the other warps fetch it
        // before they write this one's output
        bool known = false, told = false;
        auto look_ahead = [&](bool now) {
          if (!known) {
            if (now ? !wait(clc_full, n) : !mbar_test(clc_full, n & 1)) return !now;
            block = clc_block(clc_resp);
            known = true;
          }
          if (!told) {
            uint64_t* free = &item_empty[(n + 1) & 1];
            if (n > 0 && (now ? !wait(free, (n - 1) >> 1) : !mbar_test(free, ((n - 1) >> 1) & 1))) return !now;
            publish(n + 1, block, next);
            told = true;
          }
          return true;
        };
        const int t0 = I.first(), t1 = I.last();
        for (int t = t0; ok && t < t1 + 2; ++t) {  // K(t0), K(t0+1), then K(t+2) and V(t) in turn
          if (t < t1) {
            const int st = ik % C::kK;
            if (!wait(&k_empty[st], (ik / C::kK) ^ 1)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&k_full[st], C::kBlock);
            load_tile(&maps.k, maps.swap & 2, &k_full[st], smem + C::oK + st * C::kBlock, I.kvh, t * BB, kAtoms, kAtom64);
            ++ik;
          }
          if (t >= t0 + 2) {
            const int st = iv % C::kV;
            if (!wait(&v_empty[st], (iv / C::kV) ^ 1)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&v_full[st], C::kBlock);
            load_tile(&maps.v, maps.swap & 4, &v_full[st], smem + C::oV + st * C::kBlock, I.kvh, (t - 2) * BB, kAtoms,
                      kAtom64);
            ++iv;
            look_ahead(false);
          }
        }
        ok = ok && look_ahead(true);
      }
      if (!ok) {
        fail(kErrTimeoutProducer);
        // the copies in flight still write to this block's shared memory
        for (int g = max(0, ik - C::kK); g < ik; ++g) mbar_wait(&k_full[g % C::kK], (g / C::kK) & 1, kDrainNs, nullptr);
        for (int g = max(0, iv - C::kV); g < iv; ++g) mbar_wait(&v_full[g % C::kV], (g / C::kV) & 1, kDrainNs, nullptr);
        if (nc > 0) mbar_wait(clc_full, (nc - 1) & 1, kDrainNs, nullptr);
      }
    }
  } else if (warp < 3) {
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_16<T>(BT, BB, false, false);
      constexpr uint32_t idesc_o = umma_idesc_16<T>(BT, D, false, true);
      // where a query tile is: at key block t (its product with V, then the scores of t + 2) of its n-th item [t0, t1),
      // of which it uses [lo, hi)
      struct Place {
        int n, t, t0, t1, lo, hi;
        int kpos, vpos;  // ring positions of the next K and V block
        int nq;          // items begun
        uint32_t np;     // bit s: parity of the uses of score set s
        bool open, pv;   // in an item; the product with V_t (or its passing) is done
        bool end;
      };
      Place w = {};
      const int x = warp - 1;
      const uint32_t tm = tmem + x * 256;
      // the tile's next product, if what it needs is there; true if something was done
      auto step = [&]() {
        if (!w.open) {
          const int slot = w.n & 1;
          if (!mbar_test(&item_full[slot], (w.n >> 1) & 1)) return false;
          if (ring[slot * 4] < 0) {
            w.end = true;
            return true;
          }
          const FwdItem I = item_of(slot);
          mbar_arrive(&item_empty[slot]);
          w.t0 = I.first(), w.t1 = I.last(), w.lo = x ? I.lo[1] : I.lo[0], w.hi = x ? I.hi[1] : I.hi[0];
          w.t = w.t0 - 2;
          w.open = true;
          w.pv = false;
        }
        bool any = false;
        if (!w.pv && w.t >= w.t0) {
          const int t = w.t, st = w.vpos % C::kV, set = t & 1;
          if (!mbar_test(&v_full[st], (w.vpos / C::kV) & 1)) return false;
          if (t >= w.lo && t < w.hi) {  // O += P V_t; an item's first one overwrites O when the last item's has been read
            if (!mbar_test(&p_full[2 * x + set], (w.np >> set) & 1)) return false;
            if (t == w.lo && w.nq > 1 && !mbar_test(&o_empty[x], (w.nq - 2) & 1)) return false;
            w.np ^= 1u << set;
            tc_fence_after();
            const uint64_t v_desc = mn_major(smem + C::oV + st * C::kBlock, kAtom64);
#pragma unroll
            for (int kk = 0; kk < BB / 16; ++kk)
              umma_bf16_ts(tm + 128, tm + set * 64 + kk * 8, v_desc + kk * (2048 >> 4), idesc_o,
                           (t > w.lo || kk > 0) ? 1u : 0u);
            umma_commit(&v_empty[st]);
            umma_commit(&pv_done[x]);
            if (t == w.hi - 1) umma_commit(&o_done[x]);
          } else {
            mbar_arrive(&v_empty[st]);
          }
          ++w.vpos;
          any = true;
        }
        w.pv = true;
        if (w.t + 2 < w.t1) {
          const int t = w.t + 2, st = w.kpos % C::kK, set = t & 1;
          if (!mbar_test(&k_full[st], (w.kpos / C::kK) & 1)) return any;
          if (t >= w.lo && t < w.hi) {  // S = Q K_t^T
            if (t == w.lo) {
              if (!mbar_test(&q_full[x], w.nq & 1)) return any;
              ++w.nq;
            }
            tc_fence_after();
            const uint64_t q_desc = k_major(smem + C::oQ + x * C::kTile), k_desc = k_major(smem + C::oK + st * C::kBlock);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t offq = ((kk >> 2) * kAtom + (kk & 3) * 32) >> 4, offk = ((kk >> 2) * kAtom64 + (kk & 3) * 32) >> 4;
              umma_bf16_ss(tm + set * 64, q_desc + offq, k_desc + offk, idesc_s, kk > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[2 * x + set]);
            umma_commit(&k_empty[st]);
            if (t == w.hi - 1) umma_commit(&q_empty[x]);  // the item's last score product
          } else {
            mbar_arrive(&k_empty[st]);
          }
          ++w.kpos;
        }
        w.pv = false;
        if (++w.t == w.t1) {
          w.open = false;
          ++w.n;
        }
        return true;
      };
      uint64_t since = globaltimer_ns();
      bool ok = true;
      for (uint32_t spin = 0; !w.end;) {
        if (step()) {
          spin = 0;
        } else if ((++spin & 255u) == 0) {
          if (spin == 256) since = globaltimer_ns();
          if (*abort_flag || (status && *reinterpret_cast<const volatile int*>(status)) ||
              globaltimer_ns() - since > p.wait_ns) {
            ok = false;
            break;
          }
        }
      }
      if (!ok) fail(kErrTimeoutMma);
      umma_commit(&drain[x]);
      mbar_wait(&drain[x], 0, kDrainNs, nullptr);
    }
  } else if (warp == 3) {
    const int x = lane_id();
    if (x < 2) {
      tma_prefetch_desc(&maps.q);
      int nq = 0;
      bool ok = true;
      for (int n = 0;; ++n) {
        const int slot = n & 1;
        if (!wait(&item_full[slot], n >> 1)) {
          ok = false;
          break;
        }
        if (ring[slot * 4] < 0) break;
        const FwdItem I = item_of(slot);
        mbar_arrive(&item_empty[slot]);
        if ((x ? I.hi[1] : I.hi[0]) == 0) continue;
        if (nq > 0 && !wait(&q_empty[x], nq - 1)) {  // the previous item's score products have read the tile
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&q_full[x], C::kTile);
        load_tile(&maps.q, maps.swap & 1, &q_full[x], smem + C::oQ + x * C::kTile, x ? I.h[1] : I.h[0],
                  x ? I.q0[1] : I.q0[0], kAtoms, kAtom);
        ++nq;
      }
      if (!ok) {
        fail(kErrTimeoutProducer);
        if (nq > 0) mbar_wait(&q_full[x], (nq - 1) & 1, kDrainNs, nullptr);
      }
    }
    __syncwarp();
  } else {
    const int x = (warp - 4) >> 2, wq = warp & 3, lane = lane_id();
    const int r = wq * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(wq * 32) << 16) + x * 256;
    uint32_t sc = 0;  // bit s: parity of the uses of score set s
    int pv = 0, oc = 0;  // this query tile's products with V, and its finished items, so far
    int vbase = 0;    // ring position of the item's first V block
    uint8_t* out_buf = smem + C::oOut + (warp - 4) * kOutBytes;
    // an item as this thread sees it; `next` is fetched before an item's output is written, so that the spans arrive
    // meanwhile
    struct Work {
      int block, t_lo, t_hi, h, i, t0, z, vfirst;
      int2 key;
    } now, next;
    auto fetch = [&](int n, Work& w) -> bool {
      const int slot = n & 1;
      if (!mbar_wait_warp(&item_full[slot], (n >> 1) & 1, p.wait_ns, abort_flag, status)) {
        fail(kErrTimeoutEpilogue);
        return false;
      }
      w.block = ring[slot * 4];
      if (w.block < 0) return true;
      const FwdItem I = item_of(slot);
      w.z = ring[slot * 4 + 3];
      w.t0 = I.first();
      w.vfirst = vbase;
      vbase += I.last() - w.t0;
      w.t_lo = x ? I.lo[1] : I.lo[0];
      w.t_hi = x ? I.hi[1] : I.hi[0];
      w.h = x ? I.h[1] : I.h[0];
      w.i = (x ? I.q0[1] : I.q0[0]) + r;
      w.key = w.i < p.N ? keys_of(p, w.i) : make_int2(0, 0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      return true;
    };
    bool more = fetch(0, now);
    for (int n = 0; more && now.block >= 0; ++n, now = next) {
      const int t_lo = now.t_lo, t_hi = now.t_hi, h = now.h, i = now.i, t0 = now.t0, z = now.z, vfirst = now.vfirst;
      const int2 key = now.key;
      // rows of V that this thread clears before its first product (both query tiles do, neither waits for the other)
      const bool clears = t_lo == t0 && r < BB && t0 * BB + r < z;
      float m_ref = -INFINITY, l = 0.f;
      bool ok = true;
      for (int t = t_lo; t < t_hi; ++t) {
        const int set = t & 1;
        const uint32_t set_base = lane_base + set * 64;
        if (!mbar_wait_warp(&s_full[2 * x + set], (sc >> set) & 1, p.wait_ns, abort_flag, status)) {
          fail(kErrTimeoutEpilogue);
          ok = false;
          break;
        }
        sc ^= 1u << set;
        tc_fence_after();
        const int kx = key.x - t * BB, ky = key.y - t * BB;  // the row sees the keys [kx, ky) of the block
        // P = exp2(S scale - m) with the maximum so far: one pass, in which the block's own maximum is found beside
        // the exponentials. Only where that exceeds the old one by more than kGrow are the scores read again and
        // the exponentials taken anew (an item's first block finds its maximum beforehand). P replaces S once
        // it stands.
        uint32_t pk[32];
        float mx, add;
        auto pass = [&](bool first) {
          uint32_t sr[2][32];
          tmem_ld32(set_base, sr[0]);
          tmem_ld32(set_base + 32, sr[1]);
          tmem_ld_wait();
          if (!__all_sync(0xffffffffu, kx <= 0 && ky >= BB)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t vis = range_mask32(kx - 32 * c, ky - 32 * c);
#pragma unroll
              for (int e = 0; e < 32; ++e) sr[c][e] = ((vis >> e) & 1u) ? sr[c][e] : 0xff800000u;
            }
          }
          float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < BB; e += 2)
            part[(e >> 1) & 3] = fmaxf(fmaxf(part[(e >> 1) & 3], __uint_as_float(sr[e >> 5][e & 31])),
                                       __uint_as_float(sr[e >> 5][(e + 1) & 31]));
          mx = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * p.scale_log2;
          if (first) m_ref = mx;
          const float mref = m_ref == -INFINITY ? 0.f : m_ref;
          const uint64_t sc2 = f32x2(p.scale_log2, p.scale_log2), nm2 = f32x2(kRaise<T> - mref, kRaise<T> - mref);
          uint64_t l2[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < BB; e += 2) {
            const float s0 = __uint_as_float(sr[e >> 5][e & 31]), s1 = __uint_as_float(sr[e >> 5][(e + 1) & 31]);
            const float2 y = f32x2_split(fma_f32x2(f32x2(s0, s1), sc2, nm2));
            const float p0 = exp2f(y.x), p1 = exp2f(y.y);
            l2[(e >> 1) & 1] = add_f32x2(l2[(e >> 1) & 1], f32x2(p0, p1));
            pk[e / 2] = Half16<T>::pack(p0, p1);
          }
          const float2 ls = f32x2_split(add_f32x2(l2[0], l2[1]));
          add = ls.x + ls.y;
        };
        if (t == t_lo) {
          pass(true);
        } else {
          pass(false);
          // The rescale is decided per row, but tcgen05.ld/st are warp-collective: the warp rescales together
          // when any of its rows needs it, the others by 1, and after the last block's product with V (the one
          // before that has completed: it was issued before these scores).
          const bool mine = mx > m_ref + kGrow<T>;
          if (__any_sync(0xffffffffu, mine)) {
            float alpha = 1.f;
            if (mine) {
              alpha = m_ref == -INFINITY ? 0.f : exp2f(m_ref - mx);
              l *= alpha;
              m_ref = mx;
            }
            if (!mbar_wait_warp(&pv_done[x], (pv - 1) & 1, p.wait_ns, abort_flag, status)) {
              fail(kErrTimeoutEpilogue);
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t v[32];
              tmem_ld32(lane_base + 128 + c * 32, v);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
              tmem_st32(lane_base + 128 + c * 32, v);
            }
            pass(false);
          }
        }
        l += add;
        ++pv;
        tmem_st32(set_base, pk);
        if (t == t_lo && clears) {
          if (!wait(&v_full[vfirst % C::kV], vfirst / C::kV)) *abort_flag = 1;
          uint4* row = reinterpret_cast<uint4*>(smem + C::oV + vfirst % C::kV * C::kBlock + r * 128);
#pragma unroll 1
          for (int c = 0; c < D / 64 * 8; ++c) row[(c >> 3) * (kAtom64 / 16) + (c & 7)] = make_uint4(0, 0, 0, 0);
          fence_async_smem();
        }
        __syncwarp();
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[2 * x + set]);
      }
      more = ok && fetch(n + 1, next);
      if (!more) break;
      if (t_hi <= t_lo) continue;
      if (!mbar_wait_warp(&o_done[x], oc & 1, p.wait_ns, abort_flag, status)) {
        fail(kErrTimeoutEpilogue);
        break;
      }
      ++oc;
      tc_fence_after();
      const bool real = key.y > key.x;
      const float inv = 1.f / l;
      float odd = 0.f;  // becomes NaN when a value of the row is no number
      // whole warps of rows go through shared memory (rows behind the end are cut off); a warp with padding rows among
      // its own stores each row by itself
      const bool send = __all_sync(0xffffffffu, real || i >= p.N) && i - lane < p.N;
      T* orow = reinterpret_cast<T*>(p.o.p) + (int64_t)i * p.o.row + h * p.o.head;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        const int col = c * 32;
        uint32_t v[32];
        tmem_ld32(lane_base + 128 + col, v);
        if (send && lane == 0) out_wait_read();  // the buffer's last contents are on their way
        __syncwarp();
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float y[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            y[u] = __uint_as_float(v[e + u]) * inv;
            odd = fmaf(y[u], 0.f, odd);
          }
          const uint4 o = make_uint4(Half16<T>::pack(y[0], y[1]), Half16<T>::pack(y[2], y[3]),
                                     Half16<T>::pack(y[4], y[5]), Half16<T>::pack(y[6], y[7]));
          if (send) {
            out_piece(out_buf, lane, e / 8, o);
          } else if (real) {
            *reinterpret_cast<uint4*>(orow + col + e) = o;
          }
        }
        if (c == D / 32 - 1) {
          // O is read: the next item's first product of this tile may overwrite it
          tc_fence_before();
          mbar_arrive(&o_empty[x]);
        }
        if (send) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) out_send(&maps.o, maps.swap_o, out_buf, col, h, i);
        }
        __syncwarp();
      }
      if (real) p.lse[(int64_t)h * p.N + i] = (m_ref - kRaise<T> + log2f(l)) * kLn2;
      // rows that are no numbers although their scores are, and whose tiles hold foreign keys that were not cleared, or
      // hidden keys of the row's own sequence that are no numbers
      bool again = real && odd != 0.f && l == l;
      if (__any_sync(0xffffffffu, again)) {
        const int first = t_lo == t0 ? max(t_lo * BB, z) : t_lo * BB;
        const bool foreign = again && (__ldg(p.start + i) > first || __ldg(p.end + i) < t_hi * BB);
        const bool own = again && !foreign;
        const int g = h / (p.H / p.KV), row0 = i - lane;
        const int later = odd_rows<T, D>(p.v, g, g + 1, row0 + 1, min(t_hi * BB, p.N), lane).y;
        const int earlier = odd_rows<T, D>(p.v, g, g + 1, first, __reduce_max_sync(0xffffffffu, own ? key.x : 0), lane).x;
        again = foreign || (own && (later >= key.y || earlier < key.x));
      }
      uint32_t redo = __ballot_sync(0xffffffffu, again);
      if (redo) {
        if (lane == 0) out_wait_done();  // these rows' first values are in memory before the second ones
        __syncwarp();
      }
      while (redo) {
        const int b = __ffs((int)redo) - 1;
        redo &= redo - 1;
        fwd_row<T, D>(p, i - lane + b, h, lane, reinterpret_cast<float*>(out_buf));
      }
    }
    if (lane == 0) out_wait_done();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------- backward, tcgen05
// Two kernels, so that no sum is shared between blocks and the results do not depend on the schedule: dQ (one block
// per 128 query rows and head) and dK/dV (one block per 128 key rows and kv head). Both recompute the scores,
// 64 keys or queries at a time, 384 threads: warp 0 loads (TMA), warp 1 issues the MMAs, warps 4-7 and 8-11 turn
// scores into P and dS, one tile row per thread, the two groups taking the blocks in turn: while one group
// loads, computes and stores, the other's block goes through the tensor core. P and dS are rounded to 16 bits
// for their products (half a step, relative to each entry: in fp16 after a power of two, see kUp, which with its bounds
// makes 65536 rows' forward and backward 611 us instead of 556); everything else is fp32. They are written over the
// scores that they came from. On B200, 65536 rows in documents of 512 on average, 4 x 128 heads: dQ 0.20 ms, dK/dV
// 0.26 ms, where a block's start and end lie open between two tiles of an SM; 8192 rows, 16 heads of 128 on 4: dQ
// 0.36 ms (0.6 of the tensor core's cycles), dK/dV 0.53 ms, bound by the shared memory that its products read (128
// KB per block of 64 queries at 128 bytes per cycle: as long as the products) and by 256 uneven tiles on 148 SMs.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 32 fp32 columns of this warp's 32 TMEM rows, times f, as 16-bit values to columns [col, +32) of head `head` of rows
// i (one per lane); true in a lane whose row has a value that is no number. Whole warps of rows go through the
// warp's buffer in shared memory, a warp with rows that are not written among its own stores each by itself.
template <typename T>
__device__ __forceinline__ bool store_cols(uint32_t taddr, float f, const Rows& to, const CUtensorMap* map, bool swap,
                                           uint8_t* buf, int col, int head, int i, int lane, bool write, int N) {
  uint32_t v[32];
  tmem_ld32(taddr, v);
  const bool send = __all_sync(0xffffffffu, write || i >= N) && i - lane < N;
  T* dst = reinterpret_cast<T*>(to.p) + (int64_t)i * to.row + head * to.head + col;
  if (send && lane == 0) out_wait_read();
  __syncwarp();
  tmem_ld_wait();
  float odd = 0.f;
#pragma unroll
  for (int e = 0; e < 32; e += 8) {
    float y[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      y[u] = __uint_as_float(v[e + u]) * f;
      odd = fmaf(y[u], 0.f, odd);
    }
    const uint4 o = make_uint4(Half16<T>::pack(y[0], y[1]), Half16<T>::pack(y[2], y[3]), Half16<T>::pack(y[4], y[5]),
                               Half16<T>::pack(y[6], y[7]));
    if (send) {
      out_piece(buf, lane, e / 8, o);
    } else if (write) {
      *reinterpret_cast<uint4*>(dst + e) = o;
    }
  }
  if (send) {
    fence_async_smem();
    __syncwarp();
    if (lane == 0) out_send(map, swap, buf, col, head, i);
  }
  __syncwarp();
  return odd != 0.f;
}

// dQ. TMEM: two score sets (set s, for the blocks of group s: S at [128s, +64), dP at [128s + 64, +64)); dQ at
// [256, +D); the tile's Q and dO rows as 16-bit pairs at [384, +D/2) and [448, +D/2): the S and dP products read only
// K and V from shared memory. The kernel also computes delta = rowsum(dO o O) and leaves lse and delta of each row
// for the dK/dV kernel. Two roundings are undone here, since with dS rounded once and O's rounding in delta, dQ
// and dK came out 1.5 to 1.6 times as far from 64 bits as one rounding of the result alone: the tile's last two
// blocks take dS in two 16-bit parts, and the delta that goes to dK/dV is the sum of P dP itself, in fp32, which this
// kernel has at hand. The last two blocks are a compromise: rows of few keys and large weights have theirs there,
// unless their document starts a few rows before the tile does. (Both parts in every block: 219 instead of 184 us
// over 65536 packed tokens.)
template <int D>
struct DqCfg {
  static constexpr int kTile = BB * D * 2;
  static constexpr int kStages = 6;
  static constexpr int oK = 0, oV = kStages * kTile;
  // the tile's Q and dO rows wait in the ring's stages 3 and 4 until they are in TMEM, its O rows by themselves
  static constexpr int oQ = oK + 3 * kTile, oD = oV + 3 * kTile, oO = oV + kStages * kTile;
  static constexpr int oSum = oO + 2 * kTile;  // [2][128] half-row sums, [128] one group's share of delta
  static constexpr int oBar = oSum + 1536;
  static constexpr int kSmem = oBar + 256 + 1024;
  static_assert(kSmem <= 232448, "dQ shared memory");
};

struct DqMaps {
  CUtensorMap k, v, q, d, o, dq;
  int swap_kv, swap_in, swap_dq;  // bits of swap_in: q, dO, O
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) dq_tc_kernel(const __grid_constant__ DqMaps maps,
                                                       const __grid_constant__ PackedParams p, int* status) {
  using C = DqCfg<D>;
  constexpr int kAtoms = D / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::oBar);
  uint64_t* q_full = bars + 0;
  uint64_t* done = bars + 1;
  uint64_t* s_full = bars + 2;  // [2]
  uint64_t* p_full = bars + 4;  // [2]
  uint64_t* kv_full = bars + 6;
  uint64_t* kv_empty = kv_full + C::kStages;
  uint64_t* in_full = kv_empty + C::kStages;  // Q, dO and O have arrived
  uint64_t* in_read = in_full + 1;            // Q and dO are in TMEM
  uint64_t* sums_full = in_read + 1;          // both groups' shares of delta stand in shared memory
  static_assert(9 + 2 * C::kStages <= 28, "barrier region");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tile = (int)gridDim.x / p.H - 1 - (int)blockIdx.x / p.H, h = blockIdx.x % p.H;  // late rows first
  const int kvh = h / (p.H / p.KV), q0 = tile * BT;
  const int warp = warp_id();
  if (__syncthreads_or(device_failed(status))) return;  // all threads or none: the word may change meanwhile
  // spans never decrease along the rows: the first row has the first key
  const int kb_hi = min(q0 + BT, p.N) - 1 >> 6;
  const int kb_lo = min(max(keys_of(p, q0).x, 0) >> 6, kb_hi);
  const int nb = kb_hi - kb_lo + 1;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 256);  // every softmax thread has stored its Q or dO row in TMEM
    mbar_init(in_full, 1);
    mbar_init(in_read, 256);
    mbar_init(sums_full, 256);
    mbar_init(done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&](int code) {
    *abort_flag = 1;
    if (status) atomicCAS(status, 0, code);
  };
  auto wait = [&](uint64_t* bar, int phase) { return mbar_wait(bar, phase & 1, kBudgetNs, abort_flag, status); };

  if (warp == 0) {
    few_registers();
    if (elect_one()) {
      mbar_arrive_expect_tx(in_full, 3 * BT * D * 2);
      load_tile(&maps.q, maps.swap_in & 1, in_full, smem + C::oQ, h, q0, kAtoms, kAtom);
      load_tile(&maps.d, maps.swap_in & 2, in_full, smem + C::oD, h, q0, kAtoms, kAtom);
      load_tile(&maps.o, maps.swap_in & 4, in_full, smem + C::oO, h, q0, kAtoms, kAtom);
      int j = 0;
      bool ok = true;
      for (; j < nb; ++j) {
        const int st = j % C::kStages;
        if (!wait(&kv_empty[st], (j / C::kStages) ^ 1) || (j == 3 && !wait(in_read, 0))) {
          ok = false;
          break;
        }
        const int k0 = (kb_lo + j) * BB;
        mbar_arrive_expect_tx(&kv_full[st], 2 * C::kTile);
        load_tile(&maps.k, maps.swap_kv & 1, &kv_full[st], smem + C::oK + st * C::kTile, kvh, k0, kAtoms, kAtom64);
        load_tile(&maps.v, maps.swap_kv & 2, &kv_full[st], smem + C::oV + st * C::kTile, kvh, k0, kAtoms, kAtom64);
      }
      if (!ok) {
        fail(kErrTimeoutProducer);
        mbar_wait(in_full, 0, kDrainNs, nullptr);
        for (int g = max(0, j - C::kStages); g < j; ++g)
          mbar_wait(&kv_full[g % C::kStages], (g / C::kStages) & 1, kDrainNs, nullptr);
      }
    }
  } else if (warp == 1) {
    few_registers();
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_16<T>(BT, BB, false, false);
      constexpr uint32_t idesc_q = umma_idesc_16<T>(BT, D, false, true);
      bool ok = wait(q_full, 0);
      auto issue_s = [&](int j) -> bool {
        const int st = j % C::kStages, set = j & 1;
        if (!wait(&kv_full[st], j / C::kStages)) return false;
        tc_fence_after();
        const uint64_t k_desc = k_major(smem + C::oK + st * C::kTile), v_desc = k_major(smem + C::oV + st * C::kTile);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kAtom64 + (kk & 3) * 32) >> 4;
          umma_bf16_ts(tmem + set * 128, tmem + 384 + kk * 8, k_desc + off, idesc_s, kk > 0 ? 1u : 0u);
          umma_bf16_ts(tmem + set * 128 + 64, tmem + 448 + kk * 8, v_desc + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[set]);
        return true;
      };
      if (ok) ok = issue_s(0);
      if (ok && nb > 1) ok = issue_s(1);
      for (int j = 0; j < nb && ok; ++j) {
        if (!wait(&p_full[j & 1], j >> 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int st = j % C::kStages;
        const uint64_t k_desc = mn_major(smem + C::oK + st * C::kTile, kAtom64);
#pragma unroll
        for (int kk = 0; kk < BB / 16; ++kk)  // dS as 16-bit pairs at the first 32 columns of its set
          umma_bf16_ts(tmem + 256, tmem + (j & 1) * 128 + kk * 8, k_desc + kk * (2048 >> 4), idesc_q,
                       (j > 0 || kk > 0) ? 1u : 0u);
        if (j >= nb - 2) {
#pragma unroll
          for (int kk = 0; kk < BB / 16; ++kk)  // and what its rounding left, in the next 32
            umma_bf16_ts(tmem + 256, tmem + (j & 1) * 128 + 32 + kk * 8, k_desc + kk * (2048 >> 4), idesc_q, 1u);
        }
        umma_commit(&kv_empty[st]);
        if (j + 2 < nb) ok = issue_s(j + 2);  // into the set that this product has read
      }
      if (!ok) fail(kErrTimeoutMma);
      umma_commit(done);
      mbar_wait(done, 0, kBudgetNs, nullptr);
    }
  } else if (warp < 4) {
    few_registers();
  } else {
    many_registers();
    const int wq = warp & 3, lane = lane_id(), half = (warp - 4) >> 2;
    const int r = wq * 32 + lane, i = q0 + r;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    const int2 key = i < p.N ? keys_of(p, i) : make_int2(0, 0);
    const bool real = key.y > key.x;
    const float lse = real ? p.lse[(int64_t)h * p.N + i] * kLog2e : INFINITY;
    const int seq = real ? __ldg(p.start + i) : -1 - lane;
    float v_most = 0.f;
    if constexpr (kScaled<T>) {
      // the 32 rows with this one among them; before them, rows of one sequence alone are seen: that of their first row
      const float* most = p.v_most + (int64_t)kvh * p.Np;
      const int g0 = i - lane, lo = __shfl_sync(0xffffffffu, real ? key.x : g0, 0);
      float before = 0.f;
      for (int g = lo / 32 + lane; g < g0 / 32; g += 32) before = fmaxf(before, most[g * 32 + 31]);
      before = warp_max(before);
      if (real) v_most = fmaxf(most[i], key.x < g0 ? before : 0.f);
    }
    bool ok = mbar_wait_warp(in_full, 0, kBudgetNs, abort_flag, status);
    if (!ok) fail(kErrTimeoutEpilogue);
    // 16 bytes, the piece-th of this row of a tile
    auto piece_of = [&](int tile_at, int piece) {
      return *reinterpret_cast<const uint4*>(smem + tile_at + (piece >> 3) * kAtom + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
    };
    // this row's Q (first warp of the row) or dO (second warp) into TMEM: the A operands of S and dP
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      uint32_t w[32];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint4 a = piece_of(half == 0 ? C::oQ : C::oD, c * 8 + e);
        w[4 * e] = a.x;
        w[4 * e + 1] = a.y;
        w[4 * e + 2] = a.z;
        w[4 * e + 3] = a.w;
      }
      tmem_st32(lane_base + 384 + 64 * half + 32 * c, w);
    }
    tmem_st_wait();
    tc_fence_before();
    mbar_arrive(q_full);
    // delta: the two warps of a row each reduce half of its values and meet in shared memory
    float2 stat;
    int up = 0;  // dS goes to its product times 2^up
    float norm = 0.f;
    {
      float* sums = reinterpret_cast<float*>(smem + C::oSum);
      float acc = 0.f, norm2 = 0.f;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        const uint4 a = piece_of(C::oO, half * (D / 16) + e), b = piece_of(C::oD, half * (D / 16) + e);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = Half16<T>::unpack(u[k]), w = Half16<T>::unpack(y[k]);
          acc = fmaf(f.x, w.x, fmaf(f.y, w.y, acc));
          if constexpr (kScaled<T>) norm2 = fmaf(w.x, w.x, fmaf(w.y, w.y, norm2));
        }
      }
      mbar_arrive(in_read);
      sums[half * 128 + r] = acc;
      // the halves of |do|^2 meet where each thread has read O: at its first piece
      auto norm_at = [&](int x) {
        const int piece = x * (D / 16);
        return reinterpret_cast<float*>(smem + C::oO + (piece >> 3) * kAtom + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
      };
      if constexpr (kScaled<T>) *norm_at(half) = norm2;
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the eight softmax warps
      stat = make_float2(lse, real ? sums[r] + sums[128 + r] : 0.f);
      if constexpr (kScaled<T>) {
        const float n2 = *norm_at(0) + *norm_at(1);
        norm = real && n2 < INFINITY ? sqrtf(n2) : 0.f;
        up = up_for(norm * v_most + fabsf(stat.y));
      }
    }
    const float from = stat.x - (float)up;  // P times 2^up is exp2(s - from)
    const int z = __ldg(p.start + q0);  // keys before it are foreign to every row of the tile: all in block kb_lo
    const uint32_t set_base = lane_base + half * 128;
    uint64_t exact = 0;  // sum of P dP: delta without the rounding of O
    for (int j = half; ok && j < nb; j += 2) {
      if (!mbar_wait_warp(&s_full[half], (j >> 1) & 1, kBudgetNs, abort_flag, status)) {
        fail(kErrTimeoutEpilogue);
        ok = false;
        break;
      }
      tc_fence_after();
      const int k0 = (kb_lo + j) * BB;
      uint32_t pk[32], rest[32];
      // dS = P (dP - delta), 0 where the row does not see the key
      uint32_t svs[2][32], dvs[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_ld32(set_base + c * 32, svs[c]);
        tmem_ld32(set_base + 64 + c * 32, dvs[c]);
      }
      tmem_ld_wait();
      auto body = [&](int c, auto masked, auto split) {
        constexpr bool kMasked = decltype(masked)::value, kSplit = decltype(split)::value;
        const uint32_t(&sv)[32] = svs[c];
        const uint32_t(&dv)[32] = dvs[c];
        uint32_t vis = 0xffffffffu;
        if constexpr (kMasked) vis = range_mask32(key.x - k0 - 32 * c, key.y - k0 - 32 * c);
        const uint64_t dl2 = f32x2(stat.y, stat.y), sc2 = f32x2(p.scale_log2, p.scale_log2), nl2 = f32x2(-from, -from);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 y = f32x2_split(fma_f32x2(f32x2(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), sc2, nl2));
          const uint64_t pr = f32x2(exp2f(y.x), exp2f(y.y));
          const uint64_t dp = f32x2(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1]));
          float2 g = f32x2_split(mul_f32x2(pr, sub_f32x2(dp, dl2)));
          if constexpr (kMasked) {
            const bool v0 = (vis >> e) & 1u, v1 = (vis >> (e + 1)) & 1u;
            g.x = v0 ? g.x : 0.f;
            g.y = v1 ? g.y : 0.f;
            const float2 t = f32x2_split(mul_f32x2(pr, dp));
            exact = add_f32x2(exact, f32x2(v0 ? t.x : 0.f, v1 ? t.y : 0.f));
          } else {
            exact = fma_f32x2(pr, dp, exact);
          }
          const uint32_t hi = Half16<T>::pack(g.x, g.y);
          pk[c * 16 + e / 2] = hi;
          if constexpr (kSplit) {
            const float2 back = Half16<T>::unpack(hi);
            rest[c * 16 + e / 2] = Half16<T>::pack(g.x - back.x, g.y - back.y);
          }
        }
      };
      const bool split = j >= nb - 2;
      if (split) {
        body(0, std::true_type{}, std::true_type{});
        body(1, std::true_type{}, std::true_type{});
      } else if (__all_sync(0xffffffffu, key.x <= k0 && key.y >= k0 + BB)) {
        body(0, std::false_type{}, std::false_type{});
        body(1, std::false_type{}, std::false_type{});
      } else {
        body(0, std::true_type{}, std::false_type{});
        body(1, std::true_type{}, std::false_type{});
      }
      if (j == 0 && r < BB && kb_lo * BB + r < z) {
        uint4* row = reinterpret_cast<uint4*>(smem + C::oK + r * 128);
#pragma unroll 1
        for (int c = 0; c < D / 64 * 8; ++c) row[(c >> 3) * (kAtom64 / 16) + (c & 7)] = make_uint4(0, 0, 0, 0);
        fence_async_smem();
      }
      __syncwarp();
      tmem_st32(set_base, pk);
      if (split) tmem_st32(set_base + 32, rest);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[half]);
    }
    // delta for the dK/dV kernel
    {
      float* sums = reinterpret_cast<float*>(smem + C::oSum);
      const float2 e2 = f32x2_split(exact);
      const float mine = (e2.x + e2.y) * power_of_2(-up);
      if (half == 1) sums[256 + r] = mine;
      mbar_arrive(sums_full);
      if (half == 0) {
        ok = mbar_wait_warp(sums_full, 0, kBudgetNs, abort_flag, status) && ok;
        const float delta = real ? mine + sums[256 + r] : 0.f;
        p.stat[(int64_t)h * p.Np + i] = make_float2(kUp<T> - stat.x, -delta);
        if constexpr (kScaled<T>)
          p.d_most[(int64_t)h * p.Np + i] = make_float2(most_of_seq(norm, seq),
                                                        most_of_seq(fabsf(delta) < INFINITY ? fabsf(delta) : 0.f, seq));
      }
    }
    if (ok && mbar_wait_warp(done, 0, kBudgetNs, abort_flag, status)) {
      tc_fence_after();
      bool odd = false;
#pragma unroll 1
      for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c)  // through the ring's memory, which is free by now
        odd |= store_cols<T>(lane_base + 256 + c * 32, p.scale * power_of_2(-up), p.dq, &maps.dq, maps.swap_dq,
                             smem + C::oK + (warp - 4) * kOutBytes, c * 32, h, i, lane, real, p.N);
      // as in the forward: no number, though the scores and delta are, and foreign keys among the tile's that were not
      // cleared, or hidden ones that are no numbers
      bool again = real && odd && stat.x == stat.x && is_number(stat.y);
      if (__any_sync(0xffffffffu, again)) {
        const int first = max(kb_lo * BB, z);
        const bool foreign = again && (__ldg(p.start + i) > first || __ldg(p.end + i) < (kb_hi + 1) * BB);
        const bool own = again && !foreign;
        const int later = odd_rows<T, D>(p.k, kvh, kvh + 1, i - lane + 1, min((kb_hi + 1) * BB, p.N), lane).y;
        const int earlier = odd_rows<T, D>(p.k, kvh, kvh + 1, first, __reduce_max_sync(0xffffffffu, own ? key.x : 0), lane).x;
        again = foreign || (own && (later >= key.y || earlier < key.x));
      }
      uint32_t redo = __ballot_sync(0xffffffffu, again);
      if (lane == 0) out_wait_done();  // also before any row's second values
      __syncwarp();
      while (redo) {
        const int b = __ffs((int)redo) - 1;
        redo &= redo - 1;
        const float2 st = make_float2(__shfl_sync(0xffffffffu, stat.x, b), __shfl_sync(0xffffffffu, stat.y, b));
        dq_row<T, D>(p, i - lane + b, h, half, lane, st, reinterpret_cast<float*>(smem + C::oK + (warp - 4) * kOutBytes));
      }
    } else if (ok) {
      fail(kErrTimeoutEpilogue);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dK and dV. TMEM: two score sets (set s, for the blocks of group s: S^T at [128s, +64), dP^T at [128s + 64, +64)), dV at [256, +D), dK at
// [384, +D). K and V stay in shared memory as the A operands of S^T and dP^T; blocks of 64 queries (Q, dO, their
// lse and delta) go through a ring, head after head of the kv head's group.
template <int D>
struct DkvCfg {
  static constexpr int kTile = BT * D * 2, kBlock = BB * D * 2;
  static constexpr int kStages = 4;
  static constexpr int oK = 0, oV = kTile, oQ = 2 * kTile, oD = oQ + kStages * kBlock, oStat = oD + kStages * kBlock;
  static constexpr int oBar = oStat + kStages * BB * 8;
  static constexpr int kSmem = oBar + 256 + 1024;
  static_assert(kSmem <= 232448, "dK/dV shared memory");
};

struct DkvMaps {
  CUtensorMap k, v, q, d, dv, dk;
  int swap_kv, swap_qd, swap_o;  // bits of swap_o: dv, dk
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) dkv_tc_kernel(const __grid_constant__ DkvMaps maps,
                                                        const __grid_constant__ PackedParams p, int* status) {
  using C = DkvCfg<D>;
  constexpr int kAtoms = D / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::oBar);
  uint64_t* kv_full = bars + 0;
  uint64_t* done = bars + 1;
  uint64_t* s_full = bars + 2;  // [2]
  uint64_t* p_full = bars + 4;  // [2]
  uint64_t* qd_full = bars + 6;
  uint64_t* qd_empty = qd_full + C::kStages;
  static_assert(6 + 2 * C::kStages <= 28, "barrier region");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 28);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* stat = reinterpret_cast<float2*>(smem + C::oStat);

  const int kvh = blockIdx.x % p.KV, k0 = (int)blockIdx.x / p.KV * BT, group = p.H / p.KV;
  const int warp = warp_id();
  if (__syncthreads_or(device_failed(status))) return;  // all threads or none: the word may change meanwhile
  // spans never decrease along the rows: the last row is seen by the last query
  const int k_last = min(k0 + BT, p.N) - 1;
  const int qb_lo = k0 / BB, qb_hi = (max(queries_of(p, k_last), k_last + 1) - 1) / BB;
  const int nq = qb_hi - qb_lo + 1, iters = nq * group;
  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&qd_full[i], 1);
      mbar_init(&qd_empty[i], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&](int code) {
    *abort_flag = 1;
    if (status) atomicCAS(status, 0, code);
  };
  auto wait = [&](uint64_t* bar, int phase) { return mbar_wait(bar, phase & 1, kBudgetNs, abort_flag, status); };

  if (warp == 0) {
    few_registers();
    if (elect_one()) {
      mbar_arrive_expect_tx(kv_full, 2 * C::kTile);
      load_tile(&maps.k, maps.swap_kv & 1, kv_full, smem + C::oK, kvh, k0, kAtoms, kAtom);
      load_tile(&maps.v, maps.swap_kv & 2, kv_full, smem + C::oV, kvh, k0, kAtoms, kAtom);
      int it = 0;
      bool ok = true;
      for (; it < iters; ++it) {
        const int st = it % C::kStages;
        if (!wait(&qd_empty[st], (it / C::kStages) ^ 1)) {
          ok = false;
          break;
        }
        const int h = kvh * group + it / nq, q0 = (qb_lo + it % nq) * BB;
        mbar_arrive_expect_tx(&qd_full[st], 2 * C::kBlock + BB * 8);
        load_tile(&maps.q, maps.swap_qd & 1, &qd_full[st], smem + C::oQ + st * C::kBlock, h, q0, kAtoms, kAtom64);
        load_tile(&maps.d, maps.swap_qd & 2, &qd_full[st], smem + C::oD + st * C::kBlock, h, q0, kAtoms, kAtom64);
        bulk_load(stat + st * BB, p.stat + (int64_t)h * p.Np + q0, BB * 8, &qd_full[st]);
      }
      if (!ok) {
        fail(kErrTimeoutProducer);
        mbar_wait(kv_full, 0, kDrainNs, nullptr);
        for (int g = max(0, it - C::kStages); g < it; ++g)
          mbar_wait(&qd_full[g % C::kStages], (g / C::kStages) & 1, kDrainNs, nullptr);
      }
    }
  } else if (warp == 1) {
    few_registers();
    if (elect_one()) {
      constexpr uint32_t idesc_s = umma_idesc_16<T>(BT, BB, false, false);
      constexpr uint32_t idesc_g = umma_idesc_16<T>(BT, D, false, true);
      const uint64_t k_desc = k_major(smem + C::oK), v_desc = k_major(smem + C::oV);
      bool ok = wait(kv_full, 0);
      auto issue_s = [&](int it) -> bool {
        const int st = it % C::kStages, set = it & 1;
        if (!wait(&qd_full[st], it / C::kStages)) return false;
        tc_fence_after();
        const uint64_t q_desc = k_major(smem + C::oQ + st * C::kBlock), d_desc = k_major(smem + C::oD + st * C::kBlock);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t offa = ((kk >> 2) * kAtom + (kk & 3) * 32) >> 4, offb = ((kk >> 2) * kAtom64 + (kk & 3) * 32) >> 4;
          umma_bf16_ss(tmem + set * 128, k_desc + offa, q_desc + offb, idesc_s, kk > 0 ? 1u : 0u);
          umma_bf16_ss(tmem + set * 128 + 64, v_desc + offa, d_desc + offb, idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[set]);
        return true;
      };
      if (ok) ok = issue_s(0);
      if (ok && iters > 1) ok = issue_s(1);
      for (int it = 0; it < iters && ok; ++it) {
        if (!wait(&p_full[it & 1], it >> 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int st = it % C::kStages, set = it & 1;
        const uint64_t q_desc = mn_major(smem + C::oQ + st * C::kBlock, kAtom64);
        const uint64_t d_desc = mn_major(smem + C::oD + st * C::kBlock, kAtom64);
        // P^T and dS^T as 16-bit pairs at the first 32 columns of S^T and dP^T
#pragma unroll
        for (int kk = 0; kk < BB / 16; ++kk) {
          const uint32_t acc = (it > 0 || kk > 0) ? 1u : 0u;
          const uint32_t col = tmem + set * 128 + kk * 8;
          umma_bf16_ts(tmem + 256, col, d_desc + kk * (2048 >> 4), idesc_g, acc);
          umma_bf16_ts(tmem + 384, col + 64, q_desc + kk * (2048 >> 4), idesc_g, acc);
        }
        umma_commit(&qd_empty[st]);
        if (it + 2 < iters) ok = issue_s(it + 2);  // into the set that these products have read
      }
      if (!ok) fail(kErrTimeoutMma);
      umma_commit(done);
      mbar_wait(done, 0, kBudgetNs, nullptr);
    }
  } else if (warp < 4) {
    few_registers();
  } else {
    many_registers();
    const int wq = warp & 3, lane = lane_id(), half = (warp - 4) >> 2;
    const int r = wq * 32 + lane, j = k0 + r;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    // the queries that see this key row (none for a row of no sequence)
    const bool real = j < p.N && __ldg(p.start + j) <= j && queries_of(p, j) > j;
    const int q_hi = real ? queries_of(p, j) : 0;
    bool ok = true;
    int up = 0;  // dS goes to its product times 2^up
    if constexpr (kScaled<T>) {
      ok = mbar_wait_warp(kv_full, 0, kBudgetNs, abort_flag, status);
      if (!ok) fail(kErrTimeoutEpilogue);
      float v2 = 0.f;  // |v_j|^2
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint4 a = *reinterpret_cast<const uint4*>(smem + C::oV + (c >> 3) * kAtom + r * 128 + (((c & 7) ^ (r & 7)) << 4));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Half16<T>::unpack(w[e]);
          v2 = fmaf(f.x, f.x, fmaf(f.y, f.y, v2));
        }
      }
      // the 32 rows with this one among them; behind them, rows of one sequence alone see these: that of their last row
      const int g0 = j - lane, hi = __reduce_max_sync(0xffffffffu, q_hi);
      float2 own = make_float2(0.f, 0.f), behind = own;
      auto take = [](float2& m, float2 x) { m = make_float2(fmaxf(m.x, x.x), fmaxf(m.y, x.y)); };
      for (int h = kvh * group; h < (kvh + 1) * group; ++h) {
        const float2* most = p.d_most + (int64_t)h * p.Np;
        for (int i = g0 + 32 + lane * 32; i < hi; i += 32 * 32) take(behind, most[i]);
        if (real) take(own, most[j]);
      }
      behind = make_float2(warp_max(behind.x), warp_max(behind.y));
      if (q_hi > g0 + 32) take(own, behind);
      up = up_for(own.x * (v2 < INFINITY ? sqrtf(v2) : 0.f) + own.y);
    }
    const float more = power_of_2(up - (int)kUp<T>);  // P has kUp already
    const int z = __ldg(p.end + k_last);  // queries from here on are foreign to every key of the tile: all in block qb_hi
    const uint32_t set_base = lane_base + half * 128;
    int qb = half % nq;  // the iteration's query block, counted from qb_lo
    for (int it = half; ok && it < iters; it += 2) {
      const int st = it % C::kStages;
      if (!mbar_wait_warp(&s_full[half], (it >> 1) & 1, kBudgetNs, abort_flag, status)) {
        fail(kErrTimeoutEpilogue);
        ok = false;
        break;
      }
      tc_fence_after();
      const int q0 = (qb_lo + qb) * BB;
      uint32_t pp[32], ss[32], svs[2][32], dvs[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_ld32(set_base + c * 32, svs[c]);
        tmem_ld32(set_base + 64 + c * 32, dvs[c]);
      }
      tmem_ld_wait();
      auto body = [&](int c, auto masked) {
        constexpr bool kMasked = decltype(masked)::value;
        const float4* ls = reinterpret_cast<const float4*>(stat + st * BB + c * 32);
        const uint32_t(&sv)[32] = svs[c];
        const uint32_t(&dv)[32] = dvs[c];
        uint32_t vis = 0xffffffffu;
        if constexpr (kMasked) vis = range_mask32(real ? j - q0 - 32 * c : 32, q_hi - q0 - 32 * c);
        const uint64_t sc2 = f32x2(p.scale_log2, p.scale_log2);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float4 a = ls[e / 2];  // (-lse, -delta) of two queries
          const float2 y = f32x2_split(fma_f32x2(f32x2(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), sc2,
                                                 f32x2(a.x, a.z)));
          float p0 = exp2f(y.x), p1 = exp2f(y.y);
          float2 g = f32x2_split(mul_f32x2(
              f32x2(p0, p1), add_f32x2(f32x2(__uint_as_float(dv[e]), __uint_as_float(dv[e + 1])), f32x2(a.y, a.w))));
          if constexpr (kMasked) {
            const bool v0 = (vis >> e) & 1u, v1 = (vis >> (e + 1)) & 1u;
            p0 = v0 ? p0 : 0.f;
            p1 = v1 ? p1 : 0.f;
            g.x = v0 ? g.x : 0.f;
            g.y = v1 ? g.y : 0.f;
          }
          if constexpr (kScaled<T>) g = f32x2_split(mul_f32x2(f32x2(g.x, g.y), f32x2(more, more)));
          pp[c * 16 + e / 2] = Half16<T>::pack(p0, p1);
          ss[c * 16 + e / 2] = Half16<T>::pack(g.x, g.y);
        }
      };
      if (__all_sync(0xffffffffu, real && j <= q0 && q_hi >= q0 + BB)) {
        body(0, std::false_type{});
        body(1, std::false_type{});
      } else {
        body(0, std::true_type{});
        body(1, std::true_type{});
      }
      if (qb == nq - 1 && r < BB && qb_hi * BB + r >= z) {
        uint4* row = reinterpret_cast<uint4*>(smem + C::oQ + st * C::kBlock + r * 128);
        uint4* dow = reinterpret_cast<uint4*>(smem + C::oD + st * C::kBlock + r * 128);
#pragma unroll 1
        for (int c = 0; c < D / 64 * 8; ++c)
          row[(c >> 3) * (kAtom64 / 16) + (c & 7)] = dow[(c >> 3) * (kAtom64 / 16) + (c & 7)] = make_uint4(0, 0, 0, 0);
        fence_async_smem();
      }
      __syncwarp();
      tmem_st32(set_base, pp);
      tmem_st32(set_base + 64, ss);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[half]);
      qb += 2;
      while (qb >= nq) qb -= nq;
    }
    if (ok && mbar_wait_warp(done, 0, kBudgetNs, abort_flag, status)) {
      tc_fence_after();
      // half 0 writes dV, half 1 dK, through the ring's memory, which is free by now
      const Rows& to = half ? p.dk : p.dv;
      bool odd = false;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c)
        odd |= store_cols<T>(lane_base + (half ? 384 : 256) + c * 32, half ? p.scale * power_of_2(-up) : power_of_2(-(int)kUp<T>), to, half ? &maps.dk : &maps.dv,
                             (maps.swap_o >> half) & 1, smem + C::oQ + (warp - 4) * kOutBytes, c * 32, kvh, j, lane, real,
                             p.N);
      // no number, and foreign queries among the tile's that were not cleared, or hidden ones that are no numbers
      bool again = real && odd;
      if (__any_sync(0xffffffffu, again)) {
        const int end = min(z, (qb_hi + 1) * BB);
        const bool foreign = again && (__ldg(p.start + j) > k0 || __ldg(p.end + j) < end);
        const bool own = again && !foreign;
        const Rows& from = half ? p.q : p.dout;  // what the hidden weights of 0 are multiplied by
        const int earlier = odd_rows<T, D>(from, kvh * group, (kvh + 1) * group, k0, min(j - lane + 31, p.N), lane).x;
        const int later = odd_rows<T, D>(from, kvh * group, (kvh + 1) * group,
                                         __reduce_min_sync(0xffffffffu, own ? q_hi : p.N), min(end, p.N), lane).y;
        again = foreign || (own && (earlier < j || later >= q_hi));
      }
      uint32_t redo = __ballot_sync(0xffffffffu, again);
      if (lane == 0) out_wait_done();  // also before any row's second values
      __syncwarp();
      while (redo) {
        const int b = __ffs((int)redo) - 1;
        redo &= redo - 1;
        dkv_row<T, D>(p, j - lane + b, kvh, half, lane, reinterpret_cast<float*>(smem + C::oQ + (warp - 4) * kOutBytes));
      }
    } else if (ok) {
      fail(kErrTimeoutEpilogue);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
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
  // up to 32 rows of a warp by themselves: 5 us per key in all (200,000 keys, 128 wide), and four times that allowed
  p.wait_ns = kBudgetNs + 20000ull * p.window;
  p.start = start.data_ptr<int>();
  p.end = end.data_ptr<int>();
  return p;
}

// TMA maps of [rows, heads, D] tensors with boxes of box_rows rows and box_cols columns of one head; bit i of the result: the i-th map's
// coordinates are (d, row, head)
template <size_t n>
int tile_maps(const std::pair<const torch::Tensor*, CUtensorMap*> (&sides)[n], int box_rows, int box_cols = 64) {
  int swap = 0;
  for (size_t i = 0; i < n; ++i) {
    const torch::Tensor& t = *sides[i].first;
    const Rows r = rows_of(t);
    bool s = false;
    *sides[i].second = tma_map_head_rows(
        t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, r.p, t.size(2),
        t.size(1), t.size(0), r.head, r.row, box_rows, &s, box_cols);
    swap |= (int)s << i;
  }
  return swap;
}

// a kernel's attributes belong to a device: each caller (each F) runs f once for each device that it is used on
template <typename F>
void once_per_device(int device, F&& f) {
  static std::atomic<uint64_t> done{0};
  TORCH_CHECK(device >= 0 && device < 64, "bad device index");
  if (!(done.load(std::memory_order_acquire) >> device & 1)) {
    f();
    done.fetch_or(uint64_t(1) << device, std::memory_order_release);
  }
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
  check_output(what, {"out", &out}, {{"q", &q}, {"k", &k}, {"v", &v}, {"start", &start}, {"end", &end}});
  check_output(what, {"lse", &lse}, {{"out", &out}, {"q", &q}, {"k", &k}, {"v", &v}, {"start", &start}, {"end", &end}});
  TORCH_CHECK_VALUE(q.is_cuda(), what, ": q must be on a CUDA device");
  if (p.N == 0) return {out, lse};
  p.o = rows_of(out);
  p.lse = lse.data_ptr<float>();
  c10::cuda::CUDAGuard g(q.device());
  auto st = at::cuda::getCurrentCUDAStream();
  by_type(q, [&](auto t, auto d) {
    constexpr int D = d();
    using C = FwdCfg<D>;
    FwdMaps maps;
    const std::pair<const torch::Tensor*, CUtensorMap*> q_side[] = {{&q, &maps.q}}, kv_side[] = {{&k, &maps.k}, {&v, &maps.v}},
                                                        to[] = {{&out, &maps.o}};
    maps.swap = tile_maps(q_side, BT) | tile_maps(kv_side, BB) << 1;
    maps.swap_o = tile_maps(to, 32, 32);
    once_per_device(q.device().index(), [] {
      C10_CUDA_CHECK(cudaFuncSetAttribute(fwd_tc_kernel<decltype(t), D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          C::kSmem));
    });
    const int64_t tiles = (p.N + BT - 1) / BT;
    const int64_t items = p.H / p.KV % 2 == 0 ? tiles * (p.H / 2) : (tiles + 1) / 2 * p.H;
    TORCH_CHECK_VALUE(items < (int64_t(1) << 31), what, ": too many rows or heads");
    fwd_tc_kernel<decltype(t), D><<<(unsigned)items, kThreads, C::kSmem, st>>>(maps, p, status_ptr(q.device().index()));
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {out, lse};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> packed_attn_bwd(
    const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& out,
    const torch::Tensor& lse, const torch::Tensor& dout, const torch::Tensor& start, const torch::Tensor& end,
    int64_t window, double scale, c10::optional<torch::Tensor> dq_, c10::optional<torch::Tensor> dk_,
    c10::optional<torch::Tensor> dv_, c10::optional<torch::Tensor> scratch_) {
  const char* what = "packed attention_bwd";
  PackedParams p = common_params(what, q, k, v, start, end, window, scale);
  const int64_t N = p.N, H = p.H, KV = p.KV;
  check_rows(out, what, "out", N, H, q.size(2), q);
  check_rows(dout, what, "dout", N, H, q.size(2), q);
  stat_rows(lse, what, "lse", H, q, false);
  torch::Tensor dq = out_rows(dq_, what, "dq", H, q), dk = out_rows(dk_, what, "dk", KV, q),
                dv = out_rows(dv_, what, "dv", KV, q);
  p.Np = (int)((N + BT - 1) / BT * BT);
  const bool scaled = q.scalar_type() == at::kHalf;
  const int64_t entries = (int64_t)p.Np * (scaled ? 4 * H + KV : 2 * H);
  torch::Tensor scratch;
  if (scratch_.has_value() && scratch_->defined()) {
    scratch = *scratch_;
    TORCH_CHECK_VALUE(scratch.scalar_type() == at::kFloat && scratch.is_contiguous() && scratch.numel() >= entries &&
                          reinterpret_cast<uintptr_t>(scratch.data_ptr()) % 16 == 0,
                      what, ": scratch must be contiguous float32 of ", std::to_string(entries), " entries, 16-byte aligned");
    TORCH_CHECK_VALUE(scratch.device() == q.device(), what, ": scratch is on another device than q");
  } else {
    scratch = torch::empty({entries}, q.options().dtype(at::kFloat));
  }
  for (const Named& r : {Named("dq", &dq), Named("dk", &dk), Named("dv", &dv), Named("scratch", &scratch)})
    check_output(what, r, {{"q", &q}, {"k", &k}, {"v", &v}, {"out", &out}, {"lse", &lse}, {"dout", &dout},
                           {"start", &start}, {"end", &end}});
  check_output(what, {"dq", &dq}, {{"dk", &dk}, {"dv", &dv}, {"scratch", &scratch}});
  check_output(what, {"dk", &dk}, {{"dv", &dv}, {"scratch", &scratch}});
  check_output(what, {"dv", &dv}, {{"scratch", &scratch}});
  TORCH_CHECK_VALUE(q.is_cuda(), what, ": q must be on a CUDA device");
  if (N == 0) return {dq, dk, dv};
  p.o = rows_of(out);
  p.dout = rows_of(dout);
  p.dq = rows_of(dq);
  p.dk = rows_of(dk);
  p.dv = rows_of(dv);
  p.lse = lse.data_ptr<float>();
  p.stat = reinterpret_cast<float2*>(scratch.data_ptr<float>());
  p.d_most = p.stat + H * p.Np;
  p.v_most = reinterpret_cast<float*>(p.d_most + H * p.Np);
  c10::cuda::CUDAGuard g(q.device());
  auto st = at::cuda::getCurrentCUDAStream();
  by_type(q, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = d();
    DqMaps a;
    const std::pair<const torch::Tensor*, CUtensorMap*> kv64[] = {{&k, &a.k}, {&v, &a.v}};
    a.swap_kv = tile_maps(kv64, BB);
    const std::pair<const torch::Tensor*, CUtensorMap*> in[] = {{&q, &a.q}, {&dout, &a.d}, {&out, &a.o}}, to_q[] = {{&dq, &a.dq}};
    a.swap_in = tile_maps(in, BT);
    a.swap_dq = tile_maps(to_q, 32, 32);
    DkvMaps b;
    const std::pair<const torch::Tensor*, CUtensorMap*> kv[] = {{&k, &b.k}, {&v, &b.v}}, qd[] = {{&q, &b.q}, {&dout, &b.d}};
    b.swap_kv = tile_maps(kv, BT);
    b.swap_qd = tile_maps(qd, BB);
    const std::pair<const torch::Tensor*, CUtensorMap*> to_kv[] = {{&dv, &b.dv}, {&dk, &b.dk}};
    b.swap_o = tile_maps(to_kv, 32, 32);
    once_per_device(q.device().index(), [] {
      C10_CUDA_CHECK(cudaFuncSetAttribute(dq_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, DqCfg<D>::kSmem));
      C10_CUDA_CHECK(cudaFuncSetAttribute(dkv_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, DkvCfg<D>::kSmem));
    });
    const int64_t tiles = p.Np / BT;
    TORCH_CHECK_VALUE(tiles * H < (int64_t(1) << 31), what, ": too many rows or heads");
    int* status = status_ptr(q.device().index());
    if constexpr (kScaled<T>) {
      v_most_kernel<T, D><<<(unsigned)((p.Np / 32 * KV + kNormThreads / 32 - 1) / (kNormThreads / 32)), kNormThreads, 0, st>>>(p);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
    dq_tc_kernel<T, D><<<(unsigned)(tiles * H), kThreads, DqCfg<D>::kSmem, st>>>(a, p, status);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    dkv_tc_kernel<T, D><<<(unsigned)(tiles * KV), kThreads, DkvCfg<D>::kSmem, st>>>(b, p, status);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dq, dk, dv};
}

}  // namespace br
