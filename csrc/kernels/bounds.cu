// The span of each row's sequence in a packed batch: start[i] is the first row of the sequence that row i
// belongs to, end[i] the row past its last one. A row of no sequence gets the empty span [i, i).
//
// Both kernels move 4 bytes in (or a search in a table that stays in L1) and 8 out per row and compute next to
// nothing, so they are bound by the launch up to about a million rows: a call takes 6.5 us for 600 rows and for 2^18,
// two allocations with it.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <tuple>

#include "common.cuh"
#include "overlap.h"
#include "status.h"

namespace br {
namespace {

constexpr int kOffThreads = 256;

// offsets[0..n_off): sequence s holds rows [offsets[s], offsets[s + 1]). One thread per row: the number of
// offsets <= row, by bisection. The bisection's invariant offsets[ub - 1] <= row < offsets[ub] holds for any
// contents, so an unsorted table gives a wrong span but never one that leaves [0, rows); tables that are not
// sorted or reach outside [0, rows] are reported as kErrBadIndex.
__global__ void __launch_bounds__(kOffThreads) bounds_offsets_kernel(const int* __restrict__ offsets, int n_off, int rows,
                                                                     int* __restrict__ start, int* __restrict__ end,
                                                                     int* status) {
  const int64_t i = (int64_t)blockIdx.x * kOffThreads + threadIdx.x;
  if (i < rows) {
    const int row = (int)i;
    int lo = 0, hi = n_off;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(offsets + mid) <= row) {
        lo = mid + 1;
      } else {
        hi = mid;
      }
    }
    const bool inside = lo > 0 && lo < n_off;
    start[row] = inside ? max(__ldg(offsets + lo - 1), 0) : row;
    end[row] = inside ? min(__ldg(offsets + lo), rows) : row;
  }
  for (int64_t s = i; s < n_off; s += (int64_t)gridDim.x * kOffThreads) {
    const int o = __ldg(offsets + s);
    if (o < 0 || o > rows || (s > 0 && __ldg(offsets + s - 1) > o)) atomicCAS(status, 0, (int)kErrBadIndex);
  }
}

// ids [B, T]: a sequence starts at the first token of each row of ids and at each BOS. Block: one tile of
// 2048 tokens of one row, 8 consecutive tokens per thread. Within the tile the last BOS at or before a token is
// a running maximum of positions and the next BOS behind it a running minimum from the other side (warp
// shuffles, then the 8 warps' results); the tile's first tokens and its last ones look for theirs in the
// neighbouring tiles, a block-wide step of 2048 tokens at a time until one is found, which takes one step or
// two where documents are shorter than that. A row without any BOS costs every tile a walk over all the others (2^18
// tokens: up to 127 steps, one after the other).
constexpr int kIdThreads = 256, kIdPer = 8, kIdTile = kIdThreads * kIdPer;

__device__ __forceinline__ int block_max(int v, int* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();  // red may still be read from an earlier call
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int m = red[0];
#pragma unroll
  for (int w = 1; w < kIdThreads / 32; ++w) m = max(m, red[w]);
  return m;
}

__global__ void __launch_bounds__(kIdThreads) bounds_ids_kernel(const int* __restrict__ ids, int64_t ld, int T, int bos,
                                                                int* __restrict__ start, int* __restrict__ end) {
  __shared__ int red[kIdThreads / 32], pre[kIdThreads / 32], suf[kIdThreads / 32];
  const int tiles = (T + kIdTile - 1) / kIdTile;
  const int b = blockIdx.x / tiles, t0 = (blockIdx.x % tiles) * kIdTile;
  const int* row = ids + (int64_t)b * ld;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int p0 = t0 + (int)threadIdx.x * kIdPer;
  uint32_t is = 0;  // bit e: token p0 + e starts a sequence
#pragma unroll
  for (int e = 0; e < kIdPer; ++e) {
    const int p = p0 + e;
    if (p < T && (p == 0 || __ldg(row + p) == bos)) is |= 1u << e;
  }
  const int none = T;                                     // "no BOS behind"
  int last = is ? p0 + 31 - __clz(is) : -1;               // this thread's last start
  int first = is ? p0 + __ffs((int)is) - 1 : none;        // and its first
  // inclusive scans over the warp, then over the warps
  int inc = last, dec = first;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, inc, o), c = __shfl_down_sync(0xffffffffu, dec, o);
    if (lane >= o) inc = max(inc, a);
    if (lane + o < 32) dec = min(dec, c);
  }
  if (lane == 31) pre[warp] = inc;
  if (lane == 0) suf[warp] = dec;
  __syncthreads();
  int before = -1, after = none;
  for (int w = 0; w < warp; ++w) before = max(before, pre[w]);
  for (int w = kIdThreads / 32 - 1; w > warp; --w) after = min(after, suf[w]);
  const int up = __shfl_up_sync(0xffffffffu, inc, 1), down = __shfl_down_sync(0xffffffffu, dec, 1);
  if (lane > 0) before = max(before, up);
  if (lane < 31) after = min(after, down);
  // the tile's neighbours
  int carry = -1, ahead = none;
  if (t0 > 0 && row[t0] != bos) {
    for (int p = t0 - kIdTile; carry < 0; p -= kIdTile) {  // p >= 0: tiles are whole below t0; token 0 is a start
      int m = -1;
      for (int e = threadIdx.x; e < kIdTile; e += kIdThreads)
        if (p + e == 0 || __ldg(row + p + e) == bos) m = max(m, p + e);
      carry = block_max(m, red);
      if (p == 0) break;
    }
  }
  for (int p = t0 + kIdTile; p < T && ahead == none; p += kIdTile) {
    int m = -none;
    for (int e = threadIdx.x; e < kIdTile; e += kIdThreads)
      if (p + e < T && __ldg(row + p + e) == bos) m = max(m, -(p + e));
    ahead = -block_max(m, red);
  }
  const int64_t base = (int64_t)b * T;
  int s = max(before, carry);
#pragma unroll
  for (int e = 0; e < kIdPer; ++e) {
    const int p = p0 + e;
    if (p >= T) break;
    if ((is >> e) & 1u) s = p;
    const uint32_t rest = e + 1 < kIdPer ? is >> (e + 1) : 0u;
    const int n = rest ? p + __ffs((int)rest) : min(after, ahead);
    start[base + p] = (int)(base + s);
    end[base + p] = (int)(base + n);
  }
}

torch::Tensor bounds_out(const c10::optional<torch::Tensor>& t, int64_t rows, const torch::Tensor& like, const char* name) {
  if (!t.has_value() || !t->defined()) return torch::empty({rows}, like.options().dtype(at::kInt));
  TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == rows && t->is_contiguous(),
                    "bounds: ", name, " must be contiguous int32 [rows]");
  TORCH_CHECK_VALUE(t->device() == like.device(), "bounds: ", name, " is on another device");
  return *t;
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor> bounds_from_offsets(const torch::Tensor& offsets, int64_t rows,
                                                             c10::optional<torch::Tensor> start_out,
                                                             c10::optional<torch::Tensor> end_out) {
  TORCH_CHECK_VALUE(offsets.scalar_type() == at::kInt && offsets.dim() == 1 && offsets.is_contiguous(),
                    "bounds_from_offsets: offsets must be contiguous int32 [sequences + 1]");
  TORCH_CHECK_VALUE(offsets.size(0) >= 1 && offsets.size(0) < (int64_t(1) << 31),
                    "bounds_from_offsets: offsets needs at least one entry");
  TORCH_CHECK_VALUE(rows >= 0 && rows < (int64_t(1) << 31), "bounds_from_offsets: rows out of range");
  torch::Tensor start = bounds_out(start_out, rows, offsets, "start"), end = bounds_out(end_out, rows, offsets, "end");
  check_output("bounds_from_offsets", {"start", &start}, {{"end", &end}, {"offsets", &offsets}});
  check_output("bounds_from_offsets", {"end", &end}, {{"offsets", &offsets}});
  TORCH_CHECK_VALUE(offsets.is_cuda(), "bounds_from_offsets: offsets must be on a CUDA device");
  c10::cuda::CUDAGuard g(offsets.device());
  if (rows == 0) return {start, end};
  bounds_offsets_kernel<<<(unsigned)((rows + kOffThreads - 1) / kOffThreads), kOffThreads, 0,
                          at::cuda::getCurrentCUDAStream()>>>(offsets.data_ptr<int>(), (int)offsets.size(0), (int)rows,
                                                              start.data_ptr<int>(), end.data_ptr<int>(),
                                                              status_ptr(offsets.device().index()));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {start, end};
}

std::tuple<torch::Tensor, torch::Tensor> bounds_from_ids(const torch::Tensor& ids, int64_t bos,
                                                         c10::optional<torch::Tensor> start_out,
                                                         c10::optional<torch::Tensor> end_out) {
  TORCH_CHECK_VALUE(ids.scalar_type() == at::kInt && ids.dim() == 2 && (ids.size(1) <= 1 || ids.stride(1) == 1),
                    "bounds_from_ids: ids must be int32 [B, T] with contiguous rows");
  const int64_t B = ids.size(0), T = ids.size(1), rows = B * T;
  // the limit of the attention; positions and the tile behind them stay below 2^31
  TORCH_CHECK_VALUE(rows < (int64_t(1) << 30), "bounds_from_ids: too many tokens");
  TORCH_CHECK_VALUE(bos >= INT32_MIN && bos <= INT32_MAX, "bounds_from_ids: bos is not an int32");
  torch::Tensor start = bounds_out(start_out, rows, ids, "start"), end = bounds_out(end_out, rows, ids, "end");
  check_output("bounds_from_ids", {"start", &start}, {{"end", &end}, {"ids", &ids}});
  check_output("bounds_from_ids", {"end", &end}, {{"ids", &ids}});
  TORCH_CHECK_VALUE(ids.is_cuda(), "bounds_from_ids: ids must be on a CUDA device");
  c10::cuda::CUDAGuard g(ids.device());
  if (rows == 0) return {start, end};
  const int64_t tiles = (T + kIdTile - 1) / kIdTile;
  bounds_ids_kernel<<<(unsigned)(B * tiles), kIdThreads, 0, at::cuda::getCurrentCUDAStream()>>>(
      ids.data_ptr<int>(), B > 1 ? ids.stride(0) : T, (int)T, (int)bos, start.data_ptr<int>(), end.data_ptr<int>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {start, end};
}

}  // namespace br
