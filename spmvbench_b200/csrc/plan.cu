// Kernels of the expert plan (plan.cuh).
#include "plan.cuh"

namespace spmvb {
namespace {

// Up to this many blocks each of plan_scatter's adds up all counts itself;
// beyond, plan_scan does it once.
constexpr int kPlanOwnBlocks = 128;

__global__ void __launch_bounds__(kPlanThreads) plan_counts(PlanView P) {
  __shared__ int c[kPlanMaxExperts];
  for (int e = threadIdx.x; e < P.stride; e += kPlanThreads) c[e] = 0;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * P.tile_entries * P.block_tiles;
  const int n = static_cast<int>(min(static_cast<int64_t>(P.tile_entries) * P.block_tiles, P.entries - i0));
  int x[kPlanRounds];
#pragma unroll
  for (int q = 0; q < kPlanRounds; ++q) {
    const int i = q * kPlanThreads + threadIdx.x;
    x[q] = i < n ? __ldg(P.indices + i0 + i) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kPlanRounds; ++q) {
    const int e = plan_expert(x[q], P.experts, P.err);
    if (e >= 0) atomicAdd(&c[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < P.stride; e += kPlanThreads)
    P.counts[static_cast<int64_t>(blockIdx.x) * P.stride + e] = c[e];
}

// An expert a warp: running sums of its counts over the blocks.
__global__ void __launch_bounds__(kPlanThreads) plan_scan(PlanView P) {
  const int lane = threadIdx.x & 31, e = blockIdx.x * kPlanWarps + (threadIdx.x >> 5);
  if (e >= P.experts) return;
  int sum = 0;
  for (int b0 = 0; b0 < P.blocks; b0 += 32) {
    const int b = b0 + lane;
    const int v = b < P.blocks ? P.counts[static_cast<int64_t>(b) * P.stride + e] : 0;
    int incl = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += u;
    }
    if (b < P.blocks) P.prefix[static_cast<int64_t>(b) * P.stride + e] = sum + incl - v;
    sum += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) P.totals[e] = sum;
}

// Shared memory: wc[kPlanWarps][experts] (the counts' sums before that),
// before[stride], total[stride].
__global__ void __launch_bounds__(kPlanThreads) plan_scatter(PlanView P, bool scanned) {
  extern __shared__ __align__(16) int shared[];
  __shared__ int sh[kPlanWarps];
  __shared__ bool last;
  const int E = P.experts, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int* wc = shared;
  int* before = shared + kPlanWarps * max(E, 256);
  int* total = before + P.stride;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * P.tile_entries * P.block_tiles;
  const int n = static_cast<int>(min(static_cast<int64_t>(P.tile_entries) * P.block_tiles, P.entries - first));
  const auto load = [&](int i) { return __ldg(P.indices + first + i); };
  if (P.blocks == 1) {
    plan_alone<kPlanRounds>(load, n, E, P.err, wc, total, sh, P.offsets, P.order, P.position);
    return;
  }
  if (scanned) {
    for (int e = threadIdx.x; e < E; e += kPlanThreads) {
      before[e] = P.prefix[static_cast<int64_t>(blockIdx.x) * P.stride + e];
      total[e] = P.totals[e];
    }
  } else {
    // 128 experts at a time: a warp takes every eighth block, a lane four experts.
    for (int c0 = 0; c0 < P.stride; c0 += 128) {
      const int e0 = c0 + lane * 4;
      int4 a = make_int4(0, 0, 0, 0), b = a;
      if (e0 < P.stride) {
#pragma unroll 8
        for (int q = w; q < P.blocks; q += kPlanWarps) {
          const int4 v = __ldcg(reinterpret_cast<const int4*>(P.counts + static_cast<int64_t>(q) * P.stride + e0));
          const int in = q < static_cast<int>(blockIdx.x) ? -1 : 0;
          a.x += v.x; b.x += v.x & in;
          a.y += v.y; b.y += v.y & in;
          a.z += v.z; b.z += v.z & in;
          a.w += v.w; b.w += v.w & in;
        }
      }
      reinterpret_cast<int4*>(wc)[w * 64 + lane] = a;
      reinterpret_cast<int4*>(wc)[w * 64 + 32 + lane] = b;
      __syncthreads();
      const int e = c0 + (threadIdx.x & 127), half = threadIdx.x >> 7;  // totals, then those before
      if (e < P.stride) {
        int sum = 0;
#pragma unroll
        for (int i = 0; i < kPlanWarps; ++i) sum += wc[i * 256 + half * 128 + (threadIdx.x & 127)];
        (half ? before : total)[e] = sum;
      }
      __syncthreads();
    }
  }
  // The last block to have read the counts clears them.
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(P.ticket, 1u) == gridDim.x - 1;
  for (int i = threadIdx.x; i < kPlanWarps * E; i += kPlanThreads) wc[i] = 0;
  __syncthreads();
  if (last) {
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(P.blocks) * P.stride / 4; i += kPlanThreads)
      reinterpret_cast<int4*>(P.counts)[i] = make_int4(0, 0, 0, 0);
    if (threadIdx.x == 0) *P.ticket = 0u;
  }
  const int all = plan_scan_experts(total, E, sh);
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < E; e += kPlanThreads) P.offsets[e] = total[e];
    if (threadIdx.x == 0) P.offsets[E] = all;
  }
  const int rounds = (n + kPlanThreads - 1) / kPlanThreads;
  int expert[kPlanRounds], rank[kPlanRounds];
  plan_rank<kPlanRounds>(load, n, rounds, E, P.err, wc, expert, rank);
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kPlanThreads) total[e] += before[e];
  __syncthreads();
  plan_place<kPlanRounds>(total, wc, E, n, first, rounds, expert, rank, P.order, P.position);
}

}  // namespace

spmvb_status PlanSpace::alloc(int64_t tokens, int k, int experts) {
  const int64_t blocks = std::max<int64_t>(1, ceil_div(tokens, plan_tile_tokens(k) * plan_block_tiles(k)));
  const int stride = plan_stride(experts);
  SPMVB_TRY(counts.alloc(static_cast<size_t>(blocks) * stride * 4));
  SPMVB_TRY(prefix.alloc(blocks > kPlanOwnBlocks ? static_cast<size_t>(blocks) * stride * 4 : 16));
  SPMVB_TRY(totals.alloc(static_cast<size_t>(stride) * 4));
  SPMVB_TRY(ticket.alloc(4));
  return SPMVB_OK;
}

PlanView plan_view(const PlanSpace& space, const int* indices, int64_t tokens, int k, int experts, int* err) {
  PlanView P{};
  P.indices = indices;
  P.entries = tokens * k;
  P.experts = experts;
  P.stride = plan_stride(experts);
  P.tile_entries = plan_tile_tokens(k) * k;
  P.block_tiles = plan_block_tiles(k);
  P.blocks = static_cast<int>(ceil_div(tokens, plan_tile_tokens(k) * P.block_tiles));
  P.counts = space.counts.as<int>();
  P.prefix = space.prefix.as<int>();
  P.totals = space.totals.as<int>();
  P.ticket = space.ticket.as<unsigned>();
  P.err = err;
  return P;
}

spmvb_status launch_plan(const PlanView& P, bool counted, cudaStream_t s) {
  if (P.entries == 0) {
    SPMVB_TRY_CUDA(cudaMemsetAsync(P.offsets, 0, (static_cast<size_t>(P.experts) + 1) * 4, s));
    return SPMVB_OK;
  }
  const bool scanned = P.blocks > kPlanOwnBlocks;
  if (P.blocks > 1 && !counted) {
    plan_counts<<<P.blocks, kPlanThreads, 0, s>>>(P);
    count_launch();
  }
  if (scanned) {
    plan_scan<<<static_cast<int>(ceil_div(P.experts, kPlanWarps)), kPlanThreads, 0, s>>>(P);
    count_launch();
  }
  const size_t shared = (static_cast<size_t>(kPlanWarps) * std::max(P.experts, 256) + 2 * P.stride) * 4;
  plan_scatter<<<P.blocks, kPlanThreads, shared, s>>>(P, scanned);
  count_launch();
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // namespace spmvb
