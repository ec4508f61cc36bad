// Kernels of the expert plan (plan.cuh).
#include "plan.cuh"

namespace spmvb {
namespace {

// Up to this many tiles every block of plan_scatter adds up all tiles' counts
// itself; beyond, plan_scan does it once.
constexpr int kPlanOwnTiles = 64;

__global__ void __launch_bounds__(kPlanThreads) plan_counts(PlanView P) {
  __shared__ int c[kPlanMaxExperts];
  for (int e = threadIdx.x; e < P.stride; e += kPlanThreads) c[e] = 0;
  __syncthreads();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * P.tile_entries;
  int x[2];  // a tile has at most 512 choices
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int i = q * kPlanThreads + threadIdx.x;
    x[q] = i < P.tile_entries && i0 + i < P.entries ? __ldg(P.indices + i0 + i) : -1;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int e = plan_expert(x[q], P.experts, P.err);
    if (e >= 0) atomicAdd(&c[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < P.stride; e += kPlanThreads)
    P.counts[static_cast<int64_t>(blockIdx.x) * P.stride + e] = static_cast<uint16_t>(c[e]);
}

__device__ __forceinline__ void unpack8(const uint4& v, int (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = w[i] & 0xffffu;
    x[2 * i + 1] = w[i] >> 16;
  }
}

// Eight experts a block: running sums of their counts over the tiles.
__global__ void __launch_bounds__(kPlanThreads) plan_scan(PlanView P) {
  __shared__ int sh[kPlanWarps][8];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, e0 = blockIdx.x * 8;
  int sum[8] = {};
  for (int t0 = 0; t0 < P.tiles; t0 += kPlanThreads) {
    const int t = t0 + threadIdx.x;
    int x[8] = {}, incl[8];
    if (t < P.tiles) unpack8(*reinterpret_cast<const uint4*>(P.counts + static_cast<int64_t>(t) * P.stride + e0), x);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      incl[q] = x[q];
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl[q], off);
        if (lane >= off) incl[q] += u;
      }
      if (lane == 31) sh[w][q] = incl[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      int at = sum[q] + incl[q] - x[q];
#pragma unroll
      for (int i = 0; i < kPlanWarps; ++i) {
        at += i < w ? sh[i][q] : 0;
        sum[q] += sh[i][q];
      }
      if (t < P.tiles) P.prefix[static_cast<int64_t>(t) * P.stride + e0 + q] = at;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0)
#pragma unroll
    for (int q = 0; q < 8; ++q) P.totals[e0 + q] = sum[q];
}

// Shared memory: wc[kPlanWarps][experts] (the counts' sums before that),
// before[stride], total[stride].
__global__ void __launch_bounds__(kPlanThreads) plan_scatter(PlanView P, bool scanned) {
  extern __shared__ int shared[];
  __shared__ int sh[kPlanWarps];
  const int E = P.experts, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int* wc = shared;
  int* before = shared + kPlanWarps * max(E, 512);
  int* total = before + P.stride;
  const int tile0 = blockIdx.x * P.block_tiles;
  const int64_t first = static_cast<int64_t>(tile0) * P.tile_entries;
  const int n = static_cast<int>(min(static_cast<int64_t>(P.tile_entries) * P.block_tiles, P.entries - first));
  const auto load = [&](int i) { return __ldg(P.indices + first + i); };
  if (P.tiles <= P.block_tiles) {
    plan_alone<kPlanRounds>(load, n, E, P.err, wc, total, sh, P.offsets, P.order, P.position);
    return;
  }
  if (scanned) {
    for (int e = threadIdx.x; e < E; e += kPlanThreads) {
      before[e] = P.prefix[static_cast<int64_t>(tile0) * P.stride + e];
      total[e] = P.totals[e];
    }
  } else {
    // 256 experts at a time: a warp takes every eighth tile, a lane eight experts.
    for (int c0 = 0; c0 < P.stride; c0 += 256) {
      const int e0 = c0 + lane * 8;
      // Two experts' sums to a word: a warp sees at most kPlanOwnTiles / 8 tiles
      // of at most 512 choices, 2^15.
      static_assert(kPlanOwnTiles / kPlanWarps * 512 < 65536);
      uint32_t a[4] = {}, b[4] = {};
      if (e0 < P.stride) {
#pragma unroll 8
        for (int t = w; t < P.tiles; t += kPlanWarps) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(P.counts + static_cast<int64_t>(t) * P.stride + e0));
          const uint32_t in = t < tile0 ? 0xffffffffu : 0u;
          a[0] += v.x; b[0] += v.x & in;
          a[1] += v.y; b[1] += v.y & in;
          a[2] += v.z; b[2] += v.z & in;
          a[3] += v.w; b[3] += v.w & in;
        }
      }
      int* ra = wc + w * 512 + lane * 8;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        ra[q] = a[q / 2] >> (q % 2 * 16) & 0xffffu;
        ra[256 + q] = b[q / 2] >> (q % 2 * 16) & 0xffffu;
      }
      __syncthreads();
      const int e = c0 + threadIdx.x;
      if (e < P.stride) {
        int sa = 0, sb = 0;
#pragma unroll
        for (int i = 0; i < kPlanWarps; ++i) {
          sa += wc[i * 512 + threadIdx.x];
          sb += wc[i * 512 + 256 + threadIdx.x];
        }
        total[e] = sa;
        before[e] = sb;
      }
      __syncthreads();
    }
  }
  for (int i = threadIdx.x; i < kPlanWarps * E; i += kPlanThreads) wc[i] = 0;
  __syncthreads();
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
  const int64_t tiles = std::max<int64_t>(1, ceil_div(tokens, plan_tile_tokens(k)));
  const int stride = plan_stride(experts);
  SPMVB_TRY(counts.alloc(static_cast<size_t>(tiles) * stride * 2));
  SPMVB_TRY(prefix.alloc(tiles > kPlanOwnTiles ? static_cast<size_t>(tiles) * stride * 4 : 16));
  SPMVB_TRY(totals.alloc(static_cast<size_t>(stride) * 4));
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
  P.tiles = static_cast<int>(ceil_div(tokens, plan_tile_tokens(k)));
  P.counts = space.counts.as<uint16_t>();
  P.prefix = space.prefix.as<int>();
  P.totals = space.totals.as<int>();
  P.err = err;
  return P;
}

spmvb_status launch_plan(const PlanView& P, bool counted, cudaStream_t s) {
  if (P.entries == 0) {
    SPMVB_TRY_CUDA(cudaMemsetAsync(P.offsets, 0, (static_cast<size_t>(P.experts) + 1) * 4, s));
    return SPMVB_OK;
  }
  const bool one = plan_is_one_block(P), scanned = P.tiles > kPlanOwnTiles;
  if (!one && !counted) {
    plan_counts<<<P.tiles, kPlanThreads, 0, s>>>(P);
    count_launch();
  }
  if (scanned) {
    plan_scan<<<P.stride / 8, kPlanThreads, 0, s>>>(P);
    count_launch();
  }
  const size_t shared = (static_cast<size_t>(kPlanWarps) * std::max(P.experts, 512) + 2 * P.stride) * 4;
  plan_scatter<<<static_cast<int>(ceil_div(P.tiles, P.block_tiles)), kPlanThreads, shared, s>>>(P, scanned);
  count_launch();
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // namespace spmvb
