// The expert plan: a stable counting sort of the choices by expert, and its
// shares of the kernels that make it (route.cu, plan.cu).
//
// A block is up to kPlanEntries choices of whole tokens, and has a count for
// each expert: added up by the routing kernel, tile by tile, while it has the
// choices (integer atomics: the sums do not depend on their order), or made by
// plan_counts. plan_scatter adds up the counts of all blocks, before its own and
// in total, ranks its choices among the equal ones before them and writes them
// to their places. The ranks follow the entries' order, so the plan is stable
// and does not depend on timing.
#pragma once

#include "select.cuh"

namespace spmvb {

constexpr int kPlanThreads = 256;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanEntries = 2048;                         // of a block
constexpr int kPlanRounds = kPlanEntries / kPlanThreads;   // of 32 entries a warp
constexpr int kPlanMaxExperts = 1024;

// Tokens of a tile, tiles of a block.
inline int plan_tile_tokens(int k) { return std::min(32, 512 / k); }
inline int plan_block_tiles(int k) { return kPlanEntries / (plan_tile_tokens(k) * k); }
// Row length of the blocks' counts: whole 16-byte words.
inline int plan_stride(int experts) { return (experts + 3) / 4 * 4; }

struct PlanView {
  const int* indices;
  int64_t entries;
  int experts, stride;
  int tile_entries, block_tiles;
  int blocks;
  int* counts;       // blocks x stride; 0 between calls
  int* prefix;       // blocks x stride, the choices of an expert in the blocks before (plan_scan)
  int* totals;       // stride
  unsigned* ticket;  // 0 between calls
  int *offsets, *order, *position;
  int* err;
};

__device__ __forceinline__ int plan_expert(int e, int experts, int* err) {
  if (e >= experts) {
    *err = 1;
    return -1;
  }
  return e < 0 ? -1 : e;
}

// Ranks the block's n entries from `first` on: expert[r] and rank[r] of the
// entry first + (warp * rounds + r) * 32 + lane, rank among the warp's equal
// ones; wc[warp][expert] its count. wc must be zero.
template <int Rounds, typename Load>
__device__ __forceinline__ void plan_rank(Load&& load, int n, int rounds, int experts, int* err, int* wc,
                                          int (&expert)[Rounds], int (&rank)[Rounds]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int* mine = wc + w * experts;
#pragma unroll
  for (int r = 0; r < Rounds; ++r) {
    const int i = (w * rounds + r) * 32 + lane;
    expert[r] = r < rounds && i < n ? load(i) : -1;
  }
  // After all loads: the store of the report would hold the next one back.
#pragma unroll
  for (int r = 0; r < Rounds; ++r) expert[r] = plan_expert(expert[r], experts, err);
  // The lanes with the same expert, from one vote a bit: a match instruction
  // takes a microsecond for 32 different values.
  unsigned same[Rounds];
#pragma unroll
  for (int r = 0; r < Rounds; ++r) {
    if (r >= rounds) break;
    same[r] = 0xffffffffu;
    for (int bit = 1; bit <= experts; bit <<= 1) {
      const bool on = expert[r] & bit;  // -1 is all ones, more than any expert
      const unsigned vote = __ballot_sync(0xffffffffu, on);
      same[r] &= on ? vote : ~vote;
    }
  }
#pragma unroll
  for (int r = 0; r < Rounds; ++r) {
    if (r >= rounds) break;
    const int e = expert[r];
    const unsigned before = same[r] & ((1u << lane) - 1u);
    const int base = e >= 0 ? mine[e] : 0;
    rank[r] = base + __popc(before);
    __syncwarp();
    if (e >= 0 && before == 0) mine[e] = base + __popc(same[r]);
    __syncwarp();
  }
}

// Exclusive sum over v[0..experts) by the whole block, in place; returns the
// total. experts <= 4 * kPlanThreads.
__device__ __forceinline__ int plan_scan_experts(int* v, int experts, int* sh) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x[4], own = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int e = threadIdx.x * 4 + q;
    x[q] = e < experts ? v[e] : 0;
    own += x[q];
  }
  int incl = own;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += u;
  }
  if (lane == 31) sh[w] = incl;
  __syncthreads();
  int at = incl - own, all = 0;
#pragma unroll
  for (int i = 0; i < kPlanWarps; ++i) {
    at += i < w ? sh[i] : 0;
    all += sh[i];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int e = threadIdx.x * 4 + q;
    if (e < experts) v[e] = at;
    at += x[q];
  }
  __syncthreads();
  return all;
}

// From the first place of each expert in this block (base) and the warps'
// counts, each entry's place.
template <int Rounds>
__device__ __forceinline__ void plan_place(const int* base, int* wc, int experts, int n, int64_t first, int rounds,
                                           const int (&expert)[Rounds], const int (&rank)[Rounds],
                                           int* __restrict__ order, int* __restrict__ position) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < experts; e += kPlanThreads) {
    int at = base[e];
#pragma unroll
    for (int i = 0; i < kPlanWarps; ++i) {
      const int c = wc[i * experts + e];
      wc[i * experts + e] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < Rounds; ++r) {
    const int i = (w * rounds + r) * 32 + lane;
    if (r >= rounds || i >= n) continue;
    const int e = expert[r], at = e >= 0 ? wc[w * experts + e] + rank[r] : -1;
    position[first + i] = at;
    if (e >= 0) order[at] = static_cast<int>(first + i);
  }
}

// The whole plan of at most kPlanThreads * Rounds entries by one block.
// wc: kPlanWarps * experts ints, base: experts ints, sh: kPlanWarps ints.
template <int Rounds, typename Load>
__device__ __forceinline__ void plan_alone(Load&& load, int n, int experts, int* err, int* wc, int* base, int* sh,
                                           int* __restrict__ offsets, int* __restrict__ order,
                                           int* __restrict__ position) {
  for (int i = threadIdx.x; i < kPlanWarps * experts; i += kPlanThreads) wc[i] = 0;
  __syncthreads();
  const int rounds = (n + kPlanThreads - 1) / kPlanThreads;
  int expert[Rounds], rank[Rounds];
  plan_rank<Rounds>(load, n, rounds, experts, err, wc, expert, rank);
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kPlanThreads) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPlanWarps; ++i) c += wc[i * experts + e];
    base[e] = c;
  }
  __syncthreads();
  const int all = plan_scan_experts(base, experts, sh);
  for (int e = threadIdx.x; e < experts; e += kPlanThreads) offsets[e] = base[e];
  if (threadIdx.x == 0) offsets[experts] = all;
  plan_place<Rounds>(base, wc, experts, n, 0, rounds, expert, rank, order, position);
}

// ---- host ------------------------------------------------------------------------
struct PlanSpace {
  DevBuf counts, prefix, totals, ticket;
  spmvb_status alloc(int64_t tokens, int k, int experts);
};
// Fills in everything but the outputs.
PlanView plan_view(const PlanSpace& space, const int* indices, int64_t tokens, int k, int experts, int* err);
// Enqueues the plan; `counted`: the blocks' counts have been made.
spmvb_status launch_plan(const PlanView& P, bool counted, cudaStream_t s);
// One block makes the whole plan, without counts.
inline bool plan_is_one_block(const PlanView& P) { return P.blocks <= 1; }

}  // namespace spmvb
