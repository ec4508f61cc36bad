// Routing of tokens to experts: the choice, its weights and their gradient,
// and the plan that orders the choices by expert.
//
// The choice. One warp per token. The lanes are divided among the groups
// (`lanes` of them to a group, a power of two) and hold EPL experts each, so the
// order of (lane, slot) is the order of the experts. Each expert gets one
// 32-bit key: a fixed-point value q of what it is ranked by in the high bits,
// its slot number, descending, in the low ones. A lane sorts its keys once;
// a choice is then one warp-wide maximum, which names the expert and breaks
// ties by itself, and the lane that held it moves its list up.
//
// A row of 256 fp32 logits takes 2.9 us of HBM time for 16,384 tokens; the
// instructions for ranking them bound the kernel, which is why the keys are
// single words. What q stands for:
//   no bias, 16-bit logits  the logit itself, exactly
//   no bias, fp32 logits    its place between the row's least and largest
//                           logit: rounded, but in order, so only equal q of
//                           unequal logits are in doubt
//   bias                    score + bias between the least and largest that
//                           can occur, with an error of `tol` units at most
// Where two neighbours in the result lie so close that the error could have
// exchanged them (or two groups' values at the border of the kept ones), the
// row is done again in fp64 (choose_exact): about 0.5% of the rows of 256
// sigmoid scores. Two experts can lie closer together than fp32 resolves, and
// the choice between them must not depend on the rounding of exp.
#include <cmath>

#include "plan.cuh"

namespace spmvb {
namespace {

constexpr int kRouteThreads = 256;
constexpr unsigned kAll = 0xffffffffu;

template <typename A>
__device__ __forceinline__ A warp_max(A v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, off));
  return v;
}
template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(kAll, v, off);
  return v;
}

// How a router's experts lie in a warp.
struct RouteShape {
  spmvb_router_spec s;
  int per;    // experts of a group
  int lanes;  // lanes of a group
};

// Bits of a slot's number (lane * EPL + slot), and those left for q, which an
// fp32 sum with 2^23 rounds to an integer: 23 at most.
constexpr int slot_bits(int epl) { return epl == 1 ? 5 : 1 + slot_bits(epl / 2); }
constexpr int value_bits(int epl) { return slot_bits(epl) > 9 ? 32 - slot_bits(epl) : 23; }

// fp32 as an int in the same order (-0 as 0).
__device__ __forceinline__ int ordered(float v) {
  const int b = __float_as_int(v + 0.f);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int b) { return __int_as_float(b ^ ((b >> 31) & 0x7fffffff)); }

// A 16-bit float's bits in order, above 0 for every finite value.
template <typename T>
__device__ __forceinline__ unsigned ordered16(T v) {
  const unsigned b = *reinterpret_cast<const uint16_t*>(&v);
  return b & 0x8000u ? (b == 0x8000u ? 0x8000u : 0xffffu ^ b) : b | 0x8000u;
}

// Descending order of N keys (Batcher's odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b);
            k[i + j + q] = min(a, b);
          }
}

// The choice of one row in fp64, from its logits each time they are needed:
// lane j returns the j-th expert, -1 for none.
template <typename T>
__device__ __noinline__ int choose_exact(const RouteShape& S, const T* __restrict__ row, const float* __restrict__ bias,
                                         int epl) {
  const int lane = threadIdx.x & 31, group = lane / S.lanes, first = (lane % S.lanes) * epl;
  const int own = group < S.s.groups ? max(0, min(epl, S.per - first)) : 0;
  const int e0 = group * S.per + first;
  const bool softmax = S.s.score == SPMVB_SOFTMAX;
  double top = -INFINITY, sum = 0;
  if (softmax) {
#pragma unroll 1
    for (int i = 0; i < own; ++i) top = fmax(top, static_cast<double>(widen(row[e0 + i])));
    top = warp_max(top);
#pragma unroll 1
    for (int i = 0; i < own; ++i) {
      const double l = widen(row[e0 + i]);
      if (l > -INFINITY) sum += exp(l - top);
    }
    sum = warp_sum(sum);
  }
  const auto score = [&](double l) { return softmax ? exp(l - top) / sum : 1.0 / (1.0 + exp(-l)); };
  const auto rank = [&](int i) -> double {
    const double l = widen(row[e0 + i]);
    if (!(l > -INFINITY)) return -INFINITY;
    const double c = bias ? score(l) + static_cast<double>(bias[e0 + i]) : l;
    return c > -INFINITY ? c : -INFINITY;
  };
  bool open = own > 0;
  if (S.s.groups > 1) {
    double a = -INFINITY, b = -INFINITY;
#pragma unroll 1
    for (int i = 0; i < own; ++i) {
      double v = rank(i);
      if (!bias && S.s.group_top == 2 && v > -INFINITY) v = score(v);
      if (v > a) { b = a; a = v; } else if (v > b) { b = v; }
    }
    for (int off = S.lanes / 2; off > 0; off >>= 1) {
      const double a2 = __shfl_xor_sync(kAll, a, off), b2 = __shfl_xor_sync(kAll, b, off);
      b = fmax(fmin(a, a2), fmax(b, b2));
      a = fmax(a, a2);
    }
    const double level = S.s.group_top == 2 && b > -INFINITY ? a + b : a;
    int better = 0;
    for (int g = 0; g < S.s.groups; ++g) {
      const double v = __shfl_sync(kAll, level, g * S.lanes);
      better += v > level || (v == level && g < group);
    }
    open = open && better < S.s.groups_kept;
  }
  uint64_t taken = 0;
  int mine = -1;
#pragma unroll 1
  for (int j = 0; j < S.s.k; ++j) {
    double v = -INFINITY;
    int e = INT32_MAX;
#pragma unroll 1
    for (int i = 0; open && i < own; ++i) {
      if (taken >> i & 1u) continue;
      const double c = rank(i);
      if (c > v) { v = c; e = e0 + i; }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const double v2 = __shfl_xor_sync(kAll, v, off);
      const int e2 = __shfl_xor_sync(kAll, e, off);
      if (v2 > v || (v2 == v && e2 < e)) { v = v2; e = e2; }
    }
    if (!(v > -INFINITY)) break;
    if (e >= e0 && e < e0 + own) taken |= uint64_t(1) << (e - e0);
    if (lane == j) mine = e;
  }
  return mine;
}

__device__ __forceinline__ float exp_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

// What a warp keeps of the bias for all its rows: per expert its place on the
// scale of q, and the scale.
template <int EPL>
struct BiasScale {
  float at[EPL];  // 2^23 + 1 + (bias - least) * scale; NaN: not available
  float scale;    // units per score
  int zero;       // q of score + bias = 0
  bool exact;     // no scale: every row goes to choose_exact
};

template <int EPL, int Q>
__device__ __forceinline__ void load_bias(const RouteShape& S, const float* __restrict__ bias, int e0, int own,
                                          BiasScale<EPL>& B) {
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    B.at[i] = i < own ? __ldg(bias + e0 + i) : NAN;
    if (B.at[i] > -INFINITY) {
      lo = fminf(lo, B.at[i]);
      hi = fmaxf(hi, B.at[i]);
    }
  }
  lo = -warp_max(-lo);
  hi = warp_max(hi);
  // Scores are within [0, 1 + 2^-17].
  B.scale = static_cast<float>((1 << Q) - 16) / (hi - lo + 1.0001f);
  // No finite range, one that leaves q no resolution, or one that is far from 0.
  B.exact = !(B.scale > 1.f) || !(fabsf(lo) * B.scale < 8e6f);
  B.zero = B.exact ? 0 : __float2int_rn(-lo * B.scale) + 1;
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    B.at[i] = B.at[i] > -INFINITY ? fmaf(B.at[i] - lo, B.scale, 8388609.f) : NAN;
}

// Routes one row; lane j returns its j-th choice (expert or -1) and weight.
template <typename T, int EPL, bool Bias>
__device__ __forceinline__ void route_row(const RouteShape& S, const T* __restrict__ row, bool whole,
                                          const float* __restrict__ bias, const BiasScale<EPL>& B, int& mine,
                                          float& weight) {
  constexpr int Slots = slot_bits(EPL);
  constexpr bool Exact16 = !Bias && sizeof(T) == 2;
  constexpr int Shift = Exact16 ? 16 : Slots;  // key = q << Shift | (all ones - slot number)
  constexpr int Q = value_bits(EPL);
  const int lane = threadIdx.x & 31, group = lane / S.lanes, first = (lane % S.lanes) * EPL;
  const int own = group < S.s.groups ? max(0, min(EPL, S.per - first)) : 0;
  const int e0 = group * S.per + first;
  const int k = S.s.k;
  const bool softmax = S.s.score == SPMVB_SOFTMAX;

  Pack<T, EPL * static_cast<int>(sizeof(T))> in;
  if (whole) {  // every slot is an expert, the rows allow wide loads
    constexpr int VB = EPL * sizeof(T) > 16 ? 16 : EPL * static_cast<int>(sizeof(T));
    constexpr int N = Pack<T, VB>::N;
#pragma unroll
    for (int i = 0; i < EPL; i += N) {
      const Pack<T, VB> p = ld_pack<T, VB>(row + lane * EPL + i);
#pragma unroll
      for (int q = 0; q < N; ++q) in.v[i + q] = p.v[q];
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) in.v[i] = i < own ? row[e0 + i] : narrow<T, float>(-INFINITY);
  }
  float l[EPL], top = -INFINITY;
  bool poison = false;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    l[i] = widen(in.v[i]);
    poison |= !(l[i] < INFINITY);
    top = fmaxf(top, l[i]);
  }
  float sum = 0.f;
  poison = softmax && __any_sync(kAll, poison);
  if (poison) {
    mine = -1;
    weight = NAN;
    return;
  }
  // Scores, where the ranking or the weights need those of the whole row.
  const bool level_scores = !Bias && S.s.groups > 1 && S.s.group_top == 2;
  float score[EPL];
  if (softmax) top = unordered(__reduce_max_sync(kAll, ordered(top)));
  if (Bias || level_scores || (softmax && !S.s.renormalise)) {
    if (softmax) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        score[i] = l[i] > -INFINITY ? exp_fast(l[i] - top) : 0.f;
        sum += score[i];
      }
      sum = warp_sum(sum);
      const float inv = sum > 0.f ? __fdividef(1.f, sum) : 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) score[i] *= inv;
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) score[i] = __fdividef(1.f, 1.f + exp_fast(fminf(-l[i], 80.f)));
    }
  }
  // Keys. `tol`: units of q that two of them may be off against each other.
  uint32_t key[EPL];
  const uint32_t low0 = (1u << Slots) - 1u - static_cast<uint32_t>(lane * EPL);
  const uint32_t base0 = low0 - (0x4b000000u << Shift);  // takes the exponent of 2^23 + q off
  // A score's error, absolute: exp2 (2^-22) and its argument (1.5 * 2^-24 |l|),
  // 1 +, and the quotient, weighted by s (1 - s) under the sigmoid: 2.6e-7.
  // Under the softmax relative to the largest score 1 / sum: the same and the
  // sum's own error, below 4e-6.
  const float off = softmax ? 7.7e-6f * (sum > 0.f ? __fdividef(1.f, sum) : 0.f) + 1.2e-7f : 4.8e-7f;
  int tol = -1;
  bool exact = false;
  if constexpr (Bias) {
    tol = static_cast<int>(2.f * (off * B.scale + 1.5f)) + 1;
    exact = B.exact;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float f = fmaf(score[i], B.scale, B.at[i]);  // NaN: not available
      key[i] = f > 0.f && l[i] > -INFINITY ? (__float_as_uint(f) << Shift) + (base0 - i) : 0u;
    }
  } else if constexpr (Exact16) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = l[i] > -INFINITY ? ordered16(in.v[i]) << Shift | (low0 - i) : 0u;
  } else {
    tol = 0;
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (l[i] > -INFINITY) {
        lo = fminf(lo, l[i]);
        hi = fmaxf(hi, l[i]);
      }
    lo = unordered(__reduce_min_sync(kAll, ordered(lo)));
    hi = unordered(__reduce_max_sync(kAll, ordered(hi)));
    // +inf or a range past fp32: one q for all, and fp64 decides.
    float scale = static_cast<float>((1 << Q) - 16) / (hi - lo);
    if (!(scale < 1e30f)) scale = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const float f = scale > 0.f ? fmaf(l[i] - lo, scale, 8388609.f) : 8388609.f;
      key[i] = l[i] > -INFINITY ? (__float_as_uint(f) << Shift) + (base0 - i) : 0u;
    }
  }
  sort_keys<EPL>(key);
  if (S.s.groups > 1) {
    uint32_t a, b;
    int level_tol = tol;
    if (level_scores) {
      a = b = 0u;
      level_tol = static_cast<int>(4.f * (off * 8388592.f + 1.f)) + 1;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const uint32_t v = l[i] > -INFINITY ? __float_as_uint(fmaf(score[i], 8380000.f, 8388609.f)) & 0x7fffffu : 0u;
        b = max(b, min(a, v));
        a = max(a, v);
      }
    } else {
      a = key[0] >> Shift;
      b = S.s.group_top == 2 && EPL > 1 ? key[EPL > 1 ? 1 : 0] >> Shift : 0u;
      if (tol > 0 && S.s.group_top == 2) level_tol = 2 * tol;
    }
    for (int o = S.lanes / 2; o > 0; o >>= 1) {
      const uint32_t a2 = __shfl_xor_sync(kAll, a, o), b2 = __shfl_xor_sync(kAll, b, o);
      b = max(min(a, a2), max(b, b2));
      a = max(a, a2);
    }
    // A group of one available expert has no second score: 0 is added.
    const int zero = Bias ? B.zero : 1;
    const int level = a == 0u ? INT32_MIN : static_cast<int>(a) + (S.s.group_top == 1 ? 0 : b ? static_cast<int>(b) : zero);
    int better = 0;
    for (int g = 0; g < S.s.groups; ++g) {
      const int v = __shfl_sync(kAll, level, g * S.lanes);
      better += v > level || (v == level && g < group);
    }
    const bool kept = group < S.s.groups && better < S.s.groups_kept;
    const int least = __reduce_min_sync(kAll, kept ? level : INT32_MAX);
    const int next = __reduce_max_sync(kAll, kept || group >= S.s.groups ? INT32_MIN : level);
    exact |= next > INT32_MIN && least - next <= level_tol;
    if (!kept) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) key[i] = 0u;
    }
  }
  uint32_t picked = 0u, after = 0u;  // lane j: the j-th key and the one after it
  for (int j = 0; j <= k; ++j) {
    const uint32_t m = __reduce_max_sync(kAll, key[0]);
    if (lane == j) picked = m;
    if (lane == j - 1) after = m;
    if (m == 0u) break;
    if (key[0] == m) {
#pragma unroll
      for (int i = 0; i + 1 < EPL; ++i) key[i] = key[i + 1];
      key[EPL - 1] = 0u;
    }
  }
  if (lane >= k) picked = 0u;
  const auto expert = [&](uint32_t v) {
    const int slot = static_cast<int>((1u << Slots) - 1u - (v & ((1u << Slots) - 1u)));
    const int ln = slot / EPL;
    return ln / S.lanes * S.per + (ln % S.lanes) * EPL + slot % EPL;
  };
  mine = picked ? expert(picked) : -1;
  if (!Exact16 && picked && after && static_cast<int>((picked >> Shift) - (after >> Shift)) <= tol) {
    const int other = expert(after);  // the same logit and bias: equal, and in order
    const bool same = widen(row[mine]) == widen(row[other]) && (!Bias || bias[mine] == bias[other]);
    exact |= !same;
  }
  if (__any_sync(kAll, exact)) mine = choose_exact<T>(S, row, Bias ? bias : nullptr, EPL);

  const float ml = mine >= 0 ? static_cast<float>(widen(row[mine])) : -INFINITY;
  float w = 0.f;
  if (S.s.renormalise) {
    // Shares of the chosen scores, from a common factor taken out of them:
    // exp(l - m) under the softmax; under the sigmoid, where m <= 0,
    // exp(l - m) / (1 + exp(l)) = sigmoid(l) * exp(-m).
    float m = warp_max(ml);
    if (!softmax) m = fminf(m, 0.f);
    if (mine >= 0)
      w = softmax ? expf(ml - m) : ml > 0.f ? 1.f / (1.f + expf(-ml)) : expf(ml - m) / (1.f + expf(ml));
    const float all = warp_sum(w);
    w = all > 0.f ? w / all : 0.f;
  } else if (mine >= 0) {
    w = softmax ? expf(ml - top) / sum : 1.f / (1.f + expf(-ml));
  }
  weight = w * S.s.scale;
}

// A block takes the tokens of a tile (all tiles in turn where no plan is made),
// a warp one row at a time. With a plan it also leaves the tile's counts of
// each expert, or, if the tile is all there is, the plan itself.
enum class PlanPart { None, Counts, Whole };

template <typename T, int EPL, bool Bias>
__global__ void __launch_bounds__(kRouteThreads)
    route_rows(RouteShape S, const T* __restrict__ logits, int64_t ld, bool whole, const float* __restrict__ bias,
               int tokens, int tile_tokens, int* __restrict__ indices, float* __restrict__ weights, PlanPart part,
               PlanView P) {
  extern __shared__ int shared[];  // chosen[tile_entries], then the plan's
  __shared__ int sh[kPlanWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, k = S.s.k, E = S.s.experts;
  BiasScale<EPL> B{};
  if constexpr (Bias) {
    const int group = lane / S.lanes, first = (lane % S.lanes) * EPL;
    load_bias<EPL, value_bits(EPL)>(S, bias, group * S.per + first,
                                    group < S.s.groups ? max(0, min(EPL, S.per - first)) : 0, B);
  }
  int* counts = shared + tile_tokens * k;
  if (part == PlanPart::Counts) {
    for (int e = threadIdx.x; e < P.stride; e += kRouteThreads) counts[e] = 0;
    __syncthreads();
  }
  const int t0 = blockIdx.x * tile_tokens, n = min(tile_tokens, tokens - t0);
  for (int i = w; i < n; i += kRouteThreads / 32) {
    const int64_t t = t0 + i;
    int mine;
    float weight;
    route_row<T, EPL, Bias>(S, logits + t * ld, whole, bias, B, mine, weight);
    if (lane < k) {
      indices[t * k + lane] = mine;
      weights[t * k + lane] = weight;
      if (part == PlanPart::Counts && mine >= 0) atomicAdd(&counts[mine], 1);
      if (part == PlanPart::Whole) shared[i * k + lane] = mine;
    }
  }
  if (part == PlanPart::None) return;
  __syncthreads();
  if (part == PlanPart::Counts) {
    for (int e = threadIdx.x; e < P.stride; e += kRouteThreads)
      P.counts[static_cast<int64_t>(blockIdx.x) * P.stride + e] = static_cast<uint16_t>(counts[e]);
  } else {
    plan_alone<2>([&](int i) { return shared[i]; }, n * k, E, counts, counts + kPlanWarps * E, sh, P.offsets, P.order,
                  P.position);
  }
}

// dlogits of a token. With share p_j of the j-th choice and g = sum_i p_i dw_i:
//   renormalised      scale * p_j * (dw_j - g), times 1 - s_j under the sigmoid
//   sigmoid           scale * s_j * (1 - s_j) * dw_j
//   softmax           scale * p_e * ([e chosen] dw_e - g) for every expert
template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteThreads)
    route_grad_rows(spmvb_router_spec S, const T* __restrict__ logits, int64_t ld, int tokens,
                    const int* __restrict__ indices, const float* __restrict__ dweights, T* __restrict__ dlogits,
                    int64_t ldd, int* __restrict__ err) {
  const int t = blockIdx.x * (kRouteThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= tokens) return;
  const int E = S.experts, k = S.k;
  const T* row = logits + t * ld;
  int e = -1;
  float dw = 0.f, le = -INFINITY;
  if (lane < k) {
    e = indices[static_cast<int64_t>(t) * k + lane];
    if (e >= E) *err = 1;
    if (e < 0 || e >= E) e = -1;
    if (e >= 0) {
      dw = dweights[static_cast<int64_t>(t) * k + lane] * S.scale;
      le = static_cast<float>(widen(row[e]));
    }
  }
  float d = 0.f, g[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) g[i] = 0.f;
  float l[EPL], top = -INFINITY;
  bool poison = false;
  if (S.score == SPMVB_SOFTMAX) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int x = lane * EPL + i;
      l[i] = x < E ? static_cast<float>(widen(row[x])) : -INFINITY;
      poison |= isnan(l[i]) || l[i] == INFINITY;
      top = fmaxf(top, l[i]);
    }
    poison = __any_sync(kAll, poison);
  }
  if (S.renormalise) {
    float m = warp_max(le);
    if (S.score == SPMVB_SIGMOID) m = fminf(m, 0.f);
    float s = 0.f, rest = 1.f;
    if (e >= 0) {
      if (S.score == SPMVB_SOFTMAX) {
        s = expf(le - m);
      } else {
        s = le > 0 ? 1.f / (1.f + expf(-le)) : expf(le - m) / (1.f + expf(le));
        rest = 1.f / (1.f + expf(le));
      }
    }
    const float sum = warp_sum(s);
    const float p = sum > 0 ? s / sum : 0.f;
    d = p * (dw - warp_sum(p * dw)) * rest;
  } else if (S.score == SPMVB_SIGMOID) {
    if (e >= 0) d = dw / (1.f + expf(-le)) / (1.f + expf(le));
  } else {
    top = warp_max(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      l[i] = l[i] > -INFINITY ? expf(l[i] - top) : 0.f;
      sum += l[i];
    }
    sum = warp_sum(sum);
    const float inv = sum > 0 ? 1.f / sum : 0.f;
    if (e >= 0) d = dw * expf(le - top) * inv;
    const float all = warp_sum(d);
#pragma unroll
    for (int i = 0; i < EPL; ++i) g[i] = -l[i] * inv * all;
  }
  for (int j = 0; j < k; ++j) {
    const int ej = __shfl_sync(kAll, e, j);
    const float dj = __shfl_sync(kAll, d, j);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane * EPL + i == ej) g[i] += dj;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int x = lane * EPL + i;
    if (x < E) dlogits[t * ldd + x] = narrow<T, float>(poison ? NAN : g[i]);
  }
}

// Lanes of a group: the warp shared out among the groups, a power of two each.
int lanes_per_group(const spmvb_router_spec& s) {
  int lanes = 32;
  while (lanes * s.groups > 32) lanes /= 2;
  return lanes;
}
// Experts of a lane, rounded up to a power of two: at most 64, as of 1,020
// experts in 17 groups.
int slots_per_lane(const spmvb_router_spec& s) {
  int slots = 1;
  while (slots * lanes_per_group(s) < s.experts / s.groups) slots *= 2;
  return slots;
}

int slots_for(int experts) {
  int slots = 1;
  while (slots * 32 < experts) slots *= 2;
  return slots;
}

template <typename F>
spmvb_status with_logits(spmvb_dtype d, int slots, F&& f) {
  const auto by_lane = [&](auto tv) -> spmvb_status {
    using std::integral_constant;
    switch (slots) {
      case 1: return f(tv, integral_constant<int, 1>{});
      case 2: return f(tv, integral_constant<int, 2>{});
      case 4: return f(tv, integral_constant<int, 4>{});
      case 8: return f(tv, integral_constant<int, 8>{});
      case 16: return f(tv, integral_constant<int, 16>{});
      case 32: return f(tv, integral_constant<int, 32>{});
    }
    return f(tv, integral_constant<int, 64>{});
  };
  if (d == SPMVB_F32) return by_lane(float{});
  if (d == SPMVB_F16) return by_lane(__half{});
  return by_lane(__nv_bfloat16{});
}

}  // namespace
}  // namespace spmvb

struct spmvb_router_st {
  spmvb_context ctx = nullptr;
  spmvb_router_spec spec{};
  int device = 0, max_tokens = 0;
  spmvb::PlanSpace plan;
};

using namespace spmvb;

namespace {

// What every exchange call checks of its handle, sizes and positions.
spmvb_status exchange_args(spmvb_router R, spmvb_dtype dtype, int tokens, int width, int rows, const int* position) {
  if (!R) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null router");
  if (!half_or_float(dtype)) return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype");
  if (tokens < 0 || width < 1 || rows < 0)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "tokens and rows must not be negative, width must be positive");
  if (static_cast<int64_t>(tokens) * R->spec.k > INT32_MAX)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "tokens * k exceeds the int32 index range");
  const int64_t n = static_cast<int64_t>(tokens) * R->spec.k;
  return check_rows({position, n > 0, n, n, 4, "position"}, R->device);
}

RowSet entries_of(const void* p, int64_t n, const char* name) { return {p, n > 0, n, n, 4, name}; }

// Checks a plan's outputs and fills in its view.
spmvb_status plan_args(spmvb_router R, int tokens, const int* indices, int* offsets, int* order, int* position,
                       PlanView* P) {
  if (tokens < 0 || tokens > R->max_tokens)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "tokens must be in [0, max_tokens = " + std::to_string(R->max_tokens) + "]");
  const int64_t n = static_cast<int64_t>(tokens) * R->spec.k;
  const RowSet idx = entries_of(indices, n, "indices"), off = entries_of(offsets, R->spec.experts + 1, "offsets"),
               ord = entries_of(order, n, "order"), pos = entries_of(position, n, "position");
  for (const RowSet* r : {&off, &ord, &pos}) {
    SPMVB_TRY(check_rows(*r, R->device));
    SPMVB_TRY(check_apart(*r, idx));
  }
  SPMVB_TRY(check_apart(off, ord));
  SPMVB_TRY(check_apart(off, pos));
  SPMVB_TRY(check_apart(ord, pos));
  *P = plan_view(R->plan, indices, tokens, R->spec.k, R->spec.experts, R->ctx->index_err());
  P->offsets = offsets;
  P->order = order;
  P->position = position;
  return SPMVB_OK;
}

}  // namespace

extern "C" {

spmvb_status spmvb_router_check(const spmvb_router_spec* spec) {
  clear_error();
  if (!spec) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null spec");
  const auto& s = *spec;
  if (s.experts < 1 || s.experts > 1024) return fail(SPMVB_ERR_INVALID_ARGUMENT, "experts must be in [1, 1024]");
  if (s.score != SPMVB_SOFTMAX && s.score != SPMVB_SIGMOID) return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad score");
  if (s.groups < 1 || s.groups > 32 || s.experts % s.groups)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "groups must be in [1, 32] and divide experts");
  if (s.groups_kept < 1 || s.groups_kept > s.groups)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "groups_kept must be in [1, groups]");
  if (s.group_top != 1 && s.group_top != 2) return fail(SPMVB_ERR_INVALID_ARGUMENT, "group_top must be 1 or 2");
  if (s.k < 1 || s.k > 32 || s.k > s.experts / s.groups * s.groups_kept)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "k must be in [1, 32] and at most the experts of the kept groups");
  if (!std::isfinite(s.scale)) return fail(SPMVB_ERR_INVALID_ARGUMENT, "scale must be finite");
  return SPMVB_OK;
}

spmvb_status spmvb_router_create(spmvb_context ctx, const spmvb_router_spec* spec, int32_t max_tokens,
                                 spmvb_router* out) {
  SPMVB_TRY(spmvb_router_check(spec));
  if (!ctx || !out) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null context or output");
  if (max_tokens < 0 || static_cast<int64_t>(max_tokens) * spec->k > INT32_MAX)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "max_tokens * k must be in the int32 index range");
  return constructed([&]() -> spmvb_status {
    DeviceGuard g(ctx->device);
    auto R = std::make_unique<spmvb_router_st>();
    R->ctx = ctx;
    R->device = ctx->device;
    R->spec = *spec;
    R->max_tokens = max_tokens;
    SPMVB_TRY(R->plan.alloc(max_tokens, spec->k, spec->experts));
    *out = R.release();
    return SPMVB_OK;
  });
}

spmvb_status spmvb_router_destroy(spmvb_router R) {
  clear_error();
  if (R) {
    DeviceGuard g(R->device);
    delete R;
  }
  return SPMVB_OK;
}

spmvb_status spmvb_router_plan(spmvb_router R, int32_t tokens, const int32_t* d_indices, int32_t* d_offsets,
                               int32_t* d_order, int32_t* d_position, void* stream) {
  clear_error();
  if (!R) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null router");
  DeviceGuard g(R->device);
  PlanView P{};
  SPMVB_TRY(plan_args(R, tokens, d_indices, d_offsets, d_order, d_position, &P));
  SPMVB_TRY(check_rows(entries_of(d_indices, P.entries, "indices"), R->device));
  return launch_plan(P, false, static_cast<cudaStream_t>(stream));
}

spmvb_status spmvb_router_route(spmvb_router R, spmvb_dtype dtype, int32_t tokens, const void* d_logits,
                                int64_t ld_logits, const float* d_bias, int32_t* d_indices, float* d_weights,
                                int32_t* d_offsets, int32_t* d_order, int32_t* d_position, void* stream) {
  clear_error();
  if (!R) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null router");
  if (!half_or_float(dtype)) return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype");
  const bool plan = d_offsets || d_order || d_position;
  if (plan && !(d_offsets && (tokens == 0 || (d_order && d_position))))
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "offsets, order and position come together");
  if (tokens < 0) return fail(SPMVB_ERR_INVALID_ARGUMENT, "negative tokens");
  const auto& S = R->spec;
  const int dev = R->device;
  const int64_t n = static_cast<int64_t>(tokens) * S.k;
  if (n > INT32_MAX) return fail(SPMVB_ERR_INVALID_ARGUMENT, "tokens * k exceeds the int32 index range");
  const RowSet logits{d_logits, tokens, ld_logits, S.experts, dtype_size(dtype), "logits"},
      bias = entries_of(d_bias, d_bias ? S.experts : 0, "bias"), idx = entries_of(d_indices, n, "indices"),
      weights = entries_of(d_weights, n, "weights");
  const auto s = static_cast<cudaStream_t>(stream);
  DeviceGuard g(dev);
  for (const RowSet* r : {&logits, &bias, &idx, &weights}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* o : {&idx, &weights})
    for (const RowSet* r : {&logits, &bias}) SPMVB_TRY(check_apart(*o, *r));
  SPMVB_TRY(check_apart(idx, weights));
  PlanView P{};
  if (plan) {
    SPMVB_TRY(plan_args(R, tokens, d_indices, d_offsets, d_order, d_position, &P));
    for (const RowSet& o : {entries_of(d_offsets, S.experts + 1, "offsets"), entries_of(d_order, n, "order"),
                            entries_of(d_position, n, "position")})
      for (const RowSet* r : {&logits, &bias, &weights}) SPMVB_TRY(check_apart(o, *r));
  }
  const int tile = plan_tile_tokens(S.k);
  const PlanPart part = !plan ? PlanPart::None
                        : tokens <= tile ? PlanPart::Whole
                        : plan_is_one_block(P) ? PlanPart::None : PlanPart::Counts;
  if (tokens > 0) {
    SPMVB_TRY(with_logits(dtype, slots_per_lane(S), [&](auto tv, auto epl) -> spmvb_status {
      using T = decltype(tv);
      constexpr int EPL = decltype(epl)::value;
      const RouteShape shape{S, S.experts / S.groups, lanes_per_group(S)};
      const int vb = std::min<int>(16, EPL * sizeof(T));
      const bool whole = S.experts == 32 * EPL && access_bytes(sizeof(T), {{d_logits, ld_logits}}, vb / sizeof(T)) == vb;
      // Without a plan a block takes a row a warp where that many blocks have room.
      const int rows = part == PlanPart::None ? std::max(kRouteThreads / 32, static_cast<int>(ceil_div(tokens, int64_t(R->ctx->sm_count) * 4)))
                                              : tile;
      const size_t shared = part == PlanPart::None     ? 0
                            : part == PlanPart::Counts ? (static_cast<size_t>(rows) * S.k + P.stride) * 4
                                                       : (static_cast<size_t>(rows) * S.k + (kPlanWarps + 1) * S.experts) * 4;
      const auto kernel = d_bias ? route_rows<T, EPL, true> : route_rows<T, EPL, false>;
      kernel<<<static_cast<int>(ceil_div(tokens, rows)), kRouteThreads, shared, s>>>(
          shape, static_cast<const T*>(d_logits), ld_logits, whole, d_bias, tokens, rows, d_indices, d_weights, part, P);
      count_launch();
      SPMVB_TRY_CUDA(cudaGetLastError());
      return SPMVB_OK;
    }));
  }
  return plan && part != PlanPart::Whole ? launch_plan(P, part == PlanPart::Counts, s) : SPMVB_OK;
}

spmvb_status spmvb_router_route_grad(spmvb_router R, spmvb_dtype dtype, int32_t tokens, const void* d_logits,
                                     int64_t ld_logits, const int32_t* d_indices, const float* d_dweights,
                                     void* d_dlogits, int64_t ld_dlogits, void* stream) {
  clear_error();
  if (!R) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null router");
  if (!half_or_float(dtype)) return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype");
  if (tokens < 0) return fail(SPMVB_ERR_INVALID_ARGUMENT, "negative tokens");
  const auto& S = R->spec;
  const int dev = R->device;
  const int64_t n = static_cast<int64_t>(tokens) * S.k;
  if (n > INT32_MAX) return fail(SPMVB_ERR_INVALID_ARGUMENT, "tokens * k exceeds the int32 index range");
  const size_t es = dtype_size(dtype);
  const RowSet logits{d_logits, tokens, ld_logits, S.experts, es, "logits"},
      dlogits{d_dlogits, tokens, ld_dlogits, S.experts, es, "dlogits"}, idx = entries_of(d_indices, n, "indices"),
      dw = entries_of(d_dweights, n, "dweights");
  const auto s = static_cast<cudaStream_t>(stream);
  DeviceGuard g(dev);
  for (const RowSet* r : {&logits, &dlogits, &idx, &dw}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* r : {&logits, &idx, &dw}) SPMVB_TRY(check_apart(dlogits, *r));
  if (tokens == 0) return SPMVB_OK;
  return with_logits(dtype, slots_for(S.experts), [&](auto tv, auto epl) -> spmvb_status {
    using T = decltype(tv);
    route_grad_rows<T, decltype(epl)::value><<<static_cast<int>(ceil_div(tokens, kRouteThreads / 32)), kRouteThreads, 0, s>>>(
        S, static_cast<const T*>(d_logits), ld_logits, tokens, d_indices, d_dweights, static_cast<T*>(d_dlogits),
        ld_dlogits, R->ctx->index_err());
    count_launch();
    SPMVB_TRY_CUDA(cudaGetLastError());
    return SPMVB_OK;
  });
}

spmvb_status spmvb_router_dispatch(spmvb_router R, spmvb_dtype dtype, int32_t tokens, int32_t width,
                                   const int32_t* d_position, const void* d_X, int64_t ld_X, int32_t out_rows,
                                   void* d_out, int64_t ld_out, void* stream) {
  clear_error();
  SPMVB_TRY(exchange_args(R, dtype, tokens, width, out_rows, d_position));
  const int dev = R->device;
  const size_t es = dtype_size(dtype);
  const int64_t n = static_cast<int64_t>(tokens) * R->spec.k;
  const RowSet pos = entries_of(d_position, n, "position"), X{d_X, tokens, ld_X, width, es, "X"},
               out{d_out, out_rows, ld_out, width, es, "out"};
  DeviceGuard g(dev);
  for (const RowSet* r : {&X, &out}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* r : {&pos, &X}) SPMVB_TRY(check_apart(out, *r));
  return launch_dispatch(dtype, d_position, tokens, R->spec.k, X, out, R->ctx->index_err(),
                         static_cast<cudaStream_t>(stream));
}

spmvb_status spmvb_router_dispatch_grad(spmvb_router R, spmvb_dtype dtype, int32_t tokens, int32_t width,
                                        const int32_t* d_position, int32_t out_rows, const void* d_dout,
                                        int64_t ld_dout, void* d_dX, int64_t ld_dX, void* stream) {
  clear_error();
  SPMVB_TRY(exchange_args(R, dtype, tokens, width, out_rows, d_position));
  const int dev = R->device;
  const size_t es = dtype_size(dtype);
  const int64_t n = static_cast<int64_t>(tokens) * R->spec.k;
  const RowSet pos = entries_of(d_position, n, "position"), dout{d_dout, out_rows, ld_dout, width, es, "dout"},
               dX{d_dX, tokens, ld_dX, width, es, "dX"};
  DeviceGuard g(dev);
  for (const RowSet* r : {&dout, &dX}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* r : {&pos, &dout}) SPMVB_TRY(check_apart(dX, *r));
  return launch_lookup(dtype, d_position, nullptr, tokens, R->spec.k, out_rows, 1.0, dout, dX, R->ctx->index_err(),
                       static_cast<cudaStream_t>(stream));
}

spmvb_status spmvb_router_combine(spmvb_router R, spmvb_dtype dtype, int32_t tokens, int32_t width,
                                  const int32_t* d_position, const float* d_weights, int32_t y_rows, const void* d_Y,
                                  int64_t ld_Y, void* d_out, int64_t ld_out, void* stream) {
  clear_error();
  SPMVB_TRY(exchange_args(R, dtype, tokens, width, y_rows, d_position));
  const int dev = R->device;
  const size_t es = dtype_size(dtype);
  const int64_t n = static_cast<int64_t>(tokens) * R->spec.k;
  const RowSet pos = entries_of(d_position, n, "position"), w = entries_of(d_weights, n, "weights"),
               Y{d_Y, y_rows, ld_Y, width, es, "Y"}, out{d_out, tokens, ld_out, width, es, "out"};
  DeviceGuard g(dev);
  for (const RowSet* r : {&w, &Y, &out}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* r : {&pos, &w, &Y}) SPMVB_TRY(check_apart(out, *r));
  return launch_lookup(dtype, d_position, d_weights, tokens, R->spec.k, y_rows, 1.0, Y, out, R->ctx->index_err(),
                       static_cast<cudaStream_t>(stream));
}

spmvb_status spmvb_router_combine_grad(spmvb_router R, spmvb_dtype dtype, int32_t tokens, int32_t width,
                                       const int32_t* d_position, const float* d_weights, int32_t y_rows,
                                       const void* d_Y, int64_t ld_Y, const void* d_dout, int64_t ld_dout, void* d_dY,
                                       int64_t ld_dY, float* d_dweights, void* stream) {
  clear_error();
  SPMVB_TRY(exchange_args(R, dtype, tokens, width, y_rows, d_position));
  const int dev = R->device;
  const size_t es = dtype_size(dtype);
  const int64_t n = static_cast<int64_t>(tokens) * R->spec.k;
  const RowSet pos = entries_of(d_position, n, "position"), w = entries_of(d_weights, n, "weights"),
               Y{d_Y, y_rows, ld_Y, width, es, "Y"}, dout{d_dout, tokens, ld_dout, width, es, "dout"},
               dY{d_dY, y_rows, ld_dY, width, es, "dY"}, dw = entries_of(d_dweights, n, "dweights");
  DeviceGuard g(dev);
  for (const RowSet* r : {&w, &Y, &dout, &dY, &dw}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* o : {&dY, &dw})
    for (const RowSet* r : {&pos, &w, &Y, &dout}) SPMVB_TRY(check_apart(*o, *r));
  SPMVB_TRY(check_apart(dY, dw));
  return launch_combine_grad(dtype, d_position, d_weights, tokens, R->spec.k, Y, dout, dY, d_dweights,
                             R->ctx->index_err(), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
