// Routing of tokens to experts: the choice, its weights and their gradient,
// and the plan that orders the choices by expert.
//
// The choice. L lanes of a warp take a token (32, or 8 or 16 where that leaves a
// lane eight experts: the tokens of a warp share the instructions that are not
// per expert). The lanes are divided among the groups (2^lanes_log of
// them to a group) and hold EPL experts each, so the order of (lane, slot) is
// the order of the experts. Each expert gets one 32-bit key: a fixed-point
// value q of what it is ranked by in the high bits, its slot number,
// descending, in the low ones. A lane sorts its keys once; a choice is then
// one maximum over the lanes, which names the expert and breaks ties by
// itself, and the lane that held it moves its list up.
//
// What q stands for:
//   no bias, 16-bit logits  the logit itself, exactly
//   no bias, fp32 logits    its place between the row's least and largest
//                           logit: rounded, but in order, so only equal q of
//                           unequal logits are in doubt
//   bias                    score + bias between the least and largest that
//                           can occur, with an error of `tol` units at most
// Where two neighbours in the result lie so close that the error could have
// exchanged them, about 0.5% of the rows of 256 sigmoid scores, the two are
// compared in fp64; a row where more than two experts or two groups' values
// meet is done again in fp64 (route_exact). Two experts can lie closer together than fp32 resolves, and
// the choice between them must not depend on the rounding of exp.
#include <cmath>

#include "plan.cuh"

namespace spmvb {
namespace {

constexpr int kRouteThreads = 256;
constexpr int kRouteRows = 256;  // of a block, at most
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
  int per;        // experts of a group
  int lanes_log;  // 2^lanes_log lanes of a group
};

// Bits of a slot's number (lane * EPL + slot), and those left for q, which an
// fp32 sum with 2^23 rounds to an integer: 23 at most.
constexpr int slot_bits(int slots) { return slots == 1 ? 0 : 1 + slot_bits(slots / 2); }
constexpr int value_bits(int slots) { return slot_bits(slots) > 9 ? 32 - slot_bits(slots) : 23; }

// fp32 as an int in the same order (-0 as 0).
__device__ __forceinline__ int ordered(float v) {
  const int b = __float_as_int(v + 0.f);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int b) { return __int_as_float(b ^ ((b >> 31) & 0x7fffffff)); }

// Two 16-bit floats' bits in order (-0 as 0, NaN above infinity).
template <typename T>
__device__ __forceinline__ uint32_t ordered_pair(T a, T b) {
  uint32_t w;
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 v = __hadd2(__halves2half2(a, b), __halves2half2(__half(0.f), __half(0.f)));
    w = *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __hadd2(__halves2bfloat162(a, b), __halves2bfloat162(__nv_bfloat16(0.f), __nv_bfloat16(0.f)));
    w = *reinterpret_cast<const uint32_t*>(&v);
  }
  return w ^ ((w >> 15 & 0x00010001u) * 0xffffu | 0x80008000u);
}
// The infinities' places in that order: -inf is ~inf.
template <typename T>
constexpr uint32_t kInf16 = std::is_same_v<T, __half> ? 0xfc00u : 0xff80u;

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

// Shares of the chosen scores (lane j's logit l, -inf for none) in the chosen
// sum, from a common factor taken out of them: exp(l - m) under the softmax;
// under the sigmoid, where m <= 0, exp(l - m) / (1 + exp(l)) = sigmoid(l) * exp(-m).
__device__ __forceinline__ double chosen_share(double l, bool softmax) {
  double m = warp_max(l);
  if (!softmax) m = fmin(m, 0.0);
  double w = 0;
  if (l > -INFINITY) w = softmax ? exp(l - m) : l > 0 ? 1.0 / (1.0 + exp(-l)) : exp(l - m) / (1.0 + exp(l));
  const double all = warp_sum(w);
  return all > 0 ? w / all : 0.0;
}

// One row in fp64, by a warp: lane j returns the j-th expert (-1 for none) and
// its weight. Out of line, so that its registers are the kernel's only while
// it runs.
template <typename T, int EPL>
__device__ __noinline__ int route_exact(const RouteShape& S, const T* __restrict__ row,
                                        const float* __restrict__ bias, float& weight) {
  const int lane = threadIdx.x & 31, group = lane >> S.lanes_log, first = (lane & ((1 << S.lanes_log) - 1)) * EPL;
  const int own = group < S.s.groups ? max(0, min(EPL, S.per - first)) : 0;
  const int e0 = group * S.per + first;
  const bool softmax = S.s.score == SPMVB_SOFTMAX;
  double l[EPL], c[EPL], top = -INFINITY, sum = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    l[i] = i < own ? static_cast<double>(widen(row[e0 + i])) : -INFINITY;
    c[i] = l[i];
    top = fmax(top, l[i]);
  }
  if (softmax) top = warp_max(top);
  // Rolled up: a row in doubt comes alone, and the code has to be fetched first.
#pragma unroll 2
  for (int i = 0; i < EPL; ++i) {
    if (!(l[i] > -INFINITY)) continue;
    c[i] = softmax ? exp(l[i] - top) : 1.0 / (1.0 + exp(-l[i]));
    sum += c[i];
  }
  if (softmax) {
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (l[i] > -INFINITY) c[i] /= sum;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    if (bias && i < own) c[i] += static_cast<double>(bias[e0 + i]);
    if (!(l[i] > -INFINITY) || !(c[i] > -INFINITY)) c[i] = -INFINITY;
  }
  bool open = own > 0;
  if (S.s.groups > 1) {
    // A group's single best is by what the experts are ranked by: without a
    // bias the logits, as scores are equal long before the logits are.
    const bool by_logit = !bias && S.s.group_top == 1;
    double a = -INFINITY, b = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const double v = by_logit && c[i] > -INFINITY ? l[i] : c[i];
      if (v > a) { b = a; a = v; } else if (v > b) { b = v; }
    }
    for (int off = 1 << S.lanes_log >> 1; off > 0; off >>= 1) {
      const double a2 = __shfl_xor_sync(kAll, a, off), b2 = __shfl_xor_sync(kAll, b, off);
      b = fmax(fmin(a, a2), fmax(b, b2));
      a = fmax(a, a2);
    }
    const double level = S.s.group_top == 2 && b > -INFINITY ? a + b : a;
    int better = 0;
    for (int g = 0; g < S.s.groups; ++g) {
      const double v = __shfl_sync(kAll, level, g << S.lanes_log);
      better += v > level || (v == level && g < group);
    }
    open = open && better < S.s.groups_kept;
  }
  // Ranked by the values' bits, as integers in the same order; 0: not there.
  uint64_t key[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const double v = (bias ? c[i] : l[i]) + 0.0;  // -0 as 0
    const int64_t bits = __double_as_longlong(v);
    key[i] = open && v > -INFINITY ? static_cast<uint64_t>(bits) ^ (static_cast<uint64_t>(bits >> 63) | (1ull << 63)) : 0ull;
  }
  int mine = -1;
#pragma unroll 1
  for (int j = 0; j < S.s.k; ++j) {
    uint64_t v = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (key[i] > v) { v = key[i]; at = i; }
    const uint32_t high = __reduce_max_sync(kAll, static_cast<uint32_t>(v >> 32));
    if (high == 0u) break;
    const uint32_t low = __reduce_max_sync(kAll, v >> 32 == high ? static_cast<uint32_t>(v) : 0u);
    // The lowest lane that holds the largest value has the lowest index.
    const int from = __ffs(__ballot_sync(kAll, v == (static_cast<uint64_t>(high) << 32 | low))) - 1;
    const int e = __shfl_sync(kAll, e0 + at, from);
    if (lane == j) mine = e;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane == from && i == at) key[i] = 0ull;
  }
  const double ml = mine >= 0 ? static_cast<double>(widen(row[mine])) : -INFINITY;
  double w = 0;
  if (S.s.renormalise)
    w = chosen_share(ml, softmax);
  else if (mine >= 0)
    w = softmax ? exp(ml - top) / sum : 1.0 / (1.0 + exp(-ml));
  weight = static_cast<float>(w * S.s.scale);
  return mine;
}

__device__ __forceinline__ float exp_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// w / all, for 0 <= w <= all. Exactly 1 where one choice holds the whole sum: the
// fast quotient of two equal values is a step below 1 for one value in five,
// and a lone choice's gradient would not be 0.
__device__ __forceinline__ float share_of(float w, float all) {
  return w == all ? (all > 0.f ? 1.f : 0.f) : __fdividef(w, all);
}

// Maxima and sums over the L lanes of a row.
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  if constexpr (L == 32) return __reduce_max_sync(kAll, v);
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) v = max(v, __shfl_xor_sync(kAll, v, off));
  return v;
}
template <int L>
__device__ __forceinline__ int row_max(int v) {
  if constexpr (L == 32) return __reduce_max_sync(kAll, v);
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) v = max(v, __shfl_xor_sync(kAll, v, off));
  return v;
}
template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) v += __shfl_xor_sync(kAll, v, off);
  return v;
}
template <int L>
__device__ __forceinline__ bool row_any(bool v) {
  const unsigned all = __ballot_sync(kAll, v);
  if constexpr (L == 32) return all != 0u;
  return (all >> (threadIdx.x & 31 & ~(L - 1)) & ((1u << (L & 31)) - 1u)) != 0u;
}

// What the biases are on the scale of q, for a block's rows.
struct BiasScale {
  const float* at;  // per slot 2^23 + 1 + (bias - least) * scale; NaN: not available
  float scale;      // units per score
  int zero;         // q of score + bias = 0
  bool exact;       // no scale: every row goes to route_exact
};
// Rows of the slots' table: 16-byte words that fall on different banks.
constexpr int bias_row(int epl) { return epl >= 4 ? epl + 4 : epl; }

template <int L, int EPL>
__device__ __forceinline__ BiasScale load_bias(const RouteShape& S, const float* __restrict__ bias, float* table) {
  const int lane = threadIdx.x & 31;
  float lo = INFINITY, hi = -INFINITY;
  for (int e = lane; e < S.s.experts; e += 32) {
    const float b = __ldg(bias + e);
    if (b > -INFINITY) {
      lo = fminf(lo, b);
      hi = fmaxf(hi, b);
    }
  }
  lo = -warp_max(-lo);
  hi = warp_max(hi);
  BiasScale B;
  // Scores are within [0, 1 + 2^-17].
  B.scale = static_cast<float>((1 << value_bits(L * EPL)) - 16) / (hi - lo + 1.0001f);
  // No finite range, one that leaves q no resolution, or one that is far from 0.
  B.exact = !(B.scale > 1.f) || !(fabsf(lo) * B.scale < 8e6f);
  B.zero = B.exact ? 0 : __float2int_rn(-lo * B.scale) + 1;
  for (int i = threadIdx.x; i < L * EPL; i += kRouteThreads) {
    const int ln = i / EPL, e = (ln >> S.lanes_log) * S.per + (ln & ((1 << S.lanes_log) - 1)) * EPL + i % EPL;
    const int last = min(((ln >> S.lanes_log) + 1) * S.per, S.s.experts);  // of the lane's group
    const float b = e < last ? __ldg(bias + e) : NAN;
    table[ln * bias_row(EPL) + i % EPL] = b > -INFINITY ? fmaf(b - lo, B.scale, 8388609.f) : NAN;
  }
  B.at = table;
  return B;
}

// Routes the row of these L lanes; lane j returns its j-th choice (expert or
// -1) and weight. `list`: this lane's column of a 32-wide array of list_depth
// rows, the last of them 0. True: the result is in doubt.
constexpr int list_depth(int epl) { return epl <= 8 ? epl + 1 : 0; }
template <typename T, int L, int EPL, bool Bias>
__device__ __forceinline__ bool route_row(const RouteShape& S, const T* __restrict__ row, bool whole, const float* __restrict__ bias, const BiasScale& B,
                                          uint32_t* list, int& mine, float& weight) {
  constexpr int Slots = slot_bits(L * EPL);
  constexpr bool Exact16 = !Bias && sizeof(T) == 2;
  constexpr int Shift = Exact16 ? 16 : Slots;  // key = q << Shift | (all ones - slot number)
  constexpr int Q = value_bits(L * EPL);
  const int lane = threadIdx.x & (L - 1), group = lane >> S.lanes_log, first = (lane & ((1 << S.lanes_log) - 1)) * EPL;
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
    const int own = group < S.s.groups ? max(0, min(EPL, S.per - first)) : 0;
    const T* from = row + group * S.per + first;
#pragma unroll
    for (int i = 0; i < EPL; ++i) in.v[i] = i < own ? __ldg(from + i) : narrow<T, float>(-INFINITY);
  }
  float l[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) l[i] = widen(in.v[i]);
  uint32_t key[EPL];
  const uint32_t low0 = (1u << Slots) - 1u - static_cast<uint32_t>(lane * EPL);
  constexpr uint32_t Least = Exact16 ? ((0xffffu ^ kInf16<T>) + 1u) << 16 : 1u;  // key of an available expert
  // Under the softmax a NaN or +inf leaves the row without scores.
  bool poison = false, exact = false;
  if constexpr (Exact16) {
#pragma unroll
    for (int i = 0; i < EPL; i += 2) {
      const uint32_t o = ordered_pair<T>(in.v[i], in.v[i + 1 < EPL ? i + 1 : i]);
      key[i] = (o << 16) + (low0 - i);
      if (i + 1 < EPL) key[i + 1] = (o & 0xffff0000u) + (low0 - (i + 1));
    }
    sort_keys<EPL>(key);
    if (softmax)
      poison = row_any<L>(key[0] >= kInf16<T> << 16);
    else
      exact = key[0] > (kInf16<T> << 16 | 0xffffu);  // NaN: not available
  } else if (softmax) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) poison |= !(l[i] < INFINITY);
    poison = row_any<L>(poison);
  }
  // The row's largest logit and sum of exponentials, where the ranking or the
  // weights need the scores of the whole row.
  const bool level_scores = !Bias && S.s.groups > 1 && S.s.group_top == 2;
  float top = -INFINITY, sum = 0.f, inv = 0.f;
  if (softmax && (Bias || level_scores || !S.s.renormalise)) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) top = fmaxf(top, l[i]);
    top = unordered(row_max<L>(ordered(top)));
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += l[i] > -INFINITY ? exp_fast(l[i] - top) : 0.f;
    sum = row_sum<L>(sum);
    inv = sum > 0.f ? reciprocal(sum) : 0.f;
  }
  // Scores, NaN where there is none.
  const auto scores = [&](float (&v)[EPL]) {
    if (softmax) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) v[i] = l[i] > -INFINITY ? exp_fast(l[i] - top) * inv : NAN;
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) v[i] = l[i] > -INFINITY ? reciprocal(1.f + exp_fast(-l[i])) : NAN;
    }
  };
  // `tol`: units of q that two of them may be off against each other. A
  // score's error, absolute: exp2 (2^-22) and its argument (1.5 * 2^-24 |l|),
  // 1 +, and the quotient, weighted by s (1 - s) under the sigmoid: 2.6e-7.
  // Under the softmax relative to the largest score 1 / sum: the same and the
  // sum's own error, below 4e-6.
  const float off = softmax ? 7.7e-6f * inv + 1.2e-7f : 2.7e-7f;
  int tol = -1;
  uint32_t sa = 0u, sb = 0u;  // the two best scores on q's scale, for level_scores
  if constexpr (Bias) {
    const uint32_t base0 = low0 - (0x4b000000u << Shift);  // takes the exponent of 2^23 + q off
    tol = static_cast<int>(2.f * (off * B.scale + 1.5f)) + 1;
    exact = B.exact;
    float v[EPL];
    scores(v);
    constexpr int VB = EPL >= 4 ? 16 : EPL * 4;
    constexpr int N = VB / 4;
#pragma unroll
    for (int i = 0; i < EPL; i += N) {
      const Pack<float, VB> at = *reinterpret_cast<const Pack<float, VB>*>(B.at + lane * bias_row(EPL) + i);
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const float f = fmaf(v[i + q], B.scale, at.v[q]);  // NaN: not available
        key[i + q] = f > 0.f ? (__float_as_uint(f) << Shift) + (base0 - (i + q)) : 0u;
      }
    }
    sort_keys<EPL>(key);
  } else {
    if (level_scores) {
      float v[EPL];
      scores(v);
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const float f = fmaf(v[i], 8380000.f, 8388609.f);
        const uint32_t u = f > 0.f ? __float_as_uint(f) & 0x7fffffu : 0u;
        sb = max(sb, min(sa, u));
        sa = max(sa, u);
      }
    }
    if constexpr (!Exact16) {
      const uint32_t base0 = low0 - (0x4b000000u << Shift);
      tol = 0;
      float lo = INFINITY, hi = -INFINITY;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        lo = fminf(lo, l[i] > -INFINITY ? l[i] : INFINITY);
        hi = fmaxf(hi, l[i]);
      }
      lo = -unordered(row_max<L>(ordered(-lo)));
      hi = unordered(row_max<L>(ordered(hi)));
      // Equal logits, +inf or a range past fp32: one q for all, and fp64
      // decides where they differ.
      float scale = __fdividef(static_cast<float>((1 << Q) - 16), hi - lo);
      if (!(scale > 0.f) || !(scale < 1e30f)) scale = 0.f;
      if (scale == 0.f) lo = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const float f = scale == 0.f ? 8388609.f : fmaf(l[i] - lo, scale, 8388609.f);
        key[i] = l[i] > -INFINITY ? (__float_as_uint(f) << Shift) + (base0 - i) : 0u;
      }
      sort_keys<EPL>(key);
    }
  }
  uint32_t head = poison ? 0u : key[0];
  if (S.s.groups > 1) {
    uint32_t a, b;
    int level_tol = tol;
    if (level_scores) {
      a = sa;
      b = sb;
      level_tol = static_cast<int>(4.f * (off * 8388592.f + 1.f)) + 1;
    } else {
      a = key[0] < Least ? 0u : key[0] >> Shift;
      b = S.s.group_top == 2 && EPL > 1 ? key[EPL > 1 ? 1 : 0] >> Shift : 0u;
      if (tol > 0 && S.s.group_top == 2) level_tol = 2 * tol;
    }
    for (int o = 1 << S.lanes_log >> 1; o > 0; o >>= 1) {
      const uint32_t a2 = __shfl_xor_sync(kAll, a, o), b2 = __shfl_xor_sync(kAll, b, o);
      b = max(min(a, a2), max(b, b2));
      a = max(a, a2);
    }
    // A group of one available expert has no second score: 0 is added.
    const int zero = Bias ? B.zero : 1;
    const int level = a == 0u ? INT32_MIN : static_cast<int>(a) + (S.s.group_top == 1 ? 0 : b ? static_cast<int>(b) : zero);
    int better = 0;
#pragma unroll 4
    for (int g = 0; g < S.s.groups; ++g) {
      const int v = __shfl_sync(kAll, level, g << S.lanes_log, L);
      better += v > level || (v == level && g < group);
    }
    const bool kept = group < S.s.groups && better < S.s.groups_kept;
    const int least = ~row_max<L>(kept ? ~level : INT32_MIN);
    const int next = row_max<L>(kept || group >= S.s.groups ? INT32_MIN : level);
    exact |= next > INT32_MIN && least - next <= level_tol;
    if (!kept) head = 0u;  // its list is never moved up
  }
  // Lists wait in shared memory, where moving up is one load; the long ones
  // move through the registers. A list ends in a 0.
  constexpr int Depth = list_depth(EPL);
#pragma unroll
  for (int i = 1; i < Depth - 1; ++i) list[i * 32] = key[i < EPL ? i : 0];
  uint32_t picked = 0u, m = 0u;  // lane j: the j-th key
  const uint32_t* next_key = list;
#pragma unroll 3
  for (int j = 0; j <= k; ++j) {
    m = row_max<L>(head);
    if (lane == j) picked = m;
    if (L == 32 && m < Least) break;
    const bool up = head == m && (L == 32 || m >= Least);
    if constexpr (Depth > 0) {
      next_key += up ? 32 : 0;
      if (up) head = *next_key;
    } else if (up) {
#pragma unroll
      for (int i = 0; i + 1 < EPL; ++i) key[i] = key[i + 1];
      key[EPL - 1] = 0u;
      head = key[0];
    }
  }
  uint32_t after = __shfl_down_sync(kAll, picked, 1);
  if (lane == k - 1) after = m;  // the first one not chosen
  if (lane >= k || picked < Least) picked = 0u;
  if (after < Least) after = 0u;
  const auto expert = [&](uint32_t v) {
    const int slot = static_cast<int>((1u << Slots) - 1u - (v & ((1u << Slots) - 1u)));
    const int ln = slot / EPL;
    return (ln >> S.lanes_log) * S.per + (ln & ((1 << S.lanes_log) - 1)) * EPL + slot % EPL;
  };
  mine = picked ? expert(picked) : -1;
  // No lane takes a branch of its own up to here and below: the compiler
  // guards every vote and shuffle behind one with a synchronisation of its
  // own, which made half of this loop's instructions.
  const bool near = !Exact16 && picked && after && static_cast<int>((picked >> Shift) - (after >> Shift)) <= tol;
  if (!Exact16 && __any_sync(kAll, near)) {
    // The pair's values themselves, in fp64: is the order right? At the last
    // choice the one after the pair has to be further off.
    const int a = near ? mine : 0, b = near ? expert(after) : 0;
    double va = widen(row[a]), vb = widen(row[b]);
    if constexpr (Bias) {
      if (softmax) {
        double all = 0;
#pragma unroll 1
        for (int e = lane; e < S.s.experts; e += L) {
          const double v = widen(row[e]);
          if (v > -INFINITY) all += exp(v - static_cast<double>(top));
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) all += __shfl_xor_sync(kAll, all, o);
        va = exp(va - static_cast<double>(top)) / all;
        vb = exp(vb - static_cast<double>(top)) / all;
      } else {
        va = 1.0 / (1.0 + exp(-va));
        vb = 1.0 / (1.0 + exp(-vb));
      }
      va += static_cast<double>(bias[a]);
      vb += static_cast<double>(bias[b]);
    }
    const uint32_t third = row_max<L>(head);  // the loop's last turn took `after` off its list
    const bool crowded = lane == k - 1 && third >= Least && static_cast<int>((picked >> Shift) - (third >> Shift)) <= tol;
    // A pair in the wrong order that is near no other is exchanged.
    const bool wrong = near && !(va > vb || (va == vb && a < b));
    const int near_before = __shfl_up_sync(kAll, near, 1, L), near_after = __shfl_down_sync(kAll, near, 1, L);
    const int wrong_before = __shfl_up_sync(kAll, wrong, 1, L), before = __shfl_up_sync(kAll, a, 1, L);
    const bool beside = (lane > 0 && near_before) || (lane < k - 1 && near_after);
    exact |= (near && crowded) || (wrong && beside);
    mine = wrong ? b : lane > 0 && lane < k && wrong_before ? before : mine;
  }

  const float chosen = static_cast<float>(widen(row[max(mine, 0)]));
  const float ml = mine >= 0 ? chosen : -INFINITY;
  float w;
  if (S.s.renormalise) {
    // As chosen_share, in fp32.
    float m = unordered(row_max<L>(ordered(ml)));
    if (softmax) {
      w = expf(ml - m);
    } else {
      const float e = ml > 0.f ? 1.f : expf(ml - fminf(m, 0.f));
      w = __fdividef(e, 1.f + expf(-fabsf(ml)));
    }
    w = mine >= 0 ? w : 0.f;
    const float all = row_sum<L>(w);
    w = share_of(w, all);
  } else {
    w = softmax ? expf(ml - top) / sum : 1.f / (1.f + expf(-ml));
    w = mine >= 0 ? w : 0.f;
  }
  weight = poison ? NAN : w * S.s.scale;
  return row_any<L>(exact && !poison);
}

// A block takes the tokens of a tile, 32 / L rows a warp at a time. With a plan
// it also adds the tile's counts of each expert to its plan block's, or, if
// the tile is all there is, makes the plan itself.
enum class PlanPart { None, Counts, Whole };

template <typename T, int L, int EPL, bool Bias>
__global__ void __launch_bounds__(kRouteThreads, EPL > 8 ? 2 : 4)
    route_rows(RouteShape S, const T* __restrict__ logits, int64_t ld, bool whole, const float* __restrict__ bias,
               int tokens, int tile_tokens, int* __restrict__ indices, float* __restrict__ weights, PlanPart part,
               PlanView P) {
  extern __shared__ int shared[];  // chosen[tile_entries], then the plan's
  __shared__ int sh[kPlanWarps], doubtful;
  __shared__ uint16_t doubts[kRouteRows];
  __shared__ uint32_t lists[kRouteThreads / 32][list_depth(EPL) ? list_depth(EPL) * 32 : 1];
  __shared__ __align__(16) float table[Bias ? L * bias_row(EPL) : 1];
  constexpr int Rows = 32 / L;  // of a warp
  const int lane = threadIdx.x & (L - 1), w = threadIdx.x >> 5, sub = (threadIdx.x & 31) / L, k = S.s.k, E = S.s.experts;
  BiasScale B{};
  if constexpr (Bias) B = load_bias<L, EPL>(S, bias, table);
  if constexpr (list_depth(EPL) > 0) lists[w][(list_depth(EPL) - 1) * 32 + (threadIdx.x & 31)] = 0u;
  int* counts = shared + tile_tokens * k;
  if (threadIdx.x == 0) doubtful = 0;
  if (part == PlanPart::Counts)
    for (int e = threadIdx.x; e < P.stride; e += kRouteThreads) counts[e] = 0;
  __syncthreads();
  const int t0 = blockIdx.x * tile_tokens, n = min(tile_tokens, tokens - t0);
  // Every warp makes the same number of turns, so that the compiler knows the
  // lanes to be together at each vote and shuffle (a loop it takes for
  // divergent costs a synchronisation at each: 1.4x the instructions). Lanes
  // past the last row do it again and keep it to themselves.
  for (int i0 = 0; i0 < n; i0 += kRouteThreads / L) {
    const int i = i0 + w * Rows;
    const bool real = i + sub < n;
    const int64_t t = t0 + (real ? i + sub : n - 1);
    int mine;
    float weight;
    const bool doubt =
        route_row<T, L, EPL, Bias>(S, logits + t * ld, whole, bias, B, lists[w] + (threadIdx.x & 31), mine, weight);
    if (lane == 0 && real && doubt) doubts[atomicAdd(&doubtful, 1)] = static_cast<uint16_t>(i + sub);
    if (lane < k && real && !doubt) {
      indices[t * k + lane] = mine;
      weights[t * k + lane] = weight;
      if (part == PlanPart::Counts && mine >= 0) atomicAdd(&counts[mine], 1);
      if (part == PlanPart::Whole) shared[(i + sub) * k + lane] = mine;
    }
  }
  // The rows in doubt, shared out among the warps.
  __syncthreads();
  if (doubtful > 0) {
    RouteShape wide = S;
    wide.lanes_log += L == 8 ? 2 : L == 16 ? 1 : 0;
    for (int d = w; d < doubtful; d += kRouteThreads / 32) {
      const int i = doubts[d], ln = threadIdx.x & 31;
      const int64_t t = t0 + i;
      float weight;
      const int mine = route_exact<T, (EPL * L / 32 > 0 ? EPL * L / 32 : 1)>(wide, logits + t * ld, Bias ? bias : nullptr, weight);
      if (ln < k) {
        indices[t * k + ln] = mine;
        weights[t * k + ln] = weight;
        if (part == PlanPart::Counts && mine >= 0) atomicAdd(&counts[mine], 1);
        if (part == PlanPart::Whole) shared[i * k + ln] = mine;
      }
    }
  }
  if (part == PlanPart::None) return;
  __syncthreads();
  if (part == PlanPart::Counts) {
    int* to = P.counts + static_cast<int64_t>(blockIdx.x / P.block_tiles) * P.stride;
    for (int e = threadIdx.x; e < E; e += kRouteThreads)
      if (counts[e] > 0) atomicAdd(to + e, counts[e]);
  } else {
    plan_alone<2>([&](int i) { return shared[i]; }, n * k, E, P.err, counts, counts + kPlanWarps * E, sh, P.offsets, P.order,
                  P.position);
  }
}

// dlogits of a token. With share p_j of the j-th choice and g = sum_i p_i dw_i:
//   renormalised      scale * p_j * (dw_j - g), times 1 - s_j under the sigmoid
//   sigmoid           scale * s_j * (1 - s_j) * dw_j
//   softmax           scale * p_e * ([e chosen] dw_e - g) for every expert
//
// L lanes a row (8 where they hold the choices). The row is written in words of VB bytes as if nothing were
// chosen; lane j then writes the j-th choice's own value, with those of equal
// choices added.
template <typename T, int VB, int L>
__global__ void __launch_bounds__(kRouteThreads)
    route_grad_rows(spmvb_router_spec S, const T* __restrict__ logits, int64_t ld, int tokens,
                    const int* __restrict__ indices, const float* __restrict__ dweights, T* __restrict__ dlogits,
                    int64_t ldd, int* __restrict__ err) {
  constexpr int N = VB / sizeof(T);
  const int lane = threadIdx.x & (L - 1);
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kRouteThreads + threadIdx.x) / L;
  const bool real = t0 < tokens;  // lanes past the last token repeat it and write nothing
  const int64_t t = real ? t0 : tokens - 1;
  const int k = S.k, words = S.experts / N;
  const bool softmax = S.score == SPMVB_SOFTMAX;
  const T* row = logits + t * ld;
  T* to = dlogits + t * ldd;
  const int loaded = lane < k ? __ldg(indices + t * k + lane) : -1;
  // Zeros need not wait for the loads.
  if (!softmax && real)
    for (int v = lane; v < words; v += L) {
      Pack<T, VB> o;
#pragma unroll
      for (int i = 0; i < N; ++i) o.v[i] = narrow<T, float>(0.f);
      st_pack_stream<T, VB>(to + v * N, o);
    }
  int e = loaded;
  if (e >= S.experts) *err = 1;
  if (e < 0 || e >= S.experts) e = -1;
  const float dw = e >= 0 ? dweights[t * k + lane] * S.scale : 0.f;
  const float le = e >= 0 ? static_cast<float>(widen(row[e])) : -INFINITY;
  float d, top = -INFINITY, inv = 0.f, all = 0.f;
  bool poison = false;
  if (softmax) {
    float sum = 0.f;
    for (int v = lane; v < words; v += L) {
      const Pack<T, VB> p = ld_pack<T, VB>(row + v * N);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float l = widen(p.v[i]);
        poison |= !(l < INFINITY);
        top = fmaxf(top, l);
      }
    }
    poison = row_any<L>(poison);
    if (!S.renormalise) {
      top = unordered(row_max<L>(ordered(top)));
      for (int v = lane; v < words; v += L) {
        const Pack<T, VB> p = ld_pack<T, VB>(row + v * N);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float l = widen(p.v[i]);
          sum += l > -INFINITY ? expf(l - top) : 0.f;
        }
      }
      sum = row_sum<L>(sum);
      inv = sum > 0.f ? 1.f / sum : 0.f;
    }
  }
  if (S.renormalise) {
    float m = unordered(row_max<L>(ordered(le)));
    if (!softmax) m = fminf(m, 0.f);
    const float a = softmax || le <= 0.f ? expf(le - m) : 1.f, b = expf(-fabsf(le));
    const float s = e < 0 ? 0.f : softmax ? a : __fdividef(a, 1.f + b);
    const float sum = row_sum<L>(s), share = share_of(s, sum);
    // 1 - sigmoid(l) = exp(-l) / (1 + exp(-l)) or 1 / (1 + exp(l)).
    const float rest = softmax ? 1.f : __fdividef(le > 0.f ? b : 1.f, 1.f + b);
    d = share * (dw - row_sum<L>(share * dw)) * rest;
  } else if (softmax) {
    const float share = e >= 0 ? expf(le - top) * inv : 0.f;
    all = row_sum<L>(share * dw);
    d = share * (dw - all);
  } else {
    const float b = expf(-fabsf(le));
    d = e >= 0 ? dw * __fdividef(b, (1.f + b) * (1.f + b)) : 0.f;  // s (1 - s), the same for -l
  }
  // Equal choices: the first of them writes the sum of all. Under the plain
  // softmax each holds the row's own term, which counts once.
  float own = 0.f;
  if (softmax && !S.renormalise && e >= 0) own = -expf(le - top) * inv * all;
  float total = 0.f;
  bool first = true;
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const int ej = __shfl_sync(kAll, e, j, L);
    const float dj = __shfl_sync(kAll, d - own, j, L);
    total += ej == e ? dj : 0.f;
    first &= !(ej == e && j < lane);
  }
  for (int v = lane; softmax && v < words; v += L) {
    Pack<T, VB> o;
    if (!S.renormalise) {
      const Pack<T, VB> p = ld_pack<T, VB>(row + v * N);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float l = widen(p.v[i]);
        o.v[i] = narrow<T, float>(poison ? NAN : l > -INFINITY ? -expf(l - top) * inv * all : 0.f);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) o.v[i] = narrow<T, float>(poison ? NAN : 0.f);
    }
    if (real) st_pack_stream<T, VB>(to + v * N, o);
  }
  __syncwarp();
  if (real && e >= 0 && first && !poison) to[e] = narrow<T, float>(own + total);
}

// Lanes of a group: the row's lanes shared out among the groups, a power of
// two each.
int lanes_per_group(const spmvb_router_spec& s, int lanes) {
  int n = lanes;
  while (n * s.groups > lanes) n /= 2;
  return n;
}
// Experts of a lane, rounded up to a power of two: at most 64, as of 1,020
// experts in 17 groups.
int slots_per_lane(const spmvb_router_spec& s, int lanes) {
  int slots = 1;
  while (slots * lanes_per_group(s, lanes) < s.experts / s.groups) slots *= 2;
  return slots;
}

// Lanes of a row: as few as leave a lane eight experts, where the lanes can
// hold the choices and the groups and there are rows to fill the GPU.
int row_lanes(const spmvb_router_spec& s, int tokens, int sm_count) {
  if (tokens <= sm_count * 8) return 32;
  int lanes = 8;
  while (lanes < 32 && (lanes * 8 < s.experts || lanes < s.k || lanes < s.groups)) lanes *= 2;
  return (s.groups & (s.groups - 1)) == 0 ? lanes : 32;
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
  spmvb::ContextRef ctx;
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
    R->ctx.hold(ctx);
    R->device = ctx->device;
    R->spec = *spec;
    R->max_tokens = max_tokens;
    SPMVB_TRY(R->plan.alloc(max_tokens, spec->k, spec->experts));
    SPMVB_TRY(scratch_ready());
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
                        : tokens > 0 && tokens <= tile ? PlanPart::Whole
                        : plan_is_one_block(P) ? PlanPart::None : PlanPart::Counts;
  if (tokens > 0) {
    const int L = row_lanes(S, tokens, R->ctx->sm_count);
    SPMVB_TRY(with_logits(dtype, slots_per_lane(S, L), [&](auto tv, auto epl) -> spmvb_status {
      using T = decltype(tv);
      constexpr int EPL = decltype(epl)::value;
      const RouteShape shape{S, S.experts / S.groups, __builtin_ctz(lanes_per_group(S, L))};
      const int vb = std::min<int>(16, EPL * sizeof(T));
      const bool whole = S.experts == L * EPL && access_bytes(sizeof(T), {{d_logits, ld_logits}}, vb / sizeof(T)) == vb;
      // Without a plan a block takes one row a lane group where that many blocks have room.
      const int at_once = kRouteThreads / L;
      const int rows = part != PlanPart::None ? tile
                                              : std::min(kRouteRows, static_cast<int>(ceil_div(ceil_div(tokens, int64_t(R->ctx->sm_count) * 4), at_once)) * at_once);
      const size_t shared = part == PlanPart::None     ? 0
                            : part == PlanPart::Counts ? (static_cast<size_t>(rows) * S.k + P.stride) * 4
                                                       : (static_cast<size_t>(rows) * S.k + (kPlanWarps + 1) * S.experts) * 4;
      auto kernel = d_bias ? route_rows<T, 32, EPL, true> : route_rows<T, 32, EPL, false>;
      if constexpr (EPL <= 8) {
        if (L == 16) kernel = d_bias ? route_rows<T, 16, EPL, true> : route_rows<T, 16, EPL, false>;
        if (L == 8) kernel = d_bias ? route_rows<T, 8, EPL, true> : route_rows<T, 8, EPL, false>;
      }
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
  const int vb = access_bytes(es, {{d_logits, ld_logits}, {d_dlogits, ld_dlogits}}, S.experts);
  const auto run = [&](auto tv) -> spmvb_status {
    using T = decltype(tv);
    const bool few = S.k <= 8;
    const auto kernel = vb == 16  ? (few ? route_grad_rows<T, 16, 8> : route_grad_rows<T, 16, 32>)
                        : vb == 8 ? (few ? route_grad_rows<T, 8, 8> : route_grad_rows<T, 8, 32>)
                                  : (few ? route_grad_rows<T, sizeof(T), 8> : route_grad_rows<T, sizeof(T), 32>);
    kernel<<<static_cast<int>(ceil_div(tokens, kRouteThreads / (few ? 8 : 32))), kRouteThreads, 0, s>>>(
        S, static_cast<const T*>(d_logits), ld_logits, tokens, d_indices, d_dweights, static_cast<T*>(d_dlogits),
        ld_dlogits, R->ctx->index_err());
    count_launch();
    SPMVB_TRY_CUDA(cudaGetLastError());
    return SPMVB_OK;
  };
  return dtype == SPMVB_F32 ? run(float{}) : dtype == SPMVB_F16 ? run(__half{}) : run(__nv_bfloat16{});
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
  return launch_gather_sum(dtype, d_position, nullptr, tokens, R->spec.k, dout, dX, R->ctx->index_err(),
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
  return launch_gather_sum(dtype, d_position, d_weights, tokens, R->spec.k, Y, out, R->ctx->index_err(),
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
