// Routing of tokens to experts: the choice, its weights and their gradient.
//
// One warp per token; lane i holds the experts i * EPL .. i * EPL + EPL - 1,
// so the lowest lane with the largest value has the lowest index. The scores
// are computed in fp64: two experts can lie closer together than fp32
// resolves, and the choice between them must not depend on the rounding of
// exp.
#include <cmath>

#include "select.cuh"

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

template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteThreads)
    route_rows(spmvb_router_spec S, const T* __restrict__ logits, int64_t ld, const float* __restrict__ bias, int tokens,
               int* __restrict__ indices, float* __restrict__ weights) {
  const int t = blockIdx.x * (kRouteThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= tokens) return;
  const int E = S.experts, k = S.k;
  double l[EPL], c[EPL], score[EPL];
  bool poison = false;
  double top = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    l[i] = e < E ? static_cast<double>(widen(logits[t * ld + e])) : -INFINITY;
    poison |= isnan(l[i]) || l[i] == INFINITY;
    if (l[i] > top) top = l[i];
  }
  if (S.score == SPMVB_SOFTMAX) {
    poison = __any_sync(kAll, poison);
    top = warp_max(top);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      score[i] = !poison && l[i] > -INFINITY ? exp(l[i] - top) : 0.0;
      sum += score[i];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < EPL; ++i) score[i] = sum > 0 ? score[i] / sum : 0.0;
  } else {
    poison = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) score[i] = 1.0 / (1.0 + exp(-l[i]));
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane * EPL + i;
    c[i] = bias && e < E ? score[i] + static_cast<double>(bias[e]) : l[i];
    if (poison || !(l[i] > -INFINITY) || !(c[i] > -INFINITY)) c[i] = -INFINITY;
  }
  if (S.groups > 1) {
    const int per = E / S.groups;
    double level = -INFINITY;  // of group `lane`
    for (int g = 0; g < S.groups; ++g) {
      double a = -INFINITY, b = -INFINITY;  // the two best
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = lane * EPL + i;
        if (e >= E || e / per != g || !(c[i] > -INFINITY)) continue;
        const double v = bias || S.group_top == 1 ? c[i] : score[i];
        if (v > a) { b = a; a = v; } else if (v > b) { b = v; }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        const double a2 = __shfl_xor_sync(kAll, a, off), b2 = __shfl_xor_sync(kAll, b, off);
        b = fmax(fmin(a, a2), fmax(b, b2));
        a = fmax(a, a2);
      }
      if (lane == g) level = S.group_top == 2 && b > -INFINITY ? a + b : a;
    }
    int better = 0;
    for (int g = 0; g < S.groups; ++g) {
      const double v = __shfl_sync(kAll, level, g);
      better += v > level || (v == level && g < lane);
    }
    const unsigned open = __ballot_sync(kAll, lane < S.groups && better < S.groups_kept);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane * EPL + i;
      if (e < E && !(open >> (e / per) & 1u)) c[i] = -INFINITY;
    }
  }
  int mine = -1;  // lane j: the j-th choice, its logit and score
  double ml = -INFINITY, ms = 0;
  for (int j = 0; j < k; ++j) {
    double v = c[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < EPL; ++i)
      if (c[i] > v) { v = c[i]; at = i; }
    int e = lane * EPL + at;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const double v2 = __shfl_xor_sync(kAll, v, off);
      const int e2 = __shfl_xor_sync(kAll, e, off);
      if (v2 > v || (v2 == v && e2 < e)) { v = v2; e = e2; }
    }
    if (!(v > -INFINITY)) break;
    double le = 0, se = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane * EPL + i == e) { le = l[i]; se = score[i]; c[i] = -INFINITY; }
    le = __shfl_sync(kAll, le, e / EPL);
    se = __shfl_sync(kAll, se, e / EPL);
    if (lane == j) { mine = e; ml = le; ms = se; }
  }
  if (S.renormalise) {
    // Shares of the chosen scores, from a common factor taken out of them:
    // exp(l - m) under the softmax; under the sigmoid, where m <= 0,
    // exp(l - m) / (1 + exp(l)) = sigmoid(l) * exp(-m).
    double m = warp_max(ml);
    if (S.score == SPMVB_SIGMOID) m = fmin(m, 0.0);
    double s = 0;
    if (mine >= 0) s = S.score == SPMVB_SOFTMAX ? exp(ml - m) : ml > 0 ? 1.0 / (1.0 + exp(-ml)) : exp(ml - m) / (1.0 + exp(ml));
    const double sum = warp_sum(s);
    ms = sum > 0 ? s / sum : 0.0;
  }
  if (lane < k) {
    indices[static_cast<int64_t>(t) * k + lane] = mine;
    weights[static_cast<int64_t>(t) * k + lane] = poison ? NAN : static_cast<float>(mine >= 0 ? ms * S.scale : 0.0);
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

template <typename F>
spmvb_status with_logits(spmvb_dtype d, int experts, F&& f) {
  const auto by_lane = [&](auto tv) -> spmvb_status {
    using std::integral_constant;
    if (experts <= 32) return f(tv, integral_constant<int, 1>{});
    if (experts <= 64) return f(tv, integral_constant<int, 2>{});
    if (experts <= 128) return f(tv, integral_constant<int, 4>{});
    if (experts <= 256) return f(tv, integral_constant<int, 8>{});
    if (experts <= 512) return f(tv, integral_constant<int, 16>{});
    return f(tv, integral_constant<int, 32>{});
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
  spmvb::SortSpace sort;
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
    SPMVB_TRY(R->sort.alloc(static_cast<int64_t>(max_tokens) * spec->k));
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
  if (tokens < 0 || tokens > R->max_tokens)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "tokens must be in [0, max_tokens = " + std::to_string(R->max_tokens) + "]");
  const int dev = R->device;
  const int64_t n = static_cast<int64_t>(tokens) * R->spec.k;
  const RowSet idx = entries_of(d_indices, n, "indices"), offsets = entries_of(d_offsets, R->spec.experts + 1, "offsets"),
               order = entries_of(d_order, n, "order"), position = entries_of(d_position, n, "position");
  DeviceGuard g(dev);
  for (const RowSet* r : {&idx, &offsets, &order, &position}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* r : {&offsets, &order, &position}) SPMVB_TRY(check_apart(*r, idx));
  for (const RowSet* r : {&order, &position}) SPMVB_TRY(check_apart(offsets, *r));
  SPMVB_TRY(check_apart(order, position));
  return launch_plan(R->sort, d_indices, n, R->spec.experts, d_offsets, d_order, d_position, R->ctx->index_err(),
                     static_cast<cudaStream_t>(stream));
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
  if (tokens < 0 || (plan && tokens > R->max_tokens))
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "tokens must be in [0, max_tokens = " + std::to_string(R->max_tokens) + "]");
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
  if (tokens > 0) {
    SPMVB_TRY(with_logits(dtype, S.experts, [&](auto tv, auto epl) -> spmvb_status {
      using T = decltype(tv);
      route_rows<T, decltype(epl)::value><<<static_cast<int>(ceil_div(tokens, kRouteThreads / 32)), kRouteThreads, 0, s>>>(
          S, static_cast<const T*>(d_logits), ld_logits, d_bias, tokens, d_indices, d_weights);
      count_launch();
      SPMVB_TRY_CUDA(cudaGetLastError());
      return SPMVB_OK;
    }));
  }
  return plan ? spmvb_router_plan(R, tokens, d_indices, d_offsets, d_order, d_position, stream) : SPMVB_OK;
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
  return with_logits(dtype, S.experts, [&](auto tv, auto epl) -> spmvb_status {
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
