// The global 2-norm of many tensors, and their scaling by
// min(1, max_norm / (norm + eps)) in place.
//
// The tensors are cut into pieces of 4 to 16 KB. sum_squares sums each block's
// pieces in fp64; the last block to finish adds the blocks' sums in their order
// and forms the factor. scale_pieces multiplies, from the last piece to the
// first, so that it finds in the L2 what was read last, and leaves the tensors
// alone where the factor is 1. Squares of doubles past 2^480 or below 2^-480 are
// summed apart, scaled by a power of two: the norm of finite values is finite
// where fp64 holds it. HBM bounds both: the data is read twice and
// written once (no cache holds it in between). fp64 costs the bf16 sum nothing
// yet: its conversions take 0.7 of the reading time.
#include <cmath>
#include <iterator>
#include <vector>

#include "select.cuh"

namespace spmvb {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipBlocks = 148 * 6;
constexpr int64_t kMinPiece = 4096, kMaxPiece = 16384;  // bytes

struct Piece {
  void* p;
  int count;
  int dtype;
};

// Calls whole(place, word) for the 16-byte words of a piece, four loads ahead,
// and one(element) for the elements before and after them.
template <typename T, typename Whole, typename One>
__device__ __forceinline__ void each_word(const Piece& c, Whole&& whole, One&& one) {
  constexpr int N = 16 / sizeof(T);
  T* p = static_cast<T*>(c.p);
  const int head = min(c.count, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int words = (c.count - head) / N;
  uint4* w = reinterpret_cast<uint4*>(p + head) + threadIdx.x;
  int left = words - static_cast<int>(threadIdx.x);
  for (; left > 3 * kClipThreads; left -= 4 * kClipThreads, w += 4 * kClipThreads) {
    const uint4 a = w[0], b = w[kClipThreads], d = w[2 * kClipThreads], e = w[3 * kClipThreads];
    whole(w, a);
    whole(w + kClipThreads, b);
    whole(w + 2 * kClipThreads, d);
    whole(w + 3 * kClipThreads, e);
  }
  for (; left > 0; left -= kClipThreads, w += kClipThreads) whole(w, *w);
  const int tail = head + words * N;
  if (static_cast<int>(threadIdx.x) < head) one(p + threadIdx.x);
  if (tail + static_cast<int>(threadIdx.x) < c.count) one(p + tail + threadIdx.x);
}

template <typename T>
__device__ __forceinline__ Pack<T, 16> as_pack(const uint4& v) {
  Pack<T, 16> p;
  *reinterpret_cast<uint4*>(&p) = v;
  return p;
}

// Sums of squares: of doubles past 2^480 in units of 2^1200, of those below
// 2^-480 in units of 2^-1200, and of all other values. 2^40 squares of none of
// the three leave fp64, and neither do those of any fp32 value.
struct Squares {
  double mid = 0, big = 0, small = 0;
};
constexpr double kBig = 0x1p480, kSmall = 0x1p-480, kUp = 0x1p600, kDown = 0x1p-600;

// Adds x * x: to s where it is neither big nor small, which its exponent alone
// tells (zeros are small; NaN goes to s).
__device__ __forceinline__ void add_square(double x, double& s, Squares& far) {
  constexpr unsigned Least = (1023u - 480u) << 20, Most = (1023u + 480u) << 20;
  if ((static_cast<unsigned>(__double2hiint(x)) & 0x7fffffffu) - Least < Most - Least) {
    s = fma(x, x, s);
  } else if (fabs(x) >= kBig) {
    far.big = fma(x * kDown, x * kDown, far.big);
  } else if (fabs(x) < kSmall) {
    far.small = fma(x * kUp, x * kUp, far.small);
  } else {
    s += x;
  }
}
__device__ __forceinline__ void add_square(float x, double& s, Squares&) {
  const double a = static_cast<double>(x);
  s = fma(a, a, s);
}

template <typename T>
__device__ __forceinline__ void piece_squares(const Piece& c, Squares& sum) {
  double s0 = 0, s1 = 0;
  each_word<T>(
      c,
      [&](const uint4*, const uint4& v) {
        const Pack<T, 16> x = as_pack<T>(v);
#pragma unroll
        for (int i = 0; i < Pack<T, 16>::N; i += 2) {
          add_square(widen(x.v[i]), s0, sum);
          add_square(widen(x.v[i + 1]), s1, sum);
        }
      },
      [&](const T* p) { add_square(widen(*p), s0, sum); });
  sum.mid += s0 + s1;
}

// Sum over the block, valid in thread 0.
__device__ __forceinline__ double clip_block_sum(double v) {
  __shared__ double sh[kClipThreads / 32];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  if (threadIdx.x == 0)
    for (int i = 0; i < kClipThreads / 32; ++i) v += sh[i];
  return v;
}

__device__ __forceinline__ void clip_block_sums(Squares& s, bool doubles) {
  s.mid = clip_block_sum(s.mid);
  if (doubles && __syncthreads_or(s.big != 0 || s.small != 0)) {
    s.big = clip_block_sum(s.big);
    s.small = clip_block_sum(s.small);
  }
}

// Calls f(T{}) for the type of a piece; Only: that of all tensors, or -1.
template <int Only, typename F>
__device__ __forceinline__ void with_piece(const Piece& c, F&& f) {
  const int d = Only >= 0 ? Only : c.dtype;
  if (d == SPMVB_F32) f(float{});
  else if (d == SPMVB_F64) f(double{});
  else if (d == SPMVB_F16) f(__half{});
  else f(__nv_bfloat16{});
}

// sums: mid of every block, then, where there are doubles, big and small.
// factor: what values are multiplied by and, where there are doubles, a power of
// two to multiply them by before. `ticket` is 0 between calls.
template <int Only>
__global__ void __launch_bounds__(kClipThreads, kClipBlocks / 148)
    sum_squares(const Piece* __restrict__ pieces, int count, double* __restrict__ sums, unsigned* __restrict__ ticket,
                double max_norm, double eps, float* __restrict__ norm, double* __restrict__ factor) {
  constexpr bool Doubles = Only < 0 || Only == SPMVB_F64;
  __shared__ bool last;
  Squares s;
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    const Piece q = pieces[c];
    with_piece<Only>(q, [&](auto tv) { piece_squares<decltype(tv)>(q, s); });
  }
  clip_block_sums(s, Doubles);
  if (threadIdx.x == 0) {
    __stcg(sums + blockIdx.x, s.mid);
    if constexpr (Doubles) {
      __stcg(sums + gridDim.x + blockIdx.x, s.big);
      __stcg(sums + 2 * gridDim.x + blockIdx.x, s.small);
    }
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  s = Squares{};
  for (int i = threadIdx.x; i < gridDim.x; i += kClipThreads) {
    s.mid += ld_written(sums + i);
    if constexpr (Doubles) {
      s.big += ld_written(sums + gridDim.x + i);
      s.small += ld_written(sums + 2 * gridDim.x + i);
    }
  }
  clip_block_sums(s, Doubles);
  if (threadIdx.x == 0) {
    *ticket = 0u;
    double n;
    if constexpr (Doubles) {
      const bool up = s.big > 0, down = !up && s.mid == 0;
      n = sqrt(up ? s.big + s.mid * kDown * kDown : down ? s.small : s.mid + s.small * kDown * kDown);
      n *= up ? kUp : down ? kDown : 1.0;  // what a sum leaves out is below 2^-200 of it
    } else {
      n = sqrt(s.mid);
    }
    const double f = max_norm / (n + eps);
    *norm = static_cast<float>(n);
    factor[0] = n + eps > 0 ? (f > 1.0 ? 1.0 : f) : n == n ? 1.0 : n;  // NaN carries on
    if constexpr (Doubles) {
      // A factor near fp64's least is divided in two: the values that it leaves
      // more than 0 are far above those that the first of them would round.
      const bool split = f < 0x1p-900 && max_norm > 0;
      if (split) factor[0] = max_norm / ((n + eps) * kDown);
      factor[1] = split ? kDown : 1.0;
    }
  }
}

// Values times f, in fp32, or in fp64 where fp32 does not hold f (Far).
template <typename T, bool Far>
__device__ __forceinline__ void piece_scale(const Piece& c, double f, double first) {
  using Acc = typename AccOf<T>::type;
  const Acc g = static_cast<Acc>(f);
  const auto one = [&](T v) {
    if constexpr (sizeof(T) == 8) return narrow<T, Acc>(v * first * f);
    else if constexpr (Far) return narrow<T, Acc>(static_cast<Acc>(static_cast<double>(widen(v)) * f));
    else return narrow<T, Acc>(widen(v) * g);
  };
  each_word<T>(
      c,
      [&](uint4* to, const uint4& v) {
        Pack<T, 16> x = as_pack<T>(v);
#pragma unroll
        for (int i = 0; i < Pack<T, 16>::N; ++i) x.v[i] = one(x.v[i]);
        __stcs(to, *reinterpret_cast<const uint4*>(&x));
      },
      [&](T* p) { *p = one(*p); });
}

// Values as large as fp32 holds and a norm beyond make factors that are
// subnormal in fp32, or 0, and results that are neither.
constexpr double kFarFactor = 0x1p-100;

// Out of line, as only a step that diverged needs it.
template <int Only>
__device__ __noinline__ void scale_far(const Piece* __restrict__ pieces, int count, double f, double first) {
  for (int c = count - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const Piece q = pieces[c];
    with_piece<Only>(q, [&](auto tv) {
      using T = decltype(tv);
      piece_scale<T, true>(q, sizeof(T) == 8 ? f : f * first, first);
    });
  }
}

template <int Only>
__global__ void __launch_bounds__(kClipThreads, kClipBlocks / 148)
    scale_pieces(const Piece* __restrict__ pieces, int count, const double* __restrict__ factor) {
  const double f = factor[0], first = Only < 0 || Only == SPMVB_F64 ? factor[1] : 1.0, all = f * first;
  if (all == 1.0) return;
  if (all > 0 && all < kFarFactor) {
    scale_far<Only>(pieces, count, f, first);
    return;
  }
  for (int c = count - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const Piece q = pieces[c];
    with_piece<Only>(q, [&](auto tv) {
      using T = decltype(tv);
      piece_scale<T, false>(q, sizeof(T) == 8 ? f : all, first);
    });
  }
}

}  // namespace
}  // namespace spmvb

struct spmvb_clip_st {
  int device = 0, pieces = 0, blocks = 0;
  int only = -1;  // the dtype of all tensors, -1 where they differ
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;  // of the tensors' bytes, ascending
  spmvb::DevBuf table, sums, factor, ticket;
};

using namespace spmvb;

namespace {

// The norm's place must be a float on the device and outside the tensors.
spmvb_status check_norm(spmvb_clip C, const float* d_norm) {
  SPMVB_TRY(check_rows({d_norm, 1, 1, 1, 4, "norm"}, C->device));
  const auto a = reinterpret_cast<uintptr_t>(d_norm);
  const auto it = std::upper_bound(C->spans.begin(), C->spans.end(), a + 3,
                                   [](uintptr_t v, const auto& span) { return v < span.first; });
  if (it != C->spans.begin() && std::prev(it)->second > a)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "norm lies inside a tensor");
  return SPMVB_OK;
}

spmvb_status run_norm(spmvb_clip C, double max_norm, double eps, float* d_norm, cudaStream_t s) {
  const auto kernel = C->only == SPMVB_F32    ? sum_squares<SPMVB_F32>
                      : C->only == SPMVB_F64  ? sum_squares<SPMVB_F64>
                      : C->only == SPMVB_F16  ? sum_squares<SPMVB_F16>
                      : C->only == SPMVB_BF16 ? sum_squares<SPMVB_BF16>
                                              : sum_squares<-1>;
  kernel<<<C->blocks, kClipThreads, 0, s>>>(C->table.as<Piece>(), C->pieces, C->sums.as<double>(),
                                            C->ticket.as<unsigned>(), max_norm, eps, d_norm, C->factor.as<double>());
  count_launch();
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // namespace

extern "C" {

spmvb_status spmvb_clip_create(spmvb_context ctx, int32_t count, void* const* h_tensors, const int64_t* h_sizes,
                               const spmvb_dtype* h_dtypes, spmvb_clip* out) {
  clear_error();
  if (!ctx || !out) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null context or output");
  if (count < 0 || (count > 0 && (!h_tensors || !h_sizes || !h_dtypes)))
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "negative count or null tensors, sizes or dtypes");
  return constructed([&]() -> spmvb_status {
    std::vector<Piece> pieces;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    DeviceGuard g(ctx->device);
    int64_t total = 0;
    for (int32_t i = 0; i < count; ++i) {
      if (!any_float(h_dtypes[i])) return fail(SPMVB_ERR_INVALID_ARGUMENT, "tensor " + std::to_string(i) + ": bad dtype");
      if (h_sizes[i] < 0) return fail(SPMVB_ERR_INVALID_ARGUMENT, "tensor " + std::to_string(i) + ": negative size");
      const int64_t es = static_cast<int64_t>(dtype_size(h_dtypes[i]));
      // No device holds that much, and past 63 bits the length would wrap.
      if (h_sizes[i] > (INT64_MAX - total) / es)
        return fail(SPMVB_ERR_INVALID_ARGUMENT, "tensor " + std::to_string(i) + ": the tensors' bytes pass 63 bits");
      total += h_sizes[i] * es;
    }
    // Small pieces where large ones would leave SMs without any.
    int64_t piece = kMinPiece;
    while (piece < kMaxPiece && piece * 2 * kClipBlocks <= total) piece *= 2;
    for (int32_t i = 0; i < count; ++i) {
      const std::string name = "tensor " + std::to_string(i);
      if (h_sizes[i] == 0) continue;
      const size_t es = dtype_size(h_dtypes[i]);
      SPMVB_TRY(check_rows({h_tensors[i], 1, h_sizes[i], h_sizes[i], es, name.c_str()}, ctx->device));
      const auto a = reinterpret_cast<uintptr_t>(h_tensors[i]);
      spans.emplace_back(a, a + h_sizes[i] * es);
      // Pieces end on 16-byte boundaries, so that only the first can begin off one.
      for (int64_t at = 0; at < h_sizes[i];) {
        const int64_t off = static_cast<int64_t>((a + at * es) & 15) / static_cast<int64_t>(es);
        const int64_t n = std::min<int64_t>(piece / static_cast<int64_t>(es) - off, h_sizes[i] - at);
        pieces.push_back({static_cast<char*>(h_tensors[i]) + at * es, static_cast<int>(n), static_cast<int>(h_dtypes[i])});
        at += n;
      }
      if (pieces.size() > (size_t(1) << 28)) return fail(SPMVB_ERR_UNSUPPORTED, "too many elements");
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      if (spans[i].first < spans[i - 1].second) return fail(SPMVB_ERR_INVALID_ARGUMENT, "two tensors overlap");
    auto C = std::make_unique<spmvb_clip_st>();
    C->device = ctx->device;
    C->pieces = static_cast<int>(pieces.size());
    C->only = count > 0 ? static_cast<int>(h_dtypes[0]) : -1;
    for (int32_t i = 1; i < count; ++i)
      if (h_dtypes[i] != h_dtypes[0]) C->only = -1;
    C->blocks = std::max(1, std::min(C->pieces, kClipBlocks));
    SPMVB_TRY(upload(C->table, pieces.data(), pieces.size() * sizeof(Piece), 16));
    SPMVB_TRY(C->sums.alloc(static_cast<size_t>(C->blocks) * 3 * 8));
    SPMVB_TRY(C->factor.alloc(16));
    SPMVB_TRY(C->ticket.alloc(4));
    SPMVB_TRY(scratch_ready());
    C->spans = std::move(spans);
    *out = C.release();
    return SPMVB_OK;
  });
}

spmvb_status spmvb_clip_destroy(spmvb_clip C) {
  clear_error();
  if (C) {
    DeviceGuard g(C->device);
    delete C;
  }
  return SPMVB_OK;
}

spmvb_status spmvb_clip_norm(spmvb_clip C, float* d_norm, void* stream) {
  clear_error();
  if (!C) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null clip");
  DeviceGuard g(C->device);
  SPMVB_TRY(check_norm(C, d_norm));
  return run_norm(C, 0.0, 0.0, d_norm, static_cast<cudaStream_t>(stream));
}

spmvb_status spmvb_clip_run(spmvb_clip C, double max_norm, double eps, float* d_norm, void* stream) {
  clear_error();
  if (!C) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null clip");
  if (!(max_norm >= 0) || !(eps >= 0) || std::isinf(eps))
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "max_norm and eps must not be negative or NaN, eps must be finite");
  DeviceGuard g(C->device);
  SPMVB_TRY(check_norm(C, d_norm));
  const auto s = static_cast<cudaStream_t>(stream);
  SPMVB_TRY(run_norm(C, max_norm, eps, d_norm, s));
  if (C->pieces == 0) return SPMVB_OK;
  const auto kernel = C->only == SPMVB_F32    ? scale_pieces<SPMVB_F32>
                      : C->only == SPMVB_F64  ? scale_pieces<SPMVB_F64>
                      : C->only == SPMVB_F16  ? scale_pieces<SPMVB_F16>
                      : C->only == SPMVB_BF16 ? scale_pieces<SPMVB_BF16>
                                              : scale_pieces<-1>;
  kernel<<<C->blocks, kClipThreads, 0, s>>>(C->table.as<Piece>(), C->pieces, C->factor.as<double>());
  count_launch();
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // extern "C"
