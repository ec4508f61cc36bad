// The global 2-norm of many tensors, and their scaling by
// min(1, max_norm / (norm + eps)) in place.
//
// The tensors are cut into pieces of at most kPiece elements. sum_squares
// sums each block's pieces in fp64, norm_factor adds the blocks' sums in a
// fixed order and forms the factor, scale_pieces multiplies, and leaves the
// tensors alone where the factor is 1. The data is read twice and written once, so HBM
// bounds it.
#include <cmath>
#include <iterator>
#include <vector>

#include "select.cuh"

namespace spmvb {
namespace {

constexpr int kClipThreads = 256;
constexpr int kPiece = 16384;
constexpr int kMaxBlocks = 1184;  // 148 SMs x 8

struct Piece {
  void* p;
  int count;
  int dtype;
};

template <typename T>
__device__ __forceinline__ double piece_squares(const Piece& c) {
  const T* p = static_cast<const T*>(c.p);
  double s = 0;
  for (int i = threadIdx.x; i < c.count; i += kClipThreads) {
    const double v = static_cast<double>(widen(p[i]));
    s = fma(v, v, s);
  }
  return s;
}

// Sum over the block, valid in thread 0.
__device__ __forceinline__ double clip_block_sum(double v) {
  __shared__ double sh[kClipThreads / 32];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  if (threadIdx.x == 0)
    for (int i = 0; i < kClipThreads / 32; ++i) v += sh[i];
  return v;
}

__global__ void __launch_bounds__(kClipThreads)
    sum_squares(const Piece* __restrict__ pieces, int count, double* __restrict__ sums) {
  double s = 0;
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    const Piece q = pieces[c];
    switch (q.dtype) {
      case SPMVB_F32: s += piece_squares<float>(q); break;
      case SPMVB_F64: s += piece_squares<double>(q); break;
      case SPMVB_F16: s += piece_squares<__half>(q); break;
      default: s += piece_squares<__nv_bfloat16>(q); break;
    }
  }
  s = clip_block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ void __launch_bounds__(kClipThreads)
    norm_factor(const double* __restrict__ sums, int blocks, double max_norm, double eps, float* __restrict__ norm,
                double* __restrict__ factor) {
  double s = 0;
  for (int i = threadIdx.x; i < blocks; i += kClipThreads) s += sums[i];
  s = clip_block_sum(s);
  if (threadIdx.x == 0) {
    const double n = sqrt(s), f = max_norm / (n + eps);
    *norm = static_cast<float>(n);
    *factor = n + eps > 0 ? (f > 1.0 ? 1.0 : f) : n == n ? 1.0 : n;  // NaN carries on
  }
}

template <typename T>
__device__ __forceinline__ void piece_scale(const Piece& c, double factor) {
  using Acc = typename AccOf<T>::type;
  T* p = static_cast<T*>(c.p);
  const Acc f = static_cast<Acc>(factor);
  for (int i = threadIdx.x; i < c.count; i += kClipThreads) p[i] = narrow<T, Acc>(widen(p[i]) * f);
}

__global__ void __launch_bounds__(kClipThreads)
    scale_pieces(const Piece* __restrict__ pieces, int count, const double* __restrict__ factor) {
  const double f = *factor;
  if (f == 1.0) return;
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    const Piece q = pieces[c];
    switch (q.dtype) {
      case SPMVB_F32: piece_scale<float>(q, f); break;
      case SPMVB_F64: piece_scale<double>(q, f); break;
      case SPMVB_F16: piece_scale<__half>(q, f); break;
      default: piece_scale<__nv_bfloat16>(q, f); break;
    }
  }
}

}  // namespace
}  // namespace spmvb

struct spmvb_clip_st {
  int device = 0, pieces = 0, blocks = 0;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;  // of the tensors' bytes, ascending
  spmvb::DevBuf table, sums, factor;
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
  sum_squares<<<C->blocks, kClipThreads, 0, s>>>(C->table.as<Piece>(), C->pieces, C->sums.as<double>());
  norm_factor<<<1, kClipThreads, 0, s>>>(C->sums.as<double>(), C->blocks, max_norm, eps, d_norm, C->factor.as<double>());
  count_launch(2);
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
    for (int32_t i = 0; i < count; ++i) {
      const std::string name = "tensor " + std::to_string(i);
      if (!any_float(h_dtypes[i])) return fail(SPMVB_ERR_INVALID_ARGUMENT, name + ": bad dtype");
      if (h_sizes[i] < 0) return fail(SPMVB_ERR_INVALID_ARGUMENT, name + ": negative size");
      if (h_sizes[i] == 0) continue;
      const size_t es = dtype_size(h_dtypes[i]);
      SPMVB_TRY(check_rows({h_tensors[i], 1, h_sizes[i], h_sizes[i], es, name.c_str()}, ctx->device));
      const auto a = reinterpret_cast<uintptr_t>(h_tensors[i]);
      spans.emplace_back(a, a + h_sizes[i] * es);
      for (int64_t at = 0; at < h_sizes[i]; at += kPiece)
        pieces.push_back({static_cast<char*>(h_tensors[i]) + at * es,
                          static_cast<int>(std::min<int64_t>(kPiece, h_sizes[i] - at)), static_cast<int>(h_dtypes[i])});
      if (pieces.size() > (size_t(1) << 28)) return fail(SPMVB_ERR_UNSUPPORTED, "too many elements");
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
      if (spans[i].first < spans[i - 1].second) return fail(SPMVB_ERR_INVALID_ARGUMENT, "two tensors overlap");
    auto C = std::make_unique<spmvb_clip_st>();
    C->device = ctx->device;
    C->pieces = static_cast<int>(pieces.size());
    C->blocks = std::max(1, std::min(C->pieces, kMaxBlocks));
    SPMVB_TRY(upload(C->table, pieces.data(), pieces.size() * sizeof(Piece), 16));
    SPMVB_TRY(C->sums.alloc(static_cast<size_t>(C->blocks) * 8));
    SPMVB_TRY(C->factor.alloc(8));
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
  scale_pieces<<<C->blocks, kClipThreads, 0, s>>>(C->table.as<Piece>(), C->pieces, C->factor.as<double>());
  count_launch();
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // extern "C"
