// Shared by the row-selection operators (rows.cu, segment.cu, route.cu,
// clip.cu): value types, row vectors and the argument checks of their entry
// points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>
#include <type_traits>
#include <utility>

#include "common.cuh"
#include "internal.hpp"

namespace spmvb {

// Accumulator of a value type: fp32, or fp64 for doubles.
template <typename T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T, typename Acc> __device__ __forceinline__ T narrow(Acc v);
template <> __device__ __forceinline__ float narrow<float, float>(float v) { return v; }
template <> __device__ __forceinline__ double narrow<double, double>(double v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half, float>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16, float>(float v) { return __float2bfloat16_rn(v); }

// VB bytes (2, 4, 8 or 16) of a row, loaded and stored as one access.
template <int VB> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

template <typename T, int VB>
struct alignas(VB) Pack {
  static constexpr int N = VB / static_cast<int>(sizeof(T));
  T v[N];
};

template <typename T, int VB>
__device__ __forceinline__ Pack<T, VB> ld_pack(const T* p) {
  using Raw = typename RawOf<VB>::type;
  Pack<T, VB> r;
  *reinterpret_cast<Raw*>(&r) = __ldg(reinterpret_cast<const Raw*>(p));
  return r;
}
// Read once: the line is the first to be evicted.
template <typename T, int VB>
__device__ __forceinline__ Pack<T, VB> ld_pack_stream(const T* p) {
  using Raw = typename RawOf<VB>::type;
  Pack<T, VB> r;
  *reinterpret_cast<Raw*>(&r) = __ldcs(reinterpret_cast<const Raw*>(p));
  return r;
}
template <typename T, int VB>
__device__ __forceinline__ void st_pack_stream(T* p, const Pack<T, VB>& v) {
  using Raw = typename RawOf<VB>::type;
  __stcs(reinterpret_cast<Raw*>(p), *reinterpret_cast<const Raw*>(&v));
}
// The widest access that every one of a call's row sets allows: base
// addresses, row strides and the row length in bytes are multiples of it.
inline int access_bytes(size_t elem, std::initializer_list<std::pair<const void*, int64_t>> sets, int64_t width) {
  uint64_t all = 16 | static_cast<uint64_t>(width) * elem;
  for (const auto& s : sets) all |= reinterpret_cast<uint64_t>(s.first) | static_cast<uint64_t>(s.second) * elem;
  int vb = 16;
  while (all & (vb - 1)) vb >>= 1;
  return std::max<int>(vb, static_cast<int>(elem));
}

// A strided set of rows on the host side of a call.
struct RowSet {
  const void* p;
  int64_t rows, ld, width;
  size_t elem;
  const char* name;
  // From the first row's begin to the last one's end (check_rows has seen that it fits).
  size_t bytes() const { return rows > 0 ? (static_cast<size_t>(rows - 1) * ld + width) * elem : 0; }
};

inline spmvb_status check_rows(const RowSet& s, int device) {
  if (s.ld < s.width) return fail(SPMVB_ERR_INVALID_ARGUMENT, std::string(s.name) + ": row stride below the row length");
  // No sum or product of offsets within the rows may pass 63 bits: a length
  // that wrapped would be found inside any allocation.
  const int64_t most = INT64_MAX / static_cast<int64_t>(s.elem);
  if (s.rows > 0 && (s.width > most || (s.rows > 1 && s.ld > (most - s.width) / (s.rows - 1))))
    return fail(SPMVB_ERR_INVALID_ARGUMENT, std::string(s.name) + ": the rows' extent passes 63 bits");
  if (reinterpret_cast<uintptr_t>(s.p) % s.elem)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, std::string(s.name) + " is not aligned to its elements");
  return check_device_ptr(s.p, s.bytes(), device, s.name);
}

// An output may not share elements with an input. Two column ranges of the
// same rows (equal strides) do not.
inline spmvb_status check_apart(const RowSet& out, const RowSet& in) {
  const auto a = reinterpret_cast<uintptr_t>(out.p), b = reinterpret_cast<uintptr_t>(in.p);
  if (!out.bytes() || !in.bytes() || a + out.bytes() <= b || b + in.bytes() <= a) return SPMVB_OK;
  // The stride of a lone row may be anything.
  const auto pitch = [](const RowSet& s) {
    const int64_t e = static_cast<int64_t>(s.elem);
    return s.ld <= INT64_MAX / e ? s.ld * e : 0;
  };
  const int64_t row = pitch(out);
  if (row > 0 && row == pitch(in)) {
    int64_t off = (static_cast<int64_t>(b) - static_cast<int64_t>(a)) % row;
    if (off < 0) off += row;
    if (off >= out.width * static_cast<int64_t>(out.elem) && off + in.width * static_cast<int64_t>(in.elem) <= row)
      return SPMVB_OK;
  }
  return fail(SPMVB_ERR_INVALID_ARGUMENT, std::string(out.name) + " overlaps " + in.name);
}

inline bool half_or_float(spmvb_dtype d) { return d == SPMVB_F32 || d == SPMVB_F16 || d == SPMVB_BF16; }
inline bool any_float(spmvb_dtype d) { return half_or_float(d) || d == SPMVB_F64; }

// Runs a handle's construction; a failed host allocation becomes a status.
template <typename F>
spmvb_status constructed(F&& f) {
  try {
    return f();
  } catch (const std::exception&) {
    return fail(SPMVB_ERR_OUT_OF_MEMORY, "host allocation failed");
  }
}

// A load of what another block has written: not moved before the fence it
// comes after, as the read-only loads (__ldg, __ldcg) may be.
__device__ __forceinline__ double ld_written(const double* p) {
  double r;
  asm volatile("ld.global.cg.f64 %0, [%1];" : "=d"(r) : "l"(p) : "memory");
  return r;
}
__device__ __forceinline__ float ld_written(const float* p) {
  float r;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(r) : "l"(p) : "memory");
  return r;
}

// New buffers are cleared on the legacy stream, which streams made without its
// ordering do not wait for: a handle's first call may be on one of those.
inline spmvb_status scratch_ready() {
  SPMVB_TRY_CUDA(cudaStreamSynchronize(nullptr));
  return SPMVB_OK;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- row products (rows.cu) ------------------------------------------------------
// out[t] = scale * X[idx[t]].
spmvb_status launch_lookup(spmvb_dtype dtype, const int* idx, int count, double scale, const RowSet& X,
                           const RowSet& out, int* err, cudaStream_t s);
// out[t] = sum_j w[t,j] * X[idx[t,j]], j < k (w null: 1).
spmvb_status launch_gather_sum(spmvb_dtype dtype, const int* idx, const float* w, int count, int k, const RowSet& X,
                               const RowSet& out, int* err, cudaStream_t s);
// out[pos[t,j]] = X[t].
spmvb_status launch_dispatch(spmvb_dtype dtype, const int* pos, int count, int k, const RowSet& X, const RowSet& out,
                             int* err, cudaStream_t s);
// dY[pos[t,j]] = w[t,j] * dout[t], dw[t,j] = <dout[t], Y[pos[t,j]]>.
spmvb_status launch_combine_grad(spmvb_dtype dtype, const int* pos, const float* w, int count, int k, const RowSet& Y,
                                 const RowSet& dout, const RowSet& dY, float* dw, int* err, cudaStream_t s);

}  // namespace spmvb
