// Row products of the row-selection operators: embedding lookup, and the
// exchange of rows with the experts (dispatch, combine and their gradients).
//
//   lookup         out[t]          = scale * table[tokens[t]]
//   dispatch       out[pos[t,j]]   = X[t]
//   dispatch_grad  dX[t]           = sum_j dout[pos[t,j]]
//   combine        out[t]          = sum_j w[t,j] * Y[pos[t,j]]
//   combine_grad   dY[pos[t,j]]    = w[t,j] * dout[t],  dw[t,j] = <dout[t], Y[pos[t,j]]>
//
// Each is one pass over its rows: every row is read once and written once,
// so HBM bounds all of them. Sums over j run in order in fp32 (fp64 for
// doubles) and are rounded once.
#include "select.cuh"

namespace spmvb {
namespace {

constexpr int kRowThreads = 256;

// The row an index names, or -1: an index past the end is reported and left out.
__device__ __forceinline__ int checked(int i, int rows, int* __restrict__ err) {
  if (i >= rows) {
    *err = 1;
    return -1;
  }
  return i < 0 ? -1 : i;
}

// out[t] = scale * sum_j w[t,j] * X[idx[t,j]] (w null: 1). blockDim.x threads
// share a row, blockDim.y rows share a block.
template <typename T, int VB, bool Weighted>
__global__ void __launch_bounds__(kRowThreads)
    gather_sum(const int* __restrict__ idx, const float* __restrict__ w, int count, int k, int rows,
               typename AccOf<T>::type scale, const T* __restrict__ X, int64_t ldx, T* __restrict__ out, int64_t ldo,
               int packs, int* __restrict__ err) {
  using Acc = typename AccOf<T>::type;
  constexpr int N = Pack<T, VB>::N;
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= count) return;
  const int64_t e0 = static_cast<int64_t>(t) * k;
  for (int v = threadIdx.x; v < packs; v += blockDim.x) {
    Acc sum[N] = {};
    for (int j = 0; j < k; ++j) {
      const int r = checked(__ldg(idx + e0 + j), rows, err);
      if (r < 0) continue;
      const Pack<T, VB> p = ld_pack<T, VB>(X + r * ldx + static_cast<int64_t>(v) * N);
      const Acc f = Weighted ? static_cast<Acc>(__ldg(w + e0 + j)) : Acc(1);
#pragma unroll
      for (int i = 0; i < N; ++i) sum[i] += f * widen(p.v[i]);
    }
    Pack<T, VB> o;
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = narrow<T, Acc>(sum[i] * scale);
    st_pack_stream<T, VB>(out + t * ldo + static_cast<int64_t>(v) * N, o);
  }
}

// out[pos[t,j]] = X[t]: the row is read once and written to each of its places.
template <typename T, int VB>
__global__ void __launch_bounds__(kRowThreads)
    scatter_rows(const int* __restrict__ pos, int count, int k, const T* __restrict__ X, int64_t ldx, int rows,
                 T* __restrict__ out, int64_t ldo, int packs, int* __restrict__ err) {
  constexpr int N = Pack<T, VB>::N;
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= count) return;
  const int64_t e0 = static_cast<int64_t>(t) * k;
  for (int v = threadIdx.x; v < packs; v += blockDim.x) {
    const Pack<T, VB> p = ld_pack_stream<T, VB>(X + t * ldx + static_cast<int64_t>(v) * N);
    for (int j = 0; j < k; ++j) {
      const int r = checked(__ldg(pos + e0 + j), rows, err);
      if (r >= 0) st_pack_stream<T, VB>(out + r * ldo + static_cast<int64_t>(v) * N, p);
    }
  }
}

// One block per token: dout[t] is held while the token's rows of Y pass by;
// the inner products are summed over each thread's columns, then the warp,
// then the warps in order.
template <typename T, int VB>
__global__ void __launch_bounds__(kRowThreads)
    combine_grad_rows(const int* __restrict__ pos, const float* __restrict__ w, int k, int rows,
                      const T* __restrict__ Y, int64_t ldy, const T* __restrict__ dout, int64_t ldd,
                      T* __restrict__ dY, int64_t lddy, float* __restrict__ dw, int packs, int* __restrict__ err) {
  constexpr int N = Pack<T, VB>::N;
  __shared__ float part[32][kRowThreads / 32];
  const int64_t t = blockIdx.x;
  const int64_t e0 = t * k;
  const int warps = blockDim.x >> 5;
  for (int j = 0; j < k; ++j) {
    const int r = checked(__ldg(pos + e0 + j), rows, err);
    float dot = 0.f;
    if (r >= 0) {
      const float f = __ldg(w + e0 + j);
      for (int v = threadIdx.x; v < packs; v += blockDim.x) {
        const int64_t c = static_cast<int64_t>(v) * N;
        const Pack<T, VB> d = ld_pack<T, VB>(dout + t * ldd + c);
        const Pack<T, VB> y = ld_pack_stream<T, VB>(Y + r * ldy + c);
        Pack<T, VB> o;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float g = static_cast<float>(widen(d.v[i]));
          dot += g * static_cast<float>(widen(y.v[i]));
          o.v[i] = narrow<T, typename AccOf<T>::type>(f * g);
        }
        st_pack_stream<T, VB>(dY + r * lddy + c, o);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    if ((threadIdx.x & 31) == 0) part[j][threadIdx.x >> 5] = dot;
  }
  __syncthreads();
  if (threadIdx.x < k) {
    float sum = 0.f;
    for (int i = 0; i < warps; ++i) sum += part[threadIdx.x][i];
    dw[e0 + threadIdx.x] = sum;
  }
}

// Threads of a block: x along the row (a power of two of at most 256), y rows.
dim3 row_block(int packs) {
  int x = 1;
  while (x < packs && x < kRowThreads) x *= 2;
  return dim3(x, kRowThreads / x);
}

}  // namespace

spmvb_status launch_lookup(spmvb_dtype dtype, const int* idx, const float* w, int count, int k, int rows, double scale,
                           const RowSet& X, const RowSet& out, int* err, cudaStream_t s) {
  if (count == 0) return SPMVB_OK;
  const int vb = access_bytes(X.elem, {{X.p, X.ld}, {out.p, out.ld}}, X.width);
  return with_type<true>(dtype, vb, [&](auto tv, auto vbc) -> spmvb_status {
    using T = decltype(tv);
    using Acc = typename AccOf<T>::type;
    constexpr int VB = decltype(vbc)::value;
    const int packs = static_cast<int>(X.width / Pack<T, VB>::N);
    const dim3 block = row_block(packs);
    const int grid = static_cast<int>(ceil_div(count, block.y));
    const T* x = static_cast<const T*>(X.p);
    T* o = static_cast<T*>(const_cast<void*>(out.p));
    if (w)
      gather_sum<T, VB, true><<<grid, block, 0, s>>>(idx, w, count, k, rows, Acc(scale), x, X.ld, o, out.ld, packs, err);
    else
      gather_sum<T, VB, false><<<grid, block, 0, s>>>(idx, w, count, k, rows, Acc(scale), x, X.ld, o, out.ld, packs, err);
    count_launch();
    SPMVB_TRY_CUDA(cudaGetLastError());
    return SPMVB_OK;
  });
}

spmvb_status launch_dispatch(spmvb_dtype dtype, const int* pos, int count, int k, const RowSet& X, const RowSet& out,
                             int* err, cudaStream_t s) {
  if (count == 0) return SPMVB_OK;
  const int vb = access_bytes(X.elem, {{X.p, X.ld}, {out.p, out.ld}}, X.width);
  return with_type<false>(dtype, vb, [&](auto tv, auto vbc) -> spmvb_status {
    using T = decltype(tv);
    constexpr int VB = decltype(vbc)::value;
    const int packs = static_cast<int>(X.width / Pack<T, VB>::N);
    const dim3 block = row_block(packs);
    scatter_rows<T, VB><<<static_cast<int>(ceil_div(count, block.y)), block, 0, s>>>(
        pos, count, k, static_cast<const T*>(X.p), X.ld, static_cast<int>(out.rows),
        static_cast<T*>(const_cast<void*>(out.p)), out.ld, packs, err);
    count_launch();
    SPMVB_TRY_CUDA(cudaGetLastError());
    return SPMVB_OK;
  });
}

spmvb_status launch_combine_grad(spmvb_dtype dtype, const int* pos, const float* w, int count, int k, const RowSet& Y,
                                 const RowSet& dout, const RowSet& dY, float* dw, int* err, cudaStream_t s) {
  if (count == 0) return SPMVB_OK;
  const int vb = access_bytes(Y.elem, {{Y.p, Y.ld}, {dout.p, dout.ld}, {dY.p, dY.ld}}, Y.width);
  return with_type<false>(dtype, vb, [&](auto tv, auto vbc) -> spmvb_status {
    using T = decltype(tv);
    constexpr int VB = decltype(vbc)::value;
    const int packs = static_cast<int>(Y.width / Pack<T, VB>::N);
    const int threads = std::max<int>(32, static_cast<int>(row_block(packs).x));
    combine_grad_rows<T, VB><<<count, threads, 0, s>>>(
        pos, w, k, static_cast<int>(Y.rows), static_cast<const T*>(Y.p), Y.ld, static_cast<const T*>(dout.p), dout.ld,
        static_cast<T*>(const_cast<void*>(dY.p)), dY.ld, dw, packs, err);
    count_launch();
    SPMVB_TRY_CUDA(cudaGetLastError());
    return SPMVB_OK;
  });
}

}  // namespace spmvb
