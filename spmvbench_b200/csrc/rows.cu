// Row products of the row-selection operators: embedding lookup, and the
// exchange of rows with the experts (dispatch, combine and their gradients).
//
//   lookup         out[t]          = scale * table[tokens[t]]
//   dispatch       out[pos[t,j]]   = X[t]
//   dispatch_grad  dX[t]           = sum_j dout[pos[t,j]]
//   combine        out[t]          = sum_j w[t,j] * Y[pos[t,j]]
//   combine_grad   dY[pos[t,j]]    = w[t,j] * dout[t],  dw[t,j] = <dout[t], Y[pos[t,j]]>
//
// Each is one pass over its rows. Sums over j run in order in fp32 (fp64 for
// doubles) and are rounded once. Where rows begin and end on 16-byte words every
// row is read once and written once, and HBM bounds them: about 0.9 of the copy rate
// for rows of 8 KB. Other rows take 2.3 to 3.7 times their floor, for the two
// loads a word, the ends moved by element, and dispatch reading a row again for
// each of its places: the lookup of 16,384 rows of 1,001 bf16 values 22.6 us
// (floor 8.0), dispatch + combine of 3,001 tokens x 3 such rows 27 us (7.2), both
// gradients in fp32 45.7 us (19.9).
//
// Rows are moved in 16-byte words of the row that is written. Where every row
// begins on such a word (Aligned), the words of the rows read are the same;
// else a word is put together from the two that hold its bytes, and the
// elements before the first and after the last whole word are moved alone.
#include <atomic>

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

// 16 bytes from an address that is aligned to its elements alone. Only words
// that hold one of the bytes are read.
template <typename T, bool Aligned>
__device__ __forceinline__ Pack<T, 16> ld_word(const T* p) {
  Pack<T, 16> r;
  if constexpr (Aligned) {
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  } else {
    const auto a = reinterpret_cast<uintptr_t>(p);
    const unsigned off = static_cast<unsigned>(a & 15u);
    const uint4* w = reinterpret_cast<const uint4*>(a - off);
    const uint4 x = __ldg(w), y = off ? __ldg(w + 1) : make_uint4(0, 0, 0, 0);
    // Words off / 4 .. off / 4 + 4 of the eight, then the bytes within.
    uint32_t v0 = x.x, v1 = x.y, v2 = x.z, v3 = x.w, v4 = y.x;
    if (off & 8u) {
      v0 = x.z; v1 = x.w; v2 = y.x; v3 = y.y; v4 = y.z;
    }
    if (off & 4u) {
      v0 = v1; v1 = v2; v2 = v3; v3 = v4; v4 = off & 8u ? y.w : y.y;
    }
    const unsigned bits = (off & 3u) * 8u;
    uint4 o = make_uint4(v0, v1, v2, v3);
    if constexpr (sizeof(T) == 2)
      o = make_uint4(__funnelshift_r(v0, v1, bits), __funnelshift_r(v1, v2, bits), __funnelshift_r(v2, v3, bits),
                     __funnelshift_r(v3, v4, bits));
    *reinterpret_cast<uint4*>(&r) = o;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void st_word(T* p, const Pack<T, 16>& v) {
  __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
}

// The words of a row that is written: elements first .. first + 16 / size - 1
// of word v. Unaligned rows have a word 0 of the elements before the first
// 16-byte boundary and a last one of those after the last: `count` < N.
template <typename T, bool Aligned>
struct Words {
  static constexpr int N = 16 / sizeof(T);
  int head, width;
  __device__ __forceinline__ Words(const T* row, int w)
      : head(Aligned ? 0 : min(w, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T)))),
        width(w) {}
  // The last word's first element may lie past the row, and past int32: its
  // place is an unsigned one, and the count behind it an exact difference.
  __device__ __forceinline__ int first(int v) const { return static_cast<int>(place(v)); }
  __device__ __forceinline__ int count(int v) const {
    if constexpr (Aligned) return N;
    return v == 0 ? head : min(N, static_cast<int>(static_cast<unsigned>(width) - place(v)));  // <= 0: past the end
  }
  __device__ __forceinline__ unsigned place(int v) const {
    return Aligned ? static_cast<unsigned>(v) * N : v == 0 ? 0u : head + (static_cast<unsigned>(v) - 1u) * N;
  }
};
// Words of a row of any alignment, at most.
inline int words_of(int width, size_t elem, bool aligned) {
  const int n = static_cast<int>(16 / elem);
  return aligned ? width / n : (width - 1) / n + 2;
}

// out[t] = scale * X[idx[t]]. blockDim.x threads share a row and take Ahead
// words of it at a time.
constexpr int kAhead = 4;
template <typename T, bool Aligned>
__global__ void __launch_bounds__(kRowThreads)
    copy_rows(const int* __restrict__ idx, int count, int rows, typename AccOf<T>::type scale, const T* __restrict__ X,
              int64_t ldx, T* __restrict__ out, int64_t ldo, int width, int words, int* __restrict__ err) {
  using Acc = typename AccOf<T>::type;
  constexpr int N = 16 / sizeof(T);
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= count) return;
  const int r = checked(__ldg(idx + t), rows, err);
  T* to = out + t * ldo;
  const T* from = X + max(r, 0) * ldx;
  const Words<T, Aligned> W(to, width);
  for (int v0 = threadIdx.x; v0 < words; v0 += blockDim.x * kAhead) {
    Pack<T, 16> p[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int v = v0 + q * blockDim.x;
      if (v < words && r >= 0 && W.count(v) == N) p[q] = ld_word<T, Aligned>(from + W.first(v));
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int v = v0 + q * blockDim.x;
      if (v >= words) continue;
      const int e = W.first(v), n = W.count(v);
      if (n == N) {
#pragma unroll
        for (int i = 0; i < N; ++i) p[q].v[i] = r >= 0 ? narrow<T, Acc>(widen(p[q].v[i]) * scale) : narrow<T, Acc>(0);
        st_word(to + e, p[q]);
      } else {
        for (int i = 0; i < n; ++i) to[e + i] = r >= 0 ? narrow<T, Acc>(widen(__ldg(from + e + i)) * scale) : narrow<T, Acc>(0);
      }
    }
  }
}

// out[t] = sum_j w[t,j] * X[idx[t,j]], Ahead rows loaded at a time: as many as
// leave 32 warps to an SM (more loads and fewer warps were slower: 8 ahead
// 59 us, 4 ahead 52 us for 4,096 x 8 rows of 4,096 bf16 values).
template <typename T, bool Aligned, bool Weighted>
__global__ void __launch_bounds__(kRowThreads, Aligned ? 4 : 6)
    gather_sum(const int* __restrict__ idx, const float* __restrict__ w, int count, int k, int rows,
               const T* __restrict__ X, int64_t ldx, T* __restrict__ out, int64_t ldo, int width, int words,
               int* __restrict__ err) {
  constexpr int N = 16 / sizeof(T), Ahead = Aligned ? 4 : 2;
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= count) return;
  const int64_t e0 = static_cast<int64_t>(t) * k;
  T* to = out + t * ldo;
  const Words<T, Aligned> W(to, width);
  for (int v = threadIdx.x; v < words; v += blockDim.x) {
    const int e = W.first(v), n = W.count(v);
    if (n == N) {
      float sum[N] = {};
      for (int j0 = 0; j0 < k; j0 += Ahead) {
        Pack<T, 16> p[Ahead];
        int r[Ahead];
#pragma unroll
        for (int q = 0; q < Ahead; ++q) r[q] = j0 + q < k ? __ldg(idx + e0 + j0 + q) : -1;
#pragma unroll
        for (int q = 0; q < Ahead; ++q)
          if (static_cast<unsigned>(r[q]) < static_cast<unsigned>(rows)) p[q] = ld_word<T, Aligned>(X + r[q] * ldx + e);
#pragma unroll
        for (int q = 0; q < Ahead; ++q) {
          if (checked(r[q], rows, err) < 0) continue;
          const float f = Weighted ? __ldg(w + e0 + j0 + q) : 1.f;
#pragma unroll
          for (int i = 0; i < N; ++i) sum[i] += f * widen(p[q].v[i]);
        }
      }
      Pack<T, 16> o;
#pragma unroll
      for (int i = 0; i < N; ++i) o.v[i] = narrow<T, float>(sum[i]);
      st_word(to + e, o);
    } else {
      for (int i = 0; i < n; ++i) {
        float sum = 0.f;
        for (int j = 0; j < k; ++j) {
          const int r = checked(__ldg(idx + e0 + j), rows, err);
          if (r >= 0) sum += (Weighted ? __ldg(w + e0 + j) : 1.f) * widen(__ldg(X + r * ldx + e + i));
        }
        to[e + i] = narrow<T, float>(sum);
      }
    }
  }
}

// The inner product of two words, in a tree; a word times a factor.
template <typename T>
__device__ __forceinline__ float word_dot(const Pack<T, 16>& a, const Pack<T, 16>& b) {
  constexpr int N = 16 / sizeof(T);
  float x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = widen(a.v[i]) * widen(b.v[i]);
#pragma unroll
  for (int s = N / 2; s > 0; s /= 2)
#pragma unroll
    for (int i = 0; i < s; ++i) x[i] += x[i + s];
  return x[0];
}
template <typename T>
__device__ __forceinline__ Pack<T, 16> scaled(const Pack<T, 16>& a, float f) {
  Pack<T, 16> o;
#pragma unroll
  for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) o.v[i] = narrow<T, float>(f * widen(a.v[i]));
  return o;
}

// ---- up to kFew rows a token, aligned ------------------------------------------
// The words of all of a token's rows are copied to shared memory at once, each
// thread's to places of its own, so a thread waits for its own copies alone
// and the block for nothing. 64 KB a block are on their way without a
// register, three times what the registers of the kernels for any k hold. For
// 4,096 tokens of 8 rows of 4,096 bf16 values: 46 us against 57 us for the sum
// (6.5 TB/s), 90 us against 99 us for the gradient (6.3 TB/s of both ways).
constexpr int kFew = 8, kWordsHeld = 2;
constexpr size_t few_shared(int k) { return static_cast<size_t>(k) * kWordsHeld * kRowThreads * 16; }

__device__ __forceinline__ void copy_word(uint4* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `Left` of the groups issued last are on their way.
template <int Left>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(Left) : "memory");
}
template <typename T>
__device__ __forceinline__ Pack<T, 16> held_word(const uint4* from) {
  Pack<T, 16> r;
  *reinterpret_cast<uint4*>(&r) = *from;
  return r;
}

template <typename T, bool Weighted>
__global__ void __launch_bounds__(kRowThreads)
    gather_sum_few(const int* __restrict__ idx, const float* __restrict__ w, int count, int k, int rows,
                   const T* __restrict__ X, int64_t ldx, T* __restrict__ out, int64_t ldo, int words,
                   int* __restrict__ err) {
  extern __shared__ __align__(16) uint4 slots[];
  constexpr int N = 16 / sizeof(T);
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= count) return;
  uint4* mine = slots + threadIdx.y * blockDim.x + threadIdx.x;  // slot (h, j) kRowThreads * (h * k + j) on
  const int64_t e0 = static_cast<int64_t>(t) * k;
  int r[kFew];
  float f[kFew];
#pragma unroll
  for (int j = 0; j < kFew; ++j) {
    r[j] = j < k ? __ldg(idx + e0 + j) : -1;
    f[j] = !Weighted ? 1.f : j < k ? __ldg(w + e0 + j) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < kFew; ++j) r[j] = checked(r[j], rows, err);
  T* to = out + t * ldo;
  for (int v0 = threadIdx.x; v0 < words; v0 += kWordsHeld * blockDim.x) {
#pragma unroll
    for (int h = 0; h < kWordsHeld; ++h) {
      const int v = v0 + h * blockDim.x;
#pragma unroll
      for (int j = 0; j < kFew; ++j)
        if (v < words && r[j] >= 0)
          copy_word(mine + kRowThreads * (h * k + j), X + r[j] * ldx + static_cast<int64_t>(v) * N);
      copies_issued();
    }
    const auto add = [&](int h) {
      const int v = v0 + h * blockDim.x;
      if (v >= words) return;
      float sum[N] = {};
#pragma unroll
      for (int j = 0; j < kFew; ++j) {
        if (r[j] < 0) continue;
        const Pack<T, 16> p = held_word<T>(mine + kRowThreads * (h * k + j));
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] += f[j] * widen(p.v[i]);
      }
      Pack<T, 16> o;
#pragma unroll
      for (int i = 0; i < N; ++i) o.v[i] = narrow<T, float>(sum[i]);
      st_word(to + static_cast<int64_t>(v) * N, o);
    };
    static_assert(kWordsHeld == 2);
    copies_wait<1>();
    add(0);
    copies_wait<0>();
    add(1);
  }
}

// One block per token, as combine_grad_rows.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    combine_grad_few(const int* __restrict__ pos, const float* __restrict__ w, int k, int rows,
                     const T* __restrict__ Y, int64_t ldy, const T* __restrict__ dout, int64_t ldd,
                     T* __restrict__ dY, int64_t lddy, float* __restrict__ dw, int words, int* __restrict__ err) {
  extern __shared__ __align__(16) uint4 slots[];
  constexpr int N = 16 / sizeof(T);
  __shared__ float part[kFew][kRowThreads / 32];
  const int64_t t = blockIdx.x;
  const int64_t e0 = t * k;
  const int warps = blockDim.x >> 5, wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint4* mine = slots + threadIdx.x;
  int r[kFew];
  float f[kFew], dot[kFew];
#pragma unroll
  for (int j = 0; j < kFew; ++j) {
    r[j] = j < k ? __ldg(pos + e0 + j) : -1;
    f[j] = j < k ? __ldg(w + e0 + j) : 0.f;
    dot[j] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < kFew; ++j) r[j] = checked(r[j], rows, err);
  const T* d = dout + t * ldd;
  for (int v0 = threadIdx.x; v0 < words; v0 += kWordsHeld * blockDim.x) {
    Pack<T, 16> held[kWordsHeld];
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
#pragma unroll
      for (int h = 0; h < kWordsHeld; ++h) {
        const int v = v0 + h * blockDim.x;
        if (v < words && r[j] >= 0)
          copy_word(mine + kRowThreads * (h * k + j), Y + r[j] * ldy + static_cast<int64_t>(v) * N);
      }
      copies_issued();
    }
#pragma unroll
    for (int h = 0; h < kWordsHeld; ++h)
      if (v0 + h * blockDim.x < words) held[h] = ld_word<T, true>(d + static_cast<int64_t>(v0 + h * blockDim.x) * N);
    const auto one = [&](int j) {
      if (r[j] < 0) return;
#pragma unroll
      for (int h = 0; h < kWordsHeld; ++h) {
        const int v = v0 + h * blockDim.x;
        if (v >= words) continue;
        dot[j] += word_dot<T>(held[h], held_word<T>(mine + kRowThreads * (h * k + j)));
        st_word(dY + r[j] * lddy + static_cast<int64_t>(v) * N, scaled<T>(held[h], f[j]));
      }
    };
    static_assert(kFew == 8);
    copies_wait<7>(); one(0);
    copies_wait<6>(); one(1);
    copies_wait<5>(); one(2);
    copies_wait<4>(); one(3);
    copies_wait<3>(); one(4);
    copies_wait<2>(); one(5);
    copies_wait<1>(); one(6);
    copies_wait<0>(); one(7);
  }
#pragma unroll
  for (int j = 0; j < kFew; ++j) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
    if (lane == 0) part[j][wid] = dot[j];
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < k) {
    float sum = 0.f;
    for (int i = 0; i < warps; ++i) sum += part[threadIdx.x][i];
    dw[e0 + threadIdx.x] = sum;
  }
}

// out[pos[t,j]] = X[t]. Aligned rows are read once and written to each of their
// places; others are read again for each place (from the L1), as the words
// that are written lie differently in each.
template <typename T, bool Aligned>
__global__ void __launch_bounds__(kRowThreads)
    scatter_rows(const int* __restrict__ pos, int count, int k, const T* __restrict__ X, int64_t ldx, int rows,
                 T* __restrict__ out, int64_t ldo, int width, int words, int* __restrict__ err) {
  constexpr int N = 16 / sizeof(T), Two = 2;
  const int t = blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= count) return;
  const int64_t e0 = static_cast<int64_t>(t) * k;
  const T* from = X + t * ldx;
  if constexpr (Aligned) {
    for (int v = threadIdx.x; v < words; v += blockDim.x * Two) {
      Pack<T, 16> p[Two];
#pragma unroll
      for (int q = 0; q < Two; ++q)
        if (v + q * blockDim.x < words) p[q] = ld_word<T, true>(from + static_cast<int64_t>(v + q * blockDim.x) * N);
#pragma unroll 4
      for (int j = 0; j < k; ++j) {
        const int r = checked(__ldg(pos + e0 + j), rows, err);
        if (r < 0) continue;
#pragma unroll
        for (int q = 0; q < Two; ++q)
          if (v + q * blockDim.x < words) st_word(out + r * ldo + static_cast<int64_t>(v + q * blockDim.x) * N, p[q]);
      }
    }
  } else {
    for (int j = 0; j < k; ++j) {
      const int r = checked(__ldg(pos + e0 + j), rows, err);
      if (r < 0) continue;
      T* to = out + r * ldo;
      const Words<T, false> W(to, width);
#pragma unroll 2
      for (int v = threadIdx.x; v < words; v += blockDim.x) {
        const int e = W.first(v), n = W.count(v);
        if (n == N)
          st_word(to + e, ld_word<T, false>(from + e));
        else
          for (int i = 0; i < n; ++i) to[e + i] = __ldg(from + e + i);
      }
    }
  }
}

// One block per token: dout[t] is held (Held words a thread) while the token's
// rows of Y pass by, two at a time; the inner products are summed over each
// word in a tree, each thread's words, then the warp, then the warps in order.
constexpr int kHeld = 2;
template <typename T, bool Aligned>
__global__ void __launch_bounds__(kRowThreads)
    combine_grad_rows(const int* __restrict__ pos, const float* __restrict__ w, int k, int rows,
                      const T* __restrict__ Y, int64_t ldy, const T* __restrict__ dout, int64_t ldd,
                      T* __restrict__ dY, int64_t lddy, float* __restrict__ dw, int width, int words,
                      int* __restrict__ err) {
  constexpr int N = 16 / sizeof(T), Pair = 2;
  __shared__ float part[32][kRowThreads / 32];
  __shared__ int place[32];
  __shared__ float weight[32];
  const int64_t t = blockIdx.x;
  const int64_t e0 = t * k;
  const int warps = blockDim.x >> 5, wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (static_cast<int>(threadIdx.x) < k) {
    place[threadIdx.x] = checked(__ldg(pos + e0 + threadIdx.x), rows, err);
    weight[threadIdx.x] = __ldg(w + e0 + threadIdx.x);
  }
  for (int i = threadIdx.x; i < k * warps; i += blockDim.x) part[i / warps][i % warps] = 0.f;
  __syncthreads();
  const T* d = dout + t * ldd;
  const auto add_up = [&](int j, float dot) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    if (lane == 0) part[j][wid] += dot;
  };
  if constexpr (Aligned) {
    // A thread's words v0, v0 + blockDim.x; all threads make the same turns.
    for (int b = 0; b < words; b += blockDim.x * kHeld) {
      const int v0 = b + threadIdx.x;
      Pack<T, 16> held[kHeld];
#pragma unroll
      for (int q = 0; q < kHeld; ++q)
        if (v0 + q * blockDim.x < words) held[q] = ld_word<T, true>(d + static_cast<int64_t>(v0 + q * blockDim.x) * N);
      for (int j0 = 0; j0 < k; j0 += Pair) {
        Pack<T, 16> y[Pair][kHeld];
#pragma unroll
        for (int u = 0; u < Pair; ++u) {
          const int r = j0 + u < k ? place[j0 + u] : -1;
#pragma unroll
          for (int q = 0; q < kHeld; ++q)
            if (r >= 0 && v0 + q * blockDim.x < words)
              y[u][q] = ld_word<T, true>(Y + r * ldy + static_cast<int64_t>(v0 + q * blockDim.x) * N);
        }
#pragma unroll
        for (int u = 0; u < Pair; ++u) {
          const int r = j0 + u < k ? place[j0 + u] : -1;
          if (r < 0) continue;
          float dot = 0.f;
#pragma unroll
          for (int q = 0; q < kHeld; ++q) {
            if (v0 + q * blockDim.x >= words) continue;
            dot += word_dot<T>(held[q], y[u][q]);
            st_word(dY + r * lddy + static_cast<int64_t>(v0 + q * blockDim.x) * N, scaled<T>(held[q], weight[j0 + u]));
          }
          add_up(j0 + u, dot);
        }
      }
    }
  } else {
    for (int j = 0; j < k; ++j) {
      const int r = place[j];
      if (r < 0) continue;
      T* to = dY + r * lddy;
      const T* y = Y + r * ldy;
      const Words<T, false> W(to, width);
      float dot = 0.f;
#pragma unroll 2
      for (int v = threadIdx.x; v < words; v += blockDim.x) {
        const int e = W.first(v), n = W.count(v);
        if (n == N) {
          const Pack<T, 16> a = ld_word<T, false>(d + e);
          dot += word_dot<T>(a, ld_word<T, false>(y + e));
          st_word(to + e, scaled<T>(a, weight[j]));
        } else {
          for (int i = 0; i < n; ++i) {
            const float g = widen(__ldg(d + e + i));
            dot += g * widen(__ldg(y + e + i));
            to[e + i] = narrow<T, float>(weight[j] * g);
          }
        }
      }
      add_up(j, dot);
    }
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < k) {
    float sum = 0.f;
    for (int i = 0; i < warps; ++i) sum += part[threadIdx.x][i];
    dw[e0 + threadIdx.x] = sum;
  }
}

// Threads along a row for `words` words, `each` to a thread: a power of two,
// 256 at most.
int across(int words, int each, int least) {
  int x = least;
  while (x * each < words && x < kRowThreads) x *= 2;
  return x;
}

template <bool F64, typename F>
spmvb_status with_rows(spmvb_dtype d, bool aligned, F&& f) {
  const auto by = [&](auto tv) -> spmvb_status {
    return aligned ? f(tv, std::true_type{}) : f(tv, std::false_type{});
  };
  switch (d) {
    case SPMVB_F32: return by(float{});
    case SPMVB_F16: return by(__half{});
    case SPMVB_BF16: return by(__nv_bfloat16{});
    case SPMVB_F64:
      if constexpr (F64) return by(double{});
      break;
  }
  return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype");
}

// Lets a kernel have few_shared(kFew) bytes: asked of the runtime once a device.
template <auto Kernel>
spmvb_status allow_shared() {
  static std::atomic<uint64_t> asked{0};
  int device = 0;
  SPMVB_TRY_CUDA(cudaGetDevice(&device));
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (asked.load(std::memory_order_relaxed) & bit) return SPMVB_OK;
  SPMVB_TRY_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(few_shared(kFew))));
  asked.fetch_or(bit, std::memory_order_relaxed);
  return SPMVB_OK;
}

spmvb_status launched() {
  count_launch();
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

template <typename T>
T* rows_at(const RowSet& r) {
  return static_cast<T*>(const_cast<void*>(r.p));
}

}  // namespace

spmvb_status launch_lookup(spmvb_dtype dtype, const int* idx, int count, double scale, const RowSet& X,
                           const RowSet& out, int* err, cudaStream_t s) {
  if (count == 0) return SPMVB_OK;
  const bool aligned = access_bytes(X.elem, {{X.p, X.ld}, {out.p, out.ld}}, X.width) == 16;
  return with_rows<true>(dtype, aligned, [&](auto tv, auto al) -> spmvb_status {
    using T = decltype(tv);
    constexpr bool Aligned = decltype(al)::value;
    const int width = static_cast<int>(X.width), words = words_of(width, sizeof(T), Aligned);
    const int x = across(words, kAhead, 1), y = kRowThreads / x;
    copy_rows<T, Aligned><<<static_cast<int>(ceil_div(count, y)), dim3(x, y), 0, s>>>(
        idx, count, static_cast<int>(X.rows), static_cast<typename AccOf<T>::type>(scale), rows_at<const T>(X), X.ld,
        rows_at<T>(out), out.ld, width, words, err);
    return launched();
  });
}

spmvb_status launch_gather_sum(spmvb_dtype dtype, const int* idx, const float* w, int count, int k, const RowSet& X,
                               const RowSet& out, int* err, cudaStream_t s) {
  if (count == 0) return SPMVB_OK;
  const bool aligned = access_bytes(X.elem, {{X.p, X.ld}, {out.p, out.ld}}, X.width) == 16;
  return with_rows<false>(dtype, aligned, [&](auto tv, auto al) -> spmvb_status {
    using T = decltype(tv);
    constexpr bool Aligned = decltype(al)::value;
    const int width = static_cast<int>(X.width), words = words_of(width, sizeof(T), Aligned);
    if constexpr (Aligned) {
      if (k > 1 && k <= kFew) {
        const int x = across(words, kWordsHeld, 1), y = kRowThreads / x;
        const auto few = w ? gather_sum_few<T, true> : gather_sum_few<T, false>;
        SPMVB_TRY((w ? allow_shared<gather_sum_few<T, true>>() : allow_shared<gather_sum_few<T, false>>()));
        few<<<static_cast<int>(ceil_div(count, y)), dim3(x, y), few_shared(k), s>>>(
            idx, w, count, k, static_cast<int>(X.rows), rows_at<const T>(X), X.ld, rows_at<T>(out), out.ld, words, err);
        return launched();
      }
    }
    const int x = across(words, 1, 1), y = kRowThreads / x;
    const auto kernel = w ? gather_sum<T, Aligned, true> : gather_sum<T, Aligned, false>;
    kernel<<<static_cast<int>(ceil_div(count, y)), dim3(x, y), 0, s>>>(idx, w, count, k, static_cast<int>(X.rows),
                                                                      rows_at<const T>(X), X.ld, rows_at<T>(out), out.ld,
                                                                      width, words, err);
    return launched();
  });
}

spmvb_status launch_dispatch(spmvb_dtype dtype, const int* pos, int count, int k, const RowSet& X, const RowSet& out,
                             int* err, cudaStream_t s) {
  if (count == 0) return SPMVB_OK;
  const bool aligned = access_bytes(X.elem, {{X.p, X.ld}, {out.p, out.ld}}, X.width) == 16;
  return with_rows<false>(dtype, aligned, [&](auto tv, auto al) -> spmvb_status {
    using T = decltype(tv);
    constexpr bool Aligned = decltype(al)::value;
    const int width = static_cast<int>(X.width), words = words_of(width, sizeof(T), Aligned);
    const int x = across(words, Aligned ? 2 : 1, 1), y = kRowThreads / x;
    scatter_rows<T, Aligned><<<static_cast<int>(ceil_div(count, y)), dim3(x, y), 0, s>>>(
        pos, count, k, rows_at<const T>(X), X.ld, static_cast<int>(out.rows), rows_at<T>(out), out.ld, width, words, err);
    return launched();
  });
}

spmvb_status launch_combine_grad(spmvb_dtype dtype, const int* pos, const float* w, int count, int k, const RowSet& Y,
                                 const RowSet& dout, const RowSet& dY, float* dw, int* err, cudaStream_t s) {
  if (count == 0) return SPMVB_OK;
  const bool aligned = access_bytes(Y.elem, {{Y.p, Y.ld}, {dout.p, dout.ld}, {dY.p, dY.ld}}, Y.width) == 16;
  return with_rows<false>(dtype, aligned, [&](auto tv, auto al) -> spmvb_status {
    using T = decltype(tv);
    constexpr bool Aligned = decltype(al)::value;
    const int width = static_cast<int>(Y.width), words = words_of(width, sizeof(T), Aligned);
    if constexpr (Aligned) {
      if (k <= kFew) {
        SPMVB_TRY(allow_shared<combine_grad_few<T>>());
        combine_grad_few<T><<<count, across(words, kWordsHeld, 32), few_shared(k), s>>>(
            pos, w, k, static_cast<int>(Y.rows), rows_at<const T>(Y), Y.ld, rows_at<const T>(dout), dout.ld,
            rows_at<T>(dY), dY.ld, dw, words, err);
        return launched();
      }
    }
    combine_grad_rows<T, Aligned><<<count, across(words, Aligned ? kHeld : 1, 32), 0, s>>>(
        pos, w, k, static_cast<int>(Y.rows), rows_at<const T>(Y), Y.ld, rows_at<const T>(dout), dout.ld,
        rows_at<T>(dY), dY.ld, dw, width, words, err);
    return launched();
  });
}

}  // namespace spmvb
