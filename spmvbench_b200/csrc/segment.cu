// The transposed product of a selection: the stable order of the tokens by the
// row they name, and the embedding gradient made with it.
//
// Order. The entries are sorted by key (the row named, or n for none) with a
// least-significant-digit radix sort, kDigitBits at a time. One pass: every
// tile of kTile entries counts its digits (digit_counts); one warp per digit
// turns the counts of all tiles into running sums (digit_scan); every tile
// ranks its entries among the equal digits before them and writes them to
// their places (digit_scatter). Ranks follow the entries' order, so the sort
// is stable and nothing depends on timing.
//
// Gradient. dtable[r] = scale * sum of dout[t] over the tokens that name r:
// in sorted order the tokens of one row are neighbours (a run). A block takes
// kChunk sorted entries and a range of columns, adds each run in registers
// and writes the runs that lie inside its chunk. A run that crosses a chunk's
// edge leaves its part in scratch (slot 0: the run came in from the chunk
// before, slot 1: it begins here and goes on), and the chunk where it begins
// adds the parts in chunk order afterwards (join_runs). A frequent token is so
// spread over many blocks, in a fixed order of summation.
#include "select.cuh"

namespace spmvb {
namespace {

constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kPerThread = 4;
constexpr int kTile = kSortThreads * kPerThread;

__device__ __forceinline__ uint32_t key_of(int i, uint32_t n, int* err) {
  if (i >= 0 && static_cast<uint32_t>(i) >= n) *err = 1;
  return i < 0 || static_cast<uint32_t>(i) >= n ? n : static_cast<uint32_t>(i);
}

// Keys of a pass: the indices themselves (First) or the last pass's keys.
template <bool First>
__device__ __forceinline__ uint32_t load_key(const void* src, int64_t i, uint32_t n, int* err) {
  if (First) return key_of(static_cast<const int*>(src)[i], n, err);
  return static_cast<const uint32_t*>(src)[i];
}

// counts[digit * tiles + tile].
template <bool First>
__global__ void __launch_bounds__(kSortThreads)
    digit_counts(const void* __restrict__ src, int64_t count, uint32_t n, int shift, int tiles, int* __restrict__ counts,
                 int* __restrict__ err) {
  __shared__ int c[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) c[d] = 0;
  __syncthreads();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kTile;
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) {
    const int64_t i = i0 + q * kSortThreads + threadIdx.x;
    if (i < count) atomicAdd(&c[(load_key<First>(src, i, n, err) >> shift) & (kDigits - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) counts[static_cast<int64_t>(d) * tiles + blockIdx.x] = c[d];
}

// One warp per digit: counts become the number of the digit's entries in the
// tiles before, totals[digit] their sum.
__global__ void __launch_bounds__(256) digit_scan(int* __restrict__ counts, int tiles, int* __restrict__ totals) {
  const int d = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  int* c = counts + static_cast<int64_t>(d) * tiles;
  int sum = 0;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const int t = t0 + lane;
    const int v = t < tiles ? c[t] : 0;
    int incl = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += u;
    }
    if (t < tiles) c[t] = sum + incl - v;
    sum += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) totals[d] = sum;
}

// Exclusive sum of one value per digit over a block: thread t holds digits
// 2t and 2t + 1 (kDigits = 2 * kSortThreads).
__device__ __forceinline__ void scan_digits(int (&v)[2], int* sh) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int own = v[0] + v[1];
  int incl = own;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += u;
  }
  if (lane == 31) sh[w] = incl;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int i = 0; i < kSortWarps; ++i) before += i < w ? sh[i] : 0;
  const int a = v[0];
  v[0] = before + incl - own;
  v[1] = v[0] + a;
  __syncthreads();
}
static_assert(kDigits == 2 * kSortThreads);

template <bool First>
__global__ void __launch_bounds__(kSortThreads)
    digit_scatter(const void* __restrict__ src, const int* __restrict__ src_vals, int64_t count, uint32_t n, int shift,
                  int tiles, const int* __restrict__ counts, const int* __restrict__ totals,
                  uint32_t* __restrict__ dst_keys, int* __restrict__ dst_vals, int* __restrict__ err) {
  __shared__ int wc[kSortWarps][kDigits];  // a warp's count of each digit, then its first place
  __shared__ int sh[kSortWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < kSortWarps * kDigits; d += kSortThreads) (&wc[0][0])[d] = 0;
  __syncthreads();
  // A warp's entries are neighbours: 32 * kPerThread of them, in rounds of 32.
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kTile + w * (32 * kPerThread) + lane;
  uint32_t key[kPerThread];
  int rank[kPerThread];
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) {
    const int64_t i = i0 + q * 32;
    const bool in = i < count;
    key[q] = in ? load_key<First>(src, i, n, err) : 0u;
    const int d = in ? static_cast<int>((key[q] >> shift) & (kDigits - 1)) : kDigits + lane;
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const unsigned before = same & ((1u << lane) - 1u);
    const int base = in ? wc[w][d] : 0;
    rank[q] = base + __popc(before);
    __syncwarp();
    if (in && before == 0) wc[w][d] = base + __popc(same);
    __syncwarp();
  }
  __syncthreads();
  // First place of each digit: all smaller digits, then this digit in the
  // tiles and the warps before.
  int v[2] = {totals[2 * threadIdx.x], totals[2 * threadIdx.x + 1]};
  scan_digits(v, sh);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d = 2 * threadIdx.x + h;
    int at = v[h] + counts[static_cast<int64_t>(d) * tiles + blockIdx.x];
#pragma unroll
    for (int i = 0; i < kSortWarps; ++i) {
      const int c = wc[i][d];
      wc[i][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) {
    const int64_t i = i0 + q * 32;
    if (i >= count) continue;
    const int at = wc[w][(key[q] >> shift) & (kDigits - 1)] + rank[q];
    dst_keys[at] = key[q];
    dst_vals[at] = First ? static_cast<int>(i) : src_vals[i];
  }
}

// ---- embedding gradient ----------------------------------------------------------
constexpr int kChunk = 16;
constexpr int kGradThreads = 256;

template <typename T, typename G, int N>
__device__ __forceinline__ void store_row(G* dst, const typename AccOf<T>::type (&sum)[N],
                                          typename AccOf<T>::type scale, bool accumulate) {
  using Acc = typename AccOf<T>::type;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    Acc v = sum[i] * scale;
    if (accumulate) v += widen(dst[i]);
    dst[i] = narrow<G, Acc>(v);
  }
}

template <typename T, typename G, int VB>
__global__ void __launch_bounds__(kGradThreads)
    run_sums(const uint32_t* __restrict__ keys, const int* __restrict__ vals, int64_t count, uint32_t n,
             const T* __restrict__ dout, int64_t ldo, typename AccOf<T>::type scale, G* __restrict__ dtable, int64_t ldt,
             int packs, int width, bool accumulate, typename AccOf<T>::type* __restrict__ parts) {
  using Acc = typename AccOf<T>::type;
  constexpr int N = Pack<T, VB>::N;
  const int v = blockIdx.y * kGradThreads + threadIdx.x;
  if (v >= packs) return;
  const int64_t c = static_cast<int64_t>(v) * N;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kChunk;
  const int64_t last = min(first + kChunk, count);
  const bool came_in = first > 0 && keys[first - 1] == keys[first];
  const bool goes_on = last < count && keys[last] == keys[last - 1];
  Acc sum[N] = {};
  int64_t begin = first;
  for (int64_t i = first; i < last; ++i) {
    const uint32_t key = keys[i];
    if (key >= n) return;  // the entries that select nothing come last
    const Pack<T, VB> p = ld_pack_stream<T, VB>(dout + vals[i] * ldo + c);
#pragma unroll
    for (int q = 0; q < N; ++q) sum[q] += widen(p.v[q]);
    if (i + 1 < last && keys[i + 1] == key) continue;
    const bool in = begin == first && came_in, on = i + 1 == last && goes_on;
    if (in || on) {
      Acc* part = parts + (static_cast<int64_t>(blockIdx.x) * 2 + (in ? 0 : 1)) * width + c;
#pragma unroll
      for (int q = 0; q < N; ++q) part[q] = sum[q];
    } else {
      store_row<T, G, N>(dtable + key * ldt + c, sum, scale, accumulate);
    }
#pragma unroll
    for (int q = 0; q < N; ++q) sum[q] = 0;
    begin = i + 1;
  }
}

// Adds the parts of the run that begins in this chunk and goes on.
template <typename T, typename G>
__global__ void __launch_bounds__(kGradThreads)
    join_runs(const uint32_t* __restrict__ keys, int64_t count, uint32_t n, typename AccOf<T>::type scale,
              G* __restrict__ dtable, int64_t ldt, int width, bool accumulate,
              const typename AccOf<T>::type* __restrict__ parts) {
  using Acc = typename AccOf<T>::type;
  const int64_t chunk = blockIdx.x, first = chunk * kChunk, last = min(first + kChunk, count);
  if (last >= count) return;
  const uint32_t key = keys[last - 1];
  if (key >= n || keys[last] != key) return;                             // nothing goes on
  if (keys[first] == key && first > 0 && keys[first - 1] == key) return;  // it began before
  const int c = blockIdx.y * kGradThreads + threadIdx.x;
  if (c >= width) return;
  Acc sum = parts[(chunk * 2 + 1) * width + c];
  for (int64_t q = chunk + 1; q * kChunk < count && keys[q * kChunk] == key; ++q) sum += parts[q * 2 * width + c];
  const Acc one[1] = {sum};
  store_row<T, G, 1>(dtable + key * ldt + c, one, scale, accumulate);
}

}  // namespace

spmvb_status SortSpace::alloc(int64_t entries) {
  const int64_t tiles = std::max<int64_t>(1, ceil_div(entries, kTile));
  for (int i = 0; i < 2; ++i) {
    SPMVB_TRY(keys[i].alloc(entries * 4));
    SPMVB_TRY(vals[i].alloc(entries * 4));
  }
  SPMVB_TRY(counts.alloc(static_cast<size_t>(tiles) * kDigits * 4));
  SPMVB_TRY(totals.alloc(kDigits * 4));
  cap = entries;
  return SPMVB_OK;
}

spmvb_status sort_entries(SortSpace& space, const int* idx, int64_t count, int n, int* err, cudaStream_t s, Sorted* out) {
  const int tiles = static_cast<int>(ceil_div(count, kTile));
  int bits = 1;
  while (bits < 32 && (static_cast<uint64_t>(n) >> bits) != 0) ++bits;
  int* counts = space.counts.as<int>();
  int* totals = space.totals.as<int>();
  int at = 0;
  for (int shift = 0; shift < bits; shift += kDigitBits, at ^= 1) {
    const bool first = shift == 0;
    const void* src = first ? static_cast<const void*>(idx) : space.keys[at ^ 1].get();
    const int* vals = space.vals[at ^ 1].as<int>();
    uint32_t* dk = space.keys[at].as<uint32_t>();
    int* dv = space.vals[at].as<int>();
    if (first) {
      digit_counts<true><<<tiles, kSortThreads, 0, s>>>(src, count, n, shift, tiles, counts, err);
      digit_scan<<<kDigits / 8, 256, 0, s>>>(counts, tiles, totals);
      digit_scatter<true><<<tiles, kSortThreads, 0, s>>>(src, vals, count, n, shift, tiles, counts, totals, dk, dv, err);
    } else {
      digit_counts<false><<<tiles, kSortThreads, 0, s>>>(src, count, n, shift, tiles, counts, err);
      digit_scan<<<kDigits / 8, 256, 0, s>>>(counts, tiles, totals);
      digit_scatter<false><<<tiles, kSortThreads, 0, s>>>(src, vals, count, n, shift, tiles, counts, totals, dk, dv, err);
    }
    count_launch(3);
    out->keys = dk;
    out->entries = dv;
  }
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // namespace spmvb

struct spmvb_embedding_st {
  spmvb_context ctx = nullptr;
  int device = 0, rows = 0, width = 0, max_tokens = 0;
  spmvb::SortSpace sort;
  spmvb::DevBuf parts;  // 2 rows of sums (fp64 wide) per chunk
};

using namespace spmvb;

namespace {

template <typename T, typename G, int VB>
spmvb_status lookup_grad(spmvb_embedding E, const Sorted& sorted, int count, double scale, const RowSet& dout,
                         const RowSet& dtable, bool accumulate, cudaStream_t s) {
  using Acc = typename AccOf<T>::type;
  const int packs = E->width / Pack<T, VB>::N;
  const int chunks = static_cast<int>(ceil_div(count, kChunk));
  G* dt = static_cast<G*>(const_cast<void*>(dtable.p));
  run_sums<T, G, VB><<<dim3(chunks, static_cast<unsigned>(ceil_div(packs, kGradThreads))), kGradThreads, 0, s>>>(
      sorted.keys, sorted.entries, count, E->rows, static_cast<const T*>(dout.p), dout.ld, Acc(scale), dt, dtable.ld,
      packs, E->width, accumulate, E->parts.as<Acc>());
  join_runs<T, G><<<dim3(chunks, static_cast<unsigned>(ceil_div(E->width, kGradThreads))), kGradThreads, 0, s>>>(
      sorted.keys, count, E->rows, Acc(scale), dt, dtable.ld, E->width, accumulate, E->parts.as<Acc>());
  count_launch(2);
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // namespace

extern "C" {

spmvb_status spmvb_embedding_create(spmvb_context ctx, int32_t rows, int32_t width, int32_t max_tokens,
                                    spmvb_embedding* out) {
  clear_error();
  if (!ctx || !out) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null context or output");
  if (rows < 1 || width < 1 || max_tokens < 0)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "rows and width must be positive, max_tokens not negative");
  return constructed([&]() -> spmvb_status {
    DeviceGuard g(ctx->device);
    auto E = std::make_unique<spmvb_embedding_st>();
    E->ctx = ctx;
    E->device = ctx->device;
    E->rows = rows;
    E->width = width;
    E->max_tokens = max_tokens;
    SPMVB_TRY(E->sort.alloc(max_tokens));
    SPMVB_TRY(E->parts.alloc(static_cast<size_t>(ceil_div(max_tokens, kChunk)) * 2 * width * 8));
    *out = E.release();
    return SPMVB_OK;
  });
}

spmvb_status spmvb_embedding_destroy(spmvb_embedding E) {
  clear_error();
  if (E) {
    DeviceGuard g(E->device);
    delete E;
  }
  return SPMVB_OK;
}

spmvb_status spmvb_embedding_lookup(spmvb_embedding E, spmvb_dtype dtype, int32_t count, const int32_t* d_tokens,
                                    double scale, const void* d_table, int64_t ld_table, void* d_out, int64_t ld_out,
                                    void* stream) {
  clear_error();
  if (!E) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null embedding");
  if (!any_float(dtype)) return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype");
  if (count < 0) return fail(SPMVB_ERR_INVALID_ARGUMENT, "negative count");
  if (count == 0) return SPMVB_OK;
  const int dev = E->device;
  const size_t es = dtype_size(dtype);
  const RowSet idx{d_tokens, 1, count, count, 4, "tokens"}, table{d_table, E->rows, ld_table, E->width, es, "table"},
      out{d_out, count, ld_out, E->width, es, "out"};
  DeviceGuard g(dev);
  for (const RowSet* r : {&idx, &table, &out}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* r : {&idx, &table}) SPMVB_TRY(check_apart(out, *r));
  return launch_lookup(dtype, d_tokens, nullptr, count, 1, E->rows, scale, table, out, E->ctx->index_err(),
                       static_cast<cudaStream_t>(stream));
}

spmvb_status spmvb_embedding_lookup_grad(spmvb_embedding E, spmvb_dtype dtype, int32_t count, const int32_t* d_tokens,
                                         double scale, const void* d_dout, int64_t ld_dout, spmvb_dtype grad_dtype,
                                         void* d_dtable, int64_t ld_dtable, int accumulate, void* stream) {
  clear_error();
  if (!E) return fail(SPMVB_ERR_INVALID_ARGUMENT, "null embedding");
  if (!any_float(dtype) || (grad_dtype != dtype && !(grad_dtype == SPMVB_F32 && dtype != SPMVB_F64)))
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype: the gradient has the rows' type or is fp32");
  if (count < 0 || count > E->max_tokens)
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "count must be in [0, max_tokens = " + std::to_string(E->max_tokens) + "]");
  const int dev = E->device;
  const auto s = static_cast<cudaStream_t>(stream);
  const RowSet idx{d_tokens, count > 0, count, count, 4, "tokens"},
      dout{d_dout, count, ld_dout, E->width, dtype_size(dtype), "dout"},
      dtable{d_dtable, E->rows, ld_dtable, E->width, dtype_size(grad_dtype), "dtable"};
  DeviceGuard g(dev);
  for (const RowSet* r : {&idx, &dout, &dtable}) SPMVB_TRY(check_rows(*r, dev));
  for (const RowSet* r : {&idx, &dout}) SPMVB_TRY(check_apart(dtable, *r));
  if (!accumulate)
    SPMVB_TRY_CUDA(cudaMemset2DAsync(d_dtable, ld_dtable * dtable.elem, 0, E->width * dtable.elem, E->rows, s));
  if (count == 0) return SPMVB_OK;
  Sorted sorted{};
  SPMVB_TRY(sort_entries(E->sort, d_tokens, count, E->rows, E->ctx->index_err(), s, &sorted));
  const int vb = access_bytes(dout.elem, {{dout.p, dout.ld}}, E->width);
  return with_type<true>(dtype, vb, [&](auto tv, auto vbc) -> spmvb_status {
    using T = decltype(tv);
    constexpr int VB = decltype(vbc)::value;
    if (grad_dtype == dtype) return lookup_grad<T, T, VB>(E, sorted, count, scale, dout, dtable, accumulate != 0, s);
    if constexpr (sizeof(T) == 2)
      return lookup_grad<T, float, VB>(E, sorted, count, scale, dout, dtable, accumulate != 0, s);
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype");
  });
}

}  // extern "C"
