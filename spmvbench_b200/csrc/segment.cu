// The transposed product of a selection: the stable order of the tokens by the
// row they name, and the embedding gradient made with it.
//
// Order, by the number of tokens:
//   up to kSelfTokens   every block of the gradient ranks all tokens itself: a
//                       token's place is the number of smaller (row, token)
//                       pairs, 0.5 us of comparisons against a launch of 2.5
//   up to kRankTokens   the same ranks, by a kernel of one block per 64 tokens
//   up to kBlockTokens  grouped by a hash of the row (order_tokens), then by
//                       row: the gradient needs equal rows to be neighbours,
//                       not the rows in order
//   more                least-significant-digit radix sort: every tile of
//                       kTile tokens counts its digits (digit_counts), then
//                       ranks its tokens among the equal digits before them
//                       and writes them to their places (digit_scatter),
//                       which adds up the tiles' counts itself up to kOwnTiles
//                       tiles and has them summed by digit_scan beyond.
// Ranks follow the tokens' order, so the order is stable and nothing depends
// on timing.
//
// Gradient. dtable[r] = scale * sum of dout[t] over the tokens that name r:
// in that order the tokens of one row are neighbours (a run). A block takes
// chunks of 16 or 4 tokens and a range of columns and adds each run in
// registers. A run of up to 16 belongs to the chunk where it begins, whole. Of
// a longer one every chunk that holds some leaves its part in scratch (slot 0: the run came
// in from the chunk before, slot 1: it begins here and goes on); the last of
// its blocks to arrive adds the parts in chunk order, of very long runs by groups of
// chunks first. A frequent token is so spread over many blocks, in a fixed order of
// summation. Where the gradient is not added
// to what is there, the rows that no token names are written as well
// (empty_rows), by blocks of their own after those of the sums; which rows are
// named, the sort notes in a bit each. The table is written once, and that bounds the kernels
// (1.07 GB of 1.2 GB for 16,384 tokens of 4,096 bf16 values and 131,072 rows).
#include "select.cuh"

namespace spmvb {

// Scratch of the sort for a number of tokens.
struct SortSpace {
  DevBuf keys[2], vals[2], counts, totals;
  spmvb_status alloc(int64_t tokens);
};
struct Sorted {
  const uint32_t* keys;  // ascending; the number of rows for tokens that select nothing
  const int* entries;    // in token order among equal keys
};

namespace {

constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kPerThread = 4;
constexpr int kTile = kSortThreads * kPerThread;
constexpr int kOwnTiles = 64;
constexpr int kSelfTokens = 256;
constexpr int kGradThreads = 256;
constexpr int kRankTokens = 2048;
constexpr int kBlockTokens = 16384;
constexpr int kOrderThreads = 1024;

// The key of an index that has been loaded. The report comes after all loads
// of a thread: its store would hold the next one back.
__device__ __forceinline__ uint32_t key_of(int i, uint32_t n, int* err) {
  if (i >= 0 && static_cast<uint32_t>(i) >= n) *err = 1;
  return i < 0 || static_cast<uint32_t>(i) >= n ? n : static_cast<uint32_t>(i);
}

// Rows that no token names, a few to a block: pieces of 8 to 64 KB written in
// their order reach 7.4 TB/s, 1 MB a block 6.1.
constexpr int kEmptyRows = 8, kMaxEmptyRows = 256;
struct EmptyRows {
  char* table;           // null: nothing to write
  int64_t pitch, bytes;  // of a row
  int rows, per_block;   // rows of a block: a multiple of kEmptyRows
  bool wide;             // 16 bytes at a time, else `elem`
  int elem;
  uint8_t* named;        // a bit per row, set by the sort; null: look the tokens through
};

__device__ __forceinline__ void name_row(uint32_t* named, uint32_t row, uint32_t rows) {
  if (named && row < rows) atomicOr(named + (row >> 5), 1u << (row & 31));
}

// A block's rows, a warp a row. The bits are cleared for the next call.
__device__ __forceinline__ void empty_rows(const EmptyRows& Z, int block, const int* __restrict__ tokens, int count) {
  __shared__ unsigned bits[kMaxEmptyRows / kEmptyRows];  // 8 rows each
  const int64_t r0 = static_cast<int64_t>(block) * Z.per_block;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, bytes = Z.per_block / kEmptyRows;
  if (static_cast<int>(threadIdx.x) < bytes) {
    const int64_t at = r0 / kEmptyRows + threadIdx.x;
    const bool in = Z.named && at * kEmptyRows < Z.rows;
    bits[threadIdx.x] = in ? Z.named[at] : 0u;
    if (in && bits[threadIdx.x]) Z.named[at] = 0;
  }
  __syncthreads();
  if (!Z.named) {
    for (int i = threadIdx.x; i < count; i += kGradThreads) {
      const int64_t r = __ldg(tokens + i) - r0;
      if (r >= 0 && r < Z.per_block) atomicOr(&bits[r / kEmptyRows], 1u << (r % kEmptyRows));
    }
    __syncthreads();
  }
  for (int q = 0; q < bytes; ++q) {
    const int64_t r = r0 + q * kEmptyRows + w;
    if (r >= Z.rows || (bits[q] >> w & 1u)) continue;
    char* row = Z.table + r * Z.pitch;
    if (Z.wide) {
#pragma unroll 4
      for (int64_t i = lane; i < Z.bytes / 16; i += 32) __stcs(reinterpret_cast<uint4*>(row) + i, make_uint4(0, 0, 0, 0));
    } else if (Z.elem == 2) {
#pragma unroll 4
      for (int64_t i = lane; i < Z.bytes / 2; i += 32) __stcs(reinterpret_cast<uint16_t*>(row) + i, uint16_t(0));
    } else {
#pragma unroll 4
      for (int64_t i = lane; i < Z.bytes / 4; i += 32) __stcs(reinterpret_cast<uint32_t*>(row) + i, 0u);
    }
  }
}
static_assert(kEmptyRows == kGradThreads / 32 && kEmptyRows == 8);

// counts[digit * tiles + tile].
template <bool First>
__global__ void __launch_bounds__(kSortThreads)
    digit_counts(const int* __restrict__ src, int64_t count, uint32_t n, int shift, int tiles, int* __restrict__ counts,
                 uint32_t* __restrict__ named, int* __restrict__ err) {
  __shared__ int c[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) c[d] = 0;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kTile + threadIdx.x;
  int raw[kPerThread];
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) raw[q] = i0 + q * kSortThreads < count ? __ldg(src + i0 + q * kSortThreads) : -1;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) {
    const uint32_t key = First ? key_of(raw[q], n, err) : static_cast<uint32_t>(raw[q]);
    if (i0 + q * kSortThreads < count) {
      atomicAdd(&c[(key >> shift) & (kDigits - 1)], 1);
      if (First) name_row(named, key, n);
    }
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
    digit_scatter(const int* __restrict__ src, const int* __restrict__ src_vals, int64_t count, uint32_t n, int shift,
                  int tiles, bool scanned, const int* __restrict__ counts, const int* __restrict__ totals,
                  uint32_t* __restrict__ dst_keys, int* __restrict__ dst_vals, int* __restrict__ err) {
  __shared__ int wc[kSortWarps][kDigits];  // a warp's count of each digit, then its first place
  __shared__ int sh[kSortWarps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < kSortWarps * kDigits; d += kSortThreads) (&wc[0][0])[d] = 0;
  // A warp's entries are neighbours: 32 * kPerThread of them, in rounds of 32.
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kTile + w * (32 * kPerThread) + lane;
  int raw[kPerThread], val[kPerThread];
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) {
    const int64_t i = i0 + q * 32;
    raw[q] = i < count ? __ldg(src + i) : -1;
    val[q] = First ? static_cast<int>(i) : i < count ? __ldg(src_vals + i) : 0;
  }
  // The digit's entries in the tiles before, and in all.
  int v[2], at_tile[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t row = static_cast<int64_t>(2 * threadIdx.x + h) * tiles;
    if (scanned) {
      v[h] = totals[2 * threadIdx.x + h];
      at_tile[h] = counts[row + blockIdx.x];
    } else {
      v[h] = at_tile[h] = 0;
#pragma unroll 8
      for (int t = 0; t < tiles; ++t) {
        const int c = __ldg(counts + row + t);
        v[h] += c;
        at_tile[h] += t < static_cast<int>(blockIdx.x) ? c : 0;
      }
    }
  }
  __syncthreads();
  uint32_t key[kPerThread];
  int rank[kPerThread];
  unsigned same[kPerThread];
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) {
    key[q] = First ? key_of(raw[q], n, err) : static_cast<uint32_t>(raw[q]);
    // The lanes with the same digit, from one vote a bit.
    same[q] = __ballot_sync(0xffffffffu, i0 + q * 32 < count);
#pragma unroll
    for (int bit = 0; bit < kDigitBits; ++bit) {
      const bool on = key[q] >> (shift + bit) & 1u;
      const unsigned vote = __ballot_sync(0xffffffffu, on);
      same[q] &= on ? vote : ~vote;
    }
  }
#pragma unroll
  for (int q = 0; q < kPerThread; ++q) {
    const bool in = i0 + q * 32 < count;
    const int d = static_cast<int>((key[q] >> shift) & (kDigits - 1));
    const unsigned before = same[q] & ((1u << lane) - 1u);
    const int base = wc[w][d];
    rank[q] = base + __popc(before);
    __syncwarp();
    if (in && before == 0) wc[w][d] = base + __popc(same[q]);
    __syncwarp();
  }
  __syncthreads();
  // First place of each digit: all smaller digits, then this digit in the
  // tiles and the warps before.
  scan_digits(v, sh);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d = 2 * threadIdx.x + h;
    int at = v[h] + at_tile[h];
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
    if (i0 + q * 32 >= count) continue;
    const int at = wc[w][(key[q] >> shift) & (kDigits - 1)] + rank[q];
    dst_keys[at] = key[q];
    dst_vals[at] = val[q];
  }
}

// Place of a (row, token) pair, as one word, among all `count` (padded with
// ones to a multiple of 4): the smaller ones. `each` threads, a power of two
// of neighbours, share the count; all of them get it.
__device__ __forceinline__ int rank_among(uint32_t mine, const uint32_t* pairs, int count, int each, int part) {
  int below = 0;
  const uint4* p = reinterpret_cast<const uint4*>(pairs);
#pragma unroll 4
  for (int i = part; i < (count + 3) / 4; i += each) {
    const uint4 v = p[i];
    below += (v.x < mine) + (v.y < mine) + (v.z < mine) + (v.w < mine);
  }
  for (int off = each / 2; off > 0; off >>= 1) below += __shfl_xor_sync(0xffffffffu, below, off);
  return below;
}

// Sorted keys and tokens by counting: 64 tokens a block, 4 threads a token.
__global__ void __launch_bounds__(256)
    rank_tokens(const int* __restrict__ src, int count, uint32_t n, int token_bits, uint32_t* __restrict__ keys,
                int* __restrict__ vals, uint32_t* __restrict__ named, int* __restrict__ err) {
  __shared__ __align__(16) uint32_t pairs[kRankTokens];
  const int padded = (count + 3) / 4 * 4;
#pragma unroll 4
  for (int i = threadIdx.x; i < padded; i += 256) {
    const int raw = i < count ? __ldg(src + i) : -1;
    const uint32_t key = raw < 0 || static_cast<uint32_t>(raw) >= n ? n : static_cast<uint32_t>(raw);
    pairs[i] = i < count ? key << token_bits | static_cast<uint32_t>(i) : 0xffffffffu;
  }
  __syncthreads();
  const int i = blockIdx.x * 64 + (threadIdx.x >> 2);
  const int at = rank_among(pairs[min(i, count - 1)], pairs, count, 4, threadIdx.x & 3);
  if (i < count && (threadIdx.x & 3) == 0) {
    keys[at] = pairs[i] >> token_bits;
    vals[at] = i;
    name_row(named, key_of(__ldg(src + i), n, err), n);
  }
}

// ---- embedding gradient ----------------------------------------------------------
constexpr int kMinAcross = 8;  // threads along a row, at least

// N values of a row, by accesses of up to 16 bytes; the row is aligned to them.
template <typename G, int N>
struct RowPack {
  static constexpr int VB = N * sizeof(G) > 16 ? 16 : N * static_cast<int>(sizeof(G));
  static constexpr int M = VB / static_cast<int>(sizeof(G));
  Pack<G, VB> p[N / M];
  __device__ __forceinline__ void load(const G* src) {
#pragma unroll
    for (int i = 0; i < N / M; ++i) p[i] = ld_pack_stream<G, VB>(src + i * M);
  }
  __device__ __forceinline__ void store(G* dst) const {
#pragma unroll
    for (int i = 0; i < N / M; ++i) st_pack_stream<G, VB>(dst + i * M, p[i]);
  }
};

// Groups up to kBlockTokens tokens by row: block p < parts (a power of two)
// takes the rows whose hash is p, in the order of the tokens, and sorts them by
// row; its place in the result is the number of tokens of smaller hash. The
// hash spreads the frequent tokens, which have neighbouring numbers.
// Shared memory: keys, 16-bit tokens, 16-bit counts per warp and digit.
constexpr size_t kOrderShared = kBlockTokens * 6 + (kOrderThreads / 32) * kDigits * 2;
constexpr int kRankGroup = 512;  // tokens of a block ranked by counting; more by digits
__global__ void __launch_bounds__(kOrderThreads)
    order_tokens(const int* __restrict__ src, int count, uint32_t n, int bits, int parts, int hash_shift,
                 uint32_t* __restrict__ keys, int* __restrict__ vals, uint32_t* __restrict__ named, int* __restrict__ err) {
  extern __shared__ __align__(16) uint32_t shared[];
  const int part = blockIdx.x;
  constexpr int Warps = kOrderThreads / 32, Rounds = kBlockTokens / kOrderThreads;
  uint32_t* sk = shared;
  uint16_t* sv = reinterpret_cast<uint16_t*>(shared + kBlockTokens);
  uint16_t* wc = sv + kBlockTokens;
  __shared__ int sh[kDigits / 32], found[3][Warps];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const unsigned before_me = (1u << lane) - 1u;
  uint32_t key[Rounds], place[Rounds];  // place: token << 16 | rank
  int m;  // tokens of this block
  {
    const int turns = (count + kOrderThreads - 1) / kOrderThreads;  // of 32 tokens a warp, neighbours
    const int i0 = w * turns * 32 + lane;
#pragma unroll
    for (int q = 0; q < Rounds; ++q)
      key[q] = q < turns && i0 + q * 32 < count ? static_cast<uint32_t>(__ldg(src + i0 + q * 32)) : 0xffffffffu;
    unsigned mine = 0, less = 0;  // a bit a turn
    int all = 0;
#pragma unroll
    for (int q = 0; q < Rounds; ++q) {
      const bool in = key[q] < n;
      const int hash = static_cast<int>(key[q] * 2654435761u >> hash_shift);
      mine |= static_cast<unsigned>(in && hash == part) << q;
      less |= static_cast<unsigned>(in && hash < part) << q;
      all += in;
    }
    if (part == 0)
      for (int q = 0; q < Rounds; ++q) key_of(static_cast<int>(key[q]), n, err);  // reports an index past the end
    const int own_w = __reduce_add_sync(0xffffffffu, __popc(mine)), less_w = __reduce_add_sync(0xffffffffu, __popc(less)),
              all_w = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) {
      found[0][w] = own_w;
      found[1][w] = less_w;
      found[2][w] = all_w;
    }
    __syncthreads();
    int incl = found[0][lane], offset = found[1][lane];
    const int here = incl;
    all = found[2][lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += u;
      offset += __shfl_xor_sync(0xffffffffu, offset, off);
      all += __shfl_xor_sync(0xffffffffu, all, off);
    }
    m = __shfl_sync(0xffffffffu, incl, 31);
    int at = __shfl_sync(0xffffffffu, incl - here, w);
#pragma unroll
    for (int q = 0; q < Rounds; ++q) {
      if (q >= turns) break;
      const bool in = mine >> q & 1u;
      const unsigned vote = __ballot_sync(0xffffffffu, in);
      if (in) {
        name_row(named, key[q], n);
        sk[at + __popc(vote & before_me)] = key[q];
        sv[at + __popc(vote & before_me)] = static_cast<uint16_t>(i0 + q * 32);
      }
      at += __popc(vote);
    }
    keys += offset;
    vals += offset;
    // The tokens that select nothing come after all others.
    if (part == parts - 1)
      for (int i = all + threadIdx.x; i < count; i += kOrderThreads) {
        keys[i - offset] = n;
        vals[i - offset] = 0;
      }
    __syncthreads();
  }
  const int rounds = (m + kOrderThreads - 1) / kOrderThreads;
  const int i0 = w * rounds * 32 + lane;
  // A few tokens are ranked by counting. Of many, the tokens of one row are
  // taken out first, the most frequent of 32: they are in order already, and
  // where few others are left (as in text, whose commonest token alone is a
  // tenth) those are ranked by counting and step over them: the gradient of
  // 16,384 tokens added to 32,003 rows of 1,001 bf16 values takes 35 us, 39 us
  // with the passes by digits below.
  if (bits <= 23) {
    uint32_t* pairs = reinterpret_cast<uint32_t*>(wc);  // row << 9 | place in the list
    uint16_t* token = reinterpret_cast<uint16_t*>(pairs + kRankGroup + 4);
    int others = m, less = 0;  // and how many of them are of rows before the frequent one
    uint32_t frequent = 0xffffffffu;
    if (m > kRankGroup) {
      const uint32_t sample = sk[lane * m / 32];
      const int same = __popc(__match_any_sync(0xffffffffu, sample));
      const int most = __reduce_max_sync(0xffffffffu, same << 5 | lane);
      frequent = __shfl_sync(0xffffffffu, sample, most & 31);
      int other_w = 0, less_w = 0;
      for (int q = 0; q < rounds; ++q) {
        const bool in = i0 + q * 32 < m;
        const uint32_t own = in ? sk[i0 + q * 32] : frequent;
        other_w += __popc(__ballot_sync(0xffffffffu, own != frequent));
        less_w += __popc(__ballot_sync(0xffffffffu, own < frequent));
      }
      if (lane == 0) {
        found[0][w] = other_w;
        found[1][w] = less_w;
      }
      __syncthreads();
      int incl = found[0][lane];
      const int here = incl;
      less = found[1][lane];
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += u;
        less += __shfl_xor_sync(0xffffffffu, less, off);
      }
      others = __shfl_sync(0xffffffffu, incl, 31);
      int at = __shfl_sync(0xffffffffu, incl - here, w);
      if (others <= kRankGroup) {
        for (int q = 0; q < rounds; ++q) {
          const int i = i0 + q * 32;
          const uint32_t own = i < m ? sk[i] : frequent;
          const unsigned vote = __ballot_sync(0xffffffffu, own != frequent);
          const int to = at + __popc(vote & before_me);
          if (own != frequent) {
            pairs[to] = own << 9 | static_cast<uint32_t>(to);
            token[to] = sv[i];
          } else if (i < m) {
            keys[less + i - to] = frequent;
            vals[less + i - to] = sv[i];
          }
          at += __popc(vote);
        }
      }
    } else if (static_cast<int>(threadIdx.x) < m) {
      pairs[threadIdx.x] = sk[threadIdx.x] << 9 | threadIdx.x;
      token[threadIdx.x] = sv[threadIdx.x];
    }
    if (others <= kRankGroup) {
      if (threadIdx.x < 4) pairs[others + threadIdx.x] = 0xffffffffu;
      __syncthreads();
      if (others == 0) return;
      int each = 2;  // threads of a token
      while (each < 32 && others * each * 2 <= kOrderThreads) each *= 2;
      const int i = threadIdx.x / each;
      const uint32_t own = pairs[min(i, others - 1)];
      int at = rank_among(own, pairs, others, each, threadIdx.x % each);
      if (i < others && threadIdx.x % each == 0) {
        if (own >> 9 > frequent) at += m - others;
        keys[at] = own >> 9;
        vals[at] = token[i];
      }
      return;
    }
  }
  for (int shift = 0; shift < bits; shift += kDigitBits) {
    uint32_t* zero = reinterpret_cast<uint32_t*>(wc);
    for (int i = threadIdx.x; i < Warps * kDigits / 2; i += kOrderThreads) zero[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Rounds; ++q) {
      const bool in = q < rounds && i0 + q * 32 < m;
      key[q] = in ? sk[i0 + q * 32] : 0u;
      place[q] = in ? static_cast<uint32_t>(sv[i0 + q * 32]) << 16 : 0u;
    }
    uint16_t* mine = wc + w * kDigits;
#pragma unroll
    for (int q = 0; q < Rounds; ++q) {
      if (q >= rounds) break;
      // The lanes with the same digit, from one vote a bit.
      const bool in = i0 + q * 32 < m;
      unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
      for (int bit = 0; bit < kDigitBits; ++bit) {
        const bool on = key[q] >> (shift + bit) & 1u;
        const unsigned vote = __ballot_sync(0xffffffffu, on);
        same &= on ? vote : ~vote;
      }
      const int d = static_cast<int>((key[q] >> shift) & (kDigits - 1));
      const unsigned before = same & before_me;
      const int base = mine[d];
      __syncwarp();
      if (in && before == 0) mine[d] = static_cast<uint16_t>(base + __popc(same));
      place[q] = (place[q] & 0xffff0000u) | static_cast<uint32_t>(base + __popc(before));
      __syncwarp();
    }
    __syncthreads();
    // First place of each digit and warp.
    int all = 0, incl = 0;
    const int d = threadIdx.x;
    if (d < kDigits) {
#pragma unroll 8
      for (int i = 0; i < Warps; ++i) all += wc[i * kDigits + d];
      incl = all;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += u;
      }
      if (lane == 31) sh[w] = incl;
    }
    __syncthreads();
    if (d < kDigits) {
      int at = incl - all;
      for (int i = 0; i < w; ++i) at += sh[i];
#pragma unroll 8
      for (int i = 0; i < Warps; ++i) {
        const int c = wc[i * kDigits + d];
        wc[i * kDigits + d] = static_cast<uint16_t>(at);
        at += c;
      }
    }
    __syncthreads();
    const bool last = shift + kDigitBits >= bits;
#pragma unroll
    for (int q = 0; q < Rounds; ++q) {
      if (q >= rounds || i0 + q * 32 >= m) continue;
      const int at = mine[(key[q] >> shift) & (kDigits - 1)] + static_cast<int>(place[q] & 0xffffu);
      if (last) {
        keys[at] = key[q];
        vals[at] = static_cast<int>(place[q] >> 16);
      } else {
        sk[at] = key[q];
        sv[at] = static_cast<uint16_t>(place[q] >> 16);
      }
    }
    __syncthreads();
  }
}

struct GradView {
  const uint32_t* keys;  // sorted (unless the block sorts)
  const int* vals;
  const int* tokens;
  int count;
  uint32_t rows;
  int chunks, chunk_blocks;   // blocks of chunks, times `ranges` of columns
  int ranges, empty_blocks;   // the grid's other blocks write empty rows
  int width, packs, across;   // columns, packs of them, threads along a row
  int64_t ldo, ldt;
  void* parts;
  unsigned* tickets;  // 3 a chunk and range, all 0 between calls
  EmptyRows empty;
  int* err;
};

// Chunks from `from` on, in steps of `dir`, whose edge towards it continues
// the run of `key`: steps that double, then halve.
template <int Chunk>
__device__ __forceinline__ int run_reach(const uint32_t* keys, int count, uint32_t key, int from, int dir) {
  const auto on = [&](int steps) {  // does the run still hold `steps` chunks on?
    const int64_t q = from + static_cast<int64_t>(dir) * steps;
    const int64_t i = dir > 0 ? q * Chunk : (q + 1) * Chunk - 1;
    return q >= 0 && i < count && keys[i] == key;
  };
  int have = 0, step = 1;
  while (on(have + step)) {
    have += step;
    step *= 2;
  }
  for (step /= 2; step > 0; step /= 2)
    if (on(have + step)) have += step;
  return have;
}

// Tokens of a chunk: few where they would not fill the GPU.
constexpr int kChunk = 16, kSmallChunk = 4;
// A longer run is added in parts.
constexpr int kLongRun = 16;
constexpr int kJoin = 16;  // chunks in a group, where the parts of a run are added by groups:
constexpr int kJoinInGroups = 48;  // in runs that go on for so many chunks

// Parts that a block adds: chunk * 2 + slot of the first and of the next, the
// number after the first, and the groups besides this one that follow.
struct Join {
  int from, next, more, head, groups;
};

// Packs of a thread, `across` packs apart: 16 bytes in all, 4 packs at most.
constexpr int packs_of(int bytes) { return bytes >= 16 ? 1 : 16 / bytes > 4 ? 4 : 16 / bytes; }

// Wide: a block's threads lie along one row.
template <typename T, typename G, int N, int Chunk, bool Self, bool Add, bool Wide>
__global__ void __launch_bounds__(kGradThreads, sizeof(T) == 8 || (Add && N * sizeof(G) > 16) ? 2 : N * sizeof(T) < 16 ? 3 : 4)
    grad_rows(GradView A, const T* __restrict__ dout, typename AccOf<T>::type scale, G* __restrict__ dtable) {
  using Acc = typename AccOf<T>::type;
  constexpr int VB = N * sizeof(T), M = packs_of(VB);
  constexpr int Batch = 4;  // rows loaded before the first is added
  constexpr int Span = Chunk + 2 * kLongRun;
  constexpr int MaxDown = kGradThreads / kMinAcross;
  __shared__ __align__(16) uint32_t pairs[Self ? kSelfTokens : 4];
  __shared__ uint32_t self_keys[Self ? kSelfTokens : 1];
  __shared__ int self_vals[Self ? kSelfTokens : 1];
  __shared__ uint32_t ck[MaxDown * Span];
  __shared__ int cv[MaxDown * Span];
  __shared__ Join joined[MaxDown][2];  // by slot: what is to be added now
  const uint32_t* keys = A.keys;
  const int* vals = A.vals;
  // The blocks that write empty rows come last: their writes run at full rate
  // in order, and slow down the loads of the others (238 us against 207 where
  // they were spread among them).
  const int block = static_cast<int>(blockIdx.x), sums = static_cast<int>(gridDim.x) - A.empty_blocks;
  if (block >= sums) {
    empty_rows(A.empty, block - sums, A.tokens, A.count);
    return;
  }
  const int range = block % A.ranges, block_x = block / A.ranges;
  if constexpr (Self) {
    // Rows have at most 23 bits, tokens 8.
    const int padded = (A.count + 3) / 4 * 4;
    for (int i = threadIdx.x; i < padded; i += kGradThreads)
      pairs[i] = i < A.count ? key_of(__ldg(A.tokens + i), A.rows, A.err) << 8 | static_cast<uint32_t>(i) : 0xffffffffu;
    __syncthreads();
    int each = 1;  // threads of a token
    while (each < 32 && A.count * each * 2 <= kGradThreads) each *= 2;
    const int i = threadIdx.x / each;
    const int at = rank_among(pairs[min(i, A.count - 1)], pairs, A.count, each, threadIdx.x % each);
    if (i < A.count && threadIdx.x % each == 0) {
      self_keys[at] = pairs[i] >> 8;
      self_vals[at] = i;
    }
    __syncthreads();
    keys = self_keys;
    vals = self_vals;
  }

  // A chunk's keys and tokens, with kLongRun before and after it.
  const int down = Wide ? 1 : kGradThreads / A.across;
  const int x = Wide ? threadIdx.x : threadIdx.x % A.across, y = Wide ? 0 : threadIdx.x / A.across;
  for (int i = threadIdx.x; i < down * Span; i += kGradThreads) {
    const int64_t at = (static_cast<int64_t>(block_x) * down + i / Span) * Chunk + i % Span - kLongRun;
    const bool in = at >= 0 && at < A.count;
    ck[i] = in ? keys[at] : 0xffffffffu;
    cv[i] = in ? vals[at] : 0;
  }
  __syncthreads();
  const int chunk = block_x * down + y, v0 = range * A.across * M + x;
  const uint32_t* k = ck + y * Span + kLongRun;
  const int* t = cv + y * Span + kLongRun;
  Acc* parts = static_cast<Acc*>(A.parts);
  const bool mine = chunk < A.chunks;
  // The runs that cross the chunk's edges: [first_begin, first_end) and
  // [last_begin, last_end), as far as they are in view. Tokens that select
  // nothing (key = rows) and places past the end (~0) are no runs.
  bool came_in = k[0] < A.rows && k[-1] == k[0];
  bool goes_on = k[Chunk - 1] < A.rows && k[Chunk] == k[Chunk - 1];
  int begin = 0, end = Chunk;
  if (came_in) {
    int from = -1, to = 1;
    while (from > -kLongRun && k[from - 1] == k[0]) --from;
    while (to < Chunk + kLongRun && k[to] == k[0]) ++to;
    if (to - from <= kLongRun) {  // short: the chunk where it begins adds it
      came_in = false;
      begin = to;
    }
  }
  const bool through = came_in && k[0] == k[Chunk - 1];
  if (goes_on) {
    int from = Chunk - 1, to = Chunk + 1;
    while (from > -kLongRun && k[from - 1] == k[Chunk - 1]) --from;
    while (to < Chunk + kLongRun && k[to] == k[Chunk - 1]) ++to;
    if (to - from <= kLongRun) {
      goes_on = false;
      end = from < 0 ? Chunk : to;
    }
  }
  bool in_first = came_in;
  const int across = Wide ? kGradThreads : A.across;
  const int64_t c0 = static_cast<int64_t>(v0) * N;
  const T* const dout_c = dout + c0;  // this thread's first column; the others lie m * across * N on
  G* const dtable_c = dtable + c0;
  if (mine) {
    Acc sum[M][N] = {};
#pragma unroll 1
    for (int b = begin; b < end; b += Batch) {
      Pack<T, VB> p[Batch][M];
      RowPack<G, N> old[Add ? Batch : 1][M];
      uint32_t key[Batch];
      bool done[Batch];  // the run ends with this token
#pragma unroll
      for (int q = 0; q < Batch; ++q) {
        const int i = b + q;
        key[q] = i < end ? k[i] : 0xffffffffu;
        done[q] = i + 1 >= end || k[i + 1] != key[q];
        if (key[q] >= A.rows) continue;
        const T* from = dout_c + t[i] * A.ldo;
#pragma unroll
        for (int m = 0; m < M; ++m)
          if (v0 + m * across < A.packs) p[q][m] = ld_pack_stream<T, VB>(from + m * across * N);
        if (Add && done[q]) {
          const G* was = dtable_c + key[q] * A.ldt;
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (v0 + m * across < A.packs) old[Add ? q : 0][m].load(was + m * across * N);
        }
      }
#pragma unroll
      for (int q = 0; q < Batch; ++q) {
        if (key[q] >= A.rows) continue;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int n = 0; n < N; ++n) sum[m][n] += widen(p[q][m].v[n]);
        if (!done[q]) continue;
        if (in_first || (b + q == Chunk - 1 && goes_on)) {
          Acc* to = parts + (static_cast<int64_t>(chunk) * 2 + (in_first ? 0 : 1)) * A.width + c0;
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (v0 + m * across < A.packs) {
#pragma unroll
              for (int n = 0; n < N; ++n) __stcg(to + m * across * N + n, sum[m][n]);
            }
          __threadfence();
        } else {
          G* row = dtable_c + key[q] * A.ldt;
#pragma unroll
          for (int m = 0; m < M; ++m) {
            if (v0 + m * across >= A.packs) continue;
            constexpr int W = RowPack<G, N>::M;
            RowPack<G, N> o;
#pragma unroll
            for (int n = 0; n < N; ++n) {
              Acc r = sum[m][n] * scale;
              if (Add) r += widen(old[Add ? q : 0][m].p[n / W].v[n % W]);
              o.p[n / W].v[n % W] = narrow<G, Acc>(r);
            }
            o.store(row + m * across * N);
          }
        }
        in_first = false;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int n = 0; n < N; ++n) sum[m][n] = 0;
      }
    }
  }
  if (!__syncthreads_or(mine && (came_in || goes_on))) return;
  // Slot 0 is the run that came in, slot 1 one that begins here and goes on.
  // The last block of a run to arrive adds its parts. In a run of
  // kJoinInGroups chunks and more the last of each kJoin neighbours adds
  // theirs, and the last of these the sums: a token that is all of 16,384 is a
  // chain of 16 + 64 parts, not of 1,024. 16,384 tokens of 3,000 rows of 256 bf16
  // values: 65 us with one chain, 38 us so. From 16 chunks on the second ticket
  // costs 2 us at 5,003 tokens of 1,001 values; from 128 on 5,000 tokens of 256
  // take 31 us, not 25.
  unsigned* tickets = A.tickets + range;  // (chunk * 3 + which) * ranges on
  if (x < 2 && mine) {
    Join j;
    j.from = -1;
    if (x == 0 ? came_in : goes_on && !through) {
      const uint32_t key = x == 0 ? k[0] : k[Chunk - 1];
      const int head = x == 0 ? chunk - run_reach<Chunk>(keys, A.count, key, chunk, -1) : chunk;
      const int tail = x == 0 && !(through && goes_on) ? chunk : chunk + run_reach<Chunk>(keys, A.count, key, chunk, 1);
      const bool grouped = tail - head >= kJoinInGroups;
      const int first = grouped ? max(head, chunk / kJoin * kJoin) : head;
      const int last = grouped ? min(tail, chunk / kJoin * kJoin + kJoin - 1) : tail;
      unsigned* ticket = tickets + (static_cast<int64_t>(first) * 3 + (first == head)) * A.ranges;
      __threadfence();
      if (atomicAdd(ticket, 1u) == static_cast<unsigned>(last - first)) {
        *ticket = 0u;
        __threadfence();
        j.from = first * 2 + (first == head);
        j.next = first * 2 + 2;
        j.more = last - first;
        j.head = head;
        j.groups = grouped ? tail / kJoin - head / kJoin : 0;
      }
    }
    joined[y][x] = j;
  }
  __syncthreads();
  // Several parts' loads in flight: a frequent token's are the longest chain of
  // the kernel.
  constexpr int kAhead = 4;
  constexpr int W = RowPack<G, N>::M;
  int step = 2;
#pragma unroll 1
  for (;;) {
    bool on = false;  // a sum that waits for those of other groups
#pragma unroll 1
    for (int slot = 0; mine && slot < 2; ++slot) {
      const Join j = joined[y][slot];
      if (j.from < 0) continue;
      G* row = dtable_c + (slot == 0 ? k[0] : k[Chunk - 1]) * A.ldt;
      RowPack<G, N> o[M];
      Acc sum[M][N];
      Acc* from = parts + static_cast<int64_t>(j.from) * A.width + c0;
#pragma unroll
      for (int m = 0; m < M; ++m)
        if (v0 + m * across < A.packs) {
          if (Add && j.groups == 0) o[m].load(row + m * across * N);
#pragma unroll
          for (int n = 0; n < N; ++n) sum[m][n] = ld_written(from + m * across * N + n);
        }
      const Acc* next = parts + static_cast<int64_t>(j.next) * A.width + c0;
      for (int q = 0; q < j.more; q += kAhead, next += static_cast<int64_t>(kAhead * step) * A.width) {
        Acc part[kAhead][M][N];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (q + u < j.more && v0 + m * across < A.packs) {
#pragma unroll
              for (int n = 0; n < N; ++n)
                part[u][m][n] = ld_written(next + static_cast<int64_t>(u * step) * A.width + m * across * N + n);
            }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (q + u < j.more) {
#pragma unroll
              for (int n = 0; n < N; ++n) sum[m][n] += part[u][m][n];
            }
      }
      if (j.groups > 0) {
#pragma unroll
        for (int m = 0; m < M; ++m)
          if (v0 + m * across < A.packs) {
#pragma unroll
            for (int n = 0; n < N; ++n) __stcg(from + m * across * N + n, sum[m][n]);
          }
        __threadfence();
        on = true;
        continue;
      }
#pragma unroll
      for (int m = 0; m < M; ++m) {
        if (v0 + m * across >= A.packs) continue;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          Acc r = sum[m][n] * scale;
          if (Add) r += widen(o[m].p[n / W].v[n % W]);
          o[m].p[n / W].v[n % W] = narrow<G, Acc>(r);
        }
        o[m].store(row + m * across * N);
      }
    }
    if (!__syncthreads_or(on)) return;
    if (x < 2 && mine) {
      Join j = joined[y][x];
      const bool waits = j.from >= 0 && j.groups > 0;
      j.from = -1;
      if (waits) {
        unsigned* ticket = tickets + (static_cast<int64_t>(j.head) * 3 + 2) * A.ranges;
        __threadfence();
        if (atomicAdd(ticket, 1u) == static_cast<unsigned>(j.groups)) {
          *ticket = 0u;
          __threadfence();
          j.from = j.head * 2 + 1;
          j.next = (j.head / kJoin + 1) * kJoin * 2;
          j.more = j.groups;
          j.groups = 0;
        }
      }
      joined[y][x] = j;
    }
    step = 2 * kJoin;
    __syncthreads();
  }
}

int bits_of(uint64_t v) {
  int b = 0;
  while (v >> b) ++b;
  return b;
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
  return SPMVB_OK;
}

namespace {

// Sorts the tokens by row: idx[i] where it is in [0, n), else n (an index past
// the end is reported in *err). `named` (or null) receives the rows' bits.
spmvb_status order_tokens_by_row(SortSpace& space, const int* idx, int count, int n, uint32_t* named, int* err,
                                 cudaStream_t s, Sorted* out) {
  const int bits = std::max(1, bits_of(n)), token_bits = bits_of(count - 1);
  uint32_t* keys0 = space.keys[0].as<uint32_t>();
  int* vals0 = space.vals[0].as<int>();
  out->keys = keys0;
  out->entries = vals0;
  const bool ranked = count <= kRankTokens && bits + token_bits <= 32;
  if (count <= kBlockTokens && !ranked) {
    // About 128 tokens a block.
    int parts_log = 1;
    while (parts_log < 7 && (128 << parts_log) < count) ++parts_log;
    order_tokens<<<1 << parts_log, kOrderThreads, kOrderShared, s>>>(idx, count, n, bits, 1 << parts_log, 32 - parts_log,
                                                                    keys0, vals0, named, err);
    count_launch();
    SPMVB_TRY_CUDA(cudaGetLastError());
    return SPMVB_OK;
  }
  if (ranked) {
    rank_tokens<<<static_cast<int>(ceil_div(count, 64)), 256, 0, s>>>(idx, count, n, token_bits, keys0, vals0, named, err);
    count_launch();
    SPMVB_TRY_CUDA(cudaGetLastError());
    return SPMVB_OK;
  }
  const int tiles = static_cast<int>(ceil_div(count, kTile));
  const bool scanned = tiles > kOwnTiles;
  int* counts = space.counts.as<int>();
  int* totals = space.totals.as<int>();
  int at = 0;
  for (int shift = 0; shift < bits; shift += kDigitBits, at ^= 1) {
    const bool first = shift == 0;
    const int* src = first ? idx : space.keys[at ^ 1].as<int>();
    const int* vals = space.vals[at ^ 1].as<int>();
    uint32_t* dk = space.keys[at].as<uint32_t>();
    int* dv = space.vals[at].as<int>();
    const auto count_kernel = first ? digit_counts<true> : digit_counts<false>;
    const auto scatter_kernel = first ? digit_scatter<true> : digit_scatter<false>;
    count_kernel<<<tiles, kSortThreads, 0, s>>>(src, count, n, shift, tiles, counts, named, err);
    if (scanned) digit_scan<<<kDigits / 8, 256, 0, s>>>(counts, tiles, totals);
    scatter_kernel<<<tiles, kSortThreads, 0, s>>>(src, vals, count, n, shift, tiles, scanned, counts, totals, dk, dv, err);
    count_launch(scanned ? 3 : 2);
    out->keys = dk;
    out->entries = dv;
  }
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

}  // namespace
}  // namespace spmvb

struct spmvb_embedding_st {
  spmvb::ContextRef ctx;
  int device = 0, rows = 0, width = 0, max_tokens = 0;
  int64_t chunks = 0;  // that parts and tickets are for
  spmvb::SortSpace sort;
  spmvb::DevBuf parts;    // 2 rows of sums (fp64 wide) per chunk
  spmvb::DevBuf tickets;  // 3 per chunk and column range, 0 between calls
  spmvb::DevBuf named;    // a bit per row, 0 between calls
};

using namespace spmvb;

namespace {

template <typename T, typename G, int N>
spmvb_status lookup_grad(spmvb_embedding E, const Sorted& sorted, EmptyRows Z, const int* tokens, int count, double scale,
                         const RowSet& dout, const RowSet& dtable, bool accumulate, cudaStream_t s) {
  using Acc = typename AccOf<T>::type;
  constexpr int M = packs_of(N * sizeof(T));
  const bool self = !sorted.keys;
  GradView A{};
  A.keys = sorted.keys;
  A.vals = sorted.entries;
  A.tokens = tokens;
  A.count = count;
  A.rows = E->rows;
  A.width = E->width;
  A.packs = E->width / N;
  A.across = kMinAcross;
  while (A.across * M < A.packs && A.across < kGradThreads) A.across *= 2;
  A.ranges = static_cast<int>(ceil_div(A.packs, A.across * M));
  const int64_t down = kGradThreads / A.across;
  // Small chunks where large ones leave the SMs short of blocks.
  const bool small = self || ceil_div(ceil_div(count, kChunk), down) * A.ranges < E->ctx->sm_count;
  A.chunks = static_cast<int>(ceil_div(count, small ? kSmallChunk : kChunk));
  if (A.chunks > E->chunks) return fail(SPMVB_ERR_UNSUPPORTED, "the handle's scratch does not hold the chunks");
  A.chunk_blocks = static_cast<int>(ceil_div(A.chunks, down));
  A.ldo = dout.ld;
  A.ldt = dtable.ld;
  A.parts = E->parts.get();
  A.tickets = E->tickets.as<unsigned>();
  A.err = E->ctx->index_err();
  A.empty_blocks = Z.table ? static_cast<int>(ceil_div(Z.rows, Z.per_block)) : 0;
  A.empty = Z;
  const int64_t blocks = static_cast<int64_t>(A.chunk_blocks) * A.ranges + A.empty_blocks;
  if (blocks == 0) return SPMVB_OK;
  if (blocks > INT32_MAX) return fail(SPMVB_ERR_UNSUPPORTED, "too many tokens for one launch");
  const auto pick = [&](auto add, auto wide) {
    constexpr bool Add = decltype(add)::value, Wide = decltype(wide)::value;
    return self    ? grad_rows<T, G, N, kSmallChunk, true, Add, Wide>
           : small ? grad_rows<T, G, N, kSmallChunk, false, Add, Wide>
                   : grad_rows<T, G, N, kChunk, false, Add, Wide>;
  };
  const bool wide = A.across == kGradThreads;
  const auto kernel = accumulate ? (wide ? pick(std::true_type{}, std::true_type{}) : pick(std::true_type{}, std::false_type{}))
                                 : (wide ? pick(std::false_type{}, std::true_type{}) : pick(std::false_type{}, std::false_type{}));
  kernel<<<static_cast<unsigned>(blocks), kGradThreads, 0, s>>>(A, static_cast<const T*>(dout.p), Acc(scale),
                                                                static_cast<G*>(const_cast<void*>(dtable.p)));
  count_launch();
  SPMVB_TRY_CUDA(cudaGetLastError());
  return SPMVB_OK;
}

// Calls lookup_grad for the values of a pack that both row sets allow.
template <typename T, typename G>
spmvb_status lookup_grad_by_pack(int n, spmvb_embedding E, const Sorted& sorted, const EmptyRows& Z, const int* tokens,
                                 int count, double scale, const RowSet& dout, const RowSet& dtable, bool accumulate,
                                 cudaStream_t s) {
  switch (n) {
    case 8:
      if constexpr (sizeof(T) == 2) return lookup_grad<T, G, 8>(E, sorted, Z, tokens, count, scale, dout, dtable, accumulate, s);
      break;
    case 4:
      if constexpr (sizeof(T) <= 4) return lookup_grad<T, G, 4>(E, sorted, Z, tokens, count, scale, dout, dtable, accumulate, s);
      break;
    case 2: return lookup_grad<T, G, 2>(E, sorted, Z, tokens, count, scale, dout, dtable, accumulate, s);
    case 1: return lookup_grad<T, G, 1>(E, sorted, Z, tokens, count, scale, dout, dtable, accumulate, s);
  }
  return fail(SPMVB_ERR_INVALID_ARGUMENT, "row not aligned to its elements");
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
    E->ctx.hold(ctx);
    E->device = ctx->device;
    E->rows = rows;
    E->width = width;
    E->max_tokens = max_tokens;
    SPMVB_TRY(E->sort.alloc(max_tokens));
    SPMVB_TRY(E->named.alloc(static_cast<size_t>(ceil_div(rows, 32)) * 4));
    SPMVB_TRY_CUDA(cudaFuncSetAttribute(order_tokens, cudaFuncAttributeMaxDynamicSharedMemorySize, kOrderShared));
    // Small chunks are taken up to the tokens that large ones would not make
    // enough blocks of: with the fewest threads along a row (8 values each).
    int across = kMinAcross;
    while (across * 8 < width && across < kGradThreads) across *= 2;
    const int64_t few = std::max<int64_t>(kSelfTokens, int64_t(ctx->sm_count) * kChunk * (kGradThreads / across));
    E->chunks = std::max(ceil_div(max_tokens, kChunk), ceil_div(std::min<int64_t>(max_tokens, few), kSmallChunk));
    const size_t chunks = static_cast<size_t>(E->chunks);
    SPMVB_TRY(E->parts.alloc(chunks * 2 * width * 8));
    SPMVB_TRY(E->tickets.alloc(chunks * 3 * ceil_div(width, kGradThreads) * 4));
    SPMVB_TRY(scratch_ready());
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
  return launch_lookup(dtype, d_tokens, count, scale, table, out, E->ctx->index_err(), static_cast<cudaStream_t>(stream));
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
  EmptyRows Z{};
  if (!accumulate) {
    Z.table = static_cast<char*>(d_dtable);
    Z.pitch = ld_dtable * static_cast<int64_t>(dtable.elem);
    Z.bytes = E->width * static_cast<int64_t>(dtable.elem);
    Z.rows = E->rows;
    Z.per_block = kEmptyRows * static_cast<int>(std::min<int64_t>(kMaxEmptyRows / kEmptyRows, std::max<int64_t>(1, 4096 / Z.bytes)));
    Z.wide = access_bytes(dtable.elem, {{dtable.p, dtable.ld}}, E->width) == 16;
    Z.elem = dtable.elem == 2 ? 2 : 4;
  }
  Sorted sorted{};  // no keys: the kernel sorts
  if (count > kSelfTokens || (count > 0 && E->rows >= (1 << 23)))
    SPMVB_TRY(order_tokens_by_row(E->sort, d_tokens, count, E->rows, Z.table ? E->named.as<uint32_t>() : nullptr,
                                  E->ctx->index_err(), s, &sorted));
  if (sorted.keys) Z.named = E->named.as<uint8_t>();
  // Values of a pack: dout's rows allow one access for them, dtable's 16-byte
  // accesses or one.
  int n = access_bytes(dout.elem, {{dout.p, dout.ld}}, E->width) / static_cast<int>(dout.elem);
  const int vg = access_bytes(dtable.elem, {{dtable.p, dtable.ld}}, E->width);
  if (vg < 16) n = std::min(n, vg / static_cast<int>(dtable.elem));
  const bool add = accumulate != 0;
  const auto run = [&](auto tv) -> spmvb_status {
    using T = decltype(tv);
    if (grad_dtype == dtype) return lookup_grad_by_pack<T, T>(n, E, sorted, Z, d_tokens, count, scale, dout, dtable, add, s);
    if constexpr (sizeof(T) == 2)
      return lookup_grad_by_pack<T, float>(n, E, sorted, Z, d_tokens, count, scale, dout, dtable, add, s);
    return fail(SPMVB_ERR_INVALID_ARGUMENT, "bad dtype");
  };
  switch (dtype) {
    case SPMVB_F32: return run(float{});
    case SPMVB_F64: return run(double{});
    case SPMVB_F16: return run(__half{});
    default: return run(__nv_bfloat16{});
  }
}

}  // extern "C"
