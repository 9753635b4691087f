// Embedding lookup with scaling, and the dense gradient of its table.
//
//   out[i] = T(scale * table[id_i])
//   dtable[v] = T(scale * sum over i with id_i = v of dout[i]),  0 for padding and unused rows
//
// The gradient sorts the tokens by id (stably), so that the rows of one id lie together and
// their fp32 sum is taken in an order that depends on the ids alone: no floating-point
// atomics, the same bits on every call.  Up to kFewTokens one launch does all of it (few).
// Otherwise:
//
//   rank   (up to kRankTokens) each token's place by comparing its id with all others;
//   sort, merge  (more) ranges sorted in LDS, then each token's place by binary searches, runs of
//          16384 tokens first and then several runs to one;
//          the first of these launches also writes the zeros of dtable, which for a
//          vocabulary is most of the bytes;
//   sum    kTile sorted tokens per group of lanes; an id whose tokens all lie in the tile is
//          written, one that crosses a tile's edge leaves an fp32 partial row;
//   join   the partial rows of ids that cross edges, added in order.
//
// Bound by bytes where the table is large: 16384 tokens (frequencies ~ 1 / id) into 128100 x 768
// bf16 take 44 us of kernels (sort 15.8, merge 12.6, sum 11.9, join 4.0; 52 with the gaps between
// the launches), of which the 197 MB of zeros alone would take 30 (6.6 TB/s); by latency where it
// is small: 512 x 1024 fp32 37 us (sort 11.0, merge 8.1, sum 14.2 for 67 MB, join 3.9), 4096
// tokens into 5000 x 64 19 us.  The lookup of 16384 rows of 768 bf16 takes 10.8 us.  (Device times
// of single launches, traced; whole gradients, here and below, are timed by events around many in
// a row, where a launch overlaps the end of the one before it: 35 us for the 512 x 1024.)
//
// Ids outside [0, rows): the lookup returns NaN for them, the gradient leaves them out.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "device_common.h"
#include "dflash.h"
#include "training.h"

namespace dflash {
namespace {

// ---- lookup ------------------------------------------------------------------

// `lanes` (a power of two, at most 64) lanes a row; V elements an access (a chunk or 1).
template <typename T, typename I, int V>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(
    const I* __restrict__ ids, const T* __restrict__ table, T* __restrict__ out, int64_t n,
    int rows, int hidden, float scale, int lanes_log2) {
  const int lanes = 1 << lanes_log2;
  const int64_t token = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> lanes_log2;
  if (token >= n) return;
  const int64_t id = static_cast<int64_t>(ids[token]);
  const bool known = id >= 0 && id < rows;
  const T* from = table + (known ? id : 0) * hidden;
  T* to = out + token * hidden;
  for (int col = (threadIdx.x & (lanes - 1)) * V; col < hidden; col += lanes * V) {
    float v[V];
    if (known) {
      load_floats<T, V>(from + col, v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] *= scale;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = __builtin_nanf("");
    }
    store_floats<T, V>(to + col, v);
  }
}

// An id as the sort's key: ids that take no gradient become `rows`, past every other.
template <typename I>
__device__ inline int32_t key_of(I value, int rows, int64_t padding) {
  const int64_t id = static_cast<int64_t>(value);
  return id >= 0 && id < rows && id != padding ? static_cast<int32_t>(id) : rows;
}

// Zeros for bytes [begin, end) of dtable, both multiples of 16 but for the table's end (elements
// are 2 or 4 bytes), by workgroups `block` of `blocks`.
struct Fill {
  u32x4_t* table;
  int64_t begin, end;
};

template <int THREADS>
__device__ inline void fill_zeros(const Fill& f, int block, int blocks) {
  const int64_t at = static_cast<int64_t>(block) * THREADS + threadIdx.x;
  const int64_t chunks = f.end / 16;
  for (int64_t i = f.begin / 16 + at; i < chunks; i += static_cast<int64_t>(blocks) * THREADS)
    f.table[i] = u32x4_t{0, 0, 0, 0};
  if (at < (f.end - chunks * 16) / 2) reinterpret_cast<uint16_t*>(f.table + chunks)[at] = 0;
}

// ---- rank --------------------------------------------------------------------

// A token's place is the number of ids below its own and of equal ids before it: every token is
// compared with every id, two instructions a pair, ids four at a time from LDS.  A
// workgroup takes 64 >> parts_log2 tokens; its 1024 threads share out the ids, and the
// counts of a token are added.  Fewer tokens a workgroup where that fills more CUs.  Quadratic:
// the whole gradient of 4096 tokens takes 19 us this way and 31 by sort and merge, 8192 23
// and 27, 16384 44 and 41.
constexpr int kRankTokens = 8192;
constexpr int kRankThreads = 1024;

template <typename I>
__global__ __launch_bounds__(kRankThreads) void embedding_rank_kernel(
    const I* __restrict__ ids, int n, int rows, int64_t padding, int blocks, int parts_log2,
    int32_t* __restrict__ sorted_ids, int32_t* __restrict__ sorted_tokens, Fill fill) {
  typedef int32_t Four __attribute__((ext_vector_type(4)));
  extern __shared__ Four keys[];  // n of them, whole groups of four; then the counts
  if (static_cast<int>(blockIdx.x) >= blocks) {
    fill_zeros<kRankThreads>(fill, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const int quads = (n + 3) / 4;
  int32_t* flat = reinterpret_cast<int32_t*>(keys);
  int32_t* counts = flat + quads * 4;
  // (Every load is made, past the end of the last id, so that all are in flight together.)
  I given[kRankTokens / kRankThreads];
#pragma unroll
  for (int k = 0; k < kRankTokens / kRankThreads; ++k)
    given[k] = ids[min(k * kRankThreads + static_cast<int>(threadIdx.x), n - 1)];
#pragma unroll
  for (int k = 0; k < kRankTokens / kRankThreads; ++k) {
    const int j = k * kRankThreads + threadIdx.x;
    if (j < quads * 4)
      flat[j] = j < n ? key_of(given[k], rows, padding) : INT32_MAX;  // above every key
  }
  __syncthreads();
  // Neighbouring lanes hold the parts of one token.
  const int tokens = 64 >> parts_log2;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int token = blockIdx.x * tokens + (lane >> parts_log2);
  const int part = wave << parts_log2 | (lane & ((1 << parts_log2) - 1));
  const int parts = (kRankThreads / 64) << parts_log2;
  const int32_t key = flat[min(token, n - 1)];
  const int own = token / 4;  // equal ids count in the groups of four before this one
  int count = 0;
#pragma unroll 4
  for (int j = part; j < quads; j += parts) {
    const Four k = keys[j];
    const int32_t limit = key + (j < own);
#pragma unroll
    for (int e = 0; e < 4; ++e) count += k[e] < limit;
  }
  counts[threadIdx.x] = count;
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < tokens) {
    const int mine = blockIdx.x * tokens + threadIdx.x;
    if (mine < n) {
      int place = 0;
      for (int w = 0; w < kRankThreads / 64; ++w) {
        for (int i = 0; i < 1 << parts_log2; ++i)
          place += counts[w * 64 + (threadIdx.x << parts_log2 | i)];
      }
      const int32_t id = flat[mine];
      for (int j = mine / 4 * 4; j < mine; ++j) place += flat[j] == id;  // in its own group
      sorted_ids[place] = id;
      sorted_tokens[place] = mine;
    }
  }
}

// ---- sort --------------------------------------------------------------------

constexpr int kSortTokens = 2048;    // per workgroup; a place in the range is 16 bits
constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kSortRounds = kSortTokens / kSortThreads;  // tokens a lane
constexpr int kDigitBits = 9;
constexpr int kBins = 1 << kDigitBits;

struct SortLds {
  uint32_t keys[kSortTokens];
  uint32_t counters[kSortWaves][kBins];
  uint32_t wave_sums[kSortWaves];
  uint16_t places[kSortTokens];
};

// Wavefront-local order of LDS accesses: a wavefront's LDS instructions execute in order.
__device__ inline void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Stable radix sort of one range.
// Each wavefront owns a contiguous part of the range and ranks 64 keys a round: the lanes of
// equal digits are found with one ballot a bit, the digit's count so far is the
// wavefront's counter.  A scan over (digit, wavefront) gives the places.
template <typename I>
__device__ void sort_range(const I* __restrict__ ids, int64_t first, int count, int rows,
                           int64_t padding, int bits, int32_t* __restrict__ sorted_ids,
                           int32_t* __restrict__ sorted_tokens, SortLds& lds) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int rounds = (count + kSortThreads - 1) / kSortThreads;
  const int mine = wave * rounds * 64 + lane;  // + 64 a round
  const uint32_t last = bits < 32 ? (1u << bits) - 1 : ~0u;  // at least `rows`

  uint32_t key[kSortRounds], place[kSortRounds], rank[kSortRounds];
  I given[kSortRounds];  // (past the end the last id: every load in flight)
#pragma unroll
  for (int j = 0; j < kSortRounds; ++j) given[j] = ids[first + min(mine + 64 * j, count - 1)];
#pragma unroll
  for (int j = 0; j < kSortRounds; ++j) {
    place[j] = mine + 64 * j;
    // Past the end: behind every token, by its value and its place.
    key[j] = mine + 64 * j < count ? static_cast<uint32_t>(key_of(given[j], rows, padding)) : last;
  }
  const int passes = (bits + kDigitBits - 1) / kDigitBits;
  const int digit_bits = (bits + passes - 1) / passes;
  const int bins = 1 << digit_bits;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    uint32_t* counter = lds.counters[wave];
    for (int b = lane; b < bins; b += 64) counter[b] = 0;
    wave_order();
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
      if (j < rounds) {
        const uint32_t digit = (key[j] >> shift) & (bins - 1);
        uint64_t same = ~0ull;
#pragma unroll
        for (int b = 0; b < kDigitBits; ++b) {
          if (b < digit_bits) {
            const uint64_t ones = __ballot((digit >> b) & 1);
            same &= (digit >> b) & 1 ? ones : ~ones;
          }
        }
        const uint32_t before = counter[digit];
        const uint32_t ahead = __popcll(same & ((1ull << lane) - 1));
        rank[j] = before + ahead;
        wave_order();  // every lane has read the count
        if (ahead == 0) counter[digit] = before + __popcll(same);
        wave_order();
      }
    }
    __syncthreads();
    // Exclusive scan over (digit, wavefront): thread b owns digit b.
    uint32_t total = 0;
    if (threadIdx.x < bins) {
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = lds.counters[w][threadIdx.x];
        lds.counters[w][threadIdx.x] = total;
        total += c;
      }
    }
    uint32_t upto = total;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const uint32_t other = __shfl_up(upto, m);
      if (lane >= m) upto += other;
    }
    if (lane == 63) lds.wave_sums[wave] = upto;
    __syncthreads();
    if (threadIdx.x < bins) {
      uint32_t base = upto - total;
      for (int w = 0; w < wave; ++w) base += lds.wave_sums[w];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) lds.counters[w][threadIdx.x] += base;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
      if (j < rounds) {
        const uint32_t at = counter[(key[j] >> shift) & (bins - 1)] + rank[j];
        lds.keys[at] = key[j];
        lds.places[at] = static_cast<uint16_t>(place[j]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortRounds; ++j) {
      if (j < rounds) {
        key[j] = lds.keys[mine + 64 * j];
        place[j] = lds.places[mine + 64 * j];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kSortRounds; ++j) {
    const int at = mine + 64 * j;
    if (j < rounds && at < count) {
      sorted_ids[first + at] = static_cast<int32_t>(key[j]);
      sorted_tokens[first + at] = static_cast<int32_t>(first + place[j]);
    }
  }
}

template <typename I>
__global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(
    const I* __restrict__ ids, int64_t n, int rows, int64_t padding, int bits, int ranges,
    int32_t* __restrict__ sorted_ids, int32_t* __restrict__ sorted_tokens, Fill fill) {
  __shared__ SortLds lds;
  if (static_cast<int>(blockIdx.x) < ranges) {
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kSortTokens;
    const int count = n - first < kSortTokens ? static_cast<int>(n - first) : kSortTokens;
    sort_range(ids, first, count, rows, padding, bits, sorted_ids, sorted_tokens, lds);
    return;
  }
  fill_zeros<kSortThreads>(fill, blockIdx.x - ranges, gridDim.x - ranges);
}

// ---- merge -------------------------------------------------------------------

// kMergeRanges ranges become one sorted run.  A token's place in it: its place in its own range,
// and in every other range the number of ids before it (equal ids of earlier ranges come
// first).  The run's ranges lie in LDS, where each search takes 11 steps and the searches of one
// token are independent; from L2 the steps alone would take their latency 11 times over.
constexpr int kMergeRanges = 8;
constexpr int kMergeThreads = 256;
constexpr int kRunTokens = kMergeRanges * kSortTokens;

__global__ __launch_bounds__(kMergeThreads) void embedding_merge_kernel(
    const int32_t* __restrict__ ids, const int32_t* __restrict__ tokens, int64_t n,
    int32_t* __restrict__ merged_ids, int32_t* __restrict__ merged_tokens, int blocks, Fill fill) {
  typedef int32_t Four __attribute__((ext_vector_type(4)));
  constexpr int kLoads = kRunTokens / 4 / kMergeThreads;
  __shared__ Four lds4[kRunTokens / 4];
  int32_t* lds = reinterpret_cast<int32_t*>(lds4);
  if (static_cast<int>(blockIdx.x) >= blocks) {
    fill_zeros<kMergeThreads>(fill, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kMergeThreads + threadIdx.x;
  const int64_t at = i < n ? i : n - 1;
  const int32_t id = ids[at], token = tokens[at];
  // (A workgroup's tokens are of one range.)
  const int64_t first = i / kRunTokens * kRunTokens;
  const int own = static_cast<int>((i - first) / kSortTokens);
  const int held = n - first < kRunTokens ? static_cast<int>(n - first) : kRunTokens;
  // (The array is padded to 256 bytes: whole accesses, past the end the last one again.)
  Four given[kLoads];
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int j = (k * kMergeThreads + threadIdx.x) * 4;
    given[k] = *reinterpret_cast<const Four*>(ids + first + min(j, (held - 1) / 4 * 4));
  }
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int j = (k * kMergeThreads + threadIdx.x) * 4;
    Four v = given[k];  // past the end: above all ids
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e >= held) v[e] = INT32_MAX;
    lds4[j / 4] = v;
  }
  __syncthreads();
  int before[kMergeRanges];
#pragma unroll
  for (int r = 0; r < kMergeRanges; ++r) before[r] = 0;
  for (int step = kSortTokens / 2; step >= 1; step /= 2) {
#pragma unroll
    for (int r = 0; r < kMergeRanges; ++r) {
      const int32_t other = lds[r * kSortTokens + before[r] + step - 1];
      before[r] += other < id || (other == id && r < own) ? step : 0;
    }
  }
  int64_t place = i - own * kSortTokens;
#pragma unroll
  for (int r = 0; r < kMergeRanges; ++r) {
    // (The steps add up to kSortTokens - 1: the last id is still to be compared.)
    const int32_t other = lds[r * kSortTokens + before[r]];
    before[r] += other < id || (other == id && r < own) ? 1 : 0;
    if (r != own) place += before[r];
  }
  if (i < n) {
    merged_ids[place] = id;
    merged_tokens[place] = token;
  }
}

// kFan sorted runs of `length` tokens (a power of two; the last may be shorter) become one, the
// same way but from L2: neighbouring tokens search in the same places.  (Whole gradients into
// 128100 x 768 bf16, by 4 runs at a time, 8 and 16: 20000 tokens 52, 54, 57 us; 65536 89, 90, 94;
// 1048576 898, 914, 965.  Every range searched for every token, quadratic: 51, 96 and 4921.)
constexpr int kFan = 4;

__global__ __launch_bounds__(kMergeThreads) void embedding_merge_runs_kernel(
    const int32_t* __restrict__ ids, const int32_t* __restrict__ tokens, int n, int length,
    int32_t* __restrict__ merged_ids, int32_t* __restrict__ merged_tokens) {
  const int i = blockIdx.x * kMergeThreads + threadIdx.x;  // (at most kMaxTokens)
  if (i >= n) return;
  const int32_t id = ids[i], token = tokens[i];
  const int start = i / length / kFan * kFan * length;
  const int own = (i - start) / length;
  int before[kFan];
#pragma unroll
  for (int r = 0; r < kFan; ++r) before[r] = 0;
  // A token behind the end is above all ids.
  auto precedes = [&](int r, int at) {
    const int32_t other = ids[at < n ? at : n - 1];
    return at < n && (other < id || (other == id && r < own));
  };
  for (int step = length / 2; step >= 1; step /= 2) {
#pragma unroll
    for (int r = 0; r < kFan; ++r)
      before[r] += precedes(r, start + r * length + before[r] + step - 1) ? step : 0;
  }
  int place = i - own * length;
#pragma unroll
  for (int r = 0; r < kFan; ++r) {
    before[r] += precedes(r, start + r * length + before[r]) ? 1 : 0;
    if (r != own) place += before[r];
  }
  merged_ids[place] = id;
  merged_tokens[place] = token;
}

// ---- sum and join --------------------------------------------------------------

// Sorted tokens of a group of lanes.  Of 16: 2000 tokens 15 us instead of 18, but 16384 positions
// 43 instead of 36, one id alone 92 instead of 71, 65536 tokens 103 instead of 93.
constexpr int kTile = 32;
constexpr int kAhead = 16;     // rows of dout in flight
constexpr int kMinLanes = 8;   // of a group, so that its workgroup's tokens fit LDS

// The loads into `v` are all issued before the first is used: the compiler would otherwise move
// each down to where its row is added, and wait for it there.
template <typename A, int N>
__device__ inline void in_flight(A (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if constexpr (sizeof(A) > 4) {
      asm volatile("" : "+v"(v[j]));
    } else {  // a single element
      using Bits = std::conditional_t<sizeof(A) == 4, uint32_t, uint16_t>;
      uint32_t word = __builtin_bit_cast(Bits, v[j]);
      asm volatile("" : "+v"(word));
      v[j] = __builtin_bit_cast(A, static_cast<Bits>(word));
    }
  }
}

template <int V>
__device__ inline void store_partial(float* p, const float (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) p[e] = v[e];
}

// A group of `lanes` lanes sums one tile over lanes * V columns, slice `blockIdx.x % slices` of
// them: the workgroups that share rows of dout are neighbours, so that a row's pieces are
// fetched together.
// partials[tile][0]: what the tile holds of an id that began in an earlier tile;
// partials[tile][1]: of an id that begins here and goes on in the next tile.
// Bound by the latency of rows gathered from HBM: the tile's ids and tokens come through LDS
// first, so that the loads of kAhead rows depend on nothing else and are in flight together.
template <typename T, int V>
__global__ __launch_bounds__(256) void embedding_sum_kernel(
    const int32_t* __restrict__ ids, const int32_t* __restrict__ tokens, int64_t n, int rows,
    const T* __restrict__ dout, T* __restrict__ dtable, int hidden, float scale,
    float* __restrict__ partials, int lanes_log2, int slices) {
  typedef T Access __attribute__((ext_vector_type(V)));
  constexpr int kMost = 256 / kMinLanes * kTile;
  __shared__ int32_t lds_ids[kMost + 2];  // with the neighbours on both sides, -1 past the ends
  __shared__ int32_t lds_tokens[kMost];
  const int lanes = 1 << lanes_log2;
  const int tiles = 256 >> lanes_log2;
  const int64_t block = blockIdx.x / slices;
  const int slice = static_cast<int>(blockIdx.x - block * slices);
  const int64_t start = block * tiles * kTile;
  for (int i = threadIdx.x; i < tiles * kTile + 2; i += 256) {
    const int64_t at = start + i - 1;
    lds_ids[i] = at >= 0 && at < n ? ids[at] : -1;
    if (i < tiles * kTile) lds_tokens[i] = start + i < n ? tokens[start + i] : 0;
  }
  __syncthreads();
  const int group = threadIdx.x >> lanes_log2;
  const int64_t tile = block * tiles + group;
  const int64_t begin = tile * kTile;
  const int col = (slice * lanes + static_cast<int>(threadIdx.x & (lanes - 1))) * V;
  if (begin >= n || col >= hidden) return;
  const int count = n - begin < kTile ? static_cast<int>(n - begin) : kTile;
  const int32_t* id = lds_ids + 1 + group * kTile;
  const int32_t* token = lds_tokens + group * kTile;
  float* partial = partials + tile * 2 * hidden + col;

  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.0f;
  int32_t current = id[0];
  bool first = id[-1] == current;  // the sum in acc belongs to partials[tile][0]
  auto put = [&](bool goes_on) {
    if (first || goes_on) {
      store_partial(first ? partial : partial + hidden, acc);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] *= scale;
      store_floats<T, V>(dtable + static_cast<int64_t>(current) * hidden + col, acc);
    }
  };
  for (int i0 = 0; i0 < count; i0 += kAhead) {
    Access row[kAhead];
    int32_t next[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {  // (past the tile's end its last row again)
      const int at = min(i0 + j, count - 1);
      next[j] = id[at];
      row[j] =
          *reinterpret_cast<const Access*>(dout + static_cast<int64_t>(token[at]) * hidden + col);
    }
    in_flight(row);
    // (No exit from this loop: it has to unroll for its rows to stay in registers.  The tokens
    // without a gradient come last; what is added up for them is never written.)
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (next[j] != current) {
        put(false);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.0f;
        current = next[j];
        first = false;
      }
      const bool live = i0 + j < count;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += live ? static_cast<float>(row[j][e]) : 0.0f;
    }
  }
  if (current < rows) put(id[count] == current);
}

// One workgroup per tile and 256 columns.  If an id begins in the tile and goes on, its partial
// rows are added: kJoinWaves wavefronts take a contiguous part each, added in order.
constexpr int kJoinWaves = 8;

template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void embedding_join_kernel(
    const int32_t* __restrict__ ids, int64_t n, int rows, T* __restrict__ dtable, int hidden,
    float scale, const float* __restrict__ partials) {
  __shared__ float lds[kJoinWaves][256];
  const int64_t tile = blockIdx.x;
  const int64_t begin = tile * kTile;
  const int64_t end = begin + kTile;
  if (end >= n) return;  // (the last tile goes nowhere)
  // One round of loads for all that is decided on; the first token of the tile after next and of
  // those behind it, a thread each, for the count below.
  constexpr int kThreadsJoin = 64 * kJoinWaves;
  const int64_t tiles = (n + kTile - 1) / kTile;
  const int32_t id = ids[end - 1], next = ids[end], head = ids[begin];
  const int32_t ahead = begin > 0 ? ids[begin - 1] : -1;
  int64_t other = tile + 2 + threadIdx.x;
  int32_t theirs = other < tiles ? ids[other * kTile] : -1;
  if (id >= rows || next != id || (head == id && ahead == id)) return;  // ends, or began earlier
  // Tiles whose first token is of the id: [tile + 1, tile + count).
  int64_t count = 2;  // partial rows, this tile's among them
  for (;;) {
    const int found = __syncthreads_count(theirs == id);
    count += found;
    if (found < kThreadsJoin) break;
    other += kThreadsJoin;
    theirs = other < tiles ? ids[other * kTile] : -1;
  }
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t per = (count + kJoinWaves - 1) / kJoinWaves;
  const int64_t from = wave * per;
  const int64_t to = from + per < count ? from + per : count;
  const int mine = blockIdx.y * 256 + lane * 4;
  const bool whole = hidden % 4 == 0;  // then four columns are one access
  f32x4_t v{};
  if (mine < hidden) {
#pragma unroll 8
    for (int64_t i = from; i < to; ++i) {
      const float* row = partials + ((tile + i) * 2 + (i == 0)) * hidden;
      if (whole) {
        v += *reinterpret_cast<const f32x4_t*>(row + mine);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += row[min(mine + e, hidden - 1)];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) lds[wave][lane * 4 + e] = v[e];
  __syncthreads();
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (threadIdx.x < 256 && col < hidden) {
    float v = lds[0][threadIdx.x];
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w) v += lds[w][threadIdx.x];
    dtable[static_cast<int64_t>(id) * hidden + col] = static_cast<T>(v * scale);
  }
}

// ---- few tokens ----------------------------------------------------------------

// One launch for up to kFewTokens tokens: a workgroup owns rows of the table, zeroes them, picks
// the tokens of its rows out of all (in order), sorts them and adds up theirs.  256 tokens into
// two rows, the worst of it, take 24 us, as three launches do on the card; the host is spared
// two of them.
constexpr int kFewTokens = 256;

// The rows are dealt out `unit` at a time (ids next to each other are often frequent together):
// one where rows are whole 16-byte chunks, else as many as together always are.
template <typename T, typename I, int V>
__global__ __launch_bounds__(256) void embedding_few_kernel(
    const I* __restrict__ ids, int n, int rows, int64_t padding, int unit,
    const T* __restrict__ dout, T* __restrict__ dtable, int hidden, float scale, int lanes_log2) {
  typedef T Access __attribute__((ext_vector_type(V)));
  constexpr int kAheadFew = 16;
  __shared__ int32_t found[2][kFewTokens], sorted[2][kFewTokens];  // id, token
  __shared__ int32_t run[kFewTokens];  // tokens of an id, at its first one; 0 at the others
  __shared__ int32_t wave_counts[4];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int blocks = gridDim.x;
  const int32_t key = static_cast<int>(threadIdx.x) < n
                          ? key_of(ids[threadIdx.x], rows, padding) : rows;
  const bool mine = key < rows && key / unit % blocks == static_cast<int>(blockIdx.x);
  const uint64_t mask = __ballot(mine);
  if (lane == 0) wave_counts[wave] = __popcll(mask);

  const int64_t per_unit = static_cast<int64_t>(unit) * hidden / Chunk<T>::N;  // chunks
  const int64_t elements = static_cast<int64_t>(rows) * hidden;
  const int64_t chunks = elements / Chunk<T>::N;
  const int units = (rows - 1) / unit + 1;
  u32x4_t* table = reinterpret_cast<u32x4_t*>(dtable);
  if (per_unit < 256) {
    // Several units at a time, each by the lanes that hold one.
    const int at_once = 256 / static_cast<int>(per_unit);
    const int which = threadIdx.x / static_cast<int>(per_unit);
    const int64_t chunk = threadIdx.x % static_cast<int>(per_unit);
    for (int64_t u = blockIdx.x + static_cast<int64_t>(which) * blocks;
         which < at_once && u < units; u += static_cast<int64_t>(at_once) * blocks) {
      if (u * per_unit + chunk < chunks) table[u * per_unit + chunk] = u32x4_t{0, 0, 0, 0};
    }
  } else {
    for (int64_t u = blockIdx.x; u < units; u += blocks) {
      for (int64_t i = threadIdx.x; i < per_unit; i += 256)
        if (u * per_unit + i < chunks) table[u * per_unit + i] = u32x4_t{0, 0, 0, 0};
    }
  }
  // The elements behind the last whole chunk are the last unit's.
  if ((units - 1) % blocks == static_cast<int>(blockIdx.x) &&
      chunks * Chunk<T>::N + threadIdx.x < elements)
    dtable[chunks * Chunk<T>::N + threadIdx.x] = T(0);
  __syncthreads();  // the counts, and the zeros before the sums
  int count = 0, at = __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) at += wave_counts[w];
    count += wave_counts[w];
  }
  if (count == 0) return;
  if (mine) {
    found[0][at] = key;
    found[1][at] = threadIdx.x;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < count) {
    const int32_t row = found[0][threadIdx.x];
    int below = 0, equal = 0, before = 0;
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
      const int32_t other = found[0][i];
      below += other < row;
      equal += other == row;
      before += other == row && i < static_cast<int>(threadIdx.x);
    }
    sorted[0][below + before] = row;
    sorted[1][below + before] = found[1][threadIdx.x];
    run[below + before] = before == 0 ? equal : 0;
  }
  __syncthreads();
  // A group of lanes takes one id (at its first token) and a slice of the columns at a time.
  const int lanes = 1 << lanes_log2, groups = 256 >> lanes_log2;
  const int slices = (hidden / V + lanes - 1) >> lanes_log2;
  for (int task = threadIdx.x >> lanes_log2; task < count * slices; task += groups) {
    const int start = task / slices;
    const int col = ((task - start * slices) * lanes + (threadIdx.x & (lanes - 1))) * V;
    const int32_t row = sorted[0][start];
    const int end = start + run[start];
    if (col >= hidden || end == start) continue;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    for (int i = start; i < end; i += kAheadFew) {
      Access v[kAheadFew];
#pragma unroll
      for (int j = 0; j < kAheadFew; ++j)
        v[j] = *reinterpret_cast<const Access*>(
            dout + static_cast<int64_t>(sorted[1][min(i + j, end - 1)]) * hidden + col);
      in_flight(v);
#pragma unroll
      for (int j = 0; j < kAheadFew; ++j) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += i + j < end ? static_cast<float>(v[j][e]) : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= scale;
    store_floats<T, V>(dtable + static_cast<int64_t>(row) * hidden + col, acc);
  }
}

// ---- host --------------------------------------------------------------------

int lanes_log2_for(int accesses, int least, int most) {
  int log2 = least;
  while ((1 << log2) < accesses && log2 < most) ++log2;
  return log2;
}

uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

template <typename T, typename I>
int launch_fwd(const void* ids, const void* table, void* out, int64_t n, int rows, int hidden,
               float scale, hipStream_t stream) {
  constexpr int N = Chunk<T>::N;
  const bool wide = hidden % N == 0 && (address(table) | address(out)) % 16 == 0;
  const int log2 = lanes_log2_for(wide ? hidden / N : hidden, 0, 6);
  if (n > (kMaxBlocks256 * 256) >> log2) return DFLASH_ERR_TOO_LARGE;
  const int64_t blocks = ((n << log2) + 255) / 256;
  hipLaunchKernelGGL(
      (wide ? &embedding_fwd_kernel<T, I, N> : &embedding_fwd_kernel<T, I, 1>),
      dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream, static_cast<const I*>(ids),
      static_cast<const T*>(table), static_cast<T*>(out), n, rows, hidden, scale, log2);
  return static_cast<int>(hipGetLastError());
}

constexpr int kFewBlocks = 1024;   // workgroups of one launch for few tokens
// (Zeros of 197 MB: 512 workgroups 32.9 us, 2048 36.2, one access a thread 31.8.)
constexpr int kFillBlocks = 512;  // workgroups that write zeros
constexpr int64_t kMaxTokens = int64_t{1} << 26;
constexpr int kMaxHidden = 1 << 20;

// Workgroups that write `bytes` of zeros: 64 bytes a thread, kFillBlocks at most, one at least.
int fill_blocks(int64_t bytes, int threads) {
  const int64_t blocks = (bytes + 64 * threads - 1) / (64 * threads);
  return blocks < 1 ? 1 : blocks > kFillBlocks ? kFillBlocks : static_cast<int>(blocks);
}

int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }
int64_t ranges_of(int64_t n) { return (n + kSortTokens - 1) / kSortTokens; }
int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct Workspace {
  int64_t index_bytes, partial_bytes, total;
};

Workspace workspace_of(int64_t n, int hidden) {
  Workspace w{0, 0, 0};
  if (n <= kFewTokens) return w;
  w.index_bytes = aligned(n * 4);
  w.partial_bytes = aligned(tiles_of(n) * 2 * hidden * 4);
  w.total = (n > kRankTokens ? 4 : 2) * w.index_bytes + w.partial_bytes;
  return w;
}

template <typename T, typename I>
int launch_bwd(const void* ids_in, const void* dout_in, void* dtable_in, int64_t n, int rows,
               int hidden, float scale, int64_t padding, char* workspace, hipStream_t stream) {
  const Workspace w = workspace_of(n, hidden);
  int32_t* ids = reinterpret_cast<int32_t*>(workspace);
  int32_t* tokens = reinterpret_cast<int32_t*>(workspace + w.index_bytes);
  float* partials = reinterpret_cast<float*>(workspace + w.total - w.partial_bytes);
  const int64_t table_bytes = static_cast<int64_t>(rows) * hidden * sizeof(T);
  constexpr int N = Chunk<T>::N;
  const I* ids_as_given = static_cast<const I*>(ids_in);
  const T* dout = static_cast<const T*>(dout_in);
  T* dtable = static_cast<T*>(dtable_in);
  const bool wide = hidden % N == 0 && address(dout) % 16 == 0;
  const int accesses = wide ? hidden / N : hidden;
  const int log2 = lanes_log2_for(accesses, 3, 5);
  const int64_t tiles = tiles_of(n);
  const int slices = (accesses + (1 << log2) - 1) >> log2;
  const int64_t sum_blocks = ((tiles << log2) + 255) / 256 * slices;
  if (sum_blocks > kMaxBlocks256) return DFLASH_ERR_TOO_LARGE;  // (before anything is launched)
  if (n <= kFewTokens) {
    const int unit = hidden % N == 0 ? 1 : N;
    const int units = (rows - 1) / unit + 1;
    hipLaunchKernelGGL((wide ? &embedding_few_kernel<T, I, N> : &embedding_few_kernel<T, I, 1>),
                       dim3(units < kFewBlocks ? units : kFewBlocks), dim3(256), 0, stream,
                       ids_as_given, static_cast<int>(n), rows, padding, unit, dout, dtable,
                       hidden, scale, log2);
    return static_cast<int>(hipGetLastError());
  }
  // The zeros go with the first launch, and a part of them with the merge if there is one, so
  // that neither has the card to itself.  (With 2/5, 3/5, 4/5 and all of them in the first: 16384
  // tokens into 128100 x 768 bf16 54.5, 52.1, 54.8, 59.1 us, x 1536 96.9, 98.7, 98.0, 104.2,
  // 30000 x 768 37.3, 37.2, 36.5, 35.5; 65536 into 128100 x 768 97.3, 97.3, 101.4, 103.4; 10000
  // into 128100 x 1024 fp32 121.5, 120.0, 119.5, 126.4; 262144 tokens or 512 rows within 1 %.)
  const bool by_rank = n <= kRankTokens;
  const int64_t first_part = by_rank ? table_bytes : table_bytes / 5 * 3 / 16 * 16;
  const Fill fill{static_cast<u32x4_t*>(dtable_in), 0, first_part};
  int rc;
  if (by_rank) {
    // 256 workgroups or more, of 8 to 64 tokens.
    int parts_log2 = 0;
    while (parts_log2 < 3 && n <= (256 * 64) >> (parts_log2 + 1)) ++parts_log2;
    const int blocks = static_cast<int>((n + (64 >> parts_log2) - 1) >> (6 - parts_log2));
    const int lds = static_cast<int>((n + 3) / 4 * 16) + kRankThreads * 4;
    hipLaunchKernelGGL((embedding_rank_kernel<I>),
                       dim3(blocks + fill_blocks(first_part, kRankThreads)), dim3(kRankThreads),
                       lds, stream, ids_as_given, static_cast<int>(n), rows, padding, blocks,
                       parts_log2, ids, tokens, fill);
    rc = static_cast<int>(hipGetLastError());
    if (rc != DFLASH_OK) return rc;
  } else {
    const int ranges = static_cast<int>(ranges_of(n));
    int bits = 1;
    while ((int64_t{1} << bits) - 1 < rows) ++bits;
    hipLaunchKernelGGL((embedding_sort_kernel<I>),
                       dim3(ranges + fill_blocks(first_part, kSortThreads)), dim3(kSortThreads), 0,
                       stream, ids_as_given, n, rows, padding, bits, ranges, ids, tokens, fill);
    rc = static_cast<int>(hipGetLastError());
    if (rc != DFLASH_OK) return rc;
    int32_t* merged = reinterpret_cast<int32_t*>(workspace + 2 * w.index_bytes);
    int32_t* merged_tokens = reinterpret_cast<int32_t*>(workspace + 3 * w.index_bytes);
    const Fill rest{static_cast<u32x4_t*>(dtable_in), first_part, table_bytes};
    const int blocks = static_cast<int>((n + kMergeThreads - 1) / kMergeThreads);
    hipLaunchKernelGGL(embedding_merge_kernel,
                       dim3(blocks + fill_blocks(table_bytes - first_part, kMergeThreads)),
                       dim3(kMergeThreads), 0, stream, ids, tokens, n, merged, merged_tokens,
                       blocks, rest);
    rc = static_cast<int>(hipGetLastError());
    if (rc != DFLASH_OK) return rc;
    std::swap(ids, merged);
    std::swap(tokens, merged_tokens);
    for (int64_t length = kRunTokens; length < n; length *= kFan) {
      hipLaunchKernelGGL(embedding_merge_runs_kernel, dim3(blocks), dim3(kMergeThreads), 0, stream,
                         ids, tokens, static_cast<int>(n), static_cast<int>(length), merged,
                         merged_tokens);
      rc = static_cast<int>(hipGetLastError());
      if (rc != DFLASH_OK) return rc;
      std::swap(ids, merged);
      std::swap(tokens, merged_tokens);
    }
  }
  hipLaunchKernelGGL((wide ? &embedding_sum_kernel<T, N> : &embedding_sum_kernel<T, 1>),
                     dim3(static_cast<uint32_t>(sum_blocks)), dim3(256), 0, stream, ids, tokens, n,
                     rows, dout, dtable, hidden, scale, partials, log2, slices);
  rc = static_cast<int>(hipGetLastError());
  if (rc != DFLASH_OK) return rc;
  hipLaunchKernelGGL((embedding_join_kernel<T>),
                     dim3(static_cast<uint32_t>(tiles), (hidden + 255) / 256),
                     dim3(64 * kJoinWaves), 0, stream, ids, n, rows, dtable, hidden, scale, partials);
  return static_cast<int>(hipGetLastError());
}

// Calls f(T, I) with the element types of the codes.
template <typename F>
int with_types(int dtype, int id_bytes, F f) {
  if (id_bytes != 4 && id_bytes != 8) return DFLASH_ERR_DTYPE;
  auto with_ids = [&](auto t) {
    return id_bytes == 4 ? f(t, int32_t()) : f(t, int64_t());
  };
  switch (dtype) {
    case DFLASH_DTYPE_FP16: return with_ids(_Float16());
    case DFLASH_DTYPE_BF16: return with_ids(__bf16());
    case DFLASH_DTYPE_FP32: return with_ids(float());
    default: return DFLASH_ERR_DTYPE;
  }
}

bool shape_taken(int64_t n, int rows, int hidden) {
  return n >= 0 && n <= kMaxTokens && rows >= 1 && rows < INT32_MAX && hidden >= 1 &&
         hidden <= kMaxHidden;
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" int dflash_embedding_fwd(const void* ids, const void* table, void* out, int64_t n,
                                    int rows, int hidden, float scale, int id_bytes, int dtype,
                                    void* stream) {
  if (!shape_taken(n, rows, hidden)) return DFLASH_ERR_SHAPE;
  return with_types(dtype, id_bytes, [&](auto t, auto i) {
    using T = decltype(t);
    using I = decltype(i);
    if (n == 0) return static_cast<int>(DFLASH_OK);
    if (!ids || !table || !out) return static_cast<int>(DFLASH_ERR_NULL);
    if (address(ids) % sizeof(I) != 0 || (address(table) | address(out)) % sizeof(T) != 0)
      return static_cast<int>(DFLASH_ERR_ALIGN);
    return launch_fwd<T, I>(ids, table, out, n, rows, hidden, scale,
                            static_cast<hipStream_t>(stream));
  });
}

extern "C" size_t dflash_embedding_bwd_workspace_bytes(int64_t n, int hidden) {
  if (!shape_taken(n, 1, hidden)) return 0;
  return static_cast<size_t>(workspace_of(n, hidden).total);
}

extern "C" int dflash_embedding_bwd(const void* ids, const void* dout, void* dtable, int64_t n,
                                    int rows, int hidden, float scale, int64_t padding,
                                    int id_bytes, int dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (!shape_taken(n, rows, hidden)) return DFLASH_ERR_SHAPE;
  return with_types(dtype, id_bytes, [&](auto t, auto i) {
    using T = decltype(t);
    using I = decltype(i);
    if (!dtable || (n > 0 && (!ids || !dout)) || (workspace_of(n, hidden).total && !workspace))
      return static_cast<int>(DFLASH_ERR_NULL);
    if (address(ids) % sizeof(I) != 0 || address(dout) % sizeof(T) != 0 ||
        address(dtable) % 16 != 0 || address(workspace) % 16 != 0)
      return static_cast<int>(DFLASH_ERR_ALIGN);
    if (workspace_bytes < static_cast<size_t>(workspace_of(n, hidden).total))
      return static_cast<int>(DFLASH_ERR_WORKSPACE);
    return launch_bwd<T, I>(ids, dout, dtable, n, rows, hidden, scale, padding,
                            static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
  });
}
