// Disentangled attention of a training step, with dropout on the probabilities, and its gradients.
//
//   s(i, j) = scale (Q_i.K_j + Q_i.PK[t(i-j)] + K_j.PQ[t(i-j)])      t: delta -> slot
//   kept query: softmax over the kept keys; padded query: 1/L for every key
//   R = P M (M: 0 or the inverse of the kept share),  O = R V
//
//   dV = R^T dO,  G = P (M (dO V^T) - D_i), D_i = dO_i.O_i, 0 where a pair is masked
//   dQ_i = scale sum_j G_ij (K_j + PK[t(i-j)]),  dK_j = scale sum_i G_ij (Q_i + PQ[t(i-j)])
//   dPK[u] = scale sum over t(i-j) = u of G_ij Q_i,  dPQ[u] = scale sum of G_ij K_j
//
// Relative terms by delta.  A block of 16 rows against a tile of keys meets one contiguous range
// of deltas i - j, so the rows PK[t(.)] of that range (gathered into LDS, the "window") are multiplied
// by the 16 rows with MFMA, and element (i, j) is read at column i - j of the result: a skewed
// read from LDS.  The gradients go the other way: G is written into a skewed buffer
// [row][i - j], whose places outside the band stay 0, and that buffer is the operand of the
// products with PK, PQ (dQ, dK) and, transposed, with Q, K (dPK, dPQ).
//
// The backward pass: D_i; then a kernel over blocks of keys, which computes P and G, sums dV and dK
// in registers and writes G once; one over blocks of queries, which sums dQ from G; one over
// diagonals of tiles, which sums dPK and dPQ from G by delta; one that adds up a diagonal's parts; and
// one that adds up the deltas of each slot.  No atomics: every sum has an order of its own.
//
// Measured (us; heads of 64 in bf16, dropout 0.1, both terms, padded batches):
//                  dropped places   forward   D    dV dK G   dQ   by delta   parts   by slot
//   32 x 512 x 12 heads       34       247    14       264   77         96      11        16
//   2 x 2000 x 12 heads       33       283     6       301   77         98      19        58
// No unit bounds the forward and the dV dK G kernel: the matrix unit is busy 9 and 12 % of the time,
// the vector unit 32 and 25 %, LDS 23 and 34 %; a wavefront waits at barriers and for loads 42 and 37 % of its
// time and for its turn to issue 15 and 23 %.  It is the chain of products, LDS, skewed reads, exponentials
// and products again, at two wavefronts a SIMD: latency, and no limit of the card (the inference kernel computes
// the same scores, softmax and product, over all pairs, in 87).  Nor does a part stand out: without the
// window products, the skewed reads, the skewed buffer and dK, the store of G, the loads of the windows
// or dV, the latter kernel lost 14 to 28 % each.  (Comments below give both sides of a choice as measured together,
// some of them by earlier builds, whose times differ from these.)
//
// G is kept in fragments: 16 keys x 32 queries are 512 elements in the order in which the
// lanes of a wavefront hold them, so that they are written and read 16 bytes a lane.
//
// Padded rows.  Rows of K at padded keys and of Q at padded queries are taken as 0 in every product,
// and so is what is not finite in V at padded keys, so that whatever they hold, NaN too,
// reaches no kept row.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "device_common.h"
#include "dflash.h"
#include "training.h"

namespace dflash {
namespace {

constexpr int kMaxLength = 16384;
constexpr int kWords = kMaxLength / 64;
constexpr int kFragment = 512;  // elements of a fragment of G: 16 keys x 32 queries

typedef float f32x8_t __attribute__((ext_vector_type(8), aligned(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t lds_s4_t;

struct Strides {
  int64_t b, h, l;
};

struct Params {
  const void *q, *k, *v;
  Strides sq, sk, sv;
  const void *pos_key, *pos_query;  // [H, S, D], NULL: no such term
  int64_t pk_h, pk_s, pq_h, pq_s;
  const int32_t* lut;     // [2L - 1]
  const uint8_t* mask;    // [B, L], may be NULL
  const uint8_t* bits;    // dropped places, rows of `bit_row` bytes; NULL: no dropout
  int64_t bit_row;
  void* out;              // [B, L, H, D]
  void* low;              // what `out`'s rounding left off, may be NULL
  float* lse;             // [B, H, L], base 2
  const void* dout;       // [B, L, H, D]
  const float* delta;     // [B, H, L]: D_i
  void *dq, *dk, *dv;     // [B, L, H, D]
  void* g;                // fragments
  float* partial;         // sums of dPK and dPQ by tile diagonal
  uint64_t* words;        // [B][ceil(L / 64)]: the mask's bits
  int b0, h0, nb, nh;     // the (batch, head) pairs of this launch
  int B, H, L, S;
  float scale, scale_log2, keep_scale;
};

// ---- operands -------------------------------------------------------------------------

// One step is 32 deep, of eight elements a lane; a half step is 16 deep, of four.
template <typename T>
struct Op {
  using frag = typename Mma<T>::frag;
  using half = Quad<T>;
  __device__ static f32x4_t run(frag a, frag b, f32x4_t c) { return Mma<T>::run(a, b, c); }
  // (The 32-deep instruction beside zeros: the 16-deep one, on the accumulators of a 32-deep one
  // two instructions before, left half of them without the older sum.)
  __device__ static f32x4_t run_half(half a, half b, f32x4_t c) {
    const half none{};
    return run(__builtin_shufflevector(a, none, 0, 1, 2, 3, 4, 5, 6, 7),
               __builtin_shufflevector(b, none, 0, 1, 2, 3, 4, 5, 6, 7), c);
  }
};
template <>
struct Op<float> {
  using frag = f32x8_t;
  using half = Quad<float>;
  __device__ static f32x4_t run_half(half a, half b, f32x4_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
  __device__ static f32x4_t run(frag a, frag b, f32x4_t c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// Rows in LDS are padded by 16 bytes: the 16 rows that a fragment read touches lie in different banks.
// Padded by 32, so do the rows 8g + 0..3 of a transposing read of 16-bit elements, which is worth it where no
// workgroup less fits a CU for it: in the key kernel (321 -> 288 us at 32 x 512 full tokens, heads of 128
// 228 -> 207) and in the forward pass (251 -> 247 at 32 x 512 padded tokens, heads of 128 45 -> 43 at 7 x 437); the
// query kernel would lose one (91 -> 109 at 32 x 512 full tokens).
template <typename T, int D>
constexpr int kLd = D + 16 / static_cast<int>(sizeof(T));
template <typename T, int D>
constexpr int kLdWide = sizeof(T) == 2 ? D + 16 : kLd<T, D>;

// Lane (c, g): elements 8g .. 8g+7 of the row of `p` (p: the row, at the k-step's start).
template <typename T>
__device__ inline typename Op<T>::frag read_row(const T* p, int g) {
  return *reinterpret_cast<const typename Op<T>::frag*>(p + 8 * g);
}

// Lane (c, g): column c of the 16 at `p` of eight rows, `lo` + 0..3 and `hi` + 0..3 (both depend on
// g), of a tile whose rows are `ld` elements apart.
template <typename T>
__device__ inline typename Op<T>::frag read_columns(const T* p, int ld, int lo, int hi, int c) {
  if constexpr (sizeof(T) == 4) {
    f32x8_t f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = p[(lo + e) * ld + c];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[4 + e] = p[(hi + e) * ld + c];
    return f;
  } else {
    // Transposing reads: lane c supplies the address of row c / 4, columns 4 (c % 4) .. + 3.
    const T* a = p + (lo + (c >> 2)) * ld + 4 * (c & 3);
    const T* b = p + (hi + (c >> 2)) * ld + 4 * (c & 3);
    const u32x2_t x =
        __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)a));
    const u32x2_t y =
        __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)b));
    return __builtin_bit_cast(typename Op<T>::frag, u32x4_t{x[0], x[1], y[0], y[1]});
  }
}

// Lane (c, g): column c of the 16 at `p` of rows `lo` + 0..3.
template <typename T>
__device__ inline typename Op<T>::half read_columns_half(const T* p, int ld, int lo, int c) {
  if constexpr (sizeof(T) == 4) {
    Quad<float> f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = p[(lo + e) * ld + c];
    return f;
  } else {
    const T* a = p + (lo + (c >> 2)) * ld + 4 * (c & 3);
    return __builtin_bit_cast(typename Op<T>::half,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)a));
  }
}

// Scores by delta are fp32 in LDS, scaled, as the backward pass computes them again: its probabilities
// are those of the forward pass only if their rounding is the same, and fp16 would have neither
// the range of bf16 inputs (a score past 65504) nor their sums (a row of probabilities of scores of
// some hundreds adds up to 0.92 .. 1.09 beside a statistic of rounded ones).  Beside fp16 operands scores in
// fp16 were the largest error: the gradients of 16 x 384 tokens, heads of 32, were off by 4.0e-4 of their
// size, with fp32 by 3.0e-4.

// Eight values of the accumulators of two blocks of 16 rows as an operand: element e < 4 is row
// 4g + e of the first, e >= 4 row 4g + e - 4 of the second.
template <typename T>
__device__ inline typename Op<T>::frag pack(f32x4_t a, f32x4_t b) {
  typename Op<T>::frag f;
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = static_cast<T>(a[e]);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[4 + e] = static_cast<T>(b[e]);
  return f;
}

// What rounding to T left off.
template <typename T>
__device__ inline f32x4_t left(f32x4_t x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] -= static_cast<float>(static_cast<T>(x[e]));
  return x;
}

// The same from global memory; `from`: byte offset of the eight.
template <typename T>
__device__ inline typename Op<T>::frag load_frag(__amdgpu_buffer_rsrc_t memory, uint32_t from) {
  const u32x4_t lo = __builtin_amdgcn_raw_buffer_load_b128(memory, from, 0, 0);
  if constexpr (sizeof(T) == 4) {
    const u32x4_t hi = __builtin_amdgcn_raw_buffer_load_b128(memory, from + 16, 0, 0);
    f32x8_t f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = __builtin_bit_cast(float, static_cast<uint32_t>(lo[e]));
      f[4 + e] = __builtin_bit_cast(float, static_cast<uint32_t>(hi[e]));
    }
    return f;
  } else {
    return __builtin_bit_cast(typename Op<T>::frag, lo);
  }
}

template <typename T>
__device__ inline void store_frag(__amdgpu_buffer_rsrc_t memory, uint32_t at,
                                  typename Op<T>::frag f) {
  if constexpr (sizeof(T) == 4) {
    __builtin_amdgcn_raw_buffer_store_b128(
        __builtin_bit_cast(u32x4_t, f32x4_t{f[0], f[1], f[2], f[3]}), memory, at, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(
        __builtin_bit_cast(u32x4_t, f32x4_t{f[4], f[5], f[6], f[7]}), memory, at + 16, 0, 0);
  } else {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, f), memory, at, 0, 0);
  }
}

template <typename T>
__device__ inline void store4(T* p, f32x4_t v) {
  Quad<T> q;
#pragma unroll
  for (int r = 0; r < 4; ++r) q[r] = static_cast<T>(v[r]);
  *reinterpret_cast<Quad<T>*>(p) = q;
}

// ---- tiles ----------------------------------------------------------------------------

// Rows are read through buffer resources: an offset past the size gives zeros, so that rows
// that are not to be read cost no branch, and all loads of a tile are in flight together
// (behind a branch for each of them a tile of the first kernels took 11 us, most of it waiting).
constexpr uint32_t kNoRow = 0x80000000u;  // past every resource's size
constexpr int kBufferFlags = 0x00020000;  // raw buffer, gfx9 family descriptor word 3

__device__ inline __amdgpu_buffer_rsrc_t resource(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0),
                                           static_cast<int>(bytes), kBufferFlags);
}

// Tokens of one head: rows `stride` elements apart.
template <typename T, int D>
struct Tokens {
  __amdgpu_buffer_rsrc_t memory;
  uint32_t stride;  // bytes
  __device__ Tokens(const void* base, const Strides& s, int b, int h, int L)
      : memory(resource(static_cast<const T*>(base) + b * s.b + h * s.h,
                        ((L - 1) * s.l + D) * static_cast<int64_t>(sizeof(T)))),
        stride(static_cast<uint32_t>(s.l * sizeof(T))) {}
};

// ROWS rows of D elements on their way into LDS, in the registers of NT threads.
template <typename T, int D, int ROWS, int NT, int LD = kLd<T, D>>
struct Stage {
  static constexpr int kChunks = D * static_cast<int>(sizeof(T)) / 16;
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  static constexpr int N = (ROWS * kChunks + NT - 1) / NT;
  u32x4_t v[N];

  __device__ static int row(int n) { return (n * NT + threadIdx.x) / kChunks; }
  __device__ static int chunk(int n) { return (n * NT + threadIdx.x) % kChunks; }
  __device__ static bool inside(int n) { return ROWS * kChunks % NT == 0 || row(n) < ROWS; }

  // offset(n, row): the row's byte offset, or kNoRow.
  template <typename Offset>
  __device__ void load(__amdgpu_buffer_rsrc_t memory, const Offset& offset) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      v[n] = __builtin_amdgcn_raw_buffer_load_b128(memory, offset(n, row(n)) + 16 * chunk(n), 0, 0);
  }
  // Rows whose bit of `wanted` is 0 are zeros.
  __device__ void load_tokens(const Tokens<T, D>& tokens, int first, uint64_t wanted) {
    load(tokens.memory, [&](int, int r) {
      return r < ROWS && (wanted >> (r & 63)) & 1 ? (first + r) * tokens.stride : kNoRow;
    });
  }
  // Infinities and NaN in the rows whose bit of `suspect` is 1 become 0.
  __device__ void make_finite(uint64_t suspect) {
    typedef T Elements __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!((suspect >> (row(n) & 63)) & 1)) continue;
      Elements x = __builtin_bit_cast(Elements, v[n]);
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (!(fabsf(static_cast<float>(x[e])) < INFINITY)) x[e] = static_cast<T>(0.0f);
      v[n] = __builtin_bit_cast(u32x4_t, x);
    }
  }
  // Row r goes to row place(r) of the tile.
  template <typename Place>
  __device__ void store(T* tile, const Place& place) const {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (inside(n))
        *reinterpret_cast<u32x4_t*>(tile + place(row(n)) * LD + chunk(n) * kPer) = v[n];
  }
  __device__ void store(T* tile) const {
    store(tile, [](int r) { return r; });
  }
};

// A window: ROWS position rows of successive deltas in LDS.  A step moves it STEP deltas on; the
// rows form a ring, so that only the new ones are read.  They are read through the table of slots
// two steps ahead of their use: first the slots, then the rows, then LDS.  Where the ring is two
// steps long the loops are written out for both of its positions, PHASE, and every address
// is a constant; a longer one has its position in a scalar register.
template <typename T, int D, int ROWS, int STEP, int NT, int LD = kLd<T, D>>
struct Window {
  static_assert(ROWS % 16 == 0 && STEP % 16 == 0 && STEP <= ROWS, "blocks of 16 rows");
  static_assert(ROWS != 2 * STEP || (STEP & (STEP - 1)) == 0, "a power of two");
  using First = Stage<T, D, ROWS, NT, LD>;
  using Next = Stage<T, D, STEP, NT, LD>;
  __amdgpu_buffer_rsrc_t table, lut;
  uint32_t stride;  // bytes
  int L, S;
  static constexpr bool kTwo = ROWS == 2 * STEP;
  int ring;  // the first row's place, where there are not two
  int slots[Next::N];
  Next rows;

  __device__ Window(const void* base, int64_t row_stride, const int32_t* lut_, int L_, int S_)
      : table(resource(base, ((S_ - 1) * row_stride + D) * static_cast<int64_t>(sizeof(T)))),
        lut(resource(lut_, (2 * static_cast<int64_t>(L_) - 1) * 4)),
        stride(static_cast<uint32_t>(row_stride * sizeof(T))), L(L_), S(S_), ring(0) {}

  __device__ bool inside(int delta) const { return delta > -L && delta < L; }
  __device__ int slot_of(int delta) const {
    return static_cast<int>(__builtin_amdgcn_raw_buffer_load_b32(
        lut, inside(delta) ? 4 * (delta + L - 1) : kNoRow, 0, 0));
  }
  __device__ uint32_t offset_of(int slot, int delta) const {
    return inside(delta) && slot >= 0 && slot < S ? slot * stride : kNoRow;
  }
  // All rows, from the delta `first`.
  __device__ void fill(T* tile, int first) {
    int at[First::N];
#pragma unroll
    for (int n = 0; n < First::N; ++n) at[n] = slot_of(first + First::row(n));
    First all;
    all.load(table, [&](int n, int r) { return offset_of(at[n], first + r); });
    all.store(tile);
    ring = 0;
  }
  // The slots of the rows that come after those of the window from `first`, and then those rows.
  // (Nothing looks at a slot before: it would be waited for, and all other loads with it.)
  __device__ void read_slots(int first) {
#pragma unroll
    for (int n = 0; n < Next::N; ++n) slots[n] = slot_of(first + ROWS + Next::row(n));
  }
  __device__ void read_rows(int first) {
    rows.load(table, [&](int n, int r) { return offset_of(slots[n], first + ROWS + r); });
    asm volatile("" ::: "memory");  // (before slots are read into the same registers)
  }
  // To the position PHASE.
  template <int PHASE>
  __device__ void advance(T* tile) {
    if constexpr (kTwo) {
      rows.store(tile, [](int r) { return r + (PHASE ? 0 : STEP); });
    } else {
      rows.store(tile, [&](int r) { return r + ring < ROWS ? r + ring : r + ring - ROWS; });
      ring += STEP;
      if (ring >= ROWS) ring -= ROWS;
    }
  }
  // Where row r of the window lies; 16 rows from a multiple of 16 lie together.
  template <int PHASE>
  __device__ int place(int r) const {
    if constexpr (kTwo) return PHASE ? r ^ STEP : r;
    const int at = r + ring;
    return at < ROWS ? at : at - ROWS;
  }
};
// (r ^ STEP is r + STEP in a ring of 2 STEP rows, STEP a power of two.)

// step(PHASE) until it returns false.
template <bool TWO, typename Step>
__device__ inline void alternate(const Step& step) {
  for (;;) {
    if (!step(std::integral_constant<int, 0>{})) break;
    if constexpr (TWO) {
      if (!step(std::integral_constant<int, 1>{})) break;
    }
  }
}

// Bit j % 64 of words[j / 64]: token j is kept (0 for j >= L).
__device__ inline void read_mask(uint64_t* words, const uint8_t* mask, int b, int L) {
  for (int at = threadIdx.x; at < (L + 63) / 64 * 64; at += blockDim.x) {
    const bool kept = at < L && (!mask || mask[static_cast<int64_t>(b) * L + at]);
    const uint64_t word = __ballot(kept);
    if (threadIdx.x % 64 == 0) words[at / 64] = word;
  }
  __syncthreads();
}

__device__ inline bool bit_of(const uint64_t* words, int at) {
  return (words[at >> 6] >> (at & 63)) & 1;
}

// Tokens at, at + 1, .. that lie in the sequence, as bits.
__device__ inline uint64_t tokens_from(int at, int L) {
  const int n = L - at;
  return n >= 64 ? ~uint64_t{0} : n <= 0 ? 0 : (uint64_t{1} << n) - 1;
}

// Bits at .. at + 63 of the sequence's words, at a multiple of 16.
__device__ inline uint64_t kept_from(const uint64_t* words, int at, int L) {
  return at < L ? words[at >> 6] >> (at & 63) : 0;
}

// The first and last block of 64 tokens of [from, to) that holds a kept one; first > last: none.
__device__ inline void kept_range(const uint64_t* words, int from, int to, int* first, int* last) {
  while (from < to && words[from] == 0) ++from;
  while (to > from && words[to - 1] == 0) --to;
  *first = from;
  *last = to - 1;
}

// x[n][r] where bit 16 n + r is 1, else 0 (by its bits: one sign-extended field and one AND).
template <int N>
__device__ inline void drop(f32x4_t (&x)[N], uint64_t kept) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t word = static_cast<uint32_t>(kept >> (n / 2 * 32));
      const int mask = __builtin_amdgcn_sbfe(static_cast<int>(word), n % 2 * 16 + r, 1);
      x[n][r] = __builtin_bit_cast(float, __builtin_bit_cast(int, static_cast<float>(x[n][r])) & mask);
    }
}

// ---- dropped places ---------------------------------------------------------------------

// Bit j of row (b, h, i): the probability is dropped.  The element's place in the generator is its
// index in the flattened [B, H, L, L] tensor, so a byte of a row spans two of the generator's
// blocks where L is no multiple of 8.
__global__ __launch_bounds__(256) void dropped_bits_kernel(uint8_t* bits, int64_t rows, int L,
                                                           int row_bytes, Dropout d) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = at / row_bytes;
  if (row >= rows) return;
  const int byte = static_cast<int>(at - row * row_bytes);
  uint32_t value = 0;
  if (byte * 8 < L) {
    const DropoutKey key = dropout_key(d);
    const int64_t first = row * L + byte * 8;
    value = dropped_of_block(d, key, first >> 3);
    const int shift = static_cast<int>(first & 7);
    if (shift) value = (value | dropped_of_block(d, key, (first >> 3) + 1) << 8) >> shift;
  }
  bits[at] = static_cast<uint8_t>(value);
}

// ---- forward ------------------------------------------------------------------------------

// A workgroup of NW wavefronts takes 16 NW queries and walks the keys in tiles of BK, the last
// first (so that its windows move up).  Scores are computed transposed (a lane holds one query
// and four keys of a block), so that the probabilities are the operand of O^T += V^T R^T as they are.
// Padded queries have the score 0 for every key; only for them are the tiles without kept keys
// walked.  Of V at padded keys, which a kept query multiplies by 0, what is not finite is taken as 0.
template <typename T, int D, int NW, int BK>
struct FwdLayout {
  static constexpr int BQ = 16 * NW, W = BQ + BK, LDC = BK + 20, LDP = BQ + 20;
  static constexpr int LD = kLdWide<T, D>;
  T k[BK * LD], v[BK * LD], pk[W * LD], pq[W * LD];
  float c2p[BQ * LDC], p2c[BK * LDP];
  uint64_t kept[kWords];
};

template <typename T, int D, int NW, int BK, bool BOTH>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 ? 2 : 1)))
void attention_train_fwd_kernel(Params p) {
  using Y = FwdLayout<T, D, NW, BK>;
  using F = typename Op<T>::frag;
  constexpr int BQ = Y::BQ, LD = Y::LD, LDC = Y::LDC, LDP = Y::LDP, NT = 64 * NW, KB = BK / 16;
  constexpr uint64_t kBlock = BK == 64 ? ~uint64_t{0} : (uint64_t{1} << (BK % 64)) - 1;
  extern __shared__ __align__(16) unsigned char memory[];
  Y& s = *reinterpret_cast<Y*>(memory);
  const int blocks = (p.L + BQ - 1) / BQ;
  const int at = xcd_logical_block(blockIdx.x, gridDim.x);
  const int bh = at / blocks, i0 = at % blocks * BQ;
  const int b = bh / p.H, h = bh % p.H;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, c = lane % 16, g = lane / 16;
  const int i = i0 + 16 * wave + c;

  read_mask(s.kept, p.mask, b, p.L);
  const int words = (p.L + 63) / 64;
  bool any_kept = false, any_padded = false;
  for (int at2 = i0; at2 < i0 + BQ && at2 < p.L; at2 += 16) {
    const uint64_t kept = kept_from(s.kept, at2, p.L);
    any_kept |= (kept & 0xFFFF) != 0;
    any_padded |= (tokens_from(at2, p.L) & ~kept & 0xFFFF) != 0;
  }
  int first = 0, last = -1;  // blocks of 64 keys that are scored
  if (any_kept) kept_range(s.kept, 0, words, &first, &last);

  const Tokens<T, D> q(p.q, p.sq, b, h, p.L), k(p.k, p.sk, b, h, p.L), v(p.v, p.sv, b, h, p.L);
  const bool has_pk = BOTH || p.pos_key, has_pq = BOTH || p.pos_query;
  Window<T, D, Y::W, BK, NT, LD> pk(static_cast<const T*>(p.pos_key) + h * p.pk_h, p.pk_s, p.lut, p.L,
                                p.S);
  Window<T, D, Y::W, BK, NT, LD> pq(static_cast<const T*>(p.pos_query) + h * p.pq_h, p.pq_s, p.lut,
                                p.L, p.S);
  const bool mine = i < p.L && bit_of(s.kept, i);

  F qf[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) {
    const uint32_t from = mine ? i * q.stride + (32 * ks + 8 * g) * sizeof(T) : kNoRow;
    qf[ks] = load_frag<T>(q.memory, from);
  }

  f32x4_t o[D / 16] = {};
  float top = -INFINITY, sum = 0;
  const __amdgpu_buffer_rsrc_t bits = resource(
      p.bits ? p.bits + static_cast<int64_t>(bh) * p.L * p.bit_row : nullptr,
      p.bits ? p.L * p.bit_row : 0);
  const uint32_t bits_at = i < p.L ? i * static_cast<uint32_t>(p.bit_row) : kNoRow;

  Stage<T, D, BK, NT, LD> next_k, next_v;
  u32x2_t next_word;
  // V of padded keys is needed where a query is padded.
  auto read_v = [&](int j0) {
    next_word = __builtin_amdgcn_raw_buffer_load_b64(bits, bits_at + j0 / 64 * 8, 0, 0);
    next_v.load_tokens(v, j0,
                       (any_padded ? tokens_from(j0, p.L) : kept_from(s.kept, j0, p.L)) & kBlock);
  };
  auto store_v = [&](int j0) {
    const uint64_t padded = tokens_from(j0, p.L) & ~kept_from(s.kept, j0, p.L) & kBlock;
    if (any_padded && padded) next_v.make_finite(padded);
    next_v.store(s.v);
  };
  // The softmax of the scores x[kb][r] of key j0 + 16 kb + 4g + r so far, and the product with V.
  auto add_tile = [&](f32x4_t (&x)[KB], int j0, u32x2_t word) {
    const uint64_t taken =
        (mine ? kept_from(s.kept, j0, p.L) : tokens_from(j0, p.L)) & kBlock;
    if (!__all(taken == kBlock)) {
      const uint64_t lane_taken = taken >> (4 * g);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[kb][r] = (lane_taken >> (16 * kb + r)) & 1 ? x[kb][r] : -INFINITY;
    }
    float high = x[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) high = fmaxf(high, x[kb][r]);
    high = fmaxf(high, __shfl_xor(high, 16));
    high = fmaxf(high, __shfl_xor(high, 32));
    high = fmaxf(high, top);
    const float base = high == -INFINITY ? 0.0f : high;  // (no key is taken so far)
    const float shrink = __builtin_amdgcn_exp2f(top - base);
    top = high;
    sum *= shrink;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) o[db] *= shrink;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[kb][r] = __builtin_amdgcn_exp2f(x[kb][r] - base);
        sum += x[kb][r];
      }
    if (p.bits) {
      const uint64_t kept = ~((static_cast<uint64_t>(word[1]) << 32 | word[0]) >> (j0 % 64));
      drop<KB>(x, kept >> (4 * g));
    }
    // A probability of 16 bits is the operand in two parts, itself rounded and what that left off.
    // Rounded alone it puts an error into D_i = dO_i.O_i that all gradients of a query share, and
    // that weighs more where many deltas have one slot.  Over 2000 tokens in bf16 the gradients were off by
    // 2.7e-3 of their size, with both parts and with `low` by 2.5e-3, and outputs of fp16 by 2.7e-4 and
    // 2.1e-4, their own rounding.  At 32 x 512 padded tokens it takes 247 us instead of 235.
#pragma unroll
    for (int ks = 0; ks < KB / 2; ++ks) {
      const F r = pack<T>(x[2 * ks], x[2 * ks + 1]);
      F rest;
      if constexpr (sizeof(T) == 2) rest = pack<T>(left<T>(x[2 * ks]), left<T>(x[2 * ks + 1]));
#pragma unroll
      for (int db = 0; db < D / 16; ++db) {
        const F values =
            read_columns<T>(s.v + 16 * db, LD, 32 * ks + 4 * g, 32 * ks + 16 + 4 * g, c);
        if constexpr (sizeof(T) == 2) o[db] = Op<T>::run(values, rest, o[db]);
        o[db] = Op<T>::run(values, r, o[db]);
      }
    }
  };

  // The scored tiles.
  if (first <= last) {
    const int stop = first * 64;
    int j0 = last * 64 + 64 - BK;
    const bool wave_kept = __any(mine);
    auto read_tile = [&](int j) {
      read_v(j);
      next_k.load_tokens(k, j, kept_from(s.kept, j, p.L) & kBlock);
    };
    read_tile(j0);
    if (has_pk) {
      pk.fill(s.pk, i0 - j0 - BK);
      pk.read_slots(i0 - j0 - BK);
    }
    if (has_pq) {
      pq.fill(s.pq, i0 - j0 - BK);
      pq.read_slots(i0 - j0 - BK);
    }
    bool begun = false;
    alternate<decltype(pk)::kTwo>([&](auto phase) {
      constexpr int kPhase = decltype(phase)::value;
      lds_barrier();
      store_v(j0);
      next_k.store(s.k);
      if (begun && has_pk) pk.template advance<kPhase>(s.pk);
      if (begun && has_pq) pq.template advance<kPhase>(s.pq);
      lds_barrier();
      const u32x2_t word = next_word;
      if (j0 > stop) {
        read_tile(j0 - BK);
        if (has_pk) {
          pk.read_rows(i0 - j0 - BK);
          pk.read_slots(i0 - j0);
        }
        if (has_pq) {
          pq.read_rows(i0 - j0 - BK);
          pq.read_slots(i0 - j0);
        }
      }

      if (has_pq) {
        // Keys of block kb against deltas from i0 - j0 - 16 kb - 16.
#pragma unroll
        for (int n = 0; n < (KB * (NW + 1) + NW - 1) / NW; ++n) {
          const int at2 = n * NW + wave, kb = at2 % KB, wb = at2 / KB;
          if (at2 < KB * (NW + 1)) {
            const T* from = s.pq + pq.template place<kPhase>(BK - 16 - 16 * kb + 16 * wb) * LD;
            f32x4_t acc{};
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks)
              acc = Op<T>::run(read_row<T>(from + c * LD + 32 * ks, g),
                               read_row<T>(s.k + (16 * kb + c) * LD + 32 * ks, g), acc);
            store4(s.p2c + (16 * kb + c) * LDP + 16 * wb + 4 * g, acc * p.scale_log2);
          }
        }
      }
      f32x4_t x[KB] = {};
      if (wave_kept) {
        if (has_pk) {
          // This wavefront's queries against deltas from i0 + 16 wave - j0 - BK.
#pragma unroll
          for (int wb = 0; wb < KB + 1; ++wb) {
            const T* from = s.pk + pk.template place<kPhase>(16 * wave + 16 * wb) * LD;
            f32x4_t acc{};
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks)
              acc = Op<T>::run(read_row<T>(from + c * LD + 32 * ks, g), qf[ks], acc);
            store4(s.c2p + (16 * wave + c) * LDC + 16 * wb + 4 * g, acc * p.scale_log2);
          }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int ks = 0; ks < D / 32; ++ks)
            x[kb] = Op<T>::run(read_row<T>(s.k + (16 * kb + c) * LD + 32 * ks, g), qf[ks], x[kb]);
      }
      if (has_pk || has_pq) lds_barrier();
      if (wave_kept) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[kb][r] = fmaf(
                x[kb][r], p.scale_log2,
                has_pk ? s.c2p[(16 * wave + c) * LDC + BK + c - 16 * kb - 4 * g - r] : 0.0f);
        if (has_pq) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              x[kb][r] += s.p2c[(16 * kb + 4 * g + r) * LDP + 16 * wave + 16 + c - 4 * g - r];
        }
        if (!__all(mine)) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) x[kb][r] = mine ? x[kb][r] : 0.0f;
        }
      }
      add_tile(x, j0, word);
      begun = true;
      j0 -= BK;
      return j0 >= stop;
    });
  }

  // The tiles that only padded queries see.
  if (any_padded) {
    auto from = [&](int j0) {
      return j0 / 64 >= first && j0 / 64 <= last ? (last + 1) * 64 : j0;
    };
    int j0 = from(0);
    if (j0 < p.L) read_v(j0);
    while (j0 < p.L) {
      lds_barrier();
      store_v(j0);
      lds_barrier();
      const u32x2_t word = next_word;
      const int next = from(j0 + BK);
      if (next < p.L) read_v(next);
      f32x4_t x[KB] = {};
      add_tile(x, j0, word);
      j0 = next;
    }
  }

  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (i >= p.L) return;
  const float factor = p.keep_scale / sum;
  const int64_t to = ((static_cast<int64_t>(b) * p.L + i) * p.H + h) * D + 4 * g;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) {
    o[db] *= factor;
    store4(static_cast<T*>(p.out) + to + 16 * db, o[db]);
  }
  if constexpr (sizeof(T) == 2) {
    if (p.low) {
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        store4(static_cast<T*>(p.low) + to + 16 * db, left<T>(o[db]));
    }
  }
  if (p.lse && g == 0) p.lse[static_cast<int64_t>(bh) * p.L + i] = top + log2f(sum);
}

// ---- D_i = dO_i . O_i -----------------------------------------------------------------------

template <typename T, int D>
__global__ __launch_bounds__(256) void attention_delta_kernel(const T* dout, const T* out,
                                                              const T* low, float* delta, int64_t rows, int H,
                                                              int L) {
  constexpr int N = Chunk<T>::N, kLanes = D / N;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  float sum = 0;
  if (at < rows) {
    float x[N], y[N];
    load_floats<T, N>(dout + at * D + lane * N, x);
    load_floats<T, N>(out + at * D + lane * N, y);
#pragma unroll
    for (int e = 0; e < N; ++e) sum += x[e] * y[e];
    if (low) {
      load_floats<T, N>(low + at * D + lane * N, y);
#pragma unroll
      for (int e = 0; e < N; ++e) sum += x[e] * y[e];
    }
  }
#pragma unroll
  for (int step = 1; step < kLanes; step *= 2) sum += __shfl_xor(sum, step);
  if (at < rows && lane == 0) {
    const int64_t token = at / H;
    const int h = static_cast<int>(at - token * H);
    const int64_t b = token / L;
    delta[(b * H + h) * L + (token - b * L)] = sum;
  }
}

// ---- dV, dK and G ---------------------------------------------------------------------------

// A workgroup of NW wavefronts takes 16 NW keys, 16 a wavefront, and walks the queries in tiles of
// BQ.  A lane holds one key and four queries of a block.
template <typename T, int D, int NW, int BQ>
struct KeyLayout {
  static constexpr int BK = 16 * NW, WQ = BK + 16, WK = BQ + 16;
  static constexpr int LDC = WQ + 4, LDP = WK + 4;
  static constexpr int LDF = WK + 8;
  static constexpr int LD = kLdWide<T, D>;
  static constexpr int W = BQ + BK;
  static constexpr int kWide = BK < 64 ? 1 : BK / 64;  // words of the generator's bits a query
  // A wavefront's scores of its keys by delta, and after them G by delta.
  static constexpr int kScores = 16 * LDP * static_cast<int>(sizeof(float));
  static constexpr int kSkew = 16 * LDF * static_cast<int>(sizeof(T));
  T q[BQ * LD], dout[BQ * LD], pk[W * LD], pq[W * LD];
  float c2p[BQ * LDC];
  unsigned char own[NW * (kScores > kSkew ? kScores : kSkew)];
  float lse[BQ], delta[BQ];
  uint16_t places[NW][BQ];  // bit c of a wavefront's row: the place of key c is kept
  uint64_t kept[kWords];
};

template <typename T, int D, int NW, int BQ, bool BOTH>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 ? 2 : 1)))
void attention_train_key_kernel(Params p) {
  using Y = KeyLayout<T, D, NW, BQ>;
  using F = typename Op<T>::frag;
  constexpr int BK = Y::BK, LD = Y::LD, LDC = Y::LDC, LDP = Y::LDP, LDF = Y::LDF, NT = 64 * NW;
  constexpr int QB = BQ / 16, kWide = Y::kWide;
  constexpr uint64_t kBlock = BQ == 64 ? ~uint64_t{0} : (uint64_t{1} << (BQ % 64)) - 1;
  extern __shared__ __align__(16) unsigned char memory[];
  Y& s = *reinterpret_cast<Y*>(memory);
  const int words = (p.L + 63) / 64;
  const int blocks = (words * 64 + BK - 1) / BK;
  const int at = xcd_logical_block(blockIdx.x, gridDim.x);
  const int pair = at / blocks, j0 = at % blocks * BK;
  const int b = p.b0 + pair / p.nh, h = p.h0 + pair % p.nh;
  const int64_t bh = static_cast<int64_t>(b) * p.H + h;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, c = lane % 16, g = lane / 16;
  const int j = j0 + 16 * wave + c;
  float* scores = reinterpret_cast<float*>(s.own + wave * (sizeof(s.own) / NW));
  T* skew = reinterpret_cast<T*>(scores);

  read_mask(s.kept, p.mask, b, p.L);
  if (h == p.h0 && j0 == 0)
    for (int n = threadIdx.x; n < words; n += NT)
      p.words[static_cast<int64_t>(b) * words + n] = s.kept[n];
  const bool mine = j < p.L && bit_of(s.kept, j);
  const float even = 1.0f / static_cast<float>(p.L);
  // The queries' blocks that are scored; none where no key of the block is kept.
  int first = 0, last = -1, key_first, key_last;
  kept_range(s.kept, j0 / 64, min((j0 + BK + 63) / 64, words), &key_first, &key_last);
  if (key_first <= key_last) kept_range(s.kept, 0, words, &first, &last);

  const Tokens<T, D> q(p.q, p.sq, b, h, p.L), k(p.k, p.sk, b, h, p.L), v(p.v, p.sv, b, h, p.L);
  const int64_t row = static_cast<int64_t>(p.H) * D;
  const Tokens<T, D> dout(p.dout, Strides{p.L * row, D, row}, b, h, p.L);
  const bool has_pk = BOTH || p.pos_key, has_pq = BOTH || p.pos_query;
  Window<T, D, Y::W, BQ, NT, LD> pk(static_cast<const T*>(p.pos_key) + h * p.pk_h, p.pk_s, p.lut, p.L,
                                 p.S);
  Window<T, D, Y::W, BQ, NT, LD> pq(static_cast<const T*>(p.pos_query) + h * p.pq_h, p.pq_s, p.lut,
                                 p.L, p.S);
  // Fragments of this pair: [16 keys][32 queries].
  const int q32 = 2 * words;
  const int64_t pair_bytes = static_cast<int64_t>(2 * q32) * q32 * kFragment * sizeof(T);
  const __amdgpu_buffer_rsrc_t out_g =
      resource(static_cast<const char*>(p.g) + pair * pair_bytes, pair_bytes);
  // (Past the last keys' fragments nothing is written.)
  const uint32_t g_at =
      j0 + 16 * wave < 64 * words
          ? static_cast<uint32_t>(((j0 / 16 + wave) * q32 * kFragment + lane * 8) * sizeof(T))
          : kNoRow;

  F kf[D / 32], vf[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) {
    const uint32_t in_row = (32 * ks + 8 * g) * sizeof(T);
    kf[ks] = load_frag<T>(k.memory, mine ? j * k.stride + in_row : kNoRow);
    vf[ks] = load_frag<T>(v.memory, j < p.L ? j * v.stride + in_row : kNoRow);
  }
  f32x4_t dk[D / 16] = {}, dv[D / 16] = {};

  Stage<T, D, BQ, NT, LD> next_q, next_dout;
  float next_lse = 0, next_delta = 0;
  u32x2_t next_dropped{};
  static_assert(BQ * kWide <= NT, "one word of dropped places a thread");
  const __amdgpu_buffer_rsrc_t bits = resource(p.bits ? p.bits + bh * p.L * p.bit_row : nullptr,
                                               p.bits ? p.L * p.bit_row : 0);
  auto read_rest = [&](int i0) {
    next_dout.load_tokens(dout, i0, tokens_from(i0, p.L));
    const int r = threadIdx.x / kWide, word = j0 / 64 + threadIdx.x % kWide;
    next_dropped = __builtin_amdgcn_raw_buffer_load_b64(
        bits,
        r < BQ && word < words ? (i0 + r) * static_cast<uint32_t>(p.bit_row) + word * 8 : kNoRow, 0,
        0);
  };
  auto store_rest = [&]() {
    next_dout.store(s.dout);
    const int r = threadIdx.x / kWide, word = threadIdx.x % kWide;
    if (r < BQ) {
      uint64_t kept = ~(static_cast<uint64_t>(next_dropped[1]) << 32 | next_dropped[0]);
      if (NW < 4) kept >>= j0 % 64;
#pragma unroll
      for (int n = 0; n < (NW < 4 ? NW : 4); ++n)
        s.places[4 * word + n][r] = static_cast<uint16_t>(kept >> (16 * n));
    }
  };
  // Query 4g + r of block qb and this lane's key: all ones where the place is kept.
  typedef uint32_t Kept __attribute__((ext_vector_type(2)));
  auto kept_of = [&](int qb) {
    return *reinterpret_cast<const Kept*>(&s.places[wave][16 * qb + 4 * g]);
  };
  auto mask_of = [&](Kept kept, int r) {
    return __builtin_amdgcn_sbfe(static_cast<int>(kept[r / 2]), c + r % 2 * 16, 1);
  };
  auto masked = [](float x, int mask) {
    return __builtin_bit_cast(float, __builtin_bit_cast(int, x) & mask);
  };
  // dV += R^T dO of a tile, R as an operand.  (R is rounded to T: off by half a step of each.)
  auto add_dv = [&](const f32x4_t (&x)[QB]) {
#pragma unroll
    for (int ks = 0; ks < QB / 2; ++ks) {
      const F r = pack<T>(x[2 * ks], x[2 * ks + 1]);
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        dv[db] = Op<T>::run(
            read_columns<T>(s.dout + 16 * db, LD, 32 * ks + 4 * g, 32 * ks + 16 + 4 * g, c), r,
            dv[db]);
    }
  };

  if (first <= last) {
    const __amdgpu_buffer_rsrc_t lse = resource(p.lse + bh * p.L, 4 * static_cast<int64_t>(p.L));
    const __amdgpu_buffer_rsrc_t delta = resource(p.delta + bh * p.L, 4 * static_cast<int64_t>(p.L));
    auto read_tile = [&](int i0) {
      read_rest(i0);
      next_q.load_tokens(q, i0, kept_from(s.kept, i0, p.L) & kBlock);
      const uint32_t at2 = threadIdx.x < BQ ? 4 * (i0 + threadIdx.x) : kNoRow;
      next_lse = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(lse, at2, 0, 0));
      next_delta = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(delta, at2, 0, 0));
    };
    const int stop = 64 * last + 64 - BQ;
    int i0 = 64 * first;
    read_tile(i0);
    if (has_pk) {
      pk.fill(s.pk, i0 - j0 - BK);
      pk.read_slots(i0 - j0 - BK);
    }
    if (has_pq) {
      pq.fill(s.pq, i0 - j0 - BK);
      pq.read_slots(i0 - j0 - BK);
    }
    bool begun = false;
    alternate<decltype(pk)::kTwo>([&](auto phase) {
      constexpr int kPhase = decltype(phase)::value;
      lds_barrier();
      store_rest();
      next_q.store(s.q);
      if (threadIdx.x < BQ) {
        s.lse[threadIdx.x] = next_lse;
        s.delta[threadIdx.x] = next_delta;
      }
      if (begun && has_pk) pk.template advance<kPhase>(s.pk);
      if (begun && has_pq) pq.template advance<kPhase>(s.pq);
      lds_barrier();
      if (i0 < stop) {
        read_tile(i0 + BQ);
        if (has_pk) {
          pk.read_rows(i0 - j0 - BK);
          pk.read_slots(i0 + BQ - j0 - BK);
        }
        if (has_pq) {
          pq.read_rows(i0 - j0 - BK);
          pq.read_slots(i0 + BQ - j0 - BK);
        }
      }

      f32x4_t x[QB] = {}, y[QB] = {};  // [qb][r]: query i0 + 16 qb + 4g + r
      if (has_pk) {
        // Blocks of 16 queries against deltas from i0 + 16 qb - j0 - BK, shared by the wavefronts.
#pragma unroll
        for (int n = 0; n < (QB * (NW + 1) + NW - 1) / NW; ++n) {
          const int at2 = n * NW + wave, qb = at2 % QB, wb = at2 / QB;
          if (at2 < QB * (NW + 1)) {
            const T* from = s.pk + pk.template place<kPhase>(16 * qb + 16 * wb) * LD;
            f32x4_t acc{};
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks)
              acc = Op<T>::run(read_row<T>(from + c * LD + 32 * ks, g),
                               read_row<T>(s.q + (16 * qb + c) * LD + 32 * ks, g), acc);
            store4(s.c2p + (16 * qb + c) * LDC + 16 * wb + 4 * g, acc * p.scale_log2);
          }
        }
      }
      if (has_pq) {
        // This wavefront's keys against deltas from i0 - j0 - 16 wave - 16.
#pragma unroll
        for (int wb = 0; wb < QB + 1; ++wb) {
          const T* from = s.pq + pq.template place<kPhase>(BK - 16 - 16 * wave + 16 * wb) * LD;
          f32x4_t acc{};
#pragma unroll
          for (int ks = 0; ks < D / 32; ++ks)
            acc = Op<T>::run(read_row<T>(from + c * LD + 32 * ks, g), kf[ks], acc);
          store4(scores + c * LDP + 16 * wb + 4 * g, acc * p.scale_log2);
        }
      }
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
          x[qb] = Op<T>::run(read_row<T>(s.q + (16 * qb + c) * LD + 32 * ks, g), kf[ks], x[qb]);
          y[qb] = Op<T>::run(read_row<T>(s.dout + (16 * qb + c) * LD + 32 * ks, g), vf[ks], y[qb]);
        }
      if (has_pk) lds_barrier();
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[qb][r] = fmaf(
              x[qb][r], p.scale_log2,
              has_pk ? s.c2p[(16 * qb + 4 * g + r) * LDC + 4 * g + r - c - 16 * wave + BK] : 0.0f);
      if (has_pq) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[qb][r] += scores[c * LDP + 16 * qb + 4 * g + r - c + 16];
      }
      // P, and P (M dP - D).
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const f32x4_t lse = *reinterpret_cast<const f32x4_t*>(s.lse + 16 * qb + 4 * g);
        const f32x4_t delta = *reinterpret_cast<const f32x4_t*>(s.delta + 16 * qb + 4 * g);
        const Kept kept = kept_of(qb);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[qb][r] = __builtin_amdgcn_exp2f(x[qb][r] - lse[r]);
          const int mask = mask_of(kept, r);
          y[qb][r] = x[qb][r] * fmaf(masked(y[qb][r], mask), p.keep_scale, -delta[r]);
          x[qb][r] = masked(x[qb][r], mask);
        }
      }
      const uint64_t kept = kept_from(s.kept, i0, p.L) & kBlock;
      // (One token has one probability, 1, and no gradient.)
      if (kept != kBlock || !__all(mine) || p.L == 1) {
        // By bits, which drops NaN too.
        const uint64_t inside = tokens_from(i0, p.L);
        const uint64_t live = mine ? kept >> (4 * g) : 0;
        const uint64_t padded = j < p.L ? (inside & ~kept) >> (4 * g) : 0;
        const int graded = p.L > 1 ? -1 : 0;
        auto field = [](uint64_t bits, int at) {
          return __builtin_amdgcn_sbfe(static_cast<int>(bits >> (at / 32 * 32)), at % 32, 1);
        };
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const Kept places = kept_of(qb);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int scored = field(live, 16 * qb + r);
            const int uniform = field(padded, 16 * qb + r) & mask_of(places, r);
            x[qb][r] = __builtin_bit_cast(
                float, (__builtin_bit_cast(int, static_cast<float>(x[qb][r])) & scored) |
                           (__builtin_bit_cast(int, even) & uniform));
            y[qb][r] = masked(y[qb][r], scored & graded);
          }
        }
      }
      add_dv(x);
      asm volatile("" ::: "memory");  // (`skew` takes the place of `scores`)
      if (has_pq) {
        // Places outside the band, which is 16 - c .. 15 - c + BQ of row c.
        constexpr int kPer = 16 / static_cast<int>(sizeof(T));
        constexpr int kLow = 16 / kPer, kChunks = 2 * kLow;
        for (int n = lane; n < 16 * kChunks; n += 64) {
          const int chunk = n % kChunks;
          *reinterpret_cast<u32x4_t*>(skew + n / kChunks * LDF +
                                      (chunk < kLow ? chunk * kPer : BQ + (chunk - kLow) * kPer)) =
              u32x4_t{};
        }
        asm volatile("" ::: "memory");
      }
      // (G is rounded to T as an operand and as it is stored: off by half a step of each.)
#pragma unroll
      for (int ks = 0; ks < QB / 2; ++ks) {
        const F dg = pack<T>(y[2 * ks], y[2 * ks + 1]);
        store_frag<T>(out_g, g_at + (i0 / 32 + ks) * static_cast<uint32_t>(kFragment * sizeof(T)),
                      dg);
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          dk[db] = Op<T>::run(
              read_columns<T>(s.q + 16 * db, LD, 32 * ks + 4 * g, 32 * ks + 16 + 4 * g, c), dg,
              dk[db]);
        if (has_pq) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            skew[c * LDF + 32 * ks + (e < 4 ? e : 12 + e) + 4 * g - c + 16] = dg[e];
        }
      }
      if (has_pq) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int ks = 0; ks < BQ / 32; ++ks) {
          const F sk = read_row<T>(skew + c * LDF + 32 * ks, g);
          const int lo =
              pq.template place<kPhase>(BK - 16 - 16 * wave + 32 * ks + 16 * (g / 2)) + 8 * (g % 2);
#pragma unroll
          for (int db = 0; db < D / 16; ++db)
            dk[db] = Op<T>::run(read_columns<T>(s.pq + 16 * db, LD, lo, lo + 4, c), sk, dk[db]);
        }
        const auto sk = *reinterpret_cast<const Quad<T>*>(skew + c * LDF + BQ + 4 * g);
        const int lo = pq.template place<kPhase>(BK - 16 - 16 * wave + BQ) + 4 * g;
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          dk[db] = Op<T>::run_half(read_columns_half<T>(s.pq + 16 * db, LD, lo, c), sk, dk[db]);
      }
      begun = true;
      i0 += BQ;
      return i0 <= stop;
    });
  }

  // Padded queries of the tiles that are not scored: 1 / L for every key.
  auto padded_of = [&](int i0) {
    return tokens_from(i0, p.L) & ~kept_from(s.kept, i0, p.L) & kBlock;
  };
  auto from = [&](int i0) {  // the first such tile from i0 on
    while (i0 < p.L && ((i0 / 64 >= first && i0 / 64 <= last) || padded_of(i0) == 0)) i0 += BQ;
    return i0;
  };
  int i0 = from(0);
  if (i0 < p.L) read_rest(i0);
  while (i0 < p.L) {
    lds_barrier();
    store_rest();
    lds_barrier();
    const uint64_t padded = padded_of(i0) >> (4 * g);
    i0 = from(i0 + BQ);
    if (i0 < p.L) read_rest(i0);
    f32x4_t x[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const Kept kept = kept_of(qb);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        x[qb][r] = (padded >> (16 * qb + r)) & 1 && j < p.L ? masked(even, mask_of(kept, r)) : 0.0f;
    }
    add_dv(x);
  }

  if (j >= p.L) return;
  const int64_t base = ((static_cast<int64_t>(b) * p.L + j) * p.H + h) * D;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) {
    store4(static_cast<T*>(p.dk) + base + 16 * db + 4 * g, dk[db] * p.scale);
    store4(static_cast<T*>(p.dv) + base + 16 * db + 4 * g, dv[db] * p.keep_scale);
  }
}

// ---- dQ ---------------------------------------------------------------------------------------

template <typename T, int D>
struct QueryLayout {
  static constexpr int LD = kLd<T, D>, LDG = kLd<T, 64>, LDE = 80 + 8;
  static constexpr int W = 128;
  T k[64 * LD], pk[W * LD];
  T g[64 * LDG];     // [key][query]
  T skew[64 * LDE];  // [query][delta]
  uint64_t kept[kWords];
};

// Element e of lane group g's eight of a fragment: which of its 32 queries.
__device__ inline int query_of(int g, int e) { return 4 * g + (e < 4 ? e : 12 + e); }

template <typename T, int D>
__global__ __launch_bounds__(256) void attention_train_query_kernel(Params p) {
  using Y = QueryLayout<T, D>;
  using F = typename Op<T>::frag;
  constexpr int LD = Y::LD, LDG = Y::LDG, LDE = Y::LDE;
  extern __shared__ __align__(16) unsigned char memory[];
  Y& s = *reinterpret_cast<Y*>(memory);
  const int blocks = (p.L + 63) / 64;
  const int at = xcd_logical_block(blockIdx.x, gridDim.x);
  const int pair = at / blocks, i0 = at % blocks * 64;
  const int b = p.b0 + pair / p.nh, h = p.h0 + pair % p.nh;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, c = lane % 16, g = lane / 16;
  const int i = i0 + 16 * wave + c;
  read_mask(s.kept, p.mask, b, p.L);
  for (int n = threadIdx.x; n < 64 * LDE; n += 256) s.skew[n] = static_cast<T>(0.0f);

  int first, last;
  kept_range(s.kept, 0, blocks, &first, &last);
  const Tokens<T, D> k(p.k, p.sk, b, h, p.L);
  const bool has_pk = p.pos_key;
  Window<T, D, Y::W, 64, 256> pk(static_cast<const T*>(p.pos_key) + h * p.pk_h, p.pk_s, p.lut, p.L,
                                 p.S);
  const int q32 = 2 * blocks;
  const T* fragments = static_cast<const T*>(p.g) +
                       (static_cast<int64_t>(pair) * 2 * q32 + wave) * q32 * kFragment +
                       static_cast<int64_t>(i0 / 32) * kFragment + lane * 8;
  f32x4_t dq[D / 16] = {};
  if (s.kept[i0 / 64] != 0) {
    Stage<T, D, 64, 256> next_k;
    F next_g[2];
    auto read_tile = [&](int jb) {
      const uint64_t kept = s.kept[jb];
      next_k.load_tokens(k, 64 * jb, kept);
      // (G of a block of keys without a kept one may not have been written.)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        next_g[n] = F{};
        if (kept)
          next_g[n] = *reinterpret_cast<const F*>(
              fragments + (static_cast<int64_t>(4 * jb) * q32 + n) * kFragment);
      }
    };
    // The last keys first: the window moves up.
    int jb = last;
    read_tile(jb);
    if (has_pk) {
      pk.fill(s.pk, i0 - 64 * jb - 64);
      pk.read_slots(i0 - 64 * jb - 64);
    }
    bool begun = false;
    alternate<decltype(pk)::kTwo>([&](auto phase) {
      constexpr int kPhase = decltype(phase)::value;
      lds_barrier();
      next_k.store(s.k);
      const int key = 16 * wave + c;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        Quad<T> four;
#pragma unroll
        for (int e = 0; e < 4; ++e) four[e] = next_g[n / 2][4 * (n % 2) + e];
        *reinterpret_cast<Quad<T>*>(s.g + key * LDG + 16 * n + 4 * g) = four;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int query = 32 * n + query_of(g, e);
          if (has_pk) s.skew[query * LDE + query % 16 - key + 64] = next_g[n][e];
        }
      if (begun && has_pk) pk.template advance<kPhase>(s.pk);
      lds_barrier();
      if (jb > first) {
        read_tile(jb - 1);
        if (has_pk) {
          pk.read_rows(i0 - 64 * jb - 64);
          pk.read_slots(i0 - 64 * jb);
        }
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const int lo = 32 * ks + 8 * g;
        const F dg = read_columns<T>(s.g + 16 * wave, LDG, lo, lo + 4, c);
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          dq[db] = Op<T>::run(read_columns<T>(s.k + 16 * db, LD, lo, lo + 4, c), dg, dq[db]);
      }
      if (has_pk) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const F sk = read_row<T>(s.skew + (16 * wave + c) * LDE + 32 * ks, g);
          const int lo = pk.template place<kPhase>(16 * wave + 32 * ks + 16 * (g / 2)) + 8 * (g % 2);
#pragma unroll
          for (int db = 0; db < D / 16; ++db)
            dq[db] = Op<T>::run(read_columns<T>(s.pk + 16 * db, LD, lo, lo + 4, c), sk, dq[db]);
        }
        const auto sk = *reinterpret_cast<const Quad<T>*>(s.skew + (16 * wave + c) * LDE + 64 + 4 * g);
        const int lo = pk.template place<kPhase>(16 * wave + 64) + 4 * g;
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          dq[db] = Op<T>::run_half(read_columns_half<T>(s.pk + 16 * db, LD, lo, c), sk, dq[db]);
      }
      begun = true;
      return --jb >= first;
    });
  }
  if (i >= p.L) return;
  T* out = static_cast<T*>(p.dq) + ((static_cast<int64_t>(b) * p.L + i) * p.H + h) * D;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) store4(out + 16 * db + 4 * g, dq[db] * p.scale);
}

// ---- dPK and dPQ by delta -------------------------------------------------------------------

// The tiles of 64 x 64 with (query block) - (key block) = m, of all sequences of one head, share
// their deltas, 64 m - 63 .. 64 m + 63: place 64 + (i - j) - 64 m of 128.  2^`shift` of them are one
// workgroup's; the parts of a diagonal are added up by the next kernel.  Every diagonal has the
// room of the longest, m = 0.
struct Diagonals {
  int blocks, batch, shift;
  __host__ __device__ int count() const { return 2 * blocks - 1; }
  __host__ __device__ int tiles(int m) const { return batch * (blocks - (m < 0 ? -m : m)); }
  __host__ __device__ int parts(int m) const {
    return (tiles(m) + (1 << shift) - 1) >> shift;
  }
  // Diagonals in the order 0, 1, -1, 2, -2, ..: the longest first.
  __host__ __device__ static int nth(int n) { return n % 2 ? (n + 1) / 2 : -(n / 2); }
  __host__ __device__ static int order(int m) { return m > 0 ? 2 * m - 1 : -2 * m; }
  __host__ __device__ int per_head() const { return count() * parts(0); }
  // The first part of diagonal m.
  __host__ __device__ int64_t first(int head, int m) const {
    return static_cast<int64_t>(head) * per_head() + order(m) * parts(0);
  }
};

template <typename T, int D>
struct PositionLayout {
  static constexpr int LD = kLd<T, D>, LDX = kLd<T, 32>;
  T q[64 * LD], k[64 * LD];
  // [half][place][query or key]: 32 queries meet 96 of the 128 places, from 0 or 32 on, and
  // 32 keys from 32 or 0 on.  (All 128 left room for two workgroups of heads of 64 a CU, not
  // three: 112 us instead of 97 at 32 x 512 padded tokens.)
  T by_query[2 * 96 * LDX], by_key[2 * 96 * LDX];
  uint64_t kept[64][2];                      // of the part's tiles: the queries' and the keys' bits,
  int at[64][2];                             // sequence and block of queries
};

template <typename T, int D>
__global__ __launch_bounds__(256) void attention_train_position_kernel(Params p, Diagonals dg) {
  using Y = PositionLayout<T, D>;
  using F = typename Op<T>::frag;
  constexpr int LD = Y::LD, LDX = Y::LDX;
  extern __shared__ __align__(16) unsigned char memory[];
  Y& s = *reinterpret_cast<Y*>(memory);
  // Heads first, then parts: the long diagonals start first.
  const int hh = blockIdx.x % p.nh, part = blockIdx.x / p.nh % dg.parts(0);
  const int m = Diagonals::nth(blockIdx.x / p.nh / dg.parts(0));
  if (part >= dg.parts(m)) return;
  const int along = dg.blocks - (m < 0 ? -m : m);
  const int h = p.h0 + hh;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int lane = threadIdx.x % 64, c = lane % 16, g = lane / 16;
  for (int x = threadIdx.x; x < 2 * 96 * LDX; x += 256) {
    s.by_query[x] = static_cast<T>(0.0f);
    s.by_key[x] = static_cast<T>(0.0f);
  }
  const int q32 = 2 * dg.blocks;
  const bool pk = p.pos_key != nullptr, pq = p.pos_query != nullptr;
  f32x4_t dpk[2][D / 16] = {}, dpq[2][D / 16] = {};
  // The part's tiles are looked up together, one a lane, and those with kept queries and keys are
  // remembered as bits (looked up one by one, with a
  // division each, 24576 tiles took 164 us instead of 162).
  const int begin = part << dg.shift, end = min((part + 1) << dg.shift, dg.tiles(m));
  uint64_t live;
  {
    const int u = begin + lane, bb = u / along, qt = u % along + (m > 0 ? m : 0);
    uint64_t kept[2] = {0, 0};
    if (u < end) {
      const uint64_t* words = p.words + static_cast<int64_t>(p.b0 + bb) * dg.blocks;
      kept[0] = words[qt];
      kept[1] = words[qt - m];
    }
    live = __ballot(kept[0] != 0 && kept[1] != 0);
    if (wave == 0) {
      s.kept[lane][0] = kept[0];
      s.kept[lane][1] = kept[1];
      s.at[lane][0] = bb;
      s.at[lane][1] = qt;
    }
  }
  __syncthreads();
  Stage<T, D, 64, 256> next_q, next_k;
  F next_g[2];
  // Reads the next live tile.
  auto read_tile = [&]() {
    const int u = __builtin_ctzll(live);
    live &= live - 1;
    const int bb = __builtin_amdgcn_readfirstlane(s.at[u][0]);
    const int qt = __builtin_amdgcn_readfirstlane(s.at[u][1]), kt = qt - m;
    const T* fragments =
        static_cast<const T*>(p.g) +
        ((static_cast<int64_t>(bb * p.nh + hh) * 2 * q32 + 4 * kt + wave) * q32 + 2 * qt) *
            kFragment +
        lane * 8;
#pragma unroll
    for (int x = 0; x < 2; ++x)
      next_g[x] = *reinterpret_cast<const F*>(fragments + x * kFragment);
    const int b = p.b0 + bb;
    if (pk) next_q.load_tokens(Tokens<T, D>(p.q, p.sq, b, h, p.L), 64 * qt, s.kept[u][0]);
    if (pq) next_k.load_tokens(Tokens<T, D>(p.k, p.sk, b, h, p.L), 64 * kt, s.kept[u][1]);
  };
  bool more = live != 0;
  if (more) read_tile();
  while (more) {
    lds_barrier();
    if (pk) next_q.store(s.q);
    if (pq) next_k.store(s.k);
    const int key = 16 * wave + c;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int query = query_of(g, e), place = 64 + 32 * x + query - key;
        if (pk) s.by_query[(64 * x + place) * LDX + query] = next_g[x][e];
        if (pq) s.by_key[(128 * (wave / 2) - 32 + place) * LDX + key % 32] = next_g[x][e];
      }
    lds_barrier();
    more = live != 0;
    if (more) read_tile();
    // Blocks of 16 places `wave` and `wave` + 4; those that a step of 32 queries or keys does not
    // reach are left out.
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int lo = 32 * ks + 8 * g;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int wb = wave + 4 * half;
        if (pk && (ks == 0 ? wb < 6 : wb >= 2)) {
          const F x = read_row<T>(s.by_query + (64 * ks + 16 * wb + c) * LDX, g);
#pragma unroll
          for (int db = 0; db < D / 16; ++db)
            dpk[half][db] = Op<T>::run(read_columns<T>(s.q + 16 * db, LD, lo, lo + 4, c), x,
                                       dpk[half][db]);
        }
        if (pq && (ks == 0 ? wb >= 2 : wb < 6)) {
          const F x = read_row<T>(s.by_key + (128 * ks - 32 + 16 * wb + c) * LDX, g);
#pragma unroll
          for (int db = 0; db < D / 16; ++db)
            dpq[half][db] = Op<T>::run(read_columns<T>(s.k + 16 * db, LD, lo, lo + 4, c), x,
                                       dpq[half][db]);
        }
      }
    }
  }
  float* out = p.partial + (dg.first(hh, m) + part) * 256 * D;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float* to = out + (16 * (wave + 4 * half) + c) * D + 4 * g;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      *reinterpret_cast<f32x4_t*>(to + 16 * db) = dpk[half][db];
      *reinterpret_cast<f32x4_t*>(to + 128 * D + 16 * db) = dpq[half][db];
    }
  }
}

// ---- dPK and dPQ by slot --------------------------------------------------------------------

// The parts of a diagonal are added up in the place of its first.  256 threads take 1024 of its
// 256 D sums.
__global__ __launch_bounds__(256) void attention_train_parts_kernel(float* partial, int D,
                                                                    Diagonals dg) {
  const int m = Diagonals::nth(blockIdx.y), parts = dg.parts(m);
  const int64_t step = 256 * D;
  float* at = partial + dg.first(blockIdx.z, m) * step + (blockIdx.x * 256 + threadIdx.x) * 4;
  f32x4_t sum{};
#pragma unroll 4
  for (int n = 0; n < parts; ++n) sum += *reinterpret_cast<const f32x4_t*>(at + n * step);
  *reinterpret_cast<f32x4_t*>(at) = sum;
}

// One workgroup for a slot of a head: the sums of its deltas, each of two diagonals.
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_train_slot_kernel(
    const float* partial, const int32_t* lut, T* dpos_key, T* dpos_query, float* carry, int first,
    int last, int L, int S, int H, int h0, Diagonals dg, float scale) {
  constexpr int kThreads = 256, kLanes = D / 4, kGroups = kThreads / kLanes;
  constexpr int kSpan = 4096;  // deltas looked through at a time
  __shared__ f32x4_t sums[2][kThreads];
  __shared__ int16_t found[kSpan];
  __shared__ int counts[kThreads / 64];
  const int slot = blockIdx.x, hh = blockIdx.y;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int wave = threadIdx.x / 64, bit = threadIdx.x % 64;
  f32x4_t sum[2] = {};
  const __amdgpu_buffer_rsrc_t table = resource(lut, (2 * static_cast<int64_t>(L) - 1) * 4);
  for (int from = 0; from < 2 * L - 1; from += kSpan) {
    // The deltas of this slot are listed, each wavefront's 1024 in an order of its own: four loads of
    // four places a lane, all in flight together.
    constexpr int kLoads = kSpan / kThreads / 4;
    u32x4_t places[kLoads];
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      places[n] = __builtin_amdgcn_raw_buffer_load_b128(
          table, 4 * (from + (wave * kLoads + n) * 256 + 4 * bit), 0, 0);
    uint64_t match[kLoads][4];
    int mine = 0;
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = from + (wave * kLoads + n) * 256 + 4 * bit + e;
        match[n][e] = __ballot(at < 2 * L - 1 && static_cast<int>(places[n][e]) == slot);
        mine += __popcll(match[n][e]);
      }
    __syncthreads();
    if (bit == 0) counts[wave] = mine;
    __syncthreads();
    int total = 0, to = 0;
#pragma unroll
    for (int n = 0; n < kThreads / 64; ++n) {
      if (n == wave) to = total;
      total += counts[n];
    }
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if ((match[n][e] >> bit) & 1)
          found[to + __popcll(match[n][e] & ((uint64_t{1} << bit) - 1))] =
              static_cast<int16_t>((wave * kLoads + n) * 256 + 4 * bit + e);
        to += __popcll(match[n][e]);
      }
    __syncthreads();
    // Twice each: delta = 64 lower + place is place 64 + place of the diagonal `lower` and `place` of
    // the next.  (Without branches, so that eight are in flight.  Where there is no such diagonal
    // place 0 is read, which no delta has.)
#pragma unroll 8
    for (int n = group; n < 2 * total; n += kGroups) {
      const int x = n & 1, up = from + found[n >> 1] - (L - 1) + 64 * dg.blocks;
      const int m = up / 64 - dg.blocks + x;
      const bool none = m <= -dg.blocks || m >= dg.blocks;
      const float* at = partial + dg.first(hh, none ? 0 : m) * 256 * D +
                        (none ? 0 : 64 - 64 * x + up % 64) * D + lane * 4;
      sum[0] += *reinterpret_cast<const f32x4_t*>(at);
      sum[1] += *reinterpret_cast<const f32x4_t*>(at + 128 * D);
    }
  }
  sums[0][threadIdx.x] = sum[0];
  sums[1][threadIdx.x] = sum[1];
  __syncthreads();
  if (group >= 2) return;
  T* out = group ? dpos_query : dpos_key;
  if (!out) return;
  const int64_t at = (static_cast<int64_t>(slot) * H + h0 + hh) * D + lane * 4;
  f32x4_t total{};
  for (int n = 0; n < kGroups; ++n) total += sums[group][n * kLanes + lane];
  // (Launches over parts of the batch add up in `carry`.)
  f32x4_t* kept = reinterpret_cast<f32x4_t*>(carry + group * static_cast<int64_t>(S) * H * D + at);
  if (!first) total += *kept;
  if (last)
    store4(out + at, total * scale);
  else
    *kept = total;
}

// ---- host -------------------------------------------------------------------------------------

// Of 16-bit rows of 32 or 64 elements workgroups of four wavefronts, two to four to a CU by their LDS
// (34 to 67 KB); of eight, whose windows serve twice the rows, the kernels took 10 % longer there (key
// kernel 321 -> 353 us, forward, by an earlier build with scores in fp16, 220 -> 249
// at 32 x 512 full tokens).  Rows of 128 have room for one
// workgroup, of eight.  In fp32 as many wavefronts as fit.  Tiles are of 32 tokens (64 in fp32, where one
// workgroup fits a CU either way): with 64 the key kernel spilled registers.
template <typename T, int D>
struct Sizes {
  static constexpr bool kWord = sizeof(T) == 4;
  static constexpr int kFwdWaves = !kWord ? (D == 128 ? 8 : 4) : D == 32 ? 8 : D == 64 ? 4 : 2;
  static constexpr int kFwdKeys = kWord && D != 128 ? 64 : 32;
  static constexpr int kKeyWaves = !kWord ? (D == 128 ? 8 : 4) : D == 32 ? 8 : D == 64 ? 4 : 2;
  static constexpr int kKeyQueries = 32;
};

int hip_code(hipError_t e) { return static_cast<int>(e); }

template <typename T, int D, bool BOTH>
int launch_forward(const Params& p, hipStream_t stream) {
  constexpr int NW = Sizes<T, D>::kFwdWaves, BK = Sizes<T, D>::kFwdKeys;
  using Y = FwdLayout<T, D, NW, BK>;
  static_assert(sizeof(Y) <= 160 * 1024, "LDS");
  const int64_t blocks = static_cast<int64_t>((p.L + Y::BQ - 1) / Y::BQ) * p.B * p.H;
  if (blocks > kMaxBlocks256) return DFLASH_ERR_TOO_LARGE;
  hipError_t e = ensure_dynamic_lds<&attention_train_fwd_kernel<T, D, NW, BK, BOTH>>(sizeof(Y));
  if (e != hipSuccess) return hip_code(e);
  hipLaunchKernelGGL((attention_train_fwd_kernel<T, D, NW, BK, BOTH>),
                     dim3(static_cast<uint32_t>(blocks)), dim3(64 * NW), sizeof(Y), stream, p);
  return hip_code(hipGetLastError());
}

// How the backward pass divides its work.
struct Plan {
  int batch, heads;  // (batch, head) pairs of one launch: all heads, or some of one batch
  int blocks, shift;
  size_t g, partial, carry, delta, words, total;
};

constexpr size_t kMostG = size_t{2} << 30;

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

Plan make_plan(int B, int H, int L, int S, int D, int esize) {
  Plan x{};
  x.blocks = (L + 63) / 64;
  const size_t each = static_cast<size_t>(x.blocks) * x.blocks * 4096 * esize;
  const size_t fit = kMostG / each > 0 ? kMostG / each : 1;
  x.heads = fit >= static_cast<size_t>(H) ? H : static_cast<int>(fit);
  x.batch = x.heads == H ? static_cast<int>(fit / H) : 1;
  if (x.batch > B) x.batch = B;
  const int64_t all = static_cast<int64_t>(x.batch) * x.heads * x.blocks * x.blocks;
  // From 512 to 1024 workgroups, of 64 tiles at most, which a wavefront looks up together.
  while (x.shift < 6 && all >> x.shift > 1024) ++x.shift;
  const int per_head = Diagonals{x.blocks, x.batch, x.shift}.per_head();
  x.g = round_up(each * x.batch * x.heads);
  x.partial = S > 0 ? round_up(static_cast<size_t>(x.heads) * per_head * 256 * D * 4) : 0;
  x.carry = S > 0 && x.batch < B ? round_up(static_cast<size_t>(2) * S * H * D * 4) : 0;
  x.delta = round_up(static_cast<size_t>(B) * H * L * 4);
  x.words = round_up(static_cast<size_t>(B) * x.blocks * 8);
  x.total = x.g + x.partial + x.carry + x.delta + x.words;
  return x;
}

template <typename T, int D, bool BOTH>
int launch_backward(Params p, const void* out, const void* low, void* dpos_key, void* dpos_query,
                    char* workspace, hipStream_t stream) {
  constexpr int NW = Sizes<T, D>::kKeyWaves, BQ = Sizes<T, D>::kKeyQueries;
  using YK = KeyLayout<T, D, NW, BQ>;
  using YQ = QueryLayout<T, D>;
  using YP = PositionLayout<T, D>;
  static_assert(sizeof(YK) <= 160 * 1024 && sizeof(YQ) <= 160 * 1024 && sizeof(YP) <= 160 * 1024,
                "LDS");
  const Plan plan = make_plan(p.B, p.H, p.L, p.S, D, sizeof(T));
  p.g = workspace;
  p.partial = reinterpret_cast<float*>(workspace + plan.g);
  float* carry = reinterpret_cast<float*>(workspace + plan.g + plan.partial);
  float* delta = reinterpret_cast<float*>(workspace + plan.g + plan.partial + plan.carry);
  p.delta = delta;
  p.words = reinterpret_cast<uint64_t*>(workspace + plan.total - plan.words);
  hipError_t e = ensure_dynamic_lds<&attention_train_key_kernel<T, D, NW, BQ, BOTH>>(sizeof(YK));
  if (e == hipSuccess) e = ensure_dynamic_lds<&attention_train_query_kernel<T, D>>(sizeof(YQ));
  if (e == hipSuccess) e = ensure_dynamic_lds<&attention_train_position_kernel<T, D>>(sizeof(YP));
  if (e != hipSuccess) return hip_code(e);

  const int64_t rows = static_cast<int64_t>(p.B) * p.L * p.H;
  constexpr int kRows = 256 / (D / Chunk<T>::N);
  hipLaunchKernelGGL((attention_delta_kernel<T, D>),
                     dim3(static_cast<uint32_t>((rows + kRows - 1) / kRows)), dim3(256), 0, stream,
                     static_cast<const T*>(p.dout), static_cast<const T*>(out),
                     sizeof(T) == 2 ? static_cast<const T*>(low) : nullptr, delta, rows, p.H, p.L);
  for (int b0 = 0; b0 < p.B; b0 += plan.batch) {
    for (int h0 = 0; h0 < p.H; h0 += plan.heads) {
      p.b0 = b0;
      p.h0 = h0;
      p.nb = p.B - b0 < plan.batch ? p.B - b0 : plan.batch;
      p.nh = p.H - h0 < plan.heads ? p.H - h0 : plan.heads;
      const int pairs = p.nb * p.nh;
      hipLaunchKernelGGL((attention_train_key_kernel<T, D, NW, BQ, BOTH>),
                         dim3(pairs * ((64 * plan.blocks + YK::BK - 1) / YK::BK)), dim3(64 * NW),
                         sizeof(YK), stream, p);
      hipLaunchKernelGGL((attention_train_query_kernel<T, D>), dim3(pairs * plan.blocks), dim3(256),
                         sizeof(YQ), stream, p);
      if (dpos_key || dpos_query) {
        const Diagonals dg{plan.blocks, p.nb, plan.shift};
        hipLaunchKernelGGL((attention_train_position_kernel<T, D>), dim3(p.nh * dg.per_head()),
                           dim3(256), sizeof(YP), stream, p, dg);
        if (dg.parts(0) > 1)
          hipLaunchKernelGGL(attention_train_parts_kernel, dim3(D / 4, dg.count(), p.nh), dim3(256), 0,
                             stream, p.partial, D, dg);
        hipLaunchKernelGGL((attention_train_slot_kernel<T, D>), dim3(p.S, p.nh), dim3(256), 0, stream,
                           p.partial, p.lut, static_cast<T*>(dpos_key),
                           static_cast<T*>(dpos_query), carry, b0 == 0, b0 + p.nb == p.B, p.L, p.S,
                           p.H, h0, dg, p.scale);
      }
    }
  }
  return hip_code(hipGetLastError());
}

template <typename F>
int by_type(int dtype, int D, const F& call) {
  auto with = [&](auto t) {
    using T = decltype(t);
    if (D == 32) return call(t, std::integral_constant<int, 32>{});
    if (D == 64) return call(t, std::integral_constant<int, 64>{});
    return call(t, std::integral_constant<int, 128>{});
  };
  if (dtype == DFLASH_DTYPE_FP16) return with(_Float16{});
  if (dtype == DFLASH_DTYPE_BF16) return with(__bf16{});
  return with(float{});
}

bool off(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

int make_params(const dflash_attention_train* a, Params& p) {
  if (!a) return DFLASH_ERR_NULL;
  if (a->B < 0 || a->H < 1 || a->L < 1 || a->S < 0 || !(a->p >= 0.0 && a->p <= 1.0) ||
      !(a->scale > 0.0f && a->scale < INFINITY))
    return DFLASH_ERR_SHAPE;
  if (a->D != 32 && a->D != 64 && a->D != 128) return DFLASH_ERR_HEAD_DIM;
  if (a->dtype < DFLASH_DTYPE_FP16 || a->dtype > DFLASH_DTYPE_FP32) return DFLASH_ERR_DTYPE;
  if (a->L > kMaxLength || static_cast<int64_t>(a->B) * a->H > (1 << 20) ||
      static_cast<int64_t>(a->S) * a->H >= (1 << 22) || a->H > 65535)
    return DFLASH_ERR_TOO_LARGE;
  const bool relative = a->pos_key || a->pos_query;
  if (!a->query || !a->key || !a->value || (relative && (!a->delta_to_slot || a->S < 1)))
    return DFLASH_ERR_NULL;
  const int esize = a->dtype == DFLASH_DTYPE_FP32 ? 4 : 2;
  const int64_t* strides[] = {a->query_strides, a->key_strides, a->value_strides};
  int64_t every = 0;
  for (const int64_t* x : strides) every |= x[0] | x[1] | x[2];
  if (a->pos_key) every |= a->pos_key_strides[0] | a->pos_key_strides[1];
  if (a->pos_query) every |= a->pos_query_strides[0] | a->pos_query_strides[1];
  const void* tensors[] = {a->query, a->key, a->value, a->pos_key, a->pos_query};
  for (const void* t : tensors)
    if (off(t, 16)) return DFLASH_ERR_ALIGN;
  if (every * esize % 16 != 0 || off(a->delta_to_slot, 4)) return DFLASH_ERR_ALIGN;
  // A head's rows are read through 31-bit byte offsets.
  auto spans = [&](int64_t rows, int64_t stride) {
    return stride < 0 || stride > INT32_MAX ||
           ((rows - 1) * stride + a->D) * esize >= int64_t{1} << 31;
  };
  for (const int64_t* x : strides)
    if (spans(a->L, x[2])) return DFLASH_ERR_TOO_LARGE;
  if ((a->pos_key && spans(a->S, a->pos_key_strides[1])) ||
      (a->pos_query && spans(a->S, a->pos_query_strides[1])) ||
      spans(a->L, static_cast<int64_t>(a->H) * a->D))
    return DFLASH_ERR_TOO_LARGE;
  p = Params{};
  p.q = a->query;
  p.k = a->key;
  p.v = a->value;
  p.sq = Strides{a->query_strides[0], a->query_strides[1], a->query_strides[2]};
  p.sk = Strides{a->key_strides[0], a->key_strides[1], a->key_strides[2]};
  p.sv = Strides{a->value_strides[0], a->value_strides[1], a->value_strides[2]};
  p.pos_key = a->pos_key;
  p.pos_query = a->pos_query;
  p.pk_h = a->pos_key_strides[0];
  p.pk_s = a->pos_key_strides[1];
  p.pq_h = a->pos_query_strides[0];
  p.pq_s = a->pos_query_strides[1];
  p.lut = a->delta_to_slot;
  p.mask = a->mask;
  p.B = a->B;
  p.H = a->H;
  p.L = a->L;
  p.S = relative ? a->S : 0;
  p.scale = a->scale;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  Dropout d;
  if (!make_dropout(a->p, nullptr, 0, d)) return DFLASH_ERR_SHAPE;
  p.keep_scale = d.scale;
  p.bit_row = (a->L + 63) / 64 * 8;
  return DFLASH_OK;
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" {

size_t dflash_attention_train_bits_bytes(int B, int H, int L) {
  if (B < 1 || H < 1 || L < 1) return 0;
  return static_cast<size_t>(B) * H * L * ((L + 63) / 64 * 8);
}

int dflash_attention_train_fwd(const dflash_attention_train* a, const int64_t* rng, uint32_t site,
                               void* out, void* out_low, float* lse, void* bits, void* stream) {
  Params p;
  const int rc = make_params(a, p);
  if (rc != DFLASH_OK) return rc;
  if (a->B == 0) return DFLASH_OK;
  if (!out || (a->p > 0 && (!rng || !bits))) return DFLASH_ERR_NULL;
  if (off(out, 16) || off(out_low, 16) || off(lse, 4) || off(bits, 8) || off(rng, 8))
    return DFLASH_ERR_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->p > 0) {
    Dropout d;
    make_dropout(a->p, rng, site, d);
    const int64_t rows = static_cast<int64_t>(p.B) * p.H * p.L;
    const int64_t blocks = (rows * p.bit_row + 255) / 256;
    if (blocks > kMaxBlocks256) return DFLASH_ERR_TOO_LARGE;
    hipLaunchKernelGGL(dropped_bits_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, s,
                       static_cast<uint8_t*>(bits), rows, p.L, static_cast<int>(p.bit_row), d);
    p.bits = static_cast<const uint8_t*>(bits);
  }
  p.out = out;
  p.low = out_low;
  p.lse = lse;
  return by_type(a->dtype, a->D, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return p.pos_key && p.pos_query ? launch_forward<T, D, true>(p, s)
                                    : launch_forward<T, D, false>(p, s);
  });
}

size_t dflash_attention_train_bwd_workspace_bytes(const dflash_attention_train* a) {
  Params p;
  if (make_params(a, p) != DFLASH_OK || a->B == 0) return 0;
  return make_plan(p.B, p.H, p.L, p.S, a->D, a->dtype == DFLASH_DTYPE_FP32 ? 4 : 2).total;
}

int dflash_attention_train_bwd(const dflash_attention_train* a, const void* out,
                               const void* out_low, const float* lse, const void* bits,
                               const void* dout, void* dquery, void* dkey,
                               void* dvalue, void* dpos_key, void* dpos_query, void* workspace,
                               size_t workspace_bytes, void* stream) {
  Params p;
  const int rc = make_params(a, p);
  if (rc != DFLASH_OK) return rc;
  if (a->B == 0) return DFLASH_OK;
  const bool halves = a->dtype != DFLASH_DTYPE_FP32;
  if (!out || (halves && !out_low) || !lse || !dout || !dquery || !dkey || !dvalue ||
      !workspace || (a->p > 0 && !bits) || (dpos_key && !a->pos_key) || (dpos_query && !a->pos_query))
    return DFLASH_ERR_NULL;
  const void* tensors[] = {out,  out_low, dout,     dquery,    dkey,
                           dvalue, dpos_key, dpos_query, workspace};
  for (const void* t : tensors)
    if (off(t, 16)) return DFLASH_ERR_ALIGN;
  if (off(lse, 4) || off(bits, 8)) return DFLASH_ERR_ALIGN;
  if (workspace_bytes < dflash_attention_train_bwd_workspace_bytes(a)) return DFLASH_ERR_WORKSPACE;
  p.lse = const_cast<float*>(lse);
  p.bits = a->p > 0 ? static_cast<const uint8_t*>(bits) : nullptr;
  p.dout = dout;
  p.dq = dquery;
  p.dk = dkey;
  p.dv = dvalue;
  return by_type(a->dtype, a->D, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    const auto call = p.pos_key && p.pos_query ? &launch_backward<T, D, true>
                                               : &launch_backward<T, D, false>;
    return call(p, out, out_low, dpos_key, dpos_query, static_cast<char*>(workspace),
                static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
