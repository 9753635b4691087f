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
// Five kernels for the backward pass.  D_i; then one over blocks of keys, which computes P and G,
// sums dV and dK in registers and writes G once; one over blocks of queries, which sums dQ from
// G; one over diagonals of tiles, which sums dPK and dPQ from G by delta; and one that adds
// up the deltas of each slot.  No atomics: every sum has an order of its own.
//
// G is kept in fragments: 16 keys x 32 queries are 512 elements in the order in which the
// lanes of a wavefront hold them, so that they are written and read 16 bytes a lane.
//
// Padded rows.  Rows of K (and of V in the forward pass) at padded keys and rows of Q at padded
// queries are taken as 0 in every product, so that whatever they hold, NaN too, reaches no
// kept row; padded queries, whose probabilities are 1/L, have blocks of their own forward.

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
  float* lse;             // [B, H, L], base 2
  const void* dout;       // [B, L, H, D]
  const float* delta;     // [B, H, L]: D_i
  void *dq, *dk, *dv;     // [B, L, H, D]
  void* g;                // fragments
  float* partial;         // sums of dPK and dPQ by tile diagonal
  int b0, h0, nb, nh;     // the (batch, head) pairs of this launch
  int B, H, L, S;
  float scale, scale_log2, keep_scale;
};

// ---- operands -------------------------------------------------------------------------

template <typename T>
struct Op {
  using frag = typename Mma<T>::frag;
  __device__ static f32x4_t run(frag a, frag b, f32x4_t c) { return Mma<T>::run(a, b, c); }
};
template <>
struct Op<float> {
  using frag = f32x8_t;
  __device__ static f32x4_t run(frag a, frag b, f32x4_t c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// A row of D elements in LDS is padded by 16 bytes, so that the 16 rows that a fragment read
// touches lie in different banks.
template <typename T, int D>
constexpr int kLd = D + 16 / static_cast<int>(sizeof(T));

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

template <typename T>
__device__ inline void store4(T* p, f32x4_t v) {
  Quad<T> q;
#pragma unroll
  for (int r = 0; r < 4; ++r) q[r] = static_cast<T>(v[r]);
  *reinterpret_cast<Quad<T>*>(p) = q;
}

// ---- tiles ----------------------------------------------------------------------------

// ROWS rows of D elements into LDS; source(r) gives row r's address, or NULL for a row of 0.
template <typename T, int D, int ROWS, int NT, typename Source>
__device__ inline void load_rows(T* tile, const Source& source) {
  constexpr int kChunks = D * static_cast<int>(sizeof(T)) / 16, kPer = 16 / static_cast<int>(sizeof(T));
#pragma unroll
  for (int at = 0; at < (ROWS * kChunks + NT - 1) / NT; ++at) {
    const int n = at * NT + threadIdx.x;
    if (ROWS * kChunks % NT != 0 && n >= ROWS * kChunks) break;
    const int row = n / kChunks, chunk = n % kChunks;
    const T* p = source(row);
    u32x4_t v{};
    if (p) v = *reinterpret_cast<const u32x4_t*>(p + chunk * kPer);
    *reinterpret_cast<u32x4_t*>(tile + row * kLd<T, D> + chunk * kPer) = v;
  }
}

// The position rows of deltas first .. first + ROWS - 1.
template <typename T, int D, int ROWS, int NT>
__device__ inline void load_window(T* tile, const T* table, int64_t row_stride, const int32_t* lut,
                                   int first, int L, int S) {
  load_rows<T, D, ROWS, NT>(tile, [&](int r) -> const T* {
    const int at = first + r + L - 1;
    if (at < 0 || at > 2 * L - 2) return nullptr;
    const int slot = lut[at];
    return slot >= 0 && slot < S ? table + slot * row_stride : nullptr;
  });
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

template <typename T>
__device__ inline const T* head(const void* base, const Strides& s, int b, int h) {
  return static_cast<const T*>(base) + b * s.b + h * s.h;
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

// A workgroup of NW wavefronts takes 16 NW queries and walks the keys in tiles of 16 NW.  Scores
// are computed transposed (a lane holds one query and four keys of a block), so that the
// probabilities are the operand of O^T += V^T R^T as they are.
template <typename T, int D, int NW>
struct FwdLayout {
  static constexpr int BT = 16 * NW, W = BT + 16, LDW = W + 4;
  static constexpr int LD = kLd<T, D>;
  T k[BT * LD], v[BT * LD], pk[2 * BT * LD], pq[2 * BT * LD];
  float c2p[BT * LDW], p2c[BT * LDW];
  uint64_t kept[kWords];
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW) void attention_train_fwd_kernel(Params p) {
  using Y = FwdLayout<T, D, NW>;
  using F = typename Op<T>::frag;
  constexpr int BT = Y::BT, LD = Y::LD, LDW = Y::LDW, NT = 64 * NW;
  extern __shared__ __align__(16) unsigned char memory[];
  Y& s = *reinterpret_cast<Y*>(memory);
  const int blocks = (p.L + BT - 1) / BT;
  const int at = xcd_logical_block(blockIdx.x, gridDim.x);
  const int bh = at / blocks, i0 = at % blocks * BT;
  const int b = bh / p.H, h = bh % p.H;
  const bool uniform = blockIdx.y == 1;  // the block's padded queries, otherwise its kept ones
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, g = lane / 16;
  const int i = i0 + 16 * wave + c;

  read_mask(s.kept, p.mask, b, p.L);
  constexpr uint64_t kBlock = BT == 64 ? ~uint64_t{0} : (uint64_t{1} << (BT % 64)) - 1;
  const uint64_t rows = tokens_from(i0, p.L) & kBlock;
  const uint64_t kept_rows = (s.kept[i0 / 64] >> (i0 % 64)) & kBlock;
  if (uniform ? rows == kept_rows : kept_rows == 0) return;

  const T* q = head<T>(p.q, p.sq, b, h);
  const T* k = head<T>(p.k, p.sk, b, h);
  const T* v = head<T>(p.v, p.sv, b, h);
  const T* pk = p.pos_key ? static_cast<const T*>(p.pos_key) + h * p.pk_h : nullptr;
  const T* pq = p.pos_query ? static_cast<const T*>(p.pos_query) + h * p.pq_h : nullptr;
  const bool mine = (kept_rows >> (16 * wave + c)) & 1;

  F qf[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) {
    qf[ks] = F{};
    if (mine) qf[ks] = *reinterpret_cast<const F*>(q + i * p.sq.l + 32 * ks + 8 * g);
  }

  f32x4_t o[D / 16] = {};
  float top = -INFINITY, sum = 0;
  const uint8_t* bits =
      p.bits ? p.bits + (static_cast<int64_t>(bh) * p.L + (i < p.L ? i : p.L - 1)) * p.bit_row
             : nullptr;

  for (int j0 = 0; j0 < p.L; j0 += BT) {
    const uint64_t inside = tokens_from(j0, p.L) & kBlock;
    const uint64_t kept = (s.kept[j0 / 64] >> (j0 % 64)) & kBlock;
    const uint64_t taken = uniform ? inside : kept;
    if (taken == 0) continue;
    __syncthreads();
    load_rows<T, D, BT, NT>(s.v, [&](int r) {
      return (taken >> r) & 1 ? v + (j0 + r) * p.sv.l : nullptr;
    });
    if (!uniform) {
      load_rows<T, D, BT, NT>(s.k, [&](int r) {
        return (kept >> r) & 1 ? k + (j0 + r) * p.sk.l : nullptr;
      });
      if (pk) load_window<T, D, 2 * BT, NT>(s.pk, pk, p.pk_s, p.lut, i0 - j0 - BT, p.L, p.S);
      if (pq) load_window<T, D, 2 * BT, NT>(s.pq, pq, p.pq_s, p.lut, i0 - j0 - BT, p.L, p.S);
    }
    uint64_t dropped = 0;
    if (bits) {
      dropped = *reinterpret_cast<const uint64_t*>(bits + j0 / 64 * 8);
      dropped = (dropped >> (j0 % 64)) >> (4 * g);
    }
    __syncthreads();

    f32x4_t x[NW] = {};  // x[kb][r]: key j0 + 16 kb + 4g + r
    if (!uniform) {
      if (pq) {
        // Keys of block `wave` against deltas from i0 - j0 - 16 wave - 16.
#pragma unroll
        for (int wb = 0; wb < NW + 1; ++wb) {
          f32x4_t acc{};
#pragma unroll
          for (int ks = 0; ks < D / 32; ++ks)
            acc = Op<T>::run(
                read_row<T>(s.pq + (BT - 16 - 16 * wave + 16 * wb + c) * LD + 32 * ks, g),
                read_row<T>(s.k + (16 * wave + c) * LD + 32 * ks, g), acc);
          *reinterpret_cast<f32x4_t*>(s.p2c + (16 * wave + c) * LDW + 16 * wb + 4 * g) = acc;
        }
      }
      if (pk) {
        // This wavefront's queries against deltas from i0 + 16 wave - j0 - BT.
#pragma unroll
        for (int wb = 0; wb < NW + 1; ++wb) {
          f32x4_t acc{};
#pragma unroll
          for (int ks = 0; ks < D / 32; ++ks)
            acc = Op<T>::run(read_row<T>(s.pk + (16 * wave + 16 * wb + c) * LD + 32 * ks, g),
                             qf[ks], acc);
          *reinterpret_cast<f32x4_t*>(s.c2p + (16 * wave + c) * LDW + 16 * wb + 4 * g) = acc;
        }
      }
#pragma unroll
      for (int kb = 0; kb < NW; ++kb)
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks)
          x[kb] = Op<T>::run(read_row<T>(s.k + (16 * kb + c) * LD + 32 * ks, g), qf[ks], x[kb]);
      __syncthreads();
      if (pk) {
#pragma unroll
        for (int kb = 0; kb < NW; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[kb][r] += s.c2p[(16 * wave + c) * LDW + BT + c - 16 * kb - 4 * g - r];
      }
      if (pq) {
#pragma unroll
        for (int kb = 0; kb < NW; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[kb][r] += s.p2c[(16 * kb + 4 * g + r) * LDW + 16 * wave + 16 + c - 4 * g - r];
      }
    }
    const uint64_t lane_taken = taken >> (4 * g);
    float high = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NW; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[kb][r] = (lane_taken >> (16 * kb + r)) & 1 ? x[kb][r] * p.scale_log2 : -INFINITY;
        high = fmaxf(high, x[kb][r]);
      }
    high = fmaxf(high, __shfl_xor(high, 16));
    high = fmaxf(high, __shfl_xor(high, 32));
    high = fmaxf(high, top);  // (finite: the tile holds a key that is taken)
    const float shrink = __builtin_amdgcn_exp2f(top - high);
    top = high;
    sum *= shrink;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) o[db] *= shrink;
#pragma unroll
    for (int kb = 0; kb < NW; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(x[kb][r] - top);
        sum += e;
        x[kb][r] = (dropped >> (16 * kb + r)) & 1 ? 0.0f : e;
      }
    // (Rounded to T here, as the operand of the product: off by half a step of each probability.)
#pragma unroll
    for (int ks = 0; ks < NW / 2; ++ks) {
      const F r = pack<T>(x[2 * ks], x[2 * ks + 1]);
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        o[db] = Op<T>::run(
            read_columns<T>(s.v + 16 * db, LD, 32 * ks + 4 * g, 32 * ks + 16 + 4 * g, c), r,
            o[db]);
    }
  }

  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (i >= p.L || mine == uniform) return;
  const float factor = p.keep_scale / sum;
  T* out = static_cast<T*>(p.out) + ((static_cast<int64_t>(b) * p.L + i) * p.H + h) * D;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) store4(out + 16 * db + 4 * g, o[db] * factor);
  if (p.lse && g == 0) p.lse[static_cast<int64_t>(bh) * p.L + i] = top + log2f(sum);
}

// ---- D_i = dO_i . O_i -----------------------------------------------------------------------

template <typename T, int D>
__global__ __launch_bounds__(256) void attention_delta_kernel(const T* dout, const T* out,
                                                              float* delta, int64_t rows, int H,
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
  static constexpr int KF = (WK + 31) / 32 * 32, LDF = KF + 16 / static_cast<int>(sizeof(T));
  static constexpr int LD = kLd<T, D>;
  // (dK's product reads KF rows of pq from row BK - 16 - 16 wave.)
  static constexpr int PQ = BK - 16 + KF;
  T q[BQ * LD], dout[BQ * LD], pk[(BQ + BK) * LD], pq[PQ * LD];
  float c2p[BQ * LDC], p2c[BK * LDP];
  T skew[BK * LDF];
  float lse[BQ], delta[BQ];
  uint64_t dropped[BQ];
  uint64_t kept[kWords];
};

template <typename T, int D, int NW, int BQ>
__global__ __launch_bounds__(64 * NW) void attention_train_key_kernel(Params p) {
  using Y = KeyLayout<T, D, NW, BQ>;
  using F = typename Op<T>::frag;
  constexpr int BK = Y::BK, LD = Y::LD, LDC = Y::LDC, LDP = Y::LDP, LDF = Y::LDF, NT = 64 * NW;
  constexpr int QB = BQ / 16;
  extern __shared__ __align__(16) unsigned char memory[];
  Y& s = *reinterpret_cast<Y*>(memory);
  const int blocks = (p.L + 63) / 64 * (64 / BK);  // whole blocks of 64: all of G is written
  const int at = xcd_logical_block(blockIdx.x, gridDim.x);
  const int pair = at / blocks, j0 = at % blocks * BK;
  const int b = p.b0 + pair / p.nh, h = p.h0 + pair % p.nh;
  const int64_t bh = static_cast<int64_t>(b) * p.H + h;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, g = lane / 16;
  const int j = j0 + 16 * wave + c;

  read_mask(s.kept, p.mask, b, p.L);
  for (int n = threadIdx.x; n < BK * LDF; n += NT) s.skew[n] = static_cast<T>(0.0f);
  const bool any_key = s.kept[j0 / 64] != 0;
  const bool mine = j < p.L && bit_of(s.kept, j);
  const float even = 1.0f / static_cast<float>(p.L);

  const T* q = head<T>(p.q, p.sq, b, h);
  const T* k = head<T>(p.k, p.sk, b, h);
  const T* v = head<T>(p.v, p.sv, b, h);
  const T* pk = p.pos_key ? static_cast<const T*>(p.pos_key) + h * p.pk_h : nullptr;
  const T* pq = p.pos_query ? static_cast<const T*>(p.pos_query) + h * p.pq_h : nullptr;
  const T* dout = static_cast<const T*>(p.dout) + (static_cast<int64_t>(b) * p.L * p.H + h) * D;
  const int64_t row = static_cast<int64_t>(p.H) * D;
  // Fragments of this pair: [16 keys][32 queries].
  const int q32 = (p.L + 63) / 64 * 2;
  T* out_g = static_cast<T*>(p.g) +
             (static_cast<int64_t>(pair) * (2 * q32) + j0 / 16 + wave) * q32 * kFragment;

  F kf[D / 32], vf[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) {
    kf[ks] = F{};
    vf[ks] = F{};
    if (mine) kf[ks] = *reinterpret_cast<const F*>(k + j * p.sk.l + 32 * ks + 8 * g);
    if (j < p.L) vf[ks] = *reinterpret_cast<const F*>(v + j * p.sv.l + 32 * ks + 8 * g);
  }
  f32x4_t dk[D / 16] = {}, dv[D / 16] = {};

  for (int i0 = 0; i0 < (p.L + 63) / 64 * 64; i0 += BQ) {
    constexpr uint64_t kBlock = BQ == 64 ? ~uint64_t{0} : (uint64_t{1} << (BQ % 64)) - 1;
    const uint64_t inside = tokens_from(i0, p.L) & kBlock;
    const uint64_t kept = (s.kept[i0 / 64] >> (i0 % 64)) & kBlock;
    // (By whole words of 64 queries: the readers of G go by the same.)
    const bool scored = any_key && s.kept[i0 / 64] != 0;
    if (!scored && kept == inside) continue;  // no padded query either
    __syncthreads();
    load_rows<T, D, BQ, NT>(s.dout, [&](int r) {
      return (inside >> r) & 1 ? dout + (i0 + r) * row : nullptr;
    });
    if (scored) {
      load_rows<T, D, BQ, NT>(s.q, [&](int r) {
        return (kept >> r) & 1 ? q + (i0 + r) * p.sq.l : nullptr;
      });
      if (pk) load_window<T, D, BQ + BK, NT>(s.pk, pk, p.pk_s, p.lut, i0 - j0 - BK, p.L, p.S);
      if (pq) load_window<T, D, Y::PQ, NT>(s.pq, pq, p.pq_s, p.lut, i0 - j0 - BK, p.L, p.S);
    }
    if (threadIdx.x < BQ) {
      const int r = threadIdx.x, i = i0 + r < p.L ? i0 + r : p.L - 1;
      if (scored) {
        s.lse[r] = p.lse[bh * p.L + i];
        s.delta[r] = p.delta[bh * p.L + i];
      }
      s.dropped[r] = 0;
      if (p.bits)
        s.dropped[r] = *reinterpret_cast<const uint64_t*>(
                           p.bits + (bh * p.L + i) * p.bit_row + j0 / 64 * 8) >>
                       (j0 % 64);
    }
    __syncthreads();

    f32x4_t x[QB] = {}, y[QB] = {};  // [qb][r]: query i0 + 16 qb + 4g + r
    if (scored) {
      if (pk) {
        // Blocks of 16 queries against deltas from i0 + 16 qb - j0 - BK, shared by the wavefronts.
#pragma unroll
        for (int n = 0; n < (QB * (NW + 1) + NW - 1) / NW; ++n) {
          const int at2 = n * NW + wave, qb = at2 / (NW + 1), wb = at2 % (NW + 1);
          if (at2 < QB * (NW + 1)) {
            f32x4_t acc{};
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks)
              acc = Op<T>::run(read_row<T>(s.pk + (16 * qb + 16 * wb + c) * LD + 32 * ks, g),
                               read_row<T>(s.q + (16 * qb + c) * LD + 32 * ks, g), acc);
            *reinterpret_cast<f32x4_t*>(s.c2p + (16 * qb + c) * LDC + 16 * wb + 4 * g) = acc;
          }
        }
      }
      if (pq) {
        // This wavefront's keys against deltas from i0 - j0 - 16 wave - 16.
#pragma unroll
        for (int wb = 0; wb < QB + 1; ++wb) {
          f32x4_t acc{};
#pragma unroll
          for (int ks = 0; ks < D / 32; ++ks)
            acc = Op<T>::run(
                read_row<T>(s.pq + (BK - 16 - 16 * wave + 16 * wb + c) * LD + 32 * ks, g), kf[ks],
                acc);
          *reinterpret_cast<f32x4_t*>(s.p2c + (16 * wave + c) * LDP + 16 * wb + 4 * g) = acc;
        }
      }
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int ks = 0; ks < D / 32; ++ks) {
          x[qb] = Op<T>::run(read_row<T>(s.q + (16 * qb + c) * LD + 32 * ks, g), kf[ks], x[qb]);
          y[qb] = Op<T>::run(read_row<T>(s.dout + (16 * qb + c) * LD + 32 * ks, g), vf[ks], y[qb]);
        }
      __syncthreads();
      if (pk) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[qb][r] +=
                s.c2p[(16 * qb + 4 * g + r) * LDC + 4 * g + r - c - 16 * wave + BK];
      }
      if (pq) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[qb][r] += s.p2c[(16 * wave + c) * LDP + 16 * qb + 4 * g + r - c + 16];
      }
    }
    const uint64_t lane_kept = kept >> (4 * g), lane_inside = inside >> (4 * g);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at2 = 16 * qb + 4 * g + r;
        const bool live = (lane_kept >> (16 * qb + r)) & 1;
        const bool padded = ((lane_inside >> (16 * qb + r)) & 1) && !live && j < p.L;
        const float m = (s.dropped[at2] >> (16 * wave + c)) & 1 ? 0.0f : p.keep_scale;
        // (One token has one probability, 1, and no gradient.)
        float prob = 0, grad = 0;
        if (scored && live && mine) {
          prob = __builtin_amdgcn_exp2f(x[qb][r] * p.scale_log2 - s.lse[at2]);
          if (p.L > 1) grad = prob * (m == 0.0f ? -s.delta[at2] : y[qb][r] * m - s.delta[at2]);
        }
        if (padded) prob = even;
        x[qb][r] = prob * m;
        y[qb][r] = grad;
      }
    // (R and G are rounded to T as operands: off by half a step of each.)
#pragma unroll
    for (int ks = 0; ks < QB / 2; ++ks) {
      const F r = pack<T>(x[2 * ks], x[2 * ks + 1]);
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        dv[db] = Op<T>::run(
            read_columns<T>(s.dout + 16 * db, LD, 32 * ks + 4 * g, 32 * ks + 16 + 4 * g, c), r,
            dv[db]);
      if (scored) {
        const F dg = pack<T>(y[2 * ks], y[2 * ks + 1]);
        *reinterpret_cast<F*>(out_g + static_cast<int64_t>(i0 / 32 + ks) * kFragment + lane * 8) =
            dg;
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          dk[db] = Op<T>::run(
              read_columns<T>(s.q + 16 * db, LD, 32 * ks + 4 * g, 32 * ks + 16 + 4 * g, c), dg,
              dk[db]);
        if (pq) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            s.skew[(16 * wave + c) * LDF + 32 * ks + (e < 4 ? e : 12 + e) + 4 * g - c + 16] =
                dg[e];
        }
      }
    }
    if (scored && pq) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int ks = 0; ks < Y::KF / 32; ++ks) {
        const F sk = read_row<T>(s.skew + (16 * wave + c) * LDF + 32 * ks, g);
        const int lo = BK - 16 - 16 * wave + 32 * ks + 8 * g;
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          dk[db] = Op<T>::run(read_columns<T>(s.pq + 16 * db, LD, lo, lo + 4, c), sk, dk[db]);
      }
    }
  }

  if (j >= p.L) return;
  const int64_t base = ((static_cast<int64_t>(b) * p.L + j) * p.H + h) * D;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) {
    store4(static_cast<T*>(p.dk) + base + 16 * db + 4 * g, dk[db] * p.scale);
    store4(static_cast<T*>(p.dv) + base + 16 * db + 4 * g, dv[db]);
  }
}

// ---- dQ ---------------------------------------------------------------------------------------

template <typename T, int D>
struct QueryLayout {
  static constexpr int LD = kLd<T, D>, LDG = kLd<T, 64>, LDE = kLd<T, 96>;
  T k[64 * LD], pk[144 * LD];
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
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, g = lane / 16;
  const int i = i0 + 16 * wave + c;
  read_mask(s.kept, p.mask, b, p.L);
  for (int n = threadIdx.x; n < 64 * LDE; n += 256) s.skew[n] = static_cast<T>(0.0f);

  const T* k = head<T>(p.k, p.sk, b, h);
  const T* pk = p.pos_key ? static_cast<const T*>(p.pos_key) + h * p.pk_h : nullptr;
  const int q32 = 2 * blocks;
  const T* fragments = static_cast<const T*>(p.g) + static_cast<int64_t>(pair) * 2 * q32 * q32 * kFragment;
  f32x4_t dq[D / 16] = {};
  for (int jb = 0; jb < blocks && s.kept[i0 / 64] != 0; ++jb) {
    const uint64_t kept = s.kept[jb];
    if (kept == 0) continue;
    const int j0 = 64 * jb;
    F f[2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
      f[n] = *reinterpret_cast<const F*>(
          fragments + (static_cast<int64_t>(j0 / 16 + wave) * q32 + i0 / 32 + n) * kFragment +
          lane * 8);
    __syncthreads();
    load_rows<T, D, 64, 256>(s.k, [&](int r) {
      return (kept >> r) & 1 ? k + (j0 + r) * p.sk.l : nullptr;
    });
    if (pk) load_window<T, D, 144, 256>(s.pk, pk, p.pk_s, p.lut, i0 - j0 - 64, p.L, p.S);
    const int key = 16 * wave + c;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int query = 32 * n + query_of(g, e);
        s.g[key * LDG + query] = f[n][e];
        if (pk) s.skew[query * LDE + query % 16 - key + 64] = f[n][e];
      }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int lo = 32 * ks + 8 * g;
      const F dg = read_columns<T>(s.g + 16 * wave, LDG, lo, lo + 4, c);
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        dq[db] = Op<T>::run(read_columns<T>(s.k + 16 * db, LD, lo, lo + 4, c), dg, dq[db]);
    }
    if (pk) {
#pragma unroll
      for (int ks = 0; ks < 3; ++ks) {
        const F sk = read_row<T>(s.skew + (16 * wave + c) * LDE + 32 * ks, g);
        const int lo = 16 * wave + 32 * ks + 8 * g;
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
          dq[db] = Op<T>::run(read_columns<T>(s.pk + 16 * db, LD, lo, lo + 4, c), sk, dq[db]);
      }
    }
  }
  if (i >= p.L) return;
  T* out = static_cast<T*>(p.dq) + ((static_cast<int64_t>(b) * p.L + i) * p.H + h) * D;
#pragma unroll
  for (int db = 0; db < D / 16; ++db) store4(out + 16 * db + 4 * g, dq[db] * p.scale);
}

// ---- dPK and dPQ by delta -------------------------------------------------------------------

// The tiles of 64 x 64 with (query block) - (key block) = m, of all sequences of one head, share
// their deltas, 64 m - 63 .. 64 m + 63: place 64 + (i - j) - 64 m of 128.  `tiles` of them are one
// workgroup's; the parts of a diagonal are added up by the next kernel.
struct Diagonals {
  int blocks, batch, tiles;
  __host__ __device__ int parts(int m) const {
    const int n = batch * (blocks - (m < 0 ? -m : m));
    return (n + tiles - 1) / tiles;
  }
  // Diagonals in the order 0, 1, -1, 2, -2, ..: the longest first.
  __host__ __device__ static int nth(int n) { return n % 2 ? (n + 1) / 2 : -(n / 2); }
  __host__ __device__ int total() const {
    int sum = 0;
    for (int n = 0; n < 2 * blocks - 1; ++n) sum += parts(nth(n));
    return sum;
  }
};

template <typename T, int D>
struct PositionLayout {
  static constexpr int LD = kLd<T, D>, LDX = kLd<T, 64>;
  T q[64 * LD], k[64 * LD];
  T by_query[128 * LDX], by_key[128 * LDX];  // [delta][query], [delta][key]
};

template <typename T, int D>
__global__ __launch_bounds__(256) void attention_train_position_kernel(Params p, Diagonals dg,
                                                                       int per_head) {
  using Y = PositionLayout<T, D>;
  using F = typename Op<T>::frag;
  constexpr int LD = Y::LD, LDX = Y::LDX;
  extern __shared__ __align__(16) unsigned char memory[];
  Y& s = *reinterpret_cast<Y*>(memory);
  const int hh = blockIdx.x % p.nh, rest = blockIdx.x / p.nh;  // (heads first: longest first)
  int n = 0, part = rest;
  for (; part >= dg.parts(Diagonals::nth(n)); ++n) part -= dg.parts(Diagonals::nth(n));
  const int m = Diagonals::nth(n);
  const int along = dg.blocks - (m < 0 ? -m : m);
  const int h = p.h0 + hh;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, g = lane / 16;
  for (int x = threadIdx.x; x < 128 * LDX; x += 256) {
    s.by_query[x] = static_cast<T>(0.0f);
    s.by_key[x] = static_cast<T>(0.0f);
  }
  const int q32 = 2 * dg.blocks;
  const bool pk = p.pos_key != nullptr, pq = p.pos_query != nullptr;
  f32x4_t dpk[2][D / 16] = {}, dpq[2][D / 16] = {};
  const int end = min((part + 1) * dg.tiles, dg.batch * along);
  for (int u = part * dg.tiles; u < end; ++u) {
    const int bb = u / along, qt = u % along + (m > 0 ? m : 0), kt = qt - m;
    const int b = p.b0 + bb, pair = bb * p.nh + hh;
    const int i0 = 64 * qt, j0 = 64 * kt;
    // (Every wavefront reads the masks of both blocks.)
    auto kept_of = [&](int at) {
      return __ballot(at + lane < p.L &&
                      (!p.mask || p.mask[static_cast<int64_t>(b) * p.L + at + lane]));
    };
    const uint64_t kept_q = kept_of(i0), kept_k = kept_of(j0);
    if (kept_q == 0 || kept_k == 0) continue;
    const T* fragments =
        static_cast<const T*>(p.g) +
        ((static_cast<int64_t>(pair) * 2 * q32 + j0 / 16 + wave) * q32 + i0 / 32) * kFragment;
    F f[2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
      f[x] = *reinterpret_cast<const F*>(fragments + x * kFragment + lane * 8);
    __syncthreads();
    const T* q = head<T>(p.q, p.sq, b, h);
    const T* k = head<T>(p.k, p.sk, b, h);
    if (pk)
      load_rows<T, D, 64, 256>(s.q, [&](int r) {
        return (kept_q >> r) & 1 ? q + (i0 + r) * p.sq.l : nullptr;
      });
    if (pq)
      load_rows<T, D, 64, 256>(s.k, [&](int r) {
        return (kept_k >> r) & 1 ? k + (j0 + r) * p.sk.l : nullptr;
      });
    const int key = 16 * wave + c;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int query = 32 * x + query_of(g, e), place = 64 + query - key;
        if (pk) s.by_query[place * LDX + query] = f[x][e];
        if (pq) s.by_key[place * LDX + key] = f[x][e];
      }
    __syncthreads();
    // Blocks of 16 places `wave` and `wave` + 4; those that a step of 32 queries or keys does not
    // reach are left out.
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int lo = 32 * ks + 8 * g;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int wb = wave + 4 * half;
        if (pk && (ks == 0 ? wb < 6 : wb >= 2)) {
          const F x = read_row<T>(s.by_query + (16 * wb + c) * LDX + 32 * ks, g);
#pragma unroll
          for (int db = 0; db < D / 16; ++db)
            dpk[half][db] = Op<T>::run(read_columns<T>(s.q + 16 * db, LD, lo, lo + 4, c), x,
                                       dpk[half][db]);
        }
        if (pq && (ks == 0 ? wb >= 2 : wb < 6)) {
          const F x = read_row<T>(s.by_key + (16 * wb + c) * LDX + 32 * ks, g);
#pragma unroll
          for (int db = 0; db < D / 16; ++db)
            dpq[half][db] = Op<T>::run(read_columns<T>(s.k + 16 * db, LD, lo, lo + 4, c), x,
                                       dpq[half][db]);
        }
      }
    }
  }
  float* out = p.partial + (static_cast<int64_t>(hh) * per_head + rest) * 2 * 128 * D;
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

// One workgroup for a slot of a head: the sums of its deltas, each the parts of two diagonals.
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_train_slot_kernel(
    const float* partial, const int32_t* lut, T* dpos_key, T* dpos_query, float* carry, int first,
    int last, int L, int S, int H, int h0, Diagonals dg, int per_head, float scale) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ f32x4_t sums[2][256];
  const int slot = blockIdx.x, hh = blockIdx.y;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  f32x4_t sum[2] = {};
  const float* base = partial + static_cast<int64_t>(hh) * per_head * 256 * D;
  for (int at = group; at < 2 * L - 1; at += kGroups) {
    if (lut[at] != slot) continue;
    const int delta = at - (L - 1);
    const int lower = delta >= 0 ? delta / 64 : -((63 - delta) / 64), place = delta - 64 * lower;
    for (int n = 0, offset = 0, found = 0; n < 2 * dg.blocks - 1 && found < 2; ++n) {
      const int m = Diagonals::nth(n), parts = dg.parts(m);
      if (m == lower || m == lower + 1) {
        ++found;
        const int at2 = m == lower ? 64 + place : place;
        for (int x = 0; x < parts; ++x) {
          const float* from = base + static_cast<int64_t>(offset + x) * 256 * D + at2 * D + lane * 4;
          sum[0] += *reinterpret_cast<const f32x4_t*>(from);
          sum[1] += *reinterpret_cast<const f32x4_t*>(from + 128 * D);
        }
      }
      offset += parts;
    }
  }
  sums[0][threadIdx.x] = sum[0];
  sums[1][threadIdx.x] = sum[1];
  __syncthreads();
  if (group != 0) return;
  const int64_t at = (static_cast<int64_t>(slot) * H + h0 + hh) * D + lane * 4;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    T* out = x ? dpos_query : dpos_key;
    if (!out) continue;
    f32x4_t total{};
    for (int n = 0; n < kGroups; ++n) total += sums[x][n * kLanes + lane];
    // (Launches over parts of the batch add up in `carry`.)
    f32x4_t* kept = reinterpret_cast<f32x4_t*>(carry + (x * static_cast<int64_t>(S) * H * D) + at);
    if (!first) total += *kept;
    if (last)
      store4(out + at, total * scale);
    else
      *kept = total;
  }
}

// ---- host -------------------------------------------------------------------------------------

template <typename T, int D>
constexpr int kWaves16 = sizeof(T) == 4 && D == 128 ? 2 : 4;  // what fits 160 KB of LDS
template <typename T, int D>
constexpr int kQueries = sizeof(T) == 4 || D == 128 ? 32 : 64;

int hip_code(hipError_t e) { return static_cast<int>(e); }

template <typename T, int D>
int launch_forward(const Params& p, hipStream_t stream) {
  constexpr int NW = kWaves16<T, D>;
  using Y = FwdLayout<T, D, NW>;
  static_assert(sizeof(Y) <= 160 * 1024, "LDS");
  const int64_t blocks = static_cast<int64_t>((p.L + Y::BT - 1) / Y::BT) * p.B * p.H;
  if (blocks > kMaxBlocks256) return DFLASH_ERR_TOO_LARGE;
  hipError_t e = ensure_dynamic_lds<&attention_train_fwd_kernel<T, D, NW>>(sizeof(Y));
  if (e != hipSuccess) return hip_code(e);
  hipLaunchKernelGGL((attention_train_fwd_kernel<T, D, NW>),
                     dim3(static_cast<uint32_t>(blocks), p.mask ? 2 : 1), dim3(64 * NW), sizeof(Y),
                     stream, p);
  return hip_code(hipGetLastError());
}

// How the backward pass divides its work.
struct Plan {
  int batch, heads;  // (batch, head) pairs of one launch: all heads, or some of one batch
  int blocks, tiles, per_head;
  size_t g, partial, carry, delta, total;
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
  // About 1024 workgroups, of 64 tiles at most.
  int64_t tiles = (all + 1023) / 1024;
  x.tiles = static_cast<int>(tiles < 1 ? 1 : tiles > 64 ? 64 : tiles);
  x.per_head = Diagonals{x.blocks, x.batch, x.tiles}.total();
  x.g = round_up(each * x.batch * x.heads);
  x.partial = S > 0 ? round_up(static_cast<size_t>(x.heads) * x.per_head * 256 * D * 4) : 0;
  x.carry = S > 0 && x.batch < B ? round_up(static_cast<size_t>(2) * S * H * D * 4) : 0;
  x.delta = round_up(static_cast<size_t>(B) * H * L * 4);
  x.total = x.g + x.partial + x.carry + x.delta;
  return x;
}

template <typename T, int D>
int launch_backward(Params p, const void* out, void* dpos_key, void* dpos_query, char* workspace,
                    hipStream_t stream) {
  constexpr int NW = kWaves16<T, D>, BQ = kQueries<T, D>;
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
  hipError_t e = ensure_dynamic_lds<&attention_train_key_kernel<T, D, NW, BQ>>(sizeof(YK));
  if (e == hipSuccess) e = ensure_dynamic_lds<&attention_train_query_kernel<T, D>>(sizeof(YQ));
  if (e == hipSuccess) e = ensure_dynamic_lds<&attention_train_position_kernel<T, D>>(sizeof(YP));
  if (e != hipSuccess) return hip_code(e);

  const int64_t rows = static_cast<int64_t>(p.B) * p.L * p.H;
  constexpr int kRows = 256 / (D / Chunk<T>::N);
  hipLaunchKernelGGL((attention_delta_kernel<T, D>),
                     dim3(static_cast<uint32_t>((rows + kRows - 1) / kRows)), dim3(256), 0, stream,
                     static_cast<const T*>(p.dout), static_cast<const T*>(out), delta, rows, p.H,
                     p.L);
  for (int b0 = 0; b0 < p.B; b0 += plan.batch) {
    for (int h0 = 0; h0 < p.H; h0 += plan.heads) {
      p.b0 = b0;
      p.h0 = h0;
      p.nb = p.B - b0 < plan.batch ? p.B - b0 : plan.batch;
      p.nh = p.H - h0 < plan.heads ? p.H - h0 : plan.heads;
      const int pairs = p.nb * p.nh;
      hipLaunchKernelGGL((attention_train_key_kernel<T, D, NW, BQ>),
                         dim3(pairs * plan.blocks * (64 / YK::BK)), dim3(64 * NW), sizeof(YK),
                         stream, p);
      hipLaunchKernelGGL((attention_train_query_kernel<T, D>), dim3(pairs * plan.blocks), dim3(256),
                         sizeof(YQ), stream, p);
      if (dpos_key || dpos_query) {
        const Diagonals dg{plan.blocks, p.nb, plan.tiles};
        const int per_head = dg.total();
        hipLaunchKernelGGL((attention_train_position_kernel<T, D>), dim3(p.nh * per_head), dim3(256),
                           sizeof(YP), stream, p, dg, per_head);
        hipLaunchKernelGGL((attention_train_slot_kernel<T, D>), dim3(p.S, p.nh), dim3(256), 0,
                           stream, p.partial, p.lut, static_cast<T*>(dpos_key),
                           static_cast<T*>(dpos_query), carry, b0 == 0, b0 + p.nb == p.B, p.L, p.S,
                           p.H, h0, dg, per_head, p.scale);
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
  if (a->B < 0 || a->H < 1 || a->L < 1 || a->S < 0 || !(a->p >= 0.0 && a->p <= 1.0))
    return DFLASH_ERR_SHAPE;
  if (a->D != 32 && a->D != 64 && a->D != 128) return DFLASH_ERR_HEAD_DIM;
  if (a->dtype < DFLASH_DTYPE_FP16 || a->dtype > DFLASH_DTYPE_FP32) return DFLASH_ERR_DTYPE;
  if (a->L > kMaxLength || static_cast<int64_t>(a->B) * a->H > (1 << 20) ||
      static_cast<int64_t>(a->S) * a->H >= (1 << 24) || a->H > 65535)
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
                               void* out, float* lse, void* bits, void* stream) {
  Params p;
  const int rc = make_params(a, p);
  if (rc != DFLASH_OK) return rc;
  if (a->B == 0) return DFLASH_OK;
  if (!out || (a->p > 0 && (!rng || !bits))) return DFLASH_ERR_NULL;
  if (off(out, 16) || off(lse, 4) || off(bits, 8) || off(rng, 8)) return DFLASH_ERR_ALIGN;
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
  p.lse = lse;
  return by_type(a->dtype, a->D, [&](auto t, auto d) {
    return launch_forward<decltype(t), decltype(d)::value>(p, s);
  });
}

size_t dflash_attention_train_bwd_workspace_bytes(const dflash_attention_train* a) {
  Params p;
  if (make_params(a, p) != DFLASH_OK || a->B == 0) return 0;
  return make_plan(p.B, p.H, p.L, p.S, a->D, a->dtype == DFLASH_DTYPE_FP32 ? 4 : 2).total;
}

int dflash_attention_train_bwd(const dflash_attention_train* a, const void* out, const float* lse,
                               const void* bits, const void* dout, void* dquery, void* dkey,
                               void* dvalue, void* dpos_key, void* dpos_query, void* workspace,
                               size_t workspace_bytes, void* stream) {
  Params p;
  const int rc = make_params(a, p);
  if (rc != DFLASH_OK) return rc;
  if (a->B == 0) return DFLASH_OK;
  if (!out || !lse || !dout || !dquery || !dkey || !dvalue || !workspace || (a->p > 0 && !bits) ||
      (dpos_key && !a->pos_key) || (dpos_query && !a->pos_query))
    return DFLASH_ERR_NULL;
  const void* tensors[] = {out, dout, dquery, dkey, dvalue, dpos_key, dpos_query, workspace};
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
    return launch_backward<decltype(t), decltype(d)::value>(p, out, dpos_key, dpos_query,
                                                            static_cast<char*>(workspace),
                                                            static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
