// Device helpers of the training kernels (gfx950): 16-byte chunks and the dropout generator.
#pragma once

#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include "dflash.h"

namespace dflash {

// A launch may hold fewer than 2^32 work items.
constexpr int64_t kMaxBlocks256 = UINT32_MAX / 256;

// A chunk: the elements of one 16-byte access.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};

// Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC'11, whose tests 7 rounds pass): the 64-bit seed is the key, the counter is
// (block, site, step).  A block of 8 consecutive elements takes one call, 16 bits
// each (p is a multiple of 2^-16): 14 wide products for 8 elements, half of what 32 bits
// for each element would take.
struct Dropout {
  const int64_t* rng;  // device: seed, step
  uint32_t site;
  uint32_t drop_max;   // a field of 16 bits, shifted to the top of a word, is dropped up to here
  float scale;         // 1 / P(kept)
  int active;          // 0: p = 0, rng is not read
};

struct DropoutKey {
  uint32_t k0, k1, step;
};

__device__ inline DropoutKey dropout_key(const Dropout& d) {
  DropoutKey key{0, 0, 0};
  if (d.active) {
    const uint64_t seed = static_cast<uint64_t>(d.rng[0]);
    key.k0 = static_cast<uint32_t>(seed);
    key.k1 = static_cast<uint32_t>(seed >> 32);
    key.step = static_cast<uint32_t>(d.rng[1]);
  }
  return key;
}

__device__ inline void dropout_words(const Dropout& d, DropoutKey key, int64_t block,
                                     uint32_t (&w)[4]) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32);
  uint32_t c2 = d.site, c3 = key.step;
  uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int round = 0; round < 7; ++round) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// Bit e: element e of the block is dropped.
__device__ inline uint32_t dropped_of_block(const Dropout& d, DropoutKey key, int64_t block) {
  uint32_t w[4];
  dropout_words(d, key, block, w);
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t field = e % 2 ? w[e / 2] : w[e / 2] << 16;
    bits |= static_cast<uint32_t>(field <= d.drop_max) << e;
  }
  return bits;
}

// Bit e: element `first + e` of the flattened tensor is dropped, for e < N; `first` is a multiple
// of N, so that the N elements lie in one block.
template <int N>
__device__ inline uint32_t dropped_from(const Dropout& d, DropoutKey key, int64_t first) {
  const uint32_t bits = dropped_of_block(d, key, first >> 3);
  return N < 8 ? bits >> (first & 7) : bits;
}

template <int N>
__device__ inline void apply_dropout(const Dropout& d, uint32_t dropped, float (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (dropped >> e) & 1 ? 0.0f : v[e] * d.scale;
}

// Host: fills `d` for a probability in [0, 1]; false outside.  p is rounded to a multiple of
// 2^-16, but to 0 and 1 only where it is 0 or 1.
inline bool make_dropout(double p, const int64_t* rng, uint32_t site, Dropout& d) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  d = Dropout{rng, site, 0, 1.0f, 0};
  if (p == 0.0) return true;
  long limit = lrint(p * 65536.0);
  if (limit < 1) limit = 1;
  if (limit > 65535) limit = p < 1.0 ? 65535 : 65536;
  d.drop_max = (static_cast<uint32_t>(limit - 1) << 16) | 0xFFFFu;
  d.scale = limit == 65536 ? 0.0f : static_cast<float>(65536.0 / (65536.0 - limit));
  d.active = 1;
  return true;
}

// A chunk of a tensor of rows, in registers.  Chunks lie on 16-byte boundaries of the flattened
// tensor.  WHOLE: rows are whole chunks.  Otherwise a row begins and ends inside a chunk; the
// column `col` of a chunk's first element may then be negative, and elements outside
// [0, width) belong to the neighbouring rows.
// Every load is made (for a chunk past the row's end of its first chunk): a branch would wait
// for each load by itself.  STREAM: read once (past the L2's other lines).
template <typename T, bool WHOLE, bool STREAM>
struct RowChunk {
  static constexpr int N = Chunk<T>::N;
  using Vector = typename Chunk<T>::type;
  Vector v;

  // `base`: the row's first element, `first_col`: the column of its first chunk; `total`: the
  // tensor's elements, whose last chunk may be a part of one.
  __device__ void load(const T* tensor, int64_t base, int col, int first_col, int width,
                       int64_t total) {
    const int64_t at = base + (col < width ? col : first_col);
    if (WHOLE || at + N <= total) {
      const auto* p = reinterpret_cast<const Vector*>(tensor + at);
      if constexpr (STREAM)
        v = __builtin_nontemporal_load(p);
      else
        v = *p;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = tensor[at + e < total ? at + e : total - 1];
    }
  }

  __device__ void floats(int col, int width, float (&out)[N]) const {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool live = WHOLE ? col < width : col + e >= 0 && col + e < width;
      out[e] = live ? static_cast<float>(v[e]) : 0.0f;
    }
  }
};

// The weights of a chunk's columns (fp32 beside 16-bit rows: two accesses).
template <typename W, int N, bool WHOLE>
struct WeightChunk {
  static constexpr int C = Chunk<W>::N, kPieces = N / C;
  typename Chunk<W>::type v[kPieces];

  __device__ void load(const W* weights, int col, int width) {
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      if constexpr (WHOLE) {
        v[c] = *reinterpret_cast<const typename Chunk<W>::type*>(
            weights + (col < width ? col : 0) + c * C);
      } else {
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const int at = col + c * C + e;
          v[c][e] = weights[at < 0 ? 0 : at < width ? at : width - 1];
        }
      }
    }
  }

  // The same of 16-bit weights staged in LDS, weight i at staged[8 + i] and two whole chunks
  // after the last that is asked for: two aligned accesses, shifted together.
  __device__ void load_staged(const W* staged, int col) {
    static_assert(sizeof(W) == 2 && kPieces == 1, "16-bit weights of 16-bit rows");
    typedef uint32_t Four __attribute__((ext_vector_type(4)));
    const uint32_t at = col + 8;  // (col is above -8)
    const Four* p = reinterpret_cast<const Four*>(staged) + at / 8;
    const Four low = p[0], high = p[1];
    const uint32_t a[8] = {low[0], low[1], low[2], low[3], high[0], high[1], high[2], high[3]};
    uint32_t b[6], c[5];
    Four d;
    // (Values: a choice between elements of an array would put it into memory.)
    auto select = [](uint32_t bit, uint32_t one, uint32_t zero) { return bit ? one : zero; };
#pragma unroll
    for (int i = 0; i < 6; ++i) b[i] = select(at & 4, a[i + 2], a[i]);
#pragma unroll
    for (int i = 0; i < 5; ++i) c[i] = select(at & 2, b[i + 1], b[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = __builtin_amdgcn_alignbit(c[i + 1], c[i], (at & 1) * 16);
    v[0] = __builtin_bit_cast(typename Chunk<W>::type, d);
  }

  // Makes the compiler take the weights as new here: their fp32 values, the same for every
  // row, are not kept in registers across the rows' loop.
  __device__ void renew() {
#pragma unroll
    for (int c = 0; c < kPieces; ++c) asm volatile("" : "+v"(v[c]));
  }

  __device__ void floats(float (&out)[N]) const {
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
#pragma unroll
      for (int e = 0; e < C; ++e) out[c * C + e] = static_cast<float>(v[c][e]);
    }
  }
};

// Outputs are written once: non-temporal, 10 % of a pass over rows (LayerNorm forward of
// 16384 x 768 bf16 17.9 -> 15.9 us, backward 32.8 -> 30.6; of 4096 rows 6.0 -> 5.5, 14.4 -> 12.5).
template <typename T, bool WHOLE>
__device__ inline void store_chunk(T* tensor, int64_t base, int col, int width,
                                   const float (&in)[Chunk<T>::N]) {
  constexpr int N = Chunk<T>::N;
  if (WHOLE ? col < width : col >= 0 && col + N <= width) {
    typename Chunk<T>::type v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = static_cast<T>(in[e]);
    __builtin_nontemporal_store(v,
                                reinterpret_cast<typename Chunk<T>::type*>(tensor + base + col));
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (col + e >= 0 && col + e < width) tensor[base + col + e] = static_cast<T>(in[e]);
  }
}

// N elements from p, one access (N = a chunk, or 1).
template <typename T, int N>
__device__ inline void load_floats(const T* p, float (&out)[N]) {
  typedef T Access __attribute__((ext_vector_type(N)));
  const Access v = *reinterpret_cast<const Access*>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = static_cast<float>(v[e]);
}

template <typename T, int N>
__device__ inline void store_floats(T* p, const float (&in)[N]) {
  typedef T Access __attribute__((ext_vector_type(N)));
  Access v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = static_cast<T>(in[e]);
  __builtin_nontemporal_store(v, reinterpret_cast<Access*>(p));
}

}  // namespace dflash
