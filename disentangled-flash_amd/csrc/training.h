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

// Bit e: element `first + e` of the flattened tensor is dropped, for e < N.  WHOLE: first is a
// multiple of N, so that the N elements lie in one block.
template <int N, bool WHOLE>
__device__ inline uint32_t dropped_from(const Dropout& d, DropoutKey key, int64_t first) {
  const int at = static_cast<int>(first & 7);
  uint32_t bits = dropped_of_block(d, key, first >> 3);
  if constexpr (!WHOLE) {
    if (at + N > 8) bits |= dropped_of_block(d, key, (first >> 3) + 1) << 8;
  }
  if constexpr (!WHOLE || N < 8) bits >>= at;
  return bits;
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

// The chunk at column `col` of a row of `width` elements.  WIDE: rows are whole chunks from
// 16-byte boundaries.  Otherwise element loads.  Either way every load is made, past the row's
// end from a place inside it (a branch would wait for each load by itself);
// floats() puts the zeros there.  STREAM: read once (past the L2's other lines).
template <typename T, int N, bool WIDE, bool STREAM = false>
struct RowChunk {
  static constexpr int kPieces = N / Chunk<T>::N;  // 2: fp32 weights beside 16-bit rows
  typename Chunk<T>::type v[kPieces];

  __device__ void load(const T* row, int col, int width) {
    constexpr int C = Chunk<T>::N;
    if constexpr (WIDE) {
      const T* from = row + (col < width ? col : 0);
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const auto* p = reinterpret_cast<const typename Chunk<T>::type*>(from + c * C);
        if constexpr (STREAM)
          v[c] = __builtin_nontemporal_load(p);
        else
          v[c] = *p;
      }
    } else {
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const int at = col + c * C + e;
          v[c][e] = row[at < width ? at : width - 1];
        }
      }
    }
  }

  // Makes the compiler take the chunk as new here: what is computed from a chunk that is the
  // same for every row (its fp32 values) is not kept in registers across the rows' loop.
  __device__ void renew() {
#pragma unroll
    for (int c = 0; c < kPieces; ++c) asm volatile("" : "+v"(v[c]));
  }

  __device__ void floats(int col, int width, float (&out)[N]) const {
    constexpr int C = Chunk<T>::N;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const bool live = (WIDE ? col : col + c * C + e) < width;
        out[c * C + e] = live ? static_cast<float>(v[c][e]) : 0.0f;
      }
    }
  }
};

// Outputs are written once: non-temporal, 10 % of a pass over rows (LayerNorm forward of
// 16384 x 768 bf16 17.9 -> 15.9 us, backward 32.8 -> 30.6; of 4096 rows 6.0 -> 5.5, 14.4 -> 12.5).
template <typename T, int N, bool WIDE>
__device__ inline void store_chunk(T* row, int col, int width, const float (&in)[N]) {
  if constexpr (WIDE) {
    static_assert(N == Chunk<T>::N, "one chunk");
    typename Chunk<T>::type v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = static_cast<T>(in[e]);
    if (col < width)
      __builtin_nontemporal_store(v, reinterpret_cast<typename Chunk<T>::type*>(row + col));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (col + e < width) row[col + e] = static_cast<T>(in[e]);
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
