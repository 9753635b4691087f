// Dropout whose mask is drawn again wherever it is needed and never stored.
//
//   y = x / P(kept) where the element's 16 bits of the generator are at least 65536 p, else 0
//
// Forward and backward are the same kernel (dx is the same function of dy).  A dropped element
// is 0 whatever it held (infinities and NaN too): it is selected, not multiplied by 0.
// One 16-byte chunk a lane: n * sizeof(T) bytes read and written, and one generator block
// for 8 elements, drawn while the chunk is loaded.  Bound by bytes: 25 M bf16 elements take
// 19.5 us (5.2 TB/s), 4.7 M fp32 7.6 us (5.0 TB/s); 75 k fp16 2.5 us, most of it the launch.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dflash.h"
#include "training.h"

namespace dflash {
namespace {

// WIDE: x and y lie on 16-byte boundaries; otherwise element accesses.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                      int64_t n, Dropout d) {
  constexpr int N = Chunk<T>::N;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * N;
  if (first >= n) return;
  const DropoutKey key = dropout_key(d);
  typename Chunk<T>::type given{};
  if (WIDE && first + N <= n)  // in flight while the mask is drawn
    given = *reinterpret_cast<const typename Chunk<T>::type*>(x + first);
  const uint32_t dropped = dropped_from<N>(d, key, first);
  if (WIDE && first + N <= n) {
    RowChunk<T, true, false> chunk;
    chunk.v = given;
    float v[N];
    chunk.floats(0, N, v);
    apply_dropout(d, dropped, v);
    store_chunk<T, true>(y, first, 0, N, v);
  } else {  // the last chunk may be a part of one
    for (int e = 0; e < N && first + e < n; ++e) {
      const float v = static_cast<float>(x[first + e]);
      y[first + e] = static_cast<T>((dropped >> e) & 1 ? 0.0f : v * d.scale);
    }
  }
}

template <typename T>
int launch_dropout(const void* x, void* y, int64_t n, const Dropout& d, hipStream_t stream) {
  const int64_t per_block = 256 * Chunk<T>::N;
  const int64_t blocks = (n + per_block - 1) / per_block;
  if (blocks > kMaxBlocks256) return DFLASH_ERR_TOO_LARGE;
  const bool wide = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % 16 == 0;
  hipLaunchKernelGGL((wide ? &dropout_kernel<T, true> : &dropout_kernel<T, false>),
                     dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream,
                     static_cast<const T*>(x), static_cast<T*>(y), n, d);
  return static_cast<int>(hipGetLastError());
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" int dflash_dropout(const void* x, void* y, int64_t n, double p, const int64_t* rng,
                              uint32_t site, int dtype, void* stream) {
  Dropout d;
  if (n < 0 || !make_dropout(p, rng, site, d)) return DFLASH_ERR_SHAPE;
  if (dtype < DFLASH_DTYPE_FP16 || dtype > DFLASH_DTYPE_FP32) return DFLASH_ERR_DTYPE;
  if (n == 0) return DFLASH_OK;
  if (!x || !y || (d.active && !rng)) return DFLASH_ERR_NULL;
  const uintptr_t element = dtype == DFLASH_DTYPE_FP32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % element != 0 ||
      reinterpret_cast<uintptr_t>(rng) % 8 != 0)
    return DFLASH_ERR_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case DFLASH_DTYPE_FP16: return launch_dropout<_Float16>(x, y, n, d, s);
    case DFLASH_DTYPE_BF16: return launch_dropout<__bf16>(x, y, n, d, s);
    default: return launch_dropout<float>(x, y, n, d, s);
  }
}
