// LayerNorm of a training step, joined with the dropout and the residual before it
// (DebertaV2SelfOutput / DebertaV2Output in training: LayerNorm(dropout(dense(x)) + input)),
// and its backward pass.
//
//   s = drop(x) + r            xh = (s - mean(s)) * rstd,  rstd = 1 / sqrt(var(s) + eps)
//   y = xh * gamma + beta
//   g = dy * gamma             ds = rstd * (g - mean(g) - xh * mean(g * xh))
//   dr = ds,  dx = drop'(ds)   dgamma = sum over rows of dy * xh,  dbeta = sum over rows of dy
//
// All of it in fp32, each result rounded once.  s is not kept: the backward pass reads x and
// r again and draws the mask again, which moves as many bytes as writing s and
// reading it back, and does not round s to 16 bits.  What is kept is mean and rstd, 8
// bytes a row.
//
// Layout: LANES lanes hold a row, CH chunks of 16 bytes a lane, so a row is read once and
// stays in registers between its statistics and its output.  Rows that are not whole
// chunks on 16-byte boundaries take the same kernels with element accesses.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dflash.h"
#include "training.h"

namespace dflash {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHidden = 8192;
// Workgroups of the backward pass: each adds up the weight gradients of its rows and writes
// one fp32 partial row of each.
constexpr int kMaxPartials = 512;

struct Forward {
  const void *x, *residual, *gamma, *beta;
  void* y;
  float *mean, *rstd;  // null: not kept
  int64_t rows;
  int hidden;
  float eps;
  Dropout drop;
};

struct Backward {
  const void *dy, *x, *residual, *gamma;
  const float *mean, *rstd;
  void *dx, *dresidual, *dgamma, *dbeta;  // null: not wanted (dgamma and dbeta together)
  float* partials;                        // [workgroups, 2, hidden]
  int64_t rows;
  int hidden;
  Dropout drop;
};

// Sum over the LANES lanes of a row.  LANES = 256 (a row a workgroup): every thread calls it.
template <int LANES, int VALUES>
__device__ inline void row_sum(float (&v)[VALUES], float (*lds)[VALUES]) {
  constexpr int kSpan = LANES < 64 ? LANES : 64;
#pragma unroll
  for (int m = kSpan / 2; m >= 1; m >>= 1) {
#pragma unroll
    for (int i = 0; i < VALUES; ++i) v[i] += __shfl_xor(v[i], m);
  }
  if constexpr (LANES > 64) {
    constexpr int kRowWaves = LANES / 64;
    __syncthreads();  // the values of the call before have been read
    if (threadIdx.x % 64 == 0) {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) lds[threadIdx.x / 64][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
      v[i] = lds[0][i];
#pragma unroll
      for (int w = 1; w < kRowWaves; ++w) v[i] += lds[w][i];
    }
  }
}

// s = drop(x) + r of this lane's chunks (0 past the row's end); `dropped`: their mask.
template <typename T, int LANES, int CH, bool WIDE>
__device__ inline void load_sum(const T* x, const T* r, int64_t base, int hidden, int sub,
                                const Dropout& drop, DropoutKey key,
                                float (&s)[CH][Chunk<T>::N], uint32_t (&dropped)[CH]) {
  constexpr int N = Chunk<T>::N;
  float rv[CH][N];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int col = (sub + LANES * k) * N;
    const int live = hidden - col;
    dropped[k] = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) s[k][e] = rv[k][e] = 0.0f;
    if (live > 0) {
      load_floats<T, N, WIDE>(x + base + col, live, s[k]);
      if (r) load_floats<T, N, WIDE>(r + base + col, live, rv[k]);
    }
  }
  if (drop.active) {
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int col = (sub + LANES * k) * N;
      if (col < hidden) dropped[k] = dropped_from<N, WIDE>(drop, key, base + col);
#pragma unroll
      for (int e = 0; e < N; ++e) s[k][e] = (dropped[k] >> e) & 1 ? 0.0f : s[k][e] * drop.scale;
    }
  }
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < N; ++e) s[k][e] += rv[k][e];
  }
}

template <typename T, typename W, int LANES, int CH, bool WIDE>
__global__ __launch_bounds__(kThreads) void layernorm_train_fwd_kernel(Forward a) {
  constexpr int N = Chunk<T>::N;
  __shared__ float lds[LANES > 64 ? LANES / 64 : 1][1];
  const int sub = threadIdx.x % LANES;
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  if (row >= a.rows) return;  // all lanes of a row together
  const int hidden = a.hidden;
  const int64_t base = row * hidden;
  const DropoutKey key = dropout_key(a.drop);
  float s[CH][N];
  uint32_t dropped[CH];
  load_sum<T, LANES, CH, WIDE>(static_cast<const T*>(a.x), static_cast<const T*>(a.residual), base,
                               hidden, sub, a.drop, key, s, dropped);
  float sum[1] = {0.0f};
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < N; ++e) sum[0] += s[k][e];
  }
  row_sum<LANES>(sum, lds);
  // (A division, not a product with 1 / hidden: equal elements have a variance of exactly 0.)
  const float width = static_cast<float>(hidden);
  const float mean = sum[0] / width;
  float sq[1] = {0.0f};
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int col = (sub + LANES * k) * N;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      s[k][e] -= mean;
      if (WIDE ? col < hidden : col + e < hidden) sq[0] += s[k][e] * s[k][e];
    }
  }
  row_sum<LANES>(sq, lds);
  const float rstd = rsqrtf(sq[0] / width + a.eps);
  if (sub == 0 && a.mean) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const W* gamma = static_cast<const W*>(a.gamma);
  const W* beta = static_cast<const W*>(a.beta);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int col = (sub + LANES * k) * N;
    const int live = hidden - col;
    if (live > 0) {
      float g[N], b[N];
      load_floats<W, N, WIDE>(gamma + col, live, g);
      load_floats<W, N, WIDE>(beta + col, live, b);
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = s[k][e] * rstd * g[e] + b[e];
      store_floats<T, N, WIDE>(static_cast<T*>(a.y) + base + col, live, g);
    }
  }
}

// A workgroup walks its rows (every gridDim-th group of kThreads / LANES rows) with the sums
// for dgamma and dbeta of its columns in registers; at the end the lanes that hold
// the same columns are added in order and one partial row is written.
template <typename T, typename W, int LANES, int CH, bool WIDE>
__global__ __launch_bounds__(kThreads) void layernorm_train_bwd_kernel(Backward a) {
  constexpr int N = Chunk<T>::N;
  constexpr int kGroups = kThreads / LANES;
  __shared__ float lds[LANES > 64 ? LANES / 64 : 1][2];
  __shared__ float part[kGroups > 1 ? kGroups : 1][kGroups > 1 ? LANES * CH * N : 1];
  const int sub = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int hidden = a.hidden;
  const float inv_h = 1.0f / static_cast<float>(hidden);
  const DropoutKey key = dropout_key(a.drop);
  const T* dy = static_cast<const T*>(a.dy);
  float gamma[CH][N], dgamma[CH][N], dbeta[CH][N];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int col = (sub + LANES * k) * N;
#pragma unroll
    for (int e = 0; e < N; ++e) gamma[k][e] = dgamma[k][e] = dbeta[k][e] = 0.0f;
    if (col < hidden)
      load_floats<W, N, WIDE>(static_cast<const W*>(a.gamma) + col, hidden - col, gamma[k]);
  }
  // (LANES = 256: the row is the workgroup's, so every thread makes the same rounds.)
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group; row < a.rows;
       row += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t base = row * hidden;
    float g[CH][N], xh[CH][N];
    uint32_t dropped[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int col = (sub + LANES * k) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) g[k][e] = 0.0f;
      if (col < hidden) load_floats<T, N, WIDE>(dy + base + col, hidden - col, g[k]);
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    load_sum<T, LANES, CH, WIDE>(static_cast<const T*>(a.x), static_cast<const T*>(a.residual),
                                 base, hidden, sub, a.drop, key, xh, dropped);
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      // (Past the row's end g is 0, so xh adds nothing there.)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        xh[k][e] = (xh[k][e] - mean) * rstd;
        dbeta[k][e] += g[k][e];
        dgamma[k][e] += g[k][e] * xh[k][e];
        g[k][e] *= gamma[k][e];
        sums[0] += g[k][e];
        sums[1] += g[k][e] * xh[k][e];
      }
    }
    if (!a.dx && !a.dresidual) continue;
    row_sum<LANES>(sums, lds);
    const float g_mean = sums[0] * inv_h, gx_mean = sums[1] * inv_h;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int col = (sub + LANES * k) * N;
      const int live = hidden - col;
      if (live > 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) g[k][e] = rstd * (g[k][e] - g_mean - xh[k][e] * gx_mean);
        if (a.dresidual)
          store_floats<T, N, WIDE>(static_cast<T*>(a.dresidual) + base + col, live, g[k]);
        if (a.dx) {
          if (a.drop.active) {
#pragma unroll
            for (int e = 0; e < N; ++e)
              g[k][e] = (dropped[k] >> e) & 1 ? 0.0f : g[k][e] * a.drop.scale;
          }
          store_floats<T, N, WIDE>(static_cast<T*>(a.dx) + base + col, live, g[k]);
        }
      }
    }
  }
  if (!a.dgamma) return;
  float* out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * hidden;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[CH][N] = which == 0 ? dgamma : dbeta;
    if constexpr (kGroups > 1) {
      if (which == 1) __syncthreads();
#pragma unroll
      for (int k = 0; k < CH; ++k) {
#pragma unroll
        for (int e = 0; e < N; ++e) part[group][(sub + LANES * k) * N + e] = acc[k][e];
      }
      __syncthreads();
      for (int col = threadIdx.x; col < hidden; col += kThreads) {
        float v = part[0][col];
#pragma unroll
        for (int i = 1; i < kGroups; ++i) v += part[i][col];
        out[which * hidden + col] = v;
      }
    } else {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int col = (sub + LANES * k) * N;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (col + e < hidden) out[which * hidden + col + e] = acc[k][e];
      }
    }
  }
}

// dgamma and dbeta: the partial rows added in order, 16 columns a workgroup, 16 threads a
// column each adding a contiguous range of the rows.
template <typename W>
__global__ __launch_bounds__(kThreads) void layernorm_weight_grad_kernel(
    const float* __restrict__ partials, int count, int hidden, W* __restrict__ dgamma,
    W* __restrict__ dbeta) {
  __shared__ float lds[16][17];
  const int lane = threadIdx.x % 16, slice = threadIdx.x / 16;
  const int col = blockIdx.x * 16 + lane;
  const int per = (count + 15) / 16;
  const int begin = slice * per;
  const int end = begin + per < count ? begin + per : count;
  float v = 0.0f;
  if (col < 2 * hidden) {
#pragma unroll 8
    for (int i = begin; i < end; ++i) v += partials[static_cast<int64_t>(i) * 2 * hidden + col];
  }
  lds[slice][lane] = v;
  __syncthreads();
  if (slice == 0 && col < 2 * hidden) {
#pragma unroll
    for (int i = 1; i < 16; ++i) v += lds[i][lane];
    if (col < hidden)
      dgamma[col] = static_cast<W>(v);
    else
      dbeta[col - hidden] = static_cast<W>(v);
  }
}

// Calls go(LANES, CH, WIDE) with the smallest layout that holds a row of `hidden` elements.
template <typename T, typename Go>
int with_layout(int hidden, bool wide, Go go) {
  const int chunks = (hidden + Chunk<T>::N - 1) / Chunk<T>::N;
#define DFLASH_LAYOUT(L, C)                                                            \
  if (chunks <= L * C)                                                                 \
    return wide ? go(std::integral_constant<int, L>(), std::integral_constant<int, C>(), \
                     std::true_type())                                                 \
                : go(std::integral_constant<int, L>(), std::integral_constant<int, C>(), \
                     std::false_type());
  DFLASH_LAYOUT(16, 1)
  DFLASH_LAYOUT(32, 1)
  DFLASH_LAYOUT(32, 2)
  DFLASH_LAYOUT(32, 3)
  DFLASH_LAYOUT(32, 4)
  DFLASH_LAYOUT(64, 3)
  DFLASH_LAYOUT(64, 4)
  DFLASH_LAYOUT(256, 2)
  DFLASH_LAYOUT(256, 4)
  if constexpr (Chunk<T>::N == 4) {
    DFLASH_LAYOUT(256, 8)
  }
#undef DFLASH_LAYOUT
  return DFLASH_ERR_SHAPE;
}

template <typename T, typename W>
int launch_forward(const Forward& a, bool wide, hipStream_t stream) {
  return with_layout<T>(a.hidden, wide, [&](auto lanes, auto ch, auto is_wide) {
    constexpr int kLanes = decltype(lanes)::value, kCh = decltype(ch)::value;
    constexpr int kRows = kThreads / kLanes;
    const int64_t blocks = (a.rows + kRows - 1) / kRows;
    if (blocks > kMaxBlocks256) return static_cast<int>(DFLASH_ERR_TOO_LARGE);
    hipLaunchKernelGGL((layernorm_train_fwd_kernel<T, W, kLanes, kCh, decltype(is_wide)::value>),
                       dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, stream, a);
    return static_cast<int>(hipGetLastError());
  });
}

int64_t partial_rows(int64_t rows) { return rows < kMaxPartials ? rows : kMaxPartials; }

template <typename T, typename W>
int launch_backward(const Backward& a, bool wide, hipStream_t stream) {
  int count = 0;
  if (a.rows > 0) {
    const int rc = with_layout<T>(a.hidden, wide, [&](auto lanes, auto ch, auto is_wide) {
      constexpr int kLanes = decltype(lanes)::value, kCh = decltype(ch)::value;
      constexpr int kRows = kThreads / kLanes;
      const int64_t blocks = (a.rows + kRows - 1) / kRows;
      count = static_cast<int>(blocks < kMaxPartials ? blocks : kMaxPartials);
      hipLaunchKernelGGL((layernorm_train_bwd_kernel<T, W, kLanes, kCh, decltype(is_wide)::value>),
                         dim3(count), dim3(kThreads), 0, stream, a);
      return static_cast<int>(hipGetLastError());
    });
    if (rc != DFLASH_OK) return rc;
  }
  if (!a.dgamma) return DFLASH_OK;
  hipLaunchKernelGGL((layernorm_weight_grad_kernel<W>), dim3((2 * a.hidden + 15) / 16),
                     dim3(kThreads), 0, stream, a.partials, count, a.hidden,
                     static_cast<W*>(a.dgamma), static_cast<W*>(a.dbeta));
  return static_cast<int>(hipGetLastError());
}

// Calls f(T, W) with the element types of the codes; weights are of the activations' type or
// fp32.
template <typename F>
int with_types(int dtype, int weight_dtype, F f) {
  if (dtype == DFLASH_DTYPE_FP32)
    return weight_dtype == DFLASH_DTYPE_FP32 ? f(float(), float()) : DFLASH_ERR_DTYPE;
  if (dtype == DFLASH_DTYPE_FP16) {
    if (weight_dtype == DFLASH_DTYPE_FP16) return f(_Float16(), _Float16());
    if (weight_dtype == DFLASH_DTYPE_FP32) return f(_Float16(), float());
  } else if (dtype == DFLASH_DTYPE_BF16) {
    if (weight_dtype == DFLASH_DTYPE_BF16) return f(__bf16(), __bf16());
    if (weight_dtype == DFLASH_DTYPE_FP32) return f(__bf16(), float());
  }
  return DFLASH_ERR_DTYPE;
}

uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

int element_size(int dtype) { return dtype == DFLASH_DTYPE_FP32 ? 4 : 2; }

bool shape_taken(int64_t rows, int hidden) {
  return rows >= 0 && hidden >= 1 && hidden <= kMaxHidden && rows <= INT64_MAX / 4 / kMaxHidden;
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" int dflash_dropout_layernorm_fwd(const void* x, const void* residual, const void* gamma,
                                            const void* beta, void* y, float* mean, float* rstd,
                                            int64_t rows, int hidden, float eps, double p,
                                            const int64_t* rng, uint32_t site, int dtype,
                                            int weight_dtype, void* stream) {
  Forward a{x, residual, gamma, beta, y, mean, rstd, rows, hidden, eps, {}};
  if (!shape_taken(rows, hidden) || !make_dropout(p, rng, site, a.drop)) return DFLASH_ERR_SHAPE;
  return with_types(dtype, weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    if (rows == 0) return static_cast<int>(DFLASH_OK);
    if (!x || !gamma || !beta || !y || !mean != !rstd || (a.drop.active && !rng))
      return static_cast<int>(DFLASH_ERR_NULL);
    const uintptr_t rows_or = address(x) | address(residual) | address(y);
    const uintptr_t weights_or = address(gamma) | address(beta);
    if (rows_or % sizeof(T) != 0 || weights_or % sizeof(W) != 0 ||
        (address(mean) | address(rstd)) % 4 != 0 || address(rng) % 8 != 0)
      return static_cast<int>(DFLASH_ERR_ALIGN);
    const bool wide = hidden % Chunk<T>::N == 0 && (rows_or | weights_or) % 16 == 0;
    return launch_forward<T, W>(a, wide, static_cast<hipStream_t>(stream));
  });
}

extern "C" size_t dflash_dropout_layernorm_bwd_workspace_bytes(int64_t rows, int hidden) {
  if (!shape_taken(rows, hidden)) return 0;
  return static_cast<size_t>(partial_rows(rows)) * 2 * hidden * sizeof(float);
}

extern "C" int dflash_dropout_layernorm_bwd(
    const void* dy, const void* x, const void* residual, const void* gamma, const float* mean,
    const float* rstd, void* dx, void* dresidual, void* dgamma, void* dbeta, int64_t rows,
    int hidden, double p, const int64_t* rng, uint32_t site, int dtype, int weight_dtype,
    void* workspace, size_t workspace_bytes, void* stream) {
  Backward a{dy,     x,      residual, gamma, mean, rstd, dx, dresidual, dgamma,
             dbeta,  static_cast<float*>(workspace), rows, hidden, {}};
  if (!shape_taken(rows, hidden) || !make_dropout(p, rng, site, a.drop)) return DFLASH_ERR_SHAPE;
  return with_types(dtype, weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    if (!dgamma != !dbeta) return static_cast<int>(DFLASH_ERR_NULL);
    if (rows > 0 && (!dy || !x || !gamma || !mean || !rstd || (a.drop.active && !rng)))
      return static_cast<int>(DFLASH_ERR_NULL);
    const uintptr_t rows_or = address(dy) | address(x) | address(residual) | address(dx) |
                              address(dresidual);
    const uintptr_t weights_or = address(gamma) | address(dgamma) | address(dbeta);
    if (rows_or % sizeof(T) != 0 || weights_or % sizeof(W) != 0 ||
        (address(mean) | address(rstd) | address(workspace)) % 4 != 0 || address(rng) % 8 != 0)
      return static_cast<int>(DFLASH_ERR_ALIGN);
    if (dgamma && rows > 0) {
      if (!workspace) return static_cast<int>(DFLASH_ERR_NULL);
      if (workspace_bytes < dflash_dropout_layernorm_bwd_workspace_bytes(rows, hidden))
        return static_cast<int>(DFLASH_ERR_WORKSPACE);
    }
    if (!dx && !dresidual && !dgamma) return static_cast<int>(DFLASH_OK);
    const bool wide = hidden % Chunk<T>::N == 0 && rows_or % 16 == 0 && address(gamma) % 16 == 0;
    return launch_backward<T, W>(a, wide, static_cast<hipStream_t>(stream));
  });
}
