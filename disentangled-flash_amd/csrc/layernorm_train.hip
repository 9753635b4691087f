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
// stays in registers between its statistics and its output.  Rows that are not whole chunks
// take the same accesses, on the 16-byte boundaries of the flattened tensor: a row then begins
// `shift` elements inside its first chunk.  A group of lanes only meets rows of one shift (they
// are a multiple of a chunk's elements apart), so its weights and the sums for their gradients
// stay with the lanes; only a row's first and last chunk are written by elements.
//
// Bound by bytes: 16384 x 768 bf16 with residual and dropout 16.3 us forward (75 MB, 4.6 TB/s)
// and 25.0 + 4.0 backward (129 MB with the partial rows, 5.2 TB/s, and the second launch); 16384 x
// 1536 fp32 54.4 (5.6 TB/s) and 84.3 + 4.7 us (6.0).  A copy of as many bytes runs at 4.5 to
// 5.4 TB/s.  (Device times of single launches, traced; those below are of many in a row, by
// events: 15.9 and 29.7, 55 and 89.)  16384 x 769 bf16: 19.9 and 39.4 us; 3059 x 1001: 7.7 and
// 18.0 (by element accesses 17.0 and 28.0).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "device_common.h"
#include "dflash.h"
#include "training.h"

namespace dflash {
namespace {

constexpr int kMaxHidden = 8192;
// Workgroups of the backward pass: each adds up the weight gradients of its rows and writes
// one fp32 partial row of each.  (Backward, bf16, by 256, 512 and 1024: 2048 x 768 11.0, 11.0,
// 11.0 us; 4096 14.6, 13.3, 13.3; 8192 22.0, 19.8, 23.7; 65536 99.2, 93.4, 95.4; 3059 x 1000 14.5,
// 13.1, 15.2; 16384 x 769 55.2, 39.4, 44.6; 16384 x 1024 fp16 30.9, 24.4, 28.9.)
constexpr int kMaxPartials = 512;
// Up to this many rows one workgroup takes them all, and there are no partial rows to add: 17
// rows of 768 take 9.8 us alone, 5.4 + 2.7 and the gap between them in two launches, of
// which the host is spared one.
constexpr int kAloneRows = 32;
// Workgroups of the forward pass.  (16384 x 768 bf16: 1024 15.9 us, 2048 16.6; 1536 fp32 55, 58.)
constexpr int kMaxForward = 1024;

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

// Sums over groups of LANES (16, 32 or 64) neighbouring lanes, in every lane of the group:
// within 16 lanes by DPP operands of the additions (neighbour pairs, quads, halves, the whole),
// across them through scalar registers; nothing passes through LDS, whose latency
// a butterfly of shuffles takes once a step.
template <int CTRL>
__device__ inline float moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL,
                                                               0xF, 0xF, true));
}

__device__ inline float lane_value(float v, int lane) {
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

template <int LANES>
__device__ inline float group_sum(float v) {
  v += moved<0xB1>(v);   // quad_perm 1, 0, 3, 2
  v += moved<0x4E>(v);   // quad_perm 2, 3, 0, 1
  v += moved<0x141>(v);  // row_half_mirror
  v += moved<0x140>(v);  // row_mirror
  if constexpr (LANES >= 32) {
    const float low = lane_value(v, 0) + lane_value(v, 16);
    const float high = lane_value(v, 32) + lane_value(v, 48);
    // (LANES = 32: the half of a row that does not exist holds anything, and nobody takes it.)
    v = LANES == 64 ? low + high : threadIdx.x % 64 < 32 ? low : high;
  }
  return v;
}

// Sum over the LANES lanes of a row.  LANES = 256 (a row a workgroup): every thread calls it.
template <int LANES, int VALUES>
__device__ inline void row_sum(float (&v)[VALUES], float (*lds)[VALUES]) {
#pragma unroll
  for (int i = 0; i < VALUES; ++i) v[i] = group_sum<(LANES < 64 ? LANES : 64)>(v[i]);
  if constexpr (LANES > 64) {
    constexpr int kRowWaves = LANES / 64;
    // (Barriers that order LDS only: the next row's loads stay in flight.)
    lds_barrier();  // the values of the call before have been read
    if (threadIdx.x % 64 == 0) {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) lds[threadIdx.x / 64][i] = v[i];
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < VALUES; ++i) {
      v[i] = lds[0][i];
#pragma unroll
      for (int w = 1; w < kRowWaves; ++w) v[i] += lds[w][i];
    }
  }
}

// This lane's chunks of the next row to work on: loaded while the row before is worked on, so
// that the registers of their fp32 values and of the loads in flight are not the same ones.
// LAST: nobody reads them after the kernel (the forward pass's rows are read again by the
// backward pass).
template <typename T, int LANES, int CH, bool WHOLE, bool LAST>
struct RowInput {
  static constexpr int N = Chunk<T>::N;
  RowChunk<T, WHOLE, LAST> x[CH], r[CH];

  __device__ void load(const T* xs, const T* rs, int64_t base, int col, int first_col, int hidden,
                       int64_t total) {
#pragma unroll
    for (int k = 0; k < CH; ++k) x[k].load(xs, base, col + LANES * N * k, first_col, hidden, total);
    if (rs) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
        r[k].load(rs, base, col + LANES * N * k, first_col, hidden, total);
    }
  }

  // s = drop(x) + r (0 outside the row); `dropped`: the masks of the chunks, drawn while the
  // loads are in flight.
  __device__ void sum(bool has_r, int64_t base, int col, int hidden, const Dropout& drop,
                      DropoutKey key, float (&s)[CH][N], uint32_t (&dropped)[CH]) const {
    if (drop.active) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
        dropped[k] = dropped_from<N>(drop, key, base + col + LANES * N * k);
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        x[k].floats(col + LANES * N * k, hidden, s[k]);
        apply_dropout(drop, dropped[k], s[k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < CH; ++k) x[k].floats(col + LANES * N * k, hidden, s[k]);
    }
    if (has_r) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        float v[N];
        r[k].floats(col + LANES * N * k, hidden, v);
#pragma unroll
        for (int e = 0; e < N; ++e) s[k][e] += v[e];
      }
    }
  }
};

// gamma and beta in LDS, weight i of each at [8 + i], for 16-bit rows that begin inside a chunk:
// each thread loads a chunk of both, and stores it when the rows' loads are on their way.
template <typename W>
struct WeightStage {
  using Vector = typename Chunk<W>::type;
  static constexpr int C = Chunk<W>::N;
  Vector gamma, beta;
  int at;
  bool whole;

  __device__ void load(const W* gammas, const W* betas, int hidden) {
    const uintptr_t both = reinterpret_cast<uintptr_t>(gammas) | reinterpret_cast<uintptr_t>(betas);
    at = threadIdx.x * C;
    whole = both % 16 == 0 && at + C <= hidden;
    if (whole) {
      gamma = *reinterpret_cast<const Vector*>(gammas + at);
      beta = *reinterpret_cast<const Vector*>(betas + at);
    }
  }

  __device__ void store(const W* gammas, const W* betas, int hidden, W* lds_gamma, W* lds_beta) {
    if (whole) {
      *reinterpret_cast<Vector*>(lds_gamma + 8 + at) = gamma;
      *reinterpret_cast<Vector*>(lds_beta + 8 + at) = beta;
    } else {
      for (int e = at; e < at + C && e < hidden; ++e) {
        lds_gamma[8 + e] = gammas[e];
        lds_beta[8 + e] = betas[e];
      }
    }
    lds_barrier();
  }
};

// A workgroup walks its rows, every gridDim-th group of kThreads / LANES rows.  (LANES = 256:
// the row is the workgroup's, so every thread makes the same rounds.)  Without WHOLE the step is
// a multiple of N or there is no second round (the launch sees to it).
template <typename T, typename W, int LANES, int CH, bool WHOLE>
__global__ __launch_bounds__(kThreads) void layernorm_train_fwd_kernel(Forward a) {
  constexpr int N = Chunk<T>::N;
  constexpr int kGroups = kThreads / LANES;
  __shared__ float lds[LANES > 64 ? LANES / 64 : 1][1];
  const int sub = threadIdx.x % LANES;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / LANES;
  // 16-bit weights that lie askew of the row's chunks pass through LDS: 3059 x 1001 bf16, where a
  // group has one row, 7.7 us instead of 10.5 with 32 element loads a lane; 16384 x 769 20.1, 23.0.
  // (The backward pass has gamma alone and more rows a group: 0.5 us of 18 are its weights'.  Rows
  // wider than a wavefront holds are a workgroup's, which has no other group to share them with.)
  constexpr bool kStaged = !WHOLE && LANES <= 64 && sizeof(W) == 2;
  __shared__ alignas(16) W staged[2][kStaged ? (LANES * CH + 2) * 8 : 8];
  static_assert(!kStaged || LANES * CH * N <= kThreads * Chunk<W>::N, "a chunk a thread");
  WeightStage<W> stage;
  if constexpr (kStaged)
    stage.load(static_cast<const W*>(a.gamma), static_cast<const W*>(a.beta), a.hidden);
  else if (row >= a.rows)
    return;  // all lanes of a row together
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int hidden = a.hidden;
  const float width = static_cast<float>(hidden);
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.residual);
  const int64_t total = a.rows * hidden;
  const int64_t first_row = row < a.rows ? row : a.rows - 1;
  const int first_col = WHOLE ? 0 : -static_cast<int>(first_row * hidden % N);
  const int lane_col = sub * N + first_col;  // + LANES * N a chunk
  RowInput<T, LANES, CH, WHOLE, false> in;
  in.load(x, r, first_row * hidden, lane_col, first_col, hidden, total);
  if constexpr (kStaged) {
    stage.store(static_cast<const W*>(a.gamma), static_cast<const W*>(a.beta), hidden, staged[0],
                staged[1]);
    if (row >= a.rows) return;
  }
  WeightChunk<W, N, WHOLE> gamma[CH], beta[CH];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if constexpr (kStaged) {
      gamma[k].load_staged(staged[0], lane_col + LANES * N * k);
      beta[k].load_staged(staged[1], lane_col + LANES * N * k);
    } else {
      gamma[k].load(static_cast<const W*>(a.gamma), lane_col + LANES * N * k, hidden);
      beta[k].load(static_cast<const W*>(a.beta), lane_col + LANES * N * k, hidden);
    }
  }
  const DropoutKey key = dropout_key(a.drop);
  for (;;) {
    float s[CH][N];
    uint32_t dropped[CH];
    in.sum(r != nullptr, row * hidden, lane_col, hidden, a.drop, key, s, dropped);
    const int64_t next = row + step;
    if (next < a.rows) in.load(x, r, next * hidden, lane_col, first_col, hidden, total);
    float sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum[0] += s[k][e];
    }
    row_sum<LANES>(sum, lds);
    // (A division, not a product with 1 / hidden: equal elements have a variance of exactly 0.)
    const float mean = sum[0] / width;
    float sq[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int col = lane_col + LANES * N * k;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        s[k][e] -= mean;
        const bool live = WHOLE ? col < hidden : col + e >= 0 && col + e < hidden;
        sq[0] += live ? s[k][e] * s[k][e] : 0.0f;
      }
    }
    row_sum<LANES>(sq, lds);
    const float rstd = rsqrtf(sq[0] / width + a.eps);
    if (sub == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float g[N], b[N];
      gamma[k].renew();
      beta[k].renew();
      gamma[k].floats(g);
      beta[k].floats(b);
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = s[k][e] * rstd * g[e] + b[e];
      store_chunk<T, WHOLE>(static_cast<T*>(a.y), row * hidden, lane_col + LANES * N * k, hidden,
                            g);
    }
    if (next >= a.rows) return;
    row = next;
  }
}

// As above, with the sums for dgamma and dbeta of the lane's columns in registers; at the end
// the lanes that hold the same columns are added in order and one partial row is written.
template <typename T, typename W, int LANES, int CH, bool WHOLE>
__global__ __launch_bounds__(kThreads) void layernorm_train_bwd_kernel(Backward a) {
  constexpr int N = Chunk<T>::N;
  constexpr int kGroups = kThreads / LANES;
  __shared__ float lds[LANES > 64 ? LANES / 64 : 1][2];
  __shared__ float part[kGroups > 1 ? kGroups : 1][kGroups > 1 ? LANES * CH * N : 1];
  const int sub = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int hidden = a.hidden;
  const float width = static_cast<float>(hidden);
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.residual);
  const T* dy = static_cast<const T*>(a.dy);
  int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t total = a.rows * hidden;
  const int first_col = WHOLE ? 0 : -static_cast<int>(row * hidden % N);
  const int lane_col = sub * N + first_col;  // + LANES * N a chunk
  RowInput<T, LANES, CH, WHOLE, true> in;
  RowChunk<T, WHOLE, true> dys[CH];
  WeightChunk<W, N, WHOLE> gamma[CH];
  float mean = 0.0f, rstd = 0.0f;
  auto load = [&](int64_t at) {
#pragma unroll
    for (int k = 0; k < CH; ++k)
      dys[k].load(dy, at * hidden, lane_col + LANES * N * k, first_col, hidden, total);
    in.load(x, r, at * hidden, lane_col, first_col, hidden, total);
    mean = a.mean[at];
    rstd = a.rstd[at];
  };
  // Narrow rows are loaded one ahead (1024 fp16, no dropout, 16384 rows: 27.5 -> 24.2 us); where
  // their registers cost wavefronts, not (1536 fp32: 98.7 ahead, 89.6 not; 1536 bf16 52.9,
  // 52.0; 768 bf16 30.2, 29.7).
  constexpr bool kAhead = WHOLE && LANES <= 64 && CH <= 2;
  if (kAhead && row < a.rows) load(row);
  const DropoutKey key = dropout_key(a.drop);
  float dgamma[CH][N], dbeta[CH][N];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    gamma[k].load(static_cast<const W*>(a.gamma), lane_col + LANES * N * k, hidden);
#pragma unroll
    for (int e = 0; e < N; ++e) dgamma[k][e] = dbeta[k][e] = 0.0f;
  }
  while (row < a.rows) {
    if (!kAhead) load(row);
    const int64_t base = row * hidden;
    float g[CH][N], xh[CH][N];
    uint32_t dropped[CH];
    in.sum(r != nullptr, base, lane_col, hidden, a.drop, key, xh, dropped);
#pragma unroll
    for (int k = 0; k < CH; ++k) dys[k].floats(lane_col + LANES * N * k, hidden, g[k]);
    const float row_mean = mean, row_rstd = rstd;
    row += step;
    if (kAhead && row < a.rows) load(row);
    float sums[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float w[N];
      gamma[k].renew();
      gamma[k].floats(w);
      // (Outside the row g is 0, so xh adds nothing there.)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        xh[k][e] = (xh[k][e] - row_mean) * row_rstd;
        dbeta[k][e] += g[k][e];
        dgamma[k][e] += g[k][e] * xh[k][e];
        g[k][e] *= w[e];
        sums[0] += g[k][e];
        sums[1] += g[k][e] * xh[k][e];
      }
    }
    if (!a.dx && !a.dresidual) continue;
    row_sum<LANES>(sums, lds);
    const float g_mean = sums[0] / width, gx_mean = sums[1] / width;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int col = lane_col + LANES * N * k;
#pragma unroll
      for (int e = 0; e < N; ++e) g[k][e] = row_rstd * (g[k][e] - g_mean - xh[k][e] * gx_mean);
      if (a.dresidual)
        store_chunk<T, WHOLE>(static_cast<T*>(a.dresidual), base, col, hidden, g[k]);
      if (a.dx) {
        if (a.drop.active) apply_dropout(a.drop, dropped[k], g[k]);
        store_chunk<T, WHOLE>(static_cast<T*>(a.dx), base, col, hidden, g[k]);
      }
    }
  }
  if (!a.dgamma) return;
  // A workgroup alone has the whole sums.
  float* out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * hidden;
  auto put = [&](int which, int col, float v) {
    if (gridDim.x > 1)
      out[which * hidden + col] = v;
    else
      static_cast<W*>(which == 0 ? a.dgamma : a.dbeta)[col] = static_cast<W>(v);
  };
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[CH][N] = which == 0 ? dgamma : dbeta;
    if constexpr (kGroups > 1) {
      if (which == 1) __syncthreads();
#pragma unroll
      for (int k = 0; k < CH; ++k) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int col = lane_col + LANES * N * k + e;
          if (WHOLE || (col >= 0 && col < hidden)) part[group][col] = acc[k][e];
        }
      }
      __syncthreads();
      for (int col = threadIdx.x; col < hidden; col += kThreads) {
        float v = part[0][col];
#pragma unroll
        for (int i = 1; i < kGroups; ++i) v += part[i][col];
        put(which, col, v);
      }
    } else {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int col = lane_col + LANES * N * k;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (col + e >= 0 && col + e < hidden) put(which, col + e, acc[k][e]);
      }
    }
  }
}

// dgamma and dbeta: the partial rows added in order, 16 columns a workgroup, kSlices threads a
// column, each adding a contiguous range of the rows (8 of 512: one round of loads).
constexpr int kSlices = 64;

template <typename W>
__global__ __launch_bounds__(16 * kSlices) void layernorm_weight_grad_kernel(
    const float* __restrict__ partials, int count, int hidden, W* __restrict__ dgamma,
    W* __restrict__ dbeta) {
  __shared__ float lds[kSlices][17];
  const int lane = threadIdx.x % 16, slice = threadIdx.x / 16;
  const int col = blockIdx.x * 16 + lane;
  const int per = (count + kSlices - 1) / kSlices;
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
    for (int i = 1; i < kSlices; ++i) v += lds[i][lane];
    if (col < hidden)
      dgamma[col] = static_cast<W>(v);
    else
      dbeta[col - hidden] = static_cast<W>(v);
  }
}

// Calls go(LANES, CH, WHOLE) with the smallest layout that holds a row of `hidden` elements: few
// chunks a lane, for their registers (1024 16-bit: 32 lanes of 4 chunks 32.5 us backward, 64 of
// 2 24.2), but 32 lanes of 3 before 64 of 2 half empty (768: 33.0, 34.8), and a row in
// one wavefront where three chunks a lane hold it (1536: 55.4, a workgroup a row 76.3).  Above 4
// chunks a lane of one wavefront a row is a workgroup's (forward and backward, against 8 chunks a
// lane: 8192 x 2560 bf16 30.9 and 61.8 us, 38.1 and 111.7; 4096 x 4096 20.1 and 49.3, 29.0 and
// 76.7; 16384 x 1536 fp32 55.0 and 89.7, 55.6 and 96.8; 4096 x 2048 19.6 and 36.9, 22.1 and 42.4).
// By the layouts that are a workgroup's alone: 2048 x 4096 fp32 20.6 and 42.0 us, 1024 x 8192 22.0
// and 59.3, 2048 x 8192 bf16 21.0 and 76.8, 4096 x 2051 21.2 and 43.0.
template <typename T, typename Go>
int with_layout(int hidden, bool whole, Go go) {
  constexpr int N = Chunk<T>::N;
  // A row that begins inside a chunk may touch one more.
  const int chunks = whole ? hidden / N : (hidden + 2 * (N - 1)) / N;
#define DFLASH_LAYOUT(L, C)                                                              \
  if (chunks <= L * C)                                                                   \
    return whole ? go(std::integral_constant<int, L>(), std::integral_constant<int, C>(), \
                      std::true_type())                                                  \
                 : go(std::integral_constant<int, L>(), std::integral_constant<int, C>(), \
                      std::false_type());
  DFLASH_LAYOUT(16, 1)
  DFLASH_LAYOUT(32, 1)
  DFLASH_LAYOUT(32, 2)
  DFLASH_LAYOUT(32, 3)
  DFLASH_LAYOUT(64, 2)
  DFLASH_LAYOUT(64, 3)
  DFLASH_LAYOUT(64, 4)
  DFLASH_LAYOUT(256, 2)
  DFLASH_LAYOUT(256, 4)
  if constexpr (N == 4) {
    DFLASH_LAYOUT(256, 8)
    DFLASH_LAYOUT(256, 9)  // 8191 elements that begin inside a chunk
  } else {
    DFLASH_LAYOUT(256, 5)
  }
#undef DFLASH_LAYOUT
  return DFLASH_ERR_SHAPE;
}

template <typename T, typename W>
int launch_forward(const Forward& a, bool whole, hipStream_t stream) {
  return with_layout<T>(a.hidden, whole, [&](auto lanes, auto ch, auto is_whole) {
    constexpr int kLanes = decltype(lanes)::value, kCh = decltype(ch)::value;
    constexpr int kRows = kThreads / kLanes;
    const int64_t blocks = (a.rows + kRows - 1) / kRows;
    const int count = static_cast<int>(blocks < kMaxForward ? blocks : kMaxForward);
    hipLaunchKernelGGL((layernorm_train_fwd_kernel<T, W, kLanes, kCh, decltype(is_whole)::value>),
                       dim3(count), dim3(kThreads), 0, stream, a);
    return static_cast<int>(hipGetLastError());
  });
}

// (Rows that are not whole chunks have their second round only a multiple of 8 rows on, which
// kMaxForward and kMaxPartials workgroups are apart and one workgroup is not.)
static_assert(kMaxForward % 8 == 0 && kMaxPartials % 8 == 0, "a multiple of a chunk's elements");
bool alone(int64_t rows, int hidden) { return rows <= kAloneRows && hidden % 8 == 0; }

int64_t partial_rows(int64_t rows, int hidden) {
  return alone(rows, hidden) ? 0 : rows < kMaxPartials ? rows : kMaxPartials;
}

template <typename T, typename W>
int launch_backward(const Backward& a, bool whole, hipStream_t stream) {
  int count = 0;
  if (a.rows > 0) {
    const int rc = with_layout<T>(a.hidden, whole, [&](auto lanes, auto ch, auto is_whole) {
      constexpr int kLanes = decltype(lanes)::value, kCh = decltype(ch)::value;
      constexpr int kRows = kThreads / kLanes;
      const int64_t blocks = (a.rows + kRows - 1) / kRows;
      count = static_cast<int>(blocks < kMaxPartials ? blocks : kMaxPartials);
      if (alone(a.rows, a.hidden)) count = 1;
      hipLaunchKernelGGL((layernorm_train_bwd_kernel<T, W, kLanes, kCh, decltype(is_whole)::value>),
                         dim3(count), dim3(kThreads), 0, stream, a);
      return static_cast<int>(hipGetLastError());
    });
    if (rc != DFLASH_OK) return rc;
  }
  if (!a.dgamma || count == 1) return DFLASH_OK;
  hipLaunchKernelGGL((layernorm_weight_grad_kernel<W>), dim3((2 * a.hidden + 15) / 16),
                     dim3(16 * kSlices), 0, stream, a.partials, count, a.hidden,
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
    if (rows_or % 16 != 0 || weights_or % sizeof(W) != 0 ||
        (address(mean) | address(rstd)) % 4 != 0 || address(rng) % 8 != 0)
      return static_cast<int>(DFLASH_ERR_ALIGN);
    const bool whole = hidden % Chunk<T>::N == 0 && weights_or % 16 == 0;
    return launch_forward<T, W>(a, whole, static_cast<hipStream_t>(stream));
  });
}

extern "C" size_t dflash_dropout_layernorm_bwd_workspace_bytes(int64_t rows, int hidden) {
  if (!shape_taken(rows, hidden)) return 0;
  return static_cast<size_t>(partial_rows(rows, hidden)) * 2 * hidden * sizeof(float);
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
    if (rows_or % 16 != 0 || weights_or % sizeof(W) != 0 ||
        (address(mean) | address(rstd) | address(workspace)) % 4 != 0 || address(rng) % 8 != 0)
      return static_cast<int>(DFLASH_ERR_ALIGN);
    if (dgamma && partial_rows(rows, hidden) > 0) {
      if (!workspace) return static_cast<int>(DFLASH_ERR_NULL);
      if (workspace_bytes < dflash_dropout_layernorm_bwd_workspace_bytes(rows, hidden))
        return static_cast<int>(DFLASH_ERR_WORKSPACE);
    }
    if (!dx && !dresidual && !dgamma) return static_cast<int>(DFLASH_OK);
    const bool whole = hidden % Chunk<T>::N == 0 && address(gamma) % 16 == 0;
    return launch_backward<T, W>(a, whole, static_cast<hipStream_t>(stream));
  });
}
