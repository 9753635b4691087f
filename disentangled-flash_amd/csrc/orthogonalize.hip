// Newton-Schulz iterations that bring a matrix's singular values near 1 (the update of the
// Muon optimiser), for a batch of matrices of one shape.
//
//   X = G / (|G|_F + eps);  steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// on the side on which X has no more rows than columns (a tall G is transposed on its way in and out).
//
// Precision.  The products run on fp16 MFMA with fp32 sums.  X is kept in two fp16 parts, hi + lo
// (22 bits), scaled by 2^8 (its entries are below 1 / sqrt(rows) on average, where fp16 would
// lose bits); hi is the operand, and both enter a X, which alone carries the small
// singular values, the ones that grow: with hi alone there a matrix of low rank beside noise is
// 6e-3 off after five steps, with both 4e-4.  A is rounded to fp16 once, for b A as for A A: were
// b A taken from its fp32 sums, the two would not cancel near 1 (normal 512 x 2048: 3.1e-3 off
// against 1.7e-3).  bf16 operands are 1.3e-2 to 5e-2 off.  The result is bf16 (1.7e-3 by itself).
// fp16 holds 2^8 X for singular values below 255, A then too, and B while |b s^2 + c s^4| is below 65504.
// In the last step hi alone enters a X too, above 128 rows: the roundings of X in a X and in B X
// then are one and the same, which p(s) nearly cancels where s is near 1.  By emulation of 768 x 768 a normal
// matrix is 1.3e-3 off before the result's rounding instead of 1.4e-3 with both parts, one of rank 20 beside noise
// 5.8e-4 instead of 2.4e-4 (2.1e-3, 2.2e-3, 1.76e-3 and 1.68e-3 with it); X's low part is not read again.
//
// One GEMM kernel, three forms.  All operands are zero-padded to whole 128 x 128 tiles in the
// workspace, so that no access needs a bound.  A and B are symmetric: tiles below the diagonal
// alone are computed and stored twice.  The loop is the projection GEMM's: slabs of 64 k copied
// straight into LDS, fragments read a step ahead.  In B X the second operand is X's own rows, k by
// columns, read with transposing reads, so that no transposed copy of X exists.  Of up to 128 rows B X
// takes both operands in two parts.
//
// Bound by feeding the matrix unit: a step's products reach 520 to 570 TFLOP/s for 48 of 768 x 768
// (A 45 us, B 46, B X 84) and 640 to 700 for 4 of 1536 x 6144 (98, 32 and 165 us), where the card's large
// matrix product reaches 1290.  What lies between are short sums (12 to 96 slabs of 64), the diagonal
// tiles' redundant halves, and epilogues that read and write X, A and B once a step.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "device_common.h"
#include "dflash.h"
#include "gemm_tile.h"
#include "training.h"

namespace dflash {
namespace {

constexpr int kTile = 128;
constexpr float kScale = 256.0f;  // of X in its fp16 parts

enum class Form { kGram, kPolynomial, kUpdate, kResult };  // kResult: the last kUpdate

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t lds_s4_t;

struct Matrices {
  _Float16* hi[2];  // [batch, rows, columns], the steps' in turn
  _Float16* lo;
  _Float16 *gram, *poly;  // [batch, rows, rows]
  _Float16* poly_lo;      // what B's rounding left off, where it is an operand
  int rows, columns;      // padded
  int batch;
};

// 16 bytes a lane from byte `off` + `scalar` of a buffer to LDS at `lds` + 16 * lane.
__device__ inline void copy_to_lds(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t scalar,
                                   uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(lds), "v"(off), "s"(r), "s"(scalar)
      : "memory");
}

// A buffer resource in scalar registers.
__device__ inline __amdgpu_buffer_rsrc_t scalar_resource(const void* base, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uintptr_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>(static_cast<uintptr_t>(hi) << 32 | lo), static_cast<short>(0),
      static_cast<int>(__builtin_amdgcn_readfirstlane(bytes)), 0x00020000);
}

template <int N>
__device__ inline void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Chunk (16 bytes) x of row r of a slab of rows of k, 128 columns each, lies at x ^ this: the four
// rows that 16 lanes of a transposing read touch lie in different banks.
__device__ inline int k_row_swizzle(int r) { return (r & 3) << 1; }

// ---- |G|_F and the first X ---------------------------------------------------------------

constexpr int kPartials = 256;  // partial sums of a matrix, at most

// Sums of squares in fp64: no overflow and no underflow whatever the elements.
template <typename T>
__global__ __launch_bounds__(256) void norm_kernel(const T* g, double* partial, int64_t elements,
                                                   int64_t block) {
  __shared__ double sums[4];
  const T* at = g + blockIdx.y * elements;
  const int64_t first = blockIdx.x * block, end = min(first + block, elements);
  double sum = 0;
#pragma unroll 8
  for (int64_t n = first + threadIdx.x; n < end; n += 256) {
    const float x = static_cast<float>(at[n]);
    sum += static_cast<double>(x) * x;
  }
  for (int step = 32; step; step /= 2) sum += __shfl_xor(sum, step);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    partial[blockIdx.y * gridDim.x + blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// A tile of 64 x 64 of X: rows and columns of X are those of G, or the other way round (`tall`).
template <typename T>
__global__ __launch_bounds__(256) void start_kernel(const T* g, const double* partial, int partials,
                                                    Matrices x, int m, int n, int tall, int whole,
                                                    float eps) {
  __shared__ float tile[64][65];
  const int b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  __shared__ double sums[4];
  static_assert(kPartials == 256, "one a thread");
  double square = threadIdx.x < partials ? partial[b * partials + threadIdx.x] : 0.0;
  for (int step = 32; step; step /= 2) square += __shfl_xor(square, step);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = square;
  __syncthreads();
  square = sums[0] + sums[1] + sums[2] + sums[3];
  // In two factors, the first a power of two: one alone would pass fp32's range for norms below 2^-120
  // and be subnormal for those above 2^134.
  const double factor = kScale / (sqrt(square) + static_cast<double>(eps));
  const float shift = factor > 0x1p+100 ? 0x1p+64f : factor < 0x1p-100 ? 0x1p-64f : 1.0f;
  const float rest = static_cast<float>(factor / static_cast<double>(shift));
  auto scaled = [=](float x) { return x * shift * rest; };
  // G's rows and columns of this tile.
  const int gr = tall ? c0 : r0, gc = tall ? r0 : c0;
  const T* from = g + static_cast<int64_t>(b) * m * n;
  const int64_t base = (static_cast<int64_t>(b) * x.rows + r0) * x.columns + c0;
  auto put = [&](int r, int c, const float (&v)[8]) {
    half8_t hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = static_cast<_Float16>(v[e]);
      lo[e] = static_cast<_Float16>(v[e] - static_cast<float>(hi[e]));
    }
    *reinterpret_cast<half8_t*>(x.hi[0] + base + static_cast<int64_t>(r) * x.columns + c) = hi;
    *reinterpret_cast<half8_t*>(x.lo + base + static_cast<int64_t>(r) * x.columns + c) = lo;
  };
  if (!tall) {
#pragma unroll
    for (int at = 0; at < 2; ++at) {
      const int r = (at * 256 + threadIdx.x) / 8, c = threadIdx.x % 8 * 8;
      const T* row = from + static_cast<int64_t>(gr + r) * n + gc + c;
      float v[8] = {};
      if (whole) {  // rows of whole 16-byte chunks, on 16-byte boundaries
        constexpr int N = Chunk<T>::N;
        if (gr + r < m && gc + c < n) {
#pragma unroll
          for (int e = 0; e < 8; e += N) {
            float part[N];
            load_floats<T, N>(row + e, part);
#pragma unroll
            for (int x = 0; x < N; ++x) v[e + x] = scaled(part[x]);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = gr + r < m && gc + c + e < n ? scaled(static_cast<float>(row[e])) : 0.0f;
      }
      put(r, c, v);
    }
    return;
  }
#pragma unroll
  for (int at = 0; at < 16; ++at) {
    const int r = at * 4 + threadIdx.x / 64, c = threadIdx.x % 64;
    tile[r][c] = gr + r < m && gc + c < n
                     ? scaled(static_cast<float>(from[static_cast<int64_t>(gr + r) * n + gc + c]))
                     : 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int at = 0; at < 2; ++at) {
    const int r = (at * 256 + threadIdx.x) % 64, c = (at * 256 + threadIdx.x) / 64 * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[c + e][r];
    put(r, c, v);
  }
}

// ---- the products ----------------------------------------------------------------------------

struct Step {
  Matrices x;
  int from;        // which of hi the step reads; it writes the other
  float a, b, c;
  int read_lo, write_lo;
  __bf16* out;     // [batch, m, n]: kResult writes it instead of X
  int m, n, tall;  // of G
};

// PARTS: B and X are operands of B X in two parts, as one product of three times the length,
// B_hi X_hi + B_hi X_lo + B_lo X_hi.  For X of one tile of rows: then a workgroup alone reads the low parts
// of its columns, and writes them when its wavefronts have read them.
template <Form FORM, typename CF, bool PARTS>
__global__ __launch_bounds__(CF::THREADS, CF::WGS) void product_kernel(Step p) {
  constexpr int BM = CF::BM, BN = CF::BN;
  constexpr int MB = CF::MB, NB = CF::NB, S = CF::STAGES;
  // Symmetric, with the second operand by rows of k-runs.
  constexpr bool kSquare = FORM == Form::kGram || FORM == Form::kPolynomial;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int wm = wave % CF::WAVES_M, wn = wave / CF::WAVES_M;

  // The tiles of a matrix lie on one XCD.
  static_assert(!kSquare || BM == BN, "tiles on both sides of the diagonal");
  const int tiles_m = p.x.rows / BM, tiles_n = (kSquare ? p.x.rows : p.x.columns) / BN;
  const int each = kSquare ? tiles_m * (tiles_m + 1) / 2 : tiles_m * tiles_n;
  const int at = xcd_logical_block(blockIdx.x, gridDim.x);
  const int batch = at / each;
  int mt, nt;
  if (kSquare) {  // the lower triangle, row by row
    int rest = at % each;
    for (mt = 0; rest > mt; ++mt) rest -= mt + 1;
    nt = rest;
  } else {
    mt = at % each % tiles_m;
    nt = at % each / tiles_m;
  }
  const int K = FORM == Form::kGram ? p.x.columns : p.x.rows;
  const int64_t square = static_cast<int64_t>(p.x.rows) * p.x.rows;
  const int64_t whole = static_cast<int64_t>(p.x.rows) * p.x.columns;
  const _Float16* hi = p.x.hi[p.from] + batch * whole;
  const _Float16* left = FORM == Form::kGram ? hi
                         : FORM == Form::kPolynomial ? p.x.gram + batch * square
                                                     : p.x.poly + batch * square;
  const _Float16* X = left + static_cast<int64_t>(mt) * BM * K;
  const _Float16* W = kSquare ? left + static_cast<int64_t>(nt) * BN * K : hi + nt * BN;
  constexpr bool kThree = PARTS && !kSquare;
  const _Float16* X_lo = kThree ? p.x.poly_lo + batch * square + static_cast<int64_t>(mt) * BM * K : X;
  const _Float16* W_lo = kThree ? p.x.lo + batch * whole + nt * BN : W;
  const uint32_t x_row = static_cast<uint32_t>(K) * 2;
  const uint32_t w_row_bytes = kSquare ? x_row : static_cast<uint32_t>(p.x.columns) * 2;
  const int slabs = K / kSlabK, KT = kThree ? 3 * slabs : slabs;

  constexpr int kChunks = BN / 8;  // of a row of k
  // Byte offsets of this lane's 16 bytes of each copy.
  uint32_t xoff[CF::A_LOADS], woff[CF::B_LOADS];
#pragma unroll
  for (int j = 0; j < CF::A_LOADS; ++j) {
    const int r = copy_row<CF>(j, wave, lane);
    xoff[j] = r * x_row + copy_chunk(r, lane) * 16;
  }
#pragma unroll
  for (int j = 0; j < CF::B_LOADS; ++j) {
    if (kSquare) {
      const int r = copy_row<CF>(j, wave, lane);
      woff[j] = w_row(r) * w_row_bytes + copy_chunk(r, lane) * 16;
    } else {  // rows of k, BN columns each
      const int r = ((j * CF::WAVES + wave) * 64 + lane) / kChunks;
      woff[j] = r * w_row_bytes + (lane % kChunks ^ k_row_swizzle(r)) * 16;
    }
  }
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem));
  // Past the last slab the copies fetch nothing (a size of 0), so that every slab has as many.
  auto copy = [&](int j, int kt, uint32_t stage) {
    const bool is_x = j < CF::A_LOADS;
    const int jj = is_x ? j : j - CF::A_LOADS;
    const uint32_t to = __builtin_amdgcn_readfirstlane(
        lds0 + stage * CF::SLAB + (is_x ? 0 : CF::A_BYTES) + (jj * CF::WAVES + wave) * 1024);
    const bool live = kt < KT;
    const int part = kThree ? kt >= 2 * slabs ? 2 : kt >= slabs ? 1 : 0 : 0;
    kt -= part * slabs;
    if (is_x || kSquare) {
      const auto memory = scalar_resource(is_x ? (part == 2 ? X_lo : X) : W,
                                          live ? (is_x ? BM : BN) * x_row : 0);
      copy_to_lds(memory, is_x ? xoff[is_x ? jj : 0] : woff[is_x ? 0 : jj],
                  __builtin_amdgcn_readfirstlane(live ? kt * kSlabK * 2 : 0), to);
    } else {  // a resource that begins at the slab's first row
      const auto memory =
          scalar_resource((part == 1 ? W_lo : W) +
                              static_cast<int64_t>(live ? kt : 0) * kSlabK * p.x.columns,
                          live ? (kSlabK - 1) * w_row_bytes + BN * 2 : 0);
      copy_to_lds(memory, woff[is_x ? 0 : jj], 0, to);
    }
  };

  using F = half8_t;
  const int swz = slab_swizzle(c);
  const int chunk[2] = {(g ^ swz) * 16, ((4 + g) ^ swz) * 16};
  const int xrow = (wm * CF::WM + c) * (kSlabK * 2);
  const int wrow = CF::A_BYTES + (wn * CF::WN + c) * (kSlabK * 2);
  auto x_frag = [&](uint32_t base, int u, int i) {
    return *static_cast<const F*>(
        __builtin_assume_aligned(smem + base + xrow + chunk[u] + i * 16 * kSlabK * 2, 16));
  };
  auto w_frag = [&](uint32_t base, int u, int i) {
    if constexpr (kSquare) {
      return *static_cast<const F*>(
          __builtin_assume_aligned(smem + base + wrow + chunk[u] + i * 16 * kSlabK * 2, 16));
    } else {
      // Columns wn WN + 16 i + c of rows 32 u + 8g + 0..3 and + 4..7.
      const int r = 32 * u + 8 * g + (c >> 2);
      const int x = ((wn * CF::WN + 16 * i) / 8 + ((c & 3) >> 1)) ^ k_row_swizzle(r);
      const unsigned char* p0 = smem + base + CF::A_BYTES + r * (BN * 2) + x * 16 + (c & 1) * 8;
      const u32x2_t lo = __builtin_bit_cast(
          u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)p0));
      const u32x2_t up = __builtin_bit_cast(
          u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(p0 + 4 * BN * 2)));
      return __builtin_bit_cast(F, u32x4_t{lo[0], lo[1], up[0], up[1]});
    }
  };

  // X of this tile, for a X: read with the first slabs, a thread's rows and chunks of eight
  // columns as it will write them.
  constexpr int kRows = BM * BN / 8 / CF::THREADS;  // chunks a thread
  _Float16* lo = p.x.lo + batch * whole;
  half8_t h[kSquare ? 1 : kRows], l[kSquare ? 1 : kRows];
  auto place = [&](int n) {  // row and column of a thread's n-th chunk
    const int at2 = n * CF::THREADS + threadIdx.x;
    return int2{at2 / (BN / 8), at2 % (BN / 8) * 8};
  };
  auto address = [&](int2 rc) {
    return static_cast<int64_t>(mt * BM + rc.x) * p.x.columns + nt * BN + rc.y;
  };
  if constexpr (!kSquare) {
#pragma unroll
    for (int n = 0; n < kRows; ++n) {
      const int64_t to = address(place(n));
      h[n] = *reinterpret_cast<const half8_t*>(hi + to);
      l[n] = half8_t{};
      if (p.read_lo) l[n] = *reinterpret_cast<const half8_t*>(lo + to);
    }
    asm volatile("" ::: "memory");
  }

  f32x4_t acc[NB][MB] = {};
  F xf[2][MB], wf[2][NB];
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int j = 0; j < CF::LOADS; ++j) copy(j, s, s);
  wait_copies<(S - 1) * CF::LOADS>();
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int i = 0; i < NB; ++i) wf[0][i] = w_frag(0, 0, i);
#pragma unroll
  for (int i = 0; i < MB; ++i) xf[0][i] = x_frag(0, 0, i);

  constexpr int kMfmas = MB * NB, kReads = MB + NB;
  auto step = [&](auto parity, auto with_copies, uint32_t base, int kt, uint32_t stage) {
    constexpr int P = decltype(parity)::value;
    constexpr bool COPY = decltype(with_copies)::value;
#pragma unroll
    for (int q = 0; q < kMfmas; ++q) {
      __builtin_amdgcn_sched_barrier(0);
      acc[q % NB][q / NB] =
          Mma<_Float16>::run(wf[P][q % NB], xf[P][q / NB], acc[q % NB][q / NB]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int z = 0; z < kReads; ++z)
        if (z * kMfmas * 3 / 4 / kReads == q) {
          if (z < NB)
            wf[P ^ 1][z] = w_frag(base, P ^ 1, z);
          else
            xf[P ^ 1][z - NB] = x_frag(base, P ^ 1, z - NB);
        }
      if constexpr (COPY) {
#pragma unroll
        for (int z = 0; z < CF::LOADS; ++z)
          if (z * kMfmas * 3 / 4 / CF::LOADS == q) copy(z, kt, stage);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  uint32_t stage = 0;
  for (int kt = 0; kt < KT; ++kt) {
    const uint32_t next = stage + 1 == S ? 0 : stage + 1;
    step(std::integral_constant<int, 0>{}, std::false_type{}, stage * CF::SLAB, 0, 0);
    wait_copies<(S - 2) * CF::LOADS>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    step(std::integral_constant<int, 1>{}, std::true_type{}, next * CF::SLAB, kt + S, stage);
    stage = next;
  }
  // No copy may land in LDS any more (and the compiler knows that no load is left).
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  asm volatile("" ::: "memory");

  if constexpr (kSquare) {
    // Eight consecutive elements of a row a lane and pair of blocks.
    _Float16* out = (FORM == Form::kGram ? p.x.gram : p.x.poly) + batch * square;
    const _Float16* gram = p.x.gram + batch * square;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // The mirrored tile, [column][row], rows of 128 + 8.
    _Float16* mirror = reinterpret_cast<_Float16*>(smem);
    constexpr bool kRest = PARTS && FORM == Form::kPolynomial;
    constexpr int kLd = BM + 8;
    static_assert(BN * kLd * 2 <= CF::LDS, "the mirrored tile");
    _Float16* out_lo = kRest ? p.x.poly_lo + batch * square : nullptr;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int row = wm * CF::WM + 16 * j + c;
#pragma unroll
      for (int i = 0; i < NB; i += 2) {
        const int column = wn * CF::WN + 16 * i + 8 * g;
        const int64_t to = static_cast<int64_t>(mt * BM + row) * p.x.rows + nt * BN + column;
        half8_t v, rest;
        if constexpr (FORM == Form::kGram) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[e] = static_cast<_Float16>(acc[i + e / 4][j][e % 4] * (1.0f / (kScale * kScale)));
        } else {
          const half8_t a = *reinterpret_cast<const half8_t*>(gram + to);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = p.b * static_cast<float>(a[e]) + p.c * acc[i + e / 4][j][e % 4];
            v[e] = static_cast<_Float16>(x);
            rest[e] = static_cast<_Float16>(x - static_cast<float>(v[e]));
          }
        }
        *reinterpret_cast<half8_t*>(out + to) = v;
        if constexpr (kRest) *reinterpret_cast<half8_t*>(out_lo + to) = rest;
        if (mt != nt) {
#pragma unroll
          for (int e = 0; e < 8; ++e) mirror[(column + e) * kLd + row] = v[e];
        }
      }
    }
    if (mt != nt) {
      __syncthreads();
      for (int n = threadIdx.x; n < BN * BM / 8; n += CF::THREADS) {
        const int r = n / (BM / 8), k = n % (BM / 8) * 8;
        *reinterpret_cast<u32x4_t*>(out + static_cast<int64_t>(nt * BN + r) * p.x.rows +
                                    mt * BM + k) =
            *reinterpret_cast<const u32x4_t*>(mirror + r * kLd + k);
      }
    }
  } else {
    // Through LDS, so that rows are read and written 256 bytes at a time (straight from the
    // accumulators, 8 bytes a lane in 16 rows, X's accesses took 69 of 114 us of a step of 48 of
    // 768 x 768).  Chunk (four columns) x of row r lies at x ^ (r % 8).
    static_assert(BM * BN * 4 <= CF::LDS, "the tile");
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    f32x4_t* tile = reinterpret_cast<f32x4_t*>(smem);
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int r = wm * CF::WM + 16 * j + c, x = (wn * CF::WN + 16 * i) / 4 + g;
        tile[r * (BN / 4) + (x ^ (r & 7))] = acc[i][j];
      }
    __syncthreads();
    _Float16* next = p.x.hi[p.from ^ 1] + batch * whole;
    __bf16* out = p.out + static_cast<int64_t>(batch) * p.m * p.n;
    const int rows = p.tall ? p.n : p.m, columns = p.tall ? p.m : p.n;
#pragma unroll
    for (int n = 0; n < kRows; ++n) {
      const int2 rc = place(n);
      float v[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const f32x4_t sum = tile[rc.x * (BN / 4) + ((rc.y / 4 + half) ^ (rc.x & 7))];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at2 = 4 * half + e;
          v[at2] = p.a * (static_cast<float>(h[n][at2]) + static_cast<float>(l[n][at2])) + sum[e];
        }
      }
      if constexpr (FORM == Form::kUpdate) {
        half8_t nh, nl;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          nh[e] = static_cast<_Float16>(v[e]);
          nl[e] = static_cast<_Float16>(v[e] - static_cast<float>(nh[e]));
        }
        *reinterpret_cast<half8_t*>(next + address(rc)) = nh;
        if (p.write_lo) *reinterpret_cast<half8_t*>(lo + address(rc)) = nl;
      } else {
        const int row = mt * BM + rc.x, column = nt * BN + rc.y;
        if (row >= rows || column >= columns) continue;
        bf16x8_t y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = static_cast<__bf16>(v[e] * (1.0f / kScale));
        if (!p.tall && columns % 8 == 0) {
          *reinterpret_cast<bf16x8_t*>(out + static_cast<int64_t>(row) * p.n + column) = y;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (column + e < columns)
              out[p.tall ? static_cast<int64_t>(column + e) * p.n + row
                         : static_cast<int64_t>(row) * p.n + column + e] = y[e];
        }
      }
    }
  }
}

// ---- host --------------------------------------------------------------------------------------

struct Plan {
  int rows, columns, partials;
  int64_t block;  // elements of a partial sum
  // B X of operands in two parts, for one tile of rows.  The fewer rows, the more of the result is what
  // their roundings make: it was off by 1.35 times its own rounding with 256 rows, 1.42 with 128, 1.52
  // with 64, 1.79 with 8; in parts by 1.14, 1.17 and 1.37.  They cost 3 us a step of 128 x 128 (98 us
  // instead of 83 for five); two tiles of rows would take 139 us instead of 111 (150 x 140).
  bool parts;
  size_t x, square, norm, total;
};

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

Plan make_plan(int64_t batch, int64_t m, int64_t n) {
  Plan p;
  const int64_t small = m < n ? m : n, large = m < n ? n : m;
  const int64_t tile = kTile;
  p.rows = static_cast<int>((small + tile - 1) / tile * tile);
  p.columns = static_cast<int>((large + tile - 1) / tile * tile);
  p.block = (m * n + kPartials - 1) / kPartials;
  if (p.block < 8192) p.block = 8192;
  p.partials = static_cast<int>((m * n + p.block - 1) / p.block);
  p.x = round_up(static_cast<size_t>(batch) * p.rows * p.columns * 2);
  p.square = round_up(static_cast<size_t>(batch) * p.rows * p.rows * 2);
  p.norm = round_up(static_cast<size_t>(batch) * p.partials * 8);
  p.parts = p.rows == kTile;
  p.total = 3 * p.x + (p.parts ? 3 : 2) * p.square + p.norm;
  return p;
}

int refuse(int64_t batch, int64_t m, int64_t n) {
  if (batch < 0 || m < 1 || n < 1) return DFLASH_ERR_SHAPE;
  // Grids, and a tile's rows within 31-bit byte offsets.
  if (m > (1 << 20) || n > (1 << 20) || batch > 65535) return DFLASH_ERR_TOO_LARGE;
  const int64_t small = m < n ? m : n, large = m < n ? n : m;
  const int64_t rows = (small + kTile - 1) / kTile, columns = (large + kTile - 1) / kTile;
  if (rows > 32767 || batch * rows * columns > (1 << 22)) return DFLASH_ERR_TOO_LARGE;
  return DFLASH_OK;
}

template <Form FORM, typename CF, bool PARTS>
int launch_config(const Step& p, hipStream_t stream) {
  const uint32_t m = p.x.rows / CF::BM, n = p.x.columns / CF::BN;
  const uint32_t tiles = FORM == Form::kGram || FORM == Form::kPolynomial ? m * (m + 1) / 2 : m * n;
  const hipError_t e = ensure_dynamic_lds<&product_kernel<FORM, CF, PARTS>>(CF::LDS);
  if (e != hipSuccess) return static_cast<int>(e);
  hipLaunchKernelGGL((product_kernel<FORM, CF, PARTS>), dim3(p.x.batch * tiles), dim3(CF::THREADS),
                     CF::LDS, stream, p);
  return static_cast<int>(hipGetLastError());
}

// Up to one tile a CU: eight wavefronts and five slabs in flight; more: two workgroups of four a CU,
// two slabs.  us a step, deep / two: Gram of 6144 x 1536 (78 tiles) 44 / 67, of four (312) 105 / 96,
// of 48 of 768 x 768 (1008) 51 / 42; update of 256 x 256 (4) 7.5 / 9.
template <Form FORM, bool PARTS>
int launch_product(const Step& p, hipStream_t stream) {
  constexpr bool kSquare = FORM == Form::kGram || FORM == Form::kPolynomial;
  const int m = p.x.rows / kTile, n = p.x.columns / kTile;
  const int64_t tiles = static_cast<int64_t>(p.x.batch) * (kSquare ? m * (m + 1) / 2 : m * n);
  return tiles <= 256 ? launch_config<FORM, Cfg128x128Deep, PARTS>(p, stream)
                      : launch_config<FORM, Cfg128x128, PARTS>(p, stream);
}

// A step from X of `from` to that of `from` ^ 1, or to the result.
template <bool PARTS>
int launch_step(const Step& p, bool last, hipStream_t stream) {
  int rc = launch_product<Form::kGram, false>(p, stream);
  if (rc == DFLASH_OK) rc = launch_product<Form::kPolynomial, PARTS>(p, stream);
  if (rc != DFLASH_OK) return rc;
  return last ? launch_product<Form::kResult, PARTS>(p, stream)
              : launch_product<Form::kUpdate, PARTS>(p, stream);
}

template <typename T>
int launch(const T* g, __bf16* out, int64_t batch, int m, int n, int steps, float a, float b,
           float c, float eps, char* workspace, hipStream_t stream) {
  const Plan plan = make_plan(batch, m, n);
  Step p{};
  p.x.hi[0] = reinterpret_cast<_Float16*>(workspace);
  p.x.hi[1] = reinterpret_cast<_Float16*>(workspace + plan.x);
  p.x.lo = reinterpret_cast<_Float16*>(workspace + 2 * plan.x);
  char* squares = workspace + 3 * plan.x;
  p.x.gram = reinterpret_cast<_Float16*>(squares);
  p.x.poly = reinterpret_cast<_Float16*>(squares + plan.square);
  p.x.poly_lo = plan.parts ? reinterpret_cast<_Float16*>(squares + 2 * plan.square) : nullptr;
  double* partial = reinterpret_cast<double*>(workspace + plan.total - plan.norm);
  p.x.rows = plan.rows;
  p.x.columns = plan.columns;
  p.x.batch = static_cast<int>(batch);
  p.a = a;
  p.b = b;
  p.c = c;
  p.out = out;
  p.m = m;
  p.n = n;
  p.tall = m > n;
  const uint32_t count = static_cast<uint32_t>(batch);
  hipLaunchKernelGGL((norm_kernel<T>), dim3(plan.partials, count), dim3(256), 0, stream, g, partial,
                     static_cast<int64_t>(m) * n, plan.block);
  hipLaunchKernelGGL((start_kernel<T>), dim3(plan.columns / 64, plan.rows / 64, count), dim3(256), 0,
                     stream, g, partial, plan.partials, p.x, m, n, p.tall,
                     n % 8 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0, eps);
  for (int step = 0; step < steps; ++step) {
    p.from = step % 2;
    const bool last = step + 1 == steps;
    // (The last step's X has hi alone, but in parts.)
    p.read_lo = step == 0 || !last || plan.parts;
    p.write_lo = step + 2 < steps || plan.parts;
    const int rc = plan.parts ? launch_step<true>(p, last, stream)
                              : launch_step<false>(p, last, stream);
    if (rc != DFLASH_OK) return rc;
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" {

size_t dflash_orthogonalize_workspace_bytes(int64_t batch, int64_t m, int64_t n) {
  if (batch < 1 || refuse(batch, m, n) != DFLASH_OK) return 0;
  return make_plan(batch, m, n).total;
}

int dflash_orthogonalize(const void* update, void* out, int64_t batch, int64_t m, int64_t n,
                         int steps, float a, float b, float c, float eps, int dtype,
                         void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = refuse(batch, m, n);
  if (rc != DFLASH_OK) return rc;
  if (steps < 1 || !(eps >= 0.0f)) return DFLASH_ERR_SHAPE;
  if (dtype < DFLASH_DTYPE_FP16 || dtype > DFLASH_DTYPE_FP32) return DFLASH_ERR_DTYPE;
  if (batch == 0) return DFLASH_OK;
  if (!update || !out || !workspace) return DFLASH_ERR_NULL;
  const uintptr_t element = dtype == DFLASH_DTYPE_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(update) % element != 0 ||
      (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 != 0)
    return DFLASH_ERR_ALIGN;
  if (workspace_bytes < make_plan(batch, m, n).total) return DFLASH_ERR_WORKSPACE;
  auto call = [&](auto t) {
    using T = decltype(t);
    return launch(static_cast<const T*>(update), static_cast<__bf16*>(out), batch,
                  static_cast<int>(m), static_cast<int>(n), steps, a, b, c, eps,
                  static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
  };
  if (dtype == DFLASH_DTYPE_FP16) return call(_Float16{});
  if (dtype == DFLASH_DTYPE_BF16) return call(__bf16{});
  return call(float{});
}

}  // extern "C"
