// Output projection of the joiner for 8-bit operands with a float32 scale per block of
// 128 (gfx950 MFMA): the serving and scoring form of the projection in ot_project.hip.
//
//   logits[r, v] = bias[v] + sum_b xs[r, b] * ws[v / 128, b] * sum_{k in b} x[r, k] * w[v, k]
//   den[r]       = log sum_v exp(logits[r, v])      (of the float32 logits)
//
// x (rows, D) and w (V, D) are e4m3.  They are read as 8 bits and widened to bfloat16, which
// holds every e4m3 value, in front of the 16-bit matrix instructions: the 8-bit ones of this
// chip align the products of a sum to the largest and drop what lies more than about 2^-13
// below it (measured: 9e-6 of the result at K = 128 for normal weights against tanh
// activations, 2e-4 in the worst sums, where the 16-bit ones stay at 1e-8), which is not a
// float32 sum.  The inner sum of a block enters the running sum times the product of the two
// scales, one fused multiply-add per value.  As in ot_project.hip the product is formed
// transposed (vocabulary along the rows of an accumulator tile), so that a lane holds
// consecutive logits of ONE packed row: one activation scale per lane, one weight scale per
// wave, and the row's running (max, sum) without cross-lane traffic.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ot_device.hip.h"
#include "ot_transducer.h"

namespace ot {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kBlocksK = 128;      // elements per scale
constexpr int kBlocksUnit = 16;    // D is a multiple of this: one 16-byte load
constexpr int kSmallCols = 64;     // vocabulary entries of a workgroup of the small kernel
constexpr int kWideCols = 32;      // vocabulary entries of a stage of the wide kernel
constexpr int kPartCols = 16;      // least vocabulary entries behind one partial log-sum-exp

// a running log-sum-exp as (largest value, sum of exp(value - largest))
struct LogSum {
  float m, s;
};
__device__ __forceinline__ LogSum merge(LogSum a, LogSum b) {
  const float m = fmaxf(a.m, b.m);
  const float ref = __builtin_isinf(m) ? 0.f : m;
  const float ra = __builtin_isinf(a.m) ? 0.f : a.m, rb = __builtin_isinf(b.m) ? 0.f : b.m;
  return {m, (a.s == 0.f ? 0.f : a.s * expf(ra - ref)) + (b.s == 0.f ? 0.f : b.s * expf(rb - ref))};
}

template <class E>
__device__ __forceinline__ void store_logit(void *logits, int64_t i, float v) {
  static_cast<unsigned short *>(logits)[i] = from_float<E>(v);
}
template <>
__device__ __forceinline__ void store_logit<float>(void *logits, int64_t i, float v) {
  static_cast<float *>(logits)[i] = v;
}

// 8 consecutive e4m3 elements widened
__device__ __forceinline__ bf16x8 widen(int lo, int hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  const bf16x4 l = __builtin_shufflevector(a, b, 0, 1, 2, 3), h = __builtin_shufflevector(c, d, 0, 1, 2, 3);
  return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7);
}

// the block product of 16 vocabulary entries x 16 packed rows, K = 128, unscaled; which k an
// element stands for is the same in both operands
__device__ __forceinline__ f32x4 mfma_16x16x128(i32x8 w, i32x8 x) {
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[2 * i], w[2 * i + 1]), widen(x[2 * i], x[2 * i + 1]), c,
                                                0, 0, 0);
  return c;
}

// 32 consecutive elements of a row, k0 onwards; those at or past D are 0 (D and k0 are
// multiples of 16)
__device__ __forceinline__ i32x8 load_k32(const unsigned char *row, int k0, int D) {
  i32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
  if (k0 < D) a = *reinterpret_cast<const i32x4 *>(row + k0);
  if (k0 + kBlocksUnit < D) b = *reinterpret_cast<const i32x4 *>(row + k0 + kBlocksUnit);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A workgroup of 4 waves forms 16 packed rows x 64 vocabulary entries, a wave one
// accumulator tile of 16 x 16 straight from memory.  Lane l holds elements
// [32 * (l / 16), + 32) of a block of row l % 16 of either operand.
template <class T>
__global__ __launch_bounds__(kBlock) void project_blocks_small_kernel(
    const unsigned char *__restrict__ x, const float *__restrict__ xs, const unsigned char *__restrict__ w,
    const float *__restrict__ ws, const float *__restrict__ bias, int64_t rows, int D, int V, int col_tiles,
    int64_t tiles, void *__restrict__ logits, LogSum *__restrict__ parts) {
  __shared__ LogSum s_part[kWavesPerBlock][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, h = lane >> 4;
  const int nblocks = (D + kBlocksK - 1) / kBlocksK;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row0 = tile / col_tiles * 16;
    const int part = (int)(tile % col_tiles);
    const int v0 = part * kSmallCols + wave * 16;
    const int64_t row = row0 + r;
    const bool row_in = row < rows;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (v0 < V) {
      // rows and entries past the end read the last one's data; their results are not stored
      const unsigned char *xr = x + min(row, rows - 1) * D;
      const unsigned char *wr = w + (int64_t)min(v0 + r, V - 1) * D;
      const float *xsr = xs + min(row, rows - 1) * nblocks;
      const float *wsr = ws + (int64_t)(v0 / kBlocksK) * nblocks;
      for (int b = 0; b < nblocks; ++b) {
        const int k0 = b * kBlocksK + 32 * h;
        const f32x4 p = mfma_16x16x128(load_k32(wr, k0, D), load_k32(xr, k0, D));
        const float s = xsr[b] * wsr[b];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(p[i], s, acc[i]);
      }
    }
    // register i: vocabulary entry v0 + 4 h + i of row r
    LogSum run = {OT_NEG_INF, 0.f};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int v = v0 + 4 * h + i;
      y[i] = v < V ? acc[i] + (bias ? bias[v] : 0.f) : OT_NEG_INF;
      if (v < V && row_in) store_logit<T>(logits, row * V + v, y[i]);
      run.m = fmaxf(run.m, y[i]);
    }
    if (parts) {
      const float ref = __builtin_isinf(run.m) ? 0.f : run.m;
#pragma unroll
      for (int i = 0; i < 4; ++i) run.s += expf(y[i] - ref);
#pragma unroll
      for (int d = 16; d < 64; d *= 2)
        run = merge(run, {__shfl_xor(run.m, d, kWave), __shfl_xor(run.s, d, kWave)});
      __syncthreads();  // the previous tile's parts have been read
      if (h == 0) s_part[wave][r] = run;
      __syncthreads();
      if (threadIdx.x < 16 && row0 + threadIdx.x < rows) {
        LogSum t = s_part[0][threadIdx.x];
        for (int k = 1; k < kWavesPerBlock; ++k) t = merge(t, s_part[k][threadIdx.x]);
        parts[part * rows + row0 + threadIdx.x] = t;
      }
    }
  }
}

// 4 consecutive logits of a row; the row may start anywhere its type can
template <class T>
__device__ __forceinline__ void store_logits4(void *logits, int64_t i, const float y[4]) {
  if constexpr (sizeof(T) == 4) {
    typedef f32x4 unaligned __attribute__((aligned(4)));
    const f32x4 t = {y[0], y[1], y[2], y[3]};
    *reinterpret_cast<unaligned *>(static_cast<float *>(logits) + i) = t;
  } else {
    typedef u32x2 unaligned __attribute__((aligned(2)));
    const u32x2 t = {(unsigned)from_float<T>(y[0]) | ((unsigned)from_float<T>(y[1]) << 16),
                     (unsigned)from_float<T>(y[2]) | ((unsigned)from_float<T>(y[3]) << 16)};
    *reinterpret_cast<unaligned *>(static_cast<unsigned short *>(logits) + i) = t;
  }
}

// Many rows.  A workgroup of 4 waves owns 64 * TILES packed rows; a wave holds its 16 * TILES
// rows of x, widened, in registers for the whole walk over the vocabulary, so x is read and
// widened once.  The weight goes by in stages of COLS vocabulary entries (8-bit, all of D)
// through two LDS buffers: the next stage's global loads are in flight while a stage is
// multiplied, and are written to the other buffer behind it.  16-byte slots of LDS are
// XOR-swizzled by their row against bank conflicts.
//   KB: blocks of 128 in D that registers are laid out for (D may have fewer)
// Lane l holds bytes [64 q + 16 (l / 16), + 16) of a block of row l % 16 (q = 0, 1); the first 8
// feed matrix instruction 2 q and the others 2 q + 1, in both operands alike.
template <class T, int KB, int TILES, int COLS, int WAVES_PER_SIMD>
__global__ __launch_bounds__(kBlock, WAVES_PER_SIMD) void project_blocks_kernel(
    const unsigned char *__restrict__ x, const float *__restrict__ xs, const unsigned char *__restrict__ w,
    const float *__restrict__ ws, const float *__restrict__ bias, int64_t rows, int D, int V,
    int stages_per_part, void *__restrict__ logits, float *__restrict__ den, LogSum *__restrict__ parts) {
  constexpr int kRowBytes = KB * kBlocksK, kSlots = kRowBytes / 16;
  constexpr int kPieces = COLS * kSlots / kBlock;  // 16-byte pieces of a stage per thread
  static_assert(kPieces * kBlock == COLS * kSlots && COLS % 16 == 0 && kBlocksK % COLS == 0, "");
  __shared__ __attribute__((aligned(16))) unsigned char s_w[2][COLS * kRowBytes];
  __shared__ __attribute__((aligned(16))) float s_bias[2][COLS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = lane & 15, h = lane >> 4;
  const int nblocks = (D + kBlocksK - 1) / kBlocksK;
  const int stages = (V + COLS - 1) / COLS;
  const int part = blockIdx.y;
  const int stage0 = part * stages_per_part, stage1 = min(stages, stage0 + stages_per_part);

  // this thread's pieces of a stage: row, slot and place in LDS
  i32x4 piece[kPieces];
  float piece_bias;
  auto load_stage = [&](int stage) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int p = tid + i * kBlock, row = p / kSlots, slot = p % kSlots;
      const int v = min(stage * COLS + row, V - 1);  // entries past the end are masked later
      piece[i] = i32x4{0, 0, 0, 0};
      if (slot * 16 < D) piece[i] = *reinterpret_cast<const i32x4 *>(w + (int64_t)v * D + slot * 16);
    }
    if (tid < COLS) {
      const int v = stage * COLS + tid;
      piece_bias = v < V ? (bias ? bias[v] : 0.f) : OT_NEG_INF;
    }
  };
  auto store_stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int p = tid + i * kBlock, row = p / kSlots, slot = p % kSlots;
      *reinterpret_cast<i32x4 *>(&s_w[buf][row * kRowBytes + ((slot ^ (row & 7)) * 16)]) = piece[i];
    }
    if (tid < COLS) s_bias[buf][tid] = piece_bias;
  };

  load_stage(stage0);
  // x: 16 * TILES rows per wave
  const int64_t row0 = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * (64 * TILES) + wave * (16 * TILES);
  bf16x8 xf[TILES][KB][4];
  float xscale[TILES][KB];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int64_t row = min(row0 + 16 * t + r, rows - 1);
    const unsigned char *xr = x + row * D;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      xscale[t][b] = b < nblocks ? xs[row * nblocks + b] : 0.f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = b * kBlocksK + 64 * q + 16 * h;
        i32x4 c = {0, 0, 0, 0};
        if (k < D) c = *reinterpret_cast<const i32x4 *>(xr + k);
        xf[t][b][2 * q] = widen(c[0], c[1]);
        xf[t][b][2 * q + 1] = widen(c[2], c[3]);
      }
    }
  }
  store_stage(0);

  // running log-sum-exp of this lane's share of its rows, relative to ref: ref follows the
  // largest value so far at a distance of at most 20, so that few values make it move
  float ref[TILES], sum[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    ref[t] = OT_NEG_INF;
    sum[t] = 0.f;
  }
  const bool want_den = den || parts;

  for (int stage = stage0; stage < stage1; ++stage) {
    const int buf = (stage - stage0) & 1;
    lds_barrier();  // LDS only: the logits' stores stay in flight
    if (stage + 1 < stage1) load_stage(stage + 1);
    // the stage lies in one block of 128 vocabulary entries
    const float *wsr = ws + (int64_t)(stage * COLS / kBlocksK) * nblocks;
    float scale[TILES][KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const float sw = b < nblocks ? wsr[b] : 0.f;
#pragma unroll
      for (int t = 0; t < TILES; ++t) scale[t][b] = xscale[t][b] * sw;
    }
#pragma unroll 1
    for (int c = 0; c < COLS / 16; ++c) {
      const int v0 = stage * COLS + 16 * c;
      if (v0 >= V) break;
      const f32x4 b4 = *reinterpret_cast<const f32x4 *>(&s_bias[buf][16 * c + 4 * h]);
      f32x4 acc[TILES];
#pragma unroll
      for (int t = 0; t < TILES; ++t) acc[t] = b4;
      const unsigned char *wr = &s_w[buf][(16 * c + r) * kRowBytes];
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        if (KB > 4 && b >= nblocks) continue;
        f32x4 p[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) p[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const i32x4 d = *reinterpret_cast<const i32x4 *>(wr + (((b * 8 + 4 * q + h) ^ (r & 7)) * 16));
          const bf16x8 w0 = widen(d[0], d[1]), w1 = widen(d[2], d[3]);
#pragma unroll
          for (int t = 0; t < TILES; ++t)
            p[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w0, xf[t][b][2 * q], p[t], 0, 0, 0);
#pragma unroll
          for (int t = 0; t < TILES; ++t)
            p[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w1, xf[t][b][2 * q + 1], p[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] = __builtin_fmaf(p[t][i], scale[t][b], acc[t][i]);
      }
      // register i: vocabulary entry v0 + 4 h + i of row 16 t + r
      const int v = v0 + 4 * h;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = v0 + 16 <= V || v + i < V ? acc[t][i] : OT_NEG_INF;
        const int64_t row = row0 + 16 * t + r;
        if (row < rows) {
          if (v + 4 <= V) {
            store_logits4<T>(logits, row * V + v, y);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (v + i < V) store_logit<T>(logits, row * V + v + i, y[i]);
          }
        }
        if (want_den) {
          constexpr float kLog2e = 1.44269502162933349609375f;
          const float top = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
          if (top > ref[t] + 20.f) {
            if (sum[t] != 0.f) sum[t] *= expf(ref[t] - top);
            ref[t] = top;
          }
          const float shift = __builtin_isinf(ref[t]) ? 0.f : -ref[t];
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[t] += __builtin_amdgcn_exp2f((y[i] + shift) * kLog2e);
        }
      }
    }
    if (stage + 1 < stage1) store_stage(buf ^ 1);
  }
  if (!want_den) return;
  // the four lanes of a row meet
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    LogSum run = {ref[t], sum[t]};
#pragma unroll
    for (int d = 16; d < 64; d *= 2)
      run = merge(run, {__shfl_xor(run.m, d, kWave), __shfl_xor(run.s, d, kWave)});
    const int64_t row = row0 + 16 * t + r;
    if (h == 0 && row < rows) {
      if (parts) parts[(int64_t)part * rows + row] = run;
      else den[row] = logf(run.s) + (__builtin_isinf(run.m) ? 0.f : run.m);
    }
  }
}

// Many rows of up to KB blocks.  A workgroup of 4 waves owns 64 * TILES packed rows; a wave holds
// its 16 * TILES rows of x, widened, in registers for the whole walk over the vocabulary, so x is
// read and widened once.  The weight goes by in stages of 32 vocabulary entries (all of D, 8-bit)
// through two LDS buffers: the next stage's global loads are issued at the start of a stage and
// written in its last part, with one barrier per stage.  16-byte slots of LDS are XOR-swizzled by
// their row against bank conflicts.
//
// The walk advances in steps of 16 vocabulary entries x one block (4 * TILES matrix instructions);
// the LDS read of a step's weight is issued one step ahead.  Nothing in a step branches: rows past
// the end are dropped by the bounds of the store's buffer view, entries past the end have weight 0
// and a starting value of -inf.
//
// Which entry of the vocabulary a row of the accumulator tile stands for is free: it is chosen so
// that a lane ends up with 16 bytes of consecutive logits and four lanes with 64, from one group of
// 16 entries for 4-byte logits and from two for 2-byte ones.
//   ALIGNED: 4 logits start at a multiple of 4 bytes (else 2-byte logits are stored one by one)
// Lane l holds bytes [64 q + 16 (l / 16), + 16) of a block of row l % 16 (q = 0, 1); the first 8
// feed matrix instruction 2 q and the others 2 q + 1, in both operands alike.
template <class T, int KB, int TILES, int WAVES_PER_SIMD, bool ALIGNED, bool DEN>
__global__ __launch_bounds__(kBlock, WAVES_PER_SIMD) void project_blocks_wide_kernel(
    const unsigned char *__restrict__ x, const float *__restrict__ xs, const unsigned char *__restrict__ w,
    const float *__restrict__ ws, const float *__restrict__ bias, int64_t rows, int D, int V,
    int stages_per_part, void *__restrict__ logits, float *__restrict__ den, LogSum *__restrict__ parts) {
  constexpr int kCols = kWideCols;
  constexpr int kSlots = KB * 8;                    // 16-byte slots of a row
  constexpr int kPieces = kCols * kSlots / kBlock;  // of a stage per thread
  constexpr int kLdsSlots = kCols * kSlots + 8 * (kCols / 8);  // of a stage, padded (see place())
  constexpr unsigned kOut = sizeof(T) == 4 ? 4u : 2u;
  constexpr int kGroup = 16 / (int)kOut;            // consecutive entries of a lane
  constexpr int kSubs = kGroup / 4;                 // groups of 16 entries behind them
  constexpr unsigned kNowhere = 0xffffffe0u;        // an offset that a store drops
  static_assert(kPieces * kBlock == kCols * kSlots, "");
  __shared__ __attribute__((aligned(16))) i32x4 s_w[2][kLdsSlots];
  __shared__ __attribute__((aligned(16))) float s_bias[2][kCols];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = lane & 15, h = lane >> 4;
  const int nblocks = (D + kBlocksK - 1) / kBlocksK;
  const int stages = (V + kCols - 1) / kCols;
  const int part = blockIdx.y;
  const int stage0 = part * stages_per_part, stage1 = min(stages, stage0 + stages_per_part);

  // Place of a 16-byte slot of a stage's row in LDS.  A 16-byte read is served 16 lanes at a time:
  // lanes 0-7 and 24-31 of a half-wave, or 8-23, that is r < 8 of one h and r >= 8 of the other.
  // Three bits of the row that lane r reads (r & 7) spread 8 lanes over 128 bytes; the other 8 are
  // half of the 256 bytes that the banks hold away, by a pad of 128 bytes every 8 rows of r.
  auto place = [&](int row, int slot) -> int {
    const int lane8 = kSubs == 1 ? row & 7 : (row & 3) | ((row >> 1) & 4);
    const int half = kSubs == 1 ? row >> 3 : row >> 4;
    return row * kSlots + (KB % 2 == 0 ? 8 * half : 0) + (slot ^ lane8);
  };
  i32x4 piece[kPieces];
  float piece_bias = 0.f;
  auto load_stage = [&](int stage) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int p = tid + i * kBlock, row = p / kSlots, slot = p % kSlots;
      const int v = stage * kCols + row;
      piece[i] = i32x4{0, 0, 0, 0};
      if (slot * 16 < D && v < V) piece[i] = *reinterpret_cast<const i32x4 *>(w + (int64_t)v * D + slot * 16);
    }
    if (tid < kCols) {
      const int v = stage * kCols + tid;
      piece_bias = v < V ? (bias ? bias[v] : 0.f) : OT_NEG_INF;
    }
  };
  auto store_stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int p = tid + i * kBlock, row = p / kSlots, slot = p % kSlots;
      s_w[buf][place(row, slot)] = piece[i];
    }
    if (tid < kCols) s_bias[buf][tid] = piece_bias;
  };

  load_stage(stage0);
  const int64_t group0 = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * (64 * TILES);
  if (group0 >= rows) return;
  const int64_t row0 = group0 + wave * (16 * TILES);
  bf16x8 xf[TILES][KB][4];
  float xscale[TILES][KB];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int64_t row = min(row0 + 16 * t + r, rows - 1);
    const unsigned char *xr = x + row * D;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      xscale[t][b] = b < nblocks ? xs[row * nblocks + b] : 0.f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = b * kBlocksK + 64 * q + 16 * h;
        i32x4 c = {0, 0, 0, 0};
        if (k < D) c = *reinterpret_cast<const i32x4 *>(xr + k);
        xf[t][b][2 * q] = widen(c[0], c[1]);
        xf[t][b][2 * q + 1] = widen(c[2], c[3]);
      }
    }
  }
  store_stage(0);
  lds_barrier();

  // this workgroup's logits; a lane's byte offset of row t at its first entry of a stage
  const __amdgpu_buffer_rsrc_t out =
      make_buffer(static_cast<char *>(logits) + group0 * V * kOut,
                  (unsigned)min((int64_t)(64 * TILES), rows - group0) * (unsigned)V * kOut);
  const unsigned out_row = ((unsigned)(wave * (16 * TILES) + r) * (unsigned)V + (unsigned)(kGroup * h)) * kOut;
  const unsigned out_tile = 16u * (unsigned)V * kOut;

  // running log-sum-exp of this lane's share of its rows, relative to ref, which follows the
  // largest value so far at a distance of at most 20
  constexpr float kLog2e = 1.44269502162933349609375f;
  float ref[TILES], sum[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    ref[t] = -1e30f;
    sum[t] = 0.f;
  }

  // Row m = 4 h + i of the tile of group `sub` stands for entry kGroup * h + 4 * sub + i of the
  // 16 * kSubs entries.  As an operand row it is lane r = m.
  const int entry0 = kGroup * (r >> 2) + (r & 3);
  // slot 4 q + h of a block, swizzled by the entry's row in LDS: its low three bits
  auto weight_at = [&](int sub, int q) -> const i32x4 * {
    return &s_w[0][place(entry0 + 4 * sub, 4 * q + h)];
  };
  const i32x4 *read_at[kSubs][2];
#pragma unroll
  for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
    for (int q = 0; q < 2; ++q) read_at[sub][q] = weight_at(sub, q);
  // step (group of 16 entries `g` of the stage, block b) of buffer buf
  auto read_weight = [&](int buf, int g, int b, i32x4 (&f)[2]) {
    const int at = buf * kLdsSlots + (kSubs == 1 && g == 1 ? place(16, 0) : 0) + 8 * b;
#pragma unroll
    for (int q = 0; q < 2; ++q) f[q] = read_at[g % kSubs][q][at];
  };

  i32x4 raw[2][2];  // weight of a step and of the next one
  read_weight(0, 0, 0, raw[0]);
  float scale[TILES][KB];
  for (int stage = stage0; stage < stage1; ++stage) {
    const int buf = (stage - stage0) & 1;
    const bool more = stage + 1 < stage1;
    if (more) load_stage(stage + 1);
    {  // the stage lies in one block of 128 vocabulary entries
      const float *wsr = ws + (int64_t)(stage * kCols / kBlocksK) * nblocks;
#pragma unroll
      for (int c = 0; c < KB; ++c) {
        const float sw = c < nblocks ? wsr[c] : 0.f;
#pragma unroll
        for (int t = 0; t < TILES; ++t) scale[t][c] = xscale[t][c] * sw;
      }
    }
#pragma unroll
    for (int set = 0; set < kCols / (16 * kSubs); ++set) {
      f32x4 acc[kSubs][TILES];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        const int g = set * kSubs + sub;
        if (g == kCols / 16 - 1 && more) store_stage(buf ^ 1);
        const f32x4 start =
            *reinterpret_cast<const f32x4 *>(&s_bias[buf][16 * kSubs * set + kGroup * h + 4 * sub]);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const int cur = (g * KB + b) & 1;  // (a stage has an even number of steps)
          // the next step's weight; behind the last step of a stage lies the barrier
          if (b + 1 < KB) read_weight(buf, g, b + 1, raw[cur ^ 1]);
          else if (g + 1 < kCols / 16) read_weight(buf, g + 1, 0, raw[cur ^ 1]);
          else {
            lds_barrier();
            read_weight(buf ^ 1, 0, 0, raw[cur ^ 1]);
          }
          f32x4 p[TILES];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const i32x4 d = raw[cur][i / 2];
            const bf16x8 wf = i & 1 ? widen(d[2], d[3]) : widen(d[0], d[1]);
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < TILES; ++t)
              p[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[t][b][i], i == 0 ? zero : p[t], 0, 0, 0);
          }
#pragma unroll
          for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[sub][t][i] = __builtin_fmaf(p[t][i], scale[t][b], b == 0 ? start[i] : acc[sub][t][i]);
        }
      }
      // rounding, store, log-sum-exp
      const int v0 = stage * kCols + 16 * kSubs * set;  // this lane: entries v0 + kGroup * h, + kGroup
      const int v = v0 + kGroup * h;
      const unsigned at = v + kGroup <= V ? out_row + (unsigned)v0 * kOut : kNowhere;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const unsigned to = at == kNowhere ? kNowhere : at + t * out_tile;
        if constexpr (kOut == 4) {
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[0][t]), out, to, 0, 0);
        } else {
          unsigned short e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = from_float<T>(acc[i / 4][t][i % 4]);
          if constexpr (ALIGNED) {
            u32x4 four;
#pragma unroll
            for (int i = 0; i < 4; ++i) four[i] = (unsigned)e[2 * i] | ((unsigned)e[2 * i + 1] << 16);
            __builtin_amdgcn_raw_buffer_store_b128(four, out, to, 0, 0);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) __builtin_amdgcn_raw_buffer_store_b16(e[i], out, to + 2 * i, 0, 0);
          }
        }
      }
      if (v0 + 16 * kSubs > V && v < V && v + kGroup > V) {  // the lane whose entries V cuts
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const int64_t row = row0 + 16 * t + r;
#pragma unroll
          for (int i = 0; i < kGroup - 1; ++i)
            if (v + i < V && row < rows) store_logit<T>(logits, row * V + v + i, acc[i / 4][t][i % 4]);
        }
      }
      if constexpr (DEN) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          float top = acc[0][t][0];
#pragma unroll
          for (int i = 1; i < kGroup; ++i) top = fmaxf(top, acc[i / 4][t][i % 4]);
          const float to = top > ref[t] + 20.f ? fminf(top, 3e38f) : ref[t];
          float s = sum[t] * __builtin_amdgcn_exp2f((ref[t] - to) * kLog2e);
          // (a difference first: in powers of 2 the rounding of a large `to` would be an exponent)
#pragma unroll
          for (int i = 0; i < kGroup; ++i) s += __builtin_amdgcn_exp2f((acc[i / 4][t][i % 4] - to) * kLog2e);
          sum[t] = s;
          ref[t] = to;
        }
      }
    }
  }
  if constexpr (DEN) {
    // the four lanes of a row meet
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      LogSum run = {ref[t], sum[t]};
#pragma unroll
      for (int d = 16; d < 64; d *= 2)
        run = merge(run, {__shfl_xor(run.m, d, kWave), __shfl_xor(run.s, d, kWave)});
      const int64_t row = row0 + 16 * t + r;
      if (h == 0 && row < rows) {
        if (parts) parts[(int64_t)part * rows + row] = run;
        else den[row] = logf(run.s) + (__builtin_isinf(run.m) ? 0.f : run.m);
      }
    }
  }
}

// den[r] = log-sum-exp of a row's parts, merged in order
__global__ __launch_bounds__(kBlock) void project_blocks_den_kernel(const LogSum *__restrict__ parts,
                                                                   int nparts, int64_t rows,
                                                                   float *__restrict__ den) {
  const int64_t r = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (r >= rows) return;
  LogSum t = parts[r];
  for (int k = 1; k < nparts; ++k) t = merge(t, parts[(int64_t)k * rows + r]);
  den[r] = logf(t.s) + (__builtin_isinf(t.m) ? 0.f : t.m);
}

// Workgroups of a launch: a part of the vocabulary for each where the rows alone do not fill the
// chip, with the denominators merged from the parts.
struct ProjectGrid {
  dim3 grid;
  int stages_per_part, nparts;
  ProjectGrid(int64_t row_groups, int64_t stages, int64_t wanted) {
    int64_t split = row_groups >= wanted ? 1 : (wanted + row_groups - 1) / row_groups;
    if (split > stages) split = stages;
    stages_per_part = (int)((stages + split - 1) / split);
    nparts = (int)((stages + stages_per_part - 1) / stages_per_part);
    // (a launch holds 2^32 threads at most in each direction)
    constexpr int64_t kMostX = 1 << 20;
    grid = dim3((unsigned)(row_groups < kMostX ? row_groups : kMostX), (unsigned)nparts,
                (unsigned)((row_groups + kMostX - 1) / kMostX));
  }
};

template <class T, int KB, int TILES, int COLS, int WAVES_PER_SIMD>
static int launch_project_blocks_kernel(const unsigned char *x, const float *xs, const unsigned char *w,
                                        const float *ws, const float *bias, int64_t rows, int32_t D, int32_t V,
                                        void *logits, float *den, LogSum *parts, int cus, hipStream_t s) {
  const ProjectGrid g((rows + 64 * TILES - 1) / (64 * TILES), (V + COLS - 1) / COLS, (int64_t)cus * WAVES_PER_SIMD);
  const bool merged = den && g.nparts > 1;
  hipLaunchKernelGGL((project_blocks_kernel<T, KB, TILES, COLS, WAVES_PER_SIMD>),
                     g.grid, dim3(kBlock), 0, s, x, xs, w, ws, bias, rows, D, V, g.stages_per_part, logits,
                     merged ? nullptr : den, merged ? parts : nullptr);
  if (merged)
    hipLaunchKernelGGL(project_blocks_den_kernel, dim3((unsigned)((rows + kBlock - 1) / kBlock)), dim3(kBlock),
                       0, s, parts, g.nparts, rows, den);
  return (int)hipGetLastError();
}

template <class T, int KB, int TILES, int WAVES_PER_SIMD>
static int launch_project_blocks_wide(const unsigned char *x, const float *xs, const unsigned char *w,
                                      const float *ws, const float *bias, int64_t rows, int32_t D, int32_t V,
                                      void *logits, float *den, LogSum *parts, int cus, hipStream_t s) {
  const ProjectGrid g((rows + 64 * TILES - 1) / (64 * TILES), (V + kWideCols - 1) / kWideCols,
                      (int64_t)cus * WAVES_PER_SIMD);
  const bool merged = den && g.nparts > 1;
#define OT_WIDE(ALIGNED_, DEN_)                                                                             \
  hipLaunchKernelGGL((project_blocks_wide_kernel<T, KB, TILES, WAVES_PER_SIMD, ALIGNED_, DEN_>), g.grid, dim3(kBlock), 0, s, \
                     x, xs, w, ws, bias, rows, D, V, g.stages_per_part, logits, merged ? nullptr : den,      \
                     merged ? parts : nullptr)
  if (sizeof(T) == 4 || (V % 2 == 0 && (reinterpret_cast<uintptr_t>(logits) & 3) == 0)) {
    if (den) OT_WIDE(true, true);
    else OT_WIDE(true, false);
  } else if constexpr (sizeof(T) != 4) {
    if (den) OT_WIDE(false, true);
    else OT_WIDE(false, false);
  }
#undef OT_WIDE
  if (merged)
    hipLaunchKernelGGL(project_blocks_den_kernel, dim3((unsigned)((rows + kBlock - 1) / kBlock)), dim3(kBlock),
                       0, s, parts, g.nparts, rows, den);
  return (int)hipGetLastError();
}

template <class T>
static int launch_project_blocks(const unsigned char *x, const float *xs, const unsigned char *w,
                                 const float *ws, const float *bias, int64_t rows, int32_t D, int32_t V,
                                 void *logits, float *den, LogSum *parts, hipStream_t s) {
  int device = 0, cus = 0;
  if (hipGetDevice(&device) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || cus <= 0)
    return OT_E_BAD_ARG;
  const int nblocks = (D + kBlocksK - 1) / kBlocksK;
  // (the wide kernel addresses a workgroup's logits with 32 bits)
  if (rows > 64 && nblocks <= 16 && V < (1 << 21)) {
#define OT_PROJECT(KB_, TILES_, COLS_, WAVES_)                                                              \
  return launch_project_blocks_kernel<T, KB_, TILES_, COLS_, WAVES_>(x, xs, w, ws, bias, rows, D, V, logits, \
                                                                     den, parts, cus, s)
#define OT_PROJECT_WIDE(KB_, TILES_, WAVES_)                                                                         \
  return launch_project_blocks_wide<T, KB_, TILES_, WAVES_>(x, xs, w, ws, bias, rows, D, V, logits, den, parts, cus, s)
    if (nblocks == 1) OT_PROJECT_WIDE(1, 2, 2);
    if (nblocks == 2) OT_PROJECT_WIDE(2, 2, 2);
    if (nblocks == 3) OT_PROJECT_WIDE(3, 2, 2);
    if (nblocks == 4) OT_PROJECT_WIDE(4, 2, 2);
    if (nblocks <= 8) OT_PROJECT(8, 2, 32, 1);
#undef OT_PROJECT_WIDE
    OT_PROJECT(16, 1, 16, 1);
#undef OT_PROJECT
  }
  const int col_tiles = (V + kSmallCols - 1) / kSmallCols;
  const int64_t tiles = (rows + 15) / 16 * col_tiles;
  const dim3 grid((unsigned)(tiles < (1 << 22) ? tiles : (1 << 22)));
  hipLaunchKernelGGL((project_blocks_small_kernel<T>), grid, dim3(kBlock), 0, s, x, xs, w, ws, bias, rows, D,
                     V, col_tiles, tiles, logits, den ? parts : nullptr);
  if (den)
    hipLaunchKernelGGL(project_blocks_den_kernel, dim3((unsigned)((rows + kBlock - 1) / kBlock)), dim3(kBlock),
                       0, s, parts, col_tiles, rows, den);
  return (int)hipGetLastError();
}

}  // namespace ot

using namespace ot;

extern "C" {

size_t ot_joiner_project_blocks_workspace_bytes(int64_t rows, int32_t V) {
  if (rows <= 0 || V <= 0) return 0;
  return (size_t)((V + kPartCols - 1) / kPartCols) * (size_t)rows * sizeof(LogSum);
}

int ot_joiner_project_blocks(const void *x, const float *x_scale, const void *weight,
                             const float *weight_scale, const float *bias, int64_t rows, int32_t D, int32_t V,
                             void *logits, int32_t logits_dtype, float *den, void *workspace,
                             size_t workspace_bytes, void *stream) {
  if (rows == 0) return 0;
  if (!x || !x_scale || !weight || !weight_scale || !logits || rows < 0 || rows > INT32_MAX || D <= 0 ||
      V <= 0 || D % kBlocksUnit != 0 || D > INT32_MAX - 2 * kBlocksK || V > INT32_MAX - 2 * kBlocksK)
    return OT_E_BAD_ARG;
  if (den && (!workspace || workspace_bytes < ot_joiner_project_blocks_workspace_bytes(rows, V)))
    return OT_E_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(weight) & 15) ||
      (reinterpret_cast<uintptr_t>(x_scale) & 3) || (reinterpret_cast<uintptr_t>(weight_scale) & 3) ||
      (reinterpret_cast<uintptr_t>(bias) & 3) || (reinterpret_cast<uintptr_t>(den) & 3) ||
      (reinterpret_cast<uintptr_t>(workspace) & 7) ||
      (reinterpret_cast<uintptr_t>(logits) & (logits_dtype == OT_DTYPE_F32 ? 3 : 1)))
    return OT_E_MISALIGNED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned char *xp = static_cast<const unsigned char *>(x);
  const unsigned char *wp = static_cast<const unsigned char *>(weight);
  LogSum *parts = static_cast<LogSum *>(workspace);
  if (logits_dtype == OT_DTYPE_F32)
    return launch_project_blocks<float>(xp, x_scale, wp, weight_scale, bias, rows, D, V, logits, den, parts, s);
  if (logits_dtype == OT_DTYPE_F16)
    return launch_project_blocks<F16>(xp, x_scale, wp, weight_scale, bias, rows, D, V, logits, den, parts, s);
  if (logits_dtype == OT_DTYPE_BF16)
    return launch_project_blocks<BF16>(xp, x_scale, wp, weight_scale, bias, rows, D, V, logits, den, parts, s);
  return OT_E_BAD_ARG;
}

}  // extern "C"
