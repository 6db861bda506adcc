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
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kBlocksK = 128;      // elements per scale
constexpr int kBlocksUnit = 16;    // D is a multiple of this: one 16-byte load
constexpr int kPartCols = 64;      // vocabulary entries behind one partial log-sum-exp

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
    const int v0 = part * kPartCols + wave * 16;
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

template <class T>
static int launch_project_blocks(const unsigned char *x, const float *xs, const unsigned char *w,
                                 const float *ws, const float *bias, int64_t rows, int32_t D, int32_t V,
                                 void *logits, float *den, LogSum *parts, hipStream_t s) {
  const int col_tiles = (V + kPartCols - 1) / kPartCols;
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
