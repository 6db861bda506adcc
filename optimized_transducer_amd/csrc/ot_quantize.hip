// Quantisation to 8 bits in blocks of 128 (gfx950).
//
// A block is 128 consecutive elements of one row (activations) or of 128 rows
// (weights); the last block of a row and the last block of rows may be partial.
//     scale  = max(fl32(max|x| / 448), 2^-126)
//     values = e4m3(fl32(x / scale)),  both roundings to nearest even
// 448 is the largest e4m3 value, so the largest element of a block uses the whole
// range.  The scale is a stored float32 and the quotient is the IEEE one: the result
// is defined bit for bit.  A NaN or an infinity makes its block's scale NaN or
// infinite, and with it every product that the block enters.
//
// Bound by memory: every element is read once, 8 per lane in 16-byte loads, and stays in registers
// between the maximum and the quotient.  Blocks of one row need 16 lanes and four cross-lane steps,
// and no LDS: 751 992 x 512 bfloat16 takes 239 us, 4.9 TB/s (a large copy reaches 4.7).  A block of
// 128 x 128 is a workgroup's, 64 elements a lane, one barrier: 5000 x 1000 float32 takes 9.6 us, 2.6
// TB/s, of which a launch alone is 5.  32 x 512 are a launch, 5.2 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ot_device.hip.h"
#include "ot_transducer.h"

namespace ot {

constexpr int kQuantBlock = 128;   // elements of a row per scale
constexpr int kQuantUnit = 8;      // elements of a row per lane
constexpr int kQuantLanes = kQuantBlock / kQuantUnit;      // 16 lanes: one row of a block
constexpr int kQuantGroups = kBlock / kQuantLanes;         // rows of blocks per workgroup pass
constexpr float kE4m3Max = 448.0f;
constexpr float kSmallestScale = 1.17549435082228750797e-38f;  // 2^-126

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// |x| as an integer: integers order like the magnitudes, and every NaN is above infinity,
// so the maximum does not lose a NaN (fmaxf would)
__device__ __forceinline__ unsigned magnitude_bits(float x) {
  return __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true));
}

// maximum over aligned groups of 16 lanes
__device__ __forceinline__ unsigned group16_max(unsigned v) {
  v = dpp_max<kDppQuadXor1>(v);
  v = dpp_max<kDppQuadXor2>(v);
  v = dpp_max<kDppRowHalfMirror>(v);
  return dpp_max<kDppRowMirror>(v);
}

__device__ __forceinline__ float block_scale(unsigned max_bits) {
  const float s = __builtin_bit_cast(float, max_bits) / kE4m3Max;
  return s < kSmallestScale ? kSmallestScale : s;  // a NaN stays
}

// Elements [c, c + 8) of row `row`; those at or past D read as 0.  16-byte loads, which a row may
// start anywhere for (200 000 x 513 float32 113 us, 235 by single elements).  WHOLE: all are there.
template <class T, bool WHOLE>
__device__ __forceinline__ void load8(const void *x, int64_t row_stride, int64_t row, int c, int D,
                                      float v[kQuantUnit]) {
  const int64_t at = row * row_stride + c;
  if constexpr (!WHOLE) {
#pragma unroll
    for (int i = 0; i < kQuantUnit; ++i) v[i] = c + i < D ? load_element<T>(x, at + i) : 0.f;
  } else if constexpr (sizeof(T) == 4) {
    typedef f32x4 unaligned __attribute__((aligned(4)));
    const unaligned *p = reinterpret_cast<const unaligned *>(static_cast<const float *>(x) + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
    typedef u32x4 unaligned __attribute__((aligned(2)));
    const u32x4 a = *reinterpret_cast<const unaligned *>(static_cast<const unsigned short *>(x) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned w = a[i];
      v[2 * i] = to_float<T>((unsigned short)(w & 0xffffu));
      v[2 * i + 1] = to_float<T>((unsigned short)(w >> 16));
    }
  }
}

// e4m3(v / scale) to values[row, c .. c + 8)
__device__ __forceinline__ void store8(const float v[kQuantUnit], float scale, unsigned char *values,
                                       int64_t row, int c, int D) {
  unsigned w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] / scale, v[4 * h + 1] / scale, 0, false);
    w[h] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] / scale, v[4 * h + 3] / scale, t, true);
  }
  unsigned char *p = values + row * D + c;
  if (c + kQuantUnit <= D) {
    typedef u32x2 unaligned __attribute__((aligned(1)));
    const u32x2 t = {w[0], w[1]};
    *reinterpret_cast<unaligned *>(p) = t;
  } else if (c < D) {
#pragma unroll
    for (int i = 0; i < kQuantUnit; ++i)
      if (c + i < D) p[i] = (unsigned char)(w[i / 4] >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ unsigned max8(const float v[kQuantUnit]) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < kQuantUnit; ++i) m = max(m, magnitude_bits(v[i]));
  return m;
}

// blocks of 128 elements of one row: 16 lanes each
template <class T>
__global__ __launch_bounds__(kBlock) void quantize_rows_kernel(const void *__restrict__ x,
                                                               int64_t row_stride, int64_t rows, int D,
                                                               int nblocks,
                                                               unsigned char *__restrict__ values,
                                                               float *__restrict__ scale) {
  const int64_t units = rows * nblocks;
  const int l = threadIdx.x % kQuantLanes;
  for (int64_t u = (int64_t)blockIdx.x * kQuantGroups + threadIdx.x / kQuantLanes; u < units;
       u += (int64_t)gridDim.x * kQuantGroups) {
    const int64_t row = u / nblocks;
    const int c = (int)(u - row * nblocks) * kQuantBlock + l * kQuantUnit;
    float v[kQuantUnit];
    if (c + kQuantUnit <= D) load8<T, true>(x, row_stride, row, c, D, v);
    else load8<T, false>(x, row_stride, row, c, D, v);
    const float s = block_scale(group16_max(max8(v)));
    store8(v, s, values, row, c, D);
    if (l == 0) scale[u] = s;
  }
}

// blocks of 128 x 128: one workgroup each, 8 rows per group of 16 lanes
template <class T>
__global__ __launch_bounds__(kBlock) void quantize_tiles_kernel(const void *__restrict__ x,
                                                                int64_t row_stride, int64_t rows, int D,
                                                                int nblocks,
                                                                unsigned char *__restrict__ values,
                                                                float *__restrict__ scale) {
  constexpr int kRows = kQuantBlock / kQuantGroups;
  __shared__ unsigned s_max[kWavesPerBlock];
  const int64_t tile_row = blockIdx.x / nblocks;
  const int l = threadIdx.x % kQuantLanes;
  const int64_t row0 = tile_row * kQuantBlock + threadIdx.x / kQuantLanes;
  const int c = (int)(blockIdx.x - tile_row * nblocks) * kQuantBlock + l * kQuantUnit;
  float v[kRows][kQuantUnit];
  unsigned m = 0;
  // (one branch around all loads, so that they are on their way together; rows past the end read
  // the last one)
  if (c + kQuantUnit <= D) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      load8<T, true>(x, row_stride, min(row0 + i * kQuantGroups, rows - 1), c, D, v[i]);
  } else if (c < D) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      load8<T, false>(x, row_stride, min(row0 + i * kQuantGroups, rows - 1), c, D, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int k = 0; k < kQuantUnit; ++k) v[i][k] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (row0 + i * kQuantGroups < rows) m = max(m, max8(v[i]));
  m = group16_max(m);
  m = max(m, (unsigned)__shfl_xor((int)m, 16, kWave));
  m = max(m, (unsigned)__shfl_xor((int)m, 32, kWave));
  if (threadIdx.x % kWave == 0) s_max[threadIdx.x / kWave] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWavesPerBlock; ++i) m = max(m, s_max[i]);
  const float s = block_scale(m);
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t row = row0 + i * kQuantGroups;
    if (row < rows) store8(v[i], s, values, row, c, D);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
}

template <class T>
static int launch_quantize(const void *x, int64_t row_stride, int64_t rows, int32_t D, int32_t block_rows,
                           unsigned char *values, float *scale, hipStream_t s) {
  const int nblocks = (D + kQuantBlock - 1) / kQuantBlock;
  if (block_rows == 1) {
    const int64_t groups = (rows * nblocks + kQuantGroups - 1) / kQuantGroups;
    const dim3 grid((unsigned)(groups < (1 << 20) ? groups : (1 << 20)));
    hipLaunchKernelGGL((quantize_rows_kernel<T>), grid, dim3(kBlock), 0, s, x, row_stride, rows, D, nblocks, values,
                       scale);
  } else {
    const int64_t tiles = (rows + kQuantBlock - 1) / kQuantBlock * nblocks;
    if (tiles > (1 << 23)) return OT_E_TOO_LONG;  // a launch holds 2^32 threads at most
    const dim3 grid((unsigned)tiles);
    hipLaunchKernelGGL((quantize_tiles_kernel<T>), grid, dim3(kBlock), 0, s, x, row_stride, rows, D, nblocks, values,
                       scale);
  }
  return (int)hipGetLastError();
}

}  // namespace ot

using namespace ot;

extern "C" int ot_quantize_blocks(const void *x, int32_t dtype, int64_t row_stride, int64_t rows, int32_t D,
                                  int32_t block_rows, void *values, float *scale, void *stream) {
  if (rows == 0) return 0;
  if (!x || !values || !scale || rows < 0 || rows > INT32_MAX || D <= 0 || D > INT32_MAX - kQuantBlock ||
      row_stride < 0 || (block_rows != 1 && block_rows != kQuantBlock))
    return OT_E_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(x) & (dtype == OT_DTYPE_F32 ? 3 : 1)) ||
      (reinterpret_cast<uintptr_t>(scale) & 3))
    return OT_E_MISALIGNED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  unsigned char *q = static_cast<unsigned char *>(values);
  if (dtype == OT_DTYPE_F32) return launch_quantize<float>(x, row_stride, rows, D, block_rows, q, scale, s);
  if (dtype == OT_DTYPE_F16) return launch_quantize<F16>(x, row_stride, rows, D, block_rows, q, scale, s);
  if (dtype == OT_DTYPE_BF16) return launch_quantize<BF16>(x, row_stride, rows, D, block_rows, q, scale, s);
  return OT_E_BAD_ARG;
}
