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
constexpr int kSmallCols = 64;     // vocabulary entries of a workgroup of the small kernel
// the wide kernel: vocabulary entries of a stage, tiles of 16 rows of a wave, rows of a workgroup
constexpr int kWideCols = 64, kWideTiles = 2, kWideRows = kWavesPerBlock * kWideTiles * 16;
constexpr int kPartCols = 64;      // least vocabulary entries behind one partial log-sum-exp

constexpr float kLargest = 3.402823466385288598e38f;  // the largest finite float32

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

// Few rows.  A workgroup of 4 waves forms 16 packed rows x 64 vocabulary entries, a wave one
// accumulator tile of 16 x 16 straight from memory.  Lane l holds elements
// [32 * (l / 16), + 32) of a block of row l % 16 of either operand.  The loads' latency, block
// after block, is what it waits for: 1 x 1024 x 16384 takes 8.1 us, 2.1 TB/s of weight, where a
// launch alone is 5.
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
        parts[(row0 + threadIdx.x) * col_tiles + part] = t;
      }
    }
  }
}

// Many rows of up to KB blocks.  A workgroup of 4 waves owns 128 packed rows; a wave holds its 32
// rows of x, widened, in registers for the whole walk over the vocabulary, so x is read and widened
// once.  The weight goes by in stages of 64 vocabulary entries (all of D, 8-bit, 32 KB at D = 512),
// loaded straight into one of two LDS buffers, with one barrier per stage.
//
// Loads and stores share one in-order counter: whoever waits for a load waits for every store
// before it, and stores are what takes longest here.  The next stage's loads are issued at the
// start of a stage, in front of its stores, and what is waited for at its end is all but the last
// kStores operations: the loads, and the stores of the stage before, which have had a whole
// stage's time to drain.
//
// The walk advances in steps of 16 vocabulary entries x one block (8 matrix instructions); the LDS
// read of a step's weight is issued one step ahead.  Rows past the end are dropped by the bounds of
// the store's buffer view, entries past the end have weight 0 and are set to -inf.
//
// Which entry of the vocabulary a row of the accumulator tile stands for is free: it is chosen so
// that a lane ends up with 16 bytes of consecutive logits and four lanes with 64, from one group of
// 16 entries for 4-byte logits and from two for 2-byte ones.
//   ALIGNED: 16 bytes of logits start at a multiple of 4 bytes.  Else (2-byte logits of an odd V)
//   they go through ordinary stores, which any element may start at, and not the buffer view's:
//   100 000 x 512 x 501 float16 146 us with stores of single elements, 93 so
// What bounds it: vector instructions (7.3 for each matrix instruction: widening, scales, rounding,
// exponentials) and matrix instructions follow each other, with two waves a SIMD to overlap them.  751 992 x
// 512 x 500 bfloat16 with denominators: vector 64 % and matrix instructions 33 % of the cycles, 0.54 ms, 711
// TFLOP/s and 2.2 TB/s (where it takes 0.55, 0.52 without the stores, 0.37 without the matrix instructions,
// 0.49 without denominators).  149 346 x 512 x 5000 float32: 46 % and 27 %, and the stores, 1.24 ms, 617
// TFLOP/s and 2.5 TB/s (0.99 without the stores, 1.17 without the matrix instructions).  Tiles straight
// from memory, as the small kernel's, take 3.19 and 6.26 ms.
// Lane l holds bytes [64 q + 16 (l / 16), + 16) of a block of row l % 16 (q = 0, 1); the first 8
// feed matrix instruction 2 q and the others 2 q + 1, in both operands alike.
template <class T, int KB, bool ALIGNED, bool DEN>
struct WideProject {
  static constexpr int kSlots = KB * 8;  // 16-byte slots of a row
  static constexpr int kPieces = kWideCols * kSlots / kBlock;  // loads of a stage per thread
  static constexpr unsigned kOut = sizeof(T) == 4 ? 4u : 2u;
  static constexpr int kGroup = 16 / (int)kOut;  // consecutive entries of a lane
  static constexpr int kSubs = kGroup / 4;       // groups of 16 entries behind them
  static constexpr int kGroups = kWideCols / 16;
  static constexpr int kStores = kGroups / kSubs * kWideTiles;  // of a stage, at least
  typedef i32x4 Weights[kWideCols * kSlots];
  typedef float Biases[kWideCols];

  const unsigned char *w;
  const float *ws, *bias;
  int D, V, lane, wave, r, h;
  bf16x8 x[kWideTiles][KB][4];
  const float (*xs)[16][kWideTiles];  // this wave's scales of x in LDS
  __amdgpu_buffer_rsrc_t out;
  char *out_base;              // the same place
  bool rows_in;                // all rows of this wave are there
  unsigned out_row, out_tile;  // byte offsets of this lane's first logit and from tile to tile
  float ref[kWideTiles], sum[kWideTiles];
  i32x4 raw[2][2];  // weight of a step and of the next one
  int at[kSubs][2][2];

  // entry of a stage that row m of group g's tile stands for, as an operand row and as a result
  __device__ __forceinline__ static int entry(int g, int m) {
    return (g / kSubs) * (16 * kSubs) + kGroup * (m >> 2) + 4 * (g % kSubs) + (m & 3);
  }
  // A 16-byte read is served 16 lanes at a time: lanes 0-7 and 24-31 of a half-wave, or 8-23.
  // Where rows are a multiple of 256 bytes, the number of the lane that reads a row (entry()
  // backwards) spreads those over all 64 banks; with others, three bits of it and the rows' own
  // offset do.
  __device__ __forceinline__ static int swizzle(int row) {
    const int m = kSubs == 1 ? row & 15 : (row & 3) | ((row >> 1) & 12);
    return KB % 2 == 0 ? m : m & 7;
  }

  // the weight and the bias of a stage into LDS; entries past the end and elements past D are 0
  __device__ __forceinline__ void load(int stage, i32x4 *weights, float *biases) const {
    const int v0 = min(stage * kWideCols, V), n = min(kWideCols, V - v0);
    const __amdgpu_buffer_rsrc_t from = make_buffer(w + (int64_t)min(v0, V - 1) * D, (unsigned)n * (unsigned)D);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int first = (wave * kPieces + i) * kWave, p = first + lane;
      const int row = p / kSlots, slot = (p % kSlots) ^ swizzle(row);
      const unsigned src = slot * 16 < D ? (unsigned)row * (unsigned)D + 16u * slot : 0x7fffffffu;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)(weights + first), 16,
                                               src, 0, 0, 0);
    }
    if (wave == 0) {
      const __amdgpu_buffer_rsrc_t b =
          make_buffer(bias ? bias + min(v0, V - 1) : (const float *)w, bias ? (unsigned)n * 4u : 0u);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void *)biases, 4,
                                               (unsigned)lane * 4u, 0, 0, 0);
    }
  }

  // the weight of step (group g, block b)
  __device__ __forceinline__ void read(const i32x4 *weights, int g, int b, i32x4 (&f)[2]) const {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      f[q] = weights[at[g % kSubs][q][b & 1] + (g / kSubs) * (16 * kSubs) * kSlots + 8 * (b & ~1)];
  }

  // one stage: its weight and bias are in LDS, its first step in raw[0]; the next stage's, if there
  // is one, go to `next` and raw[0] (nothing may be on its way to LDS when a workgroup ends)
  __device__ __forceinline__ void run(int stage, bool more, const i32x4 *weights, const float *biases,
                                      i32x4 *next_weights, float *next_biases) {
    if (more) load(stage + 1, next_weights, next_biases);
    __builtin_amdgcn_sched_barrier(0);  // no store of this stage in front of its loads
    const int v0 = stage * kWideCols;
    const float *wsr = ws + (int64_t)(v0 / kBlocksK) * KB;  // the stage lies in one block of 128 entries
    float sw[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) sw[b] = wsr[b];
#pragma unroll
    for (int set = 0; set < kGroups / kSubs; ++set) {
      f32x4 acc[kSubs][kWideTiles];
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        const int g = set * kSubs + sub;
        const f32x4 start = *reinterpret_cast<const f32x4 *>(biases + entry(g, 4 * h));
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const int cur = (g * KB + b) & 1;  // (a stage has an even number of steps)
          if (b + 1 < KB) read(weights, g, b + 1, raw[cur ^ 1]);
          else if (g + 1 < kGroups) read(weights, g + 1, 0, raw[cur ^ 1]);
          float scale[kWideTiles];
#pragma unroll
          for (int t = 0; t < kWideTiles; ++t) scale[t] = xs[b][r][t] * sw[b];
          f32x4 p[kWideTiles];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const i32x4 d = raw[cur][i / 2];
            const bf16x8 wf = i & 1 ? widen(d[2], d[3]) : widen(d[0], d[1]);
            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < kWideTiles; ++t)
              p[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, x[t][b][i], i == 0 ? zero : p[t], 0, 0, 0);
          }
#pragma unroll
          for (int t = 0; t < kWideTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[sub][t][i] = __builtin_fmaf(p[t][i], scale[t], b == 0 ? start[i] : acc[sub][t][i]);
        }
      }
      finish(v0, set, acc);
    }
    if (more) {
      // Every set of a stage that V does not cut has stored kWideTiles times: all but the last
      // kStores operations are over (vmcnt; the other counters free).
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0x0f70 | kStores);
      lds_barrier();
      read(next_weights, 0, 0, raw[0]);
    }
  }

  // rounding, store and log-sum-exp of entries [v0 + 16 * kSubs * set, + 16 * kSubs)
  __device__ __forceinline__ void finish(int v0, int set, f32x4 (&acc)[kSubs][kWideTiles]) {
    const int v = v0 + entry(set * kSubs, 4 * h);  // of this lane: kGroup entries
    const bool whole = v0 + 16 * kSubs * (set + 1) <= V;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i)
        if (v + i >= V)
#pragma unroll
          for (int t = 0; t < kWideTiles; ++t) acc[i / 4][t][i % 4] = OT_NEG_INF;
    }
    u32x4 four[kWideTiles];
#pragma unroll
    for (int t = 0; t < kWideTiles; ++t) {
      if constexpr (kOut == 4) {
        four[t] = __builtin_bit_cast(u32x4, acc[0][t]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // the float32 sum is rounded, whatever else becomes of it: a multiply-add that rounds
          // straight to float16 gives other bits now and then
          float lo = acc[i / 2][t][2 * (i & 1)], hi = acc[i / 2][t][2 * (i & 1) + 1];
          asm("" : "+v"(lo), "+v"(hi));
          four[t][i] = (unsigned)from_float<T>(lo) | ((unsigned)from_float<T>(hi) << 16);
        }
      }
    }
    const unsigned dst = out_row + (unsigned)(v0 + 16 * kSubs * set) * kOut;
    if (ALIGNED) {
      // (a group that V cuts goes past the bounds of the view: it is stored below)
      const unsigned to = whole || v + kGroup <= V ? dst : 0xfffffff0u - out_tile;
#pragma unroll
      for (int t = 0; t < kWideTiles; ++t) __builtin_amdgcn_raw_buffer_store_b128(four[t], out, to + t * out_tile, 0, 0);
    }
    const bool single = v + kGroup > V;  // (those that there are of a group that V cuts)
    if (!ALIGNED && rows_in) {
      typedef u32x4 unaligned __attribute__((aligned(2)));
      if (whole || !single)
#pragma unroll
        for (int t = 0; t < kWideTiles; ++t) *reinterpret_cast<unaligned *>(out_base + dst + t * out_tile) = four[t];
    }
    if (!whole || (!ALIGNED && !rows_in)) {
#pragma unroll
      for (int t = 0; t < kWideTiles; ++t)
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
          if (v + i < V && (single || (!ALIGNED && !rows_in))) {
            if constexpr (kOut == 4)
              __builtin_amdgcn_raw_buffer_store_b32(four[t][i], out, dst + t * out_tile + 4 * i, 0, 0);
            else
              __builtin_amdgcn_raw_buffer_store_b16((unsigned short)(four[t][i / 2] >> (16 * (i & 1))), out,
                                                    dst + t * out_tile + 2 * i, 0, 0);
          }
    }
    if constexpr (DEN) {
      // running log-sum-exp of this lane's share of its rows, relative to ref, which follows the
      // largest value so far at a distance of at most 20; it starts at the lowest finite value, so that
      // rows of no larger logits keep their sum, and stays finite, so that differences do
      constexpr float kLog2e = 1.44269502162933349609375f;
#pragma unroll
      for (int t = 0; t < kWideTiles; ++t) {
        float top = acc[0][t][0];
#pragma unroll
        for (int i = 1; i < kGroup; ++i) top = fmaxf(top, acc[i / 4][t][i % 4]);
        const float to = top > ref[t] + 20.f ? fminf(top, kLargest) : ref[t];
        float s = sum[t] * __builtin_amdgcn_exp2f((ref[t] - to) * kLog2e);
        // (a difference first: in powers of 2 the rounding of a large `to` would be an exponent)
#pragma unroll
        for (int i = 0; i < kGroup; ++i) s += __builtin_amdgcn_exp2f((acc[i / 4][t][i % 4] - to) * kLog2e);
        sum[t] = s;
        ref[t] = to;
      }
    }
  }

  // the four lanes of a row meet
  __device__ __forceinline__ void finish_den(int64_t row0, int64_t rows, int part, int nparts, float *den,
                                             LogSum *parts) const {
#pragma unroll
    for (int t = 0; t < kWideTiles; ++t) {
      LogSum run = {ref[t], sum[t]};
#pragma unroll
      for (int d = 16; d < 64; d *= 2)
        run = merge(run, {__shfl_xor(run.m, d, kWave), __shfl_xor(run.s, d, kWave)});
      const int64_t row = row0 + 16 * t + r;
      if (h == 0 && row < rows) {
        if (parts) parts[row * nparts + part] = run;
        else den[row] = logf(run.s) + (__builtin_isinf(run.m) ? 0.f : run.m);
      }
    }
  }
};

template <class T, int KB, bool ALIGNED, bool DEN>
__global__ __launch_bounds__(kBlock, 2) void project_blocks_wide_kernel(
    const unsigned char *__restrict__ x, const float *__restrict__ xs, const unsigned char *__restrict__ w,
    const float *__restrict__ ws, const float *__restrict__ bias, int64_t rows, int D, int V,
    int stages_per_part, void *__restrict__ logits, float *__restrict__ den, LogSum *__restrict__ parts) {
  typedef WideProject<T, KB, ALIGNED, DEN> P;
  // two variables each, and not one array: the compiler then knows that the loads into one do not
  // touch what is read from the other
  __shared__ __attribute__((aligned(16))) typename P::Weights s_w0, s_w1;
  __shared__ __attribute__((aligned(16))) typename P::Biases s_b0, s_b1;
  // scales of x: those of a lane's two rows side by side
  __shared__ __attribute__((aligned(16))) float s_xs[kWavesPerBlock][KB][16][kWideTiles];
  const int tid = threadIdx.x;
  const int64_t group0 = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * kWideRows;
  if (group0 >= rows) return;
  const int stages = (V + kWideCols - 1) / kWideCols;
  const int part = blockIdx.y;
  const int stage0 = part * stages_per_part, stage1 = min(stages, stage0 + stages_per_part);

  P p;
  p.w = w;
  p.ws = ws;
  p.bias = bias;
  p.D = D;
  p.V = V;
  p.lane = tid & 63;
  p.wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  p.r = p.lane & 15;
  p.h = p.lane >> 4;
  p.load(stage0, s_w0, s_b0);
  const int64_t row0 = group0 + p.wave * (16 * kWideTiles);
#pragma unroll
  for (int t = 0; t < kWideTiles; ++t) {
    const int64_t row = min(row0 + 16 * t + p.r, rows - 1);
    const unsigned char *xr = x + row * D;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      if (p.h == 0) s_xs[p.wave][b][p.r][t] = xs[row * KB + b];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = b * kBlocksK + 64 * q + 16 * p.h;
        i32x4 c = {0, 0, 0, 0};
        if (k < D) c = *reinterpret_cast<const i32x4 *>(xr + k);
        p.x[t][b][2 * q] = widen(c[0], c[1]);
        p.x[t][b][2 * q + 1] = widen(c[2], c[3]);
      }
    }
    p.ref[t] = -kLargest;
    p.sum[t] = 0.f;
  }
  p.xs = s_xs[p.wave];
#pragma unroll
  for (int sub = 0; sub < P::kSubs; ++sub)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const int row = P::entry(sub, p.r);
        p.at[sub][q][odd] = row * P::kSlots + ((8 * odd + 4 * q + p.h) ^ P::swizzle(row));
      }
  // this workgroup's logits; rows past the end are dropped by the view's bounds
  p.out_base = static_cast<char *>(logits) + group0 * V * P::kOut;
  p.rows_in = row0 + 16 * kWideTiles <= rows;
  p.out = make_buffer(p.out_base,
                      (unsigned)min((int64_t)kWideRows, rows - group0) * (unsigned)V * P::kOut);
  p.out_row = ((unsigned)(p.wave * (16 * kWideTiles) + p.r) * (unsigned)V + (unsigned)(P::kGroup * p.h)) * P::kOut;
  p.out_tile = 16u * (unsigned)V * P::kOut;

  __builtin_amdgcn_s_waitcnt(0x0f70);  // all loads; the other counters free
  lds_barrier();
  p.read(s_w0, 0, 0, p.raw[0]);
  for (int stage = stage0;;) {
    p.run(stage, stage + 1 < stage1, s_w0, s_b0, s_w1, s_b1);
    if (++stage == stage1) break;
    p.run(stage, stage + 1 < stage1, s_w1, s_b1, s_w0, s_b0);
    if (++stage == stage1) break;
  }
  if constexpr (DEN) p.finish_den(row0, rows, part, gridDim.y, den, parts);
}

// Many rows of any length.  A workgroup of 4 waves forms 128 packed rows x COLS vocabulary entries
// (64 or 128), a wave 32 x COLS in COLS / 2 running sums per lane, block of D after block: the
// weight's block goes straight into one of two LDS buffers, a wave's block of x into registers, both
// one step ahead of the COLS / 2 matrix instructions of a step (two steps ahead spilled registers and
// took 37 us where one takes 32).  Each XCD has an eighth of the tiles in order, so that its L2
// serves x to all but the first tile of a group of rows.
//
// The matrix instructions, the widening in front of them and the LDS reads of a step follow each
// other within a wave and overlap between the two or three of a SIMD: 30 000 x 4096 x 500 float32
// logits take 170 us, 723 TFLOP/s, of the 1380 that a large bfloat16 product reaches.
template <class T, int COLS, bool ALIGNED, bool DEN>
struct DeepProject {
  typedef WideProject<T, 1, ALIGNED, DEN> Wide;  // one block: layout of a step, epilogue
  static constexpr int kSubs = Wide::kSubs;
  static constexpr int kGroups = COLS / 16;
  typedef i32x4 Weights[COLS * 8];

  Wide e;
  const unsigned char *x[kWideTiles];  // this lane's rows
  const float *xs[kWideTiles];
  int v0, nblocks;
  f32x4 acc[kGroups][kWideTiles];
  i32x4 raw[kWideTiles][2];
  float raw_scale[kWideTiles];

  __device__ __forceinline__ void load(int b, i32x4 *weights) {
    const int n = min(COLS, e.V - v0);
    const __amdgpu_buffer_rsrc_t from = make_buffer(e.w + (int64_t)v0 * e.D, (unsigned)n * (unsigned)e.D);
#pragma unroll
    for (int i = 0; i < COLS * 8 / kBlock; ++i) {
      const int first = (e.wave * (COLS * 8 / kBlock) + i) * kWave, p = first + e.lane;
      const int row = p / 8, k = b * kBlocksK + 16 * ((p % 8) ^ Wide::swizzle(row));
      const unsigned src = k < e.D ? (unsigned)row * (unsigned)e.D + (unsigned)k : 0xfffffff0u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)(weights + first), 16,
                                               src, 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < kWideTiles; ++t) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = b * kBlocksK + 64 * q + 16 * e.h;
        raw[t][q] = i32x4{0, 0, 0, 0};
        if (k < e.D) raw[t][q] = *reinterpret_cast<const i32x4 *>(x[t] + k);
      }
      raw_scale[t] = xs[t][b];
    }
  }

  __device__ __forceinline__ void run(int b, const i32x4 *weights, i32x4 *next) {
    const float sw = e.ws[(int64_t)(v0 / kBlocksK) * nblocks + b];
    bf16x8 xw[kWideTiles][4];
    float scale[kWideTiles];
#pragma unroll
    for (int t = 0; t < kWideTiles; ++t) {
      scale[t] = raw_scale[t] * sw;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        xw[t][2 * q] = widen(raw[t][q][0], raw[t][q][1]);
        xw[t][2 * q + 1] = widen(raw[t][q][2], raw[t][q][3]);
      }
    }
    if (b + 1 < nblocks) load(b + 1, next);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      i32x4 d[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) d[q] = weights[e.at[g % kSubs][q][0] + (g / kSubs) * (16 * kSubs) * 8];
      f32x4 p[kWideTiles];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 wf = i & 1 ? widen(d[i / 2][2], d[i / 2][3]) : widen(d[i / 2][0], d[i / 2][1]);
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < kWideTiles; ++t)
          p[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xw[t][i], i == 0 ? zero : p[t], 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < kWideTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][t][i] = __builtin_fmaf(p[t][i], scale[t], acc[g][t][i]);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // the next step's loads; the other counters free
    lds_barrier();
  }
};

template <class T, int COLS, bool ALIGNED, bool DEN>
__global__ __launch_bounds__(kBlock, COLS == 64 ? 3 : 2) void project_blocks_deep_kernel(
    const unsigned char *__restrict__ x, const float *__restrict__ xs, const unsigned char *__restrict__ w,
    const float *__restrict__ ws, const float *__restrict__ bias, int64_t rows, int D, int V, int chunks,
    void *__restrict__ logits, float *__restrict__ den, LogSum *__restrict__ parts) {
  typedef DeepProject<T, COLS, ALIGNED, DEN> P;
  typedef typename P::Wide E;
  __shared__ __attribute__((aligned(16))) typename P::Weights s_w0, s_w1;
  const int64_t id = (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
  // an eighth of the tiles for each XCD, in order: chunk by chunk of a group of rows
  const int64_t tiles = (rows + kWideRows - 1) / kWideRows * chunks, share = (tiles + 7) / 8;
  const int64_t tile = (id & 7) * share + (id >> 3);
  if ((id >> 3) >= share || tile >= tiles) return;
  const int64_t group0 = tile / chunks * kWideRows;
  const int chunk = (int)(tile % chunks);
  P p;
  p.e.w = w;
  p.e.ws = ws;
  p.e.D = D;
  p.e.V = V;
  p.e.lane = threadIdx.x & 63;
  p.e.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = p.e.r = p.e.lane & 15, h = p.e.h = p.e.lane >> 4;
  p.v0 = chunk * COLS;
  p.nblocks = (D + kBlocksK - 1) / kBlocksK;
  const int64_t row0 = group0 + p.e.wave * (16 * kWideTiles);
#pragma unroll
  for (int t = 0; t < kWideTiles; ++t) {
    const int64_t row = min(row0 + 16 * t + r, rows - 1);
    p.x[t] = x + row * D;
    p.xs[t] = xs + row * p.nblocks;
    p.e.ref[t] = -kLargest;
    p.e.sum[t] = 0.f;
  }
  p.load(0, s_w0);
  // sums start from the bias
#pragma unroll
  for (int g = 0; g < P::kGroups; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int v = p.v0 + E::entry(g, 4 * h + i);
      const float b = bias && v < V ? bias[v] : 0.f;
#pragma unroll
      for (int t = 0; t < kWideTiles; ++t) p.acc[g][t][i] = b;
    }
#pragma unroll
  for (int sub = 0; sub < P::kSubs; ++sub)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int row = E::entry(sub, r);
      p.e.at[sub][q][0] = row * 8 + ((4 * q + h) ^ E::swizzle(row));
    }
  p.e.out_base = static_cast<char *>(logits) + group0 * V * E::kOut;
  p.e.rows_in = row0 + 16 * kWideTiles <= rows;
  p.e.out = make_buffer(p.e.out_base,
                        (unsigned)min((int64_t)kWideRows, rows - group0) * (unsigned)V * E::kOut);
  p.e.out_row = ((unsigned)(p.e.wave * (16 * kWideTiles) + r) * (unsigned)V + (unsigned)(E::kGroup * h)) * E::kOut;
  p.e.out_tile = 16u * (unsigned)V * E::kOut;
  __builtin_amdgcn_s_waitcnt(0x0f70);
  lds_barrier();
  for (int b = 0;;) {
    p.run(b, s_w0, s_w1);
    if (++b == p.nblocks) break;
    p.run(b, s_w1, s_w0);
    if (++b == p.nblocks) break;
  }
#pragma unroll
  for (int set = 0; set < P::kGroups / P::kSubs; ++set) {
    f32x4 a[P::kSubs][kWideTiles];
#pragma unroll
    for (int sub = 0; sub < P::kSubs; ++sub)
#pragma unroll
      for (int t = 0; t < kWideTiles; ++t) a[sub][t] = p.acc[set * P::kSubs + sub][t];
    p.e.finish(p.v0, set, a);
  }
  if constexpr (DEN) p.e.finish_den(row0, rows, chunk, chunks, den, parts);
}

// den[r] = log-sum-exp of a row's parts: 16 lanes a row, merged in a fixed order
__global__ __launch_bounds__(kBlock) void project_blocks_den_kernel(const LogSum *__restrict__ parts,
                                                                   int nparts, int64_t rows,
                                                                   float *__restrict__ den) {
  for (int64_t r0 = (int64_t)blockIdx.x * (kBlock / 16); r0 < rows; r0 += (int64_t)gridDim.x * (kBlock / 16)) {
    const int64_t r = r0 + threadIdx.x / 16;
    LogSum t = {OT_NEG_INF, 0.f};
    if (r < rows)
      for (int k = threadIdx.x % 16; k < nparts; k += 16) t = merge(t, parts[r * nparts + k]);
#pragma unroll
    for (int d = 1; d < 16; d *= 2) t = merge(t, {__shfl_xor(t.m, d, kWave), __shfl_xor(t.s, d, kWave)});
    if (threadIdx.x % 16 == 0 && r < rows) den[r] = logf(t.s) + (__builtin_isinf(t.m) ? 0.f : t.m);
  }
}

static void launch_den(const LogSum *parts, int nparts, int64_t rows, float *den, hipStream_t s) {
  const int64_t groups = (rows + kBlock / 16 - 1) / (kBlock / 16);
  hipLaunchKernelGGL(project_blocks_den_kernel, dim3((unsigned)(groups < (1 << 20) ? groups : (1 << 20))),
                     dim3(kBlock), 0, s, parts, nparts, rows, den);
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

template <class T, int KB>
static int launch_project_blocks_wide(const unsigned char *x, const float *xs, const unsigned char *w,
                                      const float *ws, const float *bias, int64_t rows, int32_t D, int32_t V,
                                      void *logits, float *den, LogSum *parts, int cus, hipStream_t s) {
  const ProjectGrid g((rows + kWideRows - 1) / kWideRows, (V + kWideCols - 1) / kWideCols, 2 * (int64_t)cus);
  const bool merged = den && g.nparts > 1;
#define OT_WIDE(ALIGNED_)                                                                                 \
  if (den)                                                                                                \
    hipLaunchKernelGGL((project_blocks_wide_kernel<T, KB, ALIGNED_, true>), g.grid, dim3(kBlock), 0, \
                       s, x, xs, w, ws, bias, rows, D, V, g.stages_per_part, logits,                      \
                       merged ? nullptr : den, merged ? parts : nullptr);                                 \
  else                                                                                                    \
    hipLaunchKernelGGL((project_blocks_wide_kernel<T, KB, ALIGNED_, false>), g.grid, dim3(kBlock), 0, \
                       s, x, xs, w, ws, bias, rows, D, V, g.stages_per_part, logits, (float *)nullptr,    \
                       (LogSum *)nullptr)
  if (sizeof(T) == 4 || (V % 2 == 0 && (reinterpret_cast<uintptr_t>(logits) & 3) == 0)) {
    OT_WIDE(true);
  } else if constexpr (sizeof(T) != 4) {
    OT_WIDE(false);
  }
#undef OT_WIDE
  if (merged) launch_den(parts, g.nparts, rows, den, s);
  return (int)hipGetLastError();
}

template <class T, int COLS>
static int launch_project_blocks_deep(const unsigned char *x, const float *xs, const unsigned char *w,
                                      const float *ws, const float *bias, int64_t rows, int32_t D, int32_t V,
                                      void *logits, float *den, LogSum *parts, hipStream_t s) {
  const int chunks = (V + COLS - 1) / COLS;
  const int64_t tiles = (rows + kWideRows - 1) / kWideRows * chunks, groups = (tiles + 7) / 8 * 8;
  // (a launch holds 2^32 threads at most in each direction; a multiple of 8 keeps the ids' order)
  constexpr int64_t kMostX = 1 << 20;
  const dim3 grid((unsigned)(groups < kMostX ? groups : kMostX), 1, (unsigned)((groups + kMostX - 1) / kMostX));
  const bool merged = den && chunks > 1;
#define OT_DEEP(ALIGNED_)                                                                                     \
  if (den)                                                                                                    \
    hipLaunchKernelGGL((project_blocks_deep_kernel<T, COLS, ALIGNED_, true>), grid, dim3(kBlock), 0, s, x, xs, w, ws, \
                       bias, rows, D, V, chunks, logits, merged ? nullptr : den, merged ? parts : nullptr);   \
  else                                                                                                        \
    hipLaunchKernelGGL((project_blocks_deep_kernel<T, COLS, ALIGNED_, false>), grid, dim3(kBlock), 0, s, x, xs, w,  \
                       ws, bias, rows, D, V, chunks, logits, (float *)nullptr, (LogSum *)nullptr)
  if (sizeof(T) == 4 || (V % 2 == 0 && (reinterpret_cast<uintptr_t>(logits) & 3) == 0)) {
    OT_DEEP(true);
  } else if constexpr (sizeof(T) != 4) {
    OT_DEEP(false);
  }
#undef OT_DEEP
  if (merged) launch_den(parts, chunks, rows, den, s);
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
  const int col_tiles = (V + kSmallCols - 1) / kSmallCols;
  const int64_t tiles = (rows + 15) / 16 * col_tiles;
  // The small kernel spreads over the chip what the others would do on a few compute units, but
  // reads its operands again for every 16 x 64 logits.  Microseconds with denominators, small
  // against wide or deep, by its workgroups (256 compute units):
  //   D = 512:  32 x 5000 (158) 11 : 13, 512 x 500 (256) 10 : 12, 64 x 5000 (316) 14 : 13,
  //             1024 x 500 (512) 13 : 12, 128 x 5000 (632) 16 : 14
  //   D = 1008: 32 x 5000 (158) 12 : 15, 64 x 5000 (316) 14 : 16, 768 x 500 (384) 13 : 15,
  //             128 x 5000 (632) 20 : 16, 512 x 5000 (2528) 46 : 22;  D = 1024: 32 x 16384 (512) 24 : 21
  //   D = 2048: 32 x 5000 (158) 19 : 22, 512 x 500 (256) 17 : 25, 64 x 5000 (316) 28 : 22,
  //             640 x 500 (320) 26 : 25, 4096 x 500 (2048) 90 : 27;  D = 4096: 512 x 500 (256) 26 : 43
  const bool few = 2 * tiles <= (nblocks <= 8 ? 3 : 2) * (int64_t)cus;
  // (wide and deep address a workgroup's logits, and deep its weights, with 32 bits)
  if (!few && V < (1 << 21) && D < (1 << 24)) {
#define OT_PROJECT_WIDE(KB_) \
  return launch_project_blocks_wide<T, KB_>(x, xs, w, ws, bias, rows, D, V, logits, den, parts, cus, s)
    // us by the wide kernel and by the deep one: 1024 x 512 x 500 bfloat16 11.6 and 11.3, 8000 x 512 x 500
    // 18 and 15, 100 000 x 512 x 500 83 and 99, 751 992 x 512 x 500 511 and 723, 751 992 x 128 x 500 324 and
    // 457; float32 2000 x 512 x 5000 27 and 30, 100 000 x 384 x 1001 184 and 201
    if (nblocks == 1) OT_PROJECT_WIDE(1);
    if (nblocks == 2) OT_PROJECT_WIDE(2);
    if (nblocks == 3) OT_PROJECT_WIDE(3);
    if (nblocks == 4) OT_PROJECT_WIDE(4);
#undef OT_PROJECT_WIDE
    // 64 entries a workgroup where 128 would give fewer than two rounds on every compute unit: us with
    // 64 and 128, by the workgroups of 128 entries: 2100 x 640 x 1001 (136) 16 and 18, 600 x 1536 x
    // 8000 (315) 42 and 43, 1003 x 1008 x 4998 (320) 32 and 36; 8000 x 2048 x 5000 (2520) 278 and 214,
    // 30 000 x 4096 x 500 (940) 211 and 164
    const int64_t groups = (rows + kWideRows - 1) / kWideRows * ((V + 127) / 128);
    return groups < 2 * (int64_t)cus
               ? launch_project_blocks_deep<T, 64>(x, xs, w, ws, bias, rows, D, V, logits, den, parts, s)
               : launch_project_blocks_deep<T, 128>(x, xs, w, ws, bias, rows, D, V, logits, den, parts, s);
  }
  const dim3 grid((unsigned)(tiles < (1 << 22) ? tiles : (1 << 22)));
  hipLaunchKernelGGL((project_blocks_small_kernel<T>), grid, dim3(kBlock), 0, s, x, xs, w, ws, bias, rows, D,
                     V, col_tiles, tiles, logits, den ? parts : nullptr);
  if (den) launch_den(parts, col_tiles, rows, den, s);
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
