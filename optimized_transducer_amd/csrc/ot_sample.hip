// A symbol drawn from each row of logits (gfx950).
//
// For a row x with largest entry m, temperature T > 0 and a given number u of [0, 1):
//   weights   w_i = exp((x_i - m) / T), 0 for x_i = -inf
//   order     larger values first, equal values by lower index
//   top_k     the first top_k entries of that order remain (0: all)
//   top_p     of those, an entry remains if the weights in front of it sum to less than
//             top_p times the sum of all of them (the first one always remains)
//   min_p     of those, an entry remains if w_i >= min_p
//   symbol    the first index, in index order, whose running sum of remaining weights
//             exceeds u times their total; log_prob = log(w_symbol / total)
// T = 0: the first of the largest entries, log_prob 0.  A row with no largest finite entry
// (all -inf, a NaN, +inf) has symbol -1, log_prob -inf; so has u = NaN.
//
// Which index a symbol falls on hangs on the last bits of a running sum, so weights and sums
// are held in 64 bits.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ot_device.hip.h"
#include "ot_transducer.h"

namespace ot {

// settings of a call: a value for all rows, or one per row
struct SampleSettings {
  const float *temperature, *top_p, *min_p;
  const int32_t *top_k;
  float temperature_value, top_p_value, min_p_value;
  int32_t top_k_value;
};

// unsigned integers that order like the values (both zeros alike)
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

template <class V, class Op>
__device__ __forceinline__ V block_reduce(V v, Op op, V *s) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v = op(v, __shfl_xor(v, d, kWave));
  __syncthreads();  // the previous use of s has been read
  if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int k = 1; k < kWavesPerBlock; ++k) v = op(v, s[k]);
  return v;
}

// sum of v over the threads up to and including this one; *total: over all
template <class V>
__device__ __forceinline__ V block_scan(V v, V *s, V *total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const V up = __shfl_up(v, d, kWave);
    if (lane >= d) v += up;
  }
  __syncthreads();
  if (lane == kWave - 1) s[wave] = v;
  __syncthreads();
  V before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kWavesPerBlock; ++k) {
    if (k < wave) before += s[k];
    all += s[k];
  }
  *total = all;
  return before + v;
}

// A workgroup per row; every step reads the row again.
template <class T>
__global__ __launch_bounds__(kBlock) void sample_row_kernel(const void *__restrict__ logits, int64_t row_stride,
                                                            int64_t rows, int V,
                                                            const float *__restrict__ uniform,
                                                            SampleSettings set, int32_t *__restrict__ symbols,
                                                            float *__restrict__ log_probs) {
  __shared__ unsigned s_u[kWavesPerBlock];
  __shared__ int s_i[kWavesPerBlock];
  __shared__ double s_d[kWavesPerBlock];
  auto max_u = [](unsigned a, unsigned b) { return max(a, b); };
  auto min_i = [](int a, int b) { return min(a, b); };
  auto sum_i = [](int a, int b) { return a + b; };
  auto sum_d = [](double a, double b) { return a + b; };
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * row_stride;
    const float temperature = set.temperature ? set.temperature[row] : set.temperature_value;
    const float top_p = set.top_p ? set.top_p[row] : set.top_p_value;
    const float min_p_row = set.min_p ? set.min_p[row] : set.min_p_value;
    const double min_p = min_p_row > 0.f ? fminf(min_p_row, 1.f) : 0.f;
    const int top_k = set.top_k ? set.top_k[row] : set.top_k_value;
    const double u = uniform[row];
    auto at = [&](int i) { return load_element<T>(logits, base + i); };

    // largest entry; a NaN outranks everything
    unsigned key = 0;
    for (int i = tid; i < V; i += kBlock) {
      const float x = at(i);
      key = max(key, x != x ? 0xffffffffu : order_key(x));
    }
    const unsigned top_key = block_reduce(key, max_u, s_u);
    constexpr unsigned kNegInfKey = 0x007fffffu, kPosInfKey = 0xff800000u;
    if (top_key <= kNegInfKey || top_key >= kPosInfKey || u != u) {
      if (tid == 0) {
        symbols[row] = -1;
        log_probs[row] = OT_NEG_INF;
      }
      continue;
    }
    if (!(temperature > 0.f)) {
      int first = V;
      for (int i = tid; i < V; i += kBlock)
        if (first == V && order_key(at(i)) == top_key) first = i;
      first = block_reduce(first, min_i, s_i);
      if (tid == 0) {
        symbols[row] = first;
        log_probs[row] = 0.f;
      }
      continue;
    }
    const double m = __builtin_bit_cast(float, top_key ^ ((top_key >> 31) ? 0x80000000u : 0xffffffffu));
    const double T_ = temperature;
    auto weight = [&](float x) { return x == OT_NEG_INF ? 0.0 : exp(((double)x - m) / T_); };

    // Remaining entries: those with a key above `cut`, and the first `ties` of those at it.
    unsigned cut = 0;
    int ties = V;
    if (top_k > 0 && top_k < V) {
      // the largest key that top_k entries reach, bit by bit
      unsigned k = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const unsigned t = k | (1u << bit);
        int n = 0;
        for (int i = tid; i < V; i += kBlock) n += order_key(at(i)) >= t;
        if (block_reduce(n, sum_i, s_i) >= top_k) k = t;
      }
      int above = 0;
      for (int i = tid; i < V; i += kBlock) above += order_key(at(i)) > k;
      cut = k;
      ties = top_k - block_reduce(above, sum_i, s_i);
    }
    if (top_p < 1.f) {
      const double w_cut = weight(__builtin_bit_cast(float, cut ^ ((cut >> 31) ? 0x80000000u : 0xffffffffu)));
      double sum = 0.0;
      int at_cut = 0;
      for (int i = tid; i < V; i += kBlock) {
        const float x = at(i);
        const unsigned q = order_key(x);
        if (q > cut) sum += weight(x);
        at_cut += q == cut;
      }
      const int limit = min(ties, block_reduce(at_cut, sum_i, s_i));
      const double above_cut = block_reduce(sum, sum_d, s_d);
      const double want = (double)top_p * (above_cut + (limit > 0 ? limit * w_cut : 0.0));
      // the largest key above `cut` whose entries and those above reach `want`; none: `cut`
      unsigned k = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const unsigned t = k | (1u << bit);
        if (t <= cut) {
          k = t;  // all of them reach it
          continue;
        }
        sum = 0.0;
        for (int i = tid; i < V; i += kBlock) {
          const float x = at(i);
          if (order_key(x) >= t) sum += weight(x);
        }
        if (block_reduce(sum, sum_d, s_d) >= want && t <= top_key) k = t;
      }
      if (k < cut) k = cut;
      const float xk = __builtin_bit_cast(float, k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
      const double wk = weight(xk);
      sum = 0.0;
      at_cut = 0;
      for (int i = tid; i < V; i += kBlock) {
        const float x = at(i);
        const unsigned q = order_key(x);
        if (q > k) sum += weight(x);
        at_cut += q == k;
      }
      at_cut = block_reduce(at_cut, sum_i, s_i);
      sum = block_reduce(sum, sum_d, s_d);
      if (k == cut) at_cut = min(at_cut, ties);
      // entry number j of the ties remains if sum + j * wk < want
      int n = at_cut;
      if (wk > 0.0) {
        const double q = ceil((want - sum) / wk);
        n = q < 1.0 ? 0 : q < at_cut ? (int)q : at_cut;
      }
      if (k == top_key) n = max(n, 1);
      cut = k;
      ties = n;
    }

    // total of the remaining weights, then the index where the running sum passes u times it.
    // Thread t holds entry t of a run of 256; ties count along the way.
    double total = 0.0, target = 0.0;
    int symbol = -1, last = -1;
    for (int pass = 0; pass < 2; ++pass) {
      double run = 0.0;
      int seen = 0;
      for (int i0 = 0; i0 < V; i0 += kBlock) {
        const int i = i0 + tid;
        float x = i < V ? at(i) : OT_NEG_INF;
        const unsigned q = order_key(x);
        int tie_total;
        const int tie = block_scan(i < V && q == cut ? 1 : 0, s_i, &tie_total);
        const bool remains = i < V && (q > cut || (q == cut && seen + tie <= ties));
        double w = remains ? weight(x) : 0.0;
        if (!(w >= min_p)) w = 0.0;
        seen += tie_total;
        double sum;
        const double upto = run + block_scan(w, s_d, &sum);
        if (pass == 1) {
          const int hit = block_reduce(upto > target && w > 0.0 ? i : V, min_i, s_i);
          const int any = block_reduce(w > 0.0 ? i : -1, [](int a, int b) { return max(a, b); }, s_i);
          if (any >= 0) last = any;
          if (hit < V) {
            symbol = hit;
            break;
          }
        }
        run += sum;
      }
      if (pass == 0) {
        total = run;
        target = u * total;
      }
    }
    if (symbol < 0) symbol = last;  // u >= 1, or a sum that rounds to it
    if (tid == 0) {
      symbols[row] = symbol;
      log_probs[row] = (float)(((double)at(symbol) - m) / T_ - log(total));
    }
  }
}

template <class T>
static int launch_sample(const void *logits, int64_t row_stride, int64_t rows, int32_t V, const float *uniform,
                         const SampleSettings &set, int32_t *symbols, float *log_probs, hipStream_t s) {
  const dim3 grid((unsigned)(rows < (1 << 20) ? rows : (1 << 20)));
  hipLaunchKernelGGL((sample_row_kernel<T>), grid, dim3(kBlock), 0, s, logits, row_stride, rows, V, uniform, set,
                     symbols, log_probs);
  return (int)hipGetLastError();
}

}  // namespace ot

using namespace ot;

extern "C" int ot_sample_symbols(const void *logits, int32_t dtype, int64_t row_stride, int64_t rows, int32_t V,
                                 const float *uniform, const float *temperature, float temperature_value,
                                 const int32_t *top_k, int32_t top_k_value, const float *top_p,
                                 float top_p_value, const float *min_p, float min_p_value, int32_t *symbols,
                                 float *log_probs, void *stream) {
  if (rows == 0) return 0;
  if (!logits || !uniform || !symbols || !log_probs || rows < 0 || rows > INT32_MAX || V <= 0 ||
      V > INT32_MAX - 4096 || row_stride < 0)
    return OT_E_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(logits) & (dtype == OT_DTYPE_F32 ? 3 : 1)) ||
      (reinterpret_cast<uintptr_t>(uniform) & 3) || (reinterpret_cast<uintptr_t>(temperature) & 3) ||
      (reinterpret_cast<uintptr_t>(top_k) & 3) || (reinterpret_cast<uintptr_t>(top_p) & 3) ||
      (reinterpret_cast<uintptr_t>(min_p) & 3) || (reinterpret_cast<uintptr_t>(symbols) & 3) ||
      (reinterpret_cast<uintptr_t>(log_probs) & 3))
    return OT_E_MISALIGNED;
  const SampleSettings set = {temperature, top_p,       min_p,       top_k,
                              temperature_value, top_p_value, min_p_value, top_k_value};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == OT_DTYPE_F32) return launch_sample<float>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, s);
  if (dtype == OT_DTYPE_F16) return launch_sample<F16>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, s);
  if (dtype == OT_DTYPE_BF16) return launch_sample<BF16>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, s);
  return OT_E_BAD_ARG;
}
