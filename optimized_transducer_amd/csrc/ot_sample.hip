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
// Which index a symbol falls on, or where top_p cuts, hangs on the last bits of a sum: weights
// and sums are 64-bit.  This chip's vector units do 64-bit multiply-adds at the rate of
// (unpacked) 32-bit ones, so a weight costs 19 such instructions (a range reduction and a
// polynomial for 2^f) where a 32-bit one through the hardware's 2^x costs 8 and the transcendental
// unit.  A sum over lanes is never recovered from a difference, and a lane without a weight is never
// drawn from: its sum may be a rounding larger than its neighbour's.
//
// How the cuts are found: a wave that holds its row sorts it and reads both of them off the order
// (32 x 512 float32, settings per row, 6.3 us, 11.7 by histograms).  Longer rows are not sorted: a
// histogram of 256 bins finds the one that top_p's cut falls into, and only its entries are; for
// top_k, and where such a bin holds too many, the interval that still holds the cut is divided
// again, until one value is left or few enough entries are.
//
// Who works on a row (what bounds it; times at T = 1 and sigma 2):
//   a wave                short rows, up to 512 (float32) or 1024 elements, in registers, and no
//                         barrier.  Without cuts a wave takes a batch of them: vector instructions
//                         bound it, 44 per weight, 91 % of the cycles (751 992 x 500 float32 0.51 ms,
//                         2.9 TB/s)
//   4, 8 or 16 waves      rows up to 16384, in registers; of all the waves only the wide steps
//                         profit, so that the barriers and scans of the cuts bound it.  A top_k of
//                         512 at most is found by all of them, and one wave goes on with what is left
//                         (20 011 x 5000 float16 with all cuts 0.41 ms, 0.94 with all waves to the end)
//   slices                longer rows, several workgroups each (64 x 131 072 bfloat16, top_p: 69 us,
//                         266 by a workgroup per row; launches and the chain of steps bound it)
//   16 waves              rows beyond the slices, or with top_k: they read the row in every step,
//                         served by the caches
// Every wave owns a contiguous part of the row, so that a running sum needs one number from each
// wave.
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

constexpr int kSampleBins = 256;
// Entries that one wave takes over from the others.  us with 256, 512 and 1024: 4096 x 5000 float16 with
// top_k 200 and the other cuts 80, 85, 97, top_k 250 97, 86, 97, top_k 400 182, 86, 98, top_k 700 187, 188,
// 99; 64 x 2000 float32 with top_k 50 7.6, 8.6, 11.2
constexpr int kSampleFew = 512;
constexpr float kInf = __builtin_huge_valf();

// ---- wave-wide helpers ----------------------------------------------------------------------

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
  const int64_t b = __builtin_bit_cast(int64_t, v);
  const unsigned lo = (unsigned)dpp_or_zero<CTRL, ROWS>((int)b);
  const unsigned hi = (unsigned)dpp_or_zero<CTRL, ROWS>((int)(b >> 32));
  return __builtin_bit_cast(double, (int64_t)lo | ((int64_t)hi << 32));
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  const int64_t b = __builtin_bit_cast(int64_t, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)b, lane);
  const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __builtin_bit_cast(double, (int64_t)lo | ((int64_t)hi << 32));
}

// sum over the lanes up to and including this one: inside rows of 16 lanes (row_shr), then the
// last lane of a row to the next one (row_bcast)
template <class N>
__device__ __forceinline__ N wave_scan(N v) {
  v += dpp_or_zero<0x111, 0xf>(v);
  v += dpp_or_zero<0x112, 0xf>(v);
  v += dpp_or_zero<0x114, 0xf>(v);
  v += dpp_or_zero<0x118, 0xf>(v);
  v += dpp_or_zero<0x142, 0xa>(v);
  v += dpp_or_zero<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) { return lane_value(wave_scan(v), kWave - 1); }
__device__ __forceinline__ int wave_sum(int v) { return lane_value(wave_scan(v), kWave - 1); }

// the value of lane ^ X, X = 2^n - 1 or 2^n
template <int CTRL>
__device__ __forceinline__ float dpp_value(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int X>
__device__ __forceinline__ float lane_xor(float v) {
  if constexpr (X == 1) return dpp_value<kDppQuadXor1>(v);
  else if constexpr (X == 2) return dpp_value<kDppQuadXor2>(v);
  else if constexpr (X == 3) return dpp_value<0x1b>(v);                       // quad_perm 3 2 1 0
  else if constexpr (X == 4) return dpp_value<0x1b>(dpp_value<kDppRowHalfMirror>(v));
  else if constexpr (X == 7) return dpp_value<kDppRowHalfMirror>(v);
  else if constexpr (X == 8) return dpp_value<0x128>(v);                      // row_ror 8
  else if constexpr (X == 15) return dpp_value<kDppRowMirror>(v);
  else return __shfl_xor(v, X, kWave);
}

// Sorts the 64 * N values of a wave, larger ones first; value i of lane l ends as number l * N + i.
// A bitonic network whose merges start by comparing a block with its mirror image, so that the lower
// place always takes the larger value: within a lane a maximum and a minimum, between lanes the
// median of the two values and an infinity of the lane's side.
template <int N>
__device__ __forceinline__ void sort_in_lane(float (&v)[N], int stride) {
#pragma unroll
  for (int d = stride; d > 0; d /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!(i & d)) {
        const float a = v[i], b = v[i | d];
        v[i] = fmaxf(a, b);
        v[i | d] = fminf(a, b);
      }
}
template <int X, int N>
__device__ __forceinline__ void sort_lanes(float (&v)[N], int lane, bool mirror) {
  // (lower half of the compared pair: the bit of the lane that X's highest one is)
  constexpr int kTop = X & ~(X >> 1);
  const float side = lane & kTop ? OT_NEG_INF : kInf;
  float other[N];
#pragma unroll
  for (int i = 0; i < N; ++i) other[i] = lane_xor<X>(v[mirror ? N - 1 - i : i]);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __builtin_amdgcn_fmed3f(v[i], other[i], side);
}
template <int N>
__device__ __forceinline__ void wave_sort(float (&v)[N], int lane) {
#pragma unroll
  for (int size = 2; size <= N; size *= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = i ^ (size - 1);
      if (i < j) {
        const float a = v[i], b = v[j];
        v[i] = fmaxf(a, b);
        v[j] = fminf(a, b);
      }
    }
    sort_in_lane(v, size / 4);
  }
  sort_lanes<1>(v, lane, true);
  sort_in_lane(v, N / 2);
  sort_lanes<3>(v, lane, true);
  sort_lanes<1>(v, lane, false);
  sort_in_lane(v, N / 2);
  sort_lanes<7>(v, lane, true);
  sort_lanes<2>(v, lane, false);
  sort_lanes<1>(v, lane, false);
  sort_in_lane(v, N / 2);
  sort_lanes<15>(v, lane, true);
  sort_lanes<4>(v, lane, false);
  sort_lanes<2>(v, lane, false);
  sort_lanes<1>(v, lane, false);
  sort_in_lane(v, N / 2);
  sort_lanes<31>(v, lane, true);
  sort_lanes<8>(v, lane, false);
  sort_lanes<4>(v, lane, false);
  sort_lanes<2>(v, lane, false);
  sort_lanes<1>(v, lane, false);
  sort_in_lane(v, N / 2);
  sort_lanes<63>(v, lane, true);
  sort_lanes<16>(v, lane, false);
  sort_lanes<8>(v, lane, false);
  sort_lanes<4>(v, lane, false);
  sort_lanes<2>(v, lane, false);
  sort_lanes<1>(v, lane, false);
  sort_in_lane(v, N / 2);
}

// ---- the threads that share a row -----------------------------------------------------------

template <int WAVES>
struct SampleShared {
  // (one wave that holds its row sorts it instead)
  unsigned bins[WAVES > 1 ? kSampleBins : 1];
  float few[WAVES > 1 ? kSampleFew : 1];  // entries of one bin
  double sum[WAVES];
  float value[2][WAVES];
  int count[WAVES];
  int index;
};

template <int WAVES>
struct RowGroup {
  SampleShared<WAVES> &s;
  int lane, wave;

  __device__ __forceinline__ int thread() const { return wave * kWave + lane; }
  __device__ __forceinline__ void sync() const {
    if constexpr (WAVES == 1) {
      // one wave: LDS operations of a wave run in order
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else {
      __syncthreads();
    }
  }
  // the largest hi and the smallest lo
  __device__ __forceinline__ void extremes(float &hi, float &lo) const {
    hi = group_allreduce<kWave>(hi, MaxOp());
    lo = -group_allreduce<kWave>(-lo, MaxOp());
    if constexpr (WAVES > 1) {
      sync();
      if (lane == 0) {
        s.value[0][wave] = hi;
        s.value[1][wave] = lo;
      }
      sync();
#pragma unroll
      for (int k = 0; k < WAVES; ++k) {
        hi = fmaxf(hi, s.value[0][k]);
        lo = fminf(lo, s.value[1][k]);
      }
    }
  }
  // totals of a sum and a count, the same bits in every thread
  __device__ __forceinline__ void totals(double &sum, int &count) const {
    gather(wave_sum(sum), wave_sum(count), sum, count);
  }
  // the same from every wave's part
  __device__ __forceinline__ void gather(double part, int part_count, double &sum, int &count) const {
    sum = part;
    count = part_count;
    if constexpr (WAVES > 1) {
      sync();
      if (lane == 0) {
        s.sum[wave] = part;
        s.count[wave] = part_count;
      }
      sync();
      sum = 0.0;
      count = 0;
#pragma unroll
      for (int k = 0; k < WAVES; ++k) {
        sum += s.sum[k];
        count += s.count[k];
      }
    }
  }
};

// elements per 16-byte load
template <class T> constexpr int kSampleVec = sizeof(T) == 4 ? 4 : 8;

// elements [i, i + VEC) of a row of V; those past the end are -inf
template <class T>
__device__ __forceinline__ void load_logits(const void *row, int i, int V, float x[]) {
  constexpr int VEC = kSampleVec<T>;
  if (i + VEC <= V) {
    // the row may start anywhere its type can
    if constexpr (VEC == 4) {
      typedef f32x4 unaligned __attribute__((aligned(4)));
      const f32x4 v = *reinterpret_cast<const unaligned *>(static_cast<const float *>(row) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = v[e];
    } else {
      typedef u32x4 unaligned __attribute__((aligned(2)));
      const u32x4 v = *reinterpret_cast<const unaligned *>(static_cast<const unsigned short *>(row) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned w = v[e];
        x[2 * e] = to_float<T>((unsigned short)(w & 0xffffu));
        x[2 * e + 1] = to_float<T>((unsigned short)(w >> 16));
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = i + e < V ? load_element<T>(row, i + e) : OT_NEG_INF;
  }
}

// Coefficients of f^11 down to f in 2^f = 1 + f * q(f): q interpolates (2^f - 1) / f at the 11 Chebyshev
// nodes of [-1/2, 1/2].  Read once into scalar registers, where literals would be moved into vector
// registers in front of every use.
constexpr int kExpTerms = 11;
__constant__ double kExpSeries[kExpTerms] = {
    4.4549605981865186e-10, 7.0725859492692234e-09, 1.0178062445845774e-07, 1.3215442587921689e-06,
    1.5252733829836119e-05, 1.5403530441736050e-04, 1.3333558146416936e-03, 9.6181291076068882e-03,
    5.5504108664821597e-02, 2.4022650695910097e-01, 6.9314718055994529e-01};

// 2^t, t >= -1100, as 2^n * 2^f with n the nearest integer to t and 2^f the polynomial above for
// |f| <= 1/2: within 1.4e-16 = 2^-52.7 of it over 4e7 values of f (the exponential series needs the
// 13th power for that: 751 992 x 500 float32 524 us and 502 so)
__device__ __forceinline__ double power_of_2(double t) {
  const double n = __builtin_rint(t), f = t - n;
  double p = kExpSeries[0];
#pragma unroll
  for (int k = 1; k < kExpTerms; ++k) p = __builtin_fma(p, f, kExpSeries[k]);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// exp((x - m) / T) = 2^((x - m) * c), c = log2(e) / T.  The exponent has three roundings, so a weight is
// within (|(x - m) / T| + 1) * 2^-51.  Exactly 1 at x = m, exactly 0 at x = -inf.
struct Weight {
  double m, c;
  __device__ __forceinline__ Weight(float m_, float T) : m(m_), c(1.4426950408889634074 / (double)T) {}
  __device__ __forceinline__ double operator()(float x) const {
    // (T = inf and x = -inf make a NaN of the product, which fmax drops)
    return power_of_2(__builtin_fmax(((double)x - m) * c, -1100.0));
  }
};

// unsigned integers that order like the values (both zeros alike)
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float key_value(unsigned key) {
  return __builtin_bit_cast(float, key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// one row's answer
struct Drawn {
  int symbol;
  float log_prob;
};

// (x - m) / T - log(total) in 64 bits, rounded once; c = log2(e) / T, total >= 1.  With b the hardware's
// log2 of 32 bits, total * 2^-b = 1 + q and log(total) = b ln 2 + q - q^2 / 2: |q| < 2^-18, and what is left
// out is below 2^-55.  The polynomial of the weights serves again (the library's logarithm keeps 12 more
// registers of constants over a kernel's loop: 751 992 x 500 float32 519 us and 504 so, 4096 x 16 000 with
// top_p 712 and 629)
__device__ __forceinline__ float log_probability(float logit, float m, double c, double total) {
  const double b = __builtin_amdgcn_logf((float)total), q = __builtin_fma(total, power_of_2(-b), -1.0);
  return (float)((((double)logit - m) * c - b) * 0.69314718055994531 - (q - 0.5 * q * q));
}

// Draws from a row with a finite largest entry m at a temperature above 0.  Every thread of the
// group calls it with the same arguments and gets the same answer.
//   CHUNKS > 0: wave w holds elements [w * CHUNKS * 64 * VEC, + CHUNKS * 64 * VEC) in x, chunk by
//     chunk, lane by lane (VEC consecutive ones each); excluded entries become -inf there
//   CHUNKS = 0: the row is read from memory in every step; `per_wave` chunks per wave
template <class T, int WAVES, int CHUNKS>
struct Sampler {
  static constexpr int VEC = kSampleVec<T>;
  static constexpr bool kHeld = CHUNKS > 0;
  static constexpr bool kHeldWeights = kHeld && CHUNKS * VEC <= 24;  // else formed anew in each step

  const RowGroup<WAVES> &g;
  const void *row;
  const int V, per_wave;
  const float m;
  const Weight weight;
  float (&x)[kHeld ? CHUNKS : 1][VEC];
  double w[kHeldWeights ? CHUNKS : 1][VEC];
  // not held: entries below `floor_`, and those at it behind index `floor_last`, are excluded;
  // so are weights below least
  float floor_ = OT_NEG_INF;
  int floor_last = 0x7fffffff;
  double least = 0.0;
  // sum of the remaining weights of this wave's part, where it is known, and entries at a value
  double part = 0.0;
  int part_at = 0;
  bool part_known = false;

  __device__ __forceinline__ Sampler(const RowGroup<WAVES> &g_, const void *row_, int V_, int per_wave_, float m_,
                                     float temperature, float (&x_)[kHeld ? CHUNKS : 1][VEC])
      : g(g_), row(row_), V(V_), per_wave(per_wave_), m(m_), weight(m_, temperature), x(x_) {}

  __device__ __forceinline__ int chunks() const { return kHeld ? CHUNKS : per_wave; }
  __device__ __forceinline__ int first_index(int j) const {
    return ((g.wave * chunks() + j) * kWave + g.lane) * VEC;
  }
  // f(j, i, x of the chunk) for each chunk of this lane, i the index of its first element
  template <class F>
  __device__ __forceinline__ void each(F f) {
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) f(j, first_index(j), x[j]);
    } else {
      for (int j = 0; j < per_wave; ++j) {
        const int i = first_index(j);
        float y[VEC];
        load_logits<T>(row, i, V, y);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (y[e] < floor_ || (y[e] == floor_ && i + e > floor_last)) y[e] = OT_NEG_INF;
        f(j, i, y);
      }
    }
  }
  __device__ __forceinline__ double weight_of(int j, int e, float y) {
    if constexpr (kHeldWeights) return w[j][e];
    const double v = weight(y);
    return v >= least ? v : 0.0;
  }
  // sum of a chunk's VEC weights, pairwise
  __device__ __forceinline__ static double pairwise(const double v[VEC]) {
    if constexpr (VEC == 4) return (v[0] + v[1]) + (v[2] + v[3]);
    else return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  }

  // Excludes the entries below v, and those at v behind the first n.
  __device__ __forceinline__ void exclude(float v, int n, int at_v) {
    int last = 0x7fffffff;
    if (n < at_v) {  // the index of entry number n of those at v
      int mine = 0;
      each([&](int, int, const float *y) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) mine += y[e] == v;
      });
      const int here = wave_sum(mine);
      int before = 0;
      g.sync();
      if constexpr (WAVES > 1) {
        if (g.lane == 0) g.s.count[g.wave] = here;
      }
      if (g.thread() == 0) g.s.index = -1;
      g.sync();
      if constexpr (WAVES > 1) {
        for (int k = 0; k < g.wave; ++k) before += g.s.count[k];
      }
      if (before < n && n <= before + here) {
        each([&](int, int i, const float *y) {
          int c = 0;
#pragma unroll
          for (int e = 0; e < VEC; ++e) c += y[e] == v;
          const int upto = wave_scan(c);
          int seen = before + upto - c;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            seen += y[e] == v;
            if (y[e] == v && seen == n) g.s.index = i + e;
          }
          before += lane_value(upto, kWave - 1);
        });
      }
      g.sync();
      last = g.s.index;
    }
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (x[j][e] < v || (x[j][e] == v && first_index(j) + e > last)) {
            x[j][e] = OT_NEG_INF;
            if constexpr (kHeldWeights) w[j][e] = 0.0;
          }
    } else {
      floor_last = v == floor_ ? min(last, floor_last) : last;
      floor_ = v;
    }
  }

  // The largest value v such that the entries at or above it (their number, or with WEIGHTS
  // their weights) reach `want`, among those of [lo, m]; above: what the entries above v come to.
  // With WEIGHTS this goes by 32-bit weights in whatever order the bins are filled: close, and
  // for the caller to settle.  Without, it is content with a smaller value as soon as no more than
  // `enough` entries are at or above it; above is then -1.
  template <bool WEIGHTS>
  __device__ __forceinline__ float select(double want, float lo, double &above, int enough = 0) {
    float *const bin_weight = reinterpret_cast<float *>(g.s.bins);
    float hi = m;
    above = 0.0;
    const float per_octave = (float)weight.c;
    while (lo < hi) {
      for (int i = g.thread(); i < kSampleBins; i += WAVES * kWave) g.s.bins[i] = 0;  // (also as a float)
      g.sync();
      // bins of equal width; where that is no normal number, bins of the values' bit patterns.
      // Either way hi falls into the first bin and lo into the last.
      const float half = 0.5f * hi - 0.5f * lo;
      const bool by_value = half > 1e-30f;
      const float per_unit = by_value ? (0.5f * kSampleBins) / half : 0.f;
      const unsigned hi_key = order_key(hi);
      const int shift = max(0, 24 - __clz(hi_key - order_key(lo)));
      auto bin = [&](float y) -> int {
        return by_value ? (int)fminf((hi - y) * per_unit, kSampleBins - 1.0f)
                        : (int)((hi_key - order_key(y)) >> shift);
      };
      each([&](int, int, const float *y) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (y[e] >= lo && y[e] <= hi) {
            const int b = bin(y[e]);
            if constexpr (WEIGHTS) unsafeAtomicAdd(&bin_weight[b], __builtin_amdgcn_exp2f((y[e] - m) * per_octave));
            else atomicAdd(&g.s.bins[b], 1u);
          }
      });
      g.sync();
      // every wave looks for the bin: lane l holds bins [4 l, 4 l + 4)
      constexpr int kPer = kSampleBins / kWave;
      double amount[kPer], mine = 0.0;
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        amount[q] = WEIGHTS ? (double)bin_weight[g.lane * kPer + q] : (double)g.s.bins[g.lane * kPer + q];
        mine += amount[q];
      }
      double run = above + (wave_scan(mine) - mine);
      int reached = kSampleBins, filled = -1;
      double before_reached = 0.0, before_filled = 0.0, with_reached = 0.0;
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        if (amount[q] > 0.0) {
          filled = g.lane * kPer + q;
          before_filled = run;
          if (reached == kSampleBins && run + amount[q] >= want) {
            reached = filled;
            before_reached = run;
            with_reached = run + amount[q];
          }
        }
        run += amount[q];
      }
      const uint64_t r = __ballot(reached < kSampleBins), f = __ballot(filled >= 0);
      // (rounding can keep the last bin from reaching `want`, and all weights can be 0)
      const int src = r ? __builtin_ctzll(r) : f ? 63 - __builtin_clzll(f) : 0;
      const int pick = r ? lane_value(reached, src) : f ? lane_value(filled, src) : kSampleBins - 1;
      above = r ? lane_value(before_reached, src) : f ? lane_value(before_filled, src) : above;
      const bool content = !WEIGHTS && r && lane_value(with_reached, src) <= enough;
      float b_hi = OT_NEG_INF, b_lo = kInf;
      each([&](int, int, const float *y) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (y[e] >= lo && y[e] <= hi && bin(y[e]) == pick) {
            b_hi = fmaxf(b_hi, y[e]);
            b_lo = fminf(b_lo, y[e]);
          }
      });
      g.sync();  // the bins have been read
      g.extremes(b_hi, b_lo);
      if (!(b_lo <= b_hi)) return hi;  // nothing there (no such entries or weights)
      if (content) {
        above = -1.0;
        return b_lo;
      }
      hi = b_hi;
      lo = b_lo;
    }
    return lo;
  }

  // Copies the entries that can be among the first k of the order, kSampleFew at most, and their
  // indices, in index order; k <= kSampleFew.  Returns their number.
  __device__ __forceinline__ int gather_few(int k, float lowest, int finite, float *few, int *few_index) {
    float v = lowest;
    if (finite > kSampleFew) {
      double above;
      v = select<false>((double)k, lowest, above, kSampleFew);
      if (above >= 0.0) {  // too many entries at v: only the first of them
        int at_v = 0;
        each([&](int, int, const float *y) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) at_v += y[e] == v;
        });
        double none = 0.0;
        g.totals(none, at_v);
        exclude(v, k - (int)above, at_v);
      }
    }
    int here = 0;
    each([&](int, int, const float *y) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) here += __popcll(__ballot(y[e] >= v));
    });
    int at = 0, total = here;
    if constexpr (WAVES > 1) {
      g.sync();
      if (g.lane == 0) g.s.count[g.wave] = here;
      g.sync();
      total = 0;
      for (int q = 0; q < WAVES; ++q) {
        if (q == g.wave) at = total;
        total += g.s.count[q];
      }
    }
    each([&](int, int i, const float *y) {
      int to = at;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {  // entries of the lanes before
        const uint64_t kept = __ballot(y[e] >= v);
        to += __builtin_amdgcn_mbcnt_hi((unsigned)(kept >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)kept, 0));
        at += __popcll(kept);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (y[e] >= v) {
          few[to] = y[e];
          few_index[to] = i + e;
          ++to;
        }
    });
    g.sync();
    return total;
  }

  // `lowest`: the smallest finite entry, `finite`: how many there are
  __device__ __forceinline__ void keep_top_k(int k, float &lowest, int finite) {
    if (k >= finite) return;
    double above;
    const float v = select<false>((double)k, lowest, above);
    int at_v = 0;
    each([&](int, int, const float *y) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) at_v += y[e] == v;
    });
    double none = 0.0;
    g.totals(none, at_v);
    exclude(v, k - (int)above, at_v);
    lowest = v;
  }

  // Weights above v (those at or above it with `and_at`) and the number of entries at v: of this
  // wave's part in part and part_at, of the row in sum and at_v.
  template <bool AND_AT>
  __device__ __forceinline__ void sum_above(float v, double &sum, int &at_v) {
    part = 0.0;
    part_at = 0;
    each([&](int j, int, const float *y) {
      double t[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        t[e] = y[e] > v || (AND_AT && y[e] == v) ? weight_of(j, e, y[e]) : 0.0;
        part_at += y[e] == v;
      }
      part += pairwise(t);
    });
    part = wave_sum(part);
    part_at = wave_sum(part_at);
    g.gather(part, part_at, sum, at_v);
  }

  // Of `count` entries in s.few, in front of which weights of `above` lie: how many remain for
  // `want`; the last of them, n of the at_v entries at its value.  False if the border is not among
  // them.
  template <int N>
  __device__ __forceinline__ bool settle(int count, double above, double want, float &v, int &n, int &at_v) const {
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = g.lane * N + i < count ? g.s.few[g.lane * N + i] : OT_NEG_INF;
    wave_sort(y, g.lane);
    if (sorted_fit(y, count, above, [&](double) { return want; }, n) < want && n == count) return false;
    if (n == 0) return false;
    v = sorted_value(y, n - 1);
    int over = 0;
    at_v = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      over += __popcll(__ballot(y[e] > v));
      at_v += __popcll(__ballot(y[e] == v));
    }
    n -= over;
    return true;
  }
  // The first k of a wave's sorted entries, weights of `above` in front of them: returns the sum of
  // both, and in n how many of the entries have less than want(that sum) in front of them (the row's
  // largest entry counts anyway).
  template <int N, class W>
  __device__ __forceinline__ double sorted_fit(const float (&y)[N], int k, double above, W want_of, int &n) const {
    double t[N], mine = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      t[i] = g.lane * N + i < k ? weight(y[i]) : 0.0;
      mine += t[i];
    }
    const double upto = wave_scan(mine), total = above + lane_value(upto, kWave - 1), want = want_of(total);
    double before = above + (upto - mine);
    int fit = 0;  // of this lane's entries, in front of the first that does not remain
    bool all = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      all = all && (before < want || (g.lane * N + i == 0 && y[i] == m));
      fit += all;
      before += t[i];
    }
    n = k;
    const uint64_t end = __ballot(fit < N);
    if (end) {
      const int l = __builtin_ctzll(end);
      n = min(k, l * N + lane_value(fit, l));
    }
    return total;
  }
  // entry number `at` of a wave's sorted ones
  template <int N>
  __device__ __forceinline__ static float sorted_value(const float (&y)[N], int at) {
    float v = OT_NEG_INF;  // (a maximum, and not a choice between elements, which would index the registers)
#pragma unroll
    for (int e = 0; e < N; ++e) v = fmaxf(v, e == at % N ? y[e] : OT_NEG_INF);
    return lane_value(v, at / N);
  }

  // top_p's cut where it falls into one bin of few entries: their order settles it.  False if it
  // does not; the bins' 32-bit sums, in whatever order they are formed, decide about no more than
  // that.
  __device__ __forceinline__ bool cut_in_one_bin(double want, float from) {
    float *const bin_weight = reinterpret_cast<float *>(g.s.bins);
    const float half = 0.5f * m - 0.5f * from;
    if (!(half > 1e-30f)) return false;
    const float per_unit = (0.5f * kSampleBins) / half;
    auto bin = [&](float y) -> int { return (int)fminf((m - y) * per_unit, kSampleBins - 1.0f); };
    for (int i = g.thread(); i < kSampleBins; i += WAVES * kWave) bin_weight[i] = 0.f;
    if (g.thread() == 0) g.s.index = 0;
    g.sync();
    const float per_octave = (float)weight.c;
    each([&](int, int, const float *y) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (y[e] >= from) unsafeAtomicAdd(&bin_weight[bin(y[e])], __builtin_amdgcn_exp2f((y[e] - m) * per_octave));
    });
    g.sync();
    // every wave looks for the bin: lane l holds bins [4 l, 4 l + 4)
    constexpr int kPer = kSampleBins / kWave;
    double amount[kPer], mine = 0.0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      amount[q] = (double)bin_weight[g.lane * kPer + q];
      mine += amount[q];
    }
    double run = wave_scan(mine) - mine;
    int reached = kSampleBins;
#pragma unroll
    for (int q = kPer - 1; q >= 0; --q) {
      double upto = run;
#pragma unroll
      for (int k = 0; k <= q; ++k) upto += amount[k];
      if (amount[q] > 0.0 && upto >= want) reached = g.lane * kPer + q;
    }
    const uint64_t r = __ballot(reached < kSampleBins);
    if (!r) {
      g.sync();  // the bins have been read
      return false;
    }
    const int pick = lane_value(reached, __builtin_ctzll(r));
    double above = 0.0;
    each([&](int j, int, const float *y) {
      double t[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int b = y[e] >= from ? bin(y[e]) : kSampleBins;
        t[e] = b < pick ? weight_of(j, e, y[e]) : 0.0;
        if (b == pick) {
          const int to = atomicAdd(&g.s.index, 1);
          if (to < kSampleFew) g.s.few[to] = y[e];
        }
      }
      above += pairwise(t);
    });
    int none = 0;
    g.totals(above, none);  // (barriers: the entries are in place)
    const int count = g.s.index;
    if (count > kSampleFew) return false;
    g.sync();  // the count has been read
    if (g.wave == 0) {
      float v = 0.f;
      int n = 0, at_v = 0;
      const bool ok = count <= kWave ? settle<1>(count, above, want, v, n, at_v)
                                     : settle<kSampleFew / kWave>(count, above, want, v, n, at_v);
      if (g.lane == 0) {
        g.s.value[0][0] = v;
        g.s.count[0] = n;
        g.s.count[1] = at_v;
        g.s.index = ok;
      }
    }
    g.sync();
    const bool ok = g.s.index;
    const float v = g.s.value[0][0];
    const int n = g.s.count[0], at_v = g.s.count[1];
    g.sync();  // they have been read
    if (ok) exclude(v, n, at_v);
    return ok;
  }

  static constexpr int kNearSteps = 4;
  __device__ __forceinline__ void keep_top_p(float p, float lowest) {
    double total;
    int none;
    sum_above<true>(lowest, total, none);
    part_known = false;
    const double want = (double)p * total;
    // Entries of weights below (1 - p) * total / V come to less than what lies behind the cut.
    float from = lowest;
    const double least_weight = (1.0 - (double)p) * total / V * 0.99;
    if (least_weight > 1e-30) {
      const float z = __log2f((float)least_weight) / (float)weight.c;
      if (z > -1e30f) from = fminf(m, fmaxf(from, m + 1.001f * z));
    }
    // (rows of up to some hundred entries per bin: 64 x 50 000 float32 109 us, 138 without it;
    // 64 x 131 072, where the bin holds too many, 512 and 337)
    if (V <= kSampleBins * kSampleBins && cut_in_one_bin(want, from)) return;
    double rough, sum;
    float v = select<true>(want, from, rough);
    // Where the entries above v reach `want` already, or those at it do not, v is somewhere else: next
    // to it for a few steps, and then by halving what is left of the values' keys (32-bit sums of many
    // weights in one bin can be off by thousands of entries, and stop growing at 2^24 times a weight).
    // (keys, and not their values, which both zeros have in common: every answer takes its key out)
    unsigned key = order_key(v), below = order_key(lowest) - 1, beyond = order_key(m) + 1;
    int at_v, went = 0;
    double wv;
    bool last = false;
    for (int step = 0;; ++step) {
      sum_above<false>(v, sum, at_v);
      wv = weight(v);
      const int go = sum >= want && v < m ? 1 : sum + at_v * wv < want && v > lowest ? -1 : 0;
      if (last || go == 0 || go == -went) break;  // (back and forth: the border lies within a rounding)
      if (go > 0) below = key;
      else beyond = key;
      went = step < kNearSteps ? go : 0;
      last = step >= kNearSteps && beyond - below <= 1;  // nothing left: a rounding again
      if (step >= kNearSteps && !last) {
        key = below + (beyond - below) / 2;
        v = key_value(key);  // (`go` is not 0 where no entry is)
        continue;
      }
      if (last) v = key_value(below);
      float up = kInf, down = OT_NEG_INF;
      each([&](int, int, const float *y) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if (y[e] > v) up = fminf(up, y[e]);
          if (y[e] < v) down = fmaxf(down, y[e]);
        }
      });
      g.extremes(down, up);
      v = last || go > 0 ? up : down;
      key = order_key(v);
    }
    // of the entries at v, number j (from 0) remains if sum + j * wv < want
    int n = at_v;
    if (wv > 0.0) {
      const double q = ceil((want - sum) / wv);
      n = q < 1.0 ? 0 : q < at_v ? (int)q : at_v;
    }
    if (v == m) n = max(n, 1);
    exclude(v, n, at_v);
    // this wave's part of what remains
    int before = 0;
    if constexpr (WAVES > 1) {
      g.sync();
      if (g.lane == 0) g.s.count[g.wave] = part_at;
      g.sync();
      for (int k = 0; k < g.wave; ++k) before += g.s.count[k];
    }
    part += max(0, min(n - before, part_at)) * wv;
    part_known = true;
  }

  __device__ __forceinline__ void keep_min_p(float p) {
    least = p;
    part_known = false;
    if constexpr (kHeldWeights) {
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (!(w[j][e] >= least)) w[j][e] = 0.0;
    }
  }

  // the cuts; before them `lowest` is the smallest finite entry, of `finite` ones
  __device__ __forceinline__ void cut(int top_k, float top_p, float min_p, float lowest, int finite) {
    if constexpr (WAVES == 1) {
      const int k = top_k > 0 ? min(top_k, finite) : finite;
      if (k < finite || top_p < 1.f) cut_sorted(k, top_p, finite);
      weigh();
    } else {
      if (top_k > 0 && top_k < V) keep_top_k(top_k, lowest, finite);
      weigh();
      if (top_p < 1.f) keep_top_p(fmaxf(top_p, 0.f), lowest);
    }
    if (min_p > 0.f) keep_min_p(fminf(min_p, 1.f));
  }
  // top_k and top_p by a wave that holds the row: the entries in order
  __device__ __forceinline__ void cut_sorted(int k, float top_p, int finite) {
    constexpr int N = CHUNKS * VEC;
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = x[i / VEC][i % VEC];
    wave_sort(y, g.lane);
    int n = k;  // entries that remain
    if (top_p < 1.f) {
      const double p = fmax((double)top_p, 0.0);
      sorted_fit(y, k, 0.0, [&](double total) { return p * total; }, n);
    }
    if (n >= finite) return;
    const float v = sorted_value(y, n - 1);
    int above = 0, at_v = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      above += __popcll(__ballot(y[e] > v));
      at_v += __popcll(__ballot(y[e] == v));
    }
    exclude(v, n - above, at_v);
  }
  __device__ __forceinline__ void weigh() {
    if constexpr (kHeldWeights) {
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[j][e] = weight(x[j][e]);
    }
  }

  // Where the running sum, `run` in front of chunk j, passes the target in it: in the first lane
  // with a weight whose sum does (pass, some), else the last one with a weight, and there in the
  // first element that does, else the last one with a weight (sums in another order can fall short
  // of each other's borders by their rounding, and the scan's can grow by one over a lane that adds
  // nothing).  upto: the scan over the lanes.  What lies in front of the lane is the scan's sum at
  // the lane before, and not the difference of two sums, which loses small weights before a large one.
  __device__ __forceinline__ void find(const double t[VEC], const float *y, int i, double run, double upto,
                                       double target, uint64_t pass, uint64_t some, int &symbol, float &logit) const {
    const int l = pass & some ? __builtin_ctzll(pass & some) : 63 - __builtin_clzll(some);
    double c = l > 0 ? run + lane_value(upto, l - 1) : run;
    int at = -1;
    bool found = false;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const double next = c + t[e];
      if (!found && t[e] > 0.0) {
        at = e;
        found = next > target;
      }
      c = next;
    }
    // (a maximum, and not a choice between elements, which would index the registers)
    float at_logit = OT_NEG_INF;
#pragma unroll
    for (int e = 0; e < VEC; ++e) at_logit = fmaxf(at_logit, e == at ? y[e] : OT_NEG_INF);
    symbol = lane_value(i + at, l);
    logit = lane_value(at_logit, l);
  }

  // the same as draw() for one wave that holds the row's weights: one scan per chunk
  __device__ __forceinline__ void draw_alone(double u, int &symbol, float &logit, double &total) const {
    double mine[CHUNKS], upto[CHUNKS], before[CHUNKS + 1];
    before[0] = 0.0;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
      mine[j] = pairwise(w[j]);
      upto[j] = wave_scan(mine[j]);
      before[j + 1] = before[j] + lane_value(upto[j], kWave - 1);
    }
    total = before[CHUNKS];
    // u >= 1, or a product that rounds up to the total, takes the last entry with a weight
    const double target = fmax(u, 0.0) * total;
    const bool past = !(target < total);
    symbol = -1;
#pragma unroll
    for (int j = CHUNKS - 1; j >= 0; --j) {
      const uint64_t some = __ballot(mine[j] > 0.0);
      if (past ? symbol < 0 && some != 0 : before[j] <= target && target < before[j + 1])
        find(w[j], x[j], first_index(j), before[j], upto[j], target,
             __ballot(before[j] + upto[j] > target), some, symbol, logit);
    }
  }

  // `start`, `whole`: what lies in front of these entries and the total, where they are a slice of
  // a row
  __device__ __forceinline__ Drawn draw(double u, double start = 0.0, double whole = -1.0) {
    if constexpr (WAVES == 1) {
      int symbol;
      float logit;
      double total;
      draw_alone(u, symbol, logit, total);
      return {symbol, log_probability(logit, m, weight.c, total)};
    } else {
      // totals of the waves' parts, then the part, the chunk, the lane and the element in which
      // the running sum passes u * total
      if (!part_known) {
        part = 0.0;
        each([&](int j, int, const float *y) {
          double t[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) t[e] = weight_of(j, e, y[e]);
          part += pairwise(t);
        });
        part = wave_sum(part);
      }
      g.sync();
      if (g.lane == 0) g.s.sum[g.wave] = part;
      if (g.thread() == 0) g.s.index = -1;
      g.sync();
      double total = start, before = start;
      for (int k = 0; k < WAVES; ++k) {
        if (k == g.wave) before = total;
        total += g.s.sum[k];
      }
      if (whole >= 0.0) total = whole;
      const double product = fmax(u, 0.0) * total;
      const double target = product < total ? product : __builtin_huge_val();
      int symbol = -1;
      float logit = 0.f;
      if (before <= target && target < before + part) {  // one wave
        double run = before;
        int last = -1;  // the wave's last entry with a weight
        float last_logit = 0.f;
        each([&](int j, int i, const float *y) {
          if (symbol >= 0) return;
          double t[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) t[e] = weight_of(j, e, y[e]);
          const double mine = pairwise(t), upto = wave_scan(mine);
          const double chunk = lane_value(upto, kWave - 1);
          const uint64_t pass = __ballot(run + upto > target);
          const uint64_t some = __ballot(mine > 0.0);
          if (some) {
            find(t, y, i, run, upto, target, pass, some, last, last_logit);
            if (pass & some) symbol = last;
          }
          run += chunk;
        });
        logit = last_logit;
        if (symbol < 0) symbol = last;
        if (g.lane == 0) {
          g.s.index = symbol;
          g.s.value[0][0] = logit;
        }
      }
      g.sync();
      symbol = g.s.index;
      logit = g.s.value[0][0];
      if (symbol < 0) {  // u >= 1, or a product that rounds up to the total: the last entry with a weight
        each([&](int j, int i, const float *y) {
          int last = -1;
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (weight_of(j, e, y[e]) > 0.0) last = i + e;
          const uint64_t some = __ballot(last >= 0);
          if (some) symbol = lane_value(last, 63 - __builtin_clzll(some));
        });
        g.sync();
        if (g.lane == 0) g.s.count[g.wave] = symbol;
        g.sync();
        for (int k = 0; k < WAVES; ++k) symbol = max(symbol, g.s.count[k]);
        logit = load_element<T>(row, symbol);
      }
      return {symbol, log_probability(logit, m, weight.c, total)};
    }
  }
};

// What the cuts start from: the largest entry m, whether there is a NaN (bad < 0), the smallest
// finite entry and how many are finite; of elements, and of the group.
template <int VEC>
__device__ __forceinline__ void look(const float *y, float &m, float &bad, float &lowest, int &finite) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    m = fmaxf(m, y[e]);
    if (y[e] != y[e]) bad = -1.f;
    if (y[e] > OT_NEG_INF) {
      lowest = fminf(lowest, y[e]);
      ++finite;
    }
  }
}
template <int WAVES>
__device__ __forceinline__ void look_together(const RowGroup<WAVES> &g, float &m, float &bad, float &lowest,
                                              int &finite) {
  float none = 0.f;
  double nothing = 0.0;
  g.extremes(none, bad);
  g.extremes(m, lowest);
  g.totals(nothing, finite);
}

// One row, in x if it is held: settles the rows without an answer and the greedy ones, draws from
// the others.  FILTER: one of top_k, top_p and min_p may be in force.
template <class T, int WAVES, int CHUNKS, bool FILTER>
__device__ __forceinline__ void sample_row(const RowGroup<WAVES> &g, const void *row, int V, double u,
                                           float temperature, int top_k, float top_p, float min_p,
                                           float (&x)[CHUNKS > 0 ? CHUNKS : 1][kSampleVec<T>], int32_t *symbol,
                                           float *log_prob) {
  constexpr int VEC = kSampleVec<T>;
  constexpr bool kHeld = CHUNKS > 0;
  const int chunks = kHeld ? CHUNKS : (V + WAVES * kWave * VEC - 1) / (WAVES * kWave * VEC);
  auto first_index = [&](int j) { return ((g.wave * chunks + j) * kWave + g.lane) * VEC; };
  auto each = [&](auto f) {
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) f(j, x[j]);
    } else {
      for (int j = 0; j < chunks; ++j) {
        float y[VEC];
        load_logits<T>(row, first_index(j), V, y);
        f(j, y);
      }
    }
  };
  const bool cuts = FILTER && temperature > 0.f && ((top_k > 0 && top_k < V) || top_p < 1.f);
  float m = OT_NEG_INF, bad = 0.f, lowest = kInf;
  int finite = 0;
  if (cuts) {
    each([&](int, const float *y) { look<VEC>(y, m, bad, lowest, finite); });
    look_together(g, m, bad, lowest, finite);
  } else {
    each([&](int, const float *y) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        m = fmaxf(m, y[e]);
        if (y[e] != y[e]) bad = -1.f;
      }
    });
    g.extremes(m, bad);
  }
  Drawn d = {-1, OT_NEG_INF};
  if (bad < 0.f || __builtin_isinf(m) || u != u) {
    // no answer
  } else if (!(temperature > 0.f)) {
    int first = -1;
    each([&](int j, const float *y) {
      int at = VEC;
#pragma unroll
      for (int e = VEC - 1; e >= 0; --e)
        if (y[e] == m) at = e;
      const uint64_t hit = __ballot(at < VEC);
      if (first < 0 && hit) first = lane_value(first_index(j) + at, __builtin_ctzll(hit));
    });
    if constexpr (WAVES > 1) {
      g.sync();
      if (g.lane == 0) g.s.count[g.wave] = first;
      g.sync();
      for (int k = WAVES - 1; k >= 0; --k)
        if (g.s.count[k] >= 0) first = g.s.count[k];
    }
    d = {first, 0.f};
  } else {
    Sampler<T, WAVES, CHUNKS> sampler(g, row, V, chunks, m, temperature, x);
    if constexpr (FILTER) sampler.cut(top_k, top_p, min_p, lowest, finite);
    else sampler.weigh();
    d = sampler.draw(u);
  }
  g.sync();  // the group's shared values have been read
  if (g.thread() == 0) {
    *symbol = d.symbol;
    *log_prob = d.log_prob;
  }
}

// Rows of several waves of which top_k leaves few entries (0 < top_k <= kSampleFew, top_k < V):
// the waves of a workgroup find them together, for BATCH rows one after the other, and then a wave
// each goes on with the few of one row.
template <class T, int WAVES, int CHUNKS, int BATCH>
__global__ __launch_bounds__(WAVES * kWave, WAVES == 16 ? 4 : WAVES == 8 || CHUNKS * kSampleVec<T> > 16 ? 2 : 3) void
sample_few_kernel(const void *__restrict__ logits, int64_t row_stride, int64_t rows, int V,
                  const float *__restrict__ uniform, SampleSettings set, int32_t *__restrict__ symbols,
                  float *__restrict__ log_probs) {
  static_assert(BATCH <= WAVES, "a wave takes one row");
  constexpr int VEC = kSampleVec<T>, kLanes = kSampleFew / 256;
  __shared__ SampleShared<WAVES> s_all;
  __shared__ SampleShared<1> s_one[BATCH];
  __shared__ __attribute__((aligned(16))) float s_few[BATCH][kSampleFew];
  __shared__ int s_index[BATCH][kSampleFew];
  __shared__ float s_m[BATCH];
  __shared__ int s_n[BATCH];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const RowGroup<WAVES> g = {s_all, lane, wave};
  const int chunks = CHUNKS > 0 ? CHUNKS : (V + WAVES * kWave * VEC - 1) / (WAVES * kWave * VEC);
  const int top_k = set.top_k_value;
  for (int64_t row0 = (int64_t)blockIdx.x * BATCH; row0 < rows; row0 += (int64_t)gridDim.x * BATCH) {
#pragma unroll 1
    for (int q = 0; q < BATCH && row0 + q < rows; ++q) {
      const char *base =
          static_cast<const char *>(logits) + (row0 + q) * row_stride * (sizeof(T) == 4 ? 4 : 2);
      float x[CHUNKS > 0 ? CHUNKS : 1][VEC];
      float m = OT_NEG_INF, bad = 0.f, lowest = kInf;
      int finite = 0;
      if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) load_logits<T>(base, ((wave * CHUNKS + j) * kWave + lane) * VEC, V, x[j]);
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) look<VEC>(x[j], m, bad, lowest, finite);
      } else {
        for (int j = 0; j < chunks; ++j) {
          float y[VEC];
          load_logits<T>(base, ((wave * chunks + j) * kWave + lane) * VEC, V, y);
          look<VEC>(y, m, bad, lowest, finite);
        }
      }
      look_together(g, m, bad, lowest, finite);
      int n = -1;
      if (!(bad < 0.f || __builtin_isinf(m))) {
        Sampler<T, WAVES, CHUNKS> sampler(g, base, V, chunks, m, 1.0f, x);
        n = sampler.gather_few(top_k, lowest, finite, s_few[q], s_index[q]);
      }
      if (g.thread() == 0) {
        s_m[q] = m;
        s_n[q] = n;
      }
    }
    g.sync();
    if (wave < BATCH && row0 + wave < rows) {
      const int64_t row = row0 + wave;
      const double u = uniform[row];
      const float temperature = set.temperature ? set.temperature[row] : set.temperature_value;
      const float top_p = set.top_p ? set.top_p[row] : set.top_p_value;
      const float min_p = set.min_p ? set.min_p[row] : set.min_p_value;
      const int n = s_n[wave];
      const float m = s_m[wave];
      Drawn d = {-1, OT_NEG_INF};
      if (n > 0 && u == u) {
        float few[kLanes][4], lowest = kInf;
#pragma unroll
        for (int j = 0; j < kLanes; ++j) {
          const int i = (j * kWave + lane) * 4;
          const f32x4 y = *reinterpret_cast<const f32x4 *>(&s_few[wave][i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            few[j][e] = i + e < n ? y[e] : OT_NEG_INF;
            lowest = fminf(lowest, i + e < n ? y[e] : kInf);
          }
        }
        const RowGroup<1> one = {s_one[wave], lane, 0};
        if (!(temperature > 0.f)) {
#pragma unroll
          for (int j = kLanes - 1; j >= 0; --j) {
            int at = 4;
#pragma unroll
            for (int e = 3; e >= 0; --e)
              if (few[j][e] == m) at = e;
            const uint64_t hit = __ballot(at < 4);
            if (hit) d = {lane_value((j * kWave + lane) * 4 + at, __builtin_ctzll(hit)), 0.f};
          }
        } else {
          float none = 0.f;
          one.extremes(none, lowest);
          Sampler<float, 1, kLanes> rest(one, s_few[wave], n, kLanes, m, temperature, few);
          rest.cut(top_k, top_p, min_p, lowest, n);
          d = rest.draw(u);
        }
        d.symbol = s_index[wave][d.symbol];
      }
      if (lane == 0) {
        symbols[row] = d.symbol;
        log_probs[row] = d.log_prob;
      }
    }
    g.sync();  // the few have been read
  }
}

template <class T, int WAVES, int CHUNKS, int BATCH>
static int launch_sample_few(const void *logits, int64_t row_stride, int64_t rows, int32_t V, const float *uniform,
                             const SampleSettings &set, int32_t *symbols, float *log_probs, hipStream_t s) {
  const int64_t groups = (rows + BATCH - 1) / BATCH;
  const dim3 grid((unsigned)(groups < (1 << 20) ? groups : (1 << 20)));
  hipLaunchKernelGGL((sample_few_kernel<T, WAVES, CHUNKS, BATCH>), grid, dim3(WAVES * kWave), 0, s, logits, row_stride,
                     rows, V, uniform, set, symbols, log_probs);
  return (int)hipGetLastError();
}

// Short rows without cuts: a wave per row, `batch` rows (64 at most) one after the other with the
// next one on its way, their numbers and settings read and their answers written side by side, and
// the logarithms of a batch taken at once, a row per lane.
template <class T, int CHUNKS>
__global__ __launch_bounds__(kBlock, 4) void sample_plain_kernel(const void *__restrict__ logits, int64_t row_stride,
                                                                 int64_t rows, int V, int batch,
                                                                 const float *__restrict__ uniform,
                                                                 const float *__restrict__ temperature,
                                                                 float temperature_value,
                                                                 int32_t *__restrict__ symbols,
                                                                 float *__restrict__ log_probs) {
  constexpr int VEC = kSampleVec<T>;
  __shared__ SampleShared<1> s_unused[1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const RowGroup<1> g = {s_unused[0], (int)(threadIdx.x % kWave), 0};
  auto load = [&](int64_t row, float (&to)[CHUNKS][VEC]) {
    const char *base = static_cast<const char *>(logits) + min(row, rows - 1) * row_stride * (sizeof(T) == 4 ? 4 : 2);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) load_logits<T>(base, (j * kWave + g.lane) * VEC, V, to[j]);
  };
  const int64_t stride = (int64_t)gridDim.x * kWavesPerBlock * batch;
  int64_t row0 = ((int64_t)blockIdx.x * kWavesPerBlock + wave) * batch;
  if (row0 >= rows) return;
  float x[CHUNKS][VEC];
  load(row0, x);
  for (; row0 < rows; row0 += stride) {
    const int n = (int)min((int64_t)batch, rows - row0);
    const float my_u = g.lane < n ? uniform[row0 + g.lane] : 0.f;
    const float my_T = temperature && g.lane < n ? temperature[row0 + g.lane] : temperature_value;
    int my_symbol = -1;
    float my_logit = 0.f, my_m = 0.f;
    double my_total = 1.0;
#pragma unroll 1
    for (int q = 0; q < n; ++q) {
      float next[CHUNKS][VEC];
      load(q + 1 < n ? row0 + q + 1 : row0 + stride, next);
      float m = OT_NEG_INF;
      bool nan = false;
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          m = fmaxf(m, x[j][e]);
          nan |= x[j][e] != x[j][e];
        }
      m = group_allreduce<kWave>(m, MaxOp());
      const float u = lane_value(my_u, q), T_ = lane_value(my_T, q);
      int symbol = -1;
      float logit = m;
      double total = 1.0;
      if (__ballot(nan) || __builtin_isinf(m) || u != u) {
        // no answer
      } else if (!(T_ > 0.f)) {
#pragma unroll
        for (int j = CHUNKS - 1; j >= 0; --j) {
          int at = VEC;
#pragma unroll
          for (int e = VEC - 1; e >= 0; --e)
            if (x[j][e] == m) at = e;
          const uint64_t hit = __ballot(at < VEC);
          if (hit) symbol = lane_value((j * kWave + g.lane) * VEC + at, __builtin_ctzll(hit));
        }
      } else {
        Sampler<T, 1, CHUNKS> sampler(g, nullptr, V, CHUNKS, m, T_, x);
        sampler.weigh();
        sampler.draw_alone((double)u, symbol, logit, total);
      }
      if (g.lane == q) {
        my_symbol = symbol;
        my_logit = logit;
        my_m = m;
        my_total = total;
      }
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[j][e] = next[j][e];
    }
    if (g.lane < n) {
      symbols[row0 + g.lane] = my_symbol;
      log_probs[row0 + g.lane] = my_symbol < 0 ? OT_NEG_INF
                                 : my_T > 0.f  ? log_probability(my_logit, my_m, Weight(my_m, my_T).c, my_total)
                                               : 0.f;
    }
  }
}

// ---- long rows in slices ---------------------------------------------------------------------
//
// A row beyond the registers of a workgroup is cut into slices of kSlice entries, a workgroup
// each, so that few rows fill the chip too and every step reads the row once:
//   1 facts   a slice's largest entry, where it is, and the sum of its weights relative to it
//   2 bins    (top_p) weights of a slice by value, in 1024 bins of equal width, as integers of
//             2^-32: sums that no order of the additions changes
//   3 join    (top_p) a workgroup per row: the bin in which the weights of all slices reach top_p
//             of the total
//   4 cuts    (top_p, min_p) of a slice, the 64-bit sums of what lies above that bin, and the
//             entries in it, in index order
//   5 draw    a workgroup per row: the exact cut among the entries of the bin, the slice in which
//             the running sum passes u times what remains, and the symbol in that slice
// Where a bin holds more than kBinEntries of a slice, or the rounded sums missed the bin, step 5
// does the row in the way of the shorter ones, reading it in every step.

constexpr float kBinScale = 4294967040.f;  // the largest below 2^32
constexpr int kSlice = 8192, kSliceBins = 1024, kBinEntries = 256;
constexpr int kSliceWaves = 8, kSliceThreads = kSliceWaves * kWave;
constexpr int kMostSlices = kWave;    // of a row: a lane each
constexpr int kLongRow = 16384;       // the longest row that a workgroup holds in registers
constexpr int64_t kSliceRows = 256;   // rows whose slices are in the workspace at a time

struct SliceFacts {
  double sum;
  float m, bad;
  int first, unused;
};
struct SliceCut {
  double above, kept;  // sums of the weights above the bin: all of them, and those that min_p leaves
  int entries, unused;
};
struct BinEntry {
  float x;
  int index;
};

// A batch of rows and the workspace of their slices.
struct SlicedRows {
  const void *logits;
  int64_t row_stride, row0;  // first row of the batch
  int V, slices;
  const float *uniform;
  SampleSettings set;
  SliceFacts *facts;         // (rows, slices)
  unsigned long long *bins;  // (rows, slices, kSliceBins)
  int *cut_bin;              // (rows)
  SliceCut *cuts;            // (rows, slices)
  BinEntry *entries;         // (rows, slices, kBinEntries)
  bool binned, cut;          // steps 2 and 3, and step 4, are run
};

// What the slices of a row come to, the same in every wave; lane k holds slice k.
struct RowState {
  float m, T, from, per_unit;
  float slice_m;
  int slice_first;
  double slice_sum;  // of its weights, relative to m
  bool answer, greedy, cuts;
  double want;

  __device__ __forceinline__ RowState(const SlicedRows &a, int64_t r, int lane) {
    const int64_t row = a.row0 + r;
    SliceFacts f = {0.0, OT_NEG_INF, 0.f, -1, 0};
    if (lane < a.slices) f = a.facts[r * a.slices + lane];
    slice_m = f.m;
    slice_first = f.first;
    T = a.set.temperature ? a.set.temperature[row] : a.set.temperature_value;
    const float top_p = a.set.top_p ? a.set.top_p[row] : a.set.top_p_value, u = a.uniform[row];
    greedy = !(T > 0.f);
    m = group_allreduce<kWave>(f.m, MaxOp());
    const bool bad = __ballot(f.bad < 0.f) != 0;
    answer = !(bad || __builtin_isinf(m) || u != u);
    cuts = answer && !greedy && top_p < 1.f;
    slice_sum = want = 0.0;
    from = OT_NEG_INF;
    per_unit = 0.f;
    if (!answer || greedy) return;
    const Weight weight(m, T);
    slice_sum = f.sum * weight(f.m);
    if (!cuts) return;
    const double p = fmaxf(top_p, 0.f), total = wave_sum(slice_sum);
    want = p * total;
    // entries of weights below (1 - p) * total / V come to less than what lies behind the cut
    const float z = __log2f((float)fmax((1.0 - p) * total / a.V * 0.99, 1e-30)) / (float)weight.c;
    from = z > -1e30f ? fminf(m, m + 1.001f * z) : -3.4e38f;
    const float half = 0.5f * m - 0.5f * from;
    if (half > 1e-30f) per_unit = (0.5f * kSliceBins) / half;
  }
  // 0 for the largest entries; kSliceBins below `from`
  __device__ __forceinline__ int bin(float y) const {
    return y < from ? kSliceBins : (int)fminf((m - y) * per_unit, kSliceBins - 1.0f);
  }
};

template <class T>
struct Slice {
  static constexpr int VEC = kSampleVec<T>, CHUNKS = kSlice / kSliceThreads / VEC;
  typedef Sampler<T, kSliceWaves, CHUNKS> S;
  float x[CHUNKS][VEC];
  const void *base;
  int V;  // entries

  // thread t's elements: as Sampler holds them
  __device__ __forceinline__ Slice(const SlicedRows &a, int64_t r, int slice, int lane, int wave) {
    const int64_t first = (a.row0 + r) * a.row_stride + (int64_t)slice * kSlice;
    base = static_cast<const char *>(a.logits) + first * (sizeof(T) == 4 ? 4 : 2);
    V = min(kSlice, a.V - slice * kSlice);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) load_logits<T>(base, index(j, lane, wave), V, x[j]);
  }
  __device__ __forceinline__ static int index(int j, int lane, int wave) {
    return ((wave * CHUNKS + j) * kWave + lane) * VEC;
  }
};

#define OT_SLICE_GROUP                                                                              \
  __shared__ SampleShared<kSliceWaves> s_all;                                                       \
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave; \
  const RowGroup<kSliceWaves> g = {s_all, lane, wave}

template <class T>
__global__ __launch_bounds__(kSliceThreads, 4) void slice_facts_kernel(SlicedRows a) {
  typedef Slice<T> P;
  OT_SLICE_GROUP;
  const int slice = blockIdx.x;
  const int64_t r = blockIdx.y;
  const P p(a, r, slice, lane, wave);
  float m = OT_NEG_INF, bad = 0.f;
#pragma unroll
  for (int j = 0; j < P::CHUNKS; ++j)
#pragma unroll
    for (int e = 0; e < P::VEC; ++e) {
      m = fmaxf(m, p.x[j][e]);
      if (p.x[j][e] != p.x[j][e]) bad = -1.f;
    }
  g.extremes(m, bad);
  const float T_ = a.set.temperature ? a.set.temperature[a.row0 + r] : a.set.temperature_value;
  double sum = 0.0;
  int first = 0x7fffffff, none = 0;
  if (!__builtin_isinf(m)) {
#pragma unroll
    for (int j = P::CHUNKS - 1; j >= 0; --j)
#pragma unroll
      for (int e = P::VEC - 1; e >= 0; --e)
        if (p.x[j][e] == m) first = P::index(j, lane, wave) + e;
    if (T_ > 0.f) {
      const Weight weight(m, T_);
#pragma unroll
      for (int j = 0; j < P::CHUNKS; ++j) {
        double t[P::VEC];
#pragma unroll
        for (int e = 0; e < P::VEC; ++e) t[e] = weight(p.x[j][e]);
        sum += P::S::pairwise(t);
      }
    }
  }
  g.totals(sum, none);
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) first = min(first, __shfl_xor(first, d, kWave));
  g.sync();
  if (lane == 0) s_all.count[wave] = first;
  g.sync();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kSliceWaves; ++k) first = min(first, s_all.count[k]);
    a.facts[r * a.slices + slice] = {sum, m, bad, first == 0x7fffffff ? -1 : slice * kSlice + first, 0};
  }
}

template <class T>
__global__ __launch_bounds__(kSliceThreads, 4) void slice_bins_kernel(SlicedRows a) {
  typedef Slice<T> P;
  __shared__ unsigned long long s_bins[kSliceBins];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int64_t r = blockIdx.y;
  const RowState st(a, r, lane);
  if (!st.cuts) return;
  for (int i = threadIdx.x; i < kSliceBins; i += kSliceThreads) s_bins[i] = 0;
  const P p(a, r, blockIdx.x, lane, wave);
  const float per_octave = (float)Weight(st.m, st.T).c;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < P::CHUNKS; ++j)
#pragma unroll
    for (int e = 0; e < P::VEC; ++e)
      if (p.x[j][e] >= st.from) {
        // (a NaN, of a temperature that 32 bits do not hold, is 0)
        const float v = fmaxf(__builtin_amdgcn_exp2f((p.x[j][e] - st.m) * per_octave) * kBinScale, 0.f);
        atomicAdd(&s_bins[st.bin(p.x[j][e])], (unsigned long long)(unsigned)v);
      }
  __syncthreads();
  unsigned long long *to = a.bins + (r * a.slices + blockIdx.x) * kSliceBins;
  for (int i = threadIdx.x; i < kSliceBins; i += kSliceThreads) to[i] = s_bins[i];
}

// thread t looks at bin t
__global__ __launch_bounds__(kSliceBins) void slice_join_kernel(SlicedRows a) {
  constexpr int kWaves = kSliceBins / kWave;
  __shared__ unsigned long long s_sum[kWaves];
  __shared__ int s_bin;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t r = blockIdx.x;
  const RowState st(a, r, lane);
  if (!st.cuts) return;
  const unsigned long long *from = a.bins + r * a.slices * kSliceBins + threadIdx.x;
  unsigned long long amount = 0;
#pragma unroll 8
  for (int k = 0; k < a.slices; ++k) amount += from[k * kSliceBins];
  unsigned long long upto = amount;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const unsigned long long v = __shfl_up(upto, d, kWave);
    if (lane >= d) upto += v;
  }
  if (lane == kWave - 1) s_sum[wave] = upto;
  if (threadIdx.x == 0) s_bin = kSliceBins - 1;
  __syncthreads();
  for (int k = 0; k < wave; ++k) upto += s_sum[k];
  if (amount > 0 && (double)upto >= st.want * (double)kBinScale) atomicMin(&s_bin, (int)threadIdx.x);
  __syncthreads();
  if (threadIdx.x == 0) a.cut_bin[r] = s_bin;
}

template <class T>
__global__ __launch_bounds__(kSliceThreads, 4) void slice_cuts_kernel(SlicedRows a) {
  typedef Slice<T> P;
  OT_SLICE_GROUP;
  const int slice = blockIdx.x;
  const int64_t r = blockIdx.y;
  const RowState st(a, r, lane);
  if (!st.answer || st.greedy) return;
  const int cut_bin = st.cuts ? a.cut_bin[r] : kSliceBins;  // (all entries are above that)
  const P p(a, r, slice, lane, wave);
  const float min_p_row = a.set.min_p ? a.set.min_p[a.row0 + r] : a.set.min_p_value;
  const double least = min_p_row > 0.f ? fminf(min_p_row, 1.f) : 0.0;
  const Weight weight(st.m, st.T);
  double above = 0.0, kept = 0.0;
  int here = 0, none = 0;
#pragma unroll
  for (int j = 0; j < P::CHUNKS; ++j) {
    double t[P::VEC], l[P::VEC];
#pragma unroll
    for (int e = 0; e < P::VEC; ++e) {
      const float y = p.x[j][e];
      const int b = !(y > OT_NEG_INF) ? kSliceBins + 1 : st.cuts ? st.bin(y) : 0;
      t[e] = b < cut_bin ? weight(y) : 0.0;
      l[e] = t[e] >= least ? t[e] : 0.0;
      here += __popcll(__ballot(b == cut_bin));
    }
    above += P::S::pairwise(t);
    kept += P::S::pairwise(l);
  }
  g.totals(above, none);
  g.totals(kept, none);
  // entries of the bin, in index order
  __syncthreads();
  if (lane == 0) s_all.count[wave] = here;
  __syncthreads();
  int at = 0, total = 0;
  for (int k = 0; k < kSliceWaves; ++k) {
    if (k == wave) at = total;
    total += s_all.count[k];
  }
  if (st.cuts && total > 0 && total <= kBinEntries) {
    BinEntry *to = a.entries + (r * a.slices + slice) * kBinEntries;
#pragma unroll
    for (int j = 0; j < P::CHUNKS; ++j) {
      int place = at;
      bool in[P::VEC];
#pragma unroll
      for (int e = 0; e < P::VEC; ++e) {  // entries of the lanes before
        in[e] = st.bin(p.x[j][e]) == cut_bin;
        const uint64_t which = __ballot(in[e]);
        place += __builtin_amdgcn_mbcnt_hi((unsigned)(which >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)which, 0));
        at += __popcll(which);
      }
#pragma unroll
      for (int e = 0; e < P::VEC; ++e)
        if (in[e]) to[place++] = {p.x[j][e], slice * kSlice + P::index(j, lane, wave) + e};
    }
  }
  if (threadIdx.x == 0) a.cuts[r * a.slices + slice] = {above, kept, total, 0};
}

template <class T>
__global__ __launch_bounds__(kSliceThreads, 2) void slice_draw_kernel(SlicedRows a, int32_t *__restrict__ symbols,
                                                                      float *__restrict__ log_probs) {
  typedef Slice<T> P;
  OT_SLICE_GROUP;
  constexpr int kMost = 2048;  // entries of the bin of all slices
  __shared__ BinEntry s_entry[kMost];
  __shared__ double s_weight[kMost];
  __shared__ float s_cut;
  __shared__ unsigned s_best;
  __shared__ int s_last;
  const int64_t r = blockIdx.x, row = a.row0 + r;
  const RowState st(a, r, lane);
  if (!st.answer || st.greedy) {
    const uint64_t at = __ballot(st.slice_m == st.m);
    const int first = at ? lane_value(st.slice_first, __builtin_ctzll(at)) : -1;
    if (threadIdx.x == 0) {
      symbols[row] = st.answer ? first : -1;
      log_probs[row] = st.answer ? 0.f : OT_NEG_INF;
    }
    return;
  }
  const double u = a.uniform[row];
  const float min_p_row = a.set.min_p ? a.set.min_p[row] : a.set.min_p_value;
  const float top_p = a.set.top_p ? a.set.top_p[row] : a.set.top_p_value;
  const double least = min_p_row > 0.f ? fminf(min_p_row, 1.f) : 0.0;
  const Weight weight(st.m, st.T);
  SliceCut mine = {0.0, st.slice_sum, 0, 0};  // of this lane's slice
  if (a.cut) mine = lane < a.slices ? a.cuts[r * a.slices + lane] : SliceCut{0.0, 0.0, 0, 0};
  float cut = OT_NEG_INF;  // entries above it remain, and those at it up to index `last`
  int last = 0x7fffffff;
  if (st.cuts) {
    const int upto = wave_scan(mine.entries), from = upto - mine.entries, n = lane_value(upto, kWave - 1);
    const double above = wave_sum(mine.above);
    bool slow = n > kMost || __ballot(mine.entries > kBinEntries) != 0;
    if (!slow) {
      if (threadIdx.x == 0) {
        s_best = 0;
        s_last = -1;
      }
      for (int k = wave; k < a.slices; k += kSliceWaves) {
        const int to = lane_value(from, k), c = lane_value(mine.entries, k);
        for (int i = lane; i < c; i += kWave) {
          const BinEntry e = a.entries[(r * a.slices + k) * kBinEntries + i];
          s_entry[to + i] = e;
          s_weight[to + i] = weight(e.x);
        }
      }
      __syncthreads();
      // of each entry: the weights above it, the entries equal to it, and those of them before it
      constexpr int kPer = kMost / kSliceThreads;
      double sum[kPer];
      int same[kPer], earlier[kPer];
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int i = q * kSliceThreads + threadIdx.x;
        sum[q] = above;
        same[q] = earlier[q] = 0;
        if (i >= n) continue;
        const float x = s_entry[i].x;
#pragma unroll 8
        for (int k = 0; k < n; ++k) {
          const float y = s_entry[k].x;
          const double w = s_weight[k];
          sum[q] += y > x ? w : 0.0;
          same[q] += y == x;
          earlier[q] += y == x && k < i;
        }
        // the cut: the largest value that it can be at (roundings could make it two)
        if ((sum[q] < st.want || x == st.m) && sum[q] + same[q] * s_weight[i] >= st.want)
          atomicMax(&s_best, order_key(x));
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int i = q * kSliceThreads + threadIdx.x;
        if (i >= n || order_key(s_entry[i].x) != s_best) continue;
        // number `earlier` of those at the cut remains if sum + earlier * weight < want
        const float x = s_entry[i].x;
        const double w = s_weight[i], j = w > 0.0 ? ceil((st.want - sum[q]) / w) : same[q];
        const int keep = max(j < same[q] ? (int)j : same[q], x == st.m ? 1 : 0);
        if (earlier[q] == 0) s_cut = x;
        if (earlier[q] < keep) atomicMax(&s_last, s_entry[i].index);
      }
      __syncthreads();
      slow = s_best == 0;
    }
    if (slow) {
      float unused[1][P::VEC];
      const char *base = static_cast<const char *>(a.logits) + row * a.row_stride * (sizeof(T) == 4 ? 4 : 2);
      sample_row<T, kSliceWaves, 0, true>(g, base, a.V, u, st.T, 0, top_p, min_p_row, unused, symbols + row,
                                          log_probs + row);
      return;
    }
    cut = s_cut;
    last = s_last;
    // what remains of the bin in this lane's slice
    for (int i = from; i < upto; ++i) {
      const BinEntry e = s_entry[i];
      if ((e.x > cut || (e.x == cut && e.index <= last)) && s_weight[i] >= least) mine.kept += s_weight[i];
    }
  }
  // the slice in which the running sum passes the target; u >= 1: the last one with a weight
  const double run = wave_scan(mine.kept), total = lane_value(run, kWave - 1);
  const uint64_t some = __ballot(mine.kept > 0.0), pass = __ballot(mine.kept > 0.0 && run > fmax(u, 0.0) * total);
  const int slice = pass ? __builtin_ctzll(pass) : 63 - __builtin_clzll(some);
  // (the scan's sum can grow by a rounding over slices that add nothing, past the target)
  const double before = slice > 0 ? fmin(lane_value(run, slice - 1), fmax(u, 0.0) * total) : 0.0;
  P p(a, r, slice, lane, wave);
  if (st.cuts) {
#pragma unroll
    for (int j = 0; j < P::CHUNKS; ++j)
#pragma unroll
      for (int e = 0; e < P::VEC; ++e)
        if (p.x[j][e] < cut || (p.x[j][e] == cut && slice * kSlice + P::index(j, lane, wave) + e > last))
          p.x[j][e] = OT_NEG_INF;
  }
  typename P::S sampler(g, p.base, p.V, P::CHUNKS, st.m, st.T, p.x);
  sampler.weigh();
  if (least > 0.0) sampler.keep_min_p((float)least);
  const Drawn d = sampler.draw(u, before, total);
  if (threadIdx.x == 0) {
    symbols[row] = slice * kSlice + d.symbol;
    log_probs[row] = d.log_prob;
  }
}
#undef OT_SLICE_GROUP

// Bytes of workspace for a row (the arrays' elements need 8-byte alignment).
static size_t slice_row_bytes(int32_t V) {
  const size_t slices = ((size_t)V + kSlice - 1) / kSlice;
  return sizeof(int64_t) + slices * (sizeof(SliceFacts) + sizeof(SliceCut) +
                                     kSliceBins * sizeof(unsigned long long) + kBinEntries * sizeof(BinEntry));
}

template <class T>
static int launch_slices(const void *logits, int64_t row_stride, int64_t rows, int32_t V, const float *uniform,
                         const SampleSettings &set, int32_t *symbols, float *log_probs, void *workspace,
                         hipStream_t s) {
  SlicedRows a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.V = V;
  a.slices = (V + kSlice - 1) / kSlice;
  a.uniform = uniform;
  a.set = set;
  const int64_t most = rows < kSliceRows ? rows : kSliceRows;
  char *at = static_cast<char *>(workspace);
  a.facts = reinterpret_cast<SliceFacts *>(at);
  at += (size_t)most * a.slices * sizeof(SliceFacts);
  a.cuts = reinterpret_cast<SliceCut *>(at);
  at += (size_t)most * a.slices * sizeof(SliceCut);
  a.entries = reinterpret_cast<BinEntry *>(at);
  at += (size_t)most * a.slices * kBinEntries * sizeof(BinEntry);
  a.bins = reinterpret_cast<unsigned long long *>(at);
  at += (size_t)most * a.slices * kSliceBins * sizeof(unsigned long long);
  a.cut_bin = reinterpret_cast<int *>(at);
  a.binned = set.top_p || set.top_p_value < 1.f;
  a.cut = a.binned || set.min_p || set.min_p_value > 0.f;
  for (a.row0 = 0; a.row0 < rows; a.row0 += kSliceRows) {
    const unsigned n = (unsigned)(rows - a.row0 < kSliceRows ? rows - a.row0 : kSliceRows);
    const dim3 grid((unsigned)a.slices, n), block(kSliceThreads);
    hipLaunchKernelGGL((slice_facts_kernel<T>), grid, block, 0, s, a);
    if (a.binned) {
      hipLaunchKernelGGL((slice_bins_kernel<T>), grid, block, 0, s, a);
      hipLaunchKernelGGL(slice_join_kernel, dim3(n), dim3(kSliceBins), 0, s, a);
    }
    if (a.cut) hipLaunchKernelGGL((slice_cuts_kernel<T>), grid, block, 0, s, a);
    hipLaunchKernelGGL((slice_draw_kernel<T>), dim3(n), block, 0, s, a, symbols, log_probs);
  }
  return (int)hipGetLastError();
}

// Waves per SIMD: as many as leave the elements of a thread in registers.
constexpr int sample_occupancy(int waves, int elements, bool filter) {
  return waves == 16 || waves == 1 ? 4 : waves == 4 && (elements <= 16 || !filter) ? 3 : 2;
}

// ROWS groups of WAVES waves per workgroup, a row each
template <class T, int WAVES, int ROWS, int CHUNKS, bool FILTER>
__global__ __launch_bounds__(WAVES * ROWS * kWave, sample_occupancy(WAVES, CHUNKS * kSampleVec<T>, FILTER)) void
sample_kernel(
    const void *__restrict__ logits, int64_t row_stride, int64_t rows, int V, const float *__restrict__ uniform,
    SampleSettings set, int32_t *__restrict__ symbols, float *__restrict__ log_probs) {
  static_assert(ROWS == 1 || WAVES == 1, "barriers are per workgroup");
  constexpr int VEC = kSampleVec<T>;
  __shared__ SampleShared<WAVES> s_row[ROWS];
  // the wave's number in scalar registers, and with it the row and its settings
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const RowGroup<WAVES> g = {s_row[ROWS > 1 ? wave : 0], (int)(threadIdx.x % kWave), ROWS > 1 ? 0 : wave};
  float x[CHUNKS > 0 ? CHUNKS : 1][VEC];
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + (ROWS > 1 ? wave : 0); row < rows; row += stride) {
    const char *base = static_cast<const char *>(logits) + row * row_stride * (sizeof(T) == 4 ? 4 : 2);
    if constexpr (CHUNKS > 0) {
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
        load_logits<T>(base, ((g.wave * CHUNKS + j) * kWave + g.lane) * VEC, V, x[j]);
    }
    sample_row<T, WAVES, CHUNKS, FILTER>(g, base, V, (double)uniform[row],
                                         set.temperature ? set.temperature[row] : set.temperature_value,
                                         set.top_k ? set.top_k[row] : set.top_k_value,
                                         set.top_p ? set.top_p[row] : set.top_p_value,
                                         set.min_p ? set.min_p[row] : set.min_p_value, x, symbols + row,
                                         log_probs + row);
  }
}

template <class T, int WAVES, int ROWS, int CHUNKS, bool FILTER>
static int launch_sample_kernel(const void *logits, int64_t row_stride, int64_t rows, int32_t V,
                                const float *uniform, const SampleSettings &set, int32_t *symbols,
                                float *log_probs, hipStream_t s) {
  const int64_t groups = (rows + ROWS - 1) / ROWS;
  const dim3 grid((unsigned)(groups < (1 << 20) ? groups : (1 << 20)));
  hipLaunchKernelGGL((sample_kernel<T, WAVES, ROWS, CHUNKS, FILTER>), grid, dim3(WAVES * ROWS * kWave), 0, s,
                     logits, row_stride, rows, V, uniform, set, symbols, log_probs);
  return (int)hipGetLastError();
}

template <class T, int CHUNKS>
static int launch_sample_plain(const void *logits, int64_t row_stride, int64_t rows, int32_t V, const float *uniform,
                               const SampleSettings &set, int32_t *symbols, float *log_probs, hipStream_t s) {
  // 7 waves per SIMD of 256 compute units are resident; 16 rows a batch fill a line of answers.  us with
  // batches of 1, 4, 16 and 64 rows: 30 000 x 500 float32 29, 25, 24, 24, 751 992 x 500 633, 532, 503, 480,
  // 751 992 x 100 436, 352, 325, 302
  constexpr int64_t kWaves = 256 * 4 * 7;
  const int batch = (int)(rows <= kWaves ? 1 : rows >= 16 * kWaves ? 16 : (rows + kWaves - 1) / kWaves);
  const int64_t per_group = (int64_t)kWavesPerBlock * batch, groups = (rows + per_group - 1) / per_group;
  const dim3 grid((unsigned)(groups < kWaves / kWavesPerBlock ? groups : kWaves / kWavesPerBlock));
  hipLaunchKernelGGL((sample_plain_kernel<T, CHUNKS>), grid, dim3(kBlock), 0, s, logits, row_stride, rows, V, batch,
                     uniform, set.temperature, set.temperature_value, symbols, log_probs);
  return (int)hipGetLastError();
}

template <class T, bool FILTER>
static int launch_sample(const void *logits, int64_t row_stride, int64_t rows, int32_t V, const float *uniform,
                         const SampleSettings &set, int32_t *symbols, float *log_probs, hipStream_t s) {
  constexpr int VEC = kSampleVec<T>, kChunk = kWave * VEC;  // 256 or 512 elements
#define OT_SAMPLE(WAVES_, ROWS_, CHUNKS_)                                                                       \
  return launch_sample_kernel<T, WAVES_, ROWS_, CHUNKS_, FILTER>(logits, row_stride, rows, V, uniform, set, symbols, \
                                                                 log_probs, s)
#define OT_SAMPLE_FEW(WAVES_, CHUNKS_, BATCH_)                                                              \
  return launch_sample_few<T, WAVES_, CHUNKS_, BATCH_>(logits, row_stride, rows, V, uniform, set, symbols, \
                                                       log_probs, s)
  if constexpr (FILTER) {
    if (V > 2 * kChunk && !set.top_k && set.top_k_value > 0 && set.top_k_value <= kSampleFew) {
      // A batch of four rows per workgroup, a wave each for the few, where there are rows for all compute
      // units; us by one row and by four: 1024 x 2000 float32 14, 22, 2048 x 2000 26, 25, 4096 x 2000 49,
      // 36, 20 011 x 5000 float16 893, 404 (1024 x 5000 float16 47, 37 and 512 x 5000 25, 36: the border
      // is right for the shorter of them).  Longer rows take 8 or 16 waves, and one row at a time.
      if (rows >= 2048) {
        if (V <= 2048) OT_SAMPLE_FEW(4, 2048 / 4 / kChunk, 4);
        if (V <= 4096) OT_SAMPLE_FEW(4, 4096 / 4 / kChunk, 4);
        if (V <= 6144) OT_SAMPLE_FEW(4, 6144 / 4 / kChunk, 4);
      }
      if (V <= 2048) OT_SAMPLE_FEW(4, 2048 / 4 / kChunk, 1);
      if (V <= 4096) OT_SAMPLE_FEW(4, 4096 / 4 / kChunk, 1);
      if (V <= 8192) OT_SAMPLE_FEW(8, 8192 / 8 / kChunk, 1);
      if (V <= 16384) OT_SAMPLE_FEW(16, 16384 / 16 / kChunk, 1);
      OT_SAMPLE_FEW(16, 0, 1);
    }
  }
#undef OT_SAMPLE_FEW
  if constexpr (FILTER) {
    if (V <= kChunk) OT_SAMPLE(1, 4, 1);
    if (V <= 2 * kChunk) OT_SAMPLE(1, 4, 2);
  } else {
    if (V <= kChunk)
      return launch_sample_plain<T, 1>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, s);
    if (V <= 2 * kChunk)
      return launch_sample_plain<T, 2>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, s);
  }
  // (4 waves up to 6144 entries; 8 waves from 4097 on take 20 000 x 5000 float32 244 us without cuts and
  // 1172 with top_p, 4 waves 178 and 718; 64 x 5000 8 and 17 both)
  if (V <= 2048) OT_SAMPLE(4, 1, 2048 / 4 / kChunk);
  if (V <= 4096) OT_SAMPLE(4, 1, 4096 / 4 / kChunk);
  if (V <= 6144) OT_SAMPLE(4, 1, 6144 / 4 / kChunk);
  if (V <= 8192) OT_SAMPLE(8, 1, 8192 / 8 / kChunk);
  if (V <= 16384) OT_SAMPLE(16, 1, 16384 / 16 / kChunk);
  OT_SAMPLE(16, 1, 0);
#undef OT_SAMPLE
}

template <class T>
static int launch_sample(const void *logits, int64_t row_stride, int64_t rows, int32_t V, const float *uniform,
                         const SampleSettings &set, int32_t *symbols, float *log_probs, void *workspace,
                         hipStream_t s) {
  const bool with_top_p = set.top_p || set.top_p_value < 1.f, with_min_p = set.min_p || set.min_p_value > 0.f;
  // Slices or one workgroup of 16 waves (us, float32, slices first):
  //   top_p     64 x 20 000 36 / 50, 4096 x 20 000 815 / 782, 64 x 50 000 46 / 109, 4096 x 50 000
  //             1350 / 1836, 64 x 131 072 70 / 337; 64 x 16 000 (elements in registers) 35 / 37,
  //             4096 x 16 000 693 / 647
  //   no cuts   64 x 20 000 12 / 13, 4096 x 20 000 276 / 197, 64 x 50 000 14 / 26, 4096 x 50 000 415 / 467,
  //             64 x 131 072 20 / 55
  //   min_p     64 x 20 000 19 / 16, 64 x 50 000 23 / 31, 256 x 50 000 51 / 37, 64 x 131 072 35 / 66,
  //             1024 x 131 072 375 / 337
  if (workspace && (with_top_p || (V > 32768 && (!with_min_p || rows <= 128))))
    return launch_slices<T>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, workspace, s);
  const bool filter = set.top_k || with_top_p || with_min_p || (set.top_k_value > 0 && set.top_k_value < V);
  return filter ? launch_sample<T, true>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, s)
                : launch_sample<T, false>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, s);
}

}  // namespace ot

using namespace ot;

extern "C" {

size_t ot_sample_symbols_workspace_bytes(int64_t rows, int32_t V, int32_t with_top_k) {
  if (rows <= 0 || V <= kLongRow || V > kMostSlices * kSlice || with_top_k) return 0;
  return (size_t)(rows < kSliceRows ? rows : kSliceRows) * slice_row_bytes(V);
}

int ot_sample_symbols(const void *logits, int32_t dtype, int64_t row_stride, int64_t rows, int32_t V,
                      const float *uniform, const float *temperature, float temperature_value, const int32_t *top_k,
                      int32_t top_k_value, const float *top_p, float top_p_value, const float *min_p,
                      float min_p_value, int32_t *symbols, float *log_probs, void *workspace, size_t workspace_bytes,
                      void *stream) {
  if (rows == 0) return 0;
  if (!logits || !uniform || !symbols || !log_probs || rows < 0 || rows > INT32_MAX || V <= 0 ||
      V > INT32_MAX - 8192 || row_stride < 0)  // (indices of whole steps of 16 waves stay below 2^31)
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
  const size_t need =
      ot_sample_symbols_workspace_bytes(rows, V, top_k || (top_k_value > 0 && top_k_value < V));
  void *ws = need > 0 && workspace_bytes >= need ? workspace : nullptr;
  if (reinterpret_cast<uintptr_t>(ws) & 15) return OT_E_MISALIGNED;
  if (dtype == OT_DTYPE_F32)
    return launch_sample<float>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, ws, s);
  if (dtype == OT_DTYPE_F16)
    return launch_sample<F16>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, ws, s);
  if (dtype == OT_DTYPE_BF16)
    return launch_sample<BF16>(logits, row_stride, rows, V, uniform, set, symbols, log_probs, ws, s);
  return OT_E_BAD_ARG;
}

}  // extern "C"
