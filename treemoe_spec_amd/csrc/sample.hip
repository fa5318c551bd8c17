// One token of every row of logits from a given uniform number, after temperature,
// top-k, top-p and min-p, and the filtered distribution where asked.
//
// With l_max the row's largest logit, w_i = exp((l_i - l_max) / temperature) and the
// order "larger logit first, lower index first among equals":
//   top-k  keeps the first k of the order;
//   top-p  keeps the shortest prefix of those whose weight reaches p of theirs;
//   min-p  keeps what weighs at least min_p (l_max weighs 1);
//   token  the first index, in index order, at which the running sum of the kept
//          weights exceeds u times their sum.
//
// Arithmetic.  Weights are taken in 64 bits and summed as integers, multiples of
// 2^-44: integer sums do not depend on their order, so histograms may be filled by
// LDS atomics and every result is the same on every run.  Up to 2^18 weights of at
// most 1 fit 62 bits.  A weight below 2^-45 (logits over 31.2 temperatures under
// the largest) is 0.
//
// The order's cut, for top-k and top-p alike, is the element at which a running
// measure (count, or weight) reaches a target.  It is found from histograms: first
// over 2048 equal steps of (l_max - l) / temperature, in which few logits share a
// step, then within the step over the 64-bit keys (ordered bits of l, inverted
// index), all distinct, in 2048 steps of the remaining range at a time.
//
// One workgroup of 16 waves takes a row.  Up to 32768 logits it holds them in
// registers between its passes, above that it reads them again through L2.
#include <cmath>

#include "tm_vec.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kRound = kThreads * 4;            // logits of one round: 4 consecutive a thread
constexpr int kRegRounds = 8;                   // rounds held in registers
constexpr int kBins = 2048;
constexpr int kMaxRounds = TM_MAX_SAMPLE_VOCAB / kRound;
constexpr float kSpan = 31.25f;                 // (l_max - l) / temperature of the last bin's end
constexpr double kUnit = 17592186044416.0;      // 2^44

struct SampleParams {
  const void* logits;
  int64_t row_stride;
  const float* uniforms;
  const float *temperatures, *top_ps, *min_ps;  // one a row, or NULL
  const int32_t* top_ks;
  double temperature, top_p, min_p;             // otherwise
  int top_k;
  int vocab;
  int aligned;                                  // rows start on 4 elements
  int64_t* tokens;
  float* probs;                                 // [N, V] or NULL
  int64_t probs_stride;
};

struct Row {
  float top;       // largest logit
  float inv_t;     // 1 / temperature
  double inv_y;    // 32 log2(e) / temperature
  const double* powers;  // 2^(j / 32), j < 32
};

// Ordered bits: larger floats have larger keys.
__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  return u ^ (uint32_t)(((int32_t)u >> 31) | 0x80000000);
}
__device__ __forceinline__ uint64_t key_of(float l, int index) {
  return ((uint64_t)order_bits(l) << 32) | (uint32_t)~index;
}

// (l_max - l) / temperature in fp32, monotone in l; a logit is a candidate where
// it is below kSpan.
__device__ __forceinline__ float depth_of(const Row& r, float l) {
  return l == r.top ? 0.0f : (r.top - l) * r.inv_t;
}

// The weight of a candidate in 64 bits: e^z = 2^(k / 32) e^r with k the nearest integer
// to 32 z log2(e), 2^(k % 32 / 32) from a table and e^r, |r| <= ln 2 / 64, from its
// Taylor polynomial of degree 5 (truncation below 3e-15).  A logit equal to the
// largest weighs 1 (also infinities).
__device__ __forceinline__ double weight_of(const Row& r, float l) {
  const double y = ((double)l - (double)r.top) * r.inv_y;  // 32 z log2(e), > -1443
  const double kd = rint(y);
  const double x = (y - kd) * 0.021660849392498290;  // ln 2 / 32
  double q = fma(x, 8.3333333333333333e-3, 4.1666666666666667e-2);
  q = fma(q, x, 1.6666666666666667e-1);
  q = fma(q, x, 0.5);
  q = fma(q, x, 1.0);
  q = fma(q, x, 1.0);
  const int k = (int)kd;
  const double w = q * r.powers[k & 31];
  const uint64_t bits = (uint64_t)__double_as_longlong(w) + ((uint64_t)(int64_t)(k >> 5) << 52);
  return l == r.top ? 1.0 : __longlong_as_double((long long)bits);
}
__device__ __forceinline__ uint64_t fixed_of(double w) { return (uint64_t)(w * kUnit + 0.5); }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, m);
  const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), m);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, d);
  const uint32_t hi = (uint32_t)__shfl_up((int)(uint32_t)(v >> 32), d);
  return ((uint64_t)hi << 32) | lo;
}
// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ uint64_t scan_wave(uint64_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = shfl_up64(v, d);
    if (lane >= d) v += o;
  }
  return v;
}
__device__ __forceinline__ uint64_t sum_wave(uint64_t v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += shfl_xor64(v, m);
  return v;
}

struct Shared {
  uint64_t weight[kBins];
  uint32_t count[kBins];
  uint64_t seg[kMaxRounds * kWaves];
  uint64_t wave[kWaves];
  double powers[32];
  uint64_t lo, hi, before;
  uint32_t in_bin;
  int found;
};

template <int DT, bool REG>
struct Logits {
  float v[REG ? kRegRounds : 1][4];
  const void* row;
  int vocab, rounds;
  bool aligned;

  // The thread's 4 logits of round r; NaN and what lies past the end as -inf,
  // -0 as +0.
  __device__ __forceinline__ void fetch(int r, float (&x)[4]) const {
    const int i = r * kRound + (int)threadIdx.x * 4;
    if (aligned && i + 4 <= vocab) {
      if constexpr (DT == TM_DTYPE_F32) {
        const f32x4_t a =
            *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(row) + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e];
      } else {
        const u16x4_t a =
            *reinterpret_cast<const u16x4_t*>(reinterpret_cast<const uint16_t*>(row) + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = Half16<DT>::to_f32(a[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = i + e < vocab ? tm_load1<DT>(row, i + e) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = x[e] == x[e] ? x[e] + 0.0f : -INFINITY;
  }
  // f(round, first index, 4 logits) over the thread's logits
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    if constexpr (REG) {
#pragma unroll
      for (int r = 0; r < kRegRounds; ++r)
        if (r < rounds) f(r, r * kRound + (int)threadIdx.x * 4, v[r]);
    } else {
      for (int r = 0; r < rounds; ++r) {
        float x[4];
        fetch(r, x);
        f(r, r * kRound + (int)threadIdx.x * 4, x);
      }
    }
  }
};

__device__ __forceinline__ void clear_bins(Shared& s) {
  __syncthreads();  // the last reads are over
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.weight[i] = 0;
    s.count[i] = 0;
  }
  if (threadIdx.x == 0) {
    s.found = -1;
    s.lo = ~0ull;
    s.hi = 0;
  }
  __syncthreads();
}

// The bin at which the running measure over bins 0, 1, ... reaches `target` (>= 1):
// s.found (-1 where it does not), s.before the measure in front of it, s.in_bin its
// elements.
template <bool WEIGHT>
__device__ __forceinline__ void find_bin(Shared& s, uint64_t target) {
  __syncthreads();  // the bins are filled
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const uint64_t a = WEIGHT ? s.weight[2 * t] : (uint64_t)s.count[2 * t];
  const uint64_t b = WEIGHT ? s.weight[2 * t + 1] : (uint64_t)s.count[2 * t + 1];
  const uint64_t incl = scan_wave(a + b, lane);
  if (lane == 63) s.wave[wave] = incl;
  __syncthreads();
  uint64_t at = incl - (a + b);
  for (int w = 0; w < wave; ++w) at += s.wave[w];
  if (at < target && at + a + b >= target) {  // one thread at most
    const bool second = at + a < target;
    s.found = 2 * t + (second ? 1 : 0);
    s.before = at + (second ? a : 0);
    s.in_bin = s.count[2 * t + (second ? 1 : 0)];
  }
  __syncthreads();
}

// The key of the element at which the running measure of the candidates with
// key >= cut reaches `target`; 0 where it does not (everything stays).
template <bool WEIGHT, class L>
__device__ uint64_t cut_at(Shared& s, const L& lg, const Row& row, uint64_t cut,
                           uint64_t target) {
  constexpr float kScale = (float)kBins / kSpan;
  clear_bins(s);
  lg.each([&](int, int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = depth_of(row, x[e]);
      if (!(d < kSpan) || key_of(x[e], i + e) < cut) continue;
      const int bin = min(kBins - 1, (int)(d * kScale));
      atomicAdd(&s.count[bin], 1u);
      if constexpr (WEIGHT)
        atomicAdd((unsigned long long*)&s.weight[bin],
                  (unsigned long long)fixed_of(weight_of(row, x[e])));
    }
  });
  find_bin<WEIGHT>(s, target);
  const int step = s.found;
  if (step < 0) return 0;
  target -= s.before;
  // the keys of the step's elements
  uint64_t lo = ~0ull, hi = 0;
  lg.each([&](int, int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = depth_of(row, x[e]);
      const uint64_t key = key_of(x[e], i + e);
      if (!(d < kSpan) || key < cut || min(kBins - 1, (int)(d * kScale)) != step) continue;
      lo = key < lo ? key : lo;
      hi = key > hi ? key : hi;
    }
  });
  if (lo <= hi) {
    atomicMin((unsigned long long*)&s.lo, (unsigned long long)lo);
    atomicMax((unsigned long long*)&s.hi, (unsigned long long)hi);
  }
  __syncthreads();
  lo = s.lo;
  hi = s.hi;
  // every round leaves at most 1 / 1024 of the range; one key ends it
  while (lo < hi) {
    const int shift = max(0, 53 - (int)__clzll((long long)(hi - lo)));  // range >> shift < 2048
    clear_bins(s);
    lg.each([&](int, int i, const float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t key = key_of(x[e], i + e);
        if (key < lo || key > hi || !(depth_of(row, x[e]) < kSpan)) continue;
        const int bin = (int)((hi - key) >> shift);
        atomicAdd(&s.count[bin], 1u);
        if constexpr (WEIGHT)
          atomicAdd((unsigned long long*)&s.weight[bin],
                    (unsigned long long)fixed_of(weight_of(row, x[e])));
      }
    });
    find_bin<WEIGHT>(s, target);
    const int bin = s.found;
    if (bin < 0) return lo;  // not reached by rounding of the target: all of the step stays
    target -= s.before;
    const uint32_t n = s.in_bin;
    const uint64_t top = hi - ((uint64_t)bin << shift);
    const uint64_t width = ((uint64_t)1 << shift) - 1;
    const uint64_t low = top - lo > width ? top - width : lo;
    if (n == 1) return low;  // the one element of the bin is the last that stays
    lo = low;
    hi = top;
  }
  return lo;
}

template <int DT, bool REG>
__global__ void __launch_bounds__(kThreads) tm_sample_kernel(SampleParams p) {
  __shared__ Shared s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t n = blockIdx.x;
  Logits<DT, REG> lg;
  lg.row = reinterpret_cast<const uint8_t*>(p.logits) +
           n * p.row_stride * (DT == TM_DTYPE_F32 ? 4 : 2);
  lg.vocab = p.vocab;
  lg.rounds = (p.vocab + kRound - 1) / kRound;
  lg.aligned = p.aligned != 0;
  if constexpr (REG) {
#pragma unroll
    for (int r = 0; r < kRegRounds; ++r) {
      if (r < lg.rounds) {
        lg.fetch(r, lg.v[r]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) lg.v[r][e] = -INFINITY;
      }
    }
  }
  // the first element of the order
  uint64_t best = 0;
  lg.each([&](int, int i, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t key = key_of(x[e], i + e);
      best = key > best ? key : best;
    }
  });
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    const uint64_t o = shfl_xor64(best, m);
    best = o > best ? o : best;
  }
  if (lane == 0) s.wave[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) best = s.wave[w] > best ? s.wave[w] : best;

  Row row;
  const uint32_t ob = (uint32_t)(best >> 32);
  row.top = __uint_as_float(ob ^ ((ob >> 31) ? 0x80000000u : 0xffffffffu));
  const double temp = p.temperatures ? (double)p.temperatures[n] : p.temperature;
  const float u = p.uniforms[n];
  const int top_k = p.top_ks ? p.top_ks[n] : p.top_k;
  const double top_p = p.top_ps ? (double)p.top_ps[n] : p.top_p;
  const double min_p = p.min_ps ? (double)p.min_ps[n] : p.min_p;
  float* const probs = p.probs ? p.probs + n * p.probs_stride : nullptr;

  const int first = (int)~(uint32_t)best;
  if (row.top == -INFINITY || !(temp > 0.0)) {
    // nothing to choose from, or the largest logit itself
    const int token = row.top == -INFINITY ? -1 : first;
    if (t == 0) p.tokens[n] = token;
    if (probs)
      for (int i = t; i < p.vocab; i += kThreads) probs[i] = i == token ? 1.0f : 0.0f;
    return;
  }
  row.inv_t = (float)(1.0 / temp);
  row.inv_y = 46.166241308446828384 / temp;
  row.powers = s.powers;
  if (t < 32) s.powers[t] = exp2((double)t / 32.0);
  __syncthreads();

  uint64_t cut = 0;
  if (top_k > 0 && top_k < p.vocab) cut = cut_at<false>(s, lg, row, cut, (uint64_t)top_k);
  if (top_p < 1.0) {
    uint64_t sum = 0;
    lg.each([&](int, int i, const float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (depth_of(row, x[e]) < kSpan && key_of(x[e], i + e) >= cut)
          sum += fixed_of(weight_of(row, x[e]));
    });
    sum = sum_wave(sum);
    __syncthreads();
    if (lane == 0) s.wave[wave] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += s.wave[w];
    const double want = ceil(top_p * (double)sum);
    const uint64_t target = want > 1.0 ? (uint64_t)want : 1;
    const uint64_t c = cut_at<true>(s, lg, row, cut, target < sum ? target : sum);
    cut = c > cut ? c : cut;
  }

  // sums of 256 consecutive indices: a wave's part of a round
  const double floor_w = min_p > 0.0 ? (min_p < 1.0 ? min_p : 1.0) : 0.0;
  auto kept = [&](float x, int i) -> double {
    if (!(depth_of(row, x) < kSpan) || key_of(x, i) < cut) return 0.0;
    const double w = weight_of(row, x);
    return w >= floor_w ? w : 0.0;
  };
  __syncthreads();
  lg.each([&](int r, int i, const float (&x)[4]) {
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += fixed_of(kept(x[e], i + e));
    sum = sum_wave(sum);
    if (lane == 0) s.seg[r * kWaves + wave] = sum;
  });
  __syncthreads();
  const int segs = lg.rounds * kWaves;  // at most kThreads
  const uint64_t mine = t < segs ? s.seg[t] : 0;
  const uint64_t incl = scan_wave(mine, lane);
  if (lane == 63) s.wave[wave] = incl;
  __syncthreads();
  uint64_t at = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) at += s.wave[w];
    total += s.wave[w];
  }
  double x = floor((u > 0.0f ? (double)u : 0.0) * (double)total);
  uint64_t goal = (uint64_t)x;  // the running sum has to exceed it
  if (!(x < (double)total) || goal >= total) goal = total - 1;
  if (at <= goal && goal < at + mine) {
    s.found = t;
    s.before = at;
  }
  __syncthreads();
  const int seg = s.found;
  if (seg % kWaves == wave) {
    float l[4];
    const int r = seg / kWaves;
    lg.fetch(r, l);
    const int i = r * kRound + t * 4;
    uint64_t w[4], four = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = fixed_of(kept(l[e], i + e));
      four += w[e];
    }
    uint64_t run = s.before + scan_wave(four, lane) - four;
    if (run <= goal && goal < run + four) {
      int token = i;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (run <= goal && goal < run + w[e]) token = i + e;
        run += w[e];
      }
      p.tokens[n] = token;
    }
  }
  if (probs) {
    const double inv = kUnit / (double)total;
    lg.each([&](int, int i, const float (&l)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < p.vocab) probs[i + e] = (float)(kept(l[e], i + e) * inv);
    });
  }
}

}  // namespace

extern "C" int tm_sample_tokens(const void* logits, int dtype, int64_t N, int64_t V,
                                int64_t row_stride, const float* uniforms,
                                const float* temperatures, double temperature,
                                const int32_t* top_ks, int64_t top_k, const float* top_ps,
                                double top_p, const float* min_ps, double min_p,
                                int64_t* tokens,
                                float* probs, int64_t probs_stride, void* stream) {
  if (!tm_dtype_ok(dtype)) return TM_ERR_ARG;
  if (!temperatures && !(temperature >= 0.0 && temperature < INFINITY)) return TM_ERR_ARG;
  if (!top_ks && top_k < 0) return TM_ERR_ARG;
  if (!top_ps && !(top_p >= 0.0 && top_p <= 1.0)) return TM_ERR_ARG;
  if (!min_ps && !(min_p >= 0.0 && min_p <= 1.0)) return TM_ERR_ARG;
  if (N < 0 || N > INT32_MAX || V < 1 || V > TM_MAX_SAMPLE_VOCAB) return TM_ERR_SHAPE;
  if (N == 0) return TM_OK;
  if (N > 1 && (row_stride < 0 || (probs && probs_stride < V))) return TM_ERR_SHAPE;
  const int64_t es = tm_dtype_bytes(dtype);
  if ((uintptr_t)logits % es || (uintptr_t)uniforms % 4 || (uintptr_t)tokens % 8 ||
      (uintptr_t)probs % 4 || (uintptr_t)temperatures % 4 || (uintptr_t)top_ks % 4 ||
      (uintptr_t)top_ps % 4 || (uintptr_t)min_ps % 4)
    return TM_ERR_ALIGN;
  SampleParams p;
  p.logits = logits;
  p.row_stride = row_stride;
  p.uniforms = uniforms;
  p.temperatures = temperatures;
  p.top_ps = top_ps;
  p.min_ps = min_ps;
  p.top_ks = top_ks;
  p.temperature = temperature;
  p.top_p = top_p;
  p.min_p = min_p;
  p.top_k = (int)(top_k < V ? top_k : V);
  p.vocab = (int)V;
  p.aligned = (uintptr_t)logits % (4 * es) == 0 && (N == 1 || row_stride % 4 == 0);
  p.tokens = tokens;
  p.probs = probs;
  p.probs_stride = probs_stride;
  const bool reg = V <= kRegRounds * kRound;
  const dim3 grid((unsigned)N), block(kThreads);
  const hipStream_t st = (hipStream_t)stream;
#define TM_SAMPLE(DT)                                                        \
  if (reg)                                                                   \
    hipLaunchKernelGGL((tm_sample_kernel<DT, true>), grid, block, 0, st, p); \
  else                                                                       \
    hipLaunchKernelGGL((tm_sample_kernel<DT, false>), grid, block, 0, st, p)
  if (dtype == TM_DTYPE_BF16) {
    TM_SAMPLE(TM_DTYPE_BF16);
  } else if (dtype == TM_DTYPE_F16) {
    TM_SAMPLE(TM_DTYPE_F16);
  } else {
    TM_SAMPLE(TM_DTYPE_F32);
  }
#undef TM_SAMPLE
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}
