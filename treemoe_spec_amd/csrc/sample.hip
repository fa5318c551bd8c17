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
// One workgroup of 16 waves takes a row, up to 32768 logits in registers, more read
// again through L2.  A row is passed over two or three times: for its largest logit,
// for the first histogram, and to collect what lies above the cut's step (or min-p's
// bound) into a list in LDS, in index order.  What follows runs on the list: a few
// logits a thread where top-k or top-p leave few, the row itself where they leave
// more than the list holds.  The 64-bit exponential of a whole row, which top-p
// without top-k and plain sampling need once, is what costs most.
#include <cmath>

#include "tm_vec.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kRound = kThreads * 4;            // logits of one round: 4 consecutive a thread
constexpr int kRegRounds = 8;                   // rounds held in registers
constexpr int kBins = 2048;
constexpr int kList = 8192;                     // logits that the list holds
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
  const double* powers;  // 2^(44 + j / 32), j < 32
};

// Ordered bits: larger floats have larger keys.
__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  return u ^ (uint32_t)(((int32_t)u >> 31) | 0x80000000);
}
__device__ __forceinline__ uint64_t key_of(float l, int index) {
  return ((uint64_t)order_bits(l) << 32) | (uint32_t)~index;
}

__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

// The step of a logit, from (l_max - l) / temperature in fp32, monotone in l; -1 for
// one too far below to weigh anything.
__device__ __forceinline__ int step_of(const Row& r, float l) {
  const float d = l == r.top ? 0.0f : (r.top - l) * r.inv_t;
  return d < kSpan ? min(kBins - 1, (int)(d * ((float)kBins / kSpan))) : -1;
}

// 2^44 times the weight of a logit with a step, in 64 bits: e^z = 2^(k / 32) e^x with k
// the nearest integer to 32 z log2(e), 2^(44 + k % 32 / 32) from a table and e^x,
// |x| <= ln 2 / 64, from its Taylor polynomial of degree 5 (truncation below 3e-15).
// A logit equal to the largest weighs 1 (also infinities).
__device__ __forceinline__ double weight_of(const Row& r, float l) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to integers
  const double y = ((double)l - (double)r.top) * r.inv_y;  // 32 z log2(e), > -1443
  const double t = y + kMagic;
  const double x = (y - (t - kMagic)) * 0.021660849392498290;  // ln 2 / 32
  double q = fma(x, 8.3333333333333333e-3, 4.1666666666666667e-2);
  q = fma(q, x, 1.6666666666666667e-1);
  q = fma(q, x, 0.5);
  q = fma(q, x, 1.0);
  q = fma(q, x, 1.0);
  const int k = (int)(uint32_t)(uint64_t)__double_as_longlong(t);
  const uint64_t w = (uint64_t)__double_as_longlong(q * r.powers[k & 31]);
  const uint32_t hi = (uint32_t)(w >> 32) + ((uint32_t)(k >> 5) << 20);
  const double v = __longlong_as_double((long long)(((uint64_t)hi << 32) | (uint32_t)w));
  return l == r.top ? kUnit : v;
}
// The weight as an integer, to the nearest: the low bits of 2^52 + w.
__device__ __forceinline__ uint64_t fixed_of(double w) {
  return (uint64_t)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}

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
  uint64_t list[kList];
  uint64_t seg[kMaxRounds * kWaves];
  uint64_t wave[kWaves];
  double powers[32];
  uint64_t lo, hi, before;
  uint32_t in_bin;
  int found;
};

// Exclusive sum of v over the workgroup's threads in order, and the total.
__device__ __forceinline__ uint64_t scan_block(Shared& s, uint64_t v, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t incl = scan_wave(v, lane);
  __syncthreads();  // s.wave is free
  if (lane == 63) s.wave[wave] = incl;
  __syncthreads();
  uint64_t at = incl - v, sum = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint64_t x = s.wave[w];
    if (w < wave) at += x;
    sum += x;
  }
  *total = sum;
  return at;
}

// A row of logits.
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
  }
  static __device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
  __device__ __forceinline__ void hold() {
    if constexpr (REG) {
#pragma unroll
      for (int r = 0; r < kRegRounds; ++r)
        if (r < rounds) fetch(r, v[r]);
#pragma unroll
      for (int r = 0; r < kRegRounds; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[r][e] = r < rounds ? clean(v[r][e]) : -INFINITY;
    }
  }
  // f(round, first index, 4 logits) over the thread's logits
  template <class F>
  __device__ __forceinline__ void rounds_of(F&& f) const {
    if constexpr (REG) {
#pragma unroll
      for (int r = 0; r < kRegRounds; ++r) {
        // taken as new values, and one round at a time, so that what one pass makes of
        // them does not stay in registers for the next
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = v[r][e];
          asm volatile("" : "+v"(x[e]));
        }
        if (r < rounds) f(r, r * kRound + (int)threadIdx.x * 4, x);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      constexpr int A = 4;  // rounds read ahead
      for (int r0 = 0; r0 < rounds; r0 += A) {
        float x[A][4];
#pragma unroll
        for (int a = 0; a < A; ++a)
          if (r0 + a < rounds) fetch(r0 + a, x[a]);
#pragma unroll
        for (int a = 0; a < A; ++a)
          if (r0 + a < rounds) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[a][e] = clean(x[a][e]);
            f(r0 + a, (r0 + a) * kRound + (int)threadIdx.x * 4, x[a]);
          }
      }
    }
  }
  // f(logit, key) over the thread's logits
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    rounds_of([&](int, int i, const float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(x[e], key_of(x[e], i + e));
    });
  }
};

// The list in LDS: n keys in index order, `per` consecutive ones a thread.
struct List {
  const uint64_t* keys;
  int n, per;
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    const int end = min(n, ((int)threadIdx.x + 1) * per);
    for (int i = (int)threadIdx.x * per; i < end; ++i) f(logit_of(keys[i]), keys[i]);
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

template <bool WEIGHT>
__device__ __forceinline__ void add_to_bin(Shared& s, const Row& row, int bin, float l) {
  atomicAdd(&s.count[bin], 1u);
  if constexpr (WEIGHT)
    atomicAdd((unsigned long long*)&s.weight[bin],
              (unsigned long long)fixed_of(weight_of(row, l)));
}

// The bin at which the running measure over bins 0, 1, ... reaches a target (a number
// of elements, or the share `top_p` of the weight of all, at least 1): s.found (-1 where it
// does not), s.before the measure in front of it, s.in_bin its elements.  Returns the
// target.
template <bool WEIGHT>
__device__ __forceinline__ uint64_t find_bin(Shared& s, uint64_t target, double top_p) {
  __syncthreads();  // the bins are filled
  const int t = threadIdx.x;
  const uint64_t a = WEIGHT ? s.weight[2 * t] : (uint64_t)s.count[2 * t];
  const uint64_t b = WEIGHT ? s.weight[2 * t + 1] : (uint64_t)s.count[2 * t + 1];
  uint64_t total;
  const uint64_t at = scan_block(s, a + b, &total);
  if (target == 0) {
    const double want = ceil(top_p * (double)total);
    target = want > 1.0 ? (uint64_t)want : 1;
    target = target < total ? target : total;
  }
  if (at < target && at + a + b >= target) {  // one thread at most
    const bool second = at + a < target;
    s.found = 2 * t + (second ? 1 : 0);
    s.before = at + (second ? a : 0);
    s.in_bin = s.count[2 * t + (second ? 1 : 0)];
  }
  __syncthreads();
  return target;
}

// The key of the element of step `step` at which the running measure over the step's
// elements with key >= cut reaches `target`.
template <bool WEIGHT, class L>
__device__ uint64_t cut_in_step(Shared& s, const L& src, const Row& row, uint64_t cut, int step,
                                uint64_t target) {
  clear_bins(s);
  uint64_t lo = ~0ull, hi = 0;
  src.each([&](float l, uint64_t key) {
    if (key < cut || step_of(row, l) != step) return;
    lo = key < lo ? key : lo;
    hi = key > hi ? key : hi;
  });
  if (lo <= hi) {
    atomicMin((unsigned long long*)&s.lo, (unsigned long long)lo);
    atomicMax((unsigned long long*)&s.hi, (unsigned long long)hi);
  }
  __syncthreads();
  lo = s.lo;
  hi = s.hi;
  // every pass leaves at most 1 / 1024 of the range; one key ends it
  while (lo < hi) {
    const int shift = max(0, 53 - (int)__clzll((long long)(hi - lo)));  // range >> shift < 2048
    clear_bins(s);
    src.each([&](float l, uint64_t key) {
      if (key < lo || key > hi) return;
      add_to_bin<WEIGHT>(s, row, (int)((hi - key) >> shift), l);
    });
    find_bin<WEIGHT>(s, target, 1.0);
    const int bin = s.found;
    if (bin < 0) return lo;  // cannot be: the step holds the target
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

// First histogram over the elements with key >= cut.
template <bool WEIGHT, class L>
__device__ __forceinline__ uint64_t first_bins(Shared& s, const L& src, const Row& row,
                                               uint64_t cut, uint64_t target, double top_p) {
  clear_bins(s);
  src.each([&](float l, uint64_t key) {
    const int step = step_of(row, l);
    if (step >= 0 && key >= cut) add_to_bin<WEIGHT>(s, row, step, l);
  });
  return find_bin<WEIGHT>(s, target, top_p);
}

struct Cuts {
  int k_step, p_step;                // steps of the cuts of top-k and top-p, or kBins
  uint64_t k_target, p_target;       // within them
  bool later_p;                      // top-p is taken over what top-k keeps
  double top_p, min_w;               // min_w: 2^44 min_p
};

// The token of one source (the list, or the row): cuts, weights, and the element at
// which their running sum exceeds u times their sum.
template <class L>
__device__ __forceinline__ uint64_t cut_of(Shared& s, const L& src, const Row& row, Cuts c) {
  uint64_t cut = 0;
  if (c.k_step < kBins) cut = cut_in_step<false>(s, src, row, 0, c.k_step, c.k_target);
  if (c.later_p) {
    const uint64_t target = first_bins<true>(s, src, row, cut, 0, c.top_p);
    c.p_step = s.found;
    c.p_target = target - s.before;
  }
  if (c.p_step < kBins) {
    const uint64_t k = cut_in_step<true>(s, src, row, cut, c.p_step, c.p_target);
    cut = k > cut ? k : cut;
  }
  return cut;
}

// A kept logit's weight, or 0.
__device__ __forceinline__ double kept(const Row& row, float l, uint64_t key, uint64_t cut,
                                       double min_w) {
  if (step_of(row, l) < 0 || key < cut) return 0.0;
  const double w = weight_of(row, l);
  return w >= min_w ? w : 0.0;
}

// What the running sum has to exceed.
__device__ __forceinline__ uint64_t goal_of(float u, uint64_t total) {
  const double x = floor((u > 0.0f ? (double)u : 0.0) * (double)total);
  const uint64_t goal = (uint64_t)x;
  return x < (double)total && goal < total ? goal : total - 1;
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
  lg.hold();
  const double temp = p.temperatures ? (double)p.temperatures[n] : p.temperature;
  const float u = p.uniforms[n];
  const int top_k = p.top_ks ? p.top_ks[n] : p.top_k;
  const double top_p = p.top_ps ? (double)p.top_ps[n] : p.top_p;
  const double min_p = p.min_ps ? (double)p.min_ps[n] : p.min_p;
  float* const probs = p.probs ? p.probs + n * p.probs_stride : nullptr;
  if (t < 32) s.powers[t] = exp2((double)t / 32.0) * kUnit;

  // the first element of the order
  uint64_t best = 0;
  lg.each([&](float, uint64_t key) { best = key > best ? key : best; });
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
  row.top = logit_of(best);
  if (row.top == -INFINITY || !(temp > 0.0)) {
    // nothing to choose from, or the largest logit itself
    const int token = row.top == -INFINITY ? -1 : index_of(best);
    if (t == 0) p.tokens[n] = token;
    if (probs)
      for (int i = t; i < p.vocab; i += kThreads) probs[i] = i == token ? 1.0f : 0.0f;
    return;
  }
  row.inv_t = (float)(1.0 / temp);
  row.inv_y = 46.166241308446828384 / temp;
  row.powers = s.powers;

  const bool by_k = top_k > 0 && top_k < p.vocab, by_p = top_p < 1.0, by_m = min_p > 0.0;
  Cuts c;
  c.k_step = c.p_step = kBins;
  c.k_target = c.p_target = 0;
  c.top_p = top_p;
  c.min_w = by_m ? (min_p < 1.0 ? min_p : 1.0) * kUnit : 0.0;
  if (by_k) {
    first_bins<false>(s, lg, row, 0, (uint64_t)top_k, 1.0);
    if (s.found >= 0) {  // (fewer than k weigh anything otherwise)
      c.k_step = s.found;
      c.k_target = (uint64_t)top_k - s.before;
    }
  } else if (by_p) {
    const uint64_t target = first_bins<true>(s, lg, row, 0, 0, top_p);
    c.p_step = s.found;
    c.p_target = target - s.before;
  }
  c.later_p = by_k && by_p;
  // the last step that can be kept: that of a cut, or the one behind min-p's (whose
  // own bound is exact); top-p after top-k has to see all that top-k keeps
  int last = min(c.k_step, c.p_step);
  if (by_m && !c.later_p) {
    const float d = -logf((float)(c.min_w / kUnit));
    const int m = d < kSpan ? (int)(d * ((float)kBins / kSpan)) + 1 : kBins;
    if (m < last) {
      last = m;
      c.k_step = c.p_step = kBins;  // the cuts lie behind it
    }
  }

  // everything up to that step, in index order
  List list;
  list.keys = s.list;
  list.n = 0;
  bool listed = last < kBins;
  if (listed) {
    __syncthreads();
    lg.rounds_of([&](int r, int i, const float (&x)[4]) {
      int m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int step = step_of(row, x[e]);
        m += step >= 0 && step <= last ? 1 : 0;
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) m += __shfl_xor(m, d);
      if (lane == 0) s.seg[r * kWaves + wave] = (uint64_t)m;
    });
    __syncthreads();
    uint64_t total;
    const uint64_t mine = t < lg.rounds * kWaves ? s.seg[t] : 0;
    const uint64_t at = scan_block(s, mine, &total);
    listed = total <= (uint64_t)kList;
    if (listed) {
      __syncthreads();
      s.seg[t] = at;
      __syncthreads();
      lg.rounds_of([&](int r, int i, const float (&x)[4]) {
        const uint64_t low = ((uint64_t)1 << lane) - 1;  // lanes below this one
        int pos = (int)s.seg[r * kWaves + wave];
        bool keep[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int step = step_of(row, x[e]);
          keep[e] = step >= 0 && step <= last;
          pos += __popcll(__ballot(keep[e]) & low);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (keep[e]) s.list[pos++] = key_of(x[e], i + e);
      });
      list.n = (int)total;
      list.per = (list.n + kThreads - 1) / kThreads;
      if (probs) {
        if (((uintptr_t)probs & 15) == 0 && (p.vocab & 3) == 0) {
          const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int i = 4 * t; i < p.vocab; i += 4 * kThreads)
            *reinterpret_cast<f32x4_t*>(probs + i) = zero;
        } else {
          for (int i = t; i < p.vocab; i += kThreads) probs[i] = 0.0f;
        }
      }
      __syncthreads();
    }
  }

  if (listed) {
    const uint64_t cut = cut_of(s, list, row, c);
    uint64_t sum = 0, total;
    list.each([&](float l, uint64_t key) { sum += fixed_of(kept(row, l, key, cut, c.min_w)); });
    uint64_t run = scan_block(s, sum, &total);
    const uint64_t goal = goal_of(u, total);
    const double inv = 1.0 / (double)total;
    const bool here = run <= goal && goal < run + sum;  // one thread's
    if (here || probs)
      list.each([&](float l, uint64_t key) {
        const double w = kept(row, l, key, cut, c.min_w);
        if (probs && w > 0.0) probs[index_of(key)] = (float)(w * inv);
        const uint64_t f = fixed_of(w);
        if (here && run <= goal && goal < run + f) p.tokens[n] = index_of(key);
        run += f;
      });
    return;
  }

  const uint64_t cut = cut_of(s, lg, row, c);
  // sums of 256 consecutive indices: a wave's part of a round
  __syncthreads();
  lg.rounds_of([&](int r, int i, const float (&x)[4]) {
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      sum += fixed_of(kept(row, x[e], key_of(x[e], i + e), cut, c.min_w));
    sum = sum_wave(sum);
    if (lane == 0) s.seg[r * kWaves + wave] = sum;
  });
  __syncthreads();
  const uint64_t mine = t < lg.rounds * kWaves ? s.seg[t] : 0;
  uint64_t total;
  const uint64_t at = scan_block(s, mine, &total);
  const uint64_t goal = goal_of(u, total);
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
      l[e] = lg.clean(l[e]);
      w[e] = fixed_of(kept(row, l[e], key_of(l[e], i + e), cut, c.min_w));
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
    const double inv = 1.0 / (double)total;
    lg.rounds_of([&](int, int i, const float (&l)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < p.vocab)
          probs[i + e] = (float)(kept(row, l[e], key_of(l[e], i + e), cut, c.min_w) * inv);
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
