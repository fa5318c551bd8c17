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
// again through L2; a wave owns consecutive indices.  All that can be kept lies above a
// value that is found cheaply: min-p's own bound, or one that some k of the 1024
// threads' largest logits reach, since then k logits do.  What lies above goes into a
// list in LDS, in index order, and the rest runs on the list: up to 256 elements are
// ranked by counting, more are cut by histograms.  top-p without top-k needs the weight
// of the whole row, one pass of 64-bit exponentials; where the list turns out to hold
// too little of it, or overflows, the row itself is cut by histograms.  The form with a row
// in registers spills 16 of 128 a thread (52 bytes) beside its 32 logits.
//
// Bound by latency at few rows and by passes over a row on one CU: 1 row of 32000, top-k 50
// and top-p, 10.7 us; 64 rows with top-p, min-p and their distributions 21.7; 256 rows of
// 131072 with top-p 92 us, 29 of them the first reading (HBM, 4.7 TB/s), 18 the second, 14
// the 64-bit exponentials.  Rows that do not start on four logits, as with a vocabulary that
// is no multiple of 4, take a load a logit: 64 rows in a graph, top-k 50, of 32000 11.6 us,
// of 32001 16.4; of 131072 26.4, of 131073 64.3.
#include <cmath>
#include <type_traits>

#include "tm_vec.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kRound = kThreads * 4;            // logits of one round: 4 consecutive a thread
constexpr int kRegRounds = 8;                   // rounds held in registers
constexpr int kBins = 2048;
constexpr int kList = 1024;                     // logits of a wave that the list holds
// Up to so many elements of the list in all are ranked by counting, up to 64 of them by one
// wave.  Measured (fp32, 32000 logits), in us: 64 rows, top-k 50, ranked 11.2, by the
// histograms 15.0; top-k 200 and top-p 16.6, 20.5; 1 row, top-k 50 and top-p, by one wave
// 10.6, by the workgroup 12.7.
constexpr int kRank = 256;
constexpr int kRankStep = 8;                    // so many at a time
constexpr float kSpan = 31.25f;                 // (l_max - l) / temperature of the last bin's end
constexpr float kMaxF32 = 3.402823466e38f;      // the largest finite float
constexpr double kUnit = 17592186044416.0;      // 2^44
constexpr double kTwo52 = 4503599627370496.0;   // where doubles are integers

// 2^(44 + j / 32)
__constant__ const double kPowers[32] = {
    0x1.0000000000000p+44, 0x1.059b0d3158574p+44, 0x1.0b5586cf9890fp+44, 0x1.11301d0125b51p+44,
    0x1.172b83c7d517bp+44, 0x1.1d4873168b9aap+44, 0x1.2387a6e756238p+44, 0x1.29e9df51fdee1p+44,
    0x1.306fe0a31b715p+44, 0x1.371a7373aa9cbp+44, 0x1.3dea64c123422p+44, 0x1.44e086061892dp+44,
    0x1.4bfdad5362a27p+44, 0x1.5342b569d4f82p+44, 0x1.5ab07dd485429p+44, 0x1.6247eb03a5585p+44,
    0x1.6a09e667f3bcdp+44, 0x1.71f75e8ec5f74p+44, 0x1.7a11473eb0187p+44, 0x1.82589994cce13p+44,
    0x1.8ace5422aa0dbp+44, 0x1.93737b0cdc5e5p+44, 0x1.9c49182a3f090p+44, 0x1.a5503b23e255dp+44,
    0x1.ae89f995ad3adp+44, 0x1.b7f76f2fb5e47p+44, 0x1.c199bdd85529cp+44, 0x1.cb720dcef9069p+44,
    0x1.d5818dcfba487p+44, 0x1.dfc97337b9b5fp+44, 0x1.ea4afa2a490dap+44, 0x1.f50765b6e4540p+44};

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
  float half_top;  // half of it
  float inv_t;     // 1 / temperature
  double inv_y;    // 32 log2(e) / temperature
  double deepest;  // l_max - l at which the weight is 0 for long
  const double* powers;  // 2^(44 + j / 32), j < 32
};

// Ordered bits: larger floats have larger keys.
__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 as +0
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
// one too far below to weigh anything.  By half of that: finite logits can lie further
// apart than the largest float, and have a weight at temperatures near it.
__device__ __forceinline__ int step_of(const Row& r, float l) {
  const float half = l == r.top ? 0.0f : fmaf(l, -0.5f, r.half_top) * r.inv_t;
  return half < 0.5f * kSpan ? min(kBins - 1, (int)(half * (2.0f * (float)kBins / kSpan))) : -1;
}

// 2^44 times the weight of a logit, in 64 bits: with d = l_max - l and t = 32 d log2(e) /
// temperature, e^(-d / temperature) = 2^(-k / 32) e^x for k the integer nearest to t
// and x = (k - t) ln 2 / 32, |x| <= ln 2 / 64: 2^(44 + j / 32) from a table, e^x from its
// Taylor polynomial of degree 5 (truncation below 3e-15).  d is clamped to where the
// weight is far below 1/2.
__device__ __forceinline__ double weight_of(const Row& r, float l) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to integers
  constexpr double c = 0.021660849392498290;     // ln 2 / 32
  const double d = fmin((double)r.top - (double)l, r.deepest);
  const double t = fma(d, -r.inv_y, kMagic);
  const double x = fma(d, -r.inv_y, kMagic - t);
  double q = fma(x, c * c * c * c * c / 120.0, c * c * c * c / 24.0);
  q = fma(q, x, c * c * c / 6.0);
  q = fma(q, x, c * c / 2.0);
  q = fma(q, x, c);
  q = fma(q, x, 1.0);
  const int k = (int)(uint32_t)(uint64_t)__double_as_longlong(t);
  return ldexp(q * r.powers[k & 31], k >> 5);
}
// The weight as an integer, to the nearest: the low bits of 2^52 + w.
__device__ __forceinline__ uint64_t fixed_of(double w) {
  return (uint64_t)__double_as_longlong(w + kTwo52) & 0xfffffffffffffull;
}

// The value DPP moves into a lane: v of another lane of the wave, 0 where none is.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t plus_moved(uint64_t v) {
  return v + (((uint64_t)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) |
              moved<CTRL, ROWS>((uint32_t)v));
}
// Inclusive sum over the lanes of a wave: within rows of 16 lanes, then row to row.
__device__ __forceinline__ uint64_t scan_wave(uint64_t v) {
  v = plus_moved<0x111, 0xf>(v);  // 1, 2, 4 and 8 lanes up
  v = plus_moved<0x112, 0xf>(v);
  v = plus_moved<0x114, 0xf>(v);
  v = plus_moved<0x118, 0xf>(v);
  v = plus_moved<0x142, 0xa>(v);  // lane 15 of a row to the next row
  return plus_moved<0x143, 0xc>(v);  // lane 31 to the upper half
}
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}

struct Shared {
  uint64_t list[kWaves][kList];  // each wave's elements
  uint64_t weight[kBins];
  uint32_t count[kBins];
  uint64_t wave[kWaves];
  double powers[32];
  uint64_t lo, hi, before;
  uint32_t in_bin;
  int found;
};

// Exclusive sum of v over the workgroup's threads in order, and the total.
__device__ __forceinline__ uint64_t scan_block(Shared& s, uint64_t v, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t incl = scan_wave(v);
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
  bool infinite = false;

  // Round r of wave w: indices 256 (w rounds + r) .., 4 consecutive a lane.
  __device__ __forceinline__ int base_at(int r) const {
    return (__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) * rounds + r) * 256;
  }
  __device__ __forceinline__ int index_at(int r) const {
    return base_at(r) + (int)(threadIdx.x & 63) * 4;
  }
  // The thread's 4 logits of round r; what lies past the end as -inf.
  __device__ __forceinline__ void fetch(int r, float (&x)[4]) const {
    const int base = base_at(r), lane4 = (int)(threadIdx.x & 63) * 4;
    if (aligned && base + 256 <= vocab) {
      if constexpr (DT == TM_DTYPE_F32) {
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(
            reinterpret_cast<const float*>(row) + base + lane4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e];
      } else {
        const u16x4_t a = *reinterpret_cast<const u16x4_t*>(
            reinterpret_cast<const uint16_t*>(row) + base + lane4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = Half16<DT>::to_f32(a[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = base + lane4 + e;
        x[e] = i < vocab ? tm_load1<DT>(row, i) : -INFINITY;
      }
    }
  }
  // NaN as -inf; where +inf is the largest logit, those as 0 and all others as -inf.
  __device__ __forceinline__ float clean(float x) const {
    x = fmaxf(x, -INFINITY);
    return !infinite ? x : x == INFINITY ? 0.0f : -INFINITY;
  }
  __device__ __forceinline__ void make_infinite() {
    infinite = true;
    if constexpr (REG) {
#pragma unroll
      for (int r = 0; r < kRegRounds; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[r][e] = clean(v[r][e]);
    }
  }
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
        if (r < rounds) f(r, index_at(r), x);
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
            f(r0 + a, index_at(r0 + a), x[a]);
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

// The list in LDS: each wave's keys in index order, consecutive ones a lane.
struct List {
  const uint64_t* keys;  // this wave's
  int n;
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    const int per = (n + 63) / 64, lane = (int)threadIdx.x & 63;
    const int end = min(n, (lane + 1) * per);
    for (int i = lane * per; i < end; ++i) f(logit_of(keys[i]), keys[i]);
  }
};

template <bool WEIGHT>
__device__ __forceinline__ void clear_bins(Shared& s) {
  __syncthreads();  // the last reads are over
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    if (WEIGHT) s.weight[i] = 0;
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
  clear_bins<false>(s);
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
    clear_bins<WEIGHT>(s);
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

// Gathers a wave's chosen elements of a round into its list, in index order; `count` goes on
// where they no longer fit.
__device__ __forceinline__ void gather(uint64_t* list, const bool (&in)[4], const float (&x)[4],
                                       int i, int& count) {
  uint64_t m[4];
  int more = 0, before = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = __ballot(in[e]);
    more += __popcll(m[e]);
    before += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m[e] >> 32),
                                             __builtin_amdgcn_mbcnt_lo((uint32_t)m[e], 0u));
  }
  if (count + more <= kList) {
    int at = count + before;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (in[e]) list[at++] = key_of(x[e], i + e);
  }
  count += more;
}

// cut_in_step of a row, on a list of the step's elements where they fit: one pass over the
// row in place of two or three.  128 rows of 131072 flat logits: top-k 2000 181 -> 125 us,
// top-p 253 -> 221.
template <bool WEIGHT, class L>
__device__ __forceinline__ uint64_t cut_in_listed_step(Shared& s, const L& src, const Row& row,
                                                       uint64_t cut, int step, uint64_t target) {
  if constexpr (!std::is_same_v<L, List>) {
    const int wave = (int)(threadIdx.x >> 6);
    int count = 0;
    src.rounds_of([&](int, int i, const float (&x)[4]) {
      bool in[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        in[e] = step_of(row, x[e]) == step && key_of(x[e], i + e) >= cut;
      if (__any(in[0] || in[1] || in[2] || in[3])) gather(s.list[wave], in, x, i, count);
    });
    if (__syncthreads_count(count > kList) == 0)
      return cut_in_step<WEIGHT>(s, List{s.list[wave], count}, row, cut, step, target);
  }
  return cut_in_step<WEIGHT>(s, src, row, cut, step, target);
}

// First histogram over the elements with key >= cut.
template <bool WEIGHT, class L>
__device__ __forceinline__ uint64_t first_bins(Shared& s, const L& src, const Row& row,
                                               uint64_t cut, uint64_t target, double top_p) {
  clear_bins<WEIGHT>(s);
  src.each([&](float l, uint64_t key) {
    const int step = step_of(row, l);
    if (step >= 0 && key >= cut) add_to_bin<WEIGHT>(s, row, step, l);
  });
  return find_bin<WEIGHT>(s, target, top_p);
}

struct Filter {
  bool by_k, by_p;
  uint64_t k;
  double top_p, min_w;   // min_w: 2^44 min_p
  uint64_t p_target;     // top-p's target where it is known (without top-k), or 0
};

// The smallest key that top-k and top-p keep of the elements of `src` (0: all).
template <class L>
__device__ __forceinline__ uint64_t cut_of(Shared& s, const L& src, const Row& row,
                                           const Filter& f) {
  uint64_t cut = 0;
  if (f.by_k) {
    first_bins<false>(s, src, row, 0, f.k, 1.0);
    const int step = s.found;
    // (fewer than k weigh anything otherwise)
    if (step >= 0) cut = cut_in_listed_step<false>(s, src, row, 0, step, f.k - s.before);
  }
  if (f.by_p) {
    const uint64_t target = first_bins<true>(s, src, row, cut, f.p_target, f.top_p);
    const int step = s.found;
    if (step >= 0) {
      const uint64_t c = cut_in_listed_step<true>(s, src, row, cut, step, target - s.before);
      cut = c > cut ? c : cut;
    }
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

// The largest of v over the workgroup.
__device__ __forceinline__ float max_block(Shared& s, float v) {
#define TM_MAX(ctrl, rows)                                                                \
  v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(                     \
                   (int)__float_as_uint(v), (int)__float_as_uint(v), ctrl, rows, 0xf, false)))
  TM_MAX(0x111, 0xf);
  TM_MAX(0x112, 0xf);
  TM_MAX(0x114, 0xf);
  TM_MAX(0x118, 0xf);
  TM_MAX(0x142, 0xa);
  TM_MAX(0x143, 0xc);
#undef TM_MAX
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.wave[threadIdx.x >> 6] = __float_as_uint(v);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = fmaxf(v, __uint_as_float((uint32_t)s.wave[w]));
  return v;
}

// The logit `depth` temperatures below the largest, or a little less: 2^-19 of the terms
// covers the roundings here and in step_of, a few 2^-24 of them.  Above -infinity.
__device__ __forceinline__ float below(const Row& row, float depth) {
  const float d = depth / row.inv_t;
  return fmaxf(row.top - d - 1.9e-6f * (d + fabsf(row.top)), -kMaxF32);
}

// A value that at least `k` (<= 1024) of the threads' `most` reach, the lowest one where
// fewer of them weigh anything.
__device__ __forceinline__ float reached_by(Shared& s, const Row& row, float most, int k) {
  clear_bins<false>(s);
  const int step = step_of(row, most);
  if (step >= 0) atomicAdd(&s.count[step], 1u);
  find_bin<false>(s, (uint64_t)k, 1.0);
  if (s.found < 0) return -kMaxF32;
  return below(row, (float)(s.found + 1) * (kSpan / (float)kBins));
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
  const double power = kPowers[t & 31];
  lg.hold();
  // (a row's infinite one as the largest; NaN stays, which takes the largest logit)
  const float row_temp = p.temperatures ? p.temperatures[n] : 0.0f;
  double temp = p.temperatures ? (double)(row_temp > kMaxF32 ? kMaxF32 : row_temp)
                               : p.temperature;
  const float u = p.uniforms[n];
  const int top_k = p.top_ks ? p.top_ks[n] : p.top_k;
  const double top_p = p.top_ps ? (double)p.top_ps[n] : p.top_p;
  const double min_p = p.min_ps ? (double)p.min_ps[n] : p.min_p;
  float* const probs = p.probs ? p.probs + n * p.probs_stride : nullptr;
  if (t < 32) s.powers[t] = power;

  float most = -INFINITY;  // of this thread's logits
  lg.rounds_of([&](int, int, const float (&x)[4]) {
    most = fmaxf(fmaxf(fmaxf(most, x[0]), fmaxf(x[1], x[2])), x[3]);
  });
  Row row;
  row.top = max_block(s, most);
  if (row.top == -INFINITY || !(temp > 0.0)) {
    // nothing to choose from, or the first of the largest logits
    if (t == 0) s.lo = ~0ull;
    __syncthreads();
    if (most == row.top && row.top != -INFINITY) {
      int at = INT32_MAX;
      lg.rounds_of([&](int, int i, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x[e] == row.top && i + e < at) at = i + e;
      });
      atomicMin((unsigned long long*)&s.lo, (unsigned long long)at);
    }
    __syncthreads();
    const int token = s.lo == ~0ull ? -1 : (int)s.lo;
    if (t == 0) p.tokens[n] = token;
    if (probs)
      for (int i = t; i < p.vocab; i += kThreads) probs[i] = i == token ? 1.0f : 0.0f;
    return;
  }
  // its inverse finite, and 32.5 of it: from 1e300 on all finite logits weigh the same, while
  // an infinite `deepest` would make NaN of the weight of -inf
  temp = fmin(fmax(temp, 1e-300), 1e300);
  row.inv_t = (float)(1.0 / temp);
  if (row.top == INFINITY) {
    lg.make_infinite();
    most = most == INFINITY ? 0.0f : -INFINITY;
    row.top = 0.0f;
  }
  row.half_top = 0.5f * row.top;
  row.inv_y = 46.166241308446828384 / temp;
  row.deepest = 32.5 * temp;  // 2^44 e^-32.5 < 0.14
  row.powers = s.powers;

  Filter f;
  f.by_k = top_k > 0 && top_k < p.vocab;
  f.by_p = top_p < 1.0;
  f.k = (uint64_t)(f.by_k ? top_k : 0);
  f.top_p = top_p;
  f.p_target = 0;
  const bool by_m = min_p > 0.0;
  f.min_w = by_m ? (min_p < 1.0 ? min_p : 1.0) * kUnit : 0.0;

  // a value above which all lies that can be kept, where one is known beforehand
  bool listed = true;
  float above = 0.0f;
  if (f.by_k && top_k <= kThreads) {
    above = reached_by(s, row, most, top_k);
  } else if (f.by_k) {
    listed = false;
  } else if (by_m) {
    above = below(row, 1e-6f - logf((float)(f.min_w / kUnit)));
  } else if (f.by_p) {
    // most of the row's weight in all likelihood: all but two threads hold a logit
    // as large, so some 6000 are
    above = reached_by(s, row, most, kThreads - 2);
  } else {
    listed = false;
  }
  // the list, and for top-p without top-k the whole row's weight
  List list;
  list.keys = s.list[wave];
  list.n = 0;
  const bool whole = f.by_p && !f.by_k;
  if (listed || whole) {
    int count = 0;           // of this wave
    double sum = kTwo52;     // of this thread: whole numbers, each weight rounded to one
    lg.rounds_of([&](int, int i, const float (&x)[4]) {
      if (whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += weight_of(row, x[e]);
      }
      if (!listed) return;
      if (!__any(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= above)) return;
      bool in[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] = x[e] >= above;
      gather(s.list[wave], in, x, i, count);
    });
    if (listed) {
      list.n = min(count, kList);
      listed = __syncthreads_count(count > kList) == 0;
    }
    if (whole) {
      uint64_t total;
      scan_block(s, (uint64_t)(sum - kTwo52), &total);
      const double want = ceil(top_p * (double)total);
      f.p_target = want > 1.0 ? (uint64_t)want : 1;
      f.p_target = f.p_target < total ? f.p_target : total;
    }
  }
  if (listed && whole) {
    // whether the cut of top-p lies in the list
    uint64_t sum = 0, total;
    list.each([&](float l, uint64_t key) { sum += fixed_of(kept(row, l, key, 0, f.min_w)); });
    scan_block(s, sum, &total);
    if (total < f.p_target) {
      if (by_m)
        f.by_p = false;  // it lies behind min-p's
      else
        listed = false;
    }
  }

  if (listed) {
    if (probs) {
      if (((uintptr_t)probs & 15) == 0) {
        const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
        const int even = p.vocab & ~3;
        for (int i = 4 * t; i < even; i += 4 * kThreads)
          *reinterpret_cast<f32x4_t*>(probs + i) = zero;
        if (even + t < p.vocab) probs[even + t] = 0.0f;
      } else {
        for (int i = t; i < p.vocab; i += kThreads) probs[i] = 0.0f;
      }
    }
    uint64_t all;
    const uint64_t first = scan_block(s, lane == 63 ? (uint64_t)list.n : 0, &all);
    const int n_all = (int)all;
    if (n_all <= kRank) {
      // the waves' elements one after the other, in s.weight; then a thread each
      for (int i = lane; i < list.n; i += 64) s.weight[(int)first + i] = list.keys[i];
      if (t < kRankStep) s.weight[n_all + t] = 0;
      __syncthreads();  // (also: the zeros before the kept probabilities)
      if (n_all <= 64) {
        // one wave, without further barriers
        if (wave > 0) return;
        const uint64_t key = t < n_all ? s.weight[t] : 0;
        int rank = 0;
        for (int j = 0; j < n_all; j += kRankStep)
#pragma unroll
          for (int e = 0; e < kRankStep; ++e) rank += s.weight[j + e] > key ? 1 : 0;
        double wd = t < n_all ? kept(row, logit_of(key), key, 0, 0.0) : 0.0;
        uint64_t w = fixed_of(wd);
        int keep = f.by_k && f.k < (uint64_t)n_all ? (int)f.k : n_all;
        if (f.by_p) {
          // the order's weights, exchanged through LDS within the wave
          if (t < n_all) s.list[0][rank] = w;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          const uint64_t o = t < keep ? s.list[0][t] : 0;
          const uint64_t upto = scan_wave(o);
          if (f.p_target == 0) {
            const double want = ceil(top_p * (double)last_lane(upto));
            f.p_target = want > 1.0 ? (uint64_t)want : 1;
          }
          keep = __popcll(__ballot(t < keep && upto - o < f.p_target));
        }
        if (rank >= keep || wd < f.min_w) {
          wd = 0.0;
          w = 0;
        }
        const uint64_t upto = scan_wave(w);
        const uint64_t total = last_lane(upto), run = upto - w;
        const uint64_t goal = goal_of(u, total);
        if (run <= goal && goal < upto) p.tokens[n] = index_of(key);
        if (probs && w > 0) probs[index_of(key)] = (float)(wd / (double)total);
        return;
      }
      uint64_t key = 0, w = 0;
      double wd = 0.0;
      int rank = 0;
      if (t < n_all) {
        key = s.weight[t];
        for (int j = 0; j < n_all; j += kRankStep)
#pragma unroll
          for (int e = 0; e < kRankStep; ++e) rank += s.weight[j + e] > key ? 1 : 0;
        wd = kept(row, logit_of(key), key, 0, 0.0);
        w = fixed_of(wd);
        s.list[0][rank] = w;  // the order's weights
      }
      const int keep_k = f.by_k && f.k < (uint64_t)n_all ? (int)f.k : n_all;
      int keep = keep_k;
      if (f.by_p) {
        __syncthreads();
        uint64_t total;
        const uint64_t before = scan_block(s, t < keep_k ? s.list[0][t] : 0, &total);
        if (f.p_target == 0) {
          const double want = ceil(top_p * (double)total);
          f.p_target = want > 1.0 ? (uint64_t)want : 1;
        }
        keep = __syncthreads_count(t < keep_k && before < f.p_target);
      }
      if (rank >= keep || wd < f.min_w) {
        wd = 0.0;
        w = 0;
      }
      uint64_t total;
      const uint64_t run = scan_block(s, w, &total);
      const uint64_t goal = goal_of(u, total);
      if (run <= goal && goal < run + w) p.tokens[n] = index_of(key);
      if (probs && w > 0) probs[index_of(key)] = (float)(wd / (double)total);
      return;
    }
    __syncthreads();  // the zeros before the kept probabilities
    const uint64_t cut = cut_of(s, list, row, f);
    uint64_t sum = 0, total;
    list.each([&](float l, uint64_t key) { sum += fixed_of(kept(row, l, key, cut, f.min_w)); });
    uint64_t run = scan_block(s, sum, &total);
    const uint64_t goal = goal_of(u, total);
    const double inv = 1.0 / (double)total;
    const bool here = run <= goal && goal < run + sum;  // one thread's
    if (here || probs)
      list.each([&](float l, uint64_t key) {
        const double w = kept(row, l, key, cut, f.min_w);
        if (probs && w > 0.0) probs[index_of(key)] = (float)(w * inv);
        const uint64_t x = fixed_of(w);
        if (here && run <= goal && goal < run + x) p.tokens[n] = index_of(key);
        run += x;
      });
    return;
  }

  const uint64_t cut = cut_of(s, lg, row, f);
  uint64_t sum = 0, total;
  lg.each([&](float l, uint64_t key) { sum += fixed_of(kept(row, l, key, cut, f.min_w)); });
  // a wave's indices are consecutive: its sum, then the round, then the lane
  const uint64_t mine = last_lane(scan_wave(sum));
  // (counted at the wave's last lane, so every lane has the waves before it)
  uint64_t from = scan_block(s, lane == 63 ? mine : 0, &total);
  const uint64_t goal = goal_of(u, total);
  if (from <= goal && goal < from + mine) {
    for (int r = 0; r < lg.rounds; ++r) {
      float l[4];
      lg.fetch(r, l);
      const int i = lg.index_at(r);
      uint64_t w[4], four = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        l[e] = lg.clean(l[e]);
        w[e] = fixed_of(kept(row, l[e], key_of(l[e], i + e), cut, f.min_w));
        four += w[e];
      }
      const uint64_t upto = scan_wave(four);
      uint64_t x = from + upto - four;
      if (x <= goal && goal < x + four) {
        int token = i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (x <= goal && goal < x + w[e]) token = i + e;
          x += w[e];
        }
        p.tokens[n] = token;
      }
      from += last_lane(upto);
      if (from > goal) break;
    }
  }
  if (probs) {
    const double inv = 1.0 / (double)total;
    lg.rounds_of([&](int, int i, const float (&l)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < p.vocab)
          probs[i + e] = (float)(kept(row, l[e], key_of(l[e], i + e), cut, f.min_w) * inv);
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
  if (N < 0 || N > TM_MAX_ROWS || V < 1 || V > TM_MAX_SAMPLE_VOCAB) return TM_ERR_SHAPE;
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
