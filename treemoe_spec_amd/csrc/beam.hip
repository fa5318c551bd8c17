// Beam search's selection over beams and vocabulary, and the reordering of what the
// beams hold.
//
// Of a group's K beams with scores s_b and logits l_b, the candidates are (b, v) with
//   s_b + l_b[v] - log sum_u exp l_b[u],
// and one (b, pad) with s_b for a beam that has finished.  The `num` best come out in
// order: larger score first, of equal ones the lower beam, then the larger logit, then
// the lower token.
//
// Arithmetic.  Scores are formed in 64 bits, the sum of the exponentials too (each off by 2e-13
// at most), so that beams are not exchanged by the rounding of 32; each score is rounded to fp32
// once, when it is written.  Within a beam the order is that of the logits, so a row is cut to
// its best `num` before any score is known.
//
// A workgroup takes 4096 or 8192 logits of a row: their sum, and their best `num` as sorted
// keys (ordered bits of the logit, inverted token), all distinct.  At least `num` logits reach
// the num-th largest of the 256 threads' largest, and only the `num` threads that reach it hold
// such: the list never overflows.  Then one workgroup a group joins the sums and ranks the
// lists' heads.  Entry i of the list whose head is the r-th has r + i above it: what is left
// when that is `num` or more, and what lies below the num-th head, cannot come out; the rest
// is ranked by counting.
//
// Bound by instructions at many logits, the 64-bit exponentials 10 of 40 us (256 rows of 131072
// in 37 us and the join 7, 67 MB), and by chains of barriers and latencies at few: 4 rows of
// 32000 7.5 and 5 us.
#include <cmath>

#include "tm_vec.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// Logits of a lane, 256 times as many of a workgroup, which leaves one list.  What a list costs
// (bound, barriers, ranks, the join) is the same whatever it stands for: many where the chip
// is full anyway.  Selection in us with 16, 32 and 64 (graph replays, with the reorder): 256
// rows of 131072 bf16 59, 52, 51; 64 rows 32, 28, 27; 1024 of 32000 fp32 56, 54, 54; 256 of
// 32000 bf16 27, 28, 32; 4 of 32000 fp32 15, 17, 20.
constexpr int kFewPer = 16, kManyPer = 32;
constexpr int kMaxNum = TM_MAX_BEAMS;
constexpr int kJoin = 512;               // threads of a group's workgroup, a list each

struct BeamParams {
  const void* logits;
  int64_t row_stride;
  const float* scores;
  const uint8_t* finished;  // or NULL
  int64_t pad_token;
  uint64_t* lists;          // [rows][segs][num], sorted, 0 behind the last
  double* sums;             // [rows][segs]
  float* tops;              // [rows][segs]
  int rows, beams, vocab, segs, num;
  int aligned;              // rows start on 16 bytes
  float* out_scores;
  int32_t* parents;
  int64_t* tokens;
};

// Ordered bits: larger floats have larger keys.
__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 as +0
  return u ^ (uint32_t)(((int32_t)u >> 31) | 0x80000000);
}
__device__ __forceinline__ float float_of(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float l, int index) {
  return ((uint64_t)order_bits(l) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ int lanes_before(uint64_t ballot) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0));
}

// The logits base + index_of(e) of a lane; what lies past the end, and NaN, as -inf.  Rows that do
// not start on 16 bytes come an element at a time: 256 rows of 131072 in bf16 75 us, aligned
// 52; of 50257 44, 35; 4 of 50257 17, 15.
template <int DT>
__device__ __forceinline__ int index_of(int e) {
  constexpr int kVec = DT == TM_DTYPE_F32 ? 4 : 8;
  return e / kVec * 64 * kVec + (int)(threadIdx.x & 63) * kVec + e % kVec;
}
template <int DT, int kPer>
__device__ __forceinline__ void fetch(const BeamParams& p, int64_t row, int base,
                                      float (&x)[kPer]) {
  if (p.aligned && base + 64 * kPer <= p.vocab) {
#pragma unroll
    for (int c = 0; c < kPer / 8; ++c) {
      if constexpr (DT == TM_DTYPE_F32) {
        const float* const from = reinterpret_cast<const float*>(p.logits) + row * p.row_stride;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4_t a =
              *reinterpret_cast<const f32x4_t*>(from + base + index_of<DT>(8 * c + 4 * h));
#pragma unroll
          for (int e = 0; e < 4; ++e) x[8 * c + 4 * h + e] = a[e];
        }
      } else {
        float v[8];
        tm_load8<DT>(reinterpret_cast<const uint16_t*>(p.logits) + row * p.row_stride,
                     base + index_of<DT>(8 * c), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[8 * c + e] = v[e];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = base + index_of<DT>(e);
      x[e] = i < p.vocab ? tm_load1<DT>(p.logits, row * p.row_stride + i) : -INFINITY;
    }
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = fmaxf(x[e], -INFINITY);
}

// 2^(j / 64)
__constant__ const double kPowers[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

// e^d for d <= 0, in 64 bits: with t = 64 d log2(e) and k the integer nearest to it,
// 2^(k / 64) e^x, x = d - k ln 2 / 64, |x| <= ln 2 / 128: 2^(j / 64) from a table, e^x from
// its Taylor polynomial of degree 4 (truncation below 4e-14; the rounding of t, largest at -700,
// brings it to 2e-13).  Below -700 it is e^-700.
// A library exponential, with its wider range and half an ulp, takes three times as long.
__device__ __forceinline__ double exp_of(double d, const double* powers) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to integers
  constexpr double c = 0.010830424696249145;     // ln 2 / 64
  const double y = fmax(d, -700.0) * 92.332482616893657;
  const double t = y + kMagic;
  const double x = y - (t - kMagic);
  double q = fma(x, c * c * c * c / 24.0, c * c * c / 6.0);
  q = fma(q, x, c * c / 2.0);
  q = fma(q, x, c);
  q = fma(q, x, 1.0);
  const int k = (int)(uint32_t)(uint64_t)__double_as_longlong(t);
  // (times 2^(k / 64) by the exponent: it stays above -1011)
  return __longlong_as_double(__double_as_longlong(q * powers[k & 63]) +
                              ((int64_t)(k >> 6) << 52));
}

// The largest value from lo to hi that num or more reach, all reaching lo, or one that just
// num reach.  `reach`: how many reach a value.
template <class REACH>
__device__ __forceinline__ uint32_t last_reached(uint32_t lo, uint32_t hi, int num, REACH&& reach) {
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    const int count = reach(mid);
    if (count == num) return mid;
    if (count > num)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A bound that just num of the threads' keys reach, by one wave: of the logits' ordered bits, and
// where the logits there are equal of the tokens first .. last, inverted.
__device__ __forceinline__ uint64_t least_of(const uint64_t (&keys)[kThreads], float top, int num,
                                             int first, int last) {
  uint32_t logit[kWaves], token[kWaves];
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const uint64_t k = keys[64 * i + (threadIdx.x & 63)];
    logit[i] = (uint32_t)(k >> 32);
    token[i] = (uint32_t)k;
  }
  auto reach = [&](uint32_t v) {
    int count = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) count += __popcll(__ballot(logit[i] >= v));
    return count;
  };
  const uint32_t lowest = 0x007fffffu;  // -inf: all reach it
  const uint32_t v = last_reached(lowest, order_bits(top), num, reach);
  if (reach(v) == num) return (uint64_t)v << 32;
  const int need = num - reach(v + 1);
  const uint32_t t =
      last_reached(~(uint32_t)last, ~(uint32_t)first, need, [&](uint32_t u) {
        int count = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i)
          count += __popcll(__ballot(logit[i] == v && token[i] >= u));
        return count;
      });
  return ((uint64_t)v << 32) | t;
}

template <int DT, int kPer>
__global__ void __launch_bounds__(kThreads) tm_beam_rows_kernel(BeamParams p) {
  extern __shared__ uint64_t s_list[];  // [num * kPer]
  __shared__ uint64_t s_key[kThreads];
  __shared__ uint64_t s_least;
  __shared__ double s_sum[kWaves];
  __shared__ float s_top[kWaves];
  __shared__ int s_count;
  __shared__ double s_powers[64];
  const int tid = threadIdx.x, lane = tid & 63, num = p.num;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = blockIdx.x;
  const int row = (int)(unit / p.segs), seg = (int)(unit - (int64_t)row * p.segs);
  if (p.finished != nullptr && p.finished[row]) return;
  const int first = seg * kThreads * kPer, base = first + wave * 64 * kPer;
  uint64_t* const out = p.lists + unit * num;
  float x[kPer];
  fetch<DT, kPer>(p, row, base, x);
  if (tid < 64) s_powers[tid] = kPowers[tid];
  if (tid == 0) s_count = 0;
  float top = x[0];
#pragma unroll
  for (int e = 1; e < kPer; ++e) top = fmaxf(top, x[e]);
  int at = 0;  // of the lane's largest, the lowest index
#pragma unroll
  for (int e = kPer - 1; e >= 0; --e) at = x[e] == top ? index_of<DT>(e) : at;
  s_key[tid] = key_of(top, base + at);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) s_top[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_top[w]);
  if (top == -INFINITY) {  // no candidate, and no weight
    if (tid < num) out[tid] = 0;
    if (tid == 0) {
      p.sums[unit] = 0.0;
      p.tops[unit] = top;
    }
    return;
  }
  // one wave finds what reaches the num-th largest of the threads' largest, while the others
  // have begun with the sum
  if (wave == 0) {
    const uint64_t least = least_of(s_key, top, num, first, first + kThreads * kPer - 1);
    if (lane == 0) s_least = least;
  }
  double part[2] = {0.0, 0.0};
  if (top < INFINITY) {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      part[e & 1] += exp_of((double)x[e] - (double)top, s_powers);
  } else {  // infinite ones weigh 1, and all finite ones nothing
#pragma unroll
    for (int e = 0; e < kPer; ++e) part[e & 1] += x[e] == top ? 1.0 : 0.0;
  }
  double sum = part[0] + part[1];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  const uint64_t least = s_least;
  const float least_logit = float_of((uint32_t)(least >> 32));
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (!__any(x[e] >= least_logit)) continue;
    const uint64_t k = key_of(x[e], base + index_of<DT>(e));
    const bool in = k >= least && x[e] > -INFINITY;
    const uint64_t who = __ballot(in);
    int to = 0;
    if (lane == 0) to = atomicAdd(&s_count, __popcll(who));
    to = __builtin_amdgcn_readfirstlane(to);
    if (in) s_list[to + lanes_before(who)] = k;
  }
  __syncthreads();
  // in order, by neighbouring lanes a key: as many as the workgroup has
  const int n = s_count;
  int P = 64;
  while (P > 1 && P * n > kThreads) P /= 2;
  for (int e0 = 0; e0 < n; e0 += kThreads / P) {
    const int e = e0 + tid / P;
    const uint64_t k = e < n ? s_list[e] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = tid & (P - 1); j < n; j += P) rank += s_list[j] > k ? 1 : 0;
    for (int d = 1; d < P; d <<= 1) rank += __shfl_xor(rank, d);
    if ((tid & (P - 1)) == 0 && e < n && rank < num) out[rank] = k;
  }
  if (tid >= n && tid < num) out[tid] = 0;
  if (tid == 0) {
    p.sums[unit] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    p.tops[unit] = top;
  }
}

// A candidate: ordered bits of its score, then the beam (inverted), the logit's ordered
// bits and the token (inverted).  {0, 0}: none.
struct Cand {
  uint64_t hi, lo;
};
__device__ __forceinline__ bool above(const Cand& a, const Cand& b) {
  return a.hi > b.hi || (a.hi == b.hi && a.lo > b.lo);
}
constexpr int kTokenBits = 18;
static_assert(TM_MAX_SAMPLE_VOCAB == 1 << kTokenBits, "a token in the low bits");
static_assert(TM_MAX_BEAMS <= 64, "a beam in six bits, a lane a candidate");

__device__ __forceinline__ uint64_t order_bits64(double d) {
  const uint64_t u = (uint64_t)__double_as_longlong(d + 0.0);
  return u ^ (uint64_t)(((int64_t)u >> 63) | (int64_t)0x8000000000000000);
}
__device__ __forceinline__ double double_of(uint64_t o) {
  return __longlong_as_double((long long)(o ^ ((o >> 63) ? 0x8000000000000000ull : ~0ull)));
}
__device__ __forceinline__ Cand cand_of(double score, int beam, uint32_t logit, uint32_t token) {
  if (!(score > -INFINITY)) return {0, 0};
  return {order_bits64(score), ((uint64_t)(63 - beam) << (32 + kTokenBits)) |
                                   ((uint64_t)logit << kTokenBits) |
                                   (((1u << kTokenBits) - 1) - token)};
}

// Neighbouring lanes that count for one of n entries: as many as the workgroup has.
__device__ __forceinline__ int lanes_of(int n) {
  int P = 64;
  while (P > 1 && P * n > kJoin) P /= 2;
  return P;
}
// How many of n candidates are above c, which P lanes have.
__device__ __forceinline__ int rank_of(const Cand* all, int n, const Cand& c, int P) {
  int rank = 0;
#pragma unroll 4
  for (int j = (int)threadIdx.x & (P - 1); j < n; j += P) rank += above(all[j], c) ? 1 : 0;
  for (int d = 1; d < P; d <<= 1) rank += __shfl_xor(rank, d);
  return rank;
}

constexpr int kSteps = 128;     // lists up to which further entries bound what can come out
constexpr int kLevels = 6;      // entries 0, 1, 3, 7, 15, 31 of a list

template <bool STEPS>
struct JoinShared {
  Cand pool[kMaxNum * (kMaxNum + 1) / 2 + kMaxNum];
  Cand heads[kJoin];
  Cand steps[STEPS ? kLevels - 1 : 1][STEPS ? kSteps : 1];
  Cand best[kMaxNum];               // so far, sorted
  double base[TM_MAX_BEAMS];        // score - log of the sum, -inf for a beam without candidates
  double powers[64];
  float top[TM_MAX_BEAMS];
  Cand least[kLevels];              // the num-th of the heads, and so on
  int list[kMaxNum];                // the lists in their heads' order
  int count;                        // of the pool
};

// STEPS: few lists for many to come out.  Their heads bound little, entry i of num / (i + 1)
// lists as well bounds more: 32 of 32 lists 69 us, so 35; but up to 16 are ranked sooner than
// bounded (8 of 16 lists 17, so 20).
template <bool STEPS>
__global__ void __launch_bounds__(kJoin) tm_beam_join_kernel(BeamParams p) {
  __shared__ JoinShared<STEPS> s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = blockIdx.x, K = p.beams, num = p.num;
  const int64_t row0 = (int64_t)group * K;
  const int lists = K * p.segs;
  const uint64_t* const from = p.lists + row0 * p.segs * num;
  // (of a finished beam nothing is there, and what is read is not used)
  uint64_t head_key = tid < lists ? from[(int64_t)tid * num] : 0;
  int levels = 1;
  uint64_t step_key[kLevels - 1];
  if constexpr (STEPS) {
    while (levels < kLevels && (1 << levels) <= num) ++levels;
#pragma unroll
    for (int l = 1; l < kLevels; ++l)
      step_key[l - 1] = l < levels && tid < lists ? from[(int64_t)tid * num + (1 << l) - 1] : 0;
  }

  if (tid < 64) s.powers[tid] = kPowers[tid];
  if (tid < num) s.best[tid] = {0, 0};
  __syncthreads();
  // each beam's sum over its segments, a wave a beam
  for (int b = wave; b < K; b += kJoin / 64) {
    const int64_t at = (row0 + b) * p.segs;
    const bool over = p.finished != nullptr && p.finished[row0 + b];
    float top = -INFINITY;
    double sum = 0.0;
    // (what a finished beam's rows left there is not used)
    float t = -INFINITY;
    double u = 0.0;
    if (lane < p.segs) {
      t = p.tops[at + lane];
      u = p.sums[at + lane];
    }
    const double score = p.scores[row0 + b];
    if (!over) {
      top = t;
      for (int i = lane + 64; i < p.segs; i += 64) top = fmaxf(top, p.tops[at + i]);
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      for (int i = lane; i < p.segs; i += 64) {
        if (i > lane) {
          t = p.tops[at + i];
          u = p.sums[at + i];
        }
        if (t == top)
          sum += u;
        else if (t > -INFINITY && top < INFINITY)
          sum += u * exp_of((double)t - (double)top, s.powers);
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    }
    if (lane == 0) {
      s.top[b] = top;
      s.base[b] = top > -INFINITY && score > -INFINITY ? score - log(sum) : -INFINITY;
    }
  }
  // the finished beams are the best so far
  if (wave == 0 && p.finished != nullptr) {
    Cand c = {0, 0};
    if (lane < K && p.finished[row0 + lane])
      c = cand_of(p.scores[row0 + lane], lane, 0, (uint32_t)p.pad_token);
    int rank = 0;
    for (int l = 0; l < K; ++l) rank += above({lane_of(c.hi, l), lane_of(c.lo, l)}, c) ? 1 : 0;
    if (c.hi != 0 && rank < num) s.best[rank] = c;
  }

  auto cand = [&](int beam, uint64_t key) {
    const double base = s.base[beam];
    const float l = float_of((uint32_t)(key >> 32)), top = s.top[beam];
    // (l - top is 0 for equal infinities)
    const double score = l == top ? base : base + ((double)l - (double)top);
    return key == 0 || !(base > -INFINITY)
               ? Cand{0, 0}
               : cand_of(score, beam, (uint32_t)(key >> 32), ~(uint32_t)key);
  };
  for (int first = 0; first < lists; first += kJoin) {
    const int now = min(lists - first, kJoin);
    if (tid < num) s.list[tid] = -1;
    if (tid < kLevels) s.least[tid] = {0, 1};  // fewer heads than num: nothing lies below
    if (tid == 0) s.count = 0;
    __syncthreads();  // the sums, and the best so far
    // the heads' order, by lanes_of(now) lanes a head
    if (tid < now) {
      const int beam = (first + tid) / p.segs;
      s.heads[tid] = cand(beam, first == 0 ? head_key : from[(int64_t)(first + tid) * num]);
      if constexpr (STEPS) {
#pragma unroll
        for (int l = 1; l < kLevels; ++l)
          if (l < levels) s.steps[l - 1][tid] = cand(beam, step_key[l - 1]);
      }
    }
    __syncthreads();
    {
      const int P = lanes_of(now), h = tid / P;
      const Cand head = h < now ? s.heads[h] : Cand{0, 0};
      const int rank = rank_of(s.heads, now, head, P);
      if ((tid & (P - 1)) == 0 && head.hi != 0 && rank < num) {
        s.list[rank] = first + h;
        if (rank == num - 1) s.least[0] = head;
      }
      if constexpr (STEPS)
        for (int l = 1; l < levels; ++l) {
          const Cand c = h < now ? s.steps[l - 1][h] : Cand{0, 0};
          const int at = rank_of(s.steps[l - 1], now, c, P);
          if ((tid & (P - 1)) == 0 && c.hi != 0 && at == (num + (1 << l) - 1) / (1 << l) - 1)
            s.least[l] = c;
        }
    }
    __syncthreads();
    // what can come out, in any order
    Cand least = s.least[0];
    if constexpr (STEPS)
      for (int l = 1; l < levels; ++l)
        if (above(s.least[l], least)) least = s.least[l];
    for (int e = tid; e < num * num + num; e += kJoin) {
      const int r = e / num, i = e - r * num;
      Cand c = {0, 0};
      if (r == num) {
        c = s.best[i];
      } else if (r + i < num && s.list[r] >= 0) {
        const int list = s.list[r];
        c = cand(list / p.segs, from[(int64_t)list * num + i]);
        if (above(least, c)) c = {0, 0};
      }
      if (c.hi != 0) s.pool[atomicAdd(&s.count, 1)] = c;
    }
    __syncthreads();
    const int count = s.count;
    if (tid < num && tid >= count) s.best[tid] = {0, 0};
    const int P = lanes_of(count);
    for (int e0 = 0; e0 < count; e0 += kJoin / P) {
      const int e = e0 + tid / P;
      const Cand c = e < count ? s.pool[e] : Cand{0, 0};
      const int r = rank_of(s.pool, count, c, P);
      if ((tid & (P - 1)) == 0 && e < count && r < num) s.best[r] = c;
    }
    __syncthreads();
  }
  if (tid < num) {
    const Cand c = s.best[tid];
    const int64_t at = (int64_t)group * num + tid;
    const bool none = c.hi == 0;
    p.out_scores[at] = none ? -INFINITY : (float)double_of(c.hi);
    p.parents[at] = none ? -1 : 63 - (int)(c.lo >> (32 + kTokenBits));
    p.tokens[at] = none ? -1 : (int64_t)(((1u << kTokenBits) - 1) -
                                         (uint32_t)(c.lo & ((1u << kTokenBits) - 1)));
  }
}

// ---------------------------------------------------------------- reorder --

constexpr int kReorderPieces = 4096;  // of a workgroup

struct ReorderParams {
  const uint8_t* x;
  uint8_t* out;
  int64_t x_stride, out_stride, width;  // bytes
  const int32_t* parents;
  int64_t parents_stride;
  int beams;
};

// Rows into an output of their own, in pieces of T.
template <typename T>
__global__ void __launch_bounds__(kThreads) tm_reorder_kernel(ReorderParams p, int64_t pieces,
                                                              int blocks) {
  const int64_t row = (int)blockIdx.x / blocks;
  const int64_t i = (int64_t)((int)blockIdx.x % blocks) * kThreads + threadIdx.x;
  if (i >= pieces) return;
  const int64_t group = row / p.beams;
  const int own = (int)(row - group * p.beams);
  const int b = p.parents[group * p.parents_stride + own];
  const int64_t from = group * p.beams + (b < 0 || b >= p.beams ? own : b);
  *reinterpret_cast<T*>(p.out + row * p.out_stride + i * (int64_t)sizeof(T)) =
      *reinterpret_cast<const T*>(p.x + from * p.x_stride + i * (int64_t)sizeof(T));
}

// Rows within x: a workgroup takes `cols` pieces of a group's rows, those that are parents of
// others into LDS, and from there to where they go.  A beam that goes on from itself, or
// whose parent is no beam of the group, stays.  32 groups of 8 rows of 32 KB 7.5 us (into rows
// apart 4.6), one group of 4 of 4 KB 3.5 (2.6).
template <typename T>
__global__ void __launch_bounds__(kThreads) tm_reorder_within_kernel(ReorderParams p, int cols) {
  __shared__ __attribute__((aligned(16))) T rows[kReorderPieces];
  __shared__ int s_parent[TM_MAX_BEAMS];
  __shared__ int s_need[TM_MAX_BEAMS];
  const int K = p.beams, tid = threadIdx.x;
  const int64_t group = blockIdx.y, row0 = group * K;
  if (tid < K) s_need[tid] = 0;
  __syncthreads();
  if (tid < K) {
    int b = p.parents[group * p.parents_stride + tid];
    if (b < 0 || b >= K) b = tid;
    s_parent[tid] = b;
    if (b != tid) s_need[b] = 1;
  }
  __syncthreads();
  const int64_t col0 = (int64_t)blockIdx.x * cols, all = p.width / (int64_t)sizeof(T);
  const int n = (int)min((int64_t)cols, all - col0);
  for (int i = tid; i < K * cols; i += kThreads) {
    const int r = i / cols, c = i - r * cols;
    if (c < n && s_need[r])
      rows[i] = *reinterpret_cast<const T*>(p.x + (row0 + r) * p.x_stride +
                                            (col0 + c) * (int64_t)sizeof(T));
  }
  __syncthreads();
  for (int i = tid; i < K * cols; i += kThreads) {
    const int r = i / cols, c = i - r * cols, b = s_parent[r];
    if (c < n && b != r)
      *reinterpret_cast<T*>(p.out + (row0 + r) * p.out_stride + (col0 + c) * (int64_t)sizeof(T)) =
          rows[b * cols + c];
  }
}

// ------------------------------------------------------------------- host --

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Logits of a lane, by the workgroups that many of them would leave.
int per_of(int64_t rows, int64_t V) {
  return rows * ceil_div(V, kThreads * kManyPer) >= 2 * 256 ? kManyPer : kFewPer;
}

int check_beams(int64_t G, int64_t K, int64_t V, int64_t num) {
  if (G < 0 || K < 1 || K > TM_MAX_BEAMS || num < 1 || num > kMaxNum || V < 1 ||
      V > TM_MAX_SAMPLE_VOCAB || G > TM_MAX_ROWS / K)
    return TM_ERR_SHAPE;
  if (G * K * ceil_div(V, kThreads * kFewPer) > UINT32_MAX / kThreads) return TM_ERR_SHAPE;
  return TM_OK;
}

template <int DT>
void launch_rows(const BeamParams& p, int per, hipStream_t st) {
  const dim3 grid((unsigned)(p.rows * p.segs)), block(kThreads);
  const size_t lds = (size_t)p.num * per * sizeof(uint64_t);
  if (per == kManyPer)
    hipLaunchKernelGGL((tm_beam_rows_kernel<DT, kManyPer>), grid, block, lds, st, p);
  else
    hipLaunchKernelGGL((tm_beam_rows_kernel<DT, kFewPer>), grid, block, lds, st, p);
}

template <typename T>
int launch_reorder(const ReorderParams& p, int64_t G, hipStream_t st) {
  const int64_t pieces = p.width / (int64_t)sizeof(T);
  const bool within = p.out == p.x;
  // columns of a workgroup: all rows of a group within its LDS, and not more than a round
  int cols = kThreads;
  while (cols > 16 && cols * p.beams > kThreads) cols /= 2;
  while (cols * p.beams > kReorderPieces) cols /= 2;
  const int64_t blocks = ceil_div(pieces, within ? cols : kThreads);
  const int64_t rows = within ? G : G * p.beams;
  if (blocks > UINT32_MAX / kThreads / rows) return TM_ERR_SHAPE;  // a grid's threads in 32 bits
  const dim3 block(kThreads);
  if (within)
    hipLaunchKernelGGL((tm_reorder_within_kernel<T>), dim3((unsigned)blocks, (unsigned)G), block,
                       0, st, p, cols);
  else
    hipLaunchKernelGGL((tm_reorder_kernel<T>), dim3((unsigned)(blocks * rows)), block, 0, st, p,
                       pieces, (int)blocks);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

}  // namespace

extern "C" int tm_beam_workspace(int64_t G, int64_t K, int64_t V, int64_t num, int64_t* bytes) {
  const int rc = check_beams(G, K, V, num);
  if (rc) return rc;
  if (bytes == nullptr) return TM_ERR_ARG;
  *bytes = G * K * ceil_div(V, kThreads * per_of(G * K, V)) * (8 * num + 8 + 4);
  return TM_OK;
}

extern "C" int tm_beam_select(const void* logits, int dtype, int64_t G, int64_t K, int64_t V,
                              int64_t row_stride, const float* scores, const uint8_t* finished,
                              int64_t pad_token, int64_t num, float* out_scores,
                              int32_t* parents, int64_t* tokens, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  int64_t need = 0;
  const int rc = tm_beam_workspace(G, K, V, num, &need);
  if (rc) return rc;
  if (!tm_dtype_ok(dtype)) return TM_ERR_ARG;
  if (pad_token < 0 || pad_token >= V || (G * K > 1 && row_stride < 0) || workspace_bytes < need)
    return TM_ERR_SHAPE;
  if (G == 0) return TM_OK;
  if ((uintptr_t)logits % tm_dtype_bytes(dtype) || (uintptr_t)scores % 4 ||
      (uintptr_t)out_scores % 4 || (uintptr_t)parents % 4 || (uintptr_t)tokens % 8 ||
      (uintptr_t)workspace % 8)
    return TM_ERR_ALIGN;
  BeamParams p = {};
  p.logits = logits;
  p.row_stride = G * K > 1 ? row_stride : V;
  p.scores = scores;
  p.finished = finished;
  p.pad_token = pad_token;
  p.rows = (int)(G * K);
  p.beams = (int)K;
  p.vocab = (int)V;
  const int per = per_of(G * K, V);
  p.segs = (int)ceil_div(V, kThreads * per);
  p.num = (int)num;
  const int64_t units = (int64_t)p.rows * p.segs;
  p.lists = (uint64_t*)workspace;
  p.sums = (double*)(p.lists + units * num);
  p.tops = (float*)(p.sums + units);
  p.aligned = (uintptr_t)logits % 16 == 0 && p.row_stride * tm_dtype_bytes(dtype) % 16 == 0;
  p.out_scores = out_scores;
  p.parents = parents;
  p.tokens = tokens;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TM_DTYPE_F32)
    launch_rows<TM_DTYPE_F32>(p, per, st);
  else if (dtype == TM_DTYPE_F16)
    launch_rows<TM_DTYPE_F16>(p, per, st);
  else
    launch_rows<TM_DTYPE_BF16>(p, per, st);
  const int64_t lists = K * p.segs;
  if (num > 16 && lists <= kSteps && lists < 4 * num)
    hipLaunchKernelGGL(tm_beam_join_kernel<true>, dim3((unsigned)G), dim3(kJoin), 0, st, p);
  else
    hipLaunchKernelGGL(tm_beam_join_kernel<false>, dim3((unsigned)G), dim3(kJoin), 0, st, p);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

extern "C" int tm_reorder_rows(const void* x, int64_t x_stride, void* out, int64_t out_stride,
                               int64_t width, const int32_t* parents, int64_t parents_stride,
                               int64_t G, int64_t K, void* stream) {
  if (G < 0 || G > 65535 || K < 1 || K > TM_MAX_BEAMS || width < 0 ||
      width > (int64_t(1) << 40) || (G * K > 1 && (x_stride < width || out_stride < width)) ||
      (G > 1 && parents_stride < K))
    return TM_ERR_SHAPE;
  if (G == 0 || width == 0) return TM_OK;
  if ((uintptr_t)parents % 4) return TM_ERR_ALIGN;
  ReorderParams p = {(const uint8_t*)x, (uint8_t*)out,   x_stride,      out_stride, width,
                     parents,           parents_stride, (int)K};
  if (x == out && G * K > 1 && x_stride != out_stride) return TM_ERR_ARG;
  // pieces as large as everything is aligned to
  const uint64_t bits = (uint64_t)(uintptr_t)x | (uint64_t)(uintptr_t)out | (uint64_t)width |
                        (G * K > 1 ? (uint64_t)(x_stride | out_stride) : 0);
  const hipStream_t st = (hipStream_t)stream;
  if (bits % 16 == 0) return launch_reorder<u32x4_t>(p, G, st);
  if (bits % 4 == 0) return launch_reorder<uint32_t>(p, G, st);
  return launch_reorder<uint8_t>(p, G, st);
}
