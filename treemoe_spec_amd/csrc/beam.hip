// Beam search's selection over beams and vocabulary, and the reordering of what the
// beams hold.
//
// Of a group's K beams with scores s_b and logits l_b, the candidates are (b, v) with
//   s_b + l_b[v] - log sum_u exp l_b[u],
// and one (b, pad) with s_b for a beam that has finished.  The `num` best come out in
// order: larger score first, of equal ones the lower beam, then the larger logit, then
// the lower token.
//
// Arithmetic.  Scores are formed in 64 bits, the sum of the exponentials too, so that beams
// are not exchanged by rounding; each is rounded to fp32 once, when it is written.  Within a
// beam the order is that of the logits, so a row is cut to its best `num` before any
// score is known.
//
// A wave takes 1024 logits of a row: its sum, and its best `num` as sorted keys (ordered
// bits of the logit, inverted token), all distinct.  At least `num` logits reach the
// num-th largest of the 64 lanes' largest, and only the `num` lanes that reach it hold
// such, 16 at most each: the list never overflows.  Then one workgroup a group joins the sums,
// takes the num-th largest of the lists' heads, which bounds the result from below in
// the same way, and ranks what reaches it by binary search in the lists it came from.
#include <cmath>

#include "tm_vec.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kSeg = 1024;               // logits of a wave
constexpr int kPer = kSeg / 64;          // of a lane
constexpr int kMaxNum = TM_MAX_BEAMS;
constexpr int kJoin = 1024;              // threads of a group's workgroup

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

// The logits base + index_of(e) of a lane; what lies past the end, and NaN, as -inf.
template <int DT>
__device__ __forceinline__ int index_of(int e) {
  constexpr int kVec = DT == TM_DTYPE_F32 ? 4 : 8;
  return e / kVec * 64 * kVec + (int)(threadIdx.x & 63) * kVec + e % kVec;
}
template <int DT>
__device__ __forceinline__ void fetch(const BeamParams& p, int64_t row, int base,
                                      float (&x)[kPer]) {
  if (p.aligned && base + kSeg <= p.vocab) {
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

// How many of the lanes' first `n` keys are larger than this lane's.
__device__ __forceinline__ int rank_in_wave(uint64_t key, int n) {
  int rank = 0;
  for (int l = 0; l < n; ++l) rank += lane_of(key, l) > key ? 1 : 0;
  return rank;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) tm_beam_rows_kernel(BeamParams p) {
  __shared__ uint64_t s_list[kWaves][kSeg];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t unit = (int64_t)blockIdx.x * kWaves + wave;
  if (unit >= (int64_t)p.rows * p.segs) return;
  const int row = (int)(unit / p.segs), seg = (int)(unit - (int64_t)row * p.segs);
  if (p.finished != nullptr && p.finished[row]) return;
  const int base = seg * kSeg;
  float x[kPer];
  fetch<DT>(p, row, base, x);
  float top = x[0];
  uint64_t best = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    top = fmaxf(top, x[e]);
    const uint64_t k = key_of(x[e], base + index_of<DT>(e));
    best = k > best ? k : best;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  uint64_t* const out = p.lists + unit * p.num;
  if (top == -INFINITY) {  // nothing here: no candidate, and no weight
    if (lane < p.num) out[lane] = 0;
    if (lane == 0) {
      p.sums[unit] = 0.0;
      p.tops[unit] = top;
    }
    return;
  }
  // (an infinite largest logit weighs 1, and all finite ones nothing)
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    sum += x[e] == top ? 1.0 : exp((double)x[e] - (double)top);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) {
    p.sums[unit] = sum;
    p.tops[unit] = top;
  }
  // the num-th largest of the lanes' largest, and what reaches it
  const uint64_t at = __ballot(rank_in_wave(best, 64) == p.num - 1);
  const uint64_t least = lane_of(best, __ffsll((unsigned long long)at) - 1);
  int n = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const uint64_t k = key_of(x[e], base + index_of<DT>(e));
    const bool in = k >= least && x[e] > -INFINITY;
    const uint64_t who = __ballot(in);
    if (in) s_list[wave][n + lanes_before(who)] = k;
    n += __popcll(who);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (n <= 64) {
    const uint64_t k = lane < n ? s_list[wave][lane] : 0;
    const int rank = rank_in_wave(k, n);
    if (lane < n && rank < p.num) out[rank] = k;
  } else {
    for (int i = lane; i < n; i += 64) {
      const uint64_t k = s_list[wave][i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += s_list[wave][j] > k ? 1 : 0;
      if (rank < p.num) out[rank] = k;
    }
  }
  if (lane >= n && lane < p.num) out[lane] = 0;
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

struct JoinShared {
  Cand pool[kMaxNum + 1][kMaxNum];  // sorted lists; the last is the best so far
  Cand heads[kJoin / 64][kMaxNum];  // of each wave, sorted
  double base[TM_MAX_BEAMS];        // score - log of the sum, -inf for a beam without candidates
  float top[TM_MAX_BEAMS];
  Cand least;
  int used;                         // of the pool
};

// How many of the sorted list's n candidates are above c.
__device__ __forceinline__ int above_in(const Cand* list, int n, const Cand& c) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (above(list[mid], c))
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kJoin) tm_beam_join_kernel(BeamParams p) {
  __shared__ JoinShared s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = blockIdx.x, K = p.beams, num = p.num;
  const int64_t row0 = (int64_t)group * K;
  const int lists = K * p.segs;

  // each beam's sum over its segments, a wave a beam
  for (int b = wave; b < K; b += kJoin / 64) {
    const int64_t at = (row0 + b) * p.segs;
    const bool over = p.finished != nullptr && p.finished[row0 + b];
    float top = -INFINITY;
    double sum = 0.0;
    if (!over) {
      for (int i = lane; i < p.segs; i += 64) top = fmaxf(top, p.tops[at + i]);
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      for (int i = lane; i < p.segs; i += 64) {
        const float t = p.tops[at + i];
        if (t > -INFINITY)
          sum += p.sums[at + i] * (t == top ? 1.0 : exp((double)t - (double)top));
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    }
    if (lane == 0) {
      const double score = p.scores[row0 + b];
      s.top[b] = top;
      s.base[b] = top > -INFINITY && score > -INFINITY ? score - log(sum) : -INFINITY;
    }
  }
  // the finished beams, sorted, are the best so far
  if (wave == 0) {
    Cand c = {0, 0};
    if (lane < K && p.finished != nullptr && p.finished[row0 + lane])
      c = cand_of(p.scores[row0 + lane], lane, 0, (uint32_t)p.pad_token);
    int rank = 0;
    for (int l = 0; l < K; ++l) {
      const Cand x = {lane_of(c.hi, l), lane_of(c.lo, l)};
      rank += above(x, c) || (x.hi == 0 && c.hi == 0 && l < lane) ? 1 : 0;
    }
    if (lane < K && rank < num) s.pool[kMaxNum][rank] = c;
    if (lane >= K && lane < num) s.pool[kMaxNum][lane] = {0, 0};
  }

  for (int first = 0; first < lists; first += kJoin) {
    if (tid == 0) s.used = 0;
    __syncthreads();
    // this thread's list and its head
    const int list = first + tid;
    Cand head = {0, 0};
    int beam = 0;
    const uint64_t* from = nullptr;
    double base = -INFINITY;
    float top = 0.0f;
    auto cand = [&](uint64_t key) {
      const float l = float_of((uint32_t)(key >> 32));
      // (l - top is 0 for equal infinities)
      const double score = l == top ? base : base + ((double)l - (double)top);
      return key == 0 ? Cand{0, 0}
                      : cand_of(score, beam, (uint32_t)(key >> 32), ~(uint32_t)key);
    };
    if (list < lists) {
      beam = list / p.segs;
      base = s.base[beam];
      top = s.top[beam];
      if (base > -INFINITY) {
        from = p.lists + (row0 * p.segs + list) * num;
        head = cand(from[0]);
      }
    }
    // the waves' best heads, sorted
    int rank = 0;
#pragma unroll 4
    for (int l = 0; l < 64; ++l) {
      const Cand x = {lane_of(head.hi, l), lane_of(head.lo, l)};
      rank += above(x, head) || (x.hi == 0 && head.hi == 0 && l < lane) ? 1 : 0;
    }
    if (rank < num) s.heads[wave][rank] = head;
    if (tid == 0) s.least = {0, 1};  // fewer heads than num: all candidates
    __syncthreads();
    // the num-th largest of all heads
    const int waves = (min(lists - first, kJoin) + 63) / 64;
    if (rank < num && head.hi != 0) {
      int r = 0;
      for (int w = 0; w < waves; ++w) r += above_in(s.heads[w], num, head);
      if (r == num - 1) s.least = head;
    }
    __syncthreads();
    // the lists that reach it, num at most, up to where they do
    if (head.hi != 0 && !above(s.least, head)) {
      Cand* const to = s.pool[atomicAdd(&s.used, 1)];
      for (int i = 0; i < num; ++i) {
        const Cand c = i == 0 ? head : cand(from[i]);
        const bool in = c.hi != 0 && !above(s.least, c);
        to[i] = in ? c : Cand{0, 0};
        if (!in) {
          for (int j = i + 1; j < num; ++j) to[j] = {0, 0};
          break;
        }
      }
    }
    __syncthreads();
    // their ranks among each other and the best so far
    const int used = s.used;
    constexpr int kMine = (kMaxNum + 1) * kMaxNum / kJoin + 1;
    Cand mine[kMine];
    int place[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int at = i * kJoin + tid;
      place[i] = -1;
      if (at >= (used + 1) * num) continue;
      const int li = at / num, l = li == used ? kMaxNum : li;
      mine[i] = s.pool[l][at - li * num];
      if (mine[i].hi == 0) continue;
      int r = above_in(s.pool[kMaxNum], num, mine[i]);
      for (int j = 0; j < used && r < num; ++j) r += above_in(s.pool[j], num, mine[i]);
      place[i] = r < num ? r : -1;
    }
    __syncthreads();
    if (tid < num) s.pool[kMaxNum][tid] = {0, 0};
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (place[i] >= 0) s.pool[kMaxNum][place[i]] = mine[i];
    __syncthreads();
  }
  if (tid < num) {
    const Cand c = s.pool[kMaxNum][tid];
    const int64_t at = (int64_t)group * num + tid;
    const bool none = c.hi == 0;
    p.out_scores[at] = none ? -INFINITY : (float)double_of(c.hi);
    p.parents[at] = none ? -1 : 63 - (int)(c.lo >> (32 + kTokenBits));
    p.tokens[at] = none ? -1 : (int64_t)(((1u << kTokenBits) - 1) -
                                         (uint32_t)(c.lo & ((1u << kTokenBits) - 1)));
  }
}

// ---------------------------------------------------------------- reorder --

struct ReorderParams {
  const uint8_t* x;
  uint8_t* out;
  int64_t x_stride, out_stride, width;  // bytes
  const int32_t* parents;
  int64_t parents_stride;
  int beams;
};

// Rows of a group in pieces of T: the parents' rows into LDS, and from there to where they
// go, so that out may be x.  A beam that goes on from itself, or whose parent is no beam of
// the group, is copied only where out is not x.
template <typename T>
__global__ void __launch_bounds__(kThreads) tm_reorder_kernel(ReorderParams p, int cols) {
  __shared__ __attribute__((aligned(16))) uint8_t s_rows[kThreads * 16 * 16];
  __shared__ int s_parent[TM_MAX_BEAMS];
  __shared__ int s_need[TM_MAX_BEAMS];
  T* const rows = reinterpret_cast<T*>(s_rows);
  const int K = p.beams, tid = threadIdx.x;
  const int64_t group = blockIdx.y, row0 = group * K;
  const bool same = p.out == p.x;
  if (tid < K) s_need[tid] = 0;
  __syncthreads();
  if (tid < K) {
    int b = p.parents[group * p.parents_stride + tid];
    if (b < 0 || b >= K) b = tid;
    s_parent[tid] = b;
    if (!same || b != tid) s_need[b] = 1;
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
    if (c < n && (!same || b != r))
      *reinterpret_cast<T*>(p.out + (row0 + r) * p.out_stride + (col0 + c) * (int64_t)sizeof(T)) =
          rows[b * cols + c];
  }
}

// ------------------------------------------------------------------- host --

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int check_beams(int64_t G, int64_t K, int64_t V, int64_t num) {
  if (G < 0 || K < 1 || K > TM_MAX_BEAMS || num < 1 || num > kMaxNum || V < 1 ||
      V > TM_MAX_SAMPLE_VOCAB || G > TM_MAX_ROWS / K)
    return TM_ERR_SHAPE;
  if (ceil_div(G * K * ceil_div(V, kSeg), kWaves) > UINT32_MAX / kThreads) return TM_ERR_SHAPE;
  return TM_OK;
}

template <typename T>
int launch_reorder(const ReorderParams& p, int64_t G, hipStream_t st) {
  // columns of a workgroup: all rows of a group within its LDS
  int cols = kThreads;
  while (cols * p.beams > kThreads * 16) cols /= 2;
  const int64_t blocks = ceil_div(p.width / (int64_t)sizeof(T), cols);
  if (blocks > UINT32_MAX / kThreads / G) return TM_ERR_SHAPE;  // a grid's threads in 32 bits
  hipLaunchKernelGGL((tm_reorder_kernel<T>), dim3((unsigned)blocks, (unsigned)G), dim3(kThreads),
                     0, st, p, cols);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

}  // namespace

extern "C" int tm_beam_workspace(int64_t G, int64_t K, int64_t V, int64_t num, int64_t* bytes) {
  const int rc = check_beams(G, K, V, num);
  if (rc) return rc;
  if (bytes == nullptr) return TM_ERR_ARG;
  *bytes = G * K * ceil_div(V, kSeg) * (8 * num + 8 + 4);
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
  if (pad_token < 0 || pad_token >= V || (G * K > 1 && row_stride < V) || workspace_bytes < need)
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
  p.segs = (int)ceil_div(V, kSeg);
  p.num = (int)num;
  const int64_t units = (int64_t)p.rows * p.segs;
  p.lists = (uint64_t*)workspace;
  p.sums = (double*)(p.lists + units * num);
  p.tops = (float*)(p.sums + units);
  p.aligned = (uintptr_t)logits % 16 == 0 && p.row_stride * tm_dtype_bytes(dtype) % 16 == 0;
  p.out_scores = out_scores;
  p.parents = parents;
  p.tokens = tokens;
  const dim3 grid((unsigned)ceil_div(units, kWaves)), block(kThreads);
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TM_DTYPE_F32)
    hipLaunchKernelGGL((tm_beam_rows_kernel<TM_DTYPE_F32>), grid, block, 0, st, p);
  else if (dtype == TM_DTYPE_F16)
    hipLaunchKernelGGL((tm_beam_rows_kernel<TM_DTYPE_F16>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((tm_beam_rows_kernel<TM_DTYPE_BF16>), grid, block, 0, st, p);
  hipLaunchKernelGGL(tm_beam_join_kernel, dim3((unsigned)G), dim3(kJoin), 0, st, p);
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
