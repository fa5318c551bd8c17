// What every cached key gets of the queries' attention, and the eviction of the keys that
// get least.
//
// Mass.  For the last T of a sequence's S positions, a KV head's rows being the (token, head
// of the group) pairs,
//   mass[j] += sum over the rows that see key j of exp(s_rj - m_r) / l_r,
// with s = scale q . k, m_r the largest of a row's scores and l_r the sum of its
// exponentials.  First m and l of every row, over ranges of keys.  Up to 32 rows (the tokens
// of a decoding step) leave their scores, too, and a second launch sums them over the rows.  Of
// more rows the scores would be more to store and read than to compute twice: a wave takes 32
// keys into registers, and the rows come by.  All in fp32; the order of the sums is fixed.
//
// Bound by latencies at few rows: one token over 7777 keys 10.8 us of two launches, 16 MB of K.
// By the matrix products and exponentials together at many: 4096 tokens over themselves
// 168-181 us, twice 69 GFLOP and 0.27 G exponentials each time, 0.76-0.82 PFLOP/s; the vector
// unit is busy in 64-70 % of the CUs' busy cycles, the matrix pipe in 44-46 %.
//
// Eviction.  Of each layer's KV heads, `keep` of S keys stay: the first `sinks` and the last
// `recent` positions, and the heaviest others.  Kept keys in slots from `keep` on move into
// the holes below, the i-th into the i-th; all others stay where they are, so a cache that
// is cut every few tokens moves few keys.  Attention does not go by the order of the
// slots; the positions go along.  One workgroup a head selects, by a radix search over the
// ordered bits of the weights, and moves the keys, or leaves many moves of few heads to a
// second launch.  Selection is a chain of barriers (32 layers' heads of 1088 slots 11 us, with
// 64 moves each); with some 900 moves a head, 236 MB, it is 10 of 68 us, and the rest a copy.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_tile.h"

namespace {

struct MassParams : PromptParams {
  float2* row_stats;      // (m in base 2, l) [chunks][kvh][rows]
  float* row_consts;      // -(m + log2 l) [kvh][rows in whole stages], or NULL: the sums'
                          // workgroups take row_stats
  float* scores;          // [kvh][rows][score_stride]: few rows' scores, unscaled, -inf where a
                          // row does not see the key
  int64_t score_stride;
  float* parts;           // [splits][kvh][keys], or NULL: the mass itself
  int splits;             // of a tile's rows
  const float* before;    // [kvh, before_stride], or NULL
  int64_t before_stride;
  float* mass;            // [kvh, mass_stride]
  int64_t mass_stride;
};

// Running maximum and sum of the stage's scores, keys kb ...
__device__ __forceinline__ void mask_scores(f32x16_t (&sc)[2], int left) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int x = 0; x < 16; ++x)
      sc[kt][x] = 32 * kt + 8 * (x >> 2) + (x & 3) <= left ? sc[kt][x] : -INFINITY;
}
template <int HD>
__device__ __forceinline__ void take_stats(float scale_log2, int kb, bool mask, Rows<HD>& r) {
  if (mask) mask_scores(r.sc, r.seen - kb - 4 * ((int)(threadIdx.x & 63) >> 5));
  float mx[2] = {fmaxf(r.sc[0][0], r.sc[1][0]), fmaxf(r.sc[0][1], r.sc[1][1])};
#pragma unroll
  for (int x = 2; x < 16; ++x) mx[x & 1] = fmaxf(fmaxf(mx[x & 1], r.sc[0][x]), r.sc[1][x]);
  const float m = fmaxf(r.m, max_halves(fmaxf(mx[0], mx[1])) * scale_log2);
  const float base = m == -INFINITY ? 0.0f : -m;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    sum[x & 1] += __builtin_amdgcn_exp2f(fmaf(r.sc[0][x], scale_log2, base));
    sum[2 + (x & 1)] += __builtin_amdgcn_exp2f(fmaf(r.sc[1][x], scale_log2, base));
  }
  const float a = r.m == m ? 1.0f : __builtin_amdgcn_exp2f(r.m - m);
  r.l = fmaf(r.l, a, (sum[0] + sum[1]) + (sum[2] + sum[3]));
  r.m = m;
}
// The larger maximum of two, and the sum over both.
__device__ __forceinline__ void join_stats(float& m, float& l, float m1, float l1) {
  const float mn = fmaxf(m, m1), ref = mn == -INFINITY ? 0.0f : mn;
  l = l * __builtin_amdgcn_exp2f(m - ref) + l1 * __builtin_amdgcn_exp2f(m1 - ref);
  m = mn;
}

// What a score s in base 2 takes to become a weight, 2^(s + c); -inf, for nothing, of a row
// whose scores are all -inf.  As one number it is off by half a step below 2^6: 1.3e-6 of a
// weight.
__device__ __forceinline__ float const_of(float m, float l) {
  return l == 0.0f ? -INFINITY : -(m + __builtin_amdgcn_logf(l));
}

// Rows 128 a tile, 32 a wave, that share the stages of a range of keys.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 2) tm_mass_stats_kernel(MassParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k1[S::kTile];
  const int kvhead = (int)blockIdx.x % p.kvh, at_item = (int)blockIdx.x / p.kvh;
  Item it = item_of(p, at_item, 128);
  {
    // The tiles with the most keys first, then from the fewest up: of workgroups that are
    // given out in turn a CU gets some of each.
    const int t = at_item / p.chunks, first = (p.tiles + 1) / 2;
    it.tile = t < first ? p.tiles - 1 - t : t - first;
    const int last_token = min(it.q_len - 1, (it.tile * 128 + 127) / p.group);
    it.end = min(it.begin + p.chunk_len, it.k_len - it.q_len + last_token + 1);
  }
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = it.end > it.begin ? (it.end - it.begin + kKeys - 1) / kKeys : 0;
  Rows<HD> r;
  const Place at = begin_rows<HD>(p, it, kvhead, it.tile * 128 + wave * 32, r);
  if (n > 0) {
    Feed<HD, true, 4> feed;
    feed.start(p, it, kvhead, it.begin, kKeys);
    auto step = [&](int s, const uint8_t* kc, uint8_t* kn) TM_INLINE {
      wait_vm<0>();
      tm_lds_barrier();
      const int kb = it.begin + s * kKeys;
      if (s + 1 < n) feed.load_k(p, kn);
      products<DT, HD, false, true>(kc, kc, r);
      take_stats<HD>(p.scale_log2, kb, kb + kKeys - 1 > at.full, r);
    };
    feed.load_k(p, s_k0);
    for (int s = 0; s < n; s += 2) {
      step(s, s_k0, s_k1);
      if (s + 1 < n) step(s + 1, s_k1, s_k0);
    }
  }
  const float l = r.l + __shfl_xor(r.l, 32);
  const int rows = it.q_len * p.group;
  if ((threadIdx.x & 32) != 0) return;
  if (p.row_consts != nullptr && p.chunks == 1) {
    const int whole = (rows + kKeys - 1) / kKeys * kKeys;
    if (at.row < whole)
      p.row_consts[(int64_t)kvhead * whole + at.row] = at.ok ? const_of(r.m, l) : -INFINITY;
  } else if (at.ok) {
    p.row_stats[((int64_t)(at_item % p.chunks) * p.kvh + kvhead) * rows + at.row] =
        float2{r.m, l};
  }
}

// Up to 32 rows: the waves take the stages in turn, and keep the scores.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 2) tm_mass_stats_few_kernel(MassParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k[4][S::kTile];
  __shared__ float s_stat[4][32][2];
  const int kvhead = (int)blockIdx.x % p.kvh, at_item = (int)blockIdx.x / p.kvh;
  const Item it = item_of(p, at_item, 32);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = it.end > it.begin ? (it.end - it.begin + kKeys - 1) / kKeys : 0;
  Rows<HD> r;
  Feed<HD, true, 1> feed;
  if (wave < n) {
    feed.start(p, it, kvhead, it.begin + wave * kKeys, 4 * kKeys);
    feed.load_k(p, s_k[wave]);
  }
  const Place at = begin_rows<HD>(p, it, kvhead, it.tile * 32, r);
  for (int s = wave; s < n; s += 4) {
    const int kb = it.begin + s * kKeys;
    wait_vm<0>();
    products<DT, HD, false, true>(s_k[wave], s_k[wave], r);
    if (s + 4 < n) feed.load_k(p, s_k[wave]);
    take_stats<HD>(p.scale_log2, kb, kb + kKeys - 1 > at.full, r);
    if (at.ok) {
      float* const to = p.scores +
                        ((int64_t)kvhead * it.q_len * p.group + at.row) * p.score_stride + kb +
                        4 * (lane >> 5);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4_t*>(to + 32 * kt + 8 * j) =
              f32x4_t{r.sc[kt][4 * j], r.sc[kt][4 * j + 1], r.sc[kt][4 * j + 2],
                      r.sc[kt][4 * j + 3]};
    }
  }
  const float l = r.l + __shfl_xor(r.l, 32);
  if (lane < 32) {
    s_stat[wave][lane][0] = r.m;
    s_stat[wave][lane][1] = l;
  }
  __syncthreads();
  if (threadIdx.x >= 32 || !at.ok) return;
  float m = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) join_stats(m, sum, s_stat[w][lane][0], s_stat[w][lane][1]);
  p.row_stats[((int64_t)(at_item % p.chunks) * p.kvh + kvhead) * it.q_len * p.group + at.row] =
      float2{m, sum};
}

// The constant of a row from its ranges, P neighbouring lanes a row.
__device__ __forceinline__ float joined(const float2* st, int64_t step, int chunks, int P) {
  const int part = (int)threadIdx.x & (P - 1);
  float m = -INFINITY, l = 0.0f;
#pragma unroll 4
  for (int c = part; c < chunks; c += P) m = fmaxf(m, st[c * step].x);
  for (int d = 1; d < P; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 4
  for (int c = part; c < chunks; c += P) {
    const float2 x = st[c * step];
    l = fmaf(x.y, __builtin_amdgcn_exp2f(x.x - ref), l);
  }
  for (int d = 1; d < P; d <<= 1) l += __shfl_xor(l, d);
  return const_of(m, l);
}

// The constants of all rows, and -inf up to whole stages: where the rows are too many for
// every workgroup of the sums to do it again.
__global__ void __launch_bounds__(kThreads) tm_mass_rows_kernel(MassParams p, int rows, int whole) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= (int64_t)p.kvh * whole) return;
  const int kvhead = (int)(i / whole), row = (int)(i - (int64_t)kvhead * whole);
  p.row_consts[i] = row < rows ? joined(p.row_stats + (int64_t)kvhead * rows + row,
                                        (int64_t)p.kvh * rows, p.chunks, 1)
                               : -INFINITY;
}

// Rows whose constants a workgroup of the sums makes by itself, instead of a launch before
// it, in us: 256 rows over 7464 keys 23.3, 26.2; 500 over 7125 34, 35; 800 over 7200 49, 49; 1000
// over 3250 37, 34; 2000 over 3500 59, 51; 2048 over 512 43, 21.
constexpr int kOwnRows = 512;

// Sums over the rows: a wave has 32 keys, one a column, and 64 rows at a time come by in LDS,
// for all waves.  A lane's products with a stage belong to its key, so they are summed in
// its registers.  OWN: the workgroup joins the rows' ranges itself.
template <int DT, int HD, int WAVES, bool OWN>
__global__ void __launch_bounds__(64 * WAVES, WAVES == 8 ? 4 : 2) tm_mass_sum_kernel(MassParams p) {
  typedef Shape<HD> S;
  constexpr int kLoads = S::kTile / (1024 * WAVES);
  __shared__ __attribute__((aligned(1024))) uint8_t s_q[2][S::kTile];
  __shared__ __attribute__((aligned(16))) float s_const[OWN ? kOwnRows : 2 * kKeys];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvhead = (int)blockIdx.x % p.kvh, rest = (int)blockIdx.x / p.kvh;
  const int split = rest % p.splits;
  const int first = rest / p.splits * (32 * WAVES);  // the keys with the most rows first
  const int rows = p.q_len * p.group, past = p.k_len - p.q_len;
  const int whole = (rows + kKeys - 1) / kKeys * kKeys;
  const int key = first + 32 * wave + c32;
  // the key's first row, and that of the workgroup's last key
  const int seen = max(min(key, p.k_len - 1) - past, 0) * p.group;
  const int all = max(min(first + 32 * WAVES, p.k_len) - 1 - past, 0) * p.group;
  const int stage0 = max(min(first, p.k_len - 1) - past, 0) * p.group / kKeys;
  const int per = (whole / kKeys - stage0 + p.splits - 1) / p.splits;
  const int begin = stage0 + split * per, end = min(begin + per, whole / kKeys);
  // The rows of a stage that this wave loads.  Where a stage is whole tokens the next stage
  // lies a fixed step behind: a division for each row costs as much as its exponentials.
  const bool even = kKeys % p.group == 0;
  const int64_t stage_step = (int64_t)(kKeys / p.group) * p.q_stride;
  int64_t lane_off[kLoads];
  auto offset_of = [&](int row, int in) TM_INLINE {
    const int token = row / p.group;
    return (int64_t)token * p.q_stride +
           (int64_t)(kvhead * p.group + row - token * p.group) * HD +
           (((lane & (S::kChunks - 1)) ^ S::swz_k(in)) * 8);
  };
  auto row_in = [&](int i) TM_INLINE {
    return (wave * kLoads + i) * S::kKeysPerLoad + lane / S::kChunks;
  };
#pragma unroll
  for (int i = 0; i < kLoads; ++i) lane_off[i] = offset_of(row_in(i), row_in(i));
  auto load = [&](int stage, uint8_t* tile) TM_INLINE {
    const bool whole_stage = even && (stage + 1) * kKeys <= rows;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int64_t off = whole_stage
                              ? lane_off[i] + stage * stage_step
                              : offset_of(min(stage * kKeys + row_in(i), rows - 1), row_in(i));
      __builtin_amdgcn_global_load_lds((glb_void*)(p.q + off),
                                       (lds_void*)(tile + (wave * kLoads + i) * 1024), 16, 0, 0);
    }
  };
  Rows<HD> r;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (begin < end) {
    load(begin, s_q[0]);
    {
      const int at = min(key, p.k_len - 1);
      const int pg = min(max(p.table[at >> p.page_shift], 0), p.cache_pages - 1);
      const uint16_t* const kr = p.k + (int64_t)pg * p.stride_page +
                                 (int64_t)(at & ((1 << p.page_shift) - 1)) * p.k_stride +
                                 kvhead * HD + 8 * half;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        r.q[ks] = *reinterpret_cast<const u32x4_t*>(kr + 16 * ks);
    }
    const float* const consts = p.row_consts + (int64_t)kvhead * whole;
    float next = 0.0f;
    if constexpr (OWN) {
      int P = 1;  // lanes a row
      while (P < 64 && 2 * P * rows <= 64 * WAVES) P *= 2;
      for (int row = tid / P; row < whole; row += 64 * WAVES / P) {
        float c = -INFINITY;
        if (row < rows)
          c = joined(p.row_stats + (int64_t)kvhead * rows + row, (int64_t)p.kvh * rows, p.chunks,
                     P);
        if ((tid & (P - 1)) == 0) s_const[row] = c;
      }
    } else if (wave == 0) {
      next = consts[begin * kKeys + lane];
    }
    auto step = [&](int stage, int turn) TM_INLINE {
      wait_vm<0>();
      if (!OWN && wave == 0) s_const[turn * kKeys + lane] = next;
      tm_lds_barrier();
      if (stage + 1 < end) {
        load(stage + 1, s_q[turn ^ 1]);
        if (!OWN && wave == 0) next = consts[(stage + 1) * kKeys + lane];
      }
      products<DT, HD, false, true>(s_q[turn], s_q[turn], r);
      const float* const c = s_const + (OWN ? stage : turn) * kKeys + 4 * half;
      // rows that do not see the lane's key give 0, whatever their constant
      const int hidden = seen - stage * kKeys - 4 * half;
      auto weights = [&](auto masked) TM_INLINE {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4_t cc = *reinterpret_cast<const f32x4_t*>(c + 32 * kt + 8 * j);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float e =
                  __builtin_amdgcn_exp2f(fmaf(r.sc[kt][4 * j + x], p.scale_log2, cc[x]));
              sum[x] += !decltype(masked)::value || 32 * kt + 8 * j + x >= hidden ? e : 0.0f;
            }
          }
      };
      if (stage * kKeys < all)
        weights(std::true_type{});
      else
        weights(std::false_type{});
    };
    for (int stage = begin; stage < end; stage += 2) {
      step(stage, 0);
      if (stage + 1 < end) step(stage + 1, 1);
    }
  }
  float v = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  v += __shfl_xor(v, 32);
  if (half != 0 || key >= p.k_len) return;
  if (p.parts != nullptr) {
    p.parts[((int64_t)split * p.kvh + kvhead) * p.k_len + key] = v;
  } else {
    if (p.before != nullptr) v += p.before[kvhead * p.before_stride + key];
    p.mass[kvhead * p.mass_stride + key] = v;
  }
}

// Sums over few rows from the scores that were kept, a thread a key.  Rows that do not see the key
// give 0 by their index, not by their score of -inf: a constant that is NaN would reach it.
// Scored again by tm_mass_sum_kernel, in us: 4 rows over 7777 keys 15.8, so 10.8; over 30001 34,
// 19; 32 rows over 7008 15.3, 13.3.
__global__ void __launch_bounds__(kThreads) tm_mass_kept_kernel(MassParams p) {
  __shared__ float s_const[32];
  const int tid = threadIdx.x, rows = p.q_len * p.group;
  const int kvhead = (int)blockIdx.x % p.kvh;
  const int key = (int)blockIdx.x / p.kvh * kThreads + tid, at = min(key, p.k_len - 1);
  constexpr int kAhead = 4;
  const float* const from = p.scores + (int64_t)kvhead * rows * p.score_stride + at;
  float first[kAhead];
#pragma unroll
  for (int r = 0; r < kAhead; ++r) first[r] = r < rows ? from[r * p.score_stride] : 0.0f;
  const float before =
      p.before != nullptr ? p.before[kvhead * p.before_stride + at] : 0.0f;
  const int seen = max(at - (p.k_len - p.q_len), 0) * p.group;  // the key's first row
  int P = 64;  // lanes a row
  while (P * rows > kThreads) P /= 2;
  if (tid / P < rows) {
    const float c = joined(p.row_stats + (int64_t)kvhead * rows + tid / P, (int64_t)p.kvh * rows,
                           p.chunks, P);
    if ((tid & (P - 1)) == 0) s_const[tid / P] = c;
  }
  __syncthreads();
  float sum = 0.0f;
#pragma unroll
  for (int r = 0; r < kAhead; ++r)
    if (r < rows) {
      const float e = __builtin_amdgcn_exp2f(fmaf(first[r], p.scale_log2, s_const[r]));
      sum += r >= seen ? e : 0.0f;
    }
#pragma unroll 4
  for (int r = kAhead; r < rows; ++r) {
    const float e =
        __builtin_amdgcn_exp2f(fmaf(from[r * p.score_stride], p.scale_log2, s_const[r]));
    sum += r >= seen ? e : 0.0f;
  }
  if (key < p.k_len) p.mass[kvhead * p.mass_stride + key] = before + sum;
}

// The splits' sums, in their order.
__global__ void __launch_bounds__(kThreads) tm_mass_join_kernel(MassParams p) {
  const int key = (int)(blockIdx.x * kThreads + threadIdx.x), kvhead = blockIdx.y;
  if (key >= p.k_len) return;
  float v = 0.0f;
  for (int s = 0; s < p.splits; ++s) v += p.parts[((int64_t)s * p.kvh + kvhead) * p.k_len + key];
  if (p.before != nullptr) v += p.before[kvhead * p.before_stride + key];
  p.mass[kvhead * p.mass_stride + key] = v;
}

// --------------------------------------------------------------- eviction --

constexpr int kSelect = 1024;  // threads of a head's workgroup
constexpr int kBins = 2048;

struct EvictParams {
  uint8_t *k, *v;                 // the cache
  int64_t stride_layer, stride_page, stride_slot, stride_head;  // bytes
  int row_bytes;                  // of one key of one head
  const int32_t* table;
  int page_shift, cache_pages;
  int kvh, length, keep, moves;   // moves: the most that a head can have
  const float* mass;
  int64_t mass_layer, mass_head;  // strides
  int columns;                    // of a row of mass and of mass_out
  const int32_t* positions;       // of the first `recorded` slots
  int64_t pos_layer, pos_head;
  int recorded, next, recent, sinks;
  float* mass_out;                // [heads][columns]
  int32_t* positions_out;         // [heads][keep]
  int fused;                      // the selecting workgroup moves the keys, too
  int32_t* counts;                // [heads]: of the moves
  int32_t *holes, *movers;        // [heads][moves]
};

// Exclusive rank of the threads whose flag is set, and how many there are.
struct BlockRank {
  int* waves;  // LDS, kSelect / 64
  __device__ __forceinline__ int operator()(bool flag, int* total) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t who = __ballot(flag);
    __syncthreads();
    if (lane == 0) waves[wave] = __popcll(who);
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kSelect / 64; ++w) {
      if (w < wave) before += waves[w];
      sum += waves[w];
    }
    *total = sum;
    return before + (int)__builtin_amdgcn_mbcnt_hi(
                        (uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
  }
};

// What a head's workgroup reads.
struct Head {
  const float* mass;
  const int32_t* pos;
  const EvictParams& p;
  int index;
  __device__ __forceinline__ Head(const EvictParams& p_) : p(p_), index((int)blockIdx.x) {
    const int layer = index / p.kvh, kvhead = index - layer * p.kvh;
    mass = p.mass + layer * p.mass_layer + kvhead * p.mass_head;
    pos = p.positions + layer * p.pos_layer + kvhead * p.pos_head;
  }
  __device__ __forceinline__ int position(int s) const {
    return s < p.recorded ? pos[s] : p.next - p.length + s;
  }
  // larger: kept sooner.  NaN last; what is kept in any case first.
  __device__ __forceinline__ uint32_t key(int s) const { return key(mass[s], position(s)); }
  __device__ __forceinline__ uint32_t key(float m, int at) const {
    if (at < p.sinks || at >= p.next - p.recent) return 0xffffffffu;
    if (m != m) return 0u;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return u ^ (uint32_t)(((int32_t)u >> 31) | 0x80000000);
  }
  // Where a slot of the head lies in k and v.
  __device__ __forceinline__ int64_t slot(int s) const {
    const int layer = index / p.kvh, kvhead = index - layer * p.kvh;
    const int pg = min(max(p.table[s >> p.page_shift], 0), p.cache_pages - 1);
    return (int64_t)layer * p.stride_layer + (int64_t)kvhead * p.stride_head +
           (int64_t)pg * p.stride_page +
           (int64_t)(s & ((1 << p.page_shift) - 1)) * p.stride_slot;
  }
};

// The sum of the waves' counts before this wave's, and of all.
template <int WAVES>
__device__ __forceinline__ int sum_waves(int* waves, int mine, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) waves[wave] = mine;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int x = waves[w];
    before += w < wave ? x : 0;
    sum += x;
  }
  *total = sum;
  return before;
}
__device__ __forceinline__ int lanes_before(uint64_t who) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
}
// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int scan_wave(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(v, d);
    v += lane >= d ? up : 0;
  }
  return v;
}

// Selection with a head's keys in registers, PER a thread: the threshold from four
// histograms of eight bits.  A wave owns consecutive slots, so that ranks need one sum over the
// waves.  Few waves where few keys are: what a step costs is its barriers.
template <int PER, int THREADS>
__global__ void __launch_bounds__(THREADS) tm_evict_held_kernel(EvictParams p) {
  constexpr int kWaves = THREADS / 64, kMost = PER * THREADS / 2;  // moves
  __shared__ uint32_t s_bins[4][256];
  __shared__ int s_scan[4][4];
  __shared__ int s_rank[2][kWaves];
  __shared__ uint32_t s_digit[4];
  __shared__ int s_need[4];
  __shared__ uint16_t s_hole[kMost], s_mover[kMost];
  static_assert(PER * THREADS <= 65536, "slots in 16 bits");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Head head(p);
  const int first = wave * (64 * PER) + lane;  // slots first + 64 i
  uint32_t key[PER];
  float mass[PER];
  int pos[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = min(first + 64 * i, p.length - 1);
    mass[i] = p.length > 0 ? head.mass[s] : 0.0f;
    pos[i] = p.length > 0 ? head.position(s) : 0;
  }
  for (int i = tid; i < 4 * 256; i += THREADS) s_bins[i >> 8][i & 255] = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = head.key(mass[i], pos[i]);
  // the keep-th largest key, and how many of its equals stay
  uint32_t t = 0;
  int need = p.keep;
  if (p.keep < p.length && p.keep > 0) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int shift = 24 - 8 * d;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (first + 64 * i < p.length && (d == 0 || (key[i] >> (shift + 8)) == t))
          atomicAdd(&s_bins[d][(key[i] >> shift) & 255], 1u);
      __syncthreads();
      // from the largest digit down, one a thread of the first four waves
      int own = 0, upto = 0;
      if (tid < 256) {
        own = (int)s_bins[d][255 - tid];
        upto = scan_wave(own);
        if (lane == 63) s_scan[d][wave] = upto;
      }
      __syncthreads();
      if (tid < 256) {
        for (int w = 0; w < wave; ++w) upto += s_scan[d][w];
        if (upto >= need && upto - own < need) {
          s_digit[d] = 255 - tid;
          s_need[d] = need - (upto - own);
        }
      }
      __syncthreads();
      t = (t << 8) | s_digit[d];
      need = s_need[d];
    }
  }
  // which stay: above t, and the first `need` of its equals
  uint32_t kept = 0;
  {
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      mine += __popcll(__ballot(first + 64 * i < p.length && key[i] == t));
    int all;
    int at = sum_waves<kWaves>(s_rank[0], mine, &all);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = first + 64 * i < p.length, equal = in && key[i] == t;
      const uint64_t who = __ballot(equal);
      if (in && p.keep > 0 && (key[i] > t || (equal && at + lanes_before(who) < need)))
        kept |= 1u << i;
      at += __popcll(who);
    }
  }
  // holes below keep, movers behind it, both in the slots' order
  int mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = first + 64 * i;
    const bool stays = kept >> i & 1;
    mine += __popcll(__ballot(s < p.length && s < p.keep && !stays));
    mine += __popcll(__ballot(stays && s >= p.keep)) << 16;
  }
  int all;
  int at = sum_waves<kWaves>(s_rank[1], mine, &all);
  float* const mass_out = p.mass_out + (int64_t)head.index * p.columns;
  int32_t* const pos_out = p.positions_out + (int64_t)head.index * p.keep;
  int rank[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int s = first + 64 * i;
    const bool stays = kept >> i & 1;
    const bool hole = s < p.length && s < p.keep && !stays, mover = stays && s >= p.keep;
    const uint64_t holes = __ballot(hole), movers = __ballot(mover);
    if (hole) s_hole[(at & 0xffff) + lanes_before(holes)] = (uint16_t)s;
    rank[i] = mover ? (at >> 16) + lanes_before(movers) : -1;
    if (mover) s_mover[rank[i]] = (uint16_t)s;
    at += __popcll(holes) + (__popcll(movers) << 16);
    if (stays && !mover) {
      mass_out[s] = mass[i];
      pos_out[s] = pos[i];
    }
  }
  for (int s = p.keep + tid; s < p.columns; s += THREADS) mass_out[s] = 0.0f;
  const int moves = all >> 16;  // (as many as holes)
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (rank[i] >= 0) {
      const int to = s_hole[rank[i]];
      mass_out[to] = mass[i];
      pos_out[to] = pos[i];
    }
  if (!p.fused) {
    if (tid == 0) p.counts[head.index] = moves;
    for (int i = tid; i < moves; i += THREADS) {
      p.holes[(int64_t)head.index * p.moves + i] = s_hole[i];
      p.movers[(int64_t)head.index * p.moves + i] = s_mover[i];
    }
    return;
  }
  const int pieces = p.row_bytes / 16, all_pieces = moves * pieces;
  constexpr int kAhead = 4;  // pieces of a thread under way
  for (int i0 = tid; i0 < all_pieces; i0 += kAhead * THREADS) {
    int64_t from[kAhead], to[kAhead];
    u32x4_t k[kAhead], v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = min(i0 + u * THREADS, all_pieces - 1);  // (the last one again and again)
      const int move = i / pieces, piece = (i - move * pieces) * 16;
      from[u] = head.slot(s_mover[move]) + piece;
      to[u] = head.slot(s_hole[move]) + piece;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      k[u] = *reinterpret_cast<const u32x4_t*>(p.k + from[u]);
      v[u] = *reinterpret_cast<const u32x4_t*>(p.v + from[u]);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      *reinterpret_cast<u32x4_t*>(p.k + to[u]) = k[u];
      *reinterpret_cast<u32x4_t*>(p.v + to[u]) = v[u];
    }
  }
}

// Selection of any number of keys, read again for each pass: the threshold from histograms
// of 11, 11 and 10 bits.  With the moves, half kept: 32 heads of 16385 slots 79 us (of 16384, held
// in registers, 53), of 32768 154; 8 of 131072 408, one CU a head.
__global__ void __launch_bounds__(kSelect) tm_evict_select_kernel(EvictParams p) {
  __shared__ uint32_t s_bins[kBins];
  __shared__ int s_waves[kSelect / 64];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x;
  const Head head(p);
  // the keep-th largest key, 11, 11 and 10 bits at a time, and how many of its equals stay
  uint32_t prefix = 0;
  int need = p.keep;
  if (p.keep < p.length && p.keep > 0) {
    for (int shift = 21; shift >= 0; shift -= shift == 21 ? 11 : 10) {
      const int bits = shift == 0 ? 10 : 11;
      for (int i = tid; i < kBins; i += kSelect) s_bins[i] = 0;
      __syncthreads();
      for (int s = tid; s < p.length; s += kSelect) {
        const uint32_t k = head.key(s);
        if (shift == 21 || (k >> (shift + bits)) == prefix)
          atomicAdd(&s_bins[(k >> shift) & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      // from the largest bin down: two bins a thread
      const int hi = kBins - 1 - 2 * tid;
      const int c1 = (int)s_bins[hi], c0 = (int)s_bins[hi - 1];
      int v = c1 + c0;
      const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(v, d);
        if (lane >= d) v += up;
      }
      if (lane == 63) s_waves[wave] = v;
      __syncthreads();
      int before = v - c1 - c0;
      for (int w = 0; w < wave; ++w) before += s_waves[w];
      if (before < need && before + c1 + c0 >= need) {
        const bool first = before + c1 >= need;
        s_prefix = (prefix << bits) | (uint32_t)(first ? hi : hi - 1);
        s_need = need - before - (first ? 0 : c1);
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      if (shift == 0) break;
    }
  }
  // slot by slot: which stay, holes below keep and movers behind it
  const BlockRank ranked = {s_waves};
  int32_t* const holes = p.holes + (int64_t)head.index * p.moves;
  int32_t* const movers = p.movers + (int64_t)head.index * p.moves;
  float* const mass_out = p.mass_out + (int64_t)head.index * p.columns;
  int32_t* const pos_out = p.positions_out + (int64_t)head.index * p.keep;
  int equal0 = 0, hole0 = 0, mover0 = 0;
  const bool all = p.keep >= p.length;
  for (int s0 = 0; s0 < p.length; s0 += kSelect) {
    const int s = s0 + tid;
    const bool in = s < p.length;
    const uint32_t k = in ? head.key(s) : 0;
    int total;
    const int equal = equal0 + ranked(in && k == prefix, &total);
    equal0 += total;
    const bool kept = in && p.keep > 0 && (all || k > prefix || (k == prefix && equal < need));
    const bool hole = in && s < p.keep && !kept, mover = kept && s >= p.keep;
    const int h = hole0 + ranked(hole, &total);
    hole0 += total;
    const int m = mover0 + ranked(mover, &total);
    mover0 += total;
    if (hole && h < p.moves) holes[h] = s;
    if (mover && m < p.moves) movers[m] = s;
    if (kept && s < p.keep) {
      mass_out[s] = head.mass[s];
      pos_out[s] = head.position(s);
    }
  }
  for (int s = p.keep + tid; s < p.columns; s += kSelect) mass_out[s] = 0.0f;
  const int moves = min(min(hole0, mover0), p.moves);
  if (tid == 0) p.counts[head.index] = moves;
  __syncthreads();  // this workgroup's lists
  for (int i = tid; i < moves; i += kSelect) {
    const int to = holes[i], from = movers[i];
    mass_out[to] = head.mass[from];
    pos_out[to] = head.position(from);
  }
}

constexpr int kMovesOf = 64;  // of a workgroup

__global__ void __launch_bounds__(kThreads) tm_evict_move_kernel(EvictParams p) {
  const int head = blockIdx.y;
  const int layer = head / p.kvh, kvhead = head - layer * p.kvh;
  const int first = (int)blockIdx.x * kMovesOf;
  const int n = min(p.counts[head] - first, kMovesOf);
  const int pieces = p.row_bytes / 16;
  const int64_t base = (int64_t)layer * p.stride_layer + (int64_t)kvhead * p.stride_head;
  auto at = [&](int slot) {
    const int pg = min(max(p.table[slot >> p.page_shift], 0), p.cache_pages - 1);
    return base + (int64_t)pg * p.stride_page +
           (int64_t)(slot & ((1 << p.page_shift) - 1)) * p.stride_slot;
  };
  for (int i = threadIdx.x; i < n * pieces; i += kThreads) {
    const int move = i / pieces, piece = (i - move * pieces) * 16;
    const int64_t l = (int64_t)head * p.moves + first + move;
    const int64_t from = at(p.movers[l]) + piece, to = at(p.holes[l]) + piece;
    const u32x4_t a = *reinterpret_cast<const u32x4_t*>(p.k + from);
    const u32x4_t b = *reinterpret_cast<const u32x4_t*>(p.v + from);
    *reinterpret_cast<u32x4_t*>(p.k + to) = a;
    *reinterpret_cast<u32x4_t*>(p.v + to) = b;
  }
}

// ------------------------------------------------------------------- host --

constexpr int64_t kMaxStride = 1 << 24;
constexpr int64_t kHeld = 16 * kSelect;  // keys of a head that its workgroup holds
// Moves up to which the selecting workgroup makes them itself: a launch more against a CU a head
// that moves alone.  Measured, in us, by the workgroup and by a launch: 16 heads of 256
// moves 16.8, 18.0, of 512 19.9, 18.5; of 1000 moves 32 heads 16.7, 15.0, 64 17.6, 17.2, 128
// 24.7, 27.7, 256 39.5, 51; 128 heads of 4000 88, 75.
int64_t fused_moves(int64_t heads) { return std::max<int64_t>(256, 8 * heads); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct MassPlan {
  bool few, own, wide;
  int64_t rows, tiles, chunks, chunk_len;
  int64_t key_tiles, splits;               // of the sums
  int64_t stats, consts, parts, scores;    // floats of the workspace
  int64_t bytes;                           // of all of it
};

int plan_mass(int64_t T, int64_t S, int64_t Hq, int64_t kvh, int64_t hd, MassPlan* o) {
  if (kvh < 1 || Hq < kvh || Hq % kvh != 0 || Hq > 1024 || (hd != 64 && hd != 128))
    return TM_ERR_SHAPE;
  const int64_t group = Hq / kvh;
  if (T < 0 || S < T || S > TM_MAX_PROMPT_KEYS || T * group > INT32_MAX - 1024)
    return TM_ERR_SHAPE;
  o->rows = T * group;
  o->few = o->rows <= 32;
  o->own = o->rows <= kOwnRows;
  o->tiles = ceil_div(o->rows, o->few ? 32 : 128);
  // ranges of keys as many as fill the chip, of four stages or more.  Many tiles leave it
  // uneven with one workgroup a CU: 800 rows over 7200 keys in us with 1, 2 and 3 a CU 56, 48,
  // 50; 4000 over 4000 110, 90, 89; but 256 over 7464, whose sums join the ranges themselves,
  // 23.3 with 1, 24.2 with 2.
  const int64_t units = std::max<int64_t>(o->tiles * kvh, 1);
  const int64_t want = std::max<int64_t>(1, (units < 32 ? kCUs : 2 * kCUs) / units);
  const int64_t chunks = std::max<int64_t>(1, std::min(want, ceil_div(S, 4 * kKeys)));
  const int64_t step = o->few ? 4 * kKeys : kKeys;
  o->chunk_len = std::max(step, ceil_div(ceil_div(S, chunks), step) * step);
  o->chunks = std::max<int64_t>(1, ceil_div(S, o->chunk_len));
  // The sums' keys by eight waves where those tiles give half the CUs one, else by four (which
  // read the rows twice as often): 4096 tokens over themselves 172 us in all, by four 176; 2048
  // 67, 62; 512 27, 21.  Their rows in parts of eight or four stages or more, four workgroups a
  // CU: 4096 tokens with two a CU 189, with eight 176 where four gave 177.
  o->wide = !o->own && ceil_div(S, 256) * kvh >= kCUs / 2;
  o->key_tiles = ceil_div(S, o->wide ? 256 : 128);
  const int64_t stages = ceil_div(o->rows, kKeys);
  const int64_t splits = 4 * kCUs / std::max<int64_t>(o->key_tiles * kvh, 1);
  o->splits =
      o->own ? 1 : std::max<int64_t>(1, std::min(splits, stages / (o->wide ? 8 : 4)));
  o->stats = o->own || o->chunks > 1 ? 2 * o->chunks * kvh * o->rows : 0;
  o->consts = o->own ? 0 : kvh * stages * kKeys;
  o->parts = o->splits > 1 ? o->splits * kvh * S : 0;
  o->stats = ceil_div(o->stats, 4) * 4;    // (16-byte stores behind them)
  o->scores = o->few ? kvh * o->rows * ceil_div(S, kKeys) * kKeys : 0;
  o->bytes = 4 * (o->stats + o->consts + o->parts + o->scores);
  if (o->tiles * o->chunks * kvh > UINT32_MAX / kThreads ||
      o->key_tiles * o->splits * kvh > UINT32_MAX / 512 || kvh * stages * kKeys > UINT32_MAX)
    return TM_ERR_SHAPE;
  return TM_OK;
}

template <int DT, int HD>
void launch_mass(const MassParams& p, const MassPlan& o, hipStream_t st) {
  const dim3 block(kThreads);
  const dim3 items((unsigned)(o.tiles * o.chunks * p.kvh));
  const dim3 sums((unsigned)(o.key_tiles * o.splits * p.kvh));
  if (o.rows > 0) {
    if (o.few)
      hipLaunchKernelGGL((tm_mass_stats_few_kernel<DT, HD>), items, block, 0, st, p);
    else
      hipLaunchKernelGGL((tm_mass_stats_kernel<DT, HD>), items, block, 0, st, p);
  }
  if (o.few) {
    hipLaunchKernelGGL(tm_mass_kept_kernel,
                       dim3((unsigned)(ceil_div(p.k_len, kThreads) * p.kvh)), block, 0, st, p);
    return;
  }
  if (o.own) {
    hipLaunchKernelGGL((tm_mass_sum_kernel<DT, HD, 4, true>), sums, block, 0, st, p);
    return;
  }
  const int64_t whole = ceil_div(o.rows, kKeys) * kKeys;
  if (o.chunks > 1)
    hipLaunchKernelGGL(tm_mass_rows_kernel, dim3((unsigned)ceil_div(p.kvh * whole, kThreads)),
                       block, 0, st, p, (int)o.rows, (int)whole);
  if (o.wide)
    hipLaunchKernelGGL((tm_mass_sum_kernel<DT, HD, 8, false>), sums, dim3(512), 0, st, p);
  else
    hipLaunchKernelGGL((tm_mass_sum_kernel<DT, HD, 4, false>), sums, block, 0, st, p);
  if (o.splits > 1)
    hipLaunchKernelGGL(tm_mass_join_kernel,
                       dim3((unsigned)ceil_div(p.k_len, kThreads), (unsigned)p.kvh), block, 0, st,
                       p);
}

int page_shift_of(int64_t page_size) {
  int shift = 0;
  while ((int64_t(1) << shift) < page_size) ++shift;
  return shift;
}
bool pages_ok(int64_t page_size, int64_t cache_pages, int64_t num_table_pages, int64_t length) {
  return page_size >= 1 && page_size <= (1 << 24) && (page_size & (page_size - 1)) == 0 &&
         cache_pages >= 1 && cache_pages <= INT32_MAX && num_table_pages <= INT32_MAX &&
         ceil_div(length, page_size) <= num_table_pages;
}

struct EvictPlan {
  int64_t heads, moves, bytes;
};
int plan_evict(int64_t L, int64_t kvh, int64_t length, int64_t keep, EvictPlan* o) {
  if (L < 0 || L > 65535 || kvh < 1 || kvh > 1024 || length < 0 || length > TM_MAX_PROMPT_KEYS ||
      keep < 0 || keep > length || L * kvh > 65535)
    return TM_ERR_SHAPE;
  o->heads = L * kvh;
  o->moves = std::min(keep, length - keep);
  if (o->heads > 0 && ceil_div(o->moves, kMovesOf) > UINT32_MAX / kThreads / o->heads)
    return TM_ERR_SHAPE;  // a grid's threads in 32 bits
  o->bytes = 4 * (o->heads + 2 * o->heads * o->moves);
  return TM_OK;
}

}  // namespace

extern "C" int tm_mass_workspace(int64_t T, int64_t seq_len, int64_t Hq, int64_t kvh, int64_t hd,
                                 int64_t* bytes) {
  MassPlan o;
  const int rc = plan_mass(T, seq_len, Hq, kvh, hd, &o);
  if (rc) return rc;
  if (bytes == nullptr) return TM_ERR_ARG;
  *bytes = o.bytes;
  return TM_OK;
}

extern "C" int tm_attention_mass(const void* q, int64_t q_stride, int64_t T, const void* k_cache,
                                 int64_t stride_page, int64_t stride_slot, int64_t page_size,
                                 int64_t cache_pages, const int32_t* block_table,
                                 int64_t num_table_pages, int64_t seq_len, int64_t Hq,
                                 int64_t kvh, int64_t hd, float scale, int dtype,
                                 const float* before, int64_t before_stride, float* mass,
                                 int64_t mass_stride, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  MassPlan o;
  const int rc = plan_mass(T, seq_len, Hq, kvh, hd, &o);
  if (rc) return rc;
  if ((dtype != TM_DTYPE_BF16 && dtype != TM_DTYPE_F16) || !(scale > 0.0f) || scale == INFINITY)
    return TM_ERR_ARG;
  if (seq_len == 0) return TM_OK;
  if (!pages_ok(page_size, cache_pages, num_table_pages, seq_len) || stride_slot < kvh * hd ||
      stride_slot > kMaxStride || stride_page < page_size * stride_slot ||
      (T > 1 && q_stride < Hq * hd) || o.bytes > workspace_bytes ||
      (kvh > 1 && (mass_stride < seq_len || (before != nullptr && before_stride < seq_len))))
    return TM_ERR_SHAPE;
  if ((uintptr_t)q % 16 || (T > 1 && q_stride % 8) || (uintptr_t)k_cache % 16 ||
      stride_slot % 8 || stride_page % 8 || (uintptr_t)block_table % 4 || (uintptr_t)before % 4 ||
      (uintptr_t)mass % 4 || (uintptr_t)workspace % 16)
    return TM_ERR_ALIGN;
  MassParams p = {};
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k_cache;
  p.v = p.k;
  p.table = block_table;
  p.q_stride = q_stride;
  p.k_stride = p.v_stride = stride_slot;
  p.stride_page = stride_page;
  p.kvh = (int)kvh;
  p.group = (int)(Hq / kvh);
  p.q_len = (int)T;
  p.k_len = (int)seq_len;
  p.tiles = (int)o.tiles;
  p.chunks = (int)o.chunks;
  p.chunk_len = (int)o.chunk_len;
  p.page_shift = page_shift_of(page_size);
  p.cache_pages = (int)cache_pages;
  p.wide = page_size >= 16 ? 1 : 0;  // keys of a stage that a wave takes from one page
  p.scale_log2 = scale * 1.4426950408889634f;
  float* const at = (float*)workspace;
  p.row_stats = (float2*)at;
  p.row_consts = o.own ? nullptr : at + o.stats;
  p.parts = o.splits > 1 ? at + o.stats + o.consts : nullptr;
  p.scores = at + o.stats;  // (few only: nothing else lies there then)
  p.score_stride = ceil_div(seq_len, kKeys) * kKeys;
  p.splits = (int)o.splits;
  p.before = before;
  p.before_stride = before_stride;
  p.mass = mass;
  p.mass_stride = mass_stride;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TM_DTYPE_F16) {
    if (hd == 128)
      launch_mass<TM_DTYPE_F16, 128>(p, o, st);
    else
      launch_mass<TM_DTYPE_F16, 64>(p, o, st);
  } else {
    if (hd == 128)
      launch_mass<TM_DTYPE_BF16, 128>(p, o, st);
    else
      launch_mass<TM_DTYPE_BF16, 64>(p, o, st);
  }
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

extern "C" int tm_evict_workspace(int64_t L, int64_t kvh, int64_t seq_len, int64_t keep,
                                  int64_t* bytes) {
  EvictPlan o;
  const int rc = plan_evict(L, kvh, seq_len, keep, &o);
  if (rc) return rc;
  if (bytes == nullptr) return TM_ERR_ARG;
  *bytes = o.bytes;
  return TM_OK;
}

extern "C" int tm_evict(void* k_cache, void* v_cache, int64_t elem_bytes, int64_t L,
                        int64_t stride_layer, int64_t stride_page, int64_t stride_slot,
                        int64_t kvh, int64_t hd, int64_t page_size, int64_t cache_pages,
                        const int32_t* block_table, int64_t num_table_pages, int64_t seq_len,
                        int64_t keep, const float* mass, int64_t mass_layer, int64_t mass_head,
                        int64_t columns, const int32_t* positions, int64_t pos_layer,
                        int64_t pos_head, int64_t recorded, int64_t next_position,
                        int64_t recent, int64_t sinks, float* mass_out, int32_t* positions_out,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  EvictPlan o;
  const int rc = plan_evict(L, kvh, seq_len, keep, &o);
  if (rc) return rc;
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4) return TM_ERR_ARG;
  if (hd < 1 || hd > 65536 || columns < seq_len || columns > INT32_MAX - kSelect ||
      recorded < 0 || recorded > seq_len || (recorded > 0 && positions == nullptr) ||
      next_position < seq_len || next_position > INT32_MAX || recent < 0 || sinks < 0 ||
      sinks > INT32_MAX || o.bytes > workspace_bytes)
    return TM_ERR_SHAPE;
  if (o.heads == 0) return TM_OK;
  if (!pages_ok(page_size, cache_pages, num_table_pages, seq_len) || stride_slot < kvh * hd ||
      stride_slot > kMaxStride || stride_page < page_size * stride_slot ||
      (L > 1 && stride_layer < cache_pages * stride_page))
    return TM_ERR_SHAPE;
  if (hd * elem_bytes % 16 || stride_slot * elem_bytes % 16 || stride_page * elem_bytes % 16 ||
      (L > 1 && stride_layer * elem_bytes % 16) || (uintptr_t)k_cache % 16 ||
      (uintptr_t)v_cache % 16 || (uintptr_t)block_table % 4 || (uintptr_t)mass % 4 ||
      (uintptr_t)positions % 4 || (uintptr_t)mass_out % 4 || (uintptr_t)positions_out % 4 ||
      (uintptr_t)workspace % 4)
    return TM_ERR_ALIGN;
  EvictParams p = {};
  p.k = (uint8_t*)k_cache;
  p.v = (uint8_t*)v_cache;
  p.stride_layer = stride_layer * elem_bytes;
  p.stride_page = stride_page * elem_bytes;
  p.stride_slot = stride_slot * elem_bytes;
  p.stride_head = hd * elem_bytes;
  p.row_bytes = (int)(hd * elem_bytes);
  p.table = block_table;
  p.page_shift = page_shift_of(page_size);
  p.cache_pages = (int)cache_pages;
  p.kvh = (int)kvh;
  p.length = (int)seq_len;
  p.keep = (int)keep;
  p.moves = (int)o.moves;
  p.mass = mass;
  p.mass_layer = mass_layer;
  p.mass_head = mass_head;
  p.columns = (int)columns;
  p.positions = positions;
  p.pos_layer = pos_layer;
  p.pos_head = pos_head;
  p.recorded = (int)recorded;
  p.next = (int)next_position;
  p.recent = (int)std::min<int64_t>(recent, next_position);
  p.sinks = (int)sinks;
  p.mass_out = mass_out;
  p.positions_out = positions_out;
  p.counts = (int32_t*)workspace;
  p.holes = p.counts + o.heads;
  p.movers = p.holes + o.heads * o.moves;
  const hipStream_t st = (hipStream_t)stream;
  p.fused = seq_len <= kHeld && o.moves <= fused_moves(o.heads);
  const dim3 grid((unsigned)o.heads), block(kSelect);
  // Slots a thread and threads by what they hold, in us, and read again for each histogram:
  // 256 heads of 1088 slots by 4 of 512 threads 11, 8 of 1024 15, 16 21, read again 18; 64 of
  // 8000, half kept, by 8 48, 16 53, read again 62; 32 of 16000 by 16 58, read again 82.
  if (seq_len <= 2048)
    hipLaunchKernelGGL((tm_evict_held_kernel<4, 512>), grid, dim3(512), 0, st, p);
  else if (seq_len <= 8192)
    hipLaunchKernelGGL((tm_evict_held_kernel<8, 1024>), grid, block, 0, st, p);
  else if (seq_len <= kHeld)
    hipLaunchKernelGGL((tm_evict_held_kernel<16, 1024>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL(tm_evict_select_kernel, grid, block, 0, st, p);
  if (o.moves > 0 && !p.fused)
    hipLaunchKernelGGL(tm_evict_move_kernel,
                       dim3((unsigned)ceil_div(o.moves, kMovesOf), (unsigned)o.heads),
                       dim3(kThreads), 0, st, p);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}
