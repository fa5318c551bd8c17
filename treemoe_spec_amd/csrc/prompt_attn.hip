// Causal attention of a prompt's tokens, down to a single one, over packed sequences
// or over one sequence's pages of the KV cache:
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / group]) v[j, h / group],
//
// j over the sequence's keys 0 .. past + t, where past = its keys minus its queries.
//
// Decomposition.  The rows of a KV head are its sequence's (token, head of the group)
// pairs, token major, so neighbouring rows share every key and the causal border
// crosses a tile of 128 rows within 128 / group tokens.  A workgroup takes a tile of 32, 128
// or 256 such rows, 32 a wave, against one range of keys, 64 keys a stage; K and V rows go
// straight from memory to LDS (16 bytes a lane, no registers between), V transposed
// as it is read from there.  Few rows over many keys are split over key ranges; each
// leaves its sum, maximum and unnormalised output in fp32 in the workspace, which a
// second kernel joins in key order.  Four kernels (the rule between them: kind_of):
//   few    32 rows; four waves take the stages in turn, no barrier between them
//   short  128 rows, two workgroups a CU
//   pair   128 rows; eight waves, half of them on every other stage
//   tall   256 rows; eight waves
// In pair and tall one wave of a SIMD is in the matrix products while the other weighs.
//
// Bound by the power limit and the turns of products and exponentials at many rows: 8192
// tokens, 32 heads over 8 of 128 in bf16, 549 GFLOP in 525 us, 1.05 PFLOP/s, where a plain
// 16384^3 product reaches 1.39; the matrix pipe is busy in 48 % of the cycles, of a clock that
// power holds at 1.78 GHz.  4.0 k tokens 0.87 PFLOP/s.  Through pages of 16, in a graph: 8192
// tokens 579 us, packed 545; 4000 162, 147.  By HBM at few rows: one token over 40000 keys
// 32 us, 5.2 TB/s; over 7777 14.3 us, of which 2.5 are the second launch and about 6 the
// latency of one stage.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <utility>
#include <vector>

#include "attn_tile.h"
#include "prompt_parts.h"

namespace {

// Eight waves, two a SIMD, that take turns: one is in the matrix products of its stage
// while the other weighs, a barrier between the turns.  Tiles of 256 rows: every wave has
// 32 rows of its own, and all read the same stages.
template <int DT, int HD, bool PAGED>
__global__ void __launch_bounds__(512, 2) tm_prompt_tall_kernel(PromptParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k2[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v2[S::kTile];

  // KV heads innermost: with 8 of them a head's workgroups, which share its keys, run
  // on one XCD; the tiles with the most keys first
  const int kvhead = (int)blockIdx.x % p.kvh;
  const Item it = item_of(p, (int)blockIdx.x / p.kvh, 256);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  Rows<HD> r;
  const Place at = begin_rows<HD>(p, it, kvhead, it.tile * 256 + wave * 32, r);
  const int full = at.full;
  const int n = it.end > it.begin ? (it.end - it.begin + kKeys - 1) / kKeys : 0;
  const float scale_log2 = p.scale_log2;
  if (n > 0) {
    Feed<HD, PAGED, 8> feed;
    feed.start(p, it, kvhead, it.begin, kKeys);
    // Load group g(s), in ring slot s % 3: K of stage s and V of stage s - 1, what the
    // products M(s) = {O += V P of s - 1, S = K Q of s} read.  W(s) weighs stage s.
    // Waves 0-3 take M(s) in turn 2 s and W(s) in turn 2 s + 1, waves 4-7, which share
    // their SIMDs, one turn later.  A wave requests g(s + 2) behind its products M(s), the
    // late waves having left its slot in turn 2 s - 1; in turn 2 s + 1 all wait for their
    // part of g(s + 1).
    auto request = [&](int s, uint8_t* kn, uint8_t* vn) TM_INLINE {
      if (s > n) return;
      if (s > 0) feed.load_v(p, vn);
      if (s < n) feed.load_k(p, kn);
    };
    // this wave's part of g(s) is there; g(s + 1) may be under way
    auto await = [&](int s) TM_INLINE {
      if (s + 1 < n)
        wait_vm<Feed<HD, PAGED, 8>::kGroup>();
      else
        wait_vm<0>();
    };
    // W(s) and M(s + 1), which reads g(s + 1) at kc, vc; g(s + 3) goes to kn, vn.  (The last
    // one's scores, of a stage that is not there, are not used.)
    auto early = [&](int s, uint8_t* kc, uint8_t* vc, uint8_t* kn, uint8_t* vn) TM_INLINE {
      const int kb = it.begin + s * kKeys;
      weigh<DT, HD>(scale_log2, kb, kb + kKeys - 1 > full, r.seen, r);
      await(s + 1);
      turn_end();
      products<DT, HD, true, true>(vc, kc, r);
      request(s + 3, kn, vn);
      turn_end();
    };
    auto late = [&](int s, uint8_t* kc, uint8_t* vc, uint8_t* kn, uint8_t* vn) TM_INLINE {
      const int kb = it.begin + s * kKeys;
      weigh<DT, HD>(scale_log2, kb, kb + kKeys - 1 > full, r.seen, r);
      turn_end();
      products<DT, HD, true, true>(vc, kc, r);
      request(s + 3, kn, vn);
      await(s + 2);
      turn_end();
    };
    request(0, s_k0, s_v0);
    request(1, s_k1, s_v1);
    wait_vm<0>();
    turn_end();
    int s = 0;
    if (wave < 4) {
      products<DT, HD, false, true>(s_v0, s_k0, r);
      request(2, s_k2, s_v2);
      turn_end();
      for (; s + 3 <= n; s += 3) {
        early(s, s_k1, s_v1, s_k0, s_v0);
        early(s + 1, s_k2, s_v2, s_k1, s_v1);
        early(s + 2, s_k0, s_v0, s_k2, s_v2);
      }
      if (s < n) early(s, s_k1, s_v1, s_k0, s_v0);
      if (s + 1 < n) early(s + 1, s_k2, s_v2, s_k1, s_v1);
      turn_end();
    } else {
      turn_end();
      products<DT, HD, false, true>(s_v0, s_k0, r);
      request(2, s_k2, s_v2);
      await(1);
      turn_end();
      for (; s + 3 <= n; s += 3) {
        late(s, s_k1, s_v1, s_k0, s_v0);
        late(s + 1, s_k2, s_v2, s_k1, s_v1);
        late(s + 2, s_k0, s_v0, s_k2, s_v2);
      }
      if (s < n) late(s, s_k1, s_v1, s_k0, s_v0);
      if (s + 1 < n) late(s + 1, s_k2, s_v2, s_k1, s_v1);
    }
  }
  retake<DT, HD, Feed<HD, PAGED, 8>>(p, it, kvhead, 0, 1, n, r);
  end_rows<DT, HD>(p, it, kvhead, 256, at, r);
}

template <int DT, int HD, bool PAGED>
__global__ void __launch_bounds__(512, 2) tm_prompt_pair_kernel(PromptParams p) {
  __shared__ PairShared<HD> lds;
  const Item it = item_of(p, (int)blockIdx.x / p.kvh, 128);
  pair_body<DT, HD, Feed<HD, PAGED, 4>>(p, it, (int)blockIdx.x % p.kvh, lds);
}

template <int DT, int HD, bool PAGED>
__global__ void __launch_bounds__(kThreads, 2) tm_prompt_short_kernel(PromptParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v1[S::kTile];
  const Item it = item_of(p, (int)blockIdx.x / p.kvh, 128);
  short_body<DT, HD, Feed<HD, PAGED, 4>>(p, it, (int)blockIdx.x % p.kvh, s_k0, s_v0, s_k1, s_v1);
}

template <int DT, int HD, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) tm_prompt_few_kernel(PromptParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k[4][S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v[4][S::kTile];
  __shared__ float s_stat[4][32][2];
  const Item it = item_of(p, (int)blockIdx.x / p.kvh, 32);
  few_body<DT, HD, Feed<HD, PAGED, 1>>(p, it, (int)blockIdx.x % p.kvh, s_k, s_v, s_stat);
}

constexpr int kMaxChunks = 512;  // of one tile's keys

// The tile that a join's unit `at` stands for.
__device__ __forceinline__ Join join_of(const PromptParams& p, int at) {
  if (p.joins != nullptr) return p.joins[at];
  Join j;
  j.q0 = 0;
  j.q_len = p.q_len;
  j.tile = at;
  j.slot0 = at * p.chunks;
  j.count = p.chunks;
  return j;
}

// Joins the partials of 32 rows' 32 columns, a wave each, in chunk order: lane l has row
// l % 32 and the columns that the partials' layout gives it.  `blocks`: of 32 rows in a tile
// that may hold some.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads) tm_prompt_join_tiles_kernel(PromptParams p,
                                                                        int tile_rows,
                                                                        int blocks) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  int unit = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  const int ht = unit % (HD / 32);
  unit /= HD / 32;
  const int first = unit % blocks * 32 + (lane & 31);
  unit /= blocks;
  const int kvhead = unit % p.kvh, at = unit / p.kvh;
  if (p.joins == nullptr && at >= p.tiles) return;
  const Join j = join_of(p, at);
  const int row = j.tile * tile_rows + first;
  if (row >= j.q_len * p.group) return;
  const int64_t slot0 = ((int64_t)j.slot0 * p.kvh + kvhead) * tile_rows + first;
  const int64_t step = (int64_t)p.kvh * tile_rows;  // from chunk to chunk
  const float* const stats = p.stats + slot0 * 2;
  const float* const from = p.part + (slot0 - (lane & 31)) * HD + 1024 * ht + 4 * lane;
  float m = -INFINITY;
#pragma unroll 4
  for (int c = 0; c < j.count; ++c) m = fmaxf(m, stats[c * step * 2]);
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
  f32x4_t o[4] = {};
#pragma unroll 4
  for (int c = 0; c < j.count; ++c) {
    const float a = __builtin_amdgcn_exp2f(stats[c * step * 2] - ref);
    sum += stats[c * step * 2 + 1] * a;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(from + c * step * HD + 256 * x);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[x][e] = fmaf(v[e], a, o[x][e]);
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
    store_row<DT>(p, j.q0, row, kvhead, HD, 32 * ht + 8 * x + 4 * half, o[x], sum);
}

// Joins the partials of one row of few, a wave each: the maximum and the sum over the chunks
// first, a lane per chunk, then the weighted outputs in chunk order, four elements a
// lane and the lanes' groups a chunk each.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads) tm_prompt_join_kernel(PromptParams p, int tile_rows,
                                                                  int rows) {
  __shared__ float s_a[4][kMaxChunks];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int unit = (int)blockIdx.x * 4 + wave;
  const int r = unit % rows;          // of the tile's `rows` that may hold some
  const int kv = unit / rows;
  const int kvhead = kv % p.kvh, at = kv / p.kvh;
  if (p.joins == nullptr && at >= p.tiles) return;
  const Join j = join_of(p, at);
  const int row = j.tile * tile_rows + r;
  if (row >= j.q_len * p.group) return;
  const int64_t slot0 = ((int64_t)j.slot0 * p.kvh + kvhead) * tile_rows + r;
  const int64_t step = (int64_t)p.kvh * tile_rows;  // from chunk to chunk
  float m = -INFINITY;
  for (int c = lane; c < j.count; c += 64) m = fmaxf(m, p.stats[(slot0 + c * step) * 2]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
  for (int c = lane; c < j.count; c += 64) {
    const float a = __builtin_amdgcn_exp2f(p.stats[(slot0 + c * step) * 2] - ref);
    sum += p.stats[(slot0 + c * step) * 2 + 1] * a;
    s_a[wave][c] = a;
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  constexpr int kLanes = HD / 4, kGroups = 64 / kLanes;
  const float* const from = p.part + slot0 * HD + 4 * (lane % kLanes);
  f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int c = lane / kLanes; c < j.count; c += kGroups) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(from + c * step * HD);
    const float a = s_a[wave][c];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], a, o[e]);
  }
#pragma unroll
  for (int d = 32; d >= kLanes; d >>= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], d);
  if (lane < kLanes) store_row<DT>(p, j.q0, row, kvhead, HD, 4 * lane, o, sum);
}

// ------------------------------------------------------------------- host --

constexpr int64_t kMaxStride = 1 << 24;  // of a key's row: 64 of them from 32-bit offsets
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Keys of tile `tile` of a sequence: those before the border of its last row.
int64_t tile_keys(int64_t q_len, int64_t k_len, int64_t tile, int64_t rows, int64_t group) {
  const int64_t last = std::min(q_len - 1, (tile * rows + rows - 1) / group);
  return k_len - q_len + last + 1;
}

// How the rows are tiled, by the rows of the longest sequence, the tiles of 128 rows of all
// sequences, and their stages of 64 keys on average:
//   few    no sequence has more than 32 rows: a decoded token's heads;
//   tall   3.5 tiles a CU or more, of 24 stages or more;
//   pair   fewer tiles, of 8 stages or more;
//   short  otherwise.
// Measured on one head shape, 32 query heads over 8 of 128 elements (heads of 64, whose stages
// are half the work, take the same thresholds), the three tilings in us: one prompt of
// 517 tokens short 21, pair 21; 1000 tokens 35, 25, tall 38; 2048 59, 52, 63; 4000 164, 160,
// 150; 8192 pair 554, tall 520; 12 prompts of 1-2048 tokens (fp16) short 77, pair 102, tall
// 85; 20 of 100 short 18, pair 27, tall 22; 300 tokens over 1000 cached short 32, pair
// 30.  Where a CU goes through several tiles of few stages, the two workgroups of `short`
// hide each other's first loads and last stores.
enum Kind { kFew, kShort, kPair, kTall, kKinds };
constexpr int64_t kTileRows[kKinds] = {32, 128, 128, 256};
// Keys that a workgroup takes in one step, and workgroups that the chip holds.
constexpr int64_t kStepKeys[kKinds] = {4 * kKeys, kKeys, 2 * kKeys, kKeys};
constexpr int64_t kSlots[kKinds] = {kCUs, 2 * kCUs, kCUs, kCUs};
// Keys of a stage that a wave takes from one page (of few, one of four parts).
constexpr int64_t kPartKeys[kKinds] = {kKeys / 4, kKeys / 4, kKeys / 4, kKeys / 8};

Kind kind_of(int64_t longest, int64_t units128, int64_t stages128) {
  if (longest <= 32) return kFew;
  if (2 * units128 >= 7 * kCUs) return stages128 >= 24 * units128 ? kTall : kShort;
  return stages128 >= 8 * units128 ? kPair : kShort;
}

// Key ranges of one sequence's tiles: as many as fill the chip, at least four stages each.
int64_t chunks_of(Kind kind, int64_t units, int64_t keys) {
  const int64_t want = std::min<int64_t>(kSlots[kind] / std::max<int64_t>(units, 1), kMaxChunks);
  return std::max<int64_t>(1, std::min(want, ceil_div(keys, 4 * kKeys)));
}

int check_heads(int64_t Hq, int64_t kvh, int64_t hd) {
  if (kvh < 1 || Hq < kvh || Hq % kvh != 0 || Hq > 1024 || (hd != 64 && hd != 128))
    return TM_ERR_SHAPE;
  return TM_OK;
}

struct OnePlan {
  Kind kind;
  int64_t rows, tiles, chunks, chunk_len, bytes;
};

int plan_one(int64_t T, int64_t S, int64_t Hq, int64_t kvh, int64_t hd, OnePlan* o) {
  const int64_t group = Hq / kvh;
  if (T < 0 || S < T || S > TM_MAX_PROMPT_KEYS || T * group > INT32_MAX - 1024)
    return TM_ERR_SHAPE;
  const int64_t tiles128 = ceil_div(T * group, 128);
  int64_t stages = 0;  // of the tiles of 128, at their mean
  if (T > 0)
    stages = tiles128 * ceil_div(tile_keys(T, S, 0, 128, group) +
                                     tile_keys(T, S, tiles128 - 1, 128, group), 2 * kKeys);
  const int64_t units = tiles128 * kvh;
  o->kind = kind_of(T * group, units, stages * kvh);
  // Tiles that leave many CUs without one, in their only turn or in the last of two: a CU
  // each to `short` workgroups over a third of the keys, where the keys are many enough to
  // pay for the join.  Measured, 32 heads over 8 of 128, whole tiles and thirds in us: 517
  // tokens of 2000 36, 37; of 4613 72, 62; of 10000 147, 115; 1100 of 9000 249, 201; but 700
  // of 6000, whose thirds do not fit one turn, 91, 113.
  const bool thirds = o->kind == kPair && units > kCUs / 2 &&
                      3 * units <= 2 * kCUs * ceil_div(units, kCUs) && stages >= 48 * tiles128;
  if (thirds) o->kind = kShort;
  o->rows = kTileRows[o->kind];
  o->tiles = ceil_div(T * group, o->rows);
  o->chunks = thirds ? 3 : chunks_of(o->kind, o->tiles * kvh, S);
  const int64_t step = kStepKeys[o->kind];
  o->chunk_len = std::max(step, ceil_div(ceil_div(S, o->chunks), step) * step);
  o->chunks = std::max<int64_t>(1, ceil_div(S, o->chunk_len));
  o->bytes = o->chunks > 1 ? o->tiles * o->chunks * kvh * o->rows * (hd + 2) * 4 : 0;
  return TM_OK;
}

template <int DT, int HD, bool PAGED>
void launch_kind(const PromptParams& p, Kind kind, int64_t blocks, int64_t joins,
                 int64_t join_rows, hipStream_t st) {
  const dim3 grid((unsigned)blocks), block(kThreads);
  if (kind == kFew)
    hipLaunchKernelGGL((tm_prompt_few_kernel<DT, HD, PAGED>), grid, block, 0, st, p);
  else if (kind == kShort)
    hipLaunchKernelGGL((tm_prompt_short_kernel<DT, HD, PAGED>), grid, block, 0, st, p);
  else if (kind == kPair)
    hipLaunchKernelGGL((tm_prompt_pair_kernel<DT, HD, PAGED>), grid, dim3(512), 0, st, p);
  else
    hipLaunchKernelGGL((tm_prompt_tall_kernel<DT, HD, PAGED>), grid, dim3(512), 0, st, p);
  if (joins == 0) return;
  const int tile_rows = (int)kTileRows[kind];
  if (kind == kFew) {
    hipLaunchKernelGGL((tm_prompt_join_kernel<DT, HD>),
                       dim3((unsigned)ceil_div(joins * p.kvh * join_rows, 4)), block, 0, st, p,
                       tile_rows, (int)join_rows);
  } else {
    // (whole tiles, as packed sequences have them, make whole workgroups)
    const int64_t blocks32 = ceil_div(join_rows, 32);
    hipLaunchKernelGGL((tm_prompt_join_tiles_kernel<DT, HD>),
                       dim3((unsigned)ceil_div(joins * p.kvh * blocks32 * (HD / 32), 4)), block,
                       0, st, p, tile_rows, (int)blocks32);
  }
}

template <bool PAGED>
void launch(const PromptParams& p, int dtype, int64_t hd, Kind kind, int64_t blocks,
            int64_t joins, int64_t join_rows, hipStream_t st) {
  if (dtype == TM_DTYPE_F16) {
    if (hd == 128)
      launch_kind<TM_DTYPE_F16, 128, PAGED>(p, kind, blocks, joins, join_rows, st);
    else
      launch_kind<TM_DTYPE_F16, 64, PAGED>(p, kind, blocks, joins, join_rows, st);
  } else {
    if (hd == 128)
      launch_kind<TM_DTYPE_BF16, 128, PAGED>(p, kind, blocks, joins, join_rows, st);
    else
      launch_kind<TM_DTYPE_BF16, 64, PAGED>(p, kind, blocks, joins, join_rows, st);
  }
}

// A grid counts its threads in 32 bits.
bool grids_ok(Kind kind, int64_t blocks, int64_t joins_rows) {
  const int64_t threads = kind == kPair || kind == kTall ? 512 : kThreads;
  return blocks <= UINT32_MAX / threads && joins_rows <= UINT32_MAX / 64;
}

bool vec_ok(const void* p, int64_t stride, int64_t tokens) {
  return (uintptr_t)p % 16 == 0 && (tokens <= 1 || stride % 8 == 0);
}

}  // namespace

int tm_prefix_plan(int64_t T, int64_t S, int64_t Hq, int64_t kvh, PrefixPlan* o) {
  const int64_t group = Hq / kvh, rows = T * group;
  if (T < 0 || S < 0 || S > TM_MAX_PROMPT_KEYS || rows > INT32_MAX - 1024) return TM_ERR_SHAPE;
  const int64_t units = ceil_div(rows, 128) * kvh;
  const Kind kind = kind_of(rows, units, units * ceil_div(S, kKeys));
  o->kind = kind;
  o->tile_rows = kTileRows[kind];
  o->tiles = ceil_div(rows, o->tile_rows);
  o->part_rows = kind == kFew ? rows : o->tile_rows;
  const int64_t chunks = chunks_of(kind, o->tiles * kvh, S), step = kStepKeys[kind];
  o->chunk_len = std::max(step, ceil_div(ceil_div(S, chunks), step) * step);
  o->chunks = ceil_div(S, o->chunk_len);
  if (!grids_ok(kind, o->tiles * o->chunks * kvh, 0)) return TM_ERR_SHAPE;
  return TM_OK;
}

void tm_prefix_launch(PromptParams p, const PrefixPlan& o, int dtype, int64_t hd,
                      int64_t page_size, hipStream_t st) {
  p.tiles = (int)o.tiles;
  p.chunks = (int)o.chunks;
  p.chunk_len = (int)o.chunk_len;
  p.part_rows = (int)o.part_rows;
  p.whole = 1;
  p.wide = page_size >= kPartKeys[o.kind] ? 1 : 0;
  launch<true>(p, dtype, hd, (Kind)o.kind, o.tiles * o.chunks * p.kvh, 0, 0, st);
}

extern "C" int tm_prompt_plan(const int64_t* q_lens, const int64_t* k_lens, int64_t B, int64_t Hq,
                              int64_t kvh, int32_t* items, int64_t max_items, int32_t* joins,
                              int64_t max_joins, int64_t* sizes) try {
  int rc = check_heads(Hq, kvh, 128);
  if (rc) return rc;
  if (sizes == nullptr || B < 0 || (B > 0 && (q_lens == nullptr || k_lens == nullptr)))
    return TM_ERR_ARG;
  const int64_t group = Hq / kvh;
  int64_t units = 0, stages = 0, q_rows = 0, k_rows = 0, longest = 0;
  for (int64_t b = 0; b < B; ++b) {
    if (q_lens[b] < 0 || k_lens[b] < q_lens[b] || k_lens[b] > TM_MAX_PROMPT_KEYS)
      return TM_ERR_SHAPE;
    q_rows += q_lens[b];
    k_rows += k_lens[b];
    if (q_rows * group > INT32_MAX - 1024 || k_rows > INT32_MAX) return TM_ERR_SHAPE;
    units += ceil_div(q_lens[b] * group, 128) * kvh;
    longest = std::max(longest, q_lens[b] * group);
    for (int64_t t = 0; t * 128 < q_lens[b] * group; ++t)
      stages += ceil_div(tile_keys(q_lens[b], k_lens[b], t, 128, group), kKeys) * kvh;
  }
  const Kind kind = kind_of(longest, units, stages);
  const int64_t rows = kTileRows[kind], step = kStepKeys[kind];
  // stages of all workgroups, and how many one of them may have before its keys are
  // split: twice an even share of the chip's slots
  stages = 0;
  for (int64_t b = 0; b < B; ++b)
    for (int64_t t = 0; t * rows < q_lens[b] * group; ++t)
      stages += ceil_div(tile_keys(q_lens[b], k_lens[b], t, rows, group), kKeys) * kvh;
  const int64_t share = std::max<int64_t>(4, ceil_div(stages, kSlots[kind]));
  std::vector<std::pair<int64_t, Item>> list;  // (keys, item)
  std::vector<Join> jlist;
  int64_t q0 = 0, k0 = 0, slots = 0;
  for (int64_t b = 0; b < B; ++b) {
    for (int64_t t = 0; t * rows < q_lens[b] * group; ++t) {
      const int64_t keys = tile_keys(q_lens[b], k_lens[b], t, rows, group);
      const int64_t n = ceil_div(keys, kKeys);
      const int64_t chunks = n > 2 * share ? ceil_div(n, share) : 1;
      const int64_t len = ceil_div(ceil_div(n, chunks) * kKeys, step) * step;
      const int64_t parts = ceil_div(keys, len);
      for (int64_t c = 0; c < parts; ++c) {
        Item it;
        it.q0 = (int)q0;
        it.q_len = (int)q_lens[b];
        it.k0 = (int)k0;
        it.k_len = (int)k_lens[b];
        it.tile = (int)t;
        it.begin = (int)(c * len);
        it.end = (int)std::min(keys, (c + 1) * len);
        it.slot = parts > 1 ? (int)(slots + c) : -1;
        list.push_back({it.end - it.begin, it});
      }
      if (parts > 1) {
        Join j = {};
        j.q0 = (int)q0;
        j.q_len = (int)q_lens[b];
        j.tile = (int)t;
        j.slot0 = (int)slots;
        j.count = (int)parts;
        jlist.push_back(j);
        slots += parts;
      }
    }
    q0 += q_lens[b];
    k0 += k_lens[b];
  }
  sizes[0] = (int64_t)list.size();
  sizes[1] = (int64_t)jlist.size();
  sizes[2] = slots;
  sizes[3] = kind;
  sizes[4] = q_rows;
  sizes[5] = k_rows;
  sizes[6] = rows;
  if (items == nullptr && joins == nullptr) return TM_OK;
  if (max_items < sizes[0] || max_joins < sizes[1]) return TM_ERR_SHAPE;
  if ((items == nullptr && !list.empty()) || (joins == nullptr && !jlist.empty()))
    return TM_ERR_ARG;
  std::stable_sort(list.begin(), list.end(),
                   [](const auto& a, const auto& b) { return a.first > b.first; });
  for (size_t i = 0; i < list.size(); ++i)
    memcpy(items + 8 * i, &list[i].second, sizeof(Item));
  if (!jlist.empty()) memcpy(joins, jlist.data(), jlist.size() * sizeof(Join));
  return TM_OK;
} catch (const std::bad_alloc&) {
  return TM_ERR_SHAPE;  // more work items than the host has memory for
}

extern "C" int tm_prompt_attention(const void* q, int64_t q_stride, const void* k,
                                   int64_t k_stride, const void* v, int64_t v_stride,
                                   const int32_t* items, int64_t num_items, const int32_t* joins,
                                   int64_t num_joins, int64_t num_slots, int64_t tiling,
                                   int64_t Hq, int64_t kvh, int64_t hd, float scale, int dtype,
                                   void* out, int64_t out_stride, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  int rc = check_heads(Hq, kvh, hd);
  if (rc) return rc;
  if ((dtype != TM_DTYPE_BF16 && dtype != TM_DTYPE_F16) || !(scale > 0.0f) || scale == INFINITY)
    return TM_ERR_ARG;
  if (tiling < 0 || tiling >= kKinds) return TM_ERR_ARG;
  const int64_t tile_rows = kTileRows[tiling];
  if (num_items < 0 || num_joins < 0 || num_slots < 0 || num_items > INT32_MAX ||
      num_joins > num_items || num_slots > num_items ||
      !grids_ok((Kind)tiling, num_items * kvh, num_joins * kvh * tile_rows))
    return TM_ERR_SHAPE;
  if (q_stride < Hq * hd || out_stride < Hq * hd || k_stride < kvh * hd || v_stride < kvh * hd ||
      k_stride > kMaxStride || v_stride > kMaxStride)
    return TM_ERR_SHAPE;
  if (num_slots * kvh * tile_rows * (hd + 2) * 4 > workspace_bytes) return TM_ERR_SHAPE;
  if (num_items == 0) return TM_OK;
  if (!vec_ok(q, q_stride, 2) || !vec_ok(k, k_stride, 2) || !vec_ok(v, v_stride, 2) ||
      !vec_ok(out, out_stride, 2) || (uintptr_t)items % 32 || (uintptr_t)joins % 32 ||
      (uintptr_t)workspace % 16)
    return TM_ERR_ALIGN;
  // (without lists the kernels would take one sequence by arithmetic)
  if (items == nullptr || (num_joins > 0 && joins == nullptr)) return TM_ERR_ARG;
  PromptParams p = {};
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k;
  p.v = (const uint16_t*)v;
  p.out = (uint16_t*)out;
  p.items = (const Item*)items;
  p.joins = (const Join*)joins;
  p.part = (float*)workspace;
  p.stats = (float*)workspace + num_slots * kvh * tile_rows * hd;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.out_stride = out_stride;
  p.kvh = (int)kvh;
  p.group = (int)(Hq / kvh);
  p.part_rows = 32;
  p.scale_log2 = scale * 1.4426950408889634f;
  launch<false>(p, dtype, hd, (Kind)tiling, num_items * kvh, num_joins, tile_rows,
                (hipStream_t)stream);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

extern "C" int tm_prompt_cached_workspace(int64_t T, int64_t seq_len, int64_t Hq, int64_t kvh,
                                          int64_t hd, int64_t* bytes) {
  int rc = check_heads(Hq, kvh, hd);
  if (rc) return rc;
  if (bytes == nullptr) return TM_ERR_ARG;
  OnePlan o;
  rc = plan_one(T, seq_len, Hq, kvh, hd, &o);
  if (rc) return rc;
  *bytes = o.bytes;
  return TM_OK;
}

extern "C" int tm_prompt_attention_cached(const void* q, int64_t q_stride, int64_t T,
                                          const void* k_cache, const void* v_cache,
                                          int64_t stride_page, int64_t stride_slot,
                                          int64_t page_size, int64_t cache_pages,
                                          const int32_t* block_table, int64_t num_table_pages,
                                          int64_t seq_len, int64_t Hq, int64_t kvh, int64_t hd,
                                          float scale, int dtype, void* out, int64_t out_stride,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_heads(Hq, kvh, hd);
  if (rc) return rc;
  if ((dtype != TM_DTYPE_BF16 && dtype != TM_DTYPE_F16) || !(scale > 0.0f) || scale == INFINITY)
    return TM_ERR_ARG;
  OnePlan o;
  rc = plan_one(T, seq_len, Hq, kvh, hd, &o);
  if (rc) return rc;
  if (page_size < 1 || page_size > (1 << 24) || (page_size & (page_size - 1)) != 0 ||
      cache_pages < 0 || cache_pages > INT32_MAX || num_table_pages < 0 ||
      num_table_pages > INT32_MAX)
    return TM_ERR_SHAPE;
  if (T == 0) return TM_OK;
  if (cache_pages < 1 || ceil_div(seq_len, page_size) > num_table_pages) return TM_ERR_SHAPE;
  if ((T > 1 && (q_stride < Hq * hd || out_stride < Hq * hd)) || stride_slot < kvh * hd ||
      stride_slot > kMaxStride || stride_page < page_size * stride_slot)
    return TM_ERR_SHAPE;
  if (o.bytes > workspace_bytes ||
      !grids_ok(o.kind, o.tiles * o.chunks * kvh, o.chunks > 1 ? o.tiles * kvh * o.rows : 0))
    return TM_ERR_SHAPE;
  if (!vec_ok(q, q_stride, T) || !vec_ok(out, out_stride, T) || !vec_ok(k_cache, stride_slot, 2) ||
      !vec_ok(v_cache, stride_page, 2) || (uintptr_t)block_table % 4 || (uintptr_t)workspace % 16)
    return TM_ERR_ALIGN;
  PromptParams p = {};
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k_cache;
  p.v = (const uint16_t*)v_cache;
  p.out = (uint16_t*)out;
  p.table = block_table;
  p.part = (float*)workspace;
  p.stats = (float*)workspace + o.tiles * o.chunks * kvh * o.rows * hd;
  p.q_stride = q_stride;
  p.k_stride = p.v_stride = stride_slot;
  p.out_stride = out_stride;
  p.stride_page = stride_page;
  p.kvh = (int)kvh;
  p.group = (int)(Hq / kvh);
  p.q_len = (int)T;
  p.k_len = (int)seq_len;
  p.tiles = (int)o.tiles;
  p.chunks = (int)o.chunks;
  p.chunk_len = (int)o.chunk_len;
  int shift = 0;
  while ((int64_t(1) << shift) < page_size) ++shift;
  p.page_shift = shift;
  p.cache_pages = (int)cache_pages;
  p.wide = page_size >= kPartKeys[o.kind] ? 1 : 0;
  p.part_rows = 32;
  p.scale_log2 = scale * 1.4426950408889634f;
  launch<true>(p, dtype, hd, o.kind, o.tiles * o.chunks * kvh, o.chunks > 1 ? o.tiles : 0,
               std::min(o.rows, T * p.group), (hipStream_t)stream);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}
