// Attention of branches of one sequence: requests behind a shared prompt, beams, drafts.
// Branch b's tokens attend to all S positions of the sequence, in the pages of its cache,
// and causally to what the branch itself holds: len_b keys in the branch cache and the
// tokens of this call, whose keys and values come as k and v and are stored behind them:
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / group]) v[j, h / group].
//
// Decomposition.  The softmax over a row's keys splits into parts that leave their sum,
// maximum and unnormalised output in fp32, which a last launch joins, the shared keys'
// first, each in key order, so results are the same on every run.
//   Few rows a branch (up to 32: decoded tokens, short drafts).  One launch.  The shared keys
//   are taken once for all branches, whose (token, head of the group) pairs are one long list
//   of rows: tiles of 32 where that is all, else prompt attention's tiles of 128, without a
//   causal border.  A branch's own keys are taken by a wave or a workgroup a range.
//   Many rows a branch (prompts behind a shared one), tiles of 128 rows.  Shared and own keys
//   are one sequence for a tile, and nothing is joined but the tiles of a last partial round.
//   But where many branches are far from filling their tiles (drafts of 9 tokens, say) and the
//   shared keys are many, those go through prompt attention's kernels for all branches.
//
// Position t of branch b lies in row origin[b][t] of the branch cache, the row of the
// ancestor that stored it (without a table of origins, in row b).  So beams are reordered
// by their tables, and no key moves.
//
// Bound by latency and by HBM at few rows: 4 beams over 517 keys 7 us and the join 4; 64
// requests of up to 700 own keys over 4096 38 us for 107 MB, of which about 10 are the two
// launches' chains of latencies; own keys alone stream at 3.1 TB/s there, at
// 4.3-5.3 where they are more (256 branches of 350, 64 of 3000-6000).  By prompt attention's
// matrix products and exponentials at many: 12 prompts over 4096 0.77-0.82 PFLOP/s.
#include <algorithm>
#include <new>

#include "attn_tile.h"
#include "prompt_parts.h"

namespace {

struct BranchParams : PromptParams {   // k, v: the layer's [rows, capacity, kvh, hd]
  const uint16_t *new_k, *new_v;       // of the call's tokens
  int64_t new_k_stride, new_v_stride;
  int64_t row_stride;                  // of the branch cache; k_stride is a position's
  const int32_t* origin;               // [rows, origin_stride], or NULL
  int64_t origin_stride;
  const int32_t* lengths;              // [rows]
  const int4* units;                   // (branch, tile, first token, tokens), or NULL:
  int count, unit_tiles;               // `count` tokens of every branch
  int rows, capacity;
  int whole_units;                     // that take all keys in one part
  int span;                            // keys of a range
  int parts;                           // leaves partials even where one part has all own keys
};

// Stages of a branch's own keys into LDS by NW waves, as Feed has them.  A key's row
// stands alone: the lanes look the origins of the wave's keys up, a stage ahead, and
// pass them to each other.
template <int HD, int NW, int KEYS = kKeys>
struct BranchFeed {
  typedef Shape<HD> S;
  typedef BranchParams Params;
  static constexpr int kLoads = KEYS * S::kRow / (1024 * NW);
  static constexpr int kWaveKeys = kLoads * S::kKeysPerLoad;
  static_assert(kWaveKeys <= 64, "a lane looks up one key");
  const uint16_t *k, *v, *new_k, *new_v;  // the head's first element
  int b, len;              // the branch, and the keys that it held before the call
  int first, left, step;   // the next stage's first key, the last key from there on, and
                           // the keys to the stage behind
  int row;                 // the row of one of the wave's keys in the next stage
  int v_first, v_left, v_row;  // of the stage whose K came last

  static __device__ __forceinline__ int last_of(const BranchParams&, int, int last) {
    return last;
  }
  static __device__ __forceinline__ int wave() {
    return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) & (NW - 1);
  }
  static __device__ __forceinline__ int wave_key() { return wave() * kWaveKeys; }
  static __device__ __forceinline__ int row_of(const BranchParams& p, int b, int len, int key) {
    if (p.origin == nullptr || key >= len) return b;
    return min(max(p.origin[(int64_t)b * p.origin_stride + key], 0), p.rows - 1);
  }
  __device__ __forceinline__ void look_up(const BranchParams& p) {
    const int j = wave_key() + ((int)threadIdx.x & (kWaveKeys - 1));
    row = row_of(p, b, len, first + min(j, left));
  }
  static __device__ __forceinline__ void key_at(const BranchParams& p, const Item& it, int key,
                                                const uint16_t*& kr, const uint16_t*& vr) {
    const int len = it.k_len - it.q_len;
    if (key < len) {
      const int64_t at = (int64_t)row_of(p, it.k0, len, key) * p.row_stride + key * p.k_stride;
      kr = p.k + at;
      vr = p.v + at;
    } else {
      kr = p.new_k + (int64_t)(it.q0 + key - len) * p.new_k_stride;
      vr = p.new_v + (int64_t)(it.q0 + key - len) * p.new_v_stride;
    }
  }
  __device__ __forceinline__ void start(const BranchParams& p, const Item& it, int kvhead,
                                        int begin, int step_) {
    b = it.k0;
    len = it.k_len - it.q_len;
    k = p.k + kvhead * HD;
    v = p.v + kvhead * HD;
    new_k = p.new_k + kvhead * HD + (int64_t)(it.q0 - len) * p.new_k_stride;
    new_v = p.new_v + kvhead * HD + (int64_t)(it.q0 - len) * p.new_v_stride;
    step = step_;
    first = begin;
    left = it.k_len - 1 - begin;
    v_first = v_left = v_row = 0;
    look_up(p);
  }
  // AUX 2: non-temporal
  template <bool V, int AUX>
  __device__ __forceinline__ void load(const BranchParams& p, int first_, int left_, int row_,
                                       uint8_t* tile) const {
    const int lane = threadIdx.x & 63, mine = lane / S::kChunks;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int in = i * S::kKeysPerLoad + mine;  // among the wave's keys
      const int j = wave_key() + in;
      const int key = first_ + min(j, left_);
      const int at = __shfl(row_, in);
      const uint16_t* const held = (V ? v : k) + (int64_t)at * p.row_stride + key * p.k_stride;
      const uint16_t* const fresh_ =
          V ? new_v + (int64_t)key * p.new_v_stride : new_k + (int64_t)key * p.new_k_stride;
      const int chunk = (lane & (S::kChunks - 1)) ^ (V ? S::swz_v(j) : S::swz_k(j));
      __builtin_amdgcn_global_load_lds((glb_void*)((key < len ? held : fresh_) + chunk * 8),
                                       (lds_void*)(tile + (wave() * kLoads + i) * 1024), 16, 0,
                                       AUX);
    }
  }
  __device__ __forceinline__ void load_k(const BranchParams& p, uint8_t* tile) {
    load_any<false>(p, first, left, row, tile);
    v_first = first;
    v_left = left;
    v_row = row;
    first += step;
    left -= step;
    look_up(p);
  }
  __device__ __forceinline__ void load_v(const BranchParams& p, uint8_t* tile) {
    load_any<true>(p, v_first, v_left, v_row, tile);
  }
  // What a branch holds alone is read once, and goes past the caches: 256 branches of 350 keys
  // 81 us, else 86; 16 of up to 4000 48, 53.  (What beams share is read by several.)
  template <bool V>
  __device__ __forceinline__ void load_any(const BranchParams& p, int first_, int left_, int row_,
                                           uint8_t* tile) const {
    if (p.origin == nullptr)
      load<V, 2>(p, first_, left_, row_, tile);
    else
      load<V, 0>(p, first_, left_, row_, tile);
  }
};

// A part of a branch: rows of a tile against a range of its keys.
struct Work {
  Item it;
  int kvhead;
  int len;     // keys that the branch held
  int lo, hi;  // the new keys of the range, which are stored with it
};
// The branch, tile and tokens of a unit.
__device__ __forceinline__ Item unit_of(const BranchParams& p, int unit) {
  Item it = {};
  if (p.units != nullptr) {
    const int4 u = p.units[unit];
    it.k0 = __builtin_amdgcn_readfirstlane(u.x);
    it.tile = __builtin_amdgcn_readfirstlane(u.y);
    it.q0 = __builtin_amdgcn_readfirstlane(u.z);
    it.q_len = __builtin_amdgcn_readfirstlane(u.w);
  } else {
    it.k0 = unit / p.unit_tiles;
    it.tile = unit - it.k0 * p.unit_tiles;
    it.q0 = it.k0 * p.count;
    it.q_len = p.count;
  }
  return it;
}
// Part `at` of all.  Ranges are whole stages, and go by the branch's own length, so that
// they hold all its keys even where it is longer than the host took it for.  Before the
// branch's keys lie `base` others.
template <int STAGE>
__device__ __forceinline__ Work work_of(const BranchParams& p, int kvhead, int at, int tile_rows,
                                        int base = 0) {
  Work w;
  w.kvhead = kvhead;
  // the first units take all keys, the others' are split
  const bool split = at >= p.whole_units;
  const int rest = at - p.whole_units, chunks = split ? p.chunks : 1;
  const int chunk = split ? rest % p.chunks : 0;
  const int unit = split ? p.whole_units + rest / p.chunks : at;
  Item& it = w.it;
  it = unit_of(p, unit);
  w.len = min(max(__builtin_amdgcn_readfirstlane(p.lengths[it.k0]), 0), p.capacity);
  it.k_len = base + w.len + it.q_len;
  const int per = (it.k_len + chunks - 1) / chunks;
  const int span = max((per + STAGE - 1) / STAGE * STAGE, split ? p.span : 0);
  const int last_token = min(it.q_len - 1, (it.tile * tile_rows + tile_rows - 1) / p.group);
  it.begin = (int)min((int64_t)chunk * span, (int64_t)it.k_len);
  const int end = min(it.begin + span, it.k_len);
  it.end = min(end, base + w.len + last_token + 1);
  it.slot = p.parts && split ? rest : -1;
  w.hi = it.tile == 0 ? end - base : 0;
  w.lo = max(it.begin - base, w.len);
  return w;
}

// The new keys and values lo .. hi - 1 of the head into the branch's own row, by THREADS
// threads of which this is the `me`-th.
template <int HD, int THREADS>
__device__ __forceinline__ void store_new(const BranchParams& p, const Work& w, int me) {
  constexpr int kPieces = HD / 8;
  const int hi = min(w.hi, p.capacity);
  for (int x = me; x < (hi - w.lo) * kPieces; x += THREADS) {
    const int key = w.lo + x / kPieces, e = w.kvhead * HD + x % kPieces * 8;
    const int64_t from = w.it.q0 + key - w.len;
    const int64_t to = (int64_t)w.it.k0 * p.row_stride + key * p.k_stride + e;
    *reinterpret_cast<u32x4_t*>(const_cast<uint16_t*>(p.k) + to) =
        *reinterpret_cast<const u32x4_t*>(p.new_k + from * p.new_k_stride + e);
    *reinterpret_cast<u32x4_t*>(const_cast<uint16_t*>(p.v) + to) =
        *reinterpret_cast<const u32x4_t*>(p.new_v + from * p.new_v_stride + e);
  }
}

// Up to 32 rows against a range of keys, 32 keys a stage, the four waves in turn, each with
// its own part of LDS and no barrier between them.  Stages of 32 keys leave room for two
// workgroups a CU: most ranges are a few stages long, and one's first loads and last stores
// run under the other's products.
constexpr int kLean = 32;
template <int HD>
struct LeanShared {
  uint8_t tiles[4][2 * kLean * Shape<HD>::kRow];  // of each wave, K and V
  float stat[4][32][2];
};

// What comes behind is not begun before the fragments are in their registers.
template <int N>
__device__ __forceinline__ void refill_after(u32x4_t (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4) | (0 << 8));  // LDS reads
  __builtin_amdgcn_sched_barrier(0);
}

// S^T = K Q^T of the stage at kt_, whose place is free for `refill` once its fragments are
// read.
template <int DT, int HD, class REFILL>
__device__ __forceinline__ void lean_scores(const uint8_t* kt_, Rows<HD>& r, REFILL&& refill) {
  const int at = k_offset<HD>();
  u32x4_t f[HD / 16];
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks)
    f[ks] = *reinterpret_cast<const u32x4_t*>(kt_ + (at ^ (32 * ks)));
  refill_after(f);
  refill();
  f32x16_t sc = {};
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) sc = mfma32<DT>(f[ks], r.q[ks], sc);
  r.sc[0] = sc;
}
// O^T += V^T P^T of the stage at vt.
template <int DT, int HD, class REFILL>
__device__ __forceinline__ void lean_outputs(const uint8_t* vt, Rows<HD>& r, REFILL&& refill) {
  int lo, hi;
  v_offsets<HD>(lo, hi);
  u32x4_t vf[kLean / 16][HD / 32];
#pragma unroll
  for (int s = 0; s < kLean / 16; ++s) read_v<HD>(vt, fresh(lo), fresh(hi), s, vf[s]);
#pragma unroll
  for (int s = 0; s < kLean / 16; ++s) refill_after(vf[s]);
  refill();
#pragma unroll
  for (int s = 0; s < kLean / 16; ++s)
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht) r.o[ht] = mfma32<DT>(vf[s][ht], r.pw[s], r.o[ht]);
}

template <int DT, int HD, class FEED>
__device__ __forceinline__ void lean_body(const typename FEED::Params& p, const Item& it,
                                          int kvhead, LeanShared<HD>& lds) {
  constexpr int kLoads = FEED::kLoads;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int first = it.tile * 32, rows = min(it.q_len * p.group - first, 32);
  const int n = it.end > it.begin ? (it.end - it.begin + kLean - 1) / kLean : 0;
  uint8_t* const kt = lds.tiles[wave];
  uint8_t* const vt = kt + kLean * Shape<HD>::kRow;
  FEED feed;
  if (wave < n) {
    feed.start(p, it, kvhead, it.begin + wave * kLean, 4 * kLean);
    feed.load_k(p, kt);
    feed.load_v(p, vt);
  }
  Rows<HD> r;
  const int full = begin_rows<HD>(p, it, kvhead, first, r).full;
  for (int s = wave; s < n; s += 4) {
    const int kb = it.begin + s * kLean;
    const bool more = s + 4 < n;
    if (s == wave)
      wait_vm<0>();  // K and V, and the query rows
    else
      wait_vm<kLoads>();  // K: V is behind it
    lean_scores<DT, HD>(kt, r, [&]() TM_INLINE {
      if (more) feed.load_k(p, kt);
    });
    weigh_stage<DT, HD, FEED, 1>(p, kb, full, r);
    if (more)
      wait_vm<kLoads>();
    else
      wait_vm<0>();
    lean_outputs<DT, HD>(vt, r, [&]() TM_INLINE {
      if (more) feed.load_v(p, vt);
    });
  }
  retake<DT, HD, FEED, kLean>(p, it, kvhead, wave, 4, n, r);
  const float l = r.l + __shfl_xor(r.l, 32);
  // each wave's O [32][HD] where its K and V were
  if (c32 < rows) {
    float* const mine = reinterpret_cast<float*>(kt) + c32 * HD + 4 * half;
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<f32x4_t*>(mine + 32 * ht + 8 * x) =
            f32x4_t{r.o[ht][4 * x], r.o[ht][4 * x + 1], r.o[ht][4 * x + 2], r.o[ht][4 * x + 3]};
    if (half == 0) {
      lds.stat[wave][c32][0] = r.m;
      lds.stat[wave][c32][1] = l;
    }
  }
  __syncthreads();
  constexpr int kLanes = HD / 4;  // of a row, four elements each
  for (int row = tid / kLanes; row < rows; row += kThreads / kLanes) {
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, lds.stat[w][row][0]);
    const float ref = m == -INFINITY ? 0.0f : m;
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = __builtin_amdgcn_exp2f(lds.stat[w][row][0] - ref);
      sum += lds.stat[w][row][1] * a;
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(
          reinterpret_cast<const float*>(lds.tiles[w]) + row * HD + 4 * (tid % kLanes));
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += x[e] * a;
    }
    if (it.slot < 0) {
      store_row<DT>(p, it.q0, first + row, kvhead, HD, 4 * (tid % kLanes), o, sum);
    } else {
      const int64_t slot = ((int64_t)it.slot * p.kvh + kvhead) * p.part_rows + row;
      *reinterpret_cast<f32x4_t*>(p.part + slot * HD + 4 * (tid % kLanes)) = o;
      if (tid % kLanes == 0) {
        p.stats[slot * 2] = m;
        p.stats[slot * 2 + 1] = sum;
      }
    }
  }
}

// The sum of a part without keys, which has no output: added it changes nothing, and by its
// sign the join tells it from the sum of keys without weight.
constexpr float kNoOutput = -0.0f;

// A branch's own keys, up to 32 rows against one range by one wave: no barrier, and no
// join within the workgroup.  What such a part costs most is its chain of latencies (the
// length, the first keys, the last stores), so all of a step's are to run at once.
template <int DT, int HD>
__device__ __forceinline__ void wave_body(const BranchParams& p, const Work& w, uint8_t* kt) {
  typedef BranchFeed<HD, 1, kLean> Own;
  const Item& it = w.it;
  const int lane = threadIdx.x & 63, half = lane >> 5, c32 = lane & 31;
  const int n = it.end > it.begin ? (it.end - it.begin + kLean - 1) / kLean : 0;
  const int rows = min(it.q_len * p.group, 32);
  uint8_t* const vt = kt + kLean * Shape<HD>::kRow;
  if (n == 0) {  // no output is written, and the sum says so
    if (lane < rows && it.slot >= 0) {
      float* const st =
          p.stats + (((int64_t)it.slot * p.kvh + w.kvhead) * p.part_rows + lane) * 2;
      st[0] = -INFINITY;
      st[1] = kNoOutput;
    }
    return;
  }
  Own feed;
  feed.start(p, it, w.kvhead, it.begin, kLean);
  feed.load_k(p, kt);
  feed.load_v(p, vt);
  Rows<HD> r;
  const int full = begin_rows<HD>(p, it, w.kvhead, 0, r).full;
  for (int s = 0; s < n; ++s) {
    const int kb = it.begin + s * kLean;
    const bool more = s + 1 < n;
    if (s == 0)
      wait_vm<0>();  // K and V, and the query rows
    else
      wait_vm<Own::kLoads>();  // K: V is behind it
    lean_scores<DT, HD>(kt, r, [&]() TM_INLINE {
      if (more) feed.load_k(p, kt);
    });
    weigh_stage<DT, HD, Own, 1>(p, kb, full, r);
    if (more)
      wait_vm<Own::kLoads>();
    else
      wait_vm<0>();
    lean_outputs<DT, HD>(vt, r, [&]() TM_INLINE {
      if (more) feed.load_v(p, vt);
    });
  }
  retake<DT, HD, Own, kLean>(p, it, w.kvhead, 0, 1, n, r);
  const float l = r.l + __shfl_xor(r.l, 32);
  if (c32 >= rows) return;
  if (it.slot < 0) {
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        store_row<DT>(p, it.q0, c32, w.kvhead, HD, 32 * ht + 8 * x + 4 * half,
                      f32x4_t{r.o[ht][4 * x], r.o[ht][4 * x + 1], r.o[ht][4 * x + 2],
                              r.o[ht][4 * x + 3]},
                      l);
    return;
  }
  const int64_t slot = ((int64_t)it.slot * p.kvh + w.kvhead) * p.part_rows + c32;
#pragma unroll
  for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<f32x4_t*>(p.part + slot * HD + 32 * ht + 8 * x + 4 * half) = f32x4_t{
          r.o[ht][4 * x], r.o[ht][4 * x + 1], r.o[ht][4 * x + 2], r.o[ht][4 * x + 3]};
  if (half == 0) {
    p.stats[slot * 2] = r.m;
    p.stats[slot * 2 + 1] = l;
  }
}

// Shared keys and the branches' own, where no branch adds more than 32 rows, in one launch:
// the shared ones' workgroups first, tiles of 32 rows (where that is all) or of 128; then
// the branches' own, a workgroup or (WAVES) a wave a part.  The products over the shared keys
// run beside the reading of the others.
enum Shared { kNone, kLeanTile, kShortTile };
template <int DT, int HD, int SHARED, bool WAVES>
__global__ void __launch_bounds__(kThreads, 2) tm_branch_kernel(PromptParams s, BranchParams p,
                                                               int shared_blocks, int own_parts) {
  __shared__ __attribute__((aligned(1024))) LeanShared<HD> lds;
  static_assert(sizeof(lds.tiles) == 4 * Shape<HD>::kTile, "two stages of 64 keys");
  const int block = blockIdx.x;
  if (SHARED != kNone && block < shared_blocks) {
    // (KV heads innermost: with 8 of them a head's workgroups, which share its keys, run
    // on one XCD)
    const int kvhead = block % p.kvh, at = block / p.kvh;
    if constexpr (SHARED == kLeanTile)
      lean_body<DT, HD, Feed<HD, true, 1, kLean>>(s, item_of(s, at, 32), kvhead, lds);
    else
      short_body<DT, HD, Feed<HD, true, 4>>(s, item_of(s, at, 128), kvhead, lds.tiles[0],
                                            lds.tiles[1], lds.tiles[2], lds.tiles[3]);
    return;
  }
  if constexpr (!WAVES) {
    const int at = block - shared_blocks;
    const Work w = work_of<kLean>(p, at % p.kvh, at / p.kvh, 32);
    store_new<HD, kThreads>(p, w, threadIdx.x);
    lean_body<DT, HD, BranchFeed<HD, 1, kLean>>(p, w.it, w.kvhead, lds);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // (the waves of a workgroup take neighbouring heads of the same keys, which lie side by
  // side)
  const int id = (block - shared_blocks) * 4 + wave, at = id / p.kvh;
  if (at >= own_parts) return;
  const Work w = work_of<kLean>(p, id - at * p.kvh, at, 32);
  store_new<HD, 64>(p, w, threadIdx.x & 63);
  wave_body<DT, HD>(p, w, lds.tiles[wave]);
}

// Its own keys, tiles of 128 rows.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 2) tm_branch_short_kernel(BranchParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v1[S::kTile];
  const Work w = work_of<kKeys>(p, (int)blockIdx.x % p.kvh, (int)blockIdx.x / p.kvh, 128);
  store_new<HD, kThreads>(p, w, threadIdx.x);
  short_body<DT, HD, BranchFeed<HD, 4>>(p, w.it, w.kvhead, s_k0, s_v0, s_k1, s_v1);
}

// The shared keys and behind them the branch's own as one sequence, for tiles that one
// branch fills: nothing is left to share between branches, and nothing to join.  The own keys
// begin with a stage of theirs, `base`, the shared ones in whole stages.
struct ChainParams : BranchParams {
  PromptParams shared;
  int shared_keys, base;
};
template <int HD, int NW>
struct ChainFeed {
  typedef ChainParams Params;
  typedef Feed<HD, true, NW> Pages;
  typedef BranchFeed<HD, NW> Own;
  static constexpr int kLoads = Pages::kLoads, kGroup = Pages::kGroup;
  static_assert(kLoads == Own::kLoads, "the waits count either's loads");
  Pages pages;
  Own own;
  int at, step;  // the next stage
  bool v_own;    // of the stage whose K came last

  static __device__ __forceinline__ int last_of(const ChainParams& p, int kb, int last) {
    return kb < p.base ? min(last, p.shared_keys - 1) : last;
  }
  static __device__ __forceinline__ Item own_of(const ChainParams& p, const Item& it) {
    Item o = it;
    o.k_len -= p.base;
    return o;
  }
  static __device__ __forceinline__ void key_at(const ChainParams& p, const Item& it, int key,
                                                const uint16_t*& kr, const uint16_t*& vr) {
    if (key < p.base)
      Pages::key_at(p.shared, it, min(key, p.shared_keys - 1), kr, vr);
    else
      Own::key_at(p, own_of(p, it), key - p.base, kr, vr);
  }
  __device__ __forceinline__ void start(const ChainParams& p, const Item& it, int kvhead,
                                        int begin, int step_) {
    at = begin;
    step = step_;
    v_own = false;
    if (begin < p.base) {
      Item s = it;
      s.k_len = p.shared_keys;
      pages.start(p.shared, s, kvhead, begin, step);
    }
    const int first = begin < p.base ? begin + (p.base - begin + step - 1) / step * step : begin;
    own.start(p, own_of(p, it), kvhead, first - p.base, step);
  }
  __device__ __forceinline__ void load_k(const ChainParams& p, uint8_t* tile) {
    v_own = at >= p.base;
    if (v_own)
      own.load_k(p, tile);
    else
      pages.load_k(p.shared, tile);
    at += step;
  }
  __device__ __forceinline__ void load_v(const ChainParams& p, uint8_t* tile) {
    if (v_own)
      own.load_v(p, tile);
    else
      pages.load_v(p.shared, tile);
  }
};
template <int DT, int HD>
__global__ void __launch_bounds__(512, 2) tm_branch_chain_pair_kernel(ChainParams p) {
  __shared__ PairShared<HD> lds;
  const Work w =
      work_of<kKeys>(p, (int)blockIdx.x % p.kvh, (int)blockIdx.x / p.kvh, 128, p.base);
  store_new<HD, 512>(p, w, threadIdx.x);
  pair_body<DT, HD, ChainFeed<HD, 4>>(p, w.it, w.kvhead, lds);
}
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 2) tm_branch_chain_short_kernel(ChainParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t tiles[4][Shape<HD>::kTile];
  const Work w =
      work_of<kKeys>(p, (int)blockIdx.x % p.kvh, (int)blockIdx.x / p.kvh, 128, p.base);
  store_new<HD, kThreads>(p, w, threadIdx.x);
  short_body<DT, HD, ChainFeed<HD, 4>>(p, w.it, w.kvhead, tiles[0], tiles[1], tiles[2], tiles[3]);
}

// Branches whose call has ended hold `count` more keys, or counts[b], which lie in their own
// rows.  A workgroup a branch.
__global__ void __launch_bounds__(64) tm_branch_advance_kernel(int32_t* lengths,
                                                               const int32_t* counts, int count,
                                                               int capacity, int32_t* origin,
                                                               int64_t origin_stride) {
  const int b = blockIdx.x;
  const int len = min(max(__builtin_amdgcn_readfirstlane(lengths[b]), 0), capacity);
  const int n = counts != nullptr ? __builtin_amdgcn_readfirstlane(counts[b]) : count;
  const int end = (int)min((int64_t)len + max(n, 0), (int64_t)capacity);
  if (origin != nullptr)
    for (int t = len + (int)threadIdx.x; t < end; t += 64) origin[b * origin_stride + t] = b;
  if (threadIdx.x == 0) lengths[b] = end;
}

// Parts of one kind: `chunks` of every tile, a row's elements together or, `tiled`, 32 rows as
// end_rows lays them.
struct Parts {
  const float* part;
  const float* stats;
  int chunks, tile_rows, part_rows;
  int tiled;
};
struct BranchJoin {
  Parts shared, own;
  const int4* tokens;  // (branch, place in it, its first unit), or NULL:
  int count, unit_tiles;
  int T, Hq, kvh, group;
  uint16_t* out;
  int64_t out_stride;
};
constexpr int kMaxParts = 512;  // of each kind

// Where a row's parts lie: chunk c's statistics at stats + c * step * 2, its output at
// o + c * step * HD.
struct RowParts {
  const float *stats, *o;
  int64_t step;
};
// elements e .. e + 3 of row `row` of a KV head; tile0: its rows' first tile
template <int HD>
__device__ __forceinline__ RowParts parts_of(const Parts& s, int kvh, int kvhead, int tile0,
                                             int row, int e) {
  const int tile = row / s.tile_rows, in = row - tile * s.tile_rows;
  const int64_t slot =
      ((int64_t)(tile0 + tile) * s.chunks * kvh + kvhead) * s.part_rows + in;
  RowParts r;
  r.step = (int64_t)kvh * s.part_rows;
  r.stats = s.stats + slot * 2;
  r.o = s.tiled ? s.part + (slot - (in & 31)) * HD + (e >> 3) * 256 + ((e >> 2) & 1) * 128 +
                      (in & 31) * 4
                : s.part + slot * HD + e;
  return r;
}

// Joins 32 rows' 32 columns of a branch's tile, a wave each, shared parts first and each in
// order: lane l has row l % 32 and the columns that the partials' layout gives it.  (A wave a
// row, as below, takes 16 bytes of each of a part's lines: 8 branches of 100 tokens, split in
// two, 47 us in all, so 32.)
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads) tm_branch_join_tiles_kernel(BranchParams p,
                                                                        Parts shared, Parts own,
                                                                        int waves) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  int id = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (id >= waves) return;
  const int ht = id % (HD / 32);
  id /= HD / 32;
  const int first = id % 4 * 32 + (lane & 31);
  id /= 4;
  const int kvhead = id % p.kvh, at = id / p.kvh, unit = p.whole_units + at;
  const Item it = unit_of(p, unit);
  const int row = it.tile * 128 + first;
  if (row >= it.q_len * p.group) return;
  const int e = 32 * ht + 4 * half;
  RowParts r[2] = {{nullptr, nullptr, 0}, parts_of<HD>(own, p.kvh, kvhead, at, first, e)};
  if (shared.chunks > 0)
    r[0] = parts_of<HD>(shared, p.kvh, kvhead, 0, it.q0 * p.group + row, e);
  const int count[2] = {shared.chunks, own.chunks};
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll 4
    for (int c = 0; c < count[k]; ++c) m = fmaxf(m, r[k].stats[c * r[k].step * 2]);
  const float ref = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
  f32x4_t o[4] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll 2
    for (int c = 0; c < count[k]; ++c) {
      const float2 st = *reinterpret_cast<const float2*>(r[k].stats + c * r[k].step * 2);
      const float a = __builtin_amdgcn_exp2f(st.x - ref);
      sum = fmaf(st.y, a, sum);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(r[k].o + c * r[k].step * HD + 256 * x);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[x][i] = fmaf(v[i], a, o[x][i]);
      }
    }
#pragma unroll
  for (int x = 0; x < 4; ++x)
    store_row<DT>(p, it.q0, row, kvhead, HD, e + 8 * x, o[x], sum);
}

// Of few rows a branch: a wave joins the parts of one row: the maximum and the sum over the
// parts, a lane per part, then the weighted outputs in their order, four elements a lane and
// the lanes' groups a part each.  The first kAhead parts of a group are asked for before
// anything is known.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads) tm_branch_join_kernel(BranchJoin p) {
  __shared__ float s_a[4][2 * kMaxParts];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  if (unit >= (int64_t)p.T * p.Hq) return;
  const int t = (int)(unit / p.Hq), head = (int)(unit - (int64_t)t * p.Hq);
  const int kvhead = head / p.group, g = head - kvhead * p.group;
  constexpr int kLanes = HD / 4, kGroups = 64 / kLanes, kAhead = 8;
  const int e = 4 * (lane % kLanes), group = lane / kLanes;
  int place, unit0;
  if (p.tokens != nullptr) {
    const int4 x = p.tokens[t];
    place = x.y;
    unit0 = x.z;
  } else {
    place = t % p.count;
    unit0 = t / p.count * p.unit_tiles;
  }
  // part c: the shared ones first
  const RowParts r0 = parts_of<HD>(p.shared, p.kvh, kvhead, 0, t * p.group + g, e);
  const RowParts r1 = parts_of<HD>(p.own, p.kvh, kvhead, unit0, place * p.group + g, e);
  const int n0 = p.shared.chunks, n = n0 + p.own.chunks;
  auto out_of = [&](int c) {
    return c < n0 ? r0.o + c * r0.step * HD : r1.o + (c - n0) * r1.step * HD;
  };
  auto stat_of = [&](int c) {
    return *reinterpret_cast<const float2*>(c < n0 ? r0.stats + c * r0.step * 2
                                                   : r1.stats + (c - n0) * r1.step * 2);
  };
  // the part's factor; -1 of one that has no output
  auto factor_of = [&](const float2& st, float a) {
    return __float_as_uint(st.y) == __float_as_uint(kNoOutput) ? -1.0f : a;
  };
  f32x4_t first[kAhead] = {};
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (i * kGroups < n)
      first[i] = *reinterpret_cast<const f32x4_t*>(out_of(min(group + i * kGroups, n - 1)));
  float m = -INFINITY, sum = 0.0f;
  if (n <= 64) {
    const float2 st = lane < n ? stat_of(lane) : float2{-INFINITY, 0.0f};
    m = st.x;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float a = __builtin_amdgcn_exp2f(st.x - (m == -INFINITY ? 0.0f : m));
    sum = st.y * a;
    s_a[wave][lane] = factor_of(st, a);
  } else {
    for (int c = lane; c < n; c += 64) m = fmaxf(m, stat_of(c).x);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float ref = m == -INFINITY ? 0.0f : m;
    for (int c = lane; c < n; c += 64) {
      const float2 st = stat_of(c);
      const float a = __builtin_amdgcn_exp2f(st.x - ref);
      sum = fmaf(st.y, a, sum);
      s_a[wave][c] = factor_of(st, a);
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](int c, const f32x4_t& x) {
    const float a = s_a[wave][c];
    // (a factor of 0 makes NaN of an infinity, as any product of the sum does)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = a < 0.0f ? o[i] : fmaf(x[i], a, o[i]);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (group + i * kGroups < n) add(group + i * kGroups, first[i]);
#pragma unroll 8
  for (int c = group + kAhead * kGroups; c < n; c += kGroups)
    add(c, *reinterpret_cast<const f32x4_t*>(out_of(c)));
#pragma unroll
  for (int d = 32; d >= kLanes; d >>= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], d);
  if (lane >= kLanes) return;
  const float inv = sum > 0.0f ? 1.0f / sum : sum;  // 0 where nothing was seen; NaN stays
  u32x2_t w;
  w.x = tm_pack2<DT>(o[0] * inv, o[1] * inv);
  w.y = tm_pack2<DT>(o[2] * inv, o[3] * inv);
  *reinterpret_cast<u32x2_t*>(p.out + (int64_t)t * p.out_stride + (int64_t)head * HD + e) = w;
}

// ------------------------------------------------------------------- host --

// How the work is split, measured at 32 heads over 8 of 128 in bf16, in us of a pass (graph
// replays on changing inputs), one token a branch unless said:
//   shared keys in as many workgroups as kSharedBlocks: 64 requests over 4096 with 64, 128
//   and 256 of them 38, 40, 44; 48 chains of five tokens over 2003 29, 22, 23; 256 requests
//   over 4096 114, 105, 119;
//   own keys by workgroups (LEAN) or waves: 8 branches of up to 400 keys 14.3, 15.9; 16 16.6,
//   15.9; 32 21.8, 18.7; 64 of up to 700 42, 40; 128 of up to 60 27, 21;
//   at most kOwnWaves parts by waves: 64 of up to 700 with 8, 12 and 16 a CU 44, 40, 44; 256
//   of them 102, 103, 112; 16 of up to 4000 52, 47, 50;
//   by workgroups, of which each has more keys to itself, where a branch may hold more than
//   kLongKeys: 64 branches of 3000-6000 keys 234, by waves 248; 12 of 7000-14000 101, 110; 16 of
//   2000-4000 by workgroups 51, by waves 48.
constexpr int64_t kSharedBlocks = 128;
constexpr int64_t kOwnWaves = 12 * kCUs;
constexpr int64_t kLeanUnits = 64;     // (branch, KV head) pairs up to which a part is a workgroup
constexpr int64_t kWaveKeys = 64;      // of a wave's part, or more
constexpr int64_t kLongKeys = 4096;
constexpr int64_t kMaxStride = 1 << 24;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int check_heads(int64_t Hq, int64_t kvh, int64_t hd) {
  if (kvh < 1 || Hq < kvh || Hq % kvh != 0 || Hq > 1024 || (hd != 64 && hd != 128))
    return TM_ERR_SHAPE;
  return TM_OK;
}

// Rows of a tile of a branch: 32 where no branch has more, else 128.
int64_t own_tile_rows(int64_t max_count, int64_t group) {
  return max_count * group <= 32 ? 32 : 128;
}

struct BranchPlan {
  PrefixPlan prefix;               // the shared keys
  Shared shared;
  bool few;                        // one launch for both kinds of keys
  bool waves;                      // a wave a part of own keys
  bool chain, pair;                // both as one sequence; with eight waves
  int64_t units, chunks, span;     // of the branches' own keys
  int64_t whole_units;             // the first, which take them in one part
  int64_t own_rows;                // rows of one of their partials
  int64_t prefix_slots, own_slots; // (of one KV head)
  int64_t prefix_floats, floats;   // of the workspace
};

// T tokens, at most max_count of one branch, in `units` tiles of branches; S shared keys, at
// most `longest` held by a branch.
int plan_branches(int64_t T, int64_t units, int64_t max_count, int64_t S, int64_t longest,
                  int64_t Hq, int64_t kvh, int64_t hd, BranchPlan* o) {
  const int64_t group = Hq / kvh;
  if (units < 0 || max_count < 0 || max_count > T || longest < 0 || longest > TM_MAX_PROMPT_KEYS ||
      S < 0 || S > TM_MAX_PROMPT_KEYS || T < 0 || T * group > INT32_MAX - 1024)
    return TM_ERR_SHAPE;
  *o = {};
  const int64_t rows = own_tile_rows(max_count, group);
  o->few = rows == 32;
  o->units = units;
  if (S > 0 && o->few) {
    const int64_t all = T * group;
    o->shared = all <= 32 ? kLeanTile : kShortTile;
    PrefixPlan& f = o->prefix;
    f.kind = o->shared == kLeanTile ? 0 : 1;
    f.tile_rows = o->shared == kLeanTile ? 32 : 128;
    f.tiles = ceil_div(all, f.tile_rows);
    f.part_rows = o->shared == kLeanTile ? all : 128;
    const int64_t step = o->shared == kLeanTile ? 4 * kLean : kKeys;
    const int64_t want = std::max<int64_t>(1, kSharedBlocks / std::max<int64_t>(f.tiles * kvh, 1));
    const int64_t chunks = std::max<int64_t>(
        1, std::min(std::min<int64_t>(want, kMaxParts),
                    ceil_div(S, o->shared == kLeanTile ? 4 * kLean : 4 * kKeys)));
    f.chunk_len = std::max(step, ceil_div(ceil_div(S, chunks), step) * step);
    f.chunks = ceil_div(S, f.chunk_len);
  }
  // Shared and own keys as one sequence, or apart and joined (the same heads measured; others take
  // the same rule).  As one, the rows that a
  // branch's tiles are short of go against the shared keys, too; apart, two launches more and
  // every row's parts are stored and read.  Measured, in us, as one and apart: 32 branches of 9
  // tokens (36 rows of 128) behind 500 keys 28, 42, 1000 36, 44, 2000 53, 50; of 16 tokens
  // behind 4000 88, 72, of 20 90, 96; 128 of 9 behind 1000 102, 105, 2000 161, 133; 8 of 16
  // behind 4000 37, 42; 12 prompts of 1-333 tokens over 4096 177, 262.
  const int64_t base = ceil_div(S, kKeys) * kKeys, all_rows = T * group;
  o->chain = !o->few && (units * 128 - all_rows) * S <= all_rows * 1600 + (1 << 25) / kvh;
  if (S > 0 && !o->few && !o->chain) {
    const int rc = tm_prefix_plan(T, S, Hq, kvh, &o->prefix);
    if (rc) return rc;
  }
  const int64_t keys = longest + max_count + (o->chain ? base : 0);
  // Eight waves a tile where the tiles leave CUs idle: 8 branches of 100 tokens over 400 keys
  // 26 us, 39 with four and the keys split, joined; but 8 of 250, 512 tiles, over 400 52, 41.
  o->pair = o->chain && units * kvh <= kCUs && keys >= 4 * kKeys;
  o->waves = o->few && units * kvh > kLeanUnits && keys <= kLongKeys;
  const int64_t slots = o->waves ? kOwnWaves : o->pair ? kCUs : 2 * kCUs;
  // As one, as many tiles as fill the chip's slots some whole times stay whole, and those left are
  // split: of 600 tiles on 512 slots the last 88 (12 prompts over 4096 179 us, all whole 234).
  o->whole_units = o->chain ? units * kvh / slots * slots / kvh : 0;
  const int64_t want = std::min<int64_t>(
      slots / std::max<int64_t>((units - o->whole_units) * kvh, 1), kMaxParts);
  const int64_t least = o->waves ? kWaveKeys : 4 * kKeys;
  const int64_t stage = o->few ? kLean : o->pair ? 2 * kKeys : kKeys;
  o->chunks = std::max<int64_t>(1, std::min(want, ceil_div(keys, least)));
  if (o->chain && o->chunks == 1) o->whole_units = units;
  o->span = ceil_div(ceil_div(keys, o->chunks), stage) * stage;
  o->own_rows = o->few ? std::min<int64_t>(32, max_count * group) : rows;
  o->prefix_slots = S > 0 && !o->chain ? o->prefix.tiles * o->prefix.chunks : 0;
  const bool joined = o->prefix_slots > 0 || o->chunks > 1;
  const int64_t split = units - o->whole_units;
  o->own_slots = joined ? split * o->chunks : 0;
  if (o->own_slots > INT32_MAX ||
      (o->prefix_slots + o->whole_units + split * o->chunks) * kvh > UINT32_MAX / 512 ||
      T * Hq > UINT32_MAX / 64)
    return TM_ERR_SHAPE;
  o->prefix_floats = kvh * (hd + 2) * o->prefix_slots * o->prefix.part_rows;
  o->prefix_floats = ceil_div(o->prefix_floats, 4) * 4;  // (16-byte stores behind them)
  o->floats = o->prefix_floats + kvh * (hd + 2) * o->own_slots * o->own_rows;
  return TM_OK;
}

bool vec_ok(const void* p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride % 8 == 0; }

template <int DT, int HD, bool WAVES>
void launch_few(const PromptParams& s, const BranchParams& p, const BranchPlan& o, int64_t shared,
                int64_t own, int64_t parts, hipStream_t st) {
  const dim3 grid((unsigned)(shared + own)), block(kThreads);
  if (o.shared == kNone)
    hipLaunchKernelGGL((tm_branch_kernel<DT, HD, kNone, WAVES>), grid, block, 0, st, s, p,
                       (int)shared, (int)parts);
  else if (o.shared == kLeanTile)
    hipLaunchKernelGGL((tm_branch_kernel<DT, HD, kLeanTile, WAVES>), grid, block, 0, st, s, p,
                       (int)shared, (int)parts);
  else
    hipLaunchKernelGGL((tm_branch_kernel<DT, HD, kShortTile, WAVES>), grid, block, 0, st, s, p,
                       (int)shared, (int)parts);
}
template <int DT, int HD>
void launch_own(const PromptParams& s, const BranchParams& p, const BranchPlan& o,
                hipStream_t st) {
  const int64_t parts = o.whole_units + (o.units - o.whole_units) * o.chunks;
  const int64_t shared = o.prefix_slots * p.kvh;
  const int64_t own = o.waves ? ceil_div(parts * p.kvh, 4) : parts * p.kvh;
  const dim3 block(kThreads);
  if (o.chain) {
    ChainParams c;
    static_cast<BranchParams&>(c) = p;
    c.shared = s;
    c.shared_keys = s.k_len;
    c.base = (int)(ceil_div(s.k_len, kKeys) * kKeys);
    if (o.pair)
      hipLaunchKernelGGL((tm_branch_chain_pair_kernel<DT, HD>), dim3((unsigned)own), dim3(512), 0,
                         st, c);
    else
      hipLaunchKernelGGL((tm_branch_chain_short_kernel<DT, HD>), dim3((unsigned)own), block, 0, st,
                         c);
  } else if (!o.few)
    hipLaunchKernelGGL((tm_branch_short_kernel<DT, HD>), dim3((unsigned)own), block, 0, st, p);
  else if (o.waves)
    launch_few<DT, HD, true>(s, p, o, shared, own, parts, st);
  else
    launch_few<DT, HD, false>(s, p, o, shared, own, parts, st);
}
template <int DT, int HD>
void launch_join(const BranchParams& p, const BranchJoin& j, const BranchPlan& o, hipStream_t st) {
  if (o.few) {
    hipLaunchKernelGGL((tm_branch_join_kernel<DT, HD>),
                       dim3((unsigned)ceil_div((int64_t)j.T * j.Hq, 4)), dim3(kThreads), 0, st, j);
  } else {
    const int64_t waves = (o.units - o.whole_units) * p.kvh * 4 * (HD / 32);
    hipLaunchKernelGGL((tm_branch_join_tiles_kernel<DT, HD>), dim3((unsigned)ceil_div(waves, 4)),
                       dim3(kThreads), 0, st, p, j.shared, j.own, (int)waves);
  }
}

}  // namespace

extern "C" int tm_branch_plan(const int64_t* counts, int64_t B, int64_t Hq, int64_t kvh,
                              int32_t* units, int64_t max_units, int32_t* tokens,
                              int64_t max_tokens, int64_t* sizes) {
  int rc = check_heads(Hq, kvh, 128);
  if (rc) return rc;
  if (sizes == nullptr || B < 0 || (B > 0 && counts == nullptr)) return TM_ERR_ARG;
  if (B > INT32_MAX) return TM_ERR_SHAPE;
  const int64_t group = Hq / kvh;
  int64_t total = 0, longest = 0;
  for (int64_t b = 0; b < B; ++b) {
    if (counts[b] < 0 || counts[b] > TM_MAX_PROMPT_KEYS) return TM_ERR_SHAPE;
    total += counts[b];
    if (total * group > INT32_MAX - 1024) return TM_ERR_SHAPE;
    longest = std::max(longest, counts[b]);
  }
  const int64_t rows = own_tile_rows(longest, group);
  int64_t n = 0;
  for (int64_t b = 0; b < B; ++b) n += ceil_div(counts[b] * group, rows);
  sizes[0] = n;
  sizes[1] = total;
  sizes[2] = longest;
  if (units == nullptr && tokens == nullptr) return TM_OK;
  if (max_units < n || max_tokens < total) return TM_ERR_SHAPE;
  if ((units == nullptr && n > 0) || (tokens == nullptr && total > 0)) return TM_ERR_ARG;
  int64_t at = 0, first = 0;
  for (int64_t b = 0; b < B; ++b) {
    const int64_t tiles = ceil_div(counts[b] * group, rows);
    for (int64_t t = 0; t < tiles; ++t) {
      int32_t* const u = units + 4 * (at + t);
      u[0] = (int32_t)b;
      u[1] = (int32_t)t;
      u[2] = (int32_t)first;
      u[3] = (int32_t)counts[b];
    }
    for (int64_t i = 0; i < counts[b]; ++i) {
      int32_t* const x = tokens + 4 * (first + i);
      x[0] = (int32_t)b;
      x[1] = (int32_t)i;
      x[2] = (int32_t)at;
      x[3] = 0;
    }
    at += tiles;
    first += counts[b];
  }
  return TM_OK;
}

extern "C" int tm_branch_workspace(int64_t T, int64_t units, int64_t max_count, int64_t seq_len,
                                   int64_t longest, int64_t Hq, int64_t kvh, int64_t hd,
                                   int64_t* bytes) {
  int rc = check_heads(Hq, kvh, hd);
  if (rc) return rc;
  if (bytes == nullptr) return TM_ERR_ARG;
  BranchPlan o;
  rc = plan_branches(T, units, max_count, seq_len, longest, Hq, kvh, hd, &o);
  if (rc) return rc;
  *bytes = 4 * o.floats;
  return TM_OK;
}

extern "C" int tm_branch_attention(
    const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
    int64_t v_stride, int64_t T, const void* k_cache, const void* v_cache, int64_t stride_page,
    int64_t stride_slot, int64_t page_size, int64_t cache_pages, const int32_t* block_table,
    int64_t num_table_pages, int64_t seq_len, void* k_rows, void* v_rows, int64_t stride_row,
    int64_t stride_pos, int64_t rows, int64_t capacity, const int32_t* origin,
    int64_t origin_stride, const int32_t* lengths, int64_t longest, const int32_t* units,
    int64_t num_units, const int32_t* tokens, int64_t max_count, int64_t Hq, int64_t kvh,
    int64_t hd, float scale, int dtype, void* out, int64_t out_stride, void* workspace,
    int64_t workspace_bytes, void* stream) {
  int rc = check_heads(Hq, kvh, hd);
  if (rc) return rc;
  if ((dtype != TM_DTYPE_BF16 && dtype != TM_DTYPE_F16) || !(scale > 0.0f) || scale == INFINITY)
    return TM_ERR_ARG;
  const int64_t group = Hq / kvh;
  if (T < 0 || rows < 0 || rows > INT32_MAX || capacity < 0 || capacity > TM_MAX_PROMPT_KEYS ||
      longest > capacity)
    return TM_ERR_SHAPE;
  if (T == 0) return TM_OK;
  if ((units == nullptr) != (tokens == nullptr)) return TM_ERR_ARG;
  if (max_count < 1 || max_count > T || T > INT32_MAX) return TM_ERR_SHAPE;
  const int64_t tile = own_tile_rows(max_count, group);
  int64_t unit_tiles = 1;
  if (units == nullptr) {
    if (rows < 1 || T != rows * max_count) return TM_ERR_SHAPE;
    unit_tiles = ceil_div(max_count * group, tile);
    if (num_units != rows * unit_tiles) return TM_ERR_SHAPE;
  } else if (num_units < 1 || num_units > T * ceil_div(group, tile)) {
    return TM_ERR_SHAPE;  // (n tokens of a branch have at most n times a token's tiles)
  }
  BranchPlan o;
  rc = plan_branches(T, num_units, max_count, seq_len, longest, Hq, kvh, hd, &o);
  if (rc) return rc;
  if (seq_len > 0 &&
      (page_size < 1 || page_size > (1 << 24) || (page_size & (page_size - 1)) != 0 ||
       cache_pages < 1 || cache_pages > INT32_MAX || num_table_pages > INT32_MAX ||
       ceil_div(seq_len, page_size) > num_table_pages || stride_slot < kvh * hd ||
       stride_slot > kMaxStride || stride_page < page_size * stride_slot))
    return TM_ERR_SHAPE;
  if ((T > 1 && (q_stride < Hq * hd || out_stride < Hq * hd || k_stride < kvh * hd ||
                 v_stride < kvh * hd)) ||
      k_stride > kMaxStride || v_stride > kMaxStride || stride_pos < kvh * hd ||
      stride_pos > kMaxStride || stride_row < capacity * stride_pos ||
      (origin != nullptr && origin_stride < capacity))
    return TM_ERR_SHAPE;
  if (4 * o.floats > workspace_bytes) return TM_ERR_SHAPE;
  if (!vec_ok(q, T > 1 ? q_stride : 0) || !vec_ok(out, T > 1 ? out_stride : 0) ||
      !vec_ok(k, T > 1 ? k_stride : 0) || !vec_ok(v, T > 1 ? v_stride : 0) ||
      !vec_ok(k_rows, stride_row) || !vec_ok(v_rows, stride_pos) ||
      (seq_len > 0 && (!vec_ok(k_cache, stride_slot) || !vec_ok(v_cache, stride_page))) ||
      (uintptr_t)units % 16 || (uintptr_t)tokens % 16 || (uintptr_t)block_table % 4 ||
      (uintptr_t)origin % 4 || (uintptr_t)lengths % 4 || (uintptr_t)workspace % 16)
    return TM_ERR_ALIGN;
  const hipStream_t st = (hipStream_t)stream;
  BranchParams p = {};
  p.q = (const uint16_t*)q;
  p.out = (uint16_t*)out;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.kvh = (int)kvh;
  p.group = (int)group;
  p.scale_log2 = scale * 1.4426950408889634f;
  float* at = (float*)workspace;
  BranchJoin j = {};
  PromptParams s = p;
  if (seq_len > 0) {
    s.k = (const uint16_t*)k_cache;
    s.v = (const uint16_t*)v_cache;
    s.table = block_table;
    s.k_stride = s.v_stride = stride_slot;
    s.stride_page = stride_page;
    s.q_len = (int)T;
    s.k_len = (int)seq_len;
    while ((int64_t(1) << s.page_shift) < page_size) ++s.page_shift;
    s.cache_pages = (int)cache_pages;
    // (keys of a stage that a wave takes from one page)
    s.wide = page_size >= 16 ? 1 : 0;
    const int64_t part_rows = o.prefix_slots * kvh * o.prefix.part_rows;
    s.part = at;
    s.stats = at + part_rows * hd;
    at += o.prefix_floats;
    if (o.few) {
      s.tiles = (int)o.prefix.tiles;
      s.chunks = (int)o.prefix.chunks;
      s.chunk_len = (int)o.prefix.chunk_len;
      s.part_rows = (int)o.prefix.part_rows;
      s.whole = 1;
    } else if (!o.chain) {
      tm_prefix_launch(s, o.prefix, dtype, hd, page_size, st);
    }
  }
  j.shared.tile_rows = 1;
  if (o.prefix_slots > 0)
    j.shared = {s.part, s.stats, (int)o.prefix.chunks, (int)o.prefix.tile_rows,
                (int)o.prefix.part_rows, o.prefix.kind != 0};
  p.k = (const uint16_t*)k_rows;
  p.v = (const uint16_t*)v_rows;
  p.k_stride = p.v_stride = stride_pos;
  p.row_stride = stride_row;
  p.new_k = (const uint16_t*)k;
  p.new_v = (const uint16_t*)v;
  p.new_k_stride = k_stride;
  p.new_v_stride = v_stride;
  p.origin = origin;
  p.origin_stride = origin_stride;
  p.lengths = lengths;
  p.units = (const int4*)units;
  p.count = (int)max_count;
  p.unit_tiles = (int)unit_tiles;
  p.rows = (int)rows;
  p.capacity = (int)capacity;
  p.chunks = (int)o.chunks;
  p.whole_units = (int)o.whole_units;
  p.span = (int)o.span;
  p.parts = o.own_slots > 0;
  p.part_rows = (int)o.own_rows;
  p.part = at;
  p.stats = at + o.own_slots * kvh * o.own_rows * hd;
  j.own = {p.part, p.stats, (int)o.chunks, o.few ? 32 : 128, (int)o.own_rows, !o.few};
  j.tokens = (const int4*)tokens;
  j.count = (int)max_count;
  j.unit_tiles = (int)unit_tiles;
  j.T = (int)T;
  j.Hq = (int)Hq;
  j.kvh = (int)kvh;
  j.group = (int)group;
  j.out = (uint16_t*)out;
  j.out_stride = out_stride;
#define TM_BRANCH(DT, HD)                             \
  do {                                                \
    launch_own<DT, HD>(s, p, o, st);                  \
    if (p.parts) launch_join<DT, HD>(p, j, o, st);    \
  } while (0)
  if (dtype == TM_DTYPE_F16) {
    if (hd == 128)
      TM_BRANCH(TM_DTYPE_F16, 128);
    else
      TM_BRANCH(TM_DTYPE_F16, 64);
  } else {
    if (hd == 128)
      TM_BRANCH(TM_DTYPE_BF16, 128);
    else
      TM_BRANCH(TM_DTYPE_BF16, 64);
  }
#undef TM_BRANCH
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

extern "C" int tm_branch_advance(int32_t* lengths, const int32_t* counts, int64_t count,
                                 int64_t rows, int64_t capacity, int32_t* origin,
                                 int64_t origin_stride, void* stream) {
  if (rows < 0 || rows > UINT32_MAX / 64 || capacity < 0 || capacity > TM_MAX_PROMPT_KEYS ||
      count < 0 || count > TM_MAX_PROMPT_KEYS ||
      (origin != nullptr && rows > 1 && origin_stride < capacity))
    return TM_ERR_SHAPE;
  if (rows == 0) return TM_OK;
  if ((uintptr_t)lengths % 4 || (uintptr_t)counts % 4 || (uintptr_t)origin % 4)
    return TM_ERR_ALIGN;
  hipLaunchKernelGGL(tm_branch_advance_kernel, dim3((unsigned)rows), dim3(64), 0,
                     (hipStream_t)stream, lengths, counts, (int)count, (int)capacity, origin,
                     origin_stride);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}
