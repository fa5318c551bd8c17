// What every cached key gets of the queries' attention, and the eviction of the keys that
// get least.
//
// Mass.  For the last T of a sequence's S positions, a KV head's rows being the (token, head
// of the group) pairs,
//   mass[j] += sum over the rows that see key j of exp(s_rj - m_r) / l_r,
// with s = scale q . k, m_r the largest of a row's scores and l_r the sum of its
// exponentials.  Two launches: m and l of every row, over ranges of keys; then, key tile
// by key tile, the scores again and their sums over the rows.  K is read twice, from L2 the
// second time where a head's keys fit it (a head's workgroups share an XCD); the
// scores of many rows would be far more to store than to compute twice.  All in fp32; the
// order of the sums is fixed.
//
// Eviction.  Of each layer's KV heads, `keep` of S keys stay: the first `sinks` and the last
// `recent` positions, and the heaviest others.  Kept keys in slots from `keep` on move into
// the holes below, the i-th into the i-th; all others stay where they are, so a cache that
// is cut every few tokens moves few keys.  Attention does not go by the order of the
// slots; the positions go along.  One workgroup a head selects (a radix search over the
// ordered bits of the weights), a second launch moves.
#include <algorithm>
#include <cmath>

#include "attn_tile.h"

namespace {

struct MassParams : PromptParams {
  float2* row_stats;      // (m in base 2, l) [chunks][kvh][rows]
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

// Rows 128 a tile, 32 a wave, that share the stages of a range of keys.
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 2) tm_mass_stats_kernel(MassParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k1[S::kTile];
  const int kvhead = (int)blockIdx.x % p.kvh, at_item = (int)blockIdx.x / p.kvh;
  const Item it = item_of(p, at_item, 128);
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
  if (at.ok && (threadIdx.x & 32) == 0)
    p.row_stats[((int64_t)(at_item % p.chunks) * p.kvh + kvhead) * it.q_len * p.group + at.row] =
        float2{r.m, l};
}

// Up to 32 rows: the waves take the stages in turn.
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

// Sums over the rows, 64 keys a wave or (SHARE 4) a workgroup, whose waves take the tiles of
// 32 rows in turn.  K stays in registers, the queries stream through.
template <int DT, int HD, int SHARE>
__global__ void __launch_bounds__(kThreads, 2) tm_mass_sum_kernel(MassParams p) {
  __shared__ float s_sum[4][64];
  const int lane = threadIdx.x & 63, half = lane >> 5, c32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int kvhead = (int)blockIdx.x % p.kvh;
  const int unit = (int)blockIdx.x / p.kvh;
  const int first = (SHARE == 1 ? unit * 4 + wave : unit) * kKeys;
  const int rows = p.q_len * p.group, past = p.k_len - p.q_len;
  u32x4_t kf[2][HD / 16];
  float acc[2][16];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int x = 0; x < 16; ++x) acc[kt][x] = 0.0f;
  const int tiles = (rows + 31) / 32;
  // the first tile of rows of which one sees the first key
  const int tile0 = first > past ? (first - past) * p.group / 32 : 0;
  const int mine = SHARE == 1 ? 0 : wave;
  if (first < p.k_len && tile0 + mine < tiles) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int key = min(first + 32 * kt + c32, p.k_len - 1);
      const int pg = min(max(p.table[key >> p.page_shift], 0), p.cache_pages - 1);
      const uint16_t* const kr = p.k + (int64_t)pg * p.stride_page +
                                 (int64_t)(key & ((1 << p.page_shift) - 1)) * p.k_stride +
                                 kvhead * HD + 8 * half;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        kf[kt][ks] = *reinterpret_cast<const u32x4_t*>(kr + 16 * ks);
    }
    struct Tile {
      u32x4_t q[HD / 16];
      float m, inv;
      int seen;
    };
    auto read = [&](int tile, Tile& t) TM_INLINE {
      const int row = tile * 32 + c32;
      const bool ok = row < rows;
      const int token = ok ? row / p.group : 0;
      const int head = kvhead * p.group + (ok ? row - token * p.group : 0);
      const uint16_t* const qr = p.q + (int64_t)token * p.q_stride + (int64_t)head * HD + 8 * half;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        t.q[ks] = *reinterpret_cast<const u32x4_t*>(qr + 16 * ks);
      float m = -INFINITY, l = 0.0f;
      if (ok) {
        const float2* const st = p.row_stats + (int64_t)kvhead * rows + row;
        const int64_t step = (int64_t)p.kvh * rows;
        const float2 a = st[0];
        m = a.x;
        l = a.y;
        for (int c = 1; c < p.chunks; ++c) {
          const float2 b = st[c * step];
          join_stats(m, l, b.x, b.y);
        }
      }
      // (a row of scores -inf gives nothing)
      t.m = l == 0.0f ? 0.0f : -m;
      t.inv = l == 0.0f ? 0.0f : 1.0f / l;
      t.seen = ok ? past + token : -1;
    };
    auto add = [&](int tile, const Tile& t) TM_INLINE {
      f32x16_t sc[2];
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          const f32x16_t zero = {};
          sc[kt] = mfma32<DT>(kf[kt][ks], t.q[ks], ks == 0 ? zero : sc[kt]);
        }
      // masked where some row of the tile does not see some key
      if (tile * 32 + 32 > rows || past + tile * 32 / p.group < first + kKeys - 1)
        mask_scores(sc, t.seen - first - 4 * half);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          acc[kt][x] = fmaf(__builtin_amdgcn_exp2f(fmaf(sc[kt][x], p.scale_log2, t.m)), t.inv,
                            acc[kt][x]);
    };
    Tile a, b;
    int t = tile0 + mine;
    read(t, a);
    for (; t < tiles; t += 2 * SHARE) {
      if (t + SHARE < tiles) read(t + SHARE, b);
      add(t, a);
      if (t + SHARE < tiles) {
        if (t + 2 * SHARE < tiles) read(t + 2 * SHARE, a);
        add(t + SHARE, b);
      }
    }
  }
  // over the 32 columns of each half: lane x of a half gets key x's sum, kt 0 and 1
  float sum[2] = {0.0f, 0.0f};
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      float v = acc[kt][x];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) v += __shfl_xor(v, d);
      sum[kt] = c32 == x ? v : sum[kt];
    }
  const int in = 8 * (c32 >> 2) + 4 * half + (c32 & 3);  // the key that a lane below 16 has
  auto store = [&](int key, float v) TM_INLINE {
    if (key >= p.k_len) return;
    if (p.before != nullptr) v += p.before[kvhead * p.before_stride + key];
    p.mass[kvhead * p.mass_stride + key] = v;
  };
  if constexpr (SHARE == 1) {
    if (c32 < 16) {
      store(first + in, sum[0]);
      store(first + 32 + in, sum[1]);
    }
  } else {
    if (c32 < 16) {
      s_sum[wave][in] = sum[0];
      s_sum[wave][32 + in] = sum[1];
    }
    __syncthreads();
    if (threadIdx.x < 64)
      store(first + lane,
            (s_sum[0][lane] + s_sum[1][lane]) + (s_sum[2][lane] + s_sum[3][lane]));
  }
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

__global__ void __launch_bounds__(kSelect) tm_evict_select_kernel(EvictParams p) {
  __shared__ uint32_t s_bins[kBins];
  __shared__ int s_waves[kSelect / 64];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, head = blockIdx.x;
  const int layer = head / p.kvh, kvhead = head - layer * p.kvh;
  const float* const mass = p.mass + layer * p.mass_layer + kvhead * p.mass_head;
  const int32_t* const pos =
      p.positions == nullptr ? nullptr : p.positions + layer * p.pos_layer + kvhead * p.pos_head;
  auto position = [&](int s) { return s < p.recorded ? pos[s] : p.next - p.length + s; };
  // larger: kept sooner.  NaN last; what is kept in any case first.
  auto key_of = [&](int s) {
    const int at = position(s);
    if (at < p.sinks || at >= p.next - p.recent) return 0xffffffffu;
    const float m = mass[s];
    if (m != m) return 0u;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return u ^ (uint32_t)(((int32_t)u >> 31) | 0x80000000);
  };
  // the keep-th largest key, 11, 11 and 10 bits at a time, and how many of its equals stay
  uint32_t prefix = 0;
  int need = p.keep;
  if (p.keep < p.length && p.keep > 0) {
    for (int shift = 21; shift >= 0; shift -= shift == 21 ? 11 : 10) {
      const int bits = shift == 0 ? 10 : 11;
      for (int i = tid; i < kBins; i += kSelect) s_bins[i] = 0;
      __syncthreads();
      for (int s = tid; s < p.length; s += kSelect) {
        const uint32_t k = key_of(s);
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
  int32_t* const holes = p.holes + (int64_t)head * p.moves;
  int32_t* const movers = p.movers + (int64_t)head * p.moves;
  float* const mass_out = p.mass_out + (int64_t)head * p.columns;
  int32_t* const pos_out = p.positions_out + (int64_t)head * p.keep;
  int equal0 = 0, hole0 = 0, mover0 = 0;
  const bool all = p.keep >= p.length;
  for (int s0 = 0; s0 < p.length; s0 += kSelect) {
    const int s = s0 + tid;
    const bool in = s < p.length;
    const uint32_t k = in ? key_of(s) : 0;
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
      mass_out[s] = mass[s];
      pos_out[s] = position(s);
    }
  }
  for (int s = p.keep + tid; s < p.columns; s += kSelect) mass_out[s] = 0.0f;
  const int moves = min(min(hole0, mover0), p.moves);
  if (tid == 0) p.counts[head] = moves;
  __syncthreads();  // this workgroup's lists
  for (int i = tid; i < moves; i += kSelect) {
    const int to = holes[i], from = movers[i];
    mass_out[to] = mass[from];
    pos_out[to] = position(from);
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
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct MassPlan {
  bool few;
  int64_t rows, tiles, chunks, chunk_len, bytes;
};

int plan_mass(int64_t T, int64_t S, int64_t Hq, int64_t kvh, int64_t hd, MassPlan* o) {
  if (kvh < 1 || Hq < kvh || Hq % kvh != 0 || Hq > 1024 || (hd != 64 && hd != 128))
    return TM_ERR_SHAPE;
  const int64_t group = Hq / kvh;
  if (T < 0 || S < T || S > TM_MAX_PROMPT_KEYS || T * group > INT32_MAX - 1024)
    return TM_ERR_SHAPE;
  o->rows = T * group;
  o->few = o->rows <= 32;
  o->tiles = ceil_div(o->rows, o->few ? 32 : 128);
  // ranges of keys as many as fill the chip, of four stages or more
  const int64_t units = std::max<int64_t>(o->tiles * kvh, 1);
  const int64_t want = std::max<int64_t>(1, 2 * kCUs / units);
  const int64_t chunks = std::max<int64_t>(1, std::min(want, ceil_div(S, 4 * kKeys)));
  const int64_t step = o->few ? 4 * kKeys : kKeys;
  o->chunk_len = std::max(step, ceil_div(ceil_div(S, chunks), step) * step);
  o->chunks = std::max<int64_t>(1, ceil_div(S, o->chunk_len));
  o->bytes = o->chunks * kvh * o->rows * 8;
  if (o->tiles * o->chunks * kvh > UINT32_MAX / kThreads ||
      ceil_div(S, kKeys) * kvh > UINT32_MAX / kThreads)
    return TM_ERR_SHAPE;
  return TM_OK;
}

template <int DT, int HD>
void launch_mass(const MassParams& p, const MassPlan& o, hipStream_t st) {
  const dim3 block(kThreads);
  const dim3 items((unsigned)(o.tiles * o.chunks * p.kvh));
  const int64_t keys = ceil_div(p.k_len, kKeys);
  if (o.rows > 0) {
    if (o.few)
      hipLaunchKernelGGL((tm_mass_stats_few_kernel<DT, HD>), items, block, 0, st, p);
    else
      hipLaunchKernelGGL((tm_mass_stats_kernel<DT, HD>), items, block, 0, st, p);
  }
  if (o.rows <= 64)
    hipLaunchKernelGGL((tm_mass_sum_kernel<DT, HD, 1>),
                       dim3((unsigned)(ceil_div(keys, 4) * p.kvh)), block, 0, st, p);
  else
    hipLaunchKernelGGL((tm_mass_sum_kernel<DT, HD, 4>), dim3((unsigned)(keys * p.kvh)), block, 0,
                       st, p);
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
      (uintptr_t)mass % 4 || (uintptr_t)workspace % 8)
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
  p.row_stats = (float2*)workspace;
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
  hipLaunchKernelGGL(tm_evict_select_kernel, dim3((unsigned)o.heads), dim3(kSelect), 0, st, p);
  if (o.moves > 0)
    hipLaunchKernelGGL(tm_evict_move_kernel,
                       dim3((unsigned)ceil_div(o.moves, kMovesOf), (unsigned)o.heads),
                       dim3(kThreads), 0, st, p);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}
