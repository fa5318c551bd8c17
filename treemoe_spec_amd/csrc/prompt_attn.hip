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
//
// Per wave and stage (v_mfma_f32_32x32x16):
//   S^T = K Q^T   lane l holds S^T[key 32 kt + 8 (v / 4) + 4 (l / 32) + v % 4][query l % 32]
//                 in accumulator value v of tile kt;
//   softmax       in base 2 against a reference maximum that moves only when a stage
//                 exceeds it by 2^8 (the division by the sum undoes any reference);
//   O^T += V^T P^T   P^T is the S^T registers: the product's k slot j of lane half h
//                 in k-step (kt, m) stands for key 32 kt + 16 m + 8 (j / 4) + 4 h + j % 4,
//                 and V^T is read with the same map, four keys of a column by each
//                 transposing LDS read.
// The weights are rounded to the inputs' 16-bit type, which the product takes: a second
// product with what the rounding left would cost half as many products again.  The sums are
// taken over the rounded weights in fp32, so that the roundings weigh alike above and below the
// division.  The whole output is off by 0.0021 of its norm in bf16 over 8192 tokens, where
// its own rounding alone is 0.0016 (fp16, packed prompts: 0.00024, 0.00020).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <utility>
#include <vector>

#include "tm_vec.h"

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) void glb_void;

// A lambda kept as a call would keep what it captures, a wave's rows, in memory.
#define TM_INLINE __attribute__((always_inline))

constexpr int kThreads = 256;
constexpr int kKeys = 64;   // keys of a stage
constexpr int kCUs = 256;   // MI355X compute units

// One piece of work: tile `tile` of a sequence against its keys [begin, end).
struct Item {
  int q0, q_len;    // the sequence's first row of q and its queries
  int k0, k_len;    // its first row of k and v, and its keys
  int tile;         // rows tile * rows_per_tile ..
  int begin, end;   // keys
  int slot;         // partial slot, or -1: the output itself
};
// A tile whose partials slot0 .. slot0 + count - 1 are joined.
struct Join {
  int q0, q_len, tile, slot0, count, pad[3];
};

struct PromptParams {
  const uint16_t* q;
  const uint16_t* k;           // [S, kvh, hd], or this layer's [pages, page, kvh, hd]
  const uint16_t* v;
  uint16_t* out;
  const int32_t* table;        // block table (paged)
  const Item* items;           // NULL: one sequence, items by arithmetic
  const Join* joins;
  float* part;                 // [slot][kvh][tile rows][hd], 32 rows as end_rows lays them
  float* stats;                // [slot][kvh][tile rows][2]
  int64_t q_stride, k_stride, v_stride, out_stride;  // paged: k_stride is the slot's
  int64_t stride_page;
  int kvh, group, q_len, k_len, tiles, chunks, chunk_len;  // one sequence's
  int page_shift, cache_pages;
  int wide;                    // the keys of each part that a wave loads lie in one page
  float scale_log2;
};

template <int DT>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (DT == TM_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// acc + the two elements of x, in fp32.
template <int DT>
__device__ __forceinline__ float add_pair(uint32_t x, float acc) {
  if constexpr (DT == TM_DTYPE_F16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), one, acc, false);
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x),
                                           __builtin_bit_cast(bf16x2, 0x3f803f80u), acc, false);
  }
}

// The larger of this lane's value and that of lane ^ 32.
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

template <int HD>
struct Shape {
  static constexpr int kRow = HD * 2;              // bytes of a key's row
  static constexpr int kChunks = kRow / 16;        // 16-byte chunks of a row
  static constexpr int kTile = kKeys * kRow;       // bytes of a stage's K, or V
  static constexpr int kKeysPerLoad = 1024 / kRow;
  // Chunk c of key j lies at c ^ swizzle(j).  K is read 16 bytes a lane, 8 or more
  // keys at one logical chunk: the keys' low bits spread them over the banks.  V
  // is read by 16 lanes as 32 bytes of each of four consecutive keys: those move to
  // distinct 64-byte blocks, and the next four keys within them.
  static __device__ __forceinline__ int swz_k(int key) { return key & (kChunks - 1); }
  static __device__ __forceinline__ int swz_v(int key) {
    if constexpr (HD == 128)
      return ((key & 3) << 2) | ((key >> 2) & 3);
    else
      return ((key & 2) << 1) | ((key >> 2) & 3);
  }
};

// Stages of 64 keys into LDS by NW waves, one after the other, V of a stage at any time
// between its K and the next one's.  Keys past the sequence's last are that one again:
// their scores are masked.
template <int HD, bool PAGED, int NW>
struct Feed {
  typedef Shape<HD> S;
  static constexpr int kLoads = S::kTile / (1024 * NW);  // loads of a wave per tile
  static constexpr int kGroup = 2 * kLoads;  // of K and V of a stage
  static constexpr int kWaveKeys = kLoads * S::kKeysPerLoad;  // of a stage, by one wave
  // a wave's keys in parts of at most 16, each within a page of 16 or more
  static constexpr int kParts = kWaveKeys > 16 ? kWaveKeys / 16 : 1;
  static constexpr int kPartKeys = kWaveKeys / kParts;
  const uint16_t *k, *v;   // the next stage's first row (paged: the cache)
  int64_t k_step, v_step;  // from stage to stage
  int k_stride, v_stride;  // of a key, or of a page's slot
  int k_lane[kLoads], v_lane[kLoads];  // this lane's piece from the stage's first row
                                       // (paged: from the wave's)
  int first, left, step;   // the next stage's first key, the last key from there on, and
                           // the keys to the stage behind
  int v_first, v_left;     // of the stage whose K came last
  int64_t off[kParts];     // what its parts' rows in the cache lie past those of one page
  int page[kParts];        // the next stage's pages of the wave, asked for a stage ahead

  // of the NW waves that load a stage together
  static __device__ __forceinline__ int wave() {
    return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) & (NW - 1);
  }
  static __device__ __forceinline__ int wave_key() { return wave() * kWaveKeys; }
  static __device__ __forceinline__ int key_in(int i) {  // within the stage
    return wave_key() + i * S::kKeysPerLoad + (int)(threadIdx.x & 63) / S::kChunks;
  }
  template <bool V>
  static __device__ __forceinline__ int chunk_off(int i) {
    const int j = key_in(i);
    return (((int)threadIdx.x & (S::kChunks - 1)) ^ (V ? S::swz_v(j) : S::swz_k(j))) * 8;
  }
  static __device__ __forceinline__ void to_lds(const uint16_t* from, uint8_t* tile, int i) {
    __builtin_amdgcn_global_load_lds((glb_void*)from,
                                     (lds_void*)(tile + (wave() * kLoads + i) * 1024), 16, 0, 0);
  }
  __device__ __forceinline__ void look_up(const PromptParams& p) {
    if constexpr (PAGED) {
      // by scalar loads, which the waits for K and V do not count: the table does not change
      // during a launch
      const auto table =
          (const __attribute__((address_space(4))) int32_t*)reinterpret_cast<uintptr_t>(p.table);
      page[0] = table[(first + min(wave_key(), left)) >> p.page_shift];
      if (kParts > 1 && (1 << p.page_shift) < kWaveKeys)
#pragma unroll
        for (int j = 1; j < kParts; ++j)
          page[j] = table[(first + min(wave_key() + j * kPartKeys, left)) >> p.page_shift];
    }
  }
  // From key `begin` on of the item's sequence, `step` keys from stage to stage.
  __device__ __forceinline__ void start(const PromptParams& p, const Item& it, int kvhead,
                                        int begin, int step_) {
    k = p.k + (int64_t)kvhead * HD + (PAGED ? 0 : (int64_t)(it.k0 + begin) * p.k_stride);
    v = p.v + (int64_t)kvhead * HD + (PAGED ? 0 : (int64_t)(it.k0 + begin) * p.v_stride);
    step = step_;
    k_step = step * p.k_stride;
    v_step = step * p.v_stride;
    k_stride = (int)p.k_stride;
    v_stride = (int)p.v_stride;
    first = begin;
    left = it.k_len - 1 - begin;
    v_first = v_left = 0;
#pragma unroll
    for (int j = 0; j < kParts; ++j) off[j] = page[j] = 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int key = key_in(i) - (PAGED ? wave_key() : 0);
      k_lane[i] = key * k_stride + chunk_off<false>(i);
      v_lane[i] = key * v_stride + chunk_off<true>(i);
    }
    look_up(p);
  }
  // K or V of a stage row by row: near the sequence's end (`left_` is negative for a
  // stage behind it), or where a wave's keys lie in several pages.
  template <bool V>
  __device__ __forceinline__ void load_rows(const PromptParams& p, int first_, int left_,
                                            uint8_t* tile) const {
    const uint16_t* const base = V ? v : k;
    const int stride = V ? v_stride : k_stride;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int j = min(key_in(i), left_);
      int64_t o;
      if constexpr (PAGED) {
        const int key = first_ + j;
        const int pg = min(max(p.table[key >> p.page_shift], 0), p.cache_pages - 1);
        o = (int64_t)pg * p.stride_page +
            (int64_t)(key & ((1 << p.page_shift) - 1)) * stride + chunk_off<V>(i);
      } else {
        o = (int64_t)j * stride + chunk_off<V>(i);
      }
      to_lds(base + o, tile, i);
    }
  }
  __device__ __forceinline__ bool whole(const PromptParams& p, int left_) const {
    return left_ >= kKeys - 1 && (!PAGED || p.wide);
  }
  __device__ __forceinline__ void load_k(const PromptParams& p, uint8_t* tile) {
    if (whole(p, left)) {
      if constexpr (PAGED) {
        auto off_of = [&](int j) TM_INLINE {
          const int pg = min(max(__builtin_amdgcn_readfirstlane(page[j]), 0), p.cache_pages - 1);
          const int slot = (first + wave_key() + j * kPartKeys) & ((1 << p.page_shift) - 1);
          return (int64_t)pg * p.stride_page + (int64_t)(slot - j * kPartKeys) * k_stride;
        };
        off[0] = off_of(0);
        const bool one = kParts == 1 || (1 << p.page_shift) >= kWaveKeys;  // one page
#pragma unroll
        for (int j = 1; j < kParts; ++j) off[j] = off[0];
        if (!one)
#pragma unroll
          for (int j = 1; j < kParts; ++j) off[j] = off_of(j);
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        to_lds(k + off[i * kParts / kLoads] + (uint32_t)k_lane[i], tile, i);
    } else {
      load_rows<false>(p, first, left, tile);
    }
    v_first = first;
    v_left = left;
    first += step;
    left -= step;
    if constexpr (!PAGED) k += k_step;
    look_up(p);
  }
  __device__ __forceinline__ void load_v(const PromptParams& p, uint8_t* tile) {
    if (whole(p, v_left)) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        to_lds(v + off[i * kParts / kLoads] + (uint32_t)v_lane[i], tile, i);
    } else {
      load_rows<true>(p, v_first, v_left, tile);
    }
    if constexpr (!PAGED) v += v_step;
  }
};

// A value that the compiler takes as new, so that addresses made from it are not kept
// in registers from one stage to the next.
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ u32x2_t read_tr(const uint8_t* p) {
  return __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) s16x4_t*)(lds_void*)const_cast<uint8_t*>(p)));
}

// Byte offsets of a lane's part of V^T fragments: keys 0-3 (lo) or 8-11 (hi) of a k-step,
// head-dim tile 0; tile ht is at ^ 64 ht.
template <int HD>
__device__ __forceinline__ void v_offsets(int& lo, int& hi) {
  typedef Shape<HD> S;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int k0 = 4 * (g >> 1) + (i >> 2);
  const int chunk = 2 * (g & 1) + ((i & 3) >> 1);
  lo = k0 * S::kRow + (chunk ^ S::swz_v(k0)) * 16 + (i & 1) * 8;
  hi = (k0 + 8) * S::kRow + (chunk ^ S::swz_v(k0 + 8)) * 16 + (i & 1) * 8;
}

// The wave's 32 rows (a lane's column is one row; its lane ^ 32 holds the same).
template <int HD>
struct Rows {
  u32x4_t q[HD / 16];    // Q^T fragments
  f32x16_t o[HD / 32];   // O^T
  f32x16_t sc[2];        // S^T of a stage
  u32x4_t pw[4];         // its weights: k-step (kt, m) at 2 kt + m
  float m, l;            // reference maximum (base 2), and this lane's part of the sum
  int seen;              // the row's last visible key
};

// Fragments of k-steps 2 i and 2 i + 1 of the K stage at kt_.
template <int HD>
__device__ __forceinline__ void read_k(const uint8_t* kt_, int at, int i, u32x4_t (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    f[j] = *reinterpret_cast<const u32x4_t*>(kt_ + 32 * (j & 1) * Shape<HD>::kRow +
                                             (at ^ (32 * (2 * i + (j >> 1)))));
}
// Byte offset of chunk `half` of row l % 32 of K; k-step ks is at ^ 32 ks.
template <int HD>
__device__ __forceinline__ int k_offset() {
  const int lane = threadIdx.x & 63, c32 = lane & 31;
  return fresh(c32 * Shape<HD>::kRow + ((lane >> 5) ^ Shape<HD>::swz_k(c32)) * 16);
}
// Fragments of the 16 keys from 16 s on of the V stage at vt.
template <int HD>
__device__ __forceinline__ void read_v(const uint8_t* vt, int lo, int hi, int s,
                                       u32x4_t (&f)[HD / 32]) {
#pragma unroll
  for (int ht = 0; ht < HD / 32; ++ht) {
    const u32x2_t a = read_tr(vt + 16 * s * Shape<HD>::kRow + (lo ^ (64 * ht)));
    const u32x2_t b = read_tr(vt + 16 * s * Shape<HD>::kRow + (hi ^ (64 * ht)));
    f[ht] = u32x4_t{a.x, a.y, b.x, b.y};
  }
}

// One product, then `reads` LDS reads, `n` times: each product covers the reads of
// the step behind it.
template <int N, int READS>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
}

// O^T += V^T P^T of the stage at vt (G), then S^T = K Q^T of the stage at kt_ (S).  A
// step's fragments are read between the products of the step before it.
template <int DT, int HD, bool G, bool S>
__device__ __forceinline__ void products(const uint8_t* vt, const uint8_t* kt_, Rows<HD>& r) {
  constexpr int HT = HD / 32, KP = HD / 32;  // output tiles; pairs of k-steps
  u32x4_t kf[2][4];
  int at = 0;
  if constexpr (S) at = k_offset<HD>();
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (G) {
    u32x4_t vf[2][HT];
    int lo, hi;
    v_offsets<HD>(lo, hi);
    lo = fresh(lo);
    hi = fresh(hi);
    read_v<HD>(vt, lo, hi, 0, vf[0]);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      __builtin_amdgcn_sched_barrier(0);
      if (s < 3)
        read_v<HD>(vt, lo, hi, s + 1, vf[(s + 1) & 1]);
      else if (S)
        read_k<HD>(kt_, at, 0, kf[0]);
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) r.o[ht] = mfma32<DT>(vf[s & 1][ht], r.pw[s], r.o[ht]);
      if (s < 3)
        interleave<HT, 2>();
      else if (S)
        interleave<HT, 4 / HT>();
    }
  } else {
    read_k<HD>(kt_, at, 0, kf[0]);
  }
  if constexpr (S) {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + 1 < KP) read_k<HD>(kt_, at, i + 1, kf[(i + 1) & 1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x16_t zero = {};
        r.sc[j & 1] = mfma32<DT>(kf[i & 1][j], r.q[2 * i + (j >> 1)],
                                 i == 0 && j < 2 ? zero : r.sc[j & 1]);
      }
      if (i + 1 < KP) interleave<4, 1>();
    }
  }
  __builtin_amdgcn_sched_barrier(0);
}

// The weights of the stage's keys kb .. against the running maximum.  mask: some key
// lies past the last one that some row sees.
template <int DT, int HD>
__device__ __forceinline__ void weigh(float scale_log2, int kb, bool mask, Rows<HD>& r) {
  if (mask) {
    const int left = r.seen - kb - 4 * ((int)(threadIdx.x & 63) >> 5);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int x = 0; x < 16; ++x)
        r.sc[kt][x] = 32 * kt + 8 * (x >> 2) + (x & 3) <= left ? r.sc[kt][x] : -INFINITY;
  }
  float mx[2] = {fmaxf(r.sc[0][0], r.sc[1][0]), fmaxf(r.sc[0][1], r.sc[1][1])};
#pragma unroll
  for (int x = 2; x < 16; ++x) mx[x & 1] = fmaxf(fmaxf(mx[x & 1], r.sc[0][x]), r.sc[1][x]);
  const float cand = max_halves(fmaxf(mx[0], mx[1])) * scale_log2;
  const bool bump = cand > r.m + 8.0f;
  if (__any(bump)) {
    const float m = bump ? cand : r.m;
    const float a = bump ? __builtin_amdgcn_exp2f(r.m - m) : 1.0f;
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
      for (int x = 0; x < 16; ++x) r.o[ht][x] *= a;
    r.l *= a;
    r.m = m;
  }
  const float base = r.m == -INFINITY ? 0.0f : -r.m;
  float sum[2] = {0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int x = 8 * (s & 1) + 2 * j;
      const float e0 = __builtin_amdgcn_exp2f(fmaf(r.sc[s >> 1][x], scale_log2, base));
      const float e1 = __builtin_amdgcn_exp2f(fmaf(r.sc[s >> 1][x + 1], scale_log2, base));
      // made here, not moved into the products
      const uint32_t w = (uint32_t)fresh((int)tm_pack2<DT>(e0, e1));
      sum[j & 1] = add_pair<DT>(w, sum[j & 1]);
      r.pw[s][j] = w;
    }
  r.l += sum[0] + sum[1];
}

// What a workgroup works on.
__device__ __forceinline__ Item item_of(const PromptParams& p, int at, int rows) {
  if (p.items != nullptr) return p.items[at];
  Item it;
  it.q0 = it.k0 = 0;
  it.q_len = p.q_len;
  it.k_len = p.k_len;
  it.tile = p.tiles - 1 - at / p.chunks;
  const int chunk = at % p.chunks;
  const int last_token = min(it.q_len - 1, (it.tile * rows + rows - 1) / p.group);
  it.begin = chunk * p.chunk_len;
  it.end = min(it.begin + p.chunk_len, it.k_len - it.q_len + last_token + 1);
  it.slot = p.chunks > 1 ? it.tile * p.chunks + chunk : -1;
  return it;
}

// Elements e .. e + 3 of row `row` of a sequence whose first query is q0, divided by the
// row's sum (0 where nothing was seen; NaN stays).
template <int DT>
__device__ __forceinline__ void store_row(const PromptParams& p, int q0, int row, int kvhead,
                                          int hd, int e, f32x4_t o, float sum) {
  const float inv = sum > 0.0f ? 1.0f / sum : sum;
  const int token = row / p.group;
  const int head = kvhead * p.group + row - token * p.group;
  u32x2_t w;
  w.x = tm_pack2<DT>(o[0] * inv, o[1] * inv);
  w.y = tm_pack2<DT>(o[2] * inv, o[3] * inv);
  *reinterpret_cast<u32x2_t*>(p.out + (int64_t)(q0 + token) * p.out_stride + (int64_t)head * hd +
                              e) = w;
}

// Where a wave's rows lie.
struct Place {
  bool ok;          // this lane's column is a row
  int row;          // of the sequence
  int full;         // the last key that every row of the wave sees, within the range
};

// Rows first .. first + 31 of the sequence: their Q^T fragments, nothing seen yet.
template <int HD>
__device__ __forceinline__ Place begin_rows(const PromptParams& p, const Item& it, int kvhead,
                                            int first, Rows<HD>& r) {
  const int lane = threadIdx.x & 63, half = lane >> 5, c32 = lane & 31;
  const int past = it.k_len - it.q_len, all_rows = it.q_len * p.group;
  Place at;
  at.row = first + c32;
  at.ok = at.row < all_rows;
  const int token = at.ok ? at.row / p.group : 0;
  const int head = kvhead * p.group + (at.ok ? at.row - token * p.group : 0);
  const uint16_t* const qr =
      p.q + (int64_t)(it.q0 + token) * p.q_stride + (int64_t)head * HD + 8 * half;
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(qr + 16 * ks);
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    r.q[ks] = at.ok ? x : zero;
  }
#pragma unroll
  for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
    for (int x = 0; x < 16; ++x) r.o[ht][x] = 0.0f;
  r.m = -INFINITY;
  r.l = 0.0f;
  // a range's end hides what lies past it
  r.seen = min(at.ok ? past + token : -1, it.end - 1);
  at.full = min(first + 32 <= all_rows ? past + first / p.group : -1, it.end - 1);
  return at;
}

// The weight 0 of a key that a row does not see still makes NaN of an infinity or NaN in
// its value, by the products.  Rows whose output is not finite are therefore taken again,
// key by key over what each sees: stages s0, s0 + step, ... of the range.  Slow, and
// only reached where an input is not finite or a product overflows.
template <int DT, int HD, bool PAGED>
__device__ __forceinline__ void retake(const PromptParams& p, const Item& it, int kvhead, int s0,
                                       int step, int n, Rows<HD>& r) {
  float bad[8] = {r.l * 0.0f};  // 0 times what is not finite is NaN
#pragma unroll
  for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
    for (int x = 0; x < 16; ++x) bad[x & 7] = fmaf(r.o[ht][x], 0.0f, bad[x & 7]);
  if (!__any(((bad[0] + bad[1]) + (bad[2] + bad[3])) +
                 ((bad[4] + bad[5]) + (bad[6] + bad[7])) != 0.0f))
    return;
  const int half = (int)(threadIdx.x & 63) >> 5;
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
    for (int x = 0; x < 16; ++x) r.o[ht][x] = 0.0f;
  for (int s = s0; s < n; s += step) {
    const int first = it.begin + s * kKeys, end = min(first + kKeys, it.end);
#pragma unroll 1
    for (int key = first; key < end; ++key) {
      int64_t ka, va;
      if constexpr (PAGED) {
        const int page = min(max(p.table[key >> p.page_shift], 0), p.cache_pages - 1);
        ka = (int64_t)page * p.stride_page +
             (int64_t)(key & ((1 << p.page_shift) - 1)) * p.k_stride;
        va = ka;
      } else {
        ka = (int64_t)(it.k0 + key) * p.k_stride;
        va = (int64_t)(it.k0 + key) * p.v_stride;
      }
      const uint16_t* const kr = p.k + ka + kvhead * HD + 8 * half;
      const uint16_t* const vr = p.v + va + kvhead * HD + 4 * half;
      float dot = 0.0f;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        float a[8], b[8];
        tm_load8<DT>(kr, 16 * ks, a);
        tm_load8<DT>(&r.q[ks], 0, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(a[e], b[e], dot);
      }
      dot += __shfl_xor(dot, 32);
      if (key > r.seen) continue;
      const float x = dot * p.scale_log2;
      const float mn = fmaxf(m, x);
      const float a = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
      const float w = x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - mn);
      l = l * a + w;
      m = mn;
#pragma unroll
      for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
        for (int x4 = 0; x4 < 4; ++x4)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            r.o[ht][4 * x4 + e] =
                r.o[ht][4 * x4 + e] * a + w * tm_load1<DT>(vr, 32 * ht + 8 * x4 + e);
    }
  }
  r.m = m;
  r.l = half == 0 ? l : 0.0f;
}

// The wave's rows as the output, or as a partial of a tile of `tile_rows`: 32 rows as
// they lie in the registers, [HD / 8][64 lanes][4], 1024 bytes a store.
template <int DT, int HD>
__device__ __forceinline__ void end_rows(const PromptParams& p, const Item& it, int kvhead,
                                         int tile_rows, const Place& at, const Rows<HD>& r) {
  const int half = (int)(threadIdx.x & 63) >> 5;
  const float l = r.l + __shfl_xor(r.l, 32);
  if (!at.ok) return;
  if (it.slot < 0) {
    const float inv = l > 0.0f ? 1.0f / l : l;  // 0 where nothing was seen; NaN stays
    const int token = at.row / p.group;
    uint16_t* const o = p.out + (int64_t)(it.q0 + token) * p.out_stride +
                        (int64_t)(kvhead * p.group + at.row - token * p.group) * HD + 4 * half;
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        u32x2_t w;
        w.x = tm_pack2<DT>(r.o[ht][4 * x] * inv, r.o[ht][4 * x + 1] * inv);
        w.y = tm_pack2<DT>(r.o[ht][4 * x + 2] * inv, r.o[ht][4 * x + 3] * inv);
        *reinterpret_cast<u32x2_t*>(o + 32 * ht + 8 * x) = w;
      }
  } else {
    const int64_t slot =
        ((int64_t)it.slot * p.kvh + kvhead) * tile_rows + (at.row - it.tile * tile_rows);
    const int lane = threadIdx.x & 63;
    f32x4_t* const o = reinterpret_cast<f32x4_t*>(p.part + (slot - (lane & 31)) * HD) + lane;
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        o[64 * (4 * ht + x)] =
            f32x4_t{r.o[ht][4 * x], r.o[ht][4 * x + 1], r.o[ht][4 * x + 2], r.o[ht][4 * x + 3]};
    if (half == 0) {
      p.stats[slot * 2] = r.m;
      p.stats[slot * 2 + 1] = l;
    }
  }
}

// The end of a turn: no wave of the workgroup goes on before all have come here.  What
// a turn read from LDS its products have used, so no reads are waited for.
__device__ __forceinline__ void turn_end() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

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
      weigh<DT, HD>(scale_log2, kb, kb + kKeys - 1 > full, r);
      await(s + 1);
      turn_end();
      products<DT, HD, true, true>(vc, kc, r);
      request(s + 3, kn, vn);
      turn_end();
    };
    auto late = [&](int s, uint8_t* kc, uint8_t* vc, uint8_t* kn, uint8_t* vn) TM_INLINE {
      const int kb = it.begin + s * kKeys;
      weigh<DT, HD>(scale_log2, kb, kb + kKeys - 1 > full, r);
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
  retake<DT, HD, PAGED>(p, it, kvhead, 0, 1, n, r);
  end_rows<DT, HD>(p, it, kvhead, 256, at, r);
}

// The same turns on tiles of 128 rows: waves w and w + 4 have the same 32 rows, waves 0-3
// take the even stages and waves 4-7 the odd ones, each four with buffers of their own.
// At the end the two outputs of a row are joined through LDS.
template <int DT, int HD, bool PAGED>
__global__ void __launch_bounds__(512, 2) tm_prompt_pair_kernel(PromptParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_ka0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_va0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_ka1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_va1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_kb0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_vb0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_kb1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_vb1[S::kTile];
  __shared__ float s_stat[4][64][2];

  const int kvhead = (int)blockIdx.x % p.kvh;
  const Item it = item_of(p, (int)blockIdx.x / p.kvh, 128);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int second = wave >> 2;
  Rows<HD> r;
  const Place at = begin_rows<HD>(p, it, kvhead, it.tile * 128 + (wave & 3) * 32, r);
  const int full = at.full;
  const int n = it.end > it.begin ? (it.end - it.begin + kKeys - 1) / kKeys : 0;
  // stages of the first four waves; the last of the second four may lie past the range,
  // all of it masked
  const int rounds = (n + 1) / 2;
  const float scale_log2 = p.scale_log2;
  if (n > 0) {
    Feed<HD, PAGED, 4> feed;
    const int begin = it.begin + second * kKeys;
    feed.start(p, it, kvhead, begin, 2 * kKeys);
    // Load group g(s), in slot s % 2: K of round s and V of round s - 1, what the products
    // M(s) = {O += V P of s - 1, S = K Q of s} read.  Round s: W(s) weighs its scores, then
    // M(s + 1), and behind it g(s + 2) is requested, whose slot all four waves left with
    // M(s) two turns before; W(s) waits for g(s + 1) at its end.  The second four waves do
    // all this one turn later.
    auto request = [&](int s, uint8_t* kn, uint8_t* vn) TM_INLINE {
      if (s > rounds) return;
      if (s > 0) feed.load_v(p, vn);
      if (s < rounds) feed.load_k(p, kn);
    };
    // W(s), M(s + 1) with g(s + 1) at kc, vc; g(s + 2) goes to kn, vn.  (The last one's
    // scores, of a stage that is not there, are not used.)
    auto round = [&](int s, uint8_t* kc, uint8_t* vc, uint8_t* kn, uint8_t* vn) TM_INLINE {
      const int kb = begin + 2 * s * kKeys;
      weigh<DT, HD>(scale_log2, kb, kb + kKeys - 1 > full, r);
      wait_vm<0>();
      turn_end();
      products<DT, HD, true, true>(vc, kc, r);
      request(s + 2, kn, vn);
      turn_end();
    };
    auto all = [&](uint8_t* ka, uint8_t* va, uint8_t* kb, uint8_t* vb) TM_INLINE {
      request(0, ka, va);
      request(1, kb, vb);
      wait_vm<0>();
      turn_end();
      if (second) turn_end();
      products<DT, HD, false, true>(va, ka, r);
      turn_end();
      int s = 0;
      for (; s + 2 <= rounds; s += 2) {
        round(s, kb, vb, ka, va);
        round(s + 1, ka, va, kb, vb);
      }
      if (s < rounds) round(s, kb, vb, ka, va);
    };
    if (second) {
      all(s_kb0, s_vb0, s_kb1, s_vb1);
    } else {
      all(s_ka0, s_va0, s_ka1, s_va1);
      turn_end();
    }
  }
  retake<DT, HD, PAGED>(p, it, kvhead, second, 2, n, r);
  // the second four waves' outputs, each where a buffer was
  const int w4 = wave & 3;
  uint8_t* const box = w4 == 0 ? s_ka0 : w4 == 1 ? s_ka1 : w4 == 2 ? s_va0 : s_va1;
  f32x4_t* const mine = reinterpret_cast<f32x4_t*>(box) + lane;
  __syncthreads();
  if (second) {
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        mine[64 * (4 * ht + x)] =
            f32x4_t{r.o[ht][4 * x], r.o[ht][4 * x + 1], r.o[ht][4 * x + 2], r.o[ht][4 * x + 3]};
    s_stat[w4][lane][0] = r.m;
    s_stat[w4][lane][1] = r.l;
  }
  __syncthreads();
  if (second) return;
  const float m1 = s_stat[w4][lane][0], l1 = s_stat[w4][lane][1];
  const float m = fmaxf(r.m, m1), ref = m == -INFINITY ? 0.0f : m;
  const float a = __builtin_amdgcn_exp2f(r.m - ref), b = __builtin_amdgcn_exp2f(m1 - ref);
  r.l = r.l * a + l1 * b;
  r.m = m;
#pragma unroll
  for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const f32x4_t o = mine[64 * (4 * ht + x)];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.o[ht][4 * x + e] = r.o[ht][4 * x + e] * a + o[e] * b;
    }
  end_rows<DT, HD>(p, it, kvhead, 128, at, r);
}

// Short tiles: four waves of 32 rows, two workgroups a CU, which drift apart by themselves.
template <int DT, int HD, bool PAGED>
__global__ void __launch_bounds__(kThreads, 2) tm_prompt_short_kernel(PromptParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v1[S::kTile];

  const int kvhead = (int)blockIdx.x % p.kvh;
  const Item it = item_of(p, (int)blockIdx.x / p.kvh, 128);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int n = it.end > it.begin ? (it.end - it.begin + kKeys - 1) / kKeys : 0;
  const float scale_log2 = p.scale_log2;
  Rows<HD> r;
  const Place at = begin_rows<HD>(p, it, kvhead, it.tile * 128 + wave * 32, r);
  const int full = at.full;
  if (n > 0) {
    Feed<HD, PAGED, 4> feed;
    feed.start(p, it, kvhead, it.begin, kKeys);
    auto step = [&](int s, const uint8_t* kc, const uint8_t* vc, uint8_t* kn, uint8_t* vn) TM_INLINE {
      wait_vm<0>();      // this wave's loads of stage s
      tm_lds_barrier();  // everyone's; and the reads of stage s - 1 are over
      const int kb = it.begin + s * kKeys;
      if (s + 1 < n) {
        feed.load_k(p, kn);
        feed.load_v(p, vn);
      }
      products<DT, HD, false, true>(vc, kc, r);
      weigh<DT, HD>(scale_log2, kb, kb + kKeys - 1 > full, r);
      products<DT, HD, true, false>(vc, kc, r);
    };
    feed.load_k(p, s_k0);
    feed.load_v(p, s_v0);
    for (int s = 0; s < n; s += 2) {
      step(s, s_k0, s_v0, s_k1, s_v1);
      if (s + 1 < n) step(s + 1, s_k1, s_v1, s_k0, s_v0);
    }
  }
  retake<DT, HD, PAGED>(p, it, kvhead, 0, 1, n, r);
  end_rows<DT, HD>(p, it, kvhead, 128, at, r);
}

// Few rows (a decoded token's heads): a tile of 32, and the four waves take the stages
// of the range in turn, each with its own part of LDS and no barrier between them, so
// that a CU has 128 KB of keys under way.  A wave asks for its next K when it has the
// scores, for its next V when it has the products.  At the end the waves' outputs are
// joined through LDS.
template <int DT, int HD, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) tm_prompt_few_kernel(PromptParams p) {
  typedef Shape<HD> S;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k[4][S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v[4][S::kTile];
  __shared__ float s_stat[4][32][2];

  const int kvhead = (int)blockIdx.x % p.kvh;
  const Item it = item_of(p, (int)blockIdx.x / p.kvh, 32);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int all_rows = it.q_len * p.group;

  // row c32 of the tile, in every wave
  const int first = it.tile * 32;
  Rows<HD> r;
  const int n = it.end > it.begin ? (it.end - it.begin + kKeys - 1) / kKeys : 0;
  Feed<HD, PAGED, 1> feed;
  constexpr int kLoads = Feed<HD, PAGED, 1>::kLoads;
  uint8_t* const kt = s_k[wave];
  uint8_t* const vt = s_v[wave];
  if (wave < n) {
    feed.start(p, it, kvhead, it.begin + wave * kKeys, 4 * kKeys);
    feed.load_k(p, kt);
    feed.load_v(p, vt);
  }
  const int full = begin_rows<HD>(p, it, kvhead, first, r).full;

  for (int s = wave; s < n; s += 4) {
    const int kb = it.begin + s * kKeys;
    const bool more = s + 4 < n;
    if (s == wave)
      wait_vm<0>();  // K and V, and the query rows
    else
      wait_vm<kLoads>();  // K: V is behind it
    products<DT, HD, false, true>(vt, kt, r);
    __builtin_amdgcn_sched_barrier(0);
    if (more) feed.load_k(p, kt);
    weigh<DT, HD>(p.scale_log2, kb, kb + kKeys - 1 > full, r);
    if (more)
      wait_vm<kLoads>();
    else
      wait_vm<0>();
    products<DT, HD, true, false>(vt, kt, r);
    __builtin_amdgcn_sched_barrier(0);
    if (more) feed.load_v(p, vt);
  }
  retake<DT, HD, PAGED>(p, it, kvhead, wave, 4, n, r);
  const float l = r.l + __shfl_xor(r.l, 32);

  // each wave's O [32][HD] where its K was
  float* const mine = reinterpret_cast<float*>(kt) + c32 * HD + 4 * half;
#pragma unroll
  for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<f32x4_t*>(mine + 32 * ht + 8 * x) =
          f32x4_t{r.o[ht][4 * x], r.o[ht][4 * x + 1], r.o[ht][4 * x + 2], r.o[ht][4 * x + 3]};
  if (half == 0) {
    s_stat[wave][c32][0] = r.m;
    s_stat[wave][c32][1] = l;
  }
  __syncthreads();
  constexpr int kLanes = HD / 4;  // of a row, four elements each
  for (int row = tid / kLanes; row < 32; row += kThreads / kLanes) {
    if (first + row >= all_rows) break;
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, s_stat[w][row][0]);
    const float ref = m == -INFINITY ? 0.0f : m;
    f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = __builtin_amdgcn_exp2f(s_stat[w][row][0] - ref);
      sum += s_stat[w][row][1] * a;
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(
          reinterpret_cast<const float*>(s_k[w]) + row * HD + 4 * (tid % kLanes));
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += x[e] * a;
    }
    if (it.slot < 0) {
      store_row<DT>(p, it.q0, first + row, kvhead, HD, 4 * (tid % kLanes), o, sum);
    } else {
      const int64_t slot = ((int64_t)it.slot * p.kvh + kvhead) * 32 + row;
      *reinterpret_cast<f32x4_t*>(p.part + slot * HD + 4 * (tid % kLanes)) = o;
      if (tid % kLanes == 0) {
        p.stats[slot * 2] = m;
        p.stats[slot * 2 + 1] = sum;
      }
    }
  }
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
  p.scale_log2 = scale * 1.4426950408889634f;
  launch<true>(p, dtype, hd, o.kind, o.tiles * o.chunks * kvh, o.chunks > 1 ? o.tiles : 0,
               std::min(o.rows, T * p.group), (hipStream_t)stream);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}
