// Causal attention of a prompt's tokens, down to a single one, over packed sequences
// or over one sequence's pages of the KV cache:
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / group]) v[j, h / group],
//
// j over the sequence's keys 0 .. past + t, where past = its keys minus its queries.
//
// Decomposition.  The rows of a KV head are its sequence's (token, head of the group)
// pairs, token major, so neighbouring rows share every key and the causal border
// crosses a tile of 128 rows within 128 / group tokens.  A workgroup of 4 waves takes
// 128 QT such rows against one range of keys, 64 keys a stage; K and V rows go
// straight from memory to LDS (16 bytes a lane, no registers between), V transposed
// as it is read from there.  Few rows over many keys are split over key ranges; each
// leaves its sum, maximum and unnormalised output in fp32 in the workspace, which a
// second kernel joins in key order.
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
// The weights are rounded to the inputs' 16-bit type for the product; the sums are
// taken over the rounded weights in fp32, so that the roundings weigh alike above and
// below the division.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <utility>
#include <vector>

#include "tm_vec.h"

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) void glb_void;

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
  float* part;                 // [slot][kvh][tile rows][hd]
  float* stats;                // [slot][kvh][tile rows][2]
  int64_t q_stride, k_stride, v_stride, out_stride;  // paged: k_stride is the slot's
  int64_t stride_page;
  int kvh, group, q_len, k_len, tiles, chunks, chunk_len;  // one sequence's
  int page_shift, table_pages, cache_pages;
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
  static constexpr int kLoads = kTile / 4096;      // loads of a wave per stage and operand
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

// Keys kb .. kb + 63 of K and V into LDS.  Keys at or past the last are that of the
// last one: their scores are masked.
template <int HD, bool PAGED>
struct Loader {
  typedef Shape<HD> S;
  const uint16_t* k;
  const uint16_t* v;
  int last;          // the sequence's last key
  int page_of[S::kLoads];  // pages of the next stage's keys (paged)

  __device__ __forceinline__ int key_in(int i) const {  // within the stage
    return ((int)(threadIdx.x >> 6) * S::kLoads + i) * S::kKeysPerLoad +
           (int)(threadIdx.x & 63) / S::kChunks;
  }
  __device__ __forceinline__ void look_up(const PromptParams& p, int kb) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i)
        page_of[i] = p.table[min(kb + key_in(i), last) >> p.page_shift];
    }
  }
  __device__ __forceinline__ void load(const PromptParams& p, int kb, uint8_t* kt, uint8_t* vt) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int chunk = (int)threadIdx.x & (S::kChunks - 1);
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int j = key_in(i);
      const int key = min(kb + j, last);
      int64_t ko, vo;
      if constexpr (PAGED) {
        const int page = min(max(page_of[i], 0), p.cache_pages - 1);
        ko = (int64_t)page * p.stride_page +
             (int64_t)(key & ((1 << p.page_shift) - 1)) * p.k_stride;
        vo = ko;
      } else {
        ko = (int64_t)key * p.k_stride;
        vo = (int64_t)key * p.v_stride;
      }
      const int at = (wave * S::kLoads + i) * 1024;
      __builtin_amdgcn_global_load_lds((glb_void*)(k + ko + (chunk ^ S::swz_k(j)) * 8),
                                       (lds_void*)(kt + at), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((glb_void*)(v + vo + (chunk ^ S::swz_v(j)) * 8),
                                       (lds_void*)(vt + at), 16, 0, 0);
    }
  }
};

__device__ __forceinline__ u32x2_t read_tr(const uint8_t* p) {
  return __builtin_bit_cast(
      u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) s16x4_t*)(lds_void*)const_cast<uint8_t*>(p)));
}

// V^T fragment of head-dim tile ht for the 16 keys from `key` on.
template <int HD>
__device__ __forceinline__ u32x4_t v_frag(const uint8_t* vt, int ht, int key, int lane) {
  typedef Shape<HD> S;
  const int i = lane & 15, g = lane >> 4;
  const int k0 = 4 * (g >> 1) + (i >> 2);
  const int chunk = 4 * ht + 2 * (g & 1) + ((i & 3) >> 1);
  const uint8_t* const lo =
      vt + (key + k0) * S::kRow + ((chunk ^ S::swz_v(k0)) * 16) + (i & 1) * 8;
  const uint8_t* const hi =
      vt + (key + k0 + 8) * S::kRow + ((chunk ^ S::swz_v(k0 + 8)) * 16) + (i & 1) * 8;
  const u32x2_t a = read_tr(lo), b = read_tr(hi);
  return u32x4_t{a.x, a.y, b.x, b.y};
}

// Softmax state and output of one tile of 32 rows (a lane's column is one row).
template <int HD>
struct RowTile {
  u32x4_t q[HD / 16];
  f32x16_t o[HD / 32];
  float m, l;     // reference maximum (base 2), and this lane's part of the sum
  int seen;       // the row's last visible key
};

// Keys kb .. of the stage at kt / vt against QT row tiles.
template <int DT, int HD, int QT, bool MASK>
__device__ __forceinline__ void attend(const PromptParams& p, const uint8_t* kt_, const uint8_t* vt,
                                       int kb, RowTile<HD> (&rt)[QT]) {
  typedef Shape<HD> S;
  const int lane = threadIdx.x & 63, half = lane >> 5, c32 = lane & 31;
  f32x16_t sc[QT][2];
#pragma unroll
  for (int t = 0; t < QT; ++t)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int x = 0; x < 16; ++x) sc[t][kt][x] = 0.0f;
  const uint8_t* const krow = kt_ + c32 * S::kRow;
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const u32x4_t a = *reinterpret_cast<const u32x4_t*>(
          krow + 32 * kt * S::kRow + (((2 * ks + half) ^ S::swz_k(c32)) * 16));
#pragma unroll
      for (int t = 0; t < QT; ++t) sc[t][kt] = mfma32<DT>(a, rt[t].q[ks], sc[t][kt]);
    }
  }
  u32x4_t pw[QT][4];  // weights of k-step (kt, m) at 2 kt + m
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if constexpr (MASK) {
      const int left = rt[t].seen - kb - 4 * half;  // keys up to this one are visible
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int x = 0; x < 16; ++x)
          sc[t][kt][x] =
              32 * kt + 8 * (x >> 2) + (x & 3) <= left ? sc[t][kt][x] : -INFINITY;
    }
    float mx = fmaxf(sc[t][0][0], sc[t][1][0]);
#pragma unroll
    for (int x = 1; x < 16; ++x) mx = fmaxf(fmaxf(mx, sc[t][0][x]), sc[t][1][x]);
    const float cand = max_halves(mx) * p.scale_log2;
    const bool bump = cand > rt[t].m + 8.0f;
    if (__any(bump)) {
      const float m = bump ? cand : rt[t].m;
      const float a = bump ? __builtin_amdgcn_exp2f(rt[t].m - m) : 1.0f;
#pragma unroll
      for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
        for (int x = 0; x < 16; ++x) rt[t].o[ht][x] *= a;
      rt[t].l *= a;
      rt[t].m = m;
    }
    const float base = rt[t].m == -INFINITY ? 0.0f : -rt[t].m;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e0 = __builtin_amdgcn_exp2f(
              fmaf(sc[t][kt][8 * m + 2 * j], p.scale_log2, base));
          const float e1 = __builtin_amdgcn_exp2f(
              fmaf(sc[t][kt][8 * m + 2 * j + 1], p.scale_log2, base));
          const uint32_t w = tm_pack2<DT>(e0, e1);
          rt[t].l = add_pair<DT>(w, rt[t].l);
          pw[t][2 * kt + m][j] = w;
        }
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht) {
      const u32x4_t a = v_frag<HD>(vt, ht, 16 * s, lane);
#pragma unroll
      for (int t = 0; t < QT; ++t) rt[t].o[ht] = mfma32<DT>(a, pw[t][s], rt[t].o[ht]);
    }
  }
}

template <int DT, int HD, int QT, bool PAGED>
__global__ void __launch_bounds__(kThreads, QT == 1 ? 2 : 1) tm_prompt_attn_kernel(PromptParams p) {
  typedef Shape<HD> S;
  constexpr int kRows = 128 * QT;
  __shared__ __attribute__((aligned(1024))) uint8_t s_k0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v0[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_k1[S::kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t s_v1[S::kTile];

  // KV heads innermost: with 8 of them a head's workgroups, which share its keys, run
  // on one XCD; the tiles with the most keys first
  const int kvhead = (int)blockIdx.x % p.kvh;
  const int at = (int)blockIdx.x / p.kvh;
  Item it;
  if (p.items != nullptr) {
    it = p.items[at];
  } else {
    it.q0 = it.k0 = 0;
    it.q_len = p.q_len;
    it.k_len = p.k_len;
    it.tile = p.tiles - 1 - at / p.chunks;
    const int chunk = at % p.chunks;
    const int last_token = min(it.q_len - 1, (it.tile * kRows + kRows - 1) / p.group);
    const int keys = it.k_len - it.q_len + last_token + 1;
    it.begin = chunk * p.chunk_len;
    it.end = min(it.begin + p.chunk_len, keys);
    it.slot = p.chunks > 1 ? it.tile * p.chunks + chunk : -1;
  }
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int past = it.k_len - it.q_len;
  const int all_rows = it.q_len * p.group;

  // this lane's rows: column c32 of each of the wave's tiles
  RowTile<HD> rt[QT];
  int64_t qat[QT];   // element offset of the row's head in q, or -1
  int wave_seen = -1;  // the last key that any row of this wave sees
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int first = it.tile * kRows + (wave * QT + t) * 32;
    const int row = first + c32;
    const bool ok = row < all_rows;
    const int token = ok ? row / p.group : 0;
    const int head = kvhead * p.group + (ok ? row - token * p.group : 0);
    const uint16_t* const qr =
        p.q + (int64_t)(it.q0 + token) * p.q_stride + (int64_t)head * HD + 8 * half;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(qr + 16 * ks);
      const u32x4_t zero = {0u, 0u, 0u, 0u};
      rt[t].q[ks] = ok ? x : zero;
    }
#pragma unroll
    for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
      for (int x = 0; x < 16; ++x) rt[t].o[ht][x] = 0.0f;
    rt[t].m = -INFINITY;
    rt[t].l = 0.0f;
    rt[t].seen = ok ? past + token : -1;
    qat[t] = ok ? (int64_t)token * p.group + (head - kvhead * p.group) : -1;
    if (first < all_rows) wave_seen = past + min(it.q_len - 1, (first + 31) / p.group);
  }
  // keys that every row of the wave sees: its first row's
  const int first_row = it.tile * kRows + wave * QT * 32;
  const int wave_full = first_row + QT * 32 <= all_rows ? past + first_row / p.group : -1;

  Loader<HD, PAGED> ld;
  ld.k = p.k + (int64_t)kvhead * HD + (PAGED ? 0 : (int64_t)it.k0 * p.k_stride);
  ld.v = p.v + (int64_t)kvhead * HD + (PAGED ? 0 : (int64_t)it.k0 * p.v_stride);
  ld.last = it.k_len - 1;
  const int stages = it.end > it.begin ? (it.end - it.begin + kKeys - 1) / kKeys : 0;
  if (stages > 0) {
    ld.look_up(p, it.begin);
    ld.load(p, it.begin, s_k0, s_v0);
    ld.look_up(p, it.begin + kKeys);
  }
  // stage s in one pair of buffers while stage s + 1 loads into the other
  auto step = [&](int s, uint8_t* kc, uint8_t* vc, uint8_t* kn, uint8_t* vn) {
    wait_vm<0>();      // this wave's loads of stage s
    tm_lds_barrier();  // everyone's; and the reads of stage s - 1 are over
    const int kb = it.begin + s * kKeys;
    if (s + 1 < stages) {
      ld.load(p, kb + kKeys, kn, vn);
      ld.look_up(p, kb + 2 * kKeys);
    }
    if (kb > wave_seen) return;  // nothing of the stage is visible to this wave
    if (kb + kKeys - 1 <= wave_full && kb + kKeys <= it.end)
      attend<DT, HD, QT, false>(p, kc, vc, kb, rt);
    else
      attend<DT, HD, QT, true>(p, kc, vc, kb, rt);
  };
  // a chunk's border hides what lies past it
#pragma unroll
  for (int t = 0; t < QT; ++t) rt[t].seen = min(rt[t].seen, it.end - 1);
  for (int s = 0; s < stages; s += 2) {
    step(s, s_k0, s_v0, s_k1, s_v1);
    if (s + 1 < stages) step(s + 1, s_k1, s_v1, s_k0, s_v0);
  }

#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float l = rt[t].l + __shfl_xor(rt[t].l, 32);
    if (qat[t] < 0) continue;
    if (it.slot < 0) {
      const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays
      const int token = (int)(qat[t] / p.group), g = (int)(qat[t] - (int64_t)token * p.group);
      uint16_t* const o = p.out + (int64_t)(it.q0 + token) * p.out_stride +
                          (int64_t)(kvhead * p.group + g) * HD + 4 * half;
#pragma unroll
      for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          u32x2_t w;
          w.x = tm_pack2<DT>(rt[t].o[ht][4 * x] * inv, rt[t].o[ht][4 * x + 1] * inv);
          w.y = tm_pack2<DT>(rt[t].o[ht][4 * x + 2] * inv, rt[t].o[ht][4 * x + 3] * inv);
          *reinterpret_cast<u32x2_t*>(o + 32 * ht + 8 * x) = w;
        }
    } else {
      const int r = (wave * QT + t) * 32 + c32;
      const int64_t slot = ((int64_t)it.slot * p.kvh + kvhead) * kRows + r;
      float* const o = p.part + slot * HD + 4 * half;
#pragma unroll
      for (int ht = 0; ht < HD / 32; ++ht)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          *reinterpret_cast<f32x4_t*>(o + 32 * ht + 8 * x) =
              f32x4_t{rt[t].o[ht][4 * x], rt[t].o[ht][4 * x + 1], rt[t].o[ht][4 * x + 2],
                      rt[t].o[ht][4 * x + 3]};
      if (half == 0) {
        p.stats[slot * 2] = rt[t].m;
        p.stats[slot * 2 + 1] = l;
      }
    }
  }
}

// Joins the partials of one row in key order: a wave takes a row of one tile and KV
// head, two elements of the head dimension a lane (hd 128) or one (hd 64).
template <int DT, int HD>
__global__ void __launch_bounds__(kThreads) tm_prompt_join_kernel(PromptParams p, int rows) {
  const int lane = threadIdx.x & 63;
  const int unit = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  const int r = unit % rows;
  const int kv = unit / rows;
  const int kvhead = kv % p.kvh, at = kv / p.kvh;
  Join j;
  if (p.joins != nullptr) {
    j = p.joins[at];
  } else {
    if (at >= p.tiles) return;
    j.q0 = 0;
    j.q_len = p.q_len;
    j.tile = at;
    j.slot0 = at * p.chunks;
    j.count = p.chunks;
  }
  const int64_t row = (int64_t)j.tile * rows + r;
  if (row >= (int64_t)j.q_len * p.group) return;
  constexpr int E = HD / 64;
  float m = -INFINITY, l = 0.0f, o[E] = {};
  for (int c = 0; c < j.count; ++c) {
    const int64_t slot = ((int64_t)(j.slot0 + c) * p.kvh + kvhead) * rows + r;
    const float m1 = p.stats[slot * 2], l1 = p.stats[slot * 2 + 1];
    const float mn = fmaxf(m, m1);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float a = exp2f(m - ref), b = exp2f(m1 - ref);
    l = l * a + l1 * b;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + p.part[slot * HD + lane * E + e] * b;
    m = mn;
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
  const int token = (int)(row / p.group), g = (int)(row - (int64_t)token * p.group);
  uint16_t* const out = p.out + (int64_t)(j.q0 + token) * p.out_stride +
                        (int64_t)(kvhead * p.group + g) * HD + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = Half16<DT>::round(o[e] * inv);
}

// ------------------------------------------------------------------- host --

constexpr int64_t kSlotsPerCU = 2;   // workgroups of 128 rows a CU holds

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Keys of tile `tile` of a sequence: those before the border of its last row.
int64_t tile_keys(int64_t q_len, int64_t k_len, int64_t tile, int64_t rows, int64_t group) {
  const int64_t last = std::min(q_len - 1, (tile * rows + rows - 1) / group);
  return k_len - q_len + last + 1;
}

// Rows of a tile: 128 rows a workgroup of which a CU holds two, or 256 where these
// fill the chip twice over.
int64_t rows_of(int64_t units128) { return units128 >= 4 * kCUs * kSlotsPerCU ? 256 : 128; }

// Key ranges of one sequence's tiles: as many as fill the chip's workgroup slots, at
// least 4 stages each.
int64_t chunks_of(int64_t units, int64_t keys) {
  const int64_t want = kCUs * kSlotsPerCU / std::max<int64_t>(units, 1);
  return std::max<int64_t>(1, std::min(want, ceil_div(keys, 4 * kKeys)));
}

int check_heads(int64_t Hq, int64_t kvh, int64_t hd) {
  if (kvh < 1 || Hq < kvh || Hq % kvh != 0 || Hq > 1024 || (hd != 64 && hd != 128))
    return TM_ERR_SHAPE;
  return TM_OK;
}

struct OnePlan {
  int64_t rows, tiles, chunks, chunk_len, bytes;
};

int plan_one(int64_t T, int64_t S, int64_t Hq, int64_t kvh, int64_t hd, OnePlan* o) {
  const int64_t group = Hq / kvh;
  if (T < 0 || S < T || S > TM_MAX_PROMPT_KEYS || T * group > INT32_MAX - 1024)
    return TM_ERR_SHAPE;
  o->rows = rows_of(ceil_div(T * group, 128) * kvh);
  o->tiles = ceil_div(T * group, o->rows);
  o->chunks = chunks_of(o->tiles * kvh, S);
  o->chunk_len = std::max<int64_t>(kKeys, ceil_div(ceil_div(S, o->chunks), kKeys) * kKeys);
  o->chunks = std::max<int64_t>(1, ceil_div(S, o->chunk_len));
  o->bytes = o->chunks > 1 ? o->tiles * o->chunks * kvh * o->rows * (hd + 2) * 4 : 0;
  return TM_OK;
}

template <int DT, int HD, bool PAGED>
void launch_rows(const PromptParams& p, int64_t rows, int64_t blocks, int64_t joins,
                 hipStream_t st) {
  const dim3 grid((unsigned)blocks), block(kThreads);
  if (rows == 256)
    hipLaunchKernelGGL((tm_prompt_attn_kernel<DT, HD, 2, PAGED>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((tm_prompt_attn_kernel<DT, HD, 1, PAGED>), grid, block, 0, st, p);
  if (joins > 0)
    hipLaunchKernelGGL((tm_prompt_join_kernel<DT, HD>),
                       dim3((unsigned)(joins * p.kvh * rows / 4)), block, 0, st, p, (int)rows);
}

template <bool PAGED>
void launch(const PromptParams& p, int dtype, int64_t hd, int64_t rows, int64_t blocks,
            int64_t joins, hipStream_t st) {
  if (dtype == TM_DTYPE_F16) {
    if (hd == 128)
      launch_rows<TM_DTYPE_F16, 128, PAGED>(p, rows, blocks, joins, st);
    else
      launch_rows<TM_DTYPE_F16, 64, PAGED>(p, rows, blocks, joins, st);
  } else {
    if (hd == 128)
      launch_rows<TM_DTYPE_BF16, 128, PAGED>(p, rows, blocks, joins, st);
    else
      launch_rows<TM_DTYPE_BF16, 64, PAGED>(p, rows, blocks, joins, st);
  }
}

bool vec_ok(const void* p, int64_t stride, int64_t tokens) {
  return (uintptr_t)p % 16 == 0 && (tokens <= 1 || stride % 8 == 0);
}

}  // namespace

extern "C" int tm_prompt_plan(const int64_t* q_lens, const int64_t* k_lens, int64_t B, int64_t Hq,
                              int64_t kvh, int32_t* items, int64_t max_items, int32_t* joins,
                              int64_t max_joins, int64_t* sizes) {
  int rc = check_heads(Hq, kvh, 128);
  if (rc) return rc;
  if (sizes == nullptr || B < 0 || (B > 0 && (q_lens == nullptr || k_lens == nullptr)))
    return TM_ERR_ARG;
  const int64_t group = Hq / kvh;
  int64_t units = 0, q_rows = 0, k_rows = 0;
  for (int64_t b = 0; b < B; ++b) {
    if (q_lens[b] < 0 || k_lens[b] < q_lens[b] || k_lens[b] > TM_MAX_PROMPT_KEYS)
      return TM_ERR_SHAPE;
    q_rows += q_lens[b];
    k_rows += k_lens[b];
    if (q_rows * group > INT32_MAX - 1024 || k_rows > INT32_MAX) return TM_ERR_SHAPE;
    units += ceil_div(q_lens[b] * group, 128) * kvh;
  }
  const int64_t rows = rows_of(units);
  // stages of all workgroups, and how many one of them may have before its keys are
  // split: twice an even share of the chip's slots
  int64_t stages = 0;
  for (int64_t b = 0; b < B; ++b)
    for (int64_t t = 0; t * rows < q_lens[b] * group; ++t)
      stages += ceil_div(tile_keys(q_lens[b], k_lens[b], t, rows, group), kKeys) * kvh;
  const int64_t share = std::max<int64_t>(4, ceil_div(stages, kCUs * kSlotsPerCU));
  std::vector<std::pair<int64_t, Item>> list;  // (keys, item)
  std::vector<Join> jlist;
  int64_t q0 = 0, k0 = 0, slots = 0;
  for (int64_t b = 0; b < B; ++b) {
    for (int64_t t = 0; t * rows < q_lens[b] * group; ++t) {
      const int64_t keys = tile_keys(q_lens[b], k_lens[b], t, rows, group);
      const int64_t n = ceil_div(keys, kKeys);
      const int64_t chunks = n > 2 * share ? ceil_div(n, share) : 1;
      const int64_t len = ceil_div(n, chunks) * kKeys;
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
  sizes[3] = rows;
  sizes[4] = q_rows;
  sizes[5] = k_rows;
  if (items == nullptr && joins == nullptr) return TM_OK;
  if (max_items < sizes[0] || max_joins < sizes[1]) return TM_ERR_SHAPE;
  std::stable_sort(list.begin(), list.end(),
                   [](const auto& a, const auto& b) { return a.first > b.first; });
  for (size_t i = 0; i < list.size(); ++i)
    memcpy(items + 8 * i, &list[i].second, sizeof(Item));
  if (!jlist.empty()) memcpy(joins, jlist.data(), jlist.size() * sizeof(Join));
  return TM_OK;
}

extern "C" int tm_prompt_attention(const void* q, int64_t q_stride, const void* k,
                                   int64_t k_stride, const void* v, int64_t v_stride,
                                   const int32_t* items, int64_t num_items, const int32_t* joins,
                                   int64_t num_joins, int64_t num_slots, int64_t tile_rows,
                                   int64_t Hq, int64_t kvh, int64_t hd, float scale, int dtype,
                                   void* out, int64_t out_stride, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  int rc = check_heads(Hq, kvh, hd);
  if (rc) return rc;
  if ((dtype != TM_DTYPE_BF16 && dtype != TM_DTYPE_F16) || !(scale > 0.0f) || scale == INFINITY)
    return TM_ERR_ARG;
  if ((tile_rows != 128 && tile_rows != 256) || num_items < 0 || num_joins < 0 || num_slots < 0 ||
      num_items * kvh > INT32_MAX || num_joins * kvh * tile_rows / 4 > INT32_MAX ||
      num_slots > INT32_MAX)
    return TM_ERR_SHAPE;
  if (q_stride < Hq * hd || out_stride < Hq * hd || k_stride < kvh * hd || v_stride < kvh * hd)
    return TM_ERR_SHAPE;
  if (num_slots * kvh * tile_rows * (hd + 2) * 4 > workspace_bytes) return TM_ERR_SHAPE;
  if (num_items == 0) return TM_OK;
  if (!vec_ok(q, q_stride, 2) || !vec_ok(k, k_stride, 2) || !vec_ok(v, v_stride, 2) ||
      !vec_ok(out, out_stride, 2) || (uintptr_t)items % 32 || (uintptr_t)joins % 32 ||
      (uintptr_t)workspace % 16)
    return TM_ERR_ALIGN;
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
  launch<false>(p, dtype, hd, tile_rows, num_items * kvh, num_joins, (hipStream_t)stream);
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
      stride_page < page_size * stride_slot)
    return TM_ERR_SHAPE;
  if (o.bytes > workspace_bytes || o.tiles * o.chunks * kvh > INT32_MAX ||
      o.tiles * kvh * o.rows / 4 > INT32_MAX)
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
  p.table_pages = (int)num_table_pages;
  p.cache_pages = (int)cache_pages;
  p.scale_log2 = scale * 1.4426950408889634f;
  launch<true>(p, dtype, hd, o.rows, o.tiles * o.chunks * kvh, o.chunks > 1 ? o.tiles : 0,
               (hipStream_t)stream);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}
