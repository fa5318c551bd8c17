// Rotary positions.  Pair (a, b) of a head at frequency f_i (turns a position)
// becomes, with t = position * f_i,
//
//   a' = m (a cos 2 pi t - b sin 2 pi t),  b' = m (b cos 2 pi t + a sin 2 pi t).
//
// Pair i of a head's first `part` elements is (i, i + part / 2) in the half
// layout and (2 i, 2 i + 1) in the interleaved one; elements from `part` on are
// copied.
//
// The angle.  f_i comes as a 64-bit fixed-point fraction of a turn, F = f 2^64.  The
// integer product position * F wraps at whole turns, so its 64 bits are the angle
// mod 1 turn, off by |position| 2^-65 turns for F's rounding and |position| f 2^-52 for that
// of the frequency, a double (2^-49 where `part` is no power of two: 2 i / part is rounded
// too): no table of cosines is read and none limits the position.  The top two bits after
// rounding to the nearest quarter turn pick the quadrant, the rest is a remainder of at most
// 1/8 turn, cut to 2^-34 turn (all in all under 2^-33 up to position 2^20, 2^-24 at 2^30; for
// other parts to 2^17, and 2^-21), whose sine and cosine come from their Taylor polynomials in
// fp32 (degree 9 and 10 on |x| <= pi / 4: truncation below 2e-9).
//
// Bound by HBM at many tokens, by the launch at few.  A thread owns 8 pairs, two
// 16-byte pieces, of the same place in several heads of one token, so its 8 sines
// and cosines (about 250 instructions) serve all of them.  Measured (bf16, 32 + 8 heads of
// 128): 5003 tokens rotated and appended, 123 MB from a cold cache, 24.5 us, 5.0 TB/s of the
// 4.9 that a large copy reaches; 64 tokens 3.0 us of kernel.
#include "tm_vec.h"

namespace {

struct RotaryParams {
  const void *q, *k, *v;       // [T, heads, hd], heads contiguous
  void *q_out, *k_out;
  void *k_cache, *v_cache;     // append: this layer's [pages, page, kvh, hd]
  const int32_t* table;
  const void* positions;       // int32 or int64; NULL: start + token
  const uint64_t* turns;       // part / 2 fractions of a turn a position
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  int64_t stride_page, stride_slot, start;
  int tokens, q_heads, kv_heads, heads;  // heads: rows of a token (q, k, and v when appending)
  int slots;                   // threads of a token = slots * units
  int units;                   // hd / 16
  int hd, part, page_size, table_pages, cache_pages, long_positions;
  float magnitude;
};

// sin and cos of 2 pi u / 2^64.
__device__ __forceinline__ void sincos_turns(uint64_t u, float& sn, float& cs) {
  const uint32_t hi = (uint32_t)(u >> 32);
  const uint32_t quad = (hi + 0x20000000u) >> 30;
  // remainder in [-1/8, 1/8) turn, from all 64 bits
  const int64_t rem = (int64_t)(u - ((uint64_t)quad << 62));
  const float x = (float)(int32_t)(rem >> 30) * (6.283185307179586f / 17179869184.0f);
  const float z = x * x;
  float s = fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
  s = fmaf(s, z, 8.33333333e-3f);
  s = fmaf(s, z, -1.66666667e-1f);
  s = fmaf(s * z, x, x);
  float c = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
  c = fmaf(c, z, -1.38888889e-3f);
  c = fmaf(c, z, 4.16666667e-2f);
  c = fmaf(c, z, -0.5f);
  c = fmaf(c, z, 1.0f);
  const bool swap = (quad & 1u) != 0;
  const float a = swap ? c : s, b = swap ? s : c;
  sn = (quad & 2u) ? -a : a;
  cs = ((quad + 1u) & 2u) ? -b : b;
}

template <int DT, bool INTER, bool APPEND>
__global__ void __launch_bounds__(256) tm_rotary_kernel(RotaryParams p) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = p.slots * p.units;
  const int64_t token = gid / per;
  if (token >= p.tokens) return;
  const int within = (int)(gid - token * per);
  const int slot = within / p.units, unit = within - slot * p.units;

  int64_t pos = p.start + token;
  if (p.positions != nullptr)
    pos = p.long_positions ? reinterpret_cast<const int64_t*>(p.positions)[token]
                           : (int64_t)reinterpret_cast<const int32_t*>(p.positions)[token];
  // the unit's two pieces of 8 elements
  const bool rot = unit * 16 < p.part;
  const int lo = INTER || !rot ? unit * 16 : unit * 8;
  const int hi = INTER || !rot ? lo + 8 : lo + p.part / 2;
  float sn[8], cs[8];
  if (rot) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sincos_turns((uint64_t)pos * p.turns[unit * 8 + e], sn[e], cs[e]);
      sn[e] *= p.magnitude;
      cs[e] *= p.magnitude;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sn[e] = 0.0f;
      cs[e] = 1.0f;
    }
  }
  int64_t row_at = -1;  // the token's row in the cache, or none
  if constexpr (APPEND) {
    const int64_t pidx = pos / p.page_size;
    if (pos >= 0 && pidx < p.table_pages) {
      const int page = p.table[pidx];
      if (page >= 0 && page < p.cache_pages)
        row_at = (int64_t)page * p.stride_page + (pos - pidx * p.page_size) * p.stride_slot;
    }
  }
  for (int h = slot; h < p.heads; h += p.slots) {
    const void* src;
    void* dst;
    int64_t from, to;
    bool turn = rot, keep = true;
    if (h < p.q_heads) {
      src = p.q;
      dst = p.q_out;
      from = token * p.q_stride + (int64_t)h * p.hd;
      to = token * p.q_out_stride + (int64_t)h * p.hd;
    } else if (h < p.q_heads + p.kv_heads) {
      const int64_t at = (int64_t)(h - p.q_heads) * p.hd;
      src = p.k;
      from = token * p.k_stride + at;
      dst = APPEND ? p.k_cache : p.k_out;
      to = APPEND ? row_at + at : token * p.k_out_stride + at;
      keep = !APPEND || row_at >= 0;
    } else {
      const int64_t at = (int64_t)(h - p.q_heads - p.kv_heads) * p.hd;
      src = p.v;
      from = token * p.v_stride + at;
      dst = p.v_cache;
      to = row_at + at;
      turn = false;
      keep = row_at >= 0;
    }
    if (!keep) continue;
    float a[8], b[8];
    if (!turn) {
      // the same 16 elements whatever the layout of the pairs
      tm_load8<DT>(src, from + unit * 16, a);
      tm_load8<DT>(src, from + unit * 16 + 8, b);
      tm_store8<DT>(dst, to + unit * 16, a);
      tm_store8<DT>(dst, to + unit * 16 + 8, b);
      continue;
    }
    tm_load8<DT>(src, from + lo, a);
    tm_load8<DT>(src, from + hi, b);
    float u[8], w[8];
    if constexpr (INTER) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u[2 * j] = a[2 * j] * cs[j] - a[2 * j + 1] * sn[j];
        u[2 * j + 1] = a[2 * j + 1] * cs[j] + a[2 * j] * sn[j];
        w[2 * j] = b[2 * j] * cs[4 + j] - b[2 * j + 1] * sn[4 + j];
        w[2 * j + 1] = b[2 * j + 1] * cs[4 + j] + b[2 * j] * sn[4 + j];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[e] = a[e] * cs[e] - b[e] * sn[e];
        w[e] = b[e] * cs[e] + a[e] * sn[e];
      }
    }
    tm_store8<DT>(dst, to + lo, u);
    tm_store8<DT>(dst, to + hi, w);
  }
}

template <bool APPEND>
int launch(const RotaryParams& p, int dtype, bool inter, hipStream_t st) {
  const int64_t threads = (int64_t)p.tokens * p.slots * p.units;
  const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
#define TM_ROT(DT)                                                                         \
  if (inter)                                                                               \
    hipLaunchKernelGGL((tm_rotary_kernel<DT, true, APPEND>), grid, block, 0, st, p);       \
  else                                                                                     \
    hipLaunchKernelGGL((tm_rotary_kernel<DT, false, APPEND>), grid, block, 0, st, p)
  if (dtype == TM_DTYPE_BF16) {
    TM_ROT(TM_DTYPE_BF16);
  } else if (dtype == TM_DTYPE_F16) {
    TM_ROT(TM_DTYPE_F16);
  } else {
    TM_ROT(TM_DTYPE_F32);
  }
#undef TM_ROT
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

// Head slots of a token: one head a thread at few tokens, 16 slots (two or three heads
// each of a token's 40 rows) from 1024 tokens on, where the angles are then a smaller part.
// Measured on one head shape (bf16, 32 + 8 heads of 128), one head, 16 slots and 8 slots in
// us: 64 tokens 3.0, 3.8, 4.7; 512 tokens 4.3, 4.5, 5.4; 1024 5.8, 5.5, 5.9; 2048 9.5, 8.5, 9.3; 5003
// 18.9, 17.8, 17.8.
int head_slots(int64_t tokens, int heads) {
  return tokens < 1024 ? heads : (heads < 16 ? heads : 16);
}

int check(int64_t T, int64_t hd, int64_t part, int64_t q_heads, int64_t kv_heads, int dtype) {
  if (!tm_dtype_ok(dtype)) return TM_ERR_ARG;
  if (T < 0 || T > TM_MAX_ROWS || hd < 16 || hd > 1024 || hd % 16 != 0 || part < 16 || part > hd ||
      part % 16 != 0 || q_heads < 0 || kv_heads < 0 || q_heads > 1024 || kv_heads > 1024)
    return TM_ERR_SHAPE;
  return TM_OK;
}

// Every token starts on 16 bytes (one token has no stride).
bool vec_ok(const void* p, int64_t stride, int64_t es, int64_t tokens) {
  return (uintptr_t)p % 16 == 0 && (tokens == 1 || stride * es % 16 == 0);
}

}  // namespace

extern "C" int tm_rotary(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                         void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride,
                         const void* positions, int long_positions, const uint64_t* turns,
                         float magnitude, int64_t T, int64_t q_heads, int64_t kv_heads,
                         int64_t hd, int64_t part, int interleaved, int dtype, void* stream) {
  int rc = check(T, hd, part, q_heads, kv_heads, dtype);
  if (rc) return rc;
  if (T == 0 || q_heads + kv_heads == 0) return TM_OK;
  const int64_t es = tm_dtype_bytes(dtype);
  if (q_heads && T > 1 && (q_stride < q_heads * hd || q_out_stride < q_heads * hd))
    return TM_ERR_SHAPE;
  if (kv_heads && T > 1 && (k_stride < kv_heads * hd || k_out_stride < kv_heads * hd))
    return TM_ERR_SHAPE;
  if ((q_heads && (!vec_ok(q, q_stride, es, T) || !vec_ok(q_out, q_out_stride, es, T))) ||
      (kv_heads && (!vec_ok(k, k_stride, es, T) || !vec_ok(k_out, k_out_stride, es, T))) ||
      (uintptr_t)turns % 8 || (uintptr_t)positions % (long_positions ? 8 : 4))
    return TM_ERR_ALIGN;
  RotaryParams p = {};
  p.q = q;
  p.k = k;
  p.q_out = q_out;
  p.k_out = k_out;
  p.positions = positions;
  p.turns = turns;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.q_out_stride = q_out_stride;
  p.k_out_stride = k_out_stride;
  p.tokens = (int)T;
  p.q_heads = (int)q_heads;
  p.kv_heads = (int)kv_heads;
  p.heads = (int)(q_heads + kv_heads);
  p.units = (int)(hd / 16);
  p.slots = head_slots(T, p.heads);
  p.hd = (int)hd;
  p.part = (int)part;
  p.long_positions = long_positions ? 1 : 0;
  p.magnitude = magnitude;
  return launch<false>(p, dtype, interleaved != 0, (hipStream_t)stream);
}

extern "C" int tm_rotary_append(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                const void* v, int64_t v_stride, void* q_out,
                                int64_t q_out_stride, void* k_cache, void* v_cache,
                                int64_t stride_page, int64_t stride_slot, int64_t page_size,
                                int64_t cache_pages, const int32_t* block_table,
                                int64_t num_table_pages, int64_t start_pos,
                                const uint64_t* turns, float magnitude, int64_t T,
                                int64_t q_heads, int64_t kv_heads, int64_t hd, int64_t part,
                                int interleaved, int dtype, void* stream) {
  int rc = check(T, hd, part, q_heads, kv_heads, dtype);
  if (rc) return rc;
  if (kv_heads < 1 || page_size < 1 || page_size > (1 << 24) || cache_pages < 0 ||
      cache_pages > INT32_MAX || num_table_pages < 0 || num_table_pages > INT32_MAX ||
      start_pos < 0 || start_pos > (1 << 30))
    return TM_ERR_SHAPE;
  if (T == 0) return TM_OK;
  if ((start_pos + T - 1) / page_size >= num_table_pages) return TM_ERR_SHAPE;
  if (stride_slot < kv_heads * hd || stride_page < page_size * stride_slot) return TM_ERR_SHAPE;
  if (T > 1 && (k_stride < kv_heads * hd || v_stride < kv_heads * hd ||
                (q_heads && (q_stride < q_heads * hd || q_out_stride < q_heads * hd))))
    return TM_ERR_SHAPE;
  const int64_t es = tm_dtype_bytes(dtype);
  if ((q_heads && (!vec_ok(q, q_stride, es, T) || !vec_ok(q_out, q_out_stride, es, T))) ||
      !vec_ok(k, k_stride, es, T) || !vec_ok(v, v_stride, es, T) ||
      !vec_ok(k_cache, stride_page, es, 2) || !vec_ok(v_cache, stride_slot, es, 2) ||
      (uintptr_t)turns % 8 || (uintptr_t)block_table % 4)
    return TM_ERR_ALIGN;
  RotaryParams p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_out = q_out;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.table = block_table;
  p.turns = turns;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.q_out_stride = q_out_stride;
  p.stride_page = stride_page;
  p.stride_slot = stride_slot;
  p.start = start_pos;
  p.tokens = (int)T;
  p.q_heads = (int)q_heads;
  p.kv_heads = (int)kv_heads;
  p.heads = (int)(q_heads + 2 * kv_heads);
  p.units = (int)(hd / 16);
  p.slots = head_slots(T, p.heads);
  p.hd = (int)hd;
  p.part = (int)part;
  p.page_size = (int)page_size;
  p.table_pages = (int)num_table_pages;
  p.cache_pages = (int)cache_pages;
  p.magnitude = magnitude;
  return launch<true>(p, dtype, interleaved != 0, (hipStream_t)stream);
}
