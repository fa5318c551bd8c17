// Eight consecutive elements of a 16- or 32-bit floating type, as floats.
#pragma once

#include "tm_common.h"

template <int DT>
__device__ __forceinline__ float tm_load1(const void* p, int64_t i) {
  if constexpr (DT == TM_DTYPE_F32)
    return reinterpret_cast<const float*>(p)[i];
  else
    return Half16<DT>::to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

template <int DT>
__device__ __forceinline__ void tm_store1(void* p, int64_t i, float f) {
  if constexpr (DT == TM_DTYPE_F32)
    reinterpret_cast<float*>(p)[i] = f;
  else
    reinterpret_cast<uint16_t*>(p)[i] = Half16<DT>::round(f);
}

// Elements i .. i + 7; the address 16-byte aligned.
template <int DT>
__device__ __forceinline__ void tm_load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (DT == TM_DTYPE_F32) {
    const f32x4_t* q = reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(p) + i);
    const f32x4_t a = q[0], b = q[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  } else {
    const u32x4_t a =
        *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = Half16<DT>::to_f32((uint16_t)(a[j] & 0xffffu));
      v[2 * j + 1] = Half16<DT>::to_f32((uint16_t)(a[j] >> 16));
    }
  }
}

// Two floats as two 16-bit elements, rounded to nearest even in one conversion.
template <int DT>
__device__ __forceinline__ uint32_t tm_pack2(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {lo, hi};
  if constexpr (DT == TM_DTYPE_F16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  }
}

template <int DT>
__device__ __forceinline__ void tm_store8(void* p, int64_t i, const float (&v)[8]) {
  if constexpr (DT == TM_DTYPE_F32) {
    f32x4_t* q = reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(p) + i);
    q[0] = f32x4_t{v[0], v[1], v[2], v[3]};
    q[1] = f32x4_t{v[4], v[5], v[6], v[7]};
  } else {
    u32x4_t a;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = tm_pack2<DT>(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(p) + i) = a;
  }
}

// Bytes of one element.
inline int64_t tm_dtype_bytes(int dt) { return dt == TM_DTYPE_F32 ? 4 : 2; }
inline bool tm_dtype_ok(int dt) {
  return dt == TM_DTYPE_F32 || dt == TM_DTYPE_BF16 || dt == TM_DTYPE_F16;
}
