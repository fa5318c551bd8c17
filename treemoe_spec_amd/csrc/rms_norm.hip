// Root-mean-square norm of rows, with the residual's addition and, where asked,
// an output in 8 bits with scales:
//
//   s = x (+ r),  y = s / sqrt(mean(s^2) + eps) * w,  r' = s,
//
// s, the sum of squares and y in fp32, each output rounded once.  The 8-bit
// form scales y by the largest magnitude of a row or of a group of columns:
// scale = amax / 448 (1 where that is 0), q = e4m3(y / scale), 448 being
// e4m3's largest value.
//
// Bound by HBM: every input is read once and every output written once, a
// row staying in registers between the sum and the product.  A thread owns 8
// consecutive elements of every `threads`-th chunk of 8, so a wave's loads are
// whole cache lines; the sum runs over a thread's elements, then an xor fold over
// the lanes, then the waves in order: a fixed order.
//
// Measured in bf16 with a residual of the same type: 6011 rows of 4096, 40 us from a cold
// cache, 4.9 TB/s of the 4.9 TB/s that a 2 GiB copy reaches; 8 bits with scales of 128,
// 2048 rows, 14.4 us, 4.1 TB/s; one row 2.7 us of kernel, which is its launch.  Rows that
// do not start on 16 bytes, or whose width is no multiple of 8, take eight narrow loads for
// a wide one: 2048 rows of 4096 in a graph 37.8 us in place of 11.5, of 4100 44.3.
#include "tm_vec.h"

namespace {

struct NormParams {
  const void* x;
  const void* res;     // NULL: none
  const void* weight;
  void* out;           // x's type, or e4m3 bytes
  void* res_out;
  float* scales;
  int64_t x_stride, res_stride, out_stride, res_out_stride, scale_stride;
  int64_t rows;
  int hidden, group;   // group: columns of one scale, 0 for the whole row
  int res_dtype, weight_dtype;
  int aligned;         // every row of every tensor starts on 16 bytes, hidden % 8 == 0
  float eps;
};

// 8 elements at `i` of a row, those at or past `end` as zeros.
template <int DT>
__device__ __forceinline__ void load_chunk(const void* p, int64_t base, int i, int end,
                                           bool aligned, float (&v)[8]) {
  if (aligned) {
    tm_load8<DT>(p, base + i, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i + e < end ? tm_load1<DT>(p, base + i + e) : 0.0f;
  }
}

__device__ __forceinline__ void load_chunk_of(int dt, const void* p, int64_t base, int i, int end,
                                              bool aligned, float (&v)[8]) {
  if (dt == TM_DTYPE_BF16)
    load_chunk<TM_DTYPE_BF16>(p, base, i, end, aligned, v);
  else if (dt == TM_DTYPE_F16)
    load_chunk<TM_DTYPE_F16>(p, base, i, end, aligned, v);
  else
    load_chunk<TM_DTYPE_F32>(p, base, i, end, aligned, v);
}

template <int DT>
__device__ __forceinline__ void store_chunk(void* p, int64_t base, int i, int end, bool aligned,
                                            const float (&v)[8]) {
  if (aligned) {
    tm_store8<DT>(p, base + i, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < end) tm_store1<DT>(p, base + i + e, v[e]);
  }
}

// Two floats to two e4m3 bytes (low half of the result), to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, 0, false) & 0xffffu;
}

// The largest of v over the lane's group of `group` / 8 lanes (a power of two, 4 .. 64).
__device__ __forceinline__ uint32_t top_of_group(uint32_t v, int group) {
#define TM_MAX(ctrl) \
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, ctrl, 0xf, 0xf, false))
  TM_MAX(0xb1);   // lane ^ 1
  TM_MAX(0x4e);   // lane ^ 2
  if (group >= 64) TM_MAX(0x141);   // the other four of eight
  if (group >= 128) TM_MAX(0x140);  // the other eight of sixteen
#undef TM_MAX
  if (group >= 256) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  if (group >= 512) v = max(v, (uint32_t)__shfl_xor((int)v, 32));
  return v;
}

// The scale of a largest magnitude, given as bits: over 448, or 1 where that leaves 0.
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float scale = __uint_as_float(top) / 448.0f;
  return scale == 0.0f ? 1.0f : scale;
}

// v over `scale`, each quotient rounded to 32 bits as a division rounds it: a product with
// the inverse in 32 bits puts values next to the middle of two e4m3 steps on the wrong
// side.  In 64 bits the product is off by 2^-52 of the quotient at most, and the quotient of
// two 24-bit numbers lies at least 2^-49 of itself from where its rounding changes.  2048
// rows of 4096 with a residual and scales of 128, in a graph: 16.8 us, by eight divisions
// 17.9, by the 32-bit inverse 16.0.
__device__ __forceinline__ void divide(float (&v)[8], float scale) {
  const double inv = 1.0 / (double)scale;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)((double)v[e] * inv);
}

// NC chunks of 8 elements a thread; W waves a row.  With W = 1 the four waves of a
// workgroup take a row each and no barrier is needed.
template <int DT, int NC, int W, bool FP8>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) tm_rms_norm_kernel(NormParams p) {
  __shared__ float s_sum[W];
  __shared__ uint32_t s_max[W];
  const int lane = threadIdx.x & 63;
  const int wave = W == 1 ? 0 : (int)(threadIdx.x >> 6);
  const int64_t row =
      W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
  if (row >= p.rows) return;
  const int t = W == 1 ? lane : (int)threadIdx.x;
  constexpr int kThreads = 64 * W;
  const bool al = p.aligned != 0;

  float s[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = (c * kThreads + t) * 8;
    if (i < p.hidden) {
      load_chunk<DT>(p.x, row * p.x_stride, i, p.hidden, al, s[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] = 0.0f;
    }
  }
  if (p.res != nullptr) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = (c * kThreads + t) * 8;
      if (i >= p.hidden) continue;
      float r[8];
      if (p.res_dtype == DT)
        load_chunk<DT>(p.res, row * p.res_stride, i, p.hidden, al, r);
      else
        load_chunk<TM_DTYPE_F32>(p.res, row * p.res_stride, i, p.hidden, al, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] += r[e];
      if (p.res_dtype == DT)
        store_chunk<DT>(p.res_out, row * p.res_out_stride, i, p.hidden, al, s[c]);
      else
        store_chunk<TM_DTYPE_F32>(p.res_out, row * p.res_out_stride, i, p.hidden, al, s[c]);
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(s[c][e], s[c][e], sum);
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  if constexpr (W > 1) {
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += s_sum[w];
  }
  const float inv = rsqrtf(sum / (float)p.hidden + p.eps);

  // y over s; the largest magnitude as bits, which order NaN above infinity
  uint32_t top = 0u;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = (c * kThreads + t) * 8;
    if (i < p.hidden) {
      float w[8];
      if (p.weight_dtype == DT)
        load_chunk<DT>(p.weight, 0, i, p.hidden, al, w);
      else
        load_chunk<TM_DTYPE_F32>(p.weight, 0, i, p.hidden, al, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] = s[c][e] * inv * w[e];
    }
    if constexpr (!FP8) {
      if (i < p.hidden) store_chunk<DT>(p.out, row * p.out_stride, i, p.hidden, al, s[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(s[c][e]) & 0x7fffffffu);
      if (p.group != 0) {
        // a group is group / 8 consecutive lanes of one chunk
        const float scale = scale_of(top_of_group(top, p.group));
        if (i < p.hidden) {
          if ((i & (p.group - 1)) == 0)
            p.scales[row * p.scale_stride + i / p.group] = scale;
          divide(s[c], scale);
        }
        top = 0u;
      }
    }
  }
  if constexpr (FP8) {
    float scale = 1.0f;
    if (p.group == 0) {
#pragma unroll
      for (int m = 32; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
      if constexpr (W > 1) {
        if (lane == 0) s_max[wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) top = max(top, s_max[w]);
      }
      scale = scale_of(top);
      if (t == 0) p.scales[row * p.scale_stride] = scale;
    }
    uint8_t* const orow = reinterpret_cast<uint8_t*>(p.out) + row * p.out_stride;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = (c * kThreads + t) * 8;
      if (i >= p.hidden) continue;
      if (p.group == 0) divide(s[c], scale);
      uint32_t q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a = s[c][2 * j], b = s[c][2 * j + 1];
        // |y| / (amax / 448) can pass 448 by a rounding only; NaN stays NaN
        a = a > 448.0f ? 448.0f : a < -448.0f ? -448.0f : a;
        b = b > 448.0f ? 448.0f : b < -448.0f ? -448.0f : b;
        q[j] = pack_e4m3(a, b);
      }
      if (al) {
        typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
        *reinterpret_cast<u32x2*>(orow + i) = u32x2{q[0] | (q[1] << 16), q[2] | (q[3] << 16)};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < p.hidden) orow[i + e] = (uint8_t)(q[e >> 1] >> (8 * (e & 1)));
      }
    }
  }
}

constexpr int64_t kFewRows = 1024;

template <int DT, int NC, int W, bool FP8>
void launch(const NormParams& p, hipStream_t stream) {
  const unsigned grid = (unsigned)(W == 1 ? (p.rows + 3) / 4 : p.rows);
  hipLaunchKernelGGL((tm_rms_norm_kernel<DT, NC, W, FP8>), dim3(grid), dim3(W == 1 ? 256 : 64 * W),
                     0, stream, p);
}

// Many rows: two chunks a thread, by the row's width: one wave a row up to 1024 elements,
// then 4 waves up to 4096, 16 up to 16384; 8 chunks above.  Up to 1024 rows, which leave
// the chip partly empty, one chunk a thread.  Measured (bf16, residual), in us:
//   1 x 1024      one wave 3.0, four 2.5          1024 x 1024  3.9, 3.6
//   2048 x 1024   4.7, 4.6                        6011 x 1024  8.8, 10.5
//   1 x 4096      four waves 3.3, eight 2.7       1024 x 4096  6.5, 6.3
//   2048 x 4096   11.1, 12.6                      6011 x 4096  29.5, 31.2
//   1 x 8192      sixteen waves 3.0, eight 3.6    1 x 4096 by one wave 6.7
//   2048 x 16384  sixteen waves 40.5, four 43.4
template <int DT, bool FP8>
void dispatch(const NormParams& p, hipStream_t stream) {
  const int chunks = (p.hidden + 7) / 8;
  const bool few = p.rows <= kFewRows;
  if (chunks <= 64)
    launch<DT, 1, 1, FP8>(p, stream);
  else if (few && chunks <= 256)
    launch<DT, 1, 4, FP8>(p, stream);
  else if (few && chunks <= 512)
    launch<DT, 1, 8, FP8>(p, stream);
  else if (chunks <= 128)
    launch<DT, 2, 1, FP8>(p, stream);
  else if (chunks <= 512)
    launch<DT, 2, 4, FP8>(p, stream);
  else if (chunks <= 2048)
    launch<DT, 2, 16, FP8>(p, stream);
  else
    launch<DT, 8, 16, FP8>(p, stream);
}

template <bool FP8>
int rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t res_stride,
             int res_dtype, const void* weight, int weight_dtype, int64_t T, int64_t H, float eps,
             int dtype, void* out, int64_t out_stride, float* scales, int64_t scale_stride,
             int64_t group, void* res_out, int64_t res_out_stride, void* stream) {
  if (!tm_dtype_ok(dtype)) return TM_ERR_ARG;
  if (weight_dtype != dtype && weight_dtype != TM_DTYPE_F32) return TM_ERR_ARG;
  if (residual != nullptr && res_dtype != dtype && res_dtype != TM_DTYPE_F32) return TM_ERR_ARG;
  if (!(eps >= 0.0f)) return TM_ERR_ARG;
  if (T < 0 || T > TM_MAX_ROWS || H < 1 || H > TM_MAX_NORM_HIDDEN) return TM_ERR_SHAPE;
  if (T == 0) return TM_OK;
  if (T > 1 && (x_stride < H || out_stride < H)) return TM_ERR_SHAPE;
  if (residual != nullptr && (res_out == nullptr || (T > 1 && (res_stride < H ||
                                                               res_out_stride < H))))
    return TM_ERR_SHAPE;
  if (FP8) {
    if (group != 0 && (group < 32 || group > 512 || (group & (group - 1)) != 0 || H % group != 0))
      return TM_ERR_SHAPE;
    if (T > 1 && scale_stride < (group != 0 ? H / group : 1)) return TM_ERR_SHAPE;
  }
  const int64_t es = tm_dtype_bytes(dtype), rs = tm_dtype_bytes(res_dtype);
  // whole elements at least
  if (((uintptr_t)x % es) || ((uintptr_t)weight % tm_dtype_bytes(weight_dtype)) ||
      ((uintptr_t)scales % 4) || (!FP8 && ((uintptr_t)out % es)) ||
      (residual != nullptr && (((uintptr_t)residual % rs) || ((uintptr_t)res_out % rs))))
    return TM_ERR_ALIGN;
  bool al = H % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)weight % 16 == 0 &&
            (uintptr_t)out % 16 == 0;
  al = al && (T == 1 || (x_stride * es % 16 == 0 && out_stride * (FP8 ? 1 : es) % 8 == 0 &&
                         (FP8 || out_stride * es % 16 == 0)));
  if (residual != nullptr)
    al = al && (uintptr_t)residual % 16 == 0 && (uintptr_t)res_out % 16 == 0 &&
         (T == 1 || (res_stride * rs % 16 == 0 && res_out_stride * rs % 16 == 0));
  NormParams p;
  p.x = x;
  p.res = residual;
  p.weight = weight;
  p.out = out;
  p.res_out = res_out;
  p.scales = scales;
  p.x_stride = x_stride;
  p.res_stride = res_stride;
  p.out_stride = out_stride;
  p.res_out_stride = res_out_stride;
  p.scale_stride = scale_stride;
  p.rows = T;
  p.hidden = (int)H;
  p.group = (int)group;
  p.res_dtype = res_dtype;
  p.weight_dtype = weight_dtype;
  p.aligned = al ? 1 : 0;
  p.eps = eps;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TM_DTYPE_BF16)
    dispatch<TM_DTYPE_BF16, FP8>(p, st);
  else if (dtype == TM_DTYPE_F16)
    dispatch<TM_DTYPE_F16, FP8>(p, st);
  else
    dispatch<TM_DTYPE_F32, FP8>(p, st);
  TM_HIP_CHECK_LAUNCH();
  return TM_OK;
}

}  // namespace

extern "C" int tm_rms_norm(const void* x, int64_t x_stride, const void* residual,
                           int64_t res_stride, int res_dtype, const void* weight,
                           int weight_dtype, int64_t T, int64_t H, float eps, int dtype,
                           void* out, int64_t out_stride, void* res_out, int64_t res_out_stride,
                           void* stream) {
  return rms_norm<false>(x, x_stride, residual, res_stride, res_dtype, weight, weight_dtype, T, H,
                         eps, dtype, out, out_stride, nullptr, 0, 0, res_out, res_out_stride,
                         stream);
}

extern "C" int tm_rms_norm_fp8(const void* x, int64_t x_stride, const void* residual,
                               int64_t res_stride, int res_dtype, const void* weight,
                               int weight_dtype, int64_t T, int64_t H, float eps, int dtype,
                               void* out, int64_t out_stride, float* scales,
                               int64_t scale_stride, int64_t group, void* res_out,
                               int64_t res_out_stride, void* stream) {
  return rms_norm<true>(x, x_stride, residual, res_stride, res_dtype, weight, weight_dtype, T, H,
                        eps, dtype, out, out_stride, scales, scale_stride, group, res_out,
                        res_out_stride, stream);
}
