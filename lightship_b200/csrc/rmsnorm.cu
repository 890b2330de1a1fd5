// rmsnorm.cu -- root-mean-square norm of the rows of [rows, d] with the residual's addition and an
// int8 output (static scale, or one scale per row):
//   h = x + r;  y = (h / sqrt(mean(h^2) + eps)) * gamma;  q = clamp(R(y / s), -128, 127)
// Each element is read once and written once, with about five flops, so HBM bounds it.
//
// Rows of up to 16384 elements stay in registers (h as f32), so nothing is read twice; the sum of
// squares is reduced over the row's threads, and the largest |h gamma| with it when the row finds
// its own scale.  TPR threads share a row, from 8 for short rows to 512 for the longest, so that a
// thread holds at most 32 elements; short rows share a CTA.  A thread takes 8 neighbours at a time
// where every buffer is 16-byte aligned and the length a multiple of 8, single elements elsewhere.
// Longer rows are walked twice by one CTA.
//
// Measured: with a residual, 16384 x 8192 bf16 in 183 to 192 us (5.6 to 5.9 TB/s) and 131072 x 768 f32 to
// int8 with a scale per row in 206 us (6.4 TB/s); without one, where fewer bytes are in flight, 130 us
// (3.9 TB/s) for the same rows to int8, 8192 x 16384 bf16 105 us (5.1 TB/s) and 65536 x 2048 bf16 133 us
// (4.0 TB/s); single elements, 131072 x 1001 f16, 255 us (2.1 TB/s); a row of 4096 2.5 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "epilogue.cuh"
#include "lsc_internal.h"

namespace lsc {
namespace {

constexpr int kWalkThreads = 256;
constexpr int kMaxRow = 16384;     // elements of a row held in registers

struct RmsArgs {
  const void* x;
  const void* res;
  const float* gamma;
  void* sum_out;
  void* out;
  int8_t* q;
  float* row_scales;
  int64_t x_stride, res_stride, sum_stride, out_stride, q_stride;
  int64_t rows, d;
  float eps, s_out, inv_s_out;
  int32_t rounding;
};

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float ld1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// V (8 or 1) elements as loaded and as f32; 8 at a 16-byte aligned address
template <typename T, int V>
struct Raw {
  uint4 v[sizeof(T) / 2];
};
template <typename T>
struct Raw<T, 1> {
  T v;
};
template <int V, typename T>
__device__ __forceinline__ Raw<T, V> load(const T* p) {
  Raw<T, V> r;
  if constexpr (V == 1) {
    r.v = *p;
  } else {
    r.v[0] = *reinterpret_cast<const uint4*>(p);
    if constexpr (sizeof(T) == 4) r.v[1] = *reinterpret_cast<const uint4*>(p + 4);
  }
  return r;
}
template <int V, typename T>
__device__ __forceinline__ void widen(const Raw<T, V>& r, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = ld1(&r.v);
  } else {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
    if constexpr (sizeof(T) == 4) {
      const uint32_t u[4] = {r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = __uint_as_float(w[e]);
        f[4 + e] = __uint_as_float(u[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 v;
        if constexpr (std::is_same<T, __half>::value) v = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
        else v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
        f[2 * e] = v.x;
        f[2 * e + 1] = v.y;
      }
    }
  }
}
template <int V, typename T>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  if constexpr (V == 1) {
    st1(p, f[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The row's scale from its largest |y|: find_scale_zp's symmetric rule.
__device__ __forceinline__ float row_scale(float top) { return top > 0.0f ? __fdiv_rn(top, 127.0f) : 1.0f; }

// How the rows are worked on: CTAs that fit an SM by their registers, and whether a row is read while
// the one before it is reduced and written (by CTAs that all run at once).  That keeps reads in flight
// where few bytes per thread or one CTA per SM leave gaps; with two steps the registers for it cost more
// than it gives.  Without and with it, us, for rows without a residual and (with one): 8192 x 16384 bf16
// 162 and 105 (198 and 182), 300000 x 256 f16 84 and 63 (111 and 96), 1000000 x 64 f16 69 and 52 (92 and
// 81), 131072 x 768 f32 to int8 147 and 130 (205 and 206); two steps, 65536 x 2048 bf16 133 and 165 (178
// and 188), 32768 x 4096 f16 121 and 150 (169 and 175).  The two-step kernels spill all the same, 8 to 56
// bytes a thread in 16 bits and about 120 in f32, as do <f32, 512 x 4> (144) and single elements,
// <256 x 16> (52).
template <int V, int TPR, int STEPS>
struct RowShape {
  static constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR;
  static constexpr int kCtas = V * STEPS <= 16 ? (TPR < 512 ? 4 : 2) : (TPR < 512 ? 2 : 1);
  static constexpr bool kAhead = V == 8 && STEPS != 2;
};

// Rows in registers: TPR threads per row, STEPS steps of V elements per thread (element
// (step * TPR + thread) * V).
template <typename TX, typename TR, int V, int TPR, int STEPS>
__global__ void __launch_bounds__(RowShape<V, TPR, STEPS>::kThreads, RowShape<V, TPR, STEPS>::kCtas)
    rmsnorm_rows_kernel(const RmsArgs a) {
  using Shape = RowShape<V, TPR, STEPS>;
  constexpr int kThreads = Shape::kThreads, kRows = Shape::kRows, kWarps = TPR / 32;
  constexpr bool kAhead = Shape::kAhead;
  __shared__ float red[2][kThreads / 32];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int in_row = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int d = static_cast<int>(a.d);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  Raw<TX, V> xr[STEPS];
  Raw<TR, V> rr[STEPS];
  auto fetch = [&](int64_t r) {
    const TX* x = static_cast<const TX*>(a.x) + r * a.x_stride;
    const TR* res = static_cast<const TR*>(a.res) + r * a.res_stride;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int i = (s * TPR + in_row) * V;
      if (r < a.rows && i < d) {
        xr[s] = load<V>(x + i);
        if (a.res) rr[s] = load<V>(res + i);
      }
    }
  };
  if constexpr (kAhead) fetch(static_cast<int64_t>(blockIdx.x) * kRows + sub);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * kRows; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + sub;
    const bool live = r < a.rows;
    if constexpr (!kAhead) fetch(r);
    float h[STEPS][V];
    float ss = 0.0f, top = 0.0f;
    auto count = [&](int s) {
#pragma unroll
      for (int e = 0; e < V; ++e) ss = fmaf(h[s][e], h[s][e], ss);
      if (a.row_scales) {
        float g[V];
        if (a.gamma) widen<V>(load<V>(a.gamma + (s * TPR + in_row) * V), g);
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, fabsf(a.gamma ? h[s][e] * g[e] : h[s][e]));
      }
    };
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int i = (s * TPR + in_row) * V;
      if (live && i < d) {
        widen<V>(xr[s], h[s]);
        if (a.res) {
          float f[V];
          widen<V>(rr[s], f);
#pragma unroll
          for (int e = 0; e < V; ++e) h[s][e] = __fadd_rn(h[s][e], f[e]);
          if (a.sum_out) store<V>(static_cast<TR*>(a.sum_out) + r * a.sum_stride + i, h[s]);
        }
        if constexpr (!kAhead) count(s);
      }
    }
    if constexpr (kAhead) {
      fetch(r + step);  // on its way while this row is reduced and written
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (live && (s * TPR + in_row) * V < d) count(s);
    }
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (a.row_scales) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if constexpr (kWarps > 1) {
      __syncthreads();  // the row before has been read
      if (lane == 0) {
        red[0][warp] = ss;
        red[1][warp] = top;
      }
      __syncthreads();
      ss = 0.0f;
      top = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        ss += red[0][sub * kWarps + w];
        top = fmaxf(top, red[1][sub * kWarps + w]);
      }
    }
    if (live) {
      const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(d)), a.eps)));
      float scale = a.s_out, inv_scale = a.inv_s_out;
      if (a.row_scales) {
        scale = row_scale(top * inv);
        // a reciprocal that is not a normal number sends every value to the division
        inv_scale = scale >= 1.2e-38f && scale <= 8.0e37f ? __frcp_rn(scale) : 0.0f;
        if (in_row == 0) a.row_scales[r] = scale;
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int i = (s * TPR + in_row) * V;
        if (i < d) {
          float y[V];
          if (a.gamma) {
            float g[V];
            widen<V>(load<V>(a.gamma + i), g);
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = h[s][e] * inv * g[e];
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = h[s][e] * inv;
          }
          if (a.out) store<V>(static_cast<TX*>(a.out) + r * a.out_stride + i, y);
          if (a.q) {
            int8_t* q = a.q + r * a.q_stride + i;
            if constexpr (V == 1) {
              *q = static_cast<int8_t>(a.rounding == LSC_ROUND_HALF_EVEN
                                           ? requant_one<LSC_ROUND_HALF_EVEN>(y[0], scale, inv_scale)
                                           : requant_one<LSC_ROUND_HALF_AWAY>(y[0], scale, inv_scale));
            } else {
              uint32_t pk[2];
              requant_pack<8>(y, scale, inv_scale, false, a.rounding, pk);
              *reinterpret_cast<uint2*>(q) = make_uint2(pk[0], pk[1]);
            }
          }
        }
      }
    }
    __syncwarp();
  }
}

// Any row: one CTA walks it twice.
template <typename TX, typename TR>
__global__ void __launch_bounds__(kWalkThreads) rmsnorm_walk_kernel(const RmsArgs a) {
  __shared__ float red[2][kWalkThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  griddep_wait();
  griddep_launch_dependents();
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const TX* x = static_cast<const TX*>(a.x) + r * a.x_stride;
    const TR* res = a.res ? static_cast<const TR*>(a.res) + r * a.res_stride : nullptr;
    float ss = 0.0f, top = 0.0f;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < a.d; i += kWalkThreads) {
      const float h = res ? __fadd_rn(ld1(x + i), ld1(res + i)) : ld1(x + i);
      ss = fmaf(h, h, ss);
      top = fmaxf(top, fabsf(a.gamma ? h * a.gamma[i] : h));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    __syncthreads();
    if (lane == 0) {
      red[0][warp] = ss;
      red[1][warp] = top;
    }
    __syncthreads();
    ss = 0.0f;
    top = 0.0f;
#pragma unroll
    for (int w = 0; w < kWalkThreads / 32; ++w) {
      ss += red[0][w];
      top = fmaxf(top, red[1][w]);
    }
    const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(a.d)), a.eps)));
    float s = a.s_out;
    if (a.row_scales) {
      s = row_scale(top * inv);
      if (threadIdx.x == 0) a.row_scales[r] = s;
    }
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < a.d; i += kWalkThreads) {
      const float h = res ? __fadd_rn(ld1(x + i), ld1(res + i)) : ld1(x + i);
      const float y = a.gamma ? h * inv * a.gamma[i] : h * inv;
      if (a.sum_out) st1(static_cast<TR*>(a.sum_out) + r * a.sum_stride + i, h);
      if (a.out) st1(static_cast<TX*>(a.out) + r * a.out_stride + i, y);
      if (a.q)
        a.q[r * a.q_stride + i] = static_cast<int8_t>(a.rounding == LSC_ROUND_HALF_EVEN
                                                          ? requant_i8<LSC_ROUND_HALF_EVEN>(y, s)
                                                          : requant_i8<LSC_ROUND_HALF_AWAY>(y, s));
    }
  }
}

template <typename TX, typename TR, int V, int TPR, int STEPS>
lsc_status launch_rows(const RmsArgs& a, const DeviceState* ds, cudaStream_t st) {
  using Shape = RowShape<V, TPR, STEPS>;
  constexpr int kThreads = Shape::kThreads, kRows = Shape::kRows;
  const int64_t ctas = (a.rows + kRows - 1) / kRows;
  const int64_t cap = static_cast<int64_t>(ds->sm_count) * (Shape::kAhead ? Shape::kCtas : 32);
  LSC_CUDA_TRY(launch_dependent(ds->overlap_launches, rmsnorm_rows_kernel<TX, TR, V, TPR, STEPS>,
                                dim3(static_cast<unsigned>(ctas < cap ? ctas : cap)), dim3(kThreads), 0, st, a));
  return LSC_SUCCESS;
}

template <typename TX, typename TR>
lsc_status launch(const RmsArgs& a, const DeviceState* ds, bool vectors, cudaStream_t st) {
  // Few threads per row while they hold it in a few vectors, so that reductions stay within a warp and
  // no lane idles (measured before rows were read ahead): 12288 x 768 f32 to int8 took 30.9 us with 64 threads x 2 vectors and 22.3 with 32 x 3;
  // 100000 x 64 f16 took 26.9 with 32 threads and 9.5 with 8.  Single elements keep rows in registers
  // all the same: 16384 x 1001 f16 took 70 us when walked twice and 42.7 so.
  if (a.d <= kMaxRow && vectors) {
    const int64_t v = a.d / 8;  // vectors of a row
    if (v <= 8) return launch_rows<TX, TR, 8, 8, 1>(a, ds, st);
    if (v <= 16) return launch_rows<TX, TR, 8, 16, 1>(a, ds, st);
    if (v <= 32) return launch_rows<TX, TR, 8, 32, 1>(a, ds, st);
    if (v <= 64) return launch_rows<TX, TR, 8, 32, 2>(a, ds, st);
    if (v <= 96) return launch_rows<TX, TR, 8, 32, 3>(a, ds, st);
    if (v <= 128) return launch_rows<TX, TR, 8, 64, 2>(a, ds, st);
    if (v <= 256) return launch_rows<TX, TR, 8, 128, 2>(a, ds, st);
    if (v <= 512) return launch_rows<TX, TR, 8, 256, 2>(a, ds, st);
    if (v <= 1024) return launch_rows<TX, TR, 8, 512, 2>(a, ds, st);
    return launch_rows<TX, TR, 8, 512, 4>(a, ds, st);
  }
  if (a.d <= kMaxRow) {
    if (a.d <= 32) return launch_rows<TX, TR, 1, 8, 4>(a, ds, st);
    if (a.d <= 256) return launch_rows<TX, TR, 1, 32, 8>(a, ds, st);
    if (a.d <= 1024) return launch_rows<TX, TR, 1, 128, 8>(a, ds, st);
    if (a.d <= 4096) return launch_rows<TX, TR, 1, 256, 16>(a, ds, st);
    return launch_rows<TX, TR, 1, 512, 32>(a, ds, st);
  }
  const int64_t cap = static_cast<int64_t>(ds->sm_count) * 8;
  LSC_CUDA_TRY(launch_dependent(ds->overlap_launches, rmsnorm_walk_kernel<TX, TR>,
                                dim3(static_cast<unsigned>(a.rows < cap ? a.rows : cap)), dim3(kWalkThreads), 0, st, a));
  return LSC_SUCCESS;
}

int64_t type_size(int32_t dtype) {
  return dtype == LSC_DTYPE_F32 ? 4 : (dtype == LSC_DTYPE_F16 || dtype == LSC_DTYPE_BF16 ? 2 : 0);
}

}  // namespace
}  // namespace lsc

using namespace lsc;

extern "C" lsc_status lsc_rmsnorm(const void* x, int32_t x_dtype, int64_t x_stride, const void* residual,
                                  int32_t residual_dtype, int64_t residual_stride, int64_t rows, int64_t d,
                                  const float* gamma, float eps, void* sum_out, int64_t sum_stride, void* out,
                                  int64_t out_stride, int8_t* out_i8, int64_t i8_stride, float s_out,
                                  float* row_scales, int32_t rounding, lsc_stream stream) {
  if (rows < 0 || d < 0 || d > INT32_MAX) return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: bad sizes");
  if (!type_size(x_dtype)) return set_error(LSC_ERROR_UNSUPPORTED_DATATYPE, "rmsnorm: x is f32, f16 or bf16");
  if (residual && residual_dtype != x_dtype && residual_dtype != LSC_DTYPE_F32)
    return set_error(LSC_ERROR_UNSUPPORTED_DATATYPE, "rmsnorm: the residual has x's type or is f32");
  if (sum_out && !residual) return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: sum_out without a residual");
  if (!(eps >= 0.0f) || !(eps <= 3.0e38f))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: eps must be finite and not negative");
  if (rounding != LSC_ROUND_HALF_AWAY && rounding != LSC_ROUND_HALF_EVEN)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: bad rounding %d", rounding);
  if (row_scales && !out_i8) return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: row_scales without an int8 output");
  if (rows == 0 || d == 0) return LSC_SUCCESS;
  if (!x || (!out && !out_i8)) return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: null pointer");
  if (out_i8 && !row_scales && !(s_out > 0.0f))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: int8 output needs a scale > 0 or row_scales");
  if (x_stride < d || (residual && residual_stride < d) || (sum_out && sum_stride < d) || (out && out_stride < d) ||
      (out_i8 && i8_stride < d))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: rows overlap (a stride below d)");
  if (out && out == sum_out) return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: out and sum_out are one buffer");
  const int64_t xs = type_size(x_dtype), rs = residual ? type_size(residual_dtype) : xs;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % xs ||
      (reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(sum_out)) % rs ||
      (reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(row_scales)) % 4)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "rmsnorm: a buffer is not aligned to its elements");
  DeviceState* ds = current_device_state();
  if (!ds) return LSC_ERROR_DEVICE_ERROR;
  RmsArgs a{};
  a.x = x;
  a.res = residual;
  a.gamma = gamma;
  a.sum_out = sum_out;
  a.out = out;
  a.q = out_i8;
  a.row_scales = row_scales;
  a.x_stride = x_stride;
  a.res_stride = residual_stride;
  a.sum_stride = sum_stride;
  a.out_stride = out_stride;
  a.q_stride = i8_stride;
  a.rows = rows;
  a.d = d;
  a.eps = eps;
  a.s_out = s_out;
  a.rounding = rounding;
  a.inv_s_out = out_i8 && !row_scales ? reciprocal_or_zero(s_out) : 0.0f;
  // every vector of 8 elements aligned: bases on 16 bytes, strides multiples of 8 elements (an int8
  // row's vectors are 8 bytes)
  const uintptr_t bases = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                          reinterpret_cast<uintptr_t>(sum_out) | reinterpret_cast<uintptr_t>(out) |
                          reinterpret_cast<uintptr_t>(gamma) | (reinterpret_cast<uintptr_t>(out_i8) << 1);
  const int64_t strides = rows > 1 ? x_stride | (residual ? residual_stride : 0) | (sum_out ? sum_stride : 0) |
                                         (out ? out_stride : 0) | (out_i8 ? i8_stride : 0)
                                   : 0;
  const bool vectors = d % 8 == 0 && bases % 16 == 0 && strides % 8 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = residual && residual_dtype == LSC_DTYPE_F32;
  switch (x_dtype) {
    case LSC_DTYPE_F32: return launch<float, float>(a, ds, vectors, st);
    case LSC_DTYPE_F16:
      return wide ? launch<__half, float>(a, ds, vectors, st) : launch<__half, __half>(a, ds, vectors, st);
    default:
      return wide ? launch<__nv_bfloat16, float>(a, ds, vectors, st)
                  : launch<__nv_bfloat16, __nv_bfloat16>(a, ds, vectors, st);
  }
}
