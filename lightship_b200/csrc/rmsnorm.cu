// rmsnorm.cu -- root-mean-square norm of the rows of [rows, d] with the residual's addition and an
// int8 output (static scale, or one scale per row):
//   h = x + r;  y = (h / sqrt(mean(h^2) + eps)) * gamma;  q = clamp(R(y / s), -128, 127)
// One CTA per row; sums in f32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "epilogue.cuh"
#include "lsc_internal.h"

namespace lsc {
namespace {

constexpr int kRmsThreads = 256;

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
  float eps, s_out;
  int32_t rounding;
};

__device__ __forceinline__ float ld1(const float* p) { return *p; }
__device__ __forceinline__ float ld1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float ld1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename TX, typename TR>
__global__ void __launch_bounds__(kRmsThreads) rmsnorm_kernel(const RmsArgs a) {
  __shared__ float red[2 * kRmsThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const TX* x = static_cast<const TX*>(a.x) + r * a.x_stride;
    const TR* res = a.res ? static_cast<const TR*>(a.res) + r * a.res_stride : nullptr;
    float ss = 0.0f, top = 0.0f;
    for (int64_t i = threadIdx.x; i < a.d; i += kRmsThreads) {
      const float h = res ? __fadd_rn(ld1(x + i), ld1(res + i)) : ld1(x + i);
      ss = fmaf(h, h, ss);
      top = fmaxf(top, fabsf(a.gamma ? h * __ldg(a.gamma + i) : h));
    }
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    __syncthreads();
    if (lane == 0) {
      red[warp] = ss;
      red[kRmsThreads / 32 + warp] = top;
    }
    __syncthreads();
    ss = 0.0f;
    top = 0.0f;
    for (int w = 0; w < kRmsThreads / 32; ++w) {
      ss += red[w];
      top = fmaxf(top, red[kRmsThreads / 32 + w]);
    }
    const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(a.d)), a.eps)));
    float s = a.s_out;
    if (a.row_scales) {
      const float am = top * inv;
      s = am > 0.0f ? __fdiv_rn(am, 127.0f) : 1.0f;
      if (threadIdx.x == 0) a.row_scales[r] = s;
    }
    for (int64_t i = threadIdx.x; i < a.d; i += kRmsThreads) {
      const float h = res ? __fadd_rn(ld1(x + i), ld1(res + i)) : ld1(x + i);
      const float y = a.gamma ? h * inv * __ldg(a.gamma + i) : h * inv;
      if (a.sum_out) st1(static_cast<TR*>(a.sum_out) + r * a.sum_stride + i, h);
      if (a.out) st1(static_cast<TX*>(a.out) + r * a.out_stride + i, y);
      if (a.q)
        a.q[r * a.q_stride + i] = static_cast<int8_t>(a.rounding == LSC_ROUND_HALF_EVEN
                                                          ? requant_i8<LSC_ROUND_HALF_EVEN>(y, s)
                                                          : requant_i8<LSC_ROUND_HALF_AWAY>(y, s));
    }
  }
}

template <typename TX, typename TR>
lsc_status launch(const RmsArgs& a, int sm_count, cudaStream_t st) {
  const int64_t cap = static_cast<int64_t>(sm_count) * 8;
  rmsnorm_kernel<TX, TR><<<static_cast<int>(a.rows < cap ? a.rows : cap), kRmsThreads, 0, st>>>(a);
  LSC_CUDA_TRY(cudaGetLastError());
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = residual && residual_dtype == LSC_DTYPE_F32;
  switch (x_dtype) {
    case LSC_DTYPE_F32: return launch<float, float>(a, ds->sm_count, st);
    case LSC_DTYPE_F16:
      return wide ? launch<__half, float>(a, ds->sm_count, st) : launch<__half, __half>(a, ds->sm_count, st);
    default:
      return wide ? launch<__nv_bfloat16, float>(a, ds->sm_count, st)
                  : launch<__nv_bfloat16, __nv_bfloat16>(a, ds->sm_count, st);
  }
}
