// attention_paged.cu -- causal attention over the paged key-value cache, for ragged batches of new
// tokens and for one new token per sequence, with a sliding window and sinks:
//   O[t, h, :] = sum_j P[t, j] V[j, :],  P = softmax_j(alpha * Q[t, h, :] . K[j, :]) over the visible j
// One warp per (row, query head) walks the visible keys with the running maximum m and sum l of
// the softmax: a new score s rescales the sum and the output by exp(m - max(m, s)).
#include "attention_paged.cuh"

namespace lsc {
namespace {

template <bool BF16>
__device__ __forceinline__ float2 to_f32(uint32_t v) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool BF16, int D>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedView c, const AttnArgs a) {
  constexpr int W = D / 64;  // 32-bit words of a row per lane
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.tokens * a.q_heads;
  if (a.offsets && blockIdx.x == 0) check_rows(c, a.offsets, a.tokens);
  for (int64_t i = blockIdx.x * 4 + (threadIdx.x >> 5); i < rows; i += gridDim.x * 4) {
    const int64_t t = i / a.q_heads;
    const int h = static_cast<int>(i - t * a.q_heads), kvh = h / a.group;
    int b = 0;
    int32_t begin = 0, end = 1;
    if (a.offsets) {
      int hi = c.batch;
      while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (__ldg(a.offsets + mid) <= t) b = mid;
        else hi = mid;
      }
      query_rows(a.offsets, b, a.tokens, c.err, lane == 0, begin, end);
      if (t < begin || t >= end) continue;
    } else {
      b = static_cast<int>(t);
      begin = b;
      end = b + 1;
    }
    const int32_t len = paged_len(c, b, lane == 0);
    const int32_t pos = len - end + static_cast<int32_t>(t);
    const int32_t low = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
    float2 q[W], o[W];
    const uint32_t* qp = reinterpret_cast<const uint32_t*>(a.q + t * a.q_token + h * a.q_head) + lane * W;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      q[w] = to_f32<BF16>(qp[w]);
      o[w] = make_float2(0.0f, 0.0f);
    }
    float m = -INFINITY, l = 0.0f;
    for (int32_t j = 0; j <= pos; ++j) {
      if (!key_visible(j, pos, low, a.sinks)) {
        j = low - 1;
        continue;
      }
      const int32_t page = __ldg(c.table + b * c.table_stride + (j >> c.page_shift));
      const bool held = page >= 0 && page < c.num_pages;
      if (!held && lane == 0) raise_bad_arg(c.err);
      const int64_t at = (held ? page : 0) * c.page_stride + (j & ((1 << c.page_shift) - 1)) * c.token_stride +
                         kvh * c.head_stride;
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(c.k + at) + lane * W;
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(c.v + at) + lane * W;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 kk = to_f32<BF16>(held ? kp[w] : 0u);
        s = fmaf(q[w].x, kk.x, fmaf(q[w].y, kk.y, s));
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= a.scale_log2;
      const float m_new = s > m ? s : m;
      const float ref = m_new == -INFINITY ? 0.0f : m_new;
      const float f = ex2_approx(m - ref), e = ex2_approx(s - ref);
      m = m_new;
      l = l * f + e;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 vv = to_f32<BF16>(held ? vp[w] : 0u);
        o[w].x = o[w].x * f + e * vv.x;
        o[w].y = o[w].y * f + e * vv.y;
      }
    }
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    const int64_t at = i * D + lane * 2 * W;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float x = o[w].x * inv, y = o[w].y * inv;
      if (a.out) *reinterpret_cast<uint32_t*>(a.out + at + 2 * w) = pack16<BF16>(x, y);
      if (a.out_i8) {
        if (a.rounding == LSC_ROUND_HALF_EVEN) {
          a.out_i8[at + 2 * w] = static_cast<int8_t>(requant_i8<LSC_ROUND_HALF_EVEN>(x, a.s_out));
          a.out_i8[at + 2 * w + 1] = static_cast<int8_t>(requant_i8<LSC_ROUND_HALF_EVEN>(y, a.s_out));
        } else {
          a.out_i8[at + 2 * w] = static_cast<int8_t>(requant_i8<LSC_ROUND_HALF_AWAY>(x, a.s_out));
          a.out_i8[at + 2 * w + 1] = static_cast<int8_t>(requant_i8<LSC_ROUND_HALF_AWAY>(y, a.s_out));
        }
      }
    }
  }
}

lsc_status launch_simple(const lsc_paged_kv* cache, const DeviceState* ds, const PagedView& c, const AttnArgs& a,
                         cudaStream_t st) {
  const int64_t ctas = (a.tokens * a.q_heads + 3) / 4;
  const int64_t cap = static_cast<int64_t>(ds->sm_count) * 64;
  const int grid = static_cast<int>(ctas < cap ? ctas : cap);
  const bool bf16 = cache->dtype == LSC_DTYPE_BF16;
  if (cache->head_dim == 64) {
    if (bf16) paged_attention_kernel<true, 64><<<grid, 128, 0, st>>>(c, a);
    else paged_attention_kernel<false, 64><<<grid, 128, 0, st>>>(c, a);
  } else {
    if (bf16) paged_attention_kernel<true, 128><<<grid, 128, 0, st>>>(c, a);
    else paged_attention_kernel<false, 128><<<grid, 128, 0, st>>>(c, a);
  }
  LSC_CUDA_TRY(cudaGetLastError());
  return LSC_SUCCESS;
}

}  // namespace

lsc_status attention_args(const lsc_paged_kv* cache, const char* who, const void* q, int64_t tokens, int32_t q_heads,
                          int64_t q_token, int64_t q_head, float alpha, int64_t window, int64_t sinks, void* out,
                          int8_t* out_i8, float s_out, int32_t rounding, AttnArgs* a) {
  if (tokens < 0 || tokens > INT32_MAX) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: bad token count", who);
  if (q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: %d query heads are not a multiple of %d key-value heads", who,
                     q_heads, cache->kv_heads);
  if (!(alpha > 0.0f) || !(alpha <= 1.0e38f))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: alpha must be positive and finite", who);
  if (window < 0 || sinks < 0) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: negative window or sinks", who);
  if (rounding != LSC_ROUND_HALF_AWAY && rounding != LSC_ROUND_HALF_EVEN)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: bad rounding %d", who, rounding);
  if (tokens <= 1) q_token = 8;  // the stride of an axis of one entry is never used
  if (q_heads == 1) q_head = 8;
  if (q_token < 0 || q_head < 0 || q_token % 8 || q_head % 8 || q_token >= (int64_t{1} << 39) ||
      q_head >= (int64_t{1} << 39))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: query strides must be multiples of 8 elements", who);
  if (tokens > 0 && cache->batch > 0) {
    if (!q || (!out && !out_i8)) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: null pointer", who);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_i8)) & 15)
      return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
    if (out_i8 && !(s_out > 0.0f))
      return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: int8 output needs a scale > 0", who);
  }
  a->q = static_cast<const uint16_t*>(q);
  a->tokens = tokens;
  a->q_token = q_token;
  a->q_head = q_head;
  a->q_heads = q_heads;
  a->group = q_heads / cache->kv_heads;
  a->scale_log2 = alpha * kLog2e;
  // positions stay below 2^30: a longer window is no window, more sinks see no more
  a->window = static_cast<int32_t>(window > (1 << 30) ? 0 : window);
  a->sinks = static_cast<int32_t>(window == 0 ? 0 : (sinks > (1 << 30) ? (1 << 30) : sinks));
  a->out = static_cast<uint16_t*>(out);
  a->out_i8 = out_i8;
  a->s_out = s_out;
  a->inv_s_out = out_i8 ? reciprocal_or_zero(s_out) : 0.0f;
  a->rounding = rounding;
  a->offsets = nullptr;
  return LSC_SUCCESS;
}

lsc_status paged_tensor_map(CUtensorMap* map, const lsc_paged_kv* cache, const PagedView& view, const void* base,
                            uint32_t box_rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(cache->head_dim), static_cast<uint64_t>(cache->page_size),
                            static_cast<uint64_t>(cache->kv_heads), static_cast<uint64_t>(cache->num_pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(view.token_stride) * 2, static_cast<uint64_t>(view.head_stride) * 2,
                               static_cast<uint64_t>(view.page_stride) * 2};
  const uint32_t box[4] = {64, box_rows, 1, 1};
  const uint32_t ones[4] = {1, 1, 1, 1};
  return encode_tmap_4d(map, cache->dtype == LSC_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        base, dims, strides, box, ones, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace lsc

using namespace lsc;

extern "C" {

lsc_status lsc_paged_attention_prefill(const lsc_paged_kv* cache, const void* q, int64_t tokens, int32_t q_heads,
                                       int64_t q_token_stride, int64_t q_head_stride, const int32_t* q_offsets,
                                       float alpha, int64_t window, int64_t sinks, void* out, int8_t* out_i8,
                                       float s_out, int32_t rounding, lsc_stream stream) {
  const char* who = "paged_attention_prefill";
  PagedView c;
  AttnArgs a;
  lsc_status st = paged_view(cache, who, &c);
  if (st) return st;
  st = attention_args(cache, who, q, tokens, q_heads, q_token_stride, q_head_stride, alpha, window, sinks, out, out_i8,
                      s_out, rounding, &a);
  if (st) return st;
  if (tokens == 0 || c.batch == 0) return LSC_SUCCESS;
  if (!q_offsets) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: null offsets", who);
  a.offsets = q_offsets;
  DeviceState* ds = nullptr;
  if ((st = paged_device(who, &ds, &c))) return st;
  return launch_simple(cache, ds, c, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
