// paged_cache.cu -- the paged key-value cache: the host's check of its description and the append
// of new tokens.
#include "paged_cache.cuh"

namespace lsc {

lsc_status paged_view(const lsc_paged_kv* c, const char* who, PagedView* view) {
  if (!c) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: no cache", who);
  if (c->dtype != LSC_DTYPE_F16 && c->dtype != LSC_DTYPE_BF16)
    return set_error(LSC_ERROR_UNSUPPORTED_DATATYPE, "%s: the cache holds f16 or bf16, not dtype %d", who, c->dtype);
  if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: page_size %d is not a power of two from 8 to 256", who,
                     c->page_size);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: head_dim %d is not 64 or 128", who, c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > 1024)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: %d key-value heads (1 to 1024)", who, c->kv_heads);
  if (c->batch < 0 || c->batch > 65535)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: %d sequences (at most 65535)", who, c->batch);
  if (c->max_pages < 0 || c->num_pages < 0 || c->num_pages > INT32_MAX ||
      static_cast<int64_t>(c->max_pages) * c->page_size > (1 << 30))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: bad page counts (at most 2^30 places per sequence)", who);
  if (c->batch > 0 && (!c->kv_lens || (c->max_pages > 0 && !c->page_table)))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: null page table or lengths", who);
  if ((reinterpret_cast<uintptr_t>(c->kv_lens) | reinterpret_cast<uintptr_t>(c->page_table)) & 3)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: misaligned page table or lengths", who);
  if (c->batch > 1 && c->table_stride < c->max_pages)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: the page table's rows overlap", who);
  if (c->batch > 0 && c->num_pages < 1) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: a cache without pages", who);
  if (c->num_pages > 0 && (!c->k || !c->v)) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: null cache", who);
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: k and v must be 16-byte aligned", who);
  // the stride of an axis of one entry is never used: any value will do there
  const int64_t token = c->token_stride;
  const int64_t head = c->kv_heads > 1 ? c->head_stride : c->head_dim;
  const int64_t page = c->num_pages > 1 ? c->page_stride : c->page_size * token;
  const int64_t most = int64_t{1} << 39;  // 2^40 bytes: the tensor maps' limit of a stride
  for (int64_t s : {page, token, head})
    if (s % 8 || s < c->head_dim || s >= most)
      return set_error(LSC_ERROR_INVALID_ARGUMENT,
                       "%s: strides must be multiples of 8 elements and not shorter than a head", who);
  view->k = static_cast<uint16_t*>(c->k);
  view->v = static_cast<uint16_t*>(c->v);
  view->table = c->page_table;
  view->lens = c->kv_lens;
  view->table_stride = c->table_stride;
  view->num_pages = c->num_pages;
  view->page_stride = page;
  view->token_stride = token;
  view->head_stride = head;
  view->max_pages = c->max_pages;
  view->batch = c->batch;
  view->kv_heads = c->kv_heads;
  view->page_shift = __builtin_ctz(static_cast<unsigned>(c->page_size));
  view->err = nullptr;
  return LSC_SUCCESS;
}

lsc_status paged_device(const char* who, DeviceState** ds, PagedView* view) {
  *ds = current_device_state();
  if (!*ds) return LSC_ERROR_DEVICE_ERROR;
  if ((*ds)->cc_major != 10) return set_error(LSC_ERROR_BACKEND_NOT_AVAILABLE, "%s: needs an sm_100 device", who);
  view->err = (*ds)->err_word;
  return LSC_SUCCESS;
}

namespace {

// One thread copies 8 elements (16 bytes) of one token's key head and value head.  Every byte is read and
// written once and the page table is small, so HBM bounds it: 35k tokens of 8 heads of 128 in 49.2 us
// (5.91 TB/s).
__global__ void __launch_bounds__(256)
    kv_append_kernel(const PagedView c, const uint16_t* __restrict__ k_new, const uint16_t* __restrict__ v_new,
                     int64_t tokens, int64_t new_token, int64_t new_head, const int32_t* __restrict__ offsets,
                     int chunk_shift) {
  const int64_t per_token = static_cast<int64_t>(c.kv_heads) << chunk_shift;
  const int64_t total = tokens * per_token;
  if (blockIdx.x == 0) check_rows(c, offsets, tokens);
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = i / per_token;
    const int r = static_cast<int>(i - t * per_token);
    const int h = r >> chunk_shift, e = (r & ((1 << chunk_shift) - 1)) * 8;
    // the last sequence whose first row is at or before t
    int lo = 0, hi = c.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (offsets[mid] <= t) lo = mid;
      else hi = mid;
    }
    int32_t begin, end;
    query_rows(offsets, lo, tokens, c.err, false, begin, end);
    if (t < begin || t >= end) continue;
    const int32_t len = paged_len(c, lo, false);
    const int32_t pos = len - end + static_cast<int32_t>(t);
    if (pos < 0) {
      if (r == 0) raise_bad_arg(c.err);
      continue;
    }
    const int32_t page = c.table[lo * c.table_stride + (pos >> c.page_shift)];
    if (page < 0 || page >= c.num_pages) {
      if (r == 0) raise_bad_arg(c.err);
      continue;
    }
    const int64_t src = t * new_token + h * new_head + e;
    const int64_t dst = page * c.page_stride + (pos & ((1 << c.page_shift) - 1)) * c.token_stride +
                        h * c.head_stride + e;
    const uint4 kv = *reinterpret_cast<const uint4*>(k_new + src);
    const uint4 vv = *reinterpret_cast<const uint4*>(v_new + src);
    *reinterpret_cast<uint4*>(c.k + dst) = kv;
    *reinterpret_cast<uint4*>(c.v + dst) = vv;
  }
}

}  // namespace
}  // namespace lsc

extern "C" lsc_status lsc_kv_cache_append(const lsc_paged_kv* cache, const void* k_new, const void* v_new,
                                          int64_t tokens, int64_t new_token_stride, int64_t new_head_stride,
                                          const int32_t* q_offsets, lsc_stream stream) {
  using namespace lsc;
  PagedView c;
  lsc_status st = paged_view(cache, "kv_cache_append", &c);
  if (st) return st;
  if (tokens < 0 || tokens > (1 << 30))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "kv_cache_append: bad token count (at most 2^30)");
  if (tokens == 0 || c.batch == 0) return LSC_SUCCESS;
  if (!k_new || !v_new || !q_offsets) return set_error(LSC_ERROR_INVALID_ARGUMENT, "kv_cache_append: null pointer");
  if (reinterpret_cast<uintptr_t>(q_offsets) & 3)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "kv_cache_append: misaligned offsets");
  if ((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) & 15)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "kv_cache_append: k_new and v_new must be 16-byte aligned");
  if (tokens == 1) new_token_stride = 0;
  if (c.kv_heads == 1) new_head_stride = 0;
  if (new_token_stride < 0 || new_head_stride < 0 || new_token_stride % 8 || new_head_stride % 8)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "kv_cache_append: strides must be multiples of 8 elements");
  DeviceState* ds = nullptr;
  if ((st = paged_device("kv_cache_append", &ds, &c))) return st;
  const int shift = cache->head_dim == 64 ? 3 : 4;
  const int64_t ctas = (((tokens * c.kv_heads) << shift) + 255) / 256;
  const int64_t cap = static_cast<int64_t>(ds->sm_count) * 32;
  kv_append_kernel<<<static_cast<int>(ctas < cap ? ctas : cap), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      c, static_cast<const uint16_t*>(k_new), static_cast<const uint16_t*>(v_new), tokens, new_token_stride,
      new_head_stride, q_offsets, shift);
  LSC_CUDA_TRY(cudaGetLastError());
  return LSC_SUCCESS;
}
