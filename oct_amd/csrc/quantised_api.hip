// Entry points of the quantised decode path: validation, locking, launches.  Every
// argument is checked before the device is looked at; what lies in device memory
// (page numbers, lengths, row starts) the kernels keep within bounds themselves.
#include <math.h>

#include "reactor_internal.h"

namespace prom {
namespace {

// The device that the reactor's stream and staging belong to is current while a call
// queues its work, whatever the calling thread had chosen.
class CurrentDevice {
 public:
  explicit CurrentDevice(int device) {
    if (hipGetDevice(&before_) == hipSuccess && before_ != device) changed_ = hipSetDevice(device) == hipSuccess;
  }
  ~CurrentDevice() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

int refuse(uint32_t* stage, int* detail, uint32_t s, int d) {
  set_status(stage, detail, s, d);
  return PROM_ERROR;
}

int invalid(uint32_t* stage, int* detail) { return refuse(stage, detail, PROM_STAGE_INIT, PROM_DETAIL_INVALID_ARGUMENT); }

int bad_handle(uint32_t* stage, int* detail) {
  set_status(stage, detail, PROM_STAGE_INIT, PROM_INVALID_HANDLE);
  return PROM_INVALID_HANDLE;
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
uintptr_t dtype_size(uint32_t dtype) { return dtype == PROM_DTYPE_BF16 ? 2 : 4; }

// PROM_OK, or what the caller returns: the launch's error to a status.
int queued(hipError_t e, uint32_t* stage, int* detail, int path) {
  if (e == hipErrorOutOfMemory) return refuse(stage, detail, PROM_STAGE_TRANSFER_IN, PROM_DETAIL_HIP_ALLOC_FAILED);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    return refuse(stage, detail, PROM_STAGE_SUBMIT, PROM_DETAIL_HIP_LAUNCH_FAILED);
  }
  set_status(stage, detail, PROM_STAGE_SUBMIT, path);
  return PROM_OK;
}

bool cache_valid(const PrometheusKv4Cache* c) {
  return c != nullptr && c->struct_size >= sizeof(*c) && prometheus_reactor_kv4_page_bytes(c->head_dim, c->kv_heads) != 0 &&
         c->pages >= 1u && c->pages <= 0x7fffffffu && c->sequences >= 1u && c->sequences <= 1u << 20 &&
         (uint64_t)c->sequences * c->kv_heads <= kKv4MaxColumns && c->table_stride >= 1u && c->table_stride <= 1u << 24 &&
         c->pool != nullptr && aligned(c->pool, 16) && c->page_table != nullptr && aligned(c->page_table, 4) &&
         c->lengths != nullptr && aligned(c->lengths, 4);
}

Kv4View view(const PrometheusKv4Cache* c) {
  return Kv4View{static_cast<uint8_t*>(c->pool), c->page_table,         c->lengths, (int)c->kv_heads,
                 (int)c->sequences,              (int)c->table_stride, c->pages};
}

int kv4_rows(void* handle, const PrometheusKv4Cache* cache, const PrometheusKv4RowsRequest* r, bool write,
             uint32_t* stage, int* detail) {
  Runtime* rt = lookup(handle);
  set_status(stage, detail, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(stage, detail);
  if (!cache_valid(cache) || r == nullptr || r->struct_size < sizeof(*r)) return invalid(stage, detail);
  const bool pointers = write ? r->k != nullptr && r->v != nullptr : r->k != nullptr || r->v != nullptr;
  if (r->dtype > PROM_DTYPE_BF16 || r->rows == 0u || r->rows > 1u << 22 ||
      (uint64_t)cache->kv_heads * cache->head_dim > r->row_stride || r->row_stride >= 1u << 24 || !pointers ||
      !aligned(r->k, dtype_size(r->dtype)) || !aligned(r->v, dtype_size(r->dtype)) || r->row_starts == nullptr ||
      !aligned(r->row_starts, 4))
    return invalid(stage, detail);
  if (!rt->available) return refuse(stage, detail, PROM_STAGE_INIT, rt->init_detail);
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  const bool bf16 = r->dtype == PROM_DTYPE_BF16;
  const auto launch = [&] {
    return write ? launch_kv4_write(view(cache), (int)cache->head_dim, r->k, r->v, bf16, r->row_starts, r->rows,
                                    r->row_stride, cx.stream)
                 : launch_kv4_read(view(cache), (int)cache->head_dim, r->k, r->v, bf16, r->row_starts, r->rows,
                                   r->row_stride, cx.stream);
  };
  return queued(launch(), stage, detail, 0);
}

}  // namespace
}  // namespace prom

using namespace prom;

extern "C" {

PROM_REACTOR_API int prometheus_reactor_runtime_quantize_rows_int8_device(void* handle, const void* input,
                                                                          int8_t* output, float* scales, uint32_t rows,
                                                                          uint32_t width, uint32_t input_row_stride,
                                                                          uint32_t dtype, uint32_t* out_stage,
                                                                          int* out_detail_code) {
  Runtime* rt = lookup(handle);
  set_status(out_stage, out_detail_code, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(out_stage, out_detail_code);
  if (input == nullptr || output == nullptr || scales == nullptr || rows == 0u || width == 0u ||
      input_row_stride < width || (uint64_t)rows * input_row_stride >= 1ull << 40 || dtype > PROM_DTYPE_BF16 ||
      !aligned(input, dtype_size(dtype)) || !aligned(scales, 4))
    return invalid(out_stage, out_detail_code);
  if (!rt->available) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, rt->init_detail);
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  return queued(launch_quantize_rows_int8(input, dtype == PROM_DTYPE_BF16, output, scales, rows, width,
                                          input_row_stride, cx.stream),
                out_stage, out_detail_code, 0);
}

PROM_REACTOR_API int prometheus_reactor_runtime_gemm_int8_device(void* handle, const int8_t* a, const int8_t* w,
                                                                 const float* a_scale, const float* w_scale, void* c,
                                                                 uint32_t m, uint32_t n, uint32_t k, uint32_t dtype,
                                                                 uint32_t* out_stage, int* out_detail_code) {
  Runtime* rt = lookup(handle);
  set_status(out_stage, out_detail_code, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(out_stage, out_detail_code);
  // The order of the other products' checks: operands, dimensions, range.
  if (a == nullptr || w == nullptr || a_scale == nullptr || w_scale == nullptr || c == nullptr)
    return refuse(out_stage, out_detail_code, PROM_STAGE_TRANSFER_IN, PROM_ERROR);
  if (m == 0u || n == 0u || k == 0u) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, PROM_ERROR);
  // Rows and columns up to a tile behind the last are counted in 31 bits.
  if (!gemm_shape_fits(m, n, k) || m > PROM_GEMM_INT8_MAX_SIDE || n > PROM_GEMM_INT8_MAX_SIDE)
    return refuse(out_stage, out_detail_code, PROM_STAGE_TRANSFER_IN, PROM_DETAIL_SIZE_OVERFLOW);
  if (k > PROM_GEMM_INT8_MAX_K || dtype > PROM_DTYPE_BF16 || !aligned(a_scale, 4) || !aligned(w_scale, 4) ||
      !aligned(c, dtype_size(dtype)))
    return invalid(out_stage, out_detail_code);
  if (!rt->available) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, rt->init_detail);
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  return queued(launch_gemm_int8(a, w, a_scale, w_scale, c, dtype == PROM_DTYPE_BF16, m, n, k, cx.stream), out_stage,
                out_detail_code, PROM_DETAIL_PATH_HIP_MFMA_INT8);
}

PROM_REACTOR_API uint64_t prometheus_reactor_kv4_page_bytes(uint32_t head_dim, uint32_t kv_heads) {
  if ((head_dim != 64u && head_dim != 128u && head_dim != 256u) || kv_heads == 0u || kv_heads > 1024u) return 0;
  return (uint64_t)kv4_block_bytes((int)head_dim) * kv_heads;
}

PROM_REACTOR_API int prometheus_reactor_runtime_kv4_write_device(void* handle, const PrometheusKv4Cache* cache,
                                                                 const PrometheusKv4RowsRequest* request,
                                                                 uint32_t* out_stage, int* out_detail_code) {
  return kv4_rows(handle, cache, request, true, out_stage, out_detail_code);
}

PROM_REACTOR_API int prometheus_reactor_runtime_kv4_read_device(void* handle, const PrometheusKv4Cache* cache,
                                                                const PrometheusKv4RowsRequest* request,
                                                                uint32_t* out_stage, int* out_detail_code) {
  return kv4_rows(handle, cache, request, false, out_stage, out_detail_code);
}

PROM_REACTOR_API int prometheus_reactor_runtime_attention_kv4_device(void* handle, const PrometheusKv4Cache* cache,
                                                                     const PrometheusKv4AttentionRequest* request,
                                                                     uint32_t* out_stage, int* out_detail_code) {
  Runtime* rt = lookup(handle);
  set_status(out_stage, out_detail_code, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(out_stage, out_detail_code);
  const PrometheusKv4AttentionRequest* r = request;
  if (!cache_valid(cache) || r == nullptr || r->struct_size < sizeof(*r)) return invalid(out_stage, out_detail_code);
  const uintptr_t size = dtype_size(r->dtype);
  if (r->dtype > PROM_DTYPE_BF16 || r->rows == 0u || r->rows > 1u << 22 || r->q_heads == 0u || r->q_heads > 1u << 16 ||
      r->q_heads % cache->kv_heads != 0u || (uint64_t)r->rows * (r->q_heads / cache->kv_heads) >= 1ull << 30 ||
      (uint64_t)r->q_heads * cache->head_dim > r->q_stride ||
      (uint64_t)r->q_heads * cache->head_dim > r->out_stride || r->q_stride >= 1u << 24 || r->out_stride >= 1u << 24 ||
      r->max_rows == 0u || r->max_rows > r->rows || r->max_length == 0u || !isfinite(r->scale * kLog2E) || r->scale <= 0.0f ||
      r->q == nullptr || r->out == nullptr || r->row_starts == nullptr || !aligned(r->q, size) ||
      !aligned(r->out, size) || !aligned(r->row_starts, 4))
    return invalid(out_stage, out_detail_code);
  if (!rt->available) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, rt->init_detail);
  Kv4AttentionArgs a{};
  a.c = view(cache);
  a.q = r->q;
  a.out = r->out;
  a.row_starts = r->row_starts;
  a.rows = r->rows;
  a.q_stride = r->q_stride;
  a.out_stride = r->out_stride;
  a.window = r->window;
  a.max_rows = r->max_rows;
  a.max_length = r->max_length;
  a.q_heads = (int)r->q_heads;
  a.group = (int)(r->q_heads / cache->kv_heads);
  a.scale = r->scale;
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  const bool bf16 = r->dtype == PROM_DTYPE_BF16;
  const size_t bytes = kv4_attention_partial_bytes(a, (int)cache->head_dim, bf16);
  if (bytes > 0) {
    a.part = static_cast<float*>(staging(6, bytes));
    if (a.part == nullptr)
      return refuse(out_stage, out_detail_code, PROM_STAGE_TRANSFER_IN, PROM_DETAIL_HIP_ALLOC_FAILED);
  }
  return queued(launch_kv4_attention(a, (int)cache->head_dim, bf16, cx.stream), out_stage,
                out_detail_code, 0);
}

}  // extern "C"
