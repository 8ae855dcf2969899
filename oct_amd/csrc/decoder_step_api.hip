// Entry points of the rest of a decoder's step (4-bit weights, the mixture layer, rotary positions, residual
// norms): validation, locking, launches.  Every argument is checked before the device is looked at.
#include <math.h>

#include "api_checks.h"
#include "moe_w4.h"
#include "reactor_internal.h"

namespace prom {
namespace {

constexpr uint32_t kMaxStride = 1u << 24;

bool matrix_valid(const PrometheusW4Matrix* w) {
  return w != nullptr && w->struct_size >= sizeof(*w) && prometheus_reactor_w4_bytes(w->n, w->k, w->group) != 0 &&
         w->count >= 1u && w->count <= 1u << 16 && w->reserved0 == 0u && w->data != nullptr && aligned(w->data, 16);
}

W4View view(const PrometheusW4Matrix* w) { return w4_view(w->data, w->n, w->k, w->group, w->count); }

// Rows of `width` elements, `stride` apart.
bool rows_valid(const void* p, uint32_t stride, uint64_t width, uint32_t dtype) {
  return p != nullptr && aligned(p, dtype_size(dtype)) && stride >= width && stride < kMaxStride;
}

int w4_rows(void* handle, const PrometheusW4Matrix* matrix, const void* weights, uint32_t row_stride, uint32_t dtype,
            bool pack, uint32_t* stage, int* detail) {
  Runtime* rt = lookup(handle);
  set_status(stage, detail, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(stage, detail);
  if (!matrix_valid(matrix) || dtype > PROM_DTYPE_BF16 || !rows_valid(weights, row_stride, matrix->k, dtype))
    return invalid(stage, detail);
  if (!rt->available) return refuse(stage, detail, PROM_STAGE_INIT, rt->init_detail);
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  const bool bf16 = dtype == PROM_DTYPE_BF16;
  return queued(pack ? launch_w4_pack(view(matrix), weights, bf16, row_stride, cx.stream)
                     : launch_w4_unpack(view(matrix), const_cast<void*>(weights), bf16, row_stride, cx.stream),
                stage, detail, 0);
}

// One of a rope call's two tensors; absent ones are valid.
bool rope_tensor(const void* in, void* out, uint32_t heads, uint32_t in_stride, uint32_t out_stride,
                 const PrometheusRopeRequest* r, RopeTensor* t) {
  *t = RopeTensor{in, out, heads, in_stride, out_stride};
  if (in == nullptr && out == nullptr) return true;
  const uint64_t width = (uint64_t)heads * r->head_dim;
  return heads >= 1u && heads <= 1u << 16 && rows_valid(in, in_stride, width, r->dtype) &&
         rows_valid(out, out_stride, width, r->dtype) && (in != out || in_stride == out_stride);
}

}  // namespace
}  // namespace prom

using namespace prom;

extern "C" {

PROM_REACTOR_API uint64_t prometheus_reactor_w4_bytes(uint32_t n, uint32_t k, uint32_t group) {
  if (n == 0u || n > 1u << 24 || k == 0u || k > 1u << 20 || (group != 32u && group != 64u && group != 128u)) return 0;
  return w4_view(nullptr, n, k, group, 1).stride;
}

PROM_REACTOR_API int prometheus_reactor_runtime_w4_pack_device(void* handle, const PrometheusW4Matrix* matrix,
                                                               const void* weights, uint32_t row_stride,
                                                               uint32_t dtype, uint32_t* out_stage,
                                                               int* out_detail_code) {
  return w4_rows(handle, matrix, weights, row_stride, dtype, true, out_stage, out_detail_code);
}

PROM_REACTOR_API int prometheus_reactor_runtime_w4_unpack_device(void* handle, const PrometheusW4Matrix* matrix,
                                                                 void* weights, uint32_t row_stride, uint32_t dtype,
                                                                 uint32_t* out_stage, int* out_detail_code) {
  return w4_rows(handle, matrix, weights, row_stride, dtype, false, out_stage, out_detail_code);
}

PROM_REACTOR_API int prometheus_reactor_runtime_gemm_w4_device(void* handle, const PrometheusW4Matrix* matrix,
                                                               const PrometheusW4GemmRequest* request,
                                                               uint32_t* out_stage, int* out_detail_code) {
  Runtime* rt = lookup(handle);
  set_status(out_stage, out_detail_code, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(out_stage, out_detail_code);
  const PrometheusW4GemmRequest* r = request;
  if (!matrix_valid(matrix) || r == nullptr || r->struct_size < sizeof(*r) || r->dtype > PROM_DTYPE_BF16 ||
      r->rows == 0u || r->rows > 1u << 20 || r->reserved0 != 0u || !rows_valid(r->x, r->x_stride, matrix->k, r->dtype) ||
      !rows_valid(r->out, r->out_stride, matrix->n, r->dtype))
    return invalid(out_stage, out_detail_code);
  if (!rt->available) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, rt->init_detail);
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  return queued(launch_gemm_w4(view(matrix), r->x, r->x_stride, r->out, r->out_stride, r->dtype == PROM_DTYPE_BF16,
                               r->rows, cx.stream),
                out_stage, out_detail_code, 0);
}

PROM_REACTOR_API int prometheus_reactor_runtime_moe_w4_device(void* handle, const PrometheusW4Matrix* gate,
                                                              const PrometheusW4Matrix* up,
                                                              const PrometheusW4Matrix* down,
                                                              const PrometheusMoeRequest* request,
                                                              uint32_t* out_stage, int* out_detail_code) {
  Runtime* rt = lookup(handle);
  set_status(out_stage, out_detail_code, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(out_stage, out_detail_code);
  const PrometheusMoeRequest* r = request;
  if (!matrix_valid(gate) || !matrix_valid(up) || !matrix_valid(down) || r == nullptr || r->struct_size < sizeof(*r))
    return invalid(out_stage, out_detail_code);
  if (gate->n != up->n || gate->k != up->k || gate->group != up->group || gate->count != up->count ||
      down->n != gate->k || down->k != gate->n || down->count != gate->count || gate->count > PROM_MOE_MAX_EXPERTS ||
      r->dtype > PROM_DTYPE_BF16 || r->tokens == 0u || r->top_k == 0u || r->top_k > gate->count ||
      r->top_k > PROM_MOE_MAX_TOP_K || (uint64_t)r->tokens * r->top_k > PROM_MOE_MAX_PAIRS ||
      !rows_valid(r->x, r->x_stride, gate->k, r->dtype) || !rows_valid(r->out, r->out_stride, gate->k, r->dtype) ||
      r->activation > PROM_MOE_GELU_TANH || r->renormalise > 1u || r->router == nullptr || !aligned(r->router, 4) ||
      !aligned(r->out_experts, 4) || !aligned(r->out_weights, 4))
    return invalid(out_stage, out_detail_code);
  if (!rt->available) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, rt->init_detail);
  W4MoeArgs a{};
  a.gate = view(gate);
  a.up = view(up);
  a.down = view(down);
  a.router = r->router;
  a.x = r->x;
  a.out = r->out;
  a.out_chosen = r->out_experts;
  a.out_weights = r->out_weights;
  a.x_stride = r->x_stride;
  a.out_stride = r->out_stride;
  a.activation = r->activation;
  a.tokens = (int)r->tokens;
  a.experts = (int)gate->count;
  a.top_k = (int)r->top_k;
  a.renormalise = r->renormalise != 0u;
  const bool bf16 = r->dtype == PROM_DTYPE_BF16;
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  void* base = staging(6, moe_w4_workspace(a, nullptr));
  if (base == nullptr)
    return refuse(out_stage, out_detail_code, PROM_STAGE_TRANSFER_IN, PROM_DETAIL_HIP_ALLOC_FAILED);
  moe_w4_workspace(a, base);
  return queued(launch_moe_w4(a, bf16, cx.stream), out_stage, out_detail_code, 0);
}

PROM_REACTOR_API int prometheus_reactor_runtime_rope_device(void* handle, const PrometheusRopeRequest* request,
                                                            uint32_t* out_stage, int* out_detail_code) {
  Runtime* rt = lookup(handle);
  set_status(out_stage, out_detail_code, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(out_stage, out_detail_code);
  const PrometheusRopeRequest* r = request;
  RopeArgs a{};
  if (r == nullptr || r->struct_size < sizeof(*r) || r->dtype > PROM_DTYPE_BF16 || r->rows == 0u ||
      r->rows > 1u << 22 || r->head_dim < 2u || r->head_dim > kRopeMaxDim || r->rotary_dim < 2u ||
      r->rotary_dim % 2u != 0u || r->rotary_dim > r->head_dim || r->layout > PROM_ROPE_PAIRS ||
      !isfinite(r->magnitude) || r->reserved0 != 0u || r->positions == nullptr || !aligned(r->positions, 4) ||
      r->turns == nullptr || !aligned(r->turns, 8) || (r->q == nullptr && r->k == nullptr) ||
      !rope_tensor(r->q, r->q_out, r->q_heads, r->q_stride, r->q_out_stride, r, &a.q) ||
      !rope_tensor(r->k, r->k_out, r->k_heads, r->k_stride, r->k_out_stride, r, &a.k))
    return invalid(out_stage, out_detail_code);
  if (!rt->available) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, rt->init_detail);
  a.positions = r->positions;
  a.turns = r->turns;
  a.rows = r->rows;
  a.head_dim = r->head_dim;
  a.rotary = r->rotary_dim;
  a.magnitude = r->magnitude;
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  return queued(launch_rope(a, r->dtype == PROM_DTYPE_BF16, r->layout == PROM_ROPE_PAIRS, cx.stream), out_stage,
                out_detail_code, 0);
}

PROM_REACTOR_API int prometheus_reactor_rope_turns(const PrometheusRopeScaling* scaling, double* out_turns,
                                                   float* out_magnitude) {
  const PrometheusRopeScaling* s = scaling;
  if (s == nullptr || s->struct_size < sizeof(*s) || out_turns == nullptr || out_magnitude == nullptr ||
      s->rotary_dim < 2u || s->rotary_dim % 2u != 0u || s->rotary_dim > kRopeMaxDim ||
      s->kind > PROM_ROPE_SCALE_PARTS || s->reserved0 != 0u || !isfinite(s->base) || !(s->base > 1.0))
    return PROM_ERROR;
  if (s->kind != PROM_ROPE_SCALE_NONE && (!isfinite(s->factor) || !(s->factor >= 1.0))) return PROM_ERROR;
  if (s->kind == PROM_ROPE_SCALE_BASE && s->rotary_dim == 2u) return PROM_ERROR;
  const bool parts = s->kind == PROM_ROPE_SCALE_PARTS;
  if (parts && (!isfinite(s->context) || !(s->context >= 1.0) || !isfinite(s->fast_turns) || !(s->slow_turns > 0.0) ||
                !(s->fast_turns > s->slow_turns)))
    return PROM_ERROR;
  const double d = s->rotary_dim, two_pi = 2.0 * 3.14159265358979323846;
  double base = s->base;
  if (s->kind == PROM_ROPE_SCALE_BASE) base *= pow(s->factor, d / (d - 2.0));
  if (!isfinite(base)) return PROM_ERROR;
  // The pair that turns t times within the context: base^(2 i / d) = context / (2 pi t).
  double low = 0.0, span = 1.0;
  if (parts) {
    const auto at = [&](double t) { return d * log(s->context / (two_pi * t)) / (2.0 * log(base)); };
    low = fmax(0.0, floor(at(s->fast_turns)));
    span = fmax(fmin(d - 1.0, ceil(at(s->slow_turns))) - low, 0.001);
  }
  for (uint32_t i = 0; i < s->rotary_dim / 2u; ++i) {
    double f = pow(base, -2.0 * i / d);
    if (s->kind == PROM_ROPE_SCALE_LINEAR) f /= s->factor;
    if (parts) {
      const double slow = fmin(fmax((i - low) / span, 0.0), 1.0);
      f = f * (1.0 - slow) + f / s->factor * slow;
    }
    out_turns[i] = f / two_pi;
  }
  *out_magnitude = parts ? (float)(1.0 + 0.1 * log(s->factor)) : 1.0f;
  return PROM_OK;
}

PROM_REACTOR_API int prometheus_reactor_runtime_residual_norm_device(void* handle,
                                                                     const PrometheusResidualNormRequest* request,
                                                                     uint32_t* out_stage, int* out_detail_code) {
  Runtime* rt = lookup(handle);
  set_status(out_stage, out_detail_code, PROM_STAGE_NONE, 0);
  if (rt == nullptr) return bad_handle(out_stage, out_detail_code);
  const PrometheusResidualNormRequest* r = request;
  if (r == nullptr || r->struct_size < sizeof(*r) || r->dtype > PROM_DTYPE_BF16) return invalid(out_stage, out_detail_code);
  const auto absent_or_rows = [&](const void* p, uint32_t stride) {
    return p == nullptr || rows_valid(p, stride, r->width, r->dtype);
  };
  // An output in place of an input keeps its rows.
  const auto in_place = [&](const void* out, uint32_t stride) {
    return out == nullptr || ((out != r->h || stride == r->h_stride) && (out != r->y || stride == r->y_stride));
  };
  const bool vectors = r->gate != nullptr || r->scale != nullptr || r->shift != nullptr;
  if (r->rows == 0u || r->rows > 1u << 22 || r->width == 0u || r->width > kResidualNormMaxWidth || r->gate_tanh > 1u ||
      !isfinite(r->residual_scale) || !isfinite(r->weight_offset) || !isfinite(r->eps) || r->eps < 0.0f ||
      !rows_valid(r->h, r->h_stride, r->width, r->dtype) || !absent_or_rows(r->y, r->y_stride) ||
      !absent_or_rows(r->h_out, r->h_out_stride) || !absent_or_rows(r->out, r->out_stride) ||
      (r->h_out == nullptr && r->out == nullptr) || (r->h_out != nullptr && r->h_out == r->out) ||
      !in_place(r->h_out, r->h_out_stride) || !in_place(r->out, r->out_stride) || !aligned(r->post, 4) ||
      !aligned(r->pre, 4) || !absent_or_rows(r->gate, r->vector_stride) ||
      !absent_or_rows(r->scale, r->vector_stride) || !absent_or_rows(r->shift, r->vector_stride) ||
      (vectors && r->rows_per_vector == 0u))
    return invalid(out_stage, out_detail_code);
  if (!rt->available) return refuse(out_stage, out_detail_code, PROM_STAGE_INIT, rt->init_detail);
  ResidualNormArgs a{};
  a.h = r->h;
  a.y = r->y;
  a.gate = r->gate;
  a.scale = r->scale;
  a.shift = r->shift;
  a.post = r->post;
  a.pre = r->pre;
  a.h_out = r->h_out;
  a.out = r->out;
  a.rows = r->rows;
  a.width = r->width;
  a.h_stride = r->h_stride;
  a.y_stride = r->y_stride;
  a.h_out_stride = r->h_out_stride;
  a.out_stride = r->out_stride;
  a.vector_stride = r->vector_stride;
  a.rows_per_vector = vectors ? r->rows_per_vector : r->rows;  // else the weights are joined once for all rows
  a.residual_scale = r->residual_scale;
  a.weight_offset = r->weight_offset;
  a.eps = r->eps;
  a.over_width = 1.0 / r->width;
  a.gate_tanh = r->gate_tanh != 0u;
  DeviceContext& cx = ctx();
  std::lock_guard<std::mutex> lock(cx.mu);
  CurrentDevice device(cx.device);
  return queued(launch_residual_norm(a, r->dtype == PROM_DTYPE_BF16, cx.stream), out_stage, out_detail_code, 0);
}

}  // extern "C"
