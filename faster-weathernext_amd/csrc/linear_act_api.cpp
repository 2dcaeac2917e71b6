// C ABI of the linear layers with an epilogue (fwn_rows.h): host-side validation, then the launches.
#include <cstdint>

#include <hip/hip_runtime.h>

#include "fwn_internal.h"
#include "fwn_rows.h"
#include "linear_act.h"

namespace fwn {
namespace {

uint64_t size_of(int32_t dtype) { return dtype == FWN_F32 ? 4u : 2u; }

int check_desc(const fwn_linear_desc* d, const char* what) {
  if (!d) return fail(FWN_ERR_INVALID_ARG, "%s: null descriptor", what);
  if (d->dtype != FWN_F32 && d->dtype != FWN_BF16) return fail(FWN_ERR_UNSUPPORTED, "%s: dtype must be f32 or bf16", what);
  if (d->activation < FWN_ACT_NONE || d->activation > FWN_ACT_SILU)
    return fail(FWN_ERR_UNSUPPORTED, "%s: unknown activation %d", what, d->activation);
  if (d->ins < 1 || d->outs < 1 || d->ins > FWN_LINEAR_ACT_MAX || d->outs > FWN_LINEAR_ACT_MAX)
    return fail(FWN_ERR_INVALID_ARG, "%s: ins %d and outs %d must be 1 to %d", what, d->ins, d->outs, FWN_LINEAR_ACT_MAX);
  // Byte offsets stay inside 64 bits and grids inside 32.
  if (d->rows < 0 || d->rows > (INT64_C(1) << 31)) return fail(FWN_ERR_INVALID_ARG, "%s: %lld rows", what, (long long)d->rows);
  const int64_t widest = INT64_C(1) << 30;
  if (d->x_stride < 0 || d->w_stride < 0 || d->r_stride < 0 || d->x_stride > widest || d->w_stride > widest ||
      d->r_stride > widest)
    return fail(FWN_ERR_INVALID_ARG, "%s: strides %lld, %lld and %lld", what, (long long)d->x_stride,
                (long long)d->w_stride, (long long)d->r_stride);
  const int64_t tiles = ((d->rows + 63) / 64) * (((d->outs > d->ins ? d->outs : d->ins) + 63) / 64);
  if (tiles > (1 << 23)) return fail(FWN_ERR_INVALID_ARG, "%s: too many rows for one launch", what);
  return FWN_OK;
}

bool misaligned(const void* p, uint64_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

struct Span {
  const void* p;
  uint64_t bytes;
};

Span span(const void* p, int64_t rows, int64_t stride, int64_t width, uint64_t size) {
  return {p, rows <= 0 ? 0 : ((uint64_t)(rows - 1) * (uint64_t)stride + (uint64_t)width) * size};
}

bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}

template <int N, int M>
int check_overlap(const Span (&ins)[N], const Span (&outs)[M], const char* what) {
  for (int i = 0; i < M; ++i) {
    for (const Span& s : ins)
      if (overlap(s, outs[i])) return fail(FWN_ERR_INVALID_ARG, "%s: an output overlaps an input", what);
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return fail(FWN_ERR_INVALID_ARG, "%s: outputs overlap", what);
  }
  return FWN_OK;
}

int check_workspace(const void* p, uint64_t bytes, uint64_t need, const char* what) {
  if (need > 0 && (!p || misaligned(p, 256) || bytes < need))
    return fail(FWN_ERR_INVALID_ARG, "%s: a 256-byte aligned workspace of %llu bytes is needed", what,
                (unsigned long long)need);
  return FWN_OK;
}

int status(hipError_t e, const char* what) {
  return e == hipSuccess ? FWN_OK : fail(FWN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int forward(const fwn_linear_desc* d, int32_t op, const void* x, const float* x_scale, const void* weight,
            const float* w_scale, const void* bias, const void* residual, void* out, void* pre, void* stream,
            const char* what) {
  if (int rc = check_desc(d, what)) return rc;
  if (d->rows == 0) return FWN_OK;
  if (!x || !weight || !out || (op == kOpE4m3 && (!x_scale || !w_scale)))
    return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  const uint64_t size = size_of(d->dtype), in_size = op == kOpE4m3 ? 1 : size;
  if (misaligned(x, in_size) || misaligned(weight, in_size) || misaligned(x_scale, 4) || misaligned(w_scale, 4) ||
      misaligned(bias, size) || misaligned(residual, size) || misaligned(out, size) || misaligned(pre, size))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const Span ins[] = {span(x, d->rows, d->x_stride, d->ins, in_size), span(weight, d->outs, d->w_stride, d->ins, in_size),
                      span(x_scale, 1, 0, d->rows, 4), span(w_scale, 1, 0, d->outs, 4), span(bias, 1, 0, d->outs, size),
                      span(residual, d->rows, d->r_stride, d->outs, size)};
  const Span outs[] = {span(out, d->rows, d->outs, d->outs, size), span(pre, d->rows, d->outs, d->outs, size)};
  if (int rc = check_overlap(ins, outs, what)) return rc;
  ProductArgs a{};
  a.a = x;
  a.b = weight;
  a.a_row = d->x_stride;
  a.b_row = d->w_stride;
  a.a_k = a.b_k = 1;
  a.m = d->rows;
  a.n = d->outs;
  a.k = d->ins;
  a.op = op;
  a.dtype = d->dtype;
  a.a_scale = x_scale;
  a.b_scale = w_scale;
  a.bias = bias;
  a.residual = residual;
  a.r_row = d->r_stride;
  a.out = out;
  a.pre = pre;
  a.activation = d->activation;
  return status(launch_product(a, (hipStream_t)stream), what);
}

uint64_t bwd_bytes(const fwn_linear_desc* d) {
  return d->activation == FWN_ACT_NONE ? 0 : (uint64_t)d->rows * (uint64_t)d->outs * size_of(d->dtype);
}

int size_query(const fwn_linear_desc* d, uint64_t* bytes, const char* what) {
  clear_error();
  if (!bytes) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  *bytes = 0;
  return check_desc(d, what);
}

}  // namespace
}  // namespace fwn

extern "C" {

int fwn_linear_act_workspace_size(const fwn_linear_desc* d, uint64_t* bytes) {
  return fwn::size_query(d, bytes, "fwn_linear_act_workspace_size");
}

int fwn_linear_act_launch(const fwn_linear_desc* d, const void* x, const void* weight, const void* bias,
                          const void* residual, void* out, void* pre, void* workspace, uint64_t workspace_bytes,
                          void* stream) {
  using namespace fwn;
  clear_error();
  (void)workspace, (void)workspace_bytes;
  return forward(d, d && d->dtype == FWN_F32 ? kOpF32 : kOpBf16, x, nullptr, weight, nullptr, bias, residual, out, pre,
                 stream, "fwn_linear_act_launch");
}

int fwn_linear_act_q8_workspace_size(const fwn_linear_desc* d, uint64_t* bytes) {
  return fwn::size_query(d, bytes, "fwn_linear_act_q8_workspace_size");
}

int fwn_linear_act_q8_launch(const fwn_linear_desc* d, const uint8_t* x, const float* x_scale, const uint8_t* weight,
                             const float* w_scale, const void* bias, const void* residual, void* out,
                             void* workspace, uint64_t workspace_bytes, void* stream) {
  using namespace fwn;
  clear_error();
  (void)workspace, (void)workspace_bytes;
  return forward(d, kOpE4m3, x, x_scale, weight, w_scale, bias, residual, out, nullptr, stream,
                 "fwn_linear_act_q8_launch");
}

int fwn_linear_act_bwd_workspace_size(const fwn_linear_desc* d, uint64_t* bytes) {
  using namespace fwn;
  if (int rc = size_query(d, bytes, "fwn_linear_act_bwd_workspace_size")) return rc;
  *bytes = bwd_bytes(d);
  return FWN_OK;
}

int fwn_linear_act_bwd_launch(const fwn_linear_desc* d, const void* x, const void* weight, const void* pre,
                              const void* g, void* gx, void* gw, void* gb, void* workspace, uint64_t workspace_bytes,
                              void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_linear_act_bwd_launch";
  if (int rc = check_desc(d, what)) return rc;
  const bool act = d->activation != FWN_ACT_NONE;
  if (d->rows > 0 && (!g || (gx && !weight) || (gw && !x) || (act && !pre)))
    return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  const uint64_t size = size_of(d->dtype);
  for (const void* p : {x, weight, pre, g, (const void*)gx, (const void*)gw, (const void*)gb})
    if (misaligned(p, size)) return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const Span ins[] = {span(x, d->rows, d->x_stride, d->ins, size), span(weight, d->outs, d->w_stride, d->ins, size),
                      span(pre, d->rows, d->outs, d->outs, size), span(g, d->rows, d->outs, d->outs, size)};
  const Span outs[] = {span(gx, d->rows, d->ins, d->ins, size), span(gw, d->outs, d->ins, d->ins, size),
                       span(gb, 1, 0, d->outs, size)};
  if (int rc = check_overlap(ins, outs, what)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, bwd_bytes(d), what)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  if (gb || act) {
    SlopeArgs a{};
    a.g = g;
    a.pre = pre;
    a.dz = act ? workspace : nullptr;
    a.gb = gb;
    a.rows = d->rows;
    a.outs = d->outs;
    a.dtype = d->dtype;
    a.activation = d->activation;
    if (int rc = status(launch_slope(a, s), what)) return rc;
  }
  ProductArgs a{};
  a.a = act ? workspace : g;
  a.op = d->dtype == FWN_F32 ? kOpF32 : kOpBf16;
  a.dtype = d->dtype;
  if (gx && d->rows > 0) {
    a.b = weight;
    a.a_row = d->outs;
    a.a_k = 1;
    a.b_row = 1;
    a.b_k = d->w_stride;
    a.m = d->rows;
    a.n = d->ins;
    a.k = d->outs;
    a.out = gx;
    if (int rc = status(launch_product(a, s), what)) return rc;
  }
  if (gw) {
    a.b = x;
    a.a_row = 1;
    a.a_k = d->outs;
    a.b_row = 1;
    a.b_k = d->x_stride;
    a.m = d->outs;
    a.n = d->ins;
    a.k = d->rows;
    a.out = gw;
    if (int rc = status(launch_product(a, s), what)) return rc;
  }
  return FWN_OK;
}

}  // extern "C"
