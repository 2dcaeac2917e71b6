// C ABI of dropout and of the norms around a block (fwn_rows.h): host-side validation, then the launches.
#include <cmath>
#include <cstdint>

#include <hip/hip_runtime.h>

#include "dropout.h"
#include "fwn_internal.h"
#include "fwn_rows.h"

namespace fwn {
namespace {

struct Span {
  const void* p;
  uint64_t bytes;
};

Span rows_of(const void* p, int64_t rows, int64_t stride, int64_t width, uint64_t size) {
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

uint64_t size_of(int32_t dtype) { return dtype == FWN_F32 ? 4u : 2u; }

bool misaligned(const void* p, uint64_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

int status(hipError_t e, const char* what) {
  return e == hipSuccess ? FWN_OK : fail(FWN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int check_rows(int64_t rows, int64_t x_stride, int64_t y_stride, int32_t channels, int32_t most, int32_t dtype, const char* what) {
  if (dtype != FWN_F32 && dtype != FWN_BF16) return fail(FWN_ERR_UNSUPPORTED, "%s: dtype must be f32 or bf16", what);
  if (channels < 1 || channels > most) return fail(FWN_ERR_INVALID_ARG, "%s: %d channels (1 to %d)", what, channels, most);
  // A row's number is a word of the generator's counter; every byte offset stays inside 64 bits.
  if (rows < 0 || rows >> 32) return fail(FWN_ERR_INVALID_ARG, "%s: %lld rows", what, (long long)rows);
  const int64_t widest = INT64_MAX / 8 / (rows > 0 ? rows : 1) - channels;
  if (x_stride < 0 || y_stride < 0 || x_stride > widest || y_stride > widest || channels > widest)
    return fail(FWN_ERR_INVALID_ARG, "%s: strides %lld and %lld", what, (long long)x_stride, (long long)y_stride);
  return FWN_OK;
}

int check_dropout(const fwn_dropout& d, DropoutArgs& a, const char* what) {
  if (!(d.p >= 0 && d.p <= 1)) return fail(FWN_ERR_INVALID_ARG, "%s: p must be 0 to 1", what);
  if (misaligned(d.state, 8)) return fail(FWN_ERR_INVALID_ARG, "%s: state is not aligned to its elements", what);
  const double border = std::nearbyint(d.p * 65536);
  a.state = d.state;
  a.seed = d.seed;
  a.offset = d.offset;
  a.border = (uint32_t)border;
  a.keep = border < 65536 ? (float)(65536 / (65536 - border)) : 0.f;
  return FWN_OK;
}

int check_sandwich(const fwn_sandwich_desc* d, DropoutArgs& draw, const char* what) {
  if (!d) return fail(FWN_ERR_INVALID_ARG, "%s: null descriptor", what);
  if (int rc = check_rows(d->rows, d->x_stride, d->y_stride, d->channels, FWN_RMS_MAX_CHANNELS, d->dtype, what)) return rc;
  for (int32_t t : {d->gate_dtype, d->post_dtype, d->pre_dtype})
    if (t != d->dtype && t != FWN_F32)
      return fail(FWN_ERR_UNSUPPORTED, "%s: the gate's and the weights' dtypes must be the dtype or f32", what);
  if (d->post_norm != 0 && d->post_norm != 1) return fail(FWN_ERR_INVALID_ARG, "%s: post_norm must be 0 or 1", what);
  if (!(d->eps >= 0.f) || !std::isfinite(d->eps)) return fail(FWN_ERR_INVALID_ARG, "%s: eps must be finite and >= 0", what);
  if (!std::isfinite(d->scale)) return fail(FWN_ERR_INVALID_ARG, "%s: scale must be finite", what);
  return check_dropout(d->drop, draw, what);
}

int check_gate(const fwn_sandwich_desc* d, const char* what) {
  if (d->gate_rows < 1 || d->rows % d->gate_rows)
    return fail(FWN_ERR_INVALID_ARG, "%s: gate_rows %lld must divide %lld rows", what, (long long)d->gate_rows, (long long)d->rows);
  return FWN_OK;
}

Span gate_of(const fwn_sandwich_desc* d, const void* gate) {
  return {gate, gate ? (uint64_t)(d->rows / d->gate_rows) * (uint64_t)d->channels * size_of(d->gate_dtype) : 0};
}

// Bytes of partial sums, whichever of the weights' gradients are wanted.
uint64_t part_bytes(const fwn_sandwich_desc* d, bool gate) {
  const SandwichGrid g = sandwich_grid(d->rows, gate ? d->gate_rows : d->rows, d->channels, d->dtype);
  return (uint64_t)g.parts * (uint64_t)g.blocks * (uint64_t)d->channels * sizeof(float);
}

}  // namespace
}  // namespace fwn

extern "C" {

int fwn_dropout_launch(const fwn_dropout_desc* d, const void* x, const void* residual, void* out, void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_dropout_launch";
  if (!d) return fail(FWN_ERR_INVALID_ARG, "%s: null descriptor", what);
  if (int rc = check_rows(d->rows, d->x_stride, d->r_stride, d->channels, FWN_DROPOUT_MAX_CHANNELS, d->dtype, what)) return rc;
  DropoutRowsArgs a{};
  if (int rc = check_dropout(d->drop, a.drop, what)) return rc;
  if (d->rows == 0) return FWN_OK;
  if (!x || !out) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  const uint64_t size = size_of(d->dtype);
  if (misaligned(x, size) || misaligned(residual, size) || misaligned(out, size))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const Span to = rows_of(out, d->rows, d->channels, d->channels, size);
  if ((overlap(to, rows_of(x, d->rows, d->x_stride, d->channels, size)) && !(out == x && d->x_stride == d->channels)) ||
      (overlap(to, rows_of(residual, d->rows, d->r_stride, d->channels, size)) &&
       !(out == residual && d->r_stride == d->channels)) ||
      overlap(to, {d->drop.state, 16}))
    return fail(FWN_ERR_INVALID_ARG, "%s: the output overlaps an input", what);
  a.x = x;
  a.residual = residual;
  a.out = out;
  a.rows = d->rows;
  a.x_stride = d->x_stride;
  a.r_stride = d->r_stride;
  a.channels = d->channels;
  return status(launch_dropout(d->dtype, a, (hipStream_t)stream), what);
}

int fwn_sandwich_norm_launch(const fwn_sandwich_desc* d, const void* x, const void* y, const void* gate, const void* post_weight,
                             const void* pre_weight, void* sum, void* out, void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_sandwich_norm_launch";
  SandwichArgs a{};
  if (int rc = check_sandwich(d, a.draw, what)) return rc;
  if (d->rows == 0) return FWN_OK;
  if (!x || !y || !sum || !out) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  if (gate)
    if (int rc = check_gate(d, what)) return rc;
  const uint64_t size = size_of(d->dtype);
  if (misaligned(x, size) || misaligned(y, size) || misaligned(sum, size) || misaligned(out, size) ||
      misaligned(gate, size_of(d->gate_dtype)) || misaligned(post_weight, size_of(d->post_dtype)) ||
      misaligned(pre_weight, size_of(d->pre_dtype)))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const uint64_t c = (uint64_t)d->channels;
  const Span ins[] = {rows_of(x, d->rows, d->x_stride, d->channels, size), rows_of(y, d->rows, d->y_stride, d->channels, size),
                      gate_of(d, gate), {post_weight, c * size_of(d->post_dtype)}, {pre_weight, c * size_of(d->pre_dtype)},
                      {d->drop.state, 16}};
  const Span outs[] = {rows_of(sum, d->rows, d->channels, d->channels, size), rows_of(out, d->rows, d->channels, d->channels, size)};
  if (int rc = check_overlap(ins, outs, what)) return rc;
  a.x = x;
  a.y = y;
  a.gate = gate;
  a.post_weight = post_weight;
  a.pre_weight = pre_weight;
  a.sum = sum;
  a.out = out;
  a.rows = d->rows;
  a.gate_rows = gate ? d->gate_rows : d->rows;
  a.x_stride = d->x_stride;
  a.y_stride = d->y_stride;
  a.channels = d->channels;
  a.eps = d->eps;
  a.scale = d->scale;
  a.post_norm = d->post_norm != 0;
  a.gate_f32 = d->gate_dtype == FWN_F32;
  a.post_f32 = d->post_dtype == FWN_F32;
  a.pre_f32 = d->pre_dtype == FWN_F32;
  a.drop = a.draw.border > 0;
  return status(launch_sandwich(d->dtype, a, (hipStream_t)stream), what);
}

int fwn_sandwich_norm_bwd_workspace_size(const fwn_sandwich_desc* d, int32_t gate, uint64_t* bytes) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_sandwich_norm_bwd_workspace_size";
  if (!bytes) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  *bytes = 0;
  DropoutArgs draw;
  if (int rc = check_sandwich(d, draw, what)) return rc;
  if (gate)
    if (int rc = check_gate(d, what)) return rc;
  *bytes = part_bytes(d, gate != 0);
  return FWN_OK;
}

int fwn_sandwich_norm_bwd_launch(const fwn_sandwich_desc* d, const void* s, const void* y, const void* gate,
                                 const void* post_weight, const void* pre_weight, const void* g_sum, const void* g_out, void* gx,
                                 void* gy, void* g_gate, void* g_post, void* g_pre, void* workspace, uint64_t workspace_bytes,
                                 void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_sandwich_norm_bwd_launch";
  SandwichBwdArgs a{};
  if (int rc = check_sandwich(d, a.draw, what)) return rc;
  if (d->rows > 0 && (!s || !y)) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  if ((g_gate && !gate) || (g_post && !post_weight) || (g_pre && !pre_weight))
    return fail(FWN_ERR_INVALID_ARG, "%s: the gradient of a gate or weight that is not given", what);
  if (gate)
    if (int rc = check_gate(d, what)) return rc;
  const uint64_t size = size_of(d->dtype), gate_size = size_of(d->gate_dtype), post_size = size_of(d->post_dtype),
                 pre_size = size_of(d->pre_dtype), c = (uint64_t)d->channels;
  for (const void* p : {s, y, g_sum, g_out, (const void*)gx, (const void*)gy})
    if (misaligned(p, size)) return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  if (misaligned(gate, gate_size) || misaligned(g_gate, gate_size) || misaligned(post_weight, post_size) ||
      misaligned(g_post, post_size) || misaligned(pre_weight, pre_size) || misaligned(g_pre, pre_size))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const auto rows = [&](const void* p, int64_t stride) { return rows_of(p, d->rows, stride, d->channels, size); };
  const bool part = g_post || g_pre || (g_gate && d->gate_rows > 1);
  const uint64_t need = part ? part_bytes(d, gate != nullptr) : 0;
  if (need > 0 && (!workspace || misaligned(workspace, 16) || workspace_bytes < need))
    return fail(FWN_ERR_INVALID_ARG, "%s: a 16-byte aligned workspace of %llu bytes is needed", what, (unsigned long long)need);
  const Span ins[] = {rows(s, d->channels), rows(y, d->y_stride), gate_of(d, gate), {post_weight, c * post_size},
                      {pre_weight, c * pre_size}, rows(g_sum, d->channels), rows(g_out, d->channels), {d->drop.state, 16}};
  const Span outs[] = {rows(gx, d->channels), rows(gy, d->channels), gate_of(d, g_gate), {g_post, c * post_size},
                       {g_pre, c * pre_size}, {workspace, need}};
  if (int rc = check_overlap(ins, outs, what)) return rc;
  a.s = s;
  a.y = y;
  a.gate = gate;
  a.post_weight = post_weight;
  a.pre_weight = pre_weight;
  a.g_sum = g_sum;
  a.g_out = g_out;
  a.gx = gx;
  a.gy = gy;
  a.g_gate = d->rows > 0 ? g_gate : nullptr;
  a.g_post = g_post;
  a.g_pre = g_pre;
  a.part = (float*)workspace;
  a.rows = d->rows;
  a.gate_rows = gate ? d->gate_rows : d->rows;
  a.y_stride = d->y_stride;
  a.channels = d->channels;
  a.eps = d->eps;
  a.scale = d->scale;
  a.post_norm = d->post_norm != 0;
  a.gate_f32 = d->gate_dtype == FWN_F32;
  a.post_f32 = d->post_dtype == FWN_F32;
  a.pre_f32 = d->pre_dtype == FWN_F32;
  a.drop = a.draw.border > 0;
  if (d->rows == 0 && !g_post && !g_pre) return FWN_OK;
  return status(launch_sandwich_bwd(d->dtype, a, (hipStream_t)stream), what);
}

}  // extern "C"
