// C ABI of the RMS norm (fwn_rows.h): host-side validation, then the launches.
#include <cmath>
#include <cstdint>

#include <hip/hip_runtime.h>

#include "fwn_internal.h"
#include "fwn_rows.h"
#include "rms_kernels.h"

namespace fwn {
namespace {

int check_desc(const fwn_rms_desc* d, const char* what) {
  if (!d) return fail(FWN_ERR_INVALID_ARG, "%s: null descriptor", what);
  if (d->dtype != FWN_F32 && d->dtype != FWN_BF16) return fail(FWN_ERR_UNSUPPORTED, "%s: dtype must be f32 or bf16", what);
  if (d->weight_dtype != d->dtype && d->weight_dtype != FWN_F32)
    return fail(FWN_ERR_UNSUPPORTED, "%s: weight_dtype must be the dtype or f32", what);
  if (d->channels < 1 || d->channels > FWN_RMS_MAX_CHANNELS)
    return fail(FWN_ERR_INVALID_ARG, "%s: %d channels (1 to %d)", what, d->channels, FWN_RMS_MAX_CHANNELS);
  // Rows times channels and every byte offset stay inside 64 bits.
  const int64_t most = INT64_MAX / 8 / FWN_RMS_MAX_CHANNELS;
  if (d->rows < 0 || d->rows > most) return fail(FWN_ERR_INVALID_ARG, "%s: %lld rows", what, (long long)d->rows);
  const int64_t widest = INT64_MAX / 8 / (d->rows > 0 ? d->rows : 1);
  if (d->x_stride < 0 || d->y_stride < 0 || d->x_stride > widest || d->y_stride > widest)
    return fail(FWN_ERR_INVALID_ARG, "%s: strides %lld and %lld", what, (long long)d->x_stride, (long long)d->y_stride);
  if (!(d->eps >= 0.f) || !std::isfinite(d->eps)) return fail(FWN_ERR_INVALID_ARG, "%s: eps must be finite and >= 0", what);
  return FWN_OK;
}

struct Span {
  const void* p;
  uint64_t bytes;
};

uint64_t size_of(int32_t dtype) { return dtype == FWN_F32 ? 4u : 2u; }

Span rows_of(const fwn_rms_desc* d, const void* p, int64_t stride, uint64_t size) {
  return {p, d->rows == 0 ? 0 : ((uint64_t)(d->rows - 1) * (uint64_t)stride + (uint64_t)d->channels) * size};
}

bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}

bool misaligned(const void* p, uint64_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

// Validates one forward launch and runs it. `out` is the norm in the dtype, else q and scale.
int forward(const fwn_rms_desc* d, const void* x, const void* y, const void* weight, void* sum, void* out, uint8_t* q,
            float* scale, bool norm, void* stream, const char* what) {
  if (int rc = check_desc(d, what)) return rc;
  if (d->rows == 0) return FWN_OK;
  if (!x || (!out && (!q || !scale))) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  if (!y != !sum) return fail(FWN_ERR_INVALID_ARG, "%s: y and sum go together", what);
  const uint64_t size = size_of(d->dtype);
  if (misaligned(x, size) || misaligned(y, size) || misaligned(sum, size) || misaligned(out, size) ||
      misaligned(weight, size_of(d->weight_dtype)) || misaligned(scale, 4))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const Span ins[] = {rows_of(d, x, d->x_stride, size), rows_of(d, y, d->y_stride, size),
                      {weight, (uint64_t)d->channels * size_of(d->weight_dtype)}};
  const Span outs[] = {rows_of(d, sum, d->channels, size), rows_of(d, out, d->channels, size),
                       rows_of(d, q, d->channels, 1), {scale, (uint64_t)d->rows * 4}};
  for (int i = 0; i < 4; ++i) {
    for (const Span& s : ins)
      if (overlap(s, outs[i])) return fail(FWN_ERR_INVALID_ARG, "%s: an output overlaps an input", what);
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return fail(FWN_ERR_INVALID_ARG, "%s: outputs overlap", what);
  }
  RmsArgs a{};
  a.x = x;
  a.y = y;
  a.weight = weight;
  a.sum = sum;
  a.out = out;
  a.q = q;
  a.scale = scale;
  a.rows = d->rows;
  a.x_stride = d->x_stride;
  a.y_stride = y ? d->y_stride : 0;
  a.channels = d->channels;
  a.eps = d->eps;
  a.norm = norm;
  a.weight_f32 = d->weight_dtype == FWN_F32;
  const hipError_t e = launch_rms(d->dtype, a, (hipStream_t)stream);
  if (e != hipSuccess) return fail(FWN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return FWN_OK;
}

uint64_t part_bytes(const fwn_rms_desc* d) {
  return (uint64_t)rms_bwd_blocks(d->rows, d->channels) * (uint64_t)d->channels * sizeof(float);
}

}  // namespace
}  // namespace fwn

extern "C" {

int fwn_rms_norm_launch(const fwn_rms_desc* d, const void* x, const void* y, const void* weight, void* sum, void* out,
                        void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_rms_norm_launch";
  if (d && d->rows > 0 && !out) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  return forward(d, x, y, weight, sum, out, nullptr, nullptr, true, stream, what);
}

int fwn_rms_norm_q8_launch(const fwn_rms_desc* d, const void* x, const void* y, const void* weight, void* sum, uint8_t* q,
                           float* scale, void* stream) {
  fwn::clear_error();
  return fwn::forward(d, x, y, weight, sum, nullptr, q, scale, true, stream, "fwn_rms_norm_q8_launch");
}

int fwn_quantize_rows_launch(const fwn_rms_desc* d, const void* x, uint8_t* q, float* scale, void* stream) {
  fwn::clear_error();
  return fwn::forward(d, x, nullptr, nullptr, nullptr, nullptr, q, scale, false, stream, "fwn_quantize_rows_launch");
}

int fwn_rms_norm_bwd_workspace_size(const fwn_rms_desc* d, uint64_t* bytes) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_rms_norm_bwd_workspace_size";
  if (!bytes) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  if (int rc = check_desc(d, what)) return rc;
  *bytes = part_bytes(d);
  return FWN_OK;
}

int fwn_rms_norm_bwd_launch(const fwn_rms_desc* d, const void* s, const void* weight, const void* g_out,
                            const void* g_sum, void* gx, void* gw, void* workspace, uint64_t workspace_bytes,
                            void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_rms_norm_bwd_launch";
  if (int rc = check_desc(d, what)) return rc;
  if (d->rows > 0 && (!s || !g_out || !gx)) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  const uint64_t size = size_of(d->dtype);
  if (misaligned(s, size) || misaligned(g_out, size) || misaligned(g_sum, size) || misaligned(gx, size) ||
      misaligned(weight, size_of(d->weight_dtype)) || misaligned(gw, size_of(d->weight_dtype)))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const uint64_t channels = (uint64_t)d->channels * size_of(d->weight_dtype);
  const Span out = rows_of(d, gx, d->channels, size), sums{gw, channels};
  for (const Span& in : {rows_of(d, s, d->channels, size), rows_of(d, g_out, d->channels, size),
                         rows_of(d, g_sum, d->channels, size), Span{weight, channels}})
    if (overlap(out, in) || overlap(sums, in)) return fail(FWN_ERR_INVALID_ARG, "%s: an output overlaps an input", what);
  if (overlap(out, sums)) return fail(FWN_ERR_INVALID_ARG, "%s: outputs overlap", what);
  if (gw && (!workspace || misaligned(workspace, 16) || workspace_bytes < part_bytes(d)))
    return fail(FWN_ERR_INVALID_ARG, "%s: a 16-byte aligned workspace of %llu bytes is needed", what,
                (unsigned long long)part_bytes(d));
  if (d->rows == 0 && !gw) return FWN_OK;
  RmsBwdArgs a{};
  a.s = s;
  a.weight = weight;
  a.g_out = g_out;
  a.g_sum = g_sum;
  a.gx = gx;
  a.part = gw ? (float*)workspace : nullptr;
  a.gw = gw;
  a.rows = d->rows;
  a.channels = d->channels;
  a.blocks = rms_bwd_blocks(d->rows, d->channels);
  a.eps = d->eps;
  a.weight_f32 = d->weight_dtype == FWN_F32;
  const hipError_t e = launch_rms_bwd(d->dtype, a, (hipStream_t)stream);
  if (e != hipSuccess) return fail(FWN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return FWN_OK;
}

}  // extern "C"
