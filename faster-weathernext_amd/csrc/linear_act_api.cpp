// C ABI of the linear layers with an epilogue (fwn_rows.h): host-side validation, then the launches.
#include <algorithm>
#include <cstdint>

#include <hip/hip_runtime.h>

#include "fwn_internal.h"
#include "fwn_rows.h"
#include "linear_act.h"
#include "linear_q4.h"

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
  const int64_t widest = FWN_LINEAR_STRIDE_MAX;
  if (d->x_stride < 0 || d->w_stride < 0 || d->r_stride < 0 || d->x_stride > widest || d->w_stride > widest ||
      d->r_stride > FWN_LINEAR_ACT_MAX)
    return fail(FWN_ERR_INVALID_ARG, "%s: strides %lld, %lld and %lld", what, (long long)d->x_stride,
                (long long)d->w_stride, (long long)d->r_stride);
  const int64_t ins = (d->ins + 63) / 64, outs = (d->outs + 63) / 64, rows = (d->rows + 63) / 64, most = 1 << 23;
  if (rows * ins > most || rows * outs > most || ins * outs > most)
    return fail(FWN_ERR_INVALID_ARG, "%s: %lld rows, ins %d and outs %d are too many for one launch", what,
                (long long)d->rows, d->ins, d->outs);
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

constexpr int64_t kCus = 256;

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t parts(int64_t v, int64_t of) { return (v + of - 1) / of; }

int64_t op_size(int32_t op) { return op == kOpE4m3 ? 1 : op == kOpBf16 ? 2 : 4; }

// Hands out pieces of a workspace (base NULL: only counts them).
struct Workspace {
  char* base;
  uint64_t used = 0;
  char* take(uint64_t bytes) {
    char* p = base ? base + used : nullptr;
    used += (uint64_t)up((int64_t)bytes, 256);
    return p;
  }
};

// A matrix in rows as the product kernels read it: as it lies where it is bf16 or e4m3 in whole aligned 16 bytes or
// float32, else laid out in the workspace.
struct Matrix {
  const void* src;
  int64_t rows, cols, stride;  // elements
  int32_t op;
  char* at;
  int64_t row_bytes;
  bool laid;

  void place(const void* p, int64_t r, int64_t c, int64_t s, int32_t o, Workspace& ws, bool force = false) {
    src = p, rows = r, cols = c, stride = s, op = o;
    const int64_t size = op_size(op);
    laid = force || s * size > kMaxStride || (op != kOpF32 && (((uintptr_t)p & 15) || c * size % 16 || s * size % 16));
    row_bytes = s * size;
    at = (char*)p;
    if (!laid) return;
    row_bytes = up(c, 8) * size;
    if (row_bytes % 16) row_bytes = up(row_bytes, 16);
    at = ws.take((uint64_t)(rows * row_bytes));
  }

  hipError_t lay_out(hipStream_t stream) const {
    if (!laid) return hipSuccess;
    return launch_layout({src, rows, cols, stride, op, at, row_bytes}, stream);
  }
};

// The tiles and ranges of the sum of one product, by an estimate of its time in us: a CU takes its share of the
// workgroups one after the other, or two at a time where that fills it, each its stages and its ends (the
// first loads and the epilogue); split sums add the partial products' trip through memory. Both tiles, one range, us
// with 256 and with 128 (rows x inputs -> outputs, bf16): 40,962 x 768 -> 3,072 231 and 247, 40,962 x 3,072 -> 768 180
// and 208, 65,536 x 256 -> 1,024 64 and 71; 10,242 x 3,072 -> 768 72 and 50, 40,962 x 128 -> 512 20 and 18. Ranges: the
// weight's gradient over 40,962 rows of 768 -> 3,072 takes 840 and 492 with one and 187 with the ones taken here.
struct Plan {
  int tile;
  int32_t splits, chunk;
  double time = 0;
};

struct Cost {
  int tile;  // rows, and columns (128 at least)
  double alone, full, ends;  // a stage of the one workgroup on a CU, of one among those that fill it, a workgroup's ends
};

// `widened`: e4m3 operands multiplied as bf16, twice the products of a stage of bf16.
Plan plan(Operands how, int64_t m, int64_t n, int64_t k, int32_t op, bool widened) {
  constexpr Cost bf16[] = {{256, 1.55, 1.55, 9.0}, {128, 0.6, 0.5, 1.8}}, f32[] = {{128, 2.0, 1.1, 3.0}, {64, 1.1, 0.66, 2.0}};
  const int64_t of = op == kOpF32 ? kStageF32 : op == kOpE4m3 ? kStageBytes : kStageRows;
  const int64_t stages = std::max<int64_t>(1, parts(k, of));
  Plan best{128, 1, (int32_t)stages};
  double least = -1;
  for (int t = 0; t < (op == kOpF32 && how == Operands::kOuterOuter ? 1 : 2); ++t) {
    const Cost& c = op == kOpF32 ? f32[t] : bf16[t];
    const int64_t tiles = parts(m, c.tile) * parts(n, std::max(c.tile, 128));
    for (int64_t want = 1; want <= 64; ++want) {
      const int64_t chunk = parts(stages, want), splits = parts(stages, chunk);
      if (splits != want) continue;
      if (want > 1 && (chunk < 2 || tiles * want > 4 * kCus)) break;
      const int64_t load = parts(tiles * splits, kCus);
      const double join = splits > 1 ? 4.0 + (double)(splits + 1) * m * n * 4 / 4e6 : 0;
      const double time = load * (chunk * (load == 1 ? c.alone : c.full) * (widened ? 2 : 1) + c.ends) + join;
      if (least < 0 || time < least) {
        least = time;
        best = {c.tile, (int32_t)splits, (int32_t)chunk, time};
      }
    }
  }
  return best;
}

// How a product of bf16 rows with a 4-bit weight is formed, by an estimate of its time in us: the few rows' kernel (tile -1), tiles
// that take the codes (tile: their waves), or a widened weight and its plan (tile 0). Measured on one machine, from captured graphs,
// and estimated: 24 rows of 5,120 -> 8,192 16 in few rows, 21 in tiles; 32 of 16,384 -> 4,096 38 and 24; 512 of 4,096 -> 8,192 36 in
// tiles of four waves (38 to 40 on others), 39 of two, 62 widened; 2,048 of 2,048 -> 4,096 41 in tiles, 40 widened.
Plan plan_q4(int64_t m, int64_t n, int64_t k) {
  Plan best{0, 1, 0};
  const double weights = (double)n * k;
  double least = plan(Operands::kInnerInner, m, n, k, kOpBf16, false).time + 3.0 + weights * 2.53 / 4.6e6;
  if (m <= kFewRows) {
    // Each workgroup of 16 or 32 outputs reads all rows.
    const double reads = (double)parts(n, n > 16 * kCus ? 32 : 16) * m * k * 2;
    least = 3.0 + std::max(weights * 0.53 / 4e6, reads / 6e6);
    best.tile = -1;
  }
  const int64_t spans = std::max<int64_t>(1, parts(k, kQ4Span));
  for (int waves = 2; waves <= 4; waves += 2) {
    const int64_t tiles = parts(m, 64) * parts(n, 64 * waves), at_once = waves == 2 ? 2 * kCus : kCus;
    for (int64_t want = 1; want <= 16; ++want) {
      const int64_t chunk = parts(spans, want), splits = parts(spans, chunk), load = tiles * splits;
      if (splits != want) continue;
      if (want > 1 && (chunk < 2 || load > 2 * at_once)) break;
      const double span = waves == 2 ? (load <= kCus ? 0.8 : 1.08) : (load <= kCus / 2 ? 0.86 : 1.0);
      const double join = splits > 1 ? 5.0 + (double)(splits + 1) * m * n * 4 / 2.5e6 : 0;
      const double time = parts(load, at_once) * (chunk * span + 4.0) + join;
      if (time < least) {
        least = time;
        best = {waves, (int32_t)splits, (int32_t)chunk};
      }
    }
  }
  return best;
}

// One product's launch: its plan, operands and workspace.
struct Product {
  ProductArgs g{};
  Operands how;
  int32_t op;
  Plan p;
  bool few;  // rows: no tiles

  // `sums`: the column sums of a are wanted. `dtype`: of the outputs.
  // `given`: the plan, of a kernel of its own.
  void shape(Operands h, int64_t m, int64_t n, int64_t k, int32_t o, int32_t dtype, bool sums, Workspace& ws,
             const Plan* given = nullptr) {
    how = h, op = o;
    few = !given && how == Operands::kInnerInner && m <= kFewRows;
    p = given ? *given : few ? Plan{0, 1, 0} : plan(how, m, n, k, op, op == kOpE4m3 && dtype == FWN_F32);
    g.k = k;
    g.splits = p.splits;
    g.chunk = p.chunk;
    g.e.m = m;
    g.e.n = n;
    g.part_row = up(n, 8);
    g.part = p.splits > 1 ? (float*)ws.take((uint64_t)p.splits * m * g.part_row * sizeof(float)) : nullptr;
    g.sums = sums && p.splits > 1 ? (float*)ws.take((uint64_t)p.splits * m * sizeof(float)) : nullptr;
  }

  hipError_t launch(const Matrix& a, const Matrix& b, hipStream_t stream) {
    g.a = a.at, g.a_stride = a.row_bytes;
    g.b = b.at, g.b_stride = b.row_bytes;
    finish();
    return few ? launch_product_rows(op, g, stream) : launch_product(how, op, p.tile, g, stream);
  }

  // What the epilogue's arguments imply.
  void finish() {
    const EpilogueArgs& e = g.e;
    g.e.vec = e.n % 8 == 0 && (!e.residual || e.r_row % 8 == 0) &&
              (((uintptr_t)e.out | (uintptr_t)e.pre | (uintptr_t)e.residual) & 15) == 0;
  }
};

// Where everything of one forward launch lies; without a workspace, how large that has to be.
struct Forward {
  Matrix x, w;
  Product z;
  uint64_t bytes;

  Forward(const fwn_linear_desc* d, int32_t op, const void* xp, const void* wp, void* workspace) {
    Workspace ws{(char*)workspace};
    x.place(xp, d->rows, d->ins, d->x_stride, op, ws);
    w.place(wp, d->outs, d->ins, d->w_stride, op, ws);
    z.shape(Operands::kInnerInner, d->rows, d->outs, d->ins, op, d->dtype, false, ws);
    bytes = ws.used;
  }
};

int forward(const fwn_linear_desc* d, int32_t op, const void* x, const float* x_scale, const void* weight,
            const float* w_scale, const void* bias, const void* residual, void* out, void* pre, void* workspace,
            uint64_t workspace_bytes, void* stream, const char* what) {
  if (int rc = check_desc(d, what)) return rc;
  if (d->rows == 0) return FWN_OK;
  if (!x || !weight || !out || (op == kOpE4m3 && (!x_scale || !w_scale)))
    return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  const uint64_t size = size_of(d->dtype), in_size = (uint64_t)op_size(op);
  if (misaligned(x, in_size) || misaligned(weight, in_size) || misaligned(x_scale, 4) || misaligned(w_scale, 4) ||
      misaligned(bias, size) || misaligned(residual, size) || misaligned(out, size) || misaligned(pre, size))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned to its elements", what);
  const Span ins[] = {span(x, d->rows, d->x_stride, d->ins, in_size), span(weight, d->outs, d->w_stride, d->ins, in_size),
                      span(x_scale, 1, 0, d->rows, 4), span(w_scale, 1, 0, d->outs, 4), span(bias, 1, 0, d->outs, size),
                      span(residual, d->rows, d->r_stride, d->outs, size)};
  const Span outs[] = {span(out, d->rows, d->outs, d->outs, size), span(pre, d->rows, d->outs, d->outs, size)};
  if (int rc = check_overlap(ins, outs, what)) return rc;
  Forward f(d, op, x, weight, workspace);
  if (int rc = check_workspace(workspace, workspace_bytes, f.bytes, what)) return rc;
  EpilogueArgs& e = f.z.g.e;
  e.a_scale = x_scale;
  e.b_scale = w_scale;
  e.bias = bias;
  e.residual = residual;
  e.r_row = d->r_stride;
  e.out = out;
  e.pre = pre;
  e.dtype = d->dtype;
  e.activation = d->activation;
  const hipStream_t s = (hipStream_t)stream;
  if (int rc = status(f.x.lay_out(s), what)) return rc;
  if (int rc = status(f.w.lay_out(s), what)) return rc;
  return status(f.z.launch(f.x, f.w, s), what);
}

// Rows of a workgroup in the dz pass: about four workgroups a CU, 32 rows at least; up to 128 rows one workgroup sums
// a column, which saves the launch that joins the sums.
int64_t slope_chunk(int64_t rows, int64_t outs) {
  if (rows <= 128) return std::max<int64_t>(1, rows);
  const int64_t blocks = std::max<int64_t>(1, std::min(4 * kCus / parts(outs, 256), parts(rows, 32)));
  return std::max<int64_t>(1, parts(rows, blocks));
}

// The backward: dz (g itself where it is bf16 without an activation), its column sums, and the two products. The
// sums come from the weight gradient's product where that reads g itself, else from the pass that forms dz.
struct Backward {
  Matrix dz, w, x;
  Product to_x, to_w;
  SlopeArgs slope{};
  bool formed, sums_in_product;
  uint64_t bytes;

  Backward(const fwn_linear_desc* d, const void* xp, const void* wp, const void* gp, bool need_x, bool need_w, bool need_b,
           void* workspace) {
    Workspace ws{(char*)workspace};
    const int32_t op = d->dtype == FWN_F32 ? kOpF32 : kOpBf16;
    const bool act = d->activation != FWN_ACT_NONE, products = need_x || need_w;
    dz.place(gp, d->rows, d->outs, d->outs, op, ws, act);
    formed = products && dz.laid;
    sums_in_product = need_b && need_w && !formed && op == kOpBf16;
    slope.chunk = slope_chunk(d->rows, d->outs);
    slope.blocks = (int32_t)std::max<int64_t>(1, parts(d->rows, slope.chunk));
    if (need_b && !sums_in_product && slope.blocks > 1) slope.part = (float*)ws.take((uint64_t)slope.blocks * d->outs * sizeof(float));
    if (need_x) {
      w.place(wp, d->outs, d->ins, d->w_stride, op, ws);
      to_x.shape(Operands::kInnerOuter, d->rows, d->ins, d->outs, op, d->dtype, false, ws);
    }
    if (need_w) {
      x.place(xp, d->rows, d->ins, d->x_stride, op, ws);
      to_w.shape(Operands::kOuterOuter, d->outs, d->ins, d->rows, op, d->dtype, sums_in_product, ws);
    }
    bytes = ws.used;
  }
};

// The same with a weight of 4 bits: read as it is for few rows and by the tiles of bf16, widened in the workspace for float32's.
struct ForwardQ4 {
  Matrix x, w{}, scales{};
  Product z;
  int64_t groups;
  int waves = 0;  // of a tile that takes the codes
  uint64_t bytes;

  ForwardQ4(const fwn_linear_desc* d, const void* xp, const uint8_t* sp, void* workspace) {
    Workspace ws{(char*)workspace};
    const int32_t op = d->dtype == FWN_F32 ? kOpF32 : kOpBf16;
    groups = parts(d->ins, FWN_Q4_GROUP);
    x.place(xp, d->rows, d->ins, d->x_stride, op, ws);
    const Plan p = op == kOpBf16 && d->rows > 16 ? plan_q4(d->rows, d->outs, d->ins) : Plan{0, 1, 0};
    waves = p.tile > 0 ? p.tile : 0;
    z.shape(Operands::kInnerInner, d->rows, d->outs, d->ins, op, d->dtype, false, ws, waves ? &p : nullptr);
    scales.at = (char*)sp;
    scales.row_bytes = groups;
    if (waves && (groups % 4 || ((uintptr_t)sp & 3))) scales.place(sp, d->outs, groups, groups, kOpE4m3, ws, true);
    if (!z.few && !waves) {
      w.row_bytes = groups * FWN_Q4_GROUP * op_size(op);
      w.at = ws.take((uint64_t)d->outs * (uint64_t)w.row_bytes);
    }
    bytes = ws.used;
  }
};

int size_query(const fwn_linear_desc* d, uint64_t* bytes, const char* what) {
  clear_error();
  if (!bytes) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  *bytes = 0;
  return check_desc(d, what);
}

}  // namespace
}  // namespace fwn

extern "C" {

int fwn_linear_act_workspace_size(const fwn_linear_desc* d, const void* x, const void* weight, uint64_t* bytes) {
  using namespace fwn;
  if (int rc = size_query(d, bytes, "fwn_linear_act_workspace_size")) return rc;
  *bytes = Forward(d, d->dtype == FWN_F32 ? kOpF32 : kOpBf16, x, weight, nullptr).bytes;
  return FWN_OK;
}

int fwn_linear_act_launch(const fwn_linear_desc* d, const void* x, const void* weight, const void* bias,
                          const void* residual, void* out, void* pre, void* workspace, uint64_t workspace_bytes,
                          void* stream) {
  using namespace fwn;
  clear_error();
  return forward(d, d && d->dtype == FWN_F32 ? kOpF32 : kOpBf16, x, nullptr, weight, nullptr, bias, residual, out, pre,
                 workspace, workspace_bytes, stream, "fwn_linear_act_launch");
}

int fwn_linear_act_q8_workspace_size(const fwn_linear_desc* d, const uint8_t* x, const uint8_t* weight, uint64_t* bytes) {
  using namespace fwn;
  if (int rc = size_query(d, bytes, "fwn_linear_act_q8_workspace_size")) return rc;
  *bytes = Forward(d, kOpE4m3, x, weight, nullptr).bytes;
  return FWN_OK;
}

int fwn_linear_act_q8_launch(const fwn_linear_desc* d, const uint8_t* x, const float* x_scale, const uint8_t* weight,
                             const float* w_scale, const void* bias, const void* residual, void* out,
                             void* workspace, uint64_t workspace_bytes, void* stream) {
  using namespace fwn;
  clear_error();
  return forward(d, kOpE4m3, x, x_scale, weight, w_scale, bias, residual, out, nullptr, workspace, workspace_bytes,
                 stream, "fwn_linear_act_q8_launch");
}

int fwn_quantize_q4_launch(int64_t rows, int32_t ins, int64_t x_stride, int32_t dtype, const void* x, uint8_t* codes,
                           uint8_t* scales, void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_quantize_q4_launch";
  if (dtype != FWN_F32 && dtype != FWN_BF16) return fail(FWN_ERR_UNSUPPORTED, "%s: dtype must be f32 or bf16", what);
  if (ins < 1 || ins > FWN_LINEAR_ACT_MAX) return fail(FWN_ERR_INVALID_ARG, "%s: ins %d must be 1 to %d", what, ins, FWN_LINEAR_ACT_MAX);
  if (rows < 0 || rows > FWN_LINEAR_ACT_MAX || x_stride < 0 || x_stride > FWN_LINEAR_STRIDE_MAX)
    return fail(FWN_ERR_INVALID_ARG, "%s: %lld rows, stride %lld", what, (long long)rows, (long long)x_stride);
  if (rows == 0) return FWN_OK;
  if (!x || !codes || !scales) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  const uint64_t size = size_of(dtype);
  if (misaligned(x, size) || misaligned(codes, 16)) return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned", what);
  const int64_t groups = parts(ins, FWN_Q4_GROUP);
  const Span in[] = {span(x, rows, x_stride, ins, size)};
  const Span outs[] = {span(codes, rows, groups * 16, groups * 16, 1), span(scales, rows, groups, groups, 1)};
  if (int rc = check_overlap(in, outs, what)) return rc;
  return status(launch_quantize_q4(dtype, {x, codes, scales, rows, ins, x_stride}, (hipStream_t)stream), what);
}

int fwn_linear_act_q4_workspace_size(const fwn_linear_desc* d, const void* x, const uint8_t* scales, uint64_t* bytes) {
  using namespace fwn;
  if (int rc = size_query(d, bytes, "fwn_linear_act_q4_workspace_size")) return rc;
  *bytes = ForwardQ4(d, x, scales, nullptr).bytes;
  return FWN_OK;
}

int fwn_linear_act_q4_launch(const fwn_linear_desc* d, const void* x, const uint8_t* codes, const uint8_t* scales,
                             const void* bias, const void* residual, void* out, void* workspace, uint64_t workspace_bytes,
                             void* stream) {
  using namespace fwn;
  clear_error();
  const char* what = "fwn_linear_act_q4_launch";
  if (int rc = check_desc(d, what)) return rc;
  if (d->rows == 0) return FWN_OK;
  if (!x || !codes || !scales || !out) return fail(FWN_ERR_INVALID_ARG, "%s: null argument", what);
  const uint64_t size = size_of(d->dtype);
  if (misaligned(x, size) || misaligned(codes, 16) || misaligned(bias, size) || misaligned(residual, size) || misaligned(out, size))
    return fail(FWN_ERR_INVALID_ARG, "%s: a tensor is not aligned", what);
  ForwardQ4 f(d, x, scales, workspace);
  if (int rc = check_workspace(workspace, workspace_bytes, f.bytes, what)) return rc;
  const Span ins[] = {span(x, d->rows, d->x_stride, d->ins, size), span(codes, d->outs, f.groups * 16, f.groups * 16, 1),
                      span(scales, d->outs, f.groups, f.groups, 1), span(bias, 1, 0, d->outs, size),
                      span(residual, d->rows, d->r_stride, d->outs, size)};
  const Span outs[] = {span(out, d->rows, d->outs, d->outs, size), {workspace, f.bytes}};
  if (int rc = check_overlap(ins, outs, what)) return rc;
  EpilogueArgs& e = f.z.g.e;
  e.bias = bias;
  e.residual = residual;
  e.r_row = d->r_stride;
  e.out = out;
  e.dtype = d->dtype;
  e.activation = d->activation;
  const hipStream_t s = (hipStream_t)stream;
  const bool f32 = d->dtype == FWN_F32;
  if (int rc = status(f.x.lay_out(s), what)) return rc;
  if (f.z.few || f.waves) {
    f.z.finish();
    if (int rc = status(f.scales.lay_out(s), what)) return rc;
    Q4Args a{f.z.g, codes, (const uint8_t*)f.scales.at, f.groups, f.scales.row_bytes};
    a.p.a = f.x.at;
    a.p.a_stride = f.x.row_bytes;
    return status(f.waves ? launch_q4_tiles(f.waves, a, s) : launch_q4_rows(f32, a, s), what);
  }
  if (int rc = status(launch_widen(f32, {codes, scales, f.w.at, d->outs, d->ins, f.groups}, s), what)) return rc;
  return status(f.z.launch(f.x, f.w, s), what);
}

int fwn_linear_act_bwd_workspace_size(const fwn_linear_desc* d, const void* x, const void* weight, const void* g,
                                      const void* gx, const void* gw, const void* gb, uint64_t* bytes) {
  using namespace fwn;
  if (int rc = size_query(d, bytes, "fwn_linear_act_bwd_workspace_size")) return rc;
  *bytes = Backward(d, x, weight, g, gx && d->rows > 0, gw != nullptr, gb != nullptr, nullptr).bytes;
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
  Backward b(d, x, weight, g, gx && d->rows > 0, gw != nullptr, gb != nullptr, workspace);
  if (int rc = check_workspace(workspace, workspace_bytes, b.bytes, what)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  if (b.formed || (gb && !b.sums_in_product)) {
    SlopeArgs& a = b.slope;
    a.g = g;
    a.pre = pre;
    a.dz = b.formed ? b.dz.at : nullptr;
    a.dz_stride = b.dz.row_bytes;
    a.rows = d->rows;
    a.outs = d->outs;
    a.dtype = d->dtype;
    a.activation = d->activation;
    a.gb = gb && !b.sums_in_product && a.blocks == 1 ? gb : nullptr;
    if (int rc = status(launch_slope(a, s), what)) return rc;
    if (gb && !b.sums_in_product && a.blocks > 1)
      if (int rc = status(launch_column_sums(a.part, a.blocks, d->outs, gb, d->dtype, s), what)) return rc;
  }
  if (gx && d->rows > 0) {
    if (int rc = status(b.w.lay_out(s), what)) return rc;
    b.to_x.g.e.out = gx;
    b.to_x.g.e.dtype = d->dtype;
    if (int rc = status(b.to_x.launch(b.dz, b.w, s), what)) return rc;
  }
  if (gw) {
    if (int rc = status(b.x.lay_out(s), what)) return rc;
    b.to_w.g.e.out = gw;
    b.to_w.g.e.dtype = d->dtype;
    b.to_w.g.sums_out = b.sums_in_product && b.to_w.p.splits == 1 ? gb : nullptr;
    if (int rc = status(b.to_w.launch(b.dz, b.x, s), what)) return rc;
    if (b.sums_in_product && b.to_w.p.splits > 1)
      if (int rc = status(launch_column_sums(b.to_w.g.sums, b.to_w.p.splits, d->outs, gb, d->dtype, s), what)) return rc;
  }
  return FWN_OK;
}

}  // extern "C"
