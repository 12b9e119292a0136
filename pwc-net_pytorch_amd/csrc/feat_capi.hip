// feat_capi.hip — the extern "C" boundary of the feature operators (layer norm, rotary positions,
// linear, gated linear) declared in include/pwc_hotpath.h.
#include "../../include/pwc_hotpath.h"
#include "feat_norm.cuh"
#include "feat_product.cuh"
#include "feat_rotary.cuh"

namespace {
using namespace pwc;
using namespace pwc::feat;

constexpr long long kIntMax = 0x7fffffffLL;

// NULL if the matrix of tokens / pixels and channels can be worked on
const char* bad_shape(int layout, long long B, long long P, long long C, int dtype) {
  if (dtype < 0 || dtype > 2) return "unsupported dtype";
  if (layout != PWC_LAYOUT_MAP && layout != PWC_LAYOUT_TOKENS) return "unknown layout";
  if (B < 0 || P < 0 || C < 0) return "negative dimension";
  if (C == 0) return "no channels";
  if (layout == PWC_LAYOUT_TOKENS && B != 1) return "tokens have one batch (B must be 1)";
  // counts of values stay far below 2^63, whatever is multiplied with them
  if (B > kIntMax || P > kIntMax || C > (1 << 24)) return "dimension too large";
  if (B > 0 && P > 0 && B * P > (1LL << 40) / C) return "dimension too large";
  return nullptr;
}

const char* bad_stride(int layout, long long B, long long P, long long C, long long stride) {
  const long long rows = layout == PWC_LAYOUT_MAP ? B : P;
  const long long least = layout == PWC_LAYOUT_MAP ? P * C : C;
  // a row repeated (stride 0) or overlapped is never what a caller means
  if (rows > 1 && stride < least) return "stride smaller than a token / an image";
  if (stride > (1LL << 40)) return "stride too large";
  return nullptr;
}

ProductArgs blank() {
  ProductArgs g = {};
  g.segments = g.batches = g.splits = 1;
  return g;
}

// what the four entries of the products share
struct Problem {
  int layout, K, O, rows, act, dtype, gated;  // rows of W: O, or 2 O
  long long B, P, M, x_stride;
  float slope;
};

const char* bad_problem(const Problem& p) {
  if (const char* e = bad_shape(p.layout, p.B, p.P, p.K, p.dtype)) return e;
  if (p.O <= 0 || p.O > (1 << 23)) return "bad number of output channels";
  if (p.M > kIntMax) return "dimension too large";
  if (p.act < 0 || p.act > kActGeluTanh) return "unknown activation";
  if (p.M > (1LL << 40) / p.rows || (long long)p.rows * p.K > (1LL << 40))
    return "dimension too large";
  return bad_stride(p.layout, p.B, p.P, p.K, p.x_stride);
}

Problem problem(int layout, long long B, long long P, int K, int O, long long x_stride, int act,
                float slope, int dtype, int gated) {
  Problem p = {layout, K, O, gated ? 2 * O : O, act, dtype, gated, B, P, 0, x_stride, slope};
  p.M = layout == PWC_LAYOUT_MAP && B >= 0 && P >= 0 && B <= kIntMax && P <= kIntMax ? B * P : P;
  return p;
}

// z = x W^T + b into the epilogue `mode`, whose output has `out_rows` channels
ProductArgs forward_args(const Problem& p, const void* x, const void* w, const void* bias,
                         const void* other, void* out, int mode, int out_rows) {
  ProductArgs g = blank();
  g.K = p.K;
  g.bias = bias;
  g.other = other;
  g.out = out;
  g.mode = mode;
  g.act = p.act;
  g.slope = p.slope;
  g.pair = p.gated ? p.O : 0;
  if (p.layout == PWC_LAYOUT_TOKENS) {
    g.a = w, g.lda = p.K, g.a_k = 1, g.I = p.rows;
    g.b = x, g.ldb = p.x_stride, g.b_k = 1, g.J = (int)p.M;
    g.ldo = out_rows;
    g.ldother = p.O;
    g.channel_i = 1;
  } else {
    g.a = x, g.lda = p.P, g.a_batch = p.x_stride, g.a_k = 0, g.I = (int)p.P;
    g.b = w, g.ldb = p.K, g.b_k = 1, g.J = p.rows;
    g.batches = (int)p.B;
    g.ldo = p.P, g.out_batch = (long long)out_rows * p.P;
    g.ldother = p.P, g.other_batch = (long long)p.O * p.P;
  }
  return g;
}

bool needs_z(const Problem& p) { return p.gated || p.act != kActNone; }
size_t elem(int dtype) { return dtype == 0 ? 4 : 2; }

ProductArgs dz_args(const Problem& p, const void* x, const void* w, const void* bias,
                    const void* dy, void* dz) {
  return forward_args(p, x, w, bias, dy, dz, p.gated ? kGatedDz : kLinearDz, p.rows);
}
// dW = dz^T x in 32-bit parts (`out`), or itself where there is one split
ProductArgs dw_args(const Problem& p, const void* x, const void* dz, void* out) {
  ProductArgs g = blank();
  g.mode = kPartial;
  g.out = out;
  g.I = p.K;
  g.J = p.rows;
  g.ldo = p.K;
  if (p.layout == PWC_LAYOUT_TOKENS) {
    g.K = (int)p.M;
    g.a = x, g.lda = p.x_stride, g.a_k = 0;
    g.b = dz, g.ldb = p.rows, g.b_k = 0;
  } else {
    g.K = (int)p.P;
    g.segments = (int)p.B;
    g.a = x, g.lda = p.P, g.a_segment = p.x_stride, g.a_k = 1;
    g.b = dz, g.ldb = p.P, g.b_segment = (long long)p.rows * p.P, g.b_k = 1;
  }
  return g;
}

struct BackwardSpace {
  size_t part, sums, total;  // bytes from the start; dz lies at 0
  int splits, rows;          // rows of partial bias gradients
};
BackwardSpace backward_space(const Problem& p, int splits, int rows) {
  BackwardSpace s = {};
  s.splits = splits;
  s.rows = rows;
  s.part = needs_z(p) ? align256((size_t)p.M * p.rows * elem(p.dtype)) : 0;
  s.sums = s.part + (splits > 1 ? align256((size_t)splits * p.rows * p.K * 4) : 0);
  s.total = s.sums + align256((size_t)rows * p.rows * 4);
  return s;
}
// (of the pointers only the alignment matters)
int dw_splits(const Problem& p, const void* x, const void* dz) {
  return product_plan(dw_args(p, x, dz, nullptr), p.dtype).splits;
}
int db_rows(const Problem& p, const void* x, const void* w) {
  return needs_z(p) ? product_sum_rows(dz_args(p, x, w, nullptr, nullptr, nullptr), p.dtype)
                    : product_column_parts(p.layout, p.B, p.P, p.rows);
}
size_t most_backward_space(const Problem& p) {
  if (bad_problem(p) || p.M == 0) return 0;
  int splits = 0, rows = 0;
  for (const void* at : {(const void*)nullptr, (const void*)1}) {
    const int s = dw_splits(p, at, at), r = db_rows(p, at, at);
    if (s > splits) splits = s;
    if (r > rows) rows = r;
  }
  return backward_space(p, splits, rows).total;
}

int product_backward(const char* fn, const Problem& p, const void* x, const void* w,
                     const void* bias, const void* dy, void* dx, void* dw, void* db,
                     void* workspace, size_t bytes, hipStream_t stream) {
  if (const char* e = bad_problem(p)) return api_fail(fn, e);
  if (p.M == 0) {  // sums over no tokens
    hipError_t e = hipSuccess;
    if (dw) e = product_add_splits(nullptr, dw, (long long)p.rows * p.K, 0, p.dtype, stream);
    if (db && e == hipSuccess) e = product_add_splits(nullptr, db, p.rows, 0, p.dtype, stream);
    return api_launch(fn, e);
  }
  if (!x || !w || !dy) return api_fail(fn, "null buffer");
  if (!dx && !dw && !db) return api_launch(fn, hipSuccess);
  const BackwardSpace s = backward_space(
      p, dw ? dw_splits(p, x, needs_z(p) ? nullptr : dy) : 1, db ? db_rows(p, x, w) : 0);
  if (s.total > 0 && (!workspace || bytes < s.total)) return api_fail(fn, "workspace too small");
  if (!aligned_to(workspace, 256)) return api_fail(fn, "workspace not aligned");
  char* ws = (char*)workspace;
  const void* dz = dy;
  if (needs_z(p)) {
    ProductArgs g = dz_args(p, x, w, bias, dy, ws);
    g.sums = db ? (float*)(ws + s.sums) : nullptr;
    const hipError_t e = product_launch(g, p.dtype, stream);
    if (e != hipSuccess) return api_launch(fn, e);
    dz = ws;
  }
  const long long dz_image = (long long)p.rows * p.P;
  if (dx) {
    ProductArgs g = blank();
    g.K = p.rows;
    g.out = dx;
    g.mode = kPlain;
    if (p.layout == PWC_LAYOUT_TOKENS) {
      g.a = w, g.lda = p.K, g.a_k = 0, g.I = p.K;
      g.b = dz, g.ldb = p.rows, g.b_k = 1, g.J = (int)p.M;
      g.ldo = p.K;
    } else {
      g.a = dz, g.lda = p.P, g.a_batch = dz_image, g.a_k = 0, g.I = (int)p.P;
      g.b = w, g.ldb = p.K, g.b_k = 0, g.J = p.K;
      g.batches = (int)p.B;
      g.ldo = p.P, g.out_batch = (long long)p.K * p.P;
    }
    const hipError_t e = product_launch(g, p.dtype, stream);
    if (e != hipSuccess) return api_launch(fn, e);
  }
  if (dw) {
    ProductArgs g = dw_args(p, x, dz, s.splits > 1 ? (void*)(ws + s.part) : dw);
    g.splits = s.splits;
    hipError_t e = product_launch(g, p.dtype, stream);
    if (e == hipSuccess && s.splits > 1)
      e = product_add_splits((const float*)(ws + s.part), dw, (long long)p.rows * p.K, s.splits,
                             p.dtype, stream);
    if (e != hipSuccess) return api_launch(fn, e);
  }
  if (db) {
    float* sums = (float*)(ws + s.sums);
    hipError_t e = hipSuccess;
    if (!needs_z(p))
      e = product_column_sums(dy, sums, p.layout, p.B, p.P, p.rows, s.rows, p.dtype, stream);
    if (e == hipSuccess) e = sum_rows(sums, db, p.rows, s.rows, p.dtype, stream);
    if (e != hipSuccess) return api_launch(fn, e);
  }
  return api_launch(fn, hipSuccess);
}

int product_forward(const char* fn, const Problem& p, const void* x, const void* w,
                    const void* bias, const void* res, void* y, hipStream_t stream) {
  if (const char* e = bad_problem(p)) return api_fail(fn, e);
  if (p.M == 0) return api_launch(fn, hipSuccess);
  if (!x || !w || !y) return api_fail(fn, "null buffer");
  return api_launch(fn, product_launch(forward_args(p, x, w, bias, res, y,
                                                    p.gated ? kGated : kLinear, p.O),
                                       p.dtype, stream));
}

NormArgs norm_args(int layout, long long B, long long P, int C, long long x_stride) {
  NormArgs a = {};
  a.layout = layout;
  a.B = B;
  a.P = P;
  a.M = B * P;
  a.C = C;
  a.x_stride = x_stride;
  return a;
}
const char* bad_norm(int layout, long long B, long long P, int C, long long x_stride, int dtype) {
  if (const char* e = bad_shape(layout, B, P, C, dtype)) return e;
  // one block a row (tokens) or a 64-pixel tile (maps)
  if (B * ((P + 63) / 64) > kIntMax) return "dimension too large";
  return bad_stride(layout, B, P, C, x_stride);
}
}  // namespace

extern "C" {

PWC_API int pwc_layer_norm_forward(const void* x, const void* weight, const void* bias, void* y,
                                   void* mean, void* rstd, int layout, long long B, long long P,
                                   int C, long long x_stride, float eps, int dtype, void* stream) {
  const char* fn = "pwc_layer_norm_forward";
  if (const char* e = bad_norm(layout, B, P, C, x_stride, dtype)) return api_fail(fn, e);
  if (!(eps >= 0.f)) return api_fail(fn, "eps must not be negative");
  if ((mean == nullptr) != (rstd == nullptr)) return api_fail(fn, "mean and rstd come together");
  if (B * P == 0) return api_launch(fn, hipSuccess);
  if (!x || !y) return api_fail(fn, "null buffer");
  NormArgs a = norm_args(layout, B, P, C, x_stride);
  a.x = x;
  a.w = weight;
  a.b = bias;
  a.y = y;
  a.mean = (float*)mean;
  a.rstd = (float*)rstd;
  a.eps = eps;
  return api_launch(fn, norm_forward(a, dtype, (hipStream_t)stream));
}

PWC_API size_t pwc_layer_norm_backward_workspace_size(int layout, long long B, long long P, int C,
                                                      int dtype) {
  if (bad_shape(layout, B, P, C, dtype)) return 0;
  return align256((size_t)2 * norm_parts(layout, B, P, C, dtype) * C * sizeof(float));
}

PWC_API int pwc_layer_norm_backward(const void* x, const void* weight, const void* grad_out,
                                    const void* mean, const void* rstd, void* grad_x,
                                    void* grad_weight, void* grad_bias, int layout, long long B,
                                    long long P, int C, long long x_stride, int dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "pwc_layer_norm_backward";
  if (const char* e = bad_norm(layout, B, P, C, x_stride, dtype)) return api_fail(fn, e);
  const bool sums = grad_weight || grad_bias;
  if (!grad_x && !sums) return api_launch(fn, hipSuccess);
  NormArgs a = norm_args(layout, B, P, C, x_stride);
  if (a.M > 0 && (!x || !grad_out || !mean || !rstd)) return api_fail(fn, "null buffer");
  const int parts = norm_parts(layout, B, P, C, dtype);
  const size_t need = (size_t)2 * parts * C * sizeof(float);
  if (sums && need > 0 && (!workspace || workspace_bytes < need))
    return api_fail(fn, "workspace too small");
  a.x = x;
  a.w = weight;
  a.dy = grad_out;
  a.mean = (float*)mean;
  a.rstd = (float*)rstd;
  a.dx = grad_x;
  a.dw = grad_weight;
  a.db = grad_bias;
  a.part = sums ? (float*)workspace : nullptr;
  if (a.M == 0)
    return api_launch(fn, sums ? norm_no_rows(a, dtype, (hipStream_t)stream) : hipSuccess);
  return api_launch(fn, norm_backward(a, parts, dtype, (hipStream_t)stream));
}

PWC_API int pwc_rotary(const void* x, void* y, const void* positions, const void* inv_freq,
                       const void* axis, const pwc_rotary_shape* shape, int inverse, int dtype,
                       void* stream) {
  const char* fn = "pwc_rotary";
  if (dtype < 0 || dtype > 2) return api_fail(fn, "unsupported dtype");
  if (!shape) return api_fail(fn, "null shape");
  const pwc_rotary_shape& s = *shape;
  if (s.B < 0 || s.N < 0 || s.heads < 0 || s.D < 0) return api_fail(fn, "negative dimension");
  if (s.B > kIntMax || s.N > kIntMax || s.heads > (1 << 20) || s.D > (1 << 20))
    return api_fail(fn, "dimension too large");
  if (s.pairs < 0 || 2LL * s.pairs > s.D) return api_fail(fn, "more pairs than channels");
  if (s.axes < 1 || s.axes > kMaxAxes) return api_fail(fn, "1 to 4 axes");
  if (positions) {
    if (s.position_type < 0 || s.position_type > 2) return api_fail(fn, "unknown position type");
  } else {
    long long n = 1;
    for (int k = 0; k < s.axes; ++k) {
      if (s.grid[k] < 0 || s.grid[k] > kIntMax) return api_fail(fn, "bad grid");
      if (n > 0 && s.grid[k] > kIntMax / n) return api_fail(fn, "grid is not the tokens");
      n *= s.grid[k];
      if (s.origin[k] > (1LL << 52) || s.origin[k] < -(1LL << 52))
        return api_fail(fn, "bad origin");
    }
    if (n != s.N) return api_fail(fn, "grid is not the tokens");
  }
  const long long count = s.B * s.N;  // < 2^62
  if (count > 0 && (long long)s.heads * s.D > (1LL << 42) / count)
    return api_fail(fn, "dimension too large");
  if (count == 0 || s.heads == 0 || s.D == 0) return api_launch(fn, hipSuccess);
  if (!x || !y || (s.pairs > 0 && (!inv_freq || !axis))) return api_fail(fn, "null buffer");
  RotaryArgs a = {};
  a.x = x;
  a.y = y;
  a.positions = positions;
  a.inv_freq = (const double*)inv_freq;
  a.axis = (const int*)axis;
  a.xs_b = s.x_stride[0], a.xs_n = s.x_stride[1], a.xs_h = s.x_stride[2], a.xs_d = s.x_stride[3];
  a.ys_b = s.y_stride[0], a.ys_n = s.y_stride[1], a.ys_h = s.y_stride[2], a.ys_d = s.y_stride[3];
  a.pos_b = s.position_stride[0], a.pos_n = s.position_stride[1], a.pos_a = s.position_stride[2];
  a.B = s.B;
  a.N = s.N;
  a.H = s.heads;
  a.D = s.D;
  a.R = s.pairs;
  a.axes = s.axes;
  a.pos_type = s.position_type;
  a.interleaved = s.interleaved;
  for (int k = 0; k < s.axes; ++k) {
    a.grid[k] = s.grid[k];
    a.origin[k] = s.origin[k];
  }
  a.sign = inverse ? -1.f : 1.f;
  return api_launch(fn, rotary_launch(a, dtype, (hipStream_t)stream));
}

PWC_API int pwc_linear_forward(const void* x, const void* weight, const void* bias,
                               const void* residual, void* y, int layout, long long B, long long P,
                               int K, int O, long long x_stride, int activation,
                               float negative_slope, int dtype, void* stream) {
  return product_forward("pwc_linear_forward",
                         problem(layout, B, P, K, O, x_stride, activation, negative_slope, dtype, 0),
                         x, weight, bias, residual, y, (hipStream_t)stream);
}

PWC_API size_t pwc_linear_backward_workspace_size(int layout, long long B, long long P, int K,
                                                  int O, int activation, int dtype) {
  const Problem p = problem(layout, B, P, K, O, layout == PWC_LAYOUT_MAP ? P * K : K, activation,
                            0.f, dtype, 0);
  return most_backward_space(p);
}

PWC_API int pwc_linear_backward(const void* x, const void* weight, const void* bias,
                                const void* grad_out, void* grad_x, void* grad_weight,
                                void* grad_bias, int layout, long long B, long long P, int K,
                                int O, long long x_stride, int activation, float negative_slope,
                                int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return product_backward("pwc_linear_backward",
                          problem(layout, B, P, K, O, x_stride, activation, negative_slope, dtype,
                                  0),
                          x, weight, bias, grad_out, grad_x, grad_weight, grad_bias, workspace,
                          workspace_bytes, (hipStream_t)stream);
}

PWC_API int pwc_gated_linear_forward(const void* x, const void* weight, const void* bias, void* y,
                                     int layout, long long B, long long P, int K, int O,
                                     long long x_stride, int activation, float negative_slope,
                                     int dtype, void* stream) {
  return product_forward("pwc_gated_linear_forward",
                         problem(layout, B, P, K, O, x_stride, activation, negative_slope, dtype, 1),
                         x, weight, bias, nullptr, y, (hipStream_t)stream);
}

PWC_API size_t pwc_gated_linear_backward_workspace_size(int layout, long long B, long long P,
                                                        int K, int O, int dtype) {
  const Problem p = problem(layout, B, P, K, O, layout == PWC_LAYOUT_MAP ? P * K : K, 0, 0.f,
                            dtype, 1);
  return most_backward_space(p);
}

PWC_API int pwc_gated_linear_backward(const void* x, const void* weight, const void* bias,
                                      const void* grad_out, void* grad_x, void* grad_weight,
                                      void* grad_bias, int layout, long long B, long long P, int K,
                                      int O, long long x_stride, int activation,
                                      float negative_slope, int dtype, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  return product_backward("pwc_gated_linear_backward",
                          problem(layout, B, P, K, O, x_stride, activation, negative_slope, dtype,
                                  1),
                          x, weight, bias, grad_out, grad_x, grad_weight, grad_bias, workspace,
                          workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
