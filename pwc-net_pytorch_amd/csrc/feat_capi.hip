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

// Images of one pixel are tokens: the kernels' tiles would take one pixel each.
void by_tokens(int& layout, long long& B, long long& P) {
  if (layout != PWC_LAYOUT_MAP || P != 1) return;
  layout = PWC_LAYOUT_TOKENS;
  P = B;
  B = 1;
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
  // tokens are counted in 32 bits, up to the end of a tile, and of the tiles of a block's turn
  if (p.M > kIntMax - 0xffff) return "dimension too large";
  if (p.act < 0 || p.act > kActGeluTanh) return "unknown activation";
  if (p.M > (1LL << 40) / p.rows || (long long)p.rows * p.K > (1LL << 40))
    return "dimension too large";
  return bad_stride(p.layout, p.B, p.P, p.K, p.x_stride);
}

Problem problem(int layout, long long B, long long P, int K, int O, long long x_stride, int act,
                float slope, int dtype, int gated) {
  by_tokens(layout, B, P);
  Problem p = {layout, K, O, O, act, dtype, gated, B, P, 0, x_stride, slope};
  if (gated && O > 0 && O <= (1 << 23)) p.rows = 2 * O;  // (larger ones are refused)
  p.M = layout == PWC_LAYOUT_MAP && B >= 0 && P >= 0 && B <= kIntMax && P <= kIntMax ? B * P : P;
  return p;
}

bool tokens(const Problem& p) { return p.layout == PWC_LAYOUT_TOKENS; }
bool needs_z(const Problem& p) { return p.gated || p.act != kActNone; }
size_t elem(int dtype) { return dtype == 0 ? 4 : 2; }

// A matrix as the products read it: rows of `cols` values, `row` apart (tokens' channels, W's
// channels, or a channel's pixels), images `image` apart; `padded`: zeros to the next 16 bytes.
struct View {
  const void* at;
  long long row, image;
  int padded;
};
View x_view(const Problem& p, const void* x) {
  if (tokens(p)) return {x, p.x_stride, 0, 0};
  return {x, p.P, p.x_stride, 0};
}
View w_view(const Problem& p, const void* w) { return {w, p.K, 0, 0}; }
View dz_view(const Problem& p, const void* dz) {
  if (tokens(p)) return {dz, p.rows, 0, 0};
  return {dz, p.P, p.rows * p.P, 0};
}

// Operations of a product up to which a 16-bit dz is kept in two parts.  Rounded once it makes the
// gradients' error 1.4 times that of their own rounding (bf16 2-norms 0.0024 against 0.0017; the two
// parts 0.0017), as in a program that keeps it between its layers.  The second part is a second
// product of each gradient: up to here 2 to 12 us of a backward pass of 14 to 35 (us, one part / two:
// 64 x 96 -> 96 13.5 / 15.1, 256 x 512 -> 512 20 / 26, 8 x 96 x 24 x 28 -> 96 16 / 17), which hide
// behind the 45 us that autograd takes for the call; from there on it shows and doubles what bounds
// the call (1024 x 512 -> 512 gated, 1.1 GFLOP, 31 / 46; 1024 x 1024 -> 4096, 8.6, 62 / 81).  So a
// token's gradients in a large batch have one rounding more than in a small one.
constexpr double kKeepLow = 5e8;

// The products load directly (memory to LDS) from rows at 16-byte places.  Where a call's rows are
// not, large ones are laid out so first.  Forward alone that is worth its launch from some GFLOP on
// (us, as they lie / laid out first; bf16: 2047 x 1023 -> 1023, 4.3 GFLOP: 20 / 22; 4095 x 1023 ->
// 1023, 8.6: 31 / 29; 8191 x 1023 -> 4095: 216 / 91).  Backward the three products share the copies,
// and rows of odd 16-bit lengths that are read across k cost most (with an activation: 1001 x 511 ->
// 511: 52 / 34, fp16 2047 x 1023 -> 1023: 136 / 54; without: 301 x 511 -> 511: 44 / 22; map 5 x 96 x 37
// x 53 -> 385 gated: 57 / 48; fp32 2001 x 701 -> 1001: 128 / 121), unless so few channels meet that the
// products are all traffic anyway (map 16 x 64 x 113 x 129 -> 64: 79 / 83, fp32 127 / 144).
bool pads_pay(const Problem& p, bool backward) {
  const double operations = 2.0 * (double)p.M * p.rows * p.K;
  if (!backward) return operations >= 8e9;
  if (p.K < 96 || p.rows < 96) return operations >= 8e9;
  return operations > (tokens(p) && p.dtype != 0 ? 1e8 : 1e9);
}
long long whole(const Problem& p, long long cols) {
  const long long e = 16 / (long long)elem(p.dtype);
  return (cols + e - 1) / e * e;
}
bool lies_well(const Problem& p, const View& v, long long cols) {
  return aligned_to(v.at, 16) && whole(p, v.row) == v.row && whole(p, v.image) == v.image &&
         whole(p, cols) == cols;
}
long long x_cols(const Problem& p) { return tokens(p) ? p.K : p.P; }
long long x_rows(const Problem& p) { return tokens(p) ? p.M : p.B * p.K; }
long long dz_cols(const Problem& p) { return tokens(p) ? p.rows : p.P; }
long long dz_rows(const Problem& p) { return tokens(p) ? p.M : p.B * p.rows; }
View padded_x(const Problem& p, const void* at) {
  const long long row = whole(p, x_cols(p));
  return {at, row, tokens(p) ? 0 : p.K * row, 1};
}
View padded_w(const Problem& p, const void* at) { return {at, whole(p, p.K), 0, 1}; }
View padded_dz(const Problem& p, const void* at) {
  const long long row = whole(p, dz_cols(p));
  return {at, row, tokens(p) ? 0 : p.rows * row, 1};
}

// z = x W^T + b into the epilogue `mode`, whose output has `out_rows` channels
ProductArgs forward_args(const Problem& p, const View& x, const View& w, const void* bias,
                         const void* other, const View& out, int mode) {
  ProductArgs g = blank();
  g.K = p.K;
  g.bias = bias;
  g.other = other;
  g.out = const_cast<void*>(out.at);
  g.ldo = out.row;
  g.out_batch = out.image;
  g.mode = mode;
  g.act = p.act;
  g.slope = p.slope;
  g.pair = p.gated ? p.O : 0;
  if (tokens(p)) {
    g.a = w.at, g.lda = w.row, g.a_pad = w.padded, g.a_k = 1, g.I = p.rows;
    g.b = x.at, g.ldb = x.row, g.b_pad = x.padded, g.b_k = 1, g.J = (int)p.M;
    g.ldother = p.O;
    g.channel_i = 1;
  } else {
    g.a = x.at, g.lda = x.row, g.a_batch = x.image, g.a_pad = x.padded, g.a_k = 0, g.I = (int)p.P;
    g.b = w.at, g.ldb = w.row, g.b_pad = w.padded, g.b_k = 1, g.J = p.rows;
    g.batches = (int)p.B;
    g.ldother = p.P, g.other_batch = (long long)p.O * p.P;
  }
  return g;
}
ProductArgs y_args(const Problem& p, const View& x, const View& w, const void* bias,
                   const void* res, void* y) {
  View out = {y, p.O, 0, 0};
  if (!tokens(p)) out.row = p.P, out.image = (long long)p.O * p.P;
  return forward_args(p, x, w, bias, res, out, p.gated ? kGated : kLinear);
}
ProductArgs dz_args(const Problem& p, const View& x, const View& w, const void* bias,
                    const void* dy, const View& dz) {
  return forward_args(p, x, w, bias, dy, dz, p.gated ? kGatedDz : kLinearDz);
}
// dx = dz W, for tokens in 32-bit parts (`out`) or itself where there is one split; `low`: from dz
// to what its rounding took, one more segment of k
ProductArgs dx_args(const Problem& p, const View& dz, long long low, const View& w, void* out) {
  ProductArgs g = blank();
  g.K = p.rows;
  g.out = out;
  g.mode = tokens(p) ? kPartial : kPlain;
  g.segments = low ? 2 : 1;
  (tokens(p) ? g.b_segment : g.a_segment) = low;
  if (tokens(p)) {
    g.a = w.at, g.lda = w.row, g.a_pad = w.padded, g.a_k = 0, g.I = p.K;
    g.b = dz.at, g.ldb = dz.row, g.b_pad = dz.padded, g.b_k = 1, g.J = (int)p.M;
    g.ldo = p.K;
  } else {
    g.a = dz.at, g.lda = dz.row, g.a_batch = dz.image, g.a_pad = dz.padded, g.a_k = 0;
    g.I = (int)p.P;
    g.b = w.at, g.ldb = w.row, g.b_pad = w.padded, g.b_k = 0, g.J = p.K;
    g.batches = (int)p.B;
    g.ldo = p.P, g.out_batch = (long long)p.K * p.P;
  }
  return g;
}
// dW = dz^T x in 32-bit parts (`out`), or itself where there is one split
ProductArgs dw_args(const Problem& p, const View& x, const View& dz, long long low, void* out) {
  ProductArgs g = blank();
  g.mode = kPartial;
  g.out = out;
  g.I = p.K;
  g.J = p.rows;
  g.ldo = p.K;
  g.a = x.at, g.lda = x.row, g.a_pad = x.padded;
  g.b = dz.at, g.ldb = dz.row, g.b_pad = dz.padded;
  if (tokens(p)) {
    g.K = (int)p.M;
    g.segments = low ? 2 : 1;
    g.b_segment = low;
  } else {
    g.K = (int)p.P;
    g.segments = (int)p.B * (low ? 2 : 1);
    g.a_segment = x.image, g.a_k = 1, g.a_halves = low ? 1 : 0;
    g.b_segment = low ? low : dz.image, g.b_k = 1;
  }
  return g;
}

// ---- workspaces, as places from their start ----
size_t bytes_of(const Problem& p, long long rows, long long cols) {
  return align256((size_t)rows * whole(p, cols) * elem(p.dtype));
}
struct ForwardSpace {
  bool pad_x, pad_w;
  size_t w, part, total;  // the padded x lies at 0
  View xv, wv;            // as the product takes them
};
ForwardSpace forward_space(const Problem& p, const void* x, const void* w, const char* ws) {
  ForwardSpace s = {};
  s.xv = x_view(p, x), s.wv = w_view(p, w);
  const int kernel =
      product_plan(y_args(p, s.xv, s.wv, nullptr, nullptr, nullptr), p.dtype).kernel;
  if (kernel > kFew64 && pads_pay(p, false)) {
    s.pad_x = !lies_well(p, s.xv, x_cols(p));
    s.pad_w = !lies_well(p, s.wv, p.K);
  }
  s.w = s.pad_x ? bytes_of(p, x_rows(p), x_cols(p)) : 0;
  s.part = s.w + (s.pad_w ? bytes_of(p, p.rows, p.K) : 0);
  if (s.pad_x) s.xv = padded_x(p, ws);
  if (s.pad_w) s.wv = padded_w(p, ws + s.w);
  s.total = s.part + product_part_bytes(y_args(p, s.xv, s.wv, nullptr, nullptr, nullptr), p.dtype);
  return s;
}

struct BackwardSpace {
  bool pad_x, pad_w, pad_dz;
  // dz, or the padded dy, lies at 0
  size_t x, w, part, part_bytes, dw_part, dw_part_bytes, sums, total;
  int dx_splits, splits, rows;     // rows: of partial bias gradients
  long long dz_rows;
  long long low;  // from dz to what its rounding took (maps: image by image), or 0
  View xv, wv, dzv;                // as the products take them
};
BackwardSpace backward_space(const Problem& p, const void* x, const void* w, const void* dy,
                             const char* ws, bool dx, bool dw, bool db) {
  BackwardSpace s = {};
  const bool z = needs_z(p), pay = pads_pay(p, true);
  s.xv = x_view(p, x), s.wv = w_view(p, w), s.dzv = dz_view(p, z ? nullptr : dy);
  s.pad_x = pay && (z || dw) && !lies_well(p, s.xv, x_cols(p));
  s.pad_w = pay && (z || dx) && !lies_well(p, s.wv, p.K);
  s.pad_dz = pay && (z || dx || dw) && !lies_well(p, s.dzv, dz_cols(p));
  // (where the copies lie comes below; that they are copies decides the kernels)
  if (s.pad_x) s.xv = padded_x(p, nullptr);
  if (s.pad_w) s.wv = padded_w(p, nullptr);
  const ProductPlan dz_plan =
      z ? product_plan(dz_args(p, s.xv, s.wv, nullptr, nullptr, s.dzv), p.dtype) : ProductPlan();
  // (only the kernels of small calls can write what dz's rounding took, which follows as more k)
  if (z && p.dtype != 0 && 2.0 * (double)p.M * p.rows * p.K <= kKeepLow &&
      (dz_plan.kernel <= kTile64Any || dz_plan.splits > 1))
    s.low = (tokens(p) ? p.M : p.rows) * (s.pad_dz ? whole(p, dz_cols(p)) : dz_cols(p));
  s.dz_rows = dz_rows(p) * (s.low ? 2 : 1);
  size_t at = 0;
  if (s.pad_dz)
    at += bytes_of(p, s.dz_rows, dz_cols(p));
  else if (z)
    at += align256((size_t)s.dz_rows * dz_cols(p) * elem(p.dtype));
  s.x = at;
  if (s.pad_x) at += bytes_of(p, x_rows(p), x_cols(p));
  s.w = at;
  if (s.pad_w) at += bytes_of(p, p.rows, p.K);
  if (s.pad_x) s.xv.at = ws + s.x;
  if (s.pad_w) s.wv.at = ws + s.w;
  if (s.pad_dz)
    s.dzv = padded_dz(p, ws);
  else if (z)
    s.dzv = dz_view(p, ws);
  if (s.low && !tokens(p)) s.dzv.image *= 2;
  s.dx_splits = dx ? product_plan(dx_args(p, s.dzv, s.low, s.wv, nullptr), p.dtype).splits : 1;
  s.splits = dw ? product_plan(dw_args(p, s.xv, s.dzv, s.low, nullptr), p.dtype).splits : 1;
  // (dz's parts are done with before dx's are written)
  auto parts = [](int splits, long long values) {
    return splits > 1 ? align256((size_t)splits * values * sizeof(float)) : 0;
  };
  const size_t dz_part = parts(dz_plan.splits, p.M * p.rows);
  s.part = at;
  s.part_bytes = parts(s.dx_splits, p.M * p.K);
  if (s.part_bytes < dz_part) s.part_bytes = dz_part;
  s.dw_part = at += s.part_bytes;
  s.dw_part_bytes = parts(s.splits, (long long)p.rows * p.K);
  at += s.dw_part_bytes;
  s.sums = at;
  if (db) {
    s.rows = z ? product_sum_rows(dz_args(p, s.xv, s.wv, nullptr, nullptr, s.dzv), p.dtype)
               : product_column_parts(p.layout, p.B, p.P, p.rows);
    at += align256((size_t)s.rows * p.rows * 4);
  }
  s.total = at;
  return s;
}

LayJob lay_x(const Problem& p, const void* x, bool pad, void* to) {
  if (!pad) return {};
  const View v = x_view(p, x);
  return {v.at, to, v.row, v.image, tokens(p) ? p.M : p.K, x_rows(p), x_cols(p)};
}
LayJob lay_w(const Problem& p, const void* w, bool pad, void* to) {
  if (!pad) return {};
  return {w, to, p.K, 0, p.rows, p.rows, p.K};
}
// dy as dz, or nothing but the zeros behind a computed one
LayJob lay_dz(const Problem& p, bool computed, const void* dy, const BackwardSpace& s, void* to) {
  if (!s.pad_dz) return {};
  const View v = dz_view(p, dy);
  return {computed ? nullptr : v.at, to,       v.row, v.image, tokens(p) ? p.M : p.rows,
          s.dz_rows,                 dz_cols(p)};
}

int product_backward(const char* fn, const Problem& p, const void* x, const void* w,
                     const void* bias, const void* dy, void* dx, void* dw, void* db,
                     void* workspace, size_t bytes, hipStream_t stream) {
  if (const char* e = bad_problem(p)) return api_fail(fn, e);
  const long long values = (long long)p.rows * p.K;
  if (p.M == 0)  // sums over no tokens
    return api_launch(fn, product_sum({{nullptr, dw, dw ? values : 0, 0},
                                       {nullptr, db, db ? p.rows : 0, 0}}, p.dtype, stream));
  if (!x || !w || !dy) return api_fail(fn, "null buffer");
  if (!dx && !dw && !db) return api_launch(fn, hipSuccess);
  char* ws = (char*)workspace;
  const BackwardSpace s = backward_space(p, x, w, dy, ws, dx, dw, db);
  if (s.total > 0 && (!workspace || bytes < s.total)) return api_fail(fn, "workspace too small");
  if (!aligned_to(workspace, 256)) return api_fail(fn, "workspace not aligned");
  // the copies, and zeros behind the rows of a dz that is to come
  const bool z = needs_z(p);
  hipError_t e = product_lay_out(
      {lay_x(p, x, s.pad_x, ws + s.x), lay_w(p, w, s.pad_w, ws + s.w), lay_dz(p, z, dy, s, ws)},
      p.dtype, stream);
  if (e == hipSuccess && z) {
    ProductArgs g = dz_args(p, s.xv, s.wv, bias, dy, s.dzv);
    g.sums = db ? (float*)(ws + s.sums) : nullptr;
    g.low = s.low;
    g.part = (float*)(ws + s.part);
    g.part_bytes = s.part_bytes;
    e = product_launch(g, p.dtype, stream);
  }
  // sums of parts in one launch at the end, unless they would have left the cache by then
  SumJob sum_dx = {}, sum_dw = {}, sum_db = {};
  const bool later = s.part_bytes + s.dw_part_bytes <= (32u << 20);
  if (dx && e == hipSuccess) {
    ProductArgs g = dx_args(p, s.dzv, s.low, s.wv, s.dx_splits > 1 ? (void*)(ws + s.part) : dx);
    g.splits = s.dx_splits;
    g.part_bytes = s.part_bytes;
    e = product_launch(g, p.dtype, stream);
    if (s.dx_splits > 1) sum_dx = {(const float*)(ws + s.part), dx, p.M * p.K, s.dx_splits};
    if (e == hipSuccess && !later) {
      e = product_sum({sum_dx}, p.dtype, stream);
      sum_dx = {};
    }
  }
  if (dw && e == hipSuccess) {
    ProductArgs g = dw_args(p, s.xv, s.dzv, s.low, s.splits > 1 ? (void*)(ws + s.dw_part) : dw);
    g.splits = s.splits;
    g.part_bytes = s.dw_part_bytes;
    e = product_launch(g, p.dtype, stream);
    if (s.splits > 1) sum_dw = {(const float*)(ws + s.dw_part), dw, values, s.splits};
  }
  if (db && e == hipSuccess) {
    float* sums = (float*)(ws + s.sums);
    if (!z) e = product_column_sums(dy, sums, p.layout, p.B, p.P, p.rows, s.rows, p.dtype, stream);
    sum_db = {sums, db, p.rows, s.rows};
  }
  if (e == hipSuccess) e = product_sum({sum_dx, sum_dw, sum_db}, p.dtype, stream);
  return api_launch(fn, e);
}

int product_forward(const char* fn, const Problem& p, const void* x, const void* w,
                    const void* bias, const void* res, void* y, void* workspace, size_t bytes,
                    hipStream_t stream) {
  if (const char* e = bad_problem(p)) return api_fail(fn, e);
  if (p.M == 0) return api_launch(fn, hipSuccess);
  if (!x || !w || !y) return api_fail(fn, "null buffer");
  char* ws = (char*)workspace;
  const ForwardSpace s = forward_space(p, x, w, ws);
  if (s.total > 0 && (!workspace || bytes < s.total)) return api_fail(fn, "workspace too small");
  if (!aligned_to(workspace, 256)) return api_fail(fn, "workspace not aligned");
  hipError_t e = product_lay_out({lay_x(p, x, s.pad_x, ws), lay_w(p, w, s.pad_w, ws + s.w)},
                                 p.dtype, stream);
  if (e == hipSuccess) {
    ProductArgs g = y_args(p, s.xv, s.wv, bias, res, y);
    g.part = (float*)(ws + s.part);
    g.part_bytes = s.total - s.part;
    e = product_launch(g, p.dtype, stream);
  }
  return api_launch(fn, e);
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
  return bad_stride(layout, B, P, C, x_stride);
}
}  // namespace

extern "C" {

PWC_API int pwc_layer_norm_forward(const void* x, const void* weight, const void* bias, void* y,
                                   void* mean, void* rstd, int layout, long long B, long long P,
                                   int C, long long x_stride, float eps, int dtype, void* stream) {
  const char* fn = "pwc_layer_norm_forward";
  by_tokens(layout, B, P);
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
  by_tokens(layout, B, P);
  if (bad_shape(layout, B, P, C, dtype)) return 0;
  return align256((size_t)2 * norm_parts(layout, B, P, C, dtype) * C * sizeof(float));
}

PWC_API int pwc_layer_norm_backward(const void* x, const void* weight, const void* grad_out,
                                    const void* mean, const void* rstd, void* grad_x,
                                    void* grad_weight, void* grad_bias, int layout, long long B,
                                    long long P, int C, long long x_stride, int dtype,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "pwc_layer_norm_backward";
  by_tokens(layout, B, P);
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
  if ((long long)s.heads * s.D > kIntMax) return api_fail(fn, "dimension too large");
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

PWC_API size_t pwc_linear_forward_workspace_size(const void* x, const void* weight, int layout,
                                                 long long B, long long P, int K, int O,
                                                 long long x_stride, int dtype) {
  const Problem p = problem(layout, B, P, K, O, x_stride, 0, 0.f, dtype, 0);
  return bad_problem(p) || p.M == 0 ? 0 : forward_space(p, x, weight, nullptr).total;
}

PWC_API int pwc_linear_forward(const void* x, const void* weight, const void* bias,
                               const void* residual, void* y, int layout, long long B, long long P,
                               int K, int O, long long x_stride, int activation,
                               float negative_slope, int dtype, void* workspace,
                               size_t workspace_bytes, void* stream) {
  return product_forward("pwc_linear_forward",
                         problem(layout, B, P, K, O, x_stride, activation, negative_slope, dtype, 0),
                         x, weight, bias, residual, y, workspace, workspace_bytes,
                         (hipStream_t)stream);
}

PWC_API size_t pwc_linear_backward_workspace_size(const void* x, const void* weight,
                                                  const void* grad_out, int layout, long long B,
                                                  long long P, int K, int O, long long x_stride,
                                                  int activation, int dtype) {
  const Problem p = problem(layout, B, P, K, O, x_stride, activation, 0.f, dtype, 0);
  if (bad_problem(p) || p.M == 0) return 0;
  return backward_space(p, x, weight, grad_out, nullptr, true, true, true).total;
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

PWC_API size_t pwc_gated_linear_forward_workspace_size(const void* x, const void* weight,
                                                       int layout, long long B, long long P, int K,
                                                       int O, long long x_stride, int dtype) {
  const Problem p = problem(layout, B, P, K, O, x_stride, 0, 0.f, dtype, 1);
  return bad_problem(p) || p.M == 0 ? 0 : forward_space(p, x, weight, nullptr).total;
}

PWC_API int pwc_gated_linear_forward(const void* x, const void* weight, const void* bias, void* y,
                                     int layout, long long B, long long P, int K, int O,
                                     long long x_stride, int activation, float negative_slope,
                                     int dtype, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  return product_forward("pwc_gated_linear_forward",
                         problem(layout, B, P, K, O, x_stride, activation, negative_slope, dtype, 1),
                         x, weight, bias, nullptr, y, workspace, workspace_bytes,
                         (hipStream_t)stream);
}

PWC_API size_t pwc_gated_linear_backward_workspace_size(const void* x, const void* weight,
                                                        const void* grad_out, int layout,
                                                        long long B, long long P, int K, int O,
                                                        long long x_stride, int dtype) {
  const Problem p = problem(layout, B, P, K, O, x_stride, 0, 0.f, dtype, 1);
  if (bad_problem(p) || p.M == 0) return 0;
  return backward_space(p, x, weight, grad_out, nullptr, true, true, true).total;
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
