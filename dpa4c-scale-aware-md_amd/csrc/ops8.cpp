// C ABI of the 8-bit operators beside the gated block: checkpoints of activations, and products in 8-bit
// integers with a scale for each token and output channel.
#include <hip/hip_runtime.h>

#include "ops_host.h"

using namespace dpamd;

namespace {

// A product of two integers is at most 127 * 128 (a row's are quantised here, weights may hold -128), and a sum of so
// many of them stays below 2^31.
constexpr int64_t kMaxIn8 = 1 << 17;
static_assert(127 * 128 * kMaxIn8 < int64_t(1) << 31, "sums of 8-bit products are 32-bit integers");

void check_type(int type) {
  require(type == DP_TYPE_F32 || type == DP_TYPE_BF16 || type == DP_TYPE_F16, "unknown type");
}

KeepArgs keep_args(int type, int64_t rows, int cols, int64_t ld, const char* what) {
  check_type(type);
  require(rows >= 0 && rows <= kMaxRows, "rows out of range");
  require(cols >= 1 && cols <= kMaxDim, "cols must be 1 .. 2^20");
  KeepArgs p{};
  p.rows = (long)rows;
  p.ld = (long)row_length(ld, cols, what);
  p.cols = p.cols_out = cols;
  p.wide = kept8_wide(cols);
  return p;
}

void check_kept(const void* kept) {
  require(reinterpret_cast<uintptr_t>(kept) % 16 == 0, "kept must be 16-byte aligned");
}

// Row length of 8-bit weights: whole 16-byte chunks.
int64_t row_length8(int64_t ld, int d_in) {
  const int64_t whole = ((int64_t)d_in + 15) / 16 * 16;
  if (ld == 0) return whole;
  require(ld >= whole && ld <= kMaxLd && ld % 16 == 0,
          "ld of 8-bit weights must be a multiple of 16 of at least d_in, and not too long");
  return ld;
}

void check_weights8(const void* w) {
  require(reinterpret_cast<uintptr_t>(w) % 16 == 0, "8-bit weights must be 16-byte aligned");
}

void linear8(dp_ops* O, const dp_linear8_shape& s, const void* x, const signed char* w, const float* w_scale,
             const signed char* up, const float* up_scale, void* y, hipStream_t st) {
  const int64_t ldq = ((int64_t)s.d_in + 15) / 16 * 16;
  const Linear8Form form = linear8_form((long)s.rows, s.d_in, s.d_out);
  Linear8RowsArgs f{};
  if (form != kLinear8Tiles) {
    f.rows = (int)s.rows, f.K = s.d_in, f.N = s.d_out, f.act = s.act;
    f.w[0] = w, f.w[1] = up, f.ld_w = (long)s.ld_w;
    f.col_scale[0] = w_scale, f.col_scale[1] = up_scale;
    f.x = x, f.ld_x = (long)s.ld_x, f.y = y, f.ld_y = (long)s.ld_y;
    if (form == kLinear8Fused) return run_linear8_rows(st, elem_of(s.type), O->ncu, f);
  }
  ProductPlan plan{};
  if (form == kLinear8Tiles)
    plan = plan_product(up ? kProdGate : kProdDown, kElemI8, s.rows, s.d_out, s.d_in, 1, 1, O->ncu);
  Regions r;
  const size_t at_q = r.take((size_t)s.rows * ldq), at_s = r.take(sizeof(float) * (size_t)s.rows),
               at_part = r.take(plan.bytes);
  char* ws = workspace(O, st, r.used);
  Rows8Args q{};
  q.rows = (long)s.rows, q.ld = (long)s.ld_x, q.ld_q = (long)ldq, q.cols = s.d_in;
  q.x = x;
  q.q = reinterpret_cast<signed char*>(ws + at_q);
  q.scale = reinterpret_cast<float*>(ws + at_s);
  rows8(st, elem_of(s.type), q);
  if (form == kLinear8FewRows) {
    f.q = q.q, f.ld_q = (long)ldq, f.row_scale = q.scale;
    return run_linear8_rows(st, elem_of(s.type), O->ncu, f);
  }
  ProductArgs p = product(Operand{q.q, (long)ldq}, Operand{w, (long)s.ld_w}, s.rows, s.d_out, s.d_in);
  p.b[1].p = up;
  p.act = s.act;
  p.row_scale = q.scale;
  p.col_scale[0] = w_scale;
  p.col_scale[1] = up_scale;
  p.out_elem = elem_of(s.type);
  p.partial = reinterpret_cast<float*>(ws + at_part);
  output(p, 0, y, s.ld_y, s.type);
  run_product8(st, up != nullptr, plan, p);
}

}  // namespace

extern "C" {

size_t dp_keep8_bytes(int64_t rows, int cols) {
  if (rows < 0 || rows > kMaxRows || cols < 1 || cols > kMaxDim) return 0;
  const size_t wide = (size_t)kept8_wide(cols);
  return (size_t)rows * (wide + wide / 32);
}

int dp_keep8(dp_ops* O, int type, int64_t rows, int cols, const void* x, int64_t ld_x, void* kept, void* stream) {
  return guarded(O, [&]() {
    KeepArgs p = keep_args(type, rows, cols, ld_x, "ld_x is shorter than cols, or too long");
    check_kept(kept);
    if (rows == 0) return;
    require(x && kept, "null pointer");
    p.x = x;
    p.kept = static_cast<unsigned char*>(kept);
    DPAMD_HIP(hipSetDevice(O->device));
    keep8(static_cast<hipStream_t>(stream), elem_of(type), p);
  });
}

int dp_restore8(dp_ops* O, int type, int64_t rows, int cols, const void* kept, void* x, int64_t ld_x, void* stream) {
  return guarded(O, [&]() {
    KeepArgs p = keep_args(type, rows, cols, ld_x, "ld_x is shorter than cols, or too long");
    check_kept(kept);
    if (rows == 0) return;
    require(x && kept, "null pointer");
    p.kept = static_cast<unsigned char*>(const_cast<void*>(kept));
    p.out = x;
    DPAMD_HIP(hipSetDevice(O->device));
    restore8(static_cast<hipStream_t>(stream), elem_of(type), p);
  });
}

int dp_weights8(dp_ops* O, int type, int d_in, int d_out, const void* w, int64_t ld_w, void* w8, int64_t ld_w8,
                float* scale, void* stream) {
  return guarded(O, [&]() {
    check_type(type);
    require(d_in >= 1 && d_in <= kMaxIn8, "d_in must be 1 .. 2^17");
    require(d_out >= 1 && d_out <= kMaxDim, "d_out must be 1 .. 2^20");
    Weights8Args p{};
    p.d_in = d_in, p.d_out = d_out;
    p.ld_w = (long)row_length(ld_w, d_out, "ld_w is shorter than d_out, or too long");
    p.ld_q = (long)row_length8(ld_w8, d_in);
    require(w && w8 && scale, "null pointer");
    check_weights8(w8);
    p.w = w;
    p.q = static_cast<signed char*>(w8);
    p.scale = scale;
    DPAMD_HIP(hipSetDevice(O->device));
    weights8(static_cast<hipStream_t>(stream), elem_of(type), p);
  });
}

int dp_linear8(dp_ops* O, const dp_linear8_shape* shape, const void* x, const void* w, const float* w_scale,
               const void* w_up, const float* up_scale, void* y, void* stream) {
  return guarded(O, [&]() {
    require(shape != nullptr, "no shape");
    dp_linear8_shape s = *shape;
    check_type(s.type);
    require(s.act == DP_ACT_TANH || s.act == DP_ACT_SILU || s.act == DP_ACT_GELU || s.act == DP_ACT_NONE,
            "unknown activation");
    require(s.rows >= 0 && s.rows <= kMaxRows, "rows out of range");
    require(s.d_in >= 1 && s.d_in <= kMaxIn8, "d_in must be 1 .. 2^17");
    require(s.d_out >= 1 && s.d_out <= kMaxDim, "d_out must be 1 .. 2^20");
    s.ld_x = row_length(s.ld_x, s.d_in, "ld_x is shorter than d_in, or too long");
    s.ld_y = row_length(s.ld_y, s.d_out, "ld_y is shorter than d_out, or too long");
    s.ld_w = row_length8(s.ld_w, s.d_in);
    require(!w_up == !up_scale, "w_up and its scales are both given or both NULL");
    if (s.rows == 0) return;
    require(x && w && w_scale && y, "null pointer");
    check_weights8(w);
    check_weights8(w_up);
    DPAMD_HIP(hipSetDevice(O->device));
    linear8(O, s, x, static_cast<const signed char*>(w), w_scale, static_cast<const signed char*>(w_up), up_scale, y,
            static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
