// C ABI of the operators of trainable heads (dp_ops): argument checks, workspaces, and
// the order of the kernels of product.hip, gated.hip and lookup.hip. (ops8.cpp, norm.cpp: the other operators.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <new>
#include <string>

#include "ops_host.h"

using namespace dpamd;

namespace {

dp_gated_shape checked(const dp_gated_shape* s) {
  require(s != nullptr, "no shape");
  dp_gated_shape t = *s;
  require(t.type == DP_TYPE_F32 || t.type == DP_TYPE_BF16 || t.type == DP_TYPE_F16, "unknown type");
  require(t.act == DP_ACT_TANH || t.act == DP_ACT_SILU || t.act == DP_ACT_GELU, "unknown activation");
  require(t.rows >= 0 && t.rows <= kMaxRows, "rows out of range");
  for (int64_t d : {t.d_in, t.d_hidden, t.d_out})
    require(d >= 1 && d <= kMaxDim, "d_in, d_hidden and d_out must be 1 .. 2^20");
  t.ld_x = row_length(t.ld_x, t.d_in, "ld_x is shorter than d_in, or too long");
  t.ld_y = row_length(t.ld_y, t.d_out, "ld_y is shorter than d_out, or too long");
  t.ld_hidden = row_length(t.ld_hidden, t.d_hidden, "ld_hidden is shorter than d_hidden, or too long");
  t.ld_down = row_length(t.ld_down, t.d_out, "ld_down is shorter than d_out, or too long");
  return t;
}

// gate and up are copied both or neither: the products take one row length for the two
bool pair_direct(const dp_gated_shape& s, const void* wg, const void* wu) {
  return is_operand(s.type, wg, s.ld_hidden, s.d_hidden) && is_operand(s.type, wu, s.ld_hidden, s.d_hidden);
}

OutsArgs outs_of(const dp_gated_shape& s, const void* wd) {
  OutsArgs q{};
  q.rows = (long)s.rows;
  q.f = s.d_hidden, q.o = s.d_out, q.act = s.act;
  q.wd = wd;
  q.ldh = (s.d_hidden + 7) / 8 * 8, q.ld_down = (long)s.ld_down, q.ld_y = (long)s.ld_y;
  return q;
}

// How each product of the block is cut.
ProductPlan plan_gate(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdGate, elem_of(s.type), s.rows, s.d_hidden, s.d_in, 1, 1, ncu);
}
ProductPlan plan_down(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdDown, elem_of(s.type), s.rows, s.d_out, s.d_hidden, 1, 1, ncu);
}
ProductPlan plan_gate_grad(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdGateGrad, elem_of(s.type), s.rows, s.d_hidden, s.d_out, 1, 1, ncu);
}
// (of the backward that forms g and u again: dh first, in fp32, and then the gate with its gradient)
ProductPlan plan_dh(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdInput, elem_of(s.type), s.rows, s.d_hidden, s.d_out, 1, 1, ncu);
}
ProductPlan plan_gate_back(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdGateBack, elem_of(s.type), s.rows, s.d_hidden, s.d_in, 1, 1, ncu);
}
// The gate's product of that backward, and what it is: with up to four outputs dh is formed in its epilogue, and a
// sliced one, whose sums are elsewhere, keeps g and u for the kernels of few outputs.
struct Gate8 {
  ProductKind what;
  ProductPlan plan;
};
Gate8 plan_gate8(const dp_gated_shape& s, int ncu) {
  if (!few_outputs(s.d_hidden, s.d_out)) return {kProdGateBack, plan_gate_back(s, ncu)};
  const ProductKind outs = s.d_out == 1 ? kProdGateOne : kProdGateOuts;
  const ProductPlan p = plan_product(outs, elem_of(s.type), s.rows, s.d_hidden, s.d_in, 1, 1, ncu);
  return p.split == 1 ? Gate8{outs, p} : Gate8{kProdGate, plan_gate(s, ncu)};
}
ProductPlan plan_input(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdInput, elem_of(s.type), s.rows, s.d_in, s.d_hidden, 2, 1, ncu);
}
ProductPlan plan_weights(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdWeight, elem_of(s.type), s.d_in, s.d_hidden, s.rows, 1, 2, ncu);
}
ProductPlan plan_down_weight(const dp_gated_shape& s, int ncu) {
  return plan_product(kProdWeight, elem_of(s.type), s.d_hidden, s.d_out, s.rows, 1, 1, ncu);
}

void gated_forward(dp_ops* O, const dp_gated_shape& s, const void* x, const void* wg, const void* wu, const void* wd,
                   void* y, void* saved, hipStream_t st) {
  const int elem = elem_of(s.type);
  const int64_t n = s.rows, f8 = (s.d_hidden + 7) / 8 * 8;
  if (n <= kFewRows) {
    RowsArgs p{};
    p.rows = (int)n;
    p.d = s.d_in, p.f = s.d_hidden, p.o = s.d_out, p.act = s.act;
    p.ld_x = s.ld_x, p.ld_hidden = s.ld_hidden, p.ld_down = s.ld_down, p.ld_y = s.ld_y;
    p.x = x, p.wg = wg, p.wu = wu, p.wd = wd, p.y = y;
    p.saved = static_cast<float*>(saved);
    p.partial1 = reinterpret_cast<float*>(workspace(O, st, plan_rows(elem, O->ncu, p)));
    run_rows(st, elem, p);
    return;
  }
  Regions r;
  const Source sx = source_of(s.type, x, s.ld_x, n, s.d_in, r);
  const bool both = pair_direct(s, wg, wu);
  const Source sg = source_of(s.type, wg, s.ld_hidden, s.d_in, s.d_hidden, r, both);
  const Source su = source_of(s.type, wu, s.ld_hidden, s.d_in, s.d_hidden, r, both);
  const bool few = few_outputs(s.d_hidden, s.d_out);
  Source sd{};
  if (!few) sd = source_of(s.type, wd, s.ld_down, s.d_hidden, s.d_out, r);
  const size_t at_h = r.take((few ? sizeof(float) : bytes_of(s.type)) * (size_t)n * f8);
  const ProductPlan p1 = plan_gate(s, O->ncu);
  const ProductPlan p2 = few ? ProductPlan{} : plan_down(s, O->ncu);
  const size_t at_part = r.take(std::max(p1.bytes, p2.bytes));
  char* ws = workspace(O, st, r.used);

  PackList list{};
  const Operand ox = operand_of(sx, ws, list), og = operand_of(sg, ws, list), ou = operand_of(su, ws, list);
  const Operand od = few ? Operand{} : operand_of(sd, ws, list);
  pack_operands(st, elem, list);
  ProductArgs a = product(ox, og, n, s.d_hidden, s.d_in);
  a.b[1] = ou;
  a.cols = (int)f8;
  a.act = s.act;
  // (with few outputs h is no operand of the matrix cores, so that nothing asks for its rounding)
  if (few)
    a.epi.h32 = reinterpret_cast<float*>(ws + at_h);
  else
    a.epi.h = ws + at_h;
  a.epi.ldh = f8;
  a.epi.saved = static_cast<float*>(saved);
  a.partial = reinterpret_cast<float*>(ws + at_part);
  run_product(st, kProdGate, elem, p1, a);

  if (few) {
    OutsArgs q = outs_of(s, wd);
    q.h = a.epi.h32;
    q.y = y;
    return run_outs_down(st, elem, O->ncu, q);
  }
  const Operand oh{a.epi.h, (long)f8};
  ProductArgs b = product(oh, od, n, s.d_out, s.d_hidden);
  output(b, 0, y, s.ld_y, s.type);
  b.partial = a.partial;
  run_product(st, kProdDown, elem, p2, b);
}

// The backward from x and the kept g and u (saved), or from the 8-bit checkpoint of x alone (kept): its values
// are restored into an operand, dh is formed first, and the gate with its gradient in one product (with few outputs
// dh too, or g and u into the workspace, for the kernels of these).
void gated_backward(dp_ops* O, const dp_gated_shape& s, const void* x, const unsigned char* kept, const void* wg,
                    const void* wu, const void* wd, const void* saved, const void* dy, void* dx, void* dwg, void* dwu,
                    void* dwd, hipStream_t st) {
  const int elem = elem_of(s.type);
  const int64_t n = s.rows, f = s.d_hidden, f8 = (f + 7) / 8 * 8;
  const bool few = few_outputs(s.d_hidden, s.d_out);
  Regions r;
  Source sdy{}, sd{}, sx{}, sg{}, su{};
  if (!few) {
    sdy = source_of(s.type, dy, s.ld_y, n, s.d_out, r);
    sd = source_of(s.type, wd, s.ld_down, f, s.d_out, r);
  }
  if (dwg && !kept) sx = source_of(s.type, x, s.ld_x, n, s.d_in, r);
  if (dx || kept) {
    const bool both = pair_direct(s, wg, wu);
    sg = source_of(s.type, wg, s.ld_hidden, s.d_in, f, r, both);
    su = source_of(s.type, wu, s.ld_hidden, s.d_in, f, r, both);
  }
  const size_t hb = bytes_of(s.type) * (size_t)n * f8;
  const size_t at_dg = r.take(hb), at_du = r.take(hb), at_h = dwd && !few ? r.take(hb) : 0;
  const long ldx = (s.d_in + 7) / 8 * 8;
  const size_t at_x = kept ? r.take(bytes_of(s.type) * (size_t)n * ldx) : 0;
  const Gate8 gate = kept ? plan_gate8(s, O->ncu) : Gate8{};
  const ProductPlan& p0 = gate.plan;
  const bool outs = kept && few && gate.what != kProdGate;
  const ProductPlan p1 = few ? ProductPlan{} : kept ? plan_dh(s, O->ncu) : plan_gate_grad(s, O->ncu);
  const long f4 = (f + 3) / 4 * 4;
  const size_t at_saved =
      kept && !outs ? r.take(few ? 8 * (size_t)n * f : sizeof(float) * p1.split * (size_t)n * f4) : 0;
  const ProductPlan p2 = plan_input(s, O->ncu);
  const ProductPlan p3 = plan_weights(s, O->ncu);
  const ProductPlan p4 = few ? ProductPlan{} : plan_down_weight(s, O->ncu);
  OutsArgs q = outs_of(s, wd);
  size_t down_bytes = few ? plan_outs_grad(O->ncu, q) : p4.bytes;
  if (outs) {
    q.slices = gate_outs_slices(p0, elem, n);
    down_bytes = sizeof(float) * q.slices * (size_t)f * s.d_out;
  }
  // (dh's slices from a checkpoint are in at_saved)
  const size_t at_part = r.take(std::max({p0.bytes, kept ? 0 : p1.bytes, dx ? p2.bytes : 0, dwg ? p3.bytes : 0,
                                          dwd ? down_bytes : 0}));
  char* ws = workspace(O, st, r.used);
  float* part = reinterpret_cast<float*>(ws + at_part);

  PackList list{};
  Operand ody{}, od{}, ox{}, og{}, ou{};
  if (!few) {
    ody = operand_of(sdy, ws, list);
    od = operand_of(sd, ws, list);
  }
  if (dwg && !kept) ox = operand_of(sx, ws, list);
  if (dx || kept) {
    og = operand_of(sg, ws, list);
    ou = operand_of(su, ws, list);
  }
  pack_operands(st, elem, list);
  if (kept) {
    KeepArgs k{};
    k.rows = (long)n, k.cols = s.d_in, k.wide = kept8_wide(s.d_in);
    k.kept = const_cast<unsigned char*>(kept);
    k.out = ws + at_x;
    k.ld = ldx, k.cols_out = (int)ldx;
    restore8(st, elem, k);
    ox = Operand{ws + at_x, ldx};
    ProductArgs a = product(ox, og, n, f, s.d_in);
    a.b[1] = ou;
    a.cols = (int)f8;
    a.act = s.act;
    a.epi.ldh = f8;
    a.partial = part;
    if (outs) {
      a.epi.dg = ws + at_dg;
      a.epi.du = ws + at_du;
      a.epi.dy = dy, a.epi.ld_dy = s.ld_y;
      a.epi.wd = wd, a.epi.ld_down = s.ld_down;
      a.epi.outs = s.d_out;
      a.epi.outs_partial = dwd ? part : nullptr;
      run_product(st, gate.what, elem, p0, a);
      q.dwd = dwd;
      q.partial = part;
      if (dwd) run_outs_join(st, elem, q);
    } else if (few) {
      a.epi.h = ws + at_dg;  // (written and not read: dg comes after it)
      a.epi.saved = reinterpret_cast<float*>(ws + at_saved);
      run_product(st, kProdGate, elem, p0, a);
      saved = ws + at_saved;
    } else {
      ProductArgs d = product(ody, od, n, f, s.d_out);
      d.raw = true;
      d.partial = reinterpret_cast<float*>(ws + at_saved);
      run_product(st, kProdInput, elem, p1, d);
      a.epi.h = dwd ? ws + at_h : nullptr;
      a.epi.dg = ws + at_dg;
      a.epi.du = ws + at_du;
      a.epi.dh = d.partial;
      a.epi.dh_slices = p1.split;
      a.epi.dh_ld = f4, a.epi.dh_plane = n * f4;
      run_product(st, kProdGateBack, elem, p0, a);
    }
  }
  if (outs) {
    // (formed with the gate)
  } else if (few) {
    q.dy = dy;
    q.saved = static_cast<const float*>(saved);
    q.dg = ws + at_dg;
    q.du = ws + at_du;
    q.dwd = dwd;
    q.partial = dwd ? part : nullptr;
    run_outs_grad(st, elem, q);
  } else if (!kept) {
    ProductArgs a = product(ody, od, n, f, s.d_out);
    a.cols = (int)f8;
    a.act = s.act;
    a.epi.h = dwd ? ws + at_h : nullptr;
    a.epi.dg = ws + at_dg;
    a.epi.du = ws + at_du;
    a.epi.ldh = f8;
    a.epi.saved = static_cast<float*>(const_cast<void*>(saved));
    a.partial = part;
    run_product(st, kProdGateGrad, elem, p1, a);
  }
  const Operand odg{ws + at_dg, (long)f8}, odu{ws + at_du, (long)f8};

  if (dx) {
    ProductArgs b = product(odg, og, n, s.d_in, f);
    b.a[1] = odu;
    b.b[1] = ou;
    b.segs = 2;
    output(b, 0, dx, s.ld_x, s.type);
    b.partial = part;
    run_product(st, kProdInput, elem, p2, b);
  }
  if (dwg) {
    ProductArgs b = product(ox, odg, s.d_in, f, n);
    b.b[1] = odu;
    b.mats = 2;
    output(b, 0, dwg, s.ld_hidden, s.type);
    output(b, 1, dwu, s.ld_hidden, s.type);
    b.partial = part;
    run_product(st, kProdWeight, elem, p3, b);
  }
  if (dwd && !few) {
    ProductArgs b = product(Operand{ws + at_h, (long)f8}, ody, f, s.d_out, n);
    output(b, 0, dwd, s.ld_down, s.type);
    b.partial = part;
    run_product(st, kProdWeight, elem, p4, b);
  }
}

// The weights' gradients of a batch without rows.
void no_rows(const dp_gated_shape& s, void* dwg, void* dwu, void* dwd, hipStream_t st) {
  const long b = (long)bytes_of(s.type);
  for (void* d : {dwg, dwu})
    if (d) fill_zero(st, d, s.d_in, s.d_hidden * b, s.ld_hidden * b);
  if (dwd) fill_zero(st, dwd, s.d_hidden, s.d_out * b, s.ld_down * b);
}

void check_embed(int type, int64_t n, int vocab, int width) {
  require(type == DP_TYPE_F32 || type == DP_TYPE_BF16 || type == DP_TYPE_F16, "unknown type");
  require(n >= 0 && n <= kMaxRows, "n out of range");
  require(vocab >= 1 && vocab <= (1 << 30), "vocab must be 1 .. 2^30");
  require(width >= 1 && width <= kMaxDim, "width must be 1 .. 2^20");
}

}  // namespace

extern "C" {

int dp_ops_create(int gpu_rank, dp_ops** out) {
  if (!out) return DP_ERR_ARG;
  *out = nullptr;
  dp_ops* O = new (std::nothrow) dp_ops();
  if (!O) return DP_ERR_HIP;
  *out = O;  // kept on failure too, so that the caller can read dp_ops_last_error
  return guarded(O, [&]() {
    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev <= 0) throw OpsError{DP_ERR_NO_GPU, "no HIP device visible"};
    if (gpu_rank < 0) gpu_rank = 0;
    O->device = gpu_rank % ndev;
    DPAMD_HIP(hipSetDevice(O->device));
    hipDeviceProp_t prop;
    DPAMD_HIP(hipGetDeviceProperties(&prop, O->device));
    O->ncu = std::max(1, prop.multiProcessorCount);
    if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
      throw OpsError{DP_ERR_NO_GPU,
                     std::string("device is ") + prop.gcnArchName + ", this library is built for gfx950"};
  });
}

void dp_ops_destroy(dp_ops* O) {
  if (!O) return;
  // teardown is best effort; hipFree waits for the work that uses the memory
  if (!O->ws.empty()) (void)hipSetDevice(O->device);
  for (Workspace& w : O->ws)
    if (w.p) (void)hipFree(w.p);
  for (void* p : O->retired) (void)hipFree(p);
  delete O;
}

const char* dp_ops_last_error(const dp_ops* O) { return O ? O->err.c_str() : "null handle"; }

size_t dp_ops_device_bytes(const dp_ops* O) { return O ? O->bytes_peak : 0; }

int dp_embed(dp_ops* O, int type, int64_t n, int vocab, int width, const int* ids, const void* table, int64_t ld_table,
             float scale, void* out, int64_t ld_out, void* stream) {
  return guarded(O, [&]() {
    check_embed(type, n, vocab, width);
    const int64_t lt = row_length(ld_table, width, "ld_table is shorter than width, or too long");
    const int64_t lo = row_length(ld_out, width, "ld_out is shorter than width, or too long");
    if (n == 0) return;  // (arrays without rows may have no address)
    require(ids && table && out, "null pointer");
    DPAMD_HIP(hipSetDevice(O->device));
    lookup_rows(static_cast<hipStream_t>(stream), elem_of(type), n, vocab, width, ids, table, lt, scale, out, lo);
  });
}

int dp_embed_grad(dp_ops* O, int type, int64_t n, int vocab, int width, const int* ids, const void* dout,
                  int64_t ld_dout, float scale, void* dtable, int64_t ld_dtable, void* stream) {
  return guarded(O, [&]() {
    check_embed(type, n, vocab, width);
    require(dtable && (n == 0 || (ids && dout)), "null pointer");
    const int64_t li = row_length(ld_dout, width, "ld_dout is shorter than width, or too long");
    const int64_t lo = row_length(ld_dtable, width, "ld_dtable is shorter than width, or too long");
    DPAMD_HIP(hipSetDevice(O->device));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (n == 0) {
      fill_zero(st, dtable, vocab, width * (long)bytes_of(type), lo * (long)bytes_of(type));
      return;
    }
    const int elem = elem_of(type);
    char* ws = workspace(O, st, lookup_grad_bytes(elem, n, vocab, width, dout, li, dtable, lo));
    lookup_grad(st, elem, n, vocab, width, ids, dout, li, scale, dtable, lo, ws);
  });
}

size_t dp_gated_saved_bytes(const dp_gated_shape* shape) {
  try {
    const dp_gated_shape s = checked(shape);
    return 8 * (size_t)s.rows * (size_t)s.d_hidden;
  } catch (...) {
    return 0;
  }
}

int dp_debug_gated_plan(const dp_gated_shape* shape, int compute_units, int* plan) {
  if (!plan || compute_units < 1) return DP_ERR_ARG;
  try {
    const dp_gated_shape s = checked(shape);
    std::fill(plan, plan + 3 * DP_GATED_PRODUCTS, 0);
    if (s.rows == 0) return DP_OK;
    auto put = [&](int k, const ProductPlan& p) {
      tile_of(p.shape, elem_of(s.type), plan[3 * k], plan[3 * k + 1]);
      plan[3 * k + 2] = p.split;
    };
    const bool few = few_outputs(s.d_hidden, s.d_out);
    if (s.rows > kFewRows) put(0, plan_gate(s, compute_units));
    if (s.rows > kFewRows && !few) put(1, plan_down(s, compute_units));
    if (!few) put(2, plan_gate_grad(s, compute_units));
    put(3, plan_input(s, compute_units));
    put(4, plan_weights(s, compute_units));
    if (!few) put(5, plan_down_weight(s, compute_units));
    return DP_OK;
  } catch (...) {
    return DP_ERR_ARG;
  }
}

int dp_debug_gated_plan8(const dp_gated_shape* shape, int compute_units, int* plan) {
  if (!plan || compute_units < 1) return DP_ERR_ARG;
  try {
    const dp_gated_shape s = checked(shape);
    std::fill(plan, plan + 3 * DP_GATED_PRODUCTS8, 0);
    if (s.rows == 0) return DP_OK;
    auto put = [&](int k, const ProductPlan& p) {
      tile_of(p.shape, elem_of(s.type), plan[3 * k], plan[3 * k + 1]);
      plan[3 * k + 2] = p.split;
    };
    const bool few = few_outputs(s.d_hidden, s.d_out);
    const Gate8 gate = plan_gate8(s, compute_units);
    put(gate.what == kProdGate ? 0 : gate.what == kProdGateBack ? 1 : gate.what == kProdGateOuts ? 2 : 3, gate.plan);
    if (!few) put(4, plan_dh(s, compute_units));
    put(5, plan_input(s, compute_units));
    put(6, plan_weights(s, compute_units));
    if (!few) put(7, plan_down_weight(s, compute_units));
    return DP_OK;
  } catch (...) {
    return DP_ERR_ARG;
  }
}

int dp_gated_forward(dp_ops* O, const dp_gated_shape* shape, const void* x, const void* w_gate, const void* w_up,
                     const void* w_down, void* y, void* saved, void* stream) {
  return guarded(O, [&]() {
    const dp_gated_shape s = checked(shape);
    if (s.rows == 0) return;
    require(x && w_gate && w_up && w_down && y, "null pointer");
    require(reinterpret_cast<uintptr_t>(saved) % 16 == 0, "saved must be 16-byte aligned");
    DPAMD_HIP(hipSetDevice(O->device));
    gated_forward(O, s, x, w_gate, w_up, w_down, y, saved, static_cast<hipStream_t>(stream));
  });
}

int dp_gated_backward(dp_ops* O, const dp_gated_shape* shape, const void* x, const void* w_gate, const void* w_up,
                      const void* w_down, const void* saved, const void* dy, void* dx, void* dw_gate, void* dw_up,
                      void* dw_down, void* stream) {
  return guarded(O, [&]() {
    const dp_gated_shape s = checked(shape);
    require(!dw_gate == !dw_up, "dw_gate and dw_up are both given or both NULL");
    if (!dx && !dw_gate && !dw_down) return;
    DPAMD_HIP(hipSetDevice(O->device));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (s.rows == 0) return no_rows(s, dw_gate, dw_up, dw_down, st);
    require(x && w_gate && w_up && w_down && saved && dy, "null pointer");
    require(reinterpret_cast<uintptr_t>(saved) % 16 == 0, "saved must be 16-byte aligned");
    gated_backward(O, s, x, nullptr, w_gate, w_up, w_down, saved, dy, dx, dw_gate, dw_up, dw_down, st);
  });
}

int dp_gated_backward8(dp_ops* O, const dp_gated_shape* shape, const void* kept, const void* w_gate, const void* w_up,
                       const void* w_down, const void* dy, void* dx, void* dw_gate, void* dw_up, void* dw_down,
                       void* stream) {
  return guarded(O, [&]() {
    const dp_gated_shape s = checked(shape);
    require(!dw_gate == !dw_up, "dw_gate and dw_up are both given or both NULL");
    if (!dx && !dw_gate && !dw_down) return;
    DPAMD_HIP(hipSetDevice(O->device));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (s.rows == 0) return no_rows(s, dw_gate, dw_up, dw_down, st);
    require(kept && w_gate && w_up && w_down && dy, "null pointer");
    require(reinterpret_cast<uintptr_t>(kept) % 16 == 0, "kept must be 16-byte aligned");
    gated_backward(O, s, nullptr, static_cast<const unsigned char*>(kept), w_gate, w_up, w_down, nullptr, dy, dx,
                   dw_gate, dw_up, dw_down, st);
  });
}

}  // extern "C"
