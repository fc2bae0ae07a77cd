// C ABI of the operators of trainable heads (dp_ops): argument checks, workspaces, and
// the order of the kernels of product.hip, gated.hip and lookup.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "../../include/dp_amd.h"
#include "common.h"
#include "ops.h"

using namespace dpamd;

namespace {

struct OpsError {
  int code;
  std::string msg;
};

// The workspace of one stream. Calls on one stream run in order, so they share it.
struct Workspace {
  hipStream_t stream = nullptr;
  char* p = nullptr;
  size_t cap = 0;
  bool captured = false;  // a graph holds its address
};

// Longest side of a matrix and row length: a tile's byte offsets, up to 256 rows of the
// longest, stay below 2^32.
constexpr int64_t kMaxDim = 1 << 20;
constexpr int64_t kMaxLd = 1 << 22;
constexpr int64_t kMaxRows = 1 << 30;

}  // namespace

struct dp_ops {
  int device = 0;
  int ncu = 256;
  std::string err;
  std::vector<Workspace> ws;
  std::vector<void*> retired;  // outgrown workspaces that graphs still name
  size_t bytes_now = 0, bytes_peak = 0;
};

namespace {

template <class F>
int guarded(dp_ops* O, F&& f) {
  if (!O) return DP_ERR_ARG;
  try {
    O->err.clear();
    f();
    return DP_OK;
  } catch (const OpsError& e) {
    O->err = e.msg;
    return e.code;
  } catch (const HipError& e) {
    (void)hipGetLastError();  // (else the next call's launch check finds it)
    O->err = std::string("HIP error ") + hipGetErrorString(e.code) + " in " + e.where;
    return DP_ERR_HIP;
  } catch (const std::exception& e) {
    O->err = e.what();
    return DP_ERR_ARG;
  } catch (...) {
    O->err = "unknown error";
    return DP_ERR_ARG;
  }
}

void require(bool ok, const char* what) {
  if (!ok) throw OpsError{DP_ERR_ARG, what};
}

char* workspace(dp_ops* O, hipStream_t st, size_t bytes) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  DPAMD_HIP(hipStreamIsCapturing(st, &cs));
  const bool capturing = cs != hipStreamCaptureStatusNone;
  Workspace* w = nullptr;
  for (Workspace& k : O->ws)
    if (k.stream == st) w = &k;
  if (!w) {
    O->ws.emplace_back();
    w = &O->ws.back();
    w->stream = st;
  }
  if (bytes > w->cap) {
    require(!capturing,
            "the workspace of a stream under capture cannot grow: run the same call once on it first");
    const size_t want = bytes + bytes / 8;
    if (w->p && w->captured) {
      O->retired.push_back(w->p);
    } else if (w->p) {
      DPAMD_HIP(hipStreamSynchronize(st));
      DPAMD_HIP(hipFree(w->p));
      O->bytes_now -= w->cap;
    }
    w->p = nullptr;
    w->cap = 0;
    w->captured = false;
    void* p = nullptr;
    DPAMD_HIP(hipMalloc(&p, want));
    w->p = static_cast<char*>(p);
    w->cap = want;
    O->bytes_now += want;
    O->bytes_peak = std::max(O->bytes_peak, O->bytes_now);
  }
  w->captured = w->captured || capturing;
  return w->p;
}

// Regions of a workspace, 256-byte aligned, laid out before its size is known.
struct Regions {
  size_t used = 0;
  size_t take(size_t bytes) {
    const size_t at = used;
    used += (bytes + 255) & ~size_t(255);
    return at;
  }
};

int elem_of(int type) {
  return type == DP_TYPE_BF16 ? 0 : type == DP_TYPE_F16 ? 1 : 2;  // ElemKind
}
size_t bytes_of(int type) { return type == DP_TYPE_F32 ? 4 : 2; }

int64_t row_length(int64_t ld, int64_t cols, const char* what) {
  if (ld == 0) return cols;
  require(ld >= cols && ld <= kMaxLd, what);
  return ld;
}

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

// An operand of the products: the caller's matrix where it is one (rows of whole 16-byte
// chunks, aligned), and else a region that it is copied into.
struct Source {
  const void* src;
  long ld_src, rows, cols;
  bool direct;
  size_t at;
  long ld;
};

bool is_operand(int type, const void* p, int64_t ld, int64_t cols) {
  const int64_t chunk = 16 / (int64_t)bytes_of(type);
  return cols % chunk == 0 && ld % chunk == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

Source source_of(int type, const void* p, int64_t ld, int64_t rows, int64_t cols, Regions& r, bool direct = true) {
  Source s{p, (long)ld, (long)rows, (long)cols, false, 0, (long)ld};
  s.direct = direct && is_operand(type, p, ld, cols);
  if (!s.direct) {
    s.ld = (s.cols + 7) / 8 * 8;
    s.at = r.take(bytes_of(type) * (size_t)s.rows * s.ld);
  }
  return s;
}

// The operand's place, and what copies it there.
Operand operand_of(const Source& s, char* ws, PackList& list) {
  if (s.direct) return Operand{s.src, s.ld};
  list.item[list.count] = PackItem{s.src, s.ld_src, s.ld, (int)s.cols, ws + s.at};
  list.end[list.count] = (list.count ? list.end[list.count - 1] : 0) + s.rows * (s.ld / 8);
  ++list.count;
  return Operand{ws + s.at, s.ld};
}

// gate and up are copied both or neither: the products take one row length for the two
bool pair_direct(const dp_gated_shape& s, const void* wg, const void* wu) {
  return is_operand(s.type, wg, s.ld_hidden, s.d_hidden) && is_operand(s.type, wu, s.ld_hidden, s.d_hidden);
}

// whether `many` elements of a row of `out`, from a multiple of it on, can be stored whole
bool aligned(const void* out, int64_t ld, int type, int many) {
  return reinterpret_cast<uintptr_t>(out) % (many * bytes_of(type)) == 0 && ld % many == 0;
}

ProductArgs product(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t K) {
  ProductArgs p{};
  p.a[0] = p.a[1] = a;
  p.b[0] = p.b[1] = b;
  p.M = (int)M;
  p.N = p.cols = (int)N;
  p.K = (int)K;
  p.segs = p.mats = 1;
  return p;
}

void output(ProductArgs& p, int k, void* out, int64_t ld, int type) {
  p.out[k] = out;
  p.ldo[k] = ld;
  p.vec[k] = aligned(out, ld, type, 4);
  p.wide[k] = type != DP_TYPE_F32 && aligned(out, ld, type, 8);
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

void gated_backward(dp_ops* O, const dp_gated_shape& s, const void* x, const void* wg, const void* wu, const void* wd,
                    const void* saved, const void* dy, void* dx, void* dwg, void* dwu, void* dwd, hipStream_t st) {
  const int elem = elem_of(s.type);
  const int64_t n = s.rows, f = s.d_hidden, f8 = (f + 7) / 8 * 8;
  const bool few = few_outputs(s.d_hidden, s.d_out);
  Regions r;
  Source sdy{}, sd{}, sx{}, sg{}, su{};
  if (!few) {
    sdy = source_of(s.type, dy, s.ld_y, n, s.d_out, r);
    sd = source_of(s.type, wd, s.ld_down, f, s.d_out, r);
  }
  if (dwg) sx = source_of(s.type, x, s.ld_x, n, s.d_in, r);
  if (dx) {
    const bool both = pair_direct(s, wg, wu);
    sg = source_of(s.type, wg, s.ld_hidden, s.d_in, f, r, both);
    su = source_of(s.type, wu, s.ld_hidden, s.d_in, f, r, both);
  }
  const size_t hb = bytes_of(s.type) * (size_t)n * f8;
  const size_t at_dg = r.take(hb), at_du = r.take(hb), at_h = dwd && !few ? r.take(hb) : 0;
  const ProductPlan p1 = few ? ProductPlan{} : plan_gate_grad(s, O->ncu);
  const ProductPlan p2 = plan_input(s, O->ncu);
  const ProductPlan p3 = plan_weights(s, O->ncu);
  const ProductPlan p4 = few ? ProductPlan{} : plan_down_weight(s, O->ncu);
  OutsArgs q = outs_of(s, wd);
  const size_t down_bytes = few ? plan_outs_grad(O->ncu, q) : p4.bytes;
  const size_t at_part = r.take(
      std::max(std::max(p1.bytes, dx ? p2.bytes : 0), std::max(dwg ? p3.bytes : 0, dwd ? down_bytes : 0)));
  char* ws = workspace(O, st, r.used);
  float* part = reinterpret_cast<float*>(ws + at_part);

  PackList list{};
  Operand ody{}, od{}, ox{}, og{}, ou{};
  if (!few) {
    ody = operand_of(sdy, ws, list);
    od = operand_of(sd, ws, list);
  }
  if (dwg) ox = operand_of(sx, ws, list);
  if (dx) {
    og = operand_of(sg, ws, list);
    ou = operand_of(su, ws, list);
  }
  pack_operands(st, elem, list);
  if (few) {
    q.dy = dy;
    q.saved = static_cast<const float*>(saved);
    q.dg = ws + at_dg;
    q.du = ws + at_du;
    q.dwd = dwd;
    q.partial = dwd ? part : nullptr;
    run_outs_grad(st, elem, q);
  } else {
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
    if (s.rows == 0) {
      const long b = (long)bytes_of(s.type);
      for (void* d : {dw_gate, dw_up})
        if (d) fill_zero(st, d, s.d_in, s.d_hidden * b, s.ld_hidden * b);
      if (dw_down) fill_zero(st, dw_down, s.d_hidden, s.d_out * b, s.ld_down * b);
      return;
    }
    require(x && w_gate && w_up && w_down && saved && dy, "null pointer");
    require(reinterpret_cast<uintptr_t>(saved) % 16 == 0, "saved must be 16-byte aligned");
    gated_backward(O, s, x, w_gate, w_up, w_down, saved, dy, dx, dw_gate, dw_up, dw_down, st);
  });
}

}  // extern "C"
