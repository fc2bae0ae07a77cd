// Host side that the operators of trainable heads share: the handle, its errors and workspaces, checks of
// arguments, and operands of the tile products.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <exception>
#include <string>
#include <vector>

#include "../../include/dp_amd.h"
#include "common.h"
#include "ops.h"

namespace dpamd {

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

}  // namespace dpamd

struct dp_ops {
  int device = 0;
  int ncu = 256;
  std::string err;
  std::vector<dpamd::Workspace> ws;
  std::vector<void*> retired;  // outgrown workspaces that graphs still name
  size_t bytes_now = 0, bytes_peak = 0;
};

namespace dpamd {

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

inline void require(bool ok, const char* what) {
  if (!ok) throw OpsError{DP_ERR_ARG, what};
}

inline char* workspace(dp_ops* O, hipStream_t st, size_t bytes) {
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

inline int elem_of(int type) {
  return type == DP_TYPE_BF16 ? 0 : type == DP_TYPE_F16 ? 1 : 2;  // ElemKind
}
constexpr int kElemI8 = 3;
inline size_t bytes_of(int type) { return type == DP_TYPE_F32 ? 4 : 2; }

inline int64_t row_length(int64_t ld, int64_t cols, const char* what) {
  if (ld == 0) return cols;
  require(ld >= cols && ld <= kMaxLd, what);
  return ld;
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

inline bool is_operand(int type, const void* p, int64_t ld, int64_t cols) {
  const int64_t chunk = 16 / (int64_t)bytes_of(type);
  return cols % chunk == 0 && ld % chunk == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

inline Source source_of(int type, const void* p, int64_t ld, int64_t rows, int64_t cols, Regions& r, bool direct = true) {
  Source s{p, (long)ld, (long)rows, (long)cols, false, 0, (long)ld};
  s.direct = direct && is_operand(type, p, ld, cols);
  if (!s.direct) {
    s.ld = (s.cols + 7) / 8 * 8;
    s.at = r.take(bytes_of(type) * (size_t)s.rows * s.ld);
  }
  return s;
}

// The operand's place, and what copies it there.
inline Operand operand_of(const Source& s, char* ws, PackList& list) {
  if (s.direct) return Operand{s.src, s.ld};
  list.item[list.count] = PackItem{s.src, s.ld_src, s.ld, (int)s.cols, ws + s.at};
  list.end[list.count] = (list.count ? list.end[list.count - 1] : 0) + s.rows * (s.ld / 8);
  ++list.count;
  return Operand{ws + s.at, s.ld};
}

// whether `many` elements of a row of `out`, from a multiple of it on, can be stored whole
inline bool aligned(const void* out, int64_t ld, int type, int many) {
  return reinterpret_cast<uintptr_t>(out) % (many * bytes_of(type)) == 0 && ld % many == 0;
}

inline ProductArgs product(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t K) {
  ProductArgs p{};
  p.a[0] = p.a[1] = a;
  p.b[0] = p.b[1] = b;
  p.M = (int)M;
  p.N = p.cols = (int)N;
  p.K = (int)K;
  p.segs = p.mats = 1;
  return p;
}

inline void output(ProductArgs& p, int k, void* out, int64_t ld, int type) {
  p.out[k] = out;
  p.ldo[k] = ld;
  p.vec[k] = aligned(out, ld, type, 4);
  p.wide[k] = type != DP_TYPE_F32 && aligned(out, ld, type, 8);
}

}  // namespace dpamd
