// The gated block's products: how each is cut into tiles and slices, and the operand
// form of what is not in it already.
#include <algorithm>

#include "product.h"

namespace dpamd {

template <int KIND>
void launch_product(hipStream_t, ProductKind, int shape, ProductArgs&);
extern template void launch_product<kBf16>(hipStream_t, ProductKind, int, ProductArgs&);
extern template void launch_product<kF16>(hipStream_t, ProductKind, int, ProductArgs&);
extern template void launch_product<kF32>(hipStream_t, ProductKind, int, ProductArgs&);

namespace {

// Rows of any stride into rows of ld, zeros from cols to ld: eight elements a thread,
// the matrices of one call one after another in one launch (a launch for each costs more
// than the work of small ones: 17 launches of a training step of 31,920 rows through 70-96-1 took 139
// us, 11 take 106).
template <int KIND>
__global__ __launch_bounds__(256) void k_pack(const PackList list) {
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < list.end[list.count - 1]; at += (long)gridDim.x * 256) {
    int m = 0;
    while (at >= list.end[m]) ++m;
    const PackItem& it = list.item[m];
    const long k = at - (m ? list.end[m - 1] : 0);
    const int per = (int)(it.ld / 8);
    const long row = k / per;
    const int c0 = (int)(k % per) * 8;
    unsigned short* d = it.dst + row * it.ld + c0;
    if constexpr (KIND == kF32) {
      const float* s = static_cast<const float*>(it.src) + row * it.ld_src + c0;
      float v[8];
      if (c0 + 8 <= it.cols) {
        __builtin_memcpy(v, s, sizeof(v));  // (the hardware takes addresses of any alignment)
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c0 + e < it.cols ? s[e] : 0.0f;
      }
      put_operand8<KIND>(d, it.plane, v);
    } else {
      const unsigned short* s = static_cast<const unsigned short*>(it.src) + row * it.ld_src + c0;
      typedef unsigned short us8 __attribute__((ext_vector_type(8)));
      us8 v;
      if (c0 + 8 <= it.cols) {
        __builtin_memcpy(&v, s, sizeof(v));  // (the hardware takes addresses of any alignment)
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c0 + e < it.cols ? s[e] : (unsigned short)0;
      }
      *reinterpret_cast<us8*>(d) = v;
    }
  }
}

__global__ __launch_bounds__(256) void k_zero(unsigned char* dst, long rows, long row_bytes, long stride) {
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < rows * row_bytes; at += (long)gridDim.x * 256)
    dst[at / row_bytes * stride + at % row_bytes] = 0;
}

// (a grid holds fewer than 2^32 threads: the kernels stride over what is beyond)
unsigned blocks_for(long threads) { return (unsigned)std::min((threads + 255) / 256, 1L << 20); }

}  // namespace

void pack_operands(hipStream_t st, int elem, const PackList& list) {
  if (!list.count) return;
  const dim3 grid(blocks_for(list.end[list.count - 1]));
  if (elem == kF32)
    hipLaunchKernelGGL((k_pack<kF32>), grid, dim3(256), 0, st, list);
  else
    hipLaunchKernelGGL((k_pack<kBf16>), grid, dim3(256), 0, st, list);
  DPAMD_LAUNCH_CHECK();
}

void fill_zero(hipStream_t st, void* dst, long rows, long row_bytes, long stride) {
  if (rows <= 0 || row_bytes <= 0) return;
  hipLaunchKernelGGL(k_zero, dim3(blocks_for(rows * row_bytes)), dim3(256), 0, st, static_cast<unsigned char*>(dst),
                     rows, row_bytes, stride);
  DPAMD_LAUNCH_CHECK();
}

ProductPlan plan_product(ProductKind what, int elem, long M, long N, long K, int segs, int mats, int ncu) {
  struct S {
    int bm, bn, bk, per_cu;
    double us;  // one step of k of one block
  };
  static const S shapes[2][3] = {{{256, 256, 64, 1, 1.9}, {128, 128, 64, 2, 1.4}, {64, 128, 64, 3, 1.2}},
                                 {{256, 128, 32, 1, 1.8}, {128, 64, 32, 2, 1.1}, {64, 64, 32, 3, 0.9}}};
  const char* fs = getenv("DPAMD_SHAPE");
  const char* fz = getenv("DPAMD_SPLIT");
  const int sub = what == kProdGate ? 2 : 1;
  ProductPlan best{1, 1, ncu, 0};
  double best_us = 0;
  for (int k = fs ? atoi(fs) : 0; k < (fs ? atoi(fs) + 1 : 3); ++k) {
    const S& s = shapes[elem == kF32][k];
    const long tiles = ((M + s.bm - 1) / s.bm) * ((N + s.bn / sub - 1) / (s.bn / sub)) * mats;
    const long steps = (K + s.bk - 1) / s.bk * segs, slots = (long)ncu * s.per_cu;
    long split = 1;
    if (fz) split = std::min(steps, atol(fz)); else if (tiles < slots) split = std::max(1L, std::min(slots / tiles, steps / 4));
    const long rounds = (tiles * split + slots - 1) / slots;
    const double bytes = split > 1 ? 4.0 * split * sub * mats * M * ((N + 7) / 8 * 8) : 0;
    const double us = (double)rounds * ((steps + split - 1) / split) * s.us + (split > 1 ? 3 + 2 * bytes / 4e6 : 0);
    if (best_us == 0 || us < best_us) {
      best_us = us;
      best = ProductPlan{k, (int)split, (int)slots / 8 * 8, (size_t)bytes};
    }
  }
  return best;
}

void run_product(hipStream_t st, ProductKind what, int elem, const ProductPlan& plan, ProductArgs& p) {
  p.split = plan.split;
  p.blocks = plan.blocks;
  p.ldp = (p.cols + 3) / 4 * 4;
  if (elem == kBf16)
    launch_product<kBf16>(st, what, plan.shape, p);
  else if (elem == kF16)
    launch_product<kF16>(st, what, plan.shape, p);
  else
    launch_product<kF32>(st, what, plan.shape, p);
}

}  // namespace dpamd
