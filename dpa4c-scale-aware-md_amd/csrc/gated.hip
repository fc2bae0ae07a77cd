// The gated block's products: how each is cut into tiles and slices, and the copies of
// matrices whose rows are not whole aligned 16-byte chunks.
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
// than the work of small ones).
template <class T>
__global__ __launch_bounds__(256) void k_pack(const PackList list) {
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < list.end[list.count - 1]; at += (long)gridDim.x * 256) {
    int m = 0;
    while (at >= list.end[m]) ++m;
    const PackItem& it = list.item[m];
    const long k = at - (m ? list.end[m - 1] : 0);
    const int per = (int)(it.ld / 8);
    const long row = k / per;
    const int c0 = (int)(k % per) * 8;
    const T* s = static_cast<const T*>(it.src) + row * it.ld_src + c0;
    struct alignas(16) Eight {
      T v[8];
    } v;
    if (c0 + 8 <= it.cols) {
      __builtin_memcpy(&v, s, sizeof(v));  // (the hardware takes addresses of any alignment)
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.v[e] = c0 + e < it.cols ? s[e] : T(0);
    }
    *reinterpret_cast<Eight*>(static_cast<T*>(it.dst) + row * it.ld + c0) = v;
  }
}

__global__ __launch_bounds__(256) void k_zero(unsigned char* dst, long rows, long row_bytes, long stride) {
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < rows * row_bytes; at += (long)gridDim.x * 256)
    dst[at / row_bytes * stride + at % row_bytes] = 0;
}

// One step (128 bytes of k) of one block, measured: its share of a compute unit's time
// among others, and its time alone; what a tile's epilogue adds (a plain store, the gate, the gate's
// gradient); and the blocks that a compute unit holds. Measured with each shape forced, every
// product of training steps of ten sizes, 33 to 131,072 rows: the one picked here took within 6 % of
// the best one's time but for eleven of 108, of which the worst took 24 % more. (fp32: the
// matrix cores are slow enough that 256 x 256 tiles gain nothing over 128 x 128. 16 bits: 128 x 32
// was nowhere ahead of both neighbours.)
struct TileShape {
  int bm, bn, per_cu;
  double share_us, alone_us, end_us[3];
};
const TileShape kShapes[2][5] = {{{256, 256, 1, 1.8, 1.8, {14, 24, 66}},
                                {128, 128, 2, 0.62, 1.0, {5, 8, 23}},
                                {64, 128, 3, 0.40, 0.9, {2.2, 3.2, 7}},
                                {},
                                {64, 32, 6, 0.22, 0.55, {0.7, 1, 1.5}}},
                               {{},
                                {128, 128, 2, 2.05, 2.26, {5, 8, 23}},
                                {64, 128, 3, 1.05, 1.27, {2.2, 3.2, 7}},
                                {128, 32, 4, 0.575, 0.75, {1.5, 1.5, 3.5}},
                                {64, 32, 6, 0.33, 0.5, {0.7, 1, 1.5}}}};

// (a grid holds fewer than 2^32 threads: the kernels stride over what is beyond)
unsigned blocks_for(long threads) { return (unsigned)std::min((threads + 255) / 256, 1L << 20); }

}  // namespace

void pack_operands(hipStream_t st, int elem, const PackList& list) {
  if (!list.count) return;
  const dim3 grid(blocks_for(list.end[list.count - 1]));
  if (elem == kF32)
    hipLaunchKernelGGL((k_pack<float>), grid, dim3(256), 0, st, list);
  else
    hipLaunchKernelGGL((k_pack<unsigned short>), grid, dim3(256), 0, st, list);
  DPAMD_LAUNCH_CHECK();
}

void fill_zero(hipStream_t st, void* dst, long rows, long row_bytes, long stride) {
  if (rows <= 0 || row_bytes <= 0) return;
  hipLaunchKernelGGL(k_zero, dim3(blocks_for(rows * row_bytes)), dim3(256), 0, st, static_cast<unsigned char*>(dst),
                     rows, row_bytes, stride);
  DPAMD_LAUNCH_CHECK();
}

ProductPlan plan_product(ProductKind what, int elem, long M, long N, long K, int segs, int mats, int ncu) {
  const int sub = what == kProdGate ? 2 : 1, bk = elem == kF32 ? 32 : 64;
  ProductPlan best{};
  double best_us = 0;
  const long steps = (K + bk - 1) / bk * segs;
  for (int k = 0; k < 5; ++k) {
    const TileShape& s = kShapes[elem == kF32][k];
    if (!s.bm) continue;
    // (k-strided tiles of 32 columns have too few banks apart)
    const double share = s.share_us * (what == kProdWeight && s.bn == 32 ? 1.3 : 1.0);
    const long tiles = ((M + s.bm - 1) / s.bm) * ((N + s.bn / sub - 1) / (s.bn / sub)) * mats;
    const long slots = (long)ncu * s.per_cu;
    const long most = std::max(1L, std::min(steps / 4, 2 * slots / tiles));
    for (long split = 1; split <= most; split = split < 4 ? split + 1 : split + split / 4) {
      const long items = tiles * split, a_cu = (items + ncu - 1) / ncu, rounds = (items + slots - 1) / slots;
      const double bytes = split > 1 ? 4.0 * split * sub * mats * M * ((N + 7) / 8 * 8) : 0;
      const double end = s.end_us[split > 1 ? 0 : what == kProdGate ? 1 : what == kProdGateGrad ? 2 : 0];
      const double us = (double)((steps + split - 1) / split) * std::max(a_cu * share, rounds * s.alone_us) +
                        a_cu * end + 2.0 + (split > 1 ? 4 + 2 * bytes / 4e6 : 0);
      if (best_us == 0 || us < best_us) {
        best_us = us;
        best = ProductPlan{k, (int)split, (int)slots / 8 * 8, (size_t)bytes};
      }
    }
  }
  return best;
}

void tile_of(int shape, int elem, int& rows, int& cols) {
  rows = kShapes[elem == kF32][shape].bm;
  cols = kShapes[elem == kF32][shape].bn;
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
