// The products of one element kind (ELEM_KIND, one object file each) and their launches.
#include <algorithm>

#include "product.h"

namespace dpamd {

namespace {

// 256 x 256 with eight waves of 128 x 64 (128 KB of LDS, one block a compute unit), 128 x 128
// with four of 64 x 64 (64 KB, two), for few rows 64 x 128 with four of 64 x 32 (48 KB, three),
// and for small products 64 x 32 with four of 16 x 32 (24 KB, six). fp32 has 128 x 32 (40 KB,
// four) for narrow ones in place of the first.
using Big = Shape<256, 256, 2, 4>;
using Small = Shape<128, 128, 2, 2>;
using Thin = Shape<64, 128, 1, 4>;
using Slim = Shape<128, 32, 4, 1>;
using Tiny = Shape<64, 32, 4, 1>;

template <int KIND, int LA, int LB, int EPI, class S>
void launch(hipStream_t st, ProductArgs& p) {
  constexpr bool PAIR = EPI == kEpiGate || EPI == kEpiGateBack || EPI == kEpiGateOuts || EPI == kEpiGateOne;
  constexpr int SUB = PAIR ? 2 : 1;
  p.tiles_m = (p.M + S::BM - 1) / S::BM;
  p.tiles_n1 = (p.N + S::BN / SUB - 1) / (S::BN / SUB);
  p.tiles_n = p.tiles_n1 * p.mats;
  const long items = (long)p.tiles_m * p.tiles_n * p.split;
  if (items >= 1L << 31) throw HipError{hipErrorInvalidValue, "gated block: too many tiles"};
  // (a slice has no h of its own to sum with dy)
  constexpr bool WHOLE = EPI == kEpiGateOuts || EPI == kEpiGateOne;
  if (WHOLE && p.split > 1) throw HipError{hipErrorInvalidValue, "gated block: a sliced gate of few outputs"};
  hipLaunchKernelGGL((k_product<KIND, LA, LB, EPI, S>), dim3((unsigned)std::min(items, (long)p.blocks)),
                     dim3(S::WM * S::WN * 64), 0, st, p);
  DPAMD_LAUNCH_CHECK();
  if constexpr (!WHOLE) {
    if (p.split == 1 || p.raw) return;
    const long rows = (long)p.M * (PAIR ? 1 : p.mats), quads = p.ldp / 4;
    // threads that share a quad's slices: up to 8 slices each, more where the quads fill the card
    p.join = 1;
    while (p.join < 64 && p.split > 8 * p.join && rows * quads * p.join < 1L << 18) p.join *= 2;
    const long per = 256 / p.join;
    hipLaunchKernelGGL((k_join<KIND, EPI>), dim3((unsigned)((rows * quads + per - 1) / per)), dim3(256), 0, st, p);
    DPAMD_LAUNCH_CHECK();
  }
}

template <int KIND, class S>
void launch_kind(hipStream_t st, ProductKind what, ProductArgs& p) {
  switch (what) {
    case kProdGate: return launch<KIND, kRowK, kColK, kEpiGate, S>(st, p);
    case kProdDown: return launch<KIND, kRowK, kColK, kEpiStore, S>(st, p);
    case kProdGateGrad: return launch<KIND, kRowK, kRowK, kEpiGateGrad, S>(st, p);
    case kProdGateBack: return launch<KIND, kRowK, kColK, kEpiGateBack, S>(st, p);
    case kProdGateOuts:
      // (the plan leaves out 128 x 128)
      if constexpr (S::BM != 128 || S::BN != 128) return launch<KIND, kRowK, kColK, kEpiGateOuts, S>(st, p);
      throw HipError{hipErrorInvalidValue, "gated block: a tile that few outputs do not have"};
    case kProdGateOne: return launch<KIND, kRowK, kColK, kEpiGateOne, S>(st, p);
    case kProdInput: return launch<KIND, kRowK, kRowK, kEpiStore, S>(st, p);
    case kProdWeight: return launch<KIND, kColK, kColK, kEpiStore, S>(st, p);
  }
}

}  // namespace

template <int KIND>
void launch_product(hipStream_t st, ProductKind what, int shape, ProductArgs& p) {
  if constexpr (KIND != kF32)
    if (shape == 0) return launch_kind<KIND, Big>(st, what, p);
  if constexpr (KIND == kF32)
    if (shape == 3) return launch_kind<KIND, Slim>(st, what, p);
  if (shape == 4)
    launch_kind<KIND, Tiny>(st, what, p);
  else if (shape == 2)
    launch_kind<KIND, Thin>(st, what, p);
  else
    launch_kind<KIND, Small>(st, what, p);
}

template void launch_product<ELEM_KIND>(hipStream_t, ProductKind, int, ProductArgs&);

}  // namespace dpamd
