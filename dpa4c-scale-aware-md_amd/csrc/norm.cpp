// C ABI of the group norm: argument checks, the choice of a form, workspaces.
#include <hip/hip_runtime.h>

#include <cmath>

#include "norm.h"
#include "ops_host.h"

namespace dpamd {

template <>
void norm_launch<0>(hipStream_t, const NormArgs&);
template <>
void norm_launch<1>(hipStream_t, const NormArgs&);
template <>
void norm_launch<2>(hipStream_t, const NormArgs&);
template <>
void norm_grad_launch<0>(hipStream_t, const NormArgs&);
template <>
void norm_grad_launch<1>(hipStream_t, const NormArgs&);
template <>
void norm_grad_launch<2>(hipStream_t, const NormArgs&);

namespace {

// lanes that sum the `entries` parts of each of `groups`, of `threads` in all
int lanes_of(int groups, int entries, int threads) {
  int lanes = 0;
  while (lanes < 6 && (2 << lanes) <= entries && ((long)groups << (lanes + 1)) <= threads) ++lanes;
  return lanes;
}

}  // namespace

NormNeeds plan_norm(int elem, int ncu, bool grad, NormArgs& p) {
  const int most = elem == 2 ? 4 : 8;  // 16 bytes
  p.per = p.channels / p.groups;
  p.vec = p.channels < most ? 1 : most;
  p.general = p.per % p.vec != 0;
  p.vecs = (p.channels + p.vec - 1) / p.vec;
  p.entries = p.general ? p.channels : p.vecs;
  p.group_entries = p.general ? p.per : p.per / p.vec;
  const long length = std::max(1L, p.rows / p.frames);
  const bool affine = grad && (p.dgamma || p.dbeta);
  NormNeeds need{};
  p.inv_entries = 1.0f / (float)p.group_entries, p.inv_per = 1.0f / (float)p.per;
  p.once = past_caches((double)p.rows * p.channels * (elem == 2 ? 4 : 2));
  p.slices = p.out_slices = 1;
  if (!p.starts && p.frames == p.rows && p.vecs <= (p.general && elem != 2 ? 512 : 1024)) {
    p.form = kNormRows;
    // (threads of a row, as few of them idle as may be: bf16, forward, 30,000 x 960 24 us with 128 and 40 with 256, 60,000 x
    // 256 12 with 32 and 18 with 64, 400,000 x 12 in 2 groups 19 with 4 and 56 with 16,
    // 100,000 x 64 7.3 with 8 and 9.9 with 16)
    const int T = p.vecs <= 4 ? 4 : p.vecs <= 8 ? 8 : p.vecs <= 16 ? 16 : p.vecs <= 32 ? 32 : p.vecs <= 64 ? 64 : p.vecs <= 128 ? 128 : 256;
    p.by_lanes = !p.general && p.group_entries <= 64 && (p.group_entries & (p.group_entries - 1)) == 0;
    // (bf16, gradients, channels as entries and pieces: 30,000 x 2500 in 4 groups 667 and 349 us, 2,712 x 4042 in 2 98 and
    // 57; but fp32, whose vectors are half as long, 30,000 x 1010 in 10 110 and 120, and 20,000 x 2500 in 2 435 and 420)
    p.pieces = p.general && p.per >= p.vec && (p.vec == 8 || p.vecs > 256);
    if (p.pieces) p.entries = 2 * p.vecs;
    p.lanes = lanes_of(p.by_lanes ? 1 : p.groups, p.pieces ? p.per / p.vec + 1 : p.group_entries, T);
    p.blocks = (int)std::min((p.rows + 256 / T - 1) / (256 / T), (grad ? 4L : 8L) * ncu);
    if (affine) need.partial = 8 * (size_t)p.blocks * p.channels;
  } else {
    // whole groups a block, at least 16 vectors (256 bytes of a row) where that leaves no compute unit idle
    auto part = [&](int g) { return (int)(((long)g * p.per + p.vec - 1) / p.vec); };
    auto blocks = [&](int g) { return (long)p.frames * ((p.groups + g - 1) / g); };
    int gp = (int)std::max(1L, std::min((long)p.groups, 256L * p.vec / p.per));
    while (gp > 1 && part((gp + 1) / 2) >= 4 &&
           (blocks(gp) < ncu || (blocks(gp) < 4 * ncu && part((gp + 1) / 2) >= 16)) &&
           256 / part((gp + 1) / 2) <= 2 * length)
      gp = (gp + 1) / 2;
    // fewer columns where that lets a block hold its rows in registers (8 a thread), from 128 bytes of a row on
    while (gp > 1 && part((gp + 1) / 2) >= 8 && length > 6 * (256 / part(gp))) gp = (gp + 1) / 2;
    // us, fitted to a card's times: a block's chain of rows beyond those it holds, or the bytes, of which pieces of
    // rows shorter than a few lines waste a part; against slices, which read all twice and take two launches more.
    // (Ragged frames: up to twice the mean length. Longer ones are not seen here: their lengths are on the device, and
    // 32,768 x 1600 in fp32 with nearly all rows in one of 64 frames takes 356 us for 77.)
    const int eb = elem == 2 ? 4 : 2, hold = grad && p.vec == 8 ? 4 : 8, batch = grad ? 2 : 4;
    const double size = (double)eb * p.rows * p.channels, n_blocks = (double)blocks(gp);
    const int lanes = 256 / std::min(256, part(gp));
    const double more = std::max(0.0, (double)length * (p.starts ? 2 : 1) / lanes - hold);
    const double again = std::max(0.0, 1.0 - (double)hold * lanes / length);  // rows that are read twice
    const double waves = std::max(1.0, n_blocks / (3 * ncu)), piece = (double)gp * p.per * eb;
    const double chain = 3 + waves * (1.2 + 2.4 * std::ceil(more / batch));
    const double moved = size * (grad ? 3 + 2 * again : 2 + again) / 4.7e6 * (1 + (p.general ? 128 : 16) / piece);
    const double whole = std::max(chain, moved * std::max(1.0, ncu / n_blocks));
    // (and a block of the slices' join for each frame and group: 50,000 frames of two rows of 256 in 32 groups, bf16,
    // 2,741 us in slices and 231 as frames)
    const double cut = 10 + size * (grad ? 5 : 3) / 4.7e6 + 1.7e-3 * p.frames * p.groups;
    const bool slices = part(gp) > 256 || whole > cut;
    if (!slices) {
      p.form = kNormFrames;
      p.part = part(gp);
      p.part_channels = gp * p.per;
      p.parts = (p.groups + gp - 1) / gp;
      p.lanes = lanes_of(gp, 256 / p.part * p.group_entries, 256);
      p.blocks = grad ? std::max(1, 8 * ncu / p.parts) : 65535;
      if (affine) need.partial = 8 * (size_t)std::min(p.frames, p.blocks) * p.channels;
    } else {
      p.form = kNormSlices;
      // as few parts of equal width as leave few of a block's threads idle (from 32 vectors on): gradients in bf16 of 60,000
      // rows of 1064 in 8 groups 200 us in one part and 154 in two, 30,000 of 2080 in 16 207 us in 256 vectors and four, and
      // 146 so
      auto width = [&](int parts) { return (p.vecs + parts - 1) / parts; };
      auto used = [&](int parts) { return (double)p.vecs * (256 / width(parts)) / (256.0 * parts); };
      p.parts = (p.vecs + 255) / 256;
      for (int k = p.parts + 1; k <= p.parts + 4 && width(k) >= 32; ++k)
        if (used(k) > 1.1 * used(p.parts)) p.parts = k;
      p.part = width(p.parts);
      p.parts = (p.vecs + p.part - 1) / p.part;
      p.part_channels = p.part * p.vec;
      const long want = std::max(1L, 4L * ncu / ((long)p.parts * p.frames));
      // (of two rows a thread at least, and of one)
      const int at_once = 256 / p.part;
      p.slices = (int)std::min(want, std::max(1L, length / (2 * at_once)));
      p.out_slices = (int)std::min(2 * want, std::max(1L, length / at_once));
      p.part_groups = (int)std::min((long)p.groups, (long)p.part_channels / p.per + 2);
      p.lanes = lanes_of(std::min(p.part_groups, 256), (std::min(p.per, p.part_channels) + p.vec - 1) / p.vec, 256);
      p.blocks = (int)std::min((long)p.frames, std::max(1L, 8L * ncu / ((long)p.parts * p.slices)));
      if (!grad || p.dx) need.pairs = 8 * (size_t)p.frames * p.slices * p.parts * p.part_groups;
      if (grad && p.dx) need.sums = 8 * (size_t)p.frames * p.groups;
      if (affine) need.partial = 8 * (size_t)p.blocks * p.slices * p.channels;
      if (!grad && !p.stats) need.stats = 8 * (size_t)p.frames * p.groups;
    }
  }
  return need;
}

namespace {

template <class F>
void by_elem(int elem, F&& f) {
  if (elem == 0)
    f(std::integral_constant<int, 0>{});
  else if (elem == 1)
    f(std::integral_constant<int, 1>{});
  else
    f(std::integral_constant<int, 2>{});
}

// The arguments that forward and backward share, checked.
NormArgs norm_args(const dp_norm_shape* shape, const void* starts) {
  require(shape != nullptr, "no shape");
  const dp_norm_shape& s = *shape;
  require(s.type == DP_TYPE_F32 || s.type == DP_TYPE_BF16 || s.type == DP_TYPE_F16, "unknown type");
  require(s.act == DP_ACT_TANH || s.act == DP_ACT_SILU || s.act == DP_ACT_GELU || s.act == DP_ACT_NONE,
          "unknown activation");
  require(s.rows >= 0 && s.rows <= kMaxRows, "rows out of range");
  require(s.channels >= 1 && s.channels <= kMaxDim, "channels must be 1 .. 2^20");
  require(s.groups >= 1 && s.groups <= s.channels && s.channels % s.groups == 0, "groups must divide channels");
  // (as many frames as rows, where there are none)
  require(s.frames >= (s.rows ? 1 : 0) && s.frames <= kMaxRows, "frames must be 1 .. 2^30");
  require(starts || s.rows == 0 || s.rows % s.frames == 0, "rows are not the same number for each frame, and there are no starts");
  require(s.eps >= 0.0f && s.eps < 1e30f, "eps must be a number from 0 on");
  NormArgs p{};
  p.rows = (long)s.rows;
  p.ld_x = (long)row_length(s.ld_x, s.channels, "ld_x is shorter than channels, or too long");
  p.ld_y = (long)row_length(s.ld_y, s.channels, "ld_y is shorter than channels, or too long");
  p.channels = s.channels, p.groups = s.groups, p.frames = s.frames, p.act = s.act, p.eps = s.eps;
  p.starts = static_cast<const int*>(starts);
  return p;
}

void buffers(dp_ops* O, hipStream_t st, const NormNeeds& need, NormArgs& p) {
  Regions r;
  const size_t a = r.take(need.stats), b = r.take(need.sums), c = r.take(need.pairs), d = r.take(need.partial);
  if (!r.used) return;
  char* ws = workspace(O, st, r.used);
  if (need.stats) p.stats = reinterpret_cast<float*>(ws + a);
  if (need.sums) p.sums = reinterpret_cast<float*>(ws + b);
  if (need.pairs) p.pairs = reinterpret_cast<float*>(ws + c);
  if (need.partial) p.partial = reinterpret_cast<float*>(ws + d);
}

}  // namespace
}  // namespace dpamd

using namespace dpamd;

extern "C" {

int dp_group_norm(dp_ops* O, const dp_norm_shape* shape, const void* x, const int* starts, const void* gamma,
                  const void* beta, void* y, float* stats, void* stream) {
  return guarded(O, [&]() {
    NormArgs p = norm_args(shape, starts);
    require(reinterpret_cast<uintptr_t>(stats) % 8 == 0, "stats must be 8-byte aligned");
    if (p.rows == 0) return;
    require(x && y, "null pointer");
    p.x = x, p.gamma = gamma, p.beta = beta, p.y = y, p.stats = stats;
    DPAMD_HIP(hipSetDevice(O->device));
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int elem = elem_of(shape->type);
    buffers(O, st, plan_norm(elem, O->ncu, false, p), p);
    by_elem(elem, [&](auto k) { norm_launch<decltype(k)::value>(st, p); });
  });
}

int dp_group_norm_grad(dp_ops* O, const dp_norm_shape* shape, const void* x, const void* kept, const int* starts,
                       const void* gamma, const void* beta, const float* stats, const void* dy, void* dx, void* dgamma,
                       void* dbeta, void* stream) {
  return guarded(O, [&]() {
    NormArgs p = norm_args(shape, starts);
    require(!x || !kept, "x and its checkpoint are not both given");
    require(reinterpret_cast<uintptr_t>(kept) % 16 == 0, "kept must be 16-byte aligned");
    require(reinterpret_cast<uintptr_t>(stats) % 8 == 0, "stats must be 8-byte aligned");
    if (!dx && !dgamma && !dbeta) return;
    DPAMD_HIP(hipSetDevice(O->device));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p.rows == 0) {
      const long b = p.channels * (long)bytes_of(shape->type);
      for (void* d : {dgamma, dbeta})
        if (d) fill_zero(st, d, 1, b, b);
      return;
    }
    require((x || kept) && stats && dy, "null pointer");
    p.x = x, p.kept = static_cast<const unsigned char*>(kept), p.wide = kept8_wide(p.channels);
    p.gamma = gamma, p.beta = beta, p.stats = const_cast<float*>(stats), p.dy = dy;
    p.dx = dx, p.dgamma = dgamma, p.dbeta = dbeta;
    const int elem = elem_of(shape->type);
    buffers(O, st, plan_norm(elem, O->ncu, true, p), p);
    by_elem(elem, [&](auto k) { norm_grad_launch<decltype(k)::value>(st, p); });
  });
}

}  // extern "C"
