// Group norm with an activation: arguments of its kernels (norm.hip).
#pragma once

#include "ops.h"

namespace dpamd {

struct NormArgs {
  long rows, ld_x, ld_y;
  int channels, groups, per;  // per: channels of a group
  int frames, act;
  float eps;
  const int* starts;  // [frames + 1], or null: equal frames
  const void *x, *gamma, *beta, *dy;
  const unsigned char* kept;  // the checkpoint in place of x (gradients), or null
  int wide;                   // its row length
  void *y, *dx, *dgamma, *dbeta;
  float* stats;  // [frames][groups][2]: mean, 1 / deviation

  // how it is cut
  int vec, vecs;  // channels that a thread takes at once, and how many times that is a row
  bool general;   // groups are not multiples of `vec`: the sums' entries are channels; else vectors
  int entries, group_entries;    // of a row, of a group
  float inv_entries, inv_per;    // 1 / group_entries, 1 / per
  bool pieces;    // kNormRows: groups of `vec` channels or more, of which a vector meets two at most: two entries a vector
  int form;       // NormForm
  bool by_lanes;  // kNormRows: a group's vectors are neighbouring lanes
  int lanes;      // log2 of the lanes that sum one group's entries
  int part;       // vectors of a block's columns, `part_channels` channels (whole groups with kNormFrames)
  int part_channels, parts;
  int part_groups;  // kNormSlices: groups that a part may meet
  int slices, out_slices;  // (the output's pass has slices of its own)
  int blocks;              // of the persistent kernels
  bool once;               // y and dx are stored past the caches
  float* partial;  // dgamma and dbeta of blocks or slices, or null: none
  float* pairs;    // two sums of each group of a slice and part
  float* sums;     // [frames][groups][2]: means of gamma dz and gamma dz v
};

// kNormRows: every row a frame of its own, 4 to 256 threads a row, in registers.
// kNormFrames: a block takes whole frames over a part of the groups; each thread's first rows stay in registers, what
// is beyond them is read twice.
// kNormSlices: frames cut into slices of rows, whose sums meet in memory.
enum NormForm { kNormRows = 0, kNormFrames = 1, kNormSlices = 2 };

// Chooses the form; the bytes that its buffers take.
struct NormNeeds {
  size_t stats, sums, pairs, partial;
};
NormNeeds plan_norm(int elem, int ncu, bool grad, NormArgs& args);

template <int KIND>
void norm_launch(hipStream_t st, const NormArgs& args);
template <int KIND>
void norm_grad_launch(hipStream_t st, const NormArgs& args);

}  // namespace dpamd
