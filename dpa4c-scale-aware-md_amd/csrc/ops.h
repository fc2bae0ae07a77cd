// Operators of trainable heads (embedding lookup, gated block): arguments and launches
// of their kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace dpamd {

// activations, with the codes of the model files
enum { kActTanh = 0, kActSilu = 1, kActGelu = 2 };

// ---- tile products (product.h) ----
enum { kEpiStore = 0, kEpiGate = 1, kEpiGateGrad = 2 };

// An operand of the products, of the call's type: 16-byte aligned, rows of whole 16-byte
// chunks (ld elements), and the contiguous side ends with a chunk or is followed by zeros up to one.
struct Operand {
  const void* p;
  long ld;
};

// h, dg and du as operands [M][ldh]; saved: g and then u, [M][N] each.
//
// h, dg and du are rounded to the call's type, once, where they are operands of the next products, whose matrix
// cores take that type (h of few rows or few outputs meets none, and stays in fp32). It costs about half a bit: errors against 64 bits, relative to the outputs' size, of
// 0.0023 in bf16 training steps (0.0017 with all of it in 32 bits and only the outputs rounded) and
// 0.00029 in fp16 forwards (0.00021). As two numbers of 16 bits each they would keep 16 bits or more, for twice the
// operations of h w_down, dx and the weights' gradients: of the 2.3 ms of a step of 8,192 rows
// through 2048-8192-2048 in bf16 these take 1.3. Who needs the digits calls with fp32.
// In f16 their range matters too: beyond 65,504 they are infinite; dg and du below 6e-5 have fewer
// bits, and below 3e-8 they are zero.
struct EpiArgs {
  void *h, *dg, *du;
  float* h32;  // h, not rounded, in place of `h` where no product follows (of a gate), or null
  long ldh;
  float* saved;
};

struct ProductArgs {
  Operand a[2], b[2];
  int M, N, K;  // N: columns of one B matrix
  int cols;     // columns written: N, or N and the zeros up to ldh
  int segs;     // 2: K runs over a[0], b[0] and then over a[1], b[1]
  int mats;     // 2: the columns of b[0] and then those of b[1], each to its own out
  int split;    // slices of K, each to its own part of `partial`
  int join;     // threads that share the slices of one quad of columns (divides 256)
  int tiles_m, tiles_n, tiles_n1;  // tiles_n1: those of one matrix
  int blocks;  // at most: those that the card holds at once
  int act;
  float* partial;
  long ldp;  // cols up to a multiple of 4
  void* out[2];
  long ldo[2];
  bool vec[2], wide[2];  // whether four, and eight, columns of a row can be stored whole
  EpiArgs epi;
};

// What a product is: which layouts and epilogue.
enum ProductKind {
  kProdGate,      // x Wg, x Wu -> h                    rows k-contiguous by columns
  kProdDown,      // h Wd -> y
  kProdGateGrad,  // dy Wd^T -> dg, du, h               both k-contiguous
  kProdInput,     // dg Wg^T + du Wu^T -> dx
  kProdWeight     // x^T dg, x^T du;  h^T dy            both k-strided
};

// How a product is cut: tile shape and slices of K, and the workspace its slices need.
struct ProductPlan {
  int shape, split, blocks;
  size_t bytes;
};
ProductPlan plan_product(ProductKind what, int elem, long M, long N, long K, int segs, int mats, int ncu);
void tile_of(int shape, int elem, int& rows, int& cols);  // of a plan's shape
void run_product(hipStream_t st, ProductKind what, int elem, const ProductPlan& plan, ProductArgs& args);

// ---- the block for a few rows (gated_rows.hip) ----
constexpr int kFewRows = 8;
struct RowsArgs {
  int rows, d, f, o, act;
  long ld_x, ld_hidden, ld_down, ld_y;
  const void *x, *wg, *wu, *wd;
  void* y;
  float* saved;
  float *partial1, *partial2;  // [slices][rows][2][f], [slices][rows][o]
  int slice1, slices1, slice2, slices2;
};
size_t plan_rows(int elem, int ncu, RowsArgs& args);  // bytes of the partial sums
void run_rows(hipStream_t st, int elem, RowsArgs& args);

// ---- the block's down side for few outputs (gated_outs.hip) ----
constexpr int kFewOutputs = 4;
struct OutsArgs {
  long rows;
  int f, o, act;
  const float* h;  // rows of ldh, zeros from f on
  const void *wd, *dy;
  const float* saved;
  long ldh, ld_down, ld_y;
  void *y, *dg, *du, *dwd;
  float* partial;  // [slices][f][o], or null: no d w_down
  int quads, groups, slices;
};
bool few_outputs(int d_hidden, int d_out);
void run_outs_down(hipStream_t st, int elem, int ncu, const OutsArgs& args);
size_t plan_outs_grad(int ncu, OutsArgs& args);  // bytes of the partial sums
void run_outs_grad(hipStream_t st, int elem, const OutsArgs& args);

// Matrices [rows][cols] to be copied into rows of ld (a multiple of 8), with zeros past cols.
struct PackItem {
  const void* src;
  long ld_src, ld;
  int cols;
  void* dst;
};
constexpr int kMaxPack = 5;
struct PackList {
  PackItem item[kMaxPack];
  long end[kMaxPack];  // running sums of the items' groups of eight elements
  int count;
};
void pack_operands(hipStream_t st, int elem, const PackList& list);
// rows x row_bytes of zeros, rows `stride` bytes apart (a kernel: may be captured)
void fill_zero(hipStream_t st, void* dst, long rows, long row_bytes, long stride);

// ---- lookup (lookup.hip) ----
void lookup_rows(hipStream_t st, int elem, long n, int vocab, int width, const int* ids,
                 const void* table, long ld_table, float scale, void* out, long ld_out);
size_t lookup_grad_bytes(int elem, long n, int vocab, int width, const void* dout, long ld, const void* dtable,
                         long ld_table);
void lookup_grad(hipStream_t st, int elem, long n, int vocab, int width, const int* ids, const void* dout,
                 long ld, float scale, void* dtable, long ld_table, char* ws);

}  // namespace dpamd
