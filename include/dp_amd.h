/*
 * dp_amd.h — C ABI of the MI355X-native DeePMD evaluator (libdpamd.so): se_e2_a
 * models and the DPA4C compressed descriptor (Nano profile).
 *
 * This is the drop-in boundary for the per-step energy / force / virial call
 * that `pair_style deepmd` makes through the DeePMD C++ model API. Every entry
 * point takes plain pointers and sizes; no torch or C++ types cross it.
 * Return value: 0 on success, a negative DP_ERR_* code on failure, with the
 * message available from dp_last_error(). The C++ façade in
 * include/deepmd_amd/DeepPot.h turns failures into deepmd::deepmd_exception,
 * as the reference does (deepmd-op/overlays/api_cc/src/DeepPotPTExpt.cc:295-309,
 * caught by lammps-deepmd-plugin/src/pair_deepmd.cpp:372-374).
 *
 * Conventions (lammps-deepmd-plugin/src/pair_deepmd.cpp:293-307, :603-621):
 *   coord  [natoms][3] Angstrom, row-major;  atype [natoms] model type index,
 *          negative = virtual atom (no energy, no force, not a neighbour);
 *   box    [9] row-major h = [xx,0,0, xy,yy,0, xz,yz,zz] (lower-triangular,
 *          LAMMPS shape), or NULL for an open (non-periodic) system;
 *   energy [1] eV;  force [natoms][3] eV/A;  virial [9] eV, row-major
 *          W[3c+d] = -sum_edges g_c (x_j - x_i)_d;
 *   atom_energy [natoms];  atom_virial [natoms][9], charged to the neighbour
 *          (source) atom as in deepmd-op/overlays/op/pt/edge_force_virial.cu:1-14.
 * Any optional output pointer may be NULL.
 *
 * Threading: one handle per host thread; calls on one handle are serialised
 * by the caller (the reference keeps thread_local caches per model,
 * DeepPotPTExpt.cc:138).
 */
#ifndef DP_AMD_H
#define DP_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DP_MAX_TYPES 8

enum {
  DP_OK = 0,
  DP_ERR_ARG = -1,      /* bad argument (null pointer, bad size, bad box) */
  DP_ERR_MODEL = -2,    /* model file missing, malformed or unsupported */
  DP_ERR_HIP = -3,      /* HIP runtime failure (allocation, launch, copy) */
  DP_ERR_CAPACITY = -4, /* a neighbour count exceeded a fixed kernel capacity */
  DP_ERR_NO_GPU = -5    /* no usable gfx950 device */
};

/* DP_PREC_MODEL: the precision the model file was written for (se_e2_a files
 * carry it in their header; DPA4C models are mixed by definition). */
enum { DP_PREC_FP64 = 0, DP_PREC_MIXED = 1, DP_PREC_MODEL = -1 };

/* Model families: se_e2_a (DPAMDSEA files) and the DPA4C compressed
 * degree-wise descriptor in its Nano profile (DPAMDC4N files). */
enum { DP_MODEL_SE_E2_A = 0, DP_MODEL_DPA4C = 1 };

typedef struct dp_model dp_model;

typedef struct {
  int ntypes;
  int nnei;
  int sel[DP_MAX_TYPES];
  double rcut;
  double rcut_smth;
  int emb[3];
  int axis;
  int fit[3];
  int dim_fparam;   /* always 0 for se_e2_a energy models here */
  int dim_aparam;   /* always 0 */
  int precision;    /* DP_PREC_* in use (DP_PREC_MIXED for DPA4C: fp32 nets) */
  char type_map[DP_MAX_TYPES][16];
  int model_kind;   /* DP_MODEL_*; for DPA4C emb = {C0, C1, C2} channel widths,
                       fit[0] = hidden width, axis = rcut_smth = 0 */
} dp_model_info;

/* Stage buffers of the last evaluation that dp_debug_copy can read back. */
enum {
  DP_STAGE_NLIST = 0,      /* int32 [nloc][nnei] (extended-atom indices, -1 pad) */
  DP_STAGE_EXT_COORD = 1,  /* f64 [nall][3] extended coordinates */
  DP_STAGE_MAPPING = 2,    /* int32 [nall] owner of each extended atom */
  DP_STAGE_DESCRPT = 3,    /* f64 [nloc][M1*axis] descriptor D (fp32 values in mixed mode) */
  DP_STAGE_ATOM_ENERGY = 4,/* f64 [nloc] */
  DP_STAGE_EDGE_GRAD = 5,  /* f64 [nloc][nnei][3] dE/d(x_j - x_i) */
  DP_STAGE_DEDD = 6,       /* f64 [nloc][M1*axis] dE/dD (fp32 values in mixed mode) */
  DP_STAGE_EXT_TYPE = 7,   /* int32 [nall] */
  DP_STAGE_C4_MOMENTS = 8, /* DPA4C: f32 [nloc][44] raw sums: scalar [8], vector [3][4],
                              tensor [5][4], sum env^2, sum env^4, 2 pad */
  DP_STAGE_C4_COTANGENTS = 9 /* DPA4C: f32 [nloc][44] dE/d(raw sums), same layout */
};

/*
 * Load a model and bind it to device `gpu_rank`.
 * Replaces deepmd::DeepPot::init(model, gpu_rank, file_content)
 * (deepmd-op/overlays/api_cc/include/DeepPot.h:475-477; called at
 * lammps-deepmd-plugin/src/pair_deepmd.cpp:668). If `file_content` is non-NULL
 * the model is read from those `content_len` bytes instead of `path`.
 * `precision` DP_PREC_MODEL takes the precision recorded in the model file
 * (upstream, the evaluation precision is a property of the trained model);
 * DP_PREC_FP64 evaluates everything in fp64; DP_PREC_MIXED
 * evaluates the descriptor and the fitting net in fp32 (and the embedding
 * nets, when they are evaluated slot by slot; their expansion is summed in
 * fp64) and the env matrix, edge gradients, forces, virials and energy
 * sums in fp64 -- the reference's mixed-precision rule (fp32
 * embedding/fitting, fp64 env matrix, force and virial accumulation), checked
 * against its acceptance limits (data/numeric-tolerances.json:3-9).
 */
int dp_create(const char* path, int gpu_rank, const void* file_content, size_t content_len,
              int precision, dp_model** out);

/* Release the handle and every device buffer it owns. */
void dp_destroy(dp_model* model);

/*
 * Model metadata: cutoff(), numb_types(), dim_fparam(), dim_aparam(),
 * get_type_map() of the reference model API
 * (deepmd-op/overlays/api_cc/include/DeepPotPTExpt.h:103-154; used at
 * lammps-deepmd-plugin/src/pair_deepmd.cpp:672-677, :1000).
 */
int dp_get_info(const dp_model* model, dp_model_info* info);

/* Message of the last failure on this handle ("" if none). */
const char* dp_last_error(const dp_model* model);

/*
 * Standalone evaluation from coordinates and box: ghost images, neighbour
 * list and evaluation are built on the GPU; ghost forces / virials are folded
 * onto their owners. Replaces DeepPot::compute(ener, force, virial,
 * [atom_energy, atom_virial,] coord, atype, box)
 * (deepmd-op/overlays/api_cc/include/DeepPot.h:503-522, :605-628;
 * backend path DeepPotPTExpt.cc:1643-1957). Host pointers.
 */
int dp_compute(dp_model* model, int natoms, const double* coord, const int* atype,
               const double* box, double* energy, double* force, double* virial,
               double* atom_energy, double* atom_virial);

/*
 * LAMMPS neighbour-list evaluation. coord/atype cover nall = nloc + nghost
 * atoms; the neighbour list (inum, ilist, numneigh, firstneigh) is LAMMPS'
 * full list with skin, indices into the nall atoms (masked with `neigh_mask`,
 * pass 0x1FFFFFFF for LAMMPS' NEIGHMASK, or 0 for no mask). force and
 * atom_virial cover all nall atoms; ghost contributions stay in ghost slots for
 * LAMMPS' reverse communication. `ago == 0` means the list was rebuilt and is
 * re-uploaded; otherwise the cached list is reused and only re-filtered.
 * Replaces DeepPot::compute(ener, force, virial, [atom_energy, atom_virial,]
 * coord, atype, box, nghost, lmp_list, ago)
 * (deepmd-op/overlays/api_cc/include/DeepPot.h:551-576, :661-690; called at
 * lammps-deepmd-plugin/src/pair_deepmd.cpp:370-371, :381-383). Host pointers.
 */
int dp_compute_nlist(dp_model* model, int nall, int nghost, const double* coord,
                     const int* atype, const double* box, int inum, const int* ilist,
                     const int* numneigh, const int* const* firstneigh, int neigh_mask, int ago,
                     double* energy, double* force, double* virial, double* atom_energy,
                     double* atom_virial);

/*
 * Device-resident standalone evaluation: every array pointer is device memory
 * on the handle's GPU except `box` (host, 9 doubles); work is ordered on
 * `stream` (a hipStream_t, NULL = default stream) and the call returns after
 * the outputs are complete on that stream. `ago == 0` refreshes the per-type
 * bucketing of atype (read back once); otherwise the previous one is reused.
 * Device analog of DeepPot::compute_canonical_graph_gpu / compute_edges_gpu
 * (deepmd-op/overlays/api_cc/include/DeepPot.h:395-445), which also write in
 * place into caller-owned device buffers (DeepPotPTExpt.cc:2843-2847).
 */
int dp_compute_device(dp_model* model, int natoms, const double* d_coord, const int* d_atype,
                      const double* box, int ago, double* d_energy, double* d_force,
                      double* d_virial, double* d_atom_energy, double* d_atom_virial,
                      void* stream);

/*
 * Asynchronous form of dp_compute_device for an MD loop that keeps its data on
 * the GPU: the evaluation is enqueued on `stream` and the call returns without
 * waiting for it, so consecutive steps (and the caller's own kernels between
 * them) queue back to back with no host round trip. With ago != 0 and the
 * same natoms as the previous call nothing is read back, and nothing is
 * allocated once the buffers have grown to the system's size; ago == 0 reads
 * the types back once, as dp_compute_device does. The outputs are complete
 * when `stream` reaches the point of the call. A capacity error raised by the
 * kernels (more than 512 neighbours within rcut of one atom, more than 1024
 * edges pointing at one atom) is returned by the first later call of this
 * function that sees it, or by dp_sync; the outputs of that evaluation and of
 * those queued after it are then invalid. Any other entry point first waits
 * for the queued evaluations (and returns such an error). Analog of the
 * reference's GPU-resident step, which hands the model outputs to the MD
 * engine's stream through events with no host synchronisation
 * (deepmd-op/overlays/api_cc/include/DeepPot.h:14-18,
 * deepmd-op/overlays/api_cc/src/DeepPotPTExpt.cc:194-222, used at
 * deepmd-op/overlays/lmp/pair_deepmd_kokkos.cpp:555-606).
 */
int dp_compute_device_async(dp_model* model, int natoms, const double* d_coord,
                            const int* d_atype, const double* box, int ago, double* d_energy,
                            double* d_force, double* d_virial, double* d_atom_energy,
                            double* d_atom_virial, void* stream);

/*
 * dp_compute_device (with ago == 0) that allocates nothing: every work
 * buffer of the evaluation is carved from a static scratch array of
 * DP_NOALLOC_SCRATCH_BYTES (128 MiB) that the library holds on each GPU it
 * runs on until the process ends, and no hipMalloc, hipFree or allocating
 * library routine is called (no vendor GEMM either: the plain GEMMs run as
 * this library's own kernels, and the per-type chains on `stream` alone).
 * The caller passes inputs and outputs; the handle's own buffers are left as
 * they were. A system whose work buffers exceed the scratch is rejected
 * with DP_ERR_CAPACITY (the outputs are then unspecified; the handle keeps
 * working). Every handle on one GPU shares that GPU's scratch: the library
 * serialises the calls of several host threads on one GPU (a per-device
 * lock held for the whole call), but work the caller queues on other streams
 * that reads or writes the scratch's contents is not ordered against it.
 * The call is synchronous: it reads the atom types back to the host and
 * returns when the outputs are complete, so it cannot be recorded into a
 * HIP graph; on a stream that is being captured it returns DP_ERR_ARG
 * without touching the stream. No counterpart in the reference: for
 * callers that cannot allocate device memory (serving loops and harnesses
 * that forbid hipMalloc).
 */
#define DP_NOALLOC_SCRATCH_BYTES (128u << 20)
int dp_compute_device_noalloc(dp_model* model, int natoms, const double* d_coord,
                              const int* d_atype, const double* box, double* d_energy,
                              double* d_force, double* d_virial, double* d_atom_energy,
                              double* d_atom_virial, void* stream);

/* With the environment variable DPAMD_GRAPH=1 set when the handle is
 * created, dp_compute_device_async replays the evaluation as a HIP graph: the
 * first call with a given key (natoms, every pointer, the box, the stream)
 * runs eagerly and sizes the buffers, the second captures the evaluation on a
 * stream of the handle's own, and later calls with the same key replay it
 * (a new key captures again; a failed capture turns graphs off for the
 * handle). Stage timing (dp_stage_times) runs eagerly. As the reference's
 * DPA_MODEL_GRAPH replay (deepmd-op/overlays/api_cc/src/DeepPotPTExpt.cc:
 * 122-191), keyed on pointers and sizes. dp_graph_stats reports the captures
 * and replays so far and returns 1 while graphs are in use, 0 otherwise. */
int dp_graph_stats(const dp_model* model, long* captures, long* replays);

/* Waits for every evaluation queued by dp_compute_device_async; returns
 * DP_ERR_CAPACITY (and clears the flag) if any of them overflowed, DP_OK
 * otherwise. Stage times then refer to the last of them. No counterpart in the
 * reference, whose errors surface at the next synchronous call. */
int dp_sync(dp_model* model);

/*
 * DPA4C evaluation of a compact canonical graph, all pointers device memory:
 * d_atype [nall_nodes] int64 model types; edges sorted by destination, with
 * d_destination_row_ptr [nall_nodes + 1] their CSR over destination nodes,
 * d_source [edge_storage] the source node of each edge and d_edge_vec
 * [edge_storage][3] fp32 x_source - x_destination; d_source_row_ptr /
 * d_source_order the CSR of the same edges by source (positions into the edge
 * arrays). Only local destinations (< nloc) carry model edges; slots past them
 * are reserved. Writes d_atom_energy [nloc], d_force [nall_nodes][3] =
 * sum(dst=n) g - sum(src=n) g and d_atom_virial [nall_nodes][9] = -sum(src=n)
 * g (x) d with g = dE/dd, ghost contributions left in ghost slots; work is
 * ordered on `stream` and complete when the call returns. Replaces
 * DeepPot::compute_canonical_graph_gpu (deepmd-op/overlays/api_cc/include/
 * DeepPot.h:430-442, DeepPotPTExpt.cc:2747-2908, same argument meanings and
 * the same dimension checks); forces follow
 * deepmd-op/overlays/op/pt/edge_force_virial.cu:1-14. DP_ERR_MODEL for an
 * se_e2_a model, DP_ERR_ARG for a type or source outside the model / graph.
 */
int dp_compute_canonical_graph_device(dp_model* model, double* d_atom_energy, double* d_force,
                                      double* d_atom_virial, const int64_t* d_atype,
                                      const uint32_t* d_source, const float* d_edge_vec,
                                      const int64_t* d_destination_row_ptr,
                                      const int64_t* d_source_row_ptr,
                                      const uint32_t* d_source_order, int nloc, int nall_nodes,
                                      int64_t edge_storage, void* stream);

/*
 * Device-resident evaluation of a caller-built edge graph, all arrays device
 * memory, work ordered on `stream` and complete on return. Replaces
 * DeepPot::compute_edges_gpu (deepmd-op/overlays/api_cc/include/DeepPot.h:
 * 395-429; backend DeepPotPTExpt.cc:2402-2740; called by the Kokkos pair,
 * lmp/pair_deepmd_kokkos.cpp:586-597), with its argument meanings:
 * d_edge_index int32 [2][nedge], row 0 the neighbour (source) node and row 1
 * the centre (destination, < nloc); d_edge_vec [nedge][3] = r_neighbour -
 * r_centre (fp64, or fp32 in the _f32 form); d_atype int32 [nall_nodes]
 * model types; nall_nodes = nloc folds every edge onto local source nodes
 * (single domain), nall_nodes > nloc keeps ghost nodes whose forces the
 * caller's reverse communication folds. Edges beyond rcut (a skin) are
 * filtered; d_coord is accepted for the signature and not read (the edge
 * vectors carry the geometry). Outputs: d_atom_energy [nloc], d_force
 * [nall_nodes][3], d_atom_virial [nall_nodes][9] (charged to the source
 * node). Works for both model families; an edge naming a node outside the
 * graph gives DP_ERR_ARG. For se_e2_a the local types are read back each call
 * (nloc ints) to group centres by type.
 */
int dp_compute_edges_device(dp_model* model, double* d_atom_energy, double* d_force,
                            double* d_atom_virial, const double* d_coord, const int* d_atype,
                            const int* d_edge_index, const double* d_edge_vec, int nloc,
                            int nedge, int nall_nodes, void* stream);
int dp_compute_edges_device_f32(dp_model* model, double* d_atom_energy, double* d_force,
                                double* d_atom_virial, const double* d_coord, const int* d_atype,
                                const int* d_edge_index, const float* d_edge_vec, int nloc,
                                int nedge, int nall_nodes, void* stream);

/* Copy a stage buffer of the last evaluation (DP_STAGE_*) to host memory.
 * Returns the buffer's size in bytes (copies min(size, capacity) bytes);
 * negative on error. No counterpart in the reference: parity tests use it to
 * compare each pipeline stage with the CPU oracle (the reference's own
 * analogue is its DPA_DUMP_FRAME hook, graph_compress.cu:1354-1378). */
long dp_debug_copy(dp_model* model, int stage, void* dst, size_t capacity);

/* keep != 0: the evaluations that follow also store their per-slot edge
 * gradients, so dp_debug_copy can return DP_STAGE_EDGE_GRAD (the se_e2_a
 * force stage otherwise scatters them into the forces without writing them);
 * keep == 0 (the default) switches that off again. No counterpart in the
 * reference: a parity-test hook, like dp_debug_copy. */
int dp_debug_keep(dp_model* model, int keep);

/* se_e2_a in fp64 forms dE/dT from the fitting's input gradient with a fused
 * kernel (dE/dD never stored) when every atom type has at least `rows` atoms
 * (default 12288; 0: always), and otherwise as the plain product
 * dE/dD = dZ0 W0^T followed by a separate dE/dT pass, which is faster for
 * few atoms per type. Systems of a few hundred to a few thousand atoms in all
 * run a set of kernels of their own (both precisions); rows == 0 switches
 * those off too. All forms give the same results to rounding. No
 * counterpart in the reference: a parity-test hook, so that each form is
 * checked at the sizes the oracle evaluates. */
int dp_debug_fused_rows(dp_model* model, int rows);

/* se_e2_a: systems of at most `rows` atoms run the few-atoms fitting kernels
 * (0: none, the forms above then apply to small systems too; negative, the
 * default: the library's own rule). dp_debug_fitting_form names the form that the
 * last evaluation ran. No counterparts in the reference: parity-test hooks. */
enum {
  DP_FIT_NONE = 0,  /* no se_e2_a evaluation yet */
  DP_FIT_FEW = 1,   /* the few-atoms kernels */
  DP_FIT_PLAIN = 2, /* dE/dD = dZ0 W0^T stored, then the dE/dT pass */
  DP_FIT_FUSED = 3  /* the fused input-gradient kernel */
};
int dp_debug_few_rows(dp_model* model, int rows);
int dp_debug_fitting_form(const dp_model* model);

/* Per-stage GPU time in milliseconds (hipEvent pairs) of the last synchronous
 * evaluation, or the mean over the evaluations queued by
 * dp_compute_device_async up to the last dp_sync, filled into times[0..n-1] in
 * pipeline order; returns the number of stages and writes their names into
 * names (NUL separated) when non-NULL. `enable` switches the timers on or off
 * for the evaluations that follow. The reference's analogue is its DPA_KTIME
 * stage timer (graph_compress.cu:1394-1427). */
int dp_stage_times(dp_model* model, int enable, double* times, int n, char* names, size_t names_len);

/* Peak device bytes allocated by this handle so far (memory high-water mark). */
size_t dp_device_bytes(const dp_model* model);

/*
 * Operators of trainable heads: what a per-atom (or per-token) net on top of
 * descriptors or embeddings needs, forward and backward, and served in 8 bits. No counterpart in the
 * reference, whose nets are evaluated inside its model. Every array is device memory
 * on the handle's GPU; work is ordered on `stream` (a hipStream_t, NULL = default
 * stream) and the calls return without waiting for it. Matrices are row-major;
 * a row length (ld_*) of 0 means packed rows. Inputs and outputs of one call must
 * not overlap. Weights are [in][out], as in the model files.
 *
 * Types: DP_TYPE_F32, DP_TYPE_BF16 or DP_TYPE_F16 for every matrix of a call. Products
 * run on the matrix cores of that type (a forward of up to eight rows, and the products with w_down
 * of up to four outputs, on the vector units, in fp32); sums are held in fp32 and rounded once. Of
 * the matrices between the products only h, dg and du are rounded to the type; h is not
 * in a forward of up to eight rows, and with up to four outputs (to 8,192 hidden columns of one
 * output, 4,096 of two, 2,048 of three and four) in y and dw_down. In f16 a value
 * of theirs past 65,504 is then infinite (of h: with more outputs, y from nine rows on, and dw_down from any
 * number of rows), and dg and du lose bits below 6e-5 and are zero below 3e-8: the backward
 * is linear in dy, so a caller whose dy is small scales it by a power of two, and the
 * gradients back. tanh and gelu are evaluated to about
 * 2e-7 of themselves (4e-6 where gelu is about to vanish), silu and the derivatives of silu and gelu, which have
 * zeros, to about 2e-7 of max(1, |g|).
 * Results do not depend on the order in which blocks run: a call repeated on the
 * same inputs at the same alignment gives the same bits.
 *
 * A handle keeps one workspace for each stream it is used with, which grows to the largest call and
 * is released by dp_ops_destroy. It knows a stream by its address: destroy a stream only once its
 * work has ended, as one created later may have the same address and takes over the workspace.
 * Calls on several streams need no ordering by the caller beyond that of their own inputs
 * and outputs. The calls can be captured into a HIP graph once the same call has run
 * on that stream (so that the workspace is there; else DP_ERR_ARG); a workspace that a
 * capture has seen is kept until dp_ops_destroy, and replays must not run beside
 * other calls that use it. One handle per host thread; dp_ops_destroy waits for the
 * handle's streams' work.
 */
typedef struct dp_ops dp_ops;
enum { DP_TYPE_F32 = 0, DP_TYPE_BF16 = 1, DP_TYPE_F16 = 2 };
/* activations; the first two have the codes of the DPA4C model files */
enum { DP_ACT_TANH = 0, DP_ACT_SILU = 1, DP_ACT_GELU = 2 };

int dp_ops_create(int gpu_rank, dp_ops** out);
void dp_ops_destroy(dp_ops* ops);
const char* dp_ops_last_error(const dp_ops* ops);
/* Peak device bytes of the handle's workspaces. */
size_t dp_ops_device_bytes(const dp_ops* ops);

/*
 * out[i] = scale * table[ids[i]], i < n: the rows of a table [vocab][width] that the
 * ids name (atom types, tokens), 32-bit integers. An id outside 0 .. vocab - 1 (a virtual atom,
 * padding) gives a row of zeros. One multiplication in fp32, rounded once. ld_table
 * and ld_out: row lengths, so the rows can be columns of wider matrices (the type
 * columns of a descriptor). With n == 0 nothing is done and the arrays may be NULL.
 */
int dp_embed(dp_ops* ops, int type, int64_t n, int vocab, int width, const int* d_ids,
             const void* d_table, int64_t ld_table, float scale, void* d_out, int64_t ld_out,
             void* stream);

/*
 * The gradient of dp_embed's table: dtable[v] = scale * sum of dout[i] over the i
 * with ids[i] == v, every row of dtable written (zeros where no id names it; with n == 0,
 * where ids and dout may be NULL, all of it).
 * Each row's sum is formed in fp32 and rounded once. Its order depends on the ids, the sizes, and the
 * alignment and row lengths of dout and dtable, not on the order in which blocks run.
 */
int dp_embed_grad(dp_ops* ops, int type, int64_t n, int vocab, int width, const int* d_ids,
                  const void* d_dout, int64_t ld_dout, float scale, void* d_dtable,
                  int64_t ld_dtable, void* stream);

/*
 * The gated feed-forward block y = h w_down, h = act(x w_gate) * (x w_up):
 * x [rows][d_in], w_gate and w_up [d_in][d_hidden], w_down [d_hidden][d_out],
 * y [rows][d_out]. ld_hidden is the row length of w_gate, w_up and of their gradients
 * (2 d_hidden for the two stored side by side), ld_down that of w_down and its gradient.
 */
typedef struct {
  int64_t rows;
  int d_in, d_hidden, d_out;
  int type, act;
  int64_t ld_x;      /* x and dx */
  int64_t ld_y;      /* y and dy */
  int64_t ld_hidden; /* w_gate, w_up and their gradients */
  int64_t ld_down;   /* w_down and its gradient */
} dp_gated_shape;

/* Bytes that dp_gated_forward keeps for dp_gated_backward: x w_gate and x w_up in fp32, 8 bytes
 * for each of rows * d_hidden. 0 for a shape that the calls refuse. */
size_t dp_gated_saved_bytes(const dp_gated_shape* shape);

/* How the block's tile products are cut on a GPU of `compute_units`: rows and columns of a tile, and slices
 * of the summed axis, three integers for each of the products x w_gate and x w_up, h w_down, dh, dx, dw_gate and
 * dw_up, dw_down; zeros for those that other kernels form (up to eight rows, up to four outputs). A test hook, so
 * that each tile and its sliced form are known to be tested. */
enum { DP_GATED_PRODUCTS = 6 };
int dp_debug_gated_plan(const dp_gated_shape* shape, int compute_units, int* plan);

/* d_saved: NULL (no backward follows) or dp_gated_saved_bytes bytes, 16-byte aligned. */
int dp_gated_forward(dp_ops* ops, const dp_gated_shape* shape, const void* d_x,
                     const void* d_w_gate, const void* d_w_up, const void* d_w_down, void* d_y,
                     void* d_saved, void* stream);

/*
 * From dy and what the forward kept: dx = dg w_gate^T + du w_up^T, dw_gate = x^T dg,
 * dw_up = x^T du, dw_down = h^T dy, with dh = dy w_down^T, du = dh * act(g) and
 * dg = dh * u * act'(g). An output that is NULL is not formed (dx of frozen descriptors;
 * dw_gate and dw_up are both given or both NULL). With rows == 0 the weights'
 * gradients are zeros.
 */
int dp_gated_backward(dp_ops* ops, const dp_gated_shape* shape, const void* d_x,
                      const void* d_w_gate, const void* d_w_up, const void* d_w_down,
                      const void* d_saved, const void* d_dy, void* d_dx, void* d_dw_gate,
                      void* d_dw_up, void* d_dw_down, void* stream);

/*
 * Checkpoints of activations in 8 bits: what the forward of a layer keeps of its input x [rows][cols] for the
 * backward, 33 bits for every four values. A row's columns are in groups of 32 (the last one may be shorter). Each
 * group has a unit, a power of two, 2^(floor(log2 max |x|) - 6) (at least 2^-133), and x is held as the multiple
 * of it that is nearest (ties to the even one), at most 127 in magnitude: off by at most half a unit, or a
 * whole one in the last 127th below the next power of two. What is restored is a number of all three types
 * (in f16 where x was one); a group with an infinity or a NaN is restored as NaN.
 * `kept`: dp_keep8_bytes bytes (0 for sizes that the calls refuse), 16-byte aligned: the integers [rows][cols up
 * to a multiple of 32], then a byte for each group, the biased exponent of its largest value. With rows == 0 nothing
 * is done.
 */
size_t dp_keep8_bytes(int64_t rows, int cols);
int dp_keep8(dp_ops* ops, int type, int64_t rows, int cols, const void* d_x, int64_t ld_x,
             void* d_kept, void* stream);
int dp_restore8(dp_ops* ops, int type, int64_t rows, int cols, const void* d_kept, void* d_x,
                int64_t ld_x, void* stream);

/*
 * dp_gated_backward from the checkpoint of x [rows][d_in] alone, with nothing kept by the forward (d_saved
 * NULL): x w_gate and x w_up are formed again from the restored x, and the gradients are those of the block
 * there. It keeps d_in * 33 / 32 bytes a row in place of x and 8 d_hidden. The workspace, which the calls of all layers
 * on a stream share, takes for the time of the call x, dg, du and (for d_w_down) h in the call's type, and in fp32 dh: once, or
 * with few rows once for each slice of its sum (64 rows of 64-512-4096: 15). With up to four outputs there is neither h
 * nor dh, but x w_gate and x w_up in fp32 where their sums are sliced. (2048-8192-2048 in bf16: 84 KB a row for the call
 * of one layer, where each layer's forward would keep 64.) Beside them stand the operands that are not whole 16-byte
 * chunks and the slices of the largest product, as in dp_gated_backward.
 */
int dp_gated_backward8(dp_ops* ops, const dp_gated_shape* shape, const void* d_kept,
                       const void* d_w_gate, const void* d_w_up, const void* d_w_down,
                       const void* d_dy, void* d_dx, void* d_dw_gate, void* d_dw_up,
                       void* d_dw_down, void* stream);

/* dp_debug_gated_plan for it: the gate that keeps x w_gate and x w_up (up to four outputs, where it is sliced), the
 * gate with its gradient of five outputs and more, of two to four, of one (one of these four runs), dh, dx, dw_gate
 * and dw_up, dw_down. */
enum { DP_GATED_PRODUCTS8 = 8 };
int dp_debug_gated_plan8(const dp_gated_shape* shape, int compute_units, int* plan);

/*
 * Products in 8-bit integers, to serve what was trained: weights with a scale for each output channel, laid out once,
 * and rows of x (tokens, atoms) quantised in the call with a scale each. A row or channel is held as
 *   scale = max |x| / 127,  q = x * (127 / max |x|) to the nearest integer (ties to the even one),
 * both quotients rounded to fp32, the product with x exact. One whose largest magnitude is below 2^-119
 * counts as zeros; one with an infinity or a NaN has a scale of NaN, and all that comes of it is NaN.
 *
 * dp_weights8: w [d_in][d_out] of a type -> d_w8 [d_out][ld_w8] integers (16-byte aligned; ld_w8 a multiple of 16, 0:
 * d_in up to one) and d_scale [d_out]. Past d_in there are zeros up to a multiple of 16, and what lies between the
 * rows beyond it is left as it was.
 */
int dp_weights8(dp_ops* ops, int type, int d_in, int d_out, const void* d_w, int64_t ld_w,
                void* d_w8, int64_t ld_w8, float* d_scale, void* stream);

/*
 * y = act(g), or act(g) * u with d_up (the gate half of the block; its down half is a call on y), where
 * g = (sum over k of q_x q_w) scale_x scale_w, and u the same of the second weights: the sums are exact (d_in is at
 * most 2^17), g and u are fp32, and y is rounded once. The integers may be any, from dp_weights8 or
 * not; what lies past d_in in their rows is not looked at, but has to be readable up to a multiple of 16.
 * The activations are those of the block, and DP_ACT_NONE; with results of 16 bits gelu's normal distribution is off by
 * 2.2e-7, or by 2.2e-5 of itself in the tail, where that is less.
 */
enum { DP_ACT_NONE = 3 };
typedef struct {
  int64_t rows;
  int d_in, d_out;
  int type, act;
  int64_t ld_x, ld_y;
  int64_t ld_w; /* of the 8-bit weights, both of them, in bytes: a multiple of 16 (0: d_in up to one) */
} dp_linear8_shape;
int dp_linear8(dp_ops* ops, const dp_linear8_shape* shape, const void* d_x, const void* d_w,
               const float* d_w_scale, const void* d_up, const float* d_up_scale, void* d_y,
               void* stream);

/*
 * Group norm with an activation, channels last: rows (atoms, positions) of `channels` in `groups` of neighbouring
 * ones, rows of a frame (a cell, a sample) normalised together,
 *   y = act(gamma (x - m) r + beta),  m the mean and r = 1 / sqrt(variance + eps) of the frame's rows over the
 * group's channels (the variance around m, over their number). gamma and beta [channels] of the call's type, or
 * NULL: ones, zeros. Frames are `frames` equal parts of the rows (rows of them, 0 of 0: each row by itself), or with d_starts
 * [frames + 1] (32-bit integers) the rows starts[f] .. starts[f + 1] - 1, not descending; a frame may be empty,
 * and rows before the first and behind the last one are left as they were. What starts holds beyond the rows is cut
 * off. The work is cut by the mean length, rows / frames, as the call does not know the others: all rows of a frame over a
 * part of its columns may be one block's, so a frame of many times the mean is better given a call of its own, and
 * `frames` the number that there are (131,072 x 256 in 32 groups, bf16: 4,096 frames of like length 38 us, gradients 63;
 * one ten times as long 44 and 68; nearly all rows in one of them 9.8 and 17.9 ms). d_stats: NULL, or [frames][groups] pairs of m and r in fp32 (8-byte aligned; zeros for an empty frame), for
 * the backward. m, r and all sums are formed in fp32 or fp64 (never as a difference of large sums), y is rounded
 * once. The activations are those of the block, in 16 bits gelu as in dp_linear8. A NaN or an infinity makes
 * its frame's group NaN, and so do values whose sum, or deviations whose squares' sum, leaves fp32's range (deviations of
 * 1e19, or of 1e16 over a million values; a mean of 1e32 over as many). A variance + eps below 2^-126 (which takes an eps
 * of 0, or almost) counts as zero: r is infinite. With rows == 0 nothing is done.
 */
typedef struct {
  int64_t rows;
  int channels, groups;
  int frames;
  int type, act; /* DP_ACT_NONE too */
  float eps;
  int64_t ld_x; /* x and dx */
  int64_t ld_y; /* y and dy */
} dp_norm_shape;
int dp_group_norm(dp_ops* ops, const dp_norm_shape* shape, const void* d_x, const int* d_starts,
                  const void* d_gamma, const void* d_beta, void* d_y, float* d_stats, void* stream);

/*
 * With v = (x - m) r, dz = dy act'(gamma v + beta) and w = gamma dz: dx = r (w - mean w - v mean(w v)), the means
 * over the frame's rows and the group's channels, dgamma = sum of dz v and dbeta = sum of dz over all frames' rows.
 * x, or in its place (d_x NULL) its checkpoint from dp_keep8, at whose values the gradients are then taken, with the
 * forward's m and r. An output that is NULL is not formed; dx of rows that are in no frame is left as it was. With rows
 * == 0 dgamma and dbeta are zeros.
 */
int dp_group_norm_grad(dp_ops* ops, const dp_norm_shape* shape, const void* d_x, const void* d_kept,
                       const int* d_starts, const void* d_gamma, const void* d_beta,
                       const float* d_stats, const void* d_dy, void* d_dx, void* d_dgamma,
                       void* d_dbeta, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DP_AMD_H */
