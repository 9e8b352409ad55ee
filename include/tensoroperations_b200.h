/*
 * tensoroperations_b200.h -- C ABI of the B200 (sm_100a) evaluator for the
 * fused spectral-element stiffness path of TensorOperations.
 *
 * Everything here is plain C: pointers, sizes and integer status codes.  No
 * call traps or aborts; every failure comes back as a non-zero `to_status`
 * and `to_last_error()` holds a one-line reason for the calling thread.
 * Device pointers are CUDA device addresses of the current device; `stream`
 * arguments are `cudaStream_t` values passed as `void*` (NULL = legacy
 * default stream).  Nothing in a launch entry point allocates device memory.
 *
 * The reference interface each entry point replaces is cited as
 * path:line inside Rohit-Kakodkar/TensorOperations.
 */
#ifndef TENSOROPERATIONS_B200_H_
#define TENSOROPERATIONS_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TO_ABI_VERSION 2

typedef enum to_status {
  TO_OK = 0,
  TO_ERR_INVALID_ARGUMENT = 1, /* null pointer, bad size, bad enum          */
  TO_ERR_UNSUPPORTED = 2,      /* dtype / NGLL combination not built        */
  TO_ERR_CUDA = 3,             /* a CUDA runtime call failed                */
  TO_ERR_SCRATCH = 4,          /* shared-memory request above device limit  */
  TO_ERR_ALIGNMENT = 5,        /* a pointer is not aligned as required      */
  TO_ERR_TIMEOUT = 6,          /* a bounded device-side wait gave up        */
  TO_ERR_COMM = 7,             /* a collective / peer exchange failed       */
  TO_ERR_NO_DEVICE = 8,        /* no CUDA device visible                    */
  TO_ERR_GRID = 9              /* a LabelWhole label longer than its tile   */
} to_status;

typedef enum to_dtype {
  TO_F32 = 0,
  TO_F64 = 1,
  TO_BF16 = 2 /* the sequence operators only; the others reject it */
} to_dtype;

/* ---------------------------------------------------------------------- */
/* Library                                                                 */
/* ---------------------------------------------------------------------- */

/* ABI version of the loaded library (compare with TO_ABI_VERSION). */
int to_abi_version(void);

/* Static text for a status code. */
const char* to_status_string(int status);

/* Detail of the last failure on the calling thread ("" if none). */
const char* to_last_error(void);

/* Number of SMs of the current device, or a negative to_status. */
int to_device_sm_count(void);

/* Device status word of the current device: TO_OK, or the status a kernel
 * recorded instead of trapping (TO_ERR_TIMEOUT when a bounded wait gave up).
 * Synchronous (reads device memory).  reset != 0 clears it. */
int to_device_status(int32_t reset);

/* ---------------------------------------------------------------------- */
/* Mesh and operators (host utilities)                                     */
/* ---------------------------------------------------------------------- */

/*
 * Structured shared-node numbering of an nex x ney x nez hexahedral mesh with
 * NGLL points per direction.  Element e = (ez*ney + ey)*nex + ex; node
 *   ibool[e][k][j][i] = ((ez*(N-1)+k)*ny + ey*(N-1)+j)*nx + ex*(N-1)+i,
 * nx = nex*(N-1)+1 (same for y, z).  `ibool` is a HOST buffer of
 * nex*ney*nez*N^3 int32.  The reference has no global numbering: its SEM
 * programs are element-local (benchmarks/sem_stiffness/bench_sem_stiffness.cpp:8-11,
 * benchmarks/sem_stiffness_3d/bench_sem3d_levelgraph.cpp:104-105); this
 * defines the one the assembled mode uses.
 */
int to_mesh_structured_ibool(int32_t nex, int32_t ney, int32_t nez,
                             int32_t ngll, int32_t* ibool);

/*
 * GLL nodes, weights, derivative matrix H(i,p) = l_p'(x_i) and the weighted
 * transpose Hw(q,i) = H(q,i) * w(q) (hprimewgll), all HOST double arrays
 * (nodes/weights [N], hprime/hprimewgll [N][N]).  Any pointer may be NULL.
 * 2 <= ngll <= 16.
 */
int to_gll_operators(int32_t ngll, double* nodes, double* weights,
                     double* hprime, double* hprimewgll);

/*
 * Seeded synthetic fill of a HOST buffer: dst[n] of `dtype`.  Element m gets
 * a value derived from splitmix64(seed, m) only, so any slice can be
 * generated independently and identically anywhere.
 *   dist 0: Uniform[a, b)      dist 1: Normal(mean a, stddev b)
 */
int to_synth_fill(void* dst, int32_t dtype, int64_t n, uint64_t seed,
                  int32_t dist, double a, double b);

/* The slice [first, first + n) of the same sequence: dst[i] is element
 * first + i of to_synth_fill's output (how a z-slab rank generates exactly its
 * part of a global problem). */
int to_synth_fill_at(void* dst, int32_t dtype, int64_t first, int64_t n, uint64_t seed,
                     int32_t dist, double a, double b);

/* The same generators on the DEVICE, for problems too large for host memory:
 * dst[i] = (element first + i of the sequence) + add, converted to dtype, and
 * the structured numbering written to a device int32 buffer.  Uniform values
 * equal the host's bit for bit; normal values use the device's log / cos.
 * to_axpy2_device: y += 2 x (l2m = lambda + 2 mu in place).  Asynchronous. */
int to_synth_fill_device(void* dst, int32_t dtype, int64_t first, int64_t n, uint64_t seed,
                         int32_t dist, double a, double b, double add, void* stream);
int to_axpy2_device(void* y, const void* x, int32_t dtype, int64_t n, void* stream);
int to_mesh_structured_ibool_device(int32_t nex, int32_t ney, int32_t nez, int32_t ngll,
                                    int32_t* ibool, void* stream);

/* ---------------------------------------------------------------------- */
/* SEM 3D isotropic-elastic stiffness operator                             */
/* ---------------------------------------------------------------------- */
/*
 * One application f = K u of the pipeline the reference builds as a
 * LevelGraph in benchmarks/sem_stiffness_3d/bench_sem3d_levelgraph.cpp:247-351
 * (stage H,Hw | stage u | 9 gradient contractions | 1 nine-output combine
 * Integrand9 | 9 divergence contractions | 3 WeightedSum combines) and
 * launches through LevelOutputs::execute (include/TensorOperations/LevelGraph.hpp:664-667):
 *
 *   grad    dxi_c = sum_p H(i,p) u_c(k,j,p)   (and eta over j, gamma over k)
 *   stress  ds = chain_rule(dxi,deta,dgam,J); sigma = mu(ds+ds^T)+lambda tr(ds) I,
 *           lambda = l2m - 2 mu
 *   flux    F^r_c = jac * sum_d sigma[c][d] J[r][d]
 *   div     t^xi_c = sum_q Hw(q,i) F^xi_c(k,j,q)  (eta over j, gamma over k)
 *   force   f_c = w_j w_k t^xi_c + w_i w_k t^eta_c + w_i w_j t^gam_c
 *
 * Per-point arrays are [E][k][j][i] (i fastest), one array per quantity, as the
 * reference's Kokkos::View<T*[N][N][N], LayoutRight> fields.
 * Element-local mode (ibool == NULL): u_c and f_c are [E][N][N][N] and f is
 * overwritten.  Assembled mode: u_c and f_c are [nglob] and f_c[ibool[...]]
 * receives the scatter-add of every element's contribution; with
 * accumulate == 0 f is zeroed first (stream-ordered memset), else added to.
 */
typedef struct to_sem3d_desc {
  int32_t dtype;            /* TO_F32 or TO_F64                              */
  int32_t ngll;             /* N: 5 or 8 (f32 and f64 each)                  */
  int64_t nelem;            /* E                                              */
  int64_t nglob;            /* assembled: number of global nodes; else 0     */
  int32_t assembled;        /* 1 = through ibool, 0 = element-local          */
  int32_t node_layout;      /* assembled u, f: 0 = one [nglob] array per
                               component; 1 = interleaved [nglob][4] floats
                               (x, y, z, unused) in u[0] / f[0], 16-byte
                               aligned (f32, NGLL 5 only): one 128-bit gather
                               and one 128-bit scatter-add per point         */
  const double* hprime;     /* HOST [N][N]  H(i,p)   (reference d.H)          */
  const double* hprimewgll; /* HOST [N][N]  Hw(q,i)  (reference d.Hw)         */
  const double* wgll;       /* HOST [N]     w        (reference d.w)           */
} to_sem3d_desc;

typedef struct to_sem3d_fields {
  const void* u[3];         /* displacement components                       */
  void* f[3];               /* force components (output)                     */
  const int32_t* ibool;     /* [E][N][N][N] global node ids (assembled mode) */
  /* inverse Jacobian J[r][d] = d(xi_r)/d(x_d), then jac, l2m, mu            */
  const void* xix;  const void* xiy;  const void* xiz;
  const void* etax; const void* etay; const void* etaz;
  const void* gamx; const void* gamy; const void* gamz;
  const void* jac;  const void* l2m;  const void* mu;
  /* Assembled mode, optional (NULL: none): DEVICE double; every gathered u
   * value is read as u * (1 / sqrt(*u_norm2)), the product taken in double
   * and rounded once -- what to_scale3 writes, so a power iteration can keep
   * the unnormalised K u and fold the normalisation into the next
   * application (one pass over u and f less per step).  Appended last: a
   * zero-initialised struct has none. */
  const double* u_norm2;
} to_sem3d_fields;

typedef struct to_sem3d_plan to_sem3d_plan;

/* Validate a description and capture the operators.  Host only. */
int to_sem3d_plan_create(const to_sem3d_desc* desc, to_sem3d_plan** plan);
int to_sem3d_plan_destroy(to_sem3d_plan* plan);

/* Launch one application on `stream` (asynchronous).  Device pointers in
 * `fields` must be 4-byte (f32) or 8-byte (f64) aligned; all per-point arrays
 * hold E*N^3 values. */
int to_sem3d_apply(const to_sem3d_plan* plan, const to_sem3d_fields* fields,
                   int32_t accumulate, void* stream);

/* The contribution of elements [first, first + count) of the plan only,
 * ADDED to f (never zeroed): `fields` describes the whole batch exactly as for
 * to_sem3d_apply.  Lets a caller order element ranges -- a z-slab rank
 * computes the element layers next to its neighbours first, starts the
 * interface exchange, then computes the interior.  The reference launches
 * its whole league at once (include/TensorOperations/LevelGraph.hpp:576-628);
 * this is the same operator on a sub-range. */
int to_sem3d_apply_elements(const to_sem3d_plan* plan, const to_sem3d_fields* fields,
                            int64_t first, int64_t count, void* stream);

/* Algorithmic HBM bytes of one application of `plan` (the roofline numerator:
 * every per-point array read once, ibool read once, u read and f written once
 * per global node in assembled mode, per point in element-local mode). */
double to_sem3d_algorithmic_bytes(const to_sem3d_plan* plan);

/* Useful floating-point operations of one application (36N+159 per point). */
double to_sem3d_flops(const to_sem3d_plan* plan);

/* ---------------------------------------------------------------------- */
/* Z-slab interface planes (multi-GPU assembled mode)                      */
/* ---------------------------------------------------------------------- */
/*
 * A rank of a z-slab partition owns a contiguous range of element layers
 * and every node plane they touch; its first and last planes are shared with
 * the neighbouring ranks and hold partial sums after the rank's own scatter.
 * With the structured numbering a node plane is one contiguous range
 * [offset, offset + n) of each component (n = nx*ny).
 *   pack:        buf[c*n + i]      = f[c][offset + i]      (c = 0..2)
 *   accumulate:  f[c][offset + i] += buf[c*n + i]
 * `f` is a HOST array of 3 device pointers; `buf` is device memory of 3*n
 * values.  Both launch one kernel on `stream`.  The reference is single-GPU;
 * these are the two local steps around the neighbour exchange (NCCL
 * send/recv of `buf`).
 */
int to_sem3d_halo_pack(int32_t dtype, void* const f[3], int64_t offset, int64_t n,
                       void* buf, void* stream);
int to_sem3d_halo_accumulate(int32_t dtype, void* const f[3], int64_t offset, int64_t n,
                             const void* buf, void* stream);

/* Node layouts (f32): out[i] = (x[0][i], x[1][i], x[2][i], 0) for i < n, the
 * interleaved [nglob][4] layout of node_layout 1, from one array per component,
 * and back (x[c][i] = in[i].c).  `x` is a HOST array of 3 device pointers;
 * the interleaved array is 16-byte aligned.  One kernel on `stream`.  No
 * counterpart in the reference (it has no assembled fields). */
int to_nodes_interleave(const float* const x[3], float* out, int64_t n, void* stream);
int to_nodes_deinterleave(const float* in, float* const x[3], int64_t n, void* stream);


/* ---------------------------------------------------------------------- */
/* Z-slab operator over NCCL (one rank per GPU)                            */
/* ---------------------------------------------------------------------- */
/*
 * NCCL's communicator handle: the same typedef as nccl.h's, so a caller that
 * includes nccl.h passes its own ncclComm_t unchanged.
 */
typedef struct ncclComm* ncclComm_t;

#define TO_NCCL_UNIQUE_ID_BYTES 128

/*
 * One rank's z-slab of a structured mesh split in element layers across the
 * ranks of `comm`.  The rank's plan covers its elements (whole layers of
 * layer_elems elements, ordered layer by layer) and the nodes they touch;
 * its first node plane is shared with rank `prev` and its last with rank
 * `next` (-1: no neighbour on that side).  With the structured numbering each
 * plane is one contiguous range of plane_nodes nodes per component: nodes
 * [0, plane_nodes) and [nglob - plane_nodes, nglob).
 */
typedef struct to_slab {
  int32_t prev;          /* rank below in `comm`, or -1                      */
  int32_t next;          /* rank above in `comm`, or -1                      */
  int64_t layer_elems;   /* elements per element layer (nex * ney)           */
  int64_t plane_nodes;   /* nodes per node plane                             */
  void* recv[2];         /* device buffers of 3 * plane_nodes values (4 *
                            plane_nodes with interleaved nodes): the partial
                            sums received from prev ([0]) / next ([1])       */
  void* sync;            /* device buffer of to_slab_sync_bytes() bytes,
                            16-byte aligned (batch tickets of the launches)  */
  int32_t f_is_zero;     /* 0: the call zeroes f first (on compute_stream);
                            1: the caller has already zeroed f in stream order
                            (lets a caller time the operator without the fill) */
} to_slab;

/*
 * f = K u on this rank's slab, with the shared planes summed across the
 * neighbours, so every copy of a shared node holds the full sum and f equals
 * the slice of the single-mesh result for this rank's nodes.  Either node
 * layout of the plan: one array per component, or interleaved (u[0], f[0]
 * [nglob][4]; each shared plane then travels as one contiguous range).
 * The reference evaluates the whole mesh in one Kokkos launch on one device
 * (include/TensorOperations/LevelGraph.hpp:576-628, bench_sem3d_levelgraph.cpp
 * :247-351); this is the same operator partitioned over ranks.
 *   compute_stream: zero f (unless slab->f_is_zero); the element layers next
 *     to a neighbour (one launch); the interior layers (one launch, batches
 *     handed out by a ticket counter); then it waits for the exchange.
 *   comm_stream: after the boundary layers, one NCCL group sends this rank's
 *     shared planes (read in place from f) and receives the neighbours' into
 *     `recv`, then adds them into f's shared planes -- overlapped with the
 *     interior, which touches no shared plane.  Give comm_stream a higher
 *     priority than compute_stream (cudaStreamCreateWithPriority) so its
 *     kernels are dispatched ahead of the interior's batches.
 * Every rank must make the same sequence of calls.  Asynchronous; returns
 * TO_ERR_COMM if NCCL cannot be loaded or a call fails.  Nothing is allocated.
 */
size_t to_slab_sync_bytes(void);
int to_sem3d_elastic_mgpu(const to_sem3d_plan* plan, const to_sem3d_fields* fields,
                          const to_slab* slab, ncclComm_t comm, void* compute_stream,
                          void* comm_stream);

/*
 * The same call with u and f in HOST memory, one array per component (pinned
 * memory for asynchronous copies): on compute_stream it copies u in (and,
 * with interleaved nodes, converts it into fields->u[0] through host->stage),
 * applies the operator as to_sem3d_elastic_mgpu, and copies f out (converting
 * from fields->f[0] through host->stage).  fields->u / f are the device
 * buffers the operator uses; `stage` holds three device arrays of nglob values
 * (interleaved plans only; NULL otherwise).  Two calls on two streams with
 * two sets of device buffers overlap one call's copy-out with the next one's
 * copy-in.  The end-to-end path a caller with host data takes.
 */
typedef struct to_host_nodes {
  const void* u[3];      /* HOST: nglob values per component, read            */
  void* f[3];            /* HOST: nglob values per component, written         */
  void* stage[3];        /* DEVICE: nglob values each (interleaved plans)     */
} to_host_nodes;
int to_sem3d_elastic_mgpu_host(const to_sem3d_plan* plan, const to_sem3d_fields* fields,
                               const to_slab* slab, ncclComm_t comm, const to_host_nodes* host,
                               void* compute_stream, void* comm_stream);

/* NCCL set-up for callers without their own: rank 0 makes an id (bytes
 * TO_NCCL_UNIQUE_ID_BYTES), every rank receives it by its own means and
 * creates its communicator (the current device is the rank's GPU).  These and
 * to_nccl_allreduce_sum_f64 (in-place sum of n doubles across the ranks, on
 * `stream`) call the process's libnccl.so.2. */
int to_nccl_unique_id(void* id);
int to_nccl_comm_init(int32_t nranks, int32_t rank, const void* id, ncclComm_t* comm);
int to_nccl_comm_destroy(ncclComm_t comm);
int to_nccl_allreduce_sum_f64(double* x, int64_t n, ncclComm_t comm, void* stream);

/* ---------------------------------------------------------------------- */
/* Field reductions (repeated applications u <- K u / ||K u||)             */
/* ---------------------------------------------------------------------- */
/*
 * Sum of squares of three device arrays over [first, first + n):
 *   *result = sum_c sum_i x[c][first + i]^2        (accumulated in double)
 * `x` is a HOST array of 3 device pointers, `result` one device double.  Two
 * kernels on `stream`; the grouping of the sum is fixed by n alone (blocks of
 * 131072 values, then a fixed-order pass over the block partials), so the
 * result is bitwise the same on every device.  `workspace` is device memory
 * of at least to_sumsq3_workspace_bytes(n) bytes holding the block partials;
 * nothing in it needs to be initialised.  For a z-slab rank, [first, first+n)
 * is the nodes it owns: a shared interface plane is counted by the lower rank
 * only.  The reference's benchmark has no norm; this is the configuration's
 * steady-state loop.
 */
size_t to_sumsq3_workspace_bytes(int64_t n);
int to_sumsq3(int32_t dtype, const void* const x[3], int64_t first, int64_t n, double* result,
              void* workspace, size_t workspace_bytes, void* stream);

/* to_sumsq3 without a workspace argument, for callers that may not allocate
 * device memory: for example a solver step running inside an application
 * that owns the GPU's memory through its own pool (a cudaMalloc of ours
 * would fail or bypass its accounting), or a loop that must not stall the
 * device the way cudaFree does.  No counterpart in the reference.
 *   - The block partials live in one fixed array inside the library (256 KiB
 *     per GPU, kept until the process exits); nothing is allocated per call.
 *   - The first call on a device looks up that array's device address (with
 *     the device current); make that first call before any stream capture.
 *     The address is remembered per device and CUDA context: a call in
 *     another context (the caller's own, or a new primary context after
 *     cudaDeviceReset) looks it up again, so it too should come before any
 *     capture in that context.
 *   - n per component is limited to to_sumsq3_noalloc_max_n()
 *     (1,431,655,765); a larger n is rejected with TO_ERR_INVALID_ARGUMENT
 *     before anything is launched.
 *   - Every call shares the array and it keeps the last call's partials.
 *     Nothing in it needs to start at zero (a call writes every partial it
 *     later reads), but calls whose kernels overlap on the GPU -- on
 *     different streams, or from different host threads -- race on it and
 *     give wrong sums.  Order such calls on one stream.
 * Same result, bit for bit, as to_sumsq3 on the same inputs. */
int to_sumsq3_noalloc(int32_t dtype, const void* const x[3], int64_t first, int64_t n,
                      double* result, void* stream);
int64_t to_sumsq3_noalloc_max_n(void);

/* y[c][i] = x[c][i] / sqrt(*sumsq) for i < n (sumsq read on the device, so no
 * host synchronisation); y may equal x. */
int to_scale3(int32_t dtype, void* const y[3], const void* const x[3], int64_t n,
              const double* sumsq, void* stream);

/* ---------------------------------------------------------------------- */
/* SEM 2D elastic P-SV stiffness operator (element-local)                  */
/* ---------------------------------------------------------------------- */
/*
 * The operator of the reference's 2D benchmark
 * (benchmarks/sem_stiffness/bench_sem_stiffness.cpp: physics :319-357, host
 * loop :1335-1385), f32, NGLL 8, two components, element-local:
 *   a_c = sum_p H(i,p) u_c(j,p),  g_c = sum_p H(j,p) u_c(p,i)
 *   ds = grad u through (xix, xiz, gamx, gamz); sigma = isotropic P-SV stress
 *   Fx_c = jac (s_c0 xix + s_c1 xiz),  Fg_c = jac (s_c0 gamx + s_c1 gamz)
 *   f_c(j,i) = w_j sum_q Hw(q,i) Fx_c(j,q) + w_i sum_q Hw(q,j) Fg_c(q,i)
 * Per-point arrays [E][j][i] (i fastest), 16-byte aligned device pointers.
 * H, Hw, w: HOST doubles ([8][8], [8][8], [8]).  f is overwritten.
 */
typedef struct to_sem2d_fields {
  const void* u[2];
  void* f[2];
  const void* xix; const void* xiz; const void* gamx; const void* gamz;
  const void* jac; const void* l2m; const void* mu;
} to_sem2d_fields;

int to_sem2d_elastic_local(int32_t ngll, int64_t nelem, const double* hprime,
                           const double* hprimewgll, const double* wgll,
                           const to_sem2d_fields* fields, void* stream);

/* ---------------------------------------------------------------------- */
/* SEM 2D acoustic stiffness operator (assembled)                          */
/* ---------------------------------------------------------------------- */
/*
 * The scalar (acoustic) 2D operator of the first benchmark configuration;
 * the reference has no acoustic kernel, so this is the configuration's own
 * definition:
 *   dxi = sum_p H(i,p) u(j,p),  dgm = sum_p H(j,p) u(p,i)   (u gathered by ibool)
 *   du/dx = dxi xix + dgm gamx,  du/dz = dxi xiz + dgm gamz
 *   Fx = jac/rho (du/dx xix + du/dz xiz),  Fg = jac/rho (du/dx gamx + du/dz gamz)
 *   f(ibool(j,i)) += w_j sum_q Hw(q,i) Fx(j,q) + w_i sum_q Hw(q,j) Fg(q,i)
 * Per-point arrays [E][j][i]; u, f [nglob]; with accumulate == 0 f is zeroed
 * first.  NGLL 5, f64 or f32.  (kappa belongs to the mass matrix, not here.)
 */
typedef struct to_sem2d_acoustic_desc {
  int32_t dtype; int32_t ngll; int64_t nelem; int64_t nglob;
  const double* hprime; const double* hprimewgll; const double* wgll;  /* HOST */
} to_sem2d_acoustic_desc;
typedef struct to_sem2d_acoustic_fields {
  const void* u; void* f; const int32_t* ibool;
  const void* xix; const void* xiz; const void* gamx; const void* gamz;
  const void* jac; const void* rho;
} to_sem2d_acoustic_fields;
int to_sem2d_acoustic_apply(const to_sem2d_acoustic_desc* desc,
                            const to_sem2d_acoustic_fields* fields, int32_t accumulate,
                            void* stream);

/* ---------------------------------------------------------------------- */
/* Batched small GEMM with a shared left operand                           */
/* ---------------------------------------------------------------------- */
/*
 *   C[b][i][j] = sum_k A[i][k] * B[b][k][j],  b < batch, i < M, k < K, j < N
 * A: HOST double [M][K] (shared by every batch entry, converted to dtype);
 * B: device [batch][K][N], C: device [batch][M][N], row-major, dtype TO_F32
 * or TO_F64.  Built for (M, K) = (5, 5) and (8, 8), any N.  The batched form
 * of one gradient contraction of the SEM operator (the reference's analogue:
 * benchmarks/sem_stiffness/bench_sem_stiffness.cpp:884-896).  One kernel on
 * `stream`.
 */
int to_batched_small_gemm(int32_t dtype, int32_t M, int32_t K, int32_t N, int64_t batch,
                          const double* A, const void* B, void* C, void* stream);

/* ---------------------------------------------------------------------- */
/* Permuted multilevel contraction chain on the tensor cores               */
/* ---------------------------------------------------------------------- */
/*
 *   T[a,b,c,d] = sum_{e,f} A[a,e,c,f] * B[f,b,e,d]
 *   R[a,d]     = sum_{b,c} T[a,b,c,d] * C[c,b]
 * All six extents equal E (32, 64 or 128); row-major fp32 tensors in device
 * memory (A, B and the workspace 16-byte aligned).  The chain the reference
 * builds from ContractionNodes over permuted operands
 * (benchmarks/permuted_contraction/bench_permuted_contraction.cpp,
 * benchmarks/multilevel_contraction/bench_multilevel_contraction.cpp).  Step 1
 * runs on tcgen05 (TF32 x3 split, fp32 accumulation in TMEM) with TMA reading
 * the permuted operands in place; step 2 is fused into its epilogue, so T
 * never reaches memory unless `T` is non-NULL (then it is also stored, for
 * checking).  R is overwritten.  `workspace` holds the split operands:
 * to_chain_workspace_bytes(E) bytes.  Asynchronous on `stream`.
 */
size_t to_chain_workspace_bytes(int32_t E);
int to_chain_f32(int32_t E, const float* A, const float* B, const float* C, float* R, float* T,
                 void* workspace, size_t workspace_bytes, void* stream);
/* Useful flops of one chain: 2 E^6 + 2 E^4. */
double to_chain_flops(int32_t E);

/* One contraction as a dense GEMM on the tensor cores:
 *   C[m][n] = sum_k A[m][k] * B[n][k]
 * with both operands K-major and given split into TF32 parts, A = Ahi + Alo
 * and B = Bhi + Blo elementwise (hi = the value rounded to TF32, lo = the
 * exact remainder); the product is formed from three TF32 products (the lo*lo
 * term, about 2^-22 relative, is dropped) accumulated in fp32.  This is the
 * path the frontend lowers a large contraction of two inputs to (the
 * reference's team contraction evaluator, include/TensorOperations/Evaluator/
 * Team.hpp:318-927, with its permuted operands, Permute.hpp:127-228, packed
 * by the frontend).  Mp, Np, Kp must be positive multiples of 128, 256 and
 * 32 (pad with zeros); A* are [Mp][Kp], B* [Np][Kp], C [Mp][Np], row-major
 * fp32 in device memory, 16-byte aligned.  C is overwritten (when the tiles
 * leave the last wave of SMs less than half full, those tiles are split in K
 * between two CTAs that add into rows of C zeroed first on `stream`).
 * Asynchronous on `stream`; allocates nothing. */
int to_gemm_tf32x3(int64_t Mp, int64_t Np, int64_t Kp, const float* Ahi, const float* Alo,
                   const float* Bhi, const float* Blo, float* C, void* stream);

/* ---------------------------------------------------------------------- */
/* Level-graph lowering                                                    */
/* ---------------------------------------------------------------------- */
/*
 * The header-only C++ frontend (make_level_graph / add / outputs / execute)
 * plans a level graph at compile time -- slots, level-timeline liveness,
 * pooled scratch, tiles -- and lowers the plan to this descriptor before every
 * launch (the reference launches from LevelGraph::launch / lg_execute,
 * include/TensorOperations/LevelGraph.hpp:576-628,718-733).  The library
 * re-checks the plan independently and returns the launch shape:
 *   - every pair of slots sharing a pool has disjoint live ranges and every
 *     pool is large enough for its slots (else TO_ERR_INVALID_ARGUMENT);
 *   - a label declared whole on a staged input is not longer than its tile
 *     (TO_ERR_GRID; the reference aborts, LevelGraph.hpp:519-522);
 *   - league = product over blocked labels of ceil(extent / tile);
 *   - team: the requested size (1..1024) or, when <= 0, the smallest multiple
 *     of 32 covering the widest level, clamped to [64, 512];
 *   - with query_device != 0, the scratch must fit the current device's
 *     opt-in shared memory per block (TO_ERR_SCRATCH).
 * Host only apart from the optional device-attribute query.
 */
typedef struct to_level_plan_desc {
  int32_t value_bytes;          /* sizeof(value type)                          */
  int32_t num_levels;
  int32_t num_slots;
  int32_t num_pools;
  const int32_t* level_kind;    /* [num_levels] 0 stage, 1 contraction, 2 combine,
                                   3 contraction staging its own operand tiles */
  const int32_t* level_members; /* [num_levels]                                */
  const int64_t* level_space;   /* [num_levels] items of the level's one loop  */
  const int32_t* slot_def;      /* [num_slots] level that writes the slot      */
  const int32_t* slot_last;     /* [num_slots] last level reading it (roots: num_levels) */
  const int32_t* slot_pool;     /* [num_slots]                                 */
  const int64_t* slot_bytes;    /* [num_slots]                                 */
  const int64_t* pool_offset;   /* [num_pools + 1] byte offsets, then the total */
  int32_t grid_rank;            /* number of blocked labels carried by stages  */
  int32_t num_whole;            /* whole-label checks                          */
  const int64_t* grid_extent;   /* [grid_rank] global extent per blocked label */
  const int32_t* grid_tile;     /* [grid_rank]                                 */
  const int64_t* whole_extent;  /* [num_whole] staged extent along a whole label */
  const int32_t* whole_tile;    /* [num_whole]                                 */
  int32_t team_size;            /* <= 0: automatic                             */
  int32_t reserved0;
} to_level_plan_desc;

typedef struct to_level_launch {
  int64_t league;         /* CTAs (one per grid tile)                          */
  int64_t scratch_bytes;  /* dynamic shared memory per CTA                     */
  int32_t team;           /* threads per CTA                                   */
  int32_t reserved0;
} to_level_launch;

int to_level_plan_lower(const to_level_plan_desc* desc, int32_t query_device,
                        to_level_launch* out);

/* ---------------------------------------------------------------------- */
/* Sequence operators: rows of heads                                       */
/* ---------------------------------------------------------------------- */
/*
 * Values of [tokens][heads][width], the width contiguous; strides count
 * elements, so a head's rows may lie inside wider packed rows.  dtype is the
 * descriptor's (TO_BF16 or TO_F32).  64-bit offsets throughout.
 */
typedef struct to_rows {
  void* data;
  int64_t token_stride;
  int64_t head_stride;
} to_rows;

/* ---------------------------------------------------------------------- */
/* Query / key norm of each head with the rotation by position             */
/* ---------------------------------------------------------------------- */
/*
 * For every head x of q and of k (head_dim values):
 *   y = w * x / sqrt(mean(x^2) + eps),
 * then the first rotary_dim values of y turn in pairs: pair j by the angle
 *   positions[axis(j)][t] * theta^(-2 j / rotary_dim),
 * (a, b) -> (a cos - b sin, b cos + a sin).  Pair j is (j, j + rotary_dim/2),
 * or (2j, 2j+1) with interleaved = 1.  Axis a owns section[a] consecutive
 * pairs (sections sum to rotary_dim / 2): one axis for text, three for
 * (time, height, width).  Angles are reduced exactly (64-bit fixed-point
 * turns), so any int32 position, negative ones included, keeps f32 accuracy.
 * wq, wk: [head_dim] f32, NULL for 1.  Sums are f32; one rounding at the end.
 * head_dim even, at most 256.  k_heads may be 0 (no keys).
 * Outputs may be their own inputs (q_out q, k_out k: same pointer and strides);
 * they may share no memory with them, or with one another, otherwise.  What
 * shares memory against these rules is refused with TO_ERR_INVALID_ARGUMENT
 * where the library can tell: arrays, rows that begin at the same place, and
 * rows with one token stride that holds a token's heads.
 */
typedef struct to_qk_desc {
  int32_t dtype;
  int32_t q_heads;
  int32_t k_heads;
  int32_t head_dim;
  int32_t rotary_dim;  /* even, 0 (no rotation) .. head_dim                  */
  int32_t axes;        /* 1 .. 4                                             */
  int32_t section[4];  /* pairs of each axis                                 */
  int32_t interleaved; /* 0: halves, 1: neighbours                           */
  int32_t reserved0;
  double theta;        /* > 0                                                */
  double eps;          /* >= 0                                               */
} to_qk_desc;

typedef struct to_qk_plan to_qk_plan;

int to_qk_plan_create(const to_qk_desc* desc, to_qk_plan** out);
int to_qk_plan_destroy(to_qk_plan* plan);

/* positions: device int32 [axes][tokens] (may be NULL when rotary_dim is 0). */
int to_qk_norm_rotary(const to_qk_plan* plan, int64_t tokens, const to_rows* q, const to_rows* k,
                      const int32_t* positions, const float* wq, const float* wk,
                      const to_rows* q_out, const to_rows* k_out, void* stream);

/*
 * Gradients: gq, gk of the outputs -> dq, dk of the inputs q, k (which are the
 * forward pass's inputs) and dwq, dwk ([head_dim] f32, overwritten; both are
 * computed even where wq / wk is NULL, and either may be NULL to leave it
 * out).  Sums run in a fixed order.  workspace: 16-byte aligned device memory
 * of at least to_qk_norm_rotary_workspace_bytes.  dq may be gq or q, dk may be
 * gk or k, as above.
 */
size_t to_qk_norm_rotary_workspace_bytes(const to_qk_plan* plan, int64_t tokens);
int to_qk_norm_rotary_backward(const to_qk_plan* plan, int64_t tokens, const to_rows* q,
                               const to_rows* k, const int32_t* positions, const float* wq,
                               const float* wk, const to_rows* gq, const to_rows* gk,
                               const to_rows* dq, const to_rows* dk, float* dwq, float* dwk,
                               void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------- */
/* Linear attention with a decay for each head                             */
/* ---------------------------------------------------------------------- */
/*
 * Query head h reads key / value head h / (q_heads / kv_heads).  Within a
 * sequence of L tokens, t = 0 .. L-1, with l = exp(log_decay[h]):
 *   S_t = l S_{t-1} + k_t v_t^T          (f32 state [key_dim][value_dim])
 *   o_t = scale * S_t^T q_t
 * S_{-1} is the entering state (state_in, zero when NULL); S_{L-1} is written
 * to state_out (when not NULL).  log_decay: device f32 [q_heads], values <= 0
 * (a positive one counts as 0); -inf forgets everything at once.
 *
 * Sequences are packed: sequence n holds the tokens cu_seqlens[n] ..
 * cu_seqlens[n+1]-1 (device int32 [nseq + 1], non-decreasing, within
 * [0, tokens]; values outside are clamped).  Lengths 0 and 1 are ordinary: an
 * empty sequence hands its entering state on.  Rows of o that belong to no
 * sequence are left as they are.
 *
 * States are [slots][q_heads][key_dim][value_dim] f32, contiguous, 16-byte
 * aligned.  slots (device int32 [nseq]) names each sequence's slot in
 * state_in and state_out; NULL: slot n is sequence n.  A slot outside
 * [0, num_slots) stands for no state: the sequence starts from zero and writes
 * none.  Two sequences may not share a slot.  state_out may be state_in, and
 * may overlap it in no other way.  o may share no memory with q, k or v (in the
 * single-token call too): they are read while it is written.
 *
 * key_dim and value_dim 1 .. 256.  Products of bf16 rows run on the tensor
 * cores with f32 sums; states and their updates keep f32 accuracy.  Results take
 * one rounding to bf16 for the first 128 tokens of a sequence that nothing
 * enters (for dk and dv the last 128), the others one more of the products'
 * operands.  A value that is not finite makes what depends on it not finite
 * (NaN, it may be, where the recurrence has an infinity), and nothing else.
 *
 * Results do not depend on timing (every sum has a fixed order).  Calls on
 * different streams need workspaces of their own.
 */
typedef struct to_linear_attention_desc {
  int32_t dtype;
  int32_t q_heads;
  int32_t kv_heads;  /* divides q_heads                                      */
  int32_t key_dim;
  int32_t value_dim;
  int32_t nseq;      /* >= 0                                                 */
  int64_t tokens;    /* rows of q, k, v, o; < 2^31                           */
  int64_t num_slots; /* slots of state_in / state_out (with slots NULL: nseq) */
  double scale;      /* finite                                               */
} to_linear_attention_desc;

typedef struct to_linear_attention_args {
  to_rows q, k, v, o;
  const float* log_decay;
  const int32_t* cu_seqlens;
  const int32_t* slots;
  const float* state_in;
  float* state_out;
  void* workspace; /* device, 256-byte aligned                               */
  size_t workspace_bytes;
} to_linear_attention_args;

size_t to_linear_attention_workspace_bytes(const to_linear_attention_desc* desc);
int to_linear_attention(const to_linear_attention_desc* desc, const to_linear_attention_args* args,
                        void* stream);

/*
 * Gradients of the call above with respect to q, k, v and the entering state,
 * from d_o and dstate_out (the gradient of the state left; NULL: zero).
 * log_decay is a constant of the model.  States and their gradients are
 * [nseq][q_heads][key_dim][value_dim] (no slots).  Gradients of heads that
 * share a key / value head are summed in f32 before their one rounding.  Rows
 * of dq, dk, dv that belong to no sequence are left as they are.  dq, dk, dv and
 * dstate_in may share no memory with the inputs or with one another.
 */
typedef struct to_linear_attention_grad_args {
  to_rows q, k, v, d_o, dq, dk, dv;
  const float* log_decay;
  const int32_t* cu_seqlens;
  const float* state_in;
  const float* dstate_out;
  float* dstate_in; /* NULL: not wanted                                      */
  void* workspace;  /* device, 256-byte aligned                              */
  size_t workspace_bytes;
} to_linear_attention_grad_args;

size_t to_linear_attention_backward_workspace_bytes(const to_linear_attention_desc* desc);
int to_linear_attention_backward(const to_linear_attention_desc* desc,
                                 const to_linear_attention_grad_args* args, void* stream);

/*
 * One token of each of desc->tokens requests: the state in the request's slot
 * becomes l S + k v^T in place and o = scale * S^T q.  A request whose slot
 * lies outside [0, num_slots) touches no state and gets a row of zeros.
 * nseq, cu_seqlens, state_in and the workspace are not used; state_out is the
 * state.
 */
int to_linear_attention_step(const to_linear_attention_desc* desc,
                             const to_linear_attention_args* args, void* stream);

/* ---------------------------------------------------------------------- */
/* Rows kept in 8 bits                                                     */
/* ---------------------------------------------------------------------- */
/*
 * [tokens][width] values as int8 codes and one scale byte for every 32
 * neighbouring values (the last group of a row may be shorter):
 *   value = code * 2^(scale - 127),
 * the scale the least power of two with |x| <= 127 * 2^(scale - 127) in the
 * group (not below 2^-127), code = x / 2^(scale - 127) rounded to the nearest
 * integer, ties to even.  Both steps are exact but for that one rounding (of
 * at most half a scale, 1/127 of the group's largest |x|): codes do not depend on
 * how they were computed.  A group that holds an infinity or a NaN has the scale byte 255 and
 * reads as NaN.  Strides count elements (bytes) from token to token.
 */
typedef struct to_rows8 {
  void* codes;  /* int8  [tokens][width]                                     */
  void* scales; /* uint8 [tokens][(width + 31) / 32]                         */
  int64_t code_stride;
  int64_t scale_stride;
} to_rows8;

/* x (rows of one head, head_stride not used) into 8 bits, and back: x = the value. */
int to_rows8_pack(int32_t dtype, int32_t width, int64_t tokens, const to_rows* x,
                  const to_rows8* out, void* stream);
int to_rows8_unpack(int32_t dtype, int32_t width, int64_t tokens, const to_rows8* in,
                    const to_rows* x, void* stream);

/* ---------------------------------------------------------------------- */
/* Gated linear recurrence                                                 */
/* ---------------------------------------------------------------------- */
/*
 * For every channel c of a sequence, t = 0 .. L-1:
 *   a_t = sigmoid(f_t + bias_c)
 *   h_t = a_t h_{t-1} + (1 - a_t) x_t     (complement = 1)
 *   h_t = a_t h_{t-1} + x_t               (complement = 0)
 * x, f, h: rows [tokens][channels] (one head: head_stride is not used).  bias:
 * device f32 [channels], NULL for 0.  h_{-1} is the entering state (state_in,
 * zero when NULL); h_{L-1}, before its rounding, is written to state_out (when
 * not NULL).  a and 1 - a keep f32 accuracy relative to themselves, whatever the
 * gates of other tokens and channels are; the recurrence is f32 throughout (with
 * complement, h - x has to be finite there), h takes one rounding.
 *
 * Sequences are packed as in to_linear_attention, and so are the rules for
 * cu_seqlens, lengths 0 and 1, rows of no sequence, slots (states are f32
 * [slots][channels], 16-byte aligned) and values that are not finite.
 *
 * For the gradients the call writes, when `saved` is not NULL, the state that
 * enters each TO_RECURRENCE_SEGMENT tokens of every sequence (f32
 * [to_gated_recurrence_saved_rows][channels], 16-byte aligned), and, where
 * keep_x / keep_f have codes, x and f in 8 bits.
 *
 * h may share no memory with x or f, nor any output with another one or with
 * what the call reads, but state_out, which may be state_in.
 * Results do not depend on timing (every sum has a fixed order).  channels 1 ..
 * 65536.  Calls that overlap need workspaces of their own.
 */
#define TO_RECURRENCE_SEGMENT 128

typedef struct to_gated_recurrence_desc {
  int32_t dtype;
  int32_t channels;
  int32_t nseq;       /* >= 0                                                */
  int32_t complement; /* 0 or 1                                              */
  int64_t tokens;     /* rows of x, f, h; < 2^31                             */
  int64_t num_slots;  /* slots of state_in / state_out (slots NULL: nseq)    */
} to_gated_recurrence_desc;

typedef struct to_gated_recurrence_args {
  to_rows x, f, h;
  to_rows8 keep_x, keep_f; /* codes NULL: not kept                           */
  const float* bias;
  const int32_t* cu_seqlens;
  const int32_t* slots;
  const float* state_in;
  float* state_out;
  float* saved;
  void* workspace; /* device, 256-byte aligned                               */
  size_t workspace_bytes;
} to_gated_recurrence_args;

/* Rows of `saved`, and bytes of the workspace (0: none), of a call of this size. */
int64_t to_gated_recurrence_saved_rows(const to_gated_recurrence_desc* desc);
size_t to_gated_recurrence_workspace_bytes(const to_gated_recurrence_desc* desc);
int to_gated_recurrence(const to_gated_recurrence_desc* desc, const to_gated_recurrence_args* args,
                        void* stream);

/*
 * How long, in microseconds, the waits within a launch of later calls last at most: a
 * segment's for the maps of others (2 s), a block's warps' for one another and for rows
 * on their way (8 s).  Negative: as at the start; 0: maps that are not there at once, or any
 * wait of a block's warps, counts as run out.  At most an hour.  Where a wait runs out, to_device_status reports
 * TO_ERR_TIMEOUT, and outputs and states that depend on what did not come are NaN or
 * have not been written.  dbias is NaN then (of sequences of one segment each, which wait
 * for no maps, also as long as an earlier TO_ERR_TIMEOUT has not been read).  Holds for
 * the process; a captured call keeps the limits of its capture.
 */
int to_gated_recurrence_wait_limits(int64_t maps_us, int64_t tiles_us);

/*
 * Gradients of the call above with respect to x, f, bias and the entering
 * state, from dh and dstate_out (the gradient of the state left, NULL: zero).
 * x and f are the forward pass's, as they were or (x8, f8 with codes) as it
 * kept them; `saved` is what it saved.  With G_t = dh_t + a_{t+1} G_{t+1}
 * (behind the last token dstate_out):
 *   dx_t = (1 - a_t) G_t,  df_t = G_t a_t (1 - a_t) (h_{t-1} - x_t)   (complement)
 *   dx_t = G_t,            df_t = G_t a_t (1 - a_t) h_{t-1}
 *   dbias = sum df_t,      dstate_in = a_0 G_0  (dstate_out for an empty sequence)
 * h_{t-1} runs from the saved states over the x and f given.  State gradients
 * are [nseq][channels] (no slots).  dbias (f32 [channels]) and dstate_in are
 * overwritten, and may be NULL.  Rows of dx, df that belong to no sequence are
 * left as they are.  Outputs may share no memory with what is read or with one
 * another.
 */
typedef struct to_gated_recurrence_grad_args {
  to_rows x, f, dh, dx, df;
  to_rows8 x8, f8; /* codes not NULL: in the place of x, f                   */
  const float* bias;
  const int32_t* cu_seqlens;
  const float* saved;
  const float* dstate_out;
  float* dstate_in;
  float* dbias;
  void* workspace; /* device, 256-byte aligned                               */
  size_t workspace_bytes;
} to_gated_recurrence_grad_args;

size_t to_gated_recurrence_backward_workspace_bytes(const to_gated_recurrence_desc* desc);
int to_gated_recurrence_backward(const to_gated_recurrence_desc* desc,
                                 const to_gated_recurrence_grad_args* args, void* stream);

/*
 * One token of each of desc->tokens requests: the state in the request's slot
 * (state_out) becomes h in place.  A request whose slot lies outside
 * [0, num_slots) touches no state and gets a row of zeros.  nseq, cu_seqlens,
 * state_in, saved, keep_x, keep_f and the workspace are not used.
 */
int to_gated_recurrence_step(const to_gated_recurrence_desc* desc,
                             const to_gated_recurrence_args* args, void* stream);

/* ---------------------------------------------------------------------- */
/* Norms around a block, with its gate and residual scale                  */
/* ---------------------------------------------------------------------- */
/*
 * Between two blocks: the block's output y joins the residual stream r, and the
 * next block's input n is made of the sum, for every row:
 *   u = w_post * y / sqrt(mean(y^2) + eps)        (post_norm = 0: u = w_post * y)
 *   r_out = r + scale * u * act(g)                (gate NONE: r + scale * u)
 *   n = w_pre * r_out / sqrt(mean(r_out^2) + eps)
 * y, g, n: rows of dtype; r, r_out: rows of residual (TO_F32, or dtype), all
 * [tokens][width] (one head: head_stride is not used).  act(g): g, sigmoid(g) or
 * g * sigmoid(g).  w_post, w_pre: device f32 [width], NULL for 1.  y NULL (a model's
 * first norm): n is made of r, and there is no r_out, g or keep_y.  n NULL: only
 * r_out is made.  Sums are f32, of squares too: a row's sum of squares has to lie
 * in f32's range, and with eps = 0 above 2^-126.  Each output takes one rounding,
 * n from r_out before its own.  width 1 .. 16384.
 *
 * keep_r, keep_y, keep_g (codes not NULL): r_out before its rounding (r, where there
 * is no y), y and g are also written in 8 bits, for the gradients.
 * r_out may be r (same pointer and stride); otherwise outputs share no memory
 * with what is read or with one another.
 */
typedef enum to_gate { TO_GATE_NONE = 0, TO_GATE_LINEAR = 1, TO_GATE_SIGMOID = 2, TO_GATE_SILU = 3 } to_gate;

typedef struct to_block_norm_desc {
  int32_t dtype;
  int32_t residual;  /* dtype of r and r_out                                 */
  int32_t width;
  int32_t gate;      /* to_gate                                              */
  int32_t post_norm; /* 0 or 1                                               */
  int32_t reserved0;
  double scale;      /* finite in f32                                        */
  double eps;        /* 0, or in f32's range (not below 2^-149)              */
} to_block_norm_desc;

typedef struct to_block_norm_args {
  to_rows r, y, g, r_out, n;
  to_rows8 keep_r, keep_y, keep_g;
  const float* w_post;
  const float* w_pre;
} to_block_norm_args;

int to_block_norm(const to_block_norm_desc* desc, int64_t tokens, const to_block_norm_args* args,
                  void* stream);

/*
 * Gradients: r_out, y, g as the forward pass had them, or (r8, y8, g8 with codes)
 * as it kept them; dr_out (residual's type, NULL data: zero) and dn (NULL data:
 * zero) of its outputs -> dr (residual's type), dy, dg of its inputs, and dw_post,
 * dw_pre (f32 [width], overwritten, computed even where the weight is NULL; either
 * may be NULL).  Without y: dr and dw_pre alone.  Sums run in a fixed order.  dr may be
 * dr_out; otherwise outputs share no memory with what is read or with one another.
 * workspace: 16-byte aligned device memory.
 */
typedef struct to_block_norm_grad_args {
  to_rows r_out, y, g, dr_out, dn, dr, dy, dg;
  to_rows8 r8, y8, g8;
  const float* w_post;
  const float* w_pre;
  float* dw_post;
  float* dw_pre;
  void* workspace;
  size_t workspace_bytes;
} to_block_norm_grad_args;

size_t to_block_norm_workspace_bytes(const to_block_norm_desc* desc, int64_t tokens);
int to_block_norm_backward(const to_block_norm_desc* desc, int64_t tokens,
                           const to_block_norm_grad_args* args, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* TENSOROPERATIONS_B200_H_ */
