/*
 * pim_b200.h -- C ABI of the B200 execution backend for the flagos-pim-compiler
 * ExecutionPlan runtime.
 *
 * The reference runtime has no native boundary: its HAL (backend/hal_numpy.py) runs
 * kernel stubs as Python callables and its communication library
 * (comm/lowering.py) reduces in NumPy on the host.  Each entry point below is the
 * device implementation of one of those Python-level operations; the comment on
 * each cites the reference interface it replaces.  The B200 HAL
 * (backend/hal_cuda.py) binds them with ctypes.
 *
 * Conventions
 *   - every pointer is a device address (the rank's arena + a planner offset), except
 *     where noted; no function allocates or frees memory;
 *   - `stream` is a cudaStream_t passed as void*; work is enqueued, never synchronised;
 *   - dtype codes: PIM_F32 = 0, PIM_BF16 = 1;
 *   - return 0 on success, a PIM_E* code otherwise; pim_last_error() describes the
 *     last failure on the calling thread.
 */
#ifndef PIM_B200_H
#define PIM_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PIM_ABI_VERSION 15

enum pim_dtype { PIM_F32 = 0, PIM_BF16 = 1, PIM_I32 = 2, PIM_I64 = 3 };
enum pim_status { PIM_OK = 0, PIM_EINVAL = 1, PIM_ECUDA = 2, PIM_EUNSUPPORTED = 3 };
enum pim_projection_mode { PIM_PROJ_PLAIN = 0, PIM_PROJ_ROPE_KV = 1, PIM_PROJ_SILU_MUL = 2 };

/* Version of this ABI (PIM_ABI_VERSION). */
int pim_abi_version(void);

/* Number of kernels this library has launched in this process (every device and stream),
 * counting launches recorded into a CUDA graph once at capture (graph replays launch
 * them again without calling the library).  No counterpart in the reference. */
uint64_t pim_kernel_launches(void);

/* Message for the last non-zero status returned on this thread. */
const char* pim_last_error(void);

/* Whether kernels whose CTAs wait on one another (the decode layer / step kernels, the
 * fused projection + all-reduce) were launched on `device` as cooperative launches that
 * also carry programmatic dependent launch: 1 yes, 0 the driver refused the combination
 * (they run as plain cooperative launches), -1 no such launch was made yet.  Every such
 * launch is cooperative: a grid that cannot be resident at once is refused with a CUDA
 * error instead of waiting.  No counterpart in the reference. */
int pim_cooperative_pdl(int32_t device);

/* Lets kernels running on `device` dereference arena pointers of `peer` (one process
 * driving several GPUs).  Replaces nothing: the reference forbids device-to-device
 * copies (backend/hal_numpy.py:56-57); peers are read only inside redistribute kernels. */
int pim_enable_peer_access(int32_t device, int32_t peer);

typedef struct pim_projection_args {
  const void* x;            /* [rows, k] activations of the rank                      */
  const void* norm_weight;  /* [k] RMSNorm weight, or NULL for no normalisation        */
  const void* weight;       /* [ncols, k] weight rows of the rank (HF [out, in] layout) */
  void* out;                /* PLAIN: [rows, ncols]; ROPE_KV: q [rows, q_heads*head_dim];
                               SILU_MUL: [rows, inter]                                 */
  int64_t rows, k, ncols;
  float eps;
  /* ROPE_KV only */
  const float* rope_cos;    /* [max_seq, head_dim/2] */
  const float* rope_sin;
  const int32_t* positions; /* [rows/seq] start position of each sequence */
  int32_t seq, q_heads, kv_heads, head_dim, max_seq;
  void* kv_base;            /* K block of the layer's first local kv head              */
  int64_t kv_block_stride;  /* elements between (head, k|v) blocks                     */
  int64_t kv_seq_stride;    /* elements between sequences                              */
  /* SILU_MUL only */
  int32_t inter;
  /* PLAIN only: out = residual + x . weight^T (the residual add fused), or NULL */
  const void* residual;
  /* device int32 set to non-zero if a bounded internal wait expires (may be NULL) */
  int32_t* err_flag;
  /* PLAIN at TP > 1, rows <= 8, one process per GPU: a device descriptor written by
   * pim_p2p_desc_init.  The partial x . weight^T of this rank goes to every rank's
   * exchange buffer over NVLink and the kernel writes out = residual + (rank-order sum
   * of the partials), i.e. the linear node, its Partial -> Replicate all_reduce
   * (comm/lowering.py:137-150) and the following add node in one launch; the sum alone
   * also goes to allreduce_out when non-NULL.  NULL: no all-reduce. */
  const void* p2p_desc;
  void* allreduce_out;
  /* ROPE_KV at rows <= 8 (decode), optional: the layer's causal decode attention (the
   * `attention` node after attn_in; the tiled KV reads of PIMStaticKVCache.read_tile,
   * memory/kv_layout.py:207-230, masked as decode_mask, :239-252) computed at the end of
   * the same launch, for every q head and row, into attn_out [rows, q_heads*head_dim]:
   * the CTA that writes the last q / k / v value a head needs computes that head.
   * attn_counters: q_heads device int32, zero-filled before the first call, left zero by
   * every call and written by nothing else.  q_heads <= 64, head_dim 64 or 128; the
   * staged kernel runs whatever pim_set_projection_kernel chose.  NULL: no attention. */
  void* attn_out;
  int32_t* attn_counters;
} pim_projection_args;

/* One projection launch of a rank.  Replaces the DPU `aten.linear` kernel stub that
 * NumpyBackend.submit runs for a "launch" command (backend/hal_numpy.py:251-256; rule
 * graph/spec_prop.py:236-256) together with the host glue that surrounds it in the
 * exported graph: RMSNorm (pow/mean/rsqrt + mul), RoPE (slice/neg/cat + mul/add) and
 * the KV append of PIMStaticKVCache.update (memory/kv_layout.py:187-205) in mode
 * ROPE_KV; silu + mul in mode SILU_MUL.  rows <= 8 run as a GEMV; larger row counts
 * need `scratch` of pim_projection_scratch_bytes() bytes.  For rows <= 8 the scratch is
 * optional: while PIM_PROJ_KERNEL_DYNAMIC is selected, pim_projection_scratch_bytes()
 * asks for a work counter that must be zero-filled before the first call and not be
 * written by anything else (the kernel leaves it zero); a call without it runs the
 * staged kernel. */
int pim_projection(const pim_projection_args* a, int32_t dtype, int32_t mode, void* scratch,
                   int64_t scratch_bytes, void* stream);
int64_t pim_projection_scratch_bytes(const pim_projection_args* a, int32_t dtype, int32_t mode);

/* Kernel that runs decode projections (rows <= 8) from now on, for the whole process:
 * PIM_PROJ_KERNEL_REGISTER (weights streamed through registers), PIM_PROJ_KERNEL_STAGED
 * (cp.async-staged, every warp streams the same bytes) or PIM_PROJ_KERNEL_DYNAMIC
 * (staged, CTAs take units of work from a counter); any other value (2 included: it
 * was a bulk-copy kernel, removed) is refused with PIM_EINVAL.  All give results within
 * fp32 summation-order differences of one another; shapes a kernel cannot take run on
 * the register kernel.  The initial choice is the staged kernel unless the environment
 * variable PIM_GEMV says "reg" or "dyn".
 * Launches already recorded in a CUDA graph keep their kernel.  No counterpart in the
 * reference. */
#define PIM_PROJ_KERNEL_REGISTER 0
#define PIM_PROJ_KERNEL_STAGED 1
#define PIM_PROJ_KERNEL_DYNAMIC 3
int pim_set_projection_kernel(int32_t kernel);
int32_t pim_projection_kernel(void);

/* Bytes of the zero-filled barrier word pair that pim_decode_layer takes. */
#define PIM_DECODE_LAYER_BARRIER_BYTES 256

/* One decoder layer of a decode step with one activation row (batch 1) in ONE
 * launch: the four projections attn_in (mode ROPE_KV, with attn_out / attn_counters:
 * the layer's decode attention), o_proj (PLAIN, residual optional), mlp_in (SILU_MUL)
 * and down (PLAIN, residual optional) -- the five launch commands a layer of the decode
 * plan lowers to (pim_projection x 4 + the attention), run by one grid of at most as many
 * CTAs as the GPU holds at once, with a grid-wide barrier between phases.  Each phase
 * computes what pim_projection computes (the staged kernel's arithmetic; results equal
 * pim_projection's up to fp32 summation order).  The chain is checked: o_proj.x ==
 * attn_in.attn_out, mlp_in.x == o_proj.out, down.x == mlp_in.out, and the k of each
 * phase equals the width of the previous phase's output; attn_in and mlp_in take a
 * norm_weight, o_proj and down none.  At TP > 1 (one process per GPU) o_proj and down
 * carry the same p2p_desc (and optionally allreduce_out): each is then the row-parallel
 * projection + rank-order all-reduce + residual add of pim_projection's p2p_desc, two
 * all-reduce calls per launch on the descriptor's group (exchange rows of at least
 * ncols x element bytes).  `barrier`: PIM_DECODE_LAYER_BARRIER_BYTES
 * of device memory, zero-filled before the first call and written by nothing else (every
 * call leaves the count zero); calls on one barrier must not overlap on the GPU.
 * `err_flag` (device int32, may be NULL) is raised when a barrier wait gives up (one
 * second): the layer's output is then not valid.  PIM_EUNSUPPORTED when the shapes do not
 * fit the kernel's shared memory or the GPU cannot hold its grid.  Replaces the five
 * `launch` commands of a decode layer; no single counterpart in the reference. */
int pim_decode_layer(const pim_projection_args* attn_in, const pim_projection_args* o_proj,
                     const pim_projection_args* mlp_in, const pim_projection_args* down, void* barrier,
                     int32_t* err_flag, int32_t dtype, void* stream);

/* A whole decode step with one activation row in ONE launch: every layer as in
 * pim_decode_layer, with a grid-wide barrier in place of the kernel boundary between
 * consecutive layers (the next layer's q/k/v weights streaming across it), then, when
 * `head` is given, the lm_head_in projection (PLAIN with norm_weight: the final RMSNorm
 * and the vocabulary GEMV of the decode plan).  Replaces the 5 x nlayers + 1 launch
 * commands of a decode step between the embedding and the logits; no single counterpart
 * in the reference.
 *
 * pim_decode_step_prepare checks `layers` (4 * nlayers pointers: attn_in, o_proj, mlp_in,
 * down of each layer, each layer as pim_decode_layer checks it, layer l + 1 reading layer
 * l's output, the same p2p_desc in every layer or none) and `head` (NULL, or reading the
 * last layer's output), writes the layers' argument table into `table` (device memory of
 * pim_decode_step_table_bytes(nlayers) bytes, 16-byte aligned; a synchronous copy: not
 * during a stream capture), sizes the grid (PIM_EUNSUPPORTED when no grid fits) and returns
 * a host-side plan.  The table must stay untouched while the plan is used.
 * pim_decode_step launches it; `barrier` and `err_flag` as in pim_decode_layer (calls on
 * one barrier must not overlap on the GPU).  pim_decode_step_free releases the plan (host
 * memory only). */
typedef struct pim_decode_step_plan pim_decode_step_plan;
int64_t pim_decode_step_table_bytes(int32_t nlayers);
int pim_decode_step_prepare(const pim_projection_args* const* layers, int32_t nlayers,
                            const pim_projection_args* head, int32_t dtype, void* table, int64_t table_bytes,
                            pim_decode_step_plan** plan);
int pim_decode_step(const pim_decode_step_plan* plan, void* barrier, int32_t* err_flag, void* stream);
void pim_decode_step_free(pim_decode_step_plan* plan);

/* Kernel that runs bf16 row-batch projections (rows > 8, the tcgen05 GEMM) from now on,
 * for the whole process: PIM_ROW_BATCH_KERNEL_TILE (one 128 x 256 output tile per CTA)
 * or PIM_ROW_BATCH_KERNEL_PERSISTENT (one CTA per SM looping over the tiles, the epilogue
 * of one tile overlapping the MMAs of the next).  Both accumulate every output in the
 * same order (fp32 over K blocks in order), so results are identical.  The initial
 * choice is the persistent kernel (the faster on B200) unless the environment variable
 * PIM_GEMM says "tile".
 * Launches already recorded in a CUDA graph keep their kernel.  No counterpart in the
 * reference. */
#define PIM_ROW_BATCH_KERNEL_TILE 0
#define PIM_ROW_BATCH_KERNEL_PERSISTENT 1
int pim_set_row_batch_kernel(int32_t kernel);
int32_t pim_row_batch_kernel(void);

/* Attention of one layer over the rank's KV blocks (causal; the query at position p
 * sees keys 0..p).  Replaces the host `aten.scaled_dot_product_attention` node and
 * the tiled KV reads of PIMStaticKVCache.read_tile (memory/kv_layout.py:207-230),
 * masked as decode_mask / prefill_mask (memory/kv_layout.py:233-252).  head_dim 32,
 * 64 or 128.  Needs a caller-provided `workspace` of pim_attention_workspace_bytes()
 * bytes, used by the split-K kernel (bf16 head_dim-128 row batches of 16 or more query
 * rows per sequence run on the tensor-core kernels and leave it untouched). */
int pim_attention(const void* q, const int32_t* positions, const void* kv_base, int64_t kv_block_stride,
                  int64_t kv_seq_stride, void* out, int32_t batch, int32_t seq, int32_t q_heads,
                  int32_t kv_heads, int32_t head_dim, int32_t max_seq, int32_t dtype, void* workspace,
                  int64_t workspace_bytes, void* stream);

/* Row batches (seq >= 16) of bf16 with head_dim 128 run on the tensor cores: warp-level
 * MMA (PIM_PREFILL_ATTENTION_MMA, the default) or tcgen05 with TMEM accumulators and
 * TMA-loaded tiles (PIM_PREFILL_ATTENTION_TCGEN05), for the whole process from the call
 * on; the initial choice is tcgen05 when the environment variable PIM_ATTN says "tc".
 * Launches already recorded in a CUDA graph keep their kernel.  The tcgen05 kernel has
 * no error argument: a wait of it that gives up raises a library-wide device word, which
 * pim_attention_errors returns (1 raised, 0 clear, -1 when it cannot be read) and clears
 * when `reset` != 0 (synchronous; not during a stream capture).  No counterpart in the
 * reference. */
#define PIM_PREFILL_ATTENTION_MMA 0
#define PIM_PREFILL_ATTENTION_TCGEN05 1
int pim_set_prefill_attention_kernel(int32_t kernel);
int32_t pim_prefill_attention_kernel(void);
int32_t pim_attention_errors(int32_t reset);
int64_t pim_attention_workspace_bytes(int32_t batch, int32_t seq, int32_t q_heads, int32_t head_dim,
                                      int32_t max_seq);

/* Size of the fixed scratch behind pim_attention_noalloc (4 MiB on every GPU that loads
 * the library, held until the process exits). */
#define PIM_ATTENTION_NOALLOC_SCRATCH_BYTES (4u << 20)

/* pim_attention without a caller workspace, for callers that cannot allocate device
 * memory -- for example a plugin whose host program owns all device memory through its
 * own pool allocator, or code on a latency-critical path where cudaMalloc would
 * synchronize the device.  No counterpart in the reference (its attention runs on the
 * host).  Allocates nothing: the workspace is a file-scope device array of
 * PIM_ATTENTION_NOALLOC_SCRATCH_BYTES.  Only the split-K kernel uses it: shapes that run
 * there and whose workspace (pim_attention_workspace_bytes) is larger are rejected with
 * PIM_EINVAL; bf16 head_dim-128 row batches (16 or more query rows per sequence) run on
 * the tensor-core kernels, need no workspace and are accepted at any size.  The first
 * call on each device (and under each CUDA context) looks the array up
 * (cudaGetSymbolAddress) with that device current; make that first call before any
 * stream capture.  A cudaDeviceReset after the first call is not supported (the cached
 * address can go stale).  All calls share the array: calls that overlap on the GPU race;
 * each call clears the counters it needs zeroed. */
int pim_attention_noalloc(const void* q, const int32_t* positions, const void* kv_base, int64_t kv_block_stride,
                          int64_t kv_seq_stride, void* out, int32_t batch, int32_t seq, int32_t q_heads,
                          int32_t kv_heads, int32_t head_dim, int32_t max_seq, int32_t dtype, void* stream);

/* Embedding row gather.  Replaces the host `aten.embedding` node of the exported graph
 * (the reference keeps the table Replicate@host, docs/spec.md:1994). Out-of-range ids
 * give a zero row and set *err_flag (device int32, may be NULL). */
int pim_embedding(const int32_t* ids, const void* table, void* out, int64_t n_ids, int64_t hidden,
                  int64_t vocab, int32_t dtype, int32_t* err_flag, void* stream);

/* out = a + b (rounded to dtype).  Replaces the DPU `aten.add.Tensor` stub for the
 * residual adds (graph/spec_prop.py:265-305). */
int pim_add(const void* a, const void* b, void* out, int64_t n, int32_t dtype, void* stream);

/* out[b] = x[b, index] for b < batch (rows of row_bytes bytes).  Replaces taking the
 * prefill logits at position P-1 (docs/spec.md:1552-1553). */
int pim_select_rows(const void* x, void* out, int32_t batch, int32_t seq, int64_t row_bytes, int32_t index,
                    void* stream);

/* Greedy sampling: first index of each row's maximum.  Replaces the host argmax of
 * the decode loop (docs/spec.md:1552-1556). */
int pim_argmax(const void* x, int32_t* out, int32_t rows, int64_t n, int32_t dtype, void* stream);

/* Device copy (same device or peer).  Replaces dpu_copy_to / dpu_copy_from byte
 * moves of one segment (backend/dpu_sdk.py:139-157). */
int pim_copy(void* dst, const void* src, int64_t nbytes, void* stream);

/* Partial -> Replicate combine: dst[d][i] = ((0 + src[0][i]) + src[1][i]) + ..., rounded to
 * dtype after every add, in the given (rank) order; divided by nsrc when mean != 0.
 * Bit-identical to the host accumulation of comm/lowering.py:137-150.  src/dst are
 * HOST arrays of up to 8 device pointers each. */
int pim_ordered_sum(const void* const* src, int32_t nsrc, void* const* dst, int32_t ndst, int64_t n,
                    int32_t dtype, int32_t mean, void* stream);

/* The Partial -> Replicate combine followed by the residual add that consumes it (the
 * `add` node after o_proj / down_proj, graph/spec_prop.py:265-305):
 * out[i] = residual[i] + S[i], S the rank-order sum of pim_ordered_sum (rounded to dtype
 * after every partial) and the add rounded to dtype once more, exactly as the combine
 * followed by the add; S itself is also written to sum_out unless it is NULL.  src is a
 * HOST array of up to 8 device pointers; dtype PIM_F32 or PIM_BF16. */
int pim_ordered_sum_add(const void* const* src, int32_t nsrc, const void* residual, void* out, void* sum_out,
                        int64_t n, int32_t dtype, void* stream);

/* One process per GPU: the Partial -> Replicate combine over NVLink peer memory, one
 * kernel per call.  Every rank calls it in the same order with its partial `src`
 * (numel elements, numel * element size a multiple of 16 and at most capacity_bytes);
 * `bufs` is a HOST array of `size` device pointers: every rank's exchange buffer of
 * PIM_P2P_HEADER_BYTES + 2 * size * capacity_bytes bytes (zero-filled before the first
 * call) as mapped in this process (pim_ipc_open), this rank's own at bufs[rank].  The
 * result is the rank-order sum of pim_ordered_sum (bit-identical to comm/lowering.py:
 * 137-150), written to the `ndst` (<= 4) device pointers of the HOST array `dsts`.
 * `counter` is a device int32 of this rank, zero before the first call.  A rank that
 * waits more than 1 s for a peer raises *err_flag (when given) and returns.  Replaces
 * the host-star all_reduce of comm/lowering.py:137-150 at TP > 1; no kernel in the
 * reference. */
#define PIM_P2P_HEADER_BYTES 1024
#define PIM_P2P_MAX_RANKS 64

/* Size of the device descriptor of a P2P group, and its initialisation (synchronous):
 * the group's exchange buffers as mapped here (HOST array of `size` device pointers), the
 * row capacity, this rank's call counter (shared with pim_allreduce_p2p), two device
 * int32 tickets (zero) and the error word raised when a wait for a peer gives up. */
int64_t pim_p2p_desc_bytes(void);
int pim_p2p_desc_init(void* desc, int32_t rank, int32_t size, void* const* bufs, int64_t capacity_bytes,
                      int32_t* counter, int32_t* tickets, int32_t* err_flag);
int pim_allreduce_p2p(const void* src, void* const* dsts, int32_t ndst, int64_t numel, int32_t dtype,
                      int32_t rank, int32_t size, void* const* bufs, int64_t capacity_bytes, int32_t* counter,
                      int32_t* err_flag, void* stream);
/* pim_allreduce_p2p followed by the residual add that consumes the sum, in the same
 * kernel: y = residual + sum (the fp32 add of the rounded sum, rounded once -- the bits of
 * pim_ordered_sum_add, i.e. of the reference's all_reduce then aten.add), and the sum itself
 * into `sum_out` when it is not NULL.  Replaces the host-star all_reduce of
 * comm/lowering.py:137-150 together with the DPU `add` node after it. */
int pim_allreduce_p2p_add(const void* src, const void* residual, void* y, void* sum_out, int64_t numel,
                          int32_t dtype, int32_t rank, int32_t size, void* const* bufs, int64_t capacity_bytes,
                          int32_t* counter, int32_t* err_flag, void* stream);

/* The same bit-exact rank-order all-reduce over the same exchange buffers with the
 * low-latency protocol: every 32-bit word of the partial is stored to the peers as one
 * 64-bit word whose high half is the call's epoch, and readers poll the words themselves
 * (no system-scope fence, no separate flag).  Writes the sum to `sum_out` and/or, when
 * `residual` and `y` are given, y = residual + sum (the bits of pim_ordered_sum_add).
 * 2 * numel * element size must fit `capacity_bytes`.  A group of exchange buffers is used
 * with this protocol or with pim_allreduce_p2p / the fused projection, not both.  Replaces
 * the host-star all_reduce of comm/lowering.py:137-150 (and the add node after it). */
int pim_allreduce_p2p_ll(const void* src, const void* residual, void* y, void* sum_out, int64_t numel,
                         int32_t dtype, int32_t rank, int32_t size, void* const* bufs, int64_t capacity_bytes,
                         int32_t* counter, int32_t* err_flag, void* stream);

/* CUDA IPC for the exchange buffers: the 64-byte handle of the allocation holding `ptr`
 * and ptr's byte offset in it; opening a peer's handle maps that allocation here
 * (*base; add the peer's offset); closing unmaps it.  No reference counterpart. */
int pim_ipc_export(const void* ptr, void* handle64, int64_t* offset);
int pim_ipc_open(const void* handle64, void** base);
int pim_ipc_close(void* base);

/* Executes `count` (src, dst, nbytes) runs stored at desc_dev (device memory, 24 bytes
 * each: two pointers and an int64).  Replaces the collect / writeback transfer
 * sequences of dma_sequence (comm/plan.py:330-347) as executed by DmaEngine
 * (comm/lowering.py:55-97) for all_gather, all_to_all, scatter and broadcast. */
int pim_batched_copy(const void* desc_dev, int32_t count, int64_t max_nbytes, void* stream);

/* Seeded N(0, std^2) fill (counter-based; same seed -> same values).  Used for
 * random-init weights; no reference counterpart (HF initialises on the host). */
int pim_fill_normal(void* out, int64_t n, int32_t dtype, uint64_t seed, float std, void* stream);

/* Constant fill (e.g. RMSNorm weights = 1).  No reference counterpart. */
int pim_fill_const(void* out, int64_t n, int32_t dtype, float value, void* stream);


/* ---- paged KV cache ------------------------------------------------------------
 * A KV cache whose memory follows the tokens: pages of page_size slots, and per sequence
 * (row) a table of the pages that hold its slots 0, 1, 2, ... in order.  It stands beside
 * the contiguous [max_seq, head_dim] blocks of memory/kv_layout.py (pim_attention, the
 * KV append of pim_projection) for sequences of different lengths, for caches of bounded
 * size and for beams that share their prompt.  No counterpart in the reference, whose
 * cache is static.
 *
 * Every entry point below checks its arguments on the host before any CUDA call and
 * bounds-checks what it reads from device memory (lengths, positions, page ids, parents):
 * a bad value raises *err_flag (device int32, may be NULL) and the access it stands for is
 * left out, as stated at each.  Rows may share pages only where an entry point says so.
 * Nothing here keeps state between calls: workspaces are scratch (no initial contents,
 * none expected afterwards); calls that overlap on the GPU must not share one. */
typedef struct pim_paged_kv {
  void* k_pages;            /* page p, head h, slot i, dim d at p * page_stride + (h * page_size + i) * head_dim + d */
  void* v_pages;            /* the same layout */
  int64_t page_stride;      /* elements between pages: at least kv_heads * page_size * head_dim */
  const int32_t* table;     /* [rows, table_stride]: page ids, 0 <= id < num_pages where a row has slots */
  int64_t table_stride;     /* elements between rows, at least max_pages */
  int32_t rows;             /* sequences */
  int32_t max_pages;        /* table entries of a row: a row holds at most max_pages * page_size slots */
  int32_t num_pages;
  int32_t page_size;        /* 8, 16, 32, 64, 128 or 256 */
  int32_t kv_heads;
  int32_t head_dim;         /* 32, 64 or 128 */
} pim_paged_kv;

typedef struct pim_paged_append_args {
  pim_paged_kv kv;
  const void* q;            /* token t, head h, dim d at t * q_stride + h * head_dim + d; NULL: no q */
  const void* k;
  const void* v;
  int64_t q_stride, k_stride, v_stride;                /* elements between tokens */
  int64_t k_head_stride, v_head_stride;                /* elements between heads of k and of v */
  void* q_out;              /* token t at t * q_out_stride; may be q itself (same stride, no pair_order) */
  int64_t q_out_stride;
  const float* rope_cos;    /* [max_pos, head_dim / 2]; both NULL: no rotation */
  const float* rope_sin;
  int32_t max_pos;
  int32_t q_heads;          /* with q; any number */
  int32_t pair_order;       /* 1: element 2j of a head is dim j and 2j + 1 is dim j + head_dim / 2 (the row order of
                               qkv_proj.weight, as pim_projection PLAIN leaves it); outputs are in dim order */
  int64_t tokens;
  const int32_t* starts;    /* [rows + 1]: row b has tokens starts[b] .. starts[b + 1) (0 or more); NULL: token b is
                               row b's only one, tokens == rows.  Tokens behind starts[rows] are left out; starts that
                               decrease (the row counts as without tokens) or leave [0, tokens] raise *err_flag. */
  const int32_t* lengths;   /* [rows] slots in use: the row's tokens go to slots lengths[b], lengths[b] + 1, ... */
  const int32_t* positions; /* [rows] position of the row's first new token; NULL: lengths */
  int32_t* lengths_out;     /* [rows] lengths + new tokens (not `lengths` itself); may be NULL */
  int32_t* positions_out;   /* [rows] positions + new tokens (not `positions` itself); may be NULL */
  int32_t* slot_positions;  /* eviction state, both or neither: [rows, kv_heads, slots] position of each slot's */
  float* weights;           /* token (set) and its accumulated attention weight (set to 0) */
  int64_t state_row_stride, state_head_stride;         /* elements, of both state arrays */
  int32_t* err_flag;
} pim_paged_append_args;

/* New tokens into the pages of their rows, for every head of a layer: k rotated to its
 * position (RoPE, halves rotated against one another as in pim_projection ROPE_KV,
 * computed in fp32 and rounded once), v as it is; q rotated into q_out.  Replaces
 * PIMStaticKVCache.update (memory/kv_layout.py:187-205) over pages.  A token whose slot,
 * page or position is out of range raises *err_flag and is left out, but counted in
 * lengths_out and positions_out: what follows would read a slot that was not written. */
int pim_paged_append(const pim_paged_append_args* a, int32_t dtype, void* stream);

typedef struct pim_paged_attention_args {
  pim_paged_kv kv;
  const void* q;            /* [rows, q_heads, head_dim], q_stride elements between rows */
  void* out;                /* the same shape, out_stride elements between rows */
  int64_t q_stride, out_stride;
  const int32_t* lengths;   /* [rows] slots the row's token attends to (its own included); 0: the output row is 0 */
  int32_t q_heads;          /* a multiple of kv_heads */
  float scale;              /* of the scores; 0: 1 / sqrt(head_dim) */
  float* weights;           /* [rows, kv_heads, slots], weights_*_stride elements: every slot's probability, summed over
                               the query heads of its group, is added to it; NULL: not asked for */
  int64_t weights_row_stride, weights_head_stride;
  int32_t* err_flag;
} pim_paged_attention_args;

/* Attention of one new token per row over its pages: the decode form of pim_attention over
 * a paged cache, with query groups that share a kv head reading it once.  Rows may share
 * pages.  A length outside [0, max_pages * page_size] is clamped and a page id out of
 * range hides its slots; both raise *err_flag.  A row without slots, or without a score above
 * -inf, gives zeros; a NaN in a score of a head makes its output and probabilities NaN.  fp32
 * scores, softmax and sums; the output is rounded once.  The result does not depend on timing: no atomics. */
int pim_paged_attention(const pim_paged_attention_args* a, int32_t dtype, void* workspace, int64_t workspace_bytes,
                        void* stream);
/* Bytes of the workspace of a call with these arguments (its lengths are not read); -1 for
 * arguments that pim_paged_attention refuses. */
int64_t pim_paged_attention_workspace_bytes(const pim_paged_attention_args* a, int32_t dtype);

typedef struct pim_paged_evict_args {
  pim_paged_kv kv;
  const int32_t* lengths;          /* [rows] slots in use */
  const int32_t* positions;        /* [rows] position of the row's next token (tokens seen so far) */
  const float* weights;            /* [rows, kv_heads, slots] accumulated attention weights */
  const int32_t* slot_positions;   /* [rows, kv_heads, slots] positions of the slots' tokens */
  float* weights_out;              /* the state after eviction; each may be its input (in place) or apart */
  int32_t* slot_positions_out;
  int32_t* lengths_out;            /* [rows]; not `lengths` itself */
  int64_t state_row_stride, state_head_stride;          /* elements, of all four state arrays */
  int32_t budget;                  /* slots kept per row and head, at least 1 */
  int32_t recent, sink;            /* tokens at position >= positions - recent or < sink stay; recent + sink <= budget */
  int32_t* err_flag;
} pim_paged_evict_args;

/* Cuts every row of more than `budget` slots down to `budget`, each head by itself: the
 * newest `recent` tokens and the first `sink` ones stay, then those of the largest weight
 * (of equal ones the lower slot; a NaN weight ranks below every number).  Kept tokens at
 * slots >= budget move, K, V and state, into the slots < budget that became free, the
 * first into the first; all others stay where they are.  Attention does not depend on the
 * order of slots (K is rotated already) and slot_positions says which token a slot holds.
 * Slots >= lengths_out are left as they were.  Rows must not share pages.  A length out of
 * range is clamped, and of a move whose freed or kept slot has a page id out of range only the
 * state follows, not K and V; both raise *err_flag.  No counterpart in the reference. */
int pim_paged_evict(const pim_paged_evict_args* a, int32_t dtype, void* workspace, int64_t workspace_bytes,
                    void* stream);
int64_t pim_paged_evict_workspace_bytes(const pim_paged_evict_args* a, int32_t dtype);

typedef struct pim_beam_select_args {
  const void* logits;       /* [batch, beams, vocab], logits_stride elements between beams (batch-major) */
  int64_t logits_stride;
  const float* scores;      /* [batch, beams] log-probability of each beam so far */
  const int32_t* done;      /* [batch, beams] non-zero: the beam has ended; NULL: none has */
  float* scores_out;        /* [batch, beams_out], best first */
  int32_t* parents;         /* [batch, beams_out] beam (0 .. beams - 1) that each continues */
  int32_t* tokens;          /* [batch, beams_out] */
  int32_t* done_out;        /* [batch, beams_out] the parent had ended or the token is `eos`; may be NULL */
  int32_t batch, beams;     /* beams <= 64 */
  int32_t beams_out;        /* <= 64 */
  int32_t vocab;            /* <= 2^19 */
  int32_t eos;              /* -1: no such token */
  int32_t pad;              /* the token a beam that has ended continues with, 0 <= pad < vocab */
  int32_t* err_flag;
} pim_beam_select_args;

/* One step of beam search, per batch entry: the beams_out largest of
 * scores[w] + logits[w][t] - log(sum_u exp(logits[w][u])) over beams w and tokens t, ties to the
 * lowest w * vocab + t; a beam that has ended offers one candidate, `pad` at its score.  A
 * logit that is not finite is no candidate and no part of the sum; a beam whose score is
 * not finite offers none.  -inf is a mask, in either; NaN and +inf raise *err_flag (the logits
 * of a beam that has ended are not looked at).  Where fewer than beams_out candidates are left, the rest get
 * score -inf, parent 0, token `pad`, done 1.  Candidates of one beam are compared by their
 * logits, those of different beams by their scores in fp64 (of equal ones the lower beam is
 * first); scores_out is rounded once.
 * Stands beside pim_argmax (greedy sampling, docs/spec.md:1552-1556). */
int pim_beam_select(const pim_beam_select_args* a, int32_t dtype, void* workspace, int64_t workspace_bytes,
                    void* stream);
int64_t pim_beam_select_workspace_bytes(const pim_beam_select_args* a, int32_t dtype);

typedef struct pim_beam_reorder_args {
  void* pages;              /* num_blocks blocks (each layer's K and V), block_stride elements apart, of pages laid */
  int64_t block_stride;     /* out as in pim_paged_kv */
  int64_t page_stride;
  const int32_t* table;     /* [batch * beams, table_stride], the beams before */
  int32_t* table_out;       /* the beams after (apart from `table`); max_pages entries of a row are written */
  int64_t table_stride;     /* of both */
  const int32_t* lengths;   /* [batch] slots in use, the same for every beam of an entry */
  const int32_t* parents;   /* [batch, beams] as pim_beam_select gives them */
  int32_t batch, beams;     /* beams <= 64 */
  int32_t num_blocks;
  int32_t max_pages, num_pages, page_size, kv_heads, head_dim;
  int32_t* err_flag;
} pim_beam_reorder_args;

/* Reordering of the beams' cache states after pim_beam_select, through the page table: new
 * beam j shares its parent's full pages.  The partly filled page cannot be shared, since
 * both beams will append to it: a parent's first child takes the parent's, and each further
 * child's is a copy (of the slots in use, in every block) in the page of a beam that has no
 * child, so that no copy reads a page that another writes and no page is needed or lost.
 * Entries behind the slots in use (reserved pages) stay with the beam's index.  The partly
 * filled and reserved pages of the beams of an entry must differ.  A parent, length or page
 * id out of range raises *err_flag: that entry's beams then keep their own tables. */
int pim_beam_reorder(const pim_beam_reorder_args* a, int32_t dtype, void* stream);

/* ---- aten-level operations -------------------------------------------------------
 * For graphs compiled at aten granularity by the reference's own passes (torch.export,
 * graph/partition.py:36-81, graph/spec_prop.py:411-451): the DPU nodes (aten.linear,
 * aten.add / mul.Tensor, aten.tanh; the reference's kernel stubs) run on their rank's
 * arena and the host nodes (the torch callables the reference runs on the CPU:
 * embedding, pow / mean / rsqrt, view / reshape / transpose / slice / cat / expand,
 * to.dtype, matmul, cos / sin, scaled_dot_product_attention, silu, neg, alias) run on the
 * plan's device-resident host buffer.  Operands are strided views: element offset,
 * shape and element strides (a stride of 0 broadcasts); operand views have the output's
 * rank.  Dtypes PIM_F32, PIM_BF16, PIM_I32, PIM_I64; arithmetic in fp32 (copies convert
 * exactly between the integer types and fp32 where the value allows). */
#define PIM_MAX_DIMS 8
typedef struct pim_tensor_view {
  void* data;                    /* base pointer (device) */
  int32_t dtype;                 /* pim_dtype */
  int32_t ndim;                  /* 0..PIM_MAX_DIMS */
  int64_t offset;                /* elements from data to element [0, ..., 0] */
  int64_t shape[PIM_MAX_DIMS];
  int64_t stride[PIM_MAX_DIMS];  /* elements; 0 broadcasts */
} pim_tensor_view;

enum pim_aten_op {
  /* unary (pim_aten_unary; `scalar` is the second operand of the *_SCALAR ops and the
   * exponent of POW_SCALAR) */
  PIM_ATEN_NEG = 0, PIM_ATEN_RSQRT = 1, PIM_ATEN_SQRT = 2, PIM_ATEN_SILU = 3, PIM_ATEN_COS = 4,
  PIM_ATEN_SIN = 5, PIM_ATEN_TANH = 6, PIM_ATEN_EXP = 7, PIM_ATEN_RECIPROCAL = 8, PIM_ATEN_POW_SCALAR = 9,
  PIM_ATEN_ADD_SCALAR = 10, PIM_ATEN_MUL_SCALAR = 11, PIM_ATEN_SUB_SCALAR = 12, PIM_ATEN_DIV_SCALAR = 13,
  /* binary (pim_aten_binary) */
  PIM_ATEN_ADD = 20, PIM_ATEN_SUB = 21, PIM_ATEN_MUL = 22, PIM_ATEN_DIV = 23
};

/* dst[i] = src[i] over dst's shape, converting the element type: aten view / reshape /
 * unsqueeze / alias / transpose / slice / expand / to.dtype, and one input of aten.cat
 * (dst a view into the output).  Replaces the host FX callables of those nodes. */
int pim_aten_copy(const pim_tensor_view* dst, const pim_tensor_view* src, void* stream);
/* dst = op(src[, scalar]): aten.neg / rsqrt / silu / cos / sin / tanh / pow.Tensor_Scalar
 * and add / mul / sub / div with a scalar operand (the reference's DPU aten.add / mul stub
 * when one operand is a Python number, graph/spec_prop.py:265-305). */
int pim_aten_unary(int32_t op, const pim_tensor_view* dst, const pim_tensor_view* src, double scalar,
                   void* stream);
/* dst = a op b with broadcasting: the DPU aten.add / mul.Tensor stubs
 * (graph/spec_prop.py:265-305) and their host counterparts. */
int pim_aten_binary(int32_t op, const pim_tensor_view* dst, const pim_tensor_view* a, const pim_tensor_view* b,
                    void* stream);
/* aten.mean.dim over the last dimension with keepdim (RMSNorm's variance). */
int pim_aten_mean_last(const pim_tensor_view* dst, const pim_tensor_view* src, void* stream);
/* aten.arange: dst[i] = start + i * step (the positions of the exported model). */
int pim_aten_arange(const pim_tensor_view* dst, double start, double step, void* stream);
/* aten.matmul of batched matrices [..., M, K] x [..., K, N] (batch dims broadcast). */
int pim_aten_matmul(const pim_tensor_view* dst, const pim_tensor_view* a, const pim_tensor_view* b, void* stream);
/* aten.scaled_dot_product_attention: q [B, H, S, D], k / v [B, Hk, L, D] (H a multiple of
 * Hk), an additive mask broadcastable to [B, H, S, L] (mask->data NULL or mask NULL for
 * none), causal != 0 for is_causal; at most 8192 keys. */
int pim_aten_sdpa(const pim_tensor_view* out, const pim_tensor_view* q, const pim_tensor_view* k,
                  const pim_tensor_view* v, const pim_tensor_view* mask, double scale, int32_t causal,
                  void* stream);
/* aten.embedding with integer ids of any width; an id outside the table gives a zero
 * row and sets *err_flag (device int32, may be NULL). */
int pim_aten_embedding(const pim_tensor_view* out, const pim_tensor_view* table, const pim_tensor_view* ids,
                       int32_t* err_flag, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PIM_B200_H */
