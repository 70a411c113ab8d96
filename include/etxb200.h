/* etxb200 -- C ABI of the B200 (sm_100a) decode megakernel.
 *
 * The reference (cklxx/etx-megakernel) has no FFI: Python emits a HIP kernel plus a C++ host built on
 * etx/runtime/include/etx/host.h and runs the linked binary as a subprocess.  This library replaces that emitted
 * kernel + host with one hand-written persistent CUDA kernel behind plain C entry points, so the same program
 * surface (task graph -> plan -> session run) drives it through ctypes / cgo / JNI.  Every entry point returns an
 * int32 status (0 = OK, ETXB_E_* otherwise), never throws and never exits the process.
 *
 * Which reference interface each entry replaces (paths inside the reference project):
 *   etxb_create / etxb_bind   etx_host::alloc_args + setup      etx/runtime/include/etx/host.h:55-210
 *   etxb_set_step             vl_set_params (VlParams upload)   examples/vllm_llm/vl_tiles.hip:13-24, 92-95
 *   etxb_launch               etx_host::check_residency+launch  host.h:326-347
 *   etxb_wait                 etx_host::wait (watchdog)         host.h:351-417
 *   etxb_step                 etx_host::run                     host.h:518-531
 *   etxb_status               ctrl words + event dump           etx/runtime/include/etx/abi.h:101-105, host.h:564-580
 *   etxb_trace                ETX_TRACE_RAW per-task stamps     host.h:640-675
 *   etxb_decode_host          the host token loop               examples/vllm_llm/host.hip:819-894
 *   etxb_op_*                 one launch of a single tile type; the argument-block bytes are the tile's own
 *                             (etx/ops/gemv.py:80-94, etx/ops/topk.py:16-23, etx/ops/attnprep.py:11-15,
 *                              etx/importer/argblock.py:16-29)
 */
#ifndef ETXB200_H
#define ETXB200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ETXB_VERSION 0x00010000

/* status codes */
enum {
  ETXB_OK = 0,
  ETXB_E_ARG = 1,        /* null pointer, bad size, unknown name */
  ETXB_E_PLAN = 2,       /* plan blob malformed or inconsistent (rejected before any launch) */
  ETXB_E_CUDA = 3,       /* a CUDA runtime call failed; etxb_last_error() has the text */
  ETXB_E_RESIDENCY = 4,  /* the persistent grid cannot be co-resident on this device */
  ETXB_E_TIMEOUT = 5,    /* a device wait ran past its deadline; the kernel returned, the context is usable */
  ETXB_E_ABORTED = 6,    /* host abort requested */
  ETXB_E_UNSUPPORTED = 7,/* shape outside what the tile supports (message says which) */
  ETXB_E_FULL = 8        /* a pool has no room: nothing was changed */
};

/* tile bodies (the `body` field of a plan's task type; the symbol names a graph links are mapped to these) */
enum {
  ETXB_BODY_NOP = 0,
  ETXB_BODY_PROLOGUE = 1,     /* vl_prologue       examples/vllm_llm/vl_tiles.hip:31-45 */
  ETXB_BODY_ARGMAX = 2,       /* vl_argmax         vl_tiles.hip:47-89 */
  ETXB_BODY_GEMV = 3,         /* dsl_gemv[_fold]   etx/ops/gemv.py:816-840 */
  ETXB_BODY_MOE_UP = 4,       /* dsl_moe_up[_fold] etx/ops/gemv.py:841-911 */
  ETXB_BODY_MOE_DOWN = 5,     /* dsl_moe_down      etx/ops/gemv.py:912-953 */
  ETXB_BODY_TOPK = 6,         /* dsl_topk          etx/ops/topk.py:35-156 */
  ETXB_BODY_ATTNPREP = 7,     /* dsl_attnprep      etx/ops/attnprep.py:86-211 */
  ETXB_BODY_ATTN = 8,         /* paged GQA decode attention, one (partition, kv head) per task */
  ETXB_BODY_ATTN_REDUCE = 9,  /* merge of the partitions of one q head */
  ETXB_BODY_SPLITK_PART = 10, /* demo: partial sums of a split-K reduction (etx/operators/splitk_sum.py) */
  ETXB_BODY_SPLITK_SUM = 11,
  ETXB_BODY_ATTN_FUSED = 12,  /* prep + split-KV attention + merge by the last task to finish, one phase (general and grouped form) */
  /* batched decode (several sequences per step; the reference's column batching, etx/ops/gemv.py:40-73, and request batching,
   * examples/vllm_llm/model.py:194-211): tensor-core tiles that read a weight row once for up to 8 tokens per pass */
  ETXB_BODY_NORM_COL = 13,    /* residual add (+ expert combine in ascending expert id) + RMSNorm of one column */
  ETXB_BODY_GEMV_NB = 14,     /* dsl_gemv with nb activation columns (dsl_gemv_rows_nb, etx/ops/gemv.py:176-289) */
  ETXB_BODY_ROUTE = 15,       /* softmax top-k of every column + per-expert token lists */
  ETXB_BODY_MOE_UP_G = 16,    /* expert-grouped gate+up: an expert's rows read once for all the tokens that selected it */
  ETXB_BODY_MOE_DOWN_G = 17,  /* expert-grouped down, scaled by the routing weight */
  ETXB_BODY_PROLOGUE_NB = 18, /* vl_prologue for column c of a batch */
  ETXB_BODY_ARGMAX_NB = 19,   /* vl_argmax for column c of a batch */
  /* the same three batched grids on the Blackwell tensor cores: tcgen05.mma, weights through TMA tensor copies, fp32 accumulators
   * in tensor memory (the library builds the tensor maps when the plan is bound) */
  ETXB_BODY_GEMV_TC = 20,
  ETXB_BODY_MOE_UP_TC = 21,
  ETXB_BODY_MOE_DOWN_TC = 22,
  ETXB_BODY_MLA_ATTN = 23,    /* absorbed multi-head latent attention of one head over the whole context (DeepSeek-V2 family) */
  ETXB_BODY_COUNT = 24
};

/* The per-step scalars and buffers of the prologue / argmax tiles: field for field the reference's VlParams
 * (examples/vllm_llm/vl_tiles.hip:13-24).  `tok` is the step index t: the prologue embeds token_in[t]; argmax
 * writes token_out[t] and, when write_next, token_in[t + 1], so a greedy run needs no device->host copy per token. */
typedef struct etxb_step_params {
  int32_t tok, pos, write_next, H, V, nrep;
  const void* embed;       /* bf16 [V][H] */
  void* resid;             /* bf16 [H] */
  int64_t* positions;      /* [1] */
  int32_t* seq_lens;       /* [1] */
  int64_t* slot_mapping;   /* [1] */
  const void* logits;      /* bf16 [V] */
  int32_t* token_in;       /* [steps + 2] */
  int32_t* token_out;      /* [steps + 1] */
  uint64_t* token_time;    /* [2 * (steps + 1)] globaltimer ns at prologue / argmax, may be null */
} etxb_step_params;

typedef struct etxb_status_t {
  int32_t ctrl;            /* bit0 host abort seen, bit1 wait deadline passed, bit2 bad task table entry */
  int32_t stuck_task;      /* task index (queue order) that gave up, -1 if none */
  int32_t stuck_event;     /* event word it waited for */
  int32_t stuck_value;     /* counter value seen */
  int32_t stuck_target;    /* value it needed */
  int32_t tasks_run;       /* tasks completed in the last step (only counted when tracing is on) */
  uint32_t epoch;          /* steps launched so far */
  float last_ms;           /* device time of the last etxb_step / etxb_wait, CUDA events */
  int32_t kernel_variant;  /* the kernel the library picked for this plan.  0: the full kernel; 1..4: the lean decode kernel (grouped
                              attention with 1, 2, 4, 8 q heads per task); 10: the lean decode kernel of a latent-attention model;
                              11: the kernel of a batched step on the tensor cores.  Option "full_kernel" = 1 forces 0.  (A sharded
                              session runs its sharded counterpart of 0..4, and that of 0 for a plan that would get 10 or 11.) */
} etxb_status_t;

typedef struct etxb_device_info_t {
  int32_t sm_count, smem_per_block_optin, l2_bytes, cc_major, cc_minor;
  int32_t workers;         /* persistent CTAs the kernel will use (one per SM) */
  int32_t threads;         /* threads per CTA */
  int32_t smem_bytes;      /* dynamic shared memory per CTA */
  uint64_t hbm_bytes;
} etxb_device_info_t;

typedef struct etxb_session etxb_session;

int32_t etxb_version(void);
const char* etxb_last_error(void);   /* thread-local text of the last failure */
int32_t etxb_device_info(int device, etxb_device_info_t* out);

/* plan_blob: the serialized plan (layout in etx-megakernel_b200/csrc/etxb_abi.h, written by passes/plan.py).
 * The blob is copied; the caller may free it. */
int32_t etxb_create(const void* plan_blob, size_t bytes, int device, etxb_session** out);
/* Give a named plan tensor its device address.  The caller keeps ownership and must keep it alive. */
int32_t etxb_bind(etxb_session* s, const char* name, void* dev_ptr, size_t bytes);
int32_t etxb_set_step(etxb_session* s, const etxb_step_params* p);
/* Options: "timeout_ms" (device wait deadline), "trace" (0/1: per-task stamps + execution counts), "full_kernel" (0/1: run
 * the kernel that holds every tile even when the plan qualifies for a smaller one; see etxb_status_t.kernel_variant). */
int32_t etxb_set_option(etxb_session* s, const char* key, int64_t value);
/* Sessions may share device buffers when their steps follow one another (one stream, or synchronised in between): what a step leaves in scratch
 * memory -- words, partial results -- is never taken for another step's. */
int32_t etxb_launch(etxb_session* s, void* cuda_stream);
/* The unfused baseline: the same step as one kernel launch PER GRID, in plan order on one stream (what the reference
 * builds with kernel.py:645-681 and runs with host.h:440-457 to state the gain of the single launch).  Same results;
 * refused (ETXB_E_UNSUPPORTED) when a grid waits for a grid that comes later in the plan. */
int32_t etxb_launch_unfused(etxb_session* s, void* cuda_stream);
int32_t etxb_wait(etxb_session* s, double timeout_s);

int32_t etxb_step(etxb_session* s, void* cuda_stream, double timeout_s);
int32_t etxb_status(etxb_session* s, etxb_status_t* out);

/* ---- sharded model: one rank (process + GPU) per shard, partial rows exchanged inside the kernel ------------------
 * The reference shards a program over devices with device-scoped events and multi-device plans
 * (etx/passes/plan.py:58-86 device_of_task, etx/runtime/include/etx/host.h:79-210 one event region per device); here
 * every rank runs the SAME single-device plan on its shard of the weights and the ranks meet at the row-parallel grids
 * the plan marks as exchanged (o_proj, MoE / MLP down).  A task of such a grid publishes the bf16 rows it wrote as
 * FLAGGED WORDS -- 4 bytes: the value in the low half, a 16-bit flag derived from the step in the high half -- into
 * row `rank` of the grid's [n_ranks][M] block in EVERY rank's exchange region: plain 4-byte stores, over NVLink for
 * the peers.  A store of 4 bytes is atomic, so value and flag arrive together: no fence, no remote counter, no
 * collective call.  The norm fold that follows (mode bit 0x1000, R = n_ranks) reads the block in its own rank's
 * memory, re-reads a word until its flag is this step's (bounded by the step's deadline like every wait), and adds
 * the ranks' rows in rank order, so every rank computes bit-identical hidden states.
 *
 * A region is one device allocation holding the blocks at offsets the caller chooses -- the same on every rank (the
 * argument blocks name them in `rows`).  etxb_exchange_alloc zeroes it and exports a 64-byte inter-process handle;
 * the caller passes the handles around (any transport) and opens the peers' with etxb_exchange_open.
 * etxb_set_exchange (once, before the first step) records this rank's region and the peers' mappings (peer_bases[r]
 * for r != rank; entry `rank` is ignored).  All ranks must run the same steps; a rank whose peers stop publishing
 * returns ETXB_E_TIMEOUT at its deadline.  Every rank must have finished its last step before any rank frees or
 * closes a region (a running peer still stores into it).  etxb_launch_unfused is refused on a sharded session, and
 * etxb_launch on a rank's plan that has no exchange set.
 * lm_head split by vocabulary: each rank's step parameters name its own V / n_ranks logits; after etxb_set_exchange,
 * etxb_set_option(s, "exchange_argmax_offset", off) names n_ranks x 16 bytes of every region where the argmax tile
 * exchanges the ranks' (maximum, global index) pairs as 8-byte (payload, step flag) stores and picks the same token
 * on every rank. */
#define ETXB_IPC_HANDLE_BYTES 64
int32_t etxb_exchange_alloc(int device, size_t bytes, void** dev_ptr, unsigned char* handle /*[64]*/);
int32_t etxb_exchange_free(int device, void* dev_ptr);
int32_t etxb_exchange_open(int device, const unsigned char* handle /*[64]*/, void** peer_ptr);
int32_t etxb_exchange_close(int device, void* peer_ptr);
int32_t etxb_set_exchange(etxb_session* s, int32_t rank, int32_t n_ranks, void* local_base, size_t bytes, void* const* peer_bases);
/* Copies 8 x uint64 per task of the last traced step: {taken, deps ready, body done, worker, 4 in-body marks}
 * (globaltimer ns; a mark a tile did not set is 0). */
int32_t etxb_trace(etxb_session* s, void* host_buf, size_t bytes);
int32_t etxb_exec_counts(etxb_session* s, int32_t* host_buf, size_t count);
int32_t etxb_destroy(etxb_session* s);

/* Greedy decode with HOST buffers: token ids come from and go back to host memory every step.  One sequence: the step's prologue
 * reads its 4-byte token from pinned host memory and its argmax writes the next one there, and the host launches the following step when
 * it sees that one (a step that fails ends the call with its error; the tokens of the steps before it are in tokens_out, and the
 * session can be used again).  Plans of several columns: a 4-byte copy each way around every step.  tokens_in[n_in] are
 * fed first (teacher-forced); generation continues greedily until n_total steps ran.  tokens_out[n_total] receives
 * the argmax of every step.  start_pos is the position of tokens_in[0]. */
int32_t etxb_decode_host(etxb_session* s, const int32_t* tokens_in, int32_t n_in, int32_t n_total,
                         int32_t start_pos, int32_t* tokens_out, float* step_ms /* may be null */);

/* Stand-alone tile launches (tests, micro-benchmarks).  `argblock` is host memory holding the tile's argument block
 * (device pointers inside); ntasks tasks of the tile run on the persistent grid, task index = blockIdx-style `blk`.
 * form: ETXB_BODY_*.  The call is asynchronous on `cuda_stream`. */
int32_t etxb_op_launch(int device, int32_t body, const void* argblock, size_t bytes, int32_t ntasks,
                       const etxb_step_params* step /* may be null */, void* cuda_stream);

/* The fused attention phase with NO device allocation: its partial-result scratch lives in a fixed-size static
 * device array inside the library (about 2.1 MiB, held by every GPU that loads the library until the process exits).
 * No counterpart in the reference.  For callers that cannot allocate when they need attention (a plug-in that only
 * gets the host's buffers, a serving loop that pre-sized its pools, a caller whose free memory all went to the KV
 * cache).  `argblock`: an attn_fused block (etx-megakernel_b200/csrc/etxb_abi.h: etxb_attnf_args); its four scratch
 * pointers are ignored.  Limits: NH <= 64, max_parts <= 64 (context <= 2048), HD <= 128, else ETXB_E_UNSUPPORTED.
 * The first call on a device does the one-time set-up (symbol address, shared-memory limit): make it before any
 * stream capture.  All calls share the array; calls that overlap on the GPU race on it.  Asynchronous on the stream. */
int32_t etxb_attn_fused_static(int device, const void* argblock, size_t bytes, void* cuda_stream);

/* ---- several answers to one prompt --------------------------------------------------------------------------------
 * Three operators beside the step: tokens drawn from its logits, pages of its KV cache shared by several sequences, and decode attention that reads
 * what they share once.  They own nothing and keep nothing between calls: all memory is the caller's, a call is asynchronous on its stream (0: the
 * default stream), may be captured into a graph, and runs on `device` whatever device is current.  `bytes` = sizeof of the argument structure. */
enum { ETXB_BF16 = 0, ETXB_F16 = 1, ETXB_F32 = 2 };

/* One token per row of logits.  The live tokens of a row (neither -inf nor NaN) in the order "larger logit first, equal ones by index", token r
 * weighted w_r = exp((l_r - l_0) / temperature): top-k keeps the first k (k < 1: all), top-p of those the ones with less than p times their sum before
 * them (p not below 1: all), min-p the ones with w_r >= min_p (not above 0: all); at least one is kept.  Drawn is the first token whose inclusive
 * sum exceeds u times the sum of the kept ones.  temperature not above 0: the first of the order.  u is taken as within [0, 1 - 2^-24].  A row without a
 * live token: token -1, log-probability -inf, kept 0.
 * Weights are 64-bit numbers; 16-bit logits are counted value by value and summed in the order of the values, those of 32 bits are summed as integers in steps of
 * 2^-43 of the largest or finer: the outcome depends on no order of execution. */
#define ETXB_SAMPLE_MAX_V 524288
typedef struct etxb_sample_args {
  const void* logits;          /* [rows][V], row_stride elements apart */
  const float* u;              /* [rows] */
  const float* temperature;    /* [rows], or null: temperature_all for every row; the same for the next three */
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;             /* [rows] */
  int32_t* next;               /* [rows], the tokens once more, 0 for -1 (the next step's input), may be null */
  float* logprobs;             /* [rows] log-probability of the token among the kept ones, may be null */
  int32_t* kept;               /* [rows] number of tokens kept, may be null */
  int64_t row_stride;
  int32_t rows, V, dtype;      /* dtype: ETXB_BF16, ETXB_F16, ETXB_F32 */
  int32_t top_k_all;
  float temperature_all, top_p_all, min_p_all;
  int32_t reserved;            /* 0 */
} etxb_sample_args;
int32_t etxb_sample(int device, const etxb_sample_args* args, size_t bytes, void* cuda_stream);

/* Pages of a paged KV cache.  One call copies pages (of all layers and tensors: keys, values) and brings block tables up to date; the lists are host
 * memory, are checked (ETXB_E_ARG) and copied before the call returns, and the device needs none of its own.
 *   copies    page dst_ids[i] := page src_ids[i] of every tensor and layer.  Within one pool no page is both read and written; no page is written twice.
 *             Pages of different tensors do not overlap (they may lie between each other's: keys and values in one allocation).
 *   set       tables[set_rows[i]][set_cols[i]] := set_pages[i]
 *   share     the first `shared` entries of each of share_rows := those of row share_from
 *   remap     in the first remap_entries[i] entries of row remap_rows[i], a page that is a source of the copies gets the number it was copied to (a call
 *             without set and share) */
#define ETXB_PAGES_MAX_TENSORS 4
typedef struct etxb_page_tensor {
  const void* src; void* dst;                             /* the pools: page p of layer l lies at base + l * layer + p * page (bytes, multiples of 16), a layer behind the pages of the last */
  int64_t src_layer, src_page, dst_layer, dst_page;
  int64_t page_bytes;
} etxb_page_tensor;
typedef struct etxb_pages_args {
  etxb_page_tensor t[ETXB_PAGES_MAX_TENSORS];
  int32_t n_tensors, layers, src_pages, dst_pages;
  const int32_t* src_ids; const int32_t* dst_ids;         /* [n_copy] */
  int32_t* tables; int64_t table_stride;                  /* device memory: [table_rows][table_width], rows table_stride entries apart */
  const int32_t* set_rows; const int32_t* set_cols; const int32_t* set_pages;   /* [n_set] */
  const int32_t* share_rows;                              /* [n_share] */
  const int32_t* remap_rows; const int32_t* remap_entries;/* [n_remap] */
  int32_t n_copy, table_rows, table_width, n_set, n_share, share_from, shared, n_remap;
} etxb_pages_args;
int32_t etxb_pages_update(int device, const etxb_pages_args* args, size_t bytes, void* cuda_stream);

/* A pool: which pages are whose.  A sequence is a row of the tables with a length in positions; its pages are given out lowest first.  Forked sequences
 * share the full pages of what they have in common, and the last, partly filled one is copied for each; a shared page is never written, since only full
 * pages are shared.  The books are the host's; what changes on the device (tables, copied pages) goes through one etxb_pages_update on the call's stream.
 * A call that fails changes nothing (ETXB_E_ARG; ETXB_E_FULL: no free pages or rows).  Calls on one pool exclude one another; none is captured into a graph.
 *   create   `layout`: t[].dst and its strides, n_tensors, layers, dst_pages, tables, table_stride, table_rows, table_width (the rest is ignored).
 *            update: what carries the changes out, null: etxb_pages_update (a host without the device gives its own)
 *   open     a new sequence with pages for `length` positions
 *   extend   pages up to lengths[i] positions for rows[i] (never fewer than it has; each row once)
 *   fork     n sequences that continue `row` from `length` positions on (-1: all of them), which are written by then; rows: [n], theirs
 *   close    the sequences end: pages that nobody else holds are free (contents and table entries stay as they are)
 *   compact  moves pages until the ones in use are the lowest, the highest into the lowest hole first; moved: how many, may be null
 *   row      *length = -1 for a row without a sequence; pages: [capacity], its first pages; n: how many it has.  Pointers may be null
 *   free     free pages */
typedef struct etxb_pool etxb_pool;
typedef int32_t (*etxb_pages_fn)(int device, const etxb_pages_args* args, size_t bytes, void* cuda_stream);
int32_t etxb_pool_create(int device, const etxb_pages_args* layout, size_t bytes, int32_t page_len, etxb_pages_fn update, etxb_pool** out);
int32_t etxb_pool_destroy(etxb_pool* pool);
int32_t etxb_pool_open(etxb_pool* pool, int32_t length, int32_t* row, void* cuda_stream);
int32_t etxb_pool_extend(etxb_pool* pool, const int32_t* rows, const int32_t* lengths, int32_t n, void* cuda_stream);
int32_t etxb_pool_fork(etxb_pool* pool, int32_t row, int32_t n, int32_t length, int32_t* rows, void* cuda_stream);
int32_t etxb_pool_close(etxb_pool* pool, const int32_t* rows, int32_t n);
int32_t etxb_pool_compact(etxb_pool* pool, int32_t* moved, void* cuda_stream);
int32_t etxb_pool_row(etxb_pool* pool, int32_t row, int32_t* length, int32_t* pages, int32_t capacity, int32_t* n);
int32_t etxb_pool_free(etxb_pool* pool, int32_t* pages);

/* Decode attention of one layer for sequences that share prefixes: group g has a block table and a length of the positions its sequences have in
 * common, each sequence a table and a length of its own ones behind them (the new position's key and value are in the cache already, and counted).
 * Caches as in the step: keys [pages][NKV][HD / 8][16][8], values [pages][NKV][HD][16], bf16.  The keys and values of a prefix are read once for all
 * sequences of its group.  A sequence without a position has the output 0.
 * A page outside the cache or a length outside its table makes the outputs of the sequences it concerns NaN and sets a bit of *status (which no call
 * clears); nothing outside the buffers is read. */
#define ETXB_SHARED_MAX_SEQS 1024
enum { ETXB_SHARED_BAD_PAGE = 1, ETXB_SHARED_BAD_LENGTH = 2, ETXB_SHARED_GAVE_UP = 4 };   /* 4: a wait inside the kernel ran past two seconds */
typedef struct etxb_attn_shared_args {
  const void* q; void* out;                               /* bf16 [seqs][NH][HD], q_stride / out_stride elements between sequences */
  const void* kc; const void* vc;                         /* k_stride / v_stride elements between pages */
  const int32_t* tables; const int32_t* lens;             /* device: [seqs][table_width] (rows table_stride apart), [seqs] */
  const int32_t* prefix_tables; const int32_t* prefix_lens;   /* device: [groups][prefix_width] (rows prefix_stride apart), [groups] */
  const int32_t* group_first;                             /* host: [groups + 1], the sequences of group g are group_first[g] .. group_first[g + 1] - 1 */
  int32_t* status;                                        /* device, may be null */
  void* work; size_t work_bytes;                          /* device memory of the call alone, as much as etxb_attn_shared_work says */
  int64_t q_stride, out_stride, k_stride, v_stride, table_stride, prefix_stride;
  int32_t seqs, groups, NH, NKV, HD, pages, table_width, prefix_width;
  float scale;
  int32_t reserved;
} etxb_attn_shared_args;
int32_t etxb_attn_shared(int device, const etxb_attn_shared_args* args, size_t bytes, void* cuda_stream);
/* The bytes of `work` a call with these sizes needs (of the pointers only group_first is looked at). */
int32_t etxb_attn_shared_work(int device, const etxb_attn_shared_args* args, size_t bytes, size_t* work_bytes);

#ifdef __cplusplus
}
#endif
#endif
