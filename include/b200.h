/* b200.h — C ABI of the Blackwell (sm_100a) execution backend for arrayjit routines.
 *
 * This is the surface an OCaml `Lowered_backend` implementation binds through ctypes/C
 * stubs.  Each entry point names the reference interface member it serves (paths are
 * relative to the reference project).  Conventions:
 *   - every function returns 0 on success; a negative value is one of B200_E_*, a
 *     positive value is the CUresult / nvrtcResult / ncclResult_t that failed;
 *   - b200_last_error() returns a thread-local message for the last failure on the
 *     calling thread;
 *   - all device work is asynchronous on the device's single stream, like the cuda
 *     backend's (arrayjit/lib/cuda_backend.ml:215-238); host buffers passed to the copy
 *     functions must stay valid until the next b200_await / b200_event_sync;
 *   - there is no CPU fallback: with no usable driver or GPU every compute entry point
 *     fails with B200_E_NO_DEVICE.
 */
#ifndef B200_H
#define B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B200_E_INVALID (-1)     /* bad argument (Invalid_argument on the OCaml side) */
#define B200_E_NO_DEVICE (-2)   /* driver, NVRTC or GPU unavailable */
#define B200_E_PARSE (-3)       /* malformed b200ir */
#define B200_E_UNSUPPORTED (-4) /* valid IR that this backend cannot run */
#define B200_E_USER (-5)        /* Utils.User_error: bad static index, missing binding, ... */
#define B200_E_DEVICE (-6)      /* a kernel reported a device-side status (bounded wait expired) */
#define B200_E_NO_SPACE (-7)    /* a fixed-capacity entry point was given a larger problem */

typedef struct b200_dev b200_dev;
typedef struct b200_event b200_event;
typedef struct b200_code b200_code;
typedef struct b200_routine b200_routine;
typedef struct b200_comm b200_comm;

const char* b200_last_error(void);
const char* b200_version(void);

/* ---- devices: Backend_device_common.{num_devices, get_device, get_name, static_properties}
 *      (arrayjit/lib/backend_intf.ml:218-266; cuda: arrayjit/lib/cuda_backend.ml:215-238) */
int b200_init(void);
int b200_num_devices(int* out);
int b200_device_open(int ordinal, b200_dev** out);     /* memoised per ordinal */
int b200_device_props(b200_dev* dev, char* json, size_t cap);

/* ---- pools: Slab_alloc.{alloc_pool, free_pool, memset_zero}
 *      (arrayjit/lib/backend_intf.ml:22-37; cuda: arrayjit/lib/cuda_backend.ml:60-94).
 *      Allocating an id that exists frees the old slab first. */
int b200_pool_alloc(b200_dev* dev, int pool_id, size_t bytes, size_t alignment);
int b200_pool_free(b200_dev* dev, int pool_id);
int b200_pool_memset0(b200_dev* dev, int pool_id, size_t offset, size_t bytes);
int b200_pool_address(b200_dev* dev, int pool_id, uint64_t* device_ptr, size_t* bytes);

/* ---- copies: No_buffer_retrieval_or_syncing.{from_host, to_host, device_to_device}
 *      (arrayjit/lib/backend_impl.ml:292-315; cuda: arrayjit/lib/cuda_backend.ml:262-314) */
int b200_h2d(b200_dev* dev, int pool_id, size_t offset, const void* src, size_t bytes);
int b200_d2h(b200_dev* dev, int pool_id, size_t offset, void* dst, size_t bytes);
int b200_d2d(b200_dev* dst_dev, int dst_pool, size_t dst_offset, b200_dev* src_dev, int src_pool,
             size_t src_offset, size_t bytes);
/* `~into_merge_buffer:Copy`: grows the destination's merge slab (reserved pool id 0,
 * arrayjit/lib/backend_intf.ml:131-132) and copies the source node into it. */
int b200_merge_copy(b200_dev* dst_dev, b200_dev* src_dev, int src_pool, size_t src_offset, size_t bytes);
/* page-locked host staging memory for from_host / to_host */
int b200_host_alloc(size_t bytes, void** out);
int b200_host_free(void* p);

/* ---- events and stream: Device.{all_work, is_done, sync, will_wait_for, await, is_idle}
 *      (arrayjit/lib/backend_intf.ml:97-126; cuda: arrayjit/lib/cuda_backend.ml:107-111,256-260) */
int b200_event_record(b200_dev* dev, b200_event** out);
int b200_event_query(b200_event* ev, int* done);
int b200_event_sync(b200_event* ev);
int b200_event_elapsed_ms(b200_event* start, b200_event* stop, float* ms);
int b200_event_free(b200_event* ev);
int b200_stream_wait(b200_dev* dev, b200_event* ev);
int b200_await(b200_dev* dev);
int b200_is_idle(b200_dev* dev, int* idle);
int b200_stream_handle(b200_dev* dev, uint64_t* custream);
/* Extension (the reference has one stream per device, arrayjit/lib/cuda_backend.ml:215-238): with
 * `on`, b200_h2d copies run on a second stream.  A copy waits for everything queued before it.
 * Work queued after it waits for the copy when it may touch the copied pool: b200_launch waits for
 * the copies into the pools its routine binds (and pool 0), b200_d2h / b200_pool_memset0 for the
 * copies into their pool, every other call for all copies.  Uploading the next batch into a second
 * pool before launching the current step therefore overlaps the two. */
int b200_set_async_uploads(b200_dev* dev, int on);

/* ---- routines: Lowered_backend.{compile, link} (arrayjit/lib/backend_impl.ml:334-367;
 *      cuda: arrayjit/lib/cuda_backend.ml:898-928 compile, :983-1066 link and launch).
 *      b200_compile is device independent.  `options` is a space-separated list of
 *      key=value pairs (gemm, attn, coop, fuse, pairs, splitk, tf32, large_models, bounds, each 0|1, and
 *      gather_mb); NULL for defaults.
 *      gemm: tensor-core contractions; attn: the attention chain (scores, softmax, weights . values,
 *      lib/nn_blocks.ml:222-236) as one kernel; coop: cooperative reductions; fuse: several stages per
 *      launch; pairs: two neighbouring elements per thread with packed 16-bit arithmetic; splitk:
 *      few-tile fp32 accumulations split over K (atomic adds, order not fixed); tf32: contractions of
 *      single-precision operands on the tensor cores as tf32 (10-bit mantissas, fp32 sums; convolutions
 *      and small, narrow or unaligned products as two such parts an operand, which keeps single
 *      precision; with tf32=0 all stay on the exact generic kernels); bounds: a range-checked build of the generated
 *      kernels (generic kernels only): an access outside a node is skipped and the next wait returns
 *      B200_E_DEVICE naming the node id and the element; gather_mb: the most megabytes of the
 *      routine's device scratch a contraction may take for the copy of an operand that has to be gathered
 *      or for the windows of an input gradient, 2048 by default (windows: 1024 at most): contractions that
 *      would take more run on the generic kernels, and so do, at b200_link, those whose copies the device
 *      has no room for. */
int b200_compile(const char* name, const char* b200ir, size_t len, const char* options, b200_code** out);
int b200_code_info(b200_code* code, char* json, size_t cap);
int b200_code_source(b200_code* code, int stage, char* buf, size_t cap, size_t* needed);
int b200_code_free(b200_code* code);

typedef struct {
  int32_t tn_id;   /* tensor node id of the routine */
  int32_t pool_id; /* Backend_intf.buffer_loc: pool + byte offset */
  uint64_t offset;
} b200_binding;

/* Bindings need only be aligned to the node's element size, which is all the reference's
 * allocator promises (plan_pool_segments, arrayjit/lib/backends.ml:22-51; an offset that is not a
 * multiple of the element size is B200_E_INVALID).  Stages whose compiled form wants more (8-byte
 * pairs, 16-byte TMA operand bases) are re-planned for the addresses at hand; b200_routine_info
 * reports the plan that runs. */
int b200_link(b200_dev* dev, b200_code* code, const b200_binding* bindings, int n_bindings,
              b200_routine** out);
int b200_routine_info(b200_routine* r, char* json, size_t cap);   /* like b200_code_info, for the linked plan */
/* Runs the routine once on the device stream.  static_idx has one value per static symbol
 * of the routine, in declaration order; a negative or out-of-range value is B200_E_USER
 * (cuda: arrayjit/lib/cuda_backend.ml:1015-1030). */
int b200_launch(b200_routine* r, const int64_t* static_idx, int n_static);
/* Replays the routine's launches as one captured graph from its second run on (the first is launched
 * directly).  Routines of up to four launches, all of them kernels (a lone clear of a node is none; clears that
 * share a launch are one), and those whose only kernel takes the static indices as an argument, are launched
 * directly all the same: a graph would only add its own time. */
int b200_routine_use_graph(b200_routine* r, int enable);
int b200_routine_launch_count(b200_routine* r, int64_t* kernels_per_run);
/* Per-stage device timing (CUDA events around every launch of the next runs; disables graph
 * replay while on).  A stage that runs in the launch of another (its note says of which) has 0 runs: its
 * time is part of that stage's.  No counterpart in the reference, which has no profiler hooks. */
int b200_routine_profile(b200_routine* r, int enable);
int b200_routine_stage_time(b200_routine* r, int stage, float* total_ms, int* runs);
int b200_routine_free(b200_routine* r);

/* ---- observability: get_used_memory, get_debug_info (arrayjit/lib/cuda_backend.ml:123-126,1114-1118) */
int b200_used_memory(b200_dev* dev, size_t* bytes);
int b200_debug_info(b200_dev* dev, char* json, size_t cap);

/* ---- data parallel exchange.  Replaces the owner-reduce + broadcast of
 *      Parallel.data_parallel's grad_sync (lib/parallel.ml:247-304) by one NCCL allreduce
 *      per contiguous gradient range.  One communicator rank per process and device. */
int b200_comm_unique_id(char* id128);                                      /* 128 bytes */
int b200_comm_init_rank(b200_dev* dev, int n_ranks, int rank, const char* id128, b200_comm** out);
/* One process that holds every shard, as the reference's data_parallel does
 * (lib/parallel.ml:166-208): all communicators at once, and one range per device reduced as one
 * NCCL group (a thread that drives several devices must group its calls). */
int b200_comm_init_all(int n_devices, b200_dev* const* devs, b200_comm** out);
int b200_allreduce_all(int n, b200_comm* const* comms, const int* pool_ids, const size_t* offsets, size_t count,
                       int dtype, int op);
#define B200_SUM 0
#define B200_AVG 1
#define B200_F32 0
#define B200_BF16 1
int b200_allreduce(b200_comm* comm, int pool_id, size_t offset, size_t count, int dtype, int op);
/* Overlap of the exchange with the backward pass.  The ranges (at most a few buckets, e.g. the
 * gradients of the last layers and those of the first) are reduced on the communicator's own
 * stream, each as soon as the routine's last stage that writes into it has been queued, while the
 * remaining stages run; the compute stream waits for all of them at the end of the routine, so the
 * optimizer step that follows sees reduced gradients.  Replaces the gradient-by-gradient
 * owner-reduce that follows the whole backward pass in lib/parallel.ml:292-304.  n = 0 detaches. */
int b200_routine_overlap_allreduce(b200_routine* r, b200_comm* comm, int n, const int* pool_ids,
                                   const size_t* offsets, const size_t* counts, int dtype, int op);
/* With a timeout (> 0 ms) b200_await polls instead of blocking: an asynchronous NCCL error
 * (ncclCommGetAsyncError), or a stream still busy after the timeout (a rank that never arrived),
 * aborts the communicator (ncclCommAbort) and is returned as an error; the device stays usable,
 * the communicator does not.  No counterpart in the reference, whose shards share one process. */
int b200_comm_set_timeout(b200_comm* comm, long long timeout_ms);
int b200_comm_free(b200_comm* comm);

/* ---- allocation-free reduction.  No counterpart in the reference: added for callers that may
 *      not reach the device allocator while they run (inside a stream capture, in a serving
 *      loop that cannot afford cudaMalloc's implicit synchronisation, or under a memory budget
 *      that was handed out up front).  Writes sum(in[0..count)) as one float at the output
 *      location, in stream order on the device's stream, with its scratch in a 4 KiB array that
 *      is part of the library's device image.  count <= 2^26, else B200_E_NO_SPACE; count 0
 *      writes 0.0f.  Both offsets must be multiples of 4, else B200_E_INVALID (checked on the
 *      host: nothing is launched).  A positive return value here is a cudaError_t.  The first
 *      call on a device resolves the array's address: make it before any stream capture.
 *      Calls that overlap on the GPU race on the shared array; stream-ordered calls do not. */
int b200_sum_f32_static(b200_dev* dev, int in_pool, size_t in_offset, size_t count, int out_pool,
                        size_t out_offset);

/* ---- operators: what a decoder layer (lib/nn_blocks.ml:209-285) does between its contractions, as kernels of their own
 *      beside the fused stages that b200_compile finds in a routine.  No counterpart in the reference, which spells them as
 *      assignments.  An operator is linked to nodes once, like a routine -- arguments are checked, the kernels and the
 *      workspace chosen -- and keeps their addresses: free it before their pools.  A run queues kernels on the device's
 *      stream, in order with routines and copies; it allocates nothing, waits for nothing and may be captured into a CUDA graph.
 *      Every linked operator has a workspace of its own; runs of ONE operator, and of the graphs that hold it, may not overlap
 *      on the GPU, and a graph that holds it is released before the operator.
 *      Nodes are row-major and need only be aligned to their element size (16 bytes are faster).  An output may not overlap
 *      another operand, but where it says so.  Sums, statistics and softmax are held in single precision or better; 16-bit outputs
 *      are rounded once.  The same inputs give the same bits. */
typedef struct b200_operator b200_operator;
#define B200_F16 2               /* beside B200_F32 and B200_BF16 */
typedef struct {
  int32_t pool_id;               /* negative: not given */
  uint64_t offset;
} b200_operand;
int b200_operator_run(b200_operator* op);
int b200_operator_free(b200_operator* op);   /* waits for the device's stream */

/* Layer norm of rows of n elements (1 <= n <= 2^30) with a scale and a shift:
 *   h = x + residual;  mean = sum(h) / n;  rstd = 1 / sqrt(sum((h - mean)^2) / n + eps);  y = (h - mean) * rstd * gamma + beta
 * and, of the gradient dy of y, with u = (h - mean) * rstd and g = dy * gamma,
 *   dx = rstd * (g - sum(g) / n - u * sum(g * u) / n) + d_total;  dgamma = sum_rows(dy * u);  dbeta = sum_rows(dy).
 * (lib/nn_blocks.ml:251-258 divides the distance from the SUM by n; this is the usual norm.) */
typedef struct {
  int64_t rows, n;
  int32_t dtype;                 /* x, residual, y, total, dy, d_total, dx */
  int32_t weight_dtype;          /* gamma, beta: B200_F32 or `dtype` */
  float eps;
  b200_operand x;                /* gradient: h, that is `total` where there was a residual */
  b200_operand residual;         /* forward, optional */
  b200_operand gamma, beta;      /* [n], optional: 1 and 0 */
  b200_operand y;                /* forward */
  b200_operand total;            /* forward, optional, with a residual: h */
  b200_operand mean, rstd;       /* [rows] single: written by the forward pass (optional), read by the gradient */
  b200_operand dy, d_total;      /* gradient; d_total (optional): what reaches h from elsewhere */
  b200_operand dx;               /* gradient: of x, and of the residual as well */
  b200_operand dgamma, dbeta;    /* gradient, [n] single, each optional */
} b200_layer_norm;
int b200_layer_norm_link(b200_dev* dev, const b200_layer_norm* spec, b200_operator** out);
int b200_layer_norm_grad_link(b200_dev* dev, const b200_layer_norm* spec, b200_operator** out);

/* Rotary positions: of the first 2 * pairs elements of every head, pair i turns by the angle position * frequency[i] and is
 * multiplied by `magnitude`; the head's other elements are copied.  Pairs are (i, i + pairs) or, interleaved, (2i, 2i + 1).
 * x is [batch, seq, heads, d]; y has the same shape and may be x itself.  A second tensor (keys beside queries, with heads of its own) may
 * go with the first.  inverse: the angle negated, which is the gradient's form (dy in the place of x).  Angles are kept in 64
 * bits of a turn: far positions lose nothing. */
typedef struct {
  int64_t batch, seq;
  int32_t heads[2];              /* heads[1] 0: one tensor */
  int32_t d;
  int32_t pairs;                 /* 2 * pairs <= d */
  int32_t dtype;
  int32_t interleaved, inverse;
  float magnitude;
  const double* frequencies;     /* host, [pairs]: radians per position; copied at link */
  int64_t first_position;        /* of index 0 in seq, where no positions are given */
  b200_operand positions;        /* int32 [batch, seq], optional */
  b200_operand x[2], y[2];
} b200_rotary;
int b200_rotary_link(b200_dev* dev, const b200_rotary* spec, b200_operator** out);

/* Attention of `queries` rows over `keys` keys (the chain of lib/nn_blocks.ml:222-236 at any length, nothing of it kept):
 *   x_rj = scale * <q_r, k_j>;  c = cap * tanh(x / cap) (cap > 0) or x;  s = c - slope[h] * |position_r - j|
 *   out_r = sum_j softmax_j(s_rj) v_j over the keys j that r sees, lse_r = log(sum_j exp(s_rj));  no key: 0 and -infinity
 * q, out are [batch, queries, heads, d], k, v [batch, keys, kv_heads, d] (each key head serves heads / kv_heads query heads
 * in a row), 1 <= d <= 128.  Query r of sequence b lies at position len_b - queries + r, where len_b is lengths[b] (taken
 * between 0 and `keys`) or `keys`.  It sees key j if j < len_b, and
 *   B200_MASK_CAUSAL: j <= position;   B200_MASK_PREFIX: j <= position or j < prefix[b];
 *   and, with documents: key_documents[b, j] == query_documents[b, r] >= 0 (a negative document is padding).  Where no documents of
 *   queries are given, a query has the document of the key at its position (and none, like padding, where its position is negative).
 * What lies at a key or a query that is not seen has no influence, whatever it holds, beyond the last bits: with a cap the formula for
 * tanh, and in the gradients of half heads the scale of a row, are chosen for a warp or a tile as a whole.
 * Products: 16-bit heads multiply their own values exactly; weights, and in the gradients the gradients of scores, are rounded to
 * the heads' type once more before they are multiplied (half ones scaled by powers of two, so that small ones keep their bits).
 * Single heads are multiplied as two tf32 parts each, 2^-21 of a product; sums are in single precision.  lse is off by 2^-22 of its size, and
 * the gradients' weights by as much as lse is: scores of thousands cost them bits.
 * The gradient takes out and lse of the forward pass and gives, with p = exp(s - lse),
 *   dv_j = sum_r p_rj d_out_r;  ds_rj = p_rj (<d_out_r, v_j> - <d_out_r, out_r>);  dx = ds (1 - (c / cap)^2)
 *   dq_r = scale * sum_j dx_rj k_j;  dk_j = scale * sum_r dx_rj q_r
 * where a key head's sums run over the query heads it serves.  slopes are constants: they get no gradient. */
#define B200_MASK_NONE 0
#define B200_MASK_CAUSAL 1
#define B200_MASK_PREFIX 2
typedef struct {
  int64_t batch, queries, keys;
  int32_t heads, kv_heads, d;
  int32_t dtype;                 /* q, k, v, out and their gradients */
  int32_t mask;
  float scale, cap;              /* cap 0: none */
  b200_operand q, k, v, out;
  b200_operand lse;              /* [batch, heads, queries] single; optional in the forward pass */
  b200_operand lengths, prefix;  /* int32 [batch] */
  b200_operand query_documents;  /* int32 [batch, queries], optional beside ... */
  b200_operand key_documents;    /* int32 [batch, keys] */
  b200_operand slopes;           /* single [heads] */
  b200_operand d_out, dq, dk, dv;
} b200_attention;
int b200_attention_link(b200_dev* dev, const b200_attention* spec, b200_operator** out);
int b200_attention_grad_link(b200_dev* dev, const b200_attention* spec, b200_operator** out);

/* A cache of keys and one of values in pages, for sequences of different lengths: [pages, kv_heads, page, d] each, of the type `dtype` or in 8
 * bits (B200_E4M3: sign, 4 bits of exponent, 3 of mantissa, 448 the largest, no infinities) with a scale for each page and head, k = k_scale * code.
 * Sequence b's tokens i * page .. (i + 1) * page - 1 lie in page page_table[b, i]; a number outside 0 .. pages - 1 is no page: nothing is written there
 * and nobody sees its tokens (as with pages given back behind a window).  lengths[b] counts a sequence's tokens, the new ones included
 * (negative: 0); tokens behind max_pages pages are not kept.  New tokens are rows of packed nodes: sequence b has rows starts[b] .. starts[b + 1] - 1
 * (numbers taken between 0 and `tokens`, not falling; where they fall, a run may take rows twice or leave them), or, without starts, tokens / batch
 * rows each.  Row i of n lies at position lengths[b] - n + i, and nowhere where that is negative.  Rows of no sequence are left as they were.  The
 * table may name a page more than once, but for those that a call of cache_append writes. */
#define B200_E4M3 3
typedef struct {
  int64_t batch, tokens;
  int64_t pages, max_pages;      /* pages of the cache; of a sequence at most */
  int32_t page;                  /* tokens of a page */
  int32_t kv_heads, d;
  int32_t dtype;                 /* of the cache: that of the new tokens, or B200_E4M3 */
  b200_operand k, v;
  b200_operand k_scale, v_scale; /* single [pages, kv_heads], with B200_E4M3: between 2^-40 and 2^40 */
  b200_operand page_table;       /* int32 [batch, max_pages] */
  b200_operand lengths;          /* int32 [batch] */
  b200_operand starts;           /* int32 [batch + 1], optional */
} b200_cache;

/* New keys and values [tokens, kv_heads, d] go to their slots of the cache.  Keys, and with them queries [tokens, heads, d] if given, turn on the way
 * as b200_rotary does it (pairs 0: they do not), by the token's position or by that of `positions`, and are rounded once to what holds them.
 * 8 bits: a page's scale of a head is 2^e, the least power of two of at least 2^-40 with |x| <= 448 * 2^e for all values that the page has received;
 * where it grows, the codes that the page holds are rounded again (which changes those alone that fall below the normal range).  A page whose
 * first slot is written starts anew.  Values that are undefined, infinite or beyond 448 * 2^40 become the code of an undefined value. */
typedef struct {
  b200_cache cache;              /* k, v and the scales are written */
  int32_t dtype;                 /* of k, v, q, q_out */
  int32_t heads;                 /* of q; 0: no queries */
  int32_t pairs;                 /* 2 * pairs <= d */
  int32_t interleaved;
  float magnitude;
  const double* frequencies;     /* host, [pairs]: radians per position; copied at link */
  b200_operand positions;        /* int32 [tokens], optional: what keys and queries turn by */
  b200_operand k, v;
  b200_operand q, q_out;         /* may be one node */
} b200_cache_append;
int b200_cache_append_link(b200_dev* dev, const b200_cache_append* spec, b200_operator** out);

/* Attention of new tokens over a cache that holds them already (and all before them):
 *   x_rj = scale * <q_r, k_j>;  c = cap * tanh(x / cap) (cap > 0) or x;  s = c - slope[h] * (position_r - j)
 *   out_r = sum_j softmax_j(s_rj) v_j, lse_r = log(sum_j exp(s_rj)) over the tokens j that r sees;  none: 0 and -infinity
 * Row r sees token j <= position_r whose page is there, if the window is 0, j > position_r - window, or j < sinks.
 * q, out are [tokens, heads, d], each key head serves heads / kv_heads query heads in a row, 1 <= d <= 128.
 * What lies at tokens that are not seen, behind the last one in a page among them, has no influence, whatever it holds, beyond the last bits.
 * Products, weights and sums are those of b200_attention; codes of 8 bits are multiplied exactly, beside 16-bit heads with weights of 11 bits. */
typedef struct {
  b200_cache cache;              /* read */
  int32_t dtype;                 /* of q, out */
  int32_t heads;
  float scale, cap;              /* cap 0: none */
  int64_t window, sinks;         /* window 0: none */
  b200_operand q, out;
  b200_operand lse;              /* single [tokens, heads], optional */
  b200_operand slopes;           /* single [heads], optional */
} b200_cache_attention;
int b200_cache_attention_link(b200_dev* dev, const b200_cache_attention* spec, b200_operator** out);

/* Chooses a token for each row of logits x [rows, vocab]:  w_i = exp((x_i - max x) / temperature).  In the order of falling x (of equal ones: of
 * rising i) the first n tokens are kept, n the least of top_k (0 or less: vocab), of the fewest whose w add up to at least top_p times the sum over the
 * first top_k (1 or more: all; at least one), and of the number of w >= min_p (more than 1: 1).  The token is the first kept one, in the order of i, at which
 * the running sum of w exceeds uniform * (the kept sum) (uniform below 0 or undefined: 0; the last kept one where none does).
 * logprob = log(w_token / kept sum).  temperature 0 or less: the first largest, logprob 0.  Undefined logits count as -infinity, which is never chosen; where
 * there are infinite ones, those have w = 1 and the others 0.  A row of nothing else: token -1, logprob -infinity.
 * Every setting is one number for all rows or a node of one a row (there an undefined temperature is 0, an undefined top_p 1, an undefined min_p 0).
 * 1 <= vocab < 2^31. */
typedef struct {
  int64_t rows, vocab;
  int32_t dtype;                 /* of the logits */
  int32_t top_k;
  float temperature, top_p, min_p;
  b200_operand logits;
  b200_operand uniform;          /* single [rows] */
  b200_operand temperatures, top_ps, min_ps;   /* single [rows], each optional, in the place of the number */
  b200_operand top_ks;           /* int32 [rows], optional */
  b200_operand tokens;           /* int32 [rows] */
  b200_operand logprob;          /* single [rows], optional */
} b200_sample;
int b200_sample_link(b200_dev* dev, const b200_sample* spec, b200_operator** out);

#ifdef __cplusplus
}
#endif
#endif /* B200_H */
