/* b200fa -- C ABI of the B200 (sm_100a) FlashAttention library.
 *
 * This is the boundary a host binding (ctypes, cgo, JNI ...) calls. It replaces the launch interface of the
 * reference, `runtime.run(kernel, grid, threads, smem, signature, values, stream, ...)`
 * (reference src/zigfa/_impl/runtime.py:233-259), together with the launch planners that feed it
 * (src/zigfa/_impl/forward.py:118-265, backward.py:314-551, inter_sequence.py:223-562).
 *
 * Rules common to every entry point:
 *  - all tensor pointers are device pointers owned by the caller; unless an entry point says otherwise the
 *    library allocates and frees no device memory;
 *  - a call only enqueues work on `stream` (a cudaStream_t passed as void*) and returns; it never synchronises;
 *  - return value 0 = success, negative = error; b200fa_last_error() returns the message of the calling thread;
 *  - tensors are BF16 with a contiguous last dimension, 16-byte aligned base pointers and strides (in elements)
 *    that are multiples of 8 (reference src/zigfa/_impl/tensors.py:114-127);
 *  - `*_workspace_bytes` functions are pure host functions of the shapes and run without a GPU.
 */
#ifndef B200FA_H_
#define B200FA_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B200FA_OK 0
#define B200FA_ERR_INVALID (-1)   /* bad argument (shape, alignment, head_dim, workspace too small) */
#define B200FA_ERR_CUDA (-2)      /* a CUDA call failed */
#define B200FA_ERR_UNSUPPORTED (-3)

/* Attention problem shared by forward and backward.
 * Fixed length: q (batch, seqlen_q, heads_q, head_dim), k/v (batch, seqlen_k, heads_kv, head_dim), cu_seqlens NULL.
 * Packed (varlen / inter-sequence): q (total_q, heads_q, head_dim), k/v (total_k, heads_kv, head_dim),
 * cu_seqlens_q/k int32 prefix sums of length batch + 1; seqlen_q / seqlen_k are then the row counts of the packed
 * tensors (their shape[0]) and stride[0] is unused.
 * window_left / window_right: -1 = unbounded; causal = (left, 0). Bottom-right aligned
 * (reference tests/reference.py:10-19).
 * Inter-sequence (reference src/zigfa/_impl/ops.py:701-742): visibility_bits (batch, ceil(batch/32)) int32, bit j of
 * row i set = query sequence i sees key sequence j; visibility_bits_t is its transpose, cu_visible_k the prefix sums
 * of visible key tokens per query sequence (both from b200fa_interseq_metadata); window_sizes (2, batch) int32 or NULL.
 * All three NULL = ordinary attention. */
typedef struct b200fa_problem {
  int32_t batch;
  int32_t seqlen_q, seqlen_k;
  int32_t heads_q, heads_kv, head_dim;
  int32_t window_left, window_right;
  float softmax_scale;
  const int32_t* cu_seqlens_q;
  const int32_t* cu_seqlens_k;
  const int32_t* visibility_bits;
  const int32_t* visibility_bits_t;
  const int32_t* cu_visible_k;
  const int32_t* cu_visible_q;
  const int32_t* window_sizes;
} b200fa_problem;

/* Strides in elements: [0] batch, [1] row, [2] head. */
typedef struct b200fa_fwd_args {
  b200fa_problem problem;
  const void* q;
  const void* k;
  const void* v;
  void* out;           /* bf16, shape of q */
  float* softmax_lse;  /* fp32 (batch, heads_q, seqlen_q) or packed (heads_q, total_q); natural log; -inf = no keys */
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
  int64_t lse_stride[2]; /* [0] batch (0 when packed), [1] head; rows are contiguous */
  void* workspace;
  size_t workspace_bytes;
} b200fa_fwd_args;

/* Replaces forward.compute_scratch_shapes (reference src/zigfa/_impl/forward.py:105-115). */
size_t b200fa_fwd_workspace_bytes(const b200fa_problem* problem);
/* Replaces forward.forward (reference src/zigfa/_impl/forward.py:118-265): out = softmax(scale q k^T + mask) v. */
int b200fa_fwd(const b200fa_fwd_args* args, void* stream);

/* Forward attention without a caller workspace (no counterpart in the reference, whose forward always takes the
 * scratch tensors its op layer allocates). Meant for callers that must not allocate device memory around the call:
 * code running under a fixed device-memory plan where every byte is assigned up front, or a host-language binding
 * that owns only the input and output buffers and has no allocator to ask for a workspace. Same arguments and results as b200fa_fwd; `workspace` and
 * `workspace_bytes` are ignored. The work list of a packed batch is kept in a 64 KiB array in device memory owned by
 * the library (held by every GPU that loads it until the process exits). The limit is
 * b200fa_fwd_workspace_bytes(problem) <= 65536, i.e. at most 8192 work-list entries: one entry covers 256 query rows
 * of a sequence at head_dim <= 128 ((total_q + 255 * batch) / 256 <= 8192) and 128 rows at head_dim 256 and 512
 * ((total_q + 127 * batch) / 128 <= 8192); larger batches are rejected with B200FA_ERR_INVALID and a
 * message. (Where the query heads of a group are packed into the rows of a work item -- a power-of-two number of query
 * heads per key head, at most 16 in a packed batch, head_dim <= 128 -- an entry covers 256 / group tokens and
 * b200fa_fwd_workspace_bytes asks for that finer list; a call whose workspace holds only the list with one head per
 * work item, as this entry point's scratch may, runs unpacked (a row's sum of exponentials may then round differently
 * in its last bit; nothing else changes), so the limit above decides.) Fixed-length problems need no scratch and have no such limit. The call itself allocates and frees nothing.
 * The first call on each device looks up the array's device address (a synchronous CUDA runtime query), so make that
 * first call before any stream capture begins. All calls on a device share the one array: each call rewrites every
 * entry it uses before its kernel reads them, nothing needs clearing, but two calls whose kernels can overlap on the
 * GPU (different streams without ordering) race on it -- keep calls to this entry point stream-ordered per device. */
int b200fa_fwd_noalloc(const b200fa_fwd_args* args, void* stream);

typedef struct b200fa_bwd_args {
  b200fa_problem problem;
  const void* q;
  const void* k;
  const void* v;
  const void* out;
  const void* dout;
  const float* softmax_lse;
  void* dq;
  void* dk;
  void* dv;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3], dout_stride[3];
  int64_t dq_stride[3], dk_stride[3], dv_stride[3];
  int64_t lse_stride[2];
  void* workspace;
  size_t workspace_bytes;
} b200fa_bwd_args;

/* Replaces backward.compute_scratch_shapes (reference src/zigfa/_impl/backward.py:141-180). */
size_t b200fa_bwd_workspace_bytes(const b200fa_problem* problem);
/* Replaces backward.backward (reference src/zigfa/_impl/backward.py:314-551): preprocess, dK/dV/dQ main kernel,
 * postprocess. dQ accumulates with floating-point atomics (not deterministic), as in the reference. */
int b200fa_bwd(const b200fa_bwd_args* args, void* stream);

/* Pivot gradients (the backward half of the reference's "softmax fix": zig/fragments.zig:23-30,
 * zig/flash_bwd_sm100.zig:635-645,984-997, zig/flash_bwd_postprocess.zig:150-397). With the setting on, b200fa_bwd
 * treats a key that holds more than 3/4 of the probability of a query row as the pivot of that row: its dS is not formed
 * as P (dP - D), which cancels for P near 1, but as minus the sum of the BF16 dS of the other keys of the row, and the
 * pivot terms of dQ and dK are added by the postprocess kernels. The results of rows without a pivot do not change.
 * The setting is process-wide, read at every b200fa_bwd call; it starts as 1 when the environment variable
 * B200FA_PIVOT_DS is "1" and as 0 otherwise (the pivot path costs the backward main kernel about 16 %; without it the
 * gradients stay within the stated tolerance of the BF16 reference). Returns the previous value; a negative `enabled`
 * only queries. */
int b200fa_set_pivot_ds(int enabled);

/* Measurement hook (no counterpart in the reference): the next b200fa_bwd call of the calling thread records the four
 * cudaEvent_t handles events[0..3] on its stream -- before the preprocess kernel, before the main kernel, after the
 * main kernel, after the postprocess kernel -- so a benchmark can time the main kernel by itself. NULL clears it. */
int b200fa_bwd_timing_events(void* const* events);

/* Tuning hook (no counterpart in the reference): `counters` is a device buffer of 32 int64 that the backward main
 * kernel adds cycle counts to -- slots 0-10 = cycles its warps spent in each of its waits, 11 = cycles per CTA,
 * 12 = iterations. NULL (the default) turns tracing off. Only libraries built with -DB200FA_TRACE count; the regular
 * build accepts the call and records nothing. */
int b200fa_set_trace(void* counters);

/* Replaces inter_sequence.prepare_metadata (reference src/zigfa/_impl/inter_sequence.py:223-254).
 * Outputs: bits_t (n, ceil(n/32)) int32, cu_visible_k (n + 1) int32, cu_visible_q (n + 1) int32 (saturating). */
int b200fa_interseq_metadata(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, const int32_t* visibility_bits,
                             int32_t num_sequences, int32_t* bits_t, int32_t* cu_visible_k, int32_t* cu_visible_q,
                             void* stream);

/* Builds the sorted work list of a packed batch on the device: entry e = (sequence, block), sequences ordered by
 * descending length class of `cu_seqlens_other` within windows of 1024 sequences, padding entries (batch, 0).
 * Replaces tensors.build_scheduler_metadata (reference src/zigfa/_impl/tensors.py:87-107,
 * zig/prepare_scheduler.zig:101-170). `descending` orders the blocks of a sequence last-to-first. */
int b200fa_work_list(const int32_t* cu_seqlens, const int32_t* cu_seqlens_other, int32_t batch, int32_t block_rows,
                     int32_t descending, int32_t num_entries, int32_t* table, void* stream);
/* Host twins of the integer kernels (same code path compiled for the CPU; used by the CPU unit tests). */
int64_t b200fa_work_list_entries(int64_t rows, int64_t batch, int64_t block_rows);
int b200fa_work_list_host(const int32_t* cu_seqlens, const int32_t* cu_seqlens_other, int32_t batch, int32_t block_rows,
                          int32_t descending, int32_t num_entries, int32_t* table);
int b200fa_interseq_metadata_host(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                  const int32_t* visibility_bits, int32_t num_sequences, int32_t* bits_t,
                                  int32_t* cu_visible_k, int32_t* cu_visible_q);
/* Lists, for query rows [m0, m1) of sequence `seq`, the key blocks the forward kernel visits:
 * out[4*i..4*i+3] = (first key row in the packed tensor, first column relative to its run, run length, banded).
 * Returns the number of blocks (at most max_blocks are written). Host twin of the device cursor. */
int b200fa_key_blocks_host(const b200fa_problem* problem, int32_t seq, int32_t m0, int32_t m1, int32_t* out,
                           int32_t max_blocks);
/* Same for the backward pass: query blocks that see key columns [c0, c1) of key sequence `seq`. */
int b200fa_query_blocks_host(const b200fa_problem* problem, int32_t seq, int32_t c0, int32_t c1, int32_t* out,
                             int32_t max_blocks);

/* ---- Sliding window with sinks (no counterpart in the reference): b200fa_fwd and b200fa_bwd with the first sink_size
 * keys of every sequence visible to each query row that the right bound lets see them, in front of the window. Without a
 * left bound sink_size has no effect. Not for inter-sequence batches; softmax_scale > 0. In a packed batch, what
 * stands in rows behind the last sequence, NaN included, has no effect on any result, whatever the window and sink_size. */
size_t b200fa_sink_fwd_workspace_bytes(const b200fa_problem* problem, int32_t sink_size);
int b200fa_sink_fwd(const b200fa_fwd_args* args, int32_t sink_size, void* stream);
size_t b200fa_sink_bwd_workspace_bytes(const b200fa_problem* problem, int32_t sink_size);
int b200fa_sink_bwd(const b200fa_bwd_args* args, int32_t sink_size, void* stream);
/* The same for contiguous results (out and softmax_lse; dq, dk and dv): the rows of a packed batch that belong to no sequence,
 * in front of cu_seqlens[0] and at or behind cu_seqlens[batch], which the calls above leave as they are, are filled with
 * zeros, -inf in softmax_lse. */
int b200fa_sink_fwd_all_rows(const b200fa_fwd_args* args, int32_t sink_size, void* stream);
int b200fa_sink_bwd_all_rows(const b200fa_bwd_args* args, int32_t sink_size, void* stream);
/* b200fa_key_blocks_host and b200fa_query_blocks_host with sinks. */
int b200fa_sink_key_blocks_host(const b200fa_problem* problem, int32_t sink_size, int32_t seq, int32_t m0, int32_t m1,
                                int32_t* out, int32_t max_blocks);
int b200fa_sink_query_blocks_host(const b200fa_problem* problem, int32_t sink_size, int32_t seq, int32_t c0, int32_t c1,
                                  int32_t* out, int32_t max_blocks);

/* ---- Paged key-value cache (no counterpart in the reference).
 * A cache tensor is (num_pages, page_size, heads_kv, head_dim) BF16; key j of sequence b is row j % page_size of page
 * block_table[b][j / page_size]. A table entry outside [0, num_pages) holds no page: its positions are not visible, and
 * nothing is written there. Lengths outside [0, max_pages * page_size] are cut to that range, except for b200fa_append_kv,
 * where a length only says where the new tokens go. The integer tensors are int32 with contiguous columns. */

/* Attention of one new token per sequence over the cache: out = softmax(scale q k^T) v over the keys that the token, the
 * last of the cache_seqlens[b] keys of its sequence, sees: the last window_left + 1 of them (-1 = all) and the first
 * sink_size. A sequence that sees no key gets zeros and a log-sum-exp of -inf.
 * Strides in elements: q and out [0] sequence, [1] head; caches [0] page, [1] row, [2] head. */
typedef struct b200fa_paged_args {
  int32_t batch, heads_q, heads_kv, head_dim;
  int32_t num_pages, page_size, max_pages; /* max_pages: columns of block_table */
  int32_t window_left, sink_size;
  float softmax_scale;
  const void* q;                /* (batch, heads_q, head_dim) */
  const void* k_cache;
  const void* v_cache;
  const int32_t* block_table;   /* (batch, max_pages), row stride table_stride */
  const int32_t* cache_seqlens; /* (batch) keys per sequence, the new token's among them */
  void* out;                    /* bf16, shape of q */
  float* softmax_lse;           /* fp32 (batch, heads_q) contiguous; natural log */
  int64_t q_stride[2], k_stride[3], v_stride[3], out_stride[2], table_stride;
  void* workspace;
  size_t workspace_bytes;
} b200fa_paged_args;

/* A function of batch, heads_q, heads_kv, head_dim, page_size, max_pages, window_left and sink_size alone. */
size_t b200fa_paged_decode_workspace_bytes(const b200fa_paged_args* args);
int b200fa_paged_decode(const b200fa_paged_args* args, void* stream);
/* Host twin of the key selection: the keys that the new token of a sequence of `length` keys sees, `capacity` being
 * max_pages * page_size, in the order in which the kernel walks them. Returns their number. */
int b200fa_paged_keys_host(int32_t length, int32_t capacity, int32_t window_left, int32_t sink_size, int32_t* keys,
                           int32_t max_keys);

typedef struct b200fa_kv_cache {
  int32_t num_pages, page_size, heads_kv, head_dim; /* head_dim: a multiple of 8 of at most 1024 */
  void* k_cache;
  void* v_cache;
  int64_t k_stride[3], v_stride[3]; /* [0] page, [1] row, [2] head */
} b200fa_kv_cache;

/* Writes the keys and values of new tokens into the pages: token i of sequence b becomes key cache_seqlens[b] + i, and is
 * dropped where that lies outside [0, max_pages * page_size) or on no page.
 * Fixed length: k, v (batch, rows, heads_kv, head_dim), cu_seqlens NULL. Packed: k, v (rows, heads_kv, head_dim),
 * cu_seqlens (batch + 1); rows behind the last sequence are left out. No two sequences may write to the same page. */
typedef struct b200fa_append_args {
  b200fa_kv_cache cache;
  const void* k;
  const void* v;
  int64_t k_stride[3], v_stride[3]; /* [0] sequence, [1] row, [2] head */
  int64_t rows;
  const int32_t* cu_seqlens;
  const int32_t* cache_seqlens; /* (batch) keys held before the call */
  const int32_t* block_table;   /* (batch, max_pages) */
  int64_t table_stride;
  int32_t batch, max_pages;
} b200fa_append_args;
int b200fa_append_kv(const b200fa_append_args* args, void* stream);

/* Copies page source_pages[i] of both caches to page target_pages[i], for i < count; a pair with an entry outside
 * [0, num_pages) is skipped. The targets must differ from one another and from every source. */
int b200fa_copy_pages(const b200fa_kv_cache* cache, const int32_t* source_pages, const int32_t* target_pages, int32_t count,
                      void* stream);

/* Which sequence holds which page. page_refs (num_pages) counts the table entries that name a page; a page with a count
 * <= 0 is free. The calls read block_table and page_refs and write new ones, which must not overlap them; an entry that
 * holds no page comes out as -1. Pages are handed out lowest first, requests served in the order (sequence, entry); when
 * the free pages run out, the entries that got none are -1. */
typedef struct b200fa_pages_args {
  int32_t sequences, rows; /* rows of block_table and of block_table_out */
  int32_t max_pages, num_pages, page_size;
  const int32_t* block_table; /* (sequences, max_pages), row stride table_stride */
  int64_t table_stride;
  const int32_t* page_refs;     /* (num_pages) */
  const int32_t* cache_seqlens; /* (sequences) */
  int32_t* block_table_out;     /* (rows, max_pages) contiguous */
  int32_t* page_refs_out;       /* (num_pages) */
  int32_t* source_pages;        /* pairs for b200fa_copy_pages, -1 = none: (rows) for a fork, (num_pages / 2) for compacting */
  int32_t* target_pages;
  void* workspace; /* b200fa_pages_workspace_bytes(num_pages); not needed by b200fa_free_pages */
  size_t workspace_bytes;
} b200fa_pages_args;
size_t b200fa_pages_workspace_bytes(int32_t num_pages);
/* Pages for the next new_tokens[b] tokens of every sequence: the entries behind the ceil(cache_seqlens[b] / page_size)
 * first ones that lack a page get a free one. */
int b200fa_reserve_pages(const b200fa_pages_args* args, const int32_t* new_tokens, void* stream);
/* Row i of block_table_out becomes a continuation of sequence parents[i]: it shares the parent's full pages and gets a
 * page of its own for the partly filled last one, to be copied (source_pages[i], target_pages[i]). child_seqlens[i] is
 * the parent's length; a parent outside [0, sequences) gives an empty row. */
int b200fa_fork_pages(const b200fa_pages_args* args, const int32_t* parents, int32_t* child_seqlens, void* stream);
/* Gives the entries [first_entry[b], last_entry[b]) of every sequence back: each becomes -1 and its page loses a
 * reference. */
int b200fa_free_pages(const b200fa_pages_args* args, const int32_t* first_entry, const int32_t* last_entry, void* stream);
/* Moves the pages in use to the front of the pool: with n of them, the i-th one at or behind n goes to the i-th free page
 * in front of n. Tables and counts follow, and the pairs (source_pages, target_pages) say what to copy. */
int b200fa_compact_pages(const b200fa_pages_args* args, void* stream);

/* Reads and clears the device-side status word (synchronises the device). 0 = no kernel wait ran out of time. */
int b200fa_device_status(void);
const char* b200fa_last_error(void);
int b200fa_version(void);
/* 1 when head_dim is supported by the forward (direction 0) / backward (direction 1) kernels. */
int b200fa_supports_head_dim(int32_t head_dim, int32_t direction);

#ifdef __cplusplus
}
#endif
#endif /* B200FA_H_ */
