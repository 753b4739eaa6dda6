/*
 * sfa_b200.h — C ABI of the B200 (sm_100a) sparse flash attention library.
 *
 * The library computes block-sparse / top-k indexed attention forward and
 * backward with the semantics of the reference op
 * `SparseFlashAttentionTriton` (lilac-me/ops, SFA.py:69-306), generalised to
 * grouped-query heads, separate k and v, block_size > 1, causal masking and
 * varlen batches.  Every entry point:
 *   - takes plain device pointers, element strides and sizes (no framework types);
 *   - enqueues work on the given CUDA stream (a `cudaStream_t` passed as void*);
 *   - allocates no memory (scratch comes from the caller's workspace);
 *   - never synchronises the host with the device;
 *   - returns SFA_OK (0) or a negative SFA_ERR_* code; sfa_last_error_string()
 *     describes the last failure on the calling thread.
 *
 * Layouts.  Dense: q [B, Tq, Hq, Dqk], k [B, Tk, Hk, Dqk], v [B, Tk, Hk, Dv],
 * block_indices [B, Tq, Hk, S] (int32), o/dout [B, Tq, Hq, Dv], lse [B, Tq, Hq].
 * Varlen (cu_seqlens_q != NULL): the batch axis is dropped, rows of sequence i
 * are [cu_seqlens_q[i], cu_seqlens_q[i+1]) for q/o/lse/indices and
 * [cu_seqlens_k[i], cu_seqlens_k[i+1]) for k/v; block ids are relative to the
 * sequence start.  Strides are in elements; the innermost dimension of every
 * tensor is contiguous.  The reference's SBHD layout (SFA.py:87-90) is the
 * dense layout with batch and token strides swapped.
 *
 * Index semantics.  A selected block id e is valid iff 0 <= e < ceil(kv_len /
 * block_size); key e*block_size + j (j < block_size) is valid iff it is < kv_len
 * and, when causal, <= t + kv_len - q_len.  Entries may sit in any slot; a
 * duplicate entry counts once per slot.  lse is natural-log; a row with no valid
 * key and no sink has o = 0 and lse = -inf.
 */
#ifndef SFA_B200_H
#define SFA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SFA_ABI_VERSION 3

enum {
  SFA_OK = 0,
  SFA_ERR_INVALID_ARGUMENT = -1,   /* bad shape, stride, alignment or null pointer */
  SFA_ERR_UNSUPPORTED = -2,        /* shape outside every kernel family's limits */
  SFA_ERR_WORKSPACE = -3,          /* workspace missing or smaller than required */
  SFA_ERR_CUDA = -4,               /* a CUDA runtime/driver call failed */
  SFA_ERR_DEVICE_TIMEOUT = -5      /* a kernel's bounded wait expired (see sfa_device_status) */
};

/* dK/dV algorithm (SfaParams.dkv_mode). */
enum {
  SFA_DKV_AUTO = 0,      /* pick from the launch table (measured throughput) */
  SFA_DKV_INVERTED = 1,  /* block->query inverted index + key-centric pass; deterministic */
  SFA_DKV_ATOMIC = 2     /* query-centric pass with fp32 atomics */
};

/* dQ algorithm (SfaParams.dq_mode) of the tensor-core backward with the
 * inverted-index dK/dV pass; other paths always compute dQ in their own pass. */
enum {
  SFA_DQ_AUTO = 0,      /* FUSED where it applies */
  SFA_DQ_SEPARATE = 1,  /* query-centric pass that recomputes S and dP; deterministic */
  SFA_DQ_FUSED = 2      /* accumulated by the key-centric dK/dV pass from its dS (fp32
                           reductions into a workspace accumulator, order not fixed);
                           needs rows * h_q * d_qk * 4 more workspace bytes */
};

/* Opt-in reference arithmetic (SfaParams.compat).  SFA_COMPAT_REFERENCE_P
 * rounds the forward's probabilities the way SparseFlashAttentionTriton does
 * before its PV matmul: stored as fp16, read back as bf16 (SFA.py:446, 456); the
 * row sums keep the unrounded values, as there.  Default: one rounding to bf16. */
#define SFA_COMPAT_REFERENCE_P 1

/* kv storage (SfaParams.kv_dtype). */
enum {
  SFA_KV_BF16 = 0,
  SFA_KV_FP8_E4M3 = 1   /* e4m3 bytes + one fp32 scale per kv row (forward only) */
};

/* Kernel family (SfaParams.kernel); AUTO picks the tensor-core path when it
 * supports the shape and the general CUDA-core path otherwise. */
enum {
  SFA_KERNEL_AUTO = 0,
  SFA_KERNEL_TCGEN05 = 1,
  SFA_KERNEL_GENERAL = 2
};

typedef struct SfaParams {
  /* inputs (device pointers) */
  const void* q;              /* bf16 */
  const void* k;              /* bf16 */
  const void* v;              /* bf16 */
  const int32_t* block_indices;
  const int32_t* cu_seqlens_q; /* [num_seqs + 1] or NULL for dense */
  const int32_t* cu_seqlens_k; /* [num_seqs + 1] or NULL for dense */
  const float* attn_sink;     /* [Hq] fp32 or NULL */
  /* forward outputs / backward inputs */
  void* o;                    /* bf16 */
  float* lse;                 /* fp32, natural log */
  /* backward */
  const void* dout;           /* bf16 */
  void* dq;                   /* bf16 */
  void* dk;                   /* bf16 */
  void* dv;                   /* bf16; may equal dk when k and v are one tensor (then dk := dk + dv) */
  float* dsink;               /* [Hq] fp32 or NULL; overwritten */

  /* element strides: batch (dense only), token, head */
  int64_t q_sb, q_st, q_sh;
  int64_t k_sb, k_st, k_sh;
  int64_t v_sb, v_st, v_sh;
  int64_t i_sb, i_st, i_sh;   /* block_indices; the S axis is contiguous */
  int64_t o_sb, o_st, o_sh;
  int64_t l_sb, l_st, l_sh;   /* lse */
  int64_t do_sb, do_st, do_sh;
  int64_t dq_sb, dq_st, dq_sh;
  int64_t dk_sb, dk_st, dk_sh;
  int64_t dv_sb, dv_st, dv_sh;

  int32_t batch;      /* B (dense) or number of sequences (varlen) */
  int32_t q_len;      /* Tq (dense) or max query length over sequences (varlen) */
  int32_t kv_len;     /* Tk (dense) or max kv length over sequences (varlen) */
  int32_t total_q;    /* varlen: cu_seqlens_q[batch]; dense: ignored */
  int32_t total_kv;   /* varlen: cu_seqlens_k[batch]; dense: ignored */
  int32_t h_q, h_kv;  /* h_q % h_kv == 0 */
  int32_t d_qk, d_v;
  int32_t block_size; /* keys per selected block (1 = token-level) */
  int32_t topk;       /* S, slots per (query, kv head) */
  float scale;        /* softmax scale applied to q.k */
  int32_t causal;     /* 0 / 1 */
  int32_t dkv_mode;   /* SFA_DKV_* */
  int32_t kernel;     /* SFA_KERNEL_* */
  int32_t dq_mode;    /* SFA_DQ_* (was reserved: zero = AUTO) */
  int32_t compat;     /* SFA_COMPAT_* bits (was reserved: zero = none) */
  /* Paged kv cache (forward only; no reference counterpart): when block_table
   * is non-NULL, k and v are page pools of total_kv rows (page p holds rows
   * [p*page_size, (p+1)*page_size), row stride k_st / v_st), the call is
   * varlen, cu_seqlens_k gives only the kv lengths (cu_seqlens_k[s+1] -
   * cu_seqlens_k[s]), and kv position t of sequence s is pool row
   * block_table[s*bt_stride + t/page_size]*page_size + t%page_size.  With
   * block_size > 1, page_size must be a multiple of block_size. */
  int32_t page_size;
  const int32_t* block_table;
  int64_t bt_stride;
  /* fp8 kv (forward only; no reference counterpart): with kv_dtype =
   * SFA_KV_FP8_E4M3, k points to e4m3 bytes (strides in bytes; v must be k or
   * its leading d_v dims, the MLA latent) and kv_scale to one fp32 scale per
   * kv row, indexed b*ks_sb + t*ks_st + h*ks_sh (t the kv row, through the
   * block table when paged): key = e4m3 value * scale, rounded to bf16 for
   * the bf16 MMAs (exact when the scales are powers of two). */
  int32_t kv_dtype;   /* SFA_KV_* */
  int32_t reserved;
  const float* kv_scale;
  int64_t ks_sb, ks_st, ks_sh;
} SfaParams;

/* Library / ABI identification. */
int sfa_abi_version(void);
const char* sfa_build_info(void);

/* Message for the last non-OK return on this thread. */
const char* sfa_last_error_string(void);

/* Number of kernels this library has enqueued since it was loaded (all
 * threads); a caller brackets a region with two reads to count its launches. */
unsigned long long sfa_kernel_launches(void);

/* Launch trace, for benchmarks that time each kernel with CUDA events (no
 * counterpart in the reference).  `events` holds n_events cudaEvent_t handles
 * (as void*) created by the caller; while it is set, every kernel or memset the
 * library enqueues from the calling thread is followed by a cudaEventRecord of
 * the next unused event on the same stream, so the time between consecutive
 * events (the first one against an event the caller records before its call)
 * is one operation.  sfa_launch_trace_count() gives how many events were
 * recorded and sfa_launch_trace_name(i) the operation event i closes.  Passing
 * NULL stops tracing; a new call restarts the count.  The events must outlive
 * the trace. */
int sfa_launch_trace(void* const* events, int n_events);
int sfa_launch_trace_count(void);
const char* sfa_launch_trace_name(int i);

/* Which kernel family a call with these params would launch (SFA_KERNEL_*), or
 * a negative error code if the shape is unsupported. */
int sfa_select_kernel(const SfaParams* p, int is_backward);

/* The backward's resolved algorithms for these params: *dkv_mode gets
 * SFA_DKV_INVERTED or SFA_DKV_ATOMIC, *dq_mode SFA_DQ_SEPARATE or SFA_DQ_FUSED
 * (the launch-table counterpart of SFA.py:51-59; no reference entry point).
 * Returns the kernel family or a negative error code. */
int sfa_bwd_plan(const SfaParams* p, int32_t* dkv_mode, int32_t* dq_mode);

/* Workspace (device bytes) the forward / backward need for these params.  The
 * token-level backward above 256 head dims runs in two passes over bf16 P and
 * dS' rows (topk slots per query head); its workspace holds them for a wave of
 * query rows sized to stay within 4 GiB (the environment variable
 * SFA_MLA_WAVE_ROWS, read at each call, sets the rows per wave instead). */
size_t sfa_fwd_workspace_bytes(const SfaParams* p);
size_t sfa_bwd_workspace_bytes(const SfaParams* p);

/* Forward: writes o and lse.  Replaces SparseFlashAttentionTriton.forward
 * (SFA.py:75-164): the reference's `_attn_fwd` launch (SFA.py:122-159) and its
 * per-launch workspaces (SFA.py:117-120), without the host sync of
 * `_effective_topk` (SFA.py:62-66). */
int sfa_fwd(const SfaParams* p, void* workspace, size_t workspace_bytes, void* stream);

/* Backward: writes dq, dk, dv and (if non-NULL) dsink.  Replaces
 * SparseFlashAttentionTriton.backward (SFA.py:167-306): `_attn_bwd_dq_dsink`
 * (SFA.py:199-251) and `_attn_bwd_dk_dv` (SFA.py:266-298). */
int sfa_bwd(const SfaParams* p, void* workspace, size_t workspace_bytes, void* stream);

/* The backward's stages, for callers that schedule them separately.  Each takes
 * the same workspace as sfa_bwd.
 *  - preprocess: delta = rowsum(o * dout) in fp32 and dsink
 *    (replaces `_get_delta_split`, SFA.py:590-610, and the dsink atomics,
 *    SFA.py:964-970);
 *  - dq: replaces `_attn_bwd_dq_dsink` / `_inner_dq` (SFA.py:613-716, 856-1002);
 *    with SFA_DQ_FUSED it only clears the dQ accumulator;
 *  - dkdv: replaces `_attn_bwd_dk_dv` / `_inner_dkv` (SFA.py:719-853, 1005-1145);
 *    with SFA_DKV_INVERTED it first builds the block->query index; with
 *    SFA_DQ_FUSED it also accumulates dQ and writes dq.
 * Run them in this order on one stream. */

int sfa_bwd_preprocess(const SfaParams* p, void* workspace, size_t workspace_bytes, void* stream);
int sfa_bwd_dq(const SfaParams* p, void* workspace, size_t workspace_bytes, void* stream);
int sfa_bwd_dkdv(const SfaParams* p, void* workspace, size_t workspace_bytes, void* stream);

/* Backward for callers that cannot allocate device memory (no counterpart in the
 * reference).  Same results as sfa_bwd, but the scratch comes from a 32 MiB
 * static device array inside the library instead of a caller workspace; every
 * GPU that loads the library reserves that array until the process exits.
 * With dq_mode SFA_DQ_AUTO, dQ runs as its own pass (SFA_DQ_SEPARATE) when the
 * fused accumulator would not fit; problems whose workspace still exceeds
 * 32 MiB are refused with SFA_ERR_WORKSPACE before anything is launched.  The first call on a device
 * looks up the array's device address; make it before any stream capture.
 * Calls share the array: calls that overlap on the GPU race and must be
 * serialised by the caller.  The looked-up address is kept for the life of the
 * process: after a device reset (cudaDeviceReset, or a primary-context reset)
 * the library must be reloaded before this entry point is called again. */
int sfa_bwd_noalloc(const SfaParams* p, void* stream);

/* Inverted index alone (for tests): for every (sequence, kv head, block) the
 * list of query rows that selected it, ascending by (query, slot).  Layout in
 * the workspace is described by sfa_inverted_index_layout(). */
int sfa_build_inverted_index(const SfaParams* p, void* workspace, size_t workspace_bytes, void* stream);
/* Byte offsets inside the backward workspace of: block offsets (int32,
 * [units * nblk + 1]) and query-row entries (int32, [pairs]); also reports
 * nblk (blocks per unit) and units (= batch * h_kv). */
int sfa_inverted_index_layout(const SfaParams* p, size_t* offsets_off, size_t* entries_off,
                              int32_t* nblk, int32_t* units);

/* Device status word written by kernels whose bounded waits expired.
 * sfa_device_status copies it to *status (synchronising `stream`); sfa_reset_device_status
 * clears it (stream-ordered). 0 = healthy. */
int sfa_device_status(void* stream, int32_t* status);
int sfa_reset_device_status(void* stream);

/* Self-test of that failure path: one warp waits, with a limit of limit_us
 * (1 .. 1e6), on an mbarrier nothing ever arrives on, through the same bounded
 * wait the kernels use.  The wait runs out and the status word receives
 * SFA_SELFTEST_STATUS (unless an earlier code is still there); the kernel
 * returns and the context stays usable.  Stream-ordered. */
#define SFA_SELFTEST_STATUS ((15 << 16) | 1)
int sfa_selftest_wait_timeout(void* stream, uint32_t limit_us);

/* ------------------------------------------------------------------------
 * Top-k token indexer: the step before the op, producing its token-level
 * indices (the reference consumes topk_idxs and has no indexer, SFA.py:90).
 * Scores follow the lightning-indexer formula of DeepSeek-V3.2's sparse
 * attention:  I[t, s] = sum_h w[t, h] * ReLU(q_idx[t, h] . k_idx[s]),  s a key
 * of t's sequence (s <= t + kv_len - q_len when causal).  The output row of t
 * holds the indices of the topk highest scores (ties: the lower index first)
 * in ascending order, then -1 when fewer keys exist — the layout the op's
 * token-level surface and the reference take as-is.
 *
 * Dense layout: q_idx [B, Tq, H, D] bf16, k_idx [B, Tk, D] bf16 (one head
 * shared by every query head), weights [B, Tq, H] fp32, out [B, Tq, topk]
 * int32; strides in elements, innermost dims contiguous.  H is 64 or 32,
 * D is 64 or 128, topk <= 4096 (fp32 scores of a row go through shared
 * memory: Tk <= 49152).  The workspace holds fp32 scores for a wave of rows. */
typedef struct SfaIndexerParams {
  const void* q_idx;
  const void* k_idx;
  const float* weights;
  int32_t* out;
  int64_t q_sb, q_st, q_sh;
  int64_t k_sb, k_st;
  int64_t w_sb, w_st;
  int64_t o_sb, o_st;
  int32_t batch, q_len, kv_len, heads, dim, topk;
  int32_t causal;
  int32_t reserved;
} SfaIndexerParams;

size_t sfa_indexer_workspace_bytes(const SfaIndexerParams* p);
int sfa_indexer_topk(const SfaIndexerParams* p, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Norm and rotary positions of queries and keys: the step before the op (no
 * counterpart in the reference, which takes q and kv as they are, SFA.py:87-90).
 * For every row x (one head of one token, dim elements), in fp32:
 *     n = x * rsqrt(mean(x^2) + eps) * weight          (tensors with a weight)
 *     y = n with the pairs of its dims [start, start + rot) turned by
 *         position * frequencies[i] and scaled by amplitude (SFA_ROTARY_TURN)
 * rounded once to the tensor's type.  Pair i is (i, i + rot/2) of the rotated
 * part, or (2i, 2i + 1) when interleaved.  Angles are reduced in whole numbers:
 * the position multiplies the frequency as a fraction of a turn (127 bits with
 * pos64, 64 without), so any position has the accuracy of the first ones.  dim is at most 1024, and a tensor has fewer than
 * 2^31 rows.
 *
 * Up to three tensors go through one launch (q, k and, for the append, v with
 * neither weight nor TURN).  A tensor with SFA_ROTARY_PAGED is stored into a
 * page pool instead: y is the pool, y_st its row stride, y_sh its head stride;
 * batch must be 1 and row i of sequence s (cu_seqlens; NULL: one row each) goes
 * to cache position cache_seqlens[s] - rows(s) + i through block_table.  Rows
 * behind cu_seqlens[num_seqs], negative positions, positions behind the table
 * and page ids outside [0, num_pages) are not stored.
 * Backward: dx from x and dy, dweight (fp32, overwritten, fixed summation order). */
enum { SFA_DTYPE_BF16 = 0, SFA_DTYPE_F16 = 1, SFA_DTYPE_F32 = 2 };
enum { SFA_ROTARY_TURN = 1, SFA_ROTARY_PAGED = 2 };

typedef struct SfaRotaryTensor {
  const void* x;
  void* y;               /* forward output (or the page pool) */
  const void* dy;        /* backward */
  void* dx;
  const float* weight;   /* [dim] or NULL: no norm */
  float* dweight;        /* [dim] or NULL */
  int64_t x_sb, x_st, x_sh;   /* element strides: batch, token, head */
  int64_t y_sb, y_st, y_sh;
  int64_t dy_sb, dy_st, dy_sh;
  int64_t dx_sb, dx_st, dx_sh;
  int32_t heads;
  int32_t flags;         /* SFA_ROTARY_* */
} SfaRotaryTensor;

typedef struct SfaRotaryParams {
  SfaRotaryTensor t[3];
  const void* positions;        /* int32, or int64 with pos64 */
  const double* frequencies;    /* [rot / 2] radians per position */
  const int32_t* block_table;   /* paged tensors only, from here ... */
  const int32_t* cache_seqlens;
  const int32_t* cu_seqlens;
  int64_t bt_stride;            /* ... to here */
  int64_t p_sb, p_st;
  int32_t num_tensors, batch, len, dim, rot, start, interleaved, dtype, pos64;
  int32_t num_seqs, num_pages, page_size, table_width;
  float eps, amplitude;
  int32_t reserved;
} SfaRotaryParams;

int sfa_rotary_fwd(const SfaRotaryParams* p, void* stream);
size_t sfa_rotary_bwd_workspace_bytes(const SfaRotaryParams* p);
int sfa_rotary_bwd(const SfaRotaryParams* p, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Attention of drafted tokens over a paged kv cache (no counterpart in the
 * reference): every query row sees all of its sequence's cache rows before the
 * drafted ones, and of the drafted ones its own and its ancestors'.
 *
 * q [total_q, h_q, d_qk] holds the drafted rows of num_seqs sequences, offsets
 * cu_seqlens (NULL: one row each); cache_seqlens are the cache lengths with
 * them, so row j of sequence s is cache position cache_seqlens[s] - rows(s) + j.
 * parents[row] is the row's parent within its sequence (a number below its own;
 * anything else: the row hangs on the prefix); NULL: a chain (causal).  With
 * parents a sequence has at most SFA_TREE_MAX_NODES rows.  Keys and values are
 * read through block_table from pools of num_pages pages; a table entry outside
 * [0, num_pages) and positions behind the table hold no keys.  Values of cache
 * rows that no row of the sequence sees do not matter, NaN included, and a row
 * is not touched by what a drafted row it does not see holds.  attn_sink adds
 * exp(sink) to the denominator.  A row that sees nothing gives o = 0 and lse =
 * -inf (or its sink); so do rows outside all sequences and rows past max_q.
 * Types: bf16 or fp16 (dtype), lse fp32; d_qk and d_v multiples of 8 up to 256;
 * strides in elements, multiples of 8, bases 16-byte aligned; scale > 0. */
#define SFA_TREE_MAX_NODES 256

typedef struct SfaTreeParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* block_table;
  const int32_t* cache_seqlens;
  const int32_t* cu_seqlens;
  const int32_t* parents;
  const float* attn_sink;
  void* o;
  float* lse;
  int64_t q_st, q_sh;
  int64_t k_st, k_sh;   /* pool row and head strides; page p is rows [p*page_size, (p+1)*page_size) */
  int64_t v_st, v_sh;
  int64_t o_st, o_sh;
  int64_t l_st, l_sh;
  int64_t bt_stride;
  int32_t num_seqs, total_q;
  int32_t max_q;        /* the most rows of a sequence */
  int32_t max_k;        /* an estimate of the longest cache (sizes the split; not a limit) */
  int32_t h_q, h_kv, d_qk, d_v;
  int32_t num_pages, page_size, table_width, dtype;
  float scale;
  int32_t reserved;
} SfaTreeParams;

size_t sfa_tree_workspace_bytes(const SfaTreeParams* p);
int sfa_tree_attention(const SfaTreeParams* p, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Pages of a kv cache (no counterpart in the reference).  A pool has num_pages
 * pages; refcounts[page] says how many block-table entries hold it (0: free).
 * Sequence s holds its first ceil(cache_seqlens[s] / page_size) table entries;
 * the entries behind are -1.  New pages are the free ones of lowest number, in
 * the order of the rows that ask, so results repeat.  All state is on the
 * device and nothing is read back.  pools (a host array) are the tensors that
 * the pages index, e.g. K and V of every layer: page p is page_bytes contiguous
 * bytes at base + p * page_stride.
 *
 *  - reserve: a = [num_seqs] rows to add.  out[s] = 1 if s got the pages for
 *    them (cache_seqlens grows), 0 if nothing was changed: a negative count, a
 *    table too narrow, a partly filled last page that others share, or free
 *    pages too few for the rows up to s together;
 *  - trim: a = [num_seqs] rows to keep (negative: leave s alone).  Entries
 *    behind them are given back;
 *  - fork: a = [count] source, b = [count] target sequences.  Whole pages are
 *    shared, a partly filled last page is copied to a new one.  out[i] = 1 if
 *    done, 0 if nothing was changed: a number outside the table, a target that
 *    holds rows or is named by an earlier fork, a last page outside the pool,
 *    or free pages too few.  Sources are taken as they were before the call;
 *  - accept: a = [num_seqs, count] accepted drafted rows of each sequence,
 *    ascending, ended by -1 or the width; b = [num_seqs] drafted rows.  The
 *    accepted cache rows are moved together behind the prefix, cache_seqlens -
 *    b; out[s] = rows to keep (for trim), -1 for a sequence with b outside
 *    [0, cache_seqlens], or one whose rows would be moved into a page with a
 *    reference count above 1: nothing of it moves.  Without refcounts the caller
 *    answers for it that those pages are the sequence's alone;
 *  - accept_table: the same with counts of its own.  refcounts is scratch, which
 *    gets the number of entries of this table that hold each page;
 *  - compact: pages in use are moved to the lowest numbers, refcounts and table
 *    follow; out[0] = pages in use;
 *  - copy: page a[i] to page b[i], i < count.  out[i] = 1 if copied, 0 for a
 *    page outside the pool, a target named by an earlier pair, or a source that
 *    another pair writes. */
typedef struct SfaCachePool {
  void* base;
  int64_t page_stride;   /* bytes */
  int64_t page_bytes;    /* a multiple of page_size */
} SfaCachePool;

typedef struct SfaCacheParams {
  int32_t* refcounts;
  int32_t* block_table;
  int32_t* cache_seqlens;
  const int32_t* a;
  const int32_t* b;
  int32_t* out;
  const SfaCachePool* pools;   /* host */
  int64_t bt_stride, a_stride;
  int32_t num_pools, num_seqs, num_pages, page_size, table_width, count;
} SfaCacheParams;

size_t sfa_cache_workspace_bytes(const SfaCacheParams* p);   /* enough for every call below */
int sfa_cache_reserve(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream);
int sfa_cache_trim(const SfaCacheParams* p, void* stream);
int sfa_cache_fork(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream);
int sfa_cache_accept(const SfaCacheParams* p, void* stream);
int sfa_cache_accept_table(const SfaCacheParams* p, void* stream);
int sfa_cache_compact(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream);
int sfa_cache_copy(const SfaCacheParams* p, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SFA_B200_H */
