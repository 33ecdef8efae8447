/*
 * nsa_sel.h -- C ABI of the B200 (sm_100a) NSA selected-branch attention forward, with the
 * block selection that produces its index rows, and with the backward and the 4-bit KV cache
 * (writing, reading back, attention of single tokens, pages and block selection for them, rotary
 * positions) that the reference lacks.
 *
 * This is the drop-in boundary for the one hot path of the nsa-hopper reference: the
 * selected-branch forward that its kernels expose through pybind as
 *
 *     torch::Tensor forward(Tensor Q, Tensor K, Tensor V, Tensor sel,
 *                           int64 l_prime, int64 BQ, Tensor cyc)
 *
 * (reference nsa_v0.cu:118-146, nsa_v1.cu:125-147, nsa_v2.cu:147-170).  Every entry point
 * takes plain pointers and sizes; no torch type crosses this boundary.  The library never
 * calls cudaMalloc: all buffers belong to the caller, except one static device array inside the
 * library (16 MB) that only nsa_sel_select_noalloc uses.  All launches go to the stream
 * passed in; a call returns as soon as the work is queued (like the reference op, which is
 * asynchronous on the legacy stream).  The library is reentrant: concurrent calls from
 * several host threads are safe, and the error text is kept per host thread.  Two exceptions
 * share device state between calls: nsa_sel_select_noalloc (one static scratch per device:
 * calls on one device must be serialised, e.g. on one stream), and replays of one captured CUDA
 * graph (each captured forward launch owns one work-counter slot: replays of the same graph
 * must not overlap each other).
 *
 * Layouts (all contiguous, row-major, as in the reference):
 *   Q   bf16 [B, Hq,  T, d_qk]        K bf16 [B, Hkv, T, d_qk]      V bf16 [B, Hkv, T, d_v]
 *   sel int32 [B, Hkv, NQB, KSEL]    NQB = ceil(T / BQ); entry = block index (block = l_prime
 *                                     keys); negative entries are padding and are skipped
 *   O   [B, Hq, T, d_v]  bf16 or fp32 (every element is written; rows with no visible key = 0)
 *   LSE fp32 [B, Hq, T]  natural log of sum_j exp(scale * q.k_j) over the visible keys
 *                        (-inf for a row with no visible key)
 *   cyc int64 [NQB * B * Hkv * 2]  optional; slot (b*Hkv+kvh)*NQB+qb holds
 *                        {cycles the MMA issuer waited for K/V tiles, other cycles}
 *
 * Semantics (pinned against the reference's PyTorch oracle ref_only.py:2-20 and
 * nsa_reference.py:18-25,66-77): query token t of KV head kvh attends to every key position
 * p with p <= t inside the selected blocks of its query block; selection is a set
 * (duplicates count once); entries < 0 or >= ceil(T / l_prime) select nothing; the softmax
 * scale defaults to 1/sqrt(d_qk); a row with no visible key gives O = 0.
 */
#ifndef NSA_SEL_H_
#define NSA_SEL_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Same object as cudaStream_t; NULL is the legacy default stream. */
typedef struct CUstream_st* nsa_stream_t;

#define NSA_SEL_VERSION 10000 /* 1.0.0 */

/* Return codes (0 = success). */
#define NSA_OK 0
#define NSA_ERR_INVALID_ARG (-1) /* bad pointer, shape, stride or alignment */
#define NSA_ERR_UNSUPPORTED (-2) /* valid request outside the built kernel family */
#define NSA_ERR_CUDA (-3)        /* a CUDA runtime call failed; see nsa_sel_last_error() */
#define NSA_ERR_DRIVER (-4)      /* the driver entry point for tensor maps is unavailable */

/* Bits a kernel ORs into the optional device error word (nsa_sel_desc.err). */
#define NSA_DEVERR_TIMEOUT 1 /* a bounded wait inside the kernel ran out; outputs invalid */

/* Test hook: the MMA warp starts with a wait that nothing completes, so the launch ends through
   the bounded-wait error path (NSA_DEVERR_TIMEOUT after timeout_ms) without any fault. */
#define NSA_DEBUG_STALL 1
/* Comparison switches (same results, different schedule): hand out work units in fixed strides
   instead of from the dynamic counter; never use the row-owner kernel for 64/128-row tiles; run a
   64-row tile of the row-owner kernel as 128-row MMAs with 64 rows of zero padding instead of
   M = 64 MMAs. */
#define NSA_DEBUG_STATIC_UNITS 2
#define NSA_DEBUG_NO_ROW_OWNER 4
#define NSA_DEBUG_RO_PAD128 8

#define NSA_DTYPE_BF16 0
#define NSA_DTYPE_F32 1
#define NSA_DTYPE_F16 2 /* the cache functions only */

#define NSA_KEYMAP_CAUSAL 0     /* key position p is visible to query t iff p <= t */
#define NSA_KEYMAP_COMPRESSED 1 /* compressed key i is visible iff linspace(0, T-1, kv_len)[i] <= t */

/* Full description of one call.  Zero-initialise, then fill the fields you need. */
typedef struct nsa_sel_desc {
  const void* q;              /* bf16 [B, Hq, T, d_qk] */
  const void* k;              /* bf16 [B, Hkv, T, d_qk] */
  const void* v;              /* bf16 [B, Hkv, T, d_v] */
  const int32_t* sel;         /* int32 [B, Hkv, NQB, KSEL] */
  const int32_t* cu_seqlens;  /* optional int32 [n_seqs + 1]: packed varlen batch (B == 1, BQ == 1);
                                 block ids are relative to each sequence's first token */
  void* o;                    /* [B, Hq, T, d_v], dtype o_dtype */
  float* lse;                 /* optional fp32 [B, Hq, T] */
  int64_t* cyc;               /* optional int64 [NQB * B * Hkv * 2], accumulated into */
  int32_t* err;               /* optional device int32; NSA_DEVERR_* bits are ORed into it */
  int32_t batch, heads_q, heads_kv, seq_len, d_qk, d_v;
  int32_t n_qblocks;          /* NQB, must equal ceil(seq_len / q_block) */
  int32_t n_sel;              /* KSEL */
  int32_t block_size;         /* l_prime: 64, 128 or 256 */
  int32_t q_block;            /* BQ: query tokens sharing one selection row (1 = per token) */
  int32_t n_seqs;             /* number of sequences when cu_seqlens is set */
  int32_t o_dtype;            /* NSA_DTYPE_BF16 or NSA_DTYPE_F32 */
  float scale;                /* softmax scale; <= 0 selects 1/sqrt(d_qk) */
  /* Shard: process only (b*Hkv+kvh) in [bkv_begin, bkv_end) and query blocks in
     [qb_begin, qb_end); an end of 0 means "to the end".  Outputs outside the shard are
     left untouched. */
  int32_t bkv_begin, bkv_end, qb_begin, qb_end;
  int32_t timeout_ms;         /* bound on every in-kernel wait; 0 = default (2000 ms) */
  int32_t max_ctas;           /* 0 = one CTA per SM */
  int32_t debug_flags;        /* NSA_DEBUG_* bits; 0 in normal use */
  /* Key visibility beyond the causal default (the sliding-window and compressed branches of NSA,
     reference nsa_reference.py:59-64 and 79-82, run on the same kernel): */
  int32_t kv_len;             /* K/V rows per (b, kvh); 0 = seq_len.  Other values need
                                 key_map = NSA_KEYMAP_COMPRESSED (then K, V are [B, Hkv, kv_len, d]) */
  int32_t window;             /* > 0: key p is visible to query t only if t - p < window (causal
                                 key map only; not with cu_seqlens) */
  int32_t key_map;            /* NSA_KEYMAP_CAUSAL: key p visible to query t iff p <= t;
                                 NSA_KEYMAP_COMPRESSED: key i visible iff the float32
                                 linspace(0, seq_len-1, kv_len)[i] <= t (not with cu_seqlens) */
  /* Fused output combination (the NSA gate, reference nsa_reference.py:86-88): */
  int32_t o_accumulate;       /* 0: O is overwritten; 1: O += w * result (fp32 O only; TMA reduce-add) */
  int32_t reserved;
  const float* o_weight;      /* optional device float w multiplying the result; NULL = 1 */
} nsa_sel_desc;

/* Launch plan chosen for a description (filled by nsa_sel_plan, used by the launcher). */
typedef struct nsa_sel_plan_info {
  int32_t n_cols;       /* N of the tensor-core tiles: G * q_tokens_per_unit rounded up */
  int32_t q_per_unit;   /* query tokens per work unit */
  int32_t parts;        /* work units per query block */
  int32_t n_units;      /* work units in the shard */
  int32_t k_stages, v_stages;
  int32_t smem_bytes;
  int32_t grid;
  int32_t tmem_cols;
  int32_t reserved[7];
} nsa_sel_plan_info;

/* Replaces the reference's forward(Q,K,V,sel,l_prime,BQ,cyc) (nsa_v2.cu:147-170,
   nsa_v1.cu:125-147, nsa_v0.cu:118-146): fp32 O, d_qk == d_v == D, scale 1/sqrt(D).
   cyc may be NULL (the reference passes an empty tensor for "none", nsa_v2.cu:159). */
int nsa_sel_forward(const void* q, const void* k, const void* v, const int32_t* sel, float* o, int64_t* cyc,
                    int32_t B, int32_t Hq, int32_t Hkv, int32_t S, int32_t D, int32_t NQB, int32_t KSEL,
                    int32_t l_prime, int32_t BQ, nsa_stream_t stream);

/* The BASELINE path: bf16 O plus fp32 LSE, d_qk may differ from d_v, optional varlen.
   Extends the same reference op (nsa_v2.cu:147) with the outputs the reference lacks. */
int nsa_sel_forward_lse(const void* q, const void* k, const void* v, const int32_t* sel,
                        const int32_t* cu_seqlens, int32_t n_seqs, void* o, float* lse, int32_t o_dtype,
                        int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t d_qk, int32_t d_v, int32_t NQB,
                        int32_t KSEL, int32_t l_prime, int32_t BQ, float scale, nsa_stream_t stream);

/* General entry point: everything above plus shards, cycle counters, a device error word
   and the wait bound.  Same reference op (nsa_v2.cu:147-170). */
int nsa_sel_run(const nsa_sel_desc* desc, nsa_stream_t stream);

/* Host buffers for nsa_sel_run_host (same layouts as the device buffers of the descriptor;
   pinned host memory lets the copies overlap the kernel). */
typedef struct nsa_sel_host_io {
  const void* q;              /* [B, Hq, T, d_qk] bf16 */
  const void* k;              /* [B, Hkv, kv_len, d_qk] bf16 */
  const void* v;              /* [B, Hkv, kv_len, d_v] bf16 */
  const int32_t* sel;         /* [B, Hkv, NQB, KSEL] */
  void* o;                    /* [B, Hq, T, d_v], dtype o_dtype; receives O */
  float* lse;                 /* optional [B, Hq, T]; receives the LSE when desc->lse is set */
  int32_t token_slices;       /* query-block ranges per (b, kvh) row; 0 = automatic */
  int32_t reserved[7];
} nsa_sel_host_io;

/* The same forward for a caller whose tensors live in host memory (the reference op takes
   whatever tensors it is given, nsa_v2.cu:147-170): copies the inputs of the descriptor's shard
   into its device buffers, runs the kernel and copies O (and LSE) back, pipelined over (b, kvh)
   rows x token slices so that the host-to-device copy of slice i+1, the kernel on slice i and the
   device-to-host copy of slice i-1 overlap (two library-owned copy streams, ordered against
   `stream` with events; no device memory is allocated).  Asynchronous: the host outputs are
   complete when `stream` reaches the point after this call.  o_accumulate must be 0;
   cu_seqlens, when set, must already be in device memory. */
int nsa_sel_run_host(const nsa_sel_desc* desc, const nsa_sel_host_io* io, nsa_stream_t stream);

/* Validate a description and report the launch plan without touching the GPU.
   sm_count <= 0 means "query the current device". */
int nsa_sel_plan(const nsa_sel_desc* desc, int32_t sm_count, nsa_sel_plan_info* out);

/* Block selection: the producer of the selected branch's index rows (replaces the PyTorch
   select_blocks of reference nsa_reference.py:27-44, with compress_kv :5-16 and the group-summed
   queries of :70-71).  For every (b, kvh, token t) it scores selection block nb as
       s(t, nb) = (sum_g q[b, kvh*G + g, t, :]) . kblk[b, kvh, nb, :],
       kblk[nb] = 1/sqrt(d) * sum over compressed keys i of block nb of
                  mean_{j < cmp_block} k[b, kvh, i*cmp_stride + j, :],
   where compressed key i belongs to block floor(linspace(0, T-1, n_cmp)[i] / l_prime) (float32,
   clamped to the last block; n_cmp = (T - cmp_block) / cmp_stride + 1), and writes
       sel_out int32 [B, Hkv, T, k],  k = min(n_sel, ceil(T / l_prime)) <= 32,
   the k best visible blocks (nb * l_prime <= t) by score, highest first; -1 where fewer than k
   blocks are visible (the reference's topk returns masked future blocks there, which the
   selected branch ignores in the same way).  q, k bf16 as in nsa_sel_forward (d_qk = d,
   d % 8 == 0, d <= 256; q 16-byte aligned); kblk_workspace: caller-owned buffer of
   nsa_sel_select_workspace_bytes() bytes, 16-byte aligned.  Two kernel launches on `stream`.
   For d = 64 and 128 the scores run on the tensor cores with each operand split into two bf16
   parts (hi + lo, three products accumulated in fp32: about 16 bits of each operand, ranking
   equal to fp32 scores except at near-ties); other d use fp32 FMA.  The tensor-core kernel's
   in-kernel waits are bounded; nsa_sel_select_status() reports one that ran out. */
int nsa_sel_select(const void* q, const void* k, float* kblk_workspace, int32_t* sel_out, int32_t B, int32_t Hq,
                   int32_t Hkv, int32_t T, int32_t d, int32_t l_prime, int32_t n_sel, int32_t cmp_block,
                   int32_t cmp_stride, nsa_stream_t stream);

/* Bytes of the workspace nsa_sel_select needs (B * Hkv * ceil(T / l_prime) * d * 4), -1 if
   an argument is not positive. */
int64_t nsa_sel_select_workspace_bytes(int32_t B, int32_t Hkv, int32_t T, int32_t d, int32_t l_prime);

/* nsa_sel_select without a caller workspace and without any allocation: the block-key table is
   kept in a static device array of nsa_sel_select_static_scratch_bytes() bytes inside the
   library (its address is resolved once per device with cudaGetSymbolAddress; the library
   never calls cudaMalloc).  Requests whose workspace would exceed it return
   NSA_ERR_UNSUPPORTED without launching.  The scratch is shared per device: calls on one device
   must not run concurrently on different streams. */
int nsa_sel_select_noalloc(const void* q, const void* k, int32_t* sel_out, int32_t B, int32_t Hq, int32_t Hkv,
                           int32_t T, int32_t d, int32_t l_prime, int32_t n_sel, int32_t cmp_block,
                           int32_t cmp_stride, nsa_stream_t stream);

/* Backward of the selected-branch forward.  The reference has no backward pass (its README
   (2).md:85 lists it as missing); these entry points give the gradients of the same attention
   (ref_only.py:2-20, nsa_reference.py:18-25) with respect to Q, K and V:
       P = exp(scale * q.k - LSE),  dP = dO . v,  dS = P * (dP - sum_d dO * O),
       dQ = scale * dS K,  dK = scale * dS^T Q,  dV = P^T dO
   over the keys each query token sees in the forward (per-token selection, BQ == 1; same
   duplicate, padding and causal rules).  Supported: d_qk == d_v == 128, G = Hq / Hkv in {8, 16},
   l_prime in {64, 128, 256}, no cu_seqlens.  Zero-initialise, then fill the fields. */
typedef struct nsa_sel_bwd_desc {
  const void* q;              /* bf16 [B, Hq, T, 128] */
  const void* k;              /* bf16 [B, Hkv, T, 128] */
  const void* v;              /* bf16 [B, Hkv, T, 128] */
  const int32_t* sel;         /* int32 [B, Hkv, T, KSEL] */
  const void* o;              /* the forward's O [B, Hq, T, 128], dtype o_dtype */
  const float* lse;           /* the forward's LSE, fp32 [B, Hq, T] */
  const void* d_o;            /* bf16 [B, Hq, T, 128]: gradient of the loss with respect to O */
  float* dq;                  /* fp32 [B, Hq, T, 128]  } accumulated into (atomic adds): */
  float* dk;                  /* fp32 [B, Hkv, T, 128] } zero them first for plain gradients */
  float* dv;                  /* fp32 [B, Hkv, T, 128] } */
  void* workspace;            /* nsa_sel_backward_workspace_bytes() bytes, 16-byte aligned */
  int32_t* err;               /* optional device int32; NSA_DEVERR_* bits are ORed into it */
  int32_t batch, heads_q, heads_kv, seq_len, d;
  int32_t n_sel;              /* KSEL */
  int32_t block_size;         /* l_prime: 64, 128 or 256 */
  int32_t o_dtype;            /* NSA_DTYPE_BF16 or NSA_DTYPE_F32 */
  float scale;                /* softmax scale of the forward; <= 0 selects 1/sqrt(d) */
  int32_t timeout_ms;         /* bound on every in-kernel wait; 0 = default (2000 ms) */
  int32_t max_ctas;           /* 0 = one CTA per SM */
  int32_t reserved[5];
} nsa_sel_bwd_desc;

/* Bytes of the workspace nsa_sel_backward needs for a description, or -1 if the description is
   invalid (see nsa_sel_last_error()): the row sums dO . O (4 * B*Hq*T bytes) and the inverse
   selection index, i.e. about 4.2 bytes per (token, selected 64-key sub-block) pair (at most
   B*Hkv*T*KSEL*l_prime/64 of them) plus 32 bytes per bucket, a bucket being one (b, kvh, token
   window, sub-block): B*Hkv * ceil(T/64) * (number of windows, at most 32). */
int64_t nsa_sel_backward_workspace_bytes(const nsa_sel_bwd_desc* desc);

/* Adds dQ, dK, dV for the description on `stream` (six kernel launches and one memset, no
   allocation, asynchronous): the row sums dO . O, the inverse index (per (b, kvh, 64-key
   sub-block) the tokens that attend to it) and the tcgen05 gradient kernel.  The sums are
   accumulated with atomic adds, so the last bits may differ between runs. */
int nsa_sel_backward(const nsa_sel_bwd_desc* desc, nsa_stream_t stream);

/* ------------------------------------------------------------------ 4-bit paged KV cache
   The reference has no cache and no form for single tokens.  These functions keep a sequence's keys and
   values in 4.5 bits a value and attend to them, one token (or a few) of a sequence at a time.

   The cache is num_pages pages of 64 tokens.  Page p of KV head h is a record of nsa_cache_record_bytes(d_qk, d_v)
   = 36 * (d_qk + d_v) bytes at cache + p * page_stride + h * record bytes:
       K codes [64][d_qk / 2], K scales [64][d_qk / 16], V codes [64][d_v / 2], V scales [64][d_v / 16].
   16 neighbouring values along d share a scale byte, 5 exponent bits (bias 15) over 3 mantissa bits, no sign: `byte << 7`
   is the scale in half precision.  A code has 4 bits, sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6
   and the same with the sign; the low nibble is the even index.  Writing takes the scale nearest to max|x| / 6 (at most
   10240) and the codes nearest to x / scale, ties to even, and saturates (beyond 61440).  Groups whose largest |x| is
   below 2.3e-5 become zeros; a group that holds a NaN or an infinity reads back as NaNs.  A value has at most 6
   significant bits, so reading back into bf16, fp16 or fp32 is exact.

   (d_qk, d_v) is (64, 64), (128, 128), (192, 128) or (128, 64), as in the forward.

   The batch, the same for all three calls: sequence s has lens[s] tokens (the call's own included), token t of it is at
   place t % 64 of page pages[s][t / 64].  The call has n_rows rows; row r of sequence s (cu_seqlens[s] <= r <
   cu_seqlens[s + 1]) is the token at position lens[s] - (cu_seqlens[s + 1] - r), so a sequence's rows are its last tokens;
   without cu_seqlens row r is the last token of sequence r, and n_rows == n_seqs.  The device arrays are trusted for
   nothing: a token at a negative position, behind the page table's width or on a page outside [0, num_pages) is absent: it
   is not written, reads back as zeros and is not attended to.  (In a cu_seqlens that is out of order a row is of any one of
   the sequences whose range holds it, or of none.)  Two rows that name one place of the cache (two sequences that write
   to a shared page) leave a mixture of both there. */
typedef struct nsa_cache_batch {
  void* cache;                /* see above; 16-byte aligned (only nsa_cache_write changes it) */
  const int32_t* pages;       /* int32 [n_seqs, width] */
  const int32_t* lens;        /* int32 [n_seqs] */
  const int32_t* cu_seqlens;  /* optional int32 [n_seqs + 1] */
  int64_t page_stride;        /* bytes from one page to the next; 0 = heads_kv records, else a multiple of 16 not below */
  int64_t pages_stride;       /* entries from one row of `pages` to the next; 0 = width */
  int32_t num_pages, n_seqs, width, n_rows, heads_kv, d_qk, d_v;
  int32_t reserved;
} nsa_cache_batch;

/* Bytes of a record (one page of one KV head), -1 for a (d_qk, d_v) outside the built family. */
int64_t nsa_cache_record_bytes(int32_t d_qk, int32_t d_v);

/* Quantises the rows' K [n_rows, heads_kv, d_qk] and V [n_rows, heads_kv, d_v] into the cache; in_dtype NSA_DTYPE_BF16 or
   NSA_DTYPE_F16.  Strides in elements (multiples of 8; d has unit stride), pointers 16-byte aligned.  One launch.  Rows
   that must not meet: the call does not order itself against calls on other streams. */
int nsa_cache_write(const nsa_cache_batch* batch, const void* k, const void* v, int64_t k_row_stride, int64_t k_head_stride,
                    int64_t v_row_stride, int64_t v_head_stride, int32_t in_dtype, nsa_stream_t stream);

/* Reads the rows back: k [heads_kv, n_rows, d_qk], v [heads_kv, n_rows, d_v] (the packed layout of the varlen forward),
   contiguous, 32-byte aligned, dtype NSA_DTYPE_BF16, _F16 or _F32.  Absent tokens and rows of no sequence read as zeros.
   One launch. */
int nsa_cache_read(const nsa_cache_batch* batch, void* k, void* v, int32_t out_dtype, nsa_stream_t stream);

/* Attention of the rows over the cache: row n at position t sees key p iff p <= t, and t - p < window (if window > 0),
   and p lies in one of the blocks sel[n][kvh] (if sel is given; block_size keys each, a set as in the forward; entries < 0
   or behind t select nothing; n_sel at most 1024).  n_rows * heads_kv * tiles * (pages that a row may see: n_sel * block_size /
   64 with sel, else the table's width or the window's pages) is at most 2^31 - 1, where a KV head with up to 8 query heads is
   one tile and one with more has a tile for each 16 of them.  Beyond either: NSA_ERR_UNSUPPORTED.  A row that sees no key gets O = 0 and LSE = -inf.  Zero-initialise, then fill. */
typedef struct nsa_cache_attend_desc {
  nsa_cache_batch batch;
  const void* q;              /* [n_rows, heads_q, d_qk], dtype q_dtype, d has unit stride, 16-byte aligned */
  const int32_t* sel;         /* optional int32 [n_rows, heads_kv, n_sel] */
  void* o;                    /* [n_rows, heads_q, d_v], dtype o_dtype, contiguous, 16-byte aligned */
  float* lse;                 /* optional fp32 [n_rows, heads_q], natural log */
  const float* o_weight;      /* optional device float w multiplying the result; NULL = 1 */
  void* workspace;            /* nsa_cache_attend_workspace_bytes() bytes, 16-byte aligned, of this call alone */
  int32_t* err;               /* optional device int32; NSA_DEVERR_* bits are ORed into it */
  int64_t q_row_stride;       /* elements, multiples of 8; 0 = heads_q * d_qk */
  int64_t q_head_stride;      /* 0 = d_qk */
  int32_t heads_q;            /* a multiple of heads_kv */
  int32_t n_sel;
  int32_t block_size;         /* l_prime of sel: 64, 128 or 256 */
  int32_t window;             /* > 0: sliding window; 0: none */
  int32_t q_dtype;            /* NSA_DTYPE_BF16 or NSA_DTYPE_F16 */
  int32_t o_dtype;            /* q_dtype or NSA_DTYPE_F32 */
  int32_t o_accumulate;       /* 1: O += w * result (fp32 O only) */
  int32_t keep_rows;          /* 0: rows of no sequence get O = 0, LSE = -inf; 1: they are left as they were */
  float scale;                /* softmax scale; <= 0 selects 1/sqrt(d_qk) */
  int32_t timeout_ms;         /* bound on every in-kernel wait; 0 = default (2000 ms) */
  int32_t debug_flags;        /* NSA_DEBUG_STALL: nothing is copied, so that the waits run out; 0 in normal use */
  int32_t reserved[5];
} nsa_cache_attend_desc;

/* How nsa_cache_attend would run on a device of sm_count SMs (<= 0: the current device). */
typedef struct nsa_cache_attend_plan_info {
  int64_t workspace_bytes;
  int32_t slots;              /* (row, KV head) x page slots of a row; 0 = as many as it has pages, and then the next two are
                                 worked out on the device (0) */
  int32_t team;               /* warps of a block that take turns at a row's slots */
  int32_t cluster;            /* blocks of a cluster that share each row; 1 = none */
  int32_t share;              /* whole rows of a team, or its slots where rows are cut (merge != 0) */
  int32_t grid, threads, smem_bytes;
  int32_t merge;              /* warps that join the parts of a cut row's head; 0 = no row is cut, one launch */
  int32_t tiles;              /* tiles of a KV head's query heads: one of up to 8, or as many of 16 as they need */
} nsa_cache_attend_plan_info;
int nsa_cache_attend_plan(const nsa_cache_attend_desc* desc, int32_t sm_count, nsa_cache_attend_plan_info* out);

/* Bytes of the workspace on the current device, or -1 if the description is invalid (see nsa_sel_last_error()). */
int64_t nsa_cache_attend_workspace_bytes(const nsa_cache_attend_desc* desc);

/* Queues the attention (one or two launches).  Results do not depend on timing: the parts of a row are joined in a
   fixed order. */
int nsa_cache_attend(const nsa_cache_attend_desc* desc, nsa_stream_t stream);

/* ------------------------------------------------------------------ around the cache: pages, selection, positions
   What a decode step needs before it attends.  Nothing here has a counterpart in the reference. */

/* Gives the sequences of a batch the pages for their next tokens, or takes pages back, and works out where the rows of the
   call lie.  Sequence s holds held[s] tokens (below 0: none; more than the table has room for: as many as that).
     rows[s] > 0   it asks for that many more.  It gets them if the table has room, and if the pages that it and all sequences
                   before it still need are there (a sequence whose last page has room needs none, and gets its rows always).
                   Otherwise it stays as it is and has no rows in this call.
     rows[s] < 0   it gives its last -rows[s] tokens back (all of them if it has no more), and the pages that they alone filled.
     rows[s] == 0  it has no part in this call.
   `pool` holds the free pages, pool[0] to pool[n_free[0] - 1].  Pages that are given back are added behind them, in the order
   of the sequences and of their pages, before any are taken (those that pool_size leaves no room for are lost); then the
   last pages of the pool are taken, in its order, by the sequences in theirs.  The rows of `pages` get the pages that are taken;
   what stood there for pages that are given back stays.  A page that two sequences share would come back twice: it must not be
   given back here before the other one has ended.
   Results:
     held_out [n_seqs]      tokens after the call       (may be `held`)
     n_free_out [1]         free pages after it         (may be `n_free`)
     lens [n_seqs]          as nsa_cache_batch wants them: held_out for sequences that got rows, 0 for all others
     cu_seqlens [n_seqs+1]  sums of the rows that were asked for, so that a caller's packed rows keep their places (those of
                            a sequence that got none are absent: its lens is 0); at most 2^31 - 1.  NULL: row s is sequence
                            s's last token, and n_rows == n_seqs
     positions [n_rows]     optional: a row's position in its sequence, -1 for an absent row
     slots [n_rows]         optional: 64 * page + position % 64, -1 for an absent row
   With held_out and n_free_out apart from held and n_free nothing that counts is changed, so that a call can be tried, dropped
   and made again.  n_seqs is at most 8192 and n_seqs * width below 2^31.  Device arrays are trusted for nothing but pages
   (copied, never used as an index); one that is not aligned to its element size is refused, as are positions and slots that
   are not aligned to 16 bytes.  One launch. */
typedef struct nsa_cache_reserve_desc {
  int32_t* pages;             /* int32 [n_seqs, width] */
  const int32_t* held;
  const int32_t* rows;
  int32_t* pool;              /* int32 [pool_size] */
  const int32_t* n_free;
  int32_t* held_out;
  int32_t* n_free_out;
  int32_t* lens;
  int32_t* cu_seqlens;
  int32_t* positions;
  int64_t* slots;
  int64_t pages_stride;       /* entries from one row of `pages` to the next; 0 = width */
  int32_t n_seqs, width, pool_size, n_rows;
  int32_t reserved[4];
} nsa_cache_reserve_desc;

int nsa_cache_reserve(const nsa_cache_reserve_desc* desc, nsa_stream_t stream);

/* Block selection for single tokens: nsa_sel_select's rows for the tokens of a batch, from the compressed keys that a 4-bit
   cache holds.  batch.cache and batch.pages are the compressed cache's; batch.lens are the tokens of the sequences themselves,
   so that the row at position t sees T = t + 1 tokens as nsa_sel_select sees a sequence of T: n_cmp = (T - cmp_block) /
   cmp_stride + 1 compressed keys, key i (place i of the cache) in block floor(linspace(0, T-1, n_cmp)[i] / block_size), and
       score(block) = sum over its keys of (sum of the query heads of the KV head) . key.
   sel [n_rows, heads_kv, n_sel]: the min(n_sel, ceil(T / block_size)) best blocks, the best first, then -1.  Blocks are ranked
   by sums in 64 bits; the lower block comes first where two are equal, and scores that are not finite come last: all of them where
   the query is not finite, so that the lowest blocks are selected.  Keys that the page table does not hold count as zeros.  A row of no token, and one of more than 2^24 tokens or of more than
   64 * width * cmp_stride + cmp_block - 1 (whose keys the table cannot hold), selects nothing: -1 throughout.
   n_sel is at most 1024, heads_q / heads_kv at most 256.  Zero-initialise, then fill.  Two launches for each 1024 rows. */
typedef struct nsa_cache_select_desc {
  nsa_cache_batch batch;
  const void* q;              /* [n_rows, heads_q, d_qk], dtype q_dtype, d has unit stride, 16-byte aligned */
  int32_t* sel;               /* int32 [n_rows, heads_kv, n_sel] */
  void* workspace;            /* nsa_cache_select_workspace_bytes() bytes, 16-byte aligned, of this call alone */
  int64_t q_row_stride;       /* elements, multiples of 8; 0 = heads_q * d_qk */
  int64_t q_head_stride;      /* 0 = d_qk */
  int32_t heads_q;            /* a multiple of heads_kv */
  int32_t n_sel;
  int32_t block_size;         /* l_prime: 64, 128 or 256 */
  int32_t cmp_block, cmp_stride;
  int32_t q_dtype;            /* NSA_DTYPE_BF16 or NSA_DTYPE_F16 */
  int32_t reserved[4];
} nsa_cache_select_desc;

/* Bytes of the workspace, or -1 if the description is invalid (see nsa_sel_last_error()): 8 for each block of the longest
   sequence that the table can hold, KV head and row of a launch, however long the sequences are. */
int64_t nsa_cache_select_workspace_bytes(const nsa_cache_select_desc* desc);
int nsa_cache_select(const nsa_cache_select_desc* desc, nsa_stream_t stream);

/* Rotary positions of one to four axes (time, height, width): values a_i, b_i of a head become a_i cos w - b_i sin w and
   b_i cos w + a_i sin w with w = position[axis[i]] * inv_freq[i], for the `pairs` pairs i of the rotary part, which begins at
   value `offset`: values i and i + pairs of it, or 2 i and 2 i + 1 if `interleaved`.  The other values are copied.  `inverse`
   turns by -w: the gradient.  inv_freq is given as turns[i] = round(inv_freq[i] / (2 pi) * 2^64) modulo 2^64, so that angles of
   any int32 position are reduced to an eighth of a turn with an error below 2^-32 of a turn; that angle is then rounded to fp32 (2^-28
   of a turn at most), and so are its sine and cosine.  One or two tensors (Q and K) with the same tokens, in any layout in which d
   has unit stride; y may be x where their strides are equal.  turns and axis are host arrays, read before the call returns.  One
   launch. */
typedef struct nsa_rotary_tensor {
  const void* x;              /* NULL: no second tensor */
  void* y;
  int64_t x_stride[3];        /* elements from one batch entry, head, token to the next */
  int64_t y_stride[3];
  int32_t heads;
  int32_t reserved;
} nsa_rotary_tensor;

typedef struct nsa_rotary_desc {
  nsa_rotary_tensor t[2];
  const int32_t* positions;   /* device int32 */
  int64_t pos_stride[3];      /* elements from one axis, batch entry, token to the next */
  const uint64_t* turns;      /* host [pairs] */
  const uint8_t* axis;        /* host [pairs], below axes; NULL: all 0 */
  int32_t batch, tokens;      /* tokens of each batch entry */
  int32_t d;                  /* values of a head, at most 256 */
  int32_t offset, pairs, axes;
  int32_t interleaved, inverse;
  int32_t dtype;              /* NSA_DTYPE_BF16, _F16 or _F32, of x and y */
  int32_t reserved[3];
} nsa_rotary_desc;

int nsa_rotary(const nsa_rotary_desc* desc, nsa_stream_t stream);

/* Size in bytes of the static scratch used by nsa_sel_select_noalloc. */
int64_t nsa_sel_select_static_scratch_bytes(void);

/* NSA_DEVERR_* bits that selection launches on the current device set since the last call (0 =
   none), cleared on return; -1 if the device cannot be queried.  Synchronous: it waits for the
   device's pending work through a blocking copy. */
int32_t nsa_sel_select_status(void);

/* Text of the last error on this host thread ("" if none). */
const char* nsa_sel_last_error(void);

/* NSA_SEL_VERSION of the loaded library. */
int32_t nsa_sel_version(void);

#ifdef __cplusplus
}
#endif

#endif /* NSA_SEL_H_ */
