/*
 * flashattn_tile_b200 -- C ABI of the B200 (sm_100a) paged-attention library.
 *
 * Every entry point takes raw device pointers, element strides (in elements,
 * the innermost dimension must be contiguous), plain integer sizes and a
 * cudaStream_t passed as void*.  Nothing here allocates device memory except
 * where a function says so; scratch space is passed in by the caller.
 *
 * Each function returns a fat_status.  On failure fat_last_error() holds a
 * message for the calling thread.  Kernels that can detect a problem only on
 * the device (a page id outside the pool, a pipeline wait that timed out)
 * OR a FAT_DEVERR_* bit into the caller's int32 device error word and
 * finish without faulting; the caller reads the word when it wants to know.
 *
 * Reference interface replaced (FlashAttnTile, path:line in that project):
 *   fat_paged_decode          flashattn_tile/ops.py:35-55 (flashattn_tile::paged_decode),
 *                             kernels/decode.py:533-642 (paged_decode_attention),
 *                             kernels/decode.py:645-704 (paged_decode_attention_fp8),
 *                             csrc/paged_decode.cu:297-344 (paged_decode_cuda)
 *   fat_prefill_varlen        flashattn_tile/ops.py:76-99 (flashattn_tile::prefill_varlen),
 *                             kernels/prefill.py:236-326 (prefill_attention)
 *   fat_gather_paged          flashattn_tile/paging.py:213-256 (gather_paged)
 *   fat_lse_merge             kernels/decode.py:316-356 (_decode_reduce_kernel)
 *   fat_prefill_paged         no counterpart: prefill (kernels/prefill.py:34-138 semantics) with
 *                             K/V read through the page table instead of packed tensors
 *                             (the reference's backend requires packed K/V, backend.py:158-162)
 *   fat_append_tokens         flashattn_tile/paging.py:172-210 (append_tokens); for 8-bit
 *                             caches also quant.py:84-142 (per-page scales, applied on write)
 */
#ifndef FLASHATTN_TILE_B200_H_
#define FLASHATTN_TILE_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes. */
enum {
  FAT_OK = 0,
  FAT_ERR_INVALID_ARGUMENT = 1, /* shapes, strides, pointers or values are inconsistent */
  FAT_ERR_UNSUPPORTED = 2,      /* a valid request this build has no kernel for       */
  FAT_ERR_CUDA = 3,             /* a CUDA runtime call or kernel launch failed         */
  FAT_ERR_WORKSPACE = 4         /* the scratch buffer passed in is too small           */
};

/* Bits OR-ed into the device error word. */
enum {
  FAT_DEVERR_TIMEOUT = 1,    /* a bounded pipeline wait gave up; the output is invalid  */
  FAT_DEVERR_BAD_PAGE = 2,   /* a page id used by a sequence is outside [0, num_pages) */
  FAT_DEVERR_BAD_LENGTH = 4, /* a sequence length exceeds the page table's capacity
                                (max_pages * page_size); it was cut to that capacity   */
  FAT_DEVERR_NO_PAGE = 8,    /* a row asked for more pages than were free, or was to
                                append to a page that it does not hold alone           */
  FAT_DEVERR_BAD_ROW = 16,   /* a row index outside the page table; it was skipped     */
  FAT_DEVERR_BAD_GROUP = 32  /* group edges that fall or leave the batch, or a group of
                                more than max_group sequences (read without sharing)   */
};

/* Element types. */
enum {
  FAT_DTYPE_F16 = 0,
  FAT_DTYPE_BF16 = 1,
  FAT_DTYPE_F32 = 2,
  FAT_DTYPE_I8 = 3,  /* symmetric int8 with per-(page, kv head) fp32 scales */
  FAT_DTYPE_E4M3 = 4 /* float8_e4m3fn with per-(page, kv head) fp32 scales  */
};

/* Library version string, e.g. "flashattn_tile_b200 0.1.0 sm_100a". */
const char* fat_version(void);

/* Message of the last failed call on this thread ("" if none). */
const char* fat_last_error(void);

/* Time limit of every bounded wait inside the decode and prefill kernels,
 * for launches made after this call, from any thread (default 2 s; 0 restores
 * it).  A wait that runs out sets FAT_DEVERR_TIMEOUT; the kernel then drains
 * its own copies and tensor-core work and returns.  Returns the previous limit.
 * No reference counterpart: the reference's Triton and CUDA kernels have no
 * in-kernel waits. */
uint64_t fat_set_wait_limit_ns(uint64_t limit_ns);

/* Which capture `stream` is in (a number of its own for each), 0 when it is in none: what a
 * call of a captured graph is given (workspace, scratch) is that graph's to use for as long
 * as it is replayed, so a caller keeps it apart from what it hands to other calls. */
uint64_t fat_stream_capture_id(void* stream);

/* Failure-path testing: each of the next `launches` decode or prefill kernel
 * launches (from any thread) first waits on a barrier phase that nothing
 * completes, so that this wait runs out after the wait limit and the launch
 * ends with FAT_DEVERR_TIMEOUT (no fault, no hang).  0 cancels requests not
 * yet taken.  No reference counterpart. */
void fat_expire_next_waits(int launches);

/* How the prefill kernels feed the probabilities P into the P.V product, for
 * launches made after this call, from any thread.  The reference kernel
 * rounds P to the input dtype once (kernels/prefill.py:128); with bf16's 8-bit
 * significand that alone moves outputs of rows with few keys by up to ~4e-3.
 *   -1  automatic (default): bf16 uses mode 3 (paged K/V: mode 1), fp16 mode 0
 *    0  P rounded to the input dtype once (the reference's arithmetic)
 *    1  a key tile's P enters as a 16-bit head plus a 16-bit remainder (a
 *       second P.V pass over that tile; ~2^-16 relative) when one of its keys
 *       holds more than 1/16 of its row's probability sum so far; every other
 *       key ends with weight <= 1/16, so its rounding moves an output by at
 *       most 2^-12 of |v|
 *    2  head plus remainder on every key tile (twice the P.V work)
 *    3  bf16 with packed K/V: P.V in fp16 -- P rounded to fp16 (~2^-12
 *       relative), V read from an fp16 copy made by a pre-pass (two small
 *       kernels on the call's stream) and scaled by 2^-e per (sequence, KV
 *       head) so that any finite bf16 V fits, the output scaled back by 2^e.
 *       The copy lives in a per-(device, stream) buffer of total_k * kv_heads *
 *       head_dim * 2 bytes, grown on demand and never freed; a stream whose
 *       buffer must grow while it is captured into a graph uses mode 1.  fp16
 *       inputs treat it as mode 0, paged K/V as mode 1
 * Returns the previous setting, or -2 (message in fat_last_error) for a mode
 * outside [-1, 3].  No reference counterpart. */
int fat_set_prefill_p_split(int mode);

/*
 * Grid of the prefill launches made from now on (process-wide; both prefill
 * entry points, all dtypes):
 *    0  persistent (default): one CTA per SM, each claiming (head, sequence,
 *       256-row query pair) items, heaviest first, from a per-stream counter
 *       until none is left, so an item's first loads and Q.K^T overlap the
 *       previous item's last softmax and output stores.  The counter (8 bytes
 *       of device memory per stream) is made on a stream's first prefill; a
 *       stream first used while it is being captured into a graph runs mode 1
 *    1  one CTA per item
 * Results are bitwise identical.  Returns the previous setting, or -2 (message
 * in fat_last_error) for another value.  No reference counterpart. */
int fat_set_prefill_schedule(int mode);

/*
 * Bytes of scratch fat_paged_decode needs for this problem on `device`.
 * The caller zero-fills the buffer once; every successful call leaves it
 * zero-filled again, so one buffer serves any number of calls that are
 * ordered on one stream.
 */
size_t fat_paged_decode_workspace_size(int device, int batch, int num_heads, int num_kv_heads, int head_dim);

/*
 * Single-query paged decode: out[b, h, :] = softmax(scale * q[b, h] . K^T) V over
 * the seq_lens[b] cached tokens of sequence b, K/V read through the page table
 * (token t in page page_table[b, t / page_size], slot t % page_size), query head
 * h reading KV head h / (num_heads / num_kv_heads).
 *
 *   q          [batch, num_heads, head_dim]          q_dtype (F16 | BF16)
 *   k/v_cache  [num_pages, page_size, num_kv_heads, head_dim]
 *              kv_dtype = q_dtype, or I8 / E4M3 with k/v_scale [num_pages, num_kv_heads] fp32
 *   page_table int32 [batch, >= ceil(max seq_len / page_size)]
 *   seq_lens   int32 [batch]; a sequence of length 0 produces zeros
 *   out        [batch, num_heads, head_dim]          out_dtype (= q_dtype, or F32)
 *
 * head_dim in {32, 64, 128, 256}; page_size 8 or a multiple of 16 up to 256; K/V
 * base addresses 16-byte aligned and their page/slot/head strides multiples of
 * 16 bytes.  split_k_hint (1..64) is accepted for interface compatibility: the
 * kernel chooses its own balanced split of the pages over all SMs, and the
 * result does not depend on it.
 */
int fat_paged_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_cache,
                     const void* v_cache, int64_t kv_stride_page, int64_t kv_stride_slot, int64_t kv_stride_head,
                     int64_t num_pages, const int32_t* page_table, int64_t page_table_stride, int64_t max_pages,
                     const int32_t* seq_lens, const float* k_scale, const float* v_scale,
                     int64_t scale_stride_page, void* out, int64_t out_stride_b, int64_t out_stride_h, int batch,
                     int num_heads, int num_kv_heads, int head_dim, int page_size, int q_dtype, int kv_dtype,
                     int out_dtype, float softmax_scale, int split_k_hint, void* workspace, size_t workspace_bytes,
                     int32_t* error_word, void* stream);

/*
 * fat_paged_decode_lse's arguments in one struct, for callers that keep them
 * between calls (an op whose tensors stay put from step to step pays the
 * argument conversion once and changes only `out`).  With `stats_out` set,
 * the call first queues fat_cache_value_stats(seq_lens, page_table, ...,
 * stats_scratch, stats_out) on the same stream (and records `stats_event`
 * after it), so value checks and decode cost one crossing; `lse` may be NULL.  Same status codes and device error
 * word as fat_paged_decode.  No reference counterpart (a calling convention).
 */
typedef struct fat_decode_call {
  const void* q;
  int64_t q_stride_b, q_stride_h;
  const void* k_cache;
  const void* v_cache;
  int64_t kv_stride_page, kv_stride_slot, kv_stride_head, num_pages;
  const int32_t* page_table;
  int64_t page_table_stride, max_pages;
  const int32_t* seq_lens;
  const float* k_scale;
  const float* v_scale;
  int64_t scale_stride_page;
  void* out;
  int64_t out_stride_b, out_stride_h;
  float* lse;
  int64_t lse_stride_b;
  int32_t batch, num_heads, num_kv_heads, head_dim, page_size;
  int32_t q_dtype, kv_dtype, out_dtype;
  float softmax_scale;
  int32_t split_k_hint;
  void* workspace;
  size_t workspace_bytes;
  int32_t* error_word;
  void* stream;
  int32_t* stats_out;      /* optional: 4 int32 (pinned host or device), see fat_cache_value_stats */
  int32_t* stats_scratch;  /* 4 int32 on the device, used with stats_out */
  void* stats_event;       /* optional cudaEvent_t, recorded on `stream` right after the statistics: a
                              host that waits on it to check the values does not wait for the decode */
} fat_decode_call;

int fat_paged_decode_call(const fat_decode_call* call);

/*
 * fat_paged_decode that also writes, per (sequence, query head), the base-2
 * log-sum-exp of the scaled scores, lse[b * lse_stride_b + h] = m + log2(l)
 * (-inf for a sequence with no cached tokens).  With out_dtype F32 the pair
 * (out, lse) is the partial a sequence-parallel decode exchanges: decode each
 * GPU's own key range (a page-table column slice with per-GPU lengths), gather
 * the partials, combine them with fat_lse_merge.  Replaces the split-K partial
 * outputs of FlashAttnTile's _decode_paged_split_kernel (kernels/decode.py:223-313).
 */
int fat_paged_decode_lse(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_cache,
                         const void* v_cache, int64_t kv_stride_page, int64_t kv_stride_slot, int64_t kv_stride_head,
                         int64_t num_pages, const int32_t* page_table, int64_t page_table_stride, int64_t max_pages,
                         const int32_t* seq_lens, const float* k_scale, const float* v_scale,
                         int64_t scale_stride_page, void* out, int64_t out_stride_b, int64_t out_stride_h,
                         float* lse, int64_t lse_stride_b, int batch, int num_heads, int num_kv_heads, int head_dim,
                         int page_size, int q_dtype, int kv_dtype, int out_dtype, float softmax_scale,
                         int split_k_hint, void* workspace, size_t workspace_bytes, int32_t* error_word,
                         void* stream);

/*
 * Merge `parts` attention partials over disjoint key ranges:
 *   out[row] = sum_r o[r][row] 2^(lse[r][row] - M) / sum_r 2^(lse[r][row] - M),  M = max_r lse[r][row]
 * o: fp32 [parts][rows][head_dim] (part r at o + r * o_part_stride), lse: fp32 [parts][rows]
 * (part r at lse + r * lse_part_stride), out: [rows][head_dim] of out_dtype (F16 | BF16 | F32),
 * lse_out: optional [rows] merged log-sum-exp.  Rows whose parts are all -inf give zeros.
 * Replaces FlashAttnTile's _decode_reduce_kernel (kernels/decode.py:316-356).
 */
int fat_lse_merge(const float* o, int64_t o_part_stride, const float* lse, int64_t lse_part_stride, int parts,
                  int64_t rows, int head_dim, void* out, int out_dtype, float* lse_out, void* stream);

/*
 * fat_paged_decode for callers that cannot allocate device memory.  No
 * counterpart exists in the reference: it is an addition for engines that
 * allocate every device buffer up front and forbid allocation afterwards,
 * plugins whose host framework gives them neither an allocator nor a scratch
 * pointer, and latency-critical loops where an allocation could synchronise
 * the device.  Same arguments and result as fat_paged_decode, minus the
 * workspace: the split scratch is a fixed 4 MiB array in this library's
 * device memory, held by every GPU that loads the library until the process
 * exits.  Problems whose scratch would exceed 4 MiB (about
 * fat_paged_decode_workspace_size) are refused with FAT_ERR_WORKSPACE.  The
 * first call on a device looks up the array's device address (once per
 * device; make that first call before any stream capture).  Each call clears
 * the tickets it uses on `stream`; all calls share the array, so calls that
 * overlap on the GPU race and must be ordered by the caller.  Allocates
 * nothing (no cudaMalloc / cudaFree).
 */
int fat_paged_decode_noalloc(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k_cache,
                             const void* v_cache, int64_t kv_stride_page, int64_t kv_stride_slot,
                             int64_t kv_stride_head, int64_t num_pages, const int32_t* page_table,
                             int64_t page_table_stride, int64_t max_pages, const int32_t* seq_lens,
                             const float* k_scale, const float* v_scale, int64_t scale_stride_page, void* out,
                             int64_t out_stride_b, int64_t out_stride_h, int batch, int num_heads, int num_kv_heads,
                             int head_dim, int page_size, int q_dtype, int kv_dtype, int out_dtype,
                             float softmax_scale, int split_k_hint, int32_t* error_word, void* stream);

/*
 * Packed varlen prefill: for every sequence b (tokens cu_q[b]..cu_q[b+1] of q and
 * cu_k[b]..cu_k[b+1] of k/v) and query head h,
 *   out = softmax(scale * q k^T [+ bottom-right causal mask]) v,
 * with query i seeing key j when j <= i + kv_len - q_len (causal), query head h
 * reading KV head h / (num_heads / num_kv_heads), P rounded to the input dtype
 * before P.V and fp32 accumulation.
 *
 *   q   [total_q, num_heads, head_dim], k/v [total_k, num_kv_heads, head_dim]   dtype (F16 | BF16)
 *   out [total_q, num_heads, head_dim]   out_dtype (= dtype, or F32)
 *   cu_q, cu_k  int32 [batch + 1], non-decreasing from 0 (not checked on the device)
 *
 * head_dim in {64, 128, 256}; all bases 16-byte aligned, token/head strides multiples
 * of 16 bytes.  max_seqlen_q bounds the launch grid (queries past it are not
 * computed).  Allocates nothing.
 */
int fat_prefill_varlen(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
                       int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h, void* out,
                       int64_t out_stride_t, int64_t out_stride_h, const int32_t* cu_seqlens_q,
                       const int32_t* cu_seqlens_k, int batch, int64_t total_q, int64_t total_k, int num_heads,
                       int num_kv_heads, int head_dim, int max_seqlen_q, int max_seqlen_k, int causal,
                       float softmax_scale, int dtype, int out_dtype, int32_t* error_word, void* stream);

/*
 * Prefill / chunked prefill over a paged cache: sequence b has q_len =
 * cu_seqlens_q[b+1] - cu_seqlens_q[b] queries (packed q, as fat_prefill_varlen)
 * that are the last q_len of its seq_lens_k[b] cached tokens; keys and values
 * are those tokens, read from k_cache/v_cache [num_pages, page_size, num_kv_heads,
 * head_dim] through page_table [batch, max_pages] (bottom-right causal alignment:
 * query i sees key j <= i + seq_lens_k[b] - q_len).  fp16/bf16; head_dim 64, 128 or 256 (256: page_size >= 16);
 * page_size a power of two in [8, 128] or a multiple of 128.  Rows past a
 * sequence's end never contribute; a page id outside [0, num_pages) is skipped
 * and ORs FAT_DEVERR_BAD_PAGE into *error_word.
 */
int fat_prefill_paged(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
                      const void* v_cache, int64_t kv_stride_page, int64_t kv_stride_slot, int64_t kv_stride_head,
                      int64_t num_pages, const int32_t* page_table, int64_t page_table_stride, int64_t max_pages,
                      const int32_t* cu_seqlens_q, const int32_t* seq_lens_k, void* out, int64_t out_stride_t,
                      int64_t out_stride_h, int batch, int64_t total_q, int num_heads, int num_kv_heads,
                      int head_dim, int page_size, int max_seqlen_q, int causal, float softmax_scale, int dtype,
                      int out_dtype, int32_t* error_word, void* stream);

/*
 * Append one token per sequence: new_k/new_v [batch, num_kv_heads, head_dim]
 * (element strides new_stride_b, new_stride_h; unit stride along head_dim) go to
 * page page_table[b, seq_lens[b] / page_size], slot seq_lens[b] % page_size, then
 * seq_lens[b] += 1 -- all on the device, no host synchronisation.  A position past
 * the page table or a page id outside [0, num_pages) leaves that sequence untouched
 * and ORs FAT_DEVERR_BAD_PAGE into *error_word.
 *   16-bit caches: new_dtype == kv_dtype, bit-exact copy; k_scale/v_scale unused.
 *   INT8 / FP8-e4m3 caches: new_dtype F16 | BF16 | F32; the page's fp32 scale
 *   (k_scale/v_scale [num_pages, num_kv_heads], stride scale_stride_page) becomes
 *   max(absmax / maxval, 1e-8) over this sequence's tokens on the page (earlier ones
 *   dequantised as code * scale) and the new token; earlier codes are requantised
 *   when the scale changed; the new token is quantised with it (int8: round half to
 *   even, clamp +-127; e4m3: clamp +-448, round to nearest even).
 */
int fat_append_tokens(void* k_cache, void* v_cache, int64_t kv_stride_page, int64_t kv_stride_slot,
                      int64_t kv_stride_head, int64_t num_pages, const int32_t* page_table, int64_t page_table_stride,
                      int64_t max_pages, int32_t* seq_lens, const void* new_k, const void* new_v,
                      int64_t new_stride_b, int64_t new_stride_h, float* k_scale, float* v_scale,
                      int64_t scale_stride_page, int batch, int num_kv_heads, int head_dim, int page_size,
                      int kv_dtype, int new_dtype, int32_t* error_word, void* stream);

/*
 * Page-table gather: out_k/out_v [batch, max_len, num_kv_heads, row_bytes] (contiguous)
 * receive, bit for bit, the rows of each sequence's first seq_lens[b] tokens, and
 * zeros past that.  The cache is addressed by byte strides (page, slot, head); the
 * element type does not matter (row_bytes = head_dim * element size).
 */
int fat_gather_paged(const void* k_cache, const void* v_cache, int64_t stride_page_bytes, int64_t stride_slot_bytes,
                     int64_t stride_head_bytes, int64_t num_pages, const int32_t* page_table,
                     int64_t page_table_stride, int64_t max_pages, const int32_t* seq_lens, void* out_k, void* out_v,
                     int64_t max_len, int batch, int num_kv_heads, int page_size, int64_t row_bytes,
                     int32_t* error_word, void* stream);

/*
 * Value statistics of a paged cache's metadata, for the host-side checks of
 * flashattn_tile/paging.py:84-130 (validate_cache): host_out[0..3] = min and max
 * of seq_lens[batch], then min and max of the page-table entries a sequence of
 * the maximum length reaches (the first ceil(max / page_size) columns of every
 * row, at most max_pages; (0, -1) when there are none).  Queues one kernel on
 * `stream`: when host_out is pinned host memory mapped into the device's
 * address space (cudaHostAlloc / cudaHostRegister memory, 16-byte aligned) the
 * kernel writes it directly, otherwise it writes device_scratch and a 16-byte
 * copy into host_out follows.  Synchronise the stream (or an event recorded
 * after this call) before reading host_out.  device_scratch: 4 int32 on the
 * device (unused when host_out is written directly).  Replaces
 * the reference's torch reductions + read-back of both tensors.
 */
int fat_cache_value_stats(const int32_t* seq_lens, const int32_t* page_table, int64_t page_table_stride, int batch,
                          int64_t max_pages, int page_size, int32_t* device_scratch, int32_t* host_out, void* stream);

/*
 * Pages shared between sequences.  No counterpart in the reference, whose caches
 * give every sequence its own pages (paging.py:133-169).
 *
 * A pool is a paged K/V cache plus two counts: refs[page], the number of table
 * entries that hold the page (0: free), and owned[row], the number of leading
 * entries of a row that hold pages (later entries are never read; they become 0 where a
 * row gives pages back).  The operations below
 * keep both exact and run on the device without host synchronisation.  Their
 * results are whole numbers fixed by the arguments alone: the lowest free page
 * ids are taken first, rows are served in the order given.  Row lists hold
 * distinct rows; rows and page ids out of range are skipped and recorded in the
 * error word (FAT_DEVERR_BAD_ROW, FAT_DEVERR_BAD_PAGE).
 *
 * Strides of the K/V storage are in bytes; row_bytes = head_dim * element size.
 * k_scale/v_scale: optional fp32 [num_pages, num_kv_heads], moved with the pages.
 * released (optional, int32 [batch], zero at first): 1 for a row from its release until it
 * is a destination of a fork (which copies the source's mark) or reserved by name.  With
 * skip_released, fat_reserve_tokens without a row list and fat_append_to_pool leave such
 * rows as they are: a captured step may run while rows are idle.
 * scratch: fat_page_scratch_size bytes, zero-filled once; every call leaves its
 * counters zero again.  Calls that share a pool are ordered by the caller.
 */
typedef struct fat_page_pool {
  void* k_cache;
  void* v_cache;
  int64_t stride_page_bytes, stride_slot_bytes, stride_head_bytes, num_pages, row_bytes;
  float* k_scale;
  float* v_scale;
  int64_t scale_stride_page;
  int32_t* page_table;
  int64_t page_table_stride, max_pages;
  int32_t* seq_lens;
  int32_t* owned;
  int32_t* refs;
  void* scratch;
  size_t scratch_bytes;
  int32_t* error_word;
  void* stream;
  int32_t batch, num_kv_heads, page_size;
  int32_t skip_released;
  int32_t* released;
} fat_page_pool;

size_t fat_page_scratch_size(int64_t num_pages, int batch);

/* Page dst[i] <- page src[i] (K, V and scales), i < n.  The dst pages are distinct
 * and no page is both source and destination.  Uses the storage fields only. */
int fat_copy_pages(const fat_page_pool* pool, const int32_t* src, const int32_t* dst, int n);

/* Row dst[i] becomes a copy of row src[i]: its length, and the table entries of the
 * pages that length reaches, each counted once more; the pages that dst[i] held are
 * released.  All sources are read before any row changes (a row may be both).  No K/V moves. */
int fat_fork_sequences(const fat_page_pool* pool, const int32_t* src, const int32_t* dst, int n);

/* Rows rows[i] (NULL: rows 0..n-1) may append `tokens` more tokens each.  A partly
 * filled tail page that others hold too is copied to a free page; where all of its
 * holders are in the call, the last of them keeps it.  Missing pages are taken from
 * the free ones.  A row whose needs, added to those of the rows before it, exceed the
 * free pages is left as it is (FAT_DEVERR_NO_PAGE), and so is one whose table is too
 * narrow (FAT_DEVERR_BAD_LENGTH). */
int fat_reserve_tokens(const fat_page_pool* pool, const int32_t* rows, int n, int tokens);

/* Rows rows[i] give their pages back: counts - 1, entries 0, length and owned 0. */
int fat_release_sequences(const fat_page_pool* pool, const int32_t* rows, int n);

/* fat_append_tokens on a pool: one token per row of the table (rows 0..batch-1), written
 * only to a page that its row alone holds (otherwise FAT_DEVERR_NO_PAGE, and the row is
 * left unchanged): call fat_reserve_tokens first.  new_k/new_v: element strides. */
int fat_append_to_pool(const fat_page_pool* pool, const void* new_k, const void* new_v, int64_t new_stride_b,
                       int64_t new_stride_h, int kv_dtype, int new_dtype);

/* With L live pages, the k-th live page with id >= L moves to the k-th free id below
 * L.  The renamed table goes to table_out (row stride table_out_stride), the counts to
 * refs_out, L to live_out (optional); both may be the pool's own.  The pages moved
 * from keep their contents, so the old table stays readable until they are reused. */
int fat_compact_pages(const fat_page_pool* pool, int32_t* table_out, int64_t table_out_stride, int32_t* refs_out,
                      int32_t* live_out);

/*
 * Decode attention for groups of consecutive sequences that share a prefix: the
 * result of fat_paged_decode on the same cache, with the prefix of each group read
 * and multiplied once for all of its sequences.  No counterpart in the reference.
 *
 * Group g is sequences cu_groups[g] .. cu_groups[g + 1] - 1 (cu_groups int32
 * [num_groups + 1] from 0; sequences past the last group share nothing).  The page
 * tables of a group agree in the first prefix_lens[g] / page_size entries; a sequence
 * of length 0 takes no part (its table is not read, its output is zeros).  Another that
 * is shorter than that many pages is named (FAT_DEVERR_BAD_LENGTH), and its own output,
 * not that of the others, is then not meaningful.  Nor is that of a sequence with a page id
 * outside [0, num_pages), which is not loaded (FAT_DEVERR_BAD_PAGE).  A prefix that ends inside a page
 * is used up to the page's start.  No group has more than max_group sequences; one
 * that does is decoded as if it shared nothing (FAT_DEVERR_BAD_GROUP).  Where edges
 * fall (FAT_DEVERR_BAD_GROUP too) the output of the sequences that two groups claim is
 * not meaningful.
 *
 * `decode` holds the arguments of fat_paged_decode_call (lse and the stats_* fields
 * are not used; workspace as there).  scratch: fat_shared_prefix_scratch_size bytes
 * of any contents, one buffer per stream.
 */
typedef struct fat_shared_prefix_call {
  fat_decode_call decode;
  const int32_t* cu_groups;
  const int32_t* prefix_lens;
  int32_t num_groups, max_group;
  void* scratch;
  size_t scratch_bytes;
} fat_shared_prefix_call;

size_t fat_shared_prefix_scratch_size(int device, int batch, int num_heads, int num_kv_heads, int head_dim,
                                      int max_group);
int fat_shared_prefix_decode(const fat_shared_prefix_call* call);

/* prefix_out[g] = the tokens that group g shares: page_size * the leading page-table
 * entries in which all of its sequences agree, over whole pages that each of them
 * fills; 0 for a group of fewer than min_sequences. */
int fat_find_shared_prefix(const int32_t* page_table, int64_t page_table_stride, int64_t max_pages,
                           const int32_t* seq_lens, int batch, int page_size, const int32_t* cu_groups,
                           int num_groups, int min_sequences, int32_t* prefix_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FLASHATTN_TILE_B200_H_ */
