/*
 * ditango_b200 -- C ABI of the sm_100a kernels behind DiTango's sequence-parallel attention path.
 *
 * Every entry point takes plain device pointers, sizes and a CUDA stream handle
 * (cudaStream_t passed as void*), launches asynchronously on that stream and returns an int
 * status: 0 = launched; negative = rejected argument (nothing was launched, text in
 * dtb_last_error()).  Pointers are borrowed: the caller keeps the memory alive until the
 * stream has passed the call.  Nothing here allocates device memory.  The calling thread's
 * current CUDA device must be the one that owns the pointers.
 *
 * Citations name the reference call site each entry point replaces (paths relative to the
 * reference project root).
 */
#ifndef DITANGO_B200_H_
#define DITANGO_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define DTB_API __attribute__((visibility("default")))
#else
#define DTB_API
#endif

#define DTB_OK 0
#define DTB_ERR_ARG (-1)      /* unsupported shape / null pointer / misaligned pointer          */
#define DTB_ERR_CUDA (-2)     /* a CUDA runtime or driver call failed (launch, tensor map, ...) */
#define DTB_ERR_DEVICE (-3)   /* current device is not compute capability 10.x                  */

/* element types of partial-state outputs */
#define DTB_F32 0
#define DTB_BF16 1
/* values kept in 8 bits with one exponent byte per row (dtb_merge_rows only) */
#define DTB_I8 2
#define DTB_E4M3 3

/* layouts of a log-sum-exp tensor that belongs to tokens [B,S] x heads H
 * (packed inputs: B = 1, S = total tokens) */
#define DTB_LSE_BHS 0         /* [B, H, S]  -- what flash_attn returns                         */
#define DTB_LSE_BSH 1         /* [B, S, H]  -- the merged state's [B,S,H,1]                    */

#define DTB_MERGE_MAX_STATES 16

DTB_API int dtb_version(void);

/* Text of the last rejected call on this host thread ("" if none). */
DTB_API const char* dtb_last_error(void);

/* 0 if the current device can run these kernels (compute capability 10.x), else DTB_ERR_DEVICE. */
DTB_API int dtb_device_supported(void);

/*
 * Device-side status word.  Kernels that wait on hardware barriers bound every wait; a wait that
 * runs out records a non-zero code and the kernel returns without storing results.
 * dtb_read_status synchronises `stream`, returns the word (0 = all kernels completed normally)
 * and clears it.
 */
DTB_API int dtb_read_status(void* stream);

/*
 * The word is sticky: once a wait has run out, every later launch of these kernels sees a non-zero
 * word in its prologue and returns without doing its work, so that nothing runs on a pipeline whose
 * state is unknown -- and nothing is stored, so results from then on are not valid although every
 * launch call returns 0.  A caller must therefore look at the word, either with dtb_read_status at a
 * point where a synchronisation is acceptable, or without blocking: dtb_peek_status_async queues a
 * copy of the word into *host_word (pinned host memory, owned by the caller) on `stream`; the value
 * is valid once work queued before the call on that stream has completed (an event recorded behind
 * it has fired).  The reference has no counterpart; its failure mode for a stuck transfer is a hung
 * process (core/group_coordinate.py:664-668 waits without a limit).
 *
 * dtb_post_status lets the host set the word (code > 0), ordered on `stream`: a watchdog that learnt
 * on the host that a peer rank is gone uses it to make kernels in flight give up their waits (they
 * poll the word) and to stop later launches, instead of letting each wait run to its limit.
 *
 * The word is one per device: cleared while launches are in flight on other streams, it leaves what those store not valid, and unreported.
 */
DTB_API int dtb_peek_status_async(int* host_word, void* stream);
DTB_API int dtb_post_status(int code, void* stream);

/*
 * Copy-engine KV transport between the GPUs of one node.  Replaces the NCCL send / receive pairs behind
 * GroupCoordinator.p2p_isend / p2p_irecv / p2p_commit (core/group_coordinate.py:643-668) as used by
 * async_ring_p2p_commit (core/attention.py:37-62): the owner of a KV chunk writes it straight into a
 * receive buffer of the consumer with one asynchronous device-to-device copy, which a copy engine
 * executes -- no SM is taken from the attention kernel.
 *
 *  dtb_ipc_export_mem   consumer side: the 64-byte CUDA IPC handle of the allocation that contains
 *                       dev_ptr, and dev_ptr's byte offset inside it (the caller ships both to the peer).
 *  dtb_ipc_open_mem     owner side: maps the peer's allocation into this process for the CURRENT device
 *                       (peer access is enabled on demand) and returns its base address; add the offset.
 *                       Map a handle once and keep it; close it with dtb_ipc_close_mem at shutdown.
 *  dtb_peer_copy_async  one asynchronous copy of `bytes` from src to dst on `stream` (either may be
 *                       peer-mapped memory).  One call per copy.
 * Ordering between the two processes is the caller's job (interprocess CUDA events plus a host-side
 * handshake; see ditango_b200/core/peer_transport.py).  These calls allocate nothing.
 */
DTB_API int dtb_ipc_export_mem(const void* dev_ptr, void* handle64, int64_t* offset);
DTB_API int dtb_ipc_open_mem(const void* handle64, void** base_ptr);
DTB_API int dtb_ipc_close_mem(void* base_ptr);
DTB_API int dtb_peer_copy_async(void* dst, const void* src, int64_t bytes, void* stream);

/*
 * Partial attention state of a query chunk against ONE key/value chunk (non-causal, no dropout):
 *     S = scale * Q K^T,  lse = logsumexp_k S,  out = softmax_k(S) V
 * Replaces flash_attn_func(q, k, v, dropout_p=0, return_attn_probs=True) at
 * core/attention.py:137-143 and :185-191, flash_attn_varlen_func at :314-324 and :366-376, and
 * _flash_attn_varlen_forward at baseline/ulysses.py:99-113.
 *
 *  q, k, v        bf16.  Token t, head h, channel c of q is q[t*q_tok_stride + h*head_dim + c]
 *                 (likewise k, v): [B,S,H,D] or packed [T,H,D] tensors, or slices of wider rows.
 *                 Base pointers 16-byte aligned, strides multiples of 8 elements.
 *  out            out_dtype DTB_F32 or DTB_BF16, same indexing with out_tok_stride.
 *  lse            fp32, natural-log units, layout lse_layout over (nseg or 1, tokens, heads).
 *  accumulate     0: write this chunk's state to (out, lse).
 *                 1: merge this chunk's state INTO the state already held in (out, lse)
 *                    (out must be DTB_F32) -- the update_out_and_lse step of utils.py:24-84 done
 *                    in the kernel's epilogue.  A row whose lse holds -inf is treated as empty.
 *  cu_seqlens_q/k NULL: dense batch -- nseg sequences of exactly seqlen_q query and seqlen_k key
 *                 tokens each, stored back to back.  Otherwise device int32[nseg+1] cumulative
 *                 offsets of a packed batch; seqlen_q / seqlen_k are then upper bounds on a
 *                 segment's length.  Segment i of q attends segment i of k.  Rows of a segment
 *                 with no keys get out = 0, lse = -inf.
 *  total_q/k      number of tokens addressable behind q / k,v (rows of the 2-D view).
 *  head_dim       64 or 128.
 */
DTB_API int dtb_flash_fwd(const void* q, const void* k, const void* v,
                  int64_t q_tok_stride, int64_t k_tok_stride, int64_t v_tok_stride,
                  void* out, int out_dtype, int64_t out_tok_stride,
                  float* lse, int lse_layout, int accumulate,
                  const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                  int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int64_t total_k,
                  int num_heads, int head_dim, float softmax_scale, void* stream);

/*
 * dtb_flash_fwd with launch flags.  The reference walks the chunks of a ring block with one attention call
 * per chunk (core/attention.py:160-196); on the device these are back-to-back launches whose grids do not
 * divide evenly over the SMs, so every launch ends with a partly filled wave.
 *
 *  DTB_LAUNCH_OVERLAP_PREVIOUS   this launch may start while the operation queued just before it on `stream`
 *      is finishing: its CTAs take the SMs that launch's last wave leaves idle (programmatic dependent
 *      launch).  The kernel reads q, k, v and cu_seqlens at once, and waits for the previous launch to
 *      complete before it reads or writes (out, lse) -- so accumulating into the state the previous launch
 *      wrote is fine.  Contract: the last kernel or copy queued on `stream` before this call must be another
 *      dtb_flash_fwd / dtb_flash_fwd_ex launch, and this call's q, k, v, cu_seqlens must not be produced by
 *      it.  Event waits and event records in between are fine (they write no memory and do not stop the
 *      overlap).  After any other kernel or a copy pass 0: what the operation just before wrote is only
 *      guaranteed visible to a launch without the flag.
 */
#define DTB_LAUNCH_OVERLAP_PREVIOUS 1
DTB_API int dtb_flash_fwd_ex(const void* q, const void* k, const void* v,
                     int64_t q_tok_stride, int64_t k_tok_stride, int64_t v_tok_stride,
                     void* out, int out_dtype, int64_t out_tok_stride,
                     float* lse, int lse_layout, int accumulate,
                     const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                     int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int64_t total_k,
                     int num_heads, int head_dim, float softmax_scale, int launch_flags, void* stream);

/*
 * dtb_flash_fwd with a sliding window and first tokens that stay visible.  (The reference has full attention only.)  The query at
 * position x sees the key at position j when
 *     j <= x + right   and   (j >= x - left  or  j < sinks)
 * Key j of a sequence is at position k_start + j; query i at q_start + i, or with q_start = DTB_QUERIES_LAST at the end of the keys,
 * the last query at the last key's position.  A row that sees nothing gets out = 0, lse = -inf (with accumulate its state stays).
 *
 *  q, k, v        bf16, token t of sequence b at t * tok_stride + b * batch_stride, head h behind it at h * head_dim (batch strides are
 *                 not read for packed batches).  Strides are multiples of 8 elements, pointers 16-byte aligned.
 *  out            [total_q, num_heads, head_dim] contiguous; lse, lse_layout, accumulate as for dtb_flash_fwd
 *  num_kv_heads   divides num_heads: query head h meets key head h / (num_heads / num_kv_heads)
 *  cu_seqlens_q/k packed batch, as for dtb_flash_fwd: rows outside all segments are left alone
 *  seqlens_k      NULL, or device int32[nseg]: the keys of each sequence of a dense batch (at most seqlen_k; what the memory holds
 *                 behind them does not matter)
 *  left, right    keys visible before and behind the query's own position, -1 for all; sinks first positions
 *  scratch        dtb_flash_window_scratch_bytes(...) bytes, 16-byte aligned, of one call at a time, for the states of parts that the keys
 *                 are split into; 0 bytes where they are not.  NULL: they are not split.  (Packed batches never are.)
 * Keys and values that no query of a block of rows sees may hold anything; those that some see must be finite.
 */
#define DTB_QUERIES_LAST (-2147483647 - 1)
DTB_API int dtb_flash_window(const void* q, const void* k, const void* v,
                     int64_t q_tok_stride, int64_t q_batch_stride, int64_t k_tok_stride, int64_t k_batch_stride,
                     int64_t v_tok_stride, int64_t v_batch_stride,
                     void* out, int out_dtype, float* lse, int lse_layout, int accumulate,
                     const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, const int32_t* seqlens_k,
                     int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int64_t total_k,
                     int num_heads, int num_kv_heads, int head_dim, float softmax_scale,
                     int left, int right, int sinks, int q_start, int k_start,
                     void* scratch, int64_t scratch_bytes, void* stream);
DTB_API int64_t dtb_flash_window_scratch_bytes(int nseg, int seqlen_q, int seqlen_k, int num_heads, int num_kv_heads, int head_dim,
                                               int left, int right, int sinks);

/*
 * Keys and values of sequences that grow, in pages.  (The reference has no cache of keys and values.)  A pool holds `pages` pages of
 * `page_size` tokens, a power of two from 16 to 2^20: k_pages and v_pages, bf16, token t of head h of page n at
 * n * page_stride + t * tok_stride + h * head_stride, head_dim channels behind it; strides are multiples of 8 elements, pointers 16-byte
 * aligned.  Slot s is token s % page_size of page s / page_size.  table[b][j], int32 [streams, columns], is the page that holds the tokens
 * [j * page_size, (j + 1) * page_size) of stream b.  A row of the table has room for fewer than 2^30 tokens, the pool for fewer than 2^31.
 * free_pages, int32 [pages]: the first *free_count of it are pages that nobody holds, the last of those is taken first.
 *
 * dtb_extend_pages: room for new_lens[b] >= 0 tokens behind the seqlens[b] of each stream, for streams in their order.
 *   table           gets the new pages' numbers; its other entries stay
 *   slots           [tokens]: the new tokens' slots, stream after stream; -1 behind the last one, and for a token on a page that was given
 *                   back before (of a stream that was cut short within what a window had left behind)
 *   cu_seqlens      [streams + 1]: where each stream's new tokens begin among them, and their number
 *   seqlens_out     [streams], free_count_out: the numbers as they are now (not over seqlens or free_count)
 *   missing         0; or how many pages there were too few, or -1 where a stream's tokens do not fit its row, all of them not `tokens`, or a
 *                   number is out of range: then nothing was taken, slots are -1, cu_seqlens 0, the numbers those of before
 * dtb_release_pages: the pages of stream b whose tokens all lie in [begin[b], end[b]) go to the end of the list, streams and their pages in
 * order; their entries become -1.  A stream whose end it is (end[b] >= seqlens[b] > begin[b]) is begin[b] tokens long afterwards.
 *   table_out       the table afterwards, may be `table`; seqlens_out and free_count_out are not over seqlens or free_count
 *   streams * (columns / 256, rounded up) is at most 262144.
 * dtb_write_pages: k, v of `tokens` tokens, bf16, token t at t * tok_stride, its heads dense behind it, to the slots of slots[t]; a token whose
 * slot is -1, or not in the pool, is left out.  Slots differ from one another; two tokens with one slot leave some of either there.
 * All three are one launch.
 */
DTB_API int dtb_extend_pages(int32_t* table, const int32_t* seqlens, const int32_t* new_lens, const int32_t* free_pages, const int32_t* free_count,
                     int streams, int columns, int pages, int page_size, int32_t* slots, int64_t tokens, int32_t* cu_seqlens,
                     int32_t* seqlens_out, int32_t* free_count_out, int32_t* missing, void* stream);
DTB_API int dtb_release_pages(const int32_t* table, int32_t* table_out, const int32_t* seqlens, const int32_t* begin, const int32_t* end,
                     int32_t* free_pages, const int32_t* free_count, int streams, int columns, int pages, int page_size,
                     int32_t* seqlens_out, int32_t* free_count_out, void* stream);
DTB_API int dtb_write_pages(const void* k, const void* v, int64_t k_tok_stride, int64_t v_tok_stride, int64_t tokens, const int32_t* slots,
                     void* k_pages, int64_t k_page_stride, int64_t k_page_tok_stride, int64_t k_head_stride,
                     void* v_pages, int64_t v_page_stride, int64_t v_page_tok_stride, int64_t v_head_stride,
                     int pages, int page_size, int num_kv_heads, int head_dim, void* stream);

/*
 * dtb_flash_window over a pool: attention of each sequence's newest queries, the last at the last key's position, over its seqlens_k[b] keys,
 * which include their own.  Arguments as there and above;
 *   table          int32 [nseg, columns]; the rows together have room for fewer than 2^31 tokens.  A page number outside the pool stands for
 *                  keys and values of 0.
 *   seqlens_k      int32 [nseg], taken to be at most columns * page_size
 *   cu_seqlens_q   NULL for a dense batch of seqlen_q queries each, else device int32 [nseg + 1]; rows outside all sequences are left alone
 *   seqlen_q       the longest sequence's queries (of longer ones the first seqlen_q are attended, from their positions); seqlen_k: about the most keys that a
 *                  sequence's queries see together, which only the choice of kernels goes by
 *   scratch        dtb_flash_paged_scratch_bytes(...) bytes, 16-byte aligned, of one call at a time; may be NULL for 0 bytes
 */
DTB_API int64_t dtb_flash_paged_scratch_bytes(int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int num_heads, int num_kv_heads, int head_dim);
/* Kernels that such a call launches (packed: whether cu_seqlens_q is given), for accounting. */
DTB_API int dtb_flash_paged_launches(int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int packed, int num_heads, int num_kv_heads, int head_dim);
DTB_API int dtb_flash_paged(const void* q, int64_t q_tok_stride, int64_t q_batch_stride,
                     const void* k_pages, int64_t k_page_stride, int64_t k_tok_stride, int64_t k_head_stride,
                     const void* v_pages, int64_t v_page_stride, int64_t v_tok_stride, int64_t v_head_stride,
                     int pages, int page_size, const int32_t* table, int columns, const int32_t* seqlens_k, const int32_t* cu_seqlens_q,
                     void* out, int out_dtype, float* lse, int lse_layout, int accumulate,
                     int nseg, int seqlen_q, int seqlen_k, int64_t total_q, int num_heads, int num_kv_heads, int head_dim, float softmax_scale,
                     int left, int right, int sinks, void* scratch, int64_t scratch_bytes, void* stream);


/*
 * N-way merge of partial softmax states in one pass over HBM:
 *     lse_out = log sum_i exp(lse_i),   out = sum_i exp(lse_i - lse_out) * out_i
 * Replaces the chains of update_out_and_lse (utils.py:24-84) at core/attention.py:110-116, :144,
 * :193-196, :213 and proCache._merge_blocks (core/cache.py:28-46).
 *
 *  outs[i]       state i's values, [rows_bs, H, D] contiguous, dtype out_dtypes[i]
 *  lses[i]       state i's fp32 lse over the same tokens, layout lse_layouts[i]
 *  out / lse_out fp32 results (lse_out may be NULL); `out` and `lse_out` may alias input 0 only.
 *  out_bf16      optional copy of the result in bf16 (NULL to skip): the cast the reference's
 *                callers apply right after the call (executor/cogvideox/attention_processor.py:80).
 *                When it is given, `out` may be NULL and the fp32 result is not written at all.
 *  batch, seq    tokens are [batch, seq]; they matter for DTB_LSE_BHS indexing only.
 *  States whose lse is -inf on a row contribute nothing; a row empty in all states gets
 *  out = 0, lse = -inf.  A NaN among a row's lse makes its out and lse NaN.
 */
DTB_API int dtb_merge_states(int nstates, const void* const* outs, const int* out_dtypes,
                     const float* const* lses, const int* lse_layouts,
                     float* out, float* lse_out, int lse_out_layout, void* out_bf16,
                     int batch, int seq, int num_heads, int head_dim, void* stream);

/*
 * dtb_merge_states for states of which some are held in 8 bits, with a result that may be written in 8 bits.  (The reference caches
 * fp32 states, core/cache.py:9-128.)
 *
 * A row, one (token, head), of a state in 8 bits is D codes (DTB_I8, or DTB_E4M3) and one exponent byte b; a value is
 * code * 2^(b - 127), so it is exact in bf16.  Written, b is the smallest byte, at least 8, with max|value| <= M * 2^(b - 127), M
 * the largest code (127, 448), and a code the nearest to value * 2^(127 - b), ties to even.  A row that holds an infinity or a
 * NaN has b = 255 and codes 0, and reads back as NaN.
 *
 *  outs[i], out_dtypes[i]   [batch, seq, H, D] contiguous, DTB_F32, DTB_BF16, DTB_I8 or DTB_E4M3
 *  exponents[i]             [batch, seq, H] bytes of a state in 8 bits (not read otherwise)
 *  out, out_bf16, out_codes results in fp32, bf16 and 8 bits (out_codes_dtype, with out_exponents); at least one.  An fp32 or bf16
 *                           result may be the buffer of a state of its type, lse_out that of a state's lse in its layout.  An
 *                           8-bit result's codes and exponents are buffers of their own.
 */
DTB_API int dtb_merge_rows(int nstates, const void* const* outs, const int* out_dtypes, const uint8_t* const* exponents,
                     const float* const* lses, const int* lse_layouts,
                     float* out, float* lse_out, int lse_out_layout, void* out_bf16,
                     void* out_codes, int out_codes_dtype, uint8_t* out_exponents,
                     int batch, int seq, int num_heads, int head_dim, void* stream);

/* A single state's values, `rows` (below 2^31) rows of head_dim, written in 8 bits, and read back as fp32 or bf16. */
DTB_API int dtb_quantize_rows(const void* values, int dtype, void* codes, int codes_dtype, uint8_t* exponents, int64_t rows, int head_dim, void* stream);
DTB_API int dtb_dequantize_rows(const void* codes, int codes_dtype, const uint8_t* exponents, void* out, int out_dtype, int64_t rows, int head_dim, void* stream);

/*
 * Strided copy of contiguous chunks: for every (i0,i1,i2) in [n0,n1,n2) copies chunk_bytes from
 * src + i0*ss0 + i1*ss1 + i2*ss2 to dst + i0*ds0 + i1*ds1 + i2*ds2 (strides in bytes), for each of
 * `npairs` (src, dst) pairs in one launch.  chunk_bytes, strides and pointers are multiples of 16.
 * Used for the head<->sequence re-layouts around the Ulysses all-to-all, replacing the
 * tensor_split + contiguous + cat copies of GroupCoordinator.all_to_all
 * (core/group_coordinate.py:281-286).
 */
DTB_API int dtb_copy_chunks(int npairs, const void* const* srcs, void* const* dsts, int64_t chunk_bytes,
                    int64_t n0, int64_t n1, int64_t n2,
                    int64_t ss0, int64_t ss1, int64_t ss2,
                    int64_t ds0, int64_t ds1, int64_t ds2, void* stream);

/*
 * Layer norm over each head of the query and key projections, then rotary embedding (interleaved channel
 * pairs) of the tokens behind the first text_len of every sequence; fp32 arithmetic, one rounding to bf16.
 * The norm_q / norm_k / apply_rotary_emb steps of the attention adapter
 * (executor/cogvideox/attention_processor.py:50-72) for both tensors in one launch.
 *
 *  q, k           bf16 [batch, seq, num_heads, head_dim] contiguous; q_out, k_out likewise (may be q, k)
 *  q_weight, ...  bf16 [head_dim]
 *  cos, sin       fp32 [seq - text_len, head_dim] contiguous; not read when text_len == seq
 */
DTB_API int dtb_norm_rope(const void* q, void* q_out, const void* q_weight, const void* q_bias, float q_eps,
                          const void* k, void* k_out, const void* k_weight, const void* k_bias, float k_eps,
                          const float* cos, const float* sin,
                          int batch, int seq, int text_len, int num_heads, int head_dim, void* stream);

/*
 * Norm of each head of the query and key projections (layer norm, or RMS norm with rms != 0), then rotary positions on three axes:
 * dtb_norm_rope without tables, for tokens that are places of a grid (time, height, width), with its gradients.  Of a sequence's
 * tokens the first text_len and those behind the video_len after them are normalised only; the n-th video token is number
 * first + n of the grid's places (row-major) with their padding, and its channel pair i' of axis a, which has axes[a] channels
 * (interleaved pairs, axes in order), turns by
 *     (origin_a + step_a * index_a) * base^(-2 i' / axes[a])
 * The places lie in `shards` pieces of ceil(places / shards) tokens; where they do not divide evenly the first pieces are full and the
 * others end with padding (what split_tensor_uneven, utils.py:86-136, makes).  Padding, and a token behind the last piece, gets a
 * result of 0, as from zero-padded tables, and passes no gradient.  The reference forms such tables per model (executor/cogvideox/attention_processor.py:50-72 applies them).
 *
 *  q, k            dtype DTB_BF16 or DTB_F32 (weights, biases, results and gradients alike): token s of sequence b, head h at
 *                  b * batch_stride + s * tok_stride + h * head_dim, strides multiples of 16 bytes
 *  q_out, k_out    [batch, seq, heads, head_dim] contiguous; they may be q, k where those are contiguous
 *  q_weight, ...   [head_dim]; a bias may be NULL; q_eps, k_eps normal numbers above 0
 *  grid, axes      host int[3]: places and channels (even, head_dim in all) of the axes
 *  place           host double[7]: base, origin[3], step[3]
 *  first           0 to 2^62
 * Backward: dq_out, dk_out are the gradients of the results, with strides of their own; dq, dk contiguous.  dq_weight ... dk_bias
 * [head_dim] (each may be NULL) are sums over all rows in a fixed order.  scratch: dtb_norm_rope_grid_scratch_bytes(head_dim) bytes
 * (negative: an error code), 16-byte aligned, of one call at a time.
 */
DTB_API int dtb_norm_rope_grid(const void* q, int64_t q_tok_stride, int64_t q_batch_stride, void* q_out, const void* q_weight, const void* q_bias, float q_eps,
                               const void* k, int64_t k_tok_stride, int64_t k_batch_stride, void* k_out, const void* k_weight, const void* k_bias, float k_eps,
                               int dtype, int rms, const int* grid, const int* axes, const double* place, int64_t first, int shards,
                               int batch, int seq, int text_len, int video_len, int q_heads, int k_heads, int head_dim, void* stream);
DTB_API int64_t dtb_norm_rope_grid_scratch_bytes(int head_dim);
DTB_API int dtb_norm_rope_grid_backward(const void* dq_out, int64_t dq_tok_stride, int64_t dq_batch_stride,
                                        const void* dk_out, int64_t dk_tok_stride, int64_t dk_batch_stride,
                                        const void* q, int64_t q_tok_stride, int64_t q_batch_stride, const void* q_weight, float q_eps,
                                        const void* k, int64_t k_tok_stride, int64_t k_batch_stride, const void* k_weight, float k_eps,
                                        void* dq, void* dk, void* dq_weight, void* dq_bias, void* dk_weight, void* dk_bias,
                                        int dtype, int rms, const int* grid, const int* axes, const double* place, int64_t first, int shards,
                                        int batch, int seq, int text_len, int video_len, int q_heads, int k_heads, int head_dim,
                                        void* scratch, int64_t scratch_bytes, void* stream);

/*
 * The two elementwise steps around a transformer block's sub-layers (LayerNormZero modulation and gated residual,
 * executor/cogvideox/cogvideox_transformer_3d.py:139-190), over both streams in one launch each; fp32 arithmetic,
 * one rounding to bf16.  All tensors bf16, contiguous.
 *
 *  dtb_ln_modulate   out[b, s] = (LayerNorm(x[b, s]) * weight + bias) * (1 + scale[b]) + shift[b]
 *  dtb_gate_add      x_out[b, s] = x[b, s] + gate[b] * a[b, s]          (x_out may be x)
 *
 *  video, text   [batch, video_len, dim], [batch, text_len, dim]; out, a: [batch, text_len + video_len, dim], text first
 *  mod           [batch, 6 dim]: shift, scale, gate of the video stream, then of the text stream
 *  dim           a multiple of 256, at most 3072
 */
DTB_API int dtb_ln_modulate(const void* video, const void* text, const void* weight, const void* bias, float eps,
                            const void* mod, void* out, int batch, int video_len, int text_len, int dim, void* stream);
DTB_API int dtb_gate_add(const void* video, const void* text, const void* a, const void* mod, void* video_out, void* text_out,
                         int batch, int video_len, int text_len, int dim, void* stream);

/*
 * Drift metric of the redundancy-profiling pass, accumulated on the device:
 *     *accum += mean|cur - prev| / (mean|prev| + 1e-8)      over positions where neither is NaN
 * (mean|cur| instead when mean|prev| < 1e-6; +inf when no position is valid).  Replaces rel_l1
 * (utils.py:202-267) as called from RedundancyMap.record_out_redundancy
 * (core/redundancy_map.py:174-197), which reads three means back to the host per layer and step.
 *
 *  cur, prev     fp32 [n] on the device
 *  accum         one fp32 on the device (for example an element of the [steps, layers] map)
 *  scratch       device memory of at least dtb_drift_scratch_bytes(n) bytes, 256-byte aligned, whose
 *                first 4 bytes are zero before the first call; the call leaves them zero, so one
 *                buffer serves any number of calls that do not overlap on the device.
 */
DTB_API int64_t dtb_drift_scratch_bytes(int64_t n);
DTB_API int dtb_drift_accumulate(const float* cur, const float* prev, int64_t n, float* accum,
                                 void* scratch, int64_t scratch_bytes, void* stream);

/*
 * dtb_drift_accumulate for callers that cannot supply (or allocate) scratch memory.  It has no
 * counterpart in the reference.  Same result as dtb_drift_accumulate; the partial sums go into a
 * 1 MiB array built into the library's device image, which every GPU that loads the library holds
 * until the process exits.  No cudaMalloc / cudaFree or allocating library routine is called.
 *
 *  - n is limited to dtb_drift_noalloc_max_elements() (536,739,840); larger inputs are rejected
 *    with DTB_ERR_ARG and a message naming the limit.
 *  - The first call on a device looks up the array's device address (cudaGetSymbolAddress, with
 *    that device current) and remembers it; make that first call outside any stream capture.
 *  - All calls on a device share the one array and it keeps the previous call's contents; the
 *    entry point clears the one word that must start at zero.  Two calls that overlap on the GPU
 *    (different streams, or different host threads) race on it: serialise them.
 */
DTB_API int64_t dtb_drift_noalloc_max_elements(void);
DTB_API int dtb_drift_accumulate_noalloc(const float* cur, const float* prev, int64_t n, float* accum, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DITANGO_B200_H_ */
