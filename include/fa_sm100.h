/*
 * C ABI of the B200 (sm_100a) FlashAttention forward library
 * (libfa_sm100.so). Plain pointers, sizes and a CUDA stream handle; no
 * PyTorch types. Every function returns FA_OK (0) or a negative FA_ERR_*
 * code; fa_last_error() then holds a message for the calling thread.
 *
 * Layout of every tensor: contiguous [batch, heads, rows, 64] fp16, so one
 * (batch, head) slice is rows x 128 bytes. Pointers must be device pointers
 * on the current CUDA device and 16-byte aligned. Work is enqueued on
 * `cuda_stream` (NULL = legacy default stream); nothing synchronises.
 */
#ifndef FA_SM100_H_
#define FA_SM100_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FA_OK 0
#define FA_ERR_INVALID (-1)     /* bad sizes, pointers or alignment */
#define FA_ERR_CUDA (-2)        /* CUDA runtime / driver call failed */
#define FA_ERR_UNSUPPORTED (-3) /* device is not sm_100 */

/*
 * Attention forward, head dimension 64, equal query and key lengths.
 * O = softmax(Q K^T * scale [+ causal mask]) V with fp32 accumulation and fp16
 * output. `causal` masks key index > query index (top-left aligned).
 *
 * Replaces the launch path of the reference's production kernel:
 *   tensorcore_attention_forward_production_impl
 *     (csrc/tensorcore_attention.cu:2969-3123), which launches
 *   tensorcore_attention_forward_kernel_d64_production<kCausal>
 *     (csrc/tensorcore_attention.cu:2019-2727) with scale 1/sqrt(64)
 *     (csrc/tensorcore_attention.cu:3040-3046).
 * Unlike the reference launcher, seq_len need not be a multiple of 128 and
 * batch * heads is not limited to 65535 (persistent grid); the torch binding
 * keeps the reference's checks for drop-in behaviour.
 * batch * heads * seq_len == 0 is a no-op (reference :3003-3009).
 */
int fa_fwd_sm100(const void* q, const void* k, const void* v, void* o, int64_t batch,
                 int64_t heads, int64_t seq_len, int causal, float scale, void* cuda_stream);

/*
 * Same, with independent query and key lengths (k and v have kv_len rows,
 * q and o have q_len rows). The causal mask stays top-left aligned, as in
 * the reference oracle flash_attention/reference.py:49-56 (triu(1) on an
 * [q_len, kv_len] matrix).
 */
int fa_fwd_sm100_varlen(const void* q, const void* k, const void* v, void* o, int64_t batch,
                        int64_t heads, int64_t q_len, int64_t kv_len, int causal, float scale,
                        void* cuda_stream);

/*
 * Same computation as fa_fwd_sm100_varlen, for callers that must not allocate
 * device memory during the call: code that runs while a CUDA graph is being
 * captured (an allocation there breaks the capture), serving paths that work
 * within a memory budget fixed at start-up, and code called from inside an
 * allocator or memory-pool callback. fa_fwd_sm100_varlen allocates a scratch
 * buffer per stream the first time a problem uses the key-range split mode;
 * this entry point instead uses one fixed 12 MiB array compiled into the
 * library, which every GPU that loads the library holds until the process
 * exits, and calls no cudaMalloc or cudaFree. A problem whose split plan needs
 * more scratch than that is rejected with FA_ERR_INVALID and a message giving
 * both sizes. The caller still provides q, k, v and o.
 * The array is shared by every call on a device and keeps the last call's
 * contents (its counters are cleared at the start of each call): calls that
 * overlap on the GPU, e.g. on two streams, race and must not be made.
 * The first call into this library on a device looks up the array's device
 * address; make that first call before any stream capture.
 * No counterpart in the reference.
 */
int fa_fwd_sm100_noalloc(const void* q, const void* k, const void* v, void* o, int64_t batch,
                         int64_t heads, int64_t q_len, int64_t kv_len, int causal, float scale,
                         void* cuda_stream);

/*
 * As fa_fwd_sm100_varlen, and also writes the row log-sum-exp of the scaled
 * scores, lse[b, h, i] = log(sum_j exp(scale * q_i . k_j)) over the unmasked
 * keys (natural log, fp32, contiguous [batch, heads, q_len]), which the
 * backward pass (fa_bwd_sm100) takes as its softmax statistics.
 * No counterpart in the reference (its forward returns only O; a training
 * caller needs the statistics).
 */
int fa_fwd_sm100_lse(const void* q, const void* k, const void* v, void* o, float* lse,
                     int64_t batch, int64_t heads, int64_t q_len, int64_t kv_len, int causal,
                     float scale, void* cuda_stream);

/*
 * Attention backward, head dimension 64: given q (fp16 [batch, heads, q_len,
 * 64]), k, v (fp16 [batch, heads, kv_len, 64]), the forward output o and the
 * output gradient d_o (fp16, q's shape) and the forward's lse (fp32 [batch,
 * heads, q_len], from fa_fwd_sm100_lse), writes dq (q's shape) and dk, dv
 * (k's shape):
 *   P = exp(scale * Q K^T - lse) (causal: top-left, key j > query i masked,
 *       as in the forward),
 *   dV = P^T dO,  dP = dO V^T,  dS = P * (dP - rowsum(dO * O)),
 *   dQ = scale * dS K,  dK = scale * dS^T Q.
 * Keys that no query sees (causal with kv_len > q_len) get dK = dV = 0.
 * kv_len = 0 with q_len > 0 is rejected, as in the forward.
 * Uses the scratch buffer per (device, stream) of the split mode for the
 * fp32 dQ accumulator and the row terms (allocated or grown on first need,
 * so the first call on a stream allocates).
 * No counterpart in the reference (it has no backward).
 */
int fa_bwd_sm100_varlen(const void* q, const void* k, const void* v, const void* o,
                        const void* d_o, const float* lse, void* dq, void* dk, void* dv,
                        int64_t batch, int64_t heads, int64_t q_len, int64_t kv_len, int causal,
                        float scale, void* cuda_stream);

/* fa_bwd_sm100_varlen with q_len = kv_len = seq_len. */
int fa_bwd_sm100(const void* q, const void* k, const void* v, const void* o, const void* d_o,
                 const float* lse, void* dq, void* dk, void* dv, int64_t batch, int64_t heads,
                 int64_t seq_len, int causal, float scale, void* cuda_stream);

/* Element types of the entry points below. */
#define FA_FP16 0
#define FA_BF16 1
#define FA_FP32 2

/* One tensor of fa_rotary_sm100: x is [batch, heads, tokens, head_dim] with
 * any strides (in elements) and dense rows; y is contiguous of that shape.
 * x and y must not overlap. */
typedef struct fa_rotary_tensor {
  const void* x;
  void* y;
  int64_t heads, batch_stride, head_stride, token_stride;
} fa_rotary_tensor;

/*
 * Rotary positions: turns the first rotary_dim elements of each row of query
 * and (key != NULL) key by the token's position; the others are copied. Pair
 * i is (i, i + rotary_dim / 2), or (2i, 2i + 1) when `interleaved`:
 *   x' = factor (x cos a - y sin a),  y' = factor (y cos a + x sin a),
 *   a = position * frequencies[i] (radians; -a when `inverse`).
 * `inverse` with the same factor is the backward pass. positions: integers
 * of position_bits 32 or 64, [batch, tokens] with the given strides in
 * elements. frequencies: fp64 [rotary_dim / 2] on the device. The angle is
 * reduced in 64 bits: it is off by 3e-7 rad at most up to position 2^28 and by
 * 7e-7 at any 32-bit one.
 * No counterpart in the reference (it has no positions).
 */
int fa_rotary_sm100(const fa_rotary_tensor* query, const fa_rotary_tensor* key,
                    const void* positions, int position_bits, int64_t position_batch_stride,
                    int64_t position_token_stride, const double* frequencies, int64_t batch,
                    int64_t tokens, int64_t head_dim, int64_t rotary_dim, int interleaved,
                    int dtype, float factor, int inverse, void* cuda_stream);

/*
 * A paged key/value cache. k_pages and v_pages: contiguous [num_pages,
 * kv_heads, page_size, head_dim] of a 16-bit type, 16-byte aligned; page_size
 * a multiple of 16, head_dim 64 or 128. Slot s of sequence b is row
 * s % page_size of page block_table[b * table_stride + s / page_size],
 * s < lengths[b] <= max_pages * page_size. A cache that is one contiguous
 * [batch, kv_heads, capacity, head_dim] tensor has num_pages = batch, max_pages
 * = 1 and page_size = capacity.
 * Table, lengths and the other integer arrays are read by the kernels: an
 * entry that leads outside the cache is not followed, the rows that it stands
 * for are left out, and bit 32 of the device status word (fa_read_status) is
 * set.
 */
typedef struct fa_paged_cache {
  void* k_pages;
  void* v_pages;
  const int* block_table;
  const int* lengths;
  int64_t table_stride;
  int64_t batch, kv_heads, num_pages, page_size, max_pages, head_dim;
} fa_paged_cache;

/* Rows [batch, heads, rows, head_dim] with strides in elements, each a
 * multiple of 8; data is 16-byte aligned and rows are dense. */
typedef struct fa_rows {
  const void* data;
  int64_t batch_stride, head_stride, row_stride;
} fa_rows;

/*
 * Appends rows of key and value to a cache: row path[b * rows + i] (path NULL:
 * row i) becomes slot lengths[b] + i for i < counts[b] (counts NULL: all
 * rows); the rows of a path end before its first entry among those outside
 * [0, rows). lengths_out[b] = lengths[b] + the rows appended; lengths itself is
 * not changed. weights and positions (each may be NULL; [batch, kv_heads,
 * max_pages * page_size] contiguous) get 0 and new_positions[b * rows +
 * path[b * rows + i]] at the new slots. A page may belong to one sequence only.
 * No counterpart in the reference (it has no cache).
 */
int fa_cache_append_sm100(const fa_paged_cache* cache, const fa_rows* key, const fa_rows* value,
                          int64_t rows, const int* path, const int* counts, float* weights,
                          int* positions, const int* new_positions, int* lengths_out,
                          void* cuda_stream);

/*
 * Evicts from a cache by the weight that its slots gathered: of every
 * (sequence, kv head) with more than `budget` slots, `budget` stay: those of
 * positions below `sinks`, those of the `recent` last positions (above the
 * largest position - recent), then those of the largest weight, among equal
 * weights the lowest slot; NaN counts as the lowest weight. A kept slot at or
 * behind `budget` moves into a dropped slot before it, the i-th into the i-th
 * in slot order; the pages change in place. Where the table names no page for
 * either slot the row, its weight and its position stay where they are: the
 * slot before the budget keeps what it held. weights_out and positions_out
 * (whole, 0 and -1 behind the new length) and lengths_out = min(lengths,
 * budget) are written beside their inputs and must not be the same memory; the
 * four [batch, kv_heads, slots] arrays are contiguous and 16-byte aligned.
 * workspace: fa_cache_evict_workspace(cache, budget) bytes on the device,
 * 256-byte aligned, in use until the call's kernels have run.
 * No counterpart in the reference.
 */
int64_t fa_cache_evict_workspace(const fa_paged_cache* cache, int64_t budget);
int fa_cache_evict_sm100(const fa_paged_cache* cache, const float* weights, const int* positions,
                         float* weights_out, int* positions_out, int* lengths_out, int64_t budget,
                         int64_t recent, int64_t sinks, void* workspace, int64_t workspace_bytes,
                         void* cuda_stream);

/*
 * Attention for a tree of drafted tokens over a cache. Query t of sequence b,
 * head h (kv head h / (heads / kv_heads)) sees the cached slots [0,
 * lengths[b]) and, of the tree's own keys (k_tree, v_tree; both NULL: none),
 * key j with tree_mask[b * mask_batch_stride + t * mask_row_stride + j] != 0
 * (tree_mask NULL: j <= t). tree_sizes (NULL: tokens each): the sequence's
 * queries and tree keys from tree_sizes[b] on are padding; nothing sees them,
 * their out is 0 and their lse -inf, as for a query that sees nothing.
 * out: contiguous [batch, heads, tokens, head_dim]; lse: fp32 [batch, heads,
 * tokens], the natural log of the sum of exp(scale q . k). dtype: FA_FP16 or
 * FA_BF16. One token and no tree is plain decoding. Scores, sums and lse are in
 * 32 bits; the probabilities are rounded to the element type for their product
 * with the values (half a step of it, relative), and out is rounded once. scale
 * is positive and finite.
 * workspace: fa_tree_attention_workspace(...) bytes on the device, 256-byte
 * aligned, in use until the call's kernels have run; it does not depend on the
 * lengths.
 * No counterpart in the reference.
 */
int64_t fa_tree_attention_workspace(const fa_paged_cache* cache, int64_t heads, int64_t tokens,
                                    int has_tree);
int fa_tree_attention_sm100(const fa_paged_cache* cache, const fa_rows* query, int64_t heads,
                            int64_t tokens, const fa_rows* k_tree, const fa_rows* v_tree,
                            const unsigned char* tree_mask, int64_t mask_batch_stride,
                            int64_t mask_row_stride, const int* tree_sizes, int dtype, float scale,
                            void* out, float* lse, void* workspace, int64_t workspace_bytes,
                            void* cuda_stream);

/*
 * Adds the attention weight that each cached slot gets from the queries:
 *   weights[b, hk, s] += sum over heads h of kv head hk and tokens t of
 *                        exp(scale q . k_s - lse[b, h, t]),  s < lengths[b].
 * lse is what the attention over these keys returned (contiguous [batch,
 * heads, tokens]); a query whose lse is -inf saw nothing and adds nothing.
 * weights: contiguous [batch, kv_heads, max_pages * page_size]; slots from
 * lengths[b] on are left as they are. Each weight is summed by one thread block
 * in one order: results do not change from run to run.
 * No counterpart in the reference.
 */
int fa_attention_weight_sm100(const fa_paged_cache* cache, const fa_rows* query, int64_t heads,
                              int64_t tokens, const float* lse, float* weights, int dtype,
                              float scale, void* cuda_stream);

/* Message for the last failing call on this thread ("" if none). */
const char* fa_last_error(void);

/*
 * Reads (and with clear != 0 resets) the device status word of the current
 * device, synchronising `cuda_stream`. Nonzero bits mean a bounded wait inside
 * a kernel ran out of time and that launch's output is invalid:
 *   1 producer, 2 MMA issuer, 4 softmax, 8 drain, 16 self-test.
 * Bit 32 is set by a cache call whose table, lengths, counts or path led outside
 * the cache; it left those rows out.
 * There is one status word per device, shared by every stream, thread and
 * launch on it: a bit set by a launch on one stream is seen (and cleared) by
 * whichever caller reads next, so the word says that some launch on the
 * device since the last clear failed, not which one.
 * No counterpart in the reference (its kernel has no waits that can fail).
 */
int fa_read_status(void* cuda_stream, unsigned int* status_out, int clear);

/* Time limit for every in-kernel wait (default 2 s; 0 restores it). The
 * limit is process-wide: it applies to every later launch from any thread
 * (the setting itself is atomic). */
void fa_set_wait_limit_ns(unsigned long long limit_ns);

/*
 * Launches a one-warp kernel that waits on a barrier nothing arrives on,
 * with the given limit; afterwards fa_read_status must report bit 16.
 * Exercises the timeout path without faulting or hanging the GPU.
 */
int fa_selftest_wait_timeout(unsigned long long limit_ns, void* cuda_stream);

/* Dynamic shared memory one block of the forward kernel uses (bytes). */
int fa_smem_bytes(void);

/*
 * Policy for splitting the key range across blocks (problems with fewer query
 * pairs than SMs): 0 = automatic (default), 1 = never, k > 1 = into at most k
 * splits. In split mode each split writes an fp32 partial result to a scratch
 * buffer and the last split to finish a query tile merges them; the scratch is
 * one buffer per (device, stream), allocated on first need and kept for reuse.
 * The automatic policy does not split across blocks when the query tiles fit
 * in one wave: each tile then gets its own block, whose two softmax
 * warpgroups take one half of the key range each and merge in the block (no
 * scratch), which measured faster on a B200; k > 1 selects the cross-block
 * split for those problems too.
 * The policy is process-wide (an atomic setting read by every later launch
 * from any thread).
 * No counterpart in the reference (its grid never splits the key range).
 */
void fa_set_max_splits(int max_splits);

/*
 * Synchronises every device that holds a split-mode scratch buffer and frees
 * them all, including buffers of streams destroyed since they were made.
 * Must not run while another thread launches. No counterpart in the
 * reference.
 */
int fa_release_workspaces(void);

/*
 * Test hook: as fa_fwd_sm100, and additionally writes the first work item's
 * first masked score tile (256 x 128 fp32, raw Q K^T before scaling) to
 * score_dump. Used only by the tests to localise layout errors.
 */
int fa_fwd_sm100_debug(const void* q, const void* k, const void* v, void* o, int64_t batch,
                       int64_t heads, int64_t seq_len, int causal, float scale, void* cuda_stream,
                       float* score_dump);

#ifdef __cplusplus
}
#endif

#endif /* FA_SM100_H_ */
