/*
 * kf/attn.h -- C ABI of the MI355X (gfx950) flash-attention forward.
 *
 * This is the drop-in boundary for the reference's attention launchers:
 *   - launch_flash_attn      tests/test_flash_attn.cu:52-113  (synchronous,
 *                            q_len == kv_len == S, launcher-owned scratch)
 *   - launch_once            tests/bench_flash_attn.cu:39-54  (asynchronous,
 *                            separate q_len / kv_len, caller-owned Mi / Li)
 *   - flash_attn_kernel<D>   kernels/flash_attn.cu:384-398    (the device
 *                            entry those launchers wrap; not exported here)
 *
 * Plain C types only: device pointers, sizes and an opaque stream handle
 * (a hipStream_t passed as void*; NULL is the default stream).  No C++
 * exceptions cross this boundary; every entry point returns a status code.
 *
 * Tensor layout contract (identical to the reference's, flash_attn.cu:364-370):
 *   Q  [B, H_q,  q_len,  D]  fp16 bits (uint16_t), contiguous row-major
 *   K  [B, H_kv, kv_len, D]  fp16 bits
 *   V  [B, H_kv, kv_len, D]  fp16 bits
 *   O  [B, H_q,  q_len,  D]  fp32
 *   Mi [B, H_q,  q_len]      fp32, optional: max_j s_ij over the scaled scores
 *                            s = q.k / sqrt(D)
 *   Li [B, H_q,  q_len]      fp32, optional: sum_j exp(s_ij - Mi)
 * Query head h_q reads KV head h_q / (H_q / H_kv) (flash_attn.cu:406); H_q
 * must be a multiple of H_kv (the reference silently mis-groups otherwise).
 * kf_attn_fwd is non-causal with softmax scale 1/sqrt(D), as in the
 * reference; kf_attn_fwd_ex adds causal masking and per-sequence key
 * counts (ranked next steps of the reference's own roadmap,
 * docs/flash_attn.md:105 and reference_benchmarks/bench_flash_attn2.py:115-150).
 * D must be one of the reference's instantiations
 * {16, 64, 128, 256} (flash_attn.cu:587-600).  All device pointers must be
 * 16-byte aligned.
 */
#ifndef KF_ATTN_H
#define KF_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes returned by the kf_* entry points. */
enum kf_status {
    KF_OK = 0,
    KF_ERR_HEAD_DIM = 1,   /* D is not 16, 64, 128 or 256                      */
    KF_ERR_GQA = 2,        /* H_q is not a positive multiple of H_kv            */
    KF_ERR_SIZE = 3,       /* a size is <= 0 or overflows the kernels' indexing */
    KF_ERR_NULL = 4,       /* a required pointer is NULL                        */
    KF_ERR_WORKSPACE = 5,  /* workspace missing or smaller than required        */
    KF_ERR_ALIGN = 6,      /* a device pointer is not 16-byte aligned           */
    KF_ERR_HIP = 7,        /* a HIP runtime call failed: kf_last_hip_error()    */
    KF_ERR_FLAGS = 8,      /* unknown bits in `flags`, or F16 and BF16 together  */
    KF_ERR_SCRATCH = 9     /* kf_attn_fwd_noalloc: shape needs more scratch than
                              its static maximum                                 */
};

/* kf_attn_fwd_ex / kf_attn_decode_paged flags. */
#define KF_ATTN_CAUSAL 1   /* query i sees keys j <= i + kv_b - q_len           */
#define KF_ATTN_OUT_F16 2  /* O is written as fp16 (RNE of the fp32 result)     */
#define KF_ATTN_OUT_BF16 4 /* O is written as bf16 (RNE of the fp32 result)     */
#define KF_ATTN_LSE 8      /* row_max receives LSE = Mi + ln(Li) (natural log;
                              -inf for a row without keys); row_sumexp unused */
/* Flags of kf_attn_packed and the entry points after it. */
#define KF_BF16 16         /* 16-bit inputs (and the cache's 16-bit side) are bf16,
                              not fp16                                          */
#define KF_ROPE_INTERLEAVED 32 /* kf_qk_norm_rope: pairs (2i, 2i + 1), not
                              (i, i + rot / 2)                                  */

/* Which kernels kf_attn_fwd runs for a shape (see kf_attn_plan). */
enum kf_path {
    KF_PATH_PREFILL = 0,   /* MFMA prefill kernel, one pass over KV             */
    KF_PATH_DECODE = 1,    /* split-KV decode kernel, writes final O directly   */
    KF_PATH_DECODE_SPLIT = 2, /* split-KV decode kernel + split-merge kernel     */
    KF_PATH_PREFILL_SPLIT = 3 /* MFMA prefill kernel over KV partitions (few query
                                 rows, many keys) + split-merge kernel          */
};

typedef struct kf_attn_plan_t {
    int path;              /* enum kf_path                                      */
    int rows_per_group;    /* H_q / H_kv * q_len query rows per KV head         */
    int num_splits;        /* KV partitions per (b, h_kv); 1 = unsplit          */
    int kv_per_split;      /* KV rows per partition                             */
    int grid_blocks;       /* workgroups of the main kernel                     */
    int block_threads;     /* threads per workgroup of the main kernel          */
    size_t workspace_bytes;/* kf_attn_workspace_bytes(): may be more than this
                              plan's partials, see kf_attn_plan                 */
    int splits_per_block;  /* decode: KV partitions per workgroup (4 = the
                              short-split kernel, one partition per wave;
                              1 = the streaming decode kernel); 0 on prefill    */
} kf_attn_plan_t;

/* Describe the dispatch of an unmasked kf_attn_fwd call on the device current
 * on the calling thread.  A decode that kf_attn_kernel_names names the ragged
 * decode for has no fixed partitions; it is described as it runs with less
 * workspace than that takes, by num_splits partitions of kv_per_split keys on
 * the streaming decode kernel.  Causal calls and calls with key counts may
 * take other layouts: kf_attn_kernel_names tells.  Validates like kf_attn_fwd (sizes only, no pointers).
 * The plan is sized for that device's compute units and XCDs, read once per
 * device with hipDeviceGetAttribute (the reference's launcher likewise sizes
 * its launch from the device, tests/test_flash_attn.cu:28-48); without a
 * visible device it is the plan for a whole MI355X (256 CUs, 8 XCDs).
 * kf_attn_fwd, kf_attn_fwd_ex, kf_attn_decode_paged and the workspace
 * queries plan the same way, so a workspace sized on the current device fits
 * calls on streams of that device. */
int kf_attn_plan(int B, int q_len, int kv_len, int H_q, int H_kv, int D,
                 kf_attn_plan_t* plan);

/* The plan for a device with num_cus compute units (no device query; for
 * planning ahead and for host-only tests).  No reference counterpart.
 * num_cus <= 0 -> KF_ERR_SIZE. */
int kf_attn_plan_for_cus(int B, int q_len, int kv_len, int H_q, int H_kv, int D, int num_cus,
                         kf_attn_plan_t* plan);

/* Names of the kernels kf_attn_fwd_ex launches for this shape on the current
 * device given its best workspace (kf_attn_workspace_bytes, or _lens with
 * kv_lens), in launch order and as a profiler lists them, e.g.
 * "kf_attn_prefill_kernel<128, false, 8, 1>" or
 * "kf_attn_decode_short_kernel<128, 1> + kf_attn_split_merge_kernel<128, 8, 4>";
 * `flags` (KF_ATTN_CAUSAL) and whether kv_lens is non-NULL (never read) pick
 * the masked prefill and its layout, and kv_lens the ragged decode.  NUL-terminated into buf; KF_ERR_SIZE if buf_bytes is
 * too small.  No reference counterpart (its launchers print the launch
 * geometry, tests/test_flash_attn.cu:86-91). */
int kf_attn_kernel_names(int B, int q_len, int kv_len, int H_q, int H_kv, int D, int flags,
                         const int* kv_lens, char* buf, size_t buf_bytes);

/* Bytes of device workspace with which kf_attn_fwd runs this shape its fastest
 * (0 when the shape runs without split-KV partials: split decode and split
 * prefill need them).  A decode whose heads do not divide over the compute
 * units is shared evenly by all of their waves given this much; with less,
 * down to num_splits partials of all query rows, it runs by the plan's splits
 * (the two differ in the last bits, within the same tolerance).  Returns 0 for
 * invalid shapes too; kf_attn_plan reports why. */
size_t kf_attn_workspace_bytes(int B, int q_len, int kv_len, int H_q, int H_kv, int D);

/* Bytes of workspace with which a kf_attn_fwd_ex call with kv_lens runs its
 * fastest: at least kf_attn_workspace_bytes().  A large decode then shares the
 * keys that the sequences really hold evenly over the compute units, instead
 * of splitting every sequence by the kv_len rows allocated; a call given less,
 * down to kf_attn_workspace_bytes_least(), still runs, by those splits (the
 * two differ in the last bits, within the same tolerance).  Shared evenly, a
 * sequence's keys are cut where the shares end, so its last bits depend on the
 * other sequences' key counts; by the splits they depend on the shape alone.
 * Sequences that all fill their kv_len rows run up to about a tenth faster by
 * the splits where those take one round.  No reference counterpart. */
size_t kf_attn_workspace_bytes_lens(int B, int q_len, int kv_len, int H_q, int H_kv, int D);

/* Bytes of workspace that a caller who has any should give this shape at
 * least (with or without kv_lens, contiguous or paged): a split decode is
 * refused with less, a split prefill runs with fewer KV partitions.  0 where
 * the call is fully split over the compute units without a workspace, though
 * it may run faster given kf_attn_workspace_bytes() or _lens().  No reference
 * counterpart. */
size_t kf_attn_workspace_bytes_least(int B, int q_len, int kv_len, int H_q, int H_kv, int D);

/* Attention forward, asynchronous on `stream`.
 *
 * Replaces launch_once (tests/bench_flash_attn.cu:39-54) and the kernel
 * launch inside launch_flash_attn (tests/test_flash_attn.cu:92-93):
 * separate q_len / kv_len (q_len = 1 is decode), optional Mi / Li outputs
 * (row_max / row_sumexp may be NULL), caller-owned workspace of at least
 * kf_attn_workspace_bytes() bytes (may be NULL when that is 0; 256-byte
 * aligned).  The workspace needs no initialisation; it must not be shared by
 * calls that can run concurrently (e.g. on two streams).  Only split decode
 * (KF_PATH_DECODE_SPLIT) requires it: a split prefill (KF_PATH_PREFILL_SPLIT)
 * given no workspace, or a smaller one, runs with as many KV partitions as
 * that workspace holds, or unsplit, instead of failing (its results then
 * differ in the last bits, within the same tolerance).
 * Validation happens before any HIP call; an invalid argument returns its
 * status code and launches nothing.  Unlike launch_once, which silently
 * does nothing for an unsupported D (bench_flash_attn.cu:48-52), this
 * returns KF_ERR_HEAD_DIM. */
int kf_attn_fwd(const void* Q, const void* K, const void* V, float* O,
                float* row_max, float* row_sumexp,
                int B, int q_len, int kv_len, int H_q, int H_kv, int D,
                void* workspace, size_t workspace_bytes, void* stream);

/* kf_attn_fwd with key masking; kf_attn_fwd(...) == kf_attn_fwd_ex(...,
 * NULL, 0, ...).  No counterpart in the reference, which has neither
 * (flash_attn.cu:384-585 is non-causal over all kv_len keys).
 *
 * kv_lens: NULL, or a device array [B] of int (4-byte aligned): sequence b
 *   uses only its first kv_b = kv_lens[b] keys (clamped to [0, kv_len]) of
 *   the kv_len rows allocated per head in K / V -- a pre-allocated KV cache
 *   filled to different lengths.
 * flags & KF_ATTN_CAUSAL: query i (0 <= i < q_len) of sequence b sees keys
 *   j <= i + kv_b - q_len, i.e. the mask is aligned to the bottom-right
 *   corner (the last query sees every key; with q_len == kv_len it is the
 *   usual lower triangle; q_len = 1 decode is unaffected).
 * A query row that sees no key (kv_b = 0, or causal rows with
 * i + kv_b - q_len < 0) gets O = 0, Mi = -inf, Li = 0.
 * O is fp32 [B, H_q, q_len, D] unless flags select KF_ATTN_OUT_F16 or
 * KF_ATTN_OUT_BF16 (then 2-byte elements, still 16-byte aligned; the
 * reference's PyTorch comparator outputs fp16, bench_flash_attn2.py:11-12);
 * KF_ATTN_LSE replaces the (Mi, Li) pair by one log-sum-exp per row in
 * row_max.  KF_ATTN_OUT_F16 | KF_ATTN_OUT_BF16 -> KF_ERR_FLAGS.  Shapes and the
 * workspace needed are those of kf_attn_fwd (kf_attn_workspace_bytes; with
 * kv_lens a decode runs faster given kf_attn_workspace_bytes_lens). */
int kf_attn_fwd_ex(const void* Q, const void* K, const void* V, void* O,
                   float* row_max, float* row_sumexp,
                   int B, int q_len, int kv_len, int H_q, int H_kv, int D,
                   const int* kv_lens, int flags,
                   void* workspace, size_t workspace_bytes, void* stream);

/* kf_attn_fwd_ex without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid allocation).  No counterpart in the reference.
 *
 * The split-KV partials go to a static device array of the library, one per
 * device, of kf_attn_noalloc_scratch_bytes() bytes (16 MiB), held until the
 * process ends; the call makes no hipMalloc / hipFree or any other allocation.
 * Its address is resolved on the first call on each device (with that device
 * current on the calling thread) and kept for the life of the process; a
 * hipDeviceReset() of that device unloads the array, so the call must not be
 * used again on a device after resetting it.  Flag, pointer and alignment
 * errors are reported as by kf_attn_fwd_ex, before any scratch check.  A
 * shape whose plan needs more than that
 * (kf_attn_workspace_bytes) returns KF_ERR_SCRATCH and launches nothing,
 * except a split prefill (KF_PATH_PREFILL_SPLIT), which is planned with as
 * many KV partitions as the scratch holds -- possibly fewer than
 * kf_attn_fwd_ex takes, in which case the results differ from its in the
 * last bits (both within the same tolerance of the exact result).  Likewise a
 * decode whose even sharing (kf_attn_workspace_bytes, or _lens) needs more than
 * the scratch runs by the plan's splits, and one whose plan needs no scratch
 * takes none.
 * Every call on one device shares that device's array: calls that can run
 * concurrently on one device (two streams, two threads) race on it and must
 * be serialised by the caller; consecutive calls on one stream are safe.  The
 * kernels need no initialised scratch.  Arguments otherwise as kf_attn_fwd_ex. */
int kf_attn_fwd_noalloc(const void* Q, const void* K, const void* V, void* O,
                        float* row_max, float* row_sumexp,
                        int B, int q_len, int kv_len, int H_q, int H_kv, int D,
                        const int* kv_lens, int flags, void* stream);

/* Size of kf_attn_fwd_noalloc's static per-device scratch (bytes). */
size_t kf_attn_noalloc_scratch_bytes(void);

/* Decode over a paged K/V cache, the block-table gather fused into the
 * split-KV decode kernel.  Replaces the gather + attention of the
 * reference's paged comparison (reference_benchmarks/bench_flash_attn2.py:
 * 153-215: pools [pool_blocks, H_kv, block_size, D], block ids per page),
 * which it names as the job of a specialised paged-attention kernel; the
 * reference has no such kernel.
 *
 * K_pages, V_pages: [num_pages, H_kv, page_size, D] fp16 page pools.
 * block_table: device int [B, max_pages_per_seq]; key j of sequence b is row
 *   j % page_size of page block_table[b * max_pages_per_seq + j / page_size].
 *   An id outside [0, num_pages) contributes no keys: the kernel never reads
 *   outside the pools.
 * kv_lens: device int [B], keys of each sequence, clamped to
 *   [0, max_pages_per_seq * page_size]; required.
 * page_size: a power of two in [16, 2^20].
 * Q, O, row_max, row_sumexp, flags (KF_ATTN_CAUSAL) as in kf_attn_fwd_ex,
 * with kv_len = max_pages_per_seq * page_size.  The decode path only: at
 * most 32 query rows per KV head ((H_q / H_kv) * q_len <= 32), else
 * KF_ERR_SIZE.  Workspace: kf_attn_decode_paged_workspace_bytes() bytes,
 * 256-byte aligned, no initialisation. */
size_t kf_attn_decode_paged_workspace_bytes(int B, int q_len, int H_q, int H_kv, int D,
                                            int page_size, int max_pages_per_seq);
int kf_attn_decode_paged(const void* Q, const void* K_pages, const void* V_pages,
                         const int* block_table, const int* kv_lens,
                         void* O, float* row_max, float* row_sumexp,
                         int B, int q_len, int H_q, int H_kv, int D,
                         int page_size, int max_pages_per_seq, int num_pages, int flags,
                         void* workspace, size_t workspace_bytes, void* stream);

/* The entry points from here to kf_kv_evict: a call of which a launch would
 * have 2^32 threads or more is KF_ERR_SIZE, before anything is launched. */

/* Attention over packed sequences: the tokens of all sequences one after the
 * other, as the projections write them.  No counterpart in the reference.
 *
 * Q [tokens_q, H_q, D], K and V [tokens_kv, H_kv, D], fp16 (bf16 with
 *   KF_BF16), D = 64, 128 or 256.  `strides`: NULL (contiguous), or six host
 *   values, token and head strides of Q, K and V in elements, multiples of 8,
 *   K's and V's token strides at most 2^28; the D channels of a head are
 *   contiguous.
 * q_starts, kv_starts: device int [n_seqs + 1], not decreasing: sequence b has
 *   the queries q_starts[b] .. q_starts[b + 1] - 1 and the keys kv_starts[b] ..
 *   kv_starts[b + 1] - 1; either may be empty.  The same array for prompts;
 *   more keys than queries for a chunk of a prompt over its context (see
 *   kf_kv4_read).  Values outside the tensors are clamped to them.
 * flags & KF_ATTN_CAUSAL: query i of n sees keys j <= i + (keys of its
 *   sequence) - n, as in kf_attn_fwd_ex.  A row that sees no key gets O = 0,
 *   Mi = -inf, Li = 0 (LSE = -inf).
 * O [tokens_q, H_q, D] contiguous, fp32 or by KF_ATTN_OUT_F16 / _BF16; row_max,
 *   row_sumexp [tokens_q, H_q], optional, as in kf_attn_fwd_ex (KF_ATTN_LSE).
 *   Rows of tokens outside the sequences are left as they were.
 * What tokens outside the sequences and other sequences hold does not matter; a
 * NaN or an infinity among a sequence's own keys or values may reach any row of
 * that sequence, also one that does not see it.  The statistics of a row that one
 * has reached mean nothing: its LSE may be NaN, or -inf as of a row without keys.
 * The softmax weights are rounded to the inputs' type before they meet V (relative
 * 2^-11 in fp16, 2^-8 in bf16, whatever O's type), since that product takes 16-bit
 * operands; Li and the LSE sum them in fp32.
 * Scores q . k / sqrt(D) may reach 9e7 in magnitude; from there on their fp32 rounding
 * can pass the range of a 16-bit weight, and rows may be NaN.
 * The sizes choose one of several layouts, which add up in different orders: a
 * sequence's last bits may differ between batches of other sizes, but not between
 * calls of the same sizes.
 * tokens_q, tokens_kv and n_seqs are positive; tokens_q H_q, tokens_kv H_kv and
 * tokens_kv H_q / H_kv are at most 2^31 - 1025.  No workspace. */
int kf_attn_packed(const void* Q, const void* K, const void* V, void* O,
                   float* row_max, float* row_sumexp, const int64_t* strides,
                   const int* q_starts, const int* kv_starts,
                   int n_seqs, int tokens_q, int tokens_kv, int H_q, int H_kv, int D,
                   int flags, void* stream);

/* RMS norm of every query and key head, then rotary positions, in one pass.
 * No counterpart in the reference.
 *
 * Q, Q_out [tokens, H_q, D], K, K_out [tokens, H_kv, D], fp16 (bf16 with
 *   KF_BF16), D = 16, 64, 128 or 256; `strides`: NULL (contiguous), or eight
 *   host values, token and head strides of Q, K, Q_out and K_out in elements,
 *   multiples of 8.  Q_out may be Q and K_out may be K, with the same strides;
 *   outputs that overlap anything else give undefined rows, and an output whose
 *   own rows overlap (a broadcast view in place) is KF_ERR_SIZE.
 * q_weight, k_weight: [D] of the same type, or NULL: Q or K is not normed.
 *   With one, x -> x / sqrt(mean(x^2) + eps) * weight over the D channels.
 * The first `rot` channels (a multiple of 16, 0 to D) of a head are turned by
 *   the angles positions[token] * freqs[i], i < rot / 2 (device double, radians
 *   per position, whatever context scaling they include), in the pairs
 *   (i, i + rot / 2) or, with KF_ROPE_INTERLEAVED, (2i, 2i + 1), and multiplied
 *   by `scale`; the others keep their normed values.
 * positions: device int [tokens].  positions and freqs may be NULL if rot is 0.
 * Computed in fp32 (the angles in fp64) and rounded once; the squares of a normed
 * bf16 row whose root mean square is above 1e18 pass fp32's range. */
int kf_qk_norm_rope(const void* Q, const void* K, void* Q_out, void* K_out,
                    const int64_t* strides, const void* q_weight, const void* k_weight,
                    const int* positions, const double* freqs,
                    int tokens, int H_q, int H_kv, int D, int rot, float eps, float scale,
                    int flags, void* stream);

/* A paged K/V cache in 4 bits.  No counterpart in the reference.
 *
 * Format: the microscaling one with 4-bit elements.  Every block of 32
 * consecutive channels of a row has one scale byte E (1 .. 254), scale
 * 2^(E - 127), and 32 codes (a sign bit over 0, .5, 1, 1.5, 2, 3, 4, 6).  E is
 * the exponent field of the block's largest magnitude as fp32, less 2, at
 * least 1; a channel is rounded to the nearest code, ties to the even code,
 * magnitudes above 6 scales to 6.  A block with an infinity or a NaN gets E = 255
 * and reads back as NaN.
 * K_pages, V_pages: [num_pages, H_kv, kf_kv4_page_bytes(page_size, D)] bytes;
 *   per page and head the codes of its rows [page_size][D / 2] (channel 2i in
 *   the low half of byte i), then their scales [page_size][D / 32].  D = 64,
 *   128 or 256; page_size a power of two in [16, 2^20].
 * block_table: device int [n_seqs, max_pages_per_seq], as in
 *   kf_attn_decode_paged. */
size_t kf_kv4_page_bytes(int page_size, int D);  /* 0 for an invalid size */

/* Quantise the new tokens' K and V into the cache.  K, V [tokens, H_kv, D] fp16
 * (bf16 with KF_BF16), packed by seq_starts (device int [n_seqs + 1], as in
 * kf_attn_packed); `strides`: NULL or four host values, token and head strides
 * of K and V.  kv_lens: device int [n_seqs], the keys of each sequence with the
 * new tokens: sequence b's packed tokens become its last ones.  A token whose
 * page id is outside [0, num_pages), or whose place is outside the table, is
 * not written; nor is one outside the sequences.  Two tokens of a call whose
 * places are the same row of the same page leave an undefined row. */
int kf_kv4_append(const void* K, const void* V, const int64_t* strides,
                  void* K_pages, void* V_pages, const int* block_table,
                  const int* seq_starts, const int* kv_lens,
                  int n_seqs, int tokens, int H_kv, int D,
                  int page_size, int max_pages_per_seq, int num_pages,
                  int flags, void* stream);

/* Read rows back: K, V [tokens, H_kv, D] contiguous, fp16 (bf16 with KF_BF16),
 * exactly the values the codes stand for (fp16 cannot hold all of a cache
 * written from bf16: beyond its range the nearest, by the conversion).
 * Sequence b's packed tokens (seq_starts) are its last ones of kv_lens[b], so
 * seq_starts = the running sum of kv_lens reads whole contexts, for
 * kf_attn_packed with these as kv_starts.  Tokens of no valid page get zeros;
 * rows outside the sequences are left as they were. */
int kf_kv4_read(const void* K_pages, const void* V_pages, const int* block_table,
                const int* seq_starts, const int* kv_lens, void* K, void* V,
                int n_seqs, int tokens, int H_kv, int D,
                int page_size, int max_pages_per_seq, int num_pages,
                int flags, void* stream);

/* Decode over the 4-bit cache: kf_attn_decode_paged's call and results for
 * pages in the format above.  Q [B, H_q, q_len, D] fp16 (bf16 with KF_BF16);
 * (H_q / H_kv) * q_len <= 32, else KF_ERR_SIZE; D = 64, 128 or 256.  The
 * workspace (256-byte aligned, no initialisation, not shared by calls that can
 * run concurrently) is required.  With KF_BF16 the softmax weights are rounded
 * to bf16 before they meet V, else to fp16; K and V are exactly what kf_kv4_read
 * with the same flags gives.  So a block with E = 255 is NaN: it makes the rows that
 * see its key NaN, or their 32 channels, and may reach any other row of its sequence, as
 * in kf_attn_packed; what pages hold past a sequence's keys does not matter.  Statistics
 * of such rows, the size of scores and the order of sums: as in kf_attn_packed. */
size_t kf_attn_decode_kv4_workspace_bytes(int B, int q_len, int H_q, int H_kv, int D,
                                          int page_size, int max_pages_per_seq);
int kf_attn_decode_kv4(const void* Q, const void* K_pages, const void* V_pages,
                       const int* block_table, const int* kv_lens,
                       void* O, float* row_max, float* row_sumexp,
                       int B, int q_len, int H_q, int H_kv, int D,
                       int page_size, int max_pages_per_seq, int num_pages, int flags,
                       void* workspace, size_t workspace_bytes, void* stream);

/* A paged K/V cache in 16 bits that is filled, attended to and kept small.  No
 * counterpart in the reference.
 *
 * K_pages, V_pages: [num_pages, H_kv, page_size, D] fp16 or bf16 page pools, as in
 *   kf_attn_decode_paged, which reads an fp16 one too.  D = 64, 128 or 256;
 *   page_size a power of two in [16, 2^20].
 * weights: [num_pages, H_kv, page_size] fp32, what every key has gathered
 *   (kf_kv_weigh), by the same block table.
 * block_table: device int [n_seqs, max_pages_per_seq], as in kf_attn_decode_paged;
 *   kv_lens: device int [n_seqs], the keys of each sequence, clamped to the
 *   table's places (kf_kv_append takes the values as they are, and writes no token
 *   whose place is outside the table); seq_starts: device int [n_seqs + 1], as in
 *   kf_attn_packed: sequence b's packed tokens are the last of its kv_lens[b] keys.
 * Sequences may share pages that are only read. */

/* Write the new tokens' K and V into the cache: kf_kv4_append's call for 16-bit
 * pages, copied bit for bit, so that fp16 and bf16 are alike (`flags`: 0 or KF_BF16).
 * weights: NULL, or the pool in which the new tokens' weights become 0. */
int kf_kv_append(const void* K, const void* V, const int64_t* strides,
                 void* K_pages, void* V_pages, float* weights, const int* block_table,
                 const int* seq_starts, const int* kv_lens,
                 int n_seqs, int tokens, int H_kv, int D,
                 int page_size, int max_pages_per_seq, int num_pages,
                 int flags, void* stream);

/* Attention of packed new tokens over the pages, their own keys among them (append
 * first): a step of one token, a chunk of a prompt over its context, or any mix.
 *
 * Q [tokens, H_q, D] fp16 (bf16 with KF_BF16, as the pools); `strides`: NULL
 *   (contiguous), or two host values, Q's token and head strides in elements,
 *   multiples of 8.  O [tokens, H_q, D], row_max, row_sumexp, flags (KF_ATTN_CAUSAL,
 *   _OUT_F16, _OUT_BF16, _LSE, KF_BF16) and what they give as in kf_attn_packed,
 *   the keys of sequence b being kv_lens[b]: query i of n sees keys j <= i +
 *   kv_lens[b] - n with KF_ATTN_CAUSAL.  A key whose page id is outside [0,
 *   num_pages) counts as none, and is never read; what pages hold past a
 *   sequence's keys does not matter.  NaN and infinities among a sequence's own
 *   keys, the size of scores, the rounding of the weights and the order of sums: as in
 *   kf_attn_packed; a sequence's keys are cut where the work of the whole call is
 *   shared out, so that its last bits depend on the other sequences' lengths.
 * Steps in fp16 that have one number of tokens each take 6 to 42 % less time in
 * kf_attn_decode_paged.  The layout goes by the average rows of a sequence, empty ones
 * among them: a prompt among many empty sequences takes longer than alone.
 * Workspace: kf_attn_paged_workspace_bytes() bytes (may be 0, then NULL will do),
 *   256-byte aligned, no initialisation, not shared by calls that can run
 *   concurrently; KF_ERR_WORKSPACE without.
 * n_seqs, tokens and tokens H_q as in kf_attn_packed. */
size_t kf_attn_paged_workspace_bytes(int n_seqs, int tokens, int H_q, int H_kv, int D,
                                     int page_size, int max_pages_per_seq);
int kf_attn_paged(const void* Q, const int64_t* strides, const void* K_pages, const void* V_pages,
                  const int* block_table, const int* seq_starts, const int* kv_lens,
                  void* O, float* row_max, float* row_sumexp,
                  int n_seqs, int tokens, int H_q, int H_kv, int D,
                  int page_size, int max_pages_per_seq, int num_pages, int flags,
                  void* workspace, size_t workspace_bytes, void* stream);

/* The attention weight that the keys gather:
 *   weights[key j] += sum over the new tokens i that see j and the query heads of the
 *   KV head's group of exp(q_i . k_j / sqrt(D) - lse_i),
 * in fp32 (the products' sums too), in an order that the sizes and lengths fix.
 * Q, strides, K_pages, tables and counts as in kf_attn_paged, of which lse
 * [tokens, H_q] is the row_max with KF_ATTN_LSE (natural logarithm); a row whose lse
 * is -inf adds nothing, whatever it and the keys hold.  flags: KF_ATTN_CAUSAL, KF_BF16.
 * A NaN or an infinity in another row of Q, or a NaN in its lse, reaches the keys that
 * the row sees and no others, one in a key the key's own weight.  Sequences that share a
 * page race for its weights: they must not.
 * Workspace: kf_kv_weigh_workspace_bytes() bytes (may be 0, then NULL will do), as
 * kf_attn_paged's. */
size_t kf_kv_weigh_workspace_bytes(int n_seqs, int tokens, int H_q, int H_kv, int D,
                                   int page_size, int max_pages_per_seq);
int kf_kv_weigh(const void* Q, const int64_t* strides, const void* K_pages, float* weights,
                const int* block_table, const int* seq_starts, const int* kv_lens,
                const float* lse, int n_seqs, int tokens, int H_q, int H_kv, int D,
                int page_size, int max_pages_per_seq, int num_pages, int flags,
                void* workspace, size_t workspace_bytes, void* stream);

/* Cut every sequence from n = kv_lens[b] to m = min(n, budgets[b]) keys (device int
 * [n_seqs], a negative one counts as 0).  Of every KV head the last r = min(recent, m)
 * keys stay, and of the n - r before them the k = m - r of largest weight, ties to
 * the lowest place; a NaN counts as larger than any number, -0 as 0.
 * Attention does not depend on the order of the keys.  Of the old ones only those move
 * that have to: kept keys in places below k stay there, those from k on go, in order,
 * to the freed places below k, in order.  The last r, which stay in order, all move, to
 * k .. m - 1.  K, V and weights move alike; places from m on are left as they were.
 * kept: device int [n_seqs], receives m, or n where nothing is cut or a page id of the
 *   n keys is outside [0, num_pages): such a sequence is left as it is.  It may be
 *   kv_lens or budgets itself.
 * Sequences that are cut must not share a page with another one of the call, nor
 *   have one twice: what these pages hold is then undefined.
 * Workspace: kf_kv_evict_workspace_bytes() bytes, 256-byte aligned, no initialisation,
 *   not shared by calls that can run concurrently: 4 bytes for every place of the table and
 *   KV head (268 MB for 64 sequences, 8 heads and 131072 places), however few keys
 *   there are, and 16 for every sequence and KV head. */
size_t kf_kv_evict_workspace_bytes(int n_seqs, int H_kv, int D, int page_size,
                                   int max_pages_per_seq);
int kf_kv_evict(void* K_pages, void* V_pages, float* weights, const int* block_table,
                const int* kv_lens, const int* budgets, int* kept,
                int n_seqs, int H_kv, int D,
                int page_size, int max_pages_per_seq, int num_pages, int recent,
                void* workspace, size_t workspace_bytes, void* stream);

/* The reference launcher's contract (tests/test_flash_attn.cu:52-113):
 * q_len = kv_len = S, scratch allocated and freed by the call, stream
 * synchronised before returning.  Returns a hipError_t value:
 * hipSuccess (0), hipErrorInvalidValue for an unsupported D or an invalid
 * shape, or the HIP error of a failed allocation / launch / sync. */
int kf_launch_flash_attn(const uint16_t* Q, const uint16_t* K, const uint16_t* V,
                         float* O, int B, int S, int H_q, int H_kv, int D,
                         void* stream);

/* Human-readable text for a kf_status value (static storage). */
const char* kf_status_string(int status);

/* hipError_t of the last failed HIP call made by a kf_* entry point on the
 * calling thread (0 if none). */
int kf_last_hip_error(void);

/* Library version string. */
const char* kf_version(void);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* KF_ATTN_H */
