/*
 * muzo_b200.h — C ABI of the B200 (sm_100a) kernels behind MuZO-Clip's optimizer hot path.
 *
 * Every entry point takes plain device pointers, sizes and a cudaStream_t passed as void*,
 * enqueues its work on that stream and returns a muzo_status code. Nothing here allocates
 * device memory: tables, accumulators and workspaces are owned by the caller.
 *
 * Reference interfaces replaced (paths inside turfur44/MuZO-Clip):
 *   hash64_seed              muzo_clip/prng.py:19-36         (muzo_hash64_seed)
 *   make_zo_noise_like       muzo_clip/prng.py:39-81         (muzo_fill_noise)
 *   _perturb_selected        muzo_clip/muzo_optimizer.py:434-446 (muzo_perturb_segments)
 *   step(): momentum rebuild muzo_clip/muzo_optimizer.py:318-333 (muzo_rebuild_segments)
 *   zeropower_via_newtonschulz5 muzo_clip/newton_schulz.py:35-66
 *                            (muzo_ns_prepare, muzo_ns_normalize, muzo_ns_gemm)
 *   step(): scale/clip/apply muzo_clip/muzo_optimizer.py:340-357, _rms 73-74
 *                            (muzo_update_sumsq, muzo_apply_update)
 *   QK-Clip max-logit probe  muzo_clip/qk_clip.py:173-196     (muzo_qk_max)
 *   QK-Clip row scaling      muzo_clip/qk_clip.py:262-322     (muzo_qk_scale_rows)
 */
#ifndef MUZO_B200_H
#define MUZO_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MUZO_ABI_VERSION 2

/* Status codes. MUZO_ERR_CUDA carries the last CUDA error in muzo_last_cuda_error(). */
enum muzo_status {
  MUZO_OK = 0,
  MUZO_ERR_ARG = 1,          /* null pointer, negative size, bad enum value */
  MUZO_ERR_DTYPE = 2,        /* dtype not supported by this entry point */
  MUZO_ERR_ALIGN = 3,        /* pointer or leading dimension violates the 16-byte rule */
  MUZO_ERR_CUDA = 4,         /* a CUDA runtime call failed */
  MUZO_ERR_CAPACITY = 5,     /* caller-provided table too small */
  MUZO_ERR_UNSUPPORTED = 6   /* shape or device not supported (e.g. not sm_100) */
};

/* Element types of parameter blocks and buffers. */
enum muzo_dtype { MUZO_F32 = 0, MUZO_BF16 = 1, MUZO_F16 = 2 };

/* Noise distributions (prng.py:16, NoiseDistribution). */
enum muzo_dist { MUZO_NORMAL = 0, MUZO_RADEMACHER = 1 };

/*
 * One launch unit of the noise stream. A parameter block of `numel` elements is generated by
 * torch's CUDA generator as one grid-stride launch, or — once the noise tensor no longer fits
 * 32-bit byte offsets — as several launches over halves of it, each with its own thread count
 * and Philox offset. muzo_plan_segments() reproduces that split; non-noise kernels use one
 * segment per block. 64 bytes, naturally aligned.
 */
typedef struct muzo_segment {
  void*    param;          /* base of the parameter block (element 0 of the block) */
  void*    out;            /* base of the block's output buffer, or NULL */
  int64_t  numel;          /* elements in this segment */
  int64_t  item_begin;     /* prefix sum of work items, padded to MUZO_ITEMS_PER_CTA */
  uint64_t philox_offset;  /* Philox offset of the launch, in 32-bit words (multiple of 4) */
  uint32_t threads;        /* total threads S of the emulated launch (blockDim * gridDim) */
  int32_t  block_index;    /* index of the parameter block: keys, sums and flags are per block */
  int64_t  elem_start;     /* element offset of this segment inside its block */
  void*    kept;           /* base of the block's kept noise (muzo_rebuild_segments_kept), or NULL */
} muzo_segment;

/* Work items handled by one CTA of the segment kernels; every segment's item range is padded to
 * a multiple of it so that a CTA never straddles two segments. */
#define MUZO_ITEMS_PER_CTA 1024

/* Per-block accumulator slots (double[MUZO_NSUMS] per block) used by the step kernels. */
enum muzo_sum_slot {
  MUZO_SUM_M2 = 0,        /* sum of M^2 of the fp32 momentum (zero-norm test) */
  MUZO_SUM_X2 = 1,        /* sum of bf16(M)^2 (Newton-Schulz normalisation) */
  MUZO_SUM_W2 = 2,        /* sum of W^2 of the parameter block before the update */
  MUZO_SUM_U2 = 3,        /* sum of U^2, U = NS(M) * sqrt(max(rows, cols)) * muon_scale */
  MUZO_SUM_U2_CLIPPED = 4,/* sum of the clipped update squared (reported update_rms) */
  MUZO_NSUMS = 8
};

/* Per-block flag bits (int32 per block). */
enum muzo_block_flag {
  MUZO_FLAG_NONFINITE_INPUT = 1,   /* M had a non-finite entry: NS returns zeros */
  MUZO_FLAG_ZERO_NORM = 2,         /* ||M|| == 0 or non-finite: NS returns zeros */
  MUZO_FLAG_NONFINITE_OUTPUT = 4   /* NS output non-finite: NS returns zeros */
};

/* Per-block step statistics written by muzo_apply_update (float[MUZO_NSTATS] per block). */
enum muzo_stat_slot {
  MUZO_STAT_RATIO_BEFORE = 0,  /* lr*rms(U)/(rms(W)+1e-12) before the ratio clip */
  MUZO_STAT_CLIP_FACTOR = 1,   /* multiplier applied to U (1 when not clipped) */
  MUZO_STAT_ZEROED = 2,        /* 1 when NS returned zeros for this block */
  MUZO_NSTATS = 4
};

/* ---------------------------------------------------------------- host-only utilities */

int         muzo_abi_version(void);
const char* muzo_status_string(int status);
int         muzo_last_cuda_error(void);

/* Kernels that the attention and the gradient entry points below have enqueued in this process (their number
 * depends on the arguments; the other entry points enqueue a fixed number per call). */
int64_t     muzo_launches(void);

/* blake2b-64 of "seed|name|d0,d1|block" masked to 63 bits (prng.py:19-36). `shape` has `ndim`
 * entries. Returns the key through *key_out. Pure host code. */
int muzo_hash64_seed(uint64_t base_seed, const char* name, const int64_t* shape, int ndim,
                     int64_t block_index, uint64_t* key_out);

/* Plan the noise launch units of `nblocks` blocks (prng.py:63-79 through torch's CUDA
 * generator): numels[i] elements each, noise element size 4 (normal, fp32) or 1 (Rademacher,
 * int8), on a device with `sm_count` SMs and `max_threads_per_sm` threads per SM. params[i] and
 * outs[i] (outs may be NULL) are the block base pointers copied into the segments. Writes at
 * most `capacity` segments; *nsegs and *total_items receive the counts. Pure host code. */
int muzo_plan_segments(const int64_t* numels, void* const* params, void* const* outs, int nblocks,
                       int dist, int sm_count, int max_threads_per_sm, muzo_segment* segs,
                       int capacity, int* nsegs, int64_t* total_items);

/* Plan one plain segment per block for the element-wise step kernels: 8 elements per item. */
int muzo_plan_linear(const int64_t* numels, void* const* params, void* const* outs, int nblocks,
                     muzo_segment* segs, int capacity, int* nsegs, int64_t* total_items);

/* ---------------------------------------------------------------- noise and perturbation */

/* make_zo_noise_like (prng.py:39-81): write the noise of one block (its segments in d_segs,
 * key `key`) into segs[i].out as `out_dtype` (the value torch gives after .to(dtype)). */
int muzo_fill_noise(const muzo_segment* d_segs, int nsegs, int64_t total_items, uint64_t key,
                    int dist, int out_dtype, void* stream);

/* _perturb_selected (muzo_optimizer.py:434-446) for every segment in the table at once:
 * W <- dtype(W + alpha * dtype(Z(keys[block_index]))), in place, Z regenerated in registers. */
int muzo_perturb_segments(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                          const uint64_t* d_keys, int dtype, int dist, float alpha, void* stream);

/* Noise kept between the passes of one projection (no counterpart in the reference, whose three
 * passes +eps, -2eps, +eps each regenerate the same noise). muzo_perturb_segments with normal
 * noise that also stores the rounded noise dtype(Z) of every element to segs[i].out (a buffer of
 * the block's dtype and element layout; a segment whose out is NULL is only perturbed). */
int muzo_perturb_segments_keep_noise(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                                     const uint64_t* d_keys, int dtype, float alpha, void* stream);

/* The perturbation of a later pass from the kept noise: W <- dtype(W + alpha * Zk) per linear
 * segment (muzo_plan_linear with params = the blocks, outs = their kept noise), the same values
 * muzo_perturb_segments computes by regenerating the noise of the key the noise was kept for. */
int muzo_perturb_kept_noise(const muzo_segment* d_segs, int nsegs, int64_t total_items, int dtype,
                            float alpha, void* stream);

/* ---------------------------------------------------------------- step kernels */

/* Momentum rebuild (muzo_optimizer.py:318-333) of every block in the table:
 *   M = sum_{h<horizon} alphas[h] * float(dtype(Z(keys[block*horizon + h])))  (h = age, newest 0)
 *   M = M * inv_coeff_sum   (when normalize != 0)
 * writes bf16(M) to segs[i].out, accumulates MUZO_SUM_M2, MUZO_SUM_X2 and MUZO_SUM_W2 (reading
 * the block's current weights from segs[i].param) into d_sums, and sets
 * MUZO_FLAG_NONFINITE_INPUT in d_flags. max_ctas > 0 caps the grid (each CTA then walks several
 * chunks of MUZO_ITEMS_PER_CTA items), e.g. one CTA per SM beside a concurrent GEMM; 0 launches
 * one CTA per chunk. */
int muzo_rebuild_segments(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                          const uint64_t* d_keys, const float* d_alphas, int horizon, int dist,
                          int param_dtype, int normalize, float inv_coeff_sum, double* d_sums,
                          int32_t* d_flags, int max_ctas, void* stream);

/* muzo_rebuild_segments (normal noise only) whose newest history entry, h = 0, is read from the
 * noise kept for its key — segs[i].kept, written by muzo_perturb_segments_keep_noise in the
 * block's dtype and layout — instead of being regenerated; the older entries are regenerated.
 * The same values as muzo_rebuild_segments; a segment whose kept pointer is NULL regenerates
 * all entries. No counterpart in the reference. */
int muzo_rebuild_segments_kept(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                               const uint64_t* d_keys, const float* d_alphas, int horizon,
                               int param_dtype, int normalize, float inv_coeff_sum, double* d_sums,
                               int32_t* d_flags, int max_ctas, void* stream);

/* History-wide kept noise (no counterpart in the reference, which regenerates every history
 * entry's noise from its seed in each step). d_slot_base[h] (device, `horizon` entries, h = age,
 * newest 0) is the base address of a slot holding history entry h's rounded noise dtype(Z) for
 * every block — written by muzo_perturb_segments_keep_noise when that entry's projection ran —
 * or 0 when that entry's noise is not kept; segs[i].kept holds the block's BYTE OFFSET inside
 * every slot (not a pointer). Entries with a slot are read, the others regenerated: the same
 * values as muzo_rebuild_segments with normal noise (the same fp32 multiply-adds in the same
 * order), and the same sums and flags. Noise-stream segments (muzo_plan_segments). */
int muzo_rebuild_segments_history(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                                  const uint64_t* d_keys, const float* d_alphas, const uint64_t* d_slot_base,
                                  int horizon, int param_dtype, int normalize, float inv_coeff_sum,
                                  double* d_sums, int32_t* d_flags, int max_ctas, void* stream);

/* The history rebuild when EVERY entry is kept (all d_slot_base[h] nonzero): a plain stream over
 * linear segments (muzo_plan_linear with params = the blocks, outs = the bf16(M) buffers; kept =
 * the block's byte offset inside a slot), reading 2 * horizon + 2 bytes and writing 2 bytes per
 * 16-bit weight instead of regenerating the noise. Same values, sums and flags as
 * muzo_rebuild_segments_history. */
int muzo_rebuild_kept_linear(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                             const float* d_alphas, const uint64_t* d_slot_base, int horizon, int param_dtype,
                             int normalize, float inv_coeff_sum, double* d_sums, int32_t* d_flags,
                             void* stream);

/* Newton-Schulz input of arbitrary matrices (newton_schulz.py:35-46): segs[i].out = bf16(G) for
 * G = segs[i].param of `dtype`; accumulates MUZO_SUM_M2 (fp32 G^2) and MUZO_SUM_X2, and sets
 * MUZO_FLAG_NONFINITE_INPUT for a non-finite G. */
int muzo_ns_prepare(const muzo_segment* d_segs, int nsegs, int64_t total_items, int dtype,
                    double* d_sums, int32_t* d_flags, void* stream);

/* X <- bf16(X / (||X||_F + 1e-7)) per block (newton_schulz.py:35-53); X is segs[i].out.
 * Sets MUZO_FLAG_ZERO_NORM for blocks whose fp32 momentum norm is zero or non-finite. */
int muzo_ns_normalize(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                      const double* d_sums, int32_t* d_flags, void* stream);

/* Allocation-free variant of muzo_ns_prepare + muzo_ns_normalize (no counterpart in the
 * reference). For callers that cannot allocate device memory — a runtime that reserves the whole
 * device pool at start-up and forbids cudaMalloc afterwards, or a plugin inside another
 * framework whose allocator owns every byte — the segment table and the sums of squares live in
 * a file-scope device array of fixed size instead of caller buffers: at most
 * MUZO_NOALLOC_MAX_BLOCKS matrices per call (more returns MUZO_ERR_CAPACITY before any GPU work).
 * inputs[i] (numels[i] elements of `dtype`) becomes outputs[i] = bf16(G)/(||bf16(G)||_F + 1e-7);
 * d_flags[i] receives MUZO_FLAG_NONFINITE_INPUT / MUZO_FLAG_ZERO_NORM. inputs, outputs and
 * numels are host arrays of device pointers and sizes. The first call on a device looks up the
 * array's device address (make it before any stream capture). All calls share the array: calls
 * whose kernels overlap on one GPU race and must be serialised. The array (8 KB) stays resident
 * on every GPU that loaded the library until the process exits. */
#define MUZO_NOALLOC_MAX_BLOCKS 64
int muzo_ns_normalize_noalloc(const void* const* inputs, void* const* outputs, const int64_t* numels,
                              int nblocks, int dtype, int32_t* d_flags, void* stream);

/* Epilogues of the Newton-Schulz GEMM D = op(A) * op(B):
 *   MUZO_EPI_STORE:  D = bf16(acc)                                   (A = X X^T)
 *   MUZO_EPI_POLY:   D = bf16(bf16(c1*E) + bf16(c2*bf16(acc)))       (B = b A + c A A, E = A)
 *   MUZO_EPI_UPDATE: D = bf16(bf16(c1*E) + bf16(acc))                 (X = a X + B X,  E = X)
 * (newton_schulz.py:55-58). */
enum muzo_epilogue { MUZO_EPI_STORE = 0, MUZO_EPI_POLY = 1, MUZO_EPI_UPDATE = 2 };

/* Batched bf16 GEMM on tcgen05 tensor cores, fp32 accumulation in TMEM, fused epilogue.
 * Logical shapes: D[b] (M x N) = sum_k A[b](m, k) * B[b](k, n).
 *   a_mn = 0: A stored row-major M x K (K contiguous, leading dim lda);
 *   a_mn = 1: A stored row-major K x M (M contiguous);
 *   b_mn = 0: B stored as N x K rows (K contiguous), i.e. D = A * B_stored^T;
 *   b_mn = 1: B stored row-major K x N (N contiguous).
 * Every matrix of batch b starts at base + b * batch_stride (elements). All leading dimensions
 * must be multiples of 8 elements and all bases 16-byte aligned. E (epilogue operand) has the
 * layout of D (ldd). symmetric != 0 declares D symmetric (m == n; store and b*A + c*A*A
 * epilogues only, with E symmetric): only the tiles that hold an element on or above the
 * diagonal are computed and every such element is also written to its mirror position, which
 * halves the tensor work of X X^T and A A.
 * d_sums, d_scales, d_flags (MUZO_EPI_UPDATE only; all NULL to skip): the last iteration's update
 * epilogue also accumulates, per batch index b, d_sums[b * MUZO_NSUMS + MUZO_SUM_U2] +=
 * sum of (fp32(D[b]) * d_scales[b])^2 over the stored values, and sets MUZO_FLAG_NONFINITE_OUTPUT
 * in d_flags[b] for a non-finite D[b] — what muzo_update_sumsq computes in a separate pass.
 * d_status points to four device int32 words, zero before the first call: [0] status — every
 * wait inside the kernel is bounded, and on timeout a nonzero code (1 producer, 2 MMA, 3
 * epilogue) is written there while the kernel drains its own copies and MMAs, frees its TMEM and
 * returns; [1], [2] the tile scheduler's counters (output tiles are handed out by an atomic
 * counter so that CTAs delayed by concurrent kernels take fewer tiles; the kernel leaves both
 * zero when it ends, after a timeout too); [3] stall request, zero in normal use: a value r in
 * 1..3 makes that role (1 producer, 2 MMA issuer, 3 epilogue) wait, before its first step, on a
 * barrier nothing arrives at, so that its bounded wait expires and the launch ends through the
 * timeout path with status r (for testing the timeout path; the launch takes about 2 s). Calls
 * whose kernels may run at the same time need distinct d_status buffers. NULL selects
 * library-internal words shared by all such calls. After a nonzero status D is unspecified: the
 * caller must not consume it and must zero word [0] before the next call (the Python engine
 * raises once the step's statistics are read; the weights that step wrote are then unspecified
 * too, as the apply kernels are already queued behind the GEMMs). */
int muzo_ns_gemm(const void* a, int64_t lda, int64_t a_batch_stride, int a_mn,
                 const void* b, int64_t ldb, int64_t b_batch_stride, int b_mn,
                 void* d, int64_t ldd, int64_t d_batch_stride,
                 const void* e, int epilogue, float c1, float c2,
                 int64_t m, int64_t n, int64_t k, int64_t batch, int symmetric,
                 double* d_sums, const float* d_scales, int32_t* d_flags,
                 int32_t* d_status, void* stream);

/* Sum of U^2 and finiteness of the Newton-Schulz result X (segs[i].out) per block, with
 * U = fp32(X) * scales[block] (muzo_optimizer.py:336-342). Sets MUZO_FLAG_NONFINITE_OUTPUT. */
int muzo_update_sumsq(const muzo_segment* d_segs, int nsegs, int64_t total_items,
                      const float* d_scales, double* d_sums, int32_t* d_flags, void* stream);

/* Apply the update of every block (muzo_optimizer.py:340-353):
 *   U = fp32(X) * scales[block]; ratio = lr*rms(U)/(rms(W)+1e-12);
 *   if ratio > ratio_clip: U *= ratio_clip/ratio;
 *   W = dtype(W - lr * dtype(U)); if weight_decay: W = dtype(W * (1 - lr*wd)).
 * Blocks flagged in d_flags use U = 0. Writes d_stats (float[MUZO_NSTATS] per block) and
 * accumulates MUZO_SUM_U2_CLIPPED. `decay` = 1 - lr*wd as the reference's float scalar;
 * apply_decay = 0 skips the multiply. */
int muzo_apply_update(const muzo_segment* d_segs, int nsegs, int64_t total_items, int dtype,
                      const float* d_scales, float lr, double ratio_clip, int apply_decay,
                      float decay, double* d_sums, const int32_t* d_flags, float* d_stats,
                      void* stream);

/* ---------------------------------------------------------------- QK-Clip */

/* Per-head max of the pre-softmax logits of eager attention (qk_clip.py:173-196), computed from
 * Q [B, Hq, Sq, D] and K [B, Hkv, Sk, D] (element strides given, D contiguous; GQA kv head
 * h / (Hq / Hkv)) without materialising the logits:
 *   smax[h] = round(round(max_{b, i, j} q[b,h,i] . k[b,kv,j]) * scale) in `dtype`,
 * over j <= i + (Sk - Sq) when causal. smax (float[Hq]) is overwritten; *d_valid is set to 1, or
 * 0 when a logit is non-finite (the reference then drops the capture) or when one of the
 * tensor-core kernel's bounded waits expired (the capture is dropped the same way). */
int muzo_qk_max(const void* q, const void* k, int dtype, int64_t batch, int64_t hq, int64_t hkv,
                int64_t seq_q, int64_t seq_k, int64_t head_dim,
                int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
                int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
                int causal, float scale, float* smax, int32_t* d_valid, void* stream);

/* muzo_qk_max over the keys each batch row attends to: key j is visible to query i of batch b
 * when d_key_lo[b] <= j < d_key_hi[b] (device int32 per batch, clamped to [0, Sk]) and, when
 * causal, j <= i + (Sk - Sq). This is the eager capture of qk_clip.py:173-196 under a padding
 * mask (left or right padding, with or without causality), where the masked logits, shifted by
 * the dtype's minimum, never reach the maximum. Both pointers NULL: muzo_qk_max. */
int muzo_qk_max_ranges(const void* q, const void* k, int dtype, int64_t batch, int64_t hq, int64_t hkv,
                       int64_t seq_q, int64_t seq_k, int64_t head_dim,
                       int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
                       int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
                       int causal, const int32_t* d_key_lo, const int32_t* d_key_hi, float scale,
                       float* smax, int32_t* d_valid, void* stream);

/* Per-head max of materialised logits [B, H, Sq, Sk] of `dtype` (the softmax-input capture,
 * qk_clip.py:188-196): out (float[H]) overwritten, *d_valid = 0 if any logit is non-finite. */
int muzo_logits_head_max(const void* logits, int dtype, int64_t batch, int64_t heads, int64_t seq_q,
                         int64_t seq_k, int64_t stride_b, int64_t stride_h, int64_t stride_q,
                         int64_t stride_k, float* out, int32_t* d_valid, void* stream);

/* running[i] = max(running[i], fresh[i]) for i < n, skipped entirely when d_valid is non-NULL and
 * *d_valid == 0 (the running maximum of qk_clip.py:195-196, kept on the device). */
int muzo_max_merge(float* running, const float* fresh, const int32_t* d_valid, int64_t n, void* stream);

/* Attention forward with the per-head maximum of the pre-softmax logits as a side output: the
 * eager capture of qk_clip.py:173-196 taken from the attention the forward computes anyway, so
 * Q K^T is formed once (no counterpart in the reference, whose capture needs eager attention).
 * Q [B, Hq, Sq, D], K and V [B, Hkv, Sk, D] (element strides, D contiguous, GQA kv head
 * h / (Hq / Hkv)), bf16 or fp16, D a multiple of 8 up to 128; out[b, h, i, :] at o_stride_b * b + o_stride_h
 * * h + o_stride_s * i (for transformers' [B, Sq, Hq, D] output: Sq*Hq*D, D, Hq*D) receives
 * softmax(scale * Q K^T) V over the visible keys (fp32 accumulation, P rounded to the input
 * dtype, the products' operand type), zeros for a row without a visible key. Key j is visible to
 * query i of batch b when d_key_lo[b] <= j < d_key_hi[b] (device int32 per batch; NULL: 0 and
 * Sk) and, when causal, j <= i + Sk - Sq. With smax non-NULL, smax[h] (float[Hq], overwritten)
 * = dtype(dtype(max over the visible logits of q . k) * scale) and *d_valid = 0 when a visible
 * logit is non-finite, else 1. Forward only. d_status: two device int32 words, zero before the
 * first call: [0] status — a nonzero code (1 producer, 2 MMA, 3 softmax) when a bounded wait
 * expired (the rows of out, and of lse below, that were computed then are NaN, *d_valid is 0); [1] a stall request, 0 in normal use: a test sets a
 * role's code there to make that role's first wait expire. */
int muzo_attention_max(const void* q, const void* k, const void* v, void* out, int dtype, int64_t batch,
                       int64_t hq, int64_t hkv, int64_t seq_q, int64_t seq_k, int64_t head_dim,
                       int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
                       int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
                       int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
                       int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s, int causal, float scale,
                       const int32_t* d_key_lo, const int32_t* d_key_hi, float* smax, int32_t* d_valid,
                       int32_t* d_status, void* stream);

/* muzo_attention_max that also keeps, when lse is non-NULL, the natural logarithm of each row's sum
 * of exp(scale * logit) over its visible keys, lse[b][h][i] (float[B * Hq * Sq], -inf for a row
 * that sees none): the statistic muzo_attention_backward recomputes the probabilities from. The
 * scale must then be positive. Sk = 0 is allowed, here and in muzo_attention_max (K and V may then
 * be NULL), and writes zeros. */
int muzo_attention_max_lse(const void* q, const void* k, const void* v, void* out, float* lse, int dtype,
                           int64_t batch, int64_t hq, int64_t hkv, int64_t seq_q, int64_t seq_k, int64_t head_dim,
                           int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
                           int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
                           int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
                           int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s, int causal, float scale,
                           const int32_t* d_key_lo, const int32_t* d_key_hi, float* smax, int32_t* d_valid,
                           int32_t* d_status, void* stream);

/* Gradients of that attention (no counterpart in the reference, which trains without gradients):
 * with P = exp(scale * Q K^T - lse) over the visible pairs, dP = dO V^T, delta = rowsum(dO * O) and
 * dS = P * (dP - delta):  dV = P^T dO, dK = scale * dS^T Q, dQ = scale * dS K, dK and dV summed over
 * the Hq / Hkv query heads of a key head. A row that sees no key has no gradient and gives none, whatever
 * its Q and dO hold. P and dS enter the products in the input type, sums are
 * fp32. Nothing is added atomically: equal calls give equal bits. Any of dq, dk, dv may be NULL
 * (dq alone, or dk and dv, skip the other's work). `strides` (host memory, 24 entries): the element
 * strides (batch, head, sequence) of q, k, v, out, dout, dq, dk, dv, all multiples of 8 and, for the
 * inputs, nonzero; D contiguous, bases 16-byte aligned. d_workspace: device memory of at least
 * muzo_attention_backward_workspace(...) bytes (negative: a shape this call refuses), 16-byte
 * aligned, that no other call uses until this one has finished. d_status as in muzo_attention_max: when a
 * wait expired, the rows of dq, dk and dv that were computed then are NaN. */
int64_t muzo_attention_backward_workspace(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t seq_q,
                                          int64_t seq_k, int64_t head_dim, int causal);
int muzo_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* dout,
                            const float* lse, void* dq, void* dk, void* dv, int dtype, int64_t batch, int64_t hq,
                            int64_t hkv, int64_t seq_q, int64_t seq_k, int64_t head_dim, const int64_t* strides,
                            int causal, float scale, const int32_t* d_key_lo, const int32_t* d_key_hi,
                            void* d_workspace, int64_t workspace_bytes, int32_t* d_status, void* stream);

/* Row-group scaling of a projection weight (qk_clip.py:287-308): rows
 * [g*rows_per_group, (g+1)*rows_per_group) are multiplied by factors[g] (already rounded to
 * the weight dtype) when mask[g] != 0. w is row-major [groups*rows_per_group, cols]. */
int muzo_qk_scale_rows(void* w, int dtype, int64_t groups, int64_t rows_per_group, int64_t cols,
                       const float* d_factors, const int32_t* d_mask, void* stream);

/* ---------------------------------------------------------------- gradient norm and clipping */

/* The norm over `count` tensors at once (no counterpart in the reference, which has no gradients):
 * src, numel and dtype are host arrays of device addresses, element counts and muzo_dtype codes;
 * types may mix, empty tensors are skipped, addresses need only their element's alignment. *d_norm
 * (device float) = sqrt(sum g^2), summed in fp64 over fp32 partial squares, or max |g| when
 * inf_norm != 0 (NaN if any g is NaN). Two launches for up to 1150 tensors: the tables travel as
 * kernel parameters, so the host arrays are free again when the call returns.
 * muzo_grad_clip also writes dst[i] = dst_dtype(g * min(1, max_norm / (norm + 1e-6))): dst_dtype[i]
 * is src_dtype[i] or MUZO_F32, dst[i] may be src[i] (same type), and what is written must not
 * otherwise overlap anything the call reads or writes (MUZO_ERR_ARG). A NaN norm makes every
 * result NaN. d_workspace: muzo_grad_workspace(count, total elements) bytes of device memory,
 * 8-byte aligned, that no other call uses until this one has finished (negative: bad arguments). */
int64_t muzo_grad_workspace(int64_t count, int64_t elements);
int muzo_grad_norm(const uint64_t* src, const int64_t* numel, const int32_t* dtype, int64_t count, int inf_norm,
                   float* d_norm, void* d_workspace, int64_t workspace_bytes, void* stream);
int muzo_grad_clip(const uint64_t* src, const uint64_t* dst, const int64_t* numel, const int32_t* src_dtype,
                   const int32_t* dst_dtype, int64_t count, int inf_norm, float max_norm, float* d_norm,
                   void* d_workspace, int64_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------- weight exchange between ranks */

/* The step of a data-parallel job is sharded by matrix: each rank orthogonalises and updates the
 * blocks it owns and must then place them in every other rank's replica (no counterpart in the
 * reference, which runs in one process). These entry points give the owner direct access to the
 * peers' parameter memory on the same node and push blocks with the copy engines.
 *
 * muzo_ipc_export: the interprocess handle (MUZO_IPC_HANDLE_BYTES opaque bytes) of the device
 * allocation that contains d_ptr, d_ptr's byte offset in it and the allocation's size.
 * MUZO_ERR_UNSUPPORTED when the allocation cannot be shared this way (for example memory of a
 * virtual-memory or stream-ordered pool); the caller then exchanges through collectives.
 * muzo_ipc_import: maps a handle exported by another process of the node (once per handle and
 * process) and returns the mapping's base; muzo_ipc_close unmaps it.
 * muzo_push_blocks: n device-to-device copies dst[i] <- src[i] of bytes[i] bytes, in order on
 * `stream`, one cudaMemcpyAsync each (dst may be a peer mapping): no kernel is launched. */
#define MUZO_IPC_HANDLE_BYTES 64
int muzo_ipc_export(const void* d_ptr, void* handle_out, uint64_t* offset_out, uint64_t* alloc_bytes_out);
int muzo_ipc_import(const void* handle, void** d_base_out);
int muzo_ipc_close(void* d_base);
int muzo_push_blocks(void* const* dst, const void* const* src, const uint64_t* bytes, int n, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MUZO_B200_H */
