/*
 * mimir_prefixlm.h -- C ABI of the MI355X (gfx950) prefix-LM attention library
 * (libmimir_prefixlm.so).
 *
 * Prefix-LM attention over packed variable-length sequences: inside sequence s
 * (tokens cu_seqlens[s] .. cu_seqlens[s+1]) with prefix length p = prefix_lens[s],
 * local query i may attend local key j iff
 *
 *     j < kend(i),   kend(i) = max(p, i + 1)        (is_causal == 0)
 *     j < i + 1                                    (is_causal != 0)
 *
 * i.e. bidirectional inside the prefix and causal after it
 * (reference: src/mimir/model/flash_attention_prefixlm_dense.py:61-69 and the
 * Metal predicate src/mimir/model/flash_attention_prefixlm_mps.py:43-51).
 *
 * Layout: q [T, Hq, D], k/v [T, Hkv, D], out [T, Hq, D]; every tensor has a
 * unit stride on the last (head_dim) axis and arbitrary token / head strides
 * given in ELEMENTS.  v may therefore be the strided split of a fused
 * gate/q/k/v projection (reference: src/mimir/model/layers.py:183-184).
 * lse is float32 [Hq, T] (natural log of the softmax denominator, scale
 * included), the FlashAttention varlen convention used by
 * src/mimir/model/flash_attention_prefixlm_v2.py:159-160.
 * GQA: query head h reads kv head h / (Hq / Hkv)
 * (reference: flash_attention_prefixlm_dense.py:10-16, repeat_interleave).
 *
 * Query rows >= total_seqlen and rows outside every sequence produce O = 0,
 * lse = -inf and zero dQ (reference: flash_attention_prefixlm_dense.py:43,79-80;
 * flash_attention_prefixlm_v2.py:143,224-226).
 *
 * All device pointers are plain HIP device addresses; `stream` is a hipStream_t
 * (passed as void* so that this header needs no HIP include).  Every entry point
 * only enqueues work on `stream` and never synchronises it.  Status 0 is success;
 * on failure mimir_prefixlm_last_error() returns a thread-local message.
 */
#ifndef MIMIR_PREFIXLM_H
#define MIMIR_PREFIXLM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MIMIR_PREFIXLM_ABI_VERSION 9

/* Element types of q/k/v/out/dout/dq/dk/dv (lse and the workspace are float32). */
enum MimirDType {
  MIMIR_DTYPE_FLOAT32 = 0,
  MIMIR_DTYPE_BFLOAT16 = 1
};

/* Status codes.  The Python binding maps them to the exception types the
 * reference raises for the same conditions. */
enum MimirStatus {
  MIMIR_OK = 0,
  MIMIR_ERR_INVALID_ARGUMENT = 1, /* ValueError  (dense.py:14,54-55; fa4.py:437,460,505) */
  MIMIR_ERR_UNSUPPORTED_DTYPE = 2,/* TypeError   (mps.py:1390-1391) */
  MIMIR_ERR_UNSUPPORTED_SHAPE = 3,/* ValueError: head_dim / size not supported by the kernels */
  MIMIR_ERR_HIP = 4               /* RuntimeError: a HIP launch or runtime call failed */
};

typedef struct MimirPrefixLMFwdParams {
  const void* q;              /* [T, Hq, D]  */
  const void* k;              /* [T, Hkv, D] */
  const void* v;              /* [T, Hkv, D] */
  void* out;                  /* [T, Hq, D], written for every row 0..T-1 */
  float* lse;                 /* [Hq, T] float32, may be NULL */
  const int32_t* prefix_lens; /* device int32 [>= numseqs]     */
  const int32_t* causal_lens; /* device int32 [>= numseqs]     (only read by mimir_prefixlm_check_metadata) */
  const int32_t* cu_seqlens;  /* device int32 [>= numseqs + 1] */
  int64_t q_stride_token, q_stride_head;
  int64_t k_stride_token, k_stride_head;
  int64_t v_stride_token, v_stride_head;
  int64_t out_stride_token, out_stride_head;
  int64_t lse_stride_head;    /* lse[h * lse_stride_head + t] */
  int32_t total_tokens;       /* T = q.shape[0] */
  int32_t num_q_heads;        /* Hq */
  int32_t num_kv_heads;       /* Hkv, Hq % Hkv == 0 */
  int32_t head_dim;           /* D */
  int32_t numseqs;
  int32_t total_seqlen;
  int32_t max_seqlen_all;     /* upper bound of cu_seqlens[s+1] - cu_seqlens[s] */
  int32_t is_causal;
  int32_t dtype;              /* enum MimirDType */
  float softmax_scale;        /* > 0; the reference uses 1/sqrt(D) */
  void* workspace;            /* device memory, >= mimir_prefixlm_fwd_workspace_bytes(); 16-byte aligned */
  size_t workspace_bytes;
  /* Optional sigmoid output gate (NULL: none).  With a gate the forward also
   * writes gated_out = sigmoid(gate) * out, rounded as the reference's
   * torch.sigmoid(gate) * attn_output in the element type
   * (src/mimir/model/layers.py:239): s = round(sigmoid(gate)), then
   * round(s * round(attention)).  out keeps the ungated attention output, which
   * the backward needs. */
  const void* gate;           /* [T, Hq, D] */
  int64_t gate_stride_token, gate_stride_head;
  void* gated_out;            /* [T, Hq, D]; required with a gate */
  int64_t gated_out_stride_token, gated_out_stride_head;
  /* Optional low half of the output (NULL: not written; bf16 only): out_lo =
   * round(O - round(O)) with O the float32 attention output, so out + out_lo
   * carries ~16 significant bits.  The backward's delta = rowsum(dout * O) reads
   * it (MimirPrefixLMBwdParams.out_lo); with bf16 O alone that row sum carries
   * the output's rounding into every dS of the row.  No reference counterpart. */
  void* out_lo;               /* [T, Hq, D] */
  int64_t out_lo_stride_token, out_lo_stride_head;
  int32_t split_mode;         /* enum MimirSplitMode (bf16; P in O = P V) */
  /* Optional (NULL: none): the forward writes its split decision (0 / 1) here,
   * and then writes out_lo only when it splits.  Passed to the backward
   * (MimirPrefixLMBwdParams.split_flag), the backward follows the same decision
   * without scanning K again and reads out_lo only when it is set. */
  int32_t* split_flag;        /* device int32 [1] */
  /* Optional rotary position embedding of q inside the kernel (bf16 only;
   * rope_cos NULL: none), replacing the apply_rotary_pos_emb of q before the
   * attention call (src/mimir/model/layers.py:186-189, rotate-half convention
   * layers.py:24-40): q is then the unrotated query, rotated where the kernel
   * loads it, with the roundings of mimir_prefixlm_rope; k must already be the
   * rotated key (mimir_prefixlm_rope: the kernel streams K through LDS).  With
   * q_rope non-NULL the kernel also writes the rotated q there (the rows below
   * total_seqlen of every sequence), the q operand of the backward. */
  const float* rope_cos;      /* [T, D] float32, 16-byte aligned rows */
  const float* rope_sin;      /* [T, D] float32 */
  int64_t rope_stride_token;  /* elements between rows of rope_cos / rope_sin (multiple of 4) */
  void* q_rope;               /* optional out [T, Hq, D] */
  int64_t q_rope_stride_token, q_rope_stride_head;
} MimirPrefixLMFwdParams;

/* Whether the bf16 kernels carry the softmax probabilities P and the score
 * gradients dS as two bf16 halves.  A bf16 MFMA operand keeps 8 significant
 * bits; split, the operand is hi + lo with lo = round(x - hi) and every product
 * with it takes one more MFMA (forward O = P V, backward dK = dS^T Q and
 * dQ = dS K), which removes that rounding from the result.  dQ and dK are sums
 * of cancelling terms (every row of dS sums to zero) and delta = rowsum(dout * O)
 * inherits the rounding of O, so with large key or query entries these roundings
 * dominate the gradients' error.  AUTO splits when softmax_scale * max|K| > 0.75
 * anywhere in the call: the prologue of the forward and of the backward's DELTA
 * stage scans K on the device, and the kernels read the result (no host
 * synchronisation).  No reference counterpart. */
enum MimirSplitMode {
  MIMIR_SPLIT_AUTO = 0,
  MIMIR_SPLIT_ALWAYS = 1,
  MIMIR_SPLIT_NEVER = 2
};

typedef struct MimirPrefixLMBwdParams {
  const void* q;
  const void* k;
  const void* v;
  const void* out;            /* forward output [T, Hq, D] */
  const void* dout;           /* upstream gradient [T, Hq, D] */
  const float* lse;           /* forward lse [Hq, T] */
  void* dq;                   /* [T, Hq, D]  */
  void* dk;                   /* [T, Hkv, D] */
  void* dv;                   /* [T, Hkv, D] */
  const int32_t* prefix_lens;
  const int32_t* causal_lens;
  const int32_t* cu_seqlens;
  int64_t q_stride_token, q_stride_head;
  int64_t k_stride_token, k_stride_head;
  int64_t v_stride_token, v_stride_head;
  int64_t out_stride_token, out_stride_head;
  int64_t dout_stride_token, dout_stride_head;
  int64_t dq_stride_token, dq_stride_head;
  int64_t dk_stride_token, dk_stride_head;
  int64_t dv_stride_token, dv_stride_head;
  int64_t lse_stride_head;
  int32_t total_tokens;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t numseqs;
  int32_t total_seqlen;
  int32_t max_seqlen_all;
  int32_t is_causal;
  int32_t dtype;
  float softmax_scale;
  void* workspace;            /* device memory, >= mimir_prefixlm_bwd_workspace_size(params) */
  size_t workspace_bytes;
  /* Optional sigmoid output gate (NULL: none), the backward of
   * gated_out = sigmoid(gate) * out.  With a gate, `dout` is the gradient of
   * gated_out and `out` the ungated attention output; the DELTA stage forms the
   * attention's upstream gradient round(dout * s) in the workspace, delta from
   * it, and dgate = round(round(dout * out) * (1 - s) * s) with s =
   * round(sigmoid(gate)), in the order torch's autograd evaluates the reference
   * expression (layers.py:239; sigmoid_backward = grad * (1 - y) * y). */
  const void* gate;           /* [T, Hq, D] */
  int64_t gate_stride_token, gate_stride_head;
  void* dgate;                /* [T, Hq, D]; required with a gate */
  int64_t dgate_stride_token, dgate_stride_head;
  /* Score-gradient hand-off (bf16, head_dim 128; no reference counterpart): when
   * the bf16 dS tiles of every (q head, 32-query block, 32-key block) fit in
   * this many bytes of workspace (mimir_prefixlm_bwd_dscore_bytes), the DKDV
   * stage writes them there and the DQ stage computes dQ = dS K from them
   * instead of recomputing S and dP; DQ then reads what DKDV wrote and runs
   * after it.  0: DQ recomputes.  The stored tiles carry no low half, so when
   * dS is split (split_mode) the recomputing dQ kernel runs instead: for ALWAYS
   * the hand-off is off, for AUTO both dQ kernels are enqueued and the one the
   * device-side decision selects does the work (the other exits at once).  The
   * recompute also takes over when a stored tile would fall outside the region
   * (a sequence longer than max_seqlen_all). */
  size_t dscore_limit_bytes;
  /* Low half of the forward output (NULL: delta from out alone; with split_flag
   * read only when the flag is set); see MimirPrefixLMFwdParams.out_lo. */
  const void* out_lo;         /* [T, Hq, D] */
  int64_t out_lo_stride_token, out_lo_stride_head;
  int32_t split_mode;         /* enum MimirSplitMode (bf16; dS in dK = dS^T Q and dQ = dS K) */
  const int32_t* split_flag;  /* the forward's recorded decision (device int32 [1]) or NULL */
  /* Optional gradient of a rotary position embedding inside the kernels (bf16
   * only; rope_cos NULL: none): q and k are the rotated operands the forward
   * used, and dq / dk receive the gradients of the unrotated q / k -- the bf16
   * gradient of the rotated operand mapped back in the kernels' stores exactly
   * as mimir_prefixlm_rope with inverse = 1 maps it (what autograd does for
   * layers.py:186-189).  Same tables as MimirPrefixLMFwdParams.rope_cos. */
  const float* rope_cos;
  const float* rope_sin;
  int64_t rope_stride_token;
  /* Key-range parts of the DQ stage (bf16; no reference counterpart): non-zero
   * lets mimir_prefixlm_bwd_workspace_size include, where the grid can be small
   * (ceil(total_tokens / 128) * num_q_heads < 512), a copy of the dQ tile list
   * with room for parts, arrival counters and 1024 / num_q_heads partial slots
   * of (4 * head_dim * 128 + 2048) bytes per q head; with a workspace that
   * large the dQ kernels cut the key ranges of their heaviest query tiles into
   * up to 16 parts run as separate workgroups, and the last part of a tile to
   * arrive sums the parts in part order (deterministic) and stores dQ.  0: no
   * parts. */
  int32_t dq_key_chunks;
} MimirPrefixLMBwdParams;

/* Bytes of device workspace the forward needs: the heaviest-first tile work list
 * (16-byte entries, one per 128-row query tile of every sequence; sized
 * ceil(T / 128) + numseqs, which bounds the tiles of any packing of T tokens into
 * numseqs sequences, so it does not rely on max_seqlen_all), then, 256-byte
 * aligned, the 512 int32 slots of the K scan behind split_mode AUTO. */
size_t mimir_prefixlm_fwd_workspace_bytes(int32_t total_tokens, int32_t numseqs, int32_t max_seqlen_all);

/* Bytes of device workspace with which the bf16 forward may also cut the key
 * ranges of its heaviest query tiles into parts (at most 16 per tile), run
 * them as separate workgroups and merge their partial outputs in part order
 * (deterministic): on a small grid -- fewer than 512 (query tile, q head)
 * workgroups -- the heaviest tiles otherwise run alone on a few compute units
 * at the end.  No counterpart in the reference (an extension of the forward's
 * own scheduling).  It adds 1024 / num_q_heads chunk slots of
 * (4 * head_dim * 128 + 2048) bytes per q head and their arrival counters; it
 * equals mimir_prefixlm_fwd_workspace_bytes where the grid cannot be small
 * (ceil(min(total_tokens, total_seqlen) / 128) * num_q_heads >= 512: the
 * least number of query tiles when cu_seqlens[0] = 0, as the reference's
 * metadata has it; with leading padding rows the grid can be smaller and then
 * runs uncut) and for float32.  The forward cuts key ranges iff its
 * workspace_bytes reaches this size; any size from
 * mimir_prefixlm_fwd_workspace_bytes up is valid.  Reads only dtype,
 * total_tokens, total_seqlen, num_q_heads, head_dim, numseqs and
 * max_seqlen_all. */
size_t mimir_prefixlm_fwd_workspace_size(const MimirPrefixLMFwdParams* params);

/* Forward: out (and lse if non-NULL).
 * Replaces the FA4 two-pass forward, src/mimir/model/flash_attention_prefixlm_fa4.py:353-406
 * (+ _fa4_varlen, fa4.py:17-50), the FA3 forward custom op
 * src/mimir/model/flash_attention_prefixlm_v2.py:101-144, and the masked-SDPA loop
 * src/mimir/model/flash_attention_prefixlm_dense.py:19-81. */
int mimir_prefixlm_fwd(const MimirPrefixLMFwdParams* params, void* stream);

/* The forward for callers that cannot allocate device memory (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc).  No
 * counterpart in the reference.  It ignores params->workspace and keeps its
 * work list and K-scan slots in a fixed device array of 128 KiB inside the
 * library (one per GPU, held until the process ends): a call whose
 * mimir_prefixlm_fwd_workspace_bytes exceeds 128 KiB fails with
 * MIMIR_ERR_UNSUPPORTED_SHAPE before any device work (it fits while
 * ceil(total_tokens / 128) + numseqs <= 8064); it never cuts key ranges.  It calls no hipMalloc / hipFree.  Every call on one GPU
 * shares that array, so calls that overlap on one GPU (two streams or threads)
 * race; the array needs no clearing between calls.  The array's device address
 * is looked up once per device (the first call there) and kept: do not call it
 * after a hipDeviceReset (or another re-creation of the device's primary
 * context) in the same process.  Outputs as mimir_prefixlm_fwd. */
int mimir_prefixlm_fwd_noalloc(const MimirPrefixLMFwdParams* params, void* stream);

/* Backward: dq, dk, dv from dout, out and lse.  Deterministic: every gradient
 * element is summed in a fixed order by one owner (atomics only count work-queue
 * units and split-tile arrivals).
 * Replaces the FA3 backward custom op src/mimir/model/flash_attention_prefixlm_v2.py:165-227,
 * FA4's backward reached through fa4.py:153-179,309-331, and the Metal split
 * backward src/mimir/model/flash_attention_prefixlm_mps.py:1456-1561. */
int mimir_prefixlm_bwd(const MimirPrefixLMBwdParams* params, void* stream);

/* Backward stages, for callers that schedule them themselves (e.g. dK/dV and
 * dQ on two streams once delta is done).  mimir_prefixlm_bwd runs them all, in
 * order.  DELTA must complete before DKDV and DQ; DKDV, DQ and FILL are
 * independent of each other, except that with the score-gradient hand-off
 * (mimir_prefixlm_bwd_dscore_bytes non-zero) DQ reads what DKDV wrote.  No reference counterpart: the reference exposes
 * the backward only through autograd (flash_attention_prefixlm_v2.py:270-283). */
enum MimirBwdStage {
  MIMIR_BWD_STAGE_DELTA = 1, /* delta = rowsum(O * dO), lse * log2(e) and the tile work lists into the workspace */
  MIMIR_BWD_STAGE_DKDV = 2,  /* dK, dV for every key row inside a sequence */
  MIMIR_BWD_STAGE_DQ = 4,    /* dQ for every active query row */
  MIMIR_BWD_STAGE_FILL = 8,  /* zero dQ / dK / dV rows outside every sequence */
  MIMIR_BWD_STAGE_ALL = 15
};
int mimir_prefixlm_bwd_stages(const MimirPrefixLMBwdParams* params, int stages, void* stream);

/* Bytes of device workspace the backward needs: float32 delta = rowsum(O * dO) [Hq, T],
 * float32 lse * log2(e) [Hq, T], the tile work lists of the DQ and DKDV stages,
 * and for head_dim 128 the counters and float32 partial-sum slots of key tiles
 * that the DKDV stage splits in two (at most 384 (tile, kv head) splits, 256 KiB
 * each).  The DELTA stage writes the lists and zeroes the counters; DQ and DKDV
 * read them, and DKDV leaves the counters at zero. */
size_t mimir_prefixlm_bwd_workspace_bytes(int32_t total_tokens, int32_t num_q_heads, int32_t numseqs,
                                          int32_t max_seqlen_all);

/* Bytes of backward workspace for these parameters: mimir_prefixlm_bwd_workspace_bytes
 * plus, with a gate, the attention's upstream gradient [T, Hq, D] in the element type,
 * plus the score-gradient tiles when mimir_prefixlm_bwd_dscore_bytes(params) is non-zero,
 * plus the DQ stage's key-range parts when dq_key_chunks asks for them and the grid can
 * be small (the test of mimir_prefixlm_fwd_workspace_size).  Only the size fields
 * (total_tokens, total_seqlen, num_q_heads, numseqs, max_seqlen_all), head_dim,
 * dtype, gate, dscore_limit_bytes and dq_key_chunks are read. */
size_t mimir_prefixlm_bwd_workspace_size(const MimirPrefixLMBwdParams* params);

/* Bytes of workspace the score-gradient hand-off takes for these parameters, 0
 * when it is off: bf16 with head_dim 128 only, and only when the bf16 tiles,
 * Hq x (floor(T / 32) + numseqs + 1) x ceil(max_seqlen_all / 32) blocks of
 * 32 x 32, fit in dscore_limit_bytes.  No reference counterpart. */
size_t mimir_prefixlm_bwd_dscore_bytes(const MimirPrefixLMBwdParams* params);

/* Rotary position embedding on [T, H, D] rows, rotate-half convention
 * (reference: src/mimir/model/layers.py:24-40, apply_rotary_pos_emb on the q / k
 * splits of the fused projection, layers.py:183-189), cos / sin float32 [T, D]:
 *
 *   inverse == 0:  y = round(x * cos + rotate_half(x) * sin)   (fp32 math, one rounding)
 *   inverse != 0:  the gradient of that map, x_grad from y_grad, rounded as torch's
 *                  autograd does for the reference expression: each of the two
 *                  contributions (y_grad * cos and the rotate_half part of
 *                  y_grad * sin) is rounded to the element type, then their sum.
 *
 * rotate_half(x) = cat(-x[D/2:], x[:D/2]).  y may alias x (same pointer and
 * strides): every element pair is read before it is written.  bf16 needs
 * D % 16 == 0, float32 D % 8 == 0; rows 16-byte aligned. */
typedef struct MimirRopeParams {
  const void* x;              /* [T, H, D] */
  void* y;                    /* [T, H, D] */
  const float* cos;           /* [T, D] float32 */
  const float* sin;           /* [T, D] float32 */
  int64_t x_stride_token, x_stride_head;
  int64_t y_stride_token, y_stride_head;
  int64_t cs_stride_token;    /* cos / sin row stride (elements) */
  int32_t total_tokens;       /* T */
  int32_t num_heads;          /* H */
  int32_t head_dim;           /* D */
  int32_t dtype;              /* enum MimirDType */
  int32_t inverse;
} MimirRopeParams;
int mimir_prefixlm_rope(const MimirRopeParams* params, void* stream);

/* Attention against a static KV cache, the inference path of Mimir2's
 * Attention (reference: src/mimir/model/layers.py:134-167, _attention_with_cache,
 * with the Cache of layers.py:107-115).  For batch row b (cache row
 * r = batch_indices ? batch_indices[b] : b) and c = cache_lengths[b]:
 *
 *   1. k_new / v_new [b, i] are written to cache_k / cache_v [r, c + i], i < S;
 *   2. query i of q [b, i, h] attends the cache keys j < c + S of kv head
 *      h / (Hq / Hkv), and if `causal` only j <= c + i (the reference's mask);
 *      softmax scale `softmax_scale`, out [b, i, h] in the element type.
 *
 * c + S must not exceed cache_len (the reference raises IndexError there; this
 * entry point skips the cache writes and keys beyond the cache instead), and a
 * batch row whose cache row lies outside [0, cache_rows) gets a zero output and
 * no cache write (the reference raises IndexError).
 * max_kv_len is an upper bound of max_b(c + S) (the reference's
 * kv_len.max().item(), layers.py:143) that sizes the key split; the split itself
 * follows the batch rows' own lengths.  bf16 only, head_dim 64 or 128.
 * The workspace holds the partial results of the split (no counters and no memset:
 * the call can be captured in a graph). */
typedef struct MimirCacheAttnParams {
  const void* q;              /* [B, S, Hq, D] */
  const void* k_new;          /* [B, S, Hkv, D] */
  const void* v_new;          /* [B, S, Hkv, D] */
  void* cache_k;              /* [>= rows, cache_len, Hkv, D] */
  void* cache_v;              /* [>= rows, cache_len, Hkv, D] */
  void* out;                  /* [B, S, Hq, D] */
  const void* cache_lengths;   /* device int32 or int64 [B] (index_int64) */
  const void* batch_indices;   /* device int32 or int64 [B], or NULL (row b) */
  int64_t q_stride_batch, q_stride_token, q_stride_head;
  int64_t kn_stride_batch, kn_stride_token, kn_stride_head;
  int64_t vn_stride_batch, vn_stride_token, vn_stride_head;
  int64_t ck_stride_batch, ck_stride_token, ck_stride_head;
  int64_t cv_stride_batch, cv_stride_token, cv_stride_head;
  int64_t out_stride_batch, out_stride_token, out_stride_head;
  int32_t batch;              /* B */
  int32_t seqlen;             /* S (1 for decode) */
  int32_t cache_len;          /* positions per cache row */
  int32_t cache_rows;         /* rows of cache_k / cache_v; rows outside [0, cache_rows) are skipped */
  int32_t max_kv_len;         /* upper bound of max_b(cache_lengths[b] + S) */
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t causal;
  int32_t dtype;              /* MIMIR_DTYPE_BFLOAT16 */
  float softmax_scale;
  void* workspace;            /* >= mimir_prefixlm_cache_attn_workspace_bytes(params) */
  size_t workspace_bytes;
  int32_t index_int64;        /* 1: cache_lengths / batch_indices are int64, 0: int32 */
} MimirCacheAttnParams;
size_t mimir_prefixlm_cache_attn_workspace_bytes(const MimirCacheAttnParams* params);
int mimir_prefixlm_cache_attn(const MimirCacheAttnParams* params, void* stream);

/* Rotary positions from token positions and a frequency table: of each head of
 * q [B, S, Hq, D] and (num_kv_heads > 0) k [B, S, Hkv, D], the pairs of the first
 * rotary_dim columns are turned by the token's position times the pair's frequency,
 *
 *     a' = amplitude (a cos t - b sin t),  b' = amplitude (b cos t + a sin t),
 *     t = 2 pi frac(positions[b, i] * turns[pair] / 2^64),
 *
 * in fp32 with one rounding; the other columns are copied.  Pair i is columns
 * (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with `interleaved`.  inverse = 1 turns
 * the other way (t -> -t): the gradient's map.  head_dim and rotary_dim even; each
 * output may be its input (same pointer and strides), else the outputs share no memory
 * with an input, each other or themselves (in place: the columns that are turned);
 * MIMIR_ERR_UNSUPPORTED_SHAPE if they do.  Strides in elements. */
typedef struct MimirRotaryParams {
  const void* q;
  const void* k;              /* NULL if num_kv_heads is 0 */
  void* q_out;
  void* k_out;
  const int64_t* turns;       /* [rotary_dim / 2]: turn per position, in units of 2^-64 */
  const void* positions;      /* device int32 or int64 (index_int64), by its strides [B, S] */
  int64_t q_stride_batch, q_stride_token, q_stride_head;
  int64_t k_stride_batch, k_stride_token, k_stride_head;
  int64_t q_out_stride_batch, q_out_stride_token, q_out_stride_head;
  int64_t k_out_stride_batch, k_out_stride_token, k_out_stride_head;
  int64_t positions_stride_batch, positions_stride_token;
  int32_t batch;              /* B */
  int32_t seqlen;             /* S */
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;           /* D */
  int32_t rotary_dim;
  int32_t interleaved;
  int32_t dtype;              /* enum MimirDType */
  int32_t inverse;
  int32_t index_int64;
  float amplitude;
} MimirRotaryParams;
int mimir_prefixlm_rotary(const MimirRotaryParams* params, void* stream);

/* Heads normed, scaled by a learned weight and turned by their position, in one pass:
 * for each head's row x of q [B, S, Hq, D] and (num_kv_heads > 0) k [B, S, Hkv, D],
 *
 *     y = R (r w x),  r = 1 / sqrt(mean(x^2) + eps),  w = q_weight or k_weight [D],
 *
 * R the turn of mimir_prefixlm_rotary (amplitude, pair layout and rotary_dim as there), in
 * fp32 with one rounding.  A weight may be NULL: ones.  weight_dtype: that of the heads, or
 * float32.  The outputs share no memory with an input, each other or themselves.
 *
 * mimir_prefixlm_norm_rotary_bwd: from dq / dk, the gradients of the outputs, those of q and
 * k in q_out / k_out and (not NULL) of the weights in dq_weight / dk_weight:
 *     g = R^T dy,  dw = sum over the rows of r g x,  dx = r (w g - x r^2 mean(w g x)).
 * The workspace is needed for weight gradients only and needs no clearing. */
typedef struct MimirNormRotaryParams {
  const void* q;
  const void* k;              /* NULL if num_kv_heads is 0 */
  void* q_out;
  void* k_out;
  const void* dq;             /* gradient: of q's output; else not read */
  const void* dk;
  const void* q_weight;       /* [D], or NULL */
  const void* k_weight;
  void* dq_weight;            /* gradient: [D], or NULL; else not read */
  void* dk_weight;
  const int64_t* turns;       /* [rotary_dim / 2] */
  const void* positions;      /* int32 or int64 (index_int64) [B, S] */
  int64_t q_stride_batch, q_stride_token, q_stride_head;
  int64_t k_stride_batch, k_stride_token, k_stride_head;
  int64_t q_out_stride_batch, q_out_stride_token, q_out_stride_head;
  int64_t k_out_stride_batch, k_out_stride_token, k_out_stride_head;
  int64_t dq_stride_batch, dq_stride_token, dq_stride_head;
  int64_t dk_stride_batch, dk_stride_token, dk_stride_head;
  int64_t positions_stride_batch, positions_stride_token;
  int32_t batch, seqlen, num_q_heads, num_kv_heads, head_dim, rotary_dim;
  int32_t interleaved;
  int32_t dtype;              /* MIMIR_DTYPE_FLOAT32 or MIMIR_DTYPE_BFLOAT16 */
  int32_t weight_dtype;
  int32_t index_int64;
  float amplitude, eps;
  void* workspace;            /* gradient: >= mimir_prefixlm_norm_rotary_workspace_bytes(params) */
  size_t workspace_bytes;
} MimirNormRotaryParams;
size_t mimir_prefixlm_norm_rotary_workspace_bytes(const MimirNormRotaryParams* params);
int mimir_prefixlm_norm_rotary(const MimirNormRotaryParams* params, void* stream);
int mimir_prefixlm_norm_rotary_bwd(const MimirNormRotaryParams* params, void* stream);

/* Attention over a KV cache in pages of MIMIR_PAGE_TOKENS tokens, held in 8 bits (e4m3)
 * under one power-of-two scale for each page and kv head.
 *
 *   cache_k      e4m3 [page][Hkv][64][D],  key   = code * 2^k_exponents[page][head]
 *   cache_v      e4m3 [page][Hkv][D][64],  value = code * 2^v_exponents[page][head]
 *   exponents    int8 [page][Hkv], in [-100, 120]
 *
 * with a stride between pages each (so that the layers of a model can lie side by side in
 * a page).  Token t of batch row b lies in page page_table[row][t / 64], slot t % 64, where
 * row = batch_indices ? batch_indices[b] : b.  With c = cache_lengths[b] and
 * m = new_lengths ? new_lengths[b] : S:
 *
 *   1. k_new / v_new [b, i], i < m, are appended at tokens c + i.  Every page and head they
 *      fall in takes the smallest exponent e >= -100 with |x| <= 448 * 2^e for its new
 *      (finite) values, but not less than the one it has if it holds older tokens, whose
 *      codes are rounded again where e grew.  Codes round to nearest even; infinite
 *      values become NaN (e4m3 has no infinity).  Slots behind the row's last token keep
 *      their codes.
 *   2. query i < m of q [b, i, h] attends the tokens t < c + m of kv head h / (Hq / Hkv), and
 *      if `causal` only t <= c + i; bf16 out [b, i, h].  Queries i >= m give zeros, and so do
 *      those that see no token.
 *
 * Tokens past the table (t / 64 >= table_width) and pages outside [0, num_pages) are neither
 * written nor attended; a batch row whose table row lies outside [0, table_rows), or whose
 * length is negative, gives zeros.  A page that a batch row appends to must be that row's
 * alone in the call (neither appended to nor read for another): the rows run side by side.
 * q, k_new, v_new and out are bf16 rows, 16-byte aligned, strides in elements; head_dim 64
 * or 128.  The workspace holds partial results of split key ranges (nothing to clear: the
 * call can be captured in a graph). */
#define MIMIR_PAGE_TOKENS 64
typedef struct MimirPagedAttnParams {
  const void* q;              /* [B, S, Hq, D] */
  const void* k_new;          /* [B, S, Hkv, D] */
  const void* v_new;          /* [B, S, Hkv, D] */
  void* out;                  /* [B, S, Hq, D] */
  void* cache_k;
  void* cache_v;
  int8_t* k_exponents;
  int8_t* v_exponents;
  const int32_t* page_table;  /* [table_rows, table_width] */
  const void* cache_lengths;  /* device int32 or int64 [B] (index_int64, as the next two) */
  const void* batch_indices;  /* [B], or NULL (row b) */
  const void* new_lengths;    /* [B], or NULL (S) */
  int64_t q_stride_batch, q_stride_token, q_stride_head;
  int64_t kn_stride_batch, kn_stride_token, kn_stride_head;
  int64_t vn_stride_batch, vn_stride_token, vn_stride_head;
  int64_t out_stride_batch, out_stride_token, out_stride_head;
  int64_t k_stride_page, v_stride_page;      /* bytes */
  int64_t ke_stride_page, ve_stride_page;    /* bytes */
  int64_t table_stride;       /* int32 between rows of page_table */
  int32_t batch;              /* B */
  int32_t seqlen;             /* S */
  int32_t num_pages;
  int32_t table_rows;
  int32_t table_width;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t causal;
  int32_t dtype;              /* of q, k_new, v_new and out: MIMIR_DTYPE_BFLOAT16 */
  int32_t index_int64;
  float softmax_scale;
  void* workspace;            /* >= mimir_prefixlm_paged_attn_workspace_bytes(params) */
  size_t workspace_bytes;
} MimirPagedAttnParams;
size_t mimir_prefixlm_paged_attn_workspace_bytes(const MimirPagedAttnParams* params);
int mimir_prefixlm_paged_attn(const MimirPagedAttnParams* params, void* stream);

/* The rows of a paged cache and the pages they hold.
 *
 *   pages    int32 [rows][width]: the page of each run of 64 tokens, -1 where none
 *   lengths  int32 [rows]: tokens held
 *   counts   int32 [num_pages]: table entries that name the page (0: free)
 *   missing  int32 [1]: pages asked for that the pool did not have, added up
 *
 * and the pool's four arrays, page by page (for the calls that move data): `bytes` per
 * page each, a multiple of 16 for keys and values.  Entries outside [0, num_pages) are
 * taken for none.  Pages are handed out lowest first, so results do not depend on
 * timing.  Every call works on the device alone, without a host synchronisation.
 *
 * `workspace`: mimir_prefixlm_pages_workspace_bytes(params, items) bytes. */
typedef struct MimirPagesParams {
  int32_t* pages;
  int32_t* lengths;
  int32_t* counts;
  int32_t* missing;
  int64_t pages_stride;       /* int32 between rows of pages */
  int32_t rows;
  int32_t width;
  int32_t num_pages;
  void* data[4];              /* keys, values, key exponents, value exponents: page 0 */
  int64_t data_bytes[4];      /* of a page */
  int64_t data_stride[4];     /* bytes between pages */
  void* workspace;
  size_t workspace_bytes;
} MimirPagesParams;
size_t mimir_prefixlm_pages_workspace_bytes(const MimirPagesParams* params, int32_t items);

/* Page destination[i] of the pool becomes a copy of page source[i], i < n.  Entries outside
 * the pool are skipped; no destination may be named twice or be a source.  Uses the data
 * fields and num_pages. */
int mimir_prefixlm_pages_copy(const MimirPagesParams* params, const int32_t* source, const int32_t* destination,
                              int32_t n, void* stream);

/* Row destination[i] goes on from what row source[i] held before the call: it gives back its
 * own pages, shares the full pages of the source and gets a copy of the source's last,
 * partly filled page in a free one.  Such a page that every row holding it gives back in the call
 * (its sources are themselves replaced) goes uncopied to the first row (lowest i) that goes on
 * from it, unless a row now holds it as a full one.  So a page that is copied is held after the
 * call, and never one of those handed out.
 * Entries with source = destination leave the row alone, entries outside the table are
 * skipped, and of entries with one destination the last counts.  Where the pool has no
 * free page the last page stays -1 and `missing` counts it. */
int mimir_prefixlm_pages_fork(const MimirPagesParams* params, const int32_t* source, const int32_t* destination,
                              int32_t n, void* stream);

/* Moves the pages in use (counts > 0) to the front of the pool: those at or past their
 * number, in ascending order, into the free pages before it, in ascending order; counts and
 * pages follow.  used[0] (device) = their number. */
int mimir_prefixlm_pages_compact(const MimirPagesParams* params, int32_t* used, void* stream);

/* The listed rows (row_list int32 [n]; those outside the table are skipped, one may come
 * twice) give back their pages and hold no tokens. */
int mimir_prefixlm_pages_release(const MimirPagesParams* params, const int32_t* row_list, int32_t n, void* stream);

/* Gives every row r with new_lengths[r] > 0 (int32 [rows]) the pages it lacks for
 * lengths[r] + new_lengths[r] tokens, by row, then place; lengths stay. */
int mimir_prefixlm_pages_reserve(const MimirPagesParams* params, const int32_t* new_lengths, void* stream);

/* Device-side metadata check: writes to bad[0] (device int32 [2]) the first s in
 * [0, numseqs) whose lengths are invalid, or -1 if none, and to bad[1] why:
 *   1  prefix_lens[s] + causal_lens[s] != cu_seqlens[s+1] - cu_seqlens[s], or a
 *      negative length (the reference raises ValueError for this,
 *      src/mimir/model/flash_attention_prefixlm_dense.py:54-55);
 *   2  cu_seqlens[s+1] - cu_seqlens[s] > max_seqlen_all (the scalar sizes the
 *      score-gradient region and the per-sequence span check).
 * Asynchronous. */
int mimir_prefixlm_check_metadata(const int32_t* prefix_lens, const int32_t* causal_lens,
                                  const int32_t* cu_seqlens, int32_t numseqs, int32_t max_seqlen_all,
                                  int32_t* bad, void* stream);

/* Thread-local description of the last failure on this thread ("" if none). */
const char* mimir_prefixlm_last_error(void);

/* Cross attention over packed sequences: the queries of sequence s, rows cu_seqlens_q[s] up to
 * cu_seqlens_q[s + 1] of q, attend all of its states, rows cu_seqlens_k[s] up to cu_seqlens_k[s + 1] of k / v:
 * out = softmax(softmax_scale q k^T) v.  Both lists hold numseqs + 1 device int32, not decreasing and within the rows
 * there are (others address nothing outside, but what is then written is not defined).  A
 * sequence without states gives O = 0, and rows before the first or behind the last sequence O = 0 and
 * zero gradients.  What the backward needs of the forward besides out (both may be NULL in a forward alone):
 * lse2, float32 [Hq, total_q], the base-2 logarithm of the softmax's sum, scale included, -inf without
 * states, and out_lo, bf16 [total_q, Hq, D] contiguous, round(O - out), the low half of O.  bf16,
 * head_dim 64 or 128, 16-byte aligned rows.  The workspaces need no clearing. */
typedef struct MimirCrossParams {
  const void* q;              /* [total_q, Hq, D] */
  const void* k;              /* [total_k, Hkv, D] */
  const void* v;
  void* out;                  /* [total_q, Hq, D]: written by the forward, read by the backward */
  void* out_lo;
  float* lse2;
  const int32_t* cu_seqlens_q;
  const int32_t* cu_seqlens_k;
  const void* dout;           /* backward */
  void* dq;
  void* dk;
  void* dv;
  int64_t q_stride_token, q_stride_head;
  int64_t k_stride_token, k_stride_head;
  int64_t v_stride_token, v_stride_head;
  int64_t out_stride_token, out_stride_head;
  int64_t dout_stride_token, dout_stride_head;
  int64_t dq_stride_token, dq_stride_head;
  int64_t dk_stride_token, dk_stride_head;
  int64_t dv_stride_token, dv_stride_head;
  int32_t total_q, total_k, numseqs, num_q_heads, num_kv_heads, head_dim;
  int32_t dtype;              /* MIMIR_DTYPE_BFLOAT16 */
  float softmax_scale;        /* positive */
  void* workspace;            /* >= mimir_prefixlm_cross_workspace_bytes(params, backward), 256-byte aligned */
  size_t workspace_bytes;
} MimirCrossParams;
size_t mimir_prefixlm_cross_workspace_bytes(const MimirCrossParams* params, int32_t backward);
int mimir_prefixlm_cross_fwd(const MimirCrossParams* params, void* stream);
int mimir_prefixlm_cross_bwd(const MimirCrossParams* params, void* stream);

/* Cross attention to rows of a static cache of states: request s is the seq_tokens query rows from
 * s * seq_tokens on (all tokens of all its beams), over the first lengths[r] (clamped to [0, cache_len]) positions
 * of cache row r = rows[s] (rows NULL: s).  A row outside [0, cache_rows) has no states; without
 * states the output is 0.  bf16, head_dim 64 or 128; the workspace needs no clearing. */
typedef struct MimirStatesParams {
  const void* q;              /* [requests * seq_tokens, Hq, D] */
  const void* keys;           /* [cache_rows, cache_len, Hkv, D] */
  const void* values;
  void* out;                  /* [requests * seq_tokens, Hq, D] */
  const void* lengths;        /* device int32 or int64 (lengths_int64) [cache_rows] */
  const void* rows;           /* device int32 or int64 (rows_int64) [requests], or NULL */
  int64_t q_stride_token, q_stride_head;
  int64_t k_stride_row, k_stride_token, k_stride_head;
  int64_t v_stride_row, v_stride_token, v_stride_head;
  int64_t out_stride_token, out_stride_head;
  int32_t requests, seq_tokens, cache_rows, cache_len, num_q_heads, num_kv_heads, head_dim;
  int32_t dtype;              /* MIMIR_DTYPE_BFLOAT16 */
  int32_t lengths_int64, rows_int64;
  float softmax_scale;        /* positive */
  void* workspace;            /* >= mimir_prefixlm_states_workspace_bytes(params), 256-byte aligned */
  size_t workspace_bytes;
} MimirStatesParams;
size_t mimir_prefixlm_states_workspace_bytes(const MimirStatesParams* params);
int mimir_prefixlm_states_attn(const MimirStatesParams* params, void* stream);

/* Beam search: of each request's W beams over a vocabulary of V tokens, the `count` best
 * continuations by scores[r, w] + log_softmax(logits[r, w])[token], ties to the lowest beam,
 * then token.  Sums of exponentials are fp32 (a beam's scores are all off by the same, less than 2^-19: beams
 * whose scores lie closer than twice that may change places), scores are formed and compared in 64 bits, out_scores rounded once.
 *
 * A beam with finished[r, w] != 0 goes on with end_token alone, at its score, and its logits are not
 * read.  A beam whose score is not finite, or whose logits hold NaN or +inf or nothing above -inf, has
 * no continuation; nor has a token with logit -inf.  Where a request has fewer than
 * `count` of them, the rest are the lowest (beam, token) among the others, with score -inf.
 *
 * out_rows[r, i] is the beam's row r * W + w, out_finished[r, i] (if not NULL) whether that beam was
 * finished or the token is end_token (end_token < 0: none).  W <= 32, 1 <= count <= min(64, W * V),
 * V < 2^30.  The workspace needs no clearing. */
typedef struct MimirBeamSelectParams {
  const void* logits;         /* [R, W, V], unit stride on V */
  const float* scores;        /* [R, W] */
  const uint8_t* finished;    /* [R, W], or NULL */
  float* out_scores;          /* [R, count] */
  int32_t* out_tokens;
  int32_t* out_rows;
  uint8_t* out_finished;      /* [R, count], or NULL */
  int64_t logits_stride_request, logits_stride_beam;  /* elements */
  int64_t scores_stride_request, scores_stride_beam;
  int64_t finished_stride_request, finished_stride_beam;
  int32_t requests, beams, vocab, count;
  int32_t end_token;
  int32_t dtype;              /* of the logits: MIMIR_DTYPE_FLOAT32 or MIMIR_DTYPE_BFLOAT16 */
  void* workspace;            /* >= mimir_prefixlm_beam_select_workspace_bytes(params), 16-byte aligned */
  size_t workspace_bytes;
} MimirBeamSelectParams;
size_t mimir_prefixlm_beam_select_workspace_bytes(const MimirBeamSelectParams* params);
int mimir_prefixlm_beam_select(const MimirBeamSelectParams* params, void* stream);

/* Reordering of cache rows: row i of each of `count` tensors takes the first
 * lengths[source[i]] positions of row source[i] as they were before the call, and then (if
 * update_lengths) lengths[i] that of its source.  Rows form groups of `group` (at most 32) neighbours;
 * a row whose source lies outside its group stays as it is.  Positions past the length
 * stay as they are.  A position holds position_bytes (a multiple of 16), side by side in a row; rows lie
 * stride bytes apart (a multiple of 16, no less than max_length positions, unless there is one row). */
#define MIMIR_REORDER_TENSORS 16
typedef struct MimirReorderParams {
  void* data[MIMIR_REORDER_TENSORS];
  int64_t stride[MIMIR_REORDER_TENSORS];
  void* lengths;              /* int32 or int64 (index_int64) [rows] */
  const void* source;         /* int32 or int64 (source_int64) [rows] */
  int64_t position_bytes;
  int32_t count, rows, group, max_length;
  int32_t index_int64, source_int64, update_lengths;
} MimirReorderParams;
int mimir_prefixlm_reorder_rows(const MimirReorderParams* params, void* stream);

/* MIMIR_PREFIXLM_ABI_VERSION of the loaded library. */
int mimir_prefixlm_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* MIMIR_PREFIXLM_H */
