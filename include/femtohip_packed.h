/*
 * femtohip_packed.h -- C ABI of the MI355X (gfx950) kernels of a training step over
 * packed documents and of its answers: attention under a mask, attention over a
 * cache, the embedding with a factor, the norm of all gradients and their clipping.
 * Same library and conventions as femtohip.h (device pointers owned by the caller,
 * workspaces passed in, asynchronous on `stream`, int status with fh_last_error(),
 * thread-safe: no state of its own); versioned by itself.  Outputs and workspaces
 * overlap no operand of their call unless its comment allows it.
 */
#ifndef FEMTOHIP_PACKED_H_
#define FEMTOHIP_PACKED_H_

#include "femtohip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FH_PACKED_ABI_VERSION 1

/* FH_PACKED_ABI_VERSION of the build. */
int fh_packed_abi_version(void);

/* ------------------------------------------------- what a token sees
 * Tokens are rows 0 .. tokens-1 and documents ranges of them: document d is rows
 * [starts[d], starts[d] + lengths[d]), starts ascending; one that runs into the next
 * or past the last row ends there.  starts null: document d is the d-th range of
 * seq_len rows (tokens a multiple, n_documents of them), of its first lengths[d] rows.
 * lengths null: each ends where the next begins.  n_documents may be 0.  A token sees tokens of its own
 * document:
 *   causal != 0     those up to itself, and with `prefix` also the document's first
 *                   prefix[d];
 *   causal == 0     all of them (prefix null);
 *   window > 0      of those the ones less than `window` away (prefix null).
 * A token of no document sees nothing, and nothing sees it.
 * starts, lengths, prefix: int64 on the device.  table: fh_attn_mask_size bytes,
 * 16-byte aligned, written here and read by the calls below: what each token sees
 * and is seen by, as ranges of rows, and their bounds over 32 rows.  Values of any
 * kind in starts, lengths and prefix give ranges within the rows.
 */
size_t fh_attn_mask_size(int64_t tokens);
int fh_attn_mask(const int64_t* starts, const int64_t* lengths, const int64_t* prefix,
                 int64_t n_documents, int64_t tokens, int64_t seq_len, int64_t window, int causal,
                 void* table, hipStream_t stream);

/* ------------------------------------------------- attention under a mask
 * For each query head h, which reads kv head h / (n_heads / n_kv_heads):
 *   s_ij = scale q_i . k_j                  (0 < scale <= 2^60)
 *   z_ij = cap tanh(s_ij / cap)             (z = s for cap 0; scale / cap <= 2^60; bf16: cap
 *                                            <= 4096, whose tanh is off by 2^-23; fp32: cap <=
 *                                            2^126 and scale / cap >= 2^-126)
 *          - slopes[h] |i - j|              (without slopes: none)
 *   o_i  = sum_j softmax_j(z_ij) v_j        over the j that i sees; 0 where it sees none
 * Token-major: head h of q, o at columns h * head_dim of its row, row strides in
 * elements (multiples of 8, < 2^24); 16-byte aligned.  head_dim 32, 64 or 128.  What
 * the backward reads (nullable): lse, fp32 [n_heads, tokens], and for bf16 o_low, int8
 * [tokens, n_heads * head_dim], 16-byte aligned: the fp32 bits of o before its rounding
 * are (bits of o << 16) + (o_low << 8), to 2^-17 (the gradients of q and k take
 * rowsum(dout o) off terms of its size, and o's rounding would be the largest error in
 * them).  slopes: fp32 [n_heads] on the device.  What a token does not see does not reach it: infinities and NaN
 * there neither.  bf16: products on bf16 operands with fp32 sums, the softmax weights
 * rounded to bf16 before their product with v, o rounded once.
 */
int fh_masked_attn_fwd(fh_dtype dt, const void* q, int64_t ldq, const void* k, int64_t ldk,
                       const void* v, int64_t ldv, void* o, int64_t ldo, float* lse,
                       int8_t* o_low, const void* table, int64_t tokens, int64_t n_heads, int64_t n_kv_heads,
                       int64_t head_dim, float scale, float cap, const float* slopes,
                       hipStream_t stream);

/* Gradients of fh_masked_attn_fwd for dout, with its o, lse and (bf16; null in fp32)
 * o_low: dq, dk, dv (0 for what sees, or is seen by, nothing).  workspace: fh_masked_attn_bwd_workspace_size bytes,
 * 16-byte aligned. */
size_t fh_masked_attn_bwd_workspace_size(fh_dtype dt, int64_t tokens, int64_t n_heads,
                                         int64_t n_kv_heads, int64_t head_dim);
int fh_masked_attn_bwd(fh_dtype dt, const void* q, int64_t ldq, const void* k, int64_t ldk,
                       const void* v, int64_t ldv, const void* o, int64_t ldo, const void* dout,
                       int64_t lddo, const float* lse, const int8_t* o_low, void* dq, int64_t lddq, void* dk,
                       int64_t lddk, void* dv, int64_t lddv, const void* table, void* workspace,
                       int64_t tokens, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                       float scale, float cap, const float* slopes, hipStream_t stream);

/* ------------------------------------------------- attention over a cache
 * The scores of fh_masked_attn_fwd for the n_new latest tokens of each sequence over a
 * cache of its keys and values: token u of sequence b stands at place
 * lengths[b] - n_new + u and sees the places up to its own, with window > 0 the last
 * `window` of them; one before place 0 sees nothing and gets 0.  lengths: int64 [batch]
 * on the device, the new tokens included, taken within 0 and room.
 * q, o: [batch * n_new] rows of strides ldq, ldo, heads as in fh_masked_attn_fwd.  k, v:
 * place t of kv head h of sequence b at b * batch_stride + t * row_stride + h *
 * head_stride (elements; row strides multiples of 8 and < 2^24, the others multiples of
 * 8), t < room.  No place from lengths[b] on is read.  workspace:
 * fh_cache_attn_workspace_size bytes, 16-byte aligned. */
size_t fh_cache_attn_workspace_size(fh_dtype dt, int64_t batch, int64_t n_new, int64_t room,
                                    int64_t n_heads, int64_t n_kv_heads, int64_t head_dim);
int fh_cache_attn(fh_dtype dt, const void* q, int64_t ldq, const void* k, int64_t k_batch_stride,
                  int64_t k_row_stride, int64_t k_head_stride, const void* v,
                  int64_t v_batch_stride, int64_t v_row_stride, int64_t v_head_stride, void* o,
                  int64_t ldo, const int64_t* lengths, int64_t batch, int64_t n_new, int64_t room,
                  int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t window,
                  float scale, float cap, const float* slopes, void* workspace,
                  hipStream_t stream);

/* ------------------------------------------------- embedding with a factor
 * fh_embedding_fwd and fh_embedding_bwd of factor * weight: rows to_dtype(factor *
 * weight[id]), rounded once, and dweight factor times the sums.  factor finite. */
int fh_embedding_scaled_fwd(fh_dtype dt, const void* weight, const int64_t* ids, void* out,
                            int64_t n_tokens, int64_t vocab, int64_t hidden, float factor,
                            hipStream_t stream);
int fh_embedding_scaled_bwd(fh_dtype dt, const void* dy, const int64_t* ids, void* dweight,
                            int64_t n_tokens, int64_t vocab, int64_t hidden, int64_t padding_idx,
                            float factor, void* workspace, hipStream_t stream);

/* ------------------------------------------------- gradient norm and clipping
 * norm = sqrt(sum of the squares of all gradients), and out_i = to_dtype(c g_i) with
 * c = min(1, max_norm / (norm + 1e-6)), as torch.nn.utils.clip_grad_norm_ has it (a norm
 * that is not a number makes them so; an infinite one makes them 0 where they are
 * finite).  The squares are summed in fp64, in a fixed order.  grads: a host array, read
 * during the call; out may be the gradient itself, and overlaps nothing else; out null
 * for all: the norm alone.  norm: fp32 on the device.  workspace:
 * fh_clip_grads_workspace_size bytes, 16-byte aligned. */
typedef struct fh_grad {
  const void* grad;
  void* out;
  int64_t numel;
  int32_t grad_dtype, out_dtype; /* fh_dtype */
} fh_grad;

size_t fh_clip_grads_workspace_size(int64_t count);
int fh_clip_grads(int64_t count, const fh_grad* grads, float max_norm, float* norm, void* workspace,
                  hipStream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* FEMTOHIP_PACKED_H_ */
