/*
 * femtohip_blocks.h -- C ABI of the MI355X (gfx950) kernels around a
 * checkpointed block: activations kept in 8 bits, the norms after and before a
 * block, and rotary positions.  Same library and conventions as femtohip.h
 * (device pointers owned by the caller, workspaces passed in, asynchronous on
 * `stream`, int status with fh_last_error(), thread-safe: no state of its own);
 * versioned by itself.  Outputs and workspaces overlap no operand of their call
 * unless its comment allows it.
 */
#ifndef FEMTOHIP_BLOCKS_H_
#define FEMTOHIP_BLOCKS_H_

#include "femtohip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FH_BLOCKS_ABI_VERSION 1

/* FH_BLOCKS_ABI_VERSION of the build. */
int fh_blocks_abi_version(void);

/* ------------------------------------------------- activations in 8 bits
 * What a checkpoint keeps of a block (its input; the reference keeps it in the
 * model's dtype, torch/utils/checkpoint.py:794-831 under
 * femtotron/training/activation_ckpt.py:78-86) in 8.25 bits an element: 32
 * consecutive elements of a row (the row's last block may be shorter) share an
 * exponent E, kept as the byte E + 127, and an element is code * 2^E.  With m
 * the largest magnitude of a block and e = floor(log2 m):
 *   FH_INT8  E = e - 6, code = rint(x 2^-E), ties to even, at most 127 in
 *            magnitude: off by at most 2^(E-1), where it is cut by less than 2^E;
 *   FH_E4M3  E = e - 8, or e - 7 where m 2^-E would pass 448; code = x 2^-E
 *            rounded to e4m3, at most 240 in magnitude at E = 120 (256 * 2^120 is
 *            infinite): off by at most 2^-4 |x| or 2^(E-10).
 * E >= -118.  A block that holds an infinity or a NaN has the byte 255 and codes
 * 0, and reads as NaN.  bf16 and fp32 hold every code * 2^E exactly.
 * codes: [rows, cols] bytes (8-byte aligned); exps: [rows, ceil(cols / 32)]
 * bytes, 9 to 248 or 255.  cols % 8 == 0; rows * cols < 2^35 (the norms: rows <
 * 2^26).
 */
typedef enum fh_fmt8 {
  FH_INT8 = 0, /* two's complement */
  FH_E4M3 = 1  /* OCP float8 e4m3  */
} fh_fmt8;

int fh_pack8(fh_dtype dt, fh_fmt8 fmt, const void* x, void* codes, uint8_t* exps, int64_t rows,
             int64_t cols, hipStream_t stream);
int fh_unpack8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps, void* x,
               int64_t rows, int64_t cols, hipStream_t stream);

/* fh_rmsnorm_fwd that also packs the x it reads (as fh_pack8 does), in one pass.
 * llama_rounding != 0: the normalised value is rounded to dt before its product
 * with w, as LlamaRMSNorm does, and y is fh_rmsnorm_fwd's bit for bit; 0: it is
 * not, and y is rounded once.  cols <= 8192, as in every norm here. */
int fh_rmsnorm_fwd_pack8(fh_dtype dt, fh_fmt8 fmt, const void* x, const void* w, void* y,
                         void* codes, uint8_t* exps, float* rstd, int64_t rows, int64_t cols,
                         float eps, int llama_rounding, hipStream_t stream);

/* fh_rmsnorm_fwd, fh_add_rmsnorm_fwd (h = to_dtype(x + a); y = rmsnorm(h)) and
 * fh_rmsnorm_bwd of a packed x, read as the values that fh_unpack8 gives.  With
 * llama_rounding each equals, bit for bit, the call on the unpacked tensor; without
 * it the normalised value and dy * w stay in fp32.  dt is the dtype of every tensor
 * but the packed one. */
int fh_rmsnorm_fwd8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps,
                    const void* w, void* y, float* rstd, int64_t rows, int64_t cols, float eps,
                    int llama_rounding, hipStream_t stream);
int fh_add_rmsnorm_fwd8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps,
                        const void* a, const void* w, void* h, void* y, float* rstd, int64_t rows,
                        int64_t cols, float eps, int llama_rounding, hipStream_t stream);
size_t fh_rmsnorm_bwd8_workspace_size(int64_t rows, int64_t cols);
int fh_rmsnorm_bwd8(fh_dtype dt, fh_fmt8 fmt, const void* dy, const void* codes,
                    const uint8_t* exps, const void* w, const float* rstd, const void* dres,
                    void* dx, void* dw, void* workspace, int64_t rows, int64_t cols, float eps,
                    int llama_rounding, hipStream_t stream);

/* ------------------------------------- norms after and before a block
 * A block's output a enters the residual stream x through a norm, a gate and a
 * residual scale, and the next block reads the stream through its norm:
 *   n = a rsqrt(mean(a^2) + eps) w_post          (n = a without w_post)
 *   h = to_dtype(x + scale * gate * n)           (gate 1 without one)
 *   y = to_dtype(h rsqrt(mean(h^2) + eps) w_pre) (no y without w_pre)
 * in fp32 between the roundings written; y is the norm of h as stored.  The
 * residual adds and norms of modeling_llama.py:284-325 are the case without
 * w_post, gate and scale (fh_add_rmsnorm_fwd, which rounds the normalised value
 * as LlamaRMSNorm does).  At least one of w_post and w_pre is given.
 * x, a, h, y: [rows, cols]; w_post, w_pre: [cols]; gate: [cols], or with
 * gate_per_token [rows, cols]; rstd_post, rstd_pre (nullable): fp32 [rows], the
 * reciprocal roots, which the backward reads.  cols % 8 == 0, cols <= 8192, all
 * tensors 16-byte aligned, h none of x, a and gate.
 */
int fh_block_norms_fwd(fh_dtype dt, const void* x, const void* a, const void* w_post,
                       const void* w_pre, const void* gate, int gate_per_token, float scale, void* h,
                       void* y, float* rstd_post, float* rstd_pre, int64_t rows, int64_t cols,
                       float eps, hipStream_t stream);

/* Gradients of fh_block_norms_fwd for dh and dy (dy with w_pre only): dx and da
 * [rows, cols]; dw_post, dw_pre [cols]; dgate of the gate's shape.  h and rstd_pre
 * are read with w_pre, rstd_post with w_post, a with w_post or a gate; the others
 * may be null.  The sums over rows are fp32, in a fixed order.  workspace:
 * fh_block_norms_bwd_workspace_size bytes, 16-byte aligned. */
size_t fh_block_norms_bwd_workspace_size(int64_t rows, int64_t cols);
int fh_block_norms_bwd(fh_dtype dt, const void* dh, const void* dy, const void* h, const void* a,
                       const void* w_post, const void* w_pre, const void* gate, int gate_per_token,
                       float scale, const float* rstd_post, const float* rstd_pre, void* dx,
                       void* da, void* dw_post, void* dw_pre, void* dgate, void* workspace,
                       int64_t rows, int64_t cols, hipStream_t stream);

/* --------------------------------------------------- rotary positions
 * Rotary embedding of q and k from positions and frequencies, for part of a head
 * or all of it.  Pair i of the rot_dim rotated dims (from `offset` on) of a head is
 *   FH_ROTARY_HALF         dims (offset + i, offset + rot_dim / 2 + i)
 *   FH_ROTARY_INTERLEAVED  dims (offset + 2i, offset + 2i + 1)
 * and is turned by position * inv_freq[i] radians, cos and sin times `factor`;
 * the other dims pass.  (fh_rope_fwd, apply_rotary_pos_emb of modeling_llama.py:
 * 130-160, is the half layout over the whole head from tables in the model's
 * dtype.)  Angles are computed in fp64, the turn in fp32, rounded once.
 * Token-major: head h of q at columns h * head_dim of its row, row strides in
 * elements; n_q or n_k may be 0, q and k then null.  Outputs may be their inputs
 * (same stride) and overlap nothing else (refused).  positions: int64 [n_positions] on the
 * device, token t at positions[t % n_positions] (tokens a multiple);
 * inv_freq: fp64 [rot_dim / 2] on the device.  (n_q + n_k) * head_dim <= 2^20,
 * head_dim <= 1024, row strides <= 2^28.  The backward takes and gives gradients: the turn back.
 */
typedef enum fh_rotary_layout {
  FH_ROTARY_HALF = 0,
  FH_ROTARY_INTERLEAVED = 1
} fh_rotary_layout;

int fh_rotary_fwd(fh_dtype dt, const void* q, int64_t ldq, int64_t n_q, const void* k, int64_t ldk,
                  int64_t n_k, void* q_out, int64_t ldqo, void* k_out, int64_t ldko, int64_t tokens,
                  int64_t head_dim, int64_t rot_dim, int64_t offset, fh_rotary_layout layout,
                  const int64_t* positions, int64_t n_positions, const double* inv_freq,
                  float factor, hipStream_t stream);
int fh_rotary_bwd(fh_dtype dt, const void* dq, int64_t lddq, int64_t n_q, const void* dk,
                  int64_t lddk, int64_t n_k, void* dq_out, int64_t lddqo, void* dk_out,
                  int64_t lddko, int64_t tokens, int64_t head_dim, int64_t rot_dim, int64_t offset,
                  fh_rotary_layout layout, const int64_t* positions, int64_t n_positions,
                  const double* inv_freq, float factor, hipStream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* FEMTOHIP_BLOCKS_H_ */
