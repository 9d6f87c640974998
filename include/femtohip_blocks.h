/*
 * femtohip_blocks.h -- C ABI of the MI355X (gfx950) kernels around a
 * checkpointed block: activations kept in 8 bits, the norms after and before a
 * block, and rotary positions.  Same library and conventions as femtohip.h
 * (device pointers owned by the caller, workspaces passed in, asynchronous on
 * `stream`, int status with fh_last_error(), thread-safe: no state of its own);
 * versioned by itself.
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
 *            rounded to e4m3: off by at most 2^-4 |x| or 2^(E-10).
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

/* fh_rmsnorm_fwd that also packs the x it reads: fh_rmsnorm_fwd and fh_pack8 in
 * one pass, bit for bit.  cols <= 8192, as in every norm here. */
int fh_rmsnorm_fwd_pack8(fh_dtype dt, fh_fmt8 fmt, const void* x, const void* w, void* y,
                         void* codes, uint8_t* exps, float* rstd, int64_t rows, int64_t cols,
                         float eps, hipStream_t stream);

/* fh_rmsnorm_fwd, fh_add_rmsnorm_fwd (h = to_dtype(x + a); y = rmsnorm(h)) and
 * fh_rmsnorm_bwd of a packed x: each equals, bit for bit, the call on the tensor
 * that fh_unpack8 gives.  dt is the dtype of every tensor but the packed one. */
int fh_rmsnorm_fwd8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps,
                    const void* w, void* y, float* rstd, int64_t rows, int64_t cols, float eps,
                    hipStream_t stream);
int fh_add_rmsnorm_fwd8(fh_dtype dt, fh_fmt8 fmt, const void* codes, const uint8_t* exps,
                        const void* a, const void* w, void* h, void* y, float* rstd, int64_t rows,
                        int64_t cols, float eps, hipStream_t stream);
size_t fh_rmsnorm_bwd8_workspace_size(int64_t rows, int64_t cols);
int fh_rmsnorm_bwd8(fh_dtype dt, fh_fmt8 fmt, const void* dy, const void* codes,
                    const uint8_t* exps, const void* w, const float* rstd, const void* dres,
                    void* dx, void* dw, void* workspace, int64_t rows, int64_t cols, float eps,
                    hipStream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* FEMTOHIP_BLOCKS_H_ */
