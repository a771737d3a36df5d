/*
 * opus_dense.h - C ABI of libopus_msmv.so, dense part: the operators a decoder layer runs around the sampling
 * op of opus_msmv.h, for MI355X / gfx950.  They have no counterpart among the reference's native kernels: its
 * decoder composes them from library layers (models/opus_transformer.py:301-448).
 *
 *   linear          z = x W^T + b;  y = residual + D(act(z))
 *   residual_norm   r = scale * x + gate * D(post(block));  y = norm(r)
 *   dropout         y = residual + D(x)
 *
 * Conventions
 *   - Tensors are contiguous (rows x last dimension), of one element type (fp32, bf16 or fp16), on the device that
 *     is current when the call is made; any address that is a multiple of the element size will do.
 *   - Nothing is allocated, freed or synchronised inside; launches are asynchronous on `stream` (a hipStream_t as
 *     void*, NULL = the default stream).  The library keeps no state between calls and is thread-safe.
 *   - A workspace is a device buffer of the size its query returns, 16-byte aligned; its contents on entry do not
 *     matter, and two calls that may run at the same time need one each.  No result depends on the order in which
 *     workgroups run.
 *   - Outputs must not overlap inputs, except where an entry says so.
 *   - Return value: OPUS_DENSE_OK (0) or a negative OPUS_DENSE_E* code; text via opus_dense_strerror().  Arguments
 *     are checked before anything is launched; sizes of zero are no error (outputs that exist are still written).
 *     OPUS_DENSE_ETOOLARGE may also mean that a kernel would need more threads than a launch counts (2^32), and then
 *     come after a launch: buffers for results hold nothing of use.
 */
#ifndef OPUS_DENSE_H
#define OPUS_DENSE_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { OPUS_DENSE_F32 = 0, OPUS_DENSE_BF16 = 1, OPUS_DENSE_F16 = 2 };

enum {
    OPUS_DENSE_OK = 0,
    OPUS_DENSE_EINVAL_TYPE = -1,      /* unknown element type */
    OPUS_DENSE_EINVAL_DIMS = -2,      /* a negative size, or sizes that do not belong together */
    OPUS_DENSE_EINVAL_PTR = -3,       /* a NULL pointer where data is required, or one that is not element-aligned */
    OPUS_DENSE_ETOOLARGE = -4,        /* sizes beyond the limits below */
    OPUS_DENSE_EWORKSPACE = -5,       /* workspace missing, misaligned or too small */
    OPUS_DENSE_EINVAL_FLAGS = -6,     /* unknown activation, norm kind or dropout threshold */
    OPUS_DENSE_ELAUNCH = -7           /* a kernel launch of this call failed */
};

enum { OPUS_DENSE_ACT_NONE = 0, OPUS_DENSE_ACT_RELU = 1, OPUS_DENSE_ACT_GELU = 2, OPUS_DENSE_ACT_GELU_TANH = 3,
       OPUS_DENSE_ACT_SILU = 4 };
enum { OPUS_DENSE_NORM_LAYER = 0, OPUS_DENSE_NORM_RMS = 1 };

#define OPUS_DENSE_MAX_WIDTH 16384    /* widest row of residual_norm */

/*
 * Dropout.  An element (row, col) of a tensor of `cols` columns is kept iff its 16 random bits are >= threshold,
 * and is then scaled by 65536 / (65536 - threshold); a dropped element is exactly 0, whatever it was.  The bits
 * come from Philox 4x32-10 with counter (col / 8, row mod 2^32, row div 2^32, offset) and key `seed`: bits
 * 16 * (col % 2) upwards of output word (col % 8) / 2.  So a mask depends on (seed, offset, row, col) alone - not
 * on the type, the operator or the launch - is computed again in the backward, and is never stored.
 * `seed_ptr`, if not NULL, is a device address (8-byte aligned) the kernels read the seed from when they run, so
 * that a captured graph can be given a new seed between replays.  NULL in place of the struct: no dropout.
 */
typedef struct {
    unsigned int threshold;           /* 0 (keep all) .. 65536 (drop all) */
    unsigned int offset;
    unsigned long long seed;
    const unsigned long long *seed_ptr;
} opus_dense_dropout_t;

const char *opus_dense_strerror(int code);

/*
 * y = residual + D(act(x W^T + bias)) for x [M, K], W [N, K], bias [N] or NULL, residual [M, N] or NULL.
 * Products and sums are in fp32; y [M, N] is rounded once.  z [M, N] (NULL: not wanted) receives x W^T + bias in
 * the element type, which is what the backward needs where there is an activation; what that type cannot hold though
 * it is finite becomes the type's largest number of its sign.
 * y may be the same buffer as residual.
 */
size_t opus_dense_linear_workspace_bytes(int type, long long M, long long N, long long K);
int opus_dense_linear_forward(int type, const void *x, const void *weight, const void *bias, const void *residual,
                              long long M, long long N, long long K, int activation,
                              const opus_dense_dropout_t *dropout, void *y, void *z,
                              void *workspace, size_t workspace_bytes, void *stream);

/*
 * Its gradients: dz = D(dy) act'(z); dx [M, K] = dz W; dweight [N, K] = dz^T x; dbias [N] = sum over rows of dz.
 * Each of dx, dweight, dbias may be NULL (not computed).  z is needed with an activation.  dz is held in the
 * element type: `dz_buffer` [M, N] receives it where there is an activation or dropout (required then, where
 * anything is computed; without either, dz is dy itself); dbias is summed before that rounding.  d residual is dy.
 */
size_t opus_dense_linear_backward_workspace_bytes(int type, long long M, long long N, long long K);
int opus_dense_linear_backward(int type, const void *dy, const void *x, const void *weight, const void *z,
                               long long M, long long N, long long K, int activation,
                               const opus_dense_dropout_t *dropout, void *dz_buffer,
                               void *dx, void *dweight, void *dbias,
                               void *workspace, size_t workspace_bytes, void *stream);

/*
 * r = scale * x + gate * D(post(block)),  y = norm(r) for x, block, r, y [rows, width].
 *   kind: LayerNorm (r - mean) / sqrt(var + eps) * weight + bias, or RMS r / sqrt(mean r^2 + eps) * weight.
 *   weight, bias [width] or NULL (1 and 0).  bias / post_bias with either kind.
 *   post_weight [width]: the block's output is normed first (same kind and eps); NULL: post is the identity.
 *   gate [gate_rows, width] or NULL (1): row i of x uses gate row i / (rows / gate_rows); gate_rows divides rows.
 *   y and stream (r in the element type) may each be NULL: not wanted.
 *   stats: fp32 [rows, 4] (mean and 1/sigma of block, mean and 1/sigma of r), for the backward; NULL: not wanted.
 * y is computed from the unrounded r.  y may be the same buffer as x or block, and so may stream (not the same one).
 */
typedef struct {
    int type, kind;
    long long rows, width, gate_rows;
    float eps, scale;
    const void *x, *block, *weight, *bias, *post_weight, *post_bias, *gate;
    const opus_dense_dropout_t *dropout;
} opus_dense_norm_t;

int opus_dense_norm_forward(const opus_dense_norm_t *in, void *y, void *stream_out, float *stats, void *stream);

/*
 * Its gradients for dy and dstream (either may be NULL: zero).  dx, dblock [rows, width], dweight, dbias,
 * dpost_weight, dpost_bias [width], dgate [gate_rows, width]; each may be NULL (not computed).  `stats` is the
 * forward's.  r is computed again from x and block; nothing else is kept from the forward.
 */
typedef struct {
    void *dx, *dblock, *dweight, *dbias, *dpost_weight, *dpost_bias, *dgate;
} opus_dense_norm_grads_t;

size_t opus_dense_norm_backward_workspace_bytes(int type, long long rows, long long width, long long gate_rows);
int opus_dense_norm_backward(const opus_dense_norm_t *in, const void *dy, const void *dstream, const float *stats,
                             const opus_dense_norm_grads_t *out, void *workspace, size_t workspace_bytes,
                             void *stream);

/*
 * y = residual + D(x) for x, y [rows, cols], residual the same or NULL.  y may be the same buffer as x or
 * residual.  It is its own backward: dx = D(dy) with the same dropout argument.
 */
int opus_dense_dropout(int type, const void *x, const void *residual, long long rows, long long cols,
                       const opus_dense_dropout_t *dropout, void *y, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* OPUS_DENSE_H */
