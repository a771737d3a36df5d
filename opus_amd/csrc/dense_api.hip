// C ABI of the dense operators (include/opus_dense.h): argument checks and dispatch to the launchers.  No allocation,
// no synchronisation, no state.
#include "dense_common.h"

#include <limits.h>

namespace {

constexpr long long MAX_SIDE = INT_MAX - 255;     // of a matrix: 32-bit column indices, tile counts that fit an int

bool known_type(int type) { return type >= OPUS_DENSE_F32 && type <= OPUS_DENSE_F16; }

// element-aligned, or NULL
bool fits(const void *p, int type) { return reinterpret_cast<uintptr_t>(p) % dn_type_bytes(type) == 0; }

int make_drop(const opus_dense_dropout_t *in, DnDrop &out)
{
    out = {};
    if (!in || in->threshold == 0)
        return OPUS_DENSE_OK;
    if (in->threshold > 65536)
        return OPUS_DENSE_EINVAL_FLAGS;
    if (reinterpret_cast<uintptr_t>(in->seed_ptr) % 8)
        return OPUS_DENSE_EINVAL_PTR;
    out.threshold = in->threshold;
    out.offset = in->offset;
    out.scale = in->threshold == 65536 ? 0.f : 65536.f / (float)(65536 - in->threshold);
    out.seed = in->seed;
    out.seed_ptr = reinterpret_cast<const uint64_t *>(in->seed_ptr);
    return OPUS_DENSE_OK;
}

int status(hipError_t e)
{
    return e == hipSuccess ? OPUS_DENSE_OK : e == hipErrorInvalidValue ? OPUS_DENSE_ETOOLARGE : OPUS_DENSE_ELAUNCH;
}

int check_workspace(const void *workspace, size_t have, size_t need)
{
    if (need == 0)
        return OPUS_DENSE_OK;
    return workspace && have >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 ? OPUS_DENSE_OK
                                                                                        : OPUS_DENSE_EWORKSPACE;
}

// bytes of any of the three matrices stay within a signed 64-bit offset by far; the sides are what is limited
int check_linear(int type, long long M, long long N, long long K, int activation)
{
    if (!known_type(type))
        return OPUS_DENSE_EINVAL_TYPE;
    if (M < 0 || N < 0 || K < 0)
        return OPUS_DENSE_EINVAL_DIMS;
    if (M > MAX_SIDE || N > MAX_SIDE || K > MAX_SIDE)
        return OPUS_DENSE_ETOOLARGE;
    if (activation < OPUS_DENSE_ACT_NONE || activation > OPUS_DENSE_ACT_SILU)
        return OPUS_DENSE_EINVAL_FLAGS;
    return OPUS_DENSE_OK;
}

int check_norm(const opus_dense_norm_t *in, DnDrop &drop)
{
    if (!in)
        return OPUS_DENSE_EINVAL_PTR;
    if (!known_type(in->type))
        return OPUS_DENSE_EINVAL_TYPE;
    if (in->kind != OPUS_DENSE_NORM_LAYER && in->kind != OPUS_DENSE_NORM_RMS)
        return OPUS_DENSE_EINVAL_FLAGS;
    // (a gate without rows goes with no rows at all)
    if (in->rows < 0 || in->width < 1 || (in->gate && in->gate_rows < (in->rows > 0)) ||
        (in->gate && in->rows > 0 && in->rows % in->gate_rows))
        return OPUS_DENSE_EINVAL_DIMS;
    if (in->width > OPUS_DENSE_MAX_WIDTH || in->rows > LLONG_MAX / 8 / in->width)
        return OPUS_DENSE_ETOOLARGE;
    if (in->rows > 0 && (!in->x || !in->block))
        return OPUS_DENSE_EINVAL_PTR;
    const void *all[] = {in->x, in->block, in->weight, in->bias, in->post_weight, in->post_bias, in->gate};
    for (const void *p : all)
        if (!fits(p, in->type))
            return OPUS_DENSE_EINVAL_PTR;
    return make_drop(in->dropout, drop);
}

}  // namespace

extern "C" {

const char *opus_dense_strerror(int code)
{
    switch (code) {
    case OPUS_DENSE_OK: return "ok";
    case OPUS_DENSE_EINVAL_TYPE: return "unknown element type";
    case OPUS_DENSE_EINVAL_DIMS: return "invalid tensor dimensions";
    case OPUS_DENSE_EINVAL_PTR: return "null or misaligned pointer argument";
    case OPUS_DENSE_ETOOLARGE: return "problem too large";
    case OPUS_DENSE_EWORKSPACE: return "workspace missing, misaligned or too small";
    case OPUS_DENSE_EINVAL_FLAGS: return "unknown activation, norm kind or dropout threshold";
    case OPUS_DENSE_ELAUNCH: return "HIP kernel launch failed";
    default: return "unknown error code";
    }
}

size_t opus_dense_linear_workspace_bytes(int type, long long M, long long N, long long K)
{
    return check_linear(type, M, N, K, 0) == OPUS_DENSE_OK ? dn_linear_forward_workspace(type, M, N, K) : 0;
}

int opus_dense_linear_forward(int type, const void *x, const void *weight, const void *bias, const void *residual,
                              long long M, long long N, long long K, int activation,
                              const opus_dense_dropout_t *dropout, void *y, void *z,
                              void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_linear(type, M, N, K, activation);
    DnDrop drop;
    if (rc == OPUS_DENSE_OK)
        rc = make_drop(dropout, drop);
    if (rc != OPUS_DENSE_OK)
        return rc;
    if (M == 0 || N == 0)
        return OPUS_DENSE_OK;
    if (!y || (K > 0 && (!x || !weight)))
        return OPUS_DENSE_EINVAL_PTR;
    const void *all[] = {x, weight, bias, residual, y, z};
    for (const void *p : all)
        if (!fits(p, type))
            return OPUS_DENSE_EINVAL_PTR;
    rc = check_workspace(workspace, workspace_bytes, dn_linear_forward_workspace(type, M, N, K));
    if (rc != OPUS_DENSE_OK)
        return rc;
    return status(dn_launch_linear_forward(type, x, weight, bias, residual, M, N, K, activation, drop, y, z,
                                           static_cast<float *>(workspace), (hipStream_t)stream));
}

size_t opus_dense_linear_backward_workspace_bytes(int type, long long M, long long N, long long K)
{
    return check_linear(type, M, N, K, 0) == OPUS_DENSE_OK ? dn_linear_backward_workspace(type, M, N, K) : 0;
}

int opus_dense_linear_backward(int type, const void *dy, const void *x, const void *weight, const void *z,
                               long long M, long long N, long long K, int activation,
                               const opus_dense_dropout_t *dropout, void *dz_buffer,
                               void *dx, void *dweight, void *dbias,
                               void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_linear(type, M, N, K, activation);
    DnDrop drop;
    if (rc == OPUS_DENSE_OK)
        rc = make_drop(dropout, drop);
    if (rc != OPUS_DENSE_OK)
        return rc;
    if (!dx && !dweight && !dbias)
        return OPUS_DENSE_OK;
    const bool prepare = activation != OPUS_DENSE_ACT_NONE || drop.threshold;
    const bool any = M > 0 && N > 0;
    if (any && (!dy || (prepare && !dz_buffer) || (activation != OPUS_DENSE_ACT_NONE && !z)))
        return OPUS_DENSE_EINVAL_PTR;
    if (any && K > 0 && ((dx && !weight) || (dweight && !x)))
        return OPUS_DENSE_EINVAL_PTR;
    const void *all[] = {dy, x, weight, z, dz_buffer, dx, dweight, dbias};
    for (const void *p : all)
        if (!fits(p, type))
            return OPUS_DENSE_EINVAL_PTR;
    rc = check_workspace(workspace, workspace_bytes, dn_linear_backward_workspace(type, M, N, K));
    if (rc != OPUS_DENSE_OK)
        return rc;
    return status(dn_launch_linear_backward(type, dy, x, weight, z, M, N, K, activation, drop, dz_buffer, dx, dweight, dbias,
                                            static_cast<float *>(workspace), (hipStream_t)stream));
}

int opus_dense_norm_forward(const opus_dense_norm_t *in, void *y, void *stream_out, float *stats, void *stream)
{
    DnDrop drop;
    const int rc = check_norm(in, drop);
    if (rc != OPUS_DENSE_OK)
        return rc;
    if (!fits(y, in->type) || !fits(stream_out, in->type) || reinterpret_cast<uintptr_t>(stats) % 16)
        return OPUS_DENSE_EINVAL_PTR;
    if (in->rows == 0 || (!y && !stream_out && !stats))
        return OPUS_DENSE_OK;
    return status(dn_launch_norm_forward(*in, drop, y, stream_out, stats, (hipStream_t)stream));
}

size_t opus_dense_norm_backward_workspace_bytes(int type, long long rows, long long width, long long gate_rows)
{
    if (!known_type(type) || rows < 0 || width < 1 || width > OPUS_DENSE_MAX_WIDTH || gate_rows < 0 || gate_rows > rows ||
        rows > LLONG_MAX / 8 / width)
        return 0;
    return dn_norm_backward_workspace(rows, width, gate_rows);
}

int opus_dense_norm_backward(const opus_dense_norm_t *in, const void *dy, const void *dstream, const float *stats,
                             const opus_dense_norm_grads_t *out, void *workspace, size_t workspace_bytes,
                             void *stream)
{
    DnDrop drop;
    int rc = check_norm(in, drop);
    if (rc != OPUS_DENSE_OK)
        return rc;
    if (!out || (in->rows > 0 && !stats) || reinterpret_cast<uintptr_t>(stats) % 16)
        return OPUS_DENSE_EINVAL_PTR;
    const void *all[] = {dy, dstream, out->dx, out->dblock, out->dweight, out->dbias, out->dpost_weight, out->dpost_bias,
                         out->dgate};
    for (const void *p : all)
        if (!fits(p, in->type))
            return OPUS_DENSE_EINVAL_PTR;
    if (((out->dpost_weight || out->dpost_bias) && !in->post_weight) || (out->dgate && !in->gate))
        return OPUS_DENSE_EINVAL_FLAGS;
    const long long gate_rows = in->gate ? in->gate_rows : 0;
    rc = check_workspace(workspace, workspace_bytes, dn_norm_backward_workspace(in->rows, in->width, gate_rows));
    if (rc != OPUS_DENSE_OK)
        return rc;
    return status(dn_launch_norm_backward(*in, drop, dy, dstream, stats, *out, static_cast<float *>(workspace),
                                          (hipStream_t)stream));
}

int opus_dense_dropout(int type, const void *x, const void *residual, long long rows, long long cols,
                       const opus_dense_dropout_t *dropout, void *y, void *stream)
{
    if (!known_type(type))
        return OPUS_DENSE_EINVAL_TYPE;
    if (rows < 0 || cols < 0)
        return OPUS_DENSE_EINVAL_DIMS;
    if (cols > MAX_SIDE || (cols > 0 && rows > LLONG_MAX / 8 / cols))
        return OPUS_DENSE_ETOOLARGE;
    DnDrop drop;
    const int rc = make_drop(dropout, drop);
    if (rc != OPUS_DENSE_OK)
        return rc;
    if (rows == 0 || cols == 0)
        return OPUS_DENSE_OK;
    if (!x || !y || !fits(x, type) || !fits(y, type) || !fits(residual, type))
        return OPUS_DENSE_EINVAL_PTR;
    return status(dn_launch_elementwise(type, x, residual, nullptr, OPUS_DENSE_ACT_NONE, rows, cols, drop, y,
                                        (hipStream_t)stream));
}

}  // extern "C"
