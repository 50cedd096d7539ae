// C ABI of the short causal filter (see include/fm_scan_b200.h): argument checks, launch shapes, launches.
// No allocation, no synchronisation, no torch.
#include "capi_common.cuh"
#include "conv_kernels.cuh"

#define FMS_BY_TAPS(taps, CALL)                                          \
    switch (taps) {                                                      \
        case 2: { constexpr int K = 2; return CALL; }                    \
        case 3: { constexpr int K = 3; return CALL; }                    \
        case 4: { constexpr int K = 4; return CALL; }                    \
        case 5: { constexpr int K = 5; return CALL; }                    \
        case 6: { constexpr int K = 6; return CALL; }                    \
        case 7: { constexpr int K = 7; return CALL; }                    \
        default: { constexpr int K = 8; return CALL; }                   \
    }

namespace {

int conv_check(const fms_conv_args *a) {
    if (!a) return FMS_ERR_NULL_POINTER;
    if (!dtype_ok(a->dtype)) return FMS_ERR_BAD_DTYPE;
    if (a->batch < 0 || a->channels < 0 || a->T < 0 || a->taps < 2 || a->taps > 8) return FMS_ERR_BAD_SHAPE;
    if (a->T > 0x7fffffff - 4096) return FMS_ERR_TOO_LARGE;
    if (!product_ok({a->batch, a->channels, std::max<int64_t>(a->T, 16)})) return FMS_ERR_BAD_SHAPE;
    return FMS_OK;
}
int conv_pointers(const fms_conv_args *a) {
    if (!a->weight || (a->T && !a->tokens)) return FMS_ERR_NULL_POINTER;
    const size_t es = elem_size(a->dtype);
    if (!aligned_to(a->tokens, es) || !aligned_to(a->x0, es) || !aligned_to(a->weight, 4) || !aligned_to(a->bias, 4) ||
        !aligned_to(a->lengths, 8))
        return FMS_ERR_MISALIGNED;
    return FMS_OK;
}
// How rows are cut: lanes of a row, groups of a row and of a unit, units of a row.  `lead` positions stand in
// front of a row (backward they take in x0), and up to 15 bytes where rows do not start on a 16-byte boundary.
// A unit has as many groups as leave the GPU some 16000 warps (at (8,2048,4096) bf16 the backward takes 134 us
// with them, 153 us with a group a unit; longer units gain nothing).
struct ConvCut {
    int lpr, groups, per_unit, units;
};
ConvCut conv_cut(const fms_conv_args *a, int lead, bool aligned) {
    const int64_t es = elem_size(a->dtype), T = std::max<int64_t>(1, a->T + lead + (aligned ? 0 : 16 / es - 1));
    ConvCut c;
    c.lpr = 1;
    while (c.lpr < 32 && c.lpr * 8 * fms::kConvUnroll < T) c.lpr *= 2;
    const int64_t span = static_cast<int64_t>(c.lpr) * 8 * fms::kConvUnroll, rows = 32 / c.lpr;
    const int64_t warps = std::max<int64_t>(1, a->batch * ((a->channels + rows - 1) / rows));
    c.groups = static_cast<int>((T + span - 1) / span);
    c.units = static_cast<int>(std::min<int64_t>(c.groups, (16000 + warps - 1) / warps));
    c.per_unit = (c.groups + c.units - 1) / c.units;
    c.units = (c.groups + c.per_unit - 1) / c.per_unit;
    return c;
}

template <typename S>
fms::ConvProblem<S> conv_problem(const fms_conv_args *a, const ConvCut &c) {
    fms::ConvProblem<S> p;
    p.x = static_cast<const S *>(a->tokens);
    std::copy_n(a->tokens_stride, 2, p.xs);
    p.weight = a->weight, p.bias = a->bias, p.x0 = static_cast<const S *>(a->x0), p.lengths = a->lengths;
    p.batch = a->batch, p.channels = a->channels;
    p.T = static_cast<int>(a->T), p.silu = a->silu != 0;
    p.lpr = c.lpr, p.groups = c.groups, p.per_unit = c.per_unit, p.units = c.units;
    return p;
}
template <typename S>
bool conv_grid(const fms::ConvProblem<S> &p, dim3 &grid) {
    const int64_t per = 32 / p.lpr * fms::kConvWarps, x = (p.channels + per - 1) / per * p.units;
    grid = dim3(static_cast<unsigned>(x), static_cast<unsigned>(std::min<int64_t>(p.batch, 65535)));
    return x <= kMaxGrid;
}
// every row written starts on a 16-byte boundary
bool conv_rows16(const fms_conv_args *a, const void *written) {
    return aligned_to(written, 16) && a->T * elem_size(a->dtype) % 16 == 0;
}

template <typename S, int K>
int launch_conv_forward(const fms_conv_args *a, void *out, void *x_last, cudaStream_t st) {
    const auto p = conv_problem<S>(a, conv_cut(a, 0, conv_rows16(a, out)));
    dim3 grid;
    if (!conv_grid(p, grid)) return FMS_ERR_TOO_LARGE;
    fms::conv_forward_kernel<S, K><<<grid, fms::kConvWarps * 32, 0, st>>>(
        p, static_cast<S *>(out), static_cast<S *>(x_last));
    return check_launch();
}

template <typename S, int K>
int launch_conv_backward(const fms_conv_args *a, const void *dout, const void *dlast, void *dx, float *dw, float *db,
                         void *dx0, float *part, cudaStream_t st) {
    const auto p = conv_problem<S>(a, conv_cut(a, dx0 ? 8 : 0, conv_rows16(a, dx)));
    dim3 grid;
    if (!conv_grid(p, grid) || (p.channels + 3) / 4 > kMaxGrid) return FMS_ERR_TOO_LARGE;
    fms::conv_backward_kernel<S, K><<<grid, fms::kConvWarps * 32, 0, st>>>(
        p, static_cast<const S *>(dout), static_cast<const S *>(dlast), static_cast<S *>(dx), static_cast<S *>(dx0), part);
    if (int rc = check_launch()) return rc;
    fms::conv_weight_kernel<K><<<static_cast<unsigned>((p.channels + 3) / 4), 128, 0, st>>>(part, dw, db, p.batch,
                                                                                         p.channels, p.units);
    return check_launch();
}

template <typename S, int K>
int launch_conv_step(const fms_conv_args *a, void *state, int64_t pool, const int64_t *slots, void *out, cudaStream_t st) {
    const auto p = conv_problem<S>(a, ConvCut{});
    const int64_t blocks = (p.channels + 127) / 128;
    if (blocks > kMaxGrid || p.batch * blocks > kMaxGrid) return FMS_ERR_TOO_LARGE;
    fms::conv_step_kernel<S, K><<<static_cast<unsigned>(p.batch * blocks), 128, 0, st>>>(
        p, static_cast<S *>(state), pool, slots, static_cast<S *>(out), static_cast<int>(blocks));
    return check_launch();
}

template <typename S>
int conv_forward_t(const fms_conv_args *a, void *out, void *x_last, cudaStream_t st) {
    FMS_BY_TAPS(a->taps, (launch_conv_forward<S, K>(a, out, x_last, st)));
}
template <typename S>
int conv_backward_t(const fms_conv_args *a, const void *dout, const void *dlast, void *dx, float *dw, float *db, void *dx0,
                    float *part, cudaStream_t st) {
    FMS_BY_TAPS(a->taps, (launch_conv_backward<S, K>(a, dout, dlast, dx, dw, db, dx0, part, st)));
}
template <typename S>
int conv_step_t(const fms_conv_args *a, void *state, int64_t pool, const int64_t *slots, void *out, cudaStream_t st) {
    FMS_BY_TAPS(a->taps, (launch_conv_step<S, K>(a, state, pool, slots, out, st)));
}

}  // namespace

FMS_EXPORT int fms_conv_forward(const fms_conv_args *a, void *out, void *x_last, fms_stream_t stream) {
    if (int rc = conv_check(a)) return rc;
    if (a->batch == 0 || a->channels == 0) return FMS_OK;
    if (int rc = conv_pointers(a)) return rc;
    if (a->T && !out) return FMS_ERR_NULL_POINTER;
    if (!aligned_to(out, elem_size(a->dtype)) || !aligned_to(x_last, elem_size(a->dtype))) return FMS_ERR_MISALIGNED;
    if (a->T == 0 && !x_last) return FMS_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    FMS_BY_TYPE(a->dtype, (conv_forward_t<S>(a, out, x_last, st)));
}

FMS_EXPORT size_t fms_conv_backward_workspace_bytes(const fms_conv_args *a) {
    if (conv_check(a) != FMS_OK || a->batch == 0 || a->channels == 0) return 0;
    return round256(sizeof(float) * a->batch * a->channels * conv_cut(a, 8, false).groups * (a->taps + 1));  // units <= groups
}

FMS_EXPORT int fms_conv_backward(const fms_conv_args *a, const void *grad_out, const void *grad_last, void *grad_tokens,
                                 float *grad_weight, float *grad_bias, void *grad_x0, void *workspace,
                                 size_t workspace_bytes, fms_stream_t stream) {
    if (int rc = conv_check(a)) return rc;
    if (a->channels == 0) return FMS_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!grad_weight) return FMS_ERR_NULL_POINTER;
    if (!aligned_to(grad_weight, 4) || !aligned_to(grad_bias, 4)) return FMS_ERR_MISALIGNED;
    if (a->batch == 0) {
        if (int rc = copy_or_zero(nullptr, grad_weight, a->channels * a->taps, st)) return rc;
        return copy_or_zero(nullptr, grad_bias, a->channels, st);
    }
    if (int rc = conv_pointers(a)) return rc;
    if (a->T && (!grad_out || !grad_tokens)) return FMS_ERR_NULL_POINTER;
    for (const void *p : {grad_out, grad_last, static_cast<const void *>(grad_tokens), static_cast<const void *>(grad_x0)})
        if (!aligned_to(p, elem_size(a->dtype))) return FMS_ERR_MISALIGNED;
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < fms_conv_backward_workspace_bytes(a))
        return FMS_ERR_WORKSPACE;
    FMS_BY_TYPE(a->dtype, (conv_backward_t<S>(a, grad_out, grad_last, grad_tokens, grad_weight, grad_bias, grad_x0,
                                              static_cast<float *>(workspace), st)));
}

FMS_EXPORT int fms_conv_step(const fms_conv_args *a, void *state, int64_t pool, const int64_t *slots, void *out,
                             fms_stream_t stream) {
    if (int rc = conv_check(a)) return rc;
    if (a->T != 1 || pool < 0 || (!slots && pool < a->batch)) return FMS_ERR_BAD_SHAPE;
    if (!product_ok({pool, a->channels, 8})) return FMS_ERR_BAD_SHAPE;
    if (a->batch == 0 || a->channels == 0) return FMS_OK;
    if (int rc = conv_pointers(a)) return rc;
    if (!out || (pool && !state)) return FMS_ERR_NULL_POINTER;
    if (!aligned_to(state, elem_size(a->dtype)) || !aligned_to(slots, 8) || !aligned_to(out, elem_size(a->dtype)))
        return FMS_ERR_MISALIGNED;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    FMS_BY_TYPE(a->dtype, (conv_step_t<S>(a, state, pool, slots, out, st)));
}
