// C ABI of the selective state-space scan (see include/fm_scan_b200.h): argument
// checks, launch shapes, launches.  No allocation, no synchronisation, no torch.
#include "fm_scan_b200.h"

#include <algorithm>
#include <cstdlib>

#include "capi_common.cuh"
#include "ssm_kernels.cuh"

namespace {

int ssm_check(const fms_ssm_args *a) {
    if (!a) return FMS_ERR_NULL_POINTER;
    if (!dtype_ok(a->dtype)) return FMS_ERR_BAD_DTYPE;
    if (a->batch < 0 || a->channels < 0 || a->T < 0 || a->groups < 1 || a->states < 1) return FMS_ERR_BAD_SHAPE;
    if (a->channels % a->groups) return FMS_ERR_BAD_SHAPE;
    if (a->states > FMS_SSM_MAX_STATES || a->T > 0x7fffffff - 4096 || a->channels > 0x7fffffff) return FMS_ERR_TOO_LARGE;
    if (!product_ok({a->batch, a->channels, std::max<int64_t>(a->T, a->states)}) ||
        !product_ok({a->batch, a->groups, a->states, a->T}) ||
        !product_ok({a->batch, a->channels, a->T / fms::kSsmTile + 1, a->states}))
        return FMS_ERR_BAD_SHAPE;
    return FMS_OK;
}

inline bool ssm_empty(const fms_ssm_args *a) { return a->batch == 0 || a->channels == 0; }

int ssm_pointers(const fms_ssm_args *a, bool big) {
    const size_t es = elem_size(a->dtype);
    if (!a->A || (big && (!a->tokens || !a->delta || !a->B || !a->C))) return FMS_ERR_NULL_POINTER;
    for (const void *p : {a->tokens, a->delta, a->z, a->B, a->C})
        if (!aligned_to(p, es)) return FMS_ERR_MISALIGNED;
    for (const float *p : {a->A, a->D, a->delta_bias, a->h0})
        if (!aligned_to(p, 4)) return FMS_ERR_MISALIGNED;
    if (!aligned_to(a->lengths, 8)) return FMS_ERR_MISALIGNED;
    return FMS_OK;
}

bool ssm_aligned(const fms_ssm_args *a) {
    const int64_t es = elem_size(a->dtype);
    return a->T * es % 16 == 0 && rows16(a->tokens, a->tokens_stride, 2, es) && rows16(a->delta, a->delta_stride, 2, es) &&
           (!a->z || rows16(a->z, a->z_stride, 2, es)) && rows16(a->B, a->B_stride, 3, es) &&
           rows16(a->C, a->C_stride, 3, es);
}

template <typename S>
fms::SsmProblem<S> ssm_problem(const fms_ssm_args *a, int cw, int warps) {
    fms::SsmProblem<S> p;
    p.x = static_cast<const S *>(a->tokens), p.delta = static_cast<const S *>(a->delta), p.z = static_cast<const S *>(a->z);
    p.B = static_cast<const S *>(a->B), p.C = static_cast<const S *>(a->C);
    std::copy_n(a->tokens_stride, 2, p.xs);
    std::copy_n(a->delta_stride, 2, p.ds);
    std::copy_n(a->z_stride, 2, p.zs);
    std::copy_n(a->B_stride, 3, p.Bs);
    std::copy_n(a->C_stride, 3, p.Cs);
    p.A = a->A, p.D = a->D, p.bias = a->delta_bias, p.h0 = a->h0, p.lengths = a->lengths;
    p.batch = a->batch, p.channels = a->channels, p.groups = a->groups;
    p.T = static_cast<int>(a->T), p.N = static_cast<int>(a->states);
    p.NP = (p.N + fms::kSsmNB - 1) / fms::kSsmNB * fms::kSsmNB;
    p.per_group = static_cast<int>(a->channels / a->groups);
    p.cw = cw;
    p.chunks = (p.per_group + cw * warps - 1) / (cw * warps);
    p.tiles = static_cast<int>((a->T + fms::kSsmTile - 1) / fms::kSsmTile);
    p.softplus = a->delta_softplus != 0;
    return p;
}

inline int padded_states(const fms_ssm_args *a) {
    return static_cast<int>((a->states + fms::kSsmNB - 1) / fms::kSsmNB * fms::kSsmNB);
}

// shared memory of a CTA: as the kernels lay it out
size_t ssm_fwd_smem(const fms_ssm_args *a, int cw) {
    return a->dtype == FMS_F32
               ? fms::ssm_bc_bytes<float>() + fms::kSsmFwdWarps * fms::ssm_fwd_warp_bytes<float>(cw, padded_states(a))
               : fms::ssm_bc_bytes<__half>() + fms::kSsmFwdWarps * fms::ssm_fwd_warp_bytes<__half>(cw, padded_states(a));
}
size_t ssm_bwd_smem(const fms_ssm_args *a, int cw) {
    const size_t red = sizeof(float) * fms::kSsmBwdWarps * 64 * 32;
    return red + (a->dtype == FMS_F32
                      ? fms::ssm_bc_bytes<float>() + fms::kSsmBwdWarps * fms::ssm_bwd_warp_bytes<float>(cw, padded_states(a))
                      : fms::ssm_bc_bytes<__half>() + fms::kSsmBwdWarps * fms::ssm_bwd_warp_bytes<__half>(cw, padded_states(a)));
}

// Channels of a warp.  More of them spread a tile's B, C and barriers over more work (and, backward,
// shrink the partial sums of their gradients); fewer give more warps.  The time is taken as the number
// of waves times the channels of a warp plus the share of a channel that a tile costs on its own.
int best_cw(const fms_ssm_args *a, int warps, int most, int per_sm, double own, size_t (*smem)(const fms_ssm_args *, int)) {
    const int64_t per = a->channels / a->groups;
    int best = 1;
    double least = 0;
    for (int cw = 1; cw <= most; ++cw) {
        const size_t bytes = smem(a, cw);
        if (bytes > kMaxSmem) break;
        const int64_t ctas = a->batch * a->groups * ((per + cw * warps - 1) / (cw * warps));
        const int64_t room = 148 * std::min<int64_t>(per_sm, static_cast<int64_t>((kMaxSmem + 1024) / (bytes + 1024)));
        const double t = static_cast<double>((ctas + room - 1) / room) * (cw + own);
        if (cw == 1 || t < least) best = cw, least = t;
    }
    return best;
}
int env_int(const char *name, int dflt) { const char *s = std::getenv(name); return s ? std::atoi(s) : dflt; }
int ssm_fwd_cw(const fms_ssm_args *a) { if (int v = env_int("X_FCW", 0)) return v; return best_cw(a, fms::kSsmFwdWarps, 8, 3, 1.5, ssm_fwd_smem); }
int ssm_bwd_cw(const fms_ssm_args *a) { if (int v = env_int("X_BCW", 0)) return v; return best_cw(a, fms::kSsmBwdWarps, 8, 1, 1.5, ssm_bwd_smem); }

template <typename Kernel>
int allow_smem(Kernel kernel, size_t bytes) {
    return fms::record_cuda_error(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
}

// out[i] = sum over `count` slices of `stride` floats, in order
__global__ void sum_slices_kernel(const float *__restrict__ part, float *__restrict__ out, int64_t n, int64_t count,
                                  int64_t stride) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n) return;
    float v = 0.f;
    for (int64_t k = 0; k < count; ++k) v += part[k * stride + i];
    out[i] = v;
}
int sum_slices(const float *part, float *out, int64_t n, int64_t count, int64_t stride, cudaStream_t st) {
    if (!out || n == 0) return FMS_OK;
    if ((n + 127) / 128 > kMaxGrid) return FMS_ERR_TOO_LARGE;
    sum_slices_kernel<<<static_cast<unsigned>((n + 127) / 128), 128, 0, st>>>(part, out, n, count, stride);
    return check_launch();
}

template <typename S, bool ALIGNED>
int launch_ssm_forward(const fms_ssm_args *a, void *out, float *h_last, float *ck, cudaStream_t st) {
    const auto p = ssm_problem<S>(a, ssm_fwd_cw(a), fms::kSsmFwdWarps);
    const int64_t grid = p.batch * p.groups * p.chunks;
    if (grid > kMaxGrid) return FMS_ERR_TOO_LARGE;
    const size_t smem = ssm_fwd_smem(a, p.cw);
    if (int rc = allow_smem(fms::ssm_forward_kernel<S, ALIGNED>, smem)) return rc;
    fms::ssm_forward_kernel<S, ALIGNED><<<static_cast<unsigned>(grid), fms::kSsmFwdWarps * 32, smem, st>>>(
        p, static_cast<S *>(out), h_last, ck);
    return check_launch();
}

struct SsmScratch {
    size_t bc, a, d, total;
};
SsmScratch ssm_scratch(const fms_ssm_args *a) {
    const int64_t cw = ssm_bwd_cw(a), per = a->channels / a->groups;
    const int64_t chunks = (per + cw * fms::kSsmBwdWarps - 1) / (cw * fms::kSsmBwdWarps);
    const int64_t Tpad = (a->T + fms::kSsmTile - 1) / fms::kSsmTile * fms::kSsmTile;
    SsmScratch s;
    s.bc = round256(sizeof(float) * a->batch * a->groups * chunks * 2 * a->states * Tpad);
    s.a = round256(sizeof(float) * a->batch * a->channels * a->states);
    s.d = round256(sizeof(float) * a->batch * a->channels * 2);
    s.total = s.bc + s.a + s.d;
    return s;
}

template <typename S, bool ALIGNED>
int launch_ssm_backward(const fms_ssm_args *a, fms::SsmGrads<S> o, S *dB, S *dC, float *dA, float *dD, float *dbias,
                        char *ws, cudaStream_t st) {
    const auto p = ssm_problem<S>(a, ssm_bwd_cw(a), fms::kSsmBwdWarps);
    const SsmScratch sc = ssm_scratch(a);
    o.bc_part = reinterpret_cast<float *>(ws);
    o.a_part = reinterpret_cast<float *>(ws + sc.bc);
    o.d_part = reinterpret_cast<float *>(ws + sc.bc + sc.a);
    const int64_t grid = p.batch * p.groups * p.chunks, rows = p.batch * p.groups * 2 * p.N;
    if (grid > kMaxGrid || rows > kMaxGrid) return FMS_ERR_TOO_LARGE;
    const size_t smem = ssm_bwd_smem(a, p.cw);
    auto kernel = p.z ? fms::ssm_backward_kernel<S, ALIGNED, true> : fms::ssm_backward_kernel<S, ALIGNED, false>;
    if (int rc = allow_smem(kernel, smem)) return rc;
    kernel<<<static_cast<unsigned>(grid), fms::kSsmBwdWarps * 32, smem, st>>>(p, o);
    if (int rc = check_launch()) return rc;
    const int Tpad = p.tiles * fms::kSsmTile;
    const dim3 g2(static_cast<unsigned>(rows), static_cast<unsigned>(std::min((p.T + 255) / 256, 65535)));
    fms::ssm_bc_kernel<S><<<g2, 256, 0, st>>>(o.bc_part, dB, dC, p.groups, p.chunks, p.N, p.T, Tpad);
    if (int rc = check_launch()) return rc;
    if (int rc = sum_slices(o.a_part, dA, p.channels * p.N, p.batch, p.channels * p.N, st)) return rc;
    if (int rc = sum_slices(o.d_part, dD, p.channels, p.batch, 2 * p.channels, st)) return rc;
    return sum_slices(o.d_part + p.channels, dbias, p.channels, p.batch, 2 * p.channels, st);
}

template <typename S, bool VEC, int U>
int launch_ssm_step_u(const fms::SsmProblem<S> &p, float *state, int64_t pool, const int64_t *slots, void *out, int log_L,
                      cudaStream_t st) {
    const int per = 128 >> log_L;
    const dim3 grid(static_cast<unsigned>((p.per_group + per * U - 1) / (per * U)), static_cast<unsigned>(p.groups),
                    static_cast<unsigned>(std::min<int64_t>(p.batch, 65535)));
    const bool bc_vec = p.N % 8 == 0 && rows16(p.B, p.Bs, 2, sizeof(S)) && rows16(p.C, p.Cs, 2, sizeof(S));
    fms::ssm_step_kernel<S, VEC, U><<<grid, 128, 0, st>>>(p, state, pool, slots, static_cast<S *>(out), log_L, bc_vec);
    return check_launch();
}
template <typename S>
int launch_ssm_step(const fms_ssm_args *a, float *state, int64_t pool, const int64_t *slots, void *out, cudaStream_t st) {
    const auto p = ssm_problem<S>(a, 1, 1);
    if (p.groups > 65535) return FMS_ERR_TOO_LARGE;
    int log_L = 0;
    while (log_L < 5 && (8 << log_L) < p.N) ++log_L;
    const bool vec = p.N % 8 == 0 && aligned_to(state, 16) && aligned_to(p.A, 16);
    const bool many = (p.batch * p.channels << log_L) >= env_int("X_MANY", 148 * 1024);
    if (vec) return many ? launch_ssm_step_u<S, true, 2>(p, state, pool, slots, out, log_L, st)
                         : launch_ssm_step_u<S, true, 1>(p, state, pool, slots, out, log_L, st);
    return launch_ssm_step_u<S, false, 1>(p, state, pool, slots, out, log_L, st);
}

}  // namespace

namespace {
template <typename S>
int ssm_forward_t(const fms_ssm_args *a, void *out, float *h_last, float *ck, cudaStream_t st) {
    return ssm_aligned(a) && aligned_to(out, 16) ? launch_ssm_forward<S, true>(a, out, h_last, ck, st)
                                                 : launch_ssm_forward<S, false>(a, out, h_last, ck, st);
}
}  // namespace

FMS_EXPORT size_t fms_ssm_checkpoint_bytes(const fms_ssm_args *a) {
    if (ssm_check(a) != FMS_OK || ssm_empty(a)) return 0;
    return sizeof(float) * a->batch * a->channels * a->states * ((a->T + fms::kSsmTile - 1) / fms::kSsmTile);
}

FMS_EXPORT int fms_ssm_forward(const fms_ssm_args *a, void *out, float *h_last, float *checkpoints, fms_stream_t stream) {
    if (int rc = ssm_check(a)) return rc;
    if (ssm_empty(a)) return FMS_OK;
    if (int rc = ssm_pointers(a, a->T > 0)) return rc;
    if (a->T > 0 && !out) return FMS_ERR_NULL_POINTER;
    if (!aligned_to(out, elem_size(a->dtype)) || !aligned_to(h_last, 4) || !aligned_to(checkpoints, 4)) return FMS_ERR_MISALIGNED;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->T == 0) return copy_or_zero(a->h0, h_last, a->batch * a->channels * a->states, st);
    FMS_BY_TYPE(a->dtype, (ssm_forward_t<S>(a, out, h_last, checkpoints, st)));
}

FMS_EXPORT size_t fms_ssm_backward_workspace_bytes(const fms_ssm_args *a) {
    if (ssm_check(a) != FMS_OK || ssm_empty(a) || a->T == 0) return 0;
    return ssm_scratch(a).total;
}

FMS_EXPORT int fms_ssm_backward(const fms_ssm_args *a, const float *checkpoints, const void *grad_out,
                                const float *grad_last, void *grad_tokens, void *grad_delta, void *grad_z, void *grad_B,
                                void *grad_C, float *grad_A, float *grad_D, float *grad_delta_bias, float *grad_h0,
                                void *workspace, size_t workspace_bytes, fms_stream_t stream) {
    if (int rc = ssm_check(a)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t states = a->batch * a->channels * a->states;
    if (a->channels == 0) return FMS_OK;
    if (!grad_A) return FMS_ERR_NULL_POINTER;
    for (const float *p : {checkpoints, grad_last, static_cast<const float *>(grad_A), static_cast<const float *>(grad_D),
                           static_cast<const float *>(grad_delta_bias), static_cast<const float *>(grad_h0)})
        if (!aligned_to(p, 4)) return FMS_ERR_MISALIGNED;
    if (a->batch == 0 || a->T == 0) {  // nothing was read but h0, which went to the last state
        if (int rc = copy_or_zero(nullptr, grad_A, a->channels * a->states, st)) return rc;
        if (int rc = copy_or_zero(nullptr, grad_D, a->channels, st)) return rc;
        if (int rc = copy_or_zero(nullptr, grad_delta_bias, a->channels, st)) return rc;
        return copy_or_zero(grad_last, grad_h0, states, st);
    }
    if (int rc = ssm_pointers(a, true)) return rc;
    if (!checkpoints || !grad_out || !grad_tokens || !grad_delta || !grad_B || !grad_C || (a->z && !grad_z))
        return FMS_ERR_NULL_POINTER;
    const int64_t es = elem_size(a->dtype);
    bool all16 = ssm_aligned(a);
    for (const void *p : {grad_out, static_cast<const void *>(grad_tokens), static_cast<const void *>(grad_delta),
                          static_cast<const void *>(grad_z), static_cast<const void *>(grad_B), static_cast<const void *>(grad_C)}) {
        if (!aligned_to(p, es)) return FMS_ERR_MISALIGNED;
        all16 = all16 && aligned_to(p, 16);
    }
    if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < fms_ssm_backward_workspace_bytes(a))
        return FMS_ERR_WORKSPACE;
    auto go = [&](auto tag) -> int {
        using S = decltype(tag);
        fms::SsmGrads<S> o{};
        o.checkpoints = checkpoints;
        o.grad_out = static_cast<const S *>(grad_out);
        o.grad_last = grad_last;
        o.dx = static_cast<S *>(grad_tokens), o.ddelta = static_cast<S *>(grad_delta), o.dz = static_cast<S *>(grad_z);
        o.dh0 = grad_h0;
        auto *dB = static_cast<S *>(grad_B), *dC = static_cast<S *>(grad_C);
        char *ws = static_cast<char *>(workspace);
        return all16 ? launch_ssm_backward<S, true>(a, o, dB, dC, grad_A, grad_D, grad_delta_bias, ws, st)
                     : launch_ssm_backward<S, false>(a, o, dB, dC, grad_A, grad_D, grad_delta_bias, ws, st);
    };
    FMS_BY_TYPE(a->dtype, go(S{}));
}

FMS_EXPORT int fms_ssm_step(const fms_ssm_args *a, float *state, int64_t pool, const int64_t *slots, void *out,
                            fms_stream_t stream) {
    if (int rc = ssm_check(a)) return rc;
    if (a->T != 1 || pool < 0 || (!slots && pool < a->batch)) return FMS_ERR_BAD_SHAPE;
    if (!product_ok({pool, a->channels, a->states})) return FMS_ERR_BAD_SHAPE;
    if (ssm_empty(a)) return FMS_OK;
    if (int rc = ssm_pointers(a, true)) return rc;
    if (!out || (pool && !state)) return FMS_ERR_NULL_POINTER;
    if (!aligned_to(state, 4) || !aligned_to(slots, 8) || !aligned_to(out, elem_size(a->dtype))) return FMS_ERR_MISALIGNED;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    FMS_BY_TYPE(a->dtype, (launch_ssm_step<S>(a, state, pool, slots, out, st)));
}
