// C ABI of the selective state-space scan (see include/fm_scan_b200.h): argument
// checks, launch shapes, launches.  No allocation, no synchronisation, no torch.
#include "fm_scan_b200.h"

#include <algorithm>

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

inline int padded_states(const fms_ssm_args *a) {
    return static_cast<int>((a->states + fms::kSsmNB - 1) / fms::kSsmNB * fms::kSsmNB);
}

// shared memory of a CTA: as the kernels lay it out
template <typename F>
size_t by_width(const fms_ssm_args *a, F f) { return a->dtype == FMS_F32 ? f(float{}) : f(__half{}); }
size_t ssm_fwd_smem(const fms_ssm_args *a, int cw) {
    return by_width(a, [&](auto t) {
        using S = decltype(t);
        return fms::ssm_bc_bytes<S>() + fms::kSsmFwdWarps * fms::ssm_fwd_warp_bytes<S>(cw, padded_states(a));
    });
}
size_t ssm_bwd_smem(const fms_ssm_args *a, int cw) {
    return sizeof(float) * fms::kSsmBwdWarps * 64 * 32 + by_width(a, [&](auto t) {
               using S = decltype(t);
               return fms::ssm_bc_bytes<S>() + fms::kSsmBwdWarps * fms::ssm_bwd_warp_bytes<S>(cw, padded_states(a));
           });
}
size_t ssm_carry_smem(const fms_ssm_args *a, int cw) {
    return by_width(a, [&](auto t) {
        using S = decltype(t);
        return fms::ssm_bc_bytes<S>() + fms::kSsmFwdWarps * fms::ssm_carry_warp_bytes<S>(cw, padded_states(a));
    });
}

// How the work is cut: channels of a warp, pieces of time.  More channels spread a tile's B, C and barriers
// over more work (and, backward, shrink the partial sums of their gradients); fewer, and more pieces of
// time, give more CTAs, but pieces cost a first pass over the data, a fold and two launches.  The cut with
// the least expected time is taken.  Measured on B200 (16-bit types, N = 16): a CTA's tile takes
// (channels of a warp + `own`) x `unit[n - 1]` microseconds with n CTAs on an SM; a cut time takes `again`
// as long, plus `fixed` for its launches.
struct CutCosts {
    int warps, per_sm;
    double own, unit[2], again, fixed;
};
constexpr CutCosts kFwdCosts{fms::kSsmFwdWarps, 2, 1.9, {0.55, 0.66}, 1.75, 12};
constexpr CutCosts kBwdCosts{fms::kSsmBwdWarps, 1, 1.5, {1.85, 1.85}, 1.4, 14};

struct SsmCut {
    int cw, segs, seg_tiles;
};
SsmCut best_cut(const fms_ssm_args *a, const CutCosts &k, size_t (*smem)(const fms_ssm_args *, int)) {
    const int64_t per = a->channels / a->groups, sms = 148;
    const int tiles = static_cast<int>((a->T + fms::kSsmTile - 1) / fms::kSsmTile);
    SsmCut best{1, 1, tiles};
    double least = 0;
    for (int cw = 1; cw <= 8; ++cw) {
        const size_t bytes = smem(a, cw);
        if (bytes > kMaxSmem) break;
        const int64_t ctas = a->batch * a->groups * ((per + cw * k.warps - 1) / (cw * k.warps));
        const int64_t most = std::min<int64_t>(k.per_sm, static_cast<int64_t>((kMaxSmem + 1024) / (bytes + 1024)));
        for (int waves = 0; waves <= 4; ++waves) {  // 0: time is not cut; else as many pieces as fill the waves
            int64_t segs = waves ? std::min<int64_t>(tiles, waves * most * sms / ctas) : 1;
            if (segs < (waves ? 2 : 1)) continue;
            const int64_t len = (tiles + segs - 1) / segs;
            segs = (tiles + len - 1) / len;
            const int64_t full = ctas * segs / (most * sms), rest = (ctas * segs - full * most * sms + sms - 1) / sms;
            double t = (full * k.unit[most - 1] + (rest ? k.unit[rest - 1] : 0)) * len * (cw + k.own);
            if (segs > 1) t = t * k.again + k.fixed;
            if (least == 0 || t < least) best = SsmCut{cw, static_cast<int>(segs), static_cast<int>(len)}, least = t;
        }
    }
    return best;
}
SsmCut ssm_fwd_cut(const fms_ssm_args *a) { return best_cut(a, kFwdCosts, ssm_fwd_smem); }
SsmCut ssm_bwd_cut(const fms_ssm_args *a) { return best_cut(a, kBwdCosts, ssm_bwd_smem); }

template <typename S>
fms::SsmProblem<S> ssm_problem(const fms_ssm_args *a, const SsmCut &cut, int warps) {
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
    p.cw = cut.cw;
    p.segs = cut.segs;
    p.seg_tiles = cut.seg_tiles;
    p.chunks = (p.per_group + p.cw * warps - 1) / (p.cw * warps);
    p.tiles = static_cast<int>((a->T + fms::kSsmTile - 1) / fms::kSsmTile);
    p.softplus = a->delta_softplus != 0;
    return p;
}

template <typename Kernel>
int allow_smem(Kernel kernel, size_t bytes) {
    return fms::record_cuda_error(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
}

// The first pass over pieces of time and the fold of what they leave; REVERSE for the adjoint.
// `carries`: (batch, segs, D, N), then the sums of time steps (batch, segs, D).
template <typename S, bool ALIGNED, bool REVERSE>
int launch_ssm_carries(const fms_ssm_args *a, const SsmCut &main, int warps, const S *grad_out, const float *first,
                       float *carries, float *sums, cudaStream_t st) {
    SsmCut cut = main;
    cut.cw = std::min(4, std::max(1, main.cw * warps / fms::kSsmFwdWarps / 2));
    while (cut.cw > 1 && ssm_carry_smem(a, cut.cw) > kMaxSmem) --cut.cw;
    const auto p = ssm_problem<S>(a, cut, fms::kSsmFwdWarps);
    const int64_t grid = p.batch * p.groups * p.chunks * p.segs, states = p.batch * p.channels * p.N;
    if (grid > kMaxGrid || (states + 127) / 128 > kMaxGrid) return FMS_ERR_TOO_LARGE;
    const size_t smem = ssm_carry_smem(a, cut.cw);
    if (int rc = allow_smem(fms::ssm_carry_kernel<S, ALIGNED, REVERSE>, smem)) return rc;
    fms::ssm_carry_kernel<S, ALIGNED, REVERSE><<<static_cast<unsigned>(grid), fms::kSsmFwdWarps * 32, smem, st>>>(
        p, grad_out, carries, sums);
    if (int rc = check_launch()) return rc;
    fms::ssm_fold_kernel<<<static_cast<unsigned>((states + 127) / 128), 128, 0, st>>>(
        carries, sums, p.A, first, p.batch, p.channels, p.N, p.segs, REVERSE);
    return check_launch();
}

size_t carry_floats(const fms_ssm_args *a, const SsmCut &cut) {  // of the states; the sums follow
    return cut.segs > 1 ? static_cast<size_t>(a->batch) * cut.segs * a->channels * a->states : 0;
}
size_t carry_bytes(const fms_ssm_args *a, const SsmCut &cut) {
    return cut.segs > 1 ? round256(sizeof(float) * (carry_floats(a, cut) + static_cast<size_t>(a->batch) * cut.segs * a->channels)) : 0;
}

template <typename S, bool ALIGNED>
int launch_ssm_forward(const fms_ssm_args *a, void *out, float *h_last, float *ck, float *ws, cudaStream_t st) {
    const SsmCut cut = ssm_fwd_cut(a);
    if (cut.segs > 1)
        if (int rc = launch_ssm_carries<S, ALIGNED, false>(a, cut, fms::kSsmFwdWarps, nullptr, a->h0, ws, ws + carry_floats(a, cut), st))
            return rc;
    const auto p = ssm_problem<S>(a, cut, fms::kSsmFwdWarps);
    const int64_t grid = p.batch * p.groups * p.chunks * p.segs;
    if (grid > kMaxGrid) return FMS_ERR_TOO_LARGE;
    const size_t smem = ssm_fwd_smem(a, p.cw);
    if (int rc = allow_smem(fms::ssm_forward_kernel<S, ALIGNED>, smem)) return rc;
    fms::ssm_forward_kernel<S, ALIGNED><<<static_cast<unsigned>(grid), fms::kSsmFwdWarps * 32, smem, st>>>(
        p, cut.segs > 1 ? ws : nullptr, static_cast<S *>(out), h_last, ck);
    return check_launch();
}

struct SsmScratch {
    size_t bc, a, d, carries, total;
};
SsmScratch ssm_scratch(const fms_ssm_args *a, const SsmCut &cut) {
    const int64_t per = a->channels / a->groups, chunks = (per + cut.cw * fms::kSsmBwdWarps - 1) / (cut.cw * fms::kSsmBwdWarps);
    const int64_t Tpad = (a->T + fms::kSsmTile - 1) / fms::kSsmTile * fms::kSsmTile;
    SsmScratch s;
    s.bc = round256(sizeof(float) * a->batch * a->groups * chunks * 2 * a->states * Tpad);
    s.a = round256(sizeof(float) * a->batch * cut.segs * a->channels * a->states);
    s.d = round256(sizeof(float) * a->batch * cut.segs * a->channels * 2);
    s.carries = carry_bytes(a, cut);
    s.total = s.bc + s.a + s.d + s.carries;
    return s;
}

template <typename S, bool ALIGNED>
int launch_ssm_backward(const fms_ssm_args *a, fms::SsmGrads<S> o, S *dB, S *dC, float *dA, float *dD, float *dbias,
                        char *ws, cudaStream_t st) {
    const SsmCut cut = ssm_bwd_cut(a);
    const auto p = ssm_problem<S>(a, cut, fms::kSsmBwdWarps);
    const SsmScratch sc = ssm_scratch(a, cut);
    o.bc_part = reinterpret_cast<float *>(ws);
    o.a_part = reinterpret_cast<float *>(ws + sc.bc);
    o.d_part = reinterpret_cast<float *>(ws + sc.bc + sc.a);
    const int64_t row_blocks = (p.T + 255) / 256, bc_blocks = p.batch * p.groups * 2 * p.N * row_blocks;
    const int64_t finish = bc_blocks + (p.channels * (p.N + 2) + 255) / 256;
    const int64_t grid = p.batch * p.groups * p.chunks * p.segs;
    if (grid > kMaxGrid || finish > kMaxGrid) return FMS_ERR_TOO_LARGE;
    if (cut.segs > 1) {
        float *carries = reinterpret_cast<float *>(ws + sc.bc + sc.a + sc.d);
        if (int rc = launch_ssm_carries<S, ALIGNED, true>(a, cut, fms::kSsmBwdWarps, o.grad_out, o.grad_last, carries,
                                                          carries + carry_floats(a, cut), st))
            return rc;
        o.carries = carries;
    }
    const size_t smem = ssm_bwd_smem(a, p.cw);
    auto kernel = p.z ? fms::ssm_backward_kernel<S, ALIGNED, true> : fms::ssm_backward_kernel<S, ALIGNED, false>;
    if (int rc = allow_smem(kernel, smem)) return rc;
    kernel<<<static_cast<unsigned>(grid), fms::kSsmBwdWarps * 32, smem, st>>>(p, o);
    if (int rc = check_launch()) return rc;
    fms::ssm_finish_kernel<S><<<static_cast<unsigned>(finish), 256, 0, st>>>(p, o, dB, dC, dA, dD, dbias, static_cast<unsigned>(bc_blocks),
                                                                            static_cast<int>(row_blocks));
    return check_launch();
}

template <typename S, bool VEC>
int launch_ssm_step_v(const fms::SsmProblem<S> &p, float *state, int64_t pool, const int64_t *slots, void *out, cudaStream_t st) {
    int log_L = 0;  // lanes of a channel: 8 states each
    while (log_L < 5 && (8 << log_L) < p.N) ++log_L;
    const int per = 128 >> log_L;
    const dim3 grid(static_cast<unsigned>((p.per_group + per - 1) / per), static_cast<unsigned>(p.groups),
                    static_cast<unsigned>(std::min<int64_t>(p.batch, 65535)));
    const bool bc_vec = p.N % 8 == 0 && rows16(p.B, p.Bs, 2, sizeof(S)) && rows16(p.C, p.Cs, 2, sizeof(S));
    fms::ssm_step_kernel<S, VEC><<<grid, 128, 0, st>>>(p, state, pool, slots, static_cast<S *>(out), log_L, bc_vec);
    return check_launch();
}
template <typename S>
int launch_ssm_step(const fms_ssm_args *a, float *state, int64_t pool, const int64_t *slots, void *out, cudaStream_t st) {
    const auto p = ssm_problem<S>(a, SsmCut{1, 1, 1}, 1);
    if (p.groups > 65535) return FMS_ERR_TOO_LARGE;
    return p.N % 8 == 0 && aligned_to(state, 16) && aligned_to(p.A, 16) ? launch_ssm_step_v<S, true>(p, state, pool, slots, out, st)
                                                                       : launch_ssm_step_v<S, false>(p, state, pool, slots, out, st);
}

}  // namespace

namespace {
template <typename S>
int ssm_forward_t(const fms_ssm_args *a, void *out, float *h_last, float *ck, float *ws, cudaStream_t st) {
    return ssm_aligned(a) && aligned_to(out, 16) ? launch_ssm_forward<S, true>(a, out, h_last, ck, ws, st)
                                                 : launch_ssm_forward<S, false>(a, out, h_last, ck, ws, st);
}
}  // namespace

FMS_EXPORT size_t fms_ssm_checkpoint_bytes(const fms_ssm_args *a) {
    if (ssm_check(a) != FMS_OK || ssm_empty(a)) return 0;
    return sizeof(float) * a->batch * a->channels * a->states * ((a->T + fms::kSsmTile - 1) / fms::kSsmTile);
}

FMS_EXPORT size_t fms_ssm_forward_workspace_bytes(const fms_ssm_args *a) {
    if (ssm_check(a) != FMS_OK || ssm_empty(a) || a->T == 0) return 0;
    return carry_bytes(a, ssm_fwd_cut(a));
}

FMS_EXPORT int fms_ssm_forward(const fms_ssm_args *a, void *out, float *h_last, float *checkpoints, void *workspace,
                               size_t workspace_bytes, fms_stream_t stream) {
    if (int rc = ssm_check(a)) return rc;
    if (ssm_empty(a)) return FMS_OK;
    if (int rc = ssm_pointers(a, a->T > 0)) return rc;
    if (a->T > 0 && !out) return FMS_ERR_NULL_POINTER;
    if (!aligned_to(out, elem_size(a->dtype)) || !aligned_to(h_last, 4) || !aligned_to(checkpoints, 4)) return FMS_ERR_MISALIGNED;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->T == 0) return copy_or_zero(a->h0, h_last, a->batch * a->channels * a->states, st);
    const size_t need = fms_ssm_forward_workspace_bytes(a);
    if (need && (!workspace || !aligned_to(workspace, 16) || workspace_bytes < need)) return FMS_ERR_WORKSPACE;
    FMS_BY_TYPE(a->dtype, (ssm_forward_t<S>(a, out, h_last, checkpoints, static_cast<float *>(workspace), st)));
}

FMS_EXPORT size_t fms_ssm_backward_workspace_bytes(const fms_ssm_args *a) {
    if (ssm_check(a) != FMS_OK || ssm_empty(a) || a->T == 0) return 0;
    return ssm_scratch(a, ssm_bwd_cut(a)).total;
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
