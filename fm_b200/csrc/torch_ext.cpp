// Thin torch C++ extension over the C ABI (include/fm_scan_b200.h).
//
// It exports the two functions the reference binds into Python (fm/scan/fm_scan.py:8-16,34-35)
// with the same names, argument order and conventions:
//   at::Tensor fm_scan_forward (gates, tokens, initial_state, out)         fm/scan/fm_scan.cuh:344-358
//   void       fm_scan_backward(gates, outGrad, firstPropGrad, tokenGradOut,
//                               cached_output, input_tokens, gateGradOut)  fm/scan/fm_scan.cuh:361-381
// Every tensor, outputs included, is allocated by the caller; failures surface as c10::Error
// (RuntimeError in Python) exactly like the reference's TORCH_CHECKs.  Unlike the reference it
// installs a device guard, launches on the current stream of the tensors' device, and checks
// the launch.
//
// Layout: all big tensors are (B, D, T) -- one independent scan per (b, d) row -- or, when the
// output has one more axis than the gates, the reference's own FM layout
// gates (B,M,L) x tokens (B,D,L) -> states (B,M,D,L) with the 1 - gate token weight.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "fm_scan_b200.h"

namespace {

int dtype_tag(const at::Tensor &t) {
    switch (t.scalar_type()) {
        case at::ScalarType::Float: return FMS_F32;
        case at::ScalarType::Half: return FMS_F16;
        case at::ScalarType::BFloat16: return FMS_BF16;
        default:
            TORCH_CHECK(false, "Unsupported tensor dtype: expecting bfloat16, float16 or float32");
    }
}

void check_status(int rc, const char *what) {
    TORCH_CHECK(rc == FMS_OK, what, " failed: ", fms_status_string(rc), " (status ", rc,
                ", cuda error ", fms_last_cuda_error(), ")");
}

void check_big(const at::Tensor &t, const at::Tensor &like, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the dtype of gates");
    TORCH_CHECK(t.device() == like.device(), name, " must be on the device of gates");
    TORCH_CHECK(t.sizes() == like.sizes(), name, " must have the shape of gates");
}

// Per-row fp32 carry vector from an optional tensor of `rows` elements (any float dtype).
// Returns an fp32 contiguous tensor (possibly the argument itself) or an undefined tensor.
at::Tensor carry_f32(const c10::optional<at::Tensor> &t, int64_t rows, const at::Tensor &like,
                     const char *name) {
    if (!t.has_value() || !t->defined() || t->numel() == 0) return at::Tensor();
    TORCH_CHECK(t->is_cuda() && t->device() == like.device(), name, " must be on the device of gates");
    TORCH_CHECK(t->numel() == rows, name, " must have one element per row (", rows, "), got ",
                t->numel());
    return t->to(at::kFloat).contiguous();
}

const float *fptr(const at::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }


int64_t rows_of_shape(const at::Tensor &t) {
    int64_t r = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) r *= t.size(i);
    return r;
}

}  // namespace

// Forward.  gates, tokens, out: (..., T) of one dtype; initial_state: (...), None or empty (= zeros,
// which is what fm/scan/fm_scan.py:48 passes by default).  Returns `out`.
// FM mode (the reference's own shapes): gates (B,M,L), tokens (B,D,L), initial_state (B,M,D) or
// empty, out (B,M,D,L).  Selected when `out` has one more axis than `gates`.
static at::Tensor fm_mode_forward(const at::Tensor &gates, const at::Tensor &tokens,
                                  const c10::optional<at::Tensor> &initial_state, const at::Tensor &out) {
    TORCH_CHECK(gates.dim() == 3 && tokens.dim() == 3 && out.dim() == 4,
                "FM mode expects gates (B,M,L), tokens (B,D,L), out (B,M,D,L)");
    const int64_t B = gates.size(0), M = gates.size(1), L = gates.size(2), D = tokens.size(1);
    TORCH_CHECK(tokens.size(0) == B && tokens.size(2) == L, "tokens must be (B,D,L) with the B and L of gates");
    TORCH_CHECK(out.size(0) == B && out.size(1) == M && out.size(2) == D && out.size(3) == L,
                "out must be (B,M,D,L)");
    for (const at::Tensor *t : {&tokens, &out}) {
        TORCH_CHECK(t->is_cuda() && t->is_contiguous() && t->scalar_type() == gates.scalar_type() &&
                        t->device() == gates.device(),
                    "tokens and out must be contiguous CUDA tensors with the dtype and device of gates");
    }
    const int dtype = dtype_tag(gates);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, B * M * D, gates, "initial_state");
    check_status(fms_fm_forward(gates.data_ptr(), tokens.data_ptr(), fptr(h0), out.data_ptr(), B, M, D, L, dtype,
                                at::cuda::getCurrentCUDAStream().stream()),
                 "fm_scan_forward");
    return out;
}

at::Tensor fm_scan_forward(const at::Tensor &gates, const at::Tensor &tokens,
                           const c10::optional<at::Tensor> &initial_state, const at::Tensor &out) {
    TORCH_CHECK(gates.is_cuda(), "gates must be a CUDA tensor");
    TORCH_CHECK(gates.is_contiguous(), "gates must be contiguous");
    if (out.dim() == gates.dim() + 1) return fm_mode_forward(gates, tokens, initial_state, out);
    check_big(tokens, gates, "tokens");
    check_big(out, gates, "out");
    const int dtype = dtype_tag(gates);
    const int64_t rows = rows_of_shape(gates), T = gates.size(-1);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, rows, gates, "initial_state");
    auto stream = at::cuda::getCurrentCUDAStream().stream();
    // A handful of very long rows: cut them into segments so the whole GPU works (needs scratch).
    const size_t scratch = fms_plain_split_recommended(rows, T, dtype) ? fms_plain_split_workspace_bytes(rows, T, dtype) : 0;
    if (scratch > 0) {
        at::Tensor ws = at::empty({static_cast<int64_t>(scratch)}, gates.options().dtype(at::kByte));
        check_status(fms_plain_forward_split(gates.data_ptr(), tokens.data_ptr(), fptr(h0), out.data_ptr(),
                                             nullptr, rows, T, dtype, ws.data_ptr(), scratch, stream),
                     "fm_scan_forward");
        return out;
    }
    check_status(fms_plain_forward(gates.data_ptr(), tokens.data_ptr(), fptr(h0), out.data_ptr(),
                                   nullptr, rows, T, dtype, stream),
                 "fm_scan_forward");
    return out;
}

// Backward with every carry exposed.
//   carry_in           (...) or empty: a_T*delta_T entering from beyond the block (the reference's
//                      firstPropGrad, fm/scan/fm_scan.cuh:120-122)
//   initial_state      (...) or empty: the forward h0, i.e. h_{-1} for grad_gates at t = 0
//   grad_initial_state (...) fp32 or empty: receives dL/dh0
void fm_scan_backward_ex(const at::Tensor &gates, const at::Tensor &outGrad,
                         const c10::optional<at::Tensor> &carry_in, const at::Tensor &tokenGradOut,
                         const at::Tensor &cached_output, const at::Tensor &gateGradOut,
                         const c10::optional<at::Tensor> &initial_state,
                         const c10::optional<at::Tensor> &grad_initial_state_opt) {
    TORCH_CHECK(gates.is_cuda(), "gates must be a CUDA tensor");
    TORCH_CHECK(gates.is_contiguous(), "gates must be contiguous");
    check_big(outGrad, gates, "outGrad");
    check_big(cached_output, gates, "cached_output");
    check_big(tokenGradOut, gates, "tokenGradOut");
    check_big(gateGradOut, gates, "gateGradOut");
    const int dtype = dtype_tag(gates);
    const int64_t rows = rows_of_shape(gates), T = gates.size(-1);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor cin = carry_f32(carry_in, rows, gates, "firstPropGrad");
    at::Tensor h0 = carry_f32(initial_state, rows, gates, "initial_state");
    float *gh0 = nullptr;
    const at::Tensor grad_initial_state =
        grad_initial_state_opt.has_value() ? *grad_initial_state_opt : at::Tensor();
    if (grad_initial_state.defined() && grad_initial_state.numel() > 0) {
        TORCH_CHECK(grad_initial_state.is_cuda() && grad_initial_state.is_contiguous() &&
                        grad_initial_state.scalar_type() == at::kFloat &&
                        grad_initial_state.numel() == rows,
                    "grad_initial_state must be a contiguous fp32 CUDA tensor with one element per row");
        gh0 = grad_initial_state.data_ptr<float>();
    }
    auto stream = at::cuda::getCurrentCUDAStream().stream();
    const size_t scratch = fms_plain_split_recommended(rows, T, dtype) ? fms_plain_split_workspace_bytes(rows, T, dtype) : 0;
    if (scratch > 0) {
        at::Tensor ws = at::empty({static_cast<int64_t>(scratch)}, gates.options().dtype(at::kByte));
        check_status(fms_plain_backward_split(gates.data_ptr(), cached_output.data_ptr(), outGrad.data_ptr(),
                                              fptr(h0), fptr(cin), gateGradOut.data_ptr(),
                                              tokenGradOut.data_ptr(), gh0, rows, T, dtype, ws.data_ptr(),
                                              scratch, stream),
                     "fm_scan_backward");
        return;
    }
    check_status(fms_plain_backward(gates.data_ptr(), cached_output.data_ptr(), outGrad.data_ptr(),
                                    fptr(h0), fptr(cin), gateGradOut.data_ptr(),
                                    tokenGradOut.data_ptr(), gh0, rows, T, dtype, stream),
                 "fm_scan_backward");
}

// FM-mode backward.  tokenGradOut (B,D,L), gateGradOut (B,M,L): the reductions are fused -- the
// shapes the reference's Python reaches only after materialising two (B,M,D,L) tensors and summing
// them (fm/scan/fm_scan.py:70-78).  tokenGradOut, gateGradOut both (B,M,D,L): the reference's own
// contract, per-row terms for a caller that sums them itself.  initial_state is the forward h0;
// grad_initial_state (B,M,D) fp32.
void fm_scan_backward_fm(const at::Tensor &gates, const at::Tensor &outGrad, const at::Tensor &tokenGradOut,
                         const at::Tensor &cached_output, const at::Tensor &input_tokens,
                         const at::Tensor &gateGradOut, const c10::optional<at::Tensor> &initial_state,
                         const c10::optional<at::Tensor> &grad_initial_state_opt) {
    TORCH_CHECK(gates.is_cuda() && gates.is_contiguous() && gates.dim() == 3, "gates must be a contiguous CUDA (B,M,L) tensor");
    TORCH_CHECK(input_tokens.dim() == 3 && cached_output.dim() == 4, "expected tokens (B,D,L) and states (B,M,D,L)");
    const int64_t B = gates.size(0), M = gates.size(1), L = gates.size(2), D = input_tokens.size(1);
    auto same = [&](const at::Tensor &t, at::IntArrayRef shape, const char *name) {
        TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.scalar_type() == gates.scalar_type() &&
                        t.device() == gates.device() && t.sizes() == shape,
                    name, " must be a contiguous CUDA tensor of shape ", shape, " with the dtype of gates");
    };
    same(input_tokens, {B, D, L}, "input_tokens");
    same(cached_output, {B, M, D, L}, "cached_output");
    same(outGrad, {B, M, D, L}, "outGrad");
    // (B,M,D,L) outputs: the reference's own contract -- per-row terms, summed by the caller
    // (fm/scan/fm_scan.py:70-78); reduced shapes: the sums are fused into the kernel.
    const bool unreduced = tokenGradOut.dim() == 4 && gateGradOut.dim() == 4;
    if (unreduced) {
        same(tokenGradOut, {B, M, D, L}, "tokenGradOut");
        same(gateGradOut, {B, M, D, L}, "gateGradOut");
    } else {
        same(tokenGradOut, {B, D, L}, "tokenGradOut (fused reduction over M)");
        same(gateGradOut, {B, M, L}, "gateGradOut (fused reduction over D)");
    }
    const int dtype = dtype_tag(gates);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, B * M * D, gates, "initial_state");
    float *gh0 = nullptr;
    if (grad_initial_state_opt.has_value() && grad_initial_state_opt->defined() && grad_initial_state_opt->numel() > 0) {
        const at::Tensor &g = *grad_initial_state_opt;
        TORCH_CHECK(g.is_cuda() && g.is_contiguous() && g.scalar_type() == at::kFloat && g.numel() == B * M * D,
                    "grad_initial_state must be a contiguous fp32 CUDA tensor of B*M*D elements");
        gh0 = g.data_ptr<float>();
    }
    if (unreduced) {
        check_status(fms_fm_backward_unreduced(gates.data_ptr(), input_tokens.data_ptr(), cached_output.data_ptr(),
                                               outGrad.data_ptr(), fptr(h0), gateGradOut.data_ptr(),
                                               tokenGradOut.data_ptr(), gh0, B, M, D, L, dtype,
                                               at::cuda::getCurrentCUDAStream().stream()),
                     "fm_scan_backward");
        return;
    }
    const size_t scratch = fms_fm_backward_workspace_bytes(B, M, D, L, dtype);
    at::Tensor ws;
    if (scratch > 0) ws = at::empty({static_cast<int64_t>(scratch)}, gates.options().dtype(at::kByte));
    check_status(fms_fm_backward(gates.data_ptr(), input_tokens.data_ptr(), cached_output.data_ptr(),
                                 outGrad.data_ptr(), fptr(h0), gateGradOut.data_ptr(), tokenGradOut.data_ptr(),
                                 gh0, B, M, D, L, dtype, scratch ? ws.data_ptr() : nullptr, scratch,
                                 at::cuda::getCurrentCUDAStream().stream()),
                 "fm_scan_backward");
}

// Layer read-out without the states (inference): out (B,D,L) = sum_m weight * [rms-norm] * states.
// gates, weight (B,M,L); tokens, out (B,D,L); initial_state (B,M,D) or None.
void fm_memory_readout(const at::Tensor &gates, const at::Tensor &tokens, const at::Tensor &weight,
                       const c10::optional<at::Tensor> &initial_state, const at::Tensor &out, bool mem_norm,
                       double eps) {
    TORCH_CHECK(gates.is_cuda() && gates.is_contiguous() && gates.dim() == 3, "gates must be a contiguous CUDA (B,M,L) tensor");
    TORCH_CHECK(tokens.dim() == 3, "tokens must be (B,D,L)");
    const int64_t B = gates.size(0), M = gates.size(1), L = gates.size(2), D = tokens.size(1);
    auto same = [&](const at::Tensor &t, at::IntArrayRef shape, const char *name) {
        TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.scalar_type() == gates.scalar_type() &&
                        t.device() == gates.device() && t.sizes() == shape,
                    name, " must be a contiguous CUDA tensor of shape ", shape, " with the dtype of gates");
    };
    same(tokens, {B, D, L}, "tokens");
    same(weight, {B, M, L}, "weight");
    same(out, {B, D, L}, "out");
    const int dtype = dtype_tag(gates);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, B * M * D, gates, "initial_state");
    const size_t scratch = fms_fm_readout_workspace_bytes(B, M, D, L, dtype);
    at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(scratch, 16))}, gates.options().dtype(at::kByte));
    check_status(fms_fm_readout(gates.data_ptr(), tokens.data_ptr(), weight.data_ptr(), fptr(h0), out.data_ptr(), B,
                                M, D, L, dtype, mem_norm ? 1 : 0, static_cast<float>(eps), ws.data_ptr(), scratch,
                                at::cuda::getCurrentCUDAStream().stream()),
                 "fm_memory_readout");
}

// Training forward of the layer: writes out (B,D,L), the normalised states (B,M,D,L) and the norm
// factor rnorm (B,M,L) fp32 (ignored when mem_norm is false).
void fm_memory_forward_train(const at::Tensor &gates, const at::Tensor &tokens, const at::Tensor &weight,
                             const c10::optional<at::Tensor> &initial_state, const at::Tensor &out,
                             const at::Tensor &states_norm, const at::Tensor &rnorm, bool mem_norm, double eps) {
    TORCH_CHECK(gates.is_cuda() && gates.is_contiguous() && gates.dim() == 3 && tokens.dim() == 3,
                "gates must be a contiguous CUDA (B,M,L) tensor and tokens (B,D,L)");
    const int64_t B = gates.size(0), M = gates.size(1), L = gates.size(2), D = tokens.size(1);
    auto same = [&](const at::Tensor &t, at::IntArrayRef shape, const char *name) {
        TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.scalar_type() == gates.scalar_type() &&
                        t.device() == gates.device() && t.sizes() == shape,
                    name, " must be a contiguous CUDA tensor of shape ", shape, " with the dtype of gates");
    };
    same(tokens, {B, D, L}, "tokens");
    same(weight, {B, M, L}, "weight");
    same(out, {B, D, L}, "out");
    same(states_norm, {B, M, D, L}, "states_norm");
    TORCH_CHECK(rnorm.is_cuda() && rnorm.is_contiguous() && rnorm.scalar_type() == at::kFloat &&
                    rnorm.numel() == B * M * L, "rnorm must be a contiguous fp32 CUDA tensor of B*M*L elements");
    const int dtype = dtype_tag(gates);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, B * M * D, gates, "initial_state");
    const size_t scratch = fms_fm_readout_workspace_bytes(B, M, D, L, dtype);
    at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(scratch, 16))}, gates.options().dtype(at::kByte));
    check_status(fms_fm_layer_forward(gates.data_ptr(), tokens.data_ptr(), weight.data_ptr(), fptr(h0), out.data_ptr(),
                                      states_norm.data_ptr(), rnorm.data_ptr<float>(), B, M, D, L, dtype,
                                      mem_norm ? 1 : 0, static_cast<float>(eps), ws.data_ptr(), scratch,
                                      at::cuda::getCurrentCUDAStream().stream()),
                 "fm_memory_forward");
}

// Training backward of the layer.  grad_states_norm: None when the returned states were not used.
void fm_memory_backward(const at::Tensor &gates, const at::Tensor &tokens, const at::Tensor &weight,
                        const at::Tensor &states_norm, const at::Tensor &rnorm, bool mem_norm,
                        const at::Tensor &grad_out, const c10::optional<at::Tensor> &grad_states_norm,
                        const c10::optional<at::Tensor> &initial_state, const at::Tensor &d_gates,
                        const at::Tensor &d_tokens, const at::Tensor &d_weight,
                        const c10::optional<at::Tensor> &d_initial_state) {
    TORCH_CHECK(gates.is_cuda() && gates.is_contiguous() && gates.dim() == 3 && tokens.dim() == 3,
                "gates must be a contiguous CUDA (B,M,L) tensor and tokens (B,D,L)");
    const int64_t B = gates.size(0), M = gates.size(1), L = gates.size(2), D = tokens.size(1);
    auto same = [&](const at::Tensor &t, at::IntArrayRef shape, const char *name) {
        TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.scalar_type() == gates.scalar_type() &&
                        t.device() == gates.device() && t.sizes() == shape,
                    name, " must be a contiguous CUDA tensor of shape ", shape, " with the dtype of gates");
    };
    same(tokens, {B, D, L}, "tokens");
    same(weight, {B, M, L}, "weight");
    same(states_norm, {B, M, D, L}, "states_norm");
    same(grad_out, {B, D, L}, "grad_out");
    same(d_gates, {B, M, L}, "d_gates");
    same(d_tokens, {B, D, L}, "d_tokens");
    same(d_weight, {B, M, L}, "d_weight");
    const void *ext = nullptr;
    if (grad_states_norm.has_value() && grad_states_norm->defined()) {
        same(*grad_states_norm, {B, M, D, L}, "grad_states_norm");
        ext = grad_states_norm->data_ptr();
    }
    const float *rn = nullptr;
    if (mem_norm) {
        TORCH_CHECK(rnorm.is_cuda() && rnorm.is_contiguous() && rnorm.scalar_type() == at::kFloat &&
                        rnorm.numel() == B * M * L, "rnorm must be a contiguous fp32 CUDA tensor of B*M*L elements");
        rn = rnorm.data_ptr<float>();
    }
    float *gh0 = nullptr;
    if (d_initial_state.has_value() && d_initial_state->defined() && d_initial_state->numel() > 0) {
        TORCH_CHECK(d_initial_state->is_cuda() && d_initial_state->is_contiguous() &&
                        d_initial_state->scalar_type() == at::kFloat && d_initial_state->numel() == B * M * D,
                    "d_initial_state must be a contiguous fp32 CUDA tensor of B*M*D elements");
        gh0 = d_initial_state->data_ptr<float>();
    }
    const int dtype = dtype_tag(gates);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, B * M * D, gates, "initial_state");
    const size_t scratch = fms_fm_layer_backward_workspace_bytes(B, M, D, L, dtype);
    at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(scratch, 16))}, gates.options().dtype(at::kByte));
    check_status(fms_fm_layer_backward(gates.data_ptr(), tokens.data_ptr(), weight.data_ptr(), states_norm.data_ptr(),
                                       rn, grad_out.data_ptr(), ext, fptr(h0), d_gates.data_ptr(), d_tokens.data_ptr(),
                                       d_weight.data_ptr(), gh0, B, M, D, L, dtype, ws.data_ptr(), scratch,
                                       at::cuda::getCurrentCUDAStream().stream()),
                 "fm_memory_backward");
}

// Channel-last layout: gates, tokens, out (B, T, D); initial_state (B, D) or None.
at::Tensor fm_scan_btd_forward(const at::Tensor &gates, const at::Tensor &tokens,
                               const c10::optional<at::Tensor> &initial_state, const at::Tensor &out) {
    TORCH_CHECK(gates.is_cuda() && gates.is_contiguous() && gates.dim() == 3, "gates must be a contiguous CUDA (B,T,D) tensor");
    check_big(tokens, gates, "tokens");
    check_big(out, gates, "out");
    const int64_t B = gates.size(0), T = gates.size(1), D = gates.size(2);
    const int dtype = dtype_tag(gates);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, B * D, gates, "initial_state");
    const size_t scratch = fms_btd_workspace_bytes(B, T, D, dtype);
    at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(scratch, 16))}, gates.options().dtype(at::kByte));
    check_status(fms_btd_forward(gates.data_ptr(), tokens.data_ptr(), fptr(h0), out.data_ptr(), nullptr, B, T, D, dtype,
                                 ws.data_ptr(), scratch, at::cuda::getCurrentCUDAStream().stream()),
                 "fm_scan_forward (B,T,D)");
    return out;
}

void fm_scan_btd_backward(const at::Tensor &gates, const at::Tensor &outGrad, const at::Tensor &tokenGradOut,
                          const at::Tensor &cached_output, const at::Tensor &gateGradOut,
                          const c10::optional<at::Tensor> &initial_state,
                          const c10::optional<at::Tensor> &grad_initial_state) {
    TORCH_CHECK(gates.is_cuda() && gates.is_contiguous() && gates.dim() == 3, "gates must be a contiguous CUDA (B,T,D) tensor");
    check_big(outGrad, gates, "outGrad");
    check_big(cached_output, gates, "cached_output");
    check_big(tokenGradOut, gates, "tokenGradOut");
    check_big(gateGradOut, gates, "gateGradOut");
    const int64_t B = gates.size(0), T = gates.size(1), D = gates.size(2);
    const int dtype = dtype_tag(gates);
    const c10::cuda::CUDAGuard guard(gates.device());
    at::Tensor h0 = carry_f32(initial_state, B * D, gates, "initial_state");
    float *gh0 = nullptr;
    if (grad_initial_state.has_value() && grad_initial_state->defined() && grad_initial_state->numel() > 0) {
        TORCH_CHECK(grad_initial_state->is_cuda() && grad_initial_state->is_contiguous() &&
                        grad_initial_state->scalar_type() == at::kFloat && grad_initial_state->numel() == B * D,
                    "grad_initial_state must be a contiguous fp32 CUDA tensor of B*D elements");
        gh0 = grad_initial_state->data_ptr<float>();
    }
    const size_t scratch = fms_btd_workspace_bytes(B, T, D, dtype);
    at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(scratch, 16))}, gates.options().dtype(at::kByte));
    check_status(fms_btd_backward(gates.data_ptr(), cached_output.data_ptr(), outGrad.data_ptr(), fptr(h0),
                                  gateGradOut.data_ptr(), tokenGradOut.data_ptr(), gh0, B, T, D, dtype, ws.data_ptr(),
                                  scratch, at::cuda::getCurrentCUDAStream().stream()),
                 "fm_scan_backward (B,T,D)");
}

// Backward with the reference's seven arguments.  firstPropGrad seeds the reverse scan
// (fm/scan/fm_scan.cuh:120-122); the reference passes zeros (fm/scan/fm_scan.py:65).
// input_tokens is accepted for signature compatibility and not read: with the token weight
// dropped, grad_gates_t = delta_t * h_{t-1} needs no tokens.  h_{-1} is taken as zero, which is
// what the reference's call amounts to (its h_{-1} is firstPropGrad = zeros,
// fm/scan/fm_scan.cuh:195-196).
void fm_scan_backward(const at::Tensor &gates, const at::Tensor &outGrad,
                      const c10::optional<at::Tensor> &firstPropGrad, const at::Tensor &tokenGradOut,
                      const at::Tensor &cached_output, const c10::optional<at::Tensor> &input_tokens,
                      const at::Tensor &gateGradOut) {
    if (cached_output.dim() == gates.dim() + 1) {  // FM mode, h_{-1} = 0; outputs reduced or (B,M,D,L)
        TORCH_CHECK(input_tokens.has_value() && input_tokens->defined(), "FM mode needs input_tokens");
        fm_scan_backward_fm(gates, outGrad, tokenGradOut, cached_output, *input_tokens, gateGradOut,
                            c10::nullopt, c10::nullopt);
        return;
    }
    fm_scan_backward_ex(gates, outGrad, firstPropGrad, tokenGradOut, cached_output, gateGradOut,
                        c10::nullopt, c10::nullopt);
}

// ------------------------------------------------------------ selective state-space layer ----
// Outputs are allocated here, on the tensors' device and the current stream's pool.

using OptTensor = c10::optional<at::Tensor>;

static bool given(const OptTensor &t) { return t.has_value() && t->defined(); }

static void want_rows(const at::Tensor &t, const at::Tensor &like, at::IntArrayRef shape, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), name, " must be on the device of tokens");
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the dtype of tokens");
    TORCH_CHECK(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
    TORCH_CHECK(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, name, " must have a contiguous last axis");
}

static const float *want_f32(const OptTensor &t, const at::Tensor &like, at::IntArrayRef shape, const char *name) {
    if (!given(t)) return nullptr;
    TORCH_CHECK(t->is_cuda() && t->device() == like.device(), name, " must be a CUDA tensor on the device of tokens");
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous(), name, " must be contiguous float32");
    TORCH_CHECK(t->sizes() == shape, name, " must have shape ", shape, ", got ", t->sizes());
    return t->data_ptr<float>();
}

static const int64_t *want_index(const OptTensor &t, const at::Tensor &like, int64_t n, const char *name) {
    if (!given(t)) return nullptr;
    TORCH_CHECK(t->is_cuda() && t->device() == like.device(), name, " must be a CUDA tensor on the device of tokens");
    TORCH_CHECK(t->scalar_type() == at::kLong && t->is_contiguous() && t->dim() == 1 && t->size(0) == n, name,
                " must be a contiguous integer tensor with one element per sequence (", n, ")");
    return t->data_ptr<int64_t>();
}

static void strides_of(const at::Tensor &t, int n, int64_t *to) {
    for (int i = 0; i < n; ++i) to[i] = t.stride(i);
}

// Fills args from the tensors of a scan (time: last axis) or, with step, of one token (no time axis).
static fms_ssm_args ssm_args(const at::Tensor &x, const at::Tensor &delta, const at::Tensor &A, const at::Tensor &B,
                             const at::Tensor &C, const OptTensor &D, const OptTensor &z, const OptTensor &bias,
                             const OptTensor &h0, const OptTensor &lengths, bool softplus, bool step) {
    const char *shape = step ? "(B, D)" : "(B, D, T)";
    const int axes = step ? 2 : 3;
    TORCH_CHECK(x.is_cuda(), "tokens must be a CUDA tensor (there is no CPU path)");
    TORCH_CHECK(x.dim() == axes, "tokens must be ", shape);
    TORCH_CHECK(A.dim() == 2, "A must be (D, N)");
    TORCH_CHECK(B.dim() == axes || B.dim() == axes + 1, "B must be ", step ? "(B, N) or (B, G, N)" : "(B, N, T) or (B, G, N, T)");
    fms_ssm_args a{};
    a.batch = x.size(0), a.channels = x.size(1), a.T = step ? 1 : x.size(2);
    a.states = A.size(1);
    const bool grouped = B.dim() == axes + 1;
    a.groups = grouped ? B.size(1) : 1;
    TORCH_CHECK(a.groups >= 1 && a.channels % a.groups == 0, "the groups of B must divide the channels");
    TORCH_CHECK(a.states >= 1 && a.states <= FMS_SSM_MAX_STATES, "A must have 1 to ", FMS_SSM_MAX_STATES, " states");
    a.dtype = dtype_tag(x);
    a.delta_softplus = softplus;
    std::vector<int64_t> rows = {a.batch, a.channels}, bc = {a.batch};
    if (grouped) bc.push_back(a.groups);
    bc.push_back(a.states);
    if (!step) rows.push_back(a.T), bc.push_back(a.T);
    want_rows(x, x, rows, "tokens");
    want_rows(delta, x, rows, "delta");
    want_rows(B, x, bc, "B");
    want_rows(C, x, bc, "C");
    a.tokens = x.data_ptr(), a.delta = delta.data_ptr(), a.B = B.data_ptr(), a.C = C.data_ptr();
    strides_of(x, 2, a.tokens_stride);
    strides_of(delta, 2, a.delta_stride);
    if (given(z)) {
        want_rows(*z, x, rows, "z");
        a.z = z->data_ptr();
        strides_of(*z, 2, a.z_stride);
    }
    auto bc_strides = [&](const at::Tensor &t, int64_t *to) {
        to[0] = t.stride(0);
        to[1] = grouped ? t.stride(1) : 0;
        to[2] = t.stride(grouped ? 2 : 1);
    };
    bc_strides(B, a.B_stride);
    bc_strides(C, a.C_stride);
    a.A = want_f32(A, x, {a.channels, a.states}, "A");
    a.D = want_f32(D, x, {a.channels}, "D");
    a.delta_bias = want_f32(bias, x, {a.channels}, "delta_bias");
    a.h0 = want_f32(h0, x, {a.batch, a.channels, a.states}, "initial_state");
    a.lengths = want_index(lengths, x, a.batch, "lengths");
    return a;
}

static std::tuple<at::Tensor, OptTensor, OptTensor> ssm_forward(
    const at::Tensor &x, const at::Tensor &delta, const at::Tensor &A, const at::Tensor &B, const at::Tensor &C,
    const OptTensor &D, const OptTensor &z, const OptTensor &bias, const OptTensor &h0, const OptTensor &lengths,
    bool softplus, bool want_last, bool want_checkpoints) {
    const fms_ssm_args a = ssm_args(x, delta, A, B, C, D, z, bias, h0, lengths, softplus, false);
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options());
    OptTensor last, ck;
    if (want_last) last = at::empty({a.batch, a.channels, a.states}, A.options());
    if (want_checkpoints) ck = at::empty({static_cast<int64_t>(fms_ssm_checkpoint_bytes(&a) / 4)}, A.options());
    const size_t scratch = fms_ssm_forward_workspace_bytes(&a);
    at::Tensor ws;
    if (scratch) ws = at::empty({static_cast<int64_t>(scratch)}, x.options().dtype(at::kByte));
    check_status(fms_ssm_forward(&a, out.data_ptr(), want_last ? last->data_ptr<float>() : nullptr,
                                 want_checkpoints ? ck->data_ptr<float>() : nullptr, scratch ? ws.data_ptr() : nullptr, scratch,
                                 at::cuda::getCurrentCUDAStream().stream()),
                 "ssm_scan");
    return {out, last, ck};
}

// grads of tokens, delta, A, B, C, D, z, delta_bias, initial_state (None where the input is)
static std::vector<OptTensor> ssm_backward(
    const at::Tensor &x, const at::Tensor &delta, const at::Tensor &A, const at::Tensor &B, const at::Tensor &C,
    const OptTensor &D, const OptTensor &z, const OptTensor &bias, const OptTensor &h0, const OptTensor &lengths,
    bool softplus, const OptTensor &checkpoints, const at::Tensor &grad_out, const OptTensor &grad_last) {
    const fms_ssm_args a = ssm_args(x, delta, A, B, C, D, z, bias, h0, lengths, softplus, false);
    const c10::cuda::CUDAGuard guard(x.device());
    want_rows(grad_out, x, x.sizes(), "grad_out");
    TORCH_CHECK(grad_out.is_contiguous(), "grad_out must be contiguous");
    TORCH_CHECK(given(checkpoints), "the forward kept no states for a backward");
    const float *gl = want_f32(grad_last, x, {a.batch, a.channels, a.states}, "grad_last");
    at::Tensor dx = at::empty(x.sizes(), x.options()), dd = at::empty(x.sizes(), x.options());
    at::Tensor dA = at::empty(A.sizes(), A.options()), dB = at::empty(B.sizes(), x.options()), dC = at::empty(C.sizes(), x.options());
    OptTensor dD, dz, db, dh;
    if (given(D)) dD = at::empty(D->sizes(), D->options());
    if (given(z)) dz = at::empty(x.sizes(), x.options());
    if (given(bias)) db = at::empty(bias->sizes(), bias->options());
    if (given(h0)) dh = at::empty(h0->sizes(), h0->options());
    const size_t scratch = fms_ssm_backward_workspace_bytes(&a);
    at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(scratch, 16))}, x.options().dtype(at::kByte));
    auto f = [](const OptTensor &t) { return given(t) ? t->data_ptr<float>() : nullptr; };
    check_status(fms_ssm_backward(&a, f(checkpoints), grad_out.data_ptr(), gl, dx.data_ptr(), dd.data_ptr(),
                                  given(z) ? dz->data_ptr() : nullptr, dB.data_ptr(), dC.data_ptr(), dA.data_ptr<float>(),
                                  f(dD), f(db), f(dh), ws.data_ptr(), scratch, at::cuda::getCurrentCUDAStream().stream()),
                 "ssm_scan backward");
    return {dx, dd, dA, dB, dC, dD, dz, db, dh};
}

static at::Tensor ssm_step(const at::Tensor &x, const at::Tensor &delta, const at::Tensor &state, const at::Tensor &A,
                           const at::Tensor &B, const at::Tensor &C, const OptTensor &D, const OptTensor &z,
                           const OptTensor &bias, bool softplus, const OptTensor &slots) {
    const fms_ssm_args a = ssm_args(x, delta, A, B, C, D, z, bias, c10::nullopt, c10::nullopt, softplus, true);
    TORCH_CHECK(state.dim() == 3, "state must be (pool, D, N)");
    const float *st = want_f32(state, x, {state.size(0), a.channels, a.states}, "state");
    const int64_t *at_ = want_index(slots, x, a.batch, "slots");
    TORCH_CHECK(at_ || !(a.batch > state.size(0)), "state must hold one state per row when slots is omitted");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options());
    check_status(fms_ssm_step(&a, const_cast<float *>(st), state.size(0), at_, out.data_ptr(),
                              at::cuda::getCurrentCUDAStream().stream()),
                 "ssm_step");
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return out;
}

static fms_conv_args conv_args(const at::Tensor &x, const at::Tensor &weight, const OptTensor &bias, const OptTensor &x0,
                               const OptTensor &lengths, bool silu, bool step) {
    TORCH_CHECK(x.is_cuda(), "tokens must be a CUDA tensor (there is no CPU path)");
    TORCH_CHECK(x.dim() == (step ? 2 : 3), "tokens must be ", step ? "(B, D)" : "(B, D, T)");
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) >= 2 && weight.size(1) <= 8, "weight must be (D, K) with 2 to 8 taps");
    fms_conv_args a{};
    a.batch = x.size(0), a.channels = x.size(1), a.T = step ? 1 : x.size(2), a.taps = weight.size(1);
    a.dtype = dtype_tag(x);
    a.silu = silu;
    want_rows(x, x, x.sizes(), "tokens");
    a.tokens = x.data_ptr();
    strides_of(x, 2, a.tokens_stride);
    a.weight = want_f32(weight, x, {a.channels, a.taps}, "weight");
    a.bias = want_f32(bias, x, {a.channels}, "bias");
    if (given(x0)) {
        want_rows(*x0, x, {a.batch, a.channels, a.taps - 1}, "initial_state");
        TORCH_CHECK(x0->is_contiguous(), "initial_state must be contiguous");
        a.x0 = x0->data_ptr();
    }
    a.lengths = want_index(lengths, x, a.batch, "lengths");
    return a;
}

static std::tuple<at::Tensor, OptTensor> short_conv_forward(const at::Tensor &x, const at::Tensor &weight, const OptTensor &bias,
                                                            const OptTensor &x0, const OptTensor &lengths, bool silu,
                                                            bool want_last) {
    const fms_conv_args a = conv_args(x, weight, bias, x0, lengths, silu, false);
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options());
    OptTensor last;
    if (want_last) last = at::empty({a.batch, a.channels, a.taps - 1}, x.options());
    check_status(fms_conv_forward(&a, out.data_ptr(), want_last ? last->data_ptr() : nullptr,
                                  at::cuda::getCurrentCUDAStream().stream()),
                 "short_conv");
    return {out, last};
}

// grads of tokens, weight, bias, initial_state (None where the input is)
static std::vector<OptTensor> short_conv_backward(const at::Tensor &x, const at::Tensor &weight, const OptTensor &bias,
                                                  const OptTensor &x0, const OptTensor &lengths, bool silu,
                                                  const at::Tensor &grad_out, const OptTensor &grad_last) {
    const fms_conv_args a = conv_args(x, weight, bias, x0, lengths, silu, false);
    const c10::cuda::CUDAGuard guard(x.device());
    want_rows(grad_out, x, x.sizes(), "grad_out");
    TORCH_CHECK(grad_out.is_contiguous(), "grad_out must be contiguous");
    const void *gl = nullptr;
    if (given(grad_last)) {
        want_rows(*grad_last, x, {a.batch, a.channels, a.taps - 1}, "grad_last");
        TORCH_CHECK(grad_last->is_contiguous(), "grad_last must be contiguous");
        gl = grad_last->data_ptr();
    }
    at::Tensor dx = at::empty(x.sizes(), x.options()), dw = at::empty(weight.sizes(), weight.options());
    OptTensor db, d0;
    if (given(bias)) db = at::empty(bias->sizes(), bias->options());
    if (given(x0)) d0 = at::empty(x0->sizes(), x0->options());
    const size_t scratch = fms_conv_backward_workspace_bytes(&a);
    at::Tensor ws = at::empty({static_cast<int64_t>(std::max<size_t>(scratch, 16))}, x.options().dtype(at::kByte));
    check_status(fms_conv_backward(&a, grad_out.data_ptr(), gl, dx.data_ptr(), dw.data_ptr<float>(),
                                   given(bias) ? db->data_ptr<float>() : nullptr, given(x0) ? d0->data_ptr() : nullptr,
                                   ws.data_ptr(), scratch, at::cuda::getCurrentCUDAStream().stream()),
                 "short_conv backward");
    return {dx, dw, db, d0};
}

static at::Tensor short_conv_step(const at::Tensor &x, const at::Tensor &state, const at::Tensor &weight, const OptTensor &bias,
                                  bool silu, const OptTensor &slots) {
    const fms_conv_args a = conv_args(x, weight, bias, c10::nullopt, c10::nullopt, silu, true);
    TORCH_CHECK(state.dim() == 3, "state must be (pool, D, K-1)");
    want_rows(state, x, {state.size(0), a.channels, a.taps - 1}, "state");
    TORCH_CHECK(state.is_contiguous(), "state must be contiguous");
    const int64_t *at_ = want_index(slots, x, a.batch, "slots");
    TORCH_CHECK(at_ || !(a.batch > state.size(0)), "state must hold one state per row when slots is omitted");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options());
    check_status(fms_conv_step(&a, state.data_ptr(), state.size(0), at_, out.data_ptr(),
                               at::cuda::getCurrentCUDAStream().stream()),
                 "short_conv_step");
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return out;
}

// ---- what Python calls: casts, copies of strided tensors and autograd are done here, where they cost less
// than in Python.

// a tensor with a contiguous last axis; parameters in fp32; indexes in int64
static at::Tensor rows_of(const at::Tensor &t) {
    return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
static OptTensor rows_of(const OptTensor &t) { return given(t) ? OptTensor(rows_of(*t)) : OptTensor(); }
static at::Tensor fp32_of(const at::Tensor &t) {
    if (t.scalar_type() == at::kFloat && t.is_contiguous()) return t;
    TORCH_CHECK(t.is_floating_point(), "parameters and states must be floating point");
    return t.to(at::kFloat).contiguous();
}
static OptTensor fp32_of(const OptTensor &t) { return given(t) ? OptTensor(fp32_of(*t)) : OptTensor(); }
static OptTensor index_of(const OptTensor &t) {
    return given(t) && t->scalar_type() == at::kInt ? OptTensor(t->to(at::kLong)) : t;
}
static bool needs(const at::Tensor &t) { return t.requires_grad(); }
static bool needs(const OptTensor &t) { return given(t) && t->requires_grad(); }
template <typename... Ts>
static bool wants_grad(const Ts &...ts) {
    return at::GradMode::is_enabled() && (needs(ts) || ...);
}
static at::Tensor value(const OptTensor &t) { return given(t) ? *t : at::Tensor(); }
static OptTensor maybe(const at::Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients that cannot be differentiated again: when a graph of the backward is asked for, going
// through it raises.
static variable_list first_order(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (const at::Tensor &g : grads)
        if (g.defined()) some.push_back(g);
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative",
                                                                 static_cast<int64_t>(some.size()));
    for (at::Tensor &g : some) g.requires_grad_(true);
    some = (*error)(std::move(some));
    size_t k = 0;
    for (at::Tensor &g : grads)
        if (g.defined()) g = some[k++];
    return grads;
}

// Saved for backward: the inputs and the states in front of every 64th position; the others are recomputed.
struct SsmScan : torch::autograd::Function<SsmScan> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &delta, const at::Tensor &A,
                                 const at::Tensor &B, const at::Tensor &C, const OptTensor &D, const OptTensor &z,
                                 const OptTensor &bias, const OptTensor &h0, const OptTensor &lengths, bool softplus,
                                 bool want_last) {
        auto [out, last, ck] = ssm_forward(x, delta, A, B, C, D, z, bias, h0, lengths, softplus, want_last, true);
        ctx->save_for_backward({x, delta, A, B, C, value(D), value(z), value(bias), value(h0), value(lengths), *ck});
        ctx->saved_data["softplus"] = softplus;
        ctx->set_materialize_grads(false);
        if (want_last) return {out, *last};
        return {out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        variable_list r;
        {
            const at::AutoGradMode off(false);
            const at::Tensor up = g[0].defined() ? g[0].contiguous() : at::zeros(s[0].sizes(), s[0].options());
            const OptTensor last = g.size() > 1 && g[1].defined() ? OptTensor(g[1].contiguous()) : OptTensor();
            for (const OptTensor &t : ssm_backward(s[0], s[1], s[2], s[3], s[4], maybe(s[5]), maybe(s[6]), maybe(s[7]), maybe(s[8]),
                                                   maybe(s[9]), ctx->saved_data["softplus"].toBool(), s[10], up, last))
                r.push_back(value(t));
        }
        r = first_order(std::move(r), "ssm_scan");
        r.resize(12);
        return r;
    }
};

static py::object ssm_scan(const at::Tensor &tokens, const at::Tensor &delta, const at::Tensor &A, const at::Tensor &B,
                           const at::Tensor &C, const OptTensor &D, const OptTensor &z, const OptTensor &bias,
                           const OptTensor &initial_state, bool softplus, const OptTensor &lengths, bool want_last) {
    const at::Tensor x_ = rows_of(tokens), d_ = rows_of(delta), A_ = fp32_of(A), B_ = rows_of(B), C_ = rows_of(C);
    const OptTensor D_ = fp32_of(D), z_ = rows_of(z), b_ = fp32_of(bias), h_ = fp32_of(initial_state), n_ = index_of(lengths);
    at::Tensor out;
    OptTensor last;
    if (wants_grad(x_, d_, A_, B_, C_, D_, z_, b_, h_)) {
        const variable_list r = SsmScan::apply(x_, d_, A_, B_, C_, D_, z_, b_, h_, n_, softplus, want_last);
        out = r[0];
        if (want_last) last = r[1];
    } else {
        std::tie(out, last, std::ignore) = ssm_forward(x_, d_, A_, B_, C_, D_, z_, b_, h_, n_, softplus, want_last, false);
    }
    if (want_last) return py::make_tuple(out, *last);
    return py::cast(out);
}

// Saved for backward: the inputs; what stands before the activation is recomputed.
struct ShortConv : torch::autograd::Function<ShortConv> {
    static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const OptTensor &bias,
                                 const OptTensor &x0, const OptTensor &lengths, bool silu, bool want_last) {
        auto [out, last] = short_conv_forward(x, weight, bias, x0, lengths, silu, want_last);
        ctx->save_for_backward({x, weight, value(bias), value(x0), value(lengths)});
        ctx->saved_data["silu"] = silu;
        ctx->set_materialize_grads(false);
        if (want_last) return {out, *last};
        return {out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        variable_list r;
        {
            const at::AutoGradMode off(false);
            const at::Tensor up = g[0].defined() ? g[0].contiguous() : at::zeros(s[0].sizes(), s[0].options());
            const OptTensor last = g.size() > 1 && g[1].defined() ? OptTensor(g[1].contiguous()) : OptTensor();
            for (const OptTensor &t : short_conv_backward(s[0], s[1], maybe(s[2]), maybe(s[3]), maybe(s[4]),
                                                          ctx->saved_data["silu"].toBool(), up, last))
                r.push_back(value(t));
        }
        r = first_order(std::move(r), "short_conv");
        r.resize(7);
        return r;
    }
};

static py::object short_conv(const at::Tensor &tokens, const at::Tensor &weight, const OptTensor &bias,
                             const OptTensor &initial_state, bool silu, const OptTensor &lengths, bool want_last) {
    const at::Tensor x_ = rows_of(tokens), w_ = fp32_of(weight);
    const OptTensor b_ = fp32_of(bias), n_ = index_of(lengths);
    const OptTensor i_ = given(initial_state) ? OptTensor(initial_state->contiguous()) : OptTensor();
    at::Tensor out;
    OptTensor last;
    if (wants_grad(x_, w_, b_, i_)) {
        const variable_list r = ShortConv::apply(x_, w_, b_, i_, n_, silu, want_last);
        out = r[0];
        if (want_last) last = r[1];
    } else {
        std::tie(out, last) = short_conv_forward(x_, w_, b_, i_, n_, silu, want_last);
    }
    if (want_last) return py::make_tuple(out, *last);
    return py::cast(out);
}

static at::Tensor ssm_step_op(const at::Tensor &x, const at::Tensor &delta, const at::Tensor &state, const at::Tensor &A,
                              const at::Tensor &B, const at::Tensor &C, const OptTensor &D, const OptTensor &z,
                              const OptTensor &bias, bool softplus, const OptTensor &slots) {
    TORCH_CHECK(!wants_grad(x, delta, state, A, B, C, D, z, bias),
                "ssm_step has no gradient: call it under torch.no_grad() or on detached tensors");
    return ssm_step(rows_of(x), rows_of(delta), state, fp32_of(A), rows_of(B), rows_of(C), fp32_of(D), rows_of(z), fp32_of(bias),
                    softplus, index_of(slots));
}

static at::Tensor short_conv_step_op(const at::Tensor &x, const at::Tensor &state, const at::Tensor &weight, const OptTensor &bias,
                                     bool silu, const OptTensor &slots) {
    TORCH_CHECK(!wants_grad(x, state, weight, bias),
                "short_conv_step has no gradient: call it under torch.no_grad() or on detached tensors");
    return short_conv_step(rows_of(x), state, fp32_of(weight), fp32_of(bias), silu, index_of(slots));
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "fm_scan for B200: torch shim over the C ABI libfm_scan_b200.so";
    m.def("fm_scan_forward", &fm_scan_forward, "scan forward (writes and returns out)");
    m.def("fm_scan_backward", &fm_scan_backward, "scan backward, reference signature");
    m.def("fm_scan_backward_ex", &fm_scan_backward_ex, "scan backward with h0 / carry_in / grad_h0");
    m.def("fm_scan_backward_fm", &fm_scan_backward_fm, "FM-mode backward with fused reductions");
    m.def("fm_scan_btd_forward", &fm_scan_btd_forward, "scan forward on (B,T,D) tensors");
    m.def("fm_scan_btd_backward", &fm_scan_btd_backward, "scan backward on (B,T,D) tensors");
    m.def("fm_memory_forward_train", &fm_memory_forward_train, "layer forward: output + normalised states");
    m.def("fm_memory_backward", &fm_memory_backward, "layer backward with the state gradient generated in-kernel");
    m.def("fm_memory_readout", &fm_memory_readout, "layer read-out without materialising the states");
    m.def("ssm_scan", &ssm_scan, "state-space scan, differentiable: out or (out, last state)");
    m.def("ssm_step", &ssm_step_op, "state-space scan of one token, states advanced in place");
    m.def("short_conv", &short_conv, "causal filter, differentiable: out or (out, last inputs)");
    m.def("short_conv_step", &short_conv_step_op, "causal filter of one token, state shifted in place");
    m.def("ssm_forward", &ssm_forward, "state-space scan forward: out, last state, checkpoints");
    m.def("ssm_backward", &ssm_backward, "state-space scan backward: gradients of every input");
    m.def("short_conv_forward", &short_conv_forward, "causal filter forward: out, last inputs");
    m.def("short_conv_backward", &short_conv_backward, "causal filter backward: gradients of every input");
    m.def("abi_version", []() { return fms_version(); });
}
