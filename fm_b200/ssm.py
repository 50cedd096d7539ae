"""The selective state-space layer's operators on (B, D, T) rows: the scan, the short causal filter in
front of it, and the one-token forms of both.

``ssm_scan`` is a scan like ``fm_scan`` whose decay depends on the input and on N states per channel:

    dt_t = delta_t (+ delta_bias, through log(1 + exp(.)))       h_t = exp(dt_t A) h_{t-1} + dt_t B_t x_t
    y_t  = sum_n C_t[n] h_t[n] + D x_t                           out = y * z * sigmoid(z)

``short_conv`` is the depthwise filter ``act(bias + sum_k weight[k] x_{t-K+1+k})``.  Both are
differentiable and carry a state in and out, so that ``ssm_step`` and ``short_conv_step`` continue a
prompt token by token on states kept in a pool.

Tensors over time are (B, D, T) (B and C: (B, N, T) or (B, G, N, T) with G groups of channels), fp32,
fp16 or bf16, any batch and channel strides; a tensor whose time axis is not the contiguous one is
copied first.  Parameters and scan states are fp32 (other float types are cast), arithmetic is fp32.
As for ``fm_scan``, there is no CPU implementation.  The reference has no such layer.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._nvtx import nvtx_range
from .fm_scan import _load_ext

_ACTIVATIONS = {None: False, "silu": True}


def _rows(t):
    """``t`` with a contiguous last axis."""
    return t if t is None or t.dim() == 0 or t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _f32(t):
    return t if t is None else t.to(torch.float32).contiguous()


def _index(t):
    return t if t is None or t.dtype != torch.int32 else t.to(torch.int64)


def _silu(activation):
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError("activation must be None or 'silu'") from None


def _no_grad_only(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or on detached tensors")


class SSM_Scan(torch.autograd.Function):
    """Autograd function of ``ssm_scan``.  Saved for backward: the inputs and the states in front of every
    64th position (fp32, N / 16 bytes per element of ``tokens``); the other states are recomputed."""

    @staticmethod
    def forward(ctx, tokens, delta, A, B, C, D, z, delta_bias, initial_state, lengths, softplus, want_state):
        with nvtx_range("ssm_scan.forward"):
            out, last, checkpoints = _load_ext().ssm_forward(
                tokens, delta, A, B, C, D, z, delta_bias, initial_state, lengths, softplus, want_state,
                any(ctx.needs_input_grad))
        ctx.save_for_backward(tokens, delta, A, B, C, D, z, delta_bias, initial_state, lengths, checkpoints)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return (out, last) if want_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out, g_last=None):
        tokens, delta, A, B, C, D, z, delta_bias, initial_state, lengths, checkpoints = ctx.saved_tensors
        g_out = torch.zeros(tokens.shape, dtype=tokens.dtype, device=tokens.device) if g_out is None else g_out.contiguous()
        with nvtx_range("ssm_scan.backward"):
            grads = _load_ext().ssm_backward(tokens, delta, A, B, C, D, z, delta_bias, initial_state, lengths, ctx.softplus,
                                             checkpoints, g_out, None if g_last is None else g_last.contiguous())
        return (*grads, None, None, None)


class Short_Conv(torch.autograd.Function):
    """Autograd function of ``short_conv``; saves its inputs and recomputes what stands before the activation."""

    @staticmethod
    def forward(ctx, tokens, weight, bias, initial_state, lengths, silu, want_state):
        with nvtx_range("short_conv.forward"):
            out, last = _load_ext().short_conv_forward(tokens, weight, bias, initial_state, lengths, silu, want_state)
        ctx.save_for_backward(tokens, weight, bias, initial_state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return (out, last) if want_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_out, g_last=None):
        tokens, weight, bias, initial_state, lengths = ctx.saved_tensors
        g_out = torch.zeros(tokens.shape, dtype=tokens.dtype, device=tokens.device) if g_out is None else g_out.contiguous()
        with nvtx_range("short_conv.backward"):
            grads = _load_ext().short_conv_backward(tokens, weight, bias, initial_state, lengths, ctx.silu, g_out,
                                                    None if g_last is None else g_last.contiguous())
        return (*grads, None, None, None)


def ssm_scan(tokens, delta, A, B, C, D=None, z=None, delta_bias=None, initial_state=None, delta_softplus=False,
             lengths=None, return_state=False):
    """Selective state-space scan along the last axis; differentiable in every float argument.

    tokens, delta, z: (B, D, T) of one dtype     A: (D, N), finite     B, C: (B, N, T) or (B, G, N, T), N <= 256
    D, delta_bias: (D,)     initial_state: (B, D, N), zeros when omitted
    delta_softplus: the time step is log(1 + exp(delta + delta_bias)) instead of delta + delta_bias
    lengths: (B,) integer CUDA tensor for right-padded batches: what stands at positions from lengths[b] on
        (NaN included) is ignored, outputs and gradients there are zero, the state stops at lengths[b]

    return: out (B, D, T), and with ``return_state`` the last state (B, D, N) in fp32

    Sums run in a fixed order: equal calls give equal bits.
    """
    return SSM_Scan.apply(_rows(tokens), _rows(delta), _f32(A), _rows(B), _rows(C), _f32(D), _rows(z), _f32(delta_bias),
                          _f32(initial_state), _index(lengths), bool(delta_softplus), bool(return_state))


def ssm_step(tokens, delta, state, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, slots=None):
    """One token of ``ssm_scan``: advances ``state`` in place and returns out (B, D).  No gradient.

    tokens, delta, z: (B, D)     B, C: (B, N) or (B, G, N)     state: (pool, D, N), contiguous fp32
    slots: (B,) integer CUDA tensor, row b's place in the pool (row b itself when omitted).  A row whose slot
        lies outside the pool (-1, say), or was named by an earlier row, is padding: its output is zero and
        it changes no state.
    """
    _no_grad_only("ssm_step", tokens, delta, state, A, B, C, D, z, delta_bias)
    return _load_ext().ssm_step(_rows(tokens), _rows(delta), state, _f32(A), _rows(B), _rows(C), _f32(D), _rows(z),
                                _f32(delta_bias), bool(delta_softplus), _index(slots))


def short_conv(tokens, weight, bias=None, initial_state=None, activation=None, lengths=None, return_state=False):
    """Depthwise causal filter along the last axis; differentiable in every float argument.

    tokens: (B, D, T)     weight: (D, K), 2 <= K <= 8, the last tap on the current position     bias: (D,)
    initial_state: (B, D, K-1) of the dtype of tokens, the inputs before position 0 (zeros when omitted)
    activation: None or "silu"     lengths: as in ``ssm_scan``

    return: out (B, D, T), and with ``return_state`` the last K-1 inputs (B, D, K-1)
    """
    return Short_Conv.apply(_rows(tokens), _f32(weight), _f32(bias),
                            None if initial_state is None else initial_state.contiguous(), _index(lengths),
                            _silu(activation), bool(return_state))


def short_conv_step(tokens, state, weight, bias=None, activation=None, slots=None):
    """One token of ``short_conv``: tokens (B, D), state (pool, D, K-1) of their dtype, contiguous, shifted in
    place; returns out (B, D).  ``slots`` as in ``ssm_step``.  No gradient."""
    _no_grad_only("short_conv_step", tokens, state, weight, bias)
    return _load_ext().short_conv_step(_rows(tokens), state, _f32(weight), _f32(bias), _silu(activation), _index(slots))
