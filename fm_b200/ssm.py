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

from .fm_scan import _load_ext

_ACTIVATIONS = {None: False, "silu": True}


def _silu(activation):
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError("activation must be None or 'silu'") from None


def ssm_scan(tokens, delta, A, B, C, D=None, z=None, delta_bias=None, initial_state=None, delta_softplus=False,
             lengths=None, return_state=False):
    """Selective state-space scan along the last axis; differentiable in every float argument.

    tokens, delta, z: (B, D, T) of one dtype     A: (D, N), finite     B, C: (B, N, T) or (B, G, N, T), N <= 256
    D, delta_bias: (D,)     initial_state: (B, D, N), zeros when omitted
    delta_softplus: the time step is log(1 + exp(delta + delta_bias)) instead of delta + delta_bias
    lengths: (B,) integer CUDA tensor for right-padded batches: what stands at positions from lengths[b] on
        (NaN included) is ignored, outputs and gradients there are zero, the state stops at lengths[b]

    return: out (B, D, T), and with ``return_state`` the last state (B, D, N) in fp32

    Sums run in a fixed order: equal calls give equal bits.  For the backward the inputs are kept, and the states
    in front of every 64th position (fp32, N / 16 bytes per element of tokens); the others are recomputed.  There
    is no second derivative.
    """
    return _load_ext().ssm_scan(tokens, delta, A, B, C, D, z, delta_bias, initial_state, delta_softplus, lengths, return_state)


def ssm_step(tokens, delta, state, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, slots=None):
    """One token of ``ssm_scan``: advances ``state`` in place and returns out (B, D).  No gradient.

    tokens, delta, z: (B, D)     B, C: (B, N) or (B, G, N)     state: (pool, D, N), contiguous fp32
    slots: (B,) integer CUDA tensor, row b's place in the pool (row b itself when omitted).  A row whose slot
        lies outside the pool (-1, say), or was named by an earlier row, is padding: its output is zero and
        it changes no state.
    """
    return _load_ext().ssm_step(tokens, delta, state, A, B, C, D, z, delta_bias, delta_softplus, slots)


def short_conv(tokens, weight, bias=None, initial_state=None, activation=None, lengths=None, return_state=False):
    """Depthwise causal filter along the last axis; differentiable in every float argument.

    tokens: (B, D, T)     weight: (D, K), 2 <= K <= 8, the last tap on the current position     bias: (D,)
    initial_state: (B, D, K-1) of the dtype of tokens, the inputs before position 0 (zeros when omitted)
    activation: None or "silu"     lengths: as in ``ssm_scan``

    return: out (B, D, T), and with ``return_state`` the last K-1 inputs (B, D, K-1)
    """
    return _load_ext().short_conv(tokens, weight, bias, initial_state, _silu(activation), lengths, return_state)


def short_conv_step(tokens, state, weight, bias=None, activation=None, slots=None):
    """One token of ``short_conv``: tokens (B, D), state (pool, D, K-1) of their dtype, contiguous, shifted in
    place; returns out (B, D).  ``slots`` as in ``ssm_step``.  No gradient."""
    return _load_ext().short_conv_step(tokens, state, weight, bias, _silu(activation), slots)
