"""The recurrent layer of a state-space prediction network: a short causal convolution and a selective scan, for whole
sequences (with backward) and for single tokens.

They stand where the reference's prediction network has its LSTM (src/decoder/decoder.py:5-44): label sequences in
training, one token per emission in decoding, the state carried by the caller as the ``hidden`` of
src/rnnt/model.py:145-165.  Entry points ``rnnt_causal_conv_*`` and ``rnnt_selective_scan_*`` (include/rnnt_mi355.h)
through the compiled binding; kernels in ``csrc/state_space_mi355.hip``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _torch_binding

_ACTIVATIONS = {"silu": True, None: False}


def _silu(activation) -> bool:
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be 'silu' or None")
    return _ACTIVATIONS[activation]


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                activation: Optional[str] = "silu") -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution over time with one filter per channel: ``(y [B, L, dim], final_state [B, width - 1, dim])``.

    ``p[t] = bias + sum_k weight[:, k] * xe[t + k]`` over ``xe = [initial_state; x]``, ``y = p * sigmoid(p)`` (or ``p``).
    ``final_state`` is the last ``width - 1`` rows of ``xe`` up to the sequence's length: the ``initial_state`` of what
    follows, and the ``state`` of :func:`causal_conv_step`.  Differentiable in ``x``, ``weight``, ``bias`` and
    ``initial_state``, from both results (once, and not in forward mode).

    Args:
        x: ``[B, L, dim]`` fp32, bf16 or fp16; rows may lie apart (half of a projection's output), channels adjacent.
        weight, bias: ``[dim, width]`` (width 2, 3 or 4) and ``[dim]``, fp32.
        initial_state: ``[B, width - 1, dim]`` in ``x``'s type; None: zeros.
        lengths: int32 ``[B]`` on the device; rows from ``lengths[b]`` on are not read, and zero in ``y`` and in the
            gradient.  Values are clamped to ``[0, L]``.
    """
    return _torch_binding.load().causal_conv(x, weight, bias, initial_state, lengths, _silu(activation))


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     activation: Optional[str] = "silu",
                     state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`causal_conv` of one token per sequence: ``x [B, dim]``, ``state [B, width - 1, dim]`` -> ``(y [B, dim], new
    state)``.  ``state`` stays as it is unless it is also passed as ``state_out``.  No backward: what requires grad
    (``state_out`` too) is refused in grad mode."""
    return _torch_binding.load().causal_conv_step(x, state, weight, bias, _silu(activation), state_out)


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, initial_state: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selective state space scan: ``(y [B, L, dim], final_state [B, dim, state] fp32)``.

    ``delta = softplus(dt + dt_bias)``; ``h[t] = exp(delta A) h[t-1] + delta x[t] B[t]``; ``y[t] = (<C[t], h[t]> + D x[t])
    * z[t] sigmoid(z[t])`` (without ``z``: no factor).  Differentiable in every floating argument, from both results (once, and not in forward mode); the
    backward reads the state before every 16th step, kept in fp32 (``4 state / 16`` bytes per element of ``x``).

    Args:
        x, dt, z: ``[B, L, dim]`` fp32, bf16 or fp16, one type; rows may lie apart, channels adjacent.
        B, C: ``[B, L, state]`` in the same type, shared by all channels; rows may lie apart (parts of one projection).
        A: ``[dim, state]`` fp32 (negative in a stable layer), 8, 16 or 32 states.
        D, dt_bias: ``[dim]`` fp32.
        initial_state: ``[B, dim, state]`` fp32; None: zeros.
        lengths: int32 ``[B]`` on the device; rows from ``lengths[b]`` on are not read, and zero in ``y`` and the gradients;
            a length of 0 gives back the initial state.  Values are clamped to ``[0, L]``.
    """
    return _torch_binding.load().selective_scan(x, dt, A, B, C, D, z, dt_bias, initial_state, lengths)


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None,
                        state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`selective_scan` of one token per sequence: ``x``, ``dt``, ``z`` ``[B, dim]``, ``B``, ``C`` ``[B, state]``,
    ``state [B, dim, state]`` fp32 -> ``(y [B, dim], new state)``.  ``state`` stays as it is unless it is also passed as
    ``state_out``.  No backward: what requires grad (``state_out`` too) is refused in grad mode."""
    return _torch_binding.load().selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, state_out)
