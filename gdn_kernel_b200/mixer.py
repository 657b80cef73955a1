"""Operators that stand around a recurrent block in a serving model: the short
causal convolution before it, the selective state space scan beside GDN, the
gated norm after it, and the residual add with the next block's norm.

Prompts are packed along one token axis and indexed by ``cu_seqlens``; the step
forms take one new token per sequence against a pool of states, as
``gdn_decode_pool`` does.  The ``gdn_*`` functions take all inputs, then the
pre-allocated outputs (torch CUDA tensors), check them (raising ``ValueError``)
and run on the current torch stream; the others allocate the outputs and return
them.  Checks and calls are in the TVM-FFI module ``libgdn_b200_tvm_mixer.so``
over the C ABI of ``libgdn_b200.so``: a decode step's operators take a few
microseconds each, which checks in Python alone would exceed.

Operands may be column slices of wider activations: what a row holds is
contiguous, the stride between rows is free.  States are contiguous pools.
``state_indices`` ([N] int32 or int64) names each sequence's slot, without it
sequence i has slot i.  A negative index is no slot: a prompt starts from zero
and stores no state, a step's entry is padding (zero output, no state touched).
States may be updated in place (``new_state`` being ``state``); slots of one
call are distinct.
"""

from __future__ import annotations

import os
import threading
import types
from typing import Optional

import torch

from . import _lib

_ACTIVATIONS = {None: _lib.ACT_NONE, "silu": _lib.ACT_SILU, "sigmoid": _lib.ACT_SIGMOID}
_FUNCTIONS = ("short_conv", "short_conv_step", "ssm_prefill_workspace", "ssm_prefill", "ssm_step",
              "gated_norm", "add_norm")

_lock = threading.Lock()
_ffi = None


def _load():
    """The TVM-FFI functions, loaded once; there is no fallback."""
    global _ffi
    with _lock:
        if _ffi is None:
            if not os.path.exists(_lib.TVM_MIXER_PATH):
                raise RuntimeError(f"{_lib.TVM_MIXER_PATH} is missing: build it with "
                                   "`python -m gdn_kernel_b200.build` (it needs tvm_ffi)")
            import tvm_ffi

            module = tvm_ffi.load_module(_lib.TVM_MIXER_PATH)
            _ffi = types.SimpleNamespace(**{name: module[name] for name in _FUNCTIONS})
    return _ffi


def _activation(name, allowed) -> int:
    if name not in allowed:
        raise ValueError(f"activation must be one of {allowed}, got {name!r}")
    return _ACTIVATIONS[name]


# ------------------------------------------------------------------ short convolution
def gdn_short_conv(x, weight, bias, state, cu_seqlens, output, new_state, *,
                   activation: Optional[str] = "silu", state_indices=None,
                   has_state=None) -> None:
    """Short causal convolution per channel over packed prompts.

    ``y_t = act(bias + sum_k weight[:, k] u[t - (W - 1) + k])``, ``u`` being a
    sequence's W - 1 carried rows, then its tokens; its last W - 1 rows are the
    new state.

    x, output: [T, D] bf16, fp16 or fp32 (not overlapping); weight: [D, W], W in
    2..4; bias: [D] or None; state: [P, W - 1, D] (oldest row first) or None
    (zero); new_state: [P, W - 1, D] (may be state); all of x's type.
    cu_seqlens: [N + 1] int32 or int64; state_indices: [N] or None; has_state:
    [N] bool or None, False for sequences that start from zero whatever their
    slot holds; activation: "silu" or None.
    """
    (_ffi or _load()).short_conv(x, weight, bias, state, cu_seqlens, output, new_state,
                                 state_indices, has_state, _activation(activation, (None, "silu")))


def gdn_short_conv_step(x, weight, bias, state_pool, state_indices, output, *,
                        activation: Optional[str] = "silu", new_state_pool=None) -> None:
    """The short convolution of one new token per sequence.

    x, output: [B, D] (output may be x); state_pool: [P, W - 1, D];
    state_indices: [B] or None (entry b has slot b); new_state_pool: where the
    new states go (default: state_pool, in place).  Otherwise as
    ``gdn_short_conv``.
    """
    (_ffi or _load()).short_conv_step(x, weight, bias, state_pool, state_indices, output,
                                      new_state_pool, _activation(activation, (None, "silu")))


def short_conv(x, weight, bias, state, cu_seqlens, *, activation: Optional[str] = "silu"):
    """Allocating short convolution of packed prompts: returns ``(output, new_state)``."""
    D, W = weight.shape
    output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    new_state = torch.empty((cu_seqlens.numel() - 1, W - 1, D), dtype=x.dtype, device=x.device)
    gdn_short_conv(x, weight, bias, state, cu_seqlens, output, new_state, activation=activation)
    return output, new_state


def short_conv_step(x, weight, bias, state_pool, state_indices=None, *,
                    activation: Optional[str] = "silu"):
    """Allocating step of the short convolution: returns the output; the states are
    updated in place."""
    output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    gdn_short_conv_step(x, weight, bias, state_pool, state_indices, output, activation=activation)
    return output


# ------------------------------------------------------------------ selective scan
def ssm_prefill_workspace_bytes(num_seqs: int, total_tokens: int, num_heads: int, head_dim: int,
                                state_dim: int) -> int:
    """Device workspace of ``gdn_ssm_prefill`` for this problem size (0: none is used)."""
    return (_ffi or _load()).ssm_prefill_workspace(num_seqs, total_tokens, num_heads, head_dim,
                                                   state_dim)


def gdn_ssm_prefill(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, output, new_state, *,
                    state_indices=None, has_state=None, workspace=None) -> None:
    """Selective state space scan over packed prompts.

    Per head, with the fp32 state h [P, N]: ``step = softplus(dt + dt_bias)``,
    ``h = exp(-exp(A_log) step) h + (step x) B^T``, ``y = h C + D x``.

    x: [T, H, P] bf16; dt: [T, H] bf16; B, C: [T, G, N] bf16 (head h reads group
    h // (H // G)), each with a free token stride of 16-byte multiples (dt: any);
    A_log: [H] fp32; D, dt_bias: [H] fp32 or None; P and N are 64 or 128;
    state: [S, H, P, N] fp32 or None (zero); output: [T, H, P] bf16 (not
    overlapping the inputs); new_state: [S, H, P, N] fp32 (may be state);
    cu_seqlens, state_indices, has_state as in ``gdn_short_conv``.  workspace: a
    uint8 CUDA tensor of at least ``ssm_prefill_workspace_bytes`` bytes
    (allocated here when omitted).

    A NaN or infinity in a token's x, or a NaN in its dt, can reach outputs of
    earlier tokens of its sequence in the same chunk of 128, as the products run
    over whole chunks.  Where decays have left nothing of a token (2^-300), a NaN
    or infinity of it may reach later tokens and the new state or not.
    """
    ffi = _ffi or _load()
    if workspace is None and x.dim() == 3 and B.dim() == 3:
        T, H, P = x.shape
        need = ffi.ssm_prefill_workspace(cu_seqlens.numel() - 1, T, H, P, B.shape[-1])
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    ffi.ssm_prefill(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, output, new_state,
                    state_indices, has_state, workspace)


def gdn_ssm_step(x, dt, A_log, B, C, D, dt_bias, state_pool, state_indices, output, *,
                 new_state_pool=None, output_state_indices=None) -> None:
    """The selective scan of one new token per sequence: x, output [B, H, P];
    dt [B, H]; B, C [B, G, N]; state_pool [S, H, P, N] fp32; state_indices [B] or
    None; new_state_pool: where the new states go (default: state_pool, in
    place); output_state_indices: their slots (default: the read slots).
    Otherwise as ``gdn_ssm_prefill``."""
    (_ffi or _load()).ssm_step(x, dt, A_log, B, C, D, dt_bias, state_pool, state_indices, output,
                               new_state_pool, output_state_indices)


def ssm_prefill(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens):
    """Allocating selective scan of packed prompts: returns ``(output, new_state)``."""
    T, H, P = x.shape
    output = torch.empty((T, H, P), dtype=x.dtype, device=x.device)
    new_state = torch.empty((cu_seqlens.numel() - 1, H, P, B.shape[2]), dtype=torch.float32,
                            device=x.device)
    gdn_ssm_prefill(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, output, new_state)
    return output, new_state


def ssm_step(x, dt, A_log, B, C, D, dt_bias, state_pool, state_indices=None):
    """Allocating step of the selective scan: returns the output; the states are
    updated in place."""
    output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    gdn_ssm_step(x, dt, A_log, B, C, D, dt_bias, state_pool, state_indices, output)
    return output


# ------------------------------------------------------------------ norms
def gdn_gated_norm(x, gate, weight, output, *, group_size: Optional[int] = None,
                   eps: float = 1e-6, activation: str = "silu", norm_first: bool = True) -> None:
    """The norm after a mixer, fused with its gate, by groups of a row.

    ``rms(v) = v / sqrt(mean(v^2) + eps)`` over each group; ``norm_first``:
    ``rms(x) * weight * act(gate)``, else ``rms(x * act(gate)) * weight``.

    x, gate, output: [T, D] or [T, H, P] bf16, fp16 or fp32 (gate may be None;
    output may be x or gate); group_size: a divisor of the row's width (default:
    the last dimension); weight: [group_size], shared by the groups, or one per
    element of a row, or None (ones), of x's type; activation: "silu" or
    "sigmoid".
    """
    if group_size is not None and group_size < 1:
        raise ValueError(f"group_size must be positive, got {group_size}")
    (_ffi or _load()).gated_norm(x, gate, weight, output, group_size or 0, eps,
                                 _activation(activation, ("silu", "sigmoid")),
                                 1 if norm_first else 0)


def gdn_add_norm(x, residual, weight, output, new_residual, *, block_weight=None, scale=1.0,
                 eps: float = 1e-6, weight_offset: float = 0.0) -> None:
    """Residual add of a block's output x and the norm before the next block.

    ``new_residual = residual + scale * u`` with ``u = x``, or
    ``rms(x) * block_weight`` (a norm after the block) where that is given;
    ``output = rms(new_residual) * (weight + weight_offset)``, from the sum
    before it is rounded.

    x, output: [T, D] bf16, fp16 or fp32 (output may be x); residual,
    new_residual: [T, D] of x's type or fp32 (may be the same); weight,
    block_weight: [D] of x's type; scale: a number, or an fp32 tensor [D] (a
    scale per channel).
    """
    channel_scale = None
    if isinstance(scale, torch.Tensor):
        channel_scale, scale = scale, 1.0
    (_ffi or _load()).add_norm(x, residual, weight, output, new_residual, block_weight,
                               channel_scale, scale, eps, weight_offset)


def gated_norm(x, gate, weight, *, group_size: Optional[int] = None, eps: float = 1e-6,
               activation: str = "silu", norm_first: bool = True):
    """Allocating gated norm: returns the output."""
    output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    gdn_gated_norm(x, gate, weight, output, group_size=group_size, eps=eps, activation=activation,
                   norm_first=norm_first)
    return output


def add_norm(x, residual, weight, *, block_weight=None, scale=1.0, eps: float = 1e-6,
             weight_offset: float = 0.0):
    """Allocating residual add and norm: returns ``(output, new_residual)``."""
    output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    new_residual = torch.empty(residual.shape, dtype=residual.dtype, device=x.device)
    gdn_add_norm(x, residual, weight, output, new_residual, block_weight=block_weight, scale=scale,
                 eps=eps, weight_offset=weight_offset)
    return output, new_residual
