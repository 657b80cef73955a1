"""Operators that stand around a recurrent block in a serving model: the short
causal convolution before it, the selective state space scan beside GDN, the
gated norm after it, and the residual add with the next block's norm.

Prompts are packed along one token axis and indexed by ``cu_seqlens``; the step
forms take one new token per sequence against a pool of states, as
``gdn_decode_pool`` does.  The ``gdn_*`` functions take all inputs, then the
pre-allocated outputs (torch CUDA tensors), check them (raising ``ValueError``)
and call the C ABI of ``libgdn_b200.so`` on the current torch stream; the others
allocate the outputs and return them.

Operands may be column slices of wider activations: what a row holds is
contiguous, the stride between rows is free.  States are contiguous pools.
``state_indices`` ([N] int32 or int64) names each sequence's slot, without it
sequence i has slot i.  A negative index is no slot: a prompt starts from zero
and stores no state, a step's entry is padding (zero output, no state touched).
States may be updated in place (``new_state`` being ``state``); slots of one
call are distinct.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
_ACTIVATIONS = {None: _lib.ACT_NONE, "silu": _lib.ACT_SILU, "sigmoid": _lib.ACT_SIGMOID}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _refuse(msg: str):
    raise ValueError(msg)


def _device(t, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(f"{name} must be a CUDA tensor")
    return t.device


def _dtype_code(t, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse(f"{name}: expected bfloat16, float16 or float32, got {t.dtype}")
    return code


def _activation(name, allowed) -> int:
    if name not in allowed:
        _refuse(f"activation must be one of {allowed}, got {name!r}")
    return _ACTIVATIONS[name]


def _full(t, name: str, dtype, shape, dev) -> int:
    """Address of a contiguous tensor of this type and shape (0 for None)."""
    if t is None:
        return 0
    if (not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != dev
            or t.shape != shape or not t.is_contiguous()):
        _explain(t, name, dtype, shape, dev, "contiguous")
    return t.data_ptr()


def _rows(t, name: str, dtype, shape, dev):
    """Address and row stride of [rows, ...] whose rows are each contiguous."""
    if (not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != dev
            or t.shape != shape):
        _explain(t, name, dtype, shape, dev, "contiguous within a row")
    strides, want = t.stride(), 1
    for size, stride in zip(reversed(shape[1:]), reversed(strides[1:])):
        if stride != want and size != 1:
            if t.numel() == 0:
                break
            _explain(t, name, dtype, shape, dev, "contiguous within a row")
        want *= size
    return t.data_ptr(), (strides[0] if shape[0] > 1 else want)


def _explain(t, name, dtype, shape, dev, layout):
    if not isinstance(t, torch.Tensor):
        _refuse(f"{name}: expected a torch.Tensor")
    if t.dtype != dtype:
        _refuse(f"{name}: expected {dtype}, got {t.dtype}")
    if t.device != dev:
        _refuse(f"{name}: must be on {dev}, got {t.device}")
    if tuple(t.shape) != tuple(shape):
        _refuse(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    _refuse(f"{name}: must be {layout}")


def _index(t, name: str, n: int, dev):
    """Address and int64 flag of an [n] index tensor (0 for None)."""
    if t is None:
        return 0, 0
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        _refuse(f"{name} must be an int32 or int64 tensor")
    return _full(t, name, t.dtype, (n,), dev), 1 if t.dtype == torch.int64 else 0


def _offsets(cu, dev):
    if not isinstance(cu, torch.Tensor) or cu.dim() != 1 or cu.numel() < 1:
        _refuse("cu_seqlens must be [N + 1]")
    n = cu.numel() - 1
    ptr, is64 = _index(cu, "cu_seqlens", n + 1, dev)
    return n, ptr, is64


def _flags(t, n: int, dev) -> int:
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.bool, torch.uint8):
        _refuse("has_state must be a bool or uint8 tensor")
    return _full(t, "has_state", t.dtype, (n,), dev)


def _pool_rows(t, name: str, tail, dev, dtype):
    if not isinstance(t, torch.Tensor) or t.dim() != len(tail) + 1:
        _refuse(f"{name} must have {len(tail) + 1} dimensions")
    return _full(t, name, dtype, (t.shape[0], *tail), dev), t.shape[0]


def _need_slots(pool: int, n: int, indices) -> None:
    if indices is None and pool < n:
        _refuse(f"the states hold {pool} rows, {n} are needed")


def _call(dev, fn, *args) -> None:
    """One C call with ``dev`` current, on its current torch stream (last argument)."""
    index = dev.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index) if _raw_stream else
                torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        _lib.check(rc)


# ------------------------------------------------------------------ short convolution
def _conv_weight(x, weight, bias, dev):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        _refuse("weight must be [channels, width]")
    channels, width = weight.shape
    if not 2 <= width <= 4:
        _refuse(f"weight: width must be 2, 3 or 4, got {width}")
    return (channels, width, _full(weight, "weight", x.dtype, (channels, width), dev),
            _full(bias, "bias", x.dtype, (channels,), dev))


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
    dev = _device(x, "x")
    code = _dtype_code(x, "x")
    act = _activation(activation, (None, "silu"))
    D, W, w_ptr, b_ptr = _conv_weight(x, weight, bias, dev)
    if x.dim() != 2:
        _refuse("x must be [T, channels]")
    T = x.shape[0]
    n, cu_ptr, cu64 = _offsets(cu_seqlens, dev)
    x_ptr, x_stride = _rows(x, "x", x.dtype, (T, D), dev)
    o_ptr, o_stride = _rows(output, "output", x.dtype, (T, D), dev)
    ns_ptr, pool = _pool_rows(new_state, "new_state", (W - 1, D), dev, x.dtype)
    s_ptr = _full(state, "state", x.dtype, (pool, W - 1, D), dev)
    i_ptr, i64 = _index(state_indices, "state_indices", n, dev)
    _need_slots(pool, n, state_indices)
    _call(dev, _lib.load().gdn_b200_short_conv, x_ptr, x_stride, w_ptr, b_ptr, s_ptr, cu_ptr,
          cu64, i_ptr, i64, _flags(has_state, n, dev), act, o_ptr, o_stride, ns_ptr, n, T, pool,
          D, W, code)


def gdn_short_conv_step(x, weight, bias, state_pool, state_indices, output, *,
                        activation: Optional[str] = "silu", new_state_pool=None) -> None:
    """The short convolution of one new token per sequence.

    x, output: [B, D] (output may be x); state_pool: [P, W - 1, D];
    state_indices: [B] or None (entry b has slot b); new_state_pool: where the
    new states go (default: state_pool, in place).  Otherwise as
    ``gdn_short_conv``.
    """
    dev = _device(x, "x")
    code = _dtype_code(x, "x")
    act = _activation(activation, (None, "silu"))
    D, W, w_ptr, b_ptr = _conv_weight(x, weight, bias, dev)
    if x.dim() != 2:
        _refuse("x must be [B, channels]")
    B = x.shape[0]
    x_ptr, x_stride = _rows(x, "x", x.dtype, (B, D), dev)
    o_ptr, o_stride = _rows(output, "output", x.dtype, (B, D), dev)
    s_ptr, pool = _pool_rows(state_pool, "state_pool", (W - 1, D), dev, x.dtype)
    ns_ptr = (s_ptr if new_state_pool is None else
              _full(new_state_pool, "new_state_pool", x.dtype, (pool, W - 1, D), dev))
    i_ptr, i64 = _index(state_indices, "state_indices", B, dev)
    _need_slots(pool, B, state_indices)
    _call(dev, _lib.load().gdn_b200_short_conv_step, x_ptr, x_stride, w_ptr, b_ptr, s_ptr, i_ptr,
          i64, act, o_ptr, o_stride, ns_ptr, B, pool, D, W, code)


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
def _scan_operands(x, dt, A_log, B, C, D, dt_bias, output, dev):
    if x.dim() != 3 or not isinstance(B, torch.Tensor) or B.dim() != 3:
        _refuse("x must be [T, H, P] and B [T, G, N]")
    T, H, P = x.shape
    G, N = B.shape[1:]
    if P not in (64, 128) or N not in (64, 128):
        _refuse(f"head_dim and state_dim must be 64 or 128, got {P} and {N}")
    if H < 1 or G < 1 or H % G:
        _refuse(f"num_heads must be a multiple of num_groups, got {H} and {G}")
    bf = torch.bfloat16
    args = (*_rows(x, "x", bf, (T, H, P), dev), *_rows(dt, "dt", bf, (T, H), dev),
            _full(A_log, "A_log", torch.float32, (H,), dev),
            *_rows(B, "B", bf, (T, G, N), dev), *_rows(C, "C", bf, (T, G, N), dev),
            _full(D, "D", torch.float32, (H,), dev),
            _full(dt_bias, "dt_bias", torch.float32, (H,), dev))
    if A_log is None:
        _refuse("A_log: expected a torch.Tensor")
    if output is None:
        _refuse("output: expected a torch.Tensor")
    return T, H, P, G, N, args, _full(output, "output", bf, (T, H, P), dev)


def ssm_prefill_workspace_bytes(num_seqs: int, total_tokens: int, num_heads: int, head_dim: int,
                                state_dim: int) -> int:
    """Device workspace of ``gdn_ssm_prefill`` for this problem size (0: none is used)."""
    return int(_lib.load().gdn_b200_ssm_prefill_workspace_size(num_seqs, total_tokens, num_heads,
                                                               head_dim, state_dim))


def gdn_ssm_prefill(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, output, new_state, *,
                    state_indices=None, has_state=None, workspace=None) -> None:
    """Selective state space scan over packed prompts.

    Per head, with the fp32 state h [P, N]: ``step = softplus(dt + dt_bias)``,
    ``h = exp(-exp(A_log) step) h + (step x) B^T``, ``y = h C + D x``.

    x: [T, H, P] bf16; dt: [T, H] bf16; B, C: [T, G, N] bf16 (head h reads group
    h // (H // G)), each with a free token stride of 16-byte multiples (dt: any);
    A_log: [H] fp32; D, dt_bias: [H] fp32 or None; P and N are 64 or 128;
    state: [S, H, P, N] fp32 or None (zero); output: [T, H, P] bf16; new_state:
    [S, H, P, N] fp32 (may be state); cu_seqlens, state_indices, has_state as in
    ``gdn_short_conv``.  workspace: a uint8 CUDA tensor of at least
    ``ssm_prefill_workspace_bytes`` bytes (allocated here when omitted).

    A NaN or infinity in one token's operands can reach outputs of earlier
    tokens of its chunk, as the products run over whole chunks.
    """
    dev = _device(x, "x")
    T, H, P, G, N, args, o_ptr = _scan_operands(x, dt, A_log, B, C, D, dt_bias, output, dev)
    n, cu_ptr, cu64 = _offsets(cu_seqlens, dev)
    ns_ptr, pool = _pool_rows(new_state, "new_state", (H, P, N), dev, torch.float32)
    s_ptr = _full(state, "state", torch.float32, (pool, H, P, N), dev)
    i_ptr, i64 = _index(state_indices, "state_indices", n, dev)
    _need_slots(pool, n, state_indices)
    lib = _lib.load()
    need = int(lib.gdn_b200_ssm_prefill_workspace_size(n, T, H, P, N))
    if need and workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    w_ptr = w_bytes = 0
    if workspace is not None:
        if (not isinstance(workspace, torch.Tensor) or workspace.device != dev
                or not workspace.is_contiguous()):
            _refuse(f"workspace must be a contiguous tensor on {dev}")
        w_ptr, w_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if w_bytes < need:
            _refuse(f"workspace must have at least {need} bytes")
    _call(dev, lib.gdn_b200_ssm_prefill, *args, s_ptr, cu_ptr, cu64, i_ptr, i64,
          _flags(has_state, n, dev), o_ptr, ns_ptr, n, T, pool, H, G, P, N, w_ptr, w_bytes)


def gdn_ssm_step(x, dt, A_log, B, C, D, dt_bias, state_pool, state_indices, output, *,
                 new_state_pool=None, output_state_indices=None) -> None:
    """The selective scan of one new token per sequence: x, output [B, H, P];
    dt [B, H]; B, C [B, G, N]; state_pool [S, H, P, N] fp32; state_indices [B] or
    None; new_state_pool: where the new states go (default: state_pool, in
    place); output_state_indices: their slots (default: the read slots).
    Otherwise as ``gdn_ssm_prefill``."""
    dev = _device(x, "x")
    Bn, H, P, G, N, args, o_ptr = _scan_operands(x, dt, A_log, B, C, D, dt_bias, output, dev)
    s_ptr, pool = _pool_rows(state_pool, "state_pool", (H, P, N), dev, torch.float32)
    ns_ptr = (s_ptr if new_state_pool is None else
              _full(new_state_pool, "new_state_pool", torch.float32, (pool, H, P, N), dev))
    i_ptr, i64 = _index(state_indices, "state_indices", Bn, dev)
    wi_ptr, wi64 = _index(output_state_indices, "output_state_indices", Bn, dev)
    if output_state_indices is not None and (state_indices is None or wi64 != i64):
        _refuse("output_state_indices need state_indices of the same type")
    _need_slots(pool, Bn, state_indices)
    _call(dev, _lib.load().gdn_b200_ssm_step, *args, s_ptr, i_ptr, wi_ptr, i64, o_ptr, ns_ptr, Bn,
          pool, H, G, P, N)


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
    dev = _device(x, "x")
    code = _dtype_code(x, "x")
    act = _activation(activation, ("silu", "sigmoid"))
    shape = x.shape
    if len(shape) == 2:
        T, width = shape
    elif len(shape) == 3:
        T, width = shape[0], shape[1] * shape[2]
    else:
        _refuse("x must be [T, D] or [T, H, P]")
    group = shape[-1] if group_size is None else int(group_size)
    if group < 1 or width < 1 or width % group:
        _refuse(f"group_size must divide the row's width {width}, got {group}")
    x_ptr, x_stride = _rows(x, "x", x.dtype, shape, dev)
    g_ptr, g_stride = (0, 0) if gate is None else _rows(gate, "gate", x.dtype, shape, dev)
    o_ptr, o_stride = _rows(output, "output", x.dtype, shape, dev)
    w_ptr = shared = 0
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or weight.numel() not in (group, width):
            _refuse(f"weight: expected {group} or {width} elements")
        shared = 1 if weight.numel() == group else 0
        w_ptr = _full(weight, "weight", x.dtype, weight.shape, dev)
    _call(dev, _lib.load().gdn_b200_gated_norm, x_ptr, x_stride, g_ptr, g_stride, w_ptr, shared,
          o_ptr, o_stride, T, width, group, eps, act, 1 if norm_first else 0, code)


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
    dev = _device(x, "x")
    code = _dtype_code(x, "x")
    if x.dim() != 2:
        _refuse("x must be [T, D]")
    shape = x.shape
    T, D = shape
    if not isinstance(residual, torch.Tensor) or residual.dtype not in (x.dtype, torch.float32):
        _refuse(f"residual must be a tensor of {x.dtype} or float32")
    rdt = residual.dtype
    x_ptr, x_stride = _rows(x, "x", x.dtype, shape, dev)
    r_ptr, r_stride = _rows(residual, "residual", rdt, shape, dev)
    o_ptr, o_stride = _rows(output, "output", x.dtype, shape, dev)
    nr_ptr, nr_stride = _rows(new_residual, "new_residual", rdt, shape, dev)
    if weight is None:
        _refuse("weight: expected a torch.Tensor")
    if D < 1:
        _refuse("rows must not be empty")
    w_ptr = _full(weight, "weight", x.dtype, (D,), dev)
    bw_ptr = _full(block_weight, "block_weight", x.dtype, (D,), dev)
    cs_ptr = 0
    if isinstance(scale, torch.Tensor):
        cs_ptr, scale = _full(scale, "scale", torch.float32, (D,), dev), 1.0
    _call(dev, _lib.load().gdn_b200_add_norm, x_ptr, x_stride, r_ptr, r_stride, w_ptr, bw_ptr,
          cs_ptr, scale, o_ptr, o_stride, nr_ptr, nr_stride, T, D, eps, weight_offset, code,
          1 if rdt == torch.float32 else 0)


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
