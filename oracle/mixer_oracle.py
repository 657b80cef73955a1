"""Plain 64-bit implementations of the mixer operators: short causal
convolution, selective state space scan, gated norm, residual add and norm.

Each is the definition written out (token by token for the recurrences), on the
CPU.  The recurrences also return the same sums over absolute values, which
bound the error of any order of summation.
"""

import torch


def _slots(state_indices, n):
    return list(range(n)) if state_indices is None else [int(i) for i in state_indices]


def _act(v, activation):
    if activation is None:
        return v
    s = 1.0 / (1.0 + torch.exp(-v))
    return s if activation == "sigmoid" else torch.where(torch.isneginf(v), v, v * s)


def short_conv(x, weight, bias, state, cu_seqlens, new_state, activation="silu",
               state_indices=None, has_state=None):
    """Returns (output, new pool, magnitude of each output's sum)."""
    x, weight = x.double().cpu(), weight.double().cpu()
    D, W = weight.shape
    cu = [int(c) for c in cu_seqlens]
    out, mag = torch.zeros_like(x), torch.zeros_like(x)
    pool = new_state.double().cpu().clone()
    for i, slot in enumerate(_slots(state_indices, len(cu) - 1)):
        old = torch.zeros(W - 1, D, dtype=torch.float64)
        if state is not None and slot >= 0 and (has_state is None or bool(has_state[i])):
            old = state[slot].double().cpu()
        u = torch.cat([old, x[cu[i]:cu[i + 1]]])
        for t in range(cu[i + 1] - cu[i]):
            terms = u[t:t + W] * weight.t()
            b = torch.zeros(D, dtype=torch.float64) if bias is None else bias.double().cpu()
            out[cu[i] + t] = _act(terms.sum(0) + b, activation)
            mag[cu[i] + t] = terms.abs().sum(0) + b.abs()
        if slot >= 0:
            pool[slot] = u[u.shape[0] - (W - 1):]
    return out, pool, mag


def scan(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, new_state, state_indices=None,
         has_state=None, write_indices=None):
    """Returns (output, new pool, magnitude of the outputs, magnitude of the pool)."""
    f = lambda t: None if t is None else t.double().cpu()  # noqa: E731
    x, dt, A_log, B, C, D, dt_bias, state = map(f, (x, dt, A_log, B, C, D, dt_bias, state))
    T, H, P = x.shape
    rep = H // B.shape[1]
    cu = [int(c) for c in cu_seqlens]
    out, mag = torch.zeros_like(x), torch.zeros_like(x)
    pool = f(new_state).clone()
    pool_mag = pool.abs()
    writes = _slots(write_indices if write_indices is not None else state_indices, len(cu) - 1)
    for i, slot in enumerate(_slots(state_indices, len(cu) - 1)):
        h = torch.zeros(H, P, B.shape[2], dtype=torch.float64)
        if state is not None and slot >= 0 and (has_state is None or bool(has_state[i])):
            h = state[slot].clone()
        m = h.abs()
        for t in range(cu[i], cu[i + 1]):
            step = torch.nn.functional.softplus(dt[t] + (0 if dt_bias is None else dt_bias),
                                                threshold=50.0)
            decay = torch.exp(-torch.exp(A_log) * step)[:, None, None]
            Bt = B[t].repeat_interleave(rep, 0)[:, None]
            Ct = C[t].repeat_interleave(rep, 0)[:, None]
            xs = (x[t] * step[:, None])[:, :, None]
            h = h * decay + xs * Bt
            m = m * decay + (xs * Bt).abs()
            out[t] = (h * Ct).sum(-1)
            mag[t] = (m * Ct.abs()).sum(-1)
            if D is not None:
                out[t] += D[:, None] * x[t]
                mag[t] += (D[:, None] * x[t]).abs()
        if writes[i] >= 0:
            pool[writes[i]] = h
            pool_mag[writes[i]] = m
    return out, pool, mag, pool_mag


def _rms(v, group, eps):
    g = v.reshape(v.shape[0], -1, group)
    return (g / torch.sqrt((g * g).mean(-1, keepdim=True) + eps)).reshape(v.shape)


def gated_norm(x, gate, weight, group_size, eps, activation="silu", norm_first=True):
    x = x.double().cpu().reshape(x.shape[0], -1)
    g = 1.0 if gate is None else _act(gate.double().cpu().reshape(x.shape), activation)
    w = 1.0
    if weight is not None:
        w = weight.double().cpu().reshape(-1)
        w = w.repeat(x.shape[1] // w.numel())
    return _rms(x, group_size, eps) * w * g if norm_first else _rms(x * g, group_size, eps) * w


def add_norm(x, residual, weight, block_weight=None, scale=1.0, eps=1e-6, weight_offset=0.0):
    """Returns (output, new residual, magnitude of the residual's sum)."""
    u, r = x.double().cpu(), residual.double().cpu()
    if block_weight is not None:
        u = _rms(u, u.shape[1], eps) * block_weight.double().cpu()
    u = u * (scale.double().cpu() if isinstance(scale, torch.Tensor) else scale)
    return (_rms(r + u, r.shape[1], eps) * (weight.double().cpu() + weight_offset), r + u,
            r.abs() + u.abs())
