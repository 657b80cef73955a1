"""A small hybrid stack served with this package: Gated DeltaNet layers and selective
scan layers in turn, prompts first, then one token per sequence at a time.

Every layer is  residual add + norm -> projection -> short convolution -> recurrence
-> gated norm -> projection.  The projections are plain matrix products with random
weights; the operators between them are calls of this package:

    add_norm, short_conv / short_conv_step, prefill / gdn_decode_pool (GDN layers) or
    ssm_prefill / ssm_step (scan layers), gated_norm

A GDN layer norms q and k with two more gated_norm calls, copies v, a and b (its calls
take contiguous tensors), and stores a prompt's states to their slots itself; a scan
layer reads column slices and slots as they are.  The states stay in pools with a slot
per sequence, updated in place by the steps.

    python examples/hybrid_stack.py            # prompts, then steps; checks the two agree
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import gdn_kernel_b200 as g  # noqa: E402

BF = torch.bfloat16
HIDDEN, WIDTH = 512, 4                    # residual stream, taps of the convolution
QK_HEADS, V_HEADS, HEAD = 2, 4, 128       # GDN layer
HEADS, HEAD_DIM, GROUPS, STATE = 8, 64, 2, 128   # scan layer


def weights(gen, rows, cols):
    return (torch.randn(rows, cols, generator=gen, device="cuda") * rows ** -0.5).to(BF)


class Layer:
    """What both kinds share: the norm before the mixer, the projections, the
    convolution and its pool, the gated norm after."""

    def __init__(self, gen, slots, channels, inner, extra):
        self.norm = torch.ones(HIDDEN, dtype=BF, device="cuda")
        self.w_in = weights(gen, HIDDEN, channels + inner + extra)
        self.w_out = weights(gen, inner, HIDDEN)
        self.conv = weights(gen, channels, WIDTH)
        self.conv_pool = torch.zeros(slots, WIDTH - 1, channels, dtype=BF, device="cuda")
        self.channels, self.inner = channels, inner

    def project(self, x):
        rows = x @ self.w_in
        c, i = self.channels, self.inner
        return rows[:, :c], rows[:, c:c + i], rows[:, c + i:]

    def convolve(self, u, cu, slots):
        out = torch.empty(u.shape, dtype=BF, device="cuda")
        if cu is None:
            g.gdn_short_conv_step(u, self.conv, None, self.conv_pool, slots, out)
        else:
            g.gdn_short_conv(u, self.conv, None, None, cu, out, self.conv_pool,
                             state_indices=slots)
        return out


class GdnLayer(Layer):
    def __init__(self, gen, slots):
        qk, v = QK_HEADS * HEAD, V_HEADS * HEAD
        super().__init__(gen, slots, 2 * qk + v, v, 2 * V_HEADS)
        self.pool = torch.zeros(slots, V_HEADS, HEAD, HEAD, device="cuda")
        self.A_log = torch.log(torch.rand(V_HEADS, generator=gen, device="cuda") * 15 + 1)
        self.dt_bias = torch.randn(V_HEADS, generator=gen, device="cuda") * 0.1 - 3
        # rms(x) / sqrt(HEAD) is x over its 2-norm, which q and k need per head
        self.unit = torch.full((HEAD,), HEAD ** -0.5, dtype=BF, device="cuda")
        self.gate_norm = torch.ones(HEAD, dtype=BF, device="cuda")

    def __call__(self, x, cu, slots):
        T, qk = x.shape[0], QK_HEADS * HEAD
        u, z, ab = self.project(x)
        u = self.convolve(u, cu, slots)
        q, k = (g.gated_norm(u[:, i * qk:(i + 1) * qk].view(T, QK_HEADS, HEAD), None, self.unit)
                for i in (0, 1))
        v = u[:, 2 * qk:].contiguous().view(T, V_HEADS, HEAD)
        a, b = ab[:, :V_HEADS].contiguous(), ab[:, V_HEADS:].contiguous()
        if cu is None:
            y = torch.empty(T, 1, V_HEADS, HEAD, dtype=BF, device="cuda")
            g.gdn_decode_pool(q[:, None], k[:, None], v[:, None], self.pool, slots, self.A_log,
                              a[:, None], self.dt_bias, b[:, None], 0.0, y)
            y = y[:, 0]
        else:
            y, states = g.prefill(q, k, v, None, self.A_log, a, self.dt_bias, b, cu)
            self.pool[slots.long()] = states
        y = g.gated_norm(y, z.view(T, V_HEADS, HEAD), self.gate_norm)
        return y.view(T, -1) @ self.w_out


class ScanLayer(Layer):
    def __init__(self, gen, slots):
        inner, bc = HEADS * HEAD_DIM, GROUPS * STATE
        super().__init__(gen, slots, inner + 2 * bc, inner, HEADS)
        self.pool = torch.zeros(slots, HEADS, HEAD_DIM, STATE, device="cuda")
        self.A_log = torch.log(torch.rand(HEADS, generator=gen, device="cuda") * 15 + 1)
        self.dt_bias = torch.randn(HEADS, generator=gen, device="cuda") * 0.1 - 3
        self.D = torch.ones(HEADS, device="cuda")
        self.gate_norm = torch.ones(inner, dtype=BF, device="cuda")

    def __call__(self, x, cu, slots):
        T, inner, bc = x.shape[0], HEADS * HEAD_DIM, GROUPS * STATE
        u, z, dt = self.project(x)
        u = self.convolve(u, cu, slots)
        # slices of the convolution's rows: no copies
        xs = u[:, :inner].view(T, HEADS, HEAD_DIM)
        B = u[:, inner:inner + bc].view(T, GROUPS, STATE)
        C = u[:, inner + bc:].view(T, GROUPS, STATE)
        y = torch.empty(T, HEADS, HEAD_DIM, dtype=BF, device="cuda")
        if cu is None:
            g.gdn_ssm_step(xs, dt, self.A_log, B, C, self.D, self.dt_bias, self.pool, slots, y)
        else:
            g.gdn_ssm_prefill(xs, dt, self.A_log, B, C, self.D, self.dt_bias, None, cu, y,
                              self.pool, state_indices=slots)
        y = g.gated_norm(y.view(T, inner), z, self.gate_norm, norm_first=False)
        return y @ self.w_out


class Stack:
    def __init__(self, slots: int, layers: int = 4, seed: int = 0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.layers = [(GdnLayer if i % 2 == 0 else ScanLayer)(gen, slots) for i in range(layers)]
        self.last_norm = torch.ones(HIDDEN, dtype=BF, device="cuda")

    def __call__(self, embedded, cu, slots):
        """embedded: [T, HIDDEN] bf16; cu: offsets of the packed prompts, or None for
        one new token per sequence; slots: each sequence's slot.  Returns the normed
        residual stream."""
        residual = torch.zeros(embedded.shape, device="cuda")       # fp32 stream
        out = embedded
        for layer in self.layers:
            x, residual = g.add_norm(out, residual, layer.norm)
            out = layer(x, cu, slots)
        return g.add_norm(out, residual, self.last_norm)[0]


def prompts_then_steps(lengths, steps: int, seed: int = 0):
    """The last `steps` tokens' outputs, from steps after the prompts and from the
    whole sequences at once: ([N, steps, HIDDEN], the same)."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 1)
    whole = [n + steps for n in lengths]
    tokens = [(torch.randn(n, HIDDEN, generator=gen, device="cuda")).to(BF) for n in whole]
    slots = torch.randperm(len(lengths) + 2, generator=gen, device="cuda")[:len(lengths)].int()

    def offsets(sizes):
        return torch.tensor([0, *torch.tensor(sizes).cumsum(0)], dtype=torch.int32, device="cuda")

    stack = Stack(len(lengths) + 2, seed=seed)
    stack(torch.cat([t[:n] for t, n in zip(tokens, lengths)]), offsets(lengths), slots)
    got = [stack(torch.stack([t[n + s] for t, n in zip(tokens, lengths)]), None, slots)
           for s in range(steps)]
    full = Stack(len(lengths) + 2, seed=seed)(torch.cat(tokens), offsets(whole), slots)
    ends = torch.tensor(whole).cumsum(0).tolist()
    want = torch.stack([full[e - steps:e] for e in ends])
    return torch.stack(got, 1), want


if __name__ == "__main__":
    got, want = prompts_then_steps([700, 1, 129, 40], steps=5)
    err = ((got.float() - want.float()).norm() / want.float().norm()).item()
    print(f"5 steps after prompts of 700, 1, 129 and 40 tokens: {err:.2e} from the whole "
          f"sequences at once; status {g.device_status(0)}")
    sys.exit(0 if err < 5e-2 else 1)
