"""Cases of the mixer operators that stand around a recurrent block: the short causal
convolution before it, the selective state space scan, the norms before and after it.

Each case is one call as a serving loop makes it: prompts packed along one token axis and
indexed by ``cu_seqlens``, or one new token per sequence against a pool of states.  ``run``
computes it in plain torch operations, or through ``gdn_kernel_b200`` where ``own`` is true.
``exact`` computes the definition in 64 bits.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LOG2_CHUNK = 6          # plain scan: tokens of a chunk, as a power of two
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One long prompt through the convolution of a GDN layer of 16 qk heads and
        # 32 v heads of 128: q, k and v side by side, 8,192 channels, width 4, no bias.
        {"name": "conv_prompt_8192", "op": "conv", "tokens": 8192, "seqs": 1, "channels": 8192,
         "width": 4, "bias": False, "dtype": "bf16", "slots": 0},
        # A scheduler's mixed batch: new prompts and further pieces of running ones, their
        # states in a pool, ragged lengths with empty and one-token ones; the x, B and C
        # channels of a scan layer of 64 heads of 64.
        {"name": "conv_ragged_pool", "op": "conv", "tokens": 3001, "seqs": 13, "channels": 4352,
         "width": 4, "bias": True, "dtype": "bf16", "slots": 40},
        # The decode step of 64 running sequences, the same GDN layer.
        {"name": "conv_step_64", "op": "conv_step", "batch": 64, "channels": 8192, "width": 4,
         "bias": False, "dtype": "bf16", "slots": 96, "padded": 0},
        # A few sequences in a padded batch, 16-bit floats of the other kind, width 3.
        {"name": "conv_step_7_padded", "op": "conv_step", "batch": 7, "channels": 2304, "width": 3,
         "bias": True, "dtype": "fp16", "slots": 16, "padded": 2},
        # One long prompt through the scan: 64 heads of 64, state 128, one group.
        {"name": "scan_prompt_8192", "op": "scan", "tokens": 8192, "seqs": 1, "heads": 64,
         "head_dim": 64, "groups": 1, "state_dim": 128, "slots": 0},
        # A mixed batch of ragged prompts with carried states, 32 heads of 128, state 64.
        {"name": "scan_ragged_pool", "op": "scan", "tokens": 20011, "seqs": 12, "heads": 32,
         "head_dim": 128, "groups": 4, "state_dim": 64, "slots": 24},
        # The decode step of 64 running sequences: the fp32 states are what moves.
        {"name": "scan_step_64", "op": "scan_step", "batch": 64, "heads": 64, "head_dim": 64,
         "groups": 1, "state_dim": 128, "slots": 80, "padded": 0},
        # A small padded batch, where latency counts.
        {"name": "scan_step_5_padded", "op": "scan_step", "batch": 5, "heads": 32,
         "head_dim": 128, "groups": 4, "state_dim": 64, "slots": 9, "padded": 1},
        # The gated norm per head after GDN on a long prompt, 32 heads of 128.
        {"name": "gated_norm_8192", "op": "gated_norm", "tokens": 8192, "width": 4096,
         "group": 128, "shared": True, "norm_first": True, "dtype": "bf16"},
        # The gated norm after a scan at decode: one group over the row, the gate first.
        {"name": "gated_norm_64", "op": "gated_norm", "tokens": 64, "width": 4096,
         "group": 4096, "shared": False, "norm_first": False, "dtype": "bf16"},
        # Residual add and the next block's norm on a long prompt, fp32 residual stream,
        # with the norm after the block and a residual scale per channel.
        {"name": "add_norm_8192", "op": "add_norm", "tokens": 8192, "width": 2048,
         "post": True, "channel_scale": True, "residual": "fp32", "dtype": "bf16"},
        # The same place at decode, all in 16 bits, plain residual add.
        {"name": "add_norm_64", "op": "add_norm", "tokens": 64, "width": 2048,
         "post": False, "channel_scale": False, "residual": "bf16", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "conv_step", "scan", "scan_step", "gated_norm", "add_norm"])
    if op == "conv":
        tokens = _log(rng, 1, 8192)
        return {"op": op, "tokens": tokens, "seqs": rng.choice([1, _log(rng, 1, 24)]),
                "channels": 8 * _log(rng, 32, 1024), "width": rng.choice([2, 3, 4, 4]),
                "bias": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "slots": rng.choice([0, 32])}
    if op == "conv_step":
        batch = _log(rng, 1, 256)
        return {"op": op, "batch": batch, "channels": 8 * _log(rng, 32, 1024),
                "width": rng.choice([2, 3, 4, 4]), "bias": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "slots": batch + rng.randint(0, 40),
                "padded": rng.randint(0, batch // 2)}
    if op == "scan":
        groups = rng.choice([1, 2, 4, 8])
        return {"op": op, "tokens": _log(rng, 1, 12000), "seqs": rng.choice([1, _log(rng, 1, 16)]),
                "heads": groups * rng.randint(1, 32 // groups), "head_dim": rng.choice([64, 128]),
                "groups": groups, "state_dim": rng.choice([64, 128]), "slots": rng.choice([0, 24])}
    if op == "scan_step":
        batch, groups = _log(rng, 1, 128), rng.choice([1, 2, 4, 8])
        return {"op": op, "batch": batch, "heads": groups * rng.randint(1, 32 // groups),
                "head_dim": rng.choice([64, 128]), "groups": groups,
                "state_dim": rng.choice([64, 128]), "slots": batch + rng.randint(0, 16),
                "padded": rng.randint(0, batch // 2)}
    if op == "gated_norm":
        group = 8 * _log(rng, 8, 256)
        return {"op": op, "tokens": _log(rng, 1, 8192), "width": group * rng.randint(1, 4096 // group + 1),
                "group": group, "shared": rng.random() < 0.5, "norm_first": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return {"op": op, "tokens": _log(rng, 1, 8192), "width": 8 * _log(rng, 16, 768),
            "post": rng.random() < 0.5, "channel_scale": rng.random() < 0.5,
            "residual": rng.choice(["fp32", dtype]), "dtype": dtype}


def _lengths(case):
    """The packed lengths of a case: ragged, with an empty and a one-token sequence where
    there are more than four."""
    tokens, seqs = case["tokens"], case["seqs"]
    if seqs == 1:
        return [tokens]
    r = random.Random(tokens * 1009 + seqs)
    fixed = [0, 1] if seqs > 4 and tokens > 8 else []
    left, n = tokens - sum(fixed), seqs - len(fixed)
    cuts = sorted(r.randint(0, left) for _ in range(n - 1))
    got = [b - a for a, b in zip([0] + cuts, cuts + [left])] + fixed
    r.shuffle(got)
    return got


# ------------------------------------------------------------------ inputs
class _Maker:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.g, device=DEV) * std).to(dtype)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.g, device=DEV) * (hi - lo) + lo

    def slots(self, count, pool):
        return torch.randperm(pool, generator=self.g, device=DEV)[:count].to(torch.int32)


def _scan_inputs(m, case, rows):
    """x, B and C lie side by side in one activation row, as the convolution leaves them."""
    H, P, G, N = case["heads"], case["head_dim"], case["groups"], case["state_dim"]
    raw = m.normal(rows, H * P + 2 * G * N)
    xbc = (raw * torch.sigmoid(raw)).to(torch.bfloat16)
    x = xbc[:, :H * P].view(rows, H, P)
    B = xbc[:, H * P:H * P + G * N].view(rows, G, N)
    C = xbc[:, H * P + G * N:].view(rows, G, N)
    step = torch.exp(m.uniform(math.log(1e-3), math.log(0.1), H))
    return {"x": x, "B": B, "C": C, "dt": m.normal(rows, H, std=0.5, dtype=torch.bfloat16),
            "A_log": torch.log(m.uniform(1.0, 16.0, H)),
            "dt_bias": step + torch.log(-torch.expm1(-step)), "D": m.normal(H, std=0.5) + 1.0}


def prepare(case, seed):
    m = _Maker(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("conv", "scan"):
        cu = [0]
        for n in _lengths(case):
            cu.append(cu[-1] + n)
        s["cu_seqlens"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
        n = case["seqs"]
        s["slots"] = s["has_state"] = None
        if case["slots"]:
            s["slots"] = m.slots(n, case["slots"])
            s["has_state"] = m.uniform(0.0, 1.0, n) < 0.6
    elif op in ("conv_step", "scan_step"):
        s["slots"] = m.slots(case["batch"], case["slots"])
        if case["padded"]:
            s["slots"][-case["padded"]:] = -1
    if op in ("conv", "conv_step"):
        dt, D, W = DTYPES[case["dtype"]], case["channels"], case["width"]
        rows = case["tokens"] if op == "conv" else case["batch"]
        pool = case["slots"] or case["seqs"]
        s["x"] = m.normal(rows, D, dtype=dt)
        s["weight"] = m.normal(D, W, std=W ** -0.5, dtype=dt)
        s["bias"] = m.normal(D, std=0.2, dtype=dt) if case["bias"] else None
        s["state"] = m.normal(pool, W - 1, D, dtype=dt) if case["slots"] else None
        s["output"] = torch.empty_like(s["x"])
        s["new_state"] = torch.zeros(pool, W - 1, D, dtype=dt, device=DEV)
    elif op in ("scan", "scan_step"):
        rows = case["tokens"] if op == "scan" else case["batch"]
        pool = case["slots"] or case["seqs"]
        s |= _scan_inputs(m, case, rows)
        shape = (pool, case["heads"], case["head_dim"], case["state_dim"])
        s["state"] = m.normal(*shape, std=0.3) if case["slots"] else None
        s["output"] = torch.empty(s["x"].shape, dtype=torch.bfloat16, device=DEV)
        s["new_state"] = torch.zeros(shape, device=DEV)
    elif op == "gated_norm":
        dt = DTYPES[case["dtype"]]
        T, D = case["tokens"], case["width"]
        s["x"] = m.normal(T, D, std=0.5, dtype=dt)
        # the gate is the first part of the rows that the block's input projection wrote
        s["gate"] = m.normal(T, D + 64, dtype=dt)[:, :D]
        s["weight"] = (m.normal(case["group"] if case["shared"] else D, std=0.1) + 1.0).to(dt)
        s["output"] = torch.empty_like(s["x"])
    else:
        dt, T, D = DTYPES[case["dtype"]], case["tokens"], case["width"]
        s["x"] = m.normal(T, D, dtype=dt)
        s["residual"] = m.normal(T, D, std=2.0, dtype=DTYPES[case["residual"]])
        s["weight"] = (m.normal(D, std=0.1) + 1.0).to(dt)
        s["post"] = (m.normal(D, std=0.1) + 1.0).to(dt) if case["post"] else None
        s["channel_scale"] = m.uniform(0.05, 0.5, D) if case["channel_scale"] else None
        s["output"] = torch.empty_like(s["x"])
        s["new_residual"] = torch.empty_like(s["residual"])
    return s


# ------------------------------------------------------------------ the calls
def run(s):
    op = s["case"]["op"]
    if own:
        return _OWN[op](s)
    return _PLAIN[op](s)


def _own_conv(s):
    import gdn_kernel_b200 as g
    g.gdn_short_conv(s["x"], s["weight"], s["bias"], s["state"], s["cu_seqlens"], s["output"],
                     s["new_state"], state_indices=s["slots"], has_state=s["has_state"])
    return {"out": s["output"], "state": s["new_state"]}


def _own_conv_step(s):
    import gdn_kernel_b200 as g
    g.gdn_short_conv_step(s["x"], s["weight"], s["bias"], s["state"], s["slots"], s["output"],
                          new_state_pool=s["new_state"])
    return {"out": s["output"], "state": s["new_state"]}


def _own_scan(s):
    import gdn_kernel_b200 as g
    g.gdn_ssm_prefill(s["x"], s["dt"], s["A_log"], s["B"], s["C"], s["D"], s["dt_bias"],
                      s["state"], s["cu_seqlens"], s["output"], s["new_state"],
                      state_indices=s["slots"], has_state=s["has_state"])
    return {"out": s["output"], "state": s["new_state"]}


def _own_scan_step(s):
    import gdn_kernel_b200 as g
    g.gdn_ssm_step(s["x"], s["dt"], s["A_log"], s["B"], s["C"], s["D"], s["dt_bias"], s["state"],
                   s["slots"], s["output"], new_state_pool=s["new_state"])
    return {"out": s["output"], "state": s["new_state"]}


def _own_gated_norm(s):
    import gdn_kernel_b200 as g
    c = s["case"]
    g.gdn_gated_norm(s["x"], s["gate"], s["weight"], s["output"], group_size=c["group"], eps=EPS,
                     norm_first=c["norm_first"])
    return {"out": s["output"]}


def _own_add_norm(s):
    import gdn_kernel_b200 as g
    scale = 0.5 if s["channel_scale"] is None else s["channel_scale"]
    g.gdn_add_norm(s["x"], s["residual"], s["weight"], s["output"], s["new_residual"],
                   block_weight=s["post"], scale=scale, eps=EPS)
    return {"out": s["output"], "residual": s["new_residual"]}


_OWN = {"conv": _own_conv, "conv_step": _own_conv_step, "scan": _own_scan,
        "scan_step": _own_scan_step, "gated_norm": _own_gated_norm, "add_norm": _own_add_norm}


# ------------------------------------------------------------------ plain forms
def _silu(v):
    return v * torch.sigmoid(v)


def _carried(state, slots, has_state, n):
    """fp32 initial states of n sequences: gathered, and zero where there is none."""
    if state is None:
        return None
    at = torch.arange(n, device=state.device) if slots is None else slots.long()
    keep = at >= 0
    if has_state is not None:
        keep = keep & has_state
    got = state[at.clamp_min(0)].float()
    return torch.where(keep.view((n,) + (1,) * (state.dim() - 1)), got, torch.zeros_like(got))


def _stored(pool, slots, values):
    """The pool with `values` at the slots; entries of negative slots go nowhere."""
    values = values.to(pool.dtype)
    if slots is None:
        return values
    room = torch.cat([pool, pool[:1]])
    at = torch.where(slots >= 0, slots, pool.shape[0]).long()
    return room.index_copy(0, at, values)[:-1]


def _plain_conv(s):
    x, w, cu = s["x"].float(), s["weight"].float(), s["cu_seqlens"].long()
    T, D = x.shape
    W, n = w.shape[1], cu.numel() - 1
    first = _carried(s["state"], s["slots"], s["has_state"], n)
    if first is None:
        first = x.new_zeros(n, W - 1, D)
    # rows of every sequence's history, then its tokens: row index of (sequence, position)
    rows = torch.cat([first.reshape(n * (W - 1), D), x])
    t = torch.arange(T, device=x.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    taps = torch.arange(W, device=x.device) - (W - 1)

    def row_of(q, pos):
        return torch.where(pos < 0, q * (W - 1) + (W - 1) + pos, n * (W - 1) + cu[q] + pos)

    at = row_of(seq[:, None], (t - cu[seq])[:, None] + taps)
    y = (rows[at] * w.t()).sum(1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    q = torch.arange(n, device=x.device)[:, None]
    last = rows[row_of(q, (cu[1:] - cu[:-1])[:, None] + taps[:-1])]
    return {"out": _silu(y).to(s["x"].dtype), "state": _stored(s["new_state"], s["slots"], last)}


def _plain_conv_step(s):
    x, w = s["x"].float(), s["weight"].float()
    slots, live = s["slots"].long(), (s["slots"] >= 0)[:, None]
    hist = torch.cat([s["state"][slots.clamp_min(0)].float(), x[:, None]], 1)
    y = (hist * w.t()).sum(1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = torch.where(live, _silu(y), torch.zeros_like(y))
    return {"out": y.to(s["x"].dtype),
            "state": _stored(s["new_state"], s["slots"], hist[:, 1:])}


def _softplus(v):
    return torch.clamp_min(v, 0) + torch.log1p(torch.exp(-v.abs()))


def _segment_sums(a):
    """[..., Q] -> [..., Q, Q]: sums of a over (j, i], -inf above the diagonal."""
    Q = a.shape[-1]
    i = torch.arange(Q, device=a.device)
    grown = torch.where(i[:, None] > i[None, :], a[..., :, None], a.new_zeros(()))
    return grown.cumsum(-2).masked_fill(i[:, None] < i[None, :], -math.inf)


def _plain_scan(s):
    """Chunks of 64 tokens, each within one sequence: products inside a chunk, then the
    states at the chunks' starts through one matrix of decays between chunks."""
    x, dt, cu = s["x"], s["dt"], s["cu_seqlens"].long()
    T, H, P = x.shape
    G, N = s["B"].shape[1:]
    n, Q = cu.numel() - 1, 1 << LOG2_CHUNK
    dev = x.device
    lens = cu[1:] - cu[:-1]
    ends = ((lens + Q - 1) >> LOG2_CHUNK).cumsum(0)          # chunks up to each sequence's end
    chunks = T // Q + n                                      # no fewer than there are
    c = torch.arange(chunks, device=dev)
    seq = torch.searchsorted(ends, c, right=True).clamp_max(n - 1)
    begin = torch.cat([ends.new_zeros(1), ends[:-1]])
    at = (cu[seq] + ((c - begin[seq]) << LOG2_CHUNK))[:, None] + torch.arange(Q, device=dev)
    ok = (at < cu[seq + 1][:, None]) & (c < ends[-1])[:, None]
    at = at.clamp(0, max(T - 1, 0))
    keep = ok[:, :, None]
    d = torch.where(keep, _softplus(dt[at].float() + s["dt_bias"]), dt.new_zeros((), dtype=torch.float32))
    la = (-torch.exp(s["A_log"]) * d).transpose(1, 2)        # [chunks, H, Q]
    zero = torch.zeros((), device=dev)
    xf = torch.where(keep[..., None], x[at].float(), zero)
    Bf = torch.where(keep[..., None], s["B"][at].float(), zero)
    Cf = torch.where(keep[..., None], s["C"][at].float(), zero)
    xd = (xf * d[..., None]).permute(0, 2, 1, 3)             # [chunks, H, Q, P]
    rep = H // G
    Bh = Bf.permute(0, 2, 1, 3).repeat_interleave(rep, 1)    # [chunks, H, Q, N]
    Ch = Cf.permute(0, 2, 1, 3).repeat_interleave(rep, 1)
    y = torch.matmul(torch.matmul(Ch, Bh.transpose(2, 3)) * torch.exp(_segment_sums(la)), xd)
    after = la.flip(-1).cumsum(-1).flip(-1) - la             # decay from a token to its chunk's end
    part = torch.matmul((xd * torch.exp(after)[..., None]).transpose(2, 3), Bh)   # [chunks, H, P, N]
    # state at the start of chunk c: the parts of earlier chunks of its sequence, decayed by
    # the chunks between, and the carried state decayed by all of them
    total = la.sum(-1).t()                                   # [H, chunks]
    between = _segment_sums(total)                           # sums over (e, c]
    same = (seq[:, None] == seq[None, :]) & (c[:, None] >= c[None, :])
    upto = torch.where(same, torch.exp(between), zero)       # decay from the end of e to the end of c
    end = torch.matmul(upto, part.permute(1, 0, 2, 3).reshape(H, chunks, P * N))
    first = _carried(s["state"], s["slots"], s["has_state"], n)
    if first is None:
        first = torch.zeros(n, H, P, N, device=dev)
    own_total = torch.matmul(same.float(), total.t())        # [chunks, H] decay since the start
    end = end.view(H, chunks, P, N).transpose(0, 1) + torch.exp(own_total)[..., None, None] * first[seq]
    new = (c == begin[seq])[:, None, None, None]
    start = torch.where(new, first[seq], torch.cat([end[:1], end[:-1]]))
    y = y + torch.exp(la.cumsum(-1))[..., None] * torch.matmul(Ch, start.transpose(2, 3))
    y = (y + s["D"][:, None, None] * xf.permute(0, 2, 1, 3)).permute(0, 2, 1, 3)   # [chunks, Q, H, P]
    t = torch.arange(T, device=dev)
    q = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    p = t - cu[q]
    y = y.reshape(chunks * Q, H, P)[((begin[q] + (p >> LOG2_CHUNK)) << LOG2_CHUNK) + (p & (Q - 1))]
    last = torch.where((lens > 0)[:, None, None, None], end[(ends - 1).clamp_min(0)], first)
    return {"out": y.to(x.dtype), "state": _stored(s["new_state"], s["slots"], last)}


def _plain_scan_step(s):
    x, slots = s["x"].float(), s["slots"].long()
    live = (s["slots"] >= 0)[:, None, None]
    rep = x.shape[1] // s["B"].shape[1]
    Bf = s["B"].float().repeat_interleave(rep, 1)
    Cf = s["C"].float().repeat_interleave(rep, 1)
    d = _softplus(s["dt"].float() + s["dt_bias"])
    h = s["state"][slots.clamp_min(0)] * torch.exp(-torch.exp(s["A_log"]) * d)[..., None, None]
    h = h + (x * d[..., None])[..., None] * Bf[:, :, None]
    y = (h * Cf[:, :, None]).sum(-1) + s["D"][:, None] * x
    y = torch.where(live, y, torch.zeros_like(y))
    return {"out": y.to(s["x"].dtype), "state": _stored(s["new_state"], s["slots"], h)}


def _norm(v, group):
    g = v.view(v.shape[0], -1, group)
    return (g * torch.rsqrt(g.square().mean(-1, keepdim=True) + EPS)).view(v.shape)


def _plain_gated_norm(s):
    c = s["case"]
    x, z, w = s["x"].float(), _silu(s["gate"].float()), s["weight"].float()
    if c["shared"]:
        w = w.repeat(c["width"] // c["group"])
    y = _norm(x, c["group"]) * w * z if c["norm_first"] else _norm(x * z, c["group"]) * w
    return {"out": y.to(s["x"].dtype)}


def _plain_add_norm(s):
    u = s["x"].float()
    if s["post"] is not None:
        u = _norm(u, u.shape[1]) * s["post"].float()
    r = s["residual"].float() + u * (0.5 if s["channel_scale"] is None else s["channel_scale"])
    y = _norm(r, r.shape[1]) * s["weight"].float()
    return {"out": y.to(s["x"].dtype), "residual": r.to(s["residual"].dtype)}


_PLAIN = {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan,
          "scan_step": _plain_scan_step, "gated_norm": _plain_gated_norm,
          "add_norm": _plain_add_norm}


# ------------------------------------------------------------------ work
def work(case):
    """Inputs read once and outputs written once; multiply-adds of the recurrences count two."""
    op = case["op"]
    if op in ("conv", "conv_step"):
        e, D, W = DTYPES[case["dtype"]].itemsize, case["channels"], case["width"]
        rows = case["tokens"] if op == "conv" else case["batch"] - case["padded"]
        states = case["seqs"] if op == "conv" else rows
        b = 2 * rows * D * e + D * W * e + states * (W - 1) * D * e * (2 if case["slots"] else 1)
        return {"bytes": b, "flops": rows * D * (2 * W + 4)}
    if op in ("scan", "scan_step"):
        H, P, G, N = case["heads"], case["head_dim"], case["groups"], case["state_dim"]
        rows = case["tokens"] if op == "scan" else case["batch"] - case["padded"]
        states = case["seqs"] if op == "scan" else rows
        b = rows * (2 * H * P + 2 * G * N + H) * 2 + states * H * P * N * 4 * (2 if case["slots"] else 1)
        return {"bytes": b + 12 * H, "flops": rows * H * P * N * 5}
    D, T, e = case["width"], case["tokens"], DTYPES[case["dtype"]].itemsize
    if op == "gated_norm":
        return {"bytes": 3 * T * D * e, "flops": 10 * T * D}
    r = DTYPES[case["residual"]].itemsize
    return {"bytes": 2 * T * D * (e + r), "flops": (10 if case["post"] else 6) * T * D}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in s.items()}
    op = case["op"]
    if op in ("gated_norm", "add_norm"):
        def rms(v, group):
            u = v.reshape(-1, group)
            return (u / torch.sqrt((u * u).sum(1, keepdim=True) / group + EPS)).reshape(v.shape)

        if op == "gated_norm":
            T, D = f["x"].shape
            g = f["gate"] / (1 + torch.exp(-f["gate"]))
            w = f["weight"].repeat(D // f["weight"].numel())
            first = case["norm_first"]
            return {"out": rms(f["x"], case["group"]) * w * g if first
                    else rms(f["x"] * g, case["group"]) * w}
        u = f["x"] if f["post"] is None else rms(f["x"], case["width"]) * f["post"]
        r = f["residual"] + (u * 0.5 if f["channel_scale"] is None else u * f["channel_scale"])
        return {"out": rms(r, case["width"]) * f["weight"], "residual": r}
    if op in ("conv", "scan"):
        lens = _lengths(case)
        starts = [sum(lens[:i]) for i in range(len(lens))]
    else:
        lens, starts = [1] * case["batch"], list(range(case["batch"]))
    slots = s["slots"].tolist() if s["slots"] is not None else list(range(len(lens)))
    has = s["has_state"].tolist() if s.get("has_state") is not None else [True] * len(lens)
    pool = torch.zeros_like(f["new_state"])
    if op in ("conv", "conv_step"):
        W, out = case["width"], torch.zeros_like(f["x"])
        for i, n in enumerate(lens):
            old = torch.zeros(W - 1, case["channels"], dtype=torch.float64, device=DEV)
            if f["state"] is not None and slots[i] >= 0 and has[i]:
                old = f["state"][slots[i]]
            if op == "conv_step" and slots[i] < 0:
                continue
            h = torch.cat([old, f["x"][starts[i]:starts[i] + n]])
            y = torch.zeros(n, case["channels"], dtype=torch.float64, device=DEV)
            for k in range(W):
                y += h[k:k + n] * f["weight"][:, k]
            if f["bias"] is not None:
                y += f["bias"]
            out[starts[i]:starts[i] + n] = y / (1 + torch.exp(-y))
            if slots[i] >= 0:
                pool[slots[i]] = h[n:]
        return {"out": out, "state": pool}
    # token by token over all sequences at once, the longest first so that those still
    # running are a leading part
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    H, P, N = case["heads"], case["head_dim"], case["state_dim"]
    rep = H // case["groups"]
    h = torch.zeros(len(lens), H, P, N, dtype=torch.float64, device=DEV)
    for k, i in enumerate(order):
        if f["state"] is not None and slots[i] >= 0 and has[i]:
            h[k] = f["state"][slots[i]]
    d = torch.log1p(torch.exp(f["dt"] + f["dt_bias"]))
    decay = torch.exp(-torch.exp(f["A_log"]) * d)
    xd = f["x"] * d[..., None]
    out = torch.zeros_like(f["x"])
    where = torch.tensor([starts[i] for i in order], device=DEV)
    for t in range(max(lens)):
        k = sum(n > t for n in lens)
        at = where[:k] + t
        Bt = f["B"][at].repeat_interleave(rep, 1)
        h[:k].mul_(decay[at][..., None, None]).addcmul_(xd[at][..., None], Bt[:, :, None])
        out[at] = torch.matmul(h[:k], f["C"][at].repeat_interleave(rep, 1)[..., None])[..., 0]
    out += f["D"][:, None] * f["x"]
    for k, i in enumerate(order):
        if slots[i] >= 0:
            pool[slots[i]] = h[k]
        elif op == "scan_step":
            out[starts[i]] = 0
    return {"out": out, "state": pool}
