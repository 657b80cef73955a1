"""The mixer operators on the GPU against their 64-bit definitions.

Bounds.  An output is rounded once to its type: half a unit, ROUND below,
relative to the result.  Before that, fp32 sums of k terms are off by at most
k 2^-24 of the sum of the terms' absolute values (which the oracle returns),
and exp, rsqrt and division by a few units of 2^-23.
"""

import pytest
import torch

from gdn_kernel_b200 import _lib, mixer as M
from oracle import mixer_oracle as O

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF: 2.0 ** -8, HF: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF: 1e-30, HF: 2.0 ** -24, F32: 1e-30}       # fp16's subnormals
DTYPES = [BF, HF, F32]


def rand(*shape, dtype=F32, std=1.0, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def check(got, want, mag, rel, name):
    """|got - want| <= ROUND |want| + rel mag, elementwise."""
    want, mag = want.cuda(), mag.cuda()
    bound = 1.001 * ROUND[got.dtype] * want.abs() + rel * mag + TINY[got.dtype]
    err = (got.double().reshape(want.shape) - want).abs()
    assert torch.isfinite(got).all(), name
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} times the bound"


def offsets(lens, dtype=torch.int32):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=dtype).cuda()


def status_clean():
    assert _lib.device_status(torch.cuda.current_device()) == 0


# ------------------------------------------------------------------ short convolution
CONV_REL = 2.0 ** -20     # 5 terms, the activation's slope of at most 1.1, exp and division


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2, 3, 4], [31, 1, 32, 0, 33, 2, 95], [260]])
def test_short_conv_lengths(dtype, width, lens):
    T, n, D = sum(lens), len(lens), 136
    x, w, b = rand(T, D, dtype=dtype), rand(D, width, dtype=dtype), rand(D, dtype=dtype, seed=1)
    st = rand(n, width - 1, D, dtype=dtype, seed=2)
    cu = offsets(lens)
    out, ns = torch.full_like(x, float("nan")), torch.full_like(st, float("nan"))
    M.gdn_short_conv(x, w, b, st, cu, out, ns)
    want, pool, mag = O.short_conv(x, w, b, st, cu, ns)
    check(out, want, mag, CONV_REL, "output")
    assert torch.equal(ns.double().cpu(), pool)
    # in place: the state is read before it is replaced, wherever a sequence starts
    M.gdn_short_conv(x, w, b, st, cu, out2 := torch.empty_like(x), st)
    assert torch.equal(out2, out) and torch.equal(st, ns)
    status_clean()


@pytest.mark.parametrize("channels,stride,dtype", [(8, 8, BF), (7, 7, BF), (1032, 1040, BF),
                                                   (1032, 1037, HF), (131, 140, F32),
                                                   (2052, 2056, F32)])
def test_short_conv_strides_pool_and_flags(channels, stride, dtype):
    lens, W, P = [40, 0, 3, 129], 4, 9
    T, n = sum(lens), len(lens)
    wide = rand(T, stride, dtype=dtype)
    x = wide[:, :channels]
    w = rand(channels, W, dtype=dtype)
    st = rand(P, W - 1, channels, dtype=dtype, seed=3)
    slots = torch.tensor([5, 2, -1, 8]).cuda()
    has = torch.tensor([True, True, True, False]).cuda()
    cu = offsets(lens, torch.int64)
    out = torch.full((T, stride), 7.0, dtype=dtype).cuda()
    ns = st.clone()
    M.gdn_short_conv(x, w, None, st, cu, out[:, :channels], ns, activation=None,
                     state_indices=slots, has_state=has)
    want, pool, mag = O.short_conv(x, w, None, st, cu, st, None, slots, has)
    check(out[:, :channels], want, mag, CONV_REL, "output")
    assert torch.equal(ns.double().cpu(), pool)
    assert (out[:, channels:] == 7).all()        # nothing beside the rows is touched
    status_clean()


@pytest.mark.parametrize("lens", [[17, 16, 15, 300, 1, 1, 0, 3], [2] * 40 + [90] + [1] * 5,
                                  [200] + [1] * 63, [0] * 70, [16] * 9])
@pytest.mark.parametrize("channels", [520, 77])
def test_short_conv_short_beside_long(lens, channels):
    """Sequences on either side of the length up to which one thread does them whole."""
    T, n = sum(lens), len(lens)
    x, w = rand(T, channels, dtype=BF), rand(channels, 4, dtype=BF)
    st = rand(n + 4, 3, channels, dtype=BF, seed=2)
    slots = torch.randperm(n + 4, generator=torch.Generator().manual_seed(n))[:n].cuda()
    slots[n // 2] = -1
    cu = offsets(lens)
    out, ns = torch.full_like(x, float("nan")), st.clone()
    M.gdn_short_conv(x, w, None, st, cu, out, ns, state_indices=slots)
    want, pool, mag = O.short_conv(x, w, None, st, cu, st, "silu", slots)
    check(out, want, mag, CONV_REL, "output")
    assert torch.equal(ns.double().cpu(), pool)
    M.gdn_short_conv(x, w, None, st, cu, again := torch.empty_like(x), st, state_indices=slots)
    assert torch.equal(again, out) and torch.equal(st, ns)
    status_clean()


def test_short_conv_new_prompts_and_uncovered_tokens():
    x, w = rand(50, 64, dtype=BF), rand(64, 4, dtype=BF)
    cu = torch.tensor([5, 20, 41], dtype=torch.int32).cuda()
    out = torch.full_like(x, 3.0)
    ns = torch.empty(2, 3, 64, dtype=BF).cuda()
    M.gdn_short_conv(x, w, None, None, cu, out, ns)
    want, pool, mag = O.short_conv(x, w, None, None, cu, ns)
    check(out[5:41], want[5:41], mag[5:41], CONV_REL, "output")
    assert (out[:5] == 3).all() and (out[41:] == 3).all()
    assert torch.equal(ns.double().cpu(), pool)
    status_clean()


def test_short_conv_many_sequences_and_bad_offsets():
    lens = [(i * 37) % 5 for i in range(1500)]
    x, w = rand(sum(lens), 64, dtype=BF), rand(64, 3, dtype=BF)
    cu = offsets(lens)
    ns = torch.empty(len(lens), 2, 64, dtype=BF).cuda()
    out, new = M.short_conv(x, w, None, None, cu)
    want, pool, mag = O.short_conv(x, w, None, None, cu, ns)
    check(out, want, mag, CONV_REL, "output")
    assert torch.equal(new.double().cpu(), pool)
    status_clean()
    bad = torch.tensor([0, 9, 4, 30], dtype=torch.int32).cuda()
    M.short_conv(x[:20], w, None, None, bad)
    assert _lib.device_status(torch.cuda.current_device()) == _lib.STATUS_BAD_SEQLENS


def test_short_conv_ignores_values_of_other_sequences():
    x, w = rand(70, 64, dtype=BF), rand(64, 4, dtype=BF)
    cu = offsets([33, 37])
    clean, _ = M.short_conv(x, w, None, None, cu)
    x[:33] = float("nan")
    out, ns = M.short_conv(x, w, None, None, cu)
    assert torch.equal(out[33:], clean[33:]) and torch.isfinite(ns[1]).all()


def test_short_conv_output_beside_x_and_not_over_it():
    T, D = 70, 64
    buf = rand(T + 3, 2 * D, dtype=BF)
    x, w, cu = buf[:T, :D], rand(D, 4, dtype=BF), offsets([T])
    want, new = M.short_conv(x, w, None, None, cu)
    ns = torch.empty_like(new)
    keep = buf.clone()
    for over in (x, buf[:T, 1:D + 1], buf[:T, D - 1:2 * D - 1], buf[3:, :D], buf[2:T + 2, D - 8:2 * D - 8],
                 buf.view(-1)[:T * D].view(T, D)):
        with pytest.raises(ValueError, match="overlap"):
            M.gdn_short_conv(x, w, None, None, cu, over, ns)
    assert torch.equal(buf, keep)
    for beside in (buf[:T, D:], buf[3:, D:]):       # the other columns of the same rows, or of others
        M.gdn_short_conv(x, w, None, None, cu, beside, ns)
        assert torch.equal(beside, want) and torch.equal(ns, new) and torch.equal(x, keep[:T, :D])
    one = rand(2, D, dtype=BF)
    M.gdn_short_conv(one[:1], w, None, None, offsets([1]), one[1:], ns)
    with pytest.raises(ValueError, match="overlap"):
        M.gdn_short_conv(one[:1], w, None, None, offsets([1]), one[:1], ns)
    status_clean()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,channels,width", [(1, 64, 4), (7, 1000, 3), (33, 73, 2),
                                                  (64, 8192, 4)])
def test_short_conv_step(dtype, batch, channels, width):
    P = batch + 3
    x, w = rand(batch, channels, dtype=dtype), rand(channels, width, dtype=dtype)
    b = rand(channels, dtype=dtype, seed=5)
    st = rand(P, width - 1, channels, dtype=dtype, seed=6)
    slots = torch.randperm(P, generator=torch.Generator().manual_seed(1))[:batch].int().cuda()
    if batch > 2:
        slots[1] = -1
    cu = torch.arange(batch + 1)
    ns = st.clone()
    out = torch.full_like(x, float("nan"))
    M.gdn_short_conv_step(x, w, b, st, slots, out, new_state_pool=ns)
    want, pool, mag = O.short_conv(x, w, b, st, cu, st, "silu", slots)
    if batch > 2:
        want[1] = 0
    check(out, want, mag, CONV_REL, "output")
    assert torch.equal(ns.double().cpu(), pool)
    assert torch.equal(M.short_conv_step(x, w, b, st, slots), out) and torch.equal(st, ns)
    status_clean()


def test_conv_step_matches_prompt_and_reports_bad_slots():
    x, w = rand(20, 256, dtype=BF), rand(256, 4, dtype=BF)
    out, ns = M.short_conv(x, w, None, None, offsets([20]))
    st = torch.zeros(1, 3, 256, dtype=BF).cuda()
    rows = [M.short_conv_step(x[t:t + 1], w, None, st) for t in range(20)]
    assert torch.equal(torch.cat(rows), out) and torch.equal(st, ns)
    before = st.clone()
    y = M.short_conv_step(x[:1], w, None, st, torch.tensor([1]).cuda())
    assert (y == 0).all() and torch.equal(st, before)
    assert _lib.device_status(torch.cuda.current_device()) == _lib.STATUS_BAD_INDEX


# ------------------------------------------------------------------ selective scan
def scan_inputs(T, H, P, G, N, seed=0, strong=False):
    row = rand(T, H * P + 2 * G * N + 8, dtype=BF, seed=seed)
    x = row[:, :H * P].view(T, H, P)
    B = row[:, H * P:H * P + G * N].view(T, G, N)
    C = row[:, H * P + G * N:H * P + 2 * G * N].view(T, G, N)
    dt = rand(T, H, dtype=BF, seed=seed + 1)
    A_log = torch.log(torch.rand(H, generator=torch.Generator().manual_seed(seed)) * 15 + 1).cuda()
    bias = rand(H, seed=seed + 2) + (1.0 if strong else -3.0)
    return x, dt, A_log, B, C, rand(H, seed=seed + 3), bias


# Step: N + 2 terms in fp32, exp, expm1 and softplus of a few units each.
STEP_REL = 2.0 ** -16
# Prompts: the products' operands are rounded to bf16 (scores and states, 2^-8 of each term,
# and a term is in one of the two); the states themselves come from products split to 24 bits, exponents
# up to 2^7 in fp32 and sums of 128 products, 2^-16 each.
PROMPT_REL, PROMPT_STATE_REL = 2.0 ** -8, 2.0 ** -15


def run_scan(lens, H, P, G, N, *, slots=None, has=None, pool=None, strong=False, seed=0,
             state=True, cu_dtype=torch.int32):
    T, n = sum(lens), len(lens)
    ins = scan_inputs(T, H, P, G, N, seed, strong)
    pool = pool or n
    st = rand(pool, H, P, N, std=0.5, seed=seed + 4) if state else None
    cu = offsets(lens, cu_dtype)
    out = torch.full((T, H, P), float("nan"), dtype=BF).cuda()
    ns = st.clone() if state else torch.full((pool, H, P, N), 9.0).cuda()
    base = ns.clone()
    M.gdn_ssm_prefill(*ins, st, cu, out, ns, state_indices=slots, has_state=has)
    want, wp, mag, pmag = O.scan(*ins, st, cu, base, slots, has)
    check(out, want, mag, PROMPT_REL, "output")
    check(ns, wp, pmag, PROMPT_STATE_REL, "state")
    status_clean()
    return ins, st, cu, out, ns


@pytest.mark.parametrize("P,N", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("lens", [[1], [7, 0, 1], [64], [65, 127, 128, 129], [300, 2, 513]])
def test_scan_lengths(P, N, lens):
    run_scan(lens, 4, P, 2, N)


@pytest.mark.parametrize("P,N", [(64, 128), (128, 64)])
@pytest.mark.parametrize("lens", [[0, 0], [10], [11], [3, 0, 17, 1, 9], [2] * 40, [40] + [0] * 7])
def test_scan_short_sequences(P, N, lens):
    """Around the length below which prompts run token by token."""
    run_scan(lens, 2, P, 2, N, seed=14)


@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (5, 5), (6, 2), (24, 8)])
def test_scan_head_layouts(H, G):
    run_scan([90, 200], H, 64, G, 128, seed=3)


def test_scan_strong_decay_and_zero_state():
    run_scan([400, 129], 4, 64, 1, 128, strong=True, state=False)


# Steep tokens: on top of the roundings, a weight is the exponential of a difference of two
# sums of up to 32 decays of at most 300 in base 2, off by 2^-10 each.
STEEP_REL = PROMPT_REL + 2.0 ** -9


@pytest.mark.parametrize("size", [10.0, 100.0, 1e4, 1e6, 1e30])
@pytest.mark.parametrize("where", ["one", "some", "all"])
@pytest.mark.parametrize("lens", [[200, 70], [1500]])
def test_scan_steep_tokens(size, where, lens):
    """Steps that leave nothing of the state, between ordinary ones: what they decay must
    not cost the weights of the tokens beside them."""
    x, dt, A_log, B, C, D, bias = scan_inputs(sum(lens), 3, 64, 1, 128, seed=71)
    at = {"one": slice(100, 101), "some": slice(33, 160, 3), "all": slice(None)}[where]
    dt[at] = size
    cu, st = offsets(lens), rand(len(lens), 3, 64, 128, std=0.5, seed=72)
    out, ns = torch.empty_like(x).contiguous(), torch.empty_like(st)
    M.gdn_ssm_prefill(x, dt, A_log, B, C, D, bias, st, cu, out, ns)
    want, wp, mag, pmag = O.scan(x, dt, A_log, B, C, D, bias, st, cu, ns)
    check(out, want, mag, STEEP_REL, "output")
    check(ns, wp, pmag, PROMPT_STATE_REL, "state")
    status_clean()


def test_scan_infinite_step_stays_with_its_token_and_those_after():
    x, dt, A_log, B, C, D, bias = scan_inputs(300, 3, 64, 1, 128, seed=73)
    cu, at = offsets([300]), 170
    clean, _ = M.ssm_prefill(x, dt, A_log, B, C, D, bias, None, cu)
    dt[at, 1] = float("inf")
    out, _ = M.ssm_prefill(x, dt, A_log, B, C, D, bias, None, cu)
    assert torch.equal(out[:, [0, 2]], clean[:, [0, 2]]) and torch.equal(out[:128, 1], clean[:128, 1])
    want, _, mag, _ = O.scan(x[:at], dt[:at], A_log, B[:at], C[:at], D, bias, None, [0, at],
                             torch.zeros(1, 3, 64, 128))
    check(out[:at], want, mag, STEEP_REL, "output before")
    assert not torch.isfinite(out[at, 1]).any()
    status_clean()


def test_scan_pool_slots_and_flags():
    slots = torch.tensor([4, -1, 0, 6], dtype=torch.int64).cuda()
    has = torch.tensor([1, 1, 0, 1], dtype=torch.uint8).cuda()
    ins, st, cu, out, ns = run_scan([130, 5, 70, 0], 4, 64, 2, 64, slots=slots, has=has, pool=7,
                                    cu_dtype=torch.int64)
    for s in (1, 2, 3, 5, 6):                     # slots of no sequence, and an empty one's
        assert torch.equal(ns[s], st[s])
    # in place
    M.gdn_ssm_prefill(*ins, st, cu, out2 := torch.empty_like(out), st, state_indices=slots,
                      has_state=has)
    assert torch.equal(out2, out) and torch.equal(st, ns)


def test_scan_long_sequence():
    run_scan([2600], 2, 64, 1, 128, seed=5)
    run_scan([3000, 10, 1111], 2, 128, 2, 64, seed=6)


@pytest.mark.parametrize("strong", [False, True])
def test_scan_divided_sequences_in_place(strong):
    """Few heads and long sequences run in pieces; slots in a pool, updated in place,
    with decays that end within a piece and that reach over several."""
    lens = [1300, 3, 0, 2048, 512, 700]
    slots = torch.tensor([6, 0, 3, 1, -1, 4], dtype=torch.int32).cuda()
    has = torch.tensor([True, True, True, True, True, False]).cuda()
    assert M.ssm_prefill_workspace_bytes(len(lens), sum(lens), 3, 64, 128) > 0
    ins, st, cu, out, ns = run_scan(lens, 3, 64, 1, 128, slots=slots, has=has, pool=8,
                                    strong=strong, seed=21)
    again = torch.empty_like(out)
    M.gdn_ssm_prefill(*ins, st, cu, again, st, state_indices=slots, has_state=has)
    assert torch.equal(again, out) and torch.equal(st, ns)


def test_scan_weak_decay_over_pieces():
    """A head that hardly forgets: every piece counts to the end."""
    ins = list(scan_inputs(2000, 2, 128, 1, 64, seed=31))
    ins[2] = torch.full((2,), -9.0).cuda()               # log decay of about 1e-4 a token
    cu, st = offsets([2000]), rand(1, 2, 128, 64, seed=32)
    out, ns = torch.empty(2000, 2, 128, dtype=BF).cuda(), torch.empty_like(st)
    M.gdn_ssm_prefill(*ins, st, cu, out, ns)
    want, wp, mag, pmag = O.scan(*ins, st, cu, ns)
    check(out, want, mag, PROMPT_REL, "output")
    check(ns, wp, pmag, PROMPT_STATE_REL, "state")
    # the same without a workspace's pieces
    lib = _lib.load()
    x, dt, A_log, B, C, D, bias = ins
    one, ns1 = torch.empty_like(out), torch.empty_like(ns)
    rc = lib.gdn_b200_ssm_prefill(
        x.data_ptr(), x.stride(0), dt.data_ptr(), dt.stride(0), A_log.data_ptr(), B.data_ptr(),
        B.stride(0), C.data_ptr(), C.stride(0), D.data_ptr(), bias.data_ptr(), st.data_ptr(),
        cu.data_ptr(), 0, 0, 0, 0, one.data_ptr(), ns1.data_ptr(), 1, 2000, 1, 2, 1, 128, 64, 0, 0,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    check(one, want, mag, PROMPT_REL, "output")
    check(ns1, wp, pmag, PROMPT_STATE_REL, "state")


def test_scan_pieces_in_parts():
    """70 column units, so a sequence runs in two pieces of 17 chunks, each one's state
    made in two parts; in place."""
    H, T = 70, 34 * 128 - 31
    assert M.ssm_prefill_workspace_bytes(1, T, H, 64, 64) > 0
    x, dt, A_log, B, C, D, bias = scan_inputs(T, H, 64, 1, 64, seed=41)
    st = rand(1, H, 64, 64, seed=42)
    cu, out, ns = offsets([T]), torch.empty(T, H, 64, dtype=BF).cuda(), torch.empty_like(st)
    M.gdn_ssm_prefill(x, dt, A_log, B, C, D, bias, st, cu, out, ns)
    heads = [0, 33, 69]                      # the oracle on a few of the heads
    few = (x[:, heads], dt[:, heads], A_log[heads], B, C, D[heads], bias[heads], st[:, heads])
    want, wp, mag, pmag = O.scan(*few, cu, ns[:, heads])
    check(out[:, heads], want, mag, PROMPT_REL, "output")
    check(ns[:, heads], wp, pmag, PROMPT_STATE_REL, "state")
    again = torch.empty_like(out)
    M.gdn_ssm_prefill(x, dt, A_log, B, C, D, bias, st, cu, again, st)
    assert torch.equal(again, out) and torch.equal(st, ns)
    status_clean()


def test_scan_without_skip_and_bias():
    x, dt, A_log, B, C, _, _ = scan_inputs(150, 4, 64, 1, 64)
    dt = dt - 3
    cu = offsets([150])
    out, ns = M.ssm_prefill(x, dt, A_log, B, C, None, None, None, cu)
    want, wp, mag, pmag = O.scan(x, dt, A_log, B, C, None, None, None, cu, ns)
    check(out, want, mag, PROMPT_REL, "output")
    check(ns, wp, pmag, PROMPT_STATE_REL, "state")


def test_scan_ignores_values_of_other_sequences():
    ins = list(scan_inputs(270, 4, 64, 2, 128))
    cu = offsets([70, 100, 100])
    clean, cs = M.ssm_prefill(*ins, None, cu)
    for k in (0, 1, 3, 4):
        ins[k] = ins[k].clone()
        ins[k][:70] = float("nan")
        ins[k][170:] = float("inf")
    out, ns = M.ssm_prefill(*ins, None, cu)
    assert torch.equal(out[70:170], clean[70:170]) and torch.equal(ns[1], cs[1])


@pytest.mark.parametrize("where", ["dt", "bias", "A_log"])
def test_scan_of_pieces_with_a_nan_step(where):
    """A NaN in the steps of one head, in the last of a piece's 8 chunks, which is the
    first that its state's kernel takes: that head's outputs and state are NaN from there
    on (and from its chunk's start at most), everything else is as without it, and no wait
    runs out.  The head hardly forgets, so that no decay of 0 ends the NaN's reach."""
    H, lens = 16, [8192, 300]
    rows = (67 + 2) // 8                       # whole pieces that the workspace holds
    assert (M.ssm_prefill_workspace_bytes(2, sum(lens), H, 64, 128)
            == rows * (2 * H * 64 * 128 * 4 + H * 4))
    ins = list(scan_inputs(sum(lens), H, 64, 1, 128, seed=61))
    ins[2][3] = -9.0
    cu, at = offsets(lens), 15 * 128 + 50
    clean, cs = M.ssm_prefill(*ins, None, cu)
    k = {"dt": 1, "A_log": 2, "bias": 6}[where]
    ins[k] = ins[k].clone()
    if where == "dt":
        ins[k][at, 3] = float("nan")
    else:
        ins[k][3] = float("nan")
    out, ns = M.ssm_prefill(*ins, None, cu)
    status_clean()
    others = [h for h in range(H) if h != 3]
    assert torch.equal(out[:, others], clean[:, others]) and torch.equal(ns[:, others], cs[:, others])
    assert ns[0, 3].isnan().all()
    if where == "dt":
        begin = at // 128 * 128
        assert torch.equal(out[:begin, 3], clean[:begin, 3]) and out[at:lens[0], 3].isnan().all()
        assert torch.equal(out[lens[0]:], clean[lens[0]:]) and torch.equal(ns[1], cs[1])
    else:
        assert out[:lens[0], 3].isnan().all() and ns[1, 3].isnan().all()


def test_scan_of_nothing():
    ins = scan_inputs(0, 4, 64, 1, 128)
    st = rand(2, 4, 64, 128)
    out, ns = torch.empty(0, 4, 64, dtype=BF).cuda(), torch.empty_like(st)
    M.gdn_ssm_prefill(*ins, st, offsets([0, 0]), out, ns)
    assert torch.equal(ns, st)
    M.gdn_ssm_prefill(*ins, st, offsets([]), out, ns)
    status_clean()


@pytest.mark.parametrize("T", [8, 300, 3000])
def test_scan_output_over_x_is_refused(T):
    """Of any length: pieces of the longest would read what others have written."""
    ins = scan_inputs(T, 2, 64, 1, 128)
    x = ins[0].contiguous()
    ns, keep = torch.zeros(1, 2, 64, 128).cuda(), x.clone()
    with pytest.raises(ValueError, match="overlap"):
        M.gdn_ssm_prefill(x, *ins[1:], None, offsets([T]), x, ns)
    assert torch.equal(x, keep) and (ns == 0).all()
    bc = torch.zeros(T, 2, 128, dtype=BF).cuda()
    for k in (3, 4):
        part = list(ins)
        part[k] = bc[:, :1]
        with pytest.raises(ValueError, match="overlap"):
            M.gdn_ssm_prefill(*part, None, offsets([T]), bc.view(-1)[:T * 128].view(T, 2, 64), ns)
    both = torch.cat([x, torch.zeros_like(x)])
    M.gdn_ssm_prefill(both[:T], *ins[1:], None, offsets([T]), both[T:], ns)
    want, _ = M.ssm_prefill(*ins, None, offsets([T]))
    assert torch.equal(both[T:], want)


def test_scan_bad_offsets_and_slots():
    ins = scan_inputs(40, 4, 64, 1, 64)
    out = torch.zeros(40, 4, 64, dtype=BF).cuda()
    ns = torch.zeros(2, 4, 64, 64).cuda()
    dev = torch.cuda.current_device()
    M.gdn_ssm_prefill(*ins, None, torch.tensor([0, 50, 40], dtype=torch.int32).cuda(), out, ns)
    assert _lib.device_status(dev) == _lib.STATUS_BAD_SEQLENS
    M.gdn_ssm_prefill(*ins, None, offsets([10, 30]), out, ns,
                      state_indices=torch.tensor([0, 2]).cuda())
    assert _lib.device_status(dev) == _lib.STATUS_BAD_INDEX


@pytest.mark.parametrize("in_place", [False, True])
def test_scan_unordered_offsets_stay_in_the_workspace(in_place):
    """Offsets that return to the start: the first sequence takes the workspace that
    8192 tokens account for (16 pieces of 4 chunks, 17 rows), the later ones are skipped.
    What lies behind the workspace is NaN, and is neither read nor written."""
    H, P, N, T = 8, 64, 128, 8192
    ins = scan_inputs(T, H, P, 1, N, seed=51)
    cu = torch.tensor([0, T] * 4, dtype=torch.int32).cuda()
    need = M.ssm_prefill_workspace_bytes(7, T, H, P, N)
    assert need == 17 * (2 * H * P * N * 4 + H * 4)
    ws = torch.full((4 * need // 4,), float("nan"), device="cuda")
    st = rand(7, H, P, N, std=0.5, seed=52)
    base = st.clone()
    ns = st if in_place else st.clone()
    out = torch.empty(T, H, P, dtype=BF).cuda()
    M.gdn_ssm_prefill(*ins, st, cu, out, ns, workspace=ws.view(torch.uint8)[:need])
    assert _lib.device_status(torch.cuda.current_device()) == _lib.STATUS_BAD_SEQLENS
    want, wp, mag, pmag = O.scan(*ins, base[:1], cu[:2], base[:1])
    check(out, want, mag, PROMPT_REL, "output")
    check(ns[:1], wp, pmag, PROMPT_STATE_REL, "state")
    assert torch.equal(ns[1:], base[1:]) and ws[need // 4:].isnan().all()


@pytest.mark.parametrize("P,N", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("batch,H,G", [(1, 4, 1), (5, 6, 3), (33, 2, 2)])
def test_scan_step(P, N, batch, H, G):
    S = batch + 2
    ins = scan_inputs(batch, H, P, G, N, seed=9)
    st = rand(S, H, P, N, seed=1)
    slots = torch.randperm(S, generator=torch.Generator().manual_seed(2))[:batch].int().cuda()
    if batch > 2:
        slots[2] = -1
    cu = torch.arange(batch + 1)
    out = torch.full((batch, H, P), float("nan"), dtype=BF).cuda()
    ns = st.clone()
    M.gdn_ssm_step(*ins, st, slots, out, new_state_pool=ns)
    want, wp, mag, pmag = O.scan(*ins, st, cu, st, slots)
    if batch > 2:
        want[2], mag[2] = 0, 0
    check(out, want, mag, STEP_REL, "output")
    check(ns, wp, pmag, STEP_REL, "state")
    assert torch.equal(M.ssm_step(*ins, st, slots), out) and torch.equal(st, ns)
    status_clean()


def test_scan_step_write_slots_and_bad_slot():
    ins = scan_inputs(2, 4, 64, 1, 128)
    st = rand(6, 4, 64, 128)
    read, write = torch.tensor([0, 1]).cuda(), torch.tensor([4, -1]).cuda()
    keep = st.clone()
    out = torch.empty(2, 4, 64, dtype=BF).cuda()
    M.gdn_ssm_step(*ins, st, read, out, output_state_indices=write)
    want, wp, mag, pmag = O.scan(*ins, keep, torch.arange(3), keep, read, None, write)
    check(out, want, mag, STEP_REL, "output")
    check(st, wp, pmag, STEP_REL, "state")
    assert torch.equal(st[:4], keep[:4]) and torch.equal(st[5], keep[5])
    status_clean()
    y = M.ssm_step(*ins, st, torch.tensor([6, 0]).cuda())
    assert (y[0] == 0).all()
    assert _lib.device_status(torch.cuda.current_device()) == _lib.STATUS_BAD_INDEX


def test_scan_steps_follow_a_prompt():
    """A prompt's last tokens one by one from the state of its first part."""
    ins = scan_inputs(140, 4, 64, 1, 128, seed=11)
    out, ns = M.ssm_prefill(*ins, None, offsets([140]))
    part = [t[:132] if t.shape[0] == 140 else t for t in ins]
    _, st = M.ssm_prefill(*part, None, offsets([132]))
    want, wp, mag, pmag = O.scan(*ins, None, torch.tensor([0, 140]), ns)
    for t in range(132, 140):
        one = [v[t:t + 1] if v.shape[0] == 140 else v for v in ins]
        y = M.ssm_step(*one, st)
        check(y, want[t:t + 1], mag[t:t + 1], PROMPT_REL, "step")
    check(st, wp, pmag, PROMPT_STATE_REL, "state")


# ------------------------------------------------------------------ norms
NORM_REL = 2.0 ** -18      # the sum of squares over up to 2^13 elements by a tree, exp, rsqrt


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,group", [(128, 128), (512, 64), (96, 32), (4096, 128), (2048, 2048),
                                         (7000, 7000), (3 * 264, 264), (1000, 1000), (777, 777),
                                         (30, 3), (40960, 40960)])
@pytest.mark.parametrize("norm_first", [True, False])
def test_gated_norm(dtype, width, group, norm_first):
    rows = 5
    x, gate = rand(rows, width, dtype=dtype), rand(rows, width + 8, dtype=dtype, seed=1)[:, :width]
    for shared in (True, False):
        w = rand(group if shared else width, dtype=dtype, seed=2)
        out = torch.full_like(x, float("nan"))
        act = "silu" if shared else "sigmoid"
        M.gdn_gated_norm(x, gate, w, out, group_size=group, activation=act, norm_first=norm_first)
        want = O.gated_norm(x, gate, w, group, 1e-6, act, norm_first)
        check(out, want, want.abs(), NORM_REL, "output")


def test_gated_norm_heads_in_place_and_plain():
    x, gate = rand(37, 32, 128, dtype=BF), rand(37, 32, 128, dtype=BF, seed=1)
    w = rand(128, dtype=BF, seed=2)
    want = O.gated_norm(x, gate, w, 128, 1e-5)
    out = M.gated_norm(x, gate, w, eps=1e-5)
    assert out.shape == x.shape
    check(out, want, want.abs(), NORM_REL, "output")
    plain = M.gated_norm(x, None, None)
    wp = O.gated_norm(x, None, None, 128, 1e-6)
    check(plain, wp, wp.abs(), NORM_REL, "no gate, no weight")
    M.gdn_gated_norm(x, gate, w, x, eps=1e-5)
    assert torch.equal(x, out)


def test_gated_norm_extremes():
    x = torch.zeros(4, 256, dtype=BF).cuda()
    gate = rand(4, 256, dtype=BF)
    assert (M.gated_norm(x, gate, None) == 0).all()                 # 0 / sqrt(eps)
    x[1] = 1.0
    gate[1] = -300.0                                                # exp overflows: the gate is 0
    gate[2] = 300.0
    out = M.gated_norm(x, gate, None)
    assert torch.isfinite(out).all() and (out[1] == 0).all()
    x[3] = float("nan")
    out = M.gated_norm(x, gate, None)
    assert torch.isfinite(out[:3]).all() and out[3].isnan().all()
    assert M.gated_norm(x[:0], gate[:0], None).shape == (0, 256)


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("norm_first", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,group", [(256, 64), (1024, 1024), (154, 77)])
def test_gated_norm_keeps_a_nan_gate(activation, norm_first, dtype, width, group):
    """Of any alignment: a NaN in a gate is its element's, or through the sum of squares
    its group's, and no other's."""
    x, gate = rand(3, width, dtype=dtype), rand(3, width, dtype=dtype, seed=1)
    want = O.gated_norm(x, gate, None, group, 1e-6, activation, norm_first)
    gate[1, 5] = float("nan")
    out = M.gated_norm(x, gate, None, group_size=group, activation=activation,
                       norm_first=norm_first)
    hit = torch.zeros(3, width, dtype=torch.bool)
    hit[1, slice(5, 6) if norm_first else slice(0, group)] = True
    assert out[hit].isnan().all()
    check(out[~hit], want[~hit], want[~hit].abs(), NORM_REL, "output")


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("width", [256, 77])
def test_far_ends_of_activations(activation, width):
    """In fp32, relative to the result, down to gates of -80.  The exponent's rounding
    leaves 1.5 |v| 2^-24; the norm and the rest 2^-18 as above."""
    v = torch.linspace(-80, 80, 6 * width).view(6, width)[:, torch.randperm(
        width, generator=torch.Generator().manual_seed(3))].cuda()
    x = rand(6, width).abs() + 0.5
    rel = (2.0 ** -18 + 1.5 * 2.0 ** -24 * v.abs().double()).cpu()
    for norm_first in (True, False):
        out = M.gated_norm(x, v, None, activation=activation, norm_first=norm_first).cpu().double()
        want = O.gated_norm(x, v, None, width, 1e-6, activation, norm_first)
        normal = want.abs() > 1e-36
        assert normal.sum() > 0.9 * normal.numel()
        # before the norm, the largest gates' errors are in the sum too
        bound = rel if norm_first else rel + rel.max()
        assert ((out - want).abs() <= bound * want.abs())[normal].all()
    if activation == "silu":                  # the same of a convolution of one tap
        w = torch.tensor([0.0, 1.0]).repeat(width, 1).cuda()
        out, _ = M.short_conv(v, w, None, None, offsets([6]))
        want, _, _ = O.short_conv(v, w, None, None, [0, 6], torch.zeros(1, 1, width))
        assert ((out.cpu().double() - want).abs() <= rel * want.abs()).all()


@pytest.mark.parametrize("dtype,rdt", [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)])
@pytest.mark.parametrize("width", [8, 256, 520, 1000, 2048, 5000, 8192, 33, 36864])
@pytest.mark.parametrize("post", [True, False])
def test_add_norm(dtype, rdt, width, post):
    rows = 6
    x, r = rand(rows, width, dtype=dtype), rand(rows, width, dtype=rdt, std=2.0, seed=1)
    w, bw = rand(width, dtype=dtype, seed=2), rand(width, dtype=dtype, seed=3) if post else None
    scale = (rand(width, seed=4) if post else 0.25)
    out, nr = M.add_norm(x, r, w, block_weight=bw, scale=scale, weight_offset=1.0)
    want, wr, mag = O.add_norm(x, r, w, bw, scale, 1e-6, 1.0)
    check(nr, wr, mag, NORM_REL, "residual")
    # an error in the sum shows in the norm in the same proportion to its row's size
    rms = wr.square().mean(1, keepdim=True).sqrt()
    check(out, want, want.abs() + mag / rms * (w.double().cpu().abs() + 1), NORM_REL, "output")
    M.gdn_add_norm(x, r, w, x, r, block_weight=bw, scale=scale, weight_offset=1.0)
    assert torch.equal(x, out) and torch.equal(r, nr)


def test_add_norm_strided_rows():
    x, r = rand(9, 520, dtype=BF)[:, :512], rand(9, 515, seed=1)[:, :512]
    w = rand(512, dtype=BF, seed=2)
    out, nr = torch.zeros(9, 512, dtype=BF).cuda(), torch.zeros(9, 600).cuda()[:, 3:515]
    M.gdn_add_norm(x, r, w, out, nr)
    want, wr, mag = O.add_norm(x, r, w)
    rms = wr.square().mean(1, keepdim=True).sqrt()
    check(nr, wr, mag, NORM_REL, "residual")
    check(out, want, want.abs() + mag / rms * w.double().cpu().abs(), NORM_REL, "output")


# ------------------------------------------------------------------ streams
def test_calls_follow_the_current_stream():
    x, w = rand(4096, 1024, dtype=BF), rand(1024, 4, dtype=BF)
    cu = offsets([4096])
    want, _ = M.short_conv(x, w, None, None, cu)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    late = torch.zeros_like(x)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(20):
            late.copy_(x)
        got, _ = M.short_conv(late, w, None, None, cu)
        ref = got.clone()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(ref, want)


@pytest.mark.parametrize("lens", [[150, 50], [1450, 50]])
def test_calls_are_captured_in_a_graph(lens):
    T = sum(lens)
    ins = scan_inputs(T, 4, 64, 1, 128)
    cu = offsets(lens)
    out, ns = torch.empty(T, 4, 64, dtype=BF).cuda(), torch.empty(2, 4, 64, 128).cuda()
    need = M.ssm_prefill_workspace_bytes(2, T, 4, 64, 128)
    assert (need > 0) == (T > 1000)              # the longer one runs in pieces
    ws = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    M.gdn_ssm_prefill(*ins, None, cu, out, ns, workspace=ws)
    want, ws_want = out.clone(), ns.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        M.gdn_ssm_prefill(*ins, None, cu, out, ns, workspace=ws)
    for _ in range(3):
        out.zero_(), ns.zero_(), ws.zero_()
        g.replay()
        g.replay()
        assert torch.equal(out, want) and torch.equal(ns, ws_want)


def test_calls_on_two_streams_with_workspaces_of_their_own():
    a = [scan_inputs(T, 8, 64, 2, 128, seed=T) for T in (3000, 2500)]
    cu = [offsets([3000]), offsets([2000, 500])]
    want = [M.ssm_prefill(*i, None, c) for i, c in zip(a, cu)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(M.ssm_prefill(*a[k], None, cu[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for out, ns in got[k]:
            assert torch.equal(out, want[k][0]) and torch.equal(ns, want[k][1])
    status_clean()
