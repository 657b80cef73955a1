"""The mixer operators' refusals, at the C entry and in Python (no GPU needed),
and their oracle against torch's own forms."""

import ctypes

import pytest
import torch

from gdn_kernel_b200 import _lib, mixer as M
from oracle import mixer_oracle as O

Z = ctypes.c_void_p(0)
BAD = _lib.GDN_B200_ERR_INVALID_ARGUMENT


def _conv(lib, n=1, t=4, pool=1, channels=64, width=4, dtype=_lib.BF16, act=1, xs=64):
    return lib.gdn_b200_short_conv(Z, xs, Z, Z, Z, Z, 0, Z, 0, Z, act, Z, xs, Z, n, t, pool,
                                   channels, width, dtype, Z)


def _conv_step(lib, b=2, pool=2, channels=64, width=4, dtype=_lib.BF16, act=1):
    return lib.gdn_b200_short_conv_step(Z, 64, Z, Z, Z, Z, 0, act, Z, 64, Z, b, pool, channels,
                                        width, dtype, Z)


def _scan(lib, n=1, t=4, pool=1, H=4, G=1, P=64, N=128):
    return lib.gdn_b200_ssm_prefill(Z, 1, Z, 1, Z, Z, 1, Z, 1, Z, Z, Z, Z, 0, Z, 0, Z, Z, Z, n, t,
                                    pool, H, G, P, N, Z, 0, Z)


def _scan_step(lib, b=2, pool=2, H=4, G=1, P=64, N=128):
    return lib.gdn_b200_ssm_step(Z, 1, Z, 1, Z, Z, 1, Z, 1, Z, Z, Z, Z, Z, 0, Z, Z, b, pool, H, G,
                                 P, N, Z)


def _gated(lib, rows=2, width=128, group=64, eps=1e-6, act=1, dtype=0):
    return lib.gdn_b200_gated_norm(Z, width, Z, width, Z, 1, Z, width, rows, width, group, eps, act,
                                   1, dtype, Z)


def _add(lib, rows=2, width=128, eps=1e-6, dtype=0):
    return lib.gdn_b200_add_norm(Z, width, Z, width, Z, Z, Z, 1.0, Z, width, Z, width, rows, width,
                                 eps, 0.0, dtype, 0, Z)


@pytest.mark.parametrize("fn,kw,word", [
    (_conv, dict(width=5), b"width"), (_conv, dict(width=1), b"width"),
    (_conv, dict(channels=0), b"channels"), (_conv, dict(dtype=3), b"dtype"),
    (_conv, dict(act=2), b"activation"), (_conv, dict(t=-1), b"extents"),
    (_conv, dict(n=-1), b"num_seqs"), (_conv, {}, b"null"),
    (_conv, dict(t=2 ** 30 + 1), b"total_tokens"),
    (_conv_step, dict(width=7), b"width"), (_conv_step, dict(b=-1), b"extents"),
    (_conv_step, {}, b"null"),
    (_scan, dict(P=96), b"head_dim"), (_scan, dict(N=32), b"state_dim"),
    (_scan, dict(H=5, G=2), b"multiple"), (_scan, dict(G=0), b"multiple"),
    (_scan, dict(n=70000), b"num_seqs"), (_scan, dict(t=-2), b"extents"), (_scan, {}, b"null"),
    (_scan_step, dict(P=32), b"head_dim"), (_scan_step, dict(b=70000), b"batch"),
    (_scan_step, {}, b"null"),
    (_gated, dict(group=48), b"multiple"), (_gated, dict(group=0), b"multiple"),
    (_gated, dict(act=0), b"activation"), (_gated, dict(eps=-1.0), b"eps"),
    (_gated, dict(eps=float("nan")), b"eps"), (_gated, dict(dtype=9), b"dtype"),
    (_gated, {}, b"null"),
    (_add, dict(width=0), b"width"), (_add, dict(rows=-1), b"rows"), (_add, dict(dtype=-1), b"dtype"),
    (_add, dict(eps=-1.0), b"eps"), (_add, {}, b"null"),
])
def test_c_entry_refuses(fn, kw, word):
    lib = _lib.load()
    assert fn(lib, **kw) == BAD
    assert word in lib.gdn_b200_last_error()


@pytest.mark.parametrize("fn,kw", [(_conv, dict(n=0)), (_conv_step, dict(b=0)), (_scan, dict(n=0)),
                                   (_scan_step, dict(b=0)), (_gated, dict(rows=0)),
                                   (_add, dict(rows=0))])
def test_nothing_to_do_is_no_error(fn, kw):
    lib = _lib.load()
    assert fn(lib, **kw) == _lib.GDN_B200_OK
    assert lib.gdn_b200_last_error() == b""


@pytest.mark.skipif(torch.cuda.is_available(), reason="its addresses hold nothing")
@pytest.mark.parametrize("rows,width,stride,start", [
    (9, 64, 64, 0), (9, 64, 64, 5 * 64), (9, 64, 64, -8 * 64), (9, 64, 64, 575), (9, 64, 64, -575),
    (9, 64, 200, 63), (9, 64, 200, -63), (9, 64, 200, 137), (9, 64, 200, 8 * 200 + 63),
    (1, 64, 64, 10), (9, 64, 200, 64), (9, 64, 200, 136), (9, 64, 200, -64), (9, 64, 200, -136),
    (9, 64, 64, 576), (9, 64, 64, -576), (9, 64, 200, 8 * 200 + 64), (9, 64, 200, 9 * 200),
    (9, 64, 200, 9 * 200 - 63), (1, 64, 64, 64), (9, 64, 200, 3 * 200 + 100)])
def test_convolution_output_over_its_input(rows, width, stride, start):
    """Refused exactly where an element of a row is one of another."""
    a = {r * stride + c for r in range(rows) for c in range(width)}
    b = {start + e for e in a}
    lib, x = _lib.load(), 1 << 20
    one = ctypes.c_void_p(256)
    rc = lib.gdn_b200_short_conv(ctypes.c_void_p(x), stride, one, Z, Z, one, 0, Z, 0, Z, 1,
                                 ctypes.c_void_p(x + 2 * start), stride, one, 1, rows, 1, width, 4,
                                 _lib.BF16, Z)
    assert (rc == BAD and b"overlap" in lib.gdn_b200_last_error()) == bool(a & b)


@pytest.mark.parametrize("seqs,tokens,H,P,N", [
    (1, 512, 8, 1, 64), (1, 512, 8, 32, 64), (1, 512, 8, 63, 128), (1, 512, 8, 96, 64),
    (1, 512, 8, 256, 64), (1, 512, 8, 64, 32), (1, 512, 8, 64, 0), (1, 512, 0, 64, 64),
    (1, 512, 70000, 64, 64), (0, 512, 8, 64, 64), (-1, 512, 8, 64, 64), (70000, 2 ** 20, 8, 64, 64),
    (1, 2 ** 40, 8, 64, 64), (1, -5, 8, 64, 64)])
def test_workspace_of_refused_sizes_is_nothing(seqs, tokens, H, P, N):
    lib = _lib.load()
    assert lib.gdn_b200_ssm_prefill_workspace_size(seqs, tokens, H, P, N) == 0
    assert M.ssm_prefill_workspace_bytes(seqs, tokens, H, P, N) == 0
    assert M.ssm_prefill_workspace_bytes(1, 512, 8, 64, 64) > 0


BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


CU = torch.tensor([0, 4], dtype=torch.int32)


def conv(x=z(4, 64), weight=z(64, 4), bias=None, state=None, cu=CU, output=z(4, 64),
         new_state=z(1, 3, 64), **kw):
    M.gdn_short_conv(x, weight, bias, state, cu, output, new_state, **kw)


def conv_step(x=z(4, 64), weight=z(64, 4), bias=None, state_pool=z(4, 3, 64), slots=None,
              output=z(4, 64), **kw):
    M.gdn_short_conv_step(x, weight, bias, state_pool, slots, output, **kw)


def scan(x=z(4, 2, 64), dt=z(4, 2), A_log=z(2, dtype=torch.float32), B=z(4, 1, 128),
         C=z(4, 1, 128), D=None, dt_bias=None, state=None, cu=CU, output=z(4, 2, 64),
         new_state=z(1, 2, 64, 128, dtype=torch.float32), **kw):
    M.gdn_ssm_prefill(x, dt, A_log, B, C, D, dt_bias, state, cu, output, new_state, **kw)


def scan_step(x=z(4, 2, 64), dt=z(4, 2), A_log=z(2, dtype=torch.float32), B=z(4, 1, 128),
              C=z(4, 1, 128), D=None, dt_bias=None, pool=z(4, 2, 64, 128, dtype=torch.float32),
              slots=None, output=z(4, 2, 64), **kw):
    M.gdn_ssm_step(x, dt, A_log, B, C, D, dt_bias, pool, slots, output, **kw)


def gated(x=z(4, 64), gate=z(4, 64), weight=z(64), output=z(4, 64), **kw):
    M.gdn_gated_norm(x, gate, weight, output, **kw)


def add(x=z(4, 64), residual=z(4, 64), weight=z(64), output=z(4, 64), new_residual=z(4, 64), **kw):
    M.gdn_add_norm(x, residual, weight, output, new_residual, **kw)


F32, I32, I64 = torch.float32, torch.int32, torch.int64


@pytest.mark.parametrize("call,kw,words", [
    # what is right but not on a GPU, last of all checks
    (conv, {}, "CUDA"), (conv_step, {}, "CUDA"), (scan, {}, "CUDA"), (scan_step, {}, "CUDA"),
    (gated, {}, "CUDA"), (add, {}, "CUDA"),
    (gated, dict(x=z(4, 130)[:, :64], gate=z(4, 72)[:, :64]), "CUDA"),     # row strides are free
    (scan, dict(x=z(4, 200)[:, :128].view(4, 2, 64), D=z(2, dtype=F32)), "CUDA"),
    # types
    (conv, dict(x=z(4, 64, dtype=torch.int32)), "x: expected bfloat16"),
    (conv, dict(weight=z(64, 4, dtype=F32)), "weight: wrong dtype"),
    (conv, dict(state=z(1, 3, 64, dtype=F32)), "state: wrong dtype"),
    (conv, dict(cu=CU.float()), "cu_seqlens: must be int32 or int64"),
    (conv, dict(state_indices=z(1, dtype=F32)), "state_indices: must be"),
    (conv, dict(has_state=z(1, dtype=I32)), "has_state: must be bool or uint8"),
    (scan, dict(x=z(4, 2, 64, dtype=F32)), "x: wrong dtype"),
    (scan, dict(A_log=z(2)), "A_log: wrong dtype"), (scan, dict(dt=z(4, 2, dtype=F32)), "dt"),
    (scan_step, dict(slots=torch.arange(4), output_state_indices=torch.arange(4, dtype=I32)),
     "output_state_indices"),
    (gated, dict(weight=z(64, dtype=F32)), "weight: wrong dtype"),
    (add, dict(residual=z(4, 64, dtype=torch.float16)), "residual"),
    (add, dict(residual=z(4, 64, dtype=F32)), "new_residual: wrong dtype"),
    (add, dict(scale=z(64)), "scale: wrong dtype"),
    # shapes
    (conv, dict(weight=z(64, 5)), "width"), (conv, dict(weight=z(64)), "weight"),
    (conv, dict(x=z(4, 60)), "x: expected shape \\(4, 64\\), got \\(4, 60\\)"),
    (conv, dict(output=z(5, 64)), "output: expected shape"), (conv, dict(bias=z(63)), "bias"),
    (conv, dict(new_state=z(1, 2, 64)), "new_state"), (conv, dict(new_state=z(64)), "new_state"),
    (conv, dict(new_state=z(0, 3, 64)), "0 rows, 1 are needed"),
    (conv, dict(cu=z(1, 2, dtype=I32)), "cu_seqlens"),
    (conv, dict(state_indices=z(2, dtype=I64)), "state_indices: expected shape"),
    (conv, dict(x=z(4, 8, 8)), "two dimensions"),
    (conv_step, dict(state_pool=z(3, 3, 64)), "3 rows, 4 are needed"),
    (conv_step, dict(new_state_pool=z(3, 3, 64)), "new_state_pool"),
    (scan, dict(x=z(4, 2, 96), output=z(4, 2, 96)), "head_dim"), (scan, dict(x=z(4, 128)), "x"),
    (scan, dict(B=z(4, 1, 32)), "state_dim"), (scan, dict(C=z(4, 1, 64)), "C: expected shape"),
    (scan, dict(x=z(4, 3, 64), B=z(4, 2, 128)), "multiple"), (scan, dict(D=z(3, dtype=F32)), "D"),
    (scan, dict(dt=z(3, 2)), "dt"), (scan, dict(new_state=z(1, 2, 64, dtype=F32)), "new_state"),
    (scan_step, dict(pool=z(3, 2, 64, 128, dtype=F32)), "3 rows, 4 are needed"),
    (gated, dict(group_size=48), "divide"), (gated, dict(group_size=0), "group_size"),
    (gated, dict(weight=z(32)), "weight: expected"), (gated, dict(gate=z(4, 32)), "gate"),
    (gated, dict(x=z(64)), "must be"), (add, dict(weight=z(63)), "weight"),
    (add, dict(x=z(4, 0)), "empty"), (add, dict(block_weight=z(63)), "block_weight"),
    # layouts
    (conv, dict(x=z(64, 4).t()), "x: must be contiguous within a row"),
    (conv, dict(state=z(1, 64, 3).transpose(1, 2)), "state: must be contiguous"),
    (scan, dict(x=z(4, 2, 128)[:, :, ::2]), "x: must be contiguous within a row"),
    (scan, dict(B=z(4, 256).view(4, 2, 128)[:, ::2]), "CUDA"),
    (gated, dict(weight=z(128)[::2]), "weight: must be contiguous"),
    (add, dict(output=z(4, 128)[:, ::2]), "output: must be contiguous within a row"),
    # words
    (conv, dict(activation="sigmoid"), "activation"), (gated, dict(activation=None), "activation"),
])
def test_python_refuses(call, kw, words):
    with pytest.raises(ValueError, match=words):
        call(**kw)


@pytest.mark.parametrize("kw,words", [
    (dict(B=z()), "B: must be"), (dict(B=z(128)), "B: must be"), (dict(x=z()), "x: must be"),
    (dict(cu=torch.tensor(4)), "cu_seqlens"), (dict(cu=z(0, dtype=I32)), "cu_seqlens")])
def test_scan_refuses_what_has_no_sizes_to_plan_for(kw, words):
    with pytest.raises(ValueError, match=words):
        scan(**kw)


@pytest.mark.parametrize("P", [1, 32, 63])
def test_python_refuses_small_heads_before_planning(P):
    with pytest.raises(ValueError, match="head_dim"):
        scan(x=z(512, 2, P), dt=z(512, 2), B=z(512, 1, 128), C=z(512, 1, 128), output=z(512, 2, P),
             cu=torch.tensor([0, 512], dtype=torch.int32))


# ------------------------------------------------------------------ the oracle
def test_oracle_convolution_is_a_causal_conv1d():
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(50, 6, generator=g), torch.randn(6, 4, generator=g)
    b = torch.randn(6, generator=g)
    ns = torch.zeros(1, 3, 6)
    out, pool, _ = O.short_conv(x, w, b, None, [0, 50], ns)
    want = torch.nn.functional.conv1d(x.t()[None].double(), w[:, None].double(), b.double(),
                                      padding=3, groups=6)[0, :, :50]
    torch.testing.assert_close(out, torch.nn.functional.silu(want).t())
    # two pieces with the carried state are the whole
    first, p1, _ = O.short_conv(x[:2], w, b, None, [0, 2], ns)
    second, p2, _ = O.short_conv(x[2:], w, b, p1, [0, 48], ns)
    torch.testing.assert_close(torch.cat([first, second]), out)
    assert torch.equal(p2, pool)


def test_oracle_scan_is_its_closed_form():
    """y_t = sum_s exp(sum of log decays over (s, t]) (C_t . B_s) step_s x_s + D x_t."""
    g = torch.Generator().manual_seed(1)
    T, H, P, G, N = 20, 4, 3, 2, 5
    x, dt = torch.randn(T, H, P, generator=g), torch.randn(T, H, generator=g)
    B, C = torch.randn(T, G, N, generator=g), torch.randn(T, G, N, generator=g)
    A_log, D, bias = (torch.randn(H, generator=g) for _ in range(3))
    ns = torch.zeros(1, H, P, N)
    out, pool, mag, pmag = O.scan(x, dt, A_log, B, C, D, bias, None, [0, T], ns)
    step = torch.nn.functional.softplus(dt.double() + bias)
    c = (-torch.exp(A_log.double()) * step).cumsum(0)
    decay = torch.exp(c[:, None] - c[None]).masked_fill(
        torch.ones(T, T).triu(1).bool()[..., None], 0.0)              # [t, s, H]
    cb = torch.einsum("tgn,sgn->tsg", C.double(), B.double()).repeat_interleave(2, 2)
    want = torch.einsum("tsh,tsh,sh,shp->thp", cb, decay, step, x.double())
    torch.testing.assert_close(out, want + D.double()[:, None] * x)
    w = torch.exp(c[-1] - c) * step
    torch.testing.assert_close(pool[0], torch.einsum(
        "sh,shp,shn->hpn", w, x.double(), B.double().repeat_interleave(2, 1)))
    assert (mag >= out.abs() - 1e-12).all() and (pmag >= pool.abs() - 1e-12).all()


def test_oracle_norms_are_torchs():
    g = torch.Generator().manual_seed(2)
    x, z, w = torch.randn(5, 24, generator=g), torch.randn(5, 24, generator=g), torch.randn(24)
    rms = lambda v, n: torch.nn.functional.rms_norm(v, (n,), eps=1e-6)  # noqa: E731
    silu = torch.nn.functional.silu(z.double())
    torch.testing.assert_close(O.gated_norm(x, z, w, 24, 1e-6), rms(x.double(), 24) * w * silu)
    torch.testing.assert_close(
        O.gated_norm(x, z, w[:8], 8, 1e-6, norm_first=False),
        (rms((x * silu).view(5, 3, 8), 8) * w[:8]).view(5, 24))
    out, r, _ = O.add_norm(x, z, w, scale=0.5, weight_offset=1.0)
    torch.testing.assert_close(r, z.double() + 0.5 * x)
    torch.testing.assert_close(out, rms(z.double() + 0.5 * x, 24) * (w + 1.0))
