"""CPU checks of the recurrent-block operators: the C ABI refuses bad arguments before it looks
at any pointer or device, and the 64-bit references agree with independent formulations."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import block_ref as R
from matmulfreellmcpu_b200 import _lib, api

P = 0x1000  # a non-null pointer that no refused call touches


def conv_args(**kw):
    a = dict(out=P, x=P, weight=P, ld_out=16, ldx=16, tokens=4, seqs=1, slot_count=1, channels=16, width=4, type=0, silu=1)
    a.update(kw)
    return _lib.ConvArgs(**a)


def ssm_args(**kw):
    a = dict(out=P, x=P, dt=P, B=P, C=P, A=P, ld_out=16, ldx=16, ld_dt=16, ldb=4, ldc=4, tokens=4, seqs=1, slot_count=1,
             channels=16, states=4, groups=1, type=0, dt_softplus=1)
    a.update(kw)
    return _lib.SsmArgs(**a)


@pytest.mark.parametrize("bad", [
    dict(out=None), dict(x=None), dict(weight=None), dict(width=1), dict(width=9), dict(type=3), dict(type=-1),
    dict(channels=0), dict(channels=1 << 40), dict(seqs=2), dict(slots=P), dict(state=P, slot_count=0),
    dict(ld_out=15), dict(tokens=1 << 40), dict(seqs=70000, seq_starts=P)])
def test_conv_refusals(bad):
    lib = _lib.lib()
    assert lib.mmfree_cuda_causal_conv(C.byref(conv_args(**bad)), None) == _lib.E_INVALID
    assert b"conv" in lib.mmfree_cuda_last_error()
    step = dict(tokens=1, seqs=1, state=P)
    if set(bad) <= {"out", "x", "weight", "width", "type", "channels"}:
        assert lib.mmfree_cuda_causal_conv_step(C.byref(conv_args(**{**step, **bad})), None) == _lib.E_INVALID
    assert lib.mmfree_cuda_causal_conv_step(C.byref(conv_args(tokens=2, seqs=1, state=P)), None) == _lib.E_INVALID
    assert lib.mmfree_cuda_causal_conv(None, None) == _lib.E_INVALID


@pytest.mark.parametrize("bad", [
    dict(out=None), dict(x=None), dict(dt=None), dict(A=None), dict(B=None), dict(C=None), dict(states=0), dict(states=257),
    dict(groups=0), dict(groups=3), dict(type=4), dict(channels=0, groups=1), dict(seqs=3), dict(slots=P), dict(ld_out=3),
    dict(state=P, slot_count=0)])
def test_ssm_refusals(bad):
    lib = _lib.lib()
    assert lib.mmfree_cuda_selective_scan(C.byref(ssm_args(**bad)), None) == _lib.E_INVALID
    assert lib.mmfree_cuda_selective_step(C.byref(ssm_args(tokens=1, seqs=1)), None) == _lib.E_INVALID  # no state
    assert lib.mmfree_cuda_selective_step(None, None) == _lib.E_INVALID


def test_norm_quant_and_int4_refusals():
    lib = _lib.lib()
    good = dict(codes=P, scales=P, x=P, ldx=64, residual=None, ldr=64, weight=P, rows=2, cols=64, eps=1e-6, type=0, code=3, group=0)
    for bad in (dict(codes=None), dict(scales=None), dict(x=None), dict(weight=None), dict(cols=0), dict(cols=60000), dict(type=3),
                dict(code=0), dict(group=48), dict(residual=P, ldr=63), dict(rows=1 << 40)):
        assert lib.mmfree_cuda_add_rmsnorm_quant(*{**good, **bad}.values(), None) == _lib.E_INVALID, bad
    good = dict(out=P, x=P, ldx=64, xs=None, codes=P, ldc=32, scales=P, zeros=None, rows=1, k=64, n=8, group=32, xg=0, xt=0, st=2, ot=0)
    for bad in (dict(out=None), dict(x=None), dict(codes=None), dict(scales=None), dict(k=0), dict(n=0), dict(k=60000), dict(ldc=31),
                dict(group=0), dict(group=40), dict(xt=5), dict(xt=-1), dict(st=3), dict(ot=4), dict(xt=3), dict(xs=P), dict(xg=32),
                dict(xt=3, xs=P, xg=64)):
        assert lib.mmfree_cuda_int4_matvec(*{**good, **bad}.values(), None) == _lib.E_INVALID, bad


def test_nothing_to_do_needs_no_device():
    lib = _lib.lib()
    assert lib.mmfree_cuda_causal_conv(C.byref(conv_args(tokens=0)), None) == 0
    assert lib.mmfree_cuda_selective_scan(C.byref(ssm_args(tokens=0)), None) == 0
    assert lib.mmfree_cuda_add_rmsnorm_quant(None, None, None, 0, None, 0, None, 0, 64, 1e-6, 0, 3, 0, None) == 0
    assert lib.mmfree_cuda_int4_matvec(None, None, 0, None, None, 0, None, None, 0, 64, 8, 32, 0, 0, 2, 0, None) == 0


def test_tensors_must_be_on_a_device():
    x, w = torch.zeros(4, 16), torch.zeros(16, 4)
    for call in (lambda: api.causal_conv(x, w), lambda: api.causal_conv_step(x, w, torch.zeros(4, 3, 16)),
                 lambda: api.selective_scan(x, x, w, x[:, :4], x[:, :4]), lambda: api.add_rmsnorm_quant(x, torch.zeros(16)),
                 lambda: api.int4_matvec(x, torch.zeros(5, 8, dtype=torch.uint8), torch.zeros(5, 1), 32)):
        with pytest.raises(api.MmfreeError) as e:
            call()
        assert e.value.code == _lib.E_INVALID and "CUDA" in str(e.value)


# ---- the references against other formulations ---------------------------------------------------

def test_conv_reference_is_a_convolution():
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(30, 6, generator=g), torch.randn(6, 4, generator=g), torch.randn(6, generator=g)
    y, _, _ = R.conv_ref(x, w, b, None, [0, 30], None, False)
    want = torch.nn.functional.conv1d(torch.nn.functional.pad(x.T.double(), (3, 0)), w[:, None].double(), b.double(), groups=6).T
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-12)


def test_scan_reference_is_the_sum_over_earlier_tokens():
    g = torch.Generator().manual_seed(1)
    T, d, n = 12, 3, 4
    x, dt = torch.randn(T, d, generator=g), torch.randn(T, d, generator=g)
    A, B, C = -torch.rand(d, n, generator=g), torch.randn(T, n, generator=g), torch.randn(T, n, generator=g)
    y, bound, _, _ = R.ssm_ref(x, dt, A, B, C, None, None, None, True, None, [0, T], None)
    delta = torch.nn.functional.softplus(dt.double())
    S = torch.cumsum(delta, 0)
    for t in range(T):
        want = sum((torch.exp((S[t] - S[s])[:, None] * A.double()) * (delta[s] * x[s].double())[:, None]
                    * B[s].double() * C[t].double()).sum(1) for s in range(t + 1))
        assert torch.allclose(y[t], want, rtol=1e-12, atol=1e-12)
    assert (bound < 1e-4).all() and (bound > 0).all()
