"""GPU tests of the recurrent-block operators at the borders of their ranges: infinities, extreme rows, sequences that break
the rules, padded pools, and what torch records about tensors that are written in place."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import block_ref as R
from matmulfreellmcpu_b200 import _lib, api
from test_gpu_block_ops import SENTINEL, close, dev, int4_inputs, rng, run_ssm, sliced, ssm_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("streams,channels,states", [(3, 32, 16), (5, 33, 5), (77, 1200, 16)])
def test_a_batch_of_padding_over_an_empty_pool(cuda, streams, channels, states):
    """The C ABI's step with no state in the pool and no stream that is there: nothing is read from the pool, nothing is
    written, and only a slot that is not negative is reported."""
    d = {k: v.to(cuda) for k, v in ssm_inputs(streams, channels, states, 1, "fp32", 3, 1).items()}
    w, conv = torch.randn(channels, 4, device=cuda), torch.zeros(1, 3, channels, device=cuda)
    slots = torch.full((streams,), -1, dtype=torch.int32, device=cuda)
    out, state = torch.full((streams, channels), SENTINEL, device=cuda), d["state"].clone()
    torch.cuda.synchronize()
    s = _lib.SsmArgs(out=out.data_ptr(), x=d["x"].data_ptr(), dt=d["dt"].data_ptr(), z=d["z"].data_ptr(), B=d["B"].data_ptr(),
                     C=d["C"].data_ptr(), A=d["A"].data_ptr(), state=state.data_ptr(), slots=slots.data_ptr(), ld_out=channels,
                     ldx=channels, ld_dt=channels, ldz=channels, ldb=states, ldc=states, tokens=streams, seqs=streams, slot_count=0,
                     channels=channels, states=states, groups=1, type=_lib.T_F32, dt_softplus=1)
    c = _lib.ConvArgs(out=out.data_ptr(), x=d["x"].data_ptr(), weight=w.data_ptr(), state=conv.data_ptr(), slots=slots.data_ptr(),
                      ld_out=channels, ldx=channels, tokens=streams, seqs=streams, slot_count=0, channels=channels, width=4,
                      type=_lib.T_F32, silu=1)
    stream = torch.cuda.current_stream().cuda_stream
    api.kernel_status()
    for bad in (False, True):
        if bad:
            slots[streams // 2] = 0
        for call, args in ((_lib.lib().mmfree_cuda_selective_step, s), (_lib.lib().mmfree_cuda_causal_conv_step, c)):
            _lib.check(call(C.byref(args), stream))
            if bad:
                with pytest.raises(api.MmfreeError) as e:
                    api.kernel_status()
                assert e.value.code == _lib.E_RANGE
            else:
                api.kernel_status()
    assert (out == SENTINEL).all() and torch.equal(state, d["state"]) and (conv == 0).all()


@pytest.mark.parametrize("channels,states", [(1200, 16), (1200, 5), (600, 40)])
def test_padded_streams_among_four_of_a_thread(cuda, channels, states):
    """Streams that are not there, alone, several together and last, where a thread has four streams; the pool's states that no
    stream has are NaN."""
    streams = 77
    pool = streams + 3
    p = ssm_inputs(streams, channels, states, 1, "bf16", channels, pool)
    slots = torch.randperm(pool, generator=rng(2))[:streams].to(torch.int32)
    slots[torch.tensor([1, 8, 9, 10, 11, 40, 42, 76])] = -1
    idle = [i for i in range(pool) if i not in slots.tolist()]
    p["state"][idle] = torch.nan
    want, bound, new, nbound = R.ssm_ref(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], True, p["state"],
                                         list(range(streams + 1)), slots)
    d = {k: v.to(cuda) for k, v in p.items()}
    out = torch.full_like(d["x"], SENTINEL)
    api.selective_step(d["x"], d["dt"], d["A"], d["B"], d["C"], d["state"], d["D"], d["z"], d["dt_bias"], slots=slots.to(cuda), out=out)
    inside, live = ~torch.isnan(want), [i for i in range(pool) if i not in idle]
    assert ((out.cpu().double() - want).abs()[inside] <= bound[inside]).all() and (out.cpu()[~inside] == SENTINEL).all()
    state = d["state"].cpu()
    assert ((state.double() - new).abs()[live] <= nbound[live]).all() and torch.isnan(state[idle]).all()
    api.kernel_status()


def same_values(got, want, bound, what):
    """Infinities and NaN where the reference has them, the finite values within the bound."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f"{what}: infinities"
    finite = torch.isfinite(want)
    close(got[finite], want[finite], bound[finite], what)


def ssm_reference(p, starts, slots=None, **kw):
    return R.ssm_ref(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], True, p["state"], starts, slots, **kw)


@pytest.mark.parametrize("states", [1, 2, 3, 5, 7, 12, 20, 100, 129])
@pytest.mark.parametrize("channels", [24, 23])
def test_an_infinite_input_with_padded_states(cuda, channels, states):
    """An infinity in x makes the states of its channel infinite and leaves the others alone, whatever the shape's number of
    states is; a prompt and its tokens one by one give the same."""
    p = ssm_inputs(20, channels, states, 1, "fp32", states, 1)
    p["B"], p["C"] = p["B"].abs() + 0.1, p["C"].abs() + 0.1
    p["x"][6, 5] = torch.inf
    p["D"] = p["D"].abs() + 0.1
    want, bound, new, nbound = ssm_reference(p, [0, 20])
    out, state = run_ssm(cuda, p, [0, 20], None, 0)
    same_values(out, want, bound, "prompt")
    same_values(state, new, nbound, "state")
    d = {k: v.to(cuda) for k, v in p.items()}
    for t in range(20):
        row = slice(t, t + 1)
        y = api.selective_step(d["x"][row], d["dt"][row], d["A"], d["B"][row], d["C"][row], d["state"], d["D"], d["z"][row], d["dt_bias"])
        same_values(y, want[row], bound[row], f"token {t}")


def test_an_infinite_input_without_a_skip(cuda):
    """Without D nothing of x is added to what the states give: no 0 * infinity."""
    p = ssm_inputs(20, 24, 16, 1, "fp32", 4, 1)
    p["B"], p["C"], p["D"] = p["B"].abs() + 0.1, p["C"].abs() + 0.1, None
    p["x"][6, 5] = torch.inf
    want, bound, _, _ = ssm_reference(p, [0, 20])
    assert torch.isinf(want[6:, 5]).all()
    out, _ = run_ssm(cuda, p, [0, 20], None, 0, drop=("D",))
    same_values(out, want, bound, "prompt")
    d = {k: None if v is None else v.to(cuda) for k, v in p.items()}
    for t in range(8):
        row = slice(t, t + 1)
        y = api.selective_step(d["x"][row], d["dt"][row], d["A"], d["B"][row], d["C"][row], d["state"], None, d["z"][row], d["dt_bias"])
        same_values(y, want[row], bound[row], f"token {t}")


@pytest.mark.parametrize("tokens", [1, 5, 32, 37])
@pytest.mark.parametrize("rate", [-torch.inf, -3.4e38])
def test_an_infinite_rate_forgets_the_state(cuda, rate, tokens):
    """A rate of minus infinity (or one that is infinite in base 2) keeps nothing of the state before a token, and the tokens
    behind a sequence's end, which a tile computes all the same, change nothing."""
    p = ssm_inputs(tokens, 24, 16, 1, "fp32", 8, 1)
    p["A"][3, 5] = -1e30
    want, bound, new, nbound = ssm_reference(p, [0, tokens])
    p["A"][3, 5] = rate
    out, state = run_ssm(cuda, p, [0, tokens], None, 0)
    close(out, want, bound, "y")
    close(state, new, nbound, "state")


@pytest.mark.parametrize("states", [16, 5])
def test_an_infinite_rate_of_a_single_token(cuda, states):
    p = ssm_inputs(3, 24, states, 1, "fp32", 8, 3)
    p["A"][3, 1] = -1e30
    want, bound, new, nbound = ssm_reference(p, [0, 1, 2, 3])
    p["A"][3, 1] = -torch.inf
    d = {k: v.to(cuda) for k, v in p.items()}
    y = api.selective_step(d["x"], d["dt"], d["A"], d["B"], d["C"], d["state"], d["D"], d["z"], d["dt_bias"])
    close(y, want, bound, "y")
    close(d["state"], new, nbound, "state")


def test_an_infinite_state_across_the_pieces_of_a_split_sequence(cuda):
    """A state that is infinite stays so, also where its decay over a whole piece is below the smallest number."""
    p = ssm_inputs(3000, 8, 16, 1, "fp32", 7, 1)
    p["B"], p["C"], p["dt_bias"] = p["B"].abs() + 0.1, p["C"].abs() + 0.1, torch.full((8,), -1.0)
    p["x"][100, 2] = torch.inf
    p["D"] = p["D"].abs() + 0.1
    want, bound, new, nbound = ssm_reference(p, [0, 3000], pieces=16)
    assert torch.isinf(new[0, 2]).all()
    out, state = run_ssm(cuda, p, [0, 3000], None, 0)
    same_values(out, want, bound, "y")
    same_values(state, new, nbound, "state")


def test_an_empty_state_across_growing_pieces(cuda):
    """A state of 0 stays 0, also where its growth over a whole piece is above the largest number."""
    p = ssm_inputs(3000, 8, 16, 1, "fp32", 7, 1)
    p["A"], p["dt_bias"] = p["A"].abs(), torch.full((8,), 1.0)
    p["x"].zero_()
    p["state"].zero_()
    out, state = run_ssm(cuda, p, [0, 3000], None, 0)
    assert (out == 0).all() and (state == 0).all()


def reported(call):
    api.kernel_status()
    call()
    with pytest.raises(api.MmfreeError) as e:
        api.kernel_status()
    assert e.value.code == _lib.E_RANGE
    api.kernel_status()


@pytest.mark.parametrize("starts,slots", [
    ([0, 8, 8, 99], None), ([0, 8, 8, 4], None), ([0, 4, 4, 8], [0, 99, 1]), ([8, 8, 8, 8], [0, 1, 99]), ([0, 8, 8, -3], None)])
def test_bad_sequences_behind_the_last_row_or_empty_are_reported(cuda, starts, slots):
    """Bounds are checked in the kernels before any access, so these calls end in a status."""
    p = ssm_inputs(8, 16, 16, 1, "fp32", 3, 3)
    d = {k: v.to(cuda) for k, v in p.items()}
    sd = torch.tensor(starts, dtype=torch.int32, device=cuda)
    sl = None if slots is None else torch.tensor(slots, dtype=torch.int32, device=cuda)
    reported(lambda: api.selective_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], state=d["state"], seq_starts=sd, slots=sl))
    for channels in (16, 3):
        x = d["x"][:, :channels].contiguous()
        w, st = torch.randn(channels, 4, device=cuda), torch.randn(3, 3, channels, device=cuda)
        reported(lambda: api.causal_conv(x, w, state=st, seq_starts=sd, slots=sl))


@pytest.mark.parametrize("at", [1, 150, 699])
def test_one_bad_slot_among_many_sequences_is_reported(cuda, at):
    x, w, st = torch.randn(900, 8, device=cuda), torch.randn(8, 4, device=cuda), torch.randn(700, 3, 8, device=cuda)
    starts = torch.arange(701, dtype=torch.int32, device=cuda).clamp(max=500)  # the last 200 are empty
    slots = torch.arange(700, dtype=torch.int32, device=cuda)
    api.causal_conv(x, w, state=st, seq_starts=starts, slots=slots)
    slots[at] = 700
    reported(lambda: api.causal_conv(x, w, state=st, seq_starts=starts, slots=slots))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("kind,cols,extra", [("fp32", 96, 0), ("bf16", 2560, 0), ("bf16", 100, 3), ("fp32", 8192, 0), ("fp16", 96, 0)])
def test_norm_scales_of_very_large_and_very_small_rows(cuda, kind, cols, extra, group, code):
    """The squares of these rows are out of fp32's range; their scales are not."""
    g = rng(cols)
    sizes = torch.tensor([1.0, 1e30, 2e37, 1e-25, 1e-30, 1e-39, 1.0, 3e18, 1e-18])
    if kind == "fp16":
        sizes = torch.tensor([1.0, 1e3, 1e4, 1e-3, 1e-4, 1e-6, 1.0, 8e3, 1e-5])
    x = (torch.randn(9, cols, generator=g) * sizes[:, None]).to(R.TYPES[kind])
    res = (torch.randn(9, cols, generator=g) * sizes[:, None]).to(R.TYPES[kind])
    w = 0.25 + torch.rand(cols, generator=g) / 2
    for eps in (0.0, 1e-6, 1e-30):
        for residual in (None, res):
            q, s, r = R.norm_quant_ref(x, w, residual, eps, code, group)
            rd = None if residual is None else sliced(residual, extra, cuda)
            gq, gs = api.add_rmsnorm_quant(sliced(x, extra, cuda), w.to(cuda), rd, eps, code, group)
            # as test_norm_quant, and half a step of the smallest numbers
            close(gs, s, s * (cols / 2 + 6) * R.U + 2.0 ** -149, f"scales, eps {eps}")
            if code == "int8":
                assert torch.equal(gq.cpu(), q)
            if residual is not None:
                assert torch.equal(rd.cpu(), r)


@pytest.mark.parametrize("group", [0, 32])
def test_norm_of_a_zero_row_without_eps(cuda, group):
    x = torch.randn(3, 96, generator=rng(1))
    x[1] = 0
    q, s = api.add_rmsnorm_quant(x.to(cuda), torch.ones(96, device=cuda), eps=0.0, group=group)
    assert (q[1] == 0).all() and (s[1] == 0).all() and (s[[0, 2]] > 0).all() and torch.isfinite(s).all()


def test_norm_of_a_row_with_an_infinity(cuda):
    """The norm of an infinity is a NaN, of everything beside it 0."""
    x = torch.randn(1, 96, generator=rng(1))
    x[0, 40] = -torch.inf
    q, s = api.add_rmsnorm_quant(x.to(cuda), torch.ones(96, device=cuda), group=32)
    assert torch.isnan(s[0, 1]) and (s[0, [0, 2]] == 0).all()


@pytest.mark.parametrize("group", [0, 128])
def test_norm_of_many_rows_of_which_some_are_far(cuda, group):
    """More rows than the device holds at once, far ones among them, and rows whose every value is a NaN."""
    rows, cols = 3000, 1500
    x = torch.randn(rows, cols, generator=rng(5))
    far = torch.tensor([0, 1, 700, 1999, 2999])
    x[far] *= torch.tensor([1e25, 1e-25, 1e30, 1e-30, 1e37])[:, None]
    x[1234] = torch.nan
    w = 0.5 + torch.rand(cols, generator=rng(6)) / 2
    q, s, _ = R.norm_quant_ref(x, w, None, 0.0, "int8", group)
    gq, gs = api.add_rmsnorm_quant(x.to(cuda), w.to(cuda), eps=0.0, group=group)
    rest = [i for i in range(rows) if i != 1234]
    assert torch.equal(gq.cpu()[rest], q[rest]) and torch.isnan(gs[1234]).all()
    close(gs[rest], s[rest], s[rest] * (cols / 2 + 6) * R.U, "scales")


@pytest.mark.parametrize("k", [300, 512])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
def test_int4_matvec_infinities(cuda, kind, k):
    x, codes, scales, _, _ = int4_inputs(4, k, 40, 64, False, kind, 11)
    x[1, 17] = torch.inf
    x[2, 200], x[2, 3] = -torch.inf, torch.inf
    want, bound = R.int4_ref(x, codes, scales, 64)
    want[torch.isnan(want)] = torch.nan
    out = api.int4_matvec(*dev(cuda, x, codes, scales), 64)
    same_values(out, want, bound + R.rounding(want, out.dtype), kind)


def test_int4_matvec_a_nan_of_low_bits_only(cuda):
    """The NaN whose upper half is that of an infinity."""
    x, codes, scales, _, _ = int4_inputs(2, 512, 40, 64, False, "fp32", 11)
    x.view(torch.int32)[1, 9] = 0x7F800001
    out = api.int4_matvec(*dev(cuda, x, codes, scales), 64)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all()


@pytest.mark.parametrize("m,k,n,extra,out_type", [(9, 5632, 160, 0, torch.float32), (2, 320, 9700, 1, torch.bfloat16), (20, 321, 5000, 0, torch.float16)])
def test_int4_matvec_infinities_of_split_and_of_many_rows(cuda, m, k, n, extra, out_type):
    x, codes, scales, z, _ = int4_inputs(m, k, n, 64, True, "fp32", 12)
    scales = scales * 0.01
    x[1, k // 2], x[m - 1, 3] = -torch.inf, torch.nan
    want, bound = R.int4_ref(x, codes, scales, 64, z)
    out = api.int4_matvec(x.to(cuda), sliced(codes, extra, cuda), scales.to(cuda), 64, zeros=z.to(cuda), out_dtype=out_type)
    same_values(out, want, bound + R.rounding(want, out_type), f"{m} x {k} -> {n}")


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "int8", "e4m3"])
@pytest.mark.parametrize("n", [40, 20000])
def test_int4_matvec_zero_points(cuda, kind, n):
    """Zero points are exact, up to 127 where rows become bf16 operands; there one above is reported."""
    g = rng(n)
    limited = kind in ("fp32", "bf16")
    most = 127 if limited else 255
    codes = torch.randint(0, 256, (n, 128), generator=g, dtype=torch.uint8)
    scales = torch.ldexp(torch.ones(n, 4), torch.randint(-2, 3, (n, 4), generator=g))
    zeros = torch.randint(0, most + 1, (n, 4), generator=g, dtype=torch.uint8)
    zeros[0, 0] = zeros[n - 1, 3] = most
    x = torch.randint(-4, 5, (2, 256), generator=g).float()
    xs = None
    if kind in R.TYPES:
        x = x.to(R.TYPES[kind])
    else:
        x, xs = x.to(torch.int8 if kind == "int8" else torch.float8_e4m3fn), torch.ones(2, 1)
    want, _ = R.int4_ref(x, codes, scales, 64, zeros, xs)  # whole numbers of at most 2^20 quarters: exact in any order
    xd, cd, sd, zd, xsd = dev(cuda, x, codes, scales, zeros, xs)
    api.kernel_status()
    out = api.int4_matvec(xd, cd, sd, 64, zeros=zd, x_scales=xsd, out_dtype=torch.float32)
    assert torch.equal(out.double().cpu(), want)
    api.kernel_status()
    for row, part in ((n - 1, 3), (n // 2, 1)) if limited else ():
        bad = zd.clone()
        bad[row, part] = 128
        api.int4_matvec(xd, cd, sd, 64, zeros=bad, x_scales=xsd)
        with pytest.raises(api.MmfreeError) as e:
            api.kernel_status()
        assert e.value.code == _lib.E_RANGE and "zero point" in str(e.value)
        api.kernel_status()


def test_tensors_written_in_place_get_a_new_version(cuda):
    """A graph that saved a tensor which a call then overwrites refuses its backward pass."""
    x, w = torch.randn(4, 16, device=cuda), torch.randn(16, 4, device=cuda)
    p = {k: v.to(cuda) for k, v in ssm_inputs(4, 16, 4, 1, "fp32", 3, 4).items()}

    def written(t, call):
        leaf = torch.ones_like(t, requires_grad=True)
        before, loss = t._version, (leaf * t).sum()  # the product keeps t for leaf's gradient
        call()
        assert t._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()

    res, st, out = torch.randn(4, 16, device=cuda), torch.randn(4, 3, 16, device=cuda), torch.empty(4, 16, device=cuda)
    written(res, lambda: api.add_rmsnorm_quant(x, torch.ones(16, device=cuda), res))
    written(st, lambda: api.causal_conv(x, w, state=st))
    written(st, lambda: api.causal_conv_step(x, w, st))
    written(out, lambda: api.causal_conv(x, w, out=out))
    scan = (p["x"], p["dt"], p["A"], p["B"], p["C"])
    written(p["state"], lambda: api.selective_scan(*scan, state=p["state"]))
    written(p["state"], lambda: api.selective_step(*scan, p["state"]))
    written(out, lambda: api.selective_scan(*scan, out=out))
    with torch.inference_mode():  # tensors without versions
        state = torch.zeros(4, 3, 16, device=cuda)
        api.causal_conv_step(x, w, state)
    api.causal_conv_step(x, w, state)


def test_forward_mode_tangents_are_refused(cuda):
    import torch.autograd.forward_ad as fw
    x, w = torch.randn(4, 16, device=cuda), torch.randn(16, 4, device=cuda)
    with fw.dual_level():
        for with_grad in (True, False):
            with torch.set_grad_enabled(with_grad), pytest.raises(api.MmfreeError) as e:
                api.causal_conv(fw.make_dual(x, torch.ones_like(x)), w)
            assert e.value.code == _lib.E_INVALID and "gradient" in str(e.value)
        api.causal_conv(x, w)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_an_output_in_the_other_half_of_the_rows(cuda, kind):
    """Halves of one buffer's rows do not overlap, although their spans do."""
    p = ssm_inputs(20, 32, 16, 1, kind, 5, 1)
    d = {k: v.to(cuda) for k, v in p.items()}
    w = torch.randn(32, 4, device=cuda)
    wide = torch.cat((d["x"], torch.zeros_like(d["x"])), 1)
    left, right = wide[:, :32], wide[:, 32:]
    assert torch.equal(api.causal_conv(left, w, out=right), api.causal_conv(d["x"], w))
    scan = (d["dt"], d["A"], d["B"], d["C"])
    want = api.selective_scan(d["x"], *scan, state=d["state"].clone())
    assert torch.equal(api.selective_scan(left, *scan, state=d["state"], out=right), want) and torch.equal(left, d["x"])
    q, s = api.add_rmsnorm_quant(d["x"], torch.ones(32, device=cuda), right.clone())
    gq, gs = api.add_rmsnorm_quant(left, torch.ones(32, device=cuda), right)
    assert torch.equal(gq, q) and torch.equal(gs, s)
    for out in (wide[:, 31:63], wide[:, 1:33], wide[:, :32]):  # one column in common, or all but one, or all
        with pytest.raises(api.MmfreeError) as e:
            api.causal_conv(left, w, out=out)
        assert "overlaps" in str(e.value)
    rows = torch.zeros(24, 64, dtype=d["x"].dtype, device=cuda)
    with pytest.raises(api.MmfreeError):  # the same columns a row further
        api.causal_conv(rows[:20, :32], w, out=rows[1:21, :32])
    with pytest.raises(api.MmfreeError):  # other pitches
        api.causal_conv(rows[:20, :32], w, out=rows.view(-1)[:20 * 48].view(20, 48)[:, 16:])


def test_one_status_names_both_kinds_of_error(cuda):
    x, w, st = torch.randn(2, 64, device=cuda), torch.randn(64, 4, device=cuda), torch.zeros(2, 3, 64, device=cuda)
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8, device=cuda), torch.ones(8, 2, device=cuda)
    api.kernel_status()
    api.int4_matvec(x, codes, scales, 32, zeros=torch.full((8, 2), 200, dtype=torch.uint8, device=cuda))
    api.causal_conv_step(x, w, st, slots=torch.tensor([0, 5], dtype=torch.int32, device=cuda))
    with pytest.raises(api.MmfreeError) as e:
        api.kernel_status()
    assert e.value.code == _lib.E_RANGE and "zero point" in str(e.value) and "slot" in str(e.value)
    api.kernel_status()
