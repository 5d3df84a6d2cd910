"""GPU tests of the recurrent-block operators against the 64-bit references of block_ref.py."""
from __future__ import annotations


import pytest
import torch

import block_ref as R
from matmulfreellmcpu_b200 import _lib, api

pytestmark = pytest.mark.gpu

SENTINEL = 77.0


def rng(seed):
    return torch.Generator().manual_seed(seed)


def sliced(t, extra, cuda):
    """The tensor on the device as a slice of wider rows (``extra`` more columns, some in front)."""
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + extra, dtype=t.dtype)
    front = extra // 2
    wide[..., front:front + t.shape[-1]] = t
    return wide.to(cuda)[..., front:front + t.shape[-1]]


def close(got, want, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    i = int(over.argmax())
    assert over.max() <= 0, f"{what}: {got.flatten()[i]} for {want.flatten()[i]}, bound {bound.flatten()[i]}"


# ---- add_rmsnorm_quant -------------------------------------------------------------------------

@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols,group,extra", [
    (1, 1, 0, 0), (1, 2048, 0, 0), (3, 7, 32, 0), (5, 100, 32, 3), (4, 1003, 64, 1), (2, 2560, 128, 8),
    (3, 5632, 0, 16), (2, 2056, 128, 0), (1, 8192, 64, 0), (2, 33000, 128, 0), (1, 57344, 0, 0)])
def test_norm_quant(cuda, rows, cols, group, extra, kind, code):
    g = rng(cols + rows)
    dtype = R.TYPES[kind]
    x = torch.randn(rows, cols, generator=g).to(dtype)
    res = (torch.randn(rows, cols, generator=g) * (1 + 20 * (torch.rand(cols, generator=g) < 0.01))).to(dtype)
    w = 0.5 + torch.rand(cols, generator=g)
    for residual in (None, res):
        q, s, r = R.norm_quant_ref(x, w, residual, 1e-6, code, group)
        xd = sliced(x, extra, cuda)
        rd = None if residual is None else sliced(residual, extra, cuda)
        gq, gs = api.add_rmsnorm_quant(xd, w.to(cuda), rd, 1e-6, code, group)
        assert gq.dtype == q.dtype and gs.shape == s.shape
        if code == "int8":
            assert torch.equal(gq.cpu(), q)
        else:
            # the product t * (448 / m) has the same two fp32 roundings on both sides
            assert torch.equal(gq.cpu().view(torch.uint8), q.view(torch.uint8))
        # the squares' sum in fp32 (cols roundings at most, halved by the root) and five more steps
        close(gs, s, s * (cols / 2 + 6) * R.U, "scales")
        if residual is not None:
            assert torch.equal(rd.cpu(), r)


def test_norm_quant_borders(cuda):
    """Quotients that lie on or next to a border between two codes."""
    cols = 1024
    m = torch.tensor([127.0, 254.0, 1.0, 0.3, 1e-30, 3e38, 5e-40])
    half = (torch.arange(cols) % 127).float() + 0.5
    x = m[:, None] * half / 127
    x = torch.stack([x, torch.nextafter(x, torch.tensor(torch.inf)), torch.nextafter(x, torch.tensor(0.0))]).flatten(0, 1)
    x[:, 0] = m.repeat(3)
    x[:, 1::2] *= -1
    w = torch.ones(cols)
    q, s, _ = R.norm_quant_ref(x, w, None, 1e-6, "int8", 0)
    gq, _ = api.add_rmsnorm_quant(x.to(cuda), w.to(cuda))
    assert torch.equal(gq.cpu(), q)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("group", [0, 32])
def test_norm_quant_zero_and_nonfinite_rows(cuda, code, group):
    x = torch.randn(4, 96, generator=rng(1))
    x[0] = 0
    x[1, 5] = torch.nan
    x[2, 40] = torch.inf
    q, s = api.add_rmsnorm_quant(x.to(cuda), torch.ones(96, device=cuda), code=code, group=group)
    q, s = q.float().cpu(), s.cpu()
    assert (q[0] == 0).all() and (s[0] == 0).all()
    assert torch.isnan(s[1]).all()      # the sum of squares is a NaN
    assert torch.isnan(s[2, 40 // group if group else 0])
    want, ws, _ = R.norm_quant_ref(x[3:], torch.ones(96), None, 1e-6, code, group)
    assert torch.equal(q[3], want[0].float()) and torch.isfinite(s[3]).all()


def test_norm_quant_broadcast_row_and_no_rows(cuda):
    x = torch.randn(1, 64, generator=rng(2)).to(cuda).expand(5, 64)
    q, s = api.add_rmsnorm_quant(x, torch.ones(64, device=cuda))
    assert (q == q[0]).all() and (s == s[0]).all()
    q, s = api.add_rmsnorm_quant(x[:0], torch.ones(64, device=cuda), code="e4m3", group=32)
    assert q.shape == (0, 64) and s.shape == (0, 2)


# ---- int4_matvec -------------------------------------------------------------------------------

def int4_inputs(m, k, n, group, zeros, kind, seed, scale_type=torch.float16):
    g = rng(seed)
    parts = -(-k // group)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(n, parts, generator=g)) * 0.1).to(scale_type)
    z = torch.randint(0, 16, (n, parts), generator=g, dtype=torch.uint8) if zeros else None
    x = torch.randn(m, k, generator=g)
    if kind in R.TYPES:
        return x.to(R.TYPES[kind]), codes, scales, z, None
    xs = x.abs().amax(1, keepdim=True) / (127 if kind == "int8" else 448)
    x = x / xs
    return (x.round().to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn)), codes, scales, z, xs


def dev(cuda, *ts):
    return [None if t is None else t.to(cuda) for t in ts]


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "int8", "e4m3"])
@pytest.mark.parametrize("m,k,n,group,zeros", [
    (1, 2048, 2048, 128, False), (1, 1, 1, 32, True), (2, 33, 5, 32, True), (3, 1003, 77, 64, False),
    (7, 256, 300, 96, True), (8, 512, 64, 512, False), (9, 700, 48, 32, True), (16, 5632, 160, 64, True),
    (17, 2560, 100, 128, False), (33, 320, 31, 32, True), (1, 6912, 50, 128, True), (70, 130, 18, 64, False)])
def test_int4_matvec(cuda, m, k, n, group, zeros, kind):
    x, codes, scales, z, xs = int4_inputs(m, k, n, group, zeros, kind, m * 1000 + k)
    want, bound = R.int4_ref(x, codes, scales, group, z, xs)
    xd, cd, sd, zd, xsd = dev(cuda, x, codes, scales, z, xs)
    out = api.int4_matvec(xd, cd, sd, group, zeros=zd, x_scales=xsd)
    assert out.dtype == (x.dtype if kind in R.TYPES else torch.float32)
    close(out, want, bound + R.rounding(want, out.dtype), f"int4 {kind}")


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "int8", "e4m3"])
@pytest.mark.parametrize("m,k,n,group", [(1, 2048, 33, 128), (5, 777, 65, 32), (20, 1600, 40, 64), (2, 8192, 130, 256)])
def test_int4_matvec_whole_numbers(cuda, m, k, n, group, kind):
    """Whole inputs and scales that are powers of two: every sum is exact in any order, so the
    result is the exact one, and a misplaced element shows."""
    g = rng(m + k)
    parts = -(-k // group)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, dtype=torch.uint8)
    scales = torch.ldexp(torch.ones(n, parts), torch.randint(-2, 3, (n, parts), generator=g)).to(torch.bfloat16)
    z = torch.randint(0, 16, (n, parts), generator=g, dtype=torch.uint8)
    x = torch.randint(-4, 5, (m, k), generator=g).float()
    xs = None
    if kind in R.TYPES:
        x = x.to(R.TYPES[kind])
    else:
        x = x.to(torch.int8 if kind == "int8" else torch.float8_e4m3fn)
        xs = torch.ldexp(torch.ones(m, parts), torch.randint(-1, 2, (m, parts), generator=g))
    want, _ = R.int4_ref(x, codes, scales, group, z, xs)
    xd, cd, sd, zd, xsd = dev(cuda, x, codes, scales, z, xs)
    out = api.int4_matvec(xd, cd, sd, group, zeros=zd, x_scales=xsd, out_dtype=torch.float32)
    assert torch.equal(out.double().cpu(), want)


@pytest.mark.parametrize("scale_type", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_type", [torch.float32, torch.bfloat16, torch.float16])
def test_int4_matvec_types_and_pitches(cuda, scale_type, out_type):
    x, codes, scales, z, xs = int4_inputs(3, 416, 70, 32, True, "bf16", 5, scale_type)
    want, bound = R.int4_ref(x, codes, scales, 32, z, xs)
    for extra in (0, 1, 16):
        out = api.int4_matvec(sliced(x, extra, cuda), sliced(codes, extra, cuda), scales.to(cuda), 32,
                              zeros=z.to(cuda), out_dtype=out_type)
        close(out, want, bound + R.rounding(want, out_type), f"pitch +{extra}")


def test_int4_matvec_wide_values(cuda):
    """fp32 and bf16 rows of very large and very small values keep their range."""
    x, codes, scales, _, _ = int4_inputs(4, 256, 40, 64, False, "fp32", 9)
    x *= torch.tensor([1e30, 1e-30, 1.0, 1e-3])[:, None]
    for dtype in (torch.float32, torch.bfloat16):
        xt = x.to(dtype)
        want, bound = R.int4_ref(xt, codes, scales, 64)
        out = api.int4_matvec(xt.to(cuda), codes.to(cuda), scales.to(cuda), 64, out_dtype=torch.float32)
        close(out, want, bound + R.rounding(want, torch.float32), str(dtype))


def test_int4_matvec_nonfinite_stays_in_its_row(cuda):
    x, codes, scales, _, _ = int4_inputs(3, 300, 40, 64, False, "fp32", 11)
    x[1, 17] = torch.nan
    out = api.int4_matvec(*dev(cuda, x, codes, scales), 64).cpu()
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()


@pytest.mark.parametrize("kind", ["fp32", "bf16", "int8"])
def test_int4_matvec_row_does_not_depend_on_the_others(cuda, kind):
    x, codes, scales, z, xs = int4_inputs(40, 1536, 96, 64, True, kind, 12)
    xd, cd, sd, zd, xsd = dev(cuda, x, codes, scales, z, xs)
    every = api.int4_matvec(xd, cd, sd, 64, zeros=zd, x_scales=xsd)
    for rows in ([0], [39], [3, 4], list(range(10, 27))):
        some = api.int4_matvec(xd[rows], cd, sd, 64, zeros=zd, x_scales=None if xsd is None else xsd[rows])
        assert torch.equal(some, every[rows])


# ---- causal_conv -------------------------------------------------------------------------------

LENS = [[1], [2], [37], [5, 0, 1, 3, 33, 0, 2, 64, 1], [0, 0, 7], [31, 1, 31, 1, 2, 30, 97]]


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("width,channels,extra", [(2, 1, 0), (3, 24, 1), (4, 256, 0), (4, 264, 8), (5, 33, 0), (8, 40, 2)])
def test_causal_conv(cuda, width, channels, extra, kind):
    dtype = R.TYPES[kind]
    for i, lens in enumerate(LENS):
        g = rng(width * 100 + i)
        lead, tail = (0, 0) if i % 2 else (3, 2)
        starts = R.starts_of(lens, lead)
        rows = starts[-1] + tail
        x = torch.randn(rows, channels, generator=g).to(dtype)
        w, b = torch.randn(channels, width, generator=g), torch.randn(channels, generator=g)
        pool = len(lens) + 2
        state = torch.randn(pool, width - 1, channels, generator=g).to(dtype)
        slots = torch.randperm(pool, generator=g)[:len(lens)].to(torch.int32)
        slots[len(lens) // 2] = -1 if len(lens) > 2 else slots[len(lens) // 2]
        for with_state, silu in ((True, True), (False, False)):
            st, sl, bias = (state, slots, b) if with_state else (None, None, None)
            want, bound, new = R.conv_ref(x, w, bias, st, starts, sl, silu)
            std = None if st is None else st.to(cuda)
            out = sliced(torch.full((rows, channels), SENTINEL, dtype=dtype), extra, cuda)
            api.causal_conv(sliced(x, extra, cuda), w.to(cuda), None if bias is None else bias.to(cuda), std,
                            torch.tensor(starts, dtype=torch.int32, device=cuda),
                            None if sl is None else sl.to(cuda), silu, out=out)
            inside = ~torch.isnan(want)
            close(out.cpu()[inside], want[inside], bound[inside], f"conv {lens}")
            assert (out.cpu()[~inside] == SENTINEL).all()
            if std is not None:
                assert torch.equal(std.cpu(), new)
    api.kernel_status()


def test_causal_conv_one_sequence_without_starts(cuda):
    x, w = torch.randn(50, 16, generator=rng(3)), torch.randn(16, 4, generator=rng(4))
    want, bound, _ = R.conv_ref(x, w, None, None, [0, 50], None, True)
    close(api.causal_conv(x.to(cuda), w.to(cuda), silu=True), want, bound, "one sequence")


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("width,channels", [(4, 264), (3, 7), (6, 20)])
def test_causal_conv_step_continues_the_prompt(cuda, width, channels, kind):
    """A prompt and its tokens one by one: the same outputs and states bit for bit."""
    dtype = R.TYPES[kind]
    g = rng(width)
    lens = [9, 9, 9]
    x = torch.randn(27, channels, generator=g).to(dtype).to(cuda)
    w, b = torch.randn(channels, width, generator=g).to(cuda), torch.randn(channels, generator=g).to(cuda)
    first = torch.randn(5, width - 1, channels, generator=g).to(dtype).to(cuda)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=cuda)
    one, two = first.clone(), first.clone()
    y = api.causal_conv(x, w, b, one, torch.tensor(R.starts_of(lens), dtype=torch.int32, device=cuda), slots, True)
    for t in range(9):
        yt = api.causal_conv_step(x[t::9], w, two, b, slots, True)
        assert torch.equal(yt, y[t::9])
    assert torch.equal(one, two) and torch.equal(one[[1, 3]], first[[1, 3]])


# ---- selective_scan ----------------------------------------------------------------------------

def ssm_inputs(rows, channels, states, groups, kind, seed, pool, sharp=1.0):
    g = rng(seed)
    dtype = R.TYPES[kind]
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    step = torch.exp(torch.rand(channels, generator=g) * 4.6 - 6.9)  # 0.001 to 0.1
    return dict(x=n(rows, channels).to(dtype), dt=(n(rows, channels) * 0.5).to(dtype),
                A=-torch.arange(1, states + 1).float() * (0.9 + 0.2 * torch.rand(channels, states, generator=g)) * sharp,
                B=n(rows, groups, states).to(dtype), C=n(rows, groups, states).to(dtype), D=n(channels),
                z=n(rows, channels).to(dtype), dt_bias=step + torch.log(-torch.expm1(-step)),
                state=n(pool, channels, states) * 0.3)


def run_ssm(cuda, p, starts, slots, extra, softplus=True, drop=()):
    d = {k: (None if k in drop else sliced(v, extra, cuda) if k in ("x", "dt", "z") else v.to(cuda)) for k, v in p.items()}
    wide = sliced(torch.cat((p["B"], p["C"]), 1).flatten(1), extra, cuda)
    half = wide.shape[1] // 2
    d["B"], d["C"] = (t.unflatten(1, p["B"].shape[1:]) for t in (wide[:, :half], wide[:, half:]))
    out = sliced(torch.full(p["x"].shape, SENTINEL, dtype=p["x"].dtype), extra, cuda)
    api.selective_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"], softplus, d["state"],
                       torch.tensor(starts, dtype=torch.int32, device=cuda), None if slots is None else slots.to(cuda), out)
    return out.cpu(), None if d["state"] is None else d["state"].cpu()


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("channels,states,groups,extra", [
    (1, 1, 1, 0), (64, 16, 1, 0), (48, 16, 2, 8), (33, 16, 1, 1), (40, 5, 4, 0), (24, 64, 1, 0), (20, 100, 2, 4), (6, 256, 1, 0)])
def test_selective_scan(cuda, channels, states, groups, extra, kind):
    for i, lens in enumerate(LENS):
        lead, tail = (0, 0) if i % 2 else (3, 2)
        starts = R.starts_of(lens, lead)
        pool = len(lens) + 1
        p = ssm_inputs(starts[-1] + tail, channels, states, groups, kind, channels + i, pool)
        g = rng(i)
        slots = torch.randperm(pool, generator=g)[:len(lens)].to(torch.int32)
        if len(lens) > 2:
            slots[1] = -1
        for drop, softplus, sl in (((), True, slots), (("D", "z", "dt_bias", "state"), False, None)):
            q = {k: (None if k in drop else v) for k, v in p.items()}
            if not softplus:
                p["dt"] = q["dt"] = p["dt"].abs() * 0.1
            want, bound, new, nbound = R.ssm_ref(q["x"], q["dt"], q["A"], q["B"], q["C"], q["D"], q["z"], q["dt_bias"],
                                                 softplus, q["state"], starts, sl, pieces=16)
            out, state = run_ssm(cuda, p, starts, sl, extra, softplus, drop)
            inside = ~torch.isnan(want)
            close(out[inside], want[inside], bound[inside], f"scan {lens}")
            assert (out[~inside] == SENTINEL).all()
            if state is not None:
                close(state, new, nbound, f"state {lens}")
                idle = [s for s in range(pool) if s not in sl.tolist()]
                assert torch.equal(state[idle], p["state"][idle])
    api.kernel_status()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("lens,channels,states", [
    ([3000], 8, 16), ([700, 1, 0, 1300], 40, 16), ([1500], 4, 128), ([520], 130, 3), ([4000, 0, 2, 900, 3000], 64, 16),
    ([2500], 33, 16), ([1100], 12, 200), ([1300, 700], 72, 7)])
def test_selective_scan_long(cuda, lens, channels, states, kind):
    starts = R.starts_of(lens)
    p = ssm_inputs(starts[-1], channels, states, 1, kind, 7, len(lens))
    want, bound, new, nbound = R.ssm_ref(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], True,
                                         p["state"], starts, None, pieces=16)
    out, state = run_ssm(cuda, p, starts, None, 0)
    close(out, want, bound, "y")
    close(state, new, nbound, "state")


def test_selective_scan_extreme_steps(cuda):
    """Steps so large that a decay is 0, so small that it is 1, and a softplus past its branch."""
    p = ssm_inputs(64, 32, 16, 1, "fp32", 13, 1)
    p["dt"][::4] = 30.0
    p["dt"][1::4] = -40.0
    p["dt"][2::4] *= 20
    starts = [0, 64]
    want, bound, new, nbound = R.ssm_ref(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], True,
                                         p["state"], starts, None, pieces=16)
    out, state = run_ssm(cuda, p, starts, None, 0)
    close(out, want, bound, "y")
    close(state, new, nbound, "state")


def test_selective_scan_nonfinite_values_stay_where_they_are(cuda):
    """An infinity in a sequence's last token, and NaN in rows and sequences around it."""
    p = ssm_inputs(40, 64, 16, 1, "fp32", 21, 3)
    starts, slots = [2, 11, 11, 37], torch.tensor([0, 1, 2], dtype=torch.int32)
    for k in ("x", "dt", "B", "C", "z"):
        p[k][:2] = torch.nan   # rows in front of the first and behind the last sequence
        p[k][37:] = torch.nan
    p["B"][10, 0, 3] = torch.inf
    p["x"][10] = p["x"][10].abs() + 0.1
    clean = {k: v.clone() for k, v in p.items()}
    clean["B"][10, 0, 3] = 1.0
    want, bound, new, nbound = R.ssm_ref(clean["x"], clean["dt"], clean["A"], clean["B"], clean["C"], clean["D"], clean["z"],
                                         clean["dt_bias"], True, clean["state"], starts, slots, pieces=16)
    out, state = run_ssm(cuda, p, starts, slots, 0)
    rows = [t for t in range(2, 37) if t != 10]
    close(out[rows], want[rows], bound[rows], "y")
    assert torch.isinf(state[0, :, 3]).all()
    keep = [n for n in range(16) if n != 3]
    close(state[:, :, keep], new[:, :, keep], nbound[:, :, keep], "state")


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("streams,channels,states,groups", [(1, 2048, 16, 1), (5, 33, 16, 1), (3, 48, 5, 2), (2, 40, 128, 4),
                                                            (4, 12, 64, 1), (2, 3, 256, 1), (64, 256, 16, 1), (3, 8, 1, 1)])
def test_selective_step(cuda, streams, channels, states, groups, kind):
    pool = streams + 2
    p = ssm_inputs(streams, channels, states, groups, kind, channels, pool)
    slots = torch.randperm(pool, generator=rng(1))[:streams].to(torch.int32)
    if streams > 2:
        slots[1] = -1
    starts = list(range(streams + 1))
    want, bound, new, nbound = R.ssm_ref(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], True,
                                         p["state"], starts, slots)
    d = {k: v.to(cuda) for k, v in p.items()}
    out = torch.full_like(d["x"], SENTINEL)
    y = api.selective_step(d["x"], d["dt"], d["A"], d["B"], d["C"], d["state"], d["D"], d["z"], d["dt_bias"],
                           slots=slots.to(cuda), out=out)
    assert y is out
    inside = ~torch.isnan(want)
    close(out.cpu()[inside], want[inside], bound[inside], "y")
    assert (out.cpu()[~inside] == SENTINEL).all()
    close(d["state"], new, nbound, "state")
    api.kernel_status()


def test_two_dimensional_b_and_c(cuda):
    p = ssm_inputs(20, 16, 16, 1, "fp32", 3, 1)
    d = {k: v.to(cuda) for k, v in p.items()}
    a = api.selective_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], state=d["state"].clone())
    b = api.selective_scan(d["x"], d["dt"], d["A"], d["B"][:, 0], d["C"][:, 0], state=d["state"].clone())
    assert torch.equal(a, b)


# ---- sequences that break the rules, streams, graphs, refusals -----------------------------------

@pytest.mark.parametrize("starts,slots,good", [
    ([0, 4, 2, 8], None, [0]), ([0, 4, 4, 99], None, [0]), ([-1, 4, 8, 8], None, [1]),
    ([0, 3, 6, 8], [0, 7, 1], [0, 2])])
def test_bad_sequences_are_skipped_and_reported(cuda, starts, slots, good):
    """Bounds are checked in the kernels before any access, so these calls end in a status."""
    p = ssm_inputs(8, 16, 16, 1, "fp32", 3, 3)
    d = {k: v.to(cuda) for k, v in p.items()}
    sd = torch.tensor(starts, dtype=torch.int32, device=cuda)
    sl = None if slots is None else torch.tensor(slots, dtype=torch.int32, device=cuda)
    api.kernel_status()
    api.selective_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], state=d["state"], seq_starts=sd, slots=sl)
    with pytest.raises(api.MmfreeError) as e:
        api.kernel_status()
    assert e.value.code == _lib.E_RANGE
    api.kernel_status()  # reported once
    w = torch.randn(16, 4, device=cuda)
    st = torch.randn(3, 3, 16, device=cuda)
    api.causal_conv(d["x"], w, state=st, seq_starts=sd, slots=sl)
    with pytest.raises(api.MmfreeError) as e:
        api.kernel_status()
    assert e.value.code == _lib.E_RANGE
    if slots is not None:
        st0 = torch.randn(3, 3, 16, device=cuda)
        x3 = d["x"][:3].contiguous()
        api.causal_conv_step(x3, w, st0, slots=sl)
        with pytest.raises(api.MmfreeError):
            api.kernel_status()
        api.selective_step(x3, d["dt"][:3], d["A"], d["B"][:3], d["C"][:3], d["state"], slots=sl)
        with pytest.raises(api.MmfreeError):
            api.kernel_status()


def block(cuda, seed=0, hidden=128, inner=256, states=16):
    g = rng(seed)

    def proj(n, k):
        return (torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).to(cuda),
                ((0.5 + torch.rand(n, -(-k // 64), generator=g)) * 0.3 * k ** -0.5).half().to(cuda))

    p = ssm_inputs(1, inner, states, 1, "bf16", seed, 1)
    return dict(norm=(0.5 + torch.rand(hidden, generator=g)).to(cuda), inp=proj(2 * inner, hidden), xp=proj(inner + 2 * states, inner),
                out=proj(hidden, inner), cw=torch.randn(inner, 4, generator=g).to(cuda) * 0.5, A=p["A"].to(cuda), D=p["D"].to(cuda),
                bias=p["dt_bias"].to(cuda), inner=inner, states=states)


def run_block(b, h, conv, ssm, starts=None, slots=None):
    """One block over packed prompts, or (without starts) over one token of each stream: ``h`` bf16
    [rows, hidden] is the residual, updated by the next block's norm; returns the block's output."""
    q, s = api.add_rmsnorm_quant(torch.zeros_like(h), b["norm"], h, code="int8")
    xz = api.int4_matvec(q, *b["inp"], 64, x_scales=s, out_dtype=torch.bfloat16)
    x, z = xz[:, :b["inner"]], xz[:, b["inner"]:]
    if starts is None:
        x = api.causal_conv_step(x, b["cw"], conv, slots=slots, silu=True)
    else:
        x = api.causal_conv(x, b["cw"], state=conv, seq_starts=starts, slots=slots, silu=True)
    w = api.int4_matvec(x, *b["xp"], 64)
    dt, B, C = w.split([b["inner"], b["states"], b["states"]], 1)
    args = (x, dt, b["A"], B, C)
    kw = dict(D=b["D"], z=z, dt_bias=b["bias"], slots=slots)
    y = api.selective_step(*args, ssm, **kw) if starts is None else api.selective_scan(*args, state=ssm, seq_starts=starts, **kw)
    return api.int4_matvec(y, *b["out"], 64), (x, dt, B, C, z, y)


def test_a_block_for_prompts_and_token_by_token(cuda):
    """The operators as one block: a packed prompt against the same tokens one at a time, its
    scan against the 64-bit reference on what the other operators gave it."""
    b = block(cuda)
    streams, length = 3, 50
    h = torch.randn(streams * length, 128, generator=rng(5)).bfloat16().to(cuda)
    slots = torch.tensor([2, 0, 3], dtype=torch.int32, device=cuda)
    conv1 = torch.zeros(4, 3, 256, dtype=torch.bfloat16, device=cuda)
    ssm1 = torch.zeros(4, 256, 16, device=cuda)
    conv2, ssm2 = conv1.clone(), ssm1.clone()
    starts = torch.tensor(R.starts_of([length] * streams), dtype=torch.int32, device=cuda)
    out, (x, dt, B, C, z, y) = run_block(b, h.clone(), conv1, ssm1, starts, slots)
    c = lambda t: t.cpu()  # noqa: E731
    want, bound, new, nbound = R.ssm_ref(c(x), c(dt), c(b["A"]), c(B), c(C), c(b["D"]), c(z), c(b["bias"]), True,
                                         torch.zeros(4, 256, 16), starts.tolist(), slots.tolist(), pieces=16)
    close(y, want, bound, "prompt scan")
    close(ssm1, new, nbound, "prompt state")
    for t in range(length):
        at = torch.arange(streams, device=cuda) * length + t
        _, (xt, _, _, _, zt, yt) = run_block(b, h[at].clone(), conv2, ssm2, None, slots)
        # everything before the scan works row by row, so it does not depend on the batch
        assert torch.equal(xt, x[at]) and torch.equal(zt, z[at])
        close(yt, want[at.cpu()], bound[at.cpu()], f"token {t}")
    assert torch.equal(conv1, conv2)
    close(ssm2, new, nbound, "token state")
    assert torch.isfinite(out).all()


def test_a_captured_step_and_two_graphs_on_two_streams(cuda):
    """Steps captured into graphs give what eager calls give, two graphs replayed at once too."""
    b = block(cuda, 1)
    graphs, expect = [], []
    for k in range(2):
        h = torch.randn(2, 128, generator=rng(k)).bfloat16().to(cuda)
        conv, ssm = torch.zeros(2, 3, 256, dtype=torch.bfloat16, device=cuda), torch.zeros(2, 256, 16, device=cuda)
        e_conv, e_ssm = conv.clone(), ssm.clone()
        for _ in range(20):
            e_out, _ = run_block(b, h.clone(), e_conv, e_ssm)
        expect.append((e_out, e_conv, e_ssm))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, _ = run_block(b, h.clone(), conv, ssm)
        graphs.append((graph, stream, out, conv, ssm, h))  # a graph reads its inputs' memory
    for _ in range(20):
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, _, out, conv, ssm, _), (e_out, e_conv, e_ssm) in zip(graphs, expect):
        assert torch.equal(out, e_out) and torch.equal(conv, e_conv) and torch.equal(ssm, e_ssm)


def test_another_stream(cuda):
    x, w = torch.randn(300, 512, device=cuda), torch.randn(512, 4, device=cuda)
    want = api.causal_conv(x, w, silu=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = api.causal_conv(x, w, silu=True, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_large_calls_in_a_captured_graph(cuda):
    """Calls of many rows and tokens ask the device for its size; that is allowed in a capture."""
    x = torch.randn(600, 512, device=cuda)
    res, w = torch.randn(600, 512, device=cuda), torch.ones(512, device=cuda)
    p = {k: v.to(cuda) for k, v in ssm_inputs(600, 512, 16, 1, "fp32", 5, 1).items()}
    codes, scales = torch.randint(0, 256, (300, 256), dtype=torch.uint8, device=cuda), torch.rand(300, 4, device=cuda)

    def run(res, st):
        q, s = api.add_rmsnorm_quant(x, w, res)
        m = api.int4_matvec(q, codes, scales, 128, x_scales=s)
        return q, s, m, api.selective_scan(p["x"], p["dt"], p["A"], p["B"], p["C"], state=st)

    r1, s1 = res.clone(), p["state"].clone()
    want = run(r1, s1)
    r2, s2 = res.clone(), p["state"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(r2, s2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*want, r1, s1), (*got, r2, s2)))


def test_inputs_that_require_gradients_are_refused(cuda):
    x, w = torch.randn(4, 16, device=cuda), torch.randn(16, 4, device=cuda, requires_grad=True)
    with pytest.raises(api.MmfreeError) as e:
        api.causal_conv(x, w)
    assert e.value.code == _lib.E_INVALID and "gradient" in str(e.value)
    with torch.no_grad():
        api.causal_conv(x, w)


def test_repeated_calls_give_the_same_bits(cuda):
    p = ssm_inputs(2000, 64, 16, 1, "fp32", 3, 1)
    d = {k: v.to(cuda) for k, v in p.items()}
    x, codes, scales, _, _ = int4_inputs(9, 5632, 200, 64, False, "fp32", 3)
    first = None
    for _ in range(3):
        st = d["state"].clone()
        y = api.selective_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["dt_bias"], state=st)
        m = api.int4_matvec(*dev(cuda, x, codes, scales), 64)
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, (y, st, m)))
        first = (y, st, m)


def test_refusals(cuda):
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=cuda)  # noqa: E731
    x, w, st = f(8, 16), f(16, 4), f(2, 3, 16)
    starts = torch.tensor([0, 4, 8], dtype=torch.int32, device=cuda)
    A, B, h = f(16, 4), f(8, 4), f(2, 16, 4)
    u8 = lambda *s: f(*s, dtype=torch.uint8)  # noqa: E731
    calls = [
        lambda: api.causal_conv(x.cpu(), w), lambda: api.causal_conv(x.double(), w), lambda: api.causal_conv(x, w.half()),
        lambda: api.causal_conv(x, f(16, 9)), lambda: api.causal_conv(x, f(16, 1)), lambda: api.causal_conv(x, f(15, 4)),
        lambda: api.causal_conv(x.T, f(8, 4)), lambda: api.causal_conv(x[None], w), lambda: api.causal_conv(x, w.cpu()),
        lambda: api.causal_conv(x, w, state=f(1, 3, 16), seq_starts=starts),     # fewer states than sequences
        lambda: api.causal_conv(x, w, state=f(2, 2, 16), seq_starts=starts), lambda: api.causal_conv(x, w, state=st.half()),
        lambda: api.causal_conv(x, w, seq_starts=starts.long()), lambda: api.causal_conv(x, w, slots=starts[:1]),
        lambda: api.causal_conv(x, w, state=st, seq_starts=starts, slots=starts),  # one slot too many
        lambda: api.causal_conv(x, w, out=x), lambda: api.causal_conv(x, w, out=f(8, 15)),
        lambda: api.causal_conv(x, w, out=f(1, 16).expand(8, 16)), lambda: api.causal_conv_step(x, w, st),
        lambda: api.causal_conv_step(x, w, None), lambda: api.selective_step(x, x, A, B, B, None),
        lambda: api.selective_scan(x, x, A, B, f(8, 5)), lambda: api.selective_scan(x, x, f(16, 257), B, B),
        lambda: api.selective_scan(x, x, A, f(8, 3, 4), f(8, 3, 4)), lambda: api.selective_scan(x, x.half(), A, B, B),
        lambda: api.selective_scan(x, x, A.double(), B, B), lambda: api.selective_scan(x, x, A, B, B, state=f(2, 16, 5)),
        lambda: api.selective_scan(x, x, A, B, B, state=h.half()), lambda: api.selective_scan(x, x, A, B, B, out=x),
        lambda: api.selective_step(x, x, A, B, B, h), lambda: api.selective_scan(x, x, A, f(4, 8).T, B),
        lambda: api.add_rmsnorm_quant(x, f(15)), lambda: api.add_rmsnorm_quant(x, f(16), code="int4"),
        lambda: api.add_rmsnorm_quant(x, f(16), group=16), lambda: api.add_rmsnorm_quant(x, f(16), residual=x),
        lambda: api.add_rmsnorm_quant(x, f(16), residual=x.half()), lambda: api.add_rmsnorm_quant(f(2, 60000), f(60000)),
        lambda: api.add_rmsnorm_quant(x, f(16), residual=f(1, 16).expand(8, 16)),
        lambda: api.int4_matvec(x, u8(5, 8), f(5, 1), 16), lambda: api.int4_matvec(x, u8(5, 7), f(5, 1), 32),
        lambda: api.int4_matvec(x, u8(5, 8), f(5, 2), 32), lambda: api.int4_matvec(x, u8(5, 8), u8(5, 1), 32),
        lambda: api.int4_matvec(x, u8(5, 8), f(5, 1), 32, zeros=f(5, 1)), lambda: api.int4_matvec(x, u8(5, 8), f(5, 1), 32, x_scales=f(8, 1)),
        lambda: api.int4_matvec(f(8, 16, dtype=torch.int8), u8(5, 8), f(5, 1), 32),
        lambda: api.int4_matvec(x, u8(5, 8), f(5, 1), 32, out_dtype=torch.int8), lambda: api.int4_matvec(x, u8(5, 8).char(), f(5, 1), 32),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(api.MmfreeError) as e:
            call()
        assert e.value.code == _lib.E_INVALID, i
    # nothing to do is not an error
    assert api.causal_conv(x[:0], w).shape == (0, 16)
    assert api.selective_scan(x[:0], x[:0], A, B[:0], B[:0], seq_starts=torch.zeros(1, dtype=torch.int32, device=cuda)).shape == (0, 16)
    assert api.int4_matvec(x[:0], u8(5, 8), f(5, 1), 32).shape == (0, 5)
