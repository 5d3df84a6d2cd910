"""GPU tests of the recurrent-block operators at sizes that reach the shapes and loops of serving: several streams a thread,
several weight-row blocks and rows a CTA, two channels a lane, and split sequences in every layout."""
from __future__ import annotations

import pytest
import torch

import block_ref as R
from matmulfreellmcpu_b200 import api
from test_gpu_block_ops import SENTINEL, close, dev, int4_inputs, rng, run_ssm, sliced, ssm_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("streams,channels,states,groups", [(77, 1200, 16, 1), (78, 1201, 16, 1), (79, 1200, 5, 4), (41, 300, 100, 1), (77, 130, 256, 2)])
def test_steps_of_four_streams_a_thread(cuda, streams, channels, states, groups, kind):
    pool = streams + 3
    p = ssm_inputs(streams, channels, states, groups, kind, channels, pool)
    slots = torch.randperm(pool, generator=rng(1))[:streams].to(torch.int32)
    slots[torch.tensor([0, 6, 7, 20, 21, 22, 23, streams - 1])] = -1
    want, bound, new, nbound = R.ssm_ref(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], True, p["state"],
                                         list(range(streams + 1)), slots)
    d = {k: v.to(cuda) for k, v in p.items()}
    out = torch.full_like(d["x"], SENTINEL)
    api.selective_step(d["x"], d["dt"], d["A"], d["B"], d["C"], d["state"], d["D"], d["z"], d["dt_bias"], slots=slots.to(cuda), out=out)
    inside = ~torch.isnan(want)
    close(out.cpu()[inside], want[inside], bound[inside], "y")
    assert (out.cpu()[~inside] == SENTINEL).all()
    close(d["state"], new, nbound, "state")
    idle = [i for i in range(pool) if i not in slots.tolist()]
    assert torch.equal(d["state"].cpu()[idle], p["state"][idle])
    api.kernel_status()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("channels,states,groups,extra", [(1024, 16, 1, 0), (1024, 16, 1, 1), (1023, 13, 1, 0), (1040, 16, 2, 8), (1024, 12, 4, 2)])
def test_scans_of_two_channels_a_lane(cuda, channels, states, groups, extra, kind):
    """Many short sequences over many channels."""
    lens = [17, 1, 16, 0, 40, 3, 15, 33, 2, 18, 31, 1, 64, 5, 20, 9]
    starts = R.starts_of(lens, 2)
    p = ssm_inputs(starts[-1] + 1, channels, states, groups, kind, channels, 18)
    slots = torch.randperm(18, generator=rng(3))[:16].to(torch.int32)
    slots[4] = -1
    want, bound, new, nbound = R.ssm_ref(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], True, p["state"], starts, slots)
    out, state = run_ssm(cuda, p, starts, slots, extra)
    inside = ~torch.isnan(want)
    close(out[inside], want[inside], bound[inside], "y")
    assert (out[~inside] == SENTINEL).all()
    close(state, new, nbound, "state")
    api.kernel_status()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("lens,channels,states,groups,extra", [
    ([1500, 0, 2100, 1], 40, 16, 2, 8), ([1700], 33, 16, 1, 1), ([900, 1300], 24, 5, 4, 2), ([1200, 400, 1], 12, 100, 2, 0),
    ([2000, 700], 48, 16, 1, 3), ([63] + [1] * 2 + [2300], 64, 16, 4, 4)])
def test_split_scans_in_every_layout(cuda, lens, channels, states, groups, extra, kind):
    """Sequences that a cluster's CTAs share: groups, permuted slots and a sequence that is left out, rows in front and behind,
    strided rows; then without state, skip, gate, bias and softplus."""
    starts = R.starts_of(lens, 3)
    pool = len(lens) + 2
    p = ssm_inputs(starts[-1] + 2, channels, states, groups, kind, channels, pool)
    slots = torch.randperm(pool, generator=rng(4))[:len(lens)].to(torch.int32)
    if len(lens) > 1:
        slots[0 if len(lens) == 2 else len(lens) - 1] = -1
    for drop, softplus, sl in (((), True, slots), (("D", "z", "dt_bias", "state"), False, None)):
        if not softplus:
            p["dt"] = p["dt"].abs() * 0.1
        q = {k: (None if k in drop else v) for k, v in p.items()}
        want, bound, new, nbound = R.ssm_ref(q["x"], q["dt"], q["A"], q["B"], q["C"], q["D"], q["z"], q["dt_bias"], softplus,
                                             q["state"], starts, sl, pieces=16)
        out, state = run_ssm(cuda, p, starts, sl, extra, softplus, drop)
        inside = ~torch.isnan(want)
        close(out[inside], want[inside], bound[inside], "y")
        assert (out[~inside] == SENTINEL).all()
        if state is not None:
            close(state, new, nbound, "state")
            idle = [i for i in range(pool) if i not in sl.tolist()]
            assert torch.equal(state[idle], p["state"][idle])
    api.kernel_status()


@pytest.mark.parametrize("kind", ["fp32", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("m", [1, 9, 17])
@pytest.mark.parametrize("extra", [0, 1])
def test_int4_matvec_of_several_weight_row_blocks(cuda, m, extra, kind):
    """More weight rows than the device's CTAs hold at once."""
    x, codes, scales, z, xs = int4_inputs(m, 320, 9617, 64, True, kind, m)
    want, bound = R.int4_ref(x, codes, scales, 64, z, xs)
    xd, sd, zd, xsd = dev(cuda, x, scales, z, xs)
    out = api.int4_matvec(xd, sliced(codes, extra, cuda), sd, 64, zeros=zd, x_scales=xsd)
    close(out, want, bound + R.rounding(want, out.dtype), f"{m} rows")


def e4m3_codes(r, w, group):
    """e4m3(t * (448 / m)) with a correctly rounded quotient. (A number divided by a tensor is the number times the tensor's
    reciprocal in torch: one more rounding, and another code for one value in some hundred thousand.)"""
    t = r.float() * w
    parts = []
    for part in t.split(group or t.shape[1], 1):
        m = part.abs().amax(1, keepdim=True)
        parts.append((part * torch.div(torch.full_like(m, 448.0), m)).to(torch.float8_e4m3fn))
    return torch.cat([p.view(torch.uint8) for p in parts], 1)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols,group,extra", [(6000, 64, 0, 0), (6000, 100, 32, 3), (3001, 1032, 0, 0), (3001, 1100, 128, 4), (900, 9000, 64, 0)])
def test_norms_of_more_rows_than_the_device_holds(cuda, rows, cols, group, extra, kind, code):
    g = rng(cols)
    x, res = torch.randn(rows, cols, generator=g).to(R.TYPES[kind]), torch.randn(rows, cols, generator=g).to(R.TYPES[kind])
    w = 0.5 + torch.rand(cols, generator=g)
    for residual in (None, res):
        q, s, r = R.norm_quant_ref(x, w, residual, 1e-6, code, group)
        rd = None if residual is None else sliced(residual, extra, cuda)
        gq, gs = api.add_rmsnorm_quant(sliced(x, extra, cuda), w.to(cuda), rd, 1e-6, code, group)
        assert torch.equal(gq.cpu().view(torch.uint8), q.view(torch.uint8) if code == "int8" else e4m3_codes(r, w, group))
        close(gs, s, s * (cols / 2 + 6) * R.U, "scales")
        if residual is not None:
            assert torch.equal(rd.cpu(), r)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_convolutions_of_many_tiles(cuda, kind):
    """Sequences that begin, end and stay short across tiles of every height, a batch of single tokens among them."""
    for lens, channels in (([300, 1, 2, 0, 63, 64, 65, 700, 1], 520), ([1] * 150, 260), ([5000], 24)):
        starts = R.starts_of(lens, 1)
        g = rng(len(lens))
        x = torch.randn(starts[-1] + 2, channels, generator=g).to(R.TYPES[kind])
        w, b = torch.randn(channels, 4, generator=g), torch.randn(channels, generator=g)
        state = torch.randn(len(lens) + 1, 3, channels, generator=g).to(R.TYPES[kind])
        slots = torch.randperm(len(lens) + 1, generator=g)[:len(lens)].to(torch.int32)
        want, bound, new = R.conv_ref(x, w, b, state, starts, slots, True)
        st, out = state.to(cuda), torch.full(x.shape, SENTINEL, dtype=x.dtype, device=cuda)
        api.causal_conv(x.to(cuda), w.to(cuda), b.to(cuda), st, torch.tensor(starts, dtype=torch.int32, device=cuda), slots.to(cuda), True, out=out)
        inside = ~torch.isnan(want)
        close(out.cpu()[inside], want[inside], bound[inside], f"{len(lens)} sequences")
        assert (out.cpu()[~inside] == SENTINEL).all() and torch.equal(st.cpu(), new)
    api.kernel_status()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_rows_farther_apart_than_32_bits(cuda, kind):
    """Row pitches with which the last rows lie behind 2^32 elements."""
    dtype = R.TYPES[kind]
    rows, pitch, channels = 37, 1 << 27, 40
    wide = torch.empty(rows * pitch, dtype=dtype, device=cuda).view(rows, pitch)
    p = ssm_inputs(rows, channels, 16, 1, kind, 5, 1)
    p["B"], p["C"] = p["B"][:, 0], p["C"][:, 0]
    far = {}
    for i, k in enumerate(("x", "dt", "z", "B", "C")):
        far[k] = wide[:, 64 * i:64 * i + p[k].shape[1]]
        far[k].copy_(p[k])
    out = wide[:, 512:512 + channels]
    d = {k: v.to(cuda) for k, v in p.items()}
    scan = lambda q, st, o: api.selective_scan(q["x"], q["dt"], d["A"], q["B"], q["C"], d["D"], q["z"], d["dt_bias"], state=st, out=o)  # noqa: E731
    s1, s2 = d["state"].clone(), d["state"].clone()
    assert torch.equal(scan(far, s1, out), scan(d, s2, None)) and torch.equal(s1, s2)
    pool = torch.randn(rows, channels, 16, device=cuda)
    step = lambda q, st, o: api.selective_step(q["x"], q["dt"], d["A"], q["B"], q["C"], st, d["D"], q["z"], d["dt_bias"], out=o)  # noqa: E731
    s1, s2 = pool.clone(), pool.clone()
    assert torch.equal(step(far, s1, out), step(d, s2, None)) and torch.equal(s1, s2)
    w = torch.randn(channels, 4, device=cuda)
    assert torch.equal(api.causal_conv(far["x"], w, out=out), api.causal_conv(d["x"], w))
    s1 = torch.randn(rows, 3, channels, device=cuda).to(dtype)
    s2 = s1.clone()
    assert torch.equal(api.causal_conv_step(far["x"], w, s1, out=out), api.causal_conv_step(d["x"], w, s2)) and torch.equal(s1, s2)
    ones = torch.ones(channels, device=cuda)
    r = d["dt"].clone()
    for a, b in zip(api.add_rmsnorm_quant(far["x"], ones, far["dt"]), api.add_rmsnorm_quant(d["x"], ones, r)):
        assert torch.equal(a.float(), b.float())
    assert torch.equal(far["dt"], r)
    _, codes, scales, _, _ = int4_inputs(1, channels, 60, 32, False, "fp32", 3)
    cd, sd = dev(cuda, codes, scales)
    want = api.int4_matvec(d["x"], cd, sd, 32)
    assert torch.equal(api.int4_matvec(far["x"], cd, sd, 32), want)
    bytes_ = wide.view(-1).view(torch.uint8)
    for start in (0, 5):  # rows of codes at aligned and at odd addresses
        rows_of = bytes_[:60 * (1 << 27)].view(60, 1 << 27)[:, 4096 + start:4096 + start + codes.shape[1]]
        rows_of.copy_(codes)
        assert torch.equal(api.int4_matvec(d["x"], rows_of, sd, 32), want)
    api.kernel_status()


def test_every_operator_on_two_other_streams_at_once_and_captured(cuda):
    """Calls with ``stream``, on two streams that overlap and in graphs of two streams, give what the current stream gives: a
    split scan, products over a cluster, rows whose scales and outputs are taken again, and the steps."""
    p = {k: v.to(cuda) for k, v in ssm_inputs(2000, 48, 16, 1, "fp32", 5, 1).items()}
    w, x = torch.randn(48, 4, device=cuda), torch.randn(9, 5632, device=cuda)
    x[3] *= 1e25
    x[5, 7] = torch.inf
    _, codes, scales, _, _ = int4_inputs(1, 5632, 160, 64, False, "fp32", 3)
    cd, sd = dev(cuda, codes, scales)
    rows = slice(0, 40)

    def run(stream=None):
        st, conv, pool = p["state"].clone(), torch.zeros(40, 3, 48, device=cuda), torch.ones(40, 48, 16, device=cuda)
        y = api.selective_scan(p["x"], p["dt"], p["A"], p["B"], p["C"], p["D"], p["z"], p["dt_bias"], state=st, stream=stream)
        c = api.causal_conv(p["x"], w, stream=stream)
        cs = api.causal_conv_step(p["x"][rows], w, conv, stream=stream)
        s = api.selective_step(p["x"][rows], p["dt"][rows], p["A"], p["B"][rows], p["C"][rows], pool, stream=stream)
        q, qs = api.add_rmsnorm_quant(x, torch.ones(5632, device=cuda), eps=0.0, stream=stream)
        m = api.int4_matvec(x, cd, sd, 64, stream=stream)
        return y, st, c, cs, conv, s, pool, q, qs.nan_to_num(7.0), m.nan_to_num(7.0)

    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for side in streams:
            with torch.cuda.stream(side):
                got.append(run(side))
    graphs = []
    for side in streams:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = run()
        graphs.append((side, graph, outs))
    for side, graph, _ in graphs:
        with torch.cuda.stream(side):
            graph.replay()
    torch.cuda.synchronize()
    for outs in got + [g[2] for g in graphs]:
        for i, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), i
