"""Cases of the recurrent-block operators: the selective scan, its short causal convolution, the
residual norm with an 8-bit output, and products with 4-bit weights.

Each case is one call of one operator as a serving program makes it. With ``own`` false ``run``
computes the operator's plain form in elementary torch operations; with ``own`` true it calls the
library. ``exact`` computes the same from the definition in 64 bits.
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
         "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "int8": 1, "e4m3": 1}


def listed():
    # widths are those of the 1.3B (hidden 2048, intermediate 5632) and 2.7B (hidden 2560)
    # configurations and of blocks twice as wide as their hidden size; 64 streams and 8 x 2048
    # prompt tokens are the serving and prefill workloads
    return [
        # one short prompt of a chat turn: latency
        dict(name="scan one short prompt", op="scan", type="fp32", tokens=37, seqs=1, channels=2048, states=16, groups=1),
        # one long document: few channels in flight, so that only its length is left to split
        dict(name="scan one long prompt", op="scan", type="fp32", tokens=4099, seqs=1, channels=4096, states=16, groups=1),
        # the prefill workload: ragged prompts packed without padding
        dict(name="scan 8 prompts", op="scan", type="bf16", tokens=16384, seqs=8, channels=5120, states=16, groups=1),
        # a token of one stream
        dict(name="step 1 stream", op="step", type="fp32", seqs=1, channels=2048, states=16, groups=1),
        # a token of each of 64 streams of a pool
        dict(name="step 64 streams", op="step", type="bf16", seqs=64, channels=4096, states=16, groups=1),
        # the convolution before that scan, at prefill
        dict(name="conv 8 prompts", op="conv", type="bf16", tokens=16384, seqs=8, channels=5120, width=4),
        # and for a token of 64 streams
        dict(name="conv 64 streams", op="conv_step", type="bf16", seqs=64, channels=4096, width=4),
        # the norm of one token, codes for an integer product
        dict(name="norm 1 row", op="norm", type="fp32", code="int8", rows=1, columns=2048, group=0, residual=True),
        # the prefill workload's norm, e4m3 with a scale for 128 columns
        dict(name="norm 16384 rows", op="norm", type="bf16", code="e4m3", rows=16384, columns=2560, group=128, residual=True),
        # batch-1 decode of a feed-forward's input projection on 8-bit rows
        dict(name="matvec 1 row", op="matvec", type="int8", rows=1, inputs=2048, outputs=11264, group=128, zeros=False),
        # the vocabulary head of one stream
        dict(name="matvec head", op="matvec", type="bf16", rows=1, inputs=2048, outputs=32000, group=128, zeros=False),
        # a feed-forward's output projection for 16 streams, with zero points, rows in 32 bits
        dict(name="matvec 16 rows", op="matvec", type="fp32", rows=16, inputs=5632, outputs=2048, group=64, zeros=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("scan", "scan", "step", "conv", "conv_step", "norm", "norm", "matvec", "matvec"))
    kind = rng.choice(("fp32", "bf16", "fp16"))
    if op in ("scan", "step"):
        groups = rng.choice((1, 1, 1, 2, 4))
        states = rng.choice((16, 16, 16, 1, 5, 8, 32, 64, 128))
        channels = groups * max(1, _log(rng, 64, 5120) // groups)
        if op == "step":
            seqs = min(_log(rng, 1, 256), max(1, (64 << 20) // (channels * states)))
            return dict(op=op, type=kind, seqs=seqs, channels=channels, states=states, groups=groups)
        tokens = min(_log(rng, 1, 16384), max(1, 16384 * 5120 * 16 // (channels * states)))
        return dict(op=op, type=kind, tokens=tokens, seqs=rng.randint(1, 16), channels=channels, states=states, groups=groups)
    if op == "conv":
        return dict(op=op, type=kind, tokens=_log(rng, 1, 16384), seqs=rng.randint(1, 16), channels=_log(rng, 64, 5120),
                    width=rng.choice((2, 3, 4, 4, 4, 7)))
    if op == "conv_step":
        return dict(op=op, type=kind, seqs=_log(rng, 1, 256), channels=_log(rng, 64, 6912), width=rng.choice((2, 3, 4, 4, 4, 7)))
    if op == "norm":
        return dict(op=op, type=kind, code=rng.choice(("int8", "e4m3")), rows=_log(rng, 1, 16384), columns=_log(rng, 64, 2560),
                    group=rng.choice((0, 0, 32, 64, 128)), residual=rng.random() < 0.75)
    kind = rng.choice(("fp32", "bf16", "fp16", "int8", "e4m3"))
    return dict(op=op, type=kind, rows=_log(rng, 1, 32), inputs=_log(rng, 64, 6912), outputs=_log(rng, 16, 32000) if kind != "fp32"
                else _log(rng, 16, 12000), group=rng.choice((32, 64, 128, 128)), zeros=rng.random() < 0.5)


def _lengths(case):
    """Lengths of the packed sequences: ragged, a few of them very short or empty, the same for every seed."""
    rng = random.Random(case["tokens"] * 131 + case["seqs"])
    if case["seqs"] == 1:
        return [case["tokens"]]
    share = [rng.choice((0.0, 0.02, 0.5, 1.0, 1.0, 1.0, 1.5)) for _ in range(case["seqs"] - 1)] + [1.0]
    lens = [int(case["tokens"] * s / sum(share)) for s in share]
    lens[-1] += case["tokens"] - sum(lens)
    return lens


def _groups(columns, group):
    return -(-columns // group) if group else 1


def work(case):
    op, e = case["op"], BYTES[case["type"]]
    if op in ("scan", "step"):
        t = case["tokens"] if op == "scan" else case["seqs"]
        d, n, g = case["channels"], case["states"], case["groups"]
        return {"bytes": t * d * 4 * e + t * 2 * g * n * e + d * (n + 2) * 4 + 2 * case["seqs"] * d * n * 4,
                # the exponent's product, the exponential, the decay, the input and the output product
                "flops": t * d * n * 7 + t * d * 8}
    if op in ("conv", "conv_step"):
        t = case["tokens"] if op == "conv" else case["seqs"]
        d, w = case["channels"], case["width"]
        return {"bytes": t * d * 2 * e + 2 * case["seqs"] * (w - 1) * d * e + d * (w + 1) * 4, "flops": t * d * (2 * w + 5)}
    if op == "norm":
        r, c = case["rows"], case["columns"]
        return {"bytes": r * c * (e * (3 if case["residual"] else 1) + 1) + 4 * c + 4 * r * _groups(c, case["group"]), "flops": 8 * r * c}
    m, k, n = case["rows"], case["inputs"], case["outputs"]
    out = 2 if case["type"] in ("bf16", "fp16") else 4
    return {"bytes": n * (-(-k // 2)) + n * _groups(k, case["group"]) * (3 if case["zeros"] else 2) + m * k * e + m * n * out
            + (4 * m if e == 1 else 0), "flops": 2 * m * n * k}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, kind = case["op"], TYPES[case["type"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    def uniform(low, high, *shape):
        return low + (high - low) * torch.rand(*shape, device="cuda", generator=gen)

    s = dict(case)
    if op in ("scan", "conv"):
        lens = _lengths(case)
        s["longest"] = max(lens)
        s["starts"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        t = case["tokens"]
    if op in ("step", "conv_step"):
        t = case["seqs"]
        pool = t + t // 4 + 1  # the pool has room for streams that are not in this batch
        s["slots"] = torch.randperm(pool, device="cuda", generator=gen)[:t].to(torch.int32)
    if op in ("scan", "step"):
        d, n, g = case["channels"], case["states"], case["groups"]
        # x and its gate are the two halves of one projection's output, B and C those of another
        xz = normal(t, 2 * d).to(kind)
        s["x"], s["z"] = xz[:, :d], xz[:, d:]
        bc = normal(t, 2 * g * n).to(kind)
        s["B"], s["C"] = bc[:, : g * n].unflatten(1, (g, n)), bc[:, g * n:].unflatten(1, (g, n))
        # step sizes from 0.001 to 0.1 on a logarithmic scale, decay rates from 1 to the number of states
        s["dt"] = normal(t, d, std=0.5).to(kind)
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), d))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["A"] = -torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * uniform(0.9, 1.1, d, n)
        s["D"] = normal(d)
        s["state"] = normal(case["seqs"] if op == "scan" else pool, d, n, std=0.1)
    elif op in ("conv", "conv_step"):
        d, w = case["channels"], case["width"]
        s["x"] = normal(t, 2 * d).to(kind)[:, :d]  # the first half of a projection's output
        s["weight"], s["bias"] = normal(d, w, std=w ** -0.5), normal(d, std=0.1)
        s["state"] = normal(case["seqs"] if op == "conv" else pool, w - 1, d).to(kind)
    elif op == "norm":
        r, c = case["rows"], case["columns"]
        s["x"] = normal(r, c).to(kind)
        outlier = 1 + 9 * (uniform(0, 1, c) < 0.01)  # a few columns of a residual stream are much larger
        s["residual_in"] = (normal(r, c) * outlier).to(kind) if case["residual"] else None
        s["weight"] = uniform(0.5, 1.5, c)
    else:
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        s["codes"] = torch.randint(0, 256, (n, -(-k // 2)), device="cuda", generator=gen, dtype=torch.uint8)
        parts = _groups(k, case["group"])
        s["scales"] = (uniform(0.5, 1.5, n, parts) * 0.2 * k ** -0.5).to(torch.float16)
        s["zeros"] = torch.randint(4, 12, (n, parts), device="cuda", generator=gen, dtype=torch.uint8) if case["zeros"] else None
        x = normal(m, k)
        if case["type"] in ("int8", "e4m3"):
            most = 127.0 if case["type"] == "int8" else 448.0
            s["x_scales"] = x.abs().amax(1, keepdim=True) / most
            x = x / s["x_scales"]
            s["x"] = torch.round(x).to(kind) if case["type"] == "int8" else x.to(kind)
        else:
            s["x"], s["x_scales"] = x.to(kind), None
    return s


def run(s):
    return (_library if own else _plain)[s["op"]](s)


# ---- the library's calls ---------------------------------------------------------------------

def _scan_library(s):
    from matmulfreellmcpu_b200 import selective_scan
    y = selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                       state=s["state"], seq_starts=s["starts"])
    return y, s["state"]


def _step_library(s):
    from matmulfreellmcpu_b200 import selective_step
    y = selective_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                       slots=s["slots"])
    return y, s["state"]


def _conv_library(s):
    from matmulfreellmcpu_b200 import causal_conv
    y = causal_conv(s["x"], s["weight"], bias=s["bias"], state=s["state"], seq_starts=s["starts"], silu=True)
    return y, s["state"]


def _conv_step_library(s):
    from matmulfreellmcpu_b200 import causal_conv_step
    y = causal_conv_step(s["x"], s["weight"], s["state"], bias=s["bias"], slots=s["slots"], silu=True)
    return y, s["state"]


def _norm_library(s):
    from matmulfreellmcpu_b200 import add_rmsnorm_quant
    q, scales = add_rmsnorm_quant(s["x"], s["weight"], residual=s["residual_in"], eps=1e-6, code=s["code"], group=s["group"])
    return (q, scales) if s["residual_in"] is None else (q, scales, s["residual_in"])


def _matvec_library(s):
    from matmulfreellmcpu_b200 import int4_matvec
    return int4_matvec(s["x"], s["codes"], s["scales"], s["group"], zeros=s["zeros"], x_scales=s["x_scales"])


_library = {"scan": _scan_library, "step": _step_library, "conv": _conv_library, "conv_step": _conv_step_library,
            "norm": _norm_library, "matvec": _matvec_library}


# ---- the plain forms -------------------------------------------------------------------------

def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v)))


def _silu(v):
    return v / (1 + torch.exp(-v))


def _terms(s):
    """Decay and input of every token, channel and state."""
    x, delta = s["x"].float(), _softplus(s["dt"].float() + s["dt_bias"])
    decay = torch.exp(delta[:, :, None] * s["A"])
    b = s["B"].float().repeat_interleave(x.shape[1] // s["groups"], 1)
    return x, decay, (delta * x)[:, :, None] * b


def _outputs(s, x, h):
    """What the states give, the skip and the gate."""
    c = s["C"].float().repeat_interleave(x.shape[1] // s["groups"], 1)
    return (((h * c).sum(2) + s["D"] * x) * _silu(s["z"].float())).to(s["x"].dtype)


def _scan_plain(s):
    x, decay, h = _terms(s)
    first, after = s["starts"][:-1].long(), s["starts"][1:].long()
    held = (after > first)[:, None, None]  # sequences that have a token
    at = first.clamp(max=x.shape[0] - 1)
    h = h.index_add(0, at, torch.where(held, decay[at] * s["state"], 0))
    begins = torch.zeros(x.shape[0] + 1, dtype=torch.bool, device=x.device)
    begins[first] = True
    decay = torch.where(begins[:-1, None, None], 0, decay)
    # the recurrence by doubling: after each turn every state holds twice as many tokens
    far = 1
    while far < s["longest"]:
        h = torch.cat((h[:far], torch.addcmul(h[far:], decay[far:], h[:-far])))
        decay = torch.cat((decay[:far], decay[far:] * decay[:-far]))
        far *= 2
    s["state"].copy_(torch.where(held, h[(after - 1).clamp(min=0)], s["state"]))
    return _outputs(s, x, h), s["state"]


def _step_plain(s):
    x, decay, inputs = _terms(s)
    at = s["slots"].long()
    h = decay * s["state"][at] + inputs
    s["state"][at] = h
    return _outputs(s, x, h), s["state"]


def _conv_plain(s):
    x, w = s["x"], s["width"]
    t = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(s["starts"][1:], t.int(), right=True).long()
    first, after = s["starts"][:-1].long(), s["starts"][1:].long()

    def inputs(seq, at):
        """The sequences' inputs at these places, those before their first token from the state."""
        back = at - first[seq]
        past = s["state"][seq, (back + w - 1).clamp(0, w - 2)]
        return torch.where((back >= 0)[..., None], x[at.clamp(0, x.shape[0] - 1)], past)

    y = sum((inputs(seq, t - (w - 1) + j).float() * s["weight"][:, j] for j in range(w)), s["bias"])
    which = torch.arange(first.shape[0], device=x.device)[:, None]
    last = inputs(which, after[:, None] - (w - 1) + torch.arange(w - 1, device=x.device))
    s["state"].copy_(last)
    return _silu(y).to(x.dtype), s["state"]


def _conv_step_plain(s):
    at = s["slots"].long()
    window = torch.cat((s["state"][at], s["x"][:, None]), 1)
    s["state"][at] = window[:, 1:]
    y = (window.float() * s["weight"].T).sum(1) + s["bias"]
    return _silu(y).to(s["x"].dtype), s["state"]


def _norm_plain(s):
    r = s["x"]
    if s["residual_in"] is not None:
        r = (s["residual_in"].float() + s["x"].float()).to(s["x"].dtype)
        s["residual_in"].copy_(r)
    r = r.float()
    rows, columns = r.shape
    rstd = torch.rsqrt(r.square().mean(1, keepdim=True) + 1e-6)
    group = s["group"] or columns
    t = torch.nn.functional.pad(r * s["weight"], (0, _groups(columns, group) * group - columns)).view(rows, -1, group)
    most = t.abs().amax(2, keepdim=True)
    if s["code"] == "int8":
        # in 64 bits, so that values next to a border between two codes fall on its right side
        q = torch.round(t.double() * 127 / most.double()).to(torch.int8)
    else:
        q = (t * (448 / most)).to(torch.float8_e4m3fn)
    scales = most[..., 0] * rstd / (127 if s["code"] == "int8" else 448)
    q = q.view(rows, -1)[:, :columns].contiguous()
    return (q, scales) if s["residual_in"] is None else (q, scales, s["residual_in"])


def _matvec_plain(s):
    columns = s["inputs"]
    u = torch.stack((s["codes"] & 15, s["codes"] >> 4), 2).flatten(1)[:, :columns].float()
    scales = s["scales"].float().repeat_interleave(s["group"], 1)[:, :columns]
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(s["group"], 1)[:, :columns]
    out = s["x"].float() @ ((u - zeros) * scales).T
    return out.to(s["x"].dtype) if s["x_scales"] is None else out * s["x_scales"]


_plain = {"scan": _scan_plain, "step": _step_plain, "conv": _conv_plain, "conv_step": _conv_step_plain,
          "norm": _norm_plain, "matvec": _matvec_plain}


# ---- the definitions in 64 bits --------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("scan", "step"):
        if op == "scan":
            lens = _lengths(case)
            where = range(len(lens))
        else:
            lens, where = [1] * case["seqs"], s["slots"].tolist()
        first = torch.tensor([sum(lens[:i]) for i in range(len(lens))], device="cuda")
        per = case["channels"] // case["groups"]
        x, z = s["x"].double(), s["z"].double()
        v = s["dt"].double() + s["dt_bias"].double()
        delta = torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))
        rates = s["A"].double()
        slots = torch.tensor(list(where), device="cuda")
        final = s["state"].double()
        y = torch.zeros_like(x)
        order = sorted(range(len(lens)), key=lambda i: -lens[i])  # longest first: those that go on are a prefix
        first, slots = first[order], slots[order]
        h = final[slots]
        for t in range(max(lens)):
            live = sum(n > t for n in lens)
            at = first[:live] + t
            d = delta[at][:, :, None]
            b = s["B"][at].double().repeat_interleave(per, 1)
            c = s["C"][at].double().repeat_interleave(per, 1)
            h[:live] = torch.exp(d * rates) * h[:live] + d * x[at][:, :, None] * b
            y[at] = torch.einsum("sdn,sdn->sd", h[:live], c)
        final[slots] = h
        return (y + s["D"].double() * x) * z * torch.sigmoid(z), final
    if op in ("conv", "conv_step"):
        w = case["width"]
        lens = _lengths(case) if op == "conv" else [1] * case["seqs"]
        where = range(len(lens)) if op == "conv" else s["slots"].tolist()
        final, outs = s["state"].double(), []
        for one, slot in zip(s["x"].double().split(lens), where):
            line = torch.cat((final[slot], one))
            final[slot] = line[line.shape[0] - (w - 1):]
            if one.shape[0]:
                outs.append(torch.einsum("tdw,dw->td", line.unfold(0, w, 1), s["weight"].double()))
        y = torch.cat(outs) + s["bias"].double()
        return y * torch.sigmoid(y), final
    if op == "norm":
        r = s["x"].double()
        if s["residual_in"] is not None:
            r = r + s["residual_in"].double()
        kept = r.to(s["x"].dtype).double()  # the norm is that of the residual as it is kept
        rms = torch.sqrt((kept ** 2).mean(1, keepdim=True) + 1e-6)
        t = kept * s["weight"].double() / rms
        most = torch.stack([part.abs().amax(1) for part in t.split(case["group"] or case["columns"], 1)], 1)
        scales = most / (127 if case["code"] == "int8" else 448)
        return (None, scales) if s["residual_in"] is None else (None, scales, r)
    k, n = case["inputs"], case["outputs"]
    u = torch.empty(n, 2 * s["codes"].shape[1], dtype=torch.float64, device="cuda")
    u[:, 0::2], u[:, 1::2] = s["codes"] % 16, s["codes"] // 16
    out = torch.zeros(case["rows"], n, dtype=torch.float64, device="cuda")
    for g in range(_groups(k, case["group"])):
        part = slice(g * case["group"], min(k, (g + 1) * case["group"]))
        zero = 8 if s["zeros"] is None else s["zeros"][:, g, None].double()
        out += s["scales"][:, g].double() * (s["x"][:, part].double() @ (u[:, part] - zero).T)
    return out if s["x_scales"] is None else out * s["x_scales"].double()
