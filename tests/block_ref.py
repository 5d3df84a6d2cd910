"""64-bit references of the recurrent-block operators, each with a bound on how far an fp32
evaluation may be off, element by element. ``U`` is the largest relative error of one fp32
rounding, 2^-24; first-order terms are counted, and the bounds are doubled for the rest."""
from __future__ import annotations

import torch

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def rounding(y, dtype):
    """Half a step of the output's type, the smallest subnormal's at least."""
    return y.abs() * half_step(dtype) + torch.finfo(dtype).smallest_normal * half_step(dtype)


def starts_of(lens, lead=0):
    at = [lead]
    for n in lens:
        at.append(at[-1] + n)
    return at


def conv_ref(x, weight, bias, state, starts, slots, silu):
    """(y, bound of y, new state); rows outside the sequences are NaN in y."""
    w = weight.shape[1]
    y = torch.full(x.shape, float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(y)
    new = None if state is None else state.clone()
    for s in range(len(starts) - 1):
        slot = s if slots is None else int(slots[s])
        if slot < 0:
            continue
        old = torch.zeros(w - 1, x.shape[1], dtype=x.dtype) if state is None else state[slot]
        line = torch.cat((old, x[starts[s]:starts[s + 1]]))
        if new is not None:
            new[slot] = line[line.shape[0] - (w - 1):]
        for t in range(starts[s], starts[s + 1]):
            win = line[t - starts[s]:t - starts[s] + w].double().T
            p = win * weight.double()
            v, size = p.sum(1), p.abs().sum(1)
            if bias is not None:
                v, size = v + bias.double(), size + bias.double().abs()
            b = (w + 1) * U * size  # w products added one after another
            if silu:
                # |silu'| < 1.1; the exponential, the sum and the quotient are off by a few steps,
                # and the exponential's argument by |v| U
                v, b = v * torch.sigmoid(v), 1.1 * b + (8 + v.abs()) * U * (v * torch.sigmoid(v)).abs()
            y[t], bound[t] = v, 2 * b + rounding(v, x.dtype)
    return y, bound, new


def ssm_ref(x, dt, A, B, C, D, z, dt_bias, softplus, state, starts, slots, pieces=1):
    """(y, its bound, new state, its bound). ``pieces``: how many pieces a sequence may be
    computed in; each adds the rounding of a decay over a whole piece."""
    T, d = x.shape
    n = A.shape[1]
    B = B if B.dim() == 3 else B[:, None]
    C = C if C.dim() == 3 else C[:, None]
    per = d // B.shape[1]
    y = torch.full((T, d), float("nan"), dtype=torch.float64)
    ybound = torch.zeros_like(y)
    new = None if state is None else state.double()
    nbound = None if state is None else torch.zeros_like(new)
    Ad = A.double()
    for s in range(len(starts) - 1):
        slot = s if slots is None else int(slots[s])
        if slot < 0:
            continue
        h = torch.zeros(d, n, dtype=torch.float64) if state is None else state[slot].double()
        e = torch.zeros_like(h)
        for t in range(starts[s], starts[s + 1]):
            v = dt[t].double()
            verr = torch.zeros_like(v)
            if dt_bias is not None:
                v = v + dt_bias.double()
                verr = U * v.abs()
            delta, derr = v, verr
            if softplus:
                # the slope is a sigmoid; exp's argument, exp and log1p: a few steps each
                delta = torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))
                derr = verr * torch.sigmoid(v) + (6 + v.abs()) * U * delta
            xt = x[t].double()
            arg = delta[:, None] * Ad
            a = torch.exp(arg)
            # the decay's argument (two products, delta's own error) and the exponential (4 U,
            # the documented bound of the hardware's)
            aerr = a * (Ad.abs() * derr[:, None] + 3 * U * arg.abs() + 6 * U)
            b = (delta * xt)[:, None] * B[t].double().repeat_interleave(per, 0)
            bin_ = b.abs() * 3 * U + (xt.abs() * derr)[:, None] * B[t].double().repeat_interleave(per, 0).abs()
            e = a * e + aerr * h.abs() + bin_ + U * ((a * h).abs() + b.abs())
            h = a * h + b
            c = C[t].double().repeat_interleave(per, 0)
            v = (h * c).sum(1)
            err = (c.abs() * e).sum(1) + (n + 1) * U * (h * c).abs().sum(1)
            # a state carried over pieces: its decay's argument is a sum of the deltas
            err = err + (pieces - 1) * (c.abs() * 16 * U * h.abs()).sum(1)
            if D is not None:
                v = v + D.double() * xt
                err = err + 2 * U * ((D.double() * xt).abs() + v.abs())
            if z is not None:
                zt = z[t].double()
                g = zt * torch.sigmoid(zt)
                v, err = v * g, err * g.abs() + (10 + zt.abs()) * U * (v * g).abs()
            y[t], ybound[t] = v, 2 * err + rounding(v, x.dtype)
        if new is not None:
            new[slot], nbound[slot] = h, 2 * e + (pieces - 1) * 32 * U * h.abs() + 1e-37
    return y, ybound, new, nbound


def norm_quant_ref(x, weight, residual, eps, code, group):
    """(codes in their type, scales in 64 bits, new residual)."""
    r = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    rows, cols = x.shape
    t = r.float() * weight  # one fp32 rounding, part of the definition
    rms = torch.sqrt((r.double() ** 2).mean(1) + eps)
    g = group or cols
    parts = -(-cols // g)
    q = torch.zeros(rows, cols, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn)
    scales = torch.zeros(rows, parts, dtype=torch.float64)
    for p in range(parts):
        part = t[:, p * g:(p + 1) * g]
        most = part.abs().amax(1)
        scales[:, p] = most.double() / rms / (127 if code == "int8" else 448)
        m = most[:, None]
        if code == "int8":
            v = torch.round(part.double() * 127 / m.double()).nan_to_num(0)
            q[:, p * g:(p + 1) * g] = v.to(torch.int8)
        else:
            v = torch.where(m > 0, part * (448 / m), 0)
            q[:, p * g:(p + 1) * g] = v.to(torch.float8_e4m3fn)
    return q, scales, r


def int4_values(codes, zeros, group, in_dim):
    """u - z in 64 bits [out_dim, in_dim]."""
    u = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64)
    u[:, 0::2], u[:, 1::2] = (codes & 15).double(), (codes >> 4).double()
    u = u[:, :in_dim]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :in_dim]
    return u - z


def int4_ref(x, codes, scales, group, zeros=None, x_scales=None):
    """(out, its bound before the output's rounding)."""
    k = x.shape[1]
    w = int4_values(codes, zeros, group, k) * scales.double().repeat_interleave(group, 1)[:, :k]
    xv = x.double() if x.dtype != torch.float8_e4m3fn else x.float().double()
    if x_scales is not None:
        sx = x_scales.double()
        xv = xv * (sx if sx.shape[1] == 1 else sx.repeat_interleave(group, 1)[:, :k])
    out, size = xv @ w.T, xv.abs() @ w.abs().T
    # k products (exact, or one rounding each) added in some order in fp32, a tensor core's
    # addition being off by a whole step at most; the scales' products
    return out, (2 * k + 8) * U * size
