"""Definitions of the sequence operators in 64 bits with error bounds for a computation in the given element type.

Bounds: u = eps / 2 of the element type (one rounding), e = 2^-24 (one fp32 operation).  A sum of n products in fp32 is off by at most
(n + 2) e sum |a b| whatever its order; an operand that is rounded to the element type first adds u |a b| a product.  The bounds below are
these rules applied to each formula, worst case, so they need no allowance for luck."""
import math

import torch

E = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}       # half a step of the smallest numbers (flushed at worst)


def rounded(x, t):
    return UNIT[t] * x.abs() + TINY[t]


def attention(q, k, v, dout=None, causal=False, scale=None, mask=None, swept=False, parts=False):
    """One head: q [n, D], k, v [m, D] -> {name: (value, bound)} of out, lse (and dq, dk, dv).  mask [m]: which keys take part.
    swept: D = sum_d dout out is corrected by sum_j P_j (dP_j - D), so the rounding of `out` is not in it (blocks of at most 256 keys).
    parts: P and dS go into the gradients' products as two numbers of the element type (at most 64 keys and 32 queries): u^2 in place of u."""
    t = q.dtype
    u = 0.0 if t == torch.float32 else UNIT[t]                        # P and dS are rounded only where the matrix operand is 16 bits
    q, k, v = q.double(), k.double(), v.double()
    n, m, D = q.shape[0], k.shape[0], q.shape[1]
    scale = D ** -0.5 if scale is None else scale
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(m - n)
    if mask is not None:
        seen = seen & mask[None]
        k, v = k.masked_fill(~mask[:, None], 0.0), v.masked_fill(~mask[:, None], 0.0)
    some = seen.any(1)
    q = q.masked_fill(~some[:, None], 0.0)                            # a row that sees nothing takes no part
    S = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(S, 1) if m else torch.full((n,), -math.inf, dtype=torch.float64, device=q.device)
    base = torch.where(some, lse, torch.zeros_like(lse))[:, None]
    P = torch.exp(S - base)
    # S: a sum of D products, the scaling and the change to powers of two (the exponent's argument is off by its own size too)
    dS0 = ((D + 4) * E * scale * (q.abs() @ k.abs().T)).masked_fill(~seen, 0.0)
    top = dS0.amax(1, keepdim=True) if m else dS0.new_zeros(n, 1)
    size = (S - base).masked_fill(~seen, 0.0).abs()
    relP = torch.expm1(2 * (dS0 + top + 4 * E * (size + base.abs())) + (m + 16) * E)   # (the sum l and the exponential itself: (m + 16) e)
    out = P @ v
    b_out = (P * (u * (1 + relP) + relP + (m + 4) * E)) @ v.abs()
    b_out = b_out * (1 + UNIT[t]) + rounded(out, t)
    b_lse = torch.where(some, (top.squeeze(1) + (m + 24) * E + 4 * E * base.squeeze(1).abs()), torch.zeros_like(lse))
    r = {"out": (out, b_out), "lse": (lse, b_lse)}
    if dout is None:
        return r
    g = dout.double().masked_fill(~some[:, None], 0.0)
    dP = g @ v.T
    delta = (g * out).sum(1, keepdim=True)
    b_delta = (g.abs() * (b_out + (D + 2) * E * out.abs())).sum(1, keepdim=True)
    b_dP = (D + 2) * E * (g.abs() @ v.abs().T)
    relP = torch.expm1(torch.log1p(relP) + b_lse[:, None])            # P from the rounded lse
    if swept:                                                         # what is left of D's error: times 1 - sum P, and the errors of the sweep's own sum
        off = dP.abs() * 4 * E + b_dP + (dP - delta).abs() + b_delta
        b_delta = (P * ((1 + relP) * (b_dP + 4 * E * (dP.abs() + delta.abs())) + (relP + (m + 4) * E) * off)).sum(1, keepdim=True)
    T = P * (dP - delta)
    b_T = P * (1 + relP) * (b_dP + b_delta + 4 * E * (dP.abs() + delta.abs())) + T.abs() * relP
    if parts:
        u = u * u
    b_T = b_T + u * (T.abs() + b_T)
    if t == torch.float16:                                            # the column's power of two keeps its largest entry above 2^14: steps below 2^-14 are 2^-24
        b_T = b_T + 2.0 ** -39 * torch.maximum(T.abs().amax(0, keepdim=True) if n else T.new_zeros(1, m), T.abs().amax(1, keepdim=True) if m else T.new_zeros(n, 1))
        tinyP = 2.0 ** -40                                            # 2^15 P, half a step of 2^-24
    else:
        tinyP = 0.0
    dq, dk, dv = T @ k * scale, T.T @ q * scale, P.T @ g
    b_dq = (b_T + (m + 4) * E * T.abs()) @ k.abs() * scale
    b_dk = (b_T + (n + 4) * E * T.abs()).T @ q.abs() * scale
    b_dv = (P * (relP + u * (1 + relP) + (n + 4) * E) + tinyP).T @ g.abs()
    for name, x, b in (("dq", dq, b_dq), ("dk", dk, b_dk), ("dv", dv, b_dv)):
        r[name] = (x, b)
    return r


def add_rounding(x, b, t):
    """The bound of x after its last rounding (dq, dk, dv: after the sum over a group of heads)."""
    return b * (1 + UNIT[t]) + rounded(x, t)


def layer_norm(x, w, b, eps, dy=None, pt=torch.float32):
    """x [rows, C] -> {name: (value, bound)}."""
    t = x.dtype
    x = x.double()
    rows, C = x.shape
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    mu = x.mean(1, keepdim=True)
    c = x - mu
    var = (c * c).mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = c * rstd
    b_mu = (C + 3) * E * x.abs().mean(1, keepdim=True)
    b_c = b_mu + E * (c.abs() + b_mu)
    # var: each centred value off by b_c, a sum of C squares; + eps, the root and the division
    b_var = (2 * c.abs() * b_c + b_c ** 2).mean(1, keepdim=True) + (C + 4) * E * (var + (b_c ** 2).mean(1, keepdim=True))
    lo = (var + eps - b_var).clamp_min(eps * (1 - 4 * E))
    rel = (var + eps).sqrt() / lo.sqrt() - 1 + 6 * E
    b_xh = (b_c * (1 + rel) + c.abs() * rel) * rstd + 2 * E * xh.abs()
    y = xh * w + b
    b_y = b_xh * w.abs() + 3 * E * ((xh * w).abs() + b.abs())
    r = {"y": (y, b_y * (1 + UNIT[t]) + rounded(y, t)), "mean": (mu, b_mu), "rstd": (rstd, rstd * rel)}
    if dy is None:
        return r
    dy = dy.double()
    g = dy * w
    a, s = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    b_a = (C + 4) * E * g.abs().mean(1, keepdim=True)
    b_s = (g.abs() * (b_xh + (C + 5) * E * xh.abs())).mean(1, keepdim=True)
    z = g - a - xh * s
    b_z = E * g.abs() + b_a + xh.abs() * b_s + s.abs() * b_xh + b_xh * b_s + 4 * E * (g.abs() + a.abs() + (xh * s).abs())
    dx = rstd * z
    b_dx = rstd * (b_z * (1 + rel) + z.abs() * (rel + 2 * E))
    dw, db = (dy * xh).sum(0), dy.sum(0)
    b_dw = (dy.abs() * (b_xh + (rows + 4) * E * xh.abs())).sum(0)
    b_db = (rows + 4) * E * dy.abs().sum(0)
    for name, v, e, tt in (("dx", dx, b_dx, t), ("dw", dw, b_dw, pt), ("db", db, b_db, pt)):
        r[name] = (v, e * (1 + UNIT[tt]) + rounded(v, tt))
    return r


def rotary(x, positions, frequencies, layout, factor=1.0, transpose=False):
    """x [B, T, H, D], positions [B, T] -> (value, bound)."""
    t = x.dtype
    x = x.double()
    R = 2 * frequencies.numel()
    angle = positions.double()[:, :, None, None] * frequencies.to(x.device)
    c, s = factor * angle.cos(), factor * angle.sin() * (-1.0 if transpose else 1.0)
    ia = torch.arange(0, R, 2) if layout == "interleaved" else torch.arange(0, R // 2)
    ib = ia + 1 if layout == "interleaved" else ia + R // 2
    a, b = x[..., ia], x[..., ib]
    y, e = x.clone(), torch.zeros_like(x)
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    # the table is rounded once (its angle is exact to 2^-53 of itself), two products and a sum in fp32
    # (an angle of n turns in 64 bits is off by 2^-52 of itself: positions up to 2^17)
    far = 2.0 ** -52 * angle.abs() * factor
    e[..., ia] = 4 * E * ((a * c).abs() + (b * s).abs()) + far * (a.abs() + b.abs())
    e[..., ib] = 4 * E * ((a * s).abs() + (b * c).abs()) + far * (a.abs() + b.abs())
    bound = e * (1 + UNIT[t])
    bound[..., :R] += rounded(y[..., :R], t)
    return y, bound
