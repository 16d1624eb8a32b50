"""Plain restatements, in 64 bits on the CPU, of layer norm, the gated recurrence and clipping by the global norm, with bounds on how
far a correct kernel may be from them.  They follow the formulas of include/adhip.h and share no code with the kernels or their
callers.

Bounds are sums of what each rounding can do, element by element, with u = 2^-24 for a 32-bit operation and w = 2^-8 for a
rounding to bf16 (0 where the result is f32).
"""
import math

import torch

U = 2.0 ** -24
W = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def rounded(x, err, dtype):
    """The error of a result that was off by err, after its rounding to dtype."""
    return err + (W[dtype] or U) * (x.abs() + err)


# Additions that a number of a row passes on its way into the row's sum: 16 of its lane, 6 between lanes, 16 between wavefronts; two
# more operations on the sum.
ROW = 40 * U


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, centered=True, added=None, out_grad=None, total_grad=None, grad_type=torch.float32):
    """Results and bounds over the last dim.  The total is the kernel's exactly: one addition of 32 bits and one rounding."""
    kind, r, e = x.dtype, {}, {}
    if added is not None:
        x = (x.float() + added.float()).to(kind)
        r["total"], e["total"] = x.double(), torch.zeros_like(x, dtype=torch.float64)
    t, n = x.double(), x.shape[-1]
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.double()
    mean = t.mean(-1, keepdim=True) if centered else torch.zeros_like(t[..., :1])
    e_mean = ROW * t.abs().mean(-1, keepdim=True) * centered
    d = t - mean
    e_d = e_mean + U * d.abs()
    var = (d * d).mean(-1, keepdim=True)
    e_var = (2 * d.abs() * e_d + e_d * e_d).mean(-1, keepdim=True) + ROW * var
    root = (var + eps) ** -0.5
    low = torch.clamp(var + eps - e_var, min=1e-300)
    e_root = (low ** -0.5 - root) + 5 * U * root
    unit = d * root
    e_unit = d.abs() * e_root + (root + e_root) * e_d + U * unit.abs()
    out = unit * w + b
    r["out"], r["stats"] = out, torch.cat((mean, root), -1)
    e["out"] = rounded(out, w.abs() * e_unit + 2 * U * ((unit * w).abs() + b.abs()), kind)
    e["stats"] = torch.cat((e_mean, e_root), -1)
    if out_grad is None:
        return r, e
    dy = out_grad.double()
    u = dy * w
    along = (u * unit).mean(-1, keepdim=True)
    e_along = (u.abs() * e_unit).mean(-1, keepdim=True) + (ROW + 3 * U) * (u * unit).abs().mean(-1, keepdim=True)
    level = u.mean(-1, keepdim=True) * centered
    e_level = (ROW + 2 * U) * u.abs().mean(-1, keepdim=True) * centered
    inner = u - level - unit * along
    e_inner = e_level + unit.abs() * e_along + along.abs() * e_unit + e_unit * e_along + 4 * U * (u.abs() + level.abs() + (unit * along).abs())
    dx = root * inner
    e_dx = root * e_inner + inner.abs() * e_root + e_root * e_inner + U * dx.abs()
    if total_grad is not None:
        dx = dx + total_grad.double()
        e_dx = e_dx + U * dx.abs()
    r["x_grad"], e["x_grad"] = dx, rounded(dx, e_dx, kind)
    rows = dy.numel() // max(1, n)
    flat = lambda a: a.reshape(-1, n)  # noqa: E731
    many = (min(rows, 80 + rows // 256) + 40) * U  # rows of a lane, then lanes, wavefronts and workgroups
    r["weight_grad"], r["bias_grad"] = flat(dy * unit).sum(0), flat(dy).sum(0)
    e["weight_grad"] = rounded(r["weight_grad"], flat(dy.abs() * e_unit).sum(0) + many * flat((dy * unit).abs()).sum(0), grad_type)
    e["bias_grad"] = rounded(r["bias_grad"], many * flat(dy.abs()).sum(0), grad_type)
    return r, e


def recurrence(x, gates, *, factors=False, initial=None, lengths=None, documents=None, out_grad=None, final_grad=None, block=256):
    """Position by position.  Every state is a sum over the positions s before it of b[s] times the factors between: a factor brings its
    own error and two roundings (the product's and the sum's), b its own, and exchanges between threads, wavefronts and ranges
    of positions at most 64 more of the sum; M is the sum of magnitudes and N that sum with each term counted once for every factor."""
    kind, (B, L, C) = x.dtype, x.shape
    count = torch.full((B,), L) if lengths is None else lengths.long().clamp(0, L)
    live = torch.arange(L)[None] < count[:, None]
    behind = ~live
    cut = torch.zeros((B, L), dtype=torch.bool)
    if documents is not None:
        cut[:, 1:] = documents[:, 1:] != documents[:, :-1]
        cut |= documents < 0
        cut &= live
        live = live & (documents >= 0)
    here = live[..., None]
    clean = lambda a: torch.where(here, a.double(), torch.zeros((), dtype=torch.float64))  # noqa: E731
    xs, g = clean(x), clean(gates)
    if factors:
        own, rest, eps_a = g, torch.ones_like(g), 0.0
        b = xs
    else:
        own, rest = torch.sigmoid(g), torch.sigmoid(-g)
        b = rest * xs
        # exp2 and the reciprocal to one unit of their last place, a product and a sum; in bf16 the exponent is rounded once more
        eps_a = 12 * U + (1.5 * U * float(g.abs().max()) if kind == torch.bfloat16 and g.numel() else 0.0)
    a = torch.where(cut[..., None], torch.zeros_like(own), torch.where(behind[..., None], torch.ones_like(own), own))
    h = torch.zeros(B, C, dtype=torch.float64) if initial is None else initial.double()
    M, N = h.abs(), torch.zeros_like(h)
    before, e_before, out, e_out = (torch.zeros(B, L, C, dtype=torch.float64) for _ in range(4))

    def error(M, N):
        return (eps_a + 2 * U) * N + (eps_a + 66 * U) * M

    def onward(a, h, b):  # a factor of zero drops what was there, whatever it is
        return torch.where(a == 0, b, a * h + b)

    for t in range(L):
        before[:, t], e_before[:, t] = h, error(M, N)
        h = onward(a[:, t], h, b[:, t])
        N = onward(a[:, t].abs(), N + M, torch.zeros_like(M))
        M = onward(a[:, t].abs(), M, b[:, t].abs())
        out[:, t], e_out[:, t] = h, error(M, N)
    out = torch.where(here, out, torch.zeros_like(out))
    r = {"out": out, "final": h, "states": before[:, ::block]}
    e = {"out": torch.where(here, rounded(out, e_out, kind), torch.zeros_like(out)), "final": error(M, N), "states": e_before[:, ::block]}
    if out_grad is None:
        return r, e
    d = clean(out_grad)
    mu = torch.zeros(B, C, dtype=torch.float64) if final_grad is None else final_grad.double()
    M, N = mu.abs(), torch.zeros_like(mu)
    for n in ("x_grad", "gates_grad"):
        r[n], e[n] = torch.zeros(B, L, C, dtype=torch.float64), torch.zeros(B, L, C, dtype=torch.float64)
    for t in range(L - 1, -1, -1):
        l = d[:, t] + mu
        M, N = M + d[:, t].abs(), N + M + d[:, t].abs()
        e_l = error(M, N)
        q = torch.where(cut[:, t, None], torch.zeros_like(l), before[:, t])
        e_q = torch.where(cut[:, t, None], torch.zeros_like(l), e_before[:, t])
        if factors:
            dx, e_dx, dg = l, e_l, l * q
            e_dg = e_l * q.abs() + l.abs() * e_q + e_l * e_q + U * dg.abs()
        else:
            p, s = own[:, t], rest[:, t]
            dx, q = l * s, q - xs[:, t]
            e_q = e_q + U * (before[:, t].abs() + xs[:, t].abs())
            e_dx = s * e_l + (eps_a + 2 * U) * (dx.abs() + s * e_l)
            dg = dx * q * p
            e_dg = p * (e_dx * q.abs() + dx.abs() * e_q + e_dx * e_q) + (eps_a + 4 * U) * dg.abs()
        r["x_grad"][:, t], r["gates_grad"][:, t] = dx, dg
        e["x_grad"][:, t], e["gates_grad"][:, t] = rounded(dx, e_dx, kind), rounded(dg, e_dg, kind)
        mu = onward(a[:, t], l, torch.zeros_like(l))
        M, N = (onward(a[:, t].abs(), y, torch.zeros_like(y)) for y in (M, N))
    for n in ("x_grad", "gates_grad"):
        r[n], e[n] = (torch.where(here, y, torch.zeros_like(y)) for y in (r[n], e[n]))
    r["initial_grad"], e["initial_grad"] = mu, error(M, N)
    return r, e


def clip(gradients, limit, grad_scale=1.0):
    """norm, factor and clipped gradients.  The sum is taken in 64 bits (2^-40 covers any order), the results rounded once; the scale is
    a product of two rounded numbers, and its product with a gradient is rounded.  Below 2^-126 f32 numbers are multiples of 2^-149, so a
    rounding is off by up to 2^-150 whatever the number; a norm of 2^128 and more is f32's infinity."""
    squares = sum((float((g.double() ** 2).sum()) for g in gradients), 0.0)
    norm = abs(grad_scale) * math.sqrt(squares)
    factor = 1.0 if norm <= limit else limit / norm
    one = lambda v: torch.tensor([v], dtype=torch.float64)  # noqa: E731
    least = 2.0 ** -150
    r = {"norm": one(norm if norm < 2.0 ** 128 else math.inf), "factor": one(factor), "g": [g.double() * (grad_scale * factor) for g in gradients]}
    e = {"norm": one(norm * (U + 2.0 ** -40)), "factor": one(factor * (U + 2.0 ** -39) + least if factor != 1.0 else 0.0),
         "g": [rounded(y, 4 * U * y.abs() + (abs(grad_scale) + 1) * least * g.double().abs(), g.dtype) + least for y, g in zip(r["g"], gradients)]}
    return r, e
