"""Plain restatements, in 64 bits on the CPU, of the operators on device arrays, with bounds on how far a correct kernel may
be from them.  They follow the formulas of include/adhip.h and share no code with the kernels or their callers.

Bounds are sums of what each rounding can do, element by element, with u = 2^-24 for a 32-bit operation and w = 2^-8 for a
rounding to bf16 (0 where the arrays are f32):
  a score is a sum of D products (D u |q|.|k| at worst) whose exponential carries that error over, tanh included
  (6e-7 of the cap); a sum over L keys or rows of terms t has L u sum|t|; probabilities and score gradients are rounded to
  the arrays' type once (w), so is every result (w), and delta = dout.out takes out as it was rounded (w |dout|.|out|).
"""
import numpy as np
import torch

U = 2.0 ** -24


def attention(q, k, v, *, scale, causal=False, window=0, cap=0.0, slopes=None, lengths=None, prefix=None, query_documents=None,
              key_documents=None, out_grad=None, rounding=0.0):
    """q [B, Lq, H, D], k and v [B, Lk, Hk, D] (tensors of any type) -> results and their bounds, two dicts of float64
    tensors: out, lse and, with out_grad, dq, dk, dv.  Arrays may hold anything where nothing may be used."""
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    w = rounding
    r = {"out": torch.zeros(B, Lq, H, D, dtype=torch.float64), "lse": torch.full((B, Lq, H), -np.inf, dtype=torch.float64)}
    e = {"out": torch.zeros(B, Lq, H, D, dtype=torch.float64), "lse": torch.zeros(B, Lq, H, dtype=torch.float64)}
    if out_grad is not None:
        for d in (r, e):
            d["dq"] = torch.zeros(B, Lq, H, D, dtype=torch.float64)
            d["dk"], d["dv"] = (torch.zeros(B, Lk, Hk, D, dtype=torch.float64) for _ in "kv")
    for b in range(B):
        n = Lk if lengths is None else min(max(int(lengths[b]), 0), Lk)
        sees = torch.zeros(Lq, Lk, dtype=torch.bool)
        for i in range(Lq):
            at = i + n - Lq
            j = torch.arange(Lk)
            band = torch.ones(Lk, dtype=torch.bool)
            if causal:
                band &= j <= at
            if window:
                band &= (at - j).abs() < window
            if prefix is not None:
                band |= j < int(prefix[b])
            band &= j < n
            if query_documents is not None:
                band &= (key_documents[b] == query_documents[b, i]) & (query_documents[b, i] >= 0)
            sees[i] = band
        rows, keys = sees.any(1), sees.any(0)
        for h in range(H):
            c = h // (H // Hk)
            clean = lambda x, used: torch.where(used[:, None], x.double(), torch.zeros(()).double())  # noqa: E731
            Q, K, V = clean(q[b, :, h], rows), clean(k[b, :, c], keys), clean(v[b, :, c], keys)
            raw = scale * Q @ K.T
            err = abs(scale) * (D + 4) * U * (Q.abs() @ K.abs().T)
            z, bend = raw, torch.ones_like(raw)
            if cap:
                y = torch.tanh(raw / cap)
                z, bend = cap * y, 1 - y * y
                err = err + cap * 6e-7
            if slopes is not None:
                far = (torch.arange(Lq)[:, None] + n - Lq - torch.arange(Lk)[None, :]).abs().double()
                z = z - float(slopes[h]) * far
                err = err + 4 * U * float(abs(slopes[h])) * far
            err = err + 8 * U * (z.abs() + 1)
            z = torch.where(sees, z, torch.full_like(z, -np.inf))
            lse = torch.logsumexp(z, 1)
            p = torch.where(sees, torch.exp(z - lse.masked_fill(~rows, 0.0)[:, None]), torch.zeros_like(z))
            sums = (Lk + 16) * U
            top = torch.where(sees, err, torch.zeros_like(err)).amax(1) if Lk else torch.zeros(Lq).double()
            pe = err + top[:, None] + sums  # of a probability, relative to it
            r["lse"][b, :, h] = lse
            e["lse"][b, :, h] = torch.where(rows, top + sums + 8 * U * lse.masked_fill(~rows, 0.0).abs() + 4 * U, torch.zeros_like(top))
            o = p @ V
            r["out"][b, :, h] = o
            e["out"][b, :, h] = (p * (pe + w)) @ V.abs() + sums * (p @ V.abs()) + (w + 4 * U) * o.abs()
            if out_grad is None:
                continue
            G = clean(out_grad[b, :, h], rows)
            dp, dpe = G @ V.T, (D + 4) * U * (G.abs() @ V.abs().T)
            delta = (G * o).sum(1, keepdim=True)
            delta_e = (G.abs() * (e["out"][b, :, h] + (D + 4) * U * o.abs())).sum(1, keepdim=True)
            ds = p * (dp - delta) * bend
            dse = p * (dpe + delta_e) + p * (dp - delta).abs() * (pe + 8 * U + (4e-6 if cap else 0.0)) + w * ds.abs()
            r["dq"][b, :, h] = scale * ds @ K
            e["dq"][b, :, h] = abs(scale) * (dse @ K.abs() + sums * (ds.abs() @ K.abs())) + (w + 4 * U) * r["dq"][b, :, h].abs()
            long = (Lq * (H // Hk) + 16) * U
            r["dk"][b, :, c] += scale * ds.T @ Q
            e["dk"][b, :, c] += abs(scale) * (dse.T @ Q.abs() + long * (ds.abs().T @ Q.abs()))
            r["dv"][b, :, c] += p.T @ G
            e["dv"][b, :, c] += ((p * (pe + w)).T @ G.abs()) + long * (p.T @ G.abs())
    if out_grad is not None:
        for name in ("dk", "dv"):
            e[name] += (w + 4 * U) * r[name].abs()
    return r, e


def rotary(x, cos, sin, positions, interleaved, inverse):
    """x [B, L, H, D] -> float64 result and bound (w of the caller's to add)."""
    x = x.double()
    pairs = cos.shape[1]
    y, size = x.clone(), torch.zeros_like(x)
    for b in range(x.shape[0]):
        for t in range(x.shape[1]):
            at = int(positions[b, t])
            for i in range(pairs):
                one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
                if not 0 <= at < cos.shape[0]:
                    y[b, t, :, one] = y[b, t, :, two] = float("nan")
                    continue
                c, s = float(cos[at, i]), float(sin[at, i]) * (-1.0 if inverse else 1.0)
                y[b, t, :, one] = x[b, t, :, one] * c - x[b, t, :, two] * s
                y[b, t, :, two] = x[b, t, :, one] * s + x[b, t, :, two] * c
                size[b, t, :, one] = size[b, t, :, two] = x[b, t, :, one].abs() + x[b, t, :, two].abs()
    return y, 3 * U * size


def adamw(p, g, m, v, *, step, rate, beta1, beta2, eps, decay, grad_scale):
    """float64 arrays -> new (p, m, v) and bounds on them in 32-bit arithmetic."""
    g = grad_scale * g
    m1, v1 = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    under = np.sqrt(v1 / (1 - beta2 ** step)) + eps
    update = rate / (1 - beta1 ** step) * m1 / under
    p1 = p * (1 - rate * decay) - update
    me, ve = 5 * U * (np.abs(beta1 * m) + np.abs((1 - beta1) * g)), 7 * U * v1
    pe = 4 * U * (np.abs(p) + np.abs(update)) + np.abs(update) * 10 * U + rate / (1 - beta1 ** step) * me / under
    return (p1, m1, v1), (pe, me, ve)
